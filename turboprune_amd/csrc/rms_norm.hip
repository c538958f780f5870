// Root-mean-square norm with the residual's addition, and an 8-bit output.
//
//   h = round(x + r)                      (h = x without a residual)
//   y = h * rsqrt(mean(h^2) + eps) * w
//   kept = y in the 8-bit format of act8.h, from the unrounded y
//
// The norm is that of the h which is handed on, so the pair (h, y) is what
// an addition followed by a norm would give, and the backward pass, which
// reads h, differentiates exactly what was computed:
//
//   dh += rstd (w dy - hhat mean(w dy hhat)),  hhat = h rstd
//   dw  = sum over rows of dy hhat
//
// Sums are in fp32. Every row is read once and held in registers: TPR
// threads to a row, each with NCH chunks of 8 neighbouring values, TPR and
// NCH growing with the row's length so that short rows do not idle a wave
// and long ones stay in registers (up to 16384 values; longer rows take the
// two-pass kernels at the end).
//
// Bound by memory: 50432 x 768, bf16 x on a 32-bit stream with codes, forward
// 97 us (5.2 TB/s), backward 126 us (4.9 TB/s); the vectors' sums 5 us.

#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>

#include "act8.h"

namespace turboprune {

using namespace act8;

std::pair<at::Tensor, at::Tensor> act8_empty(at::IntArrayRef,
                                             const at::TensorOptions&);

namespace {

// sum over the TPR threads of a row, in every one of them; TPR = 256 joins
// its four waves through LDS, and `lds` is free again at the next call only
// after a barrier, which the alternating half provides
template <int TPR, typename V>
TP_DEVICE V row_sum(V v, V* lds, int& turn) {
#pragma unroll
  for (int off = (TPR < kWave ? TPR : kWave) / 2; off > 0; off >>= 1)
    v += __shfl_xor(v, off, kWave);
  if constexpr (TPR > kWave) {
    V* l = lds + (turn & 1) * 4;
    ++turn;
    if ((threadIdx.x & (kWave - 1)) == 0) l[threadIdx.x / kWave] = v;
    __syncthreads();
    v = (l[0] + l[1]) + (l[2] + l[3]);
  }
  return v;
}

// x^-1/2 in 64 bits, from the estimate by one Newton step
TP_DEVICE double inv_root(double x) {
  float f = (float)x;
  double r = rsqrtf(f);
  return f > 0.f && f < __builtin_inff() ? r + .5 * r * (1. - x * r * r) : r;
}

// v r w for codes (r is hi + lo): the products with what each leaves, rounded
// towards zero with the last bit set where anything is cut off, so that
// rounding to fewer bits gives what rounding v r w would. Where codes are
// written a row's sum is joined in 64 bits, too: rounded at every step in 32,
// one code in two million would be the neighbour of the formula's, a sixteenth
// of its value off, and so it is one in ten million (2 us of 97 at 50432 x
// 768).
TP_DEVICE float scaled(float v, float hi, float lo, float w) {
#pragma clang fp contract(off)
  float t = v * hi, e = fmaf(v, lo, fmaf(v, hi, -t));
  float y = t * w, d = fmaf(e, w, fmaf(t, w, -y));
  float z = y + d, left = d - (z - y);
  uint32_t b = __float_as_uint(z), l = __float_as_uint(left);
  // one step down where what is left points to zero
  b = left != 0.f ? (b - ((b ^ l) >> 31)) | 1 : b;
  return fabsf(y) < __builtin_inff() ? __uint_as_float(b) : y;
}

struct NormFwd {
  const void *x, *r;
  void *h, *y;
  const float* w;
  float* rstd;
  uint8_t *codes, *scales;
  int64_t rows, ldx, ldr;
  int C;
  double eps, inv;   // inv: 1 / C
};

// TX: x; TH: residual and h (x's own type without a residual); TY: y.
template <typename TX, typename TH, typename TY, int TPR, int NCH>
__global__ __launch_bounds__(kBlock) void rms_fwd_kernel(NormFwd p) {
  __shared__ float lds[8];
  __shared__ double lds64[8];
  int turn = 0;
  constexpr int RPB = kBlock / TPR;
  int t = threadIdx.x % TPR;
  int sblk = (p.C + kBlk - 1) / kBlk;
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
       row - threadIdx.x / TPR < p.rows; row += (int64_t)gridDim.x * RPB) {
    bool live = row < p.rows;   // rows of one block end together for TPR=256
    const TX* x = (const TX*)p.x + row * p.ldx;
    const TH* r = (const TH*)p.r + row * p.ldr;
    TH* h = (TH*)p.h + row * p.C;
    float v[NCH][8];
    float ss = 0.f;
    double ss64 = 0.;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      int c = (t + j * TPR) * 8, n = live ? p.C - c : 0;
      load8n(x + c, n, v[j]);
      if (p.r) {
        float rv[8];
        load8n(r + c, n, rv);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = rounded<TH>(v[j][i] + rv[i]);
        store8n(h + c, n, v[j]);
      }
      float s8 = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s8 = fmaf(v[j][i], v[j][i], s8);
      ss += s8;
      if (p.codes) ss64 += s8;
    }
    float rstd, low = 0.f;
    if (p.codes) {
      double s = row_sum<TPR>(ss64, lds64, turn);
      s = inv_root(fma(s, p.inv, p.eps));
      rstd = (float)s;
      low = (float)(s - rstd);
    } else {
      rstd = rsqrtf(row_sum<TPR>(ss, lds, turn) / p.C + (float)p.eps);
    }
    if (live && t == 0 && p.rstd) p.rstd[row] = rstd;
    TY* y = (TY*)p.y + row * p.C;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      int c = (t + j * TPR) * 8, n = live ? p.C - c : 0;
      float w[8];
      load8n(p.w + c, n, w);
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        o[i] = p.codes ? scaled(v[j][i], rstd, low, w[i])
                       : v[j][i] * rstd * w[i];
      store8n(y + c, n, o);
      if (p.codes) {
        int e;
        uint2 q = encode8(o, e, QuadMax());
        if (n > 0) {
          store_codes(p.codes + row * p.C + c, n, q);
          if ((t & 3) == 0)
            p.scales[row * sblk + c / kBlk] = (uint8_t)(e + 127);
        }
      }
    }
  }
}

struct NormBwd {
  const void *dy, *dh, *h;
  void *dx, *dr;
  const float *w, *rstd;
  float* part;   // (blocks, C) partial sums of dw
  int64_t rows, ldh;
  int C;
};

// Blocks of the backward kernel that a CU holds at once, by the registers of
// a row: the grid is that many for each of the 256 CUs, so that no block of it
// waits for another to end (50432 rows of 768, 16-bit x, 32-bit stream: 126 us,
// 4.9 TB/s, with 768 blocks; 153 with 1024, of which a quarter runs alone).
constexpr int bwd_blocks(int nch) {
  return nch <= 1 ? 5 : nch == 2 ? 3 : nch == 4 ? 2 : 1;
}

// dx is written when its type is not h's (or there is no residual, when
// TX == TH and dr is null); the two gradients of one type are one tensor.
template <typename TX, typename TH, typename TY, int TPR, int NCH>
__global__ __launch_bounds__(kBlock, bwd_blocks(NCH)) void rms_bwd_kernel(
    NormBwd p) {
  __shared__ float lds[8];
  int turn = 0;
  constexpr int RPB = kBlock / TPR;
  int t = threadIdx.x % TPR;
  float dw[NCH][8];
  float w[NCH][8];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    int c = (t + j * TPR) * 8;
    load8n(p.w + c, p.C - c, w[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[j][i] = 0.f;
  }
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
       row - threadIdx.x / TPR < p.rows; row += (int64_t)gridDim.x * RPB) {
    bool live = row < p.rows;
    const TH* hp = (const TH*)p.h + row * p.ldh;
    const TY* gp = (const TY*)p.dy + row * p.C;
    const TH* ap = (const TH*)p.dh + row * p.C;
    float rstd = live ? p.rstd[row] : 0.f;
    float h[NCH][8], g[NCH][8], a[NCH][8];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      int c = (t + j * TPR) * 8, n = live ? p.C - c : 0;
      load8n(hp + c, n, h[j]);
      load8n(gp + c, n, g[j]);
      if (p.dh) load8n(ap + c, n, a[j]);
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[j][i] *= rstd;                             // hhat
        dw[j][i] = fmaf(g[j][i], h[j][i], dw[j][i]);
        g[j][i] *= w[j][i];
        s = fmaf(g[j][i], h[j][i], s);
      }
    s = row_sum<TPR>(s, lds, turn) / p.C;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      int c = (t + j * TPR) * 8, n = live ? p.C - c : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float d = rstd * (g[j][i] - h[j][i] * s);
        g[j][i] = p.dh ? d + a[j][i] : d;
      }
      if (p.dr) store8n((TH*)p.dr + row * p.C + c, n, g[j]);
      if (p.dx) store8n((TX*)p.dx + row * p.C + c, n, g[j]);
    }
  }
  // the block's rows, added in a fixed order
  if constexpr (RPB > 1) {
    __shared__ float sum[RPB][TPR * 8 + 1];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[threadIdx.x / TPR][t * 8 + i] = dw[j][i];
      __syncthreads();
      for (int c = threadIdx.x; c < TPR * 8; c += kBlock) {
        int col = j * TPR * 8 + c;
        if (col >= p.C) continue;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < RPB; ++k) v += sum[k][c];
        p.part[(int64_t)blockIdx.x * p.C + col] = v;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      int c = (t + j * TPR) * 8;
      store8n(p.part + (int64_t)blockIdx.x * p.C + c, p.C - c, dw[j]);
    }
  }
}

// out[c] = sum over n rows of part: 64 columns a block, 16 row lanes, joined
// through LDS in a fixed order
__global__ __launch_bounds__(1024) void rms_dw_kernel(
    const float* __restrict__ part, float* __restrict__ out, int n, int C) {
  __shared__ float sum[16][64];
  int c = blockIdx.x * 64 + (threadIdx.x & 63), k = threadIdx.x >> 6;
  float v = 0.f;
  if (c < C) {
    // eight loads in flight; one at a time is all latency
    int r = k;
    for (; r + 7 * 16 < n; r += 8 * 16) {
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = part[(int64_t)(r + i * 16) * C + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) v += t[i];
    }
    for (; r < n; r += 16) v += part[(int64_t)r * C + c];
  }
  sum[k][threadIdx.x & 63] = v;
  __syncthreads();
  if (k == 0 && c < C) {
#pragma unroll
    for (int i = 1; i < 16; ++i) v += sum[i][threadIdx.x];
    out[c] = v;
  }
}

// ---- rows longer than the registers hold: a block to a row, two passes ----
template <typename TX, typename TH, typename TY>
__global__ __launch_bounds__(kBlock) void rms_fwd_long_kernel(NormFwd p) {
  __shared__ float lds[8];
  __shared__ double lds64[8];
  int turn = 0;
  int sblk = (p.C + kBlk - 1) / kBlk;
  int span = (p.C + kBlk - 1) / kBlk * kBlk;   // whole quads
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const TX* x = (const TX*)p.x + row * p.ldx;
    const TH* r = (const TH*)p.r + row * p.ldr;
    TH* h = (TH*)p.h + row * p.C;
    float ss = 0.f;
    double ss64 = 0.;
    for (int c = threadIdx.x * 8; c < p.C; c += kBlock * 8) {
      float v[8], rv[8];
      load8n(x + c, p.C - c, v);
      if (p.r) {
        load8n(r + c, p.C - c, rv);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = rounded<TH>(v[i] + rv[i]);
        store8n(h + c, p.C - c, v);
      }
      float s8 = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s8 = fmaf(v[i], v[i], s8);
      ss += s8;
      if (p.codes) ss64 += s8;
    }
    float rstd, low = 0.f;
    if (p.codes) {
      double s = row_sum<kBlock>(ss64, lds64, turn);
      s = inv_root(fma(s, p.inv, p.eps));
      rstd = (float)s;
      low = (float)(s - rstd);
    } else {
      rstd = rsqrtf(row_sum<kBlock>(ss, lds, turn) / p.C + (float)p.eps);
    }
    if (threadIdx.x == 0 && p.rstd) p.rstd[row] = rstd;
    for (int c = threadIdx.x * 8; c < span; c += kBlock * 8) {
      float v[8], rv[8], w[8];
      int n = p.C - c;
      load8n(x + c, n, v);
      if (p.r) {
        load8n(r + c, n, rv);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = rounded<TH>(v[i] + rv[i]);
      }
      load8n(p.w + c, n, w);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = p.codes ? scaled(v[i], rstd, low, w[i]) : v[i] * rstd * w[i];
      store8n((TY*)p.y + row * p.C + c, n, v);
      if (p.codes) {
        int e;
        uint2 q = encode8(v, e, QuadMax());
        if (n > 0) {
          store_codes(p.codes + row * p.C + c, n, q);
          if ((threadIdx.x & 3) == 0)
            p.scales[row * sblk + c / kBlk] = (uint8_t)(e + 127);
        }
      }
    }
  }
}

template <typename TX, typename TH, typename TY>
__global__ __launch_bounds__(kBlock) void rms_bwd_long_kernel(NormBwd p) {
  __shared__ float lds[8];
  int turn = 0;
  float* part = p.part + (int64_t)blockIdx.x * p.C;
  bool first = true;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const TH* hp = (const TH*)p.h + row * p.ldh;
    const TY* gp = (const TY*)p.dy + row * p.C;
    const TH* ap = (const TH*)p.dh + row * p.C;
    float rstd = p.rstd[row], s = 0.f;
    for (int c = threadIdx.x * 8; c < p.C; c += kBlock * 8) {
      float h[8], g[8], w[8];
      load8n(hp + c, p.C - c, h);
      load8n(gp + c, p.C - c, g);
      load8n(p.w + c, p.C - c, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(g[i] * w[i], h[i] * rstd, s);
    }
    s = row_sum<kBlock>(s, lds, turn) / p.C;
    for (int c = threadIdx.x * 8; c < p.C; c += kBlock * 8) {
      float h[8], g[8], w[8], a[8], d[8];
      int n = p.C - c;
      load8n(hp + c, n, h);
      load8n(gp + c, n, g);
      load8n(p.w + c, n, w);
      if (p.dh) load8n(ap + c, n, a);
      // a thread owns its columns of the block's partial row
      if (first)
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = 0.f;
      else
        load8n(part + c, n, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float hat = h[i] * rstd;
        d[i] = fmaf(g[i], hat, d[i]);
        float v = rstd * (g[i] * w[i] - hat * s);
        g[i] = p.dh ? v + a[i] : v;
      }
      store8n(part + c, n, d);
      if (p.dr) store8n((TH*)p.dr + row * p.C + c, n, g);
      if (p.dx) store8n((TX*)p.dx + row * p.C + c, n, g);
    }
    first = false;
  }
}

// Threads and chunks of a row of C values.
template <typename F>
void by_length(int64_t C, F&& f) {
  using std::integral_constant;
#define TP_LEN(TPR, NCH) \
  f(integral_constant<int, TPR>(), integral_constant<int, NCH>())
  if (C <= 128) TP_LEN(16, 1);
  else if (C <= 256) TP_LEN(32, 1);
  else if (C <= 512) TP_LEN(64, 1);
  else if (C <= 1024) TP_LEN(64, 2);
  else if (C <= 2048) TP_LEN(64, 4);
  else if (C <= 4096) TP_LEN(256, 2);
  else if (C <= 8192) TP_LEN(256, 4);
  else if (C <= 16384) TP_LEN(256, 8);
  else TP_LEN(256, 0);   // 0: the two-pass kernels
#undef TP_LEN
}

template <typename T> struct Is { using type = T; };

// the types of (x, h, y) that there are kernels for
template <typename F>
void by_types(at::ScalarType x, at::ScalarType h, at::ScalarType y, F&& f) {
  using B = __hip_bfloat16;
  using H = _Float16;
  auto is = [&](at::ScalarType a, at::ScalarType b, at::ScalarType c) {
    return x == a && h == b && y == c;
  };
  if (is(at::kBFloat16, at::kBFloat16, at::kBFloat16))
    f(Is<B>(), Is<B>(), Is<B>());
  else if (is(at::kBFloat16, at::kFloat, at::kBFloat16))
    f(Is<B>(), Is<float>(), Is<B>());
  else if (is(at::kHalf, at::kHalf, at::kHalf))
    f(Is<H>(), Is<H>(), Is<H>());
  else if (is(at::kHalf, at::kFloat, at::kHalf))
    f(Is<H>(), Is<float>(), Is<H>());
  else if (is(at::kFloat, at::kFloat, at::kFloat))
    f(Is<float>(), Is<float>(), Is<float>());
  else if (is(at::kFloat, at::kFloat, at::kBFloat16))
    f(Is<float>(), Is<float>(), Is<B>());
  else if (is(at::kFloat, at::kFloat, at::kHalf))
    f(Is<float>(), Is<float>(), Is<H>());
  else
    TORCH_CHECK(false, "rms_norm: no kernel for x ", x, ", residual ", h,
                ", output ", y,
                " (x in float32, bfloat16 or float16; the residual in x's "
                "type or float32; the output in x's type, or in 16 bits "
                "where x is float32)");
}

// rows of C neighbouring values, with any distance between them
at::Tensor as_rows(const at::Tensor& t, int64_t C) {
  auto r = t.dim() == 2 ? t : t.reshape({-1, C});
  return r.size(1) <= 1 || r.stride(1) == 1 ? r : r.contiguous();
}

}  // namespace

// (y, h, rstd, codes, scales): h undefined without a residual, rstd without
// want_rstd, codes and scales without keep.
std::tuple<at::Tensor, c10::optional<at::Tensor>, c10::optional<at::Tensor>,
           c10::optional<at::Tensor>, c10::optional<at::Tensor>>
rms_fwd(const at::Tensor& x, const c10::optional<at::Tensor>& residual,
        const at::Tensor& weight, double eps, at::ScalarType out_dtype,
        bool want_rstd, bool keep) {
  TORCH_CHECK(x.is_cuda() && x.dim() >= 1 && x.size(-1) >= 1,
              "rms_fwd: x on a GPU, with rows of at least one value");
  int64_t C = x.size(-1);
  TORCH_CHECK(C <= (int64_t(1) << 30), "rms_fwd: rows of at most 2^30 values");
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == C &&
                  weight.device() == x.device(),
              "rms_fwd: weight of x's last dimension, on x's device");
  bool has_r = residual.has_value();
  if (has_r)
    TORCH_CHECK(residual->sizes() == x.sizes() &&
                    residual->device() == x.device(),
                "rms_fwd: residual of x's shape, on x's device");
  c10::DeviceGuard guard(x.device());
  auto th = has_r ? residual->scalar_type() : x.scalar_type();
  auto opt = x.options();
  auto y = at::empty(x.sizes(), opt.dtype(out_dtype));
  c10::optional<at::Tensor> h, rstd, codes, scales;
  if (has_r) h = at::empty(x.sizes(), opt.dtype(th));
  int64_t rows = x.numel() / C;
  if (want_rstd) rstd = at::empty({rows}, opt.dtype(at::kFloat));
  if (keep) std::tie(codes, scales) = act8_empty(x.sizes(), opt);
  auto xr = as_rows(x, C);
  auto w = weight.to(at::kFloat).contiguous();
  NormFwd p{};
  at::Tensor rr;
  p.x = xr.data_ptr();
  p.ldx = xr.stride(0);
  if (has_r) {
    rr = as_rows(*residual, C);
    p.r = rr.data_ptr();
    p.ldr = rr.stride(0);
    p.h = h->data_ptr();
  }
  p.y = y.data_ptr();
  p.w = w.data_ptr<float>();
  if (want_rstd) p.rstd = rstd->data_ptr<float>();
  if (keep) {
    p.codes = (uint8_t*)codes->data_ptr();
    p.scales = (uint8_t*)scales->data_ptr();
  }
  p.rows = rows;
  p.C = (int)C;
  p.eps = eps;
  p.inv = 1. / (double)C;
  auto stream = at::hip::getCurrentHIPStream();
  by_types(x.scalar_type(), th, out_dtype, [&](auto a, auto b, auto c) {
    using TX = typename decltype(a)::type;
    using TH = typename decltype(b)::type;
    using TY = typename decltype(c)::type;
    if (rows == 0) return;
    by_length(C, [&](auto tpr, auto nch) {
      constexpr int TPR = decltype(tpr)::value, NCH = decltype(nch)::value;
      int64_t per = kBlock / TPR;
      int grid = (int)std::min<int64_t>((rows + per - 1) / per, 1 << 20);
      if constexpr (NCH == 0)
        rms_fwd_long_kernel<TX, TH, TY><<<grid, kBlock, 0, stream>>>(p);
      else
        rms_fwd_kernel<TX, TH, TY, TPR, NCH><<<grid, kBlock, 0, stream>>>(p);
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
  });
  return {y, h, rstd, codes, scales};
}

// (dx, dres, dweight): dres is dx itself where the two types are one, and
// undefined without a residual. h is what the forward pass normalised; dh
// may be missing. dy has y's shape and type, dh that of h.
std::tuple<at::Tensor, c10::optional<at::Tensor>, at::Tensor> rms_bwd(
    const at::Tensor& dy_in, const c10::optional<at::Tensor>& dh_in,
    const at::Tensor& h, const at::Tensor& weight, const at::Tensor& rstd,
    at::ScalarType x_dtype, bool has_residual) {
  int64_t C = h.size(-1), rows = h.numel() / C;
  TORCH_CHECK(h.is_cuda() && dy_in.device() == h.device() &&
                  dy_in.sizes() == h.sizes() && rstd.numel() == rows &&
                  weight.numel() == C,
              "rms_bwd: shapes or devices differ from the forward pass");
  c10::DeviceGuard guard(h.device());
  auto dy = dy_in.contiguous();
  auto hr = as_rows(h, C);
  auto w = weight.to(at::kFloat).contiguous();
  at::Tensor dhc, dx, dr;
  auto th = h.scalar_type();
  bool two = has_residual && th != x_dtype;
  NormBwd p{};
  if (dh_in.has_value()) {
    TORCH_CHECK(dh_in->sizes() == h.sizes() && dh_in->scalar_type() == th &&
                    dh_in->device() == h.device(),
                "rms_bwd: dh differs from h in shape, type or device");
    dhc = dh_in->contiguous();
    p.dh = dhc.data_ptr();
  }
  dx = at::empty(h.sizes(), h.options().dtype(x_dtype));
  if (two) {
    dr = at::empty(h.sizes(), h.options());
    p.dr = dr.data_ptr();
  }
  auto dw = at::empty({C}, h.options().dtype(at::kFloat));
  p.dy = dy.data_ptr();
  p.h = hr.data_ptr();
  p.ldh = hr.stride(0);
  p.dx = dx.data_ptr();
  p.w = w.data_ptr<float>();
  p.rstd = rstd.data_ptr<float>();
  p.rows = rows;
  p.C = (int)C;
  auto stream = at::hip::getCurrentHIPStream();
  by_types(x_dtype, th, dy.scalar_type(), [&](auto a, auto b, auto c) {
    using TX = typename decltype(a)::type;
    using TH = typename decltype(b)::type;
    using TY = typename decltype(c)::type;
    if (rows == 0) {
      dw.zero_();
      return;
    }
    by_length(C, [&](auto tpr, auto nch) {
      constexpr int TPR = decltype(tpr)::value, NCH = decltype(nch)::value;
      int64_t per = kBlock / TPR;
      // partial rows of at most 256 MB
      int64_t most = std::max<int64_t>(1, std::min<int64_t>(
          256 * (NCH ? bwd_blocks(NCH) : 4), (int64_t(1) << 26) / C));
      int grid = (int)std::min<int64_t>((rows + per - 1) / per, most);
      auto part = at::empty({grid, C}, dw.options());
      p.part = part.template data_ptr<float>();
      if constexpr (NCH == 0)
        rms_bwd_long_kernel<TX, TH, TY><<<grid, kBlock, 0, stream>>>(p);
      else
        rms_bwd_kernel<TX, TH, TY, TPR, NCH><<<grid, kBlock, 0, stream>>>(p);
      C10_HIP_KERNEL_LAUNCH_CHECK();
      rms_dw_kernel<<<(int)((C + 63) / 64), 1024, 0, stream>>>(
          p.part, dw.data_ptr<float>(), grid, (int)C);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    });
  });
  c10::optional<at::Tensor> dres;
  if (has_residual) dres = two ? dr : dx;
  return {dx, dres, dw};
}

}  // namespace turboprune
