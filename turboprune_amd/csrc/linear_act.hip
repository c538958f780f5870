// Masked linear layer with bias, GELU and residual in the product's
// epilogue, and its gradients, from inputs kept in 8 or 16 bits.
//
//   z = x w^T + b,  y = act(z) + r            x (M,K), w (N,K) masked
//   dz = dy act'(z kept),  dx = dz w,  dw = (dz^T x kept) . mask,
//   db = column sums of dz,  dr = dy
//
// All three products run on one tiled matrix kernel (mm_kernel below), a few
// rows on one that stages nothing (rows_kernel).
//
// Sizes are rows x K -> N throughout, as of the product that a launch computes.
// Times are of launches after a pause or a few of them; ten large products in a
// row lower the chip's clock and take up to a fifth longer (25216 x 4096 ->
// 1024 208 us, then 250).

#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>

#include <type_traits>

#include "act8.h"

namespace turboprune {

using namespace act8;

std::pair<at::Tensor, at::Tensor> act8_empty(at::IntArrayRef,
                                             const at::TensorOptions&);
namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

#define TP_LDS __attribute__((address_space(3)))

template <typename T>
TP_DEVICE f32x4 mma(s16x8 a, s16x8 b, f32x4 c) {
  if constexpr (__is_same(T, _Float16))
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(
        __builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
        0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
        0);
}

// What a product writes.
struct Epi {
  const void* bias;      // N values, or null
  const void* res;       // (M,N) residual, or null
  void* out;             // (M,N)
  void* z;               // (M,N) kept pre-activation: 16-bit values or codes
  uint8_t* zscale;       // its scales; null: z holds 16-bit values
  const float* mask;     // weight gradient: 0/1 per value, or null
  int bias_f32, res_f32, out_f32;
};

// C[q][p] = sum_k Q P. An operand is a matrix of 16-bit values, with
// kRowK: row q (or p) holding the values along k, or
// kColK: row k holding the values along q (or p);
// kCodes is kColK with 8-bit codes and their scales in place of values.
enum { kRowK = 0, kColK = 1, kCodes = 2 };

struct Mm {
  const char *q, *p;     // 16-byte aligned, row distances multiples of 16 B
  int64_t ldq, ldp;      // row distance in bytes
  int nq, np;            // rows (kRowK) or columns (kColK) that can be read
  const uint8_t* pscale; // kCodes: a scale for every 32 codes of a row
  uint8_t *qcodes, *qscale;   // kRowK: Q in 8 bits, to be written, or null
  int M, N, K;           // rows and columns of C, length of the sum
  int tiles_n, tiles;    // tile grid
  int ksplit, kper;      // k-tiles of one slab; slab s writes out + s M N
  Epi e;
};

// LDS image of a kRowK tile: rows of BK values (64 or 128 B); the 16-byte
// chunk c of row r sits at c ^ (r / (256 B / row)), so that the 16 rows of a
// fragment read spread over all 64 banks. Of a kColK tile: BK rows (along k)
// of W values; the 32-byte block b of row r sits at b ^ f(r) with
// f(r) = (r & 3) | (r >> 3 & 1) << 2: the rows that one transposing read
// touches together then differ in bank.
template <int W, int BK, bool TR>
struct Tile {
  static constexpr int kBytes = W * BK * 2;
  static constexpr int kLoads = kBytes / 1024;   // wave-wide 16 B loads
  static constexpr int kChunks = BK / 8;         // of a kRowK row
  TP_DEVICE static int swap(int row) {
    return BK == 64 ? row / 2 % 8 : (row / 8 % 2) * 3;
  }
};

// f(r) of a kColK tile; rows of 64 values, two to 256 B, need only two bits
template <int W>
TP_DEVICE int col_swap(int row) {
  return W == 64 ? (row >> 1 & 1) | (row >> 3 & 1) << 1
                 : (row & 3) | (row >> 3 & 1) << 2;
}

typedef __amdgpu_buffer_rsrc_t rsrc_t;
TP_DEVICE rsrc_t rsrc(const void* p, int64_t bytes) {
  int n = (int)(bytes < 0x7ffffff0 ? bytes : 0x7ffffff0);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, n,
                                           0x00020000);
}
constexpr int kOut = 0x7ffffff8;   // an offset that no buffer reaches

// Wave `w` of NW brings its share of a tile into LDS with asynchronous
// 16-byte loads; what lies outside the matrix arrives as zeros.
template <int W, int BK, bool TR, int NW>
TP_DEVICE void stage(TP_LDS char* dst, const char* base, int64_t ld,
                     int first, int count, int kt, int K, int wave,
                     int lane) {
  typedef Tile<W, BK, TR> L;
  constexpr int PER = L::kLoads / NW;
  static_assert(PER * NW == L::kLoads, "loads divide evenly");
  if constexpr (!TR) {
    int rows = min(W, count - first);
    rsrc_t r = rsrc(base + (int64_t)first * ld,
                    (int64_t)(rows - 1) * ld + (K + 7) / 8 * 16);
    constexpr int RPL = 64 / L::kChunks;   // rows of one load
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int row = (wave * PER + i) * RPL + lane / L::kChunks;
      int c = lane % L::kChunks ^ L::swap(row);
      int off = row * (int)ld + c * 16;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          r, (TP_LDS void*)(dst + (wave * PER + i) * 1024), 16,
          kt * BK + c * 8 < K ? off : kOut, kt * BK * 2, 0, 0);
    }
  } else {
    int k0 = kt * BK, rows = min(BK, K - k0);
    constexpr int LPR = W * 2 / 16;       // lanes to a row
    rsrc_t r = rsrc(base + (int64_t)k0 * ld + (int64_t)first * 2,
                    (int64_t)(rows - 1) * ld + (int64_t)(count - first) * 2);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int chunk = (wave * PER + i) * 64 + lane;
      int row = chunk / LPR, c = chunk % LPR;
      int f = col_swap<W>(row);
      int col = ((c >> 1) ^ f) * 32 + (c & 1) * 16;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          r, (TP_LDS void*)(dst + (wave * PER + i) * 1024), 16,
          row * (int)ld + col, 0, 0, 0);
    }
  }
}

// Fragment of 16 rows (columns) from `at` and 32 values of k from ks * 32:
// lane l holds number l % 16, k from (l / 16) * 8.
template <int W, int BK, bool TR>
TP_DEVICE s16x8 frag(TP_LDS const char* t, int at, int ks, int lane) {
  int g = lane >> 4, i = lane & 15;
  if constexpr (!TR) {
    int row = at + i;
    int c = (ks * 4 + g) ^ Tile<W, BK, TR>::swap(row);
    return *reinterpret_cast<TP_LDS const s16x8*>(t + row * (BK * 2) + c * 16);
  } else {
    int row = ks * 32 + g * 8 + (i >> 2);   // and 4 rows on: the same swap
    int f = col_swap<W>(row);
    TP_LDS const char* a =
        t + row * (W * 2) + (((at >> 4) ^ f) * 32) + (i & 3) * 8;
    s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TP_LDS s16x4*)a);
    s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (TP_LDS s16x4*)(a + 4 * W * 2));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// kCodes tiles go through registers: 16 codes of one row, with their scale,
// become 16 values in two LDS stores. A code times a power of two is exact in
// bf16; in fp16 it is brought into range first.
template <typename T, int W, int BK, int THREADS>
struct CodeTile {
  static constexpr int kAll = W * BK / 16;
  static constexpr int kPer = (kAll + THREADS - 1) / THREADS;
  u32x4 code[kPer];
  uint32_t scale[kPer];

  TP_DEVICE void load(const Mm& a, int first, int kt) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      int at = i * THREADS + threadIdx.x;
      int row = at / (W / 16), col = first + at % (W / 16) * 16;
      int64_t k = (int64_t)kt * BK + row;
      int n = k < a.K && at < kAll ? a.np - col : 0;
      const uint8_t* p = (const uint8_t*)a.p + k * a.ldp + col;
      uint2 lo = load_codes(p, n), hi = load_codes(p + 8, n - 8);
      code[i] = u32x4{lo.x, lo.y, hi.x, hi.y};
      scale[i] = n > 0 ? a.pscale[k * ((a.np + 31) / 32) + col / 32] : 0;
    }
  }

  TP_DEVICE void store(TP_LDS char* dst) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      int at = i * THREADS + threadIdx.x;
      if (kAll % THREADS && at >= kAll) break;
      int row = at / (W / 16), blk = at % (W / 16);
      int f = col_swap<W>(row);
      float sc = __uint_as_float(scale[i] << 23);
      u32x4 v[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (__is_same(T, _Float16)) {
          f32x2v x = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[i][j], false);
          f32x2v y = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[i][j], true);
          v[j / 2][j % 2 * 2] =
              pack2<T>(held_in<T>(x[0] * sc), held_in<T>(x[1] * sc));
          v[j / 2][j % 2 * 2 + 1] =
              pack2<T>(held_in<T>(y[0] * sc), held_in<T>(y[1] * sc));
        } else {
          v[j / 2][j % 2 * 2] = __builtin_bit_cast(
              uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(
                            code[i][j], sc, false));
          v[j / 2][j % 2 * 2 + 1] = __builtin_bit_cast(
              uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(
                            code[i][j], sc, true));
        }
      }
      TP_LDS u32x4* d = (TP_LDS u32x4*)(dst + row * (W * 2) + (blk ^ f) * 32);
      d[0] = v[0];
      d[1] = v[1];
    }
  }
};

// Q's values of one k-tile, from LDS, in 8 bits. The column tiles of a row of
// tiles take the k-tiles in turn, so that each of them does its share and the
// input is read once for product and codes: 50432 x 1536 -> 384 with a 32-bit
// residual 144 us, with a pass of its own 42 + 105 and a launch more (332 and
// 354 us for the layer forward and backward when both were measured).
template <typename T, int BQ, int BK, int THREADS>
TP_DEVICE void keep_tile(TP_LDS const char* t, const Mm& a, int m0, int kt) {
  constexpr int C = BK / 8;
  static_assert(BQ * C % THREADS == 0, "whole rounds");
  // all rounds at once where registers allow, one by one beside 16 waves' sums
  constexpr int R = BQ * C / THREADS, U = THREADS == 1024 ? 1 : R;
#pragma unroll 1
  for (int i0 = 0; i0 < R; i0 += U) {
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      int at = (i0 + u) * THREADS + threadIdx.x, r = at / C, c = at % C;
      unpack8<T>(*reinterpret_cast<TP_LDS const u32x4*>(
                     t + r * (BK * 2) + (c ^ Tile<BQ, BK, false>::swap(r)) * 16),
                 v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      int at = (i0 + u) * THREADS + threadIdx.x, r = at / C, c = at % C;
      int e, col = kt * BK + c * 8;
      uint2 q = encode8(v[u], e, QuadMax());
      int64_t row = m0 + r;
      int n = row < a.M ? a.K - col : 0;
      if (n <= 0) continue;
      store_codes(a.qcodes + row * a.K + col, n, q);
      if ((c & 3) == 0)
        a.qscale[row * ((a.K + 31) / 32) + col / 32] = (uint8_t)(e + 127);
    }
  }
}

template <int N>
TP_DEVICE void wait_and_meet() {
  // this wave's loads but the newest N have landed and its reads are done;
  // then every wave's
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N)
               : "memory");
}

struct LanesMax {   // over lanes l, l^16, l^32, l^48
  TP_DEVICE float operator()(float v) const {
    uint32_t u = __float_as_uint(v);
    auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    u = __float_as_uint(v);
    a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
};

// When a k-tile's successor is fetched: behind the reads of the first fragments
// (the waves' first products then do not wait behind address arithmetic: 131 ->
// 120 us for 50432 x 384 -> 1536 with GELU and codes), behind those of all, or
// between the two halves of the products. Which is best goes by the registers
// that are left: all fragments of 16 waves at once spill.
enum { kAfterFirst = 0, kAfterReads = 1, kBetween = 2 };

// What follows the sum: nothing but the residual, GELU with z kept in 16 bits
// (or not at all), GELU with z kept in 8.
enum { kNoAct = 0, kGelu = 1, kGelu8 = 2 };

template <bool FULL, typename T>
TP_DEVICE void put8(T* p, int n, const float (&v)[8]) {
  if constexpr (FULL)
    store8(p, v);
  else
    store8n(p, n, v);
}
template <bool FULL, typename T>
TP_DEVICE void add8(const T* p, int n, float (&v)[8]) {
  float r[8];
  if constexpr (FULL)
    load8(p, r);
  else
    load8n(p, n, r);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += r[i];
}

// GELU of a lane's 8 values. gelu_short holds from -6.5 on; behind that, and
// at -inf, the tail is the longer form's. One value in 10^10 of a normal
// distribution lies there, so a wave seldom takes the branch. 32-bit results
// (wide) have the longer form throughout: the short one's 8.5e-7 is more than
// their own rounding.
TP_DEVICE void gelu_all(float (&v)[8], bool wide) {
  float low = v[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) low = fminf(low, v[i]);   // passes NaN over
  if (!wide && (low >= -6.5f || low != low)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = gelu_short(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = gelu(v[i]);
  }
}

// v: the sums of 8 neighbouring columns of one row; n of them exist (<= 0:
// none; FULL: all). The lanes l, l^16, l^32 and l^48 hold one 32-column block.
// PLAIN: no residual, no mask, 16-bit output, known beforehand (choosing here
// costs the registers' moves where the choices meet again, a tenth of the
// epilogue).
template <typename T, int ACT, bool FULL, bool PLAIN>
TP_DEVICE void epilogue8(const Epi& e, int64_t at, int64_t blk, int n,
                         bool first, float (&v)[8]) {
  if constexpr (ACT == kGelu8) {
    int x;
    uint2 q = encode8(v, x, LanesMax());
    if (FULL || n > 0) {
      store_codes((uint8_t*)e.z + at, FULL ? 8 : n, q);
      if (first) e.zscale[blk] = (uint8_t)(x + 127);
    }
  }
  if constexpr (ACT == kGelu)
    if (e.z) {
      // within the finite range: the slope of an fp16 infinity would be NaN
      // beside a result that is finite in 32 bits
      float k[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) k[i] = held_in<T>(v[i]);
      put8<FULL>((T*)e.z + at, n, k);
    }
  if constexpr (ACT != kNoAct) gelu_all(v, !PLAIN && e.out_f32);
  if constexpr (PLAIN) {
    put8<FULL>((T*)e.out + at, n, v);
    return;
  }
  if (e.res) {
    if (e.res_f32)
      add8<FULL>((const float*)e.res + at, n, v);
    else
      add8<FULL>((const T*)e.res + at, n, v);
  }
  if constexpr (ACT == kNoAct)
    if (e.mask) {
      float m[8];
      load8n(e.mask + at, n, m);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = m[i] != 0.f ? v[i] : 0.f;
    }
  if (e.out_f32)
    put8<FULL>((float*)e.out + at, n, v);
  else
    put8<FULL>((T*)e.out + at, n, v);
}

// C = Q P, a tile to a block: BK values of the sum at a time go into LDS by
// asynchronous 16-byte loads, a step ahead of the one that is multiplied, with
// one barrier a step; WQ x WP waves share the tile, their sums in registers
// until the epilogue. 25216 x 4096 -> 1024 in 256 x 256 takes 200 us (1060
// TF/s): 1.6 us for a step of 64, which is what a library product of 8192 x
// 8192 x 8192 takes for as much (1370 TF/s), but 396 tiles occupy 256 CUs
// twice. Tried without gain: three and four stages of 32 (a barrier costs more
// than the longer lead gives), fragments of the next half read ahead of the
// products, lines brought into L2 two and three steps ahead, steps begun at
// another place in every block.
template <typename T, int BQ, int BP, int BK, int WQ, int WP, int QF, int PF,
          int STAGES, int MINW, int WHEN, int ACT, bool PLAIN>
__global__ __launch_bounds__(WQ * WP * 64, MINW) void mm_kernel(Mm a) {
  constexpr int NW = WQ * WP;
  constexpr bool QTR = QF != kRowK, PTR = PF != kRowK;
  constexpr int QB = Tile<BQ, BK, QTR>::kBytes, PB = Tile<BP, BK, PTR>::kBytes;
  // asynchronous loads of a wave for one k-tile
  constexpr int LOADS = (QB + (PF == kCodes ? 0 : PB)) / 1024 / NW;
  constexpr int MI = BQ / WQ / 16, NI = BP / WP / 16;
  static_assert(NI % 2 == 0, "columns in pairs of fragments");
  __shared__ __attribute__((aligned(1024))) char smem[STAGES * (QB + PB)];
  TP_LDS char* lds = (TP_LDS char*)smem;

  // Workgroups go to the 8 XCDs in turn; each XCD takes a contiguous run of
  // tiles, so that neighbouring tiles meet in its L2.
  int wg = blockIdx.x;
  {
    int q = a.tiles / 8, r = a.tiles % 8, x = wg % 8;
    wg = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + wg / 8;
  }
  int m0 = wg / a.tiles_n * BQ, n0 = wg % a.tiles_n * BP;
  int lane = threadIdx.x & 63;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  int wq = wave / WP * (BQ / WQ), wp = wave % WP * (BP / WP);

  int kt0 = blockIdx.y * a.kper;
  int kt1 = min((a.K + BK - 1) / BK, kt0 + a.kper);

  auto place = [&](int kt) {
    return lds + (kt - kt0) % STAGES * (QB + PB);
  };
  auto fetch = [&](int kt) {
    TP_LDS char* b = place(kt);
    stage<BQ, BK, QTR, NW>(b, a.q, a.ldq, m0, a.nq, kt, a.K, wave, lane);
    if constexpr (PF != kCodes)
      stage<BP, BK, PTR, NW>(b + QB, a.p, a.ldp, n0, a.np, kt, a.K, wave, lane);
  };
  CodeTile<T, BP, BK, NW * 64> ct;

  // the sum begins with the bias: lane l holds four columns from l / 16 * 4
  f32x4 acc[NI][MI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    f32x4 b = {};
    int col = n0 + wp + i * 16 + (lane >> 4) * 4;
    if (a.e.bias)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (col + k < a.N)
          b[k] = a.e.bias_f32 ? ((const float*)a.e.bias)[col + k]
                              : to_float<T>(((const T*)a.e.bias)[col + k]);
#pragma unroll
    for (int j = 0; j < MI; ++j) acc[i][j] = b;
  }
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (kt0 + s < kt1) fetch(kt0 + s);
  if constexpr (PF == kCodes) {
    if (kt0 < kt1) {
      ct.load(a, n0, kt0);
      ct.store(place(kt0) + QB);
    }
    if (kt0 + 1 < kt1) ct.load(a, n0, kt0 + 1);
  }
  for (int kt = kt0; kt < kt1; ++kt) {
    // All but the newest STAGES - 2 tiles' loads: tile kt is there. Loads of
    // codes in flight only make the wait longer than it need be.
    if (kt + STAGES - 2 < kt1)
      wait_and_meet<(STAGES - 2) * LOADS>();
    else
      wait_and_meet<0>();
    // Every wave has read tile kt - 1, whose place tile kt + STAGES - 1 takes.
    TP_LDS const char* b = place(kt);
    auto more = [&]() {
      if (kt + STAGES - 1 < kt1) fetch(kt + STAGES - 1);
      if constexpr (PF == kCodes) {
        if (kt + 1 < kt1) ct.store(place(kt + 1) + QB);
        if (kt + 2 < kt1) ct.load(a, n0, kt + 2);
      }
    };
    constexpr int KS = BK / 32;
    s16x8 fq[KS][MI], fp[KS][NI];
    auto read = [&](int ks) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
        fq[ks][i] = frag<BQ, BK, QTR>(b, wq + i * 16, ks, lane);
#pragma unroll
      for (int i = 0; i < NI; ++i)
        fp[ks][i] = frag<BP, BK, PTR>(b + QB, wp + i * 16, ks, lane);
    };
    auto multiply = [&](int ks) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j)
          acc[i][j] = mma<T>(fp[ks][i], fq[ks][j], acc[i][j]);
    };
    read(0);
    if constexpr (WHEN == kAfterFirst) {
      more();
      multiply(0);
#pragma unroll
      for (int ks = 1; ks < KS; ++ks) {
        read(ks);
        multiply(ks);
      }
      // last, when no fragment is alive
      if constexpr (QF == kRowK && PF == kRowK)
        if (a.qcodes && kt % a.tiles_n == wg % a.tiles_n)
          keep_tile<T, BQ, BK, NW * 64>(b, a, m0, kt);
    } else {
#pragma unroll
      for (int ks = 1; ks < KS; ++ks) read(ks);
      if constexpr (WHEN == kAfterReads) more();
      multiply(0);
      if constexpr (WHEN == kBetween) more();
#pragma unroll
      for (int ks = 1; ks < KS; ++ks) multiply(ks);
    }
  }

  // Lane l of a fragment holds row l % 16 of C and four columns from
  // (l / 16) * 4. Swapping 16-lane groups between two neighbouring fragments
  // leaves every lane with eight neighbouring columns: one 16-byte store.
  a.e.out = (char*)a.e.out + (int64_t)blockIdx.y * a.M * a.N * 4;
  int g = lane >> 4, nblk = (a.N + 31) / 32;
  auto finish = [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
#pragma unroll
    for (int j = 0; j < MI; ++j) {
      int row = m0 + wq + j * 16 + (lane & 15);
      int c0 = n0 + wp + (g & 1) * 16 + (g >> 1) * 8;
      int64_t at = (int64_t)row * a.N + c0;
      int64_t blk = (int64_t)row * nblk + (n0 + wp) / 32;
#pragma unroll
      for (int i = 0; i < NI; i += 2) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          auto s = __builtin_amdgcn_permlane16_swap(
              __float_as_uint(acc[i][j][k]),
              __float_as_uint(acc[i + 1][j][k]), false, false);
          v[k] = __uint_as_float(s[0]);
          v[4 + k] = __uint_as_float(s[1]);
        }
        epilogue8<T, ACT, FULL, PLAIN>(a.e, at + i * 16, blk + i / 2,
                                row < a.M ? a.N - c0 - i * 16 : 0, g == 0, v);
      }
    }
  };
  if (m0 + BQ <= a.M && n0 + BP <= a.N && a.N % 8 == 0)
    finish(std::true_type());
  else
    finish(std::false_type());
}

// Few rows (single tokens, one image, a classifier's batch): nothing is used
// often enough for tiles to pay, and the staged kernel would give 29 x 2875 ->
// 768 to 12 CUs, each waiting for 45 loads in turn. A block takes 32 columns
// and MI x 16 rows; its 8 waves take 32 values of k each in turn, straight from
// global memory into fragments (rows at any address), and their sums meet in
// LDS, wave j finishing 16 rows. Bound by the latency of the few steps that
// each wave makes (1 x 384 -> 1000 and 1 x 768 -> 768 4 us), then by what a
// block reads: 1 x 4096 -> 4096 13 us, 2.6 TB/s, weights from memory.
//
// 8 values of a row from p on. Where rows have an odd length they start between
// two dwords every other time, and a 16-byte load there is taken apart by the
// memory pipe: such lanes load the five dwords around their values and shift
// (29 x 2875 -> 768: 17 us, 27 with loads at odd addresses; 12 where K is
// even).
template <typename T, bool ODD>
struct Few {
  u32x4 d;
  uint32_t e, odd;
  TP_DEVICE void load(const T* p) {   // ODD: needs two values behind the eight
    odd = ODD ? (uint32_t)(uintptr_t)p & 2 : 0;
    const char* c = (const char*)p - odd;
    d = *reinterpret_cast<const u32x4_a4*>(c);
    if constexpr (ODD) e = *reinterpret_cast<const uint32_t*>(c + 16);
  }
  TP_DEVICE s16x8 get() const {
    if constexpr (!ODD) return __builtin_bit_cast(s16x8, d);
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = __builtin_amdgcn_alignbyte(i < 3 ? d[i + 1] : e, d[i], odd);
    return __builtin_bit_cast(s16x8, r);
  }
};
// the end of a row: n of 8 values exist (none where n <= 0)
template <typename T>
TP_DEVICE s16x8 last_of(const T* p, int n) {
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
  u32x4 d = {};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) d[i / 2] |= (uint32_t)h[i] << (16 * (i & 1));
  return __builtin_bit_cast(s16x8, d);
}

template <typename T, int MI, int ACT, bool ODD>
__global__ __launch_bounds__(512) void rows_kernel(Mm a) {
  constexpr int NW = 8, U = 4;   // waves; steps of k in flight
  __shared__ f32x4 part[NW][2 * MI][64];
  int lane = threadIdx.x & 63, g = lane >> 4;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  int n0 = blockIdx.x * 32, m0 = blockIdx.y * (MI * 16);
  // rows behind the last are the last one again: what they give is not stored
  const T* q[MI];
  const T* p[2];
#pragma unroll
  for (int j = 0; j < MI; ++j)
    q[j] = (const T*)(a.q + min(m0 + j * 16 + (lane & 15), a.M - 1) * a.ldq);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    p[i] = (const T*)(a.p + min(n0 + i * 16 + (lane & 15), a.N - 1) * a.ldp);
  f32x4 acc[2][MI] = {};
  // whole steps: with ODD those that have two values behind them
  constexpr int W = ODD ? 34 : 32;
  int whole = a.K >= W ? (a.K - W) / 32 + 1 : 0;
  for (int s = wave; s < whole; s += NW * U) {
    Few<T, ODD> fq[U][MI], fp[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u * NW >= whole) break;
      int k = (s + u * NW) * 32 + g * 8;
#pragma unroll
      for (int i = 0; i < 2; ++i) fp[u][i].load(p[i] + k);
#pragma unroll
      for (int j = 0; j < MI; ++j) fq[u][j].load(q[j] + k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u * NW >= whole) break;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j)
          acc[i][j] = mma<T>(fp[u][i].get(), fq[u][j].get(), acc[i][j]);
    }
  }
  // the one or two steps that end the rows
  for (int s = whole; s * 32 < a.K; ++s) {
    if (s % NW != wave) continue;
    int k = s * 32 + g * 8;
    s16x8 wq[MI], wp[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) wp[i] = last_of(p[i] + k, a.K - k);
#pragma unroll
    for (int j = 0; j < MI; ++j) wq[j] = last_of(q[j] + k, a.K - k);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < MI; ++j)
        acc[i][j] = mma<T>(wp[i], wq[j], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < MI; ++j) part[wave][i * MI + j][lane] = acc[i][j];
  __syncthreads();
  if (wave >= MI) return;
  int j = wave, row = m0 + j * 16 + (lane & 15);
  f32x4 s[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s[i] = part[0][i * MI + j][lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) s[i] += part[w][i * MI + j][lane];
    int col = n0 + i * 16 + g * 4;
    if (a.e.bias)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (col + k < a.N)
          s[i][k] += a.e.bias_f32 ? ((const float*)a.e.bias)[col + k]
                                  : to_float<T>(((const T*)a.e.bias)[col + k]);
  }
  float v[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    auto t = __builtin_amdgcn_permlane16_swap(
        __float_as_uint(s[0][k]), __float_as_uint(s[1][k]), false, false);
    v[k] = __uint_as_float(t[0]);
    v[4 + k] = __uint_as_float(t[1]);
  }
  int c0 = n0 + (g & 1) * 16 + (g >> 1) * 8;
  epilogue8<T, ACT, false, false>(
      a.e, (int64_t)row * a.N + c0,
      (int64_t)row * ((a.N + 31) / 32) + blockIdx.x,
      row < a.M ? a.N - c0 : 0, g == 0, v);
}

// The ends of both sums over rows: the dz pass's parts of the bias gradient, 16
// columns to a block, and the slabs of a split product, masked and rounded, by
// the blocks behind those. Alone each takes 5 to 8 us, most of it latency (14
// slabs of 1536 x 384, 37 MB in all, 8).
struct Join {
  const float* part;   // (slabs, n)
  const float* mask;   // n values, or null
  void* out;
  int64_t n;
  int slabs;
  const float* colpart;   // (rows, C)
  void* colout;
  int rows, C, coltype;   // type of colout: 0 float32, 1 bfloat16, 2 float16
};
template <typename T>
__global__ __launch_bounds__(kBlock) void join_kernel(Join a) {
  __shared__ float sum[16][17];
  int first = (int)blockIdx.x - (a.C + 15) / 16;
  if (first >= 0) {
    int64_t i = ((int64_t)first * kBlock + threadIdx.x) * 8;
    int m = (int)min((int64_t)8, a.n - i);
    if (m <= 0) return;
    float s[8];
    load8n(a.part + i, m, s);
    for (int k = 1; k < a.slabs; ++k) {
      float v[8];
      load8n(a.part + (int64_t)k * a.n + i, m, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
    }
    if (a.mask) {
      float v[8];
      load8n(a.mask + i, m, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = v[j] != 0.f ? s[j] : 0.f;
    }
    store8n((T*)a.out + i, m, s);
    return;
  }
  int k = threadIdx.x / 16, l = threadIdx.x % 16;
  int c = (int)blockIdx.x * 16 + l;
  float v = 0.f;
  if (c < a.C) {
    const float* p = a.colpart + c;
    int r = k;
    for (; r + 7 * 16 < a.rows; r += 8 * 16) {
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = p[(int64_t)(r + i * 16) * a.C];
#pragma unroll
      for (int i = 0; i < 8; ++i) v += t[i];
    }
    for (; r < a.rows; r += 16) v += p[(int64_t)r * a.C];
  }
  sum[k][l] = v;
  __syncthreads();
  if (k || c >= a.C) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) v += sum[i][l];
  if (a.coltype == 0)
    ((float*)a.colout)[c] = v;
  else if (a.coltype == 1)
    ((__hip_bfloat16*)a.colout)[c] = from_float<__hip_bfloat16>(v);
  else
    ((_Float16*)a.colout)[c] = from_float<_Float16>(v);
}

// w (N, K), rows ldw apart, to (K, N8) with zeros behind N: 64 x 64 tiles
// through LDS
struct Turn {
  const void* w;
  void* out;
  int64_t ldw;
  int N, K, N8;
};
template <typename T>
TP_DEVICE void turn_tile(const Turn& a, int tile, char* lds) {
  T(*l)[66] = reinterpret_cast<T(*)[66]>(lds);
  int tn = (a.N8 + 63) / 64;
  int n0 = tile % tn * 64, k0 = tile / tn * 64;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int at = i * kBlock + threadIdx.x, r = at / 8, c = at % 8 * 8;
    int n = n0 + r;
    float v[8];
    load8n((const T*)a.w + (int64_t)n * a.ldw + k0 + c,
           n < a.N ? a.K - k0 - c : 0, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) l[c + j][r] = from_float<T>(v[j]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int at = i * kBlock + threadIdx.x, r = at / 8, c = at % 8 * 8;
    if (k0 + r >= a.K || n0 + c >= a.N8) continue;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_float<T>(l[r][c + j]);
    store8((T*)a.out + (int64_t)(k0 + r) * a.N8 + n0 + c, v);
  }
}
int64_t turn_tiles(const Turn& t) {
  return (int64_t)((t.N8 + 63) / 64) * ((t.K + 63) / 64);
}
constexpr int kTurnBytes = 64 * 66 * 2;
template <typename T>
__global__ __launch_bounds__(kBlock) void turn_kernel(Turn a) {
  __shared__ __attribute__((aligned(16))) char lds[kTurnBytes];
  turn_tile<T>(a, blockIdx.x, lds);
}

// dz = dy act'(z), rounded to the products' 16 bits (matrix instructions take
// no more of them at that rate; it adds as much to a gradient's error as the
// rounding of the gradient itself, and in fp16 it has that type's range: what
// overflows arrives as an infinity, by which a gradient scaler finds it), and
// the column sums of dz, unrounded. 32 threads take 256 neighbouring columns, 8
// rows at a time; a block adds its rows in registers and joins them in LDS, so
// the sums need no atomics and keep their order. Bound by memory: 50432 x 1536
// with z in 8 bits 84 us, 4.6 TB/s. The blocks behind the rows' turn the weight
// over meanwhile, which takes 5 us by itself, of latency.
struct Dz {
  const void* dy;
  const void* z;           // 16-bit values or codes; null without act
  const uint8_t* zscale;
  void* dz;                // (M, ldz), ldz a multiple of 8; null: only sums
  float* part;             // (blocks, N); null without a bias
  int64_t M;
  int N, ldz;
  int rows;                // blocks along M; those behind them turn
  Turn turn;
};
template <typename T, typename TG, int CT>
__global__ __launch_bounds__(kBlock) void dz_kernel(Dz a) {
  constexpr int RL = kBlock / CT;
  constexpr int SUM = RL * (CT * 8 + 1) * 4;
  __shared__ __attribute__((aligned(16))) char
      lds[SUM > kTurnBytes ? SUM : kTurnBytes];
  if ((int)blockIdx.y >= a.rows) {
    int64_t t = (int64_t)(blockIdx.y - a.rows) * gridDim.x + blockIdx.x;
    if (t < (int64_t)((a.turn.N8 + 63) / 64) * ((a.turn.K + 63) / 64))
      turn_tile<T>(a.turn, (int)t, lds);
    return;
  }
  int c = (blockIdx.x * CT + threadIdx.x % CT) * 8;
  int n = a.N - c, rl = threadIdx.x / CT;
  float s[8] = {};
  if (n > 0) {
    for (int64_t r = (int64_t)blockIdx.y * RL + rl; r < a.M;
         r += (int64_t)a.rows * RL) {
      float g[8];
      load8n((const TG*)a.dy + r * a.N + c, n, g);
      if (a.z) {
        float z[8];
        if (a.zscale) {
          uint2 q = load_codes((const uint8_t*)a.z + r * a.N + c, n);
          int e = (int)a.zscale[r * ((a.N + 31) / 32) + c / 32] - 127;
          decode8(q, pow2(e), z);
        } else {
          load8n((const T*)a.z + r * a.N + c, n, z);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] *= gelu_slope(z[i]);
      }
      // the rows end with zeros up to a multiple of 8: g is 0 there
      if (a.dz) store8((T*)a.dz + r * a.ldz + c, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += g[i];
    }
  }
  if (!a.part) return;
  float(*sum)[CT * 8 + 1] = reinterpret_cast<float(*)[CT * 8 + 1]>(lds);
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[rl][threadIdx.x % CT * 8 + i] = s[i];
  __syncthreads();
  for (int k = threadIdx.x; k < CT * 8; k += kBlock) {
    int col = blockIdx.x * CT * 8 + k;
    if (col >= a.N) continue;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < RL; ++i) v += sum[i][k];
    a.part[(int64_t)blockIdx.y * a.N + col] = v;
  }
}

// rows of C values to rows of ldo values (a multiple of 8), zeros behind
template <typename T>
__global__ __launch_bounds__(kBlock) void pad_kernel(
    const T* __restrict__ x, T* __restrict__ out, int64_t chunks, int64_t ldx,
    int C, int cpr) {
  int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= chunks) return;
  int64_t row = i / cpr;
  int c = (int)(i - row * cpr) * 8;
  float v[8];
  load8n(x + row * ldx + c, C - c, v);
  store8(out + (row * cpr) * 8 + c, v);
}

bool is16(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }

template <typename F>
void by16(at::ScalarType t, F&& f) {
  if (t == at::kBFloat16)
    f(__hip_bfloat16());
  else
    f(_Float16());
}

hipStream_t current() { return at::hip::getCurrentHIPStream(); }

// blocks of a launch, which may have fewer than 2^32 threads
unsigned grid_of(int64_t blocks, int threads) {
  TORCH_CHECK(blocks * threads < (int64_t(1) << 32),
              "linear_act: a matrix too large for one launch");
  return (unsigned)blocks;
}

constexpr int kMaxCols = 1 << 20;   // row offsets of a tile fit 31 bits

// A 2-D matrix that the tiles can load: values of a row together, rows 16
// bytes aligned and a multiple of 8 values long; a copy where it is not.
at::Tensor loadable(const at::Tensor& t) {
  int64_t R = t.size(0), C = t.size(1);
  bool fits = C % 8 == 0 && (C <= 1 || t.stride(1) == 1) &&
              (R <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= C &&
                          t.stride(0) <= kMaxCols)) &&
              reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  if (fits) return t;
  auto s = C <= 1 || t.stride(1) == 1 ? t : t.contiguous();
  int64_t C8 = (C + 7) / 8 * 8;
  auto out = at::empty({R, C8}, t.options());
  int64_t chunks = R * C8 / 8;
  if (chunks)
    by16(t.scalar_type(), [&](auto z) {
      using T = decltype(z);
      pad_kernel<T><<<grid_of((chunks + kBlock - 1) / kBlock, kBlock), kBlock,
                      0, current()>>>(
          (const T*)s.data_ptr(), (T*)out.data_ptr(), chunks, s.stride(0),
          (int)C, (int)(C8 / 8));
      C10_HIP_KERNEL_LAUNCH_CHECK();
    });
  return out;
}
int64_t row_bytes(const at::Tensor& t) {
  return (t.size(0) <= 1 ? t.size(1) : t.stride(0)) * 2;
}

template <typename T, int BQ, int BP, int BK, int WQ, int WP, int QF, int PF,
          int ST, int MINW, int WHEN, int ACT = kNoAct>
void launch_mm(Mm a, int slabs = 1) {
  // across the sum (weight gradients) the output is masked or in slabs
  constexpr bool kRows = PF == kRowK;
  bool plain = kRows && !a.e.res && !a.e.mask && !a.e.out_f32;
  a.tiles_n = (a.N + BP - 1) / BP;
  a.tiles = (int)grid_of((int64_t)((a.M + BQ - 1) / BQ) * a.tiles_n,
                         WQ * WP * 64);
  int kt = (a.K + BK - 1) / BK;
  a.kper = (kt + slabs - 1) / slabs;
  dim3 grid(a.tiles, slabs);
  if (kRows && plain)
    mm_kernel<T, BQ, BP, BK, WQ, WP, QF, PF, ST, MINW, WHEN, ACT,
              kRows>
        <<<grid, WQ * WP * 64, 0, current()>>>(a);
  else
    mm_kernel<T, BQ, BP, BK, WQ, WP, QF, PF, ST, MINW, WHEN, ACT,
              false>
        <<<grid, WQ * WP * 64, 0, current()>>>(a);
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

int64_t tiles_of(int64_t M, int64_t N, int q, int p) {
  return (M + q - 1) / q * ((N + p - 1) / p);
}
int64_t tiles_of(const Mm& a, int q, int p) {
  return tiles_of(a.M, a.N, q, p);
}

// Groups of 16 rows that a block of rows_kernel takes, 0: the tiles. Such
// blocks hold little and read much, so they win while the chip has a CU for
// each, and the smallest that still have one win most (fp16, us, with 1, 2 and
// 4 groups to a block, and the staged kernel in 64 x 64): 64 x 4096 -> 1024
// 13.4, 16.8, 23.7, 32.6; 197 x 768 -> 768 6.7, 5.6, 6.9, 7.3; 128 x 4096 ->
// 4096 (128 column blocks, so 4 groups) 47, 32, 25, 34. Past that many blocks
// the tiles win, 197 x 1024 -> 4096 in 11.6 against 14.7, but for a weight that
// is read once all the same: 16 x 1024 -> 16384 8.2 against 11.5, 32 rows 10.0
// against 11.6, 64 rows 15.2 against 11.6.
int row_groups(int64_t M, int64_t N) {
  int64_t cols = (N + 31) / 32;
  for (int g = 1; g <= 4; g *= 2)
    if ((M + g * 16 - 1) / (g * 16) * cols <= 256) return g;
  return M <= 16 ? 1 : M <= 32 ? 2 : 0;
}
template <typename T, int ACT>
void run_few(const Mm& a, int groups) {
  dim3 grid((a.N + 31) / 32, (a.M + groups * 16 - 1) / (groups * 16));
  auto run = [&](auto odd) {
    constexpr bool ODD = decltype(odd)::value;
    auto s = current();
    if (groups == 1)
      rows_kernel<T, 1, ACT, ODD><<<grid, 512, 0, s>>>(a);
    else if (groups == 2)
      rows_kernel<T, 2, ACT, ODD><<<grid, 512, 0, s>>>(a);
    else
      rows_kernel<T, 4, ACT, ODD><<<grid, 512, 0, s>>>(a);
    C10_HIP_KERNEL_LAUNCH_CHECK();
  };
  if (((uintptr_t)a.q | (uintptr_t)a.p | a.ldq | a.ldp) & 2)
    run(std::true_type());
  else
    run(std::false_type());
}

// Both operands along the sum. Short products end soonest in many small tiles:
// 1576 x 768 -> 768 10.2 us in 64 x 64, 12.0 in 128 x 128; 3152 x 384 -> 1536
// (1200 small tiles) 13.8 against 12.9.
//
// Of the large tiles 256 x 256 by 16 waves moves the fewest bytes into LDS per
// product, but a CU holds one, and one tile more than CUs doubles the time. Of
// 160 x 128 by 4 waves and 128 x 128 by 8 a CU holds two, the epilogue of one
// behind the product of the other. What decides is how often the CU that has
// most has to begin anew; per value of the output the smaller ones take 1.2 and
// 1.25 times as long, and an odd one, alone at the end, half as long again as
// in company. Over 60 sizes (6304 to 50432 rows, N and K of 384 to 4096, with
// and without a 32-bit residual) this finds the fastest within 1 % on average
// and 14 % at most; 256 x 256 wherever it is well filled, else 128 x 128, is
// 7 % and 47 % off. In us, 256 x 256, 160 x 128, 128 x 128:
//   50432 x 384 -> 1536, GELU, codes   118  135  137
//   50432 x 1536 -> 384, residual      126   99  110
//   25216 x 4096 -> 1024               199  211  225
//   25216 x 2560 -> 768                120   94  108
//   6304 x 4096 -> 1024                 85   76   63
std::tuple<int64_t, int64_t> rows_tile(int64_t M, int64_t N) {
  if (tiles_of(M, N, 64, 64) <= 600) return {64, 64};
  auto cost = [&](int q, int p, int one) {
    int64_t n = (tiles_of(M, N, q, p) + 255) / 256;
    return one * n + (p < 256 && n > 1 && n % 2 ? one / 2 : 0);
  };
  int64_t big = cost(256, 256, 32), mid = cost(160, 128, 12),
          low = cost(128, 128, 10);
  if (mid <= low && mid <= big) return {160, 128};
  if (low <= big) return {128, 128};
  return {256, 256};
}
template <typename T, int ACT>
void run_rows(const Mm& a) {
  switch (std::get<0>(rows_tile(a.M, a.N))) {
    case 64:
      return launch_mm<T, 64, 64, 64, 2, 2, kRowK, kRowK, 2, 1, kAfterFirst,
                       ACT>(a);
    case 160:
      return launch_mm<T, 160, 128, 64, 2, 2, kRowK, kRowK, 2, 2, kAfterFirst,
                       ACT>(a);
    case 128:
      return launch_mm<T, 128, 128, 64, 2, 4, kRowK, kRowK, 2, 2, kAfterFirst,
                       ACT>(a);
    default:
      return launch_mm<T, 256, 256, 64, 4, 4, kRowK, kRowK, 2, 4, kAfterFirst,
                       ACT>(a);
  }
}

// Both across the sum (weight gradients), in slabs of it: as many as go into
// one round of the chip (256 blocks, 512 of the smaller tiles), none shorter
// than four k-tiles. Rounds are not counted, so a weight of just over half a
// round's tiles (129 of 256) has one slab and leaves the other CUs idle. A
// gradient of 4096 x 1024 over 25216 rows takes 197 us in 256 x 256 tiles and
// 235 in 128 x 128; 1536 x 384 over 50432 rows 88 us in 128 x 128 and 95 in 256
// x 256, whose third column tile is half empty. Codes go through registers,
// which 16 waves leave too few of: 8 waves there (200 us against 285; 128 x 128
// 266).
struct Split {
  int tile, slabs;
};
Split split_of(const Mm& a) {
  int big = (int)std::min<int64_t>(tiles_of(a, 256, 256), 1 << 20);
  int64_t kt = (a.K + 63) / 64;
  bool even = (a.M % 256 == 0 || a.M % 256 > 192 || a.M > 2048) &&
              (a.N % 256 == 0 || a.N % 256 > 192 || a.N > 2048);
  int tile = big >= 12 && even ? 256 : 128;
  if (tile == 128 && tiles_of(a, 128, 128) * (kt / 4) < 128) tile = 64;
  int64_t tiles = tiles_of(a, tile, tile);
  int64_t fill = tile == 256 ? 256 : 512;
  int64_t most = std::max<int64_t>(1, kt / (tile == 64 ? 2 : 4));
  return {tile, (int)std::max<int64_t>(1, std::min(most, fill / tiles))};
}
template <typename T, int PF>
void run_cols(const Mm& a, Split s) {
  if (s.tile == 256) {
    if constexpr (PF == kCodes)
      return launch_mm<T, 256, 256, 64, 2, 4, kColK, PF, 2, 2, kBetween>(
          a, s.slabs);
    else
      return launch_mm<T, 256, 256, 64, 4, 4, kColK, PF, 2, 4, kAfterFirst>(
          a, s.slabs);
  }
  if (s.tile == 128)
    return launch_mm<T, 128, 128, 64, 2, 4, kColK, PF, 2, 2, kAfterReads>(
        a, s.slabs);
  launch_mm<T, 64, 64, 64, 2, 2, kColK, PF, 2, 1, kAfterReads>(a, s.slabs);
}

void check_size(int64_t M, int64_t N, int64_t K) {
  TORCH_CHECK(M <= (int64_t(1) << 30) && N <= kMaxCols && K <= kMaxCols,
              "linear_act: at most 2^30 rows of ", kMaxCols, " values");
}

}  // namespace

// rows and columns of the tiles that a product of M x N values along both rows
// runs in (few rows without a gradient aside)
std::tuple<int64_t, int64_t> linear_act_tile(int64_t M, int64_t N) {
  TORCH_CHECK(M > 0 && N > 0, "linear_act_tile: sizes from 1 on");
  check_size(M, N, 1);
  return rows_tile(M, N);
}
// rows and columns of the tiles, and slabs, of the gradient of an N x K weight
// over M rows
std::tuple<int64_t, int64_t> linear_act_split(int64_t M, int64_t N, int64_t K) {
  TORCH_CHECK(M > 0 && N > 0 && K > 0, "linear_act_split: sizes from 1 on");
  check_size(M, N, K);
  Mm a{};
  a.M = (int)N;
  a.N = (int)K;
  a.K = (int)M;
  Split s = split_of(a);
  return {s.tile, s.slabs};
}

// (y, z, scales of z, x's codes, their scales). keep: 0 keeps nothing, 1 the
// pre-activation in 16 bits, 2 in 8 bits (only with act); keep_x: x in 8 bits.
std::tuple<at::Tensor, c10::optional<at::Tensor>, c10::optional<at::Tensor>,
           c10::optional<at::Tensor>, c10::optional<at::Tensor>>
linear_act_fwd(const at::Tensor& x, const at::Tensor& w,
               const c10::optional<at::Tensor>& bias,
               const c10::optional<at::Tensor>& residual, bool act,
               int64_t keep, bool keep_x) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && w.dim() == 2 &&
                  x.size(1) == w.size(1) && x.size(0) > 0 && x.size(1) > 0 &&
                  w.size(0) > 0,
              "linear_act_fwd: x (M,K) and w (N,K) on a GPU, none empty");
  TORCH_CHECK(is16(x.scalar_type()) && w.scalar_type() == x.scalar_type() &&
                  w.device() == x.device(),
              "linear_act_fwd: x and w in bfloat16 or float16, on one device");
  int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  check_size(M, N, K);
  c10::DeviceGuard guard(x.device());
  auto st = x.scalar_type();
  Mm a{};
  at::Tensor b, r;
  if (bias.has_value()) {
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == N &&
                    bias->device() == x.device() &&
                    (bias->scalar_type() == st ||
                     bias->scalar_type() == at::kFloat),
                "linear_act_fwd: bias of N values in x's type or float32");
    b = bias->contiguous();
    a.e.bias = b.data_ptr();
    a.e.bias_f32 = b.scalar_type() == at::kFloat;
  }
  auto ot = st;
  if (residual.has_value()) {
    TORCH_CHECK(residual->dim() == 2 && residual->size(0) == M &&
                    residual->size(1) == N &&
                    residual->device() == x.device() &&
                    (residual->scalar_type() == st ||
                     residual->scalar_type() == at::kFloat),
                "linear_act_fwd: residual (M,N) in x's type or float32");
    r = residual->contiguous();
    a.e.res = r.data_ptr();
    a.e.res_f32 = r.scalar_type() == at::kFloat;
    ot = r.scalar_type();
  }
  // few outputs without a backward pass to come (in training every sum is the
  // tiles', so that it does not go by what is kept); they need neither
  // alignment nor padding
  int few = keep == 0 && !keep_x ? row_groups(M, N) : 0;
  auto in_rows = [](const at::Tensor& t) {
    return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous();
  };
  auto xl = few ? in_rows(x) : loadable(x), wl = few ? in_rows(w) : loadable(w);
  auto y = at::empty({M, N}, x.options().dtype(ot));
  c10::optional<at::Tensor> z, zs;
  if (act && keep == 1) z = at::empty({M, N}, x.options());
  if (act && keep == 2) std::tie(z, zs) = act8_empty({M, N}, x.options());
  c10::optional<at::Tensor> xc, xs;
  if (keep_x) {
    std::tie(xc, xs) = act8_empty({M, K}, x.options());
    a.qcodes = (uint8_t*)xc->data_ptr();
    a.qscale = (uint8_t*)xs->data_ptr();
  }
  if (z) a.e.z = z->data_ptr();
  if (zs) a.e.zscale = (uint8_t*)zs->data_ptr();
  a.e.out = y.data_ptr();
  a.e.out_f32 = ot == at::kFloat;
  a.q = (const char*)xl.data_ptr();
  a.p = (const char*)wl.data_ptr();
  a.ldq = row_bytes(xl);
  a.ldp = row_bytes(wl);
  a.nq = a.M = (int)M;
  a.np = a.N = (int)N;
  a.K = (int)K;
  by16(st, [&](auto t) {
    using T = decltype(t);
    if (few)
      act ? run_few<T, kGelu>(a, few) : run_few<T, kNoAct>(a, few);
    else if (!act)
      run_rows<T, kNoAct>(a);
    else if (zs)
      run_rows<T, kGelu8>(a);
    else
      run_rows<T, kGelu>(a);
  });
  return {y, z, zs, xc, xs};
}

// (dx, dw, db), each only where asked for. z: the kept pre-activation (16-bit
// values, or codes with zscale), null without an activation. xk: the kept
// input (16-bit values, or codes with xscale). dw has dw_type and the mask
// applied, db has db_type.
std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>,
           c10::optional<at::Tensor>>
linear_act_bwd(const at::Tensor& dy_in, const c10::optional<at::Tensor>& z,
               const c10::optional<at::Tensor>& zscale,
               const c10::optional<at::Tensor>& xkept,
               const c10::optional<at::Tensor>& xscale, const at::Tensor& w,
               const c10::optional<at::Tensor>& mask, bool want_dx,
               c10::optional<at::ScalarType> dw_type,
               c10::optional<at::ScalarType> db_type) {
  TORCH_CHECK(dy_in.is_cuda() && dy_in.dim() == 2 && w.dim() == 2 &&
                  is16(w.scalar_type()) && dy_in.device() == w.device() &&
                  (xkept.has_value() || !dw_type.has_value()),
              "linear_act_bwd: dy (M,N), x (M,K) and w (N,K) on a GPU");
  int64_t M = dy_in.size(0), N = dy_in.size(1), K = w.size(1);
  auto st = w.scalar_type();
  TORCH_CHECK(w.size(0) == N && M > 0 && N > 0 && K > 0,
              "linear_act_bwd: shapes differ from the forward pass");
  TORCH_CHECK(dy_in.scalar_type() == st || dy_in.scalar_type() == at::kFloat,
              "linear_act_bwd: dy in w's type or float32");
  check_size(M, N, K);
  c10::DeviceGuard guard(w.device());
  auto dy = dy_in.contiguous();
  bool g32 = dy.scalar_type() == at::kFloat;
  int64_t ldz = (N + 7) / 8 * 8;
  auto opt = w.options();
  // dy is dz itself where nothing has to be done to it
  bool same = !z.has_value() && !g32 && N == ldz &&
              reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16 == 0;
  bool products = want_dx || dw_type.has_value();
  at::Tensor dz = same ? dy : at::empty({products ? M : 0, ldz}, opt), part;
  c10::optional<at::Tensor> dx, dw, db;
  // w along the sum: turned over first where the product is long enough to win
  // it back (50432 x 1536 -> 384 in 128 x 128: 95 us and 5 for the turn, 111
  // across; 25216 x 4096 -> 1024: 214 and 6, 282 across)
  Mm in{};
  in.M = (int)M;
  in.N = (int)K;
  in.K = (int)N;
  bool long_in = want_dx && tiles_of(in, 64, 64) > 600, turned = long_in;
  at::Tensor ws, wt;
  Turn turn{};
  if (long_in) {
    ws = K <= 1 || w.stride(1) == 1 ? w : w.contiguous();
    wt = at::empty({K, ldz}, opt);
    turn = {ws.data_ptr(), wt.data_ptr(), ws.stride(0), (int)N, (int)K,
            (int)ldz};
  }
  Join end{};
  if ((!same && products) || db_type.has_value()) {
    Dz d{};
    d.dy = dy.data_ptr();
    if (z.has_value()) {
      TORCH_CHECK(z->sizes() == dy.sizes() && z->is_contiguous() &&
                      z->device() == w.device() &&
                      (zscale.has_value()
                           ? z->scalar_type() == at::kFloat8_e4m3fn &&
                                 zscale->is_contiguous() &&
                                 zscale->device() == w.device() &&
                                 zscale->numel() == M * ((N + 31) / 32)
                           : z->scalar_type() == st),
                  "linear_act_bwd: kept pre-activation not of the forward "
                  "pass");
      d.z = z->data_ptr();
      if (zscale.has_value()) d.zscale = (const uint8_t*)zscale->data_ptr();
    }
    if (!same && products) d.dz = dz.data_ptr();
    d.M = M;
    d.N = (int)N;
    d.ldz = (int)ldz;
    bool wide = N > 64;
    int ct = wide ? 32 : 8, rl = kBlock / ct;
    int strips = (int)((N + ct * 8 - 1) / (ct * 8));
    int gy = (int)std::min<int64_t>((M + rl - 1) / rl,
                                    std::max(1, 1536 / strips));
    if (db_type.has_value()) {
      part = at::empty({gy, N}, opt.dtype(at::kFloat));
      d.part = part.data_ptr<float>();
    }
    d.rows = gy;
    if (turned) d.turn = turn;
    int64_t more = turned ? (turn_tiles(turn) + strips - 1) / strips : 0;
    turned = more > 0 && gy + more < 65536;
    by16(st, [&](auto t) {
      using T = decltype(t);
      dim3 grid(strips, (unsigned)(gy + (turned ? more : 0)));
      auto s = current();
      if (wide && g32)
        dz_kernel<T, float, 32><<<grid, kBlock, 0, s>>>(d);
      else if (wide)
        dz_kernel<T, T, 32><<<grid, kBlock, 0, s>>>(d);
      else if (g32)
        dz_kernel<T, float, 8><<<grid, kBlock, 0, s>>>(d);
      else
        dz_kernel<T, T, 8><<<grid, kBlock, 0, s>>>(d);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    });
    if (db_type.has_value()) {
      db = at::empty({N}, opt.dtype(*db_type));
      end.colpart = d.part;
      end.colout = db->data_ptr();
      end.rows = gy;
      end.C = (int)N;
      end.coltype = *db_type == at::kFloat ? 0 : *db_type == at::kBFloat16 ? 1
                                                                          : 2;
    }
  } else {
    turned = false;
  }
  if (want_dx) {
    dx = at::empty({M, K}, opt);
    in.q = (const char*)dz.data_ptr();
    in.ldq = ldz * 2;
    in.nq = (int)M;
    in.e.out = dx->data_ptr();
    if (long_in) {
      in.p = (const char*)wt.data_ptr();
      in.ldp = ldz * 2;
      in.np = (int)K;
      by16(st, [&](auto t) {
        using T = decltype(t);
        if (!turned) {
          turn_kernel<T><<<grid_of(turn_tiles(turn), kBlock), kBlock, 0,
                           current()>>>(turn);
          C10_HIP_KERNEL_LAUNCH_CHECK();
        }
        run_rows<T, kNoAct>(in);
      });
    } else {
      auto wl = loadable(w);
      in.p = (const char*)wl.data_ptr();
      in.ldp = row_bytes(wl);
      in.np = (int)wl.size(1);
      by16(st, [&](auto t) {
        launch_mm<decltype(t), 64, 64, 64, 2, 2, kRowK, kColK, 2, 1,
                  kAfterFirst>(in);
      });
    }
  }
  at::Tensor part2, m;   // until the last launch
  if (dw_type.has_value()) {
    dw = at::empty({N, K}, opt.dtype(*dw_type));
    Mm a{};
    const at::Tensor& xk = *xkept;
    TORCH_CHECK(xk.dim() == 2 && xk.size(0) == M && xk.size(1) == K,
                "linear_act_bwd: kept input not of the forward pass");
    at::Tensor xl = xk;
    a.q = (const char*)dz.data_ptr();
    a.ldq = ldz * 2;
    a.nq = (int)ldz;
    a.M = (int)N;
    a.N = (int)K;
    a.K = (int)M;
    at::Tensor xs;
    if (xscale.has_value()) {
      TORCH_CHECK(xk.scalar_type() == at::kFloat8_e4m3fn &&
                      xscale->scalar_type() == at::kFloat8_e8m0fnu &&
                      xscale->dim() == 2 && xscale->size(0) == M &&
                      xscale->size(1) == (K + 31) / 32 &&
                      xk.device() == w.device() &&
                      xscale->device() == w.device(),
                  "linear_act_bwd: kept input not of the forward pass");
      xl = xk.contiguous();
      xs = xscale->contiguous();
      a.p = (const char*)xl.data_ptr();
      a.ldp = K;
      a.np = (int)K;
      a.pscale = (const uint8_t*)xs.data_ptr();
    } else {
      TORCH_CHECK(xk.scalar_type() == st && xk.device() == w.device(),
                  "linear_act_bwd: kept input not of the forward pass");
      xl = loadable(xk);
      a.p = (const char*)xl.data_ptr();
      a.ldp = row_bytes(xl);
      a.np = (int)xl.size(1);
    }
    if (mask.has_value()) {
      TORCH_CHECK(mask->numel() == N * K && mask->scalar_type() == at::kFloat,
                  "linear_act_bwd: float32 mask of w's shape");
      m = mask->contiguous();
    }
    Split split = split_of(a);
    int slabs = split.slabs;
    bool join = slabs > 1 || *dw_type != st;
    if (join) {
      part2 = at::empty({slabs, N, K}, opt.dtype(at::kFloat));
      a.e.out = part2.data_ptr();
      a.e.out_f32 = 1;
    } else {
      a.e.out = dw->data_ptr();
      if (m.defined()) a.e.mask = m.data_ptr<float>();
    }
    by16(st, [&](auto t) {
      using T = decltype(t);
      if (xscale.has_value())
        run_cols<T, kCodes>(a, split);
      else
        run_cols<T, kColK>(a, split);
    });
    if (join) {
      end.part = part2.data_ptr<float>();
      end.mask = m.defined() ? m.data_ptr<float>() : nullptr;
      end.out = dw->data_ptr();
      end.n = N * K;
      end.slabs = slabs;
    }
  }
  if (end.n || end.C) {
    unsigned grid = grid_of(
        (end.n + kBlock * 8 - 1) / (kBlock * 8) + (end.C + 15) / 16, kBlock);
    auto s = current();
    if (!end.n || *dw_type == at::kFloat)
      join_kernel<float><<<grid, kBlock, 0, s>>>(end);
    else
      by16(*dw_type, [&](auto t) {
        join_kernel<decltype(t)><<<grid, kBlock, 0, s>>>(end);
      });
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {dx, dw, db};
}

}  // namespace turboprune
