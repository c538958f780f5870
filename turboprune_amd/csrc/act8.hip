// Activations kept in 8 bits: conversion to and from the format of act8.h,
// and exact GELU whose input is kept that way for the backward pass.
//
// All four kernels are bound by memory (per element of a 16-bit tensor:
// quantise 2 + 1.03 B, dequantise 1.03 + 2, GELU forward 2 + 2 + 1.03,
// backward 1.03 + 2 + 2). A thread takes chunks of 8 neighbouring values,
// one 16-byte load each, and the 4 lanes that share a scale sit in one quad,
// so a block's largest magnitude is two quad permutes away and no LDS or
// barrier is needed. Each thread has two chunks in flight.
//
// 50432 x 1536 bf16: quantise 41 us (5.7 TB/s), GELU forward 64 (6.1), backward
// 76 (5.1); dequantise 50432 x 768 20 us (5.9). A copy of 2 GiB runs at 4.9.

#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>

#include "act8.h"

namespace turboprune {

using namespace act8;

namespace {

constexpr int kPer = 2;   // chunks in flight per thread

// Chunk q of the launch: row q / cpr, columns from 8 (q mod cpr). cpr is
// rounded up to whole blocks, so a quad never straddles two rows. Where C is
// a multiple of 32 (FLAT) rows need not be told apart.
struct At {
  int64_t off, blk;   // element and scale offsets
  int n;              // values of this chunk that exist
};
template <bool FLAT>
TP_DEVICE At at(uint32_t q, uint32_t cpr, int C) {
  if constexpr (FLAT) {
    return {(int64_t)q * 8, (int64_t)(q >> 2), 8};
  } else {
    uint32_t row = q / cpr, c = q - row * cpr;
    return {(int64_t)row * C + c * 8, (int64_t)row * (cpr >> 2) + (c >> 2),
            C - (int)c * 8};
  }
}

// what a kernel does between load and store
enum { kQuant = 0, kGelu = 1 };

template <typename T, int OP, bool FLAT>
__global__ __launch_bounds__(kBlock) void keep_kernel(
    const T* __restrict__ x, T* __restrict__ y, uint8_t* __restrict__ codes,
    uint8_t* __restrict__ scales, uint32_t chunks, uint32_t cpr, int C) {
  uint32_t q0 = blockIdx.x * (kBlock * kPer) + threadIdx.x;
  float v[kPer][8];
  At a[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    uint32_t q = q0 + u * kBlock;
    a[u] = at<FLAT>(q, cpr, C);
    if (q >= chunks) a[u].n = 0;
    load8n(x + a[u].off, a[u].n, v[u]);
  }
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    int e, n = a[u].n;
    uint2 c = encode8(v[u], e, QuadMax());
    if (n <= 0) continue;
    store_codes(codes + a[u].off, n, c);
    if ((threadIdx.x & 3) == 0) scales[a[u].blk] = (uint8_t)(e + 127);
    if constexpr (OP == kGelu) {
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = gelu(v[u][i]);
      store8n(y + a[u].off, n, o);
    }
  }
}

template <typename T, int OP, bool FLAT>
__global__ __launch_bounds__(kBlock) void use_kernel(
    const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
    const T* __restrict__ dy, T* __restrict__ out, uint32_t chunks,
    uint32_t cpr, int C) {
  uint32_t q0 = blockIdx.x * (kBlock * kPer) + threadIdx.x;
  uint2 c[kPer];
  float g[kPer][8], s[kPer];
  At a[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    uint32_t q = q0 + u * kBlock;
    a[u] = at<FLAT>(q, cpr, C);
    if (q >= chunks) a[u].n = 0;
    c[u] = load_codes(codes + a[u].off, a[u].n);
    s[u] = a[u].n > 0 ? pow2((int)scales[a[u].blk] - 127) : 0.f;
    if constexpr (OP == kGelu) load8n(dy + a[u].off, a[u].n, g[u]);
  }
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    if (a[u].n <= 0) continue;
    float v[8];
    decode8(c[u], s[u], v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (OP == kGelu)
        v[i] = g[u][i] * gelu_slope(v[i]);
      else
        v[i] = held_in<T>(v[i]);
    }
    store8n(out + a[u].off, a[u].n, v);
  }
}

int64_t blocks_of(int64_t C) { return (C + kBlk - 1) / kBlk; }

// launches over slabs of rows, so that chunk numbers fit 32 bits
template <typename F>
void over_slabs(int64_t rows, int64_t C, F&& launch) {
  uint32_t cpr = (uint32_t)(4 * blocks_of(C));
  int64_t most = std::max<int64_t>(1, (int64_t(1) << 30) / cpr);
  for (int64_t r = 0; r < rows; r += most) {
    int64_t n = std::min(most, rows - r);
    uint32_t chunks = (uint32_t)(n * cpr);
    launch(r * C, r * blocks_of(C), chunks, cpr,
           (chunks + kBlock * kPer - 1) / (kBlock * kPer));
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
}

void check_cols(int64_t C) {
  TORCH_CHECK(C <= (int64_t(1) << 30), "act8: rows of at most 2^30 values");
}

template <typename T, int OP>
void run_keep(const at::Tensor& x, at::Tensor* y, at::Tensor& codes,
              at::Tensor& scales) {
  int64_t C = x.size(-1), rows = x.numel() / C;
  auto stream = at::hip::getCurrentHIPStream();
  auto* xp = reinterpret_cast<const T*>(x.data_ptr());
  auto* yp = y ? reinterpret_cast<T*>(y->data_ptr()) : nullptr;
  auto* cp = reinterpret_cast<uint8_t*>(codes.data_ptr());
  auto* sp = reinterpret_cast<uint8_t*>(scales.data_ptr());
  over_slabs(rows, C, [&](int64_t o, int64_t b, uint32_t chunks,
                          uint32_t cpr, uint32_t grid) {
    if (C % kBlk == 0)
      keep_kernel<T, OP, true><<<grid, kBlock, 0, stream>>>(
          xp + o, yp ? yp + o : yp, cp + o, sp + b, chunks, cpr, (int)C);
    else
      keep_kernel<T, OP, false><<<grid, kBlock, 0, stream>>>(
          xp + o, yp ? yp + o : yp, cp + o, sp + b, chunks, cpr, (int)C);
  });
}

template <typename T, int OP>
void run_use(const at::Tensor& codes, const at::Tensor& scales,
             const at::Tensor* dy, at::Tensor& out) {
  int64_t C = codes.size(-1), rows = codes.numel() / C;
  auto stream = at::hip::getCurrentHIPStream();
  auto* cp = reinterpret_cast<const uint8_t*>(codes.data_ptr());
  auto* sp = reinterpret_cast<const uint8_t*>(scales.data_ptr());
  auto* gp = dy ? reinterpret_cast<const T*>(dy->data_ptr()) : nullptr;
  auto* op = reinterpret_cast<T*>(out.data_ptr());
  over_slabs(rows, C, [&](int64_t o, int64_t b, uint32_t chunks,
                          uint32_t cpr, uint32_t grid) {
    if (C % kBlk == 0)
      use_kernel<T, OP, true><<<grid, kBlock, 0, stream>>>(
          cp + o, sp + b, gp ? gp + o : gp, op + o, chunks, cpr, (int)C);
    else
      use_kernel<T, OP, false><<<grid, kBlock, 0, stream>>>(
          cp + o, sp + b, gp ? gp + o : gp, op + o, chunks, cpr, (int)C);
  });
}

#define TP_BY_TYPE(st, what, ...)                                         \
  [&] {                                                                   \
    if ((st) == at::kBFloat16) {                                          \
      using T = __hip_bfloat16;                                           \
      __VA_ARGS__;                                                        \
    } else if ((st) == at::kHalf) {                                       \
      using T = _Float16;                                                 \
      __VA_ARGS__;                                                        \
    } else if ((st) == at::kFloat) {                                      \
      using T = float;                                                    \
      __VA_ARGS__;                                                        \
    } else {                                                              \
      TORCH_CHECK(false, what ": float32, bfloat16 or float16, not ", st); \
    }                                                                     \
  }()

void check_kept(const at::Tensor& codes, const at::Tensor& scales) {
  TORCH_CHECK(codes.is_cuda() && scales.is_cuda() &&
                  codes.device() == scales.device(),
              "act8: codes and scales on one GPU");
  TORCH_CHECK(codes.scalar_type() == at::kFloat8_e4m3fn &&
                  scales.scalar_type() == at::kFloat8_e8m0fnu,
              "act8: float8_e4m3fn codes and float8_e8m0fnu scales");
  TORCH_CHECK(codes.dim() >= 1 && codes.dim() == scales.dim(),
              "act8: codes and scales of the same rows");
  for (int64_t i = 0; i + 1 < codes.dim(); ++i)
    TORCH_CHECK(codes.size(i) == scales.size(i),
                "act8: codes and scales of the same rows");
  TORCH_CHECK(scales.size(-1) == blocks_of(codes.size(-1)),
              "act8: one scale for every ", kBlk, " values of a row");
}

}  // namespace

// (codes, scales) for a tensor of x's shape; shared with the kernels that
// write the format themselves
std::pair<at::Tensor, at::Tensor> act8_empty(at::IntArrayRef sizes,
                                             const at::TensorOptions& o) {
  auto s = sizes.vec();
  auto codes = at::empty(s, o.dtype(at::kFloat8_e4m3fn));
  s.back() = blocks_of(s.back());
  return {codes, at::empty(s, o.dtype(at::kFloat8_e8m0fnu))};
}

std::tuple<at::Tensor, at::Tensor> act8_quantize(const at::Tensor& x_in) {
  TORCH_CHECK(x_in.is_cuda() && x_in.dim() >= 1,
              "act8_quantize: a GPU tensor of at least one dimension");
  check_cols(x_in.size(-1));
  c10::DeviceGuard guard(x_in.device());
  auto x = x_in.contiguous();
  auto kept = act8_empty(x.sizes(), x.options());
  TP_BY_TYPE(x.scalar_type(), "act8_quantize", {
    if (x.numel()) run_keep<T, kQuant>(x, nullptr, kept.first, kept.second);
  });
  return {kept.first, kept.second};
}

at::Tensor act8_dequantize(const at::Tensor& codes_in,
                           const at::Tensor& scales_in,
                           at::ScalarType dtype) {
  check_kept(codes_in, scales_in);
  check_cols(codes_in.size(-1));
  c10::DeviceGuard guard(codes_in.device());
  auto codes = codes_in.contiguous(), scales = scales_in.contiguous();
  auto out = at::empty(codes.sizes(), codes.options().dtype(dtype));
  TP_BY_TYPE(dtype, "act8_dequantize", {
    if (out.numel()) run_use<T, kQuant>(codes, scales, nullptr, out);
  });
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> gelu_keep8_fwd(
    const at::Tensor& x_in) {
  TORCH_CHECK(x_in.is_cuda() && x_in.dim() >= 1,
              "gelu_keep8_fwd: a GPU tensor of at least one dimension");
  check_cols(x_in.size(-1));
  c10::DeviceGuard guard(x_in.device());
  auto x = x_in.contiguous();
  auto y = at::empty_like(x);
  auto kept = act8_empty(x.sizes(), x.options());
  TP_BY_TYPE(x.scalar_type(), "gelu_keep8_fwd", {
    if (x.numel()) run_keep<T, kGelu>(x, &y, kept.first, kept.second);
  });
  return {y, kept.first, kept.second};
}

at::Tensor gelu_keep8_bwd(const at::Tensor& codes_in,
                          const at::Tensor& scales_in,
                          const at::Tensor& dy_in) {
  check_kept(codes_in, scales_in);
  check_cols(codes_in.size(-1));
  TORCH_CHECK(dy_in.device() == codes_in.device() &&
                  dy_in.sizes() == codes_in.sizes(),
              "gelu_keep8_bwd: dy and the kept input differ in shape or "
              "device");
  c10::DeviceGuard guard(codes_in.device());
  auto codes = codes_in.contiguous(), scales = scales_in.contiguous();
  auto dy = dy_in.contiguous();
  auto dx = at::empty_like(dy);
  TP_BY_TYPE(dy.scalar_type(), "gelu_keep8_bwd", {
    if (dy.numel()) run_use<T, kGelu>(codes, scales, &dy, dx);
  });
  return dx;
}

}  // namespace turboprune
