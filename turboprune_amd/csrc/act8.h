// The 8-bit format of kept activations, and the vector helpers of the
// kernels that read and write it.
//
// A row of C values is cut into blocks of 32. A block holds one power of
// two 2^e (e8m0: the byte is e + 127) and 32 e4m3 codes; a code c stands
// for c * 2^e. e is the smallest for which the block's largest finite
// magnitude is at most 448 * 2^e, within [-126, 126], so nothing
// saturates (but for the last 6 % below the largest float, whose rounding up
// would be infinite) and 2^e and 2^-e are both normal floats. NaN and infinities
// take the code NaN (e4m3 has no infinity) and do not raise e, so one bad
// value does not cost its neighbours their precision.
//
// Why this format: a code has 4 significant bits and the scale is a power
// of two, so c * 2^e is exact in bf16 (and in fp16 within its range) and
// matrix instructions on 16-bit operands lose nothing more.
#pragma once

#include "common.h"

namespace turboprune {
namespace act8 {

constexpr int kBlk = 32;

typedef __attribute__((ext_vector_type(2))) float f32x2v;

// Rows of any length start at any address that their type allows; the
// memory pipe takes wide accesses at such addresses, so these types only
// tell the compiler not to assume more.
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef u32x4 __attribute__((aligned(4))) u32x4_a4;
typedef u32x4 __attribute__((aligned(2))) u32x4_a2;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef u32x2 __attribute__((aligned(1))) u32x2_a1;

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2v;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2v;

// ---- one 8-element chunk of a row in registers ---------------------------
template <typename T>
TP_DEVICE void load8(const T* p, float (&v)[8]);
template <>
TP_DEVICE void load8<float>(const float* p, float (&v)[8]) {
  u32x4 a = *reinterpret_cast<const u32x4_a4*>(p);
  u32x4 b = *reinterpret_cast<const u32x4_a4*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = __uint_as_float(a[i]);
    v[i + 4] = __uint_as_float(b[i]);
  }
}
template <typename T>
TP_DEVICE void unpack8(u32x4 d, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (__is_same(T, _Float16)) {
      f16x2v e = __builtin_bit_cast(f16x2v, (uint32_t)d[i]);
      v[2 * i] = (float)e[0];
      v[2 * i + 1] = (float)e[1];
    } else {
      v[2 * i] = __uint_as_float(d[i] << 16);
      v[2 * i + 1] = __uint_as_float(d[i] & 0xffff0000u);
    }
  }
}
template <>
TP_DEVICE void load8<__hip_bfloat16>(const __hip_bfloat16* p, float (&v)[8]) {
  unpack8<__hip_bfloat16>(*reinterpret_cast<const u32x4_a2*>(p), v);
}
template <>
TP_DEVICE void load8<_Float16>(const _Float16* p, float (&v)[8]) {
  unpack8<_Float16>(*reinterpret_cast<const u32x4_a2*>(p), v);
}

// two floats to two packed 16-bit values, each rounded to nearest even
template <typename T>
TP_DEVICE uint32_t pack2(float a, float b);
template <>
TP_DEVICE uint32_t pack2<__hip_bfloat16>(float a, float b) {
  bf16x2v r;
  r[0] = (__bf16)a;
  r[1] = (__bf16)b;
  return __builtin_bit_cast(uint32_t, r);
}
template <>
TP_DEVICE uint32_t pack2<_Float16>(float a, float b) {
  f16x2v r;
  r[0] = (_Float16)a;
  r[1] = (_Float16)b;
  return __builtin_bit_cast(uint32_t, r);
}

template <typename T>
TP_DEVICE void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    u32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = __float_as_uint(v[i]);
      b[i] = __float_as_uint(v[i + 4]);
    }
    *reinterpret_cast<u32x4_a4*>(p) = a;
    *reinterpret_cast<u32x4_a4*>(p + 4) = b;
  } else {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<u32x4_a2*>(p) = r;
  }
}

// n of 8 values of a row (the last chunk of a row has fewer than 8; n <= 0
// for a lane behind it); the others read as zero and are not written
template <typename T>
TP_DEVICE void load8n(const T* p, int n, float (&v)[8]) {
  if (n >= 8) {
    load8(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_float<T>(p[i]) : 0.f;
  }
}
template <typename T>
TP_DEVICE void store8n(T* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    store8(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_float<T>(v[i]);
  }
}

// the value that is read back after a store as T
template <typename T>
TP_DEVICE float rounded(float v) { return to_float<T>(from_float<T>(v)); }
template <>
TP_DEVICE float rounded<float>(float v) { return v; }

// ---- scale and codes -----------------------------------------------------
// largest over the 4 lanes that hold one block (lanes 4k .. 4k+3)
struct QuadMax {
  TP_DEVICE float operator()(float v) const {
    int o = __builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xf, 0xf, true);
    v = fmaxf(v, __int_as_float(o));   // quad_perm [1,0,3,2]
    o = __builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xf, 0xf, true);
    return fmaxf(v, __int_as_float(o));   // quad_perm [2,3,0,1]
  }
};

// e of the block: amax = m 2^k gives k - 8, one more where m > 1.75
// (adding 0x1fffff carries into the exponent exactly then)
TP_DEVICE int block_exp(float amax) {
  int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 135;
  return max(-126, min(126, e));
}
TP_DEVICE float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

typedef __attribute__((ext_vector_type(2))) short s16x2v;

TP_DEVICE uint2 convert8(const float (&v)[8], float scale) {
  s16x2v lo = {0, 0}, hi = {0, 0};
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, v[0], v[1], scale, false);
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, v[2], v[3], scale, true);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, v[4], v[5], scale, false);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, v[6], v[7], scale, true);
  return make_uint2(__builtin_bit_cast(uint32_t, lo),
                    __builtin_bit_cast(uint32_t, hi));
}

// The codes of a lane's 8 values and its block's e; `over` takes a lane's
// number to the largest over the lanes of the block. The instructions do the
// whole of it (1.5 to a value) but for blocks with infinities, with nothing
// but NaN, or with magnitudes that 256 * 2^120, no finite float, would stand
// for: those take the second path, all lanes of a block together.
template <typename Over>
TP_DEVICE uint2 encode8(const float (&v)[8], int& e, Over over) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));   // passes NaN over
  m = over(m);
  if (m <= 3.1e38f) {
    e = block_exp(m);
    return convert8(v, pow2(e));
  }
  m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    m = fmaxf(m, fabsf(v[i]) <= 3.402823466e38f ? fabsf(v[i]) : 0.f);
  e = block_exp(over(m));
  float top = e < 120 ? 3.402823466e38f : 240.f * pow2(120), s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    s[i] = fabsf(v[i]) <= 3.402823466e38f
               ? __builtin_amdgcn_fmed3f(v[i], -top, top)
               : __uint_as_float(0x7fc00000u);
  return convert8(s, pow2(e));
}

TP_DEVICE void decode8(uint2 c, float scale, float (&v)[8]) {
  f32x2v a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.x, scale, false);
  f32x2v b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.x, scale, true);
  f32x2v d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.y, scale, false);
  f32x2v e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.y, scale, true);
  v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
  v[4] = d[0]; v[5] = d[1]; v[6] = e[0]; v[7] = e[1];
}

// a value (a code's, a sum) within T's finite range: in fp16 what is larger
// would round to infinity. NaN stays.
template <typename T>
TP_DEVICE float held_in(float v) {
  if constexpr (__is_same(T, _Float16))
    return fabsf(v) > 65504.f ? copysignf(65504.f, v) : v;
  else
    return v;
}

TP_DEVICE void store_codes(uint8_t* p, int n, uint2 c) {
  if (n >= 8) {
    u32x2 w = {c.x, c.y};
    *reinterpret_cast<u32x2_a1*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
  }
}
TP_DEVICE uint2 load_codes(const uint8_t* p, int n) {
  if (n >= 8) {
    u32x2 w = *reinterpret_cast<const u32x2_a1*>(p);
    return make_uint2(w[0], w[1]);
  }
  uint32_t x = 0, y = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) x |= (uint32_t)p[i] << (8 * i);
#pragma unroll
  for (int i = 4; i < 8; ++i)
    if (i < n) y |= (uint32_t)p[i] << (8 * (i - 4));
  return make_uint2(x, y);
}

// ---- GELU ------------------------------------------------------------------
// Phi(-t) = exp(-t^2/2) g(t) for t >= 0, with g(t) = u P(u), u = 1/(1+0.315t):
// g falls smoothly from 1/2 towards 1/(t sqrt(2 pi)), which u P(u) follows.
// P (degree 7, fitted here to the least largest relative error over [0, 40]
// with g(0) = 1/2 held, and that exactly in fp32) brings u P(u) within 6.7e-7
// of g, relative, and within 8.1e-7 as it is computed in fp32. The exponential
// adds the rounding of its argument, about 1e-7 t^2: the tail is off by
// (1.5e-6 + 1e-7 t^2) of itself at most. erff would be a two-sided branch of
// about twice the instructions, and this form shares its exponential with the
// density that the slope needs.
TP_DEVICE float normal_tail(float t, float e) {   // e = exp(-t^2/2)
  float u = __builtin_amdgcn_rcpf(fmaf(0.315f, t, 1.f));
  float p = 0.03447515890002251f;
  p = fmaf(p, u, -0.1291443556547165f);
  p = fmaf(p, u, 0.12537990510463715f);
  p = fmaf(p, u, 0.005099183414131403f);
  p = fmaf(p, u, 0.10150090605020523f);
  p = fmaf(p, u, 0.11120770126581192f);
  p = fmaf(p, u, 0.12581922113895416f);
  p = fmaf(p, u, 0.12566225230693817f);
  return e * (p * u);
}
TP_DEVICE float bell_exp(float z) {   // exp(-z^2/2) = 2^(-z^2 / (2 ln 2))
  return __builtin_amdgcn_exp2f(-0.72134752f * z * z);
}
TP_DEVICE float gelu(float z) {
  float q = normal_tail(fabsf(z), bell_exp(z));
  return z * (z < 0.f ? q : 1.f - q);
}
// The same for 16-bit results behind a product, where these instructions
// bound the epilogue: gelu(z) = max(z, 0) - t Phi(-t), t = |z|, with
// Phi(-t) = 2^-h(t), h a polynomial (fitted here over [0, 6.5] and exactly 1
// at 0): 14 instruction slots a value against 25. Off by 5e-6 of t Phi(-t) up
// to t = 4, by 5e-5 up to 6.5. Above 6.5 t stays there and the result within
// 3e-10 of z; it is not for z below -6.5, where the tail is all there is.
TP_DEVICE float gelu_short(float z) {
  float t = fminf(fabsf(z), 6.5f);
  float h = 1.7347767879982712e-06f;
  h = fmaf(h, t, -5.966168100712821e-05f);
  h = fmaf(h, t, 0.00091591477394104f);
  h = fmaf(h, t, -0.008453256450593472f);
  h = fmaf(h, t, 0.05385367572307587f);
  h = fmaf(h, t, 0.4585675299167633f);
  h = fmaf(h, t, 1.1512086391448975f);
  float q = __builtin_amdgcn_exp2f(-fmaf(h, t, 1.f));
  // this maximum is NaN where z is
  return fmaf(-t, q, __builtin_elementwise_maximum(z, 0.f));
}
TP_DEVICE float gelu_slope(float z) {
  float e = bell_exp(z);
  float q = normal_tail(fabsf(z), e);
  return fmaf(z * 0.39894228040143268f, e, z < 0.f ? q : 1.f - q);
}

}  // namespace act8
}  // namespace turboprune
