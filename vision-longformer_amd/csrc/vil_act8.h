// vil_act8.h -- the 8-bit form of activations and the GELU around it, as device functions: vil_act8.hip's kernels and the epilogues of
// the MLP block's products (vil_gemm_fused.hip) share them.
//
// Form.  32 neighbouring channels of a row share a power of two 2^e, the smallest with max |x| <= 127 * 2^e; a value is held
// as the integer c = round(x / 2^e), ties to even, |c| <= 127, and stands for c * 2^e.  One byte holds e + 127 (>= 1), so a
// value costs 1 + 1/32 bytes.  With a power of two, x / 2^e and c * 2^e are exact: the rounding to the integer is the only one, at
// most 2^e / 2, i.e. max|x| / 127 in the worst block (max|x| just over 127 * 2^(e-1)) and half of that in the best.  Against
// a 4-bit significand (relative half step 2^-4 for every value) that is 8 to 16 times closer for the large values, which
// carry the gradient.  A value of the topmost block (e = 10 in fp16, 122 otherwise) that would round past the type's largest
// finite number is held as 63, the largest code that stays finite.  A block that holds an infinity or a NaN is marked by the
// byte 255 and comes back as NaN throughout: an overflow stays visible to a gradient scaler.
//
// GELU.  a = x Phi(x), a' = Phi(x) + x phi(x).  Phi(-|x|) = erfcx(z) exp(-z^2) / 2 with z = |x| / sqrt 2, and erfcx(z) as a polynomial
// in t = 1 / (1 + p z), fitted to the least maximum of the RELATIVE error over z in [0, 10]: the negative tail keeps its
// digits, which 1 - erf would cancel.  Six terms: 5.2e-6, against a half step of 2^-11 (fp16) and 2^-9 (bf16); eight terms for
// fp32: 9e-8, 4e-7 with the rounding of the evaluation.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

static constexpr int A8_BLOCK = 32;

__device__ __forceinline__ float a8_pow2(int biased) { return __int_as_float(biased << 23); }

// biased exponent (e + 127) of a block from the bits of its largest |x|; 255 for an infinity or a NaN.  max|x| = m 2^E with m in
// [1, 2): e = E - 6 for m <= 127/64 (mantissa <= 0x7e0000), E - 5 above; at least 1, so that 2^e is no subnormal.
__device__ __forceinline__ int a8_exponent(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255;
  const int e = (int)((amax + 0x1ffffu) >> 23) - 6;
  return e < 1 ? 1 : e;
}
// the exponent whose code 64 would be past the largest finite number of T
template <typename T> struct A8Top { static constexpr int biased = 127 + 122; };
template <> struct A8Top<_Float16> { static constexpr int biased = 127 + 10; };
// 1 / 2^e of a biased exponent in [1, 249]
__device__ __forceinline__ float a8_inverse(int biased) { return a8_pow2(254 - biased); }

// Phi(-|x|) = hx s^2 and phi(x) = s^2 / sqrt(2 pi) with s = exp(-x^2 / 4): one factor s at a time, so that results keep their
// digits down to the smallest numbers (the hardware's exponential has no subnormal results).
template <bool F32>
__device__ __forceinline__ void a8_gelu(float x, float& hx, float& s) {
  const float ax = fabsf(x), v = x * x;
  s = __builtin_amdgcn_exp2f(v * -0.36067376022224085f);
  float q, t;
  if (F32) {
    const float lost = v < 300.f ? fmaf(x, x, -v) : 0.f;               // x^2's rounding error, which the exponential magnifies
    s *= fmaf(lost, -0.25f, 1.0f);
    t = 1.0f / fmaf(ax, 0.23334523779156072f, 1.0f);
    q = fmaf(t, -0.06767178326845169f, 0.23011423647403717f);
    q = fmaf(q, t, -0.17556753754615784f);
    q = fmaf(q, t, 0.20424333214759827f);
    q = fmaf(q, t, 0.02361382730305195f);
    q = fmaf(q, t, 0.1006108820438385f);
    q = fmaf(q, t, 0.0914781466126442f);
    q = fmaf(q, t, 0.0931788906455040f);
  } else {
    t = __builtin_amdgcn_rcpf(fmaf(ax, 0.3111269837220809f, 1.0f));
    q = fmaf(t, -0.07305202633142471f, 0.17532400786876678f);
    q = fmaf(q, t, 0.02036788314580917f);
    q = fmaf(q, t, 0.13179205358028412f);
    q = fmaf(q, t, 0.12128501385450363f);
    q = fmaf(q, t, 0.12428048998117447f);
  }
  hx = q * t;
}
// x Phi(x)
__device__ __forceinline__ float a8_act(float x, float hx, float s) {
  const float w = x * s * hx;
  return x < 0.f ? w * s : fmaf(-w, s, x);
}
// g (Phi(x) + x phi(x)):  Phi(-|x|) - |x| phi(x) = s^2 (hx - |x| / sqrt(2 pi)) on the left, 1 - that on the right
__device__ __forceinline__ float a8_slope(float g, float x, float hx, float s) {
  const float u = g * s * fmaf(fabsf(x), -0.39894228040143268f, hx);
  return x < 0.f ? u * s : fmaf(-u, s, g);
}

// the bits of the largest |x| of a lane, as fp32 bits: the types' bits without the sign order as the magnitudes do, NaN last
template <typename T, typename A8V> __device__ __forceinline__ uint32_t a8_lane_max(const A8V& x) {
  if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
      m = b > m ? b : m;
    }
    return m;
  } else {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    const u4 w = __builtin_bit_cast(u4, x) & 0x7fff7fffu;
    const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3];             // (a bit cast of a vector's element reads its first)
    const us2 m = __builtin_elementwise_max(__builtin_elementwise_max(__builtin_bit_cast(us2, w0), __builtin_bit_cast(us2, w1)),
                                            __builtin_elementwise_max(__builtin_bit_cast(us2, w2), __builtin_bit_cast(us2, w3)));
    const unsigned short h = m[0] > m[1] ? m[0] : m[1];
    return __float_as_uint((float)__builtin_bit_cast(T, h));
  }
}

// codes of eight values of a block with biased exponent e
typedef unsigned a8_codes8 __attribute__((ext_vector_type(2)));
template <typename T> __device__ __forceinline__ a8_codes8 a8_encode(const float (&v)[8], int e) {
  const float inv = a8_inverse(e == 255 ? 1 : e);
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = __float_as_uint(fmaf(v[i], inv, 12582912.f));   // 1.5 * 2^23: the sum's last byte is the rounded integer
  if (e >= A8Top<T>::biased) {                                               // (rare: the type's largest numbers, or a marked block)
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = e == 255 ? 0u : (uint32_t)(int)fminf(fmaxf(rintf(v[i] * inv), -63.f), 63.f);
  }
  a8_codes8 o;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __builtin_amdgcn_perm(c[4 * i + 1], c[4 * i], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[4 * i + 3], c[4 * i + 2], 0x0c0c0400u);
    o[i] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
  return o;
}
__device__ __forceinline__ void a8_decode(a8_codes8 c, int e, float (&v)[8]) {
  const float step = e == 255 ? __uint_as_float(0x7fc00000u) : a8_pow2(e);
  const uint32_t c0 = c[0], c1 = c[1];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)(int)(int8_t)((i < 4 ? c0 : c1) >> (8 * (i % 4))) * step;
}
// gelu of eight values of a block with biased exponent e (an infinity, which only a marked block holds, is its own)
template <bool F32> __device__ __forceinline__ void a8_act8(const float (&v)[8], int e, float (&a)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float hx, s;
    a8_gelu<F32>(v[i], hx, s);
    a[i] = a8_act(v[i], hx, s);
  }
  if (e == 255)
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = v[i] == INFINITY ? v[i] : a[i];
}
