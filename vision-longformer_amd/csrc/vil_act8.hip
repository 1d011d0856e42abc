// vil_act8.hip -- activations held in 8 bits between the forward and the backward pass, and the exact GELU whose backward
// pass reads its pre-activation from there.
//
// Form.  32 neighbouring channels of a row share a power of two 2^e, the smallest with max |x| <= 127 * 2^e; a value is held
// as the integer c = round(x / 2^e), ties to even, |c| <= 127, and stands for c * 2^e.  One byte holds e + 127 (>= 1), so a
// value costs 1 + 1/32 bytes.  With a power of two, x / 2^e and c * 2^e are exact: the rounding to the integer is the only one, at
// most 2^e / 2, i.e. max|x| / 127 in the worst block (max|x| just over 127 * 2^(e-1)) and half of that in the best.  Against
// a 4-bit significand (relative half step 2^-4 for every value) that is 8 to 16 times closer for the large values, which
// carry the gradient.  A value of the topmost block (e = 10 in fp16, 122 otherwise) that would round past the type's largest
// finite number is held as 63, the largest code that stays finite.  A block that holds an infinity or a NaN is marked by the byte 255 and comes back as NaN throughout: an
// overflow stays visible to a gradient scaler.
//
// GELU.  a = x Phi(x), a' = Phi(x) + x phi(x).  Phi(-|x|) = erfcx(z) exp(-z^2) / 2 with z = |x| / sqrt 2, and erfcx(z) as a polynomial
// in t = 1 / (1 + p z), fitted to the least maximum of the RELATIVE error over z in [0, 10]: the negative tail keeps its
// digits, which 1 - erf would cancel.  Six terms: 5.2e-6, against a half step of 2^-11 (fp16) and 2^-9 (bf16); eight terms for
// fp32: 9e-8, 4e-7 with the rounding of the evaluation.
#include "vil_internal.h"

namespace {

constexpr int A8_BLOCK = 32;

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

// One block of 32 channels to 32 lanes, one value to a lane.  GELU: a = gelu(x) beside the packed x.
template <typename T, bool GELU>
__global__ __launch_bounds__(256) void k_act8_pack(const T* x, int64_t x_rs, int64_t rows, int cols, T* a, int8_t* codes, uint8_t* scales) {
  const int nb = (cols + A8_BLOCK - 1) / A8_BLOCK;
  const int64_t blk = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t row = blk / nb;
  const int ib = (int)(blk - row * nb), c = ib * A8_BLOCK + (threadIdx.x & 31);
  const bool ok = row < rows && c < cols;
  const float v = ok ? (float)x[row * x_rs + c] : 0.f;
  uint32_t m = __float_as_uint(v) & 0x7fffffffu;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint32_t other = __shfl_xor(m, o, 32);
    m = other > m ? other : m;
  }
  const int e = a8_exponent(m);
  if (!ok) return;
  float r = e == 255 ? 0.f : rintf(v * a8_inverse(e));
  if (e == A8Top<T>::biased) r = fminf(fmaxf(r, -63.f), 63.f);
  codes[row * cols + c] = (int8_t)(int)r;
  if ((threadIdx.x & 31) == 0) scales[blk] = (uint8_t)e;
  if (GELU) {
    float hx, s;
    a8_gelu<sizeof(T) == 4>(v, hx, s);
    a[row * cols + c] = (T)(v == INFINITY ? v : a8_act(v, hx, s));
  }
}

// values from codes; GELU: dh = da * gelu'(value) and, where `a` is wanted, gelu(value)
template <typename T, bool GELU>
__global__ __launch_bounds__(256) void k_act8_unpack(const int8_t* codes, const uint8_t* scales, const T* da, int64_t da_rs,
                                                     int64_t rows, int cols, T* out, T* a) {
  const int nb = (cols + A8_BLOCK - 1) / A8_BLOCK;
  const int64_t blk = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t row = blk / nb;
  const int ib = (int)(blk - row * nb), c = ib * A8_BLOCK + (threadIdx.x & 31);
  if (row >= rows || c >= cols) return;
  const int e = scales[blk];
  const float v = e == 255 ? __uint_as_float(0x7fc00000u) : (float)codes[row * cols + c] * a8_pow2(e);
  if (!GELU) { out[row * cols + c] = (T)v; return; }
  float hx, s;
  a8_gelu<sizeof(T) == 4>(v, hx, s);
  out[row * cols + c] = (T)a8_slope((float)da[row * da_rs + c], v, hx, s);
  if (a) a[row * cols + c] = (T)a8_act(v, hx, s);
}

int a8_check(int dtype, int64_t rows, int cols, int64_t rs) {
  if (dtype != VIL_DTYPE_F32 && dtype != VIL_DTYPE_BF16 && dtype != VIL_DTYPE_F16) return VIL_E_DTYPE;
  if (rows < 0 || cols < 0 || (rows > 1 && rs < cols)) return VIL_E_SHAPE;
  // (one workgroup to 256 values at the most: the grid's first axis holds 2^31 - 1)
  if (cols > 0 && rows > ((int64_t)1 << 37) / cols) return VIL_E_SHAPE;
  return VIL_OK;
}
unsigned a8_grid(int64_t rows, int cols) { return (unsigned)((rows * ((cols + A8_BLOCK - 1) / A8_BLOCK) + 7) / 8); }

template <bool GELU>
int a8_pack(const void* x, int dtype, int64_t rows, int cols, int64_t rs, void* a, void* codes, void* scales, hipStream_t s) {
  const dim3 grid(a8_grid(rows, cols)), block(256);
  if (dtype == VIL_DTYPE_F32) k_act8_pack<float, GELU><<<grid, block, 0, s>>>((const float*)x, rs, rows, cols, (float*)a, (int8_t*)codes, (uint8_t*)scales);
  else if (dtype == VIL_DTYPE_BF16) k_act8_pack<__bf16, GELU><<<grid, block, 0, s>>>((const __bf16*)x, rs, rows, cols, (__bf16*)a, (int8_t*)codes, (uint8_t*)scales);
  else k_act8_pack<_Float16, GELU><<<grid, block, 0, s>>>((const _Float16*)x, rs, rows, cols, (_Float16*)a, (int8_t*)codes, (uint8_t*)scales);
  return (int)hipGetLastError();
}

template <bool GELU>
int a8_unpack(const void* codes, const void* scales, const void* da, int64_t da_rs, int dtype, int64_t rows, int cols, void* out,
              void* a, hipStream_t s) {
  const dim3 grid(a8_grid(rows, cols)), block(256);
  const int8_t* c = (const int8_t*)codes;
  const uint8_t* e = (const uint8_t*)scales;
  if (dtype == VIL_DTYPE_F32) k_act8_unpack<float, GELU><<<grid, block, 0, s>>>(c, e, (const float*)da, da_rs, rows, cols, (float*)out, (float*)a);
  else if (dtype == VIL_DTYPE_BF16) k_act8_unpack<__bf16, GELU><<<grid, block, 0, s>>>(c, e, (const __bf16*)da, da_rs, rows, cols, (__bf16*)out, (__bf16*)a);
  else k_act8_unpack<_Float16, GELU><<<grid, block, 0, s>>>(c, e, (const _Float16*)da, da_rs, rows, cols, (_Float16*)out, (_Float16*)a);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" int vil_act8_pack(const void* x, int dtype, int64_t rows, int cols, int64_t x_row_stride, void* codes, void* scales,
                             void* stream) {
  if (int e = a8_check(dtype, rows, cols, x_row_stride)) return e;
  if (rows == 0 || cols == 0) return VIL_OK;
  if (!x || !codes || !scales) return VIL_E_NULL;
  return a8_pack<false>(x, dtype, rows, cols, x_row_stride, nullptr, codes, scales, (hipStream_t)stream);
}

extern "C" int vil_act8_unpack(const void* codes, const void* scales, int64_t rows, int cols, void* y, int dtype, void* stream) {
  if (int e = a8_check(dtype, rows, cols, cols)) return e;
  if (rows == 0 || cols == 0) return VIL_OK;
  if (!codes || !scales || !y) return VIL_E_NULL;
  return a8_unpack<false>(codes, scales, nullptr, 0, dtype, rows, cols, y, nullptr, (hipStream_t)stream);
}

extern "C" int vil_gelu_act8_fwd(const void* h, int dtype, int64_t rows, int cols, int64_t h_row_stride, void* a, void* codes,
                                 void* scales, void* stream) {
  if (int e = a8_check(dtype, rows, cols, h_row_stride)) return e;
  if (rows == 0 || cols == 0) return VIL_OK;
  if (!h || !a || !codes || !scales) return VIL_E_NULL;
  return a8_pack<true>(h, dtype, rows, cols, h_row_stride, a, codes, scales, (hipStream_t)stream);
}

extern "C" int vil_gelu_act8_bwd(const void* codes, const void* scales, const void* da, int dtype, int64_t rows, int cols,
                                 int64_t da_row_stride, void* dh, void* a, void* stream) {
  if (int e = a8_check(dtype, rows, cols, da_row_stride)) return e;
  if (rows == 0 || cols == 0) return VIL_OK;
  if (!codes || !scales || !da || !dh) return VIL_E_NULL;
  return a8_unpack<true>(codes, scales, da, da_row_stride, dtype, rows, cols, dh, a, (hipStream_t)stream);
}
