// vil_act8.hip -- activations held in 8 bits between the forward and the backward pass, and the exact GELU whose backward
// pass reads its pre-activation from there.
//
// The form and the mathematics: vil_act8.h.
//
// Bound: memory, the GELU nearly as much by vector instructions.  bf16, 401536 x 384, MI355X: GELU forward 134 us (775 MB, 5.8 TB/s;
// 103 us of it issue vector instructions), backward 189 us (1.08 GB, 5.7 TB/s; 121); pack + unpack of 100480 x 192 21 us (5.4 TB/s, partly
// from the last-level cache).  A large copy runs at 5.3 TB/s.
#include "vil_internal.h"
#include "vil_act8.h"

namespace {

// Eight neighbouring channels to a lane, four lanes to a block of 32: one 16-byte load of a 16-bit type, and a block's maximum in two
// register moves.  A workgroup takes A8_CHUNKS chunks of 256 lanes, all loads first.  FLAT: rows without gaps whose channels fill
// their blocks are one long row.  Otherwise a lane finds its row by a division; rows need no alignment (the memory system takes
// 16 bytes at any address of the type), and only a row's last lane goes value by value.
constexpr int A8_THREADS = 256, A8_CHUNKS = 2;
template <typename T> using a8_vec = T __attribute__((ext_vector_type(8), aligned(sizeof(T))));
template <typename T> using a8_vec16 = T __attribute__((ext_vector_type(8)));
typedef unsigned a8_codes __attribute__((ext_vector_type(2), aligned(1)));

struct A8At { int64_t row, blk; int c, n; };               // row, block, first channel, channels of this lane (0: none)
template <bool FLAT>
__device__ __forceinline__ A8At a8_at(int64_t lane, int64_t rows, int cols, int nb) {
  A8At w;
  w.blk = lane >> 2;
  if (FLAT) {                                              // (cols: of the one row; 64-bit offsets in `row`)
    w.row = lane * 8;
    w.c = 0;
    w.n = w.row < rows ? 8 : 0;                            // (rows: the number of values)
    return w;
  }
  w.row = (uint32_t)w.blk / (uint32_t)nb;                  // (blocks: under 2^31, a8_check)
  w.c = (int)(w.blk - w.row * nb) * A8_BLOCK + (int)(lane & 3) * 8;
  w.n = w.row < rows ? cols - w.c : 0;
  w.n = w.n < 0 ? 0 : w.n > 8 ? 8 : w.n;
  return w;
}

template <typename T, bool FLAT> __device__ __forceinline__ a8_vec16<T> a8_load(const T* p, int n) {
  if (FLAT) return n ? *(const a8_vec16<T>*)p : (a8_vec16<T>)(T)0;
  if (n == 8) return *(const a8_vec<T>*)p;
  a8_vec16<T> v = (a8_vec16<T>)(T)0;
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < n) v[i] = p[i];
  return v;
}
template <typename T, bool FLAT> __device__ __forceinline__ void a8_store(T* p, const float (&v)[8], int n) {
  a8_vec16<T> o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = (T)v[i];
  if (FLAT) { if (n) *(a8_vec16<T>*)p = o; return; }
  if (n == 8) { *(a8_vec<T>*)p = o; return; }
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < n) p[i] = o[i];
}

template <int CTRL> __device__ __forceinline__ uint32_t a8_quad(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
  return o > v ? o : v;
}

// GELU: a = gelu(x) beside the packed x
template <typename T, bool GELU, bool FLAT>
__global__ __launch_bounds__(A8_THREADS) void k_act8_pack(const T* x, int64_t x_rs, int64_t rows, int cols, int nb, T* a, int8_t* codes,
                                                           uint8_t* scales) {
  const int64_t lane0 = (int64_t)blockIdx.x * (A8_THREADS * A8_CHUNKS) + threadIdx.x;
  a8_vec16<T> in[A8_CHUNKS];
  A8At at[A8_CHUNKS];
#pragma unroll
  for (int k = 0; k < A8_CHUNKS; ++k) {
    at[k] = a8_at<FLAT>(lane0 + k * A8_THREADS, rows, cols, nb);
    in[k] = a8_load<T, FLAT>(x + (FLAT ? at[k].row : at[k].row * x_rs + at[k].c), at[k].n);
  }
#pragma unroll
  for (int k = 0; k < A8_CHUNKS; ++k) {
    const A8At& w = at[k];
    const int e = a8_exponent(a8_quad<0x4e>(a8_quad<0xb1>(a8_lane_max<T>(in[k]))));
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)in[k][i];
    const a8_codes8 o = a8_encode<T>(v, e);
    if (!w.n) continue;
    const int64_t to = FLAT ? w.row : w.row * cols + w.c;
    if (FLAT) *(a8_codes8*)(codes + to) = o;
    else if (w.n == 8) *(a8_codes*)(codes + to) = o;
    else
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < w.n) codes[to + i] = (int8_t)(o[i / 4] >> (8 * (i % 4)));
    if ((threadIdx.x & 3) == 0) scales[w.blk] = (uint8_t)e;
    if (GELU) {
      float r[8];
      a8_act8<sizeof(T) == 4>(v, e, r);
      a8_store<T, FLAT>(a + to, r, w.n);
    }
  }
}

// values from codes; GELU: dh = da * gelu'(value) and, where `a` is wanted, gelu(value)
template <typename T, bool GELU, bool FLAT>
__global__ __launch_bounds__(A8_THREADS) void k_act8_unpack(const int8_t* codes, const uint8_t* scales, const T* da, int64_t da_rs,
                                                            int64_t rows, int cols, int nb, T* out, T* a) {
  const int64_t lane0 = (int64_t)blockIdx.x * (A8_THREADS * A8_CHUNKS) + threadIdx.x;
  a8_codes8 in[A8_CHUNKS];
  a8_vec16<T> g[A8_CHUNKS];
  int e[A8_CHUNKS];
  A8At at[A8_CHUNKS];
#pragma unroll
  for (int k = 0; k < A8_CHUNKS; ++k) {
    const A8At w = at[k] = a8_at<FLAT>(lane0 + k * A8_THREADS, rows, cols, nb);
    const int8_t* from = codes + (FLAT ? w.row : w.row * cols + w.c);
    in[k] = (a8_codes8)0u;
    e[k] = 1;
    if (FLAT) { if (w.n) in[k] = *(const a8_codes8*)from; }
    else if (w.n == 8) in[k] = *(const a8_codes*)from;
    else
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < w.n) in[k][i / 4] |= (uint32_t)(uint8_t)from[i] << (8 * (i % 4));
    if (w.n) e[k] = scales[w.blk];
    if (GELU) g[k] = a8_load<T, FLAT>(da + (FLAT ? w.row : w.row * da_rs + w.c), w.n);
  }
#pragma unroll
  for (int k = 0; k < A8_CHUNKS; ++k) {
    const A8At& w = at[k];
    const int64_t to = FLAT ? w.row : w.row * cols + w.c;
    float v[8], r[8];
    a8_decode(in[k], e[k], v);
    if (GELU) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float hx, s;
        a8_gelu<sizeof(T) == 4>(v[i], hx, s);
        r[i] = a8_slope((float)g[k][i], v[i], hx, s);
        v[i] = a8_act(v[i], hx, s);
      }
      a8_store<T, FLAT>(out + to, r, w.n);
      if (a) a8_store<T, FLAT>(a + to, v, w.n);
    } else {
      a8_store<T, FLAT>(out + to, v, w.n);
    }
  }
}

int a8_check(int dtype, int64_t rows, int cols, int64_t rs) {
  if (dtype != VIL_DTYPE_F32 && dtype != VIL_DTYPE_BF16 && dtype != VIL_DTYPE_F16) return VIL_E_DTYPE;
  if (rows < 0 || cols < 0 || (rows > 1 && rs < cols)) return VIL_E_SHAPE;
  // a block of 32, filled or not, is four lanes, and a launch takes fewer than 2^32: 2^24 - 1 workgroups of A8_CHUNKS * A8_THREADS / 4 blocks
  if (cols > 0 && rows > ((int64_t)(1 << 24) - 1) * (A8_CHUNKS * A8_THREADS / 4) / ((cols - 1) / A8_BLOCK + 1)) return VIL_E_SHAPE;
  return VIL_OK;
}
// FLAT: rows of whole blocks without gaps, at addresses that the widest access fits; `rows` is then the number of values
struct A8Shape { int64_t rows; int cols, nb; bool flat; unsigned grid; };
A8Shape a8_shape(int64_t rows, int cols, int64_t rs, uintptr_t addresses) {
  A8Shape w;
  w.nb = (cols - 1) / A8_BLOCK + 1;
  w.cols = cols;
  w.flat = cols % A8_BLOCK == 0 && (rs == cols || rows == 1) && addresses % 16 == 0;
  const int64_t lanes = rows * w.nb * 4, per = A8_THREADS * A8_CHUNKS;
  w.rows = w.flat ? rows * cols : rows;
  w.grid = (unsigned)((lanes + per - 1) / per);
  return w;
}

template <typename T, bool GELU>
int a8_pack_t(const void* x, int64_t rows, int cols, int64_t rs, void* a, void* codes, void* scales, hipStream_t s) {
  const A8Shape w = a8_shape(rows, cols, rs, (uintptr_t)x | (uintptr_t)a | (uintptr_t)codes);
  if (w.flat) k_act8_pack<T, GELU, true><<<dim3(w.grid), dim3(A8_THREADS), 0, s>>>((const T*)x, rs, w.rows, w.cols, w.nb, (T*)a, (int8_t*)codes, (uint8_t*)scales);
  else k_act8_pack<T, GELU, false><<<dim3(w.grid), dim3(A8_THREADS), 0, s>>>((const T*)x, rs, w.rows, w.cols, w.nb, (T*)a, (int8_t*)codes, (uint8_t*)scales);
  return (int)hipGetLastError();
}
template <bool GELU>
int a8_pack(const void* x, int dtype, int64_t rows, int cols, int64_t rs, void* a, void* codes, void* scales, hipStream_t s) {
  if (dtype == VIL_DTYPE_F32) return a8_pack_t<float, GELU>(x, rows, cols, rs, a, codes, scales, s);
  if (dtype == VIL_DTYPE_BF16) return a8_pack_t<__bf16, GELU>(x, rows, cols, rs, a, codes, scales, s);
  return a8_pack_t<_Float16, GELU>(x, rows, cols, rs, a, codes, scales, s);
}

template <typename T, bool GELU>
int a8_unpack_t(const void* codes, const void* scales, const void* da, int64_t da_rs, int64_t rows, int cols, void* out, void* a, hipStream_t s) {
  const A8Shape w = a8_shape(rows, cols, GELU ? da_rs : cols, (uintptr_t)codes | (uintptr_t)da | (uintptr_t)out | (uintptr_t)a);
  const int8_t* c = (const int8_t*)codes;
  const uint8_t* e = (const uint8_t*)scales;
  if (w.flat) k_act8_unpack<T, GELU, true><<<dim3(w.grid), dim3(A8_THREADS), 0, s>>>(c, e, (const T*)da, da_rs, w.rows, w.cols, w.nb, (T*)out, (T*)a);
  else k_act8_unpack<T, GELU, false><<<dim3(w.grid), dim3(A8_THREADS), 0, s>>>(c, e, (const T*)da, da_rs, w.rows, w.cols, w.nb, (T*)out, (T*)a);
  return (int)hipGetLastError();
}
template <bool GELU>
int a8_unpack(const void* codes, const void* scales, const void* da, int64_t da_rs, int dtype, int64_t rows, int cols, void* out,
              void* a, hipStream_t s) {
  if (dtype == VIL_DTYPE_F32) return a8_unpack_t<float, GELU>(codes, scales, da, da_rs, rows, cols, out, a, s);
  if (dtype == VIL_DTYPE_BF16) return a8_unpack_t<__bf16, GELU>(codes, scales, da, da_rs, rows, cols, out, a, s);
  return a8_unpack_t<_Float16, GELU>(codes, scales, da, da_rs, rows, cols, out, a, s);
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
