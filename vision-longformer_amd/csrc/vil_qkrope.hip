// vil_qkrope.hip -- q and k of an attention layer between their projection and the attention: rotary positions with several
// axes, alone or behind the root-mean-square norm of every head, forward and backward.
//
// Mathematics.  Pair p of a head (p < R) is rotated by theta = pos[axis(p)] * freq[p]:
//     (u, v) -> (u cos - v sin, v cos + u sin)         u, v = channels p, R + p (VIL_ROPE_HALF) or 2p, 2p + 1 (INTERLEAVED)
// channels from 2R on pass through.  With the norm, y = R(theta) (x r w), r = 1 / sqrt(mean x^2 + eps); its backward with
// g = R(-theta) dy:   dw = sum over rows of g x r,   dx = r (g w - x r^2 mean(g w x)).  The mean, r and every sum are fp32;
// a value is rounded once, where it is stored.
//
// Angles.  pos * freq / 2 pi is taken in fp64 and reduced to a quarter turn there, so that positions far into a stream keep
// their angle (fp32 would lose 2^-24 of 10^5 radians: the whole fractional turn); sine and cosine of the remainder in
// [-pi/4, pi/4] are their Taylor series in fp32 (next terms 2e-9 and 1e-10).
//
// Bound: memory.  Forward 2, backward 3 bytes a byte of q and k.  bf16, 128 x 3137 tokens, 3 heads of 32 of a packed projection (154 MB of
// q and k), MI355X: norm forward 68 us = 4.5 TB/s (192-byte slices at a stride of 576 share their end lines with v: 1.18 times
// the bytes are read), norm backward 87 us = 5.3 TB/s, dw 4 us; rotation alone at 32 x 9217: 50 us = 4.6 TB/s each way; a large
// copy runs at 5.3.
#include "vil_internal.h"
#include <string.h>

namespace {

constexpr int RO_AXES = 4;
constexpr int RO_M_MAX = 256;
constexpr int RO_THREADS = 256;

struct RoSide {               // q or k
  const void* x; const void* g; void* y; const void* w;
  int64_t x_sb, x_st, x_sh, g_sb, g_st, g_sh, y_sb, y_st, y_sh;
  int H;
};
struct RoParams {
  RoSide s[2];
  const void* pos; int64_t pos_sb, pos_st;
  const void* freq;
  float* parts;               // backward: (2, nblocks, M) partial sums of dw
  int nblocks;                // workgroups of one side
  int B, N, M, R, pos_dtype, freq_f64, w_dtype, interleaved;
  int axes, sec_end[RO_AXES];
  float eps, sign;            // sign: +1 rotates by theta, -1 back
  // tiled kernels: tokens of a tile, tiles of a segment, segments, segments of a workgroup, tokens of a segment; magic numbers of
  // x / H, x / N, x / R
  int sides, tile, ntiles, nseg, spg, flat, shared;
  int64_t T;
  unsigned h_magic[2], n_magic, r_magic;
  float inv_m;
};

// (the bf16 conversions of the compiler round to nearest even, v_cvt_pk_bf16_f32)
template <typename T> __device__ __forceinline__ float ro_ld(const T* p) { return (float)*p; }
template <typename T> __device__ __forceinline__ void ro_st(T* p, float v) { *p = (T)v; }

__device__ __forceinline__ float ro_w(const void* w, int dtype, int i) {
  if (!w) return 1.0f;
  return dtype == VIL_DTYPE_F32 ? ((const float*)w)[i] : dtype == VIL_DTYPE_BF16 ? (float)((const __bf16*)w)[i] : (float)((const _Float16*)w)[i];
}

__device__ __forceinline__ void ro_sincos(const RoParams& p, int b, int n, int j, float& sn, float& cs) {
  int axis = 0;
  while (axis + 1 < p.axes && j >= p.sec_end[axis]) ++axis;
  const int64_t at = b * p.pos_sb + n * p.pos_st + axis;
  const double x = p.pos_dtype == VIL_POS_F32 ? (double)((const float*)p.pos)[at]
                 : p.pos_dtype == VIL_POS_I32 ? (double)((const int32_t*)p.pos)[at] : (double)((const int64_t*)p.pos)[at];
  const double f = p.freq_f64 ? ((const double*)p.freq)[j] : (double)((const float*)p.freq)[j];
  double t = x * f * 0.15915494309189533577;           // turns
  t = 4.0 * (t - floor(t));                            // quarter turns, [0, 4]
  const double k = rint(t);
  const float a = (float)(t - k) * 1.57079632679489662f, a2 = a * a;
  float s0 = fmaf(a2, 2.7557319e-6f, -1.9841270e-4f), c0 = fmaf(a2, -2.7557319e-7f, 2.4801587e-5f);
  s0 = fmaf(a2, s0, 8.3333333e-3f);  c0 = fmaf(a2, c0, -1.3888889e-3f);
  s0 = fmaf(a2, s0, -1.6666667e-1f); c0 = fmaf(a2, c0, 4.1666667e-2f);
  s0 = fmaf(a2 * a, s0, a);          c0 = fmaf(a2, c0, -0.5f);
  c0 = fmaf(a2, c0, 1.0f);
  const int q = (int)k;
  const bool odd = q & 1;
  const float s1 = odd ? c0 : s0, c1 = odd ? s0 : c0;
  sn = (q & 2) ? -s1 : s1;
  cs = ((q + 1) & 2) ? -c1 : c1;
}

template <int LPR>
__device__ __forceinline__ float ro_row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Any even head of up to 256 channels, any strides: LPR lanes to a head row, NP pairs to a lane, one element at a time.
// blockIdx.y: q or k.  BWD: y = dx, g = dy, x = the forward's input (read with NORM only).
template <typename T, int LPR, int NP, bool NORM, bool BWD>
__global__ __launch_bounds__(RO_THREADS) void k_rope_any(RoParams p) {
  constexpr int RPW = 64 / LPR;
  const RoSide& S = p.s[blockIdx.y];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % LPR, slot = lane / LPR;
  const int64_t rows = (int64_t)p.B * p.N * S.H, per_pass = (int64_t)gridDim.x * 4 * RPW;
  int c0[NP], c1[NP];
  bool on[NP];
  float w0[NP], w1[NP], d0[NP], d1[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int j = sub + i * LPR;
    on[i] = j < p.M / 2;
    const bool apart = j < p.R && !p.interleaved;
    c0[i] = on[i] ? (apart ? j : 2 * j) : 0;
    c1[i] = on[i] ? (apart ? p.R + j : 2 * j + 1) : 0;
    w0[i] = NORM && on[i] ? ro_w(S.w, p.w_dtype, c0[i]) : 0.f;
    w1[i] = NORM && on[i] ? ro_w(S.w, p.w_dtype, c1[i]) : 0.f;
    d0[i] = d1[i] = 0.f;
  }
  for (int64_t r0 = ((int64_t)blockIdx.x * 4 + wave) * RPW; r0 < rows; r0 += per_pass) {
    const int64_t row = r0 + slot;
    const bool rok = row < rows;
    const int64_t tok = row / S.H;
    const int h = (int)(row - tok * S.H), b = (int)(tok / p.N), n = (int)(tok - (int64_t)b * p.N);
    const T* x = (const T*)S.x + b * S.x_sb + n * S.x_st + h * S.x_sh;
    const T* g = (const T*)S.g + b * S.g_sb + n * S.g_st + h * S.g_sh;
    T* y = (T*)S.y + b * S.y_sb + n * S.y_st + h * S.y_sh;
    float u[NP], v[NP], gu[NP], gv[NP], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const bool ok = rok && on[i];
      const int j = sub + i * LPR;
      u[i] = v[i] = gu[i] = gv[i] = 0.f;
      if (ok) {
        if (NORM || !BWD) { u[i] = ro_ld(x + c0[i]); v[i] = ro_ld(x + c1[i]); }
        if (BWD) { gu[i] = ro_ld(g + c0[i]); gv[i] = ro_ld(g + c1[i]); }
        if (BWD && j < p.R) {                       // g = R(-theta) dy
          float sn, cs;
          ro_sincos(p, b, n, j, sn, cs);
          const float a = gu[i] * cs + gv[i] * sn;
          gv[i] = gv[i] * cs - gu[i] * sn;
          gu[i] = a;
        }
      }
      if (NORM) { s1 = fmaf(u[i], u[i], s1); s1 = fmaf(v[i], v[i], s1); }
      if (NORM && BWD) { s2 = fmaf(gu[i] * w0[i], u[i], s2); s2 = fmaf(gv[i] * w1[i], v[i], s2); }
    }
    float r = 1.f, m = 0.f;
    if (NORM) {
      r = __builtin_amdgcn_rsqf(fmaf(ro_row_sum<LPR>(s1), p.inv_m, p.eps));
      if (BWD) m = r * r * (ro_row_sum<LPR>(s2) * p.inv_m);
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int j = sub + i * LPR;
      if (!(rok && on[i])) continue;
      if (!BWD) {
        float a = NORM ? u[i] * r * w0[i] : u[i], c = NORM ? v[i] * r * w1[i] : v[i];
        if (j < p.R) {
          float sn, cs;
          ro_sincos(p, b, n, j, sn, cs);
          const float a2 = a * cs - c * sn;
          c = c * cs + a * sn;
          a = a2;
        }
        ro_st(y + c0[i], a); ro_st(y + c1[i], c);
      } else if (NORM) {
        d0[i] = fmaf(gu[i], u[i] * r, d0[i]); d1[i] = fmaf(gv[i], v[i] * r, d1[i]);
        ro_st(y + c0[i], r * (gu[i] * w0[i] - u[i] * m));
        ro_st(y + c1[i], r * (gv[i] * w1[i] - v[i] * m));
      } else {
        ro_st(y + c0[i], gu[i]); ro_st(y + c1[i], gv[i]);
      }
    }
  }
  if (NORM && BWD && p.parts) {                       // rows of a wave, waves of a workgroup: one partial row of dw
    __shared__ float red[4][RO_M_MAX];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
#pragma unroll
      for (int o = LPR; o < 64; o <<= 1) { d0[i] += __shfl_xor(d0[i], o, 64); d1[i] += __shfl_xor(d1[i], o, 64); }
      if (slot == 0 && on[i]) { red[wave][c0[i]] = d0[i]; red[wave][c1[i]] = d1[i]; }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.M; c += RO_THREADS)
      p.parts[((int64_t)blockIdx.y * p.nblocks + blockIdx.x) * p.M + c] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
  }
}

// dw of q and k from the workgroups' partial rows, in a fixed order.  One workgroup to 16 channels of a side; thread (i, c) adds the
// rows i, i + 64, ... of its channel, four at a time, then 64 sums of a channel meet in LDS.  Up to 1024 rows: 16 loads of a
// thread, all under way together (the pass is one trip to L2 long, not its bytes).
__global__ __launch_bounds__(1024) void k_rope_dw(const float* parts, int nblocks, int M, void* dwq, void* dwk, int w_dtype) {
  __shared__ float red[64][17];
  void* dw = blockIdx.y ? dwk : dwq;
  if (!dw) return;                                     // (uniform over the workgroup)
  const int cl = threadIdx.x & 15, sl = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float s = 0.f;
  if (c < M) {
    const float* at = parts + (int64_t)blockIdx.y * nblocks * M + c;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = sl + 64 * i;
      v[i] = row < nblocks ? at[(int64_t)row * M] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; i += 4) s += (v[i] + v[i + 1]) + (v[i + 2] + v[i + 3]);
  }
  red[sl][cl] = s;
  __syncthreads();
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) {
    if (sl < k) red[sl][cl] += red[sl + k][cl];
    __syncthreads();
  }
  if (sl == 0 && c < M) {
    s = red[0][cl];
    if (w_dtype == VIL_DTYPE_F32) ((float*)dw)[c] = s;
    else if (w_dtype == VIL_DTYPE_BF16) ((__bf16*)dw)[c] = (__bf16)s;
    else ((_Float16*)dw)[c] = (_Float16)s;
  }
}

constexpr int RO_BWD_BLOCKS = 1024;                    // workgroups of one side at the most: rows of partial sums (k_rope_dw reads 16 x 64)

// ---- tiled kernels: heads whose halves come in chunks of CH channels that a lane loads at once (16 bytes, or 8).
// A lane owns CH pairs of a head row: two chunks, R apart (half) or side by side (interleaved, and channels that pass
// through), so that a rotation needs no other lane and a row's statistics meet in LPR = M / (2 CH) neighbouring lanes
// (rounded up to a power of two).  A workgroup takes a tile of tokens of one segment with all their heads, q's then k's; the
// angles of a token are taken once, into LDS, and serve every head of q and k.  Segments are the images; where all share
// their positions a workgroup walks several of them with the same angles.  Where a tensor's images follow each other
// (stride of an image = N tokens) and positions are each image's own, all tokens are one segment, so that short images fill a tile.
// A workgroup's segments lie gridDim.y apart: the workgroups of a moment read one window of the tensors, in order (their own
// consecutive segments each: 8 % slower).
// Addresses: a scalar base per segment and 32-bit byte offsets inside the tile (products of 24-bit factors).
template <typename T, int CH> using ro_vec = T __attribute__((ext_vector_type(CH)));

// x / d for x d < 2^31, magic = ceil(2^31 / d): the excess x (magic d - 2^31) < x d stays under 2^31
__device__ __forceinline__ unsigned ro_div(unsigned x, unsigned magic) { return __umulhi(2 * x, magic); }

template <int CTRL> __device__ __forceinline__ float ro_dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
// sum over LPR neighbouring lanes, in all of them (the mirrors pair lanes whose quads / eights already agree)
template <int LPR> __device__ __forceinline__ float ro_lane_sum(float v) {
  if (LPR >= 2) v += ro_dpp<0xb1>(v);           // quad_perm 1,0,3,2
  if (LPR >= 4) v += ro_dpp<0x4e>(v);           // quad_perm 2,3,0,1
  if (LPR >= 8) v += ro_dpp<0x141>(v);          // row_half_mirror
  if (LPR >= 16) v += ro_dpp<0x140>(v);         // row_mirror
  if (LPR >= 32) v += __shfl_xor(v, 16, 64);
  return v;
}

// cosines and sines of the tile's tokens, trig[tt * R + j]
__device__ __forceinline__ void ro_tile_angles(const RoParams& p, float2* trig, int seg, int64_t t0, int ntok) {
  // (a segment of its own per image: image seg, token t0 + tt; one segment of all: token t0 + tt counted through the images)
  const int b0 = p.flat ? (int)(t0 / p.N) : seg, n0 = p.flat ? (int)(t0 - (int64_t)b0 * p.N) : (int)t0;
  for (int e = threadIdx.x; e < ntok * p.R; e += RO_THREADS) {
    const int tt = (int)ro_div(e, p.r_magic), j = e - tt * p.R;
    int b = b0, n = n0 + tt;
    if (p.flat) {
      const int q = p.n_magic ? (int)ro_div(n, p.n_magic) : n >= p.N;   // (0: an image is no shorter than a tile)
      b += q;
      n -= q * p.N;
    }
    float sn, cs;
    ro_sincos(p, b, n, j, sn, cs);
    trig[e] = make_float2(cs, sn * p.sign);
  }
}

// a lane's pairs: chunk a at channel ca, chunk b at cb; HALF pairs a[i] with b[i], INTERLEAVED neighbours
struct RoUnit { int ca, cb, j0; bool on, turns; };
template <int CH, bool INTER> __device__ __forceinline__ RoUnit ro_unit(const RoParams& p, int sub) {
  RoUnit u;
  u.on = sub * 2 * CH < p.M;
  u.j0 = sub * CH;
  u.turns = u.on && u.j0 < p.R;
  const bool apart = u.turns && !INTER;
  u.ca = u.on ? (apart ? u.j0 : 2 * u.j0) : 0;
  u.cb = u.on ? (apart ? p.R + u.j0 : 2 * u.j0 + CH) : CH;
  return u;
}

// cs: CH pairs (cos, sin), 32-byte aligned
template <int CH, bool INTER>
__device__ __forceinline__ void ro_turn(float (&a)[CH], float (&b)[CH], const float4* cs) {
#pragma unroll
  for (int i = 0; i < CH; i += 2) {
    const float4 t = cs[i / 2];                  // cos, sin of pairs i, i + 1 of the lane
    float x0, y0, x1, y1;
    if (!INTER) { x0 = a[i]; y0 = b[i]; x1 = a[i + 1]; y1 = b[i + 1]; }
    else if (i < CH / 2) { x0 = a[2 * i]; y0 = a[2 * i + 1]; x1 = a[2 * i + 2]; y1 = a[2 * i + 3]; }
    else { x0 = b[2 * i - CH]; y0 = b[2 * i + 1 - CH]; x1 = b[2 * i + 2 - CH]; y1 = b[2 * i + 3 - CH]; }
    const float u0 = x0 * t.x - y0 * t.y, v0 = y0 * t.x + x0 * t.y, u1 = x1 * t.z - y1 * t.w, v1 = y1 * t.z + x1 * t.w;
    if (!INTER) { a[i] = u0; b[i] = v0; a[i + 1] = u1; b[i + 1] = v1; }
    else if (i < CH / 2) { a[2 * i] = u0; a[2 * i + 1] = v0; a[2 * i + 2] = u1; a[2 * i + 3] = v1; }
    else { b[2 * i - CH] = u0; b[2 * i + 1 - CH] = v0; b[2 * i + 2 - CH] = u1; b[2 * i + 3 - CH] = v1; }
  }
}

template <typename T, int CH> __device__ __forceinline__ ro_vec<T, CH> ro_load(const char* base, unsigned off) {
  return *(const ro_vec<T, CH>*)(base + off);
}
template <typename T, int CH> __device__ __forceinline__ void ro_store(char* base, unsigned off, const float (&v)[CH]) {
  ro_vec<T, CH> o;
#pragma unroll
  for (int c = 0; c < CH; ++c) o[c] = (T)v[c];
  __builtin_nontemporal_store(o, (ro_vec<T, CH>*)(base + off));   // (streams past the caches: 10 to 15 % of the large cases' time)
}

// Head rows of a tile, one side: IPT rows to a thread and step, the next step's loads issued before this one's arithmetic, so that
// loads stay under way while a wave computes (norm forward at 128 x 3137 x 3 heads of 32: 82 us without, 73 with it; a copy of the
// same slices takes 61).
// Rows past the end load the last row again and store nothing.
template <typename T, int CH, int LPR, int IPT> struct RoRows {
  static constexpr int ROWS = RO_THREADS / LPR;
  int items, H;
  unsigned magic;
  __device__ __forceinline__ void at(int base, int i, int& tt, int& h, bool& ok) const {
    int idx = base + i * ROWS + (int)threadIdx.x / LPR;
    ok = idx < items;
    idx = ok ? idx : items - 1;
    tt = (int)ro_div(idx, magic);
    h = idx - tt * H;
  }
};

// The forward pass; without the norm the backward pass too (sign -1).
template <typename T, int CH, int LPR, bool NORM, bool INTER>
__global__ __launch_bounds__(RO_THREADS, NORM ? 4 : 5) void k_rope_tile(RoParams p) {
  constexpr int IPT = 2, STEP = IPT * RO_THREADS / LPR, SZ = sizeof(T);
  extern __shared__ float4 ro_lds4[];
  float* wl = (float*)ro_lds4;                                   // (2, M) weights of q, k
  float2* trig = (float2*)(wl + (NORM ? 2 * p.M : 0));
  const int64_t t0 = (int64_t)blockIdx.x * p.tile;
  const int ntok = p.T - t0 < p.tile ? (int)(p.T - t0) : p.tile;
  const RoUnit u = ro_unit<CH, INTER>(p, threadIdx.x % LPR);
  if (NORM)
    for (int c = threadIdx.x; c < 2 * p.M; c += RO_THREADS) wl[c] = c < p.M ? ro_w(p.s[0].w, p.w_dtype, c) : ro_w(p.s[1].w, p.w_dtype, c - p.M);
  const int stride = gridDim.y;
  for (int first = blockIdx.y; first < p.nseg; first += stride) {
    const int last = p.shared ? p.nseg : first + 1;              // segments that the same angles serve
    if (first != (int)blockIdx.y) __syncthreads();               // the angles before are no longer read
    ro_tile_angles(p, trig, first, t0, ntok);
    __syncthreads();
    for (int side = 0; side < p.sides; ++side) {
      const RoSide& S = p.s[side];
      const unsigned xt = S.x_st * SZ, xh = S.x_sh * SZ, yt = S.y_st * SZ, yh = S.y_sh * SZ;
      const RoRows<T, CH, LPR, IPT> rows = {ntok * S.H, S.H, p.h_magic[side]};
      float wa[CH], wb[CH];
      if (NORM)
#pragma unroll
        for (int c = 0; c < CH; ++c) { wa[c] = wl[side * p.M + u.ca + c]; wb[c] = wl[side * p.M + u.cb + c]; }
      ro_vec<T, CH> xa[IPT], xb[IPT], na[IPT], nb[IPT];
      const auto load = [&](int seg, int base, ro_vec<T, CH>(&va)[IPT], ro_vec<T, CH>(&vb)[IPT]) {
        const char* x = (const char*)S.x + (seg * S.x_sb + t0 * S.x_st) * SZ;
#pragma unroll
        for (int i = 0; i < IPT; ++i) {
          int tt, h;
          bool ok;
          rows.at(base, i, tt, h, ok);
          const unsigned xo = __umul24(tt, xt) + __umul24(h, xh);
          va[i] = ro_load<T, CH>(x, xo + u.ca * SZ);
          vb[i] = ro_load<T, CH>(x, xo + u.cb * SZ);
        }
      };
      int seg = first, base = 0;
      load(seg, 0, xa, xb);
      for (;;) {
        int nseg = seg, nbase = base + STEP;
        if (nbase >= rows.items) { nbase = 0; nseg += stride; }
        const bool more = nseg < last;
        if (more) load(nseg, nbase, na, nb);
        char* y = (char*)S.y + (seg * S.y_sb + t0 * S.y_st) * SZ;
#pragma unroll
        for (int i = 0; i < IPT; ++i) {
          int tt, h;
          bool ok;
          rows.at(base, i, tt, h, ok);
          float a[CH], b[CH];
#pragma unroll
          for (int c = 0; c < CH; ++c) { a[c] = (float)xa[i][c]; b[c] = (float)xb[i][c]; }
          if (NORM) {
            float s = 0.f;
#pragma unroll
            for (int c = 0; c < CH; ++c) { s = fmaf(a[c], a[c], s); s = fmaf(b[c], b[c], s); }
            if (LPR > 2 && !u.on) s = 0.f;                       // (lanes past a head that is no power of two)
            const float r = __builtin_amdgcn_rsqf(fmaf(ro_lane_sum<LPR>(s), p.inv_m, p.eps));
#pragma unroll
            for (int c = 0; c < CH; ++c) { a[c] = a[c] * r * wa[c]; b[c] = b[c] * r * wb[c]; }
          }
          if (u.turns) ro_turn<CH, INTER>(a, b, (const float4*)(trig + tt * p.R + u.j0));
          if (ok && u.on) {
            const unsigned yo = __umul24(tt, yt) + __umul24(h, yh);
            ro_store<T, CH>(y, yo + u.ca * SZ, a);
            ro_store<T, CH>(y, yo + u.cb * SZ, b);
          }
        }
        if (!more) break;
#pragma unroll
        for (int i = 0; i < IPT; ++i) { xa[i] = na[i]; xb[i] = nb[i]; }
        seg = nseg;
        base = nbase;
      }
    }
    if (p.shared) break;
  }
}

// sum over the lanes of 16 that share lane % LPR, in all of them
template <int LPR> __device__ __forceinline__ float ro_row_of_16(float v) {
  if (LPR <= 8) v += ro_dpp<0x128>(v);          // row_ror 8
  if (LPR <= 4) v += ro_dpp<0x124>(v);
  if (LPR <= 2) v += ro_dpp<0x122>(v);
  if (LPR <= 1) v += ro_dpp<0x121>(v);
  return v;
}

// The norm's backward pass.  blockIdx.z: q or k; a workgroup walks tiles and segments and keeps its share of dw in registers.
template <typename T, int CH, int LPR, bool INTER>
__global__ __launch_bounds__(RO_THREADS, 4) void k_rope_norm_bwd(RoParams p) {
  constexpr int STEP = RO_THREADS / LPR, SZ = sizeof(T);
  extern __shared__ float4 ro_lds4[];                  // the weights; a tile's angles; at the end 16 shares of dw
  float* wl = (float*)ro_lds4;
  float2* trig = (float2*)ro_lds4;
  const int side = blockIdx.z;
  const RoSide& S = p.s[side];
  const RoUnit u = ro_unit<CH, INTER>(p, threadIdx.x % LPR);
  const unsigned xt = S.x_st * SZ, xh = S.x_sh * SZ, yt = S.y_st * SZ, yh = S.y_sh * SZ, gt = S.g_st * SZ, gh = S.g_sh * SZ;
  float wa[CH], wb[CH], da[CH], db[CH];
  if ((int)threadIdx.x < p.M) wl[threadIdx.x] = ro_w(S.w, p.w_dtype, threadIdx.x);
  __syncthreads();
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    wa[c] = wl[u.ca + c];
    wb[c] = wl[u.cb + c];
    da[c] = db[c] = 0.f;
  }
  const int stride = gridDim.y;
  for (int tile = blockIdx.x; tile < p.ntiles; tile += gridDim.x) {
    const int64_t t0 = (int64_t)tile * p.tile;
    const int ntok = p.T - t0 < p.tile ? (int)(p.T - t0) : p.tile;
    const RoRows<T, CH, LPR, 1> rows = {ntok * S.H, S.H, p.h_magic[side]};
    for (int first = blockIdx.y; first < p.nseg; first += stride) {
      const int last = p.shared ? p.nseg : first + 1;
      __syncthreads();                                 // the weights, or the angles before, are no longer read
      ro_tile_angles(p, trig, first, t0, ntok);
      __syncthreads();
      ro_vec<T, CH> xa, xb, ga_, gb_, nxa, nxb, nga, ngb;
      const auto load = [&](int seg, int base, ro_vec<T, CH>& va, ro_vec<T, CH>& vb, ro_vec<T, CH>& vc, ro_vec<T, CH>& vd) {
        const char* x = (const char*)S.x + (seg * S.x_sb + t0 * S.x_st) * SZ;
        const char* g = (const char*)S.g + (seg * S.g_sb + t0 * S.g_st) * SZ;
        int tt, h;
        bool ok;
        rows.at(base, 0, tt, h, ok);
        const unsigned xo = __umul24(tt, xt) + __umul24(h, xh), go = __umul24(tt, gt) + __umul24(h, gh);
        va = ro_load<T, CH>(x, xo + u.ca * SZ);
        vb = ro_load<T, CH>(x, xo + u.cb * SZ);
        vc = ro_load<T, CH>(g, go + u.ca * SZ);
        vd = ro_load<T, CH>(g, go + u.cb * SZ);
      };
      int seg = first, base = 0;
      load(seg, 0, xa, xb, ga_, gb_);
      for (;;) {
        int nseg = seg, nbase = base + STEP;
        if (nbase >= rows.items) { nbase = 0; nseg += stride; }
        const bool more = nseg < last;
        if (more) load(nseg, nbase, nxa, nxb, nga, ngb);
        int tt, h;
        bool ok;
        rows.at(base, 0, tt, h, ok);
        float a[CH], b[CH], ga[CH], gb[CH], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          a[c] = (float)xa[c]; b[c] = (float)xb[c];
          ga[c] = (float)ga_[c]; gb[c] = (float)gb_[c];
        }
        if (u.turns) ro_turn<CH, INTER>(ga, gb, (const float4*)(trig + tt * p.R + u.j0));
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          s1 = fmaf(a[c], a[c], s1); s1 = fmaf(b[c], b[c], s1);
          s2 = fmaf(ga[c] * wa[c], a[c], s2); s2 = fmaf(gb[c] * wb[c], b[c], s2);
        }
        if (LPR > 2 && !u.on) s1 = s2 = 0.f;
        const float r = __builtin_amdgcn_rsqf(fmaf(ro_lane_sum<LPR>(s1), p.inv_m, p.eps));
        const float m = r * (r * (r * (ro_lane_sum<LPR>(s2) * p.inv_m)));    // (r^3 alone leaves fp32 past |x| = 10^12 and 10^-13)
        if (ok && u.on) {
          char* y = (char*)S.y + (seg * S.y_sb + t0 * S.y_st) * SZ;
          const unsigned yo = __umul24(tt, yt) + __umul24(h, yh);
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            ga[c] *= r; gb[c] *= r;
            da[c] = fmaf(ga[c], a[c], da[c]);
            db[c] = fmaf(gb[c], b[c], db[c]);
            a[c] = ga[c] * wa[c] - a[c] * m;
            b[c] = gb[c] * wb[c] - b[c] * m;
          }
          ro_store<T, CH>(y, yo + u.ca * SZ, a);
          ro_store<T, CH>(y, yo + u.cb * SZ, b);
        }
        if (!more) break;
        xa = nxa; xb = nxb; ga_ = nga; gb_ = ngb;
        seg = nseg;
        base = nbase;
      }
      if (p.shared) break;
    }
  }
  if (!p.parts) return;
  // rows of 16 lanes by register moves, the 16 rows of the workgroup through LDS (for 32 lanes to a head, two rows hold it)
  __syncthreads();
  float* red = (float*)ro_lds4;                        // (shares, M)
  constexpr int SPAN = LPR < 16 ? 16 : LPR, SHARES = RO_THREADS / SPAN;
#pragma unroll
  for (int c = 0; c < CH; ++c) { da[c] = ro_row_of_16<LPR>(da[c]); db[c] = ro_row_of_16<LPR>(db[c]); }
  if ((int)threadIdx.x % SPAN < LPR && u.on)
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      red[threadIdx.x / SPAN * p.M + u.ca + c] = da[c];
      red[threadIdx.x / SPAN * p.M + u.cb + c] = db[c];
    }
  __syncthreads();
  const int64_t row = (int64_t)side * p.nblocks + blockIdx.y * gridDim.x + blockIdx.x;
  if ((int)threadIdx.x < p.M) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < SHARES; ++i) s += red[i * p.M + threadIdx.x];
    p.parts[row * p.M + threadIdx.x] = s;
  }
}

unsigned ro_magic(int d) { return (unsigned)(((1ull << 31) + d - 1) / d); }

// Channels of a chunk: 16 bytes where the head, the rotated part and every stride and address allow it, else 8 bytes of a 16-bit
// type, else 0: one element at a time (as where a token or head stride passes the 24 bits of a factor).
int ro_chunk(const RoParams& p, int dtype, bool bwd_norm) {
  const int size = dtype == VIL_DTYPE_F32 ? 4 : 2;
  for (int ch = 16 / size; ch >= 4; ch /= 2) {
    if (p.M % (2 * ch) || p.R % ch) continue;
    uintptr_t bits = 0;
    bool small = true;
    for (int i = 0; i < 2; ++i) {
      const RoSide& S = p.s[i];
      if (!S.H) continue;
      const int64_t strides[6] = {S.x_st, S.x_sh, S.y_st, S.y_sh, bwd_norm ? S.g_st : 0, bwd_norm ? S.g_sh : 0};
      for (int64_t st : strides) {
        bits |= (uintptr_t)(st * size);
        small = small && st >= 0 && st * size < (1 << 24);
      }
      // (offsets in a tile stay under 2^32: the heads under 2^30 here, the tokens in ro_plan)
      small = small && S.H <= (1 << 15) && S.H * S.x_sh * size < (1 << 30) && S.H * S.y_sh * size < (1 << 30) && (!bwd_norm || S.H * S.g_sh * size < (1 << 30));
      bits |= (uintptr_t)S.x | (uintptr_t)S.y | (uintptr_t)((S.x_sb | S.y_sb) * size);
      if (bwd_norm) bits |= (uintptr_t)S.g | (uintptr_t)(S.g_sb * size);
    }
    if (small && bits % (ch * size) == 0) return ch;
  }
  return 0;
}

// Tiles and segments of a launch: a tile's rows fill whole steps of the workgroup (`step` head rows; up to four), its angles 16 KB
// at the most (32 KB: 15 % slower), and there are at least `want` workgroups where there is work for them.  Segments that share their
// angles are walked by one workgroup only past `rounds` times `want` of them: the forward pass at 32 x 9217 x 3 heads of 32 takes
// 50 us with a workgroup to each of 3488 tiles, 54 with 1744, 57 with 1163.
void ro_plan(RoParams& p, int size, int wave_rows, int step, int64_t want, int rounds) {
  bool flat = true;                                    // images follow each other in every tensor
  int64_t st = 1;
  for (int i = 0; i < p.sides; ++i) {
    const RoSide& S = p.s[i];
    flat = flat && S.x_sb == p.N * S.x_st && S.y_sb == p.N * S.y_st && (!S.g || S.g_sb == p.N * S.g_st);
    for (int64_t v : {S.x_st, S.y_st, S.g ? S.g_st : 0}) st = v > st ? v : st;
  }
  const bool shared = p.R == 0 || p.pos_sb == 0 || p.B == 1;
  const int H = p.s[0].H > p.s[1].H ? p.s[0].H : p.s[1].H;
  const int64_t tokens = (int64_t)p.B * p.N;
  int64_t tile = 512;
  if (p.R > 0 && tile > 2048 / p.R) tile = 2048 / p.R;
  if (tile > (1 << 30) / (st * size)) tile = (1 << 30) / (st * size);
  const int64_t share = (tokens + want - 1) / want, wave = (wave_rows + H - 1) / H;      // (a wave's worth of rows at least)
  if (tile > (share > wave ? share : wave)) tile = share > wave ? share : wave;
  int64_t steps = tile * H / step;
  if (steps > 4) steps = 4;
  if (steps >= 1) tile = steps * step / H;
  if (tile < 1) tile = 1;
  // one segment of all tokens for positions of each image's own, and for images shorter than a tile
  p.flat = flat && p.B > 1 && (!shared || p.N < tile);
  p.nseg = p.flat ? 1 : p.B;
  p.T = p.flat ? tokens : p.N;
  if (tile > p.T) tile = p.T;
  p.tile = (int)tile;
  p.ntiles = (int)((p.T + tile - 1) / tile);
  p.spg = 1;
  p.shared = shared;
  if (shared && p.nseg > 1) {
    const int64_t units = (int64_t)p.ntiles * p.nseg, most = want * rounds, spg = (units + most - 1) / most;
    p.spg = spg > p.nseg ? p.nseg : (int)spg;
  }
  for (int i = 0; i < p.sides; ++i) p.h_magic[i] = ro_magic(p.s[i].H);      // x: rows of a tile, <= 2^11 or the heads of one token
  p.n_magic = p.flat && p.N < p.tile ? ro_magic(p.N) : 0;                   // x < 2^10, N < 2^9
  p.r_magic = p.R ? ro_magic(p.R) : 0;                                      // x: angles of a tile, <= 2^11
}

template <typename T, int CH, int LPR, bool NORM>
int ro_tile_launch(RoParams& p, hipStream_t s) {
  ro_plan(p, sizeof(T), 64 / LPR, 2 * RO_THREADS / LPR, 5 * vil_cu_count(), 8);
  if (p.nseg > 65535 * (int64_t)p.spg) p.spg = (p.nseg + 65534) / 65535;         // (the grid's second axis)
  const dim3 grid(p.ntiles, (p.nseg + p.spg - 1) / p.spg), block(RO_THREADS);
  const size_t lds = (size_t)p.tile * p.R * sizeof(float2) + (NORM ? 2 * p.M * sizeof(float) : 0);
  if (p.interleaved) k_rope_tile<T, CH, LPR, NORM, true><<<grid, block, lds, s>>>(p);
  else k_rope_tile<T, CH, LPR, NORM, false><<<grid, block, lds, s>>>(p);
  return (int)hipGetLastError();
}

template <typename T, int CH, int LPR>
int ro_bwd_launch(RoParams& p, hipStream_t s) {
  // two workgroups to a CU: every one ends in a row of partial sums (four: 7 % slower at 128 x 3137 x 3 heads of 32, one: 14 %)
  const int held = 2 * vil_cu_count() / p.sides;
  ro_plan(p, sizeof(T), 64 / LPR, RO_THREADS / LPR, held < RO_BWD_BLOCKS ? held : RO_BWD_BLOCKS, 1);
  if (p.nseg > RO_BWD_BLOCKS * (int64_t)p.spg) p.spg = (p.nseg + RO_BWD_BLOCKS - 1) / RO_BWD_BLOCKS;   // (short images)
  const int groups = (p.nseg + p.spg - 1) / p.spg, x = RO_BWD_BLOCKS / groups;
  const dim3 grid(x < p.ntiles ? x : p.ntiles, groups, p.sides), block(RO_THREADS);
  p.nblocks = grid.x * grid.y;
  const size_t angles = (size_t)p.tile * p.R * sizeof(float2), shares = (size_t)16 * p.M * sizeof(float), lds = angles > shares ? angles : shares;
  if (p.interleaved) k_rope_norm_bwd<T, CH, LPR, true><<<grid, block, lds, s>>>(p);
  else k_rope_norm_bwd<T, CH, LPR, false><<<grid, block, lds, s>>>(p);
  return (int)hipGetLastError();
}

template <typename T, int CH, bool NORM, bool BWD>
int ro_lanes(RoParams& p, hipStream_t s) {
  const int lanes = p.M / (2 * CH);
#define RO_LANES(L)                                                   \
  if (lanes <= L) {                                                   \
    if constexpr (NORM && BWD) return ro_bwd_launch<T, CH, L>(p, s);  \
    else return ro_tile_launch<T, CH, L, NORM>(p, s);                 \
  }
  RO_LANES(1) RO_LANES(2) RO_LANES(4) RO_LANES(8) RO_LANES(16)
  if constexpr (CH == 4) { RO_LANES(32) }
#undef RO_LANES
  return VIL_E_HEAD_DIM;                                               // (not reached: M <= 256)
}
template <typename T, bool NORM, bool BWD>
int ro_tiled(RoParams& p, int ch, hipStream_t s) {
  p.sign = BWD ? -1.0f : 1.0f;
  if constexpr (sizeof(T) == 2)
    if (ch == 8) return ro_lanes<T, 8, NORM, BWD>(p, s);
  return ro_lanes<T, 4, NORM, BWD>(p, s);
}

// k_rope_any: lanes of a head row, workgroups of a side
int ro_lpr(int M) { return M <= 16 ? 8 : M <= 32 ? 16 : M <= 64 ? 32 : 64; }
int ro_nblocks(const VilRopeDesc* d, int lpr) {
  const int64_t rows = (int64_t)d->B * d->N * (d->Hq > d->Hk ? d->Hq : d->Hk);
  const int64_t need = (rows + 4 * (64 / lpr) - 1) / (4 * (64 / lpr));
  return (int)(need < RO_BWD_BLOCKS ? (need < 1 ? 1 : need) : RO_BWD_BLOCKS);
}

template <typename T, bool NORM, bool BWD>
int ro_launch(RoParams& p, int dtype, int sides, hipStream_t s) {
  // (without the norm the backward pass reads g alone)
  if (BWD && !NORM)
    for (int i = 0; i < 2; ++i) { p.s[i].x = p.s[i].g; p.s[i].x_sb = p.s[i].g_sb; p.s[i].x_st = p.s[i].g_st; p.s[i].x_sh = p.s[i].g_sh; }
  p.sides = sides;
  if (const int ch = ro_chunk(p, dtype, NORM && BWD)) return ro_tiled<T, NORM, BWD>(p, ch, s);
  const dim3 grid(p.nblocks, sides), block(RO_THREADS);
  const int pairs = p.M / 2;
  if (pairs <= 8) k_rope_any<T, 8, 1, NORM, BWD><<<grid, block, 0, s>>>(p);
  else if (pairs <= 16) k_rope_any<T, 16, 1, NORM, BWD><<<grid, block, 0, s>>>(p);
  else if (pairs <= 32) k_rope_any<T, 32, 1, NORM, BWD><<<grid, block, 0, s>>>(p);
  else if (pairs <= 64) k_rope_any<T, 64, 1, NORM, BWD><<<grid, block, 0, s>>>(p);
  else k_rope_any<T, 64, 2, NORM, BWD><<<grid, block, 0, s>>>(p);
  return (int)hipGetLastError();
}

template <bool BWD>
int ro_dispatch(const VilRopeDesc* d, RoParams& p, hipStream_t s) {
  const int sides = d->Hk > 0 ? 2 : 1;
  switch (d->dtype * 2 + (d->norm ? 1 : 0)) {
    case VIL_DTYPE_F32 * 2: return ro_launch<float, false, BWD>(p, d->dtype, sides, s);
    case VIL_DTYPE_F32 * 2 + 1: return ro_launch<float, true, BWD>(p, d->dtype, sides, s);
    case VIL_DTYPE_BF16 * 2: return ro_launch<__bf16, false, BWD>(p, d->dtype, sides, s);
    case VIL_DTYPE_BF16 * 2 + 1: return ro_launch<__bf16, true, BWD>(p, d->dtype, sides, s);
    case VIL_DTYPE_F16 * 2: return ro_launch<_Float16, false, BWD>(p, d->dtype, sides, s);
    default: return ro_launch<_Float16, true, BWD>(p, d->dtype, sides, s);
  }
}

int ro_check(const VilRopeDesc* d) {
  if (!d) return VIL_E_NULL;
  if (d->B < 0 || d->N < 0 || d->Hq <= 0 || d->Hk < 0) return VIL_E_SHAPE;
  if ((int64_t)d->B * d->N > INT32_MAX) return VIL_E_SHAPE;
  if (d->M < 2 || d->M % 2 || d->M > RO_M_MAX) return VIL_E_HEAD_DIM;
  if (d->R < 0 || 2 * d->R > d->M || d->axes < 0 || d->axes > RO_AXES || (d->R > 0 && d->axes < 1)) return VIL_E_SHAPE;
  int sum = 0;
  for (int a = 0; a < d->axes; ++a) {
    if (d->sections[a] < 0 || d->sections[a] > RO_M_MAX) return VIL_E_SHAPE;
    sum += d->sections[a];
  }
  if (sum != d->R) return VIL_E_SHAPE;
  if (d->layout != VIL_ROPE_HALF && d->layout != VIL_ROPE_INTERLEAVED) return VIL_E_MODE;
  if (d->dtype != VIL_DTYPE_F32 && d->dtype != VIL_DTYPE_BF16 && d->dtype != VIL_DTYPE_F16) return VIL_E_DTYPE;
  if (d->R > 0 && d->pos_dtype != VIL_POS_F32 && d->pos_dtype != VIL_POS_I32 && d->pos_dtype != VIL_POS_I64) return VIL_E_DTYPE;
  if (d->R > 0 && d->freq_dtype != VIL_DTYPE_F32 && d->freq_dtype != VIL_DTYPE_F64) return VIL_E_DTYPE;
  if (d->norm && d->w_dtype != VIL_DTYPE_F32 && d->w_dtype != VIL_DTYPE_BF16 && d->w_dtype != VIL_DTYPE_F16) return VIL_E_DTYPE;
  if (!d->norm && d->R == 0) return VIL_E_SHAPE;          // nothing to do
  return VIL_OK;
}

void ro_fill(RoParams& p, const VilRopeDesc* d, const void* pos, const void* freq) {
  memset(&p, 0, sizeof(p));
  p.B = d->B; p.N = d->N; p.M = d->M; p.R = d->R;
  p.pos = pos; p.pos_sb = d->pos_sb; p.pos_st = d->pos_st; p.pos_dtype = d->pos_dtype;
  p.freq = freq; p.freq_f64 = d->freq_dtype == VIL_DTYPE_F64;
  p.w_dtype = d->w_dtype; p.interleaved = d->layout == VIL_ROPE_INTERLEAVED;
  p.axes = d->axes;
  for (int a = 0, e = 0; a < RO_AXES; ++a) p.sec_end[a] = e += a < d->axes ? d->sections[a] : 0;
  p.eps = d->eps;
  p.inv_m = 1.0f / d->M;
  p.s[0].H = d->Hq; p.s[1].H = d->Hk;
}
#define RO_STRIDES(SIDE, F, NAME) SIDE.F##_sb = d->NAME##_sb, SIDE.F##_st = d->NAME##_st, SIDE.F##_sh = d->NAME##_sh

}  // namespace

extern "C" size_t vil_qk_rope_workspace_bytes(const VilRopeDesc* d) {
  if (ro_check(d) || !d->norm) return 0;
  // a row of partial sums to a workgroup of either kernel: the tiled one has at most one to a token
  const int64_t tokens = (int64_t)d->B * d->N, tiled = tokens < RO_BWD_BLOCKS ? tokens : RO_BWD_BLOCKS;
  const int64_t any = ro_nblocks(d, ro_lpr(d->M));
  return (size_t)2 * (tiled > any ? tiled : any) * d->M * sizeof(float);
}

extern "C" int vil_qk_rope_fwd(const VilRopeDesc* d, const void* q, const void* k, const void* wq, const void* wk,
                               const void* pos, const void* freq, void* yq, void* yk, void* stream) {
  if (int e = ro_check(d)) return e;
  if (d->B == 0 || d->N == 0) return VIL_OK;
  if (!q || !yq || (d->Hk > 0 && (!k || !yk)) || (d->R > 0 && (!pos || !freq))) return VIL_E_NULL;
  RoParams p;
  ro_fill(p, d, pos, freq);
  p.s[0].x = q; p.s[0].y = yq; p.s[0].w = wq;
  p.s[1].x = k; p.s[1].y = yk; p.s[1].w = wk;
  RO_STRIDES(p.s[0], x, q); RO_STRIDES(p.s[0], y, yq);
  RO_STRIDES(p.s[1], x, k); RO_STRIDES(p.s[1], y, yk);
  p.nblocks = ro_nblocks(d, ro_lpr(d->M));
  return ro_dispatch<false>(d, p, (hipStream_t)stream);
}

extern "C" int vil_qk_rope_bwd(const VilRopeDesc* d, const void* gq, const void* gk, const void* q, const void* k,
                               const void* wq, const void* wk, const void* pos, const void* freq, void* dq, void* dk,
                               void* dwq, void* dwk, void* workspace, void* stream) {
  if (int e = ro_check(d)) return e;
  const bool empty = d->B == 0 || d->N == 0;
  if (!empty && (!gq || !dq || (d->Hk > 0 && (!gk || !dk)) || (d->R > 0 && (!pos || !freq)))) return VIL_E_NULL;
  if (!empty && d->norm && (!q || (d->Hk > 0 && !k))) return VIL_E_NULL;
  if ((dwq && (!d->norm || !wq)) || (dwk && (!d->norm || !wk || d->Hk == 0))) return VIL_E_NULL;
  const bool dw = dwq || dwk;
  if (dw && !workspace) return VIL_E_WORKSPACE;
  RoParams p;
  ro_fill(p, d, pos, freq);
  p.s[0].g = gq; p.s[0].x = q; p.s[0].y = dq; p.s[0].w = wq;
  p.s[1].g = gk; p.s[1].x = k; p.s[1].y = dk; p.s[1].w = wk;
  RO_STRIDES(p.s[0], g, gq); RO_STRIDES(p.s[0], x, q); RO_STRIDES(p.s[0], y, dq);
  RO_STRIDES(p.s[1], g, gk); RO_STRIDES(p.s[1], x, k); RO_STRIDES(p.s[1], y, dk);
  p.parts = dw ? (float*)workspace : nullptr;
  p.nblocks = empty ? 0 : ro_nblocks(d, ro_lpr(d->M));
  if (!empty)
    if (int e = ro_dispatch<true>(d, p, (hipStream_t)stream)) return e;
  if (dw) {                                   // (an empty batch: zeros)
    k_rope_dw<<<dim3((d->M + 15) / 16, 2), dim3(1024), 0, (hipStream_t)stream>>>((const float*)workspace, p.nblocks, d->M, dwq, dwk, d->w_dtype);
    return (int)hipGetLastError();
  }
  return VIL_OK;
}
