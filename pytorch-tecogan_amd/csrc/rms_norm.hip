// Root-mean-square norm over the last dimension, with the residual's addition in front of it, its gradient, and an 8-bit output.
//
//   s = x + r          y = s * rstd * w          rstd = 1 / sqrt(mean_c s^2 + eps)
//   e4m3:  scale = max(max_c |y|, 2^-100) / 448,  q = e4m3(y / scale)            (448: the largest e4m3 value)
//   backward, g = dy * w, xhat = s * rstd:
//          dx = rstd * (g - xhat * mean_c(g * xhat)) + ds                       (the gradient of x and of r alike)
//          dw = sum over rows of dy * xhat
//
// One pass: a row lives in the registers of L lanes (8 .. 64 of a wave, or the 256 of a workgroup), 16 bytes per load; longer rows are
// read again for each pass over them.  The sum
// of squares, the row's maximum and dw are held in 32 bits.  y is computed from the UNROUNDED sum, so storing s in 16 bits costs y
// nothing, and the backward pass adds x and r again for the same reason (dw from a 16-bit s would be off by 2^-9 of each term: 1.6e-3 of
// the sum instead of 1e-7, for one operand less to read).  dw: every workgroup adds the rows it walks in registers and writes one partial row,
// a second launch adds those in index order - no atomics, the same bits every time.
//
// Bound by memory once the rows are many: 655360 bf16 rows of 64 with a residual to e4m3 58 us, 296 MB at 5.1 TB/s; 40960 rows 6.6 us forward (3.2 us
// is an empty machine's start and end), gradient 6.7 + 2.6.
#include "common.h"

namespace {

// One 16-byte piece of a row - W consecutive elements - as floats.  EVEN: every piece is whole and aligned.  Otherwise C or an address
// does not fill 16 bytes: the loads and stores are unaligned ones, which the hardware takes (fp16 rows of 1001 channels: forward 6.6 us
// instead of the 13.4 of single elements, gradient 10.6 instead of 25.4), and a row's last piece goes element by element.  n: elements left.
template <typename T, bool EVEN> struct Piece {
  static constexpr int W = 16 / ElemTraits<T>::kBytes;
  __device__ __forceinline__ static void load(const void* base, int64_t i, int n, float* v) {
    const char* p = reinterpret_cast<const char*>(base) + i * ElemTraits<T>::kBytes;
    if (EVEN) {
      Vec<T>::load(p, v);
    } else if (n >= W) {
      u32x4 t;
      __builtin_memcpy(&t, p, 16);
      Vec<T>::load(&t, v);
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = k < n ? load_elem<T>(p, k) : 0.f;
    }
  }
  __device__ __forceinline__ static void store(void* base, int64_t i, int n, const float* v) {
    char* p = reinterpret_cast<char*>(base) + i * ElemTraits<T>::kBytes;
    if (EVEN) {
      Vec<T>::store(p, v);
    } else if (n >= W) {
      u32x4 t;
      Vec<T>::pack(&t, v);
      __builtin_memcpy(p, &t, 16);
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k)
        if (k < n) store_elem<T>(p, k, v[k]);
    }
  }
};
template <int W, bool EVEN> __device__ __forceinline__ void load_f32(const float* p, int i, int n, float* v) {
  if (EVEN || n >= W) {
#pragma unroll
    for (int k = 0; k < W; k += 4) {
      f32x4 t;
      if (EVEN) t = *reinterpret_cast<const f32x4*>(p + i + k);
      else __builtin_memcpy(&t, p + i + k, 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k + e] = t[e];
    }
  } else {
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] = k < n ? p[i + k] : 0.f;
  }
}

// W floats -> W e4m3 bytes (v_cvt_pk_fp8_f32: round to nearest even; |v| <= 448 up to one rounding by construction, NaN stays NaN)
template <int W, bool EVEN> __device__ __forceinline__ void store_e4m3(unsigned char* p, int n, const float* v) {
  int d[W / 4];
#pragma unroll
  for (int k = 0; k < W / 4; ++k) {
    d[k] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k], v[4 * k + 1], 0, false);
    d[k] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k + 2], v[4 * k + 3], d[k], true);
  }
  if (EVEN) {
    if constexpr (W == 8) *reinterpret_cast<int2*>(p) = make_int2(d[0], d[1]);
    else *reinterpret_cast<int*>(p) = d[0];
  } else if (n >= W) {
    __builtin_memcpy(p, d, W);
  } else {
#pragma unroll
    for (int k = 0; k < W; ++k)
      if (k < n) p[k] = (unsigned char)(d[k / 4] >> (8 * (k & 3)));
  }
}

// sum / maximum over the L lanes of a row; every lane gets it.  L = 256: the whole workgroup (red: 4 floats of LDS)
template <int L> __device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = (L < 64 ? L : 64) / 2; o; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (L > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}
// of the BITS of non-negative floats: their order is the integers', and a NaN is above everything, so it reaches the scale
template <int L> __device__ __forceinline__ unsigned row_max(unsigned v, unsigned* red) {
#pragma unroll
  for (int o = (L < 64 ? L : 64) / 2; o; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
  if constexpr (L > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = max(max(red[0], red[1]), max(red[2], red[3]));
  }
  return v;
}
// the floor keeps 1 / scale finite; a row whose largest |y| is below 2^-100 (an all-zero row above all) gets that scale
__device__ __forceinline__ float e4m3_scale(unsigned amax_bits) {
  const unsigned lo = 0x0d800000u;   // 2^-100
  return __uint_as_float(max(amax_bits, lo)) / 448.f;
}
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct FwdArgs {
  const void *x, *res;
  const float* w;
  void *y, *s;          // y: T rows, or e4m3 bytes
  float *rstd, *scale;
  int64_t xs, rs, rows; // row strides of x and res (elements)
  int C;
  float eps;
};

template <typename T, bool EVEN, int L, int NV, bool Q8> __global__ __launch_bounds__(256) void rms_fwd_kernel(FwdArgs a) {
  typedef Piece<T, EVEN> P;
  constexpr int W = P::W;
  __shared__ float red[4];
  const int li = threadIdx.x & (L - 1);
  const int64_t rpb = 256 / L;
  const float inv_c = 1.f / (float)a.C;
  for (int64_t row = (int64_t)blockIdx.x * rpb + threadIdx.x / L; ; row += (int64_t)gridDim.x * rpb) {
    if (row - threadIdx.x / L >= a.rows) break;   // the whole workgroup leaves together
    const bool live = row < a.rows;
    float v[NV][W];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (li + L * i) * W;
#pragma unroll
      for (int k = 0; k < W; ++k) v[i][k] = 0.f;
      if (live && e < a.C) {
        P::load(a.x, row * a.xs + e, a.C - e, v[i]);
        if (a.res) {
          float r[W];
          P::load(a.res, row * a.rs + e, a.C - e, r);
#pragma unroll
          for (int k = 0; k < W; ++k) v[i][k] += r[k];
          if (a.s) P::store(a.s, row * a.C + e, a.C - e, v[i]);
        }
      }
#pragma unroll
      for (int k = 0; k < W; ++k) ss = fmaf(v[i][k], v[i][k], ss);
    }
    const float rstd = 1.f / sqrtf(row_sum<L>(ss, red) * inv_c + a.eps);
    if (a.rstd && live && li == 0) a.rstd[row] = rstd;
    unsigned amax = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (li + L * i) * W;
      float w[W];
#pragma unroll
      for (int k = 0; k < W; ++k) w[k] = 1.f;
      if (a.w && e < a.C) load_f32<W, EVEN>(a.w, e, a.C - e, w);
#pragma unroll
      for (int k = 0; k < W; ++k) v[i][k] = v[i][k] * rstd * w[k];
      if constexpr (Q8) {
#pragma unroll
        for (int k = 0; k < W; ++k) amax = max(amax, e < a.C ? abs_bits(v[i][k]) : 0u);
      } else {
        if (live && e < a.C) P::store(a.y, row * a.C + e, a.C - e, v[i]);
      }
    }
    if constexpr (Q8) {
      const float scale = e4m3_scale(row_max<L>(amax, reinterpret_cast<unsigned*>(red)));
      const float inv = 1.f / scale;
      if (live && li == 0) a.scale[row] = scale;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (li + L * i) * W;
#pragma unroll
        for (int k = 0; k < W; ++k) v[i][k] *= inv;
        if (live && e < a.C) store_e4m3<W, EVEN>(reinterpret_cast<unsigned char*>(a.y) + row * a.C + e, a.C - e, v[i]);
      }
    }
  }
}

// rows longer than the registers hold: one workgroup per row, the row read again for each pass over it
template <typename T, bool EVEN, bool Q8> __global__ __launch_bounds__(256) void rms_fwd_long_kernel(FwdArgs a) {
  typedef Piece<T, EVEN> P;
  constexpr int W = P::W;
  __shared__ float red[4];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    auto load = [&](int e, float* v) {
      P::load(a.x, row * a.xs + e, a.C - e, v);
      if (a.res) {
        float r[W];
        P::load(a.res, row * a.rs + e, a.C - e, r);
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] += r[k];
      }
    };
    float ss = 0.f;
    for (int e = threadIdx.x * W; e < a.C; e += 256 * W) {
      float v[W];
      load(e, v);
      if (a.res && a.s) P::store(a.s, row * a.C + e, a.C - e, v);
#pragma unroll
      for (int k = 0; k < W; ++k) ss = fmaf(v[k], v[k], ss);
    }
    const float rstd = 1.f / sqrtf(row_sum<256>(ss, red) / (float)a.C + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
    auto out = [&](int e, float* v) {
      load(e, v);
      float w[W];
#pragma unroll
      for (int k = 0; k < W; ++k) w[k] = 1.f;
      if (a.w) load_f32<W, EVEN>(a.w, e, a.C - e, w);
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = v[k] * rstd * w[k];
    };
    float inv = 1.f;
    if constexpr (Q8) {
      unsigned amax = 0;
      for (int e = threadIdx.x * W; e < a.C; e += 256 * W) {
        float v[W];
        out(e, v);
#pragma unroll
        for (int k = 0; k < W; ++k) amax = max(amax, abs_bits(v[k]));
      }
      const float scale = e4m3_scale(row_max<256>(amax, reinterpret_cast<unsigned*>(red)));
      inv = 1.f / scale;
      if (threadIdx.x == 0) a.scale[row] = scale;
    }
    for (int e = threadIdx.x * W; e < a.C; e += 256 * W) {
      float v[W];
      out(e, v);
      if constexpr (Q8) {
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] *= inv;
        store_e4m3<W, EVEN>(reinterpret_cast<unsigned char*>(a.y) + row * a.C + e, a.C - e, v);
      } else {
        P::store(a.y, row * a.C + e, a.C - e, v);
      }
    }
  }
}

struct BwdArgs {
  const void *dy, *x, *res, *ds;
  const float *rstd, *w;
  void* dx;
  float* partial;        // [gridDim.x][C], or null: no dw
  int64_t dys, xs, rs, dss, rows;
  int C;
};

template <typename T, bool EVEN> __device__ __forceinline__ void load_sum(const BwdArgs& a, int64_t row, int e, float* v) {
  typedef Piece<T, EVEN> P;
  constexpr int W = P::W;
  P::load(a.x, row * a.xs + e, a.C - e, v);
  if (a.res) {
    float r[W];
    P::load(a.res, row * a.rs + e, a.C - e, r);
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] += r[k];
  }
}

template <typename T, bool EVEN, int L, int NV> __global__ __launch_bounds__(256) void rms_bwd_kernel(BwdArgs a) {
  typedef Piece<T, EVEN> P;
  constexpr int W = P::W;
  __shared__ float red[4];
  __shared__ float fold[L >= 256 ? 1 : 256 * W];
  const int li = threadIdx.x & (L - 1);
  const int64_t rpb = 256 / L;
  const float inv_c = 1.f / (float)a.C;
  float w[NV][W], dw[NV][W];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (li + L * i) * W;
#pragma unroll
    for (int k = 0; k < W; ++k) { w[i][k] = 1.f; dw[i][k] = 0.f; }
    if (a.w && e < a.C) load_f32<W, EVEN>(a.w, e, a.C - e, w[i]);
  }
  for (int64_t row = (int64_t)blockIdx.x * rpb + threadIdx.x / L; ; row += (int64_t)gridDim.x * rpb) {
    if (row - threadIdx.x / L >= a.rows) break;
    const bool live = row < a.rows;
    const float rstd = live ? a.rstd[row] : 0.f;
    float g[NV][W], xh[NV][W];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (li + L * i) * W;
#pragma unroll
      for (int k = 0; k < W; ++k) g[i][k] = xh[i][k] = 0.f;
      if (live && e < a.C) {
        P::load(a.dy, row * a.dys + e, a.C - e, g[i]);
        load_sum<T, EVEN>(a, row, e, xh[i]);
      }
#pragma unroll
      for (int k = 0; k < W; ++k) {
        xh[i][k] *= rstd;
        dw[i][k] = fmaf(g[i][k], xh[i][k], dw[i][k]);
        g[i][k] *= w[i][k];
        dot = fmaf(g[i][k], xh[i][k], dot);
      }
    }
    const float m = row_sum<L>(dot, red) * inv_c;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (li + L * i) * W;
      if (!live || e >= a.C) continue;
      float d[W];
#pragma unroll
      for (int k = 0; k < W; ++k) d[k] = 0.f;
      if (a.ds) P::load(a.ds, row * a.dss + e, a.C - e, d);
#pragma unroll
      for (int k = 0; k < W; ++k) d[k] = fmaf(rstd, fmaf(-xh[i][k], m, g[i][k]), d[k]);
      P::store(a.dx, row * a.C + e, a.C - e, d);
    }
  }
  if (!a.partial) return;
  if constexpr (L >= 256) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (li + L * i) * W;
#pragma unroll
      for (int k = 0; k < W; ++k)
        if (e + k < a.C) a.partial[(int64_t)blockIdx.x * a.C + e + k] = dw[i][k];
    }
  } else {   // the workgroup's 256 / L rows meet in LDS, one vector index at a time
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < W; ++k) fold[(threadIdx.x / L) * (L * W) + li * W + k] = dw[i][k];
      __syncthreads();
      for (int c = threadIdx.x; c < L * W; c += 256) {
        float t = 0.f;
        for (int r = 0; r < 256 / L; ++r) t += fold[r * (L * W) + c];
        if (L * W * i + c < a.C) a.partial[(int64_t)blockIdx.x * a.C + L * W * i + c] = t;
      }
    }
  }
}

template <typename T, bool EVEN> __global__ __launch_bounds__(256) void rms_bwd_long_kernel(BwdArgs a) {   // dx of rows longer than the registers hold
  typedef Piece<T, EVEN> P;
  constexpr int W = P::W;
  __shared__ float red[4];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float rstd = a.rstd[row];
    auto load = [&](int e, float* g, float* xh) {
      P::load(a.dy, row * a.dys + e, a.C - e, g);
      load_sum<T, EVEN>(a, row, e, xh);
      float w[W];
#pragma unroll
      for (int k = 0; k < W; ++k) w[k] = 1.f;
      if (a.w) load_f32<W, EVEN>(a.w, e, a.C - e, w);
#pragma unroll
      for (int k = 0; k < W; ++k) { g[k] *= w[k]; xh[k] *= rstd; }
    };
    float dot = 0.f;
    for (int e = threadIdx.x * W; e < a.C; e += 256 * W) {
      float g[W], xh[W];
      load(e, g, xh);
#pragma unroll
      for (int k = 0; k < W; ++k) dot = fmaf(g[k], xh[k], dot);
    }
    const float m = row_sum<256>(dot, red) / (float)a.C;
    for (int e = threadIdx.x * W; e < a.C; e += 256 * W) {
      float g[W], xh[W], d[W];
      load(e, g, xh);
#pragma unroll
      for (int k = 0; k < W; ++k) d[k] = 0.f;
      if (a.ds) P::load(a.ds, row * a.dss + e, a.C - e, d);
#pragma unroll
      for (int k = 0; k < W; ++k) d[k] = fmaf(rstd, fmaf(-xh[k], m, g[k]), d[k]);
      P::store(a.dx, row * a.C + e, a.C - e, d);
    }
  }
}
// and their dw: a thread per column, gridDim.y slabs of rows
template <typename T> __global__ __launch_bounds__(256) void rms_dw_long_kernel(BwdArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  float t = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float v = load_elem<T>(a.x, row * a.xs + c);
    if (a.res) v += load_elem<T>(a.res, row * a.rs + c);
    t = fmaf(load_elem<T>(a.dy, row * a.dys + c), v * a.rstd[row], t);
  }
  a.partial[(int64_t)blockIdx.y * a.C + c] = t;
}

// dw[c] = sum over the n partial rows: 16 columns a workgroup, thread (slice, 4 columns) adds every 256th row with four loads in flight, the slices of
// a wave meet in a tree and the waves in order (64 columns a workgroup and 64 slices, single elements for an odd C: 8.5 us for 512 rows of
// 1001; 3.7 so.  One thread per column and 16 slices waited for each of its loads: 16.6 us for 1024 rows of 64)
__global__ __launch_bounds__(1024) void rms_dw_fold_kernel(const float* partial, float* dw, int n, int C) {
  __shared__ float t[16][16];
  const int q = (threadIdx.x & 3) * 4, c = blockIdx.x * 16 + q;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = threadIdx.x >> 2; i < n && c < C; i += 256 * 4) {
    float w[4][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[k][e] = 0.f;
      if (i + 256 * k < n) load_f32<4, false>(partial + (int64_t)(i + 256 * k) * C, c, C - c, w[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += w[k][e];
  }
#pragma unroll
  for (int o = 4; o < 64; o <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += __shfl_xor(v[e], o, 64);
  if ((threadIdx.x & 63) < 4)
#pragma unroll
    for (int e = 0; e < 4; ++e) t[threadIdx.x >> 6][q + e] = v[e];
  __syncthreads();
  if (threadIdx.x < 16 && blockIdx.x * 16 + threadIdx.x < C) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) sum += t[k][threadIdx.x];
    dw[blockIdx.x * 16 + threadIdx.x] = sum;
  }
}

constexpr int kMaxGrid = 1 << 20;      // (forward) workgroups; rows beyond are walked
constexpr int kBwdGrid = 512;         // (backward) workgroups = partial rows of dw
constexpr int kMaxChannels = 1 << 30;  // channel indices, and a workgroup's step beyond the last one, are 32-bit

struct Shape { int L, NV; };           // lanes of a row and 16-byte pieces of a lane; 0: the long form
inline Shape pick(int pieces) {
  if (pieces <= 8) return {8, 1};
  if (pieces <= 16) return {16, 1};
  if (pieces <= 32) return {32, 1};
  if (pieces <= 64) return {64, 1};
  if (pieces <= 128) return {64, 2};
  if (pieces <= 256) return {64, 4};
  if (pieces <= 512) return {256, 2};
  if (pieces <= 1024) return {256, 4};
  return {0, 0};
}
inline int bwd_grid(int64_t rows, int L) {
  const int64_t rpb = L ? 256 / L : 1, n = (rows + rpb - 1) / rpb;
  return (int)(n < kBwdGrid ? n : kBwdGrid);
}
#define TG_RMS_SHAPES TG_RMS(8, 1) TG_RMS(16, 1) TG_RMS(32, 1) TG_RMS(64, 1) TG_RMS(64, 2) TG_RMS(64, 4) TG_RMS(256, 2) TG_RMS(256, 4)

template <typename T, bool EVEN, bool Q8> int launch_fwd(const FwdArgs& a, hipStream_t st) {
  constexpr int W = Piece<T, EVEN>::W;
  const Shape sh = pick((a.C + W - 1) / W);
  const int64_t rpb = sh.L ? 256 / sh.L : 1, need = (a.rows + rpb - 1) / rpb;
  const int grid = (int)(need < kMaxGrid ? need : kMaxGrid);
#define TG_RMS(LL, NN) if (sh.L == LL && sh.NV == NN) { rms_fwd_kernel<T, EVEN, LL, NN, Q8><<<grid, 256, 0, st>>>(a); return tg_launch_status(); }
  TG_RMS_SHAPES
#undef TG_RMS
  rms_fwd_long_kernel<T, EVEN, Q8><<<grid, 256, 0, st>>>(a);
  return tg_launch_status();
}

template <typename T, bool EVEN> int launch_bwd(const BwdArgs& a, float* dw, hipStream_t st) {
  constexpr int W = Piece<T, EVEN>::W;
  const Shape sh = pick((a.C + W - 1) / W);
  const int grid = bwd_grid(a.rows, sh.L);
  auto go = [&]() -> int {
#define TG_RMS(LL, NN) if (sh.L == LL && sh.NV == NN) { rms_bwd_kernel<T, EVEN, LL, NN><<<grid, 256, 0, st>>>(a); return tg_launch_status(); }
    TG_RMS_SHAPES
#undef TG_RMS
    rms_bwd_long_kernel<T, EVEN><<<grid, 256, 0, st>>>(a);
    if (a.partial) rms_dw_long_kernel<T><<<dim3((a.C + 255) / 256, grid), 256, 0, st>>>(a);
    return tg_launch_status();
  };
  const int rc = go();
  if (rc != TG_OK || !dw) return rc;
  rms_dw_fold_kernel<<<(a.C + 15) / 16, 1024, 0, st>>>(a.partial, dw, grid, a.C);
  return tg_launch_status();
}

inline int elem_bytes(int dtype) { return dtype == TG_F32 ? 4 : 2; }
inline bool known(int dtype) { return dtype == TG_F32 || dtype == TG_BF16 || dtype == TG_F16; }
inline bool elem_aligned(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (elem_bytes(dtype) - 1)) == 0; }
inline bool wide(int dtype, int C, int64_t stride, const void* p) {   // 16-byte accesses possible for this operand?
  const int n = 16 / elem_bytes(dtype);
  return !p || (C % n == 0 && stride % n == 0 && tg_aligned16(p));
}

template <bool Q8>
int rms_fwd(int dtype, const FwdArgs& a, hipStream_t st) {
  if (!known(dtype) || a.rows < 0 || a.C <= 0 || a.xs < 0 || a.rs < 0 || !(a.eps >= 0.f)) return TG_E_BADARG;
  if (a.C > kMaxChannels) return TG_E_UNSUPPORTED;
  if (a.rows == 0) return TG_OK;
  if (!a.x || !a.y || (Q8 && !a.scale)) return TG_E_BADARG;
  if (!elem_aligned(a.x, dtype) || !elem_aligned(a.res, dtype) || !elem_aligned(a.s, dtype) || (!Q8 && !elem_aligned(a.y, dtype)) ||
      (reinterpret_cast<uintptr_t>(a.w) & 3) || (reinterpret_cast<uintptr_t>(a.rstd) & 3) || (reinterpret_cast<uintptr_t>(a.scale) & 3))
    return TG_E_ALIGN;
  const bool v = wide(dtype, a.C, a.xs, a.x) && wide(dtype, a.C, a.rs, a.res) && wide(dtype, a.C, a.C, a.s) && wide(dtype, a.C, a.C, a.y) &&
                 (!a.w || tg_aligned16(a.w));
  TG_DISPATCH_DTYPE(dtype, return v ? (launch_fwd<BF16, true, Q8>(a, st)) : (launch_fwd<BF16, false, Q8>(a, st)),
                    return v ? (launch_fwd<F16, true, Q8>(a, st)) : (launch_fwd<F16, false, Q8>(a, st)),
                    return v ? (launch_fwd<F32, true, Q8>(a, st)) : (launch_fwd<F32, false, Q8>(a, st)));
}

}  // namespace

extern "C" int tg_rms_norm(int dtype, const void* x, int64_t x_stride, const void* res, int64_t res_stride, const float* weight, void* y,
                           void* s, float* rstd, int64_t rows, int C, float eps, void* stream) {
  return rms_fwd<false>(dtype, FwdArgs{x, res, weight, y, s, rstd, nullptr, x_stride, res_stride, rows, C, eps}, (hipStream_t)stream);
}

extern "C" int tg_rms_norm_e4m3(int dtype, const void* x, int64_t x_stride, const void* res, int64_t res_stride, const float* weight,
                                void* q, float* scale, void* s, int64_t rows, int C, float eps, void* stream) {
  return rms_fwd<true>(dtype, FwdArgs{x, res, weight, q, s, nullptr, scale, x_stride, res_stride, rows, C, eps}, (hipStream_t)stream);
}

extern "C" int64_t tg_rms_norm_bwd_scratch_floats(int64_t rows, int C) {
  if (rows <= 0 || C <= 0) return 0;
  return (rows < kBwdGrid ? rows : kBwdGrid) * (int64_t)C;
}

extern "C" int tg_rms_norm_bwd(int dtype, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* res,
                               int64_t res_stride, const float* rstd, const float* weight, const void* ds, int64_t ds_stride, void* dx,
                               float* dweight, float* scratch, int64_t rows, int C, void* stream) {
  if (!known(dtype) || rows < 0 || C <= 0 || dy_stride < 0 || x_stride < 0 || res_stride < 0 || ds_stride < 0 || (dweight && rows && !scratch))
    return TG_E_BADARG;
  if (C > kMaxChannels) return TG_E_UNSUPPORTED;
  const BwdArgs a{dy, x, res, ds, rstd, weight, dx, dweight ? scratch : nullptr, dy_stride, x_stride, res_stride, ds_stride, rows, C};
  hipStream_t st = (hipStream_t)stream;
  if (rows == 0) {   // the gradient of no rows
    if (dweight) rms_dw_fold_kernel<<<(C + 15) / 16, 1024, 0, st>>>(nullptr, dweight, 0, C);
    return tg_launch_status();
  }
  if (!dy || !x || !rstd || !dx) return TG_E_BADARG;
  if (!elem_aligned(dy, dtype) || !elem_aligned(x, dtype) || !elem_aligned(res, dtype) || !elem_aligned(ds, dtype) || !elem_aligned(dx, dtype) ||
      ((reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(rstd) | reinterpret_cast<uintptr_t>(dweight) |
        reinterpret_cast<uintptr_t>(scratch)) & 3))
    return TG_E_ALIGN;
  const bool v = wide(dtype, C, dy_stride, dy) && wide(dtype, C, x_stride, x) && wide(dtype, C, res_stride, res) && wide(dtype, C, ds_stride, ds) &&
                 wide(dtype, C, C, dx) && (!weight || tg_aligned16(weight));
  TG_DISPATCH_DTYPE(dtype, return v ? (launch_bwd<BF16, true>(a, dweight, st)) : (launch_bwd<BF16, false>(a, dweight, st)),
                    return v ? (launch_bwd<F16, true>(a, dweight, st)) : (launch_bwd<F16, false>(a, dweight, st)),
                    return v ? (launch_bwd<F32, true>(a, dweight, st)) : (launch_bwd<F32, false>(a, dweight, st)));
}
