// Linear attention with a decay for each head.  Per sequence and head, with g = exp(log_decay) and a state S of Dk x Dv floats:
//
//   S_t = g S_{t-1} + k_t v_t^T            o_t = scale q_t S_t                                    (single tokens: la_step_kernel)
//
// and for 16 tokens at a time (i, j inside the chunk, S the state in front of it, n its tokens):
//
//   o_i = scale ( g^{i+1} q_i S  +  sum_{j <= i} g^{i-j} (q_i . k_j) v_j )         S' = g^n S + sum_j g^{n-1-j} k_j v_j^T
//
// The three gradients are the same sums with the operands in other places (do: the gradient of o, dS: of the state, running backwards):
//
//   dq_i = scale (g^{i+1} do_i S^T + sum_{j <= i} g^{i-j} (do_i . v_j) k_j)                      - forward in time, a = do, b = v, c = k
//   dk_j = g^{n-1-j} v_j dS^T + scale sum_{i >= j} g^{i-j} (v_j . do_i) q_i                       - backward in time, a = v, b = do, c = q
//   dv_j = g^{n-1-j} k_j dS   + scale sum_{i >= j} g^{i-j} (k_j . q_i) do_i                       - backward in time, a = k, b = q, c = do
//
// so ONE kernel serves all four: out_i = za g^{i+1-sh} a_i S + scale sum_{j<=i} g^{i-j} (a_i . b_j) c_j,
// S' = g^n S + zs sum_j g^{n-1-j+sh} b_j c_j^T over tokens taken forwards (sh = 0, za = scale, zs = 1) or backwards (sh = 1, za = 1, zs = scale).
//
// Layout: a wave owns 16 columns of c (and of S and out) of one sequence and head.  Everything is made of 16 x 16 tiles in the matrix
// instructions' own shape: lane (c = lane % 16, g = lane / 16) holds 4 consecutive values 4g .. 4g+3 of row / column c.  An accumulator
// tile X[k][c] has the shape of an operand with c along its free dimension and k along the summed one, so the scores (b a^T, tile [j][i])
// and the state (tiles [m][n]) go from accumulators to operands without leaving the registers.
//
// Rounding: raw inputs are multiplied as they are (exact products, fp32 sums).  Scores and state are fp32; as operands beside 16-bit
// inputs they are split into TWO bf16 halves (hi + lo: 16 bits of mantissa) instead of one rounding to 8 bits - the products cost twice
// the matrix instructions of a kernel that waits for memory, and the result is off by its own last rounding alone.  fp16 inputs are
// split the same way beside them (exactly: 11 bits), because a score or a state may pass fp16's range.  What is ADDED to the state is
// split into three (24 bits): the state leaves in fp32 and is as exact as one summed in fp32.  fp32 inputs run on the fp32 matrix
// instructions.
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

// ---- one 16 x 16 x 16 product: operand types Raw<T> (inputs) and Split<T> (computed floats)
template <typename T> struct Mat;
template <> struct Mat<F32> {
  typedef f32x4 Raw;
  typedef f32x4 Split;
  typedef f32x4 Split3;
  __device__ __forceinline__ static Split split(f32x4 v) { return v; }
  __device__ __forceinline__ static Split3 split3(f32x4 v) { return v; }
  __device__ __forceinline__ static f32x4 raw_split3(Raw a, Split3 b, f32x4 c) { return raw_raw(a, b, c); }
  __device__ __forceinline__ static f32x4 raw_raw(Raw a, Raw b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static f32x4 raw_split(Raw a, Split b, f32x4 c) { return raw_raw(a, b, c); }
  __device__ __forceinline__ static f32x4 split_raw(Split a, Raw b, f32x4 c) { return raw_raw(a, b, c); }
  __device__ __forceinline__ static f32x4 to_float(Raw v) { return v; }
};
struct Halves { s16x4 hi, lo; };
__device__ __forceinline__ f32x4 mma_bf16(s16x4 a, s16x4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0); }
__device__ __forceinline__ Halves halves(f32x4 v) {
  Halves h;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const unsigned short b = f32_to_bf16_bits(v[e]);
    h.hi[e] = (short)b;
    h.lo[e] = (short)f32_to_bf16_bits(v[e] - bf16_bits_to_f32(b));
  }
  return h;
}
struct Thirds { s16x4 hi, mid, lo; };
__device__ __forceinline__ Thirds thirds(f32x4 v) {
  Thirds h;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const unsigned short a = f32_to_bf16_bits(v[e]);
    const float r = v[e] - bf16_bits_to_f32(a);
    const unsigned short b = f32_to_bf16_bits(r);
    h.hi[e] = (short)a;
    h.mid[e] = (short)b;
    h.lo[e] = (short)f32_to_bf16_bits(r - bf16_bits_to_f32(b));
  }
  return h;
}
template <> struct Mat<BF16> {
  typedef s16x4 Raw;
  typedef Halves Split;
  typedef Thirds Split3;
  __device__ __forceinline__ static Split3 split3(f32x4 v) { return thirds(v); }
  __device__ __forceinline__ static f32x4 raw_split3(Raw a, Split3 b, f32x4 c) { return mma_bf16(a, b.hi, mma_bf16(a, b.mid, mma_bf16(a, b.lo, c))); }
  __device__ __forceinline__ static Split split(f32x4 v) { return halves(v); }
  __device__ __forceinline__ static f32x4 raw_raw(Raw a, Raw b, f32x4 c) { return mma_bf16(a, b, c); }
  __device__ __forceinline__ static f32x4 raw_split(Raw a, Split b, f32x4 c) { return mma_bf16(a, b.hi, mma_bf16(a, b.lo, c)); }
  __device__ __forceinline__ static f32x4 split_raw(Split a, Raw b, f32x4 c) { return mma_bf16(a.hi, b, mma_bf16(a.lo, b, c)); }
  __device__ __forceinline__ static f32x4 to_float(Raw v) {
    f32x4 f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = bf16_bits_to_f32((unsigned short)v[e]);
    return f;
  }
};
template <> struct Mat<F16> {
  typedef s16x4 Raw;
  typedef Halves Split;
  typedef Thirds Split3;
  __device__ __forceinline__ static Split3 split3(f32x4 v) { return thirds(v); }
  __device__ __forceinline__ static f32x4 raw_split3(Raw a, Split3 b, f32x4 c) {   // (lo * lo: below 24 bits)
    const Halves h = halves(to_float(a));
    return mma_bf16(h.hi, b.hi, mma_bf16(h.hi, b.mid, mma_bf16(h.lo, b.hi, mma_bf16(h.hi, b.lo, mma_bf16(h.lo, b.mid, c)))));
  }
  __device__ __forceinline__ static Split split(f32x4 v) { return halves(v); }
  __device__ __forceinline__ static f32x4 to_float(Raw v) {
    f32x4 f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = f16_bits_to_f32((unsigned short)v[e]);
    return f;
  }
  __device__ __forceinline__ static f32x4 raw_raw(Raw a, Raw b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
  __device__ __forceinline__ static f32x4 both(Halves a, Halves b, f32x4 c) { return mma_bf16(a.hi, b.hi, mma_bf16(a.hi, b.lo, mma_bf16(a.lo, b.hi, c))); }
  __device__ __forceinline__ static f32x4 raw_split(Raw a, Split b, f32x4 c) { return both(halves(to_float(a)), b, c); }
  __device__ __forceinline__ static f32x4 split_raw(Split a, Raw b, f32x4 c) { return both(a, halves(to_float(b)), c); }
};

// 4 consecutive elements at p + i; `wide`: one load (the address is aligned to 4 elements), n: how many of them exist
template <typename T> __device__ __forceinline__ typename Mat<T>::Raw load4(const void* p, int64_t i, int n, bool wide) {
  typename Mat<T>::Raw v = {0, 0, 0, 0};
  if constexpr (ElemTraits<T>::kBytes == 4) {
    const float* f = reinterpret_cast<const float*>(p) + i;
    if (wide && n >= 4) return *reinterpret_cast<const f32x4*>(f);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) v[e] = f[e];
  } else {
    const short* f = reinterpret_cast<const short*>(p) + i;
    if (wide && n >= 4) return *reinterpret_cast<const s16x4*>(f);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) v[e] = f[e];
  }
  return v;
}
template <typename T> __device__ __forceinline__ void put(typename Mat<T>::Raw& v, int e, const void* p, int64_t i) {
  if constexpr (ElemTraits<T>::kBytes == 4) v[e] = reinterpret_cast<const float*>(p)[i];
  else v[e] = reinterpret_cast<const short*>(p)[i];
}

struct Operand { const void* p; int64_t sb, st, sh; int shared; int wide; };   // element strides of sequence, token, head; heads per stored head; 4-element loads possible

struct LaArgs {
  Operand a, b, c;
  void* out;               // [B][T][H][N], element type T, or float where out_f32
  const float* s0;         // first state, or null: zeros
  float* s1;               // last state, or null
  const float* log_decay;  // [H]
  const int* lengths;      // [B], or null
  int B, T, H, M, N;
  int64_t sm, sn;          // strides of m and n inside one state of M x N floats (the transposed roles read S^T)
  float za, zs, scale;
  int sh, reverse, out_f32, out_wide;
};

__device__ __forceinline__ float decay_pow(float la, int n) { return n == 0 ? 1.f : expf(la * (float)n); }   // (0 * -inf: g = 0 is a decay too)

template <typename T, int MT> __global__ __launch_bounds__(256) void la_wave_kernel(LaArgs p) {
  typedef Mat<T> X;
  typedef typename X::Raw Raw;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int slices = (p.N + 15) / 16;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= (int64_t)p.B * p.H * slices) return;   // (whole waves; no barrier below)
  const int slice = (int)(unit % slices), h = (int)(unit / slices % p.H);
  const int64_t bi = unit / slices / p.H;
  const int n = p.lengths ? min(max(p.lengths[bi], 0), p.T) : p.T;
  const float la = p.log_decay[h];
  const int64_t oa = bi * p.a.sb + (h / p.a.shared) * p.a.sh, ob = bi * p.b.sb + (h / p.b.shared) * p.b.sh, oc = bi * p.c.sb + (h / p.c.shared) * p.c.sh;
  const int col = slice * 16 + c;                       // this lane's column of c, S and the state
  const bool has_col = col < p.N;
  const int64_t state = ((int64_t)bi * p.H + h) * p.M * p.N;

  f32x4 S[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    S[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (p.s0 && has_col)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (16 * t + 4 * g + e < p.M) S[t][e] = p.s0[state + (16 * t + 4 * g + e) * p.sm + col * p.sn];
  }
  f32x4 inside, into;                                    // scale g^{i-j} (0 above the diagonal), i = c, j = 4g + e;  zs g^{15-j+sh}
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int j = 4 * g + e;
    inside[e] = j <= c ? p.scale * decay_pow(la, c - j) : 0.f;
    into[e] = p.zs * decay_pow(la, 15 - j + p.sh);
  }
  const float from = p.za * decay_pow(la, c + 1 - p.sh);
  float keep1 = expm1f(la * 16.f);                       // g^16 - 1: S + (g^16 - 1) S keeps slow decays' last bits

  for (int t0 = 0; t0 < p.T; t0 += 16) {
    const int cnt = min(16, n - t0);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const int ti = p.reverse ? n - 1 - (t0 + c) : t0 + c;   // token of this lane's row of a / b and column of out (valid if c < cnt)
    if (cnt > 0) {
      if (cnt < 16) {
        keep1 = expm1f(la * (float)cnt);
#pragma unroll
        for (int e = 0; e < 4; ++e) into[e] = 4 * g + e < cnt ? p.zs * decay_pow(la, cnt - 1 - (4 * g + e) + p.sh) : 0.f;
      }
      // c's tile: column `col`, tokens 4g .. 4g+3; and the tile weighted for the state
      Raw cv = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = t0 + 4 * g + e;
        if (4 * g + e < cnt && has_col) put<T>(cv, e, p.c.p, oc + (int64_t)(p.reverse ? n - 1 - j : j) * p.c.st + col);
      }
      f32x4 scores = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int m = 16 * t + 4 * g;
        Raw av = {0, 0, 0, 0}, bv = {0, 0, 0, 0};
        if (c < cnt && m < p.M) {
          av = load4<T>(p.a.p, oa + (int64_t)ti * p.a.st + m, p.M - m, p.a.wide);
          bv = load4<T>(p.b.p, ob + (int64_t)ti * p.b.st + m, p.M - m, p.b.wide);
        }
        scores = X::raw_raw(bv, av, scores);             // [j][i] = b_j . a_i
        acc = X::split_raw(X::split(S[t]), av, acc);     // [n][i] += S[m][n] a_i[m]
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[e] *= from;
        scores[e] = 4 * g + e <= c ? scores[e] * inside[e] : 0.f;
      }
      const typename X::Split ps = X::split(scores);
      // a later token's infinity or NaN in c must not reach an earlier token's sum as 0 * inf: such a chunk goes token by token
      const f32x4 cf = X::to_float(cv);
      bool odd = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) odd |= !(__builtin_fabsf(cf[e]) <= 3.4028234e38f);
      if (__builtin_expect(__any(odd), 0)) {
        const f32x4 before = acc;
        for (int i = 0; i < cnt; ++i) {
          Raw only = cv;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * g + e > i) only[e] = 0;
          const f32x4 r = X::raw_split(only, ps, before);
          if (c == i) acc = r;
        }
      } else {
        acc = X::raw_split(cv, ps, acc);                 // [n][i] += c_j[n] scores[j][i]
      }
      f32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = cf[e] * into[e];
      const typename X::Split3 ws = X::split3(w);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        Raw bt = {0, 0, 0, 0};                           // b's tile the other way: row m = 16 t + c, tokens 4g .. 4g+3
        const int m = 16 * t + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = t0 + 4 * g + e;
          if (4 * g + e < cnt && m < p.M) put<T>(bt, e, p.b.p, ob + (int64_t)(p.reverse ? n - 1 - j : j) * p.b.st + m);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) S[t][e] = fmaf(S[t][e], keep1, S[t][e]);
        S[t] = X::raw_split3(bt, ws, S[t]);              // [m][n] += b_j[m] (w_j c_j[n])
      }
    }
    // tokens behind the sequence's length get zeros
    const int to = c < cnt ? ti : t0 + c;
    const int n0 = slice * 16 + 4 * g;
    if (t0 + c < p.T && n0 < p.N) {
      if (c >= cnt) acc = f32x4{0.f, 0.f, 0.f, 0.f};
      const int64_t at = (((int64_t)bi * p.T + to) * p.H + h) * p.N + n0;
      if (p.out_f32 || ElemTraits<T>::kBytes == 4) {
        float* o = reinterpret_cast<float*>(p.out) + at;
        if (p.out_wide) *reinterpret_cast<f32x4*>(o) = acc;
        else
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n0 + e < p.N) o[e] = acc[e];
      } else if constexpr (ElemTraits<T>::kBytes == 2) {
        s16x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (short)f32_to_bits16<T>(acc[e]);
        short* o = reinterpret_cast<short*>(p.out) + at;
        if (p.out_wide) *reinterpret_cast<s16x4*>(o) = r;
        else
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n0 + e < p.N) o[e] = r[e];
      }
    }
  }
  if (p.s1 && has_col)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (16 * t + 4 * g + e < p.M) p.s1[state + (16 * t + 4 * g + e) * p.sm + col * p.sn] = S[t][e];
}

// gradient of a shared head: the sum of its `share` heads' gradients, in order: in [rows][H][D] floats -> out [rows][H / share][D]
template <typename T> __global__ __launch_bounds__(256) void la_share_kernel(const float* in, void* out, int64_t rows, int heads, int share, int D) {
  const int64_t total = rows * heads * D;   // (heads: of the output)
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int d = (int)(i % D);
    const int64_t rh = i / D;               // row * heads + head
    float t = 0.f;
    for (int s = 0; s < share; ++s) t += in[(rh * share + s) * D + d];
    store_elem<T>(out, i, t);
  }
}

struct StepArgs {
  const void *q, *k, *v;
  void* o;
  float* state;
  const float* log_decay;
  int64_t qb, qh, kb, kh, vb, vh;   // element strides of sequence and head
  int64_t units;                    // B H
  int H, share, M, N;
  float scale;
};

// one token: a wave per sequence and head, W floats of a state row per lane, 64 / LN rows at a time
template <typename T, int W> __global__ __launch_bounds__(256) void la_step_kernel(StepArgs p) {
  const int lane = threadIdx.x & 63;
  const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (u >= p.units) return;
  const int h = (int)(u % p.H);
  const int64_t bi = u / p.H;
  int LN = 1;
  while (LN < 64 && LN * W < p.N) LN *= 2;
  const int ln = lane & (LN - 1), lm = lane / LN, rows = 64 / LN;
  const float decay = expf(p.log_decay[h]);
  const int64_t oq = bi * p.qb + h * p.qh, ok = bi * p.kb + h / p.share * p.kh, ov = bi * p.vb + h / p.share * p.vh;
  float* S = p.state + u * p.M * p.N;
  for (int n = ln * W; n < ((p.N + W * LN - 1) / (W * LN)) * W * LN; n += W * LN) {
    const bool live = n < p.N;
    float v[W], acc[W];
#pragma unroll
    for (int e = 0; e < W; ++e) { v[e] = live ? load_elem<T>(p.v, ov + n + e) : 0.f; acc[e] = 0.f; }
    for (int m = lm; m < p.M; m += rows) {
      const float k = load_elem<T>(p.k, ok + m), q = load_elem<T>(p.q, oq + m);
      if (live) {
        float s[W];
        float* at = S + (int64_t)m * p.N + n;
        if constexpr (W == 4) Vec<F32>::load(at, s); else s[0] = at[0];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          s[e] = fmaf(decay, s[e], k * v[e]);
          acc[e] = fmaf(q, s[e], acc[e]);
        }
        if constexpr (W == 4) Vec<F32>::store(at, s); else at[0] = s[0];
      }
    }
#pragma unroll
    for (int e = 0; e < W; ++e) {
      for (int o = 32; o >= LN; o >>= 1) acc[e] += __shfl_xor(acc[e], o, 64);
      if (live && lm == 0) store_elem<T>(p.o, u * p.N + n + e, acc[e] * p.scale);
    }
  }
}

inline bool known(int dtype) { return dtype == TG_F32 || dtype == TG_BF16 || dtype == TG_F16; }
inline int elem_bytes(int dtype) { return dtype == TG_F32 ? 4 : 2; }
inline bool elem_aligned(int dtype, const void* p) { return (reinterpret_cast<uintptr_t>(p) & (elem_bytes(dtype) - 1)) == 0; }
inline bool word_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

template <typename T> int launch_wave(const LaArgs& a, hipStream_t st) {
  const int64_t units = (int64_t)a.B * a.H * ((a.N + 15) / 16), wgs = (units + 3) / 4;
  if (wgs > 0x7fffffff) return TG_E_UNSUPPORTED;
  const int mt = (a.M + 15) / 16;
  if (mt <= 1) la_wave_kernel<T, 1><<<(int)wgs, 256, 0, st>>>(a);
  else if (mt <= 2) la_wave_kernel<T, 2><<<(int)wgs, 256, 0, st>>>(a);
  else if (mt <= 4) la_wave_kernel<T, 4><<<(int)wgs, 256, 0, st>>>(a);
  else la_wave_kernel<T, 8><<<(int)wgs, 256, 0, st>>>(a);
  return tg_launch_status();
}
int launch_la(int dtype, const LaArgs& a, hipStream_t st) {
  TG_DISPATCH_DTYPE(dtype, return launch_wave<BF16>(a, st), return launch_wave<F16>(a, st), return launch_wave<F32>(a, st));
}

constexpr int kMaxHead = 128;

Operand operand(int dtype, const void* p, const int64_t* stride, int shared) {
  const int bytes = 4 * elem_bytes(dtype);
  const bool wide = ((reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0) && stride[0] % 4 == 0 && stride[1] % 4 == 0 && stride[2] % 4 == 0;
  return Operand{p, stride[0], stride[1], stride[2], shared, wide};
}

int check(int dtype, const tg_la_desc* d) {
  if (!d || !known(dtype) || d->B < 0 || d->T < 0 || d->H <= 0 || d->HK <= 0 || d->DK <= 0 || d->DV <= 0) return TG_E_BADARG;
  if (d->H % d->HK || d->DK > kMaxHead || d->DV > kMaxHead) return TG_E_UNSUPPORTED;
  return TG_OK;
}

}  // namespace

extern "C" int tg_linear_attention(int dtype, const tg_la_desc* d, const void* q, const void* k, const void* v, const float* log_decay,
                                   const int32_t* lengths, const float* state_in, void* o, float* state_out, void* stream) {
  const int rc = check(dtype, d);
  if (rc != TG_OK) return rc;
  if (d->B == 0) return TG_OK;
  if (!log_decay || !state_out || (d->T > 0 && (!q || !k || !v || !o))) return TG_E_BADARG;
  if (!elem_aligned(dtype, q) || !elem_aligned(dtype, k) || !elem_aligned(dtype, v) || !elem_aligned(dtype, o) || !word_aligned(log_decay) ||
      !word_aligned(lengths) || !word_aligned(state_in) || !word_aligned(state_out))
    return TG_E_ALIGN;
  const int G = d->H / d->HK;
  LaArgs a{};
  a.a = operand(dtype, q, d->q_stride, 1);
  a.b = operand(dtype, k, d->k_stride, G);
  a.c = operand(dtype, v, d->v_stride, G);
  a.out = o;
  a.s0 = state_in;
  a.s1 = state_out;
  a.log_decay = log_decay;
  a.lengths = lengths;
  a.B = d->B; a.T = d->T; a.H = d->H; a.M = d->DK; a.N = d->DV;
  a.sm = d->DV; a.sn = 1;
  a.za = a.scale = d->scale;
  a.zs = 1.f;
  a.out_wide = d->DV % 4 == 0 && (reinterpret_cast<uintptr_t>(o) & (4 * elem_bytes(dtype) - 1)) == 0;
  return launch_la(dtype, a, (hipStream_t)stream);
}

extern "C" int64_t tg_linear_attention_bwd_scratch_floats(const tg_la_desc* d) {
  if (check(TG_F32, d) != TG_OK) return 0;
  return d->H == d->HK ? 0 : (int64_t)d->B * d->T * d->H * (d->DK + d->DV);
}

extern "C" int tg_linear_attention_bwd(int dtype, const tg_la_desc* d, const void* q, const void* k, const void* v, const void* dout,
                                       const int64_t* dout_stride, const float* log_decay, const int32_t* lengths, const float* state_in,
                                       const float* dstate_out, void* dq, void* dk, void* dv, float* dstate_in, float* scratch, void* stream) {
  int rc = check(dtype, d);
  if (rc != TG_OK) return rc;
  if (d->B == 0) return TG_OK;
  const int G = d->H / d->HK;
  if (!log_decay || !dout_stride || (d->T > 0 && (!q || !k || !v || !dout || !dq || !dk || !dv || (G > 1 && !scratch)))) return TG_E_BADARG;
  if (!elem_aligned(dtype, q) || !elem_aligned(dtype, k) || !elem_aligned(dtype, v) || !elem_aligned(dtype, dout) || !elem_aligned(dtype, dq) ||
      !elem_aligned(dtype, dk) || !elem_aligned(dtype, dv) || !word_aligned(log_decay) || !word_aligned(lengths) || !word_aligned(state_in) ||
      !word_aligned(dstate_out) || !word_aligned(dstate_in) || !word_aligned(scratch))
    return TG_E_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  const Operand Q = operand(dtype, q, d->q_stride, 1), K = operand(dtype, k, d->k_stride, G), V = operand(dtype, v, d->v_stride, G),
                D = operand(dtype, dout, dout_stride, 1);
  LaArgs a{};
  a.log_decay = log_decay;
  a.lengths = lengths;
  a.B = d->B; a.T = d->T; a.H = d->H;
  a.scale = d->scale;
  auto wide = [&](const void* p, int n, int bytes) { return n % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & (4 * bytes - 1)) == 0; };
  // dq: forwards, the state read transposed
  a.a = D; a.b = V; a.c = K; a.out = dq; a.s0 = state_in; a.s1 = nullptr; a.M = d->DV; a.N = d->DK; a.sm = 1; a.sn = d->DV;
  a.za = d->scale; a.zs = 1.f; a.sh = 0; a.reverse = 0; a.out_f32 = 0; a.out_wide = wide(dq, d->DK, elem_bytes(dtype));
  if ((rc = launch_la(dtype, a, st)) != TG_OK) return rc;
  // dv: backwards
  float* sv = scratch;
  float* sk = G > 1 ? scratch + (int64_t)d->B * d->T * d->H * d->DV : nullptr;
  a.a = K; a.b = Q; a.c = D; a.out = G > 1 ? (void*)sv : dv; a.s0 = dstate_out; a.s1 = dstate_in; a.M = d->DK; a.N = d->DV; a.sm = d->DV; a.sn = 1;
  a.za = 1.f; a.zs = d->scale; a.sh = 1; a.reverse = 1; a.out_f32 = G > 1; a.out_wide = wide(a.out, d->DV, G > 1 ? 4 : elem_bytes(dtype));
  if ((rc = launch_la(dtype, a, st)) != TG_OK) return rc;
  // dk: backwards, the state's gradient read transposed
  a.a = V; a.b = D; a.c = Q; a.out = G > 1 ? (void*)sk : dk; a.s1 = nullptr; a.M = d->DV; a.N = d->DK; a.sm = 1; a.sn = d->DV;
  a.out_wide = wide(a.out, d->DK, G > 1 ? 4 : elem_bytes(dtype));
  if ((rc = launch_la(dtype, a, st)) != TG_OK) return rc;
  if (G > 1 && d->T > 0) {
    const int64_t rows = (int64_t)d->B * d->T;
    for (int w = 0; w < 2; ++w) {
      const int D_ = w ? d->DK : d->DV;
      const int64_t wgs = (rows * d->HK * D_ + 255) / 256;
      const int grid = (int)(wgs < (1 << 20) ? wgs : (1 << 20));
      const float* in = w ? sk : sv;
      void* out = w ? dk : dv;
      if (dtype == TG_BF16) la_share_kernel<BF16><<<grid, 256, 0, st>>>(in, out, rows, d->HK, G, D_);
      else if (dtype == TG_F16) la_share_kernel<F16><<<grid, 256, 0, st>>>(in, out, rows, d->HK, G, D_);
      else la_share_kernel<F32><<<grid, 256, 0, st>>>(in, out, rows, d->HK, G, D_);
      if ((rc = tg_launch_status()) != TG_OK) return rc;
    }
  }
  return TG_OK;
}

extern "C" int tg_linear_attention_step(int dtype, const tg_la_desc* d, const void* q, const void* k, const void* v, const float* log_decay,
                                        void* o, float* state, void* stream) {
  const int rc = check(dtype, d);
  if (rc != TG_OK) return rc;
  if (d->B == 0) return TG_OK;
  if (!q || !k || !v || !log_decay || !o || !state) return TG_E_BADARG;
  if (!elem_aligned(dtype, q) || !elem_aligned(dtype, k) || !elem_aligned(dtype, v) || !elem_aligned(dtype, o) || !word_aligned(log_decay) ||
      !word_aligned(state))
    return TG_E_ALIGN;
  StepArgs a{q, k, v, o, state, log_decay, d->q_stride[0], d->q_stride[2], d->k_stride[0], d->k_stride[2], d->v_stride[0], d->v_stride[2],
             (int64_t)d->B * d->H, d->H, d->H / d->HK, d->DK, d->DV, d->scale};
  const int64_t wgs = (a.units + 3) / 4;
  if (wgs > 0x7fffffff) return TG_E_UNSUPPORTED;
  const bool wide = d->DV % 4 == 0 && tg_aligned16(state);
  hipStream_t st = (hipStream_t)stream;
#define TG_STEP(TT) { if (wide) la_step_kernel<TT, 4><<<(int)wgs, 256, 0, st>>>(a); else la_step_kernel<TT, 1><<<(int)wgs, 256, 0, st>>>(a); }
  TG_DISPATCH_DTYPE(dtype, TG_STEP(BF16), TG_STEP(F16), TG_STEP(F32));
#undef TG_STEP
  return tg_launch_status();
}
