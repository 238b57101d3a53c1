// Linear attention with a decay for each head.  Per sequence and head, with g = exp(log_decay) and a state S of Dk x Dv floats:
//
//   S_t = g S_{t-1} + k_t v_t^T            o_t = scale q_t S_t                                    (single tokens: la_step_kernel)
//
// and for a chunk of tokens at a time (i, j inside the chunk, S the state in front of it, n its tokens):
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
// Layout: a wave owns 16 columns of c (and of S and out) of one sequence and head and walks its tokens in chunks of 16 CT.  Everything is
// made of 16 x 16 tiles in the matrix instructions' own shape: lane (c = lane % 16, g = lane / 16) holds 4 consecutive values 4g .. 4g+3
// of row / column c.  An accumulator tile X[k][c] has the shape of an operand with c along its free dimension and k along the summed one,
// so the scores (b a^T, tile [j][i]) and the state (tiles [m][n]) go from accumulators to operands without leaving the registers, and a
// product with the identity turns a tile that was loaded by rows into one by columns (exactly) - no LDS, no second load.
//
// Long sequences: T is cut into segments of `seg` tokens so that a few heads fill the machine.  la_kernel<STATE> sums each segment's own state,
// la_scan_kernel joins them into the state in front of every segment, and the segments then run side by side.
//
// Rounding: raw inputs are multiplied as they are (exact products, fp32 sums).  Scores and state are fp32; as operands beside 16-bit
// inputs they are split into TWO bf16 halves (hi + lo: 16 bits of mantissa) instead of one rounding to 8 bits - the products cost twice
// the matrix instructions of a kernel that waits for memory, and the result is off by its own last rounding alone.  fp16 inputs are
// split the same way beside them (exactly: 11 bits), because a score or a state may pass fp16's range.  What is ADDED to the state is
// split into three (24 bits): the state leaves in fp32 and is as exact as one summed in fp32.  fp32 inputs run on the fp32 matrix
// instructions.
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

// ---- products of 16 x 16 tiles, summed dimension 16 (mma) or 32 (mma2: two tiles of each operand).  Raw: an input as loaded; Op: an input
// beside a computed operand; Split / Split3: a computed operand
__device__ __forceinline__ f32x4 mma_bf16(s16x4 a, s16x4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0); }
__device__ __forceinline__ s16x8 join(s16x4 a, s16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ f32x4 mma2_bf16(s16x4 a0, s16x4 a1, s16x4 b0, s16x4 b1, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, join(a0, a1)), __builtin_bit_cast(bf16x8, join(b0, b1)), c, 0, 0, 0);
}
__device__ __forceinline__ s16x4 to_bf16(f32x4 v) { return __builtin_bit_cast(s16x4, __builtin_convertvector(v, bf16x4)); }
__device__ __forceinline__ f32x4 from_bf16(s16x4 v) {
  const uint2 u = __builtin_bit_cast(uint2, v);
  return f32x4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u)};
}
struct Halves { s16x4 hi, lo; };
struct Thirds { s16x4 hi, mid, lo; };
__device__ __forceinline__ Halves halves(f32x4 v) {
  Halves h;
  h.hi = to_bf16(v);
  h.lo = to_bf16(v - from_bf16(h.hi));
  return h;
}
__device__ __forceinline__ Thirds thirds(f32x4 v) {
  Thirds h;
  h.hi = to_bf16(v);
  const f32x4 r = v - from_bf16(h.hi);
  h.mid = to_bf16(r);
  h.lo = to_bf16(r - from_bf16(h.mid));
  return h;
}

template <typename T> struct Mat;
template <> struct Mat<F32> {
  typedef f32x4 Raw;
  typedef f32x4 Op;
  typedef f32x4 Split;
  typedef f32x4 Split3;
  __device__ __forceinline__ static f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static Raw one(int d) { return Raw{d == 0 ? 1.f : 0.f, d == 1 ? 1.f : 0.f, d == 2 ? 1.f : 0.f, d == 3 ? 1.f : 0.f}; }
  __device__ __forceinline__ static Op op(Raw v) { return v; }
  __device__ __forceinline__ static Op op_of(f32x4 v) { return v; }
  __device__ __forceinline__ static Split split(f32x4 v) { return v; }
  __device__ __forceinline__ static Split3 split3(f32x4 v) { return v; }
  __device__ __forceinline__ static f32x4 raw(Raw a, Raw b, f32x4 c) { return mma(a, b, c); }
  __device__ __forceinline__ static f32x4 raw2(Raw a0, Raw a1, Raw b0, Raw b1, f32x4 c) { return mma(a1, b1, mma(a0, b0, c)); }
  __device__ __forceinline__ static f32x4 state(Split s, Op a, f32x4 c) { return mma(s, a, c); }
  __device__ __forceinline__ static f32x4 state2(Split s0, Split s1, Op a0, Op a1, f32x4 c) { return mma(s1, a1, mma(s0, a0, c)); }
  __device__ __forceinline__ static f32x4 score(Op v, Split p, f32x4 c) { return mma(v, p, c); }
  __device__ __forceinline__ static f32x4 score2(Op v0, Op v1, Split p0, Split p1, f32x4 c) { return mma(v1, p1, mma(v0, p0, c)); }
  __device__ __forceinline__ static f32x4 add(Op b, Split3 w, f32x4 c) { return mma(b, w, c); }
  __device__ __forceinline__ static f32x4 add2(Op b0, Op b1, Split3 w0, Split3 w1, f32x4 c) { return mma(b1, w1, mma(b0, w0, c)); }
  __device__ __forceinline__ static Op upto(Op v, int n) {   // the first n of the 4 values, zeros behind
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? v[e] : 0.f;
    return v;
  }
};
template <> struct Mat<BF16> {
  typedef s16x4 Raw;
  typedef s16x4 Op;
  typedef Halves Split;
  typedef Thirds Split3;
  __device__ __forceinline__ static Raw one(int d) { return Raw{(short)(d == 0 ? 0x3f80 : 0), (short)(d == 1 ? 0x3f80 : 0), (short)(d == 2 ? 0x3f80 : 0), (short)(d == 3 ? 0x3f80 : 0)}; }
  __device__ __forceinline__ static Op op(Raw v) { return v; }
  __device__ __forceinline__ static Op op_of(f32x4 v) { return to_bf16(v); }   // (of values that are bf16)
  __device__ __forceinline__ static Split split(f32x4 v) { return halves(v); }
  __device__ __forceinline__ static Split3 split3(f32x4 v) { return thirds(v); }
  __device__ __forceinline__ static f32x4 raw(Raw a, Raw b, f32x4 c) { return mma_bf16(a, b, c); }
  __device__ __forceinline__ static f32x4 raw2(Raw a0, Raw a1, Raw b0, Raw b1, f32x4 c) { return mma2_bf16(a0, a1, b0, b1, c); }
  __device__ __forceinline__ static f32x4 state(Split s, Op a, f32x4 c) { return mma_bf16(s.hi, a, mma_bf16(s.lo, a, c)); }
  __device__ __forceinline__ static f32x4 state2(Split s0, Split s1, Op a0, Op a1, f32x4 c) { return mma2_bf16(s0.hi, s1.hi, a0, a1, mma2_bf16(s0.lo, s1.lo, a0, a1, c)); }
  __device__ __forceinline__ static f32x4 score(Op v, Split p, f32x4 c) { return mma_bf16(v, p.hi, mma_bf16(v, p.lo, c)); }
  __device__ __forceinline__ static f32x4 score2(Op v0, Op v1, Split p0, Split p1, f32x4 c) { return mma2_bf16(v0, v1, p0.hi, p1.hi, mma2_bf16(v0, v1, p0.lo, p1.lo, c)); }
  __device__ __forceinline__ static f32x4 add(Op b, Split3 w, f32x4 c) { return mma_bf16(b, w.hi, mma_bf16(b, w.mid, mma_bf16(b, w.lo, c))); }
  __device__ __forceinline__ static f32x4 add2(Op b0, Op b1, Split3 w0, Split3 w1, f32x4 c) {
    return mma2_bf16(b0, b1, w0.hi, w1.hi, mma2_bf16(b0, b1, w0.mid, w1.mid, mma2_bf16(b0, b1, w0.lo, w1.lo, c)));
  }
  __device__ __forceinline__ static Op upto(Op v, int n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? v[e] : (short)0;
    return v;
  }
};
template <> struct Mat<F16> {
  typedef s16x4 Raw;
  typedef Halves Op;
  typedef Halves Split;
  typedef Thirds Split3;
  __device__ __forceinline__ static Raw one(int d) { return Raw{(short)(d == 0 ? 0x3c00 : 0), (short)(d == 1 ? 0x3c00 : 0), (short)(d == 2 ? 0x3c00 : 0), (short)(d == 3 ? 0x3c00 : 0)}; }
  __device__ __forceinline__ static Op op(Raw v) { return halves(__builtin_convertvector(__builtin_bit_cast(f16x4, v), f32x4)); }
  __device__ __forceinline__ static Op op_of(f32x4 v) { return halves(v); }
  __device__ __forceinline__ static Split split(f32x4 v) { return halves(v); }
  __device__ __forceinline__ static Split3 split3(f32x4 v) { return thirds(v); }
  __device__ __forceinline__ static f32x4 raw(Raw a, Raw b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
  __device__ __forceinline__ static f32x4 raw2(Raw a0, Raw a1, Raw b0, Raw b1, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, join(a0, a1)), __builtin_bit_cast(f16x8, join(b0, b1)), c, 0, 0, 0);
  }
  // (lo * lo: below 16 bits of the product, and 24 of the state's increment, respectively)
  __device__ __forceinline__ static f32x4 state(Split s, Op a, f32x4 c) { return mma_bf16(s.hi, a.hi, mma_bf16(s.hi, a.lo, mma_bf16(s.lo, a.hi, c))); }
  __device__ __forceinline__ static f32x4 state2(Split s0, Split s1, Op a0, Op a1, f32x4 c) {
    return mma2_bf16(s0.hi, s1.hi, a0.hi, a1.hi, mma2_bf16(s0.hi, s1.hi, a0.lo, a1.lo, mma2_bf16(s0.lo, s1.lo, a0.hi, a1.hi, c)));
  }
  __device__ __forceinline__ static f32x4 score(Op v, Split p, f32x4 c) { return state(v, p, c); }
  __device__ __forceinline__ static f32x4 score2(Op v0, Op v1, Split p0, Split p1, f32x4 c) { return state2(v0, v1, p0, p1, c); }
  __device__ __forceinline__ static f32x4 add(Op b, Split3 w, f32x4 c) {
    return mma_bf16(b.hi, w.hi, mma_bf16(b.hi, w.mid, mma_bf16(b.lo, w.hi, mma_bf16(b.hi, w.lo, mma_bf16(b.lo, w.mid, c)))));
  }
  __device__ __forceinline__ static f32x4 add2(Op b0, Op b1, Split3 w0, Split3 w1, f32x4 c) {
    c = mma2_bf16(b0.lo, b1.lo, w0.mid, w1.mid, c);
    c = mma2_bf16(b0.hi, b1.hi, w0.lo, w1.lo, c);
    c = mma2_bf16(b0.lo, b1.lo, w0.hi, w1.hi, c);
    c = mma2_bf16(b0.hi, b1.hi, w0.mid, w1.mid, c);
    return mma2_bf16(b0.hi, b1.hi, w0.hi, w1.hi, c);
  }
  __device__ __forceinline__ static Op upto(Op v, int n) {
    v.hi = Mat<BF16>::upto(v.hi, n);
    v.lo = Mat<BF16>::upto(v.lo, n);
    return v;
  }
};

// 4 consecutive elements at p; n of them exist, `wide`: the address is aligned to 4 elements
template <typename T> __device__ __forceinline__ typename Mat<T>::Raw load4(const char* p, int n, bool wide) {
  typedef typename Mat<T>::Raw Raw;
  if (wide && n >= 4) return *reinterpret_cast<const Raw*>(p);
  Raw v = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) {
      if constexpr (ElemTraits<T>::kBytes == 4) v[e] = reinterpret_cast<const float*>(p)[e];
      else v[e] = reinterpret_cast<const short*>(p)[e];
    }
  return v;
}

struct Operand {
  const void* p;
  int64_t sb, sh;        // element strides of sequence and head
  int st;                // of the token
  int shared;            // heads per stored head
};

// what one pass over the tokens computes (see the top): an output, or a gradient, or (la_kernel<STATE>) segments' states alone
struct Role {
  Operand a, b, c;
  void* out;             // [B][T][H / fold][N]
  const float* s0;       // first state, or null: zeros
  float* s1;             // last state, or null
  float* seg;            // [B][H][segments] states: in front of each segment (read), or of each segment's own tokens one place further on (STATE)
  int M, N;
  int sm, sn;            // strides of m and n inside one state (the transposed roles read S^T)
  float za, zs;
  int sh, reverse;
  int fold;              // heads whose outputs are summed (dk, dv of shared heads): waves of one workgroup
  int out_f32, wide;     // out holds floats; all addresses aligned to 4 elements
};

struct LaArgs {
  const float* log_decay;  // [H]
  const int* lengths;      // [B], or null
  int B, T, H;
  int group;               // waves of a workgroup that belong to one (sequence, stored head, slice)
  int seg, segments;       // tokens in a segment (a multiple of 64)
  float scale;
  Role r[3];
};

// g^n = 2^(n log2 g), the exponent in two floats: the power's error does not grow with n
struct Decay {
  float la, hi, lo;
  __device__ __forceinline__ Decay(float l) : la(l) {
    hi = l * 1.44269502f;
    lo = fmaf(l, 1.44269502f, -hi) + l * 1.92596303e-8f;
  }
  __device__ __forceinline__ float pow(int n) const {
    const float f = (float)n, x = hi * f, r = fmaf(hi, f, -x) + lo * f;
    const float y = __builtin_amdgcn_exp2f(x) * fmaf(r, 0.693147182f, 1.f);
    return n == 0 ? 1.f : x < -149.f ? 0.f : y;   // (n = 0 and g = 0: 1; g = 0 otherwise: r is NaN, x -inf)
  }
};

template <typename T, int MT, int CT, bool WHOLE, bool STATE> __global__ __launch_bounds__(256) void la_kernel(LaArgs p) {
  typedef Mat<T> X;
  typedef typename X::Raw Raw;
  typedef typename X::Op Op;
  constexpr int kBytes = ElemTraits<T>::kBytes;
  constexpr int C = 16 * CT;
  __shared__ f32x4 sums[STATE ? 1 : 2][STATE ? 1 : 4][CT][64];
  const Role& r = p.r[blockIdx.y];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slices = (r.N + 15) >> 4, stored = p.H / p.group;
  const int per = (blockDim.x >> 6) / p.group;                       // (sequence, stored head, slice) triples of a workgroup
  const int f = blockIdx.x * per + wave / p.group, member = wave % p.group;
  const bool active = f < p.B * stored * slices;                    // (a wave without work still meets the barriers of the summed roles)
  const int slice = f % slices, bi = active ? f / slices / stored : 0, h = (active ? f / slices % stored : 0) * p.group + member;
  const int segment = blockIdx.z;
  const int n = p.lengths ? min(max(p.lengths[bi], 0), p.T) : p.T;
  const int begin = segment * p.seg, end = min(begin + p.seg, p.T);
  const Decay decay(p.log_decay[h]);
  const char* pa = reinterpret_cast<const char*>(r.a.p) + (bi * r.a.sb + (h / r.a.shared) * r.a.sh) * kBytes;
  const char* pb = reinterpret_cast<const char*>(r.b.p) + (bi * r.b.sb + (h / r.b.shared) * r.b.sh) * kBytes;
  const char* pc = reinterpret_cast<const char*>(r.c.p) + (bi * r.c.sb + (h / r.c.shared) * r.c.sh) * kBytes;
  const int col = slice * 16 + c;                       // this lane's column of S and of c's transposed tile
  const int n0 = slice * 16 + 4 * g;                    // its 4 columns of c's rows and of out
  const int64_t pair = (int64_t)bi * p.H + h, states = (int64_t)r.M * r.N;
  const Raw unit = X::one(c - 4 * g);

  f32x4 S[MT];
  const float* s0 = STATE ? nullptr : p.segments > 1 ? r.seg + (pair * p.segments + segment) * states : r.s0 ? r.s0 + pair * states : nullptr;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    S[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (s0 && active && (WHOLE || col < r.N))
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = 16 * t + 4 * g + e;
        if (WHOLE || m < r.M) S[t][e] = s0[m * r.sm + col * r.sn];
      }
  }
  // scale g^{i-j} (i = 16 it + c, j = 16 jt + 4g + e; 0 above the diagonal) by it - jt, zs g^{C-1-j+sh}, za g^{i+1-sh}, g^C - 1
  f32x4 inside[CT], into[CT];
  float from[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (!STATE) inside[t][e] = p.scale * decay.pow(max(16 * t + c - 4 * g - e, 0));
      into[t][e] = r.zs * decay.pow(C - 1 - (16 * t + 4 * g + e) + r.sh);
    }
    from[t] = r.za * decay.pow(16 * t + c + 1 - r.sh);
  }
  float keep1 = expm1f(decay.la * (float)C);            // S + (g^C - 1) S keeps a slow decay's last bits

  for (int t0 = begin; t0 < end; t0 += C) {
    const int cnt = active ? min(C, n - t0) : 0;
    f32x4 acc[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (cnt > 0) {
      if (cnt < C) {
        keep1 = expm1f(decay.la * (float)cnt);
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = 16 * t + 4 * g + e;
            into[t][e] = j < cnt ? r.zs * decay.pow(cnt - 1 - j + r.sh) : 0.f;
          }
      }
      // rows (tokens) of a, b, c; behind the last token its row again: those scores lie above every valid token's diagonal and `into` is 0
      Raw av[CT][MT], bv[CT][MT], cv[CT];
#pragma unroll
      for (int it = 0; it < CT; ++it) {
        const int idx = min(t0 + 16 * it + c, n - 1), tok = r.reverse ? n - 1 - idx : idx;
        const char* ra = pa + ((int64_t)tok * r.a.st + 4 * g) * kBytes;
        const char* rb = pb + ((int64_t)tok * r.b.st + 4 * g) * kBytes;
        const char* rc = pc + ((int64_t)tok * r.c.st + n0) * kBytes;
        if constexpr (WHOLE) {
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            if (!STATE) av[it][t] = *reinterpret_cast<const Raw*>(ra + 16 * t * kBytes);
            bv[it][t] = *reinterpret_cast<const Raw*>(rb + 16 * t * kBytes);
          }
          cv[it] = *reinterpret_cast<const Raw*>(rc);
        } else {
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const int left = r.M - 16 * t - 4 * g;
            if (!STATE) av[it][t] = load4<T>(ra + 16 * t * kBytes, left, r.wide);
            bv[it][t] = load4<T>(rb + 16 * t * kBytes, left, r.wide);
          }
          cv[it] = load4<T>(rc, r.N - n0, r.wide);
        }
      }
      f32x4 cf[CT];                                      // c by columns: tokens 4g .. 4g+3 of column `col`
#pragma unroll
      for (int t = 0; t < CT; ++t) cf[t] = X::raw(cv[t], unit, f32x4{0.f, 0.f, 0.f, 0.f});
      if constexpr (!STATE) {
        // scores[jt][it][j][i] = b_j . a_i
        typename X::Split ps[CT][CT];
#pragma unroll
        for (int it = 0; it < CT; ++it)
#pragma unroll
          for (int jt = 0; jt <= it; ++jt) {
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
            if constexpr (MT == 1) {
              x = X::raw(bv[jt][0], av[it][0], x);
            } else {
#pragma unroll
              for (int t = 0; t < MT; t += 2) x = X::raw2(bv[jt][t], bv[jt][t + 1], av[it][t], av[it][t + 1], x);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = jt < it || 4 * g + e <= c ? x[e] * inside[it - jt][e] : 0.f;
            ps[jt][it] = X::split(x);
          }
        // acc[it][n][i] = za g^{i+1-sh} sum_m S[m][n] a_i[m]
#pragma unroll
        for (int t = 0; t < MT; t += 2) {
          const typename X::Split s = X::split(S[t]);
          if constexpr (MT == 1) {
#pragma unroll
            for (int it = 0; it < CT; ++it) acc[it] = X::state(s, X::op(av[it][0]), acc[it]);
          } else {
            const typename X::Split u = X::split(S[t + 1]);
#pragma unroll
            for (int it = 0; it < CT; ++it) acc[it] = X::state2(s, u, X::op(av[it][t]), X::op(av[it][t + 1]), acc[it]);
          }
        }
        Op co[CT];
        bool odd = false;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
          acc[t] *= from[t];
          co[t] = X::op_of(cf[t]);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= !(__builtin_fabsf(cf[t][e]) <= 3.4028234e38f);
        }
        // acc[it][n][i] += sum_j c_j[n] scores[j][i].  A later token's infinity or NaN must not reach an earlier token's sum as 0 * inf: a
        // chunk that holds one goes token by token
        auto inner = [&](int it, Op last, f32x4 x) {
          if constexpr (CT == 1) return X::score(last, ps[0][0], x);
          else return it == 0 ? X::score(last, ps[0][0], x) : X::score2(co[0], last, ps[0][1], ps[1][1], x);
        };
        if (__builtin_expect(__any(odd), 0)) {
#pragma unroll
          for (int it = 0; it < CT; ++it) {
            const f32x4 before = acc[it];
            for (int i = 0; i < 16; ++i) {
              const f32x4 x = inner(it, X::upto(co[it], i + 1 - 4 * g), before);
              if (c == i) acc[it] = x;
            }
          }
        } else {
#pragma unroll
          for (int it = 0; it < CT; ++it) acc[it] = inner(it, co[it], acc[it]);
        }
      }
      // S[m][n] = g^n S[m][n] + sum_j b_j[m] (into_j c_j[n])
      typename X::Split3 ws[CT];
#pragma unroll
      for (int t = 0; t < CT; ++t) ws[t] = X::split3(cf[t] * into[t]);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        Op bt[CT];
#pragma unroll
        for (int jt = 0; jt < CT; ++jt) bt[jt] = X::op_of(X::raw(bv[jt][t], unit, f32x4{0.f, 0.f, 0.f, 0.f}));
#pragma unroll
        for (int e = 0; e < 4; ++e) S[t][e] = fmaf(S[t][e], keep1, S[t][e]);
        if constexpr (CT == 1) S[t] = X::add(bt[0], ws[0], S[t]);
        else S[t] = X::add2(bt[0], bt[1], ws[0], ws[1], S[t]);
      }
    }
    if constexpr (!STATE) {
      bool writes = active;
      if (r.fold > 1) {   // (uniform over the launch's role) the heads of one stored head add up in the first one's wave
        const int buf = (t0 / C) & 1;
#pragma unroll
        for (int t = 0; t < CT; ++t) sums[buf][wave][t][lane] = acc[t];
        __syncthreads();   // (two buffers: who writes this one again has passed the next barrier, and so have its readers)
        writes = active && member == 0;
        if (writes)
          for (int k = 1; k < r.fold; ++k)
#pragma unroll
            for (int t = 0; t < CT; ++t) acc[t] += sums[buf][wave + k][t][lane];
      }
      // (tokens behind the sequence's length get zeros)
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        const int idx = t0 + 16 * t + c;
        if (!writes || idx >= end || (!WHOLE && n0 >= r.N)) continue;
        if (idx >= n) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int tok = r.reverse && idx < n ? n - 1 - idx : idx;
        const int64_t at = (((int64_t)bi * p.T + tok) * (p.H / r.fold) + h / r.fold) * r.N + n0;
        if (r.out_f32 || kBytes == 4) {
          float* o = reinterpret_cast<float*>(r.out) + at;
          if (WHOLE || r.wide) *reinterpret_cast<f32x4*>(o) = acc[t];
          else
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n0 + e < r.N) o[e] = acc[t][e];
        } else if constexpr (kBytes == 2) {
          s16x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = (short)f32_to_bits16<T>(acc[t][e]);
          short* o = reinterpret_cast<short*>(r.out) + at;
          if (WHOLE || r.wide) *reinterpret_cast<s16x4*>(o) = v;
          else
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n0 + e < r.N) o[e] = v[e];
        }
      }
    }
  }
  float* s1 = STATE ? r.seg + (pair * p.segments + segment + 1) * states : segment == p.segments - 1 && r.s1 ? r.s1 + pair * states : nullptr;
  if (s1 && active && (WHOLE || col < r.N))
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = 16 * t + 4 * g + e;
        if (WHOLE || m < r.M) s1[m * r.sm + col * r.sn] = S[t][e];
      }
}

// the state in front of every segment, from each segment's own (written one place further on) and the first state: in place.  A workgroup
// takes 64 elements of one state; 16 groups of threads take consecutive segments each and meet through LDS
constexpr int kMaxSegments = 256;
__global__ __launch_bounds__(1024) void la_scan_kernel(LaArgs p) {
  __shared__ float total[16][64];
  const Role& r = p.r[blockIdx.z];
  const int states = r.M * r.N, x = threadIdx.x & 63, z = threadIdx.x >> 6, at = blockIdx.x * 64 + x;
  const int64_t pair = blockIdx.y;
  const int h = (int)(pair % p.H);
  const int64_t bi = pair / p.H;
  const int n = p.lengths ? min(max(p.lengths[bi], 0), p.T) : p.T;
  const Decay decay(p.log_decay[h]);
  const bool live = at < states;
  float* seg = r.seg + pair * p.segments * states + at;
  const int K = (p.segments - 1 + 15) / 16, s_begin = min(z * K, p.segments - 1), s_end = min(s_begin + K, p.segments - 1);
  auto tokens = [&](int s) { return min(max(n - s * p.seg, 0), p.seg); };   // of segment s
  auto count = [&](int a, int b) { return min(max(n - a * p.seg, 0), (b - a) * p.seg); };   // of segments a .. b - 1 (all but the last are whole)
  float own[kMaxSegments / 16], run = 0.f;
#pragma unroll
  for (int k = 0; k < kMaxSegments / 16; ++k)
    if (s_begin + k < s_end && live) own[k] = seg[(int64_t)(s_begin + k + 1) * states];
#pragma unroll
  for (int k = 0; k < kMaxSegments / 16; ++k)
    if (s_begin + k < s_end && live) run = fmaf(decay.pow(tokens(s_begin + k)), run, own[k]);
  total[z][x] = run;
  __syncthreads();
  const float first = r.s0 && live ? r.s0[pair * states + at] : 0.f;
  run = first;
  for (int y = 0; y < z; ++y) {
    const int a = min(y * K, p.segments - 1), b = min(a + K, p.segments - 1);
    run = fmaf(decay.pow(count(a, b)), run, total[y][x]);
  }
  if (!live) return;
  if (z == 0) seg[0] = first;
#pragma unroll
  for (int k = 0; k < kMaxSegments / 16; ++k)
    if (s_begin + k < s_end) {
      run = fmaf(decay.pow(tokens(s_begin + k)), run, own[k]);
      seg[(int64_t)(s_begin + k + 1) * states] = run;
    }
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

constexpr int kMaxHead = 128;
constexpr int kFold = 4;   // shared heads that are summed inside a workgroup; more: through `scratch` and la_share_kernel

inline int tiles(int m) { return m <= 16 ? 1 : m <= 32 ? 2 : m <= 64 ? 4 : 8; }

// Waves that the machine wants at once, and the fewest tokens that are worth a segment
constexpr int64_t kWaves = 2048;
constexpr int kMinSegment = 128;

// (tokens in a segment, segments) for `waves` waves per segment
void segmentation(int T, int64_t waves, int* seg, int* segments) {
  int64_t want = waves > 0 ? kWaves / waves : 1, most = T / kMinSegment;
  if (want > most) want = most;
  if (want > kMaxSegments) want = kMaxSegments;
  if (want < 2) { *seg = (T + 63) / 64 * 64; *segments = 1; return; }
  int64_t s = (T + want - 1) / want;
  s = (s + 63) / 64 * 64;
  *seg = (int)s;
  *segments = (int)((T + s - 1) / s);
}

template <typename T, int MT, int CT, bool STATE> int go(const LaArgs& a, bool whole, dim3 grid, int threads, hipStream_t st) {
  if (whole) la_kernel<T, MT, CT, true, STATE><<<grid, threads, 0, st>>>(a);
  else la_kernel<T, MT, CT, false, STATE><<<grid, threads, 0, st>>>(a);
  return tg_launch_status();
}
template <typename T, int MT> int go_mt(const LaArgs& a, bool whole, bool state, dim3 grid, int threads, hipStream_t st) {
  // chunks of 32 tokens halve the work on the state per token; sequences of one chunk of 16 would waste half of them
  if (state) return go<T, MT, 2, true>(a, whole, grid, threads, st);
  return a.T <= 16 ? go<T, MT, 1, false>(a, whole, grid, threads, st) : go<T, MT, 2, false>(a, whole, grid, threads, st);
}
// `roles` roles with the same number of m tiles in one launch
template <typename T> int launch(const LaArgs& a, int roles, bool state, hipStream_t st) {
  int mt = 1, slices = 1;
  bool whole = true;
  for (int i = 0; i < roles; ++i) {
    const Role& r = a.r[i];
    if (tiles(r.M) > mt) mt = tiles(r.M);
    if ((r.N + 15) / 16 > slices) slices = (r.N + 15) / 16;
  }
  for (int i = 0; i < roles; ++i) whole = whole && a.r[i].wide && a.r[i].M == 16 * mt && a.r[i].N % 16 == 0;
  const int per = kFold / a.group, threads = 64 * per * a.group;
  const int64_t wgs = ((int64_t)a.B * (a.H / a.group) * slices + per - 1) / per;
  if ((int64_t)a.B * a.H * slices > 0x7fffffff - 64) return TG_E_UNSUPPORTED;
  const dim3 grid((unsigned)wgs, roles, state ? a.segments - 1 : a.segments);
  if (mt == 1) return go_mt<T, 1>(a, whole, state, grid, threads, st);
  if (mt == 2) return go_mt<T, 2>(a, whole, state, grid, threads, st);
  if (mt == 4) return go_mt<T, 4>(a, whole, state, grid, threads, st);
  return go_mt<T, 8>(a, whole, state, grid, threads, st);
}
int launch_dt(int dtype, const LaArgs& a, int roles, bool state, hipStream_t st) {
  TG_DISPATCH_DTYPE(dtype, return launch<BF16>(a, roles, state, st), return launch<F16>(a, roles, state, st), return launch<F32>(a, roles, state, st));
}

struct Strided { Operand o; bool wide; };
Strided operand(int dtype, const void* p, const int64_t* stride, int shared) {
  const int bytes = 4 * elem_bytes(dtype);
  const bool wide = ((reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0) && stride[0] % 4 == 0 && stride[1] % 4 == 0 && stride[2] % 4 == 0;
  return {Operand{p, stride[0], stride[2], (int)stride[1], shared}, wide};
}

int check(int dtype, const tg_la_desc* d) {
  if (!d || !known(dtype) || d->B < 0 || d->T < 0 || d->H <= 0 || d->HK <= 0 || d->DK <= 0 || d->DV <= 0) return TG_E_BADARG;
  if (d->H % d->HK || d->DK > kMaxHead || d->DV > kMaxHead || d->T > 0x7fffff00) return TG_E_UNSUPPORTED;
  for (const int64_t* s : {d->q_stride, d->k_stride, d->v_stride})
    if (s[0] < 0 || s[1] < 0 || s[2] < 0) return TG_E_BADARG;
    else if (s[1] > 0x7fffffff) return TG_E_UNSUPPORTED;
  return TG_OK;
}

inline int64_t slices_of(int n) { return (n + 15) / 16; }
// segments of the forward pass (one role) and of the backward pass (three)
void forward_segments(const tg_la_desc* d, int* seg, int* segments) { segmentation(d->T, (int64_t)d->B * d->H * slices_of(d->DV), seg, segments); }
void backward_segments(const tg_la_desc* d, int* seg, int* segments) {
  segmentation(d->T, (int64_t)d->B * d->H * (2 * slices_of(d->DK) + slices_of(d->DV)), seg, segments);
}
inline int64_t states(const tg_la_desc* d) { return (int64_t)d->B * d->H * d->DK * d->DV; }
inline int64_t fold_floats(const tg_la_desc* d) { return d->H / d->HK > kFold ? (int64_t)d->B * d->T * d->H * (d->DK + d->DV) : 0; }

// segments' states: own ones, then joined
int join_segments(int dtype, const LaArgs& a, int roles, hipStream_t st) {
  const int rc = launch_dt(dtype, a, roles, true, st);
  if (rc != TG_OK) return rc;
  la_scan_kernel<<<dim3((a.r[0].M * a.r[0].N + 63) / 64, (unsigned)(a.B * a.H), roles), 1024, 0, st>>>(a);
  return tg_launch_status();
}

}  // namespace

extern "C" int64_t tg_linear_attention_scratch_floats(const tg_la_desc* d) {
  if (check(TG_F32, d) != TG_OK) return 0;
  int seg, segments;
  forward_segments(d, &seg, &segments);
  return segments > 1 ? segments * states(d) : 0;
}

extern "C" int tg_linear_attention(int dtype, const tg_la_desc* d, const void* q, const void* k, const void* v, const float* log_decay,
                                   const int32_t* lengths, const float* state_in, void* o, float* state_out, float* scratch, void* stream) {
  int rc = check(dtype, d);
  if (rc != TG_OK) return rc;
  if (d->B == 0) return TG_OK;
  LaArgs a{};
  forward_segments(d, &a.seg, &a.segments);
  if (!log_decay || !state_out || (d->T > 0 && (!q || !k || !v || !o)) || (a.segments > 1 && !scratch)) return TG_E_BADARG;
  if (!elem_aligned(dtype, q) || !elem_aligned(dtype, k) || !elem_aligned(dtype, v) || !elem_aligned(dtype, o) || !word_aligned(log_decay) ||
      !word_aligned(lengths) || !word_aligned(state_in) || !word_aligned(state_out) || !word_aligned(scratch))
    return TG_E_ALIGN;
  const int G = d->H / d->HK;
  const Strided Q = operand(dtype, q, d->q_stride, 1), K = operand(dtype, k, d->k_stride, G), V = operand(dtype, v, d->v_stride, G);
  hipStream_t st = (hipStream_t)stream;
  a.log_decay = log_decay;
  a.lengths = lengths;
  a.B = d->B; a.T = d->T; a.H = d->H;
  a.group = 1;
  a.scale = d->scale;
  const bool wide = Q.wide && K.wide && V.wide && d->DK % 4 == 0 && d->DV % 4 == 0 && (reinterpret_cast<uintptr_t>(o) & (4 * elem_bytes(dtype) - 1)) == 0;
  a.r[0] = Role{Q.o, K.o, V.o, o, state_in, state_out, scratch, d->DK, d->DV, d->DV, 1, d->scale, 1.f, 0, 0, 1, 0, wide};
  if (a.segments > 1 && (rc = join_segments(dtype, a, 1, st)) != TG_OK) return rc;
  return launch_dt(dtype, a, 1, false, st);
}

extern "C" int64_t tg_linear_attention_bwd_scratch_floats(const tg_la_desc* d) {
  if (check(TG_F32, d) != TG_OK) return 0;
  int seg, segments;
  backward_segments(d, &seg, &segments);
  return fold_floats(d) + (segments > 1 ? 2 * segments * states(d) : 0);
}

extern "C" int tg_linear_attention_bwd(int dtype, const tg_la_desc* d, const void* q, const void* k, const void* v, const void* dout,
                                       const int64_t* dout_stride, const float* log_decay, const int32_t* lengths, const float* state_in,
                                       const float* dstate_out, void* dq, void* dk, void* dv, float* dstate_in, float* scratch, void* stream) {
  int rc = check(dtype, d);
  if (rc != TG_OK) return rc;
  if (d->B == 0) return TG_OK;
  LaArgs a{};
  backward_segments(d, &a.seg, &a.segments);
  const int G = d->H / d->HK;
  if (!log_decay || !dout_stride || (d->T > 0 && (!q || !k || !v || !dout || !dq || !dk || !dv)) || (tg_linear_attention_bwd_scratch_floats(d) && !scratch))
    return TG_E_BADARG;
  if (dout_stride[0] < 0 || dout_stride[1] < 0 || dout_stride[2] < 0) return TG_E_BADARG;
  if (dout_stride[1] > 0x7fffffff) return TG_E_UNSUPPORTED;
  if (!elem_aligned(dtype, q) || !elem_aligned(dtype, k) || !elem_aligned(dtype, v) || !elem_aligned(dtype, dout) || !elem_aligned(dtype, dq) ||
      !elem_aligned(dtype, dk) || !elem_aligned(dtype, dv) || !word_aligned(log_decay) || !word_aligned(lengths) || !word_aligned(state_in) ||
      !word_aligned(dstate_out) || !word_aligned(dstate_in) || !word_aligned(scratch))
    return TG_E_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  const Strided Q = operand(dtype, q, d->q_stride, 1), K = operand(dtype, k, d->k_stride, G), V = operand(dtype, v, d->v_stride, G),
                D = operand(dtype, dout, dout_stride, 1);
  const bool apart = G > kFold;   // dk, dv of every head through scratch
  float* const part_v = scratch;
  float* const part_k = apart ? scratch + (int64_t)d->B * d->T * d->H * d->DV : nullptr;
  float* const seg_s = scratch + fold_floats(d);
  float* const seg_d = seg_s + a.segments * states(d);
  a.log_decay = log_decay;
  a.lengths = lengths;
  a.B = d->B; a.T = d->T; a.H = d->H;
  a.group = apart ? 1 : G;
  a.scale = d->scale;
  const int fold = a.group, DK = d->DK, DV = d->DV;
  bool wide = Q.wide && K.wide && V.wide && D.wide && DK % 4 == 0 && DV % 4 == 0;
  for (const void* p : {(const void*)dq, (const void*)(apart ? part_k : dk), (const void*)(apart ? part_v : dv)})
    wide = wide && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
  if (a.segments > 1) {
    a.r[0] = Role{Q.o, K.o, V.o, nullptr, state_in, nullptr, seg_s, DK, DV, DV, 1, 0.f, 1.f, 0, 0, 1, 0, wide};
    a.r[1] = Role{K.o, Q.o, D.o, nullptr, dstate_out, nullptr, seg_d, DK, DV, DV, 1, 0.f, d->scale, 1, 1, 1, 0, wide};
    if ((rc = join_segments(dtype, a, 2, st)) != TG_OK) return rc;
  }
  const Role rq{D.o, V.o, K.o, dq, state_in, nullptr, seg_s, DV, DK, 1, DV, d->scale, 1.f, 0, 0, 1, 0, wide};
  const Role rk{V.o, D.o, Q.o, apart ? (void*)part_k : dk, dstate_out, nullptr, seg_d, DV, DK, 1, DV, 1.f, d->scale, 1, 1, fold, apart, wide};
  const Role rv{K.o, Q.o, D.o, apart ? (void*)part_v : dv, dstate_out, dstate_in, seg_d, DK, DV, DV, 1, 1.f, d->scale, 1, 1, fold, apart, wide};
  a.r[0] = rq;
  a.r[1] = rk;
  a.r[2] = rv;
  if (tiles(DK) == tiles(DV)) {
    rc = launch_dt(dtype, a, 3, false, st);
  } else {
    if ((rc = launch_dt(dtype, a, 2, false, st)) != TG_OK) return rc;
    a.r[0] = rv;
    rc = launch_dt(dtype, a, 1, false, st);
  }
  if (rc != TG_OK || !apart || d->T == 0) return rc;
  const int64_t rows = (int64_t)d->B * d->T;
  for (int w = 0; w < 2; ++w) {
    const int D_ = w ? DK : DV;
    const int64_t wgs = (rows * d->HK * D_ + 255) / 256;
    const int grid = (int)(wgs < (1 << 20) ? wgs : (1 << 20));
    const float* in = w ? part_k : part_v;
    void* out = w ? dk : dv;
    if (dtype == TG_BF16) la_share_kernel<BF16><<<grid, 256, 0, st>>>(in, out, rows, d->HK, G, D_);
    else if (dtype == TG_F16) la_share_kernel<F16><<<grid, 256, 0, st>>>(in, out, rows, d->HK, G, D_);
    else la_share_kernel<F32><<<grid, 256, 0, st>>>(in, out, rows, d->HK, G, D_);
    if ((rc = tg_launch_status()) != TG_OK) return rc;
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
