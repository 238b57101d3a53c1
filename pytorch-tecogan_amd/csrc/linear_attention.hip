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
// Layout: a wave owns 16 columns of c (and of S and out) of one head, or twice as many, and walks the tokens in chunks of 16 CT.  Everything is
// made of 16 x 16 tiles in the matrix instructions' own shape: lane (c = lane % 16, g = lane / 16) holds 4 consecutive values 4g .. 4g+3
// of row / column c.  An accumulator tile X[k][c] has the shape of an operand with c along its free dimension and k along the summed one,
// so the scores (b a^T, tile [j][i]) and the state (tiles [m][n]) go from accumulators to operands without leaving the registers.
//
// Long sequences: T is cut into segments of `seg` tokens so that a few heads fill the machine.  la_kernel with STATE sums each segment's own state,
// la_scan_kernel joins them into the state in front of every segment, and the segments then run side by side.
//
// Rounding: raw inputs are multiplied as they are (exact products, fp32 sums).  Scores, states and what is added to a state are fp32; as
// operands beside 16-bit inputs they are split into THREE bf16 parts (hi + mid + lo: all 24 bits), so the products are those of fp32 and a result is off by
// fp32 sums and its own last rounding.  (Two parts, 16 bits, were up to 14 % faster where instruction issue is the bound, and lost what neighbouring tokens
// differ by: keys that differ by 2^-8 with opposite values, fp16 9e-4 off where 2.1e-4 is the type's own.)  fp16 inputs are split into two bf16 parts beside
// them (exactly: 11 bits), because a score or a state may pass fp16's range.  fp32 inputs run on the fp32 matrix instructions.
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

// ---- products of 16 x 16 tiles, summed dimension 16 (mma) or 32 (mma2: two tiles of each operand).  Raw: an input as loaded; Op: an input
// beside a computed operand; Split: a computed operand
__device__ __forceinline__ f32x4 mma_bf16(s16x4 a, s16x4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0); }
__device__ __forceinline__ s16x8 join(s16x4 a, s16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ f32x4 mma2_bf16(s16x4 a0, s16x4 a1, s16x4 b0, s16x4 b1, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, join(a0, a1)), __builtin_bit_cast(bf16x8, join(b0, b1)), c, 0, 0, 0);
}
__device__ __forceinline__ unsigned pack_bf16(float a, float b) {   // v_cvt_pk_bf16_f32
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
__device__ __forceinline__ s16x4 to_bf16(f32x4 v) { return __builtin_bit_cast(s16x4, make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]))); }
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
  __device__ __forceinline__ static f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static f32x4 to_float(Raw v) { return v; }
  __device__ __forceinline__ static Op op(Raw v) { return v; }
  __device__ __forceinline__ static Split split(f32x4 v) { return v; }
  __device__ __forceinline__ static f32x4 raw(Raw a, Raw b, f32x4 c) { return mma(a, b, c); }
  __device__ __forceinline__ static f32x4 raw2(Raw a0, Raw a1, Raw b0, Raw b1, f32x4 c) { return mma(a1, b1, mma(a0, b0, c)); }
  __device__ __forceinline__ static f32x4 state(Split s, Op a, f32x4 c) { return mma(s, a, c); }
  __device__ __forceinline__ static f32x4 state2(Split s0, Split s1, Op a0, Op a1, f32x4 c) { return mma(s1, a1, mma(s0, a0, c)); }
  __device__ __forceinline__ static f32x4 add(Op b, Split w, f32x4 c) { return mma(b, w, c); }
  __device__ __forceinline__ static f32x4 add2(Op b0, Op b1, Split w0, Split w1, f32x4 c) { return mma(b1, w1, mma(b0, w0, c)); }
  template <int CT> __device__ __forceinline__ static f32x4 grown(f32x4 s, const Op* b, const Split* w) {
    if constexpr (CT == 1) return add(b[0], w[0], s);
    else return add2(b[0], b[1], w[0], w[1], s);
  }
  __device__ __forceinline__ static Op upto(Op v, int n) {   // the first n of the 4 values, zeros behind
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? v[e] : 0.f;
    return v;
  }
  __device__ __forceinline__ static Op behind(Op v, int n) {   // zeros in place of the first n
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? 0.f : v[e];
    return v;
  }
};
template <> struct Mat<BF16> {
  typedef s16x4 Raw;
  typedef s16x4 Op;
  typedef Thirds Split;
  __device__ __forceinline__ static s16x4 to_out(f32x4 v) { return to_bf16(v); }
  __device__ __forceinline__ static f32x4 to_float(Raw v) { return from_bf16(v); }
  __device__ __forceinline__ static Op op(Raw v) { return v; }
  __device__ __forceinline__ static Split split(f32x4 v) { return thirds(v); }
  __device__ __forceinline__ static f32x4 raw(Raw a, Raw b, f32x4 c) { return mma_bf16(a, b, c); }
  __device__ __forceinline__ static f32x4 raw2(Raw a0, Raw a1, Raw b0, Raw b1, f32x4 c) { return mma2_bf16(a0, a1, b0, b1, c); }
  __device__ __forceinline__ static f32x4 state(Split s, Op a, f32x4 c) { return mma_bf16(s.hi, a, mma_bf16(s.mid, a, mma_bf16(s.lo, a, c))); }
  __device__ __forceinline__ static f32x4 state2(Split s0, Split s1, Op a0, Op a1, f32x4 c) {
    return mma2_bf16(s0.hi, s1.hi, a0, a1, mma2_bf16(s0.mid, s1.mid, a0, a1, mma2_bf16(s0.lo, s1.lo, a0, a1, c)));
  }
  __device__ __forceinline__ static f32x4 add(Op b, Split w, f32x4 c) { return mma_bf16(b, w.hi, mma_bf16(b, w.mid, mma_bf16(b, w.lo, c))); }
  __device__ __forceinline__ static f32x4 add2(Op b0, Op b1, Split w0, Split w1, f32x4 c) {
    return mma2_bf16(b0, b1, w0.hi, w1.hi, mma2_bf16(b0, b1, w0.mid, w1.mid, mma2_bf16(b0, b1, w0.lo, w1.lo, c)));
  }
  template <int CT> __device__ __forceinline__ static f32x4 grown(f32x4 s, const Op* b, const Split* w) {
    if constexpr (CT == 1) return add(b[0], w[0], s);
    else return add2(b[0], b[1], w[0], w[1], s);
  }
  __device__ __forceinline__ static Op upto(Op v, int n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? v[e] : (short)0;
    return v;
  }
  __device__ __forceinline__ static Op behind(Op v, int n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? (short)0 : v[e];
    return v;
  }
};
template <> struct Mat<F16> {
  typedef s16x4 Raw;
  typedef Halves Op;
  typedef Thirds Split;
  __device__ __forceinline__ static s16x4 to_out(f32x4 v) { return __builtin_bit_cast(s16x4, __builtin_convertvector(v, f16x4)); }
  __device__ __forceinline__ static f32x4 to_float(Raw v) { return __builtin_convertvector(__builtin_bit_cast(f16x4, v), f32x4); }
  __device__ __forceinline__ static Op op(Raw v) { return halves(to_float(v)); }
  __device__ __forceinline__ static Split split(f32x4 v) { return thirds(v); }
  __device__ __forceinline__ static f32x4 raw(Raw a, Raw b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
  __device__ __forceinline__ static f32x4 raw2(Raw a0, Raw a1, Raw b0, Raw b1, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, join(a0, a1)), __builtin_bit_cast(f16x8, join(b0, b1)), c, 0, 0, 0);
  }
  // (lo * lo: 2^-9 of the input by 2^-18 of the operand, below 24 bits of the product)
  __device__ __forceinline__ static f32x4 state(Split s, Op a, f32x4 c) {
    return mma_bf16(s.hi, a.hi, mma_bf16(s.mid, a.hi, mma_bf16(s.hi, a.lo, mma_bf16(s.lo, a.hi, mma_bf16(s.mid, a.lo, c)))));
  }
  __device__ __forceinline__ static f32x4 state2(Split s0, Split s1, Op a0, Op a1, f32x4 c) {
    c = mma2_bf16(s0.mid, s1.mid, a0.lo, a1.lo, c);
    c = mma2_bf16(s0.lo, s1.lo, a0.hi, a1.hi, c);
    c = mma2_bf16(s0.hi, s1.hi, a0.lo, a1.lo, c);
    c = mma2_bf16(s0.mid, s1.mid, a0.hi, a1.hi, c);
    return mma2_bf16(s0.hi, s1.hi, a0.hi, a1.hi, c);
  }
  __device__ __forceinline__ static f32x4 add(Op b, Split w, f32x4 c) {
    return mma_bf16(b.hi, w.hi, mma_bf16(b.hi, w.mid, mma_bf16(b.lo, w.hi, mma_bf16(b.hi, w.lo, mma_bf16(b.lo, w.mid, c)))));
  }
  __device__ __forceinline__ static f32x4 add2(Op b0, Op b1, Split w0, Split w1, f32x4 c) {
    c = mma2_bf16(b0.lo, b1.lo, w0.mid, w1.mid, c);
    c = mma2_bf16(b0.hi, b1.hi, w0.lo, w1.lo, c);
    c = mma2_bf16(b0.lo, b1.lo, w0.hi, w1.hi, c);
    c = mma2_bf16(b0.hi, b1.hi, w0.mid, w1.mid, c);
    return mma2_bf16(b0.hi, b1.hi, w0.hi, w1.hi, c);
  }
  template <int CT> __device__ __forceinline__ static f32x4 grown(f32x4 s, const Op* b, const Split* w) {
    if constexpr (CT == 1) return add(b[0], w[0], s);
    else return add2(b[0], b[1], w[0], w[1], s);
  }
  __device__ __forceinline__ static Op upto(Op v, int n) {
    v.hi = Mat<BF16>::upto(v.hi, n);
    v.lo = Mat<BF16>::upto(v.lo, n);
    return v;
  }
  __device__ __forceinline__ static Op behind(Op v, int n) {
    v.hi = Mat<BF16>::behind(v.hi, n);
    v.lo = Mat<BF16>::behind(v.lo, n);
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

// what one pass over the tokens computes (see the top): an output, or a gradient, or (STATE) segments' states alone
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
  int out_f32, wide, pieces;   // out holds floats; all addresses aligned to 4 elements; to 16 bytes, and M and N fill 16 bytes
};

struct LaArgs {
  const float* log_decay;  // [H]
  const int* lengths;      // [B], or null
  int B, T, H;
  int group;               // waves of a workgroup that belong to one (stored head, slice)
  int columns, bgroups;    // blockIdx.x = bgroup * columns + column: workgroups over (stored head, slice), and over the sequences
  int seg, segments;       // tokens in a segment (a multiple of 32)
  bool wide;               // (for the launch) slices of 32 columns where they can be
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

// A state's factor g^n = e^a as two floats, whose product with the state rounds once.  Slow decays: in a single float a rate of -1e-6 would be off by 1.3 %,
// the same way at every use.  Fast ones (and growth), where 1 + (g^n - 1) would lose the digits of a small power: `fast`, e^a in one float.
struct Factor {
  float hi, lo;
  Factor() = default;
  __device__ __forceinline__ static Factor of(float hi, float lo) {
    Factor f;
    f.hi = hi;
    f.lo = lo;
    return f;
  }
  __device__ __forceinline__ Factor(float a, float fast) {
    const float m = expm1f(a);
    hi = 1.f + m;
    lo = (1.f - hi) + m;   // (exact: |m| < 1)
    if (!(__builtin_fabsf(a) < 0.5f)) {
      hi = fast;
      lo = 0.f;
    }
  }
  __device__ __forceinline__ Factor(const Decay& d, int n) : Factor(d.la * (float)n, d.pow(n)) {}
  __device__ __forceinline__ float operator()(float s) const { return fmaf(s, hi, s * lo); }
  __device__ __forceinline__ float plus(float s, float x) const {   // g^n s + x; an infinite s stays (0 * infinity would be NaN)
    return fmaf(hi, s, fmaf(lo, __builtin_amdgcn_fmed3f(s, -3.4028234e38f, 3.4028234e38f), x));
  }
};

__device__ __forceinline__ void wave_fence() {   // the wave's own LDS writes and reads keep their order
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// What a wave works on: NS x 16 columns (a slice) of one head, and the sequences bgroup, bgroup + bgroups, .. of it.  A wave without work does another's
// and writes nothing (it meets the barriers of the summed roles).
template <typename T, int MT, int NS = 1> struct Wave {
  int lane, c, g, wave, waves, member, bgroup, slice, h;
  bool active;
  Decay decay;
  __device__ __forceinline__ explicit Wave(const LaArgs& p) : decay(0.f) {
    const Role& r = p.r[blockIdx.y];
    lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int slices = (r.N + 16 * NS - 1) / (16 * NS), per = waves / p.group;   // (stored head, slice) pairs of a workgroup
    bgroup = blockIdx.x / p.columns;
    int f = (blockIdx.x - bgroup * p.columns) * per + wave / p.group;
    member = wave % p.group;
    active = f < p.H / p.group * slices;
    if (!active) f = 0;
    slice = f % slices;
    h = f / slices * p.group + member;
    decay = Decay(p.log_decay[h]);
  }
  __device__ __forceinline__ bool whole(const Role& r) const { return r.M == 16 * MT && r.N % (16 * NS) == 0; }   // no part tiles
  __device__ __forceinline__ int col(int s) const { return (slice * NS + s) * 16 + c; }
  // sequence bgroup's states of this wave's head, and how far it is to the next sequence's: in front of the first token (null: zeros), and
  // behind the last one (null: not wanted)
  template <bool STATE> __device__ __forceinline__ const float* first_at(const LaArgs& p, const Role& r, int64_t* next) const {
    const int64_t pair = (int64_t)bgroup * p.H + h, states = (int64_t)r.M * r.N;
    *next = (int64_t)p.bgroups * p.H * p.segments * states;
    if (STATE) return nullptr;
    if (p.segments > 1) return r.seg + (pair * p.segments + blockIdx.z) * states;
    return r.s0 ? r.s0 + pair * states : nullptr;
  }
  template <bool STATE> __device__ __forceinline__ float* last_at(const LaArgs& p, const Role& r, int64_t* next) const {
    const int64_t pair = (int64_t)bgroup * p.H + h, states = (int64_t)r.M * r.N;
    *next = (int64_t)p.bgroups * p.H * (STATE ? p.segments : 1) * states;
    if (STATE) return r.seg + (pair * p.segments + blockIdx.z + 1) * states;
    return (int)blockIdx.z == p.segments - 1 && r.s1 ? r.s1 + pair * states : nullptr;
  }
  __device__ __forceinline__ void load(const Role& r, const float* s0, f32x4 (&S)[NS][MT]) const {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
#pragma unroll
      for (int t = 0; t < MT; ++t) S[s][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (!s0) continue;
      const int at = 4 * g * r.sm + col(s) * r.sn;
      if (whole(r)) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[s][t][e] = s0[at + (16 * t + e) * r.sm];
      } else if (col(s) < r.N) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (16 * t + 4 * g + e < r.M) S[s][t][e] = s0[at + (16 * t + e) * r.sm];
      }
    }
  }
  __device__ __forceinline__ void store(const Role& r, float* s1, const f32x4 (&S)[NS][MT]) const {
    if (!s1 || !active) return;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int at = 4 * g * r.sm + col(s) * r.sn;
      if (whole(r)) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s1[at + (16 * t + e) * r.sm] = S[s][t][e];
      } else if (col(s) < r.N) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (16 * t + 4 * g + e < r.M) s1[at + (16 * t + e) * r.sm] = S[s][t][e];
      }
    }
  }
  // the heads of one stored head add up, in order, in the first one's wave; whether this wave writes.  (Uniform over the launch's role.  Two
  // buffers: who writes one again has passed the next barrier, and so have its readers.)
  template <int CT> __device__ __forceinline__ bool fold(f32x4 (&acc)[NS][CT], f32x4* sums, int heads, int turn) const {
    if (heads == 1) return active;
    f32x4* const buf = sums + (turn & 1) * waves * NS * CT * 64;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int t = 0; t < CT; ++t) buf[((wave * NS + s) * CT + t) * 64 + lane] = acc[s][t];
    __syncthreads();
    if (!writer(heads)) return false;
    for (int k = 1; k < heads; ++k)
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int t = 0; t < CT; ++t) acc[s][t] += buf[(((wave + k) * NS + s) * CT + t) * 64 + lane];
    return true;
  }
  __device__ __forceinline__ bool writer(int heads) const { return active && (heads == 1 || member == 0); }
};

// The decay's powers for chunks of 16 CT tokens
template <int CT> struct Weights {
  static constexpr int C = 16 * CT;
  f32x4 inside[CT], whole[CT], tail[CT];   // scale g^{i-j} by tile distance (i = c, j = 4g + e); zs g^{n-1-j+sh} of whole chunks, and of the one of `tokens` that ends a sequence
  float from[CT], g1;   // za g^{i+1-sh}; g
  Factor whole_keep, tail_keep;   // g^n
  int tokens;
  __device__ __forceinline__ Weights(const Decay& decay, int c, int g, float scale, float za, float zs, int sh) : whole_keep(decay, C), tail_keep(0.f, 1.f) {
    g1 = decay.pow(1);
    tokens = 0;
#pragma unroll
    for (int t = 0; t < CT; ++t) {   // (the fourth of four neighbouring powers, the others by one more factor each)
      const int d = 16 * t + c - 4 * g, j = 16 * t + 4 * g;
      inside[t][3] = scale * decay.pow(max(d - 3, 0));
      whole[t][3] = zs * decay.pow(C - 4 - j + sh);
#pragma unroll
      for (int e = 2; e >= 0; --e) {
        inside[t][e] = d - e > 0 ? inside[t][e + 1] * g1 : scale;
        whole[t][e] = whole[t][e + 1] * g1;
      }
      tail[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      from[t] = za * decay.pow(16 * t + c + 1 - sh);
    }
  }
  __device__ __forceinline__ void length(const Decay& decay, int cnt, int g, float zs, int sh) {   // a sequence's last chunk has cnt tokens
    if (cnt >= C || cnt == tokens) return;
    tokens = cnt;
    tail_keep = Factor(decay, cnt);
    const float w0 = zs * decay.pow(sh);
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const int d = cnt - 1 - 16 * t - 4 * g;   // tokens behind the first of the four
      float w = zs * decay.pow(max(d - 3, 0) + sh);
#pragma unroll
      for (int e = 3; e >= 0; --e) {
        if (e < 3) w = d - e > 0 ? w * g1 : w0;
        tail[t][e] = d - e >= 0 ? w : 0.f;
      }
    }
  }
  __device__ __forceinline__ f32x4 into(int cnt, int t) const { return cnt < C ? tail[t] : whole[t]; }
  __device__ __forceinline__ f32x4 kept(f32x4 s, int cnt) const {   // g^n S
    const Factor k = Factor::of(cnt < C ? tail_keep.hi : whole_keep.hi, cnt < C ? tail_keep.lo : whole_keep.lo);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = k(s[e]);
    return s;
  }
  __device__ __forceinline__ f32x4 masked(f32x4 x, int it, int jt, int c, int g) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = jt < it || 4 * g + e <= c ? x[e] * inside[it - jt][e] : 0.f;
    return x;
  }
};

// acc[it][n][i] += sum_j c_j[n] scores[j][i].  A later token's infinity or NaN must not reach an earlier token's sum as 0 * inf: a chunk that
// holds one goes token by token
template <typename T, int CT>
__device__ __forceinline__ void weighted_sum(f32x4* acc, const typename Mat<T>::Split (&ps)[CT][CT], const typename Mat<T>::Op* co, const f32x4* cf, int c, int g) {
  typedef Mat<T> X;
  float top = 0.f;
#pragma unroll
  for (int t = 0; t < CT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = __builtin_elementwise_maximum(top, __builtin_fabsf(cf[t][e]));   // (a NaN stays)
  auto inner = [&](int it, typename X::Op last, f32x4 y) {
    if constexpr (CT == 1) return X::add(last, ps[0][0], y);
    else return it == 0 ? X::add(last, ps[0][0], y) : X::add2(co[0], last, ps[0][1], ps[1][1], y);
  };
  if (__builtin_expect(__any(!(top <= 3.4028234e38f)), 0)) {
#pragma unroll
    for (int it = 0; it < CT; ++it) {
      const f32x4 before = acc[it];
#pragma unroll 1
      for (int i = 0; i < 16; ++i) {
        const f32x4 y = inner(it, X::upto(co[it], i + 1 - 4 * g), before);
        if (c == i) acc[it] = y;
      }
    }
  } else {
#pragma unroll
    for (int it = 0; it < CT; ++it) acc[it] = inner(it, co[it], acc[it]);
  }
}

// staged rows by columns: rows row0 + 4g .. + 3 of channel 16 t + c - a transposing read (16-bit), or one channel of four rows
template <typename T> __device__ __forceinline__ typename Mat<T>::Raw columns(const char* area, int row_bytes, int row0, int t, int c, int g) {
  if constexpr (ElemTraits<T>::kBytes == 2) {
    typedef __attribute__((address_space(3))) s16x4* Lds;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(area + (row0 + 4 * g + (c >> 2)) * row_bytes + (16 * t + 4 * (c & 3)) * 2));
  } else {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const float*>(area + (row0 + 4 * g + e) * row_bytes + (16 * t + c) * 4);
    return v;
  }
}

// Operands that are not aligned to 16 bytes, or whose channels do not fill them: every lane loads its tiles' elements itself.  Columns (of b and
// c) come from the wave's own part of the LDS, never out of a product with the identity, which would spread one channel's infinity over a tile.
template <typename T, int MT, int CT> struct Turn {
  static constexpr int kRow = 16 * MT * ElemTraits<T>::kBytes + 16, kCRow = 16 * ElemTraits<T>::kBytes + 16;   // bytes between rows (see Stage)
  static constexpr int kArea = 16 * CT * (kRow + kCRow);
};
template <typename T, int MT, int CT, bool STATE> __global__ __launch_bounds__(256, 2) void la_plain_kernel(LaArgs p) {
  typedef Mat<T> X;
  typedef Turn<T, MT, CT> G;
  typedef typename X::Raw Raw;
  typedef typename X::Op Op;
  constexpr int kBytes = ElemTraits<T>::kBytes;
  constexpr int C = 16 * CT;
  constexpr f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  extern __shared__ __align__(16) char lds[];           // [waves][kArea], then [2][waves][CT][64] sums of 4 floats if a role folds
  const Wave<T, MT> w(p);
  const Role& r = p.r[blockIdx.y];
  const int c = w.c, g = w.g;
  const int begin = blockIdx.z * p.seg, end = min(begin + p.seg, p.T);
  const char* pa = reinterpret_cast<const char*>(r.a.p) + (w.h / r.a.shared) * r.a.sh * kBytes;
  const char* pb = reinterpret_cast<const char*>(r.b.p) + (w.h / r.b.shared) * r.b.sh * kBytes;
  const char* pc = reinterpret_cast<const char*>(r.c.p) + ((w.h / r.c.shared) * r.c.sh + w.slice * 16) * kBytes;
  const int n0 = w.slice * 16 + 4 * g;                  // this lane's 4 columns of c's rows and of out
  const int row_out = p.H / r.fold * r.N, out_bytes = r.out_f32 ? 4 : kBytes;
  char* const area_b = lds + w.wave * G::kArea;
  char* const area_c = area_b + C * G::kRow;
  f32x4* const sums = reinterpret_cast<f32x4*>(lds + w.waves * G::kArea);
  Weights<CT> k(w.decay, c, g, p.scale, r.za, r.zs, r.sh);
  int64_t next0, next1;
  const float* s0 = w.template first_at<STATE>(p, r, &next0);
  float* s1 = w.template last_at<STATE>(p, r, &next1);
  int turn = 0;
  for (int bi = w.bgroup; bi < p.B; bi += p.bgroups, s0 += s0 ? next0 : 0, s1 += s1 ? next1 : 0) {
    const int n = p.lengths ? min(max(p.lengths[bi], 0), p.T) : p.T;
    const char *qa = pa + bi * r.a.sb * kBytes, *qb = pb + bi * r.b.sb * kBytes, *qc = pc + bi * r.c.sb * kBytes;
    f32x4 Ss[1][MT], (&S)[MT] = Ss[0];
    w.load(r, s0, Ss);
    for (int t0 = begin; t0 < end; t0 += C, ++turn) {
      const int cnt = min(C, n - t0);
      f32x4 accs[1][CT], (&acc)[CT] = accs[0];
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[t] = zero;
      if (cnt > 0) {
        // (behind the last token its row again: those scores lie above every valid token's diagonal and their weights in the state are 0)
        Raw av[CT][MT], bv[CT][MT], craw[CT];
        f32x4 cf[CT];
#pragma unroll
        for (int it = 0; it < CT; ++it) {
          const int idx = min(t0 + 16 * it + c, n - 1);
          const int64_t tok = r.reverse ? n - 1 - idx : idx;
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const int m = 16 * t + 4 * g;
            if (!STATE) av[it][t] = load4<T>(qa + (tok * r.a.st + m) * kBytes, r.M - m, r.wide);
            bv[it][t] = load4<T>(qb + (tok * r.b.st + m) * kBytes, r.M - m, r.wide);
          }
          craw[it] = load4<T>(qc + (tok * r.c.st + 4 * g) * kBytes, r.N - n0, r.wide);
        }
        wave_fence();
#pragma unroll
        for (int it = 0; it < CT; ++it) {
          char* const row = area_b + (16 * it + c) * G::kRow + 4 * g * kBytes;
#pragma unroll
          for (int t = 0; t < MT; ++t) *reinterpret_cast<Raw*>(row + 16 * t * kBytes) = bv[it][t];
          *reinterpret_cast<Raw*>(area_c + (16 * it + c) * G::kCRow + 4 * g * kBytes) = craw[it];
        }
        wave_fence();
#pragma unroll
        for (int it = 0; it < CT; ++it) {
          craw[it] = columns<T>(area_c, G::kCRow, 16 * it, 0, c, g);
          cf[it] = X::to_float(craw[it]);
        }
        if constexpr (!STATE) {
          typename X::Split ps[CT][CT];
#pragma unroll
          for (int it = 0; it < CT; ++it)
#pragma unroll
            for (int jt = 0; jt <= it; ++jt) {
              f32x4 x = zero;
              if constexpr (MT == 1) x = X::raw(bv[jt][0], av[it][0], x);
              else
#pragma unroll
                for (int t = 0; t < MT; t += 2) x = X::raw2(bv[jt][t], bv[jt][t + 1], av[it][t], av[it][t + 1], x);
              ps[jt][it] = X::split(k.masked(x, it, jt, c, g));
            }
          if (s0 || t0 > begin) {
#pragma unroll
            for (int t = 0; t < MT; t += MT == 1 ? 1 : 2)
#pragma unroll
              for (int it = 0; it < CT; ++it) {
                if constexpr (MT == 1) acc[it] = X::state(X::split(S[0]), X::op(av[it][0]), acc[it]);
                else acc[it] = X::state2(X::split(S[t]), X::split(S[t + 1]), X::op(av[it][t]), X::op(av[it][t + 1]), acc[it]);
              }
#pragma unroll
            for (int t = 0; t < CT; ++t) acc[t] *= k.from[t];
          }
          Op co[CT];
#pragma unroll
          for (int t = 0; t < CT; ++t) co[t] = X::op(craw[t]);
          weighted_sum<T, CT>(acc, ps, co, cf, c, g);
        }
        k.length(w.decay, cnt, g, r.zs, r.sh);
        typename X::Split ws[CT];
#pragma unroll
        for (int t = 0; t < CT; ++t) ws[t] = X::split(cf[t] * k.into(cnt, t));
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          Op b[CT];
#pragma unroll
          for (int jt = 0; jt < CT; ++jt) b[jt] = X::op(columns<T>(area_b, G::kRow, 16 * jt, t, c, g));
          S[t] = X::template grown<CT>(k.kept(S[t], cnt), b, ws);
        }
      }
      if constexpr (!STATE) {
        const bool writes = w.template fold<CT>(accs, sums, r.fold, turn);
        // (tokens behind the sequence's length get zeros)
        char* const base = reinterpret_cast<char*>(r.out) + ((int64_t)bi * p.T * row_out + w.h / r.fold * r.N + n0) * out_bytes;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
          const int idx = t0 + 16 * t + c;
          if (!writes || idx >= end || n0 >= r.N) continue;
          if (idx >= n) acc[t] = zero;
          char* const o = base + (int64_t)(r.reverse && idx < n ? n - 1 - idx : idx) * row_out * out_bytes;
          if (kBytes == 4 || out_bytes == 4) {
            if (r.wide) *reinterpret_cast<f32x4*>(o) = acc[t];
            else
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (n0 + e < r.N) reinterpret_cast<float*>(o)[e] = acc[t][e];
          } else if constexpr (kBytes == 2) {
            const s16x4 v = X::to_out(acc[t]);
            if (r.wide) *reinterpret_cast<s16x4*>(o) = v;
            else
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (n0 + e < r.N) reinterpret_cast<short*>(o)[e] = v[e];
          }
        }
      }
    }
    w.store(r, s1, Ss);
  }
}

// How a chunk's rows reach a wave.  Where operands are aligned to 16 bytes and their channels fill 16-byte pieces, a wave reads whole rows, 16 bytes per
// lane and neighbouring lanes side by side, into its own part of the LDS and takes the tiles from there.  (Tiles straight from memory -
// 16 rows at a time, 8 bytes per lane - cost one L1 access per LANE: 54 per load instruction, and the L1s became the bound: for 65536 sequences of
// 120 tokens 370 us where the first staged form took 311, the more waves the worse.)  The next chunk's rows are on their way, in registers,
// while this one is worked on.
template <typename T, int MT, int CT, int NS = 1> struct Stage {
  static constexpr int kBytes = ElemTraits<T>::kBytes;
  static constexpr int C = 16 * CT;
  static constexpr int kLanes = kBytes * MT;                      // lanes (16-byte pieces) of a row of a or b
  static constexpr int kRow = 16 * kLanes + 16;                   // bytes between rows: 16 rows x 16 bytes hit every bank once
  static constexpr int kCLanes = kBytes * NS, kCRow = 16 * kCLanes + 16;   // the same for c: NS x 16 columns
  static constexpr int kLoads = (C * kLanes + 63) / 64, kCLoads = (C * kCLanes + 63) / 64;
  static constexpr int kRows = C < 64 / kLanes ? C : 64 / kLanes, kCRows = C < 64 / kCLanes ? C : 64 / kCLanes;   // rows of one load
  static constexpr int kArea = C * (2 * kRow + kCRow);            // LDS of a wave
};

// The staged form.  Addresses are a uniform pointer to the chunk's lowest token, which moves on by a constant, and every lane's own offset:
// the loop holds no multiplication and no scalar load (with both, 187 scalar instructions and 7 loads stood beside 325 vector ones a chunk).
// Measured: 65536 sequences of 120 tokens x 16 fp16 channels 247 - 260 us (269 under the profiler), 1.0 GB at 3.9 - 4.1 TB/s, bound by memory; two of
// 16384 tokens, 4 bf16 heads of 64 channels: 25 us, the gradients 67 us, bound by issuing a chunk's vector instructions (splits, masks, the state's
// factor) beside its 36 matrix ones at two waves per SIMD, with no registers for a third.  The four slices of such a head stage the same rows and compute
// the same scores, each wave for itself.
template <typename T, int MT, int CT, int NS, bool STATE> __global__ __launch_bounds__(256, 2) void la_kernel(LaArgs p) {
  typedef Mat<T> X;
  typedef Stage<T, MT, CT, NS> G;
  typedef typename X::Raw Raw;
  typedef typename X::Op Op;
  constexpr int kBytes = ElemTraits<T>::kBytes;
  constexpr int C = 16 * CT;
  // Rows of less than 128 bytes: the cache lines hold other heads' rows as well, so the heads' waves load at the same time (65536 sequences of 120
  // tokens x 16 channels: 260 us, 310 with each wave in its own time; wider rows only lose, 2 x 16384 tokens x 64 channels 44 us and gradients 94, 47 and
  // 102 so)
  constexpr bool kTogether = 16 * MT * kBytes < 128;
  constexpr f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  extern __shared__ __align__(16) char lds[];           // [waves][kArea], then [2][waves][NS][CT][64] sums of 4 floats if a role folds
  const Wave<T, MT, NS> w(p);
  const Role& r = p.r[blockIdx.y];
  const int lane = w.lane, c = w.c, g = w.g, reverse = r.reverse, N = r.N, B = p.B, step = p.bgroups;
  const int begin = blockIdx.z * p.seg, end = min(begin + p.seg, p.T);
  char* const area_a = lds + w.wave * G::kArea;
  char* const area_b = area_a + C * G::kRow;
  char* const area_c = area_b + C * G::kRow;
  f32x4* const sums = reinterpret_cast<f32x4*>(lds + w.waves * G::kArea);
  const int cols_bytes = r.out_f32 ? 4 : kBytes, to = p.H / r.fold * N * cols_bytes;   // bytes of a column, and of a token of out
  const int ta = r.a.st * kBytes, tb = r.b.st * kBytes, tc = r.c.st * kBytes;
  Weights<CT> k(w.decay, c, g, p.scale, r.za, r.zs, r.sh);

  // this lane's piece of a row, its row of a load, and its place in one of a whole chunk's loads
  const int piece = lane % G::kLanes * 16, piece_c = lane % G::kCLanes * 16, row_a = lane / G::kLanes, row_c = lane / G::kCLanes;
  const bool live_a = piece < r.M * kBytes && row_a < C, live_c = w.slice * 16 * G::kCLanes + piece_c < N * kBytes && row_c < C;
  // (lanes without a piece of their own bring another's again: a load for all lanes can stay in flight into the loop's registers, one for some is
  // merged with the old values by copies that wait for it)
  const int piece_r = live_a ? piece : 0, row_r = min(row_a, C - 1), piece_rc = live_c ? piece_c : 0, row_rc = min(row_c, C - 1);
  const int up_a = reverse ? C - 1 - row_r : row_r, up_c = reverse ? C - 1 - row_rc : row_rc;   // from a chunk's lowest token
  const unsigned va = (unsigned)(up_a * ta + piece_r), vb = (unsigned)(up_a * tb + piece_r), vc = (unsigned)(up_c * tc + piece_rc);
  const unsigned vo = (unsigned)((reverse ? G::kCRows - 1 - row_c : row_c) * to + piece_c);
  const int sign = reverse ? -1 : 1;
  const unsigned la = (unsigned)(sign * G::kRows * ta), lb = (unsigned)(sign * G::kRows * tb), lc = (unsigned)(sign * G::kCRows * tc);   // from load to load
  // uniform: the lowest token of the chunk in the registers, of a, b and c, from chunk to chunk; of the next store of out
  const char *ca = nullptr, *cb = nullptr, *cc = nullptr;
  char* co_at = nullptr;
  const int64_t da = (int64_t)sign * C * ta, db = (int64_t)sign * C * tb, dc = (int64_t)sign * C * tc, d_out = (int64_t)sign * G::kCRows * to;
  // a sequence's rows, and how far it is to the wave's next one
  const char *qa = reinterpret_cast<const char*>(r.a.p) + (w.bgroup * r.a.sb + (w.h / r.a.shared) * r.a.sh) * kBytes;
  const char *qb = reinterpret_cast<const char*>(r.b.p) + (w.bgroup * r.b.sb + (w.h / r.b.shared) * r.b.sh) * kBytes;
  const char *qc = reinterpret_cast<const char*>(r.c.p) + (w.bgroup * r.c.sb + (w.h / r.c.shared) * r.c.sh + w.slice * 16 * NS) * kBytes;
  char* out = reinterpret_cast<char*>(r.out) + (int64_t)w.bgroup * p.T * to + (w.h / r.fold * N + w.slice * 16 * NS) * cols_bytes;
  const int64_t next_a = step * r.a.sb * kBytes, next_b = step * r.b.sb * kBytes, next_c = step * r.c.sb * kBytes, next_out = (int64_t)step * p.T * to;
  auto place = [&](int n) {   // at a sequence's first chunk
    const int64_t tok = reverse ? n - begin - C : begin;
    ca = qa + tok * ta;
    cb = qb + tok * tb;
    cc = qc + tok * tc;
  };
  u32x4 fa[G::kLoads], fb[G::kLoads], fc[G::kCLoads];
  auto fetch = [&](int cnt) {   // the chunk at ca, cb, cc; its tokens
    unsigned oa[G::kLoads], ob[G::kLoads], oc[G::kCLoads];
    if (cnt >= C) {
#pragma unroll
      for (int i = 0; i < G::kLoads; ++i) {
        oa[i] = va + i * la;
        ob[i] = vb + i * lb;
      }
#pragma unroll
      for (int i = 0; i < G::kCLoads; ++i) oc[i] = vc + i * lc;
    } else {   // (behind the last one its row again: those scores lie above every valid token's diagonal and their weights in the state are 0)
      auto at = [&](int row) {
        const int r = min(row, cnt - 1);
        return (unsigned)(reverse ? C - 1 - r : r);
      };
#pragma unroll
      for (int i = 0; i < G::kLoads; ++i) {
        const unsigned row = at(i * G::kRows + row_r);
        oa[i] = row * ta + piece_r;
        ob[i] = row * tb + piece_r;
      }
#pragma unroll
      for (int i = 0; i < G::kCLoads; ++i) oc[i] = at(i * G::kCRows + row_rc) * tc + piece_rc;
    }
#pragma unroll
    for (int i = 0; i < G::kLoads; ++i) {
      if (!STATE) fa[i] = *reinterpret_cast<const u32x4*>(ca + oa[i]);
      fb[i] = *reinterpret_cast<const u32x4*>(cb + ob[i]);
    }
#pragma unroll
    for (int i = 0; i < G::kCLoads; ++i) fc[i] = *reinterpret_cast<const u32x4*>(cc + oc[i]);
  };
  // into the wave's LDS, which the wave alone reads (its LDS operations run in order).  Channels behind M and N were cleared once
  auto stage = [&]() {
    wave_fence();
    if (live_a)
#pragma unroll
      for (int i = 0; i < G::kLoads; ++i) {
        if (!STATE) *reinterpret_cast<u32x4*>(area_a + (i * G::kRows + row_a) * G::kRow + piece) = fa[i];
        *reinterpret_cast<u32x4*>(area_b + (i * G::kRows + row_a) * G::kRow + piece) = fb[i];
      }
    if (live_c)
#pragma unroll
      for (int i = 0; i < G::kCLoads; ++i) *reinterpret_cast<u32x4*>(area_c + (i * G::kCRows + row_c) * G::kCRow + piece_c) = fc[i];
    wave_fence();
  };
  if (!w.whole(r))
    for (int i = lane * 16; i < G::kArea; i += 1024) *reinterpret_cast<u32x4*>(area_a + i) = u32x4{0, 0, 0, 0};
  auto A = [&](int it, int t) { return *reinterpret_cast<const Raw*>(area_a + (16 * it + c) * G::kRow + (16 * t + 4 * g) * kBytes); };
  auto Bm = [&](int it, int t) { return *reinterpret_cast<const Raw*>(area_b + (16 * it + c) * G::kRow + (16 * t + 4 * g) * kBytes); };

  auto length = [&](int bi) { return bi >= B ? 0 : p.lengths ? min(max(p.lengths[bi], 0), p.T) : p.T; };
  int n = length(w.bgroup), n_next = length(w.bgroup + step), turn = 0;
  bool ready = false;   // the sequence's first chunk is on its way
  int64_t next0, next1;
  const float* s0 = w.template first_at<STATE>(p, r, &next0);
  float* s1 = w.template last_at<STATE>(p, r, &next1);
  for (int bi = w.bgroup; bi < B; bi += step, n = n_next, n_next = length(bi + step)) {
    const int stop = min(n, end);
    f32x4 S[NS][MT];
    w.load(r, s0, S);
    co_at = out + (int64_t)(reverse ? n - begin - G::kCRows : begin) * to;
    if (!ready && begin < n) {
      place(n);
      ca -= da;
      cb -= db;
      cc -= dc;
    }
    // a sequence whose first chunk is not there begins with a turn that only brings it: the loads stand in one place, where they stay in flight
    int t0 = ready ? begin : begin - C;
    ready = false;
    qa += next_a;
    qb += next_b;
    qc += next_c;
    for (; begin < n && t0 < stop; t0 += C) {
      const int cnt = min(C, stop - t0);
      if (t0 >= begin) stage();
      if constexpr (kTogether) __builtin_amdgcn_s_barrier();   // (no data is handed over)
      if (t0 + C < stop) {
        ca += da;
        cb += db;
        cc += dc;
        fetch(stop - t0 - C);
      } else {
        ready = begin < n_next;
        if (ready) place(n_next);
        fetch(ready ? n_next - begin : cnt);   // (nothing to come: the same rows again)
      }
      if (t0 < begin) continue;
      f32x4 acc[NS][CT];
      Raw craw[NS][CT];
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int t = 0; t < CT; ++t) {
          craw[s][t] = columns<T>(area_c, G::kCRow, 16 * t, s, c, g);
          acc[s][t] = zero;
        }
      if constexpr (!STATE) {
        // scores x[jt][it][j][i] = b_j . a_i
        f32x4 x[CT][CT];
#pragma unroll
        for (int it = 0; it < CT; ++it)
#pragma unroll
          for (int jt = 0; jt <= it; ++jt) x[jt][it] = zero;
        if constexpr (MT == 1) {
          Raw b[CT];
#pragma unroll
          for (int it = 0; it < CT; ++it) {
            b[it] = Bm(it, 0);
#pragma unroll
            for (int jt = 0; jt <= it; ++jt) x[jt][it] = X::raw(b[jt], A(it, 0), zero);
          }
        } else {
#pragma unroll
          for (int t = 0; t < MT; t += 2) {
            Raw b0[CT], b1[CT];
#pragma unroll
            for (int it = 0; it < CT; ++it) {
              b0[it] = Bm(it, t);
              b1[it] = Bm(it, t + 1);
#pragma unroll
              for (int jt = 0; jt <= it; ++jt) x[jt][it] = X::raw2(b0[jt], b1[jt], A(it, t), A(it, t + 1), x[jt][it]);
            }
          }
        }
        if (s0 || t0 > begin) {   // acc[it][n][i] = za g^{i+1-sh} sum_m S[m][n] a_i[m]; nothing is read from a state of zeros
          if constexpr (MT == 1) {
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
              for (int it = 0; it < CT; ++it) acc[s][it] = X::state(X::split(S[s][0]), X::op(A(it, 0)), zero);
          } else {
#pragma unroll
            for (int t = 0; t < MT; t += 2) {
              Op a0[CT], a1[CT];
#pragma unroll
              for (int it = 0; it < CT; ++it) {
                a0[it] = X::op(A(it, t));
                a1[it] = X::op(A(it, t + 1));
              }
#pragma unroll
              for (int s = 0; s < NS; ++s) {
                const typename X::Split u = X::split(S[s][t]), v = X::split(S[s][t + 1]);
#pragma unroll
                for (int it = 0; it < CT; ++it) acc[s][it] = X::state2(u, v, a0[it], a1[it], acc[s][it]);
              }
            }
          }
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int t = 0; t < CT; ++t) acc[s][t] *= k.from[t];
        }
        typename X::Split ps[CT][CT];
#pragma unroll
        for (int it = 0; it < CT; ++it)
#pragma unroll
          for (int jt = 0; jt <= it; ++jt) ps[jt][it] = X::split(k.masked(x[jt][it], it, jt, c, g));
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          Op co[CT];
          f32x4 cf[CT];
#pragma unroll
          for (int t = 0; t < CT; ++t) {
            cf[t] = X::to_float(craw[s][t]);
            co[t] = X::op(craw[s][t]);
          }
          weighted_sum<T, CT>(acc[s], ps, co, cf, c, g);
        }
      }
      if (s1 || t0 + C < stop) {   // (nothing is added to a state that nobody reads)
        k.length(w.decay, cnt, g, r.zs, r.sh);
        typename X::Split ws[NS][CT];
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int t = 0; t < CT; ++t) ws[s][t] = X::split(X::to_float(craw[s][t]) * k.into(cnt, t));
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          Op b[CT];
#pragma unroll
          for (int jt = 0; jt < CT; ++jt) b[jt] = X::op(columns<T>(area_b, G::kRow, 16 * jt, t, c, g));
#pragma unroll
          for (int s = 0; s < NS; ++s) S[s][t] = X::template grown<CT>(k.kept(S[s][t], cnt), b, ws[s]);
        }
      }
      if constexpr (!STATE) {
        const bool writes = w.template fold<CT>(acc, sums, r.fold, turn++);
        if (writes && cols_bytes == kBytes) {   // through c's place in the LDS: whole rows again, 16 bytes per lane
          wave_fence();
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int t = 0; t < CT; ++t) {
              char* const o = area_c + (16 * t + c) * G::kCRow + (16 * s + 4 * g) * kBytes;
              if constexpr (kBytes == 4) *reinterpret_cast<f32x4*>(o) = acc[s][t];
              else *reinterpret_cast<s16x4*>(o) = X::to_out(acc[s][t]);
            }
          wave_fence();
          if (live_c)
#pragma unroll
            for (int i = 0; i < G::kCLoads; ++i) {
              const int row = i * G::kCRows + row_c;
              if (row < cnt)
                *reinterpret_cast<u32x4*>(co_at + i * d_out + vo) = *reinterpret_cast<const u32x4*>(area_c + row * G::kCRow + piece_c);
            }
        } else if (writes) {
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int t = 0; t < CT; ++t) {
              const int row = 16 * t + c;
              if (row < cnt && (w.slice * NS + s) * 16 + 4 * g < N)
                *reinterpret_cast<f32x4*>(co_at + (int64_t)(reverse ? G::kCRows - 1 - row : row) * to + 64 * s + 16 * g) = acc[s][t];
            }
        }
        co_at += G::kCLoads * d_out;
      }
    }
    if (!STATE && w.writer(r.fold)) {   // tokens behind the sequence's length get zeros
      const int wide = 16 * NS * cols_bytes;   // bytes of the slice in a row: pieces of 16
      for (int i = lane; i < max(end - max(n, begin), 0) * (wide / 16); i += 64) {
        const int at = i % (wide / 16) * 16, tok = max(n, begin) + i / (wide / 16);
        if (w.slice * wide + at < N * cols_bytes) *reinterpret_cast<u32x4*>(out + (int64_t)tok * to + at) = u32x4{0, 0, 0, 0};
      }
    }
    w.store(r, s1, S);
    out += next_out;
    if (s0) s0 += next0;
    if (s1) s1 += next1;
  }
}

// Sequences of at most 16 tokens (a training clip's frames): the same arithmetic for ONE chunk, straight through.  A wave walks its sequences with
// addresses that move on by a constant, the next one's rows on their way; what depends on the length is made again only where it changes.
// (la_kernel's loops over segments and chunks cost more scalar instructions and branches here than the chunk itself: 39 us for the gradients
// of 16384 sequences of 10 tokens x 16 channels, 23 us here, when both were built.)  Forward 13.5 us, 38 MB at 2.8 TB/s (four sequences a wave: the
// launch and the decay's powers are a third of it); 65536 sequences, 4 heads of 16 channels, states in and out: 171 - 185 us, 872 MB at 4.7 - 5.1 TB/s.
// Heads of up to 32 channels are held to the registers of four waves per SIMD, which they fit (4096 sequences of 10 tokens x 32 fp16 channels 34.3 us, 37.4
// with 131 registers and three waves).
template <typename T, int MT> __global__ __launch_bounds__(256, MT <= 2 ? 4 : 2) void la_short_kernel(LaArgs p) {
  typedef Mat<T> X;
  typedef Stage<T, MT, 1> G;
  typedef typename X::Raw Raw;
  typedef typename X::Op Op;
  constexpr int kBytes = ElemTraits<T>::kBytes;
  constexpr f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  extern __shared__ __align__(16) char lds[];
  const Role& r = p.r[blockIdx.y];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int slices = (r.N + 15) >> 4, per = waves / p.group;
  const int bgroup = blockIdx.x / p.columns, f = (blockIdx.x - bgroup * p.columns) * per + wave / p.group, member = wave % p.group;
  const bool active = f < p.H / p.group * slices;
  const int slice = f % slices, h = active ? f / slices * p.group + member : 0;
  const Decay decay(p.log_decay[h]);
  const int step = p.bgroups, B = p.B, Tn = p.T, M = r.M, N = r.N, reverse = r.reverse, fold = r.fold;
  const int col = slice * 16 + c;
  const bool has_col = active && col < N;
  char* const area_a = lds + wave * G::kArea;
  char* const area_b = area_a + 16 * G::kRow;
  char* const area_c = area_b + 16 * G::kRow;
  f32x4* const sums = reinterpret_cast<f32x4*>(lds + waves * G::kArea);
  const int64_t states = (int64_t)M * N, next_states = (int64_t)step * p.H * states;
  const float* s0 = r.s0 ? r.s0 + ((int64_t)bgroup * p.H + h) * states : nullptr;
  float* s1 = r.s1 ? r.s1 + ((int64_t)bgroup * p.H + h) * states : nullptr;
  const int row_bytes = p.H / fold * N * (r.out_f32 ? 4 : kBytes), cols_bytes = r.out_f32 ? 4 : kBytes;
  char* out = reinterpret_cast<char*>(r.out) + (int64_t)bgroup * Tn * row_bytes + (h / fold * N + slice * 16) * cols_bytes;
  const int64_t next_out = (int64_t)step * Tn * row_bytes;
  const char* qa = reinterpret_cast<const char*>(r.a.p) + (bgroup * r.a.sb + (h / r.a.shared) * r.a.sh) * kBytes;
  const char* qb = reinterpret_cast<const char*>(r.b.p) + (bgroup * r.b.sb + (h / r.b.shared) * r.b.sh) * kBytes;
  const char* qc = reinterpret_cast<const char*>(r.c.p) + (bgroup * r.c.sb + (h / r.c.shared) * r.c.sh + slice * 16) * kBytes;
  const int64_t next_a = step * r.a.sb * kBytes, next_b = step * r.b.sb * kBytes, next_c = step * r.c.sb * kBytes;
  const int ta = r.a.st * kBytes, tb = r.b.st * kBytes, tc = r.c.st * kBytes;

  const int piece = lane % G::kLanes * 16, piece_c = lane % kBytes * 16, row_a = lane / G::kLanes, row_c = lane / kBytes;
  const bool live_a = piece < M * kBytes && row_a < 16, live_c = slice * 16 * kBytes + piece_c < N * kBytes && row_c < 16;
  const int piece_r = live_a ? piece : 0, piece_rc = live_c ? piece_c : 0;   // (lanes without a piece bring another's again: see la_kernel)
  constexpr bool kTogether = 16 * MT * kBytes < 128;   // (see la_kernel; 65536 sequences of 10 tokens, 4 heads of 16 channels: 171 - 185 us, 216 without.
                                                       // The gradients in one pass have fewer waves and lose by it: 417 us, 407 - 414 without)
  // lengths, and what goes by them: the lanes' places in a sequence, the weights in the state, the rows of out
  auto length = [&](int bi) { return p.lengths ? min(max(p.lengths[bi], 0), Tn) : Tn; };
  unsigned oa[G::kLoads], ob[G::kLoads], oc;
  auto places = [&](int n) {
    auto token = [&](int row) {
      const int idx = min(row, max(n, 1) - 1);
      return reverse ? max(n, 1) - 1 - idx : idx;
    };
#pragma unroll
    for (int i = 0; i < G::kLoads; ++i) {
      const int tok = token(i * G::kRows + row_a);
      oa[i] = (unsigned)(tok * ta + piece_r);
      ob[i] = (unsigned)(tok * tb + piece_r);
    }
    oc = (unsigned)(token(row_c) * tc + piece_rc);
  };
  u32x4 fa[G::kLoads], fb[G::kLoads], fc;
  auto fetch = [&]() {
#pragma unroll
    for (int i = 0; i < G::kLoads; ++i) {
      fa[i] = *reinterpret_cast<const u32x4*>(qa + oa[i]);
      fb[i] = *reinterpret_cast<const u32x4*>(qb + ob[i]);
    }
    fc = *reinterpret_cast<const u32x4*>(qc + oc);
  };
  auto columns = [&](const char* area, int row, int t) {
    if constexpr (kBytes == 2) {
      typedef __attribute__((address_space(3))) s16x4* Lds;
      return __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(area + (4 * g + (c >> 2)) * row + (16 * t + 4 * (c & 3)) * 2));
    } else {
      Raw v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const float*>(area + (4 * g + e) * row + (16 * t + c) * 4);
      return v;
    }
  };
  f32x4 inside, into;
  Factor keep(0.f, 1.f);
  const float g1 = decay.pow(1), from = r.za * decay.pow(c + 1 - r.sh);
  {
    const int d = c - 4 * g;
    inside[3] = p.scale * decay.pow(max(d - 3, 0));
#pragma unroll
    for (int e = 2; e >= 0; --e) inside[e] = d - e > 0 ? inside[e + 1] * g1 : p.scale;
  }
  auto weights = [&](int n) {
    keep = Factor(decay, n);
    const int d = n - 1 - 4 * g;
    const float w0 = r.zs * decay.pow(r.sh);
    float w = r.zs * decay.pow(max(d - 3, 0) + r.sh);
#pragma unroll
    for (int e = 3; e >= 0; --e) {
      if (e < 3) w = d - e > 0 ? w * g1 : w0;
      into[e] = d - e >= 0 ? w : 0.f;
    }
  };

  if (M != 16 * MT || N % 16 != 0)   // channels behind M and N
    for (int i = lane * 16; i < G::kArea; i += 1024) *reinterpret_cast<u32x4*>(area_a + i) = u32x4{0, 0, 0, 0};
  int n = active && bgroup < B ? length(bgroup) : 0, placed = n, weighted = -1, turn = 0;
  places(n);
  if (n > 0) fetch();
  for (int bi = bgroup; bi < B; bi += step, ++turn) {
    f32x4 S[MT];
    if (s0) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int m = 16 * t + 4 * g + e;
          const float v = s0[min(m, M - 1) * r.sm + min(col, N - 1) * r.sn];
          S[t][e] = m < M && has_col ? v : 0.f;
        }
      s0 += next_states;
    }
    if (n > 0) {   // into the wave's LDS
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (live_a)
#pragma unroll
        for (int i = 0; i < G::kLoads; ++i) {
          *reinterpret_cast<u32x4*>(area_a + (i * G::kRows + row_a) * G::kRow + piece) = fa[i];
          *reinterpret_cast<u32x4*>(area_b + (i * G::kRows + row_a) * G::kRow + piece) = fb[i];
        }
      if (live_c) *reinterpret_cast<u32x4*>(area_c + row_c * G::kCRow + piece_c) = fc;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    if constexpr (kTogether) __builtin_amdgcn_s_barrier();
    int n_next = 0;
    if (active && bi + step < B) {
      qa += next_a;
      qb += next_b;
      qc += next_c;
      n_next = length(bi + step);
      if (n_next != placed) {
        placed = n_next;
        places(n_next);
      }
      if (n_next > 0) fetch();
    }
    f32x4 acc = zero;
    if (n > 0) {
      auto A = [&](int t) { return *reinterpret_cast<const Raw*>(area_a + c * G::kRow + (16 * t + 4 * g) * kBytes); };
      auto Bm = [&](int t) { return *reinterpret_cast<const Raw*>(area_b + c * G::kRow + (16 * t + 4 * g) * kBytes); };
      const Raw craw = columns(area_c, G::kCRow, 0);
      f32x4 x = zero;
      if constexpr (MT == 1) {
        x = X::raw(Bm(0), A(0), x);
      } else {
#pragma unroll
        for (int t = 0; t < MT; t += 2) x = X::raw2(Bm(t), Bm(t + 1), A(t), A(t + 1), x);
      }
      if (s0) {
#pragma unroll
        for (int t = 0; t < MT; t += MT == 1 ? 1 : 2) {
          if constexpr (MT == 1) acc = X::state(X::split(S[0]), X::op(A(0)), acc);
          else acc = X::state2(X::split(S[t]), X::split(S[t + 1]), X::op(A(t)), X::op(A(t + 1)), acc);
        }
        acc *= from;
      }
      const f32x4 cf = X::to_float(craw);
      const Op co = X::op(craw);
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = 4 * g + e <= c ? x[e] * inside[e] : 0.f;
        top = __builtin_elementwise_maximum(top, __builtin_fabsf(cf[e]));
      }
      const typename X::Split ps = X::split(x);
      if (__builtin_expect(__any(!(top <= 3.4028234e38f)), 0)) {   // (see la_kernel)
        const f32x4 before = acc;
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
          const f32x4 y = X::add(X::upto(co, i + 1 - 4 * g), ps, before);
          if (c == i) acc = y;
        }
      } else {
        acc = X::add(co, ps, acc);
      }
      if (s1) {
        if (n != weighted) {
          weighted = n;
          weights(n);
        }
        const typename X::Split ws = X::split(cf * into);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          f32x4 v = zero;
          if (s0)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = keep(S[t][e]);
          S[t] = X::add(X::op(columns(area_b, G::kRow, t)), ws, v);
        }
      }
    } else if (!s0) {
#pragma unroll
      for (int t = 0; t < MT; ++t) S[t] = zero;
    }
    if (s1) {
      if (has_col)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int m = 16 * t + 4 * g + e;
            if (m < M) s1[m * r.sm + col * r.sn] = S[t][e];
          }
      s1 += next_states;
    }
    bool writes = active;
    if (fold > 1) {   // (see la_kernel)
      f32x4* const buf = sums + (turn & 1) * waves * 64;
      buf[wave * 64 + lane] = acc;
      __syncthreads();
      writes = active && member == 0;
      if (writes)
        for (int k = 1; k < fold; ++k) acc += buf[(wave + k) * 64 + lane];
    }
    if (writes) {
      if (c >= n) acc = zero;
      if (kBytes == 4 || cols_bytes == kBytes) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        char* const o = area_c + c * G::kCRow + 4 * g * kBytes;
        if constexpr (kBytes == 4) *reinterpret_cast<f32x4*>(o) = acc;
        else *reinterpret_cast<s16x4*>(o) = X::to_out(acc);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int tok = reverse && row_c < n ? n - 1 - row_c : row_c;
        if (live_c && row_c < Tn) *reinterpret_cast<u32x4*>(out + (unsigned)(tok * row_bytes + piece_c)) = *reinterpret_cast<const u32x4*>(area_c + row_c * G::kCRow + piece_c);
      } else if (c < Tn && slice * 16 + 4 * g < N) {
        const int tok = reverse && c < n ? n - 1 - c : c;
        *reinterpret_cast<f32x4*>(out + (unsigned)(tok * row_bytes + 16 * g)) = acc;
      }
    }
    out += next_out;
    n = n_next;
  }
}

// The three gradients of such sequences in one pass: a wave brings q, k, v and do once instead of nine rows' worth for three roles, and takes one
// slice of dq, dk and dv from them, tokens in their own order (15.9 us for 16384 sequences of 10 tokens x 16 channels; as three roles of
// la_short_kernel, when this was built, 23 where it took 15.6).  p.r[] are the roles of the general form.  Heads of up to 16 channels are held to the
// registers of four waves per SIMD, which they fit (65536 sequences, bf16: 98 us, 133 with the 171 registers and two waves that the compiler takes by itself).
template <typename T, int MT> __global__ __launch_bounds__(256, MT == 1 ? 4 : 2) void la_short_grad_kernel(LaArgs p) {
  typedef Mat<T> X;
  typedef Stage<T, MT, 1> G;
  typedef typename X::Raw Raw;
  typedef typename X::Op Op;
  constexpr int kBytes = ElemTraits<T>::kBytes;
  constexpr f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  extern __shared__ __align__(16) char lds[];
  const Role &rq = p.r[0], &rk = p.r[1], &rv = p.r[2];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int DK = rv.M, DV = rv.N, slices = (max(DK, DV) + 15) >> 4, per = waves / p.group;
  const int bgroup = blockIdx.x / p.columns, member = wave % p.group;
  int f = (blockIdx.x - bgroup * p.columns) * per + wave / p.group;
  const bool active = f < p.H / p.group * slices;
  if (!active) f = 0;
  const int slice = f % slices, h = f / slices * p.group + member, fold = rv.fold, step = p.bgroups, B = p.B;
  const Decay decay(p.log_decay[h]);
  constexpr int kRows16 = 16 * G::kRow;
  char* const area = lds + wave * 4 * kRows16;   // q, k, v, do
  f32x4* const sums = reinterpret_cast<f32x4*>(lds + waves * 4 * kRows16);

  // operand x of head h of sequence bgroup; its token stride in bytes; the way to the next sequence
  const Operand* const ops[4] = {&rk.c, &rq.c, &rq.b, &rq.a};
  const char* at[4];
  int64_t next[4];
  int ts[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    at[x] = reinterpret_cast<const char*>(ops[x]->p) + (bgroup * ops[x]->sb + (h / ops[x]->shared) * ops[x]->sh) * kBytes;
    next[x] = step * ops[x]->sb * kBytes;
    ts[x] = ops[x]->st * kBytes;
  }
  const int piece = lane % G::kLanes * 16, row = lane / G::kLanes;
  const bool live_k = piece < DK * kBytes && row < 16, live_v = piece < DV * kBytes && row < 16;
  const int piece_k = live_k ? piece : 0, piece_v = live_v ? piece : 0;   // (lanes without a piece bring another's again: see la_kernel)
  auto length = [&](int bi) { return bi >= B ? 0 : p.lengths ? min(max(p.lengths[bi], 0), p.T) : p.T; };
  u32x4 in[4][G::kLoads];
  auto fetch = [&](int n) {
#pragma unroll
    for (int i = 0; i < G::kLoads; ++i) {
      const int tok = min(i * G::kRows + row, n - 1);
#pragma unroll
      for (int x = 0; x < 4; ++x) in[x][i] = *reinterpret_cast<const u32x4*>(at[x] + (unsigned)(tok * ts[x] + (x < 2 ? piece_k : piece_v)));
    }
  };
  auto rows = [&](int x, int t) { return *reinterpret_cast<const Raw*>(area + x * kRows16 + c * G::kRow + (16 * t + 4 * g) * kBytes); };
  auto cols = [&](int x, int t) { return columns<T>(area + x * kRows16, G::kRow, 0, t, c, g); };
  if (DK != 16 * MT || DV != 16 * MT)   // (channels behind DK and DV)
    for (int i = lane * 16; i < 4 * kRows16; i += 1024) *reinterpret_cast<u32x4*>(area + i) = u32x4{0, 0, 0, 0};

  // scale g^{i-j}: [j][i] for dq, [i][j] for dk and dv;  scale g^{i+1} by lane and by element;  g^{n-1-j} by lane, and g^n
  f32x4 below, above, into;
  const float g1 = decay.pow(1), from = p.scale * decay.pow(c + 1);
  float back = 0.f;
  Factor keep(0.f, 1.f);
  int known = -1;
  {
    const int d = c - 4 * g;
    below[3] = p.scale * decay.pow(max(d - 3, 0));
    above[0] = p.scale * decay.pow(max(-d, 0));
    into[0] = p.scale * decay.pow(4 * g + 1);
#pragma unroll
    for (int e = 2; e >= 0; --e) below[e] = d - e > 0 ? below[e + 1] * g1 : p.scale;
#pragma unroll
    for (int e = 1; e < 4; ++e) {
      above[e] = e - d > 0 ? above[e - 1] * g1 : p.scale;
      into[e] = into[e - 1] * g1;
    }
  }
  // states: S of M x N read through the strides, this wave's 16 columns of it
  auto state = [&](const float* s, int M, int N, int sm, int sn, f32x4* S) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = 16 * t + 4 * g + e, n = slice * 16 + c;
        S[t][e] = 0.f;
        if (m < M && n < N) S[t][e] = s[m * sm + n * sn];
      }
  };
  const int64_t states = (int64_t)DK * DV, first = ((int64_t)bgroup * p.H + h) * states, next_states = (int64_t)step * p.H * states;
  const float *s0 = rq.s0 ? rq.s0 + first : nullptr, *d1 = rv.s0 ? rv.s0 + first : nullptr;
  float* d0 = rv.s1 ? rv.s1 + first : nullptr;
  const int tq = p.H * DK * kBytes, tk = p.H / fold * DK * kBytes, tv = p.H / fold * DV * kBytes;   // bytes of a token of dq, dk, dv
  char* oq = reinterpret_cast<char*>(rq.out) + (int64_t)bgroup * p.T * tq + (h * DK + slice * 16) * kBytes;
  char* ok = reinterpret_cast<char*>(rk.out) + (int64_t)bgroup * p.T * tk + (h / fold * DK + slice * 16) * kBytes;
  char* ov = reinterpret_cast<char*>(rv.out) + (int64_t)bgroup * p.T * tv + (h / fold * DV + slice * 16) * kBytes;
  const int piece_c = lane % kBytes * 16, row_c = lane / kBytes;
  const bool out_k = row_c < p.T && slice * 16 * kBytes + piece_c < DK * kBytes && row_c < 16, out_v = row_c < p.T && slice * 16 * kBytes + piece_c < DV * kBytes && row_c < 16;

  // acc[n][.] += sum over tokens of c[token][n] scores[token][.]; a masked token's infinity or NaN must not come through as 0 * inf.  later:
  // the tokens behind the lane's own count (dk, dv), not those in front of it (dq)
  auto sum = [&](Raw craw, f32x4 x, f32x4 acc, bool later) {
    const Op co = X::op(craw);
    const f32x4 cf = X::to_float(craw);
    const typename X::Split ps = X::split(x);
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = __builtin_elementwise_maximum(top, __builtin_fabsf(cf[e]));
    if (__builtin_expect(__any(!(top <= 3.4028234e38f)), 0)) {
      const f32x4 before = acc;
#pragma unroll 1
      for (int i = 0; i < 16; ++i) {
        const f32x4 y = X::add(later ? X::behind(co, i - 4 * g) : X::upto(co, i + 1 - 4 * g), ps, before);
        if (c == i) acc = y;
      }
      return acc;
    }
    return X::add(co, ps, acc);
  };

  int n = length(bgroup), n_next = length(bgroup + step), turn = 0;
  if (n > 0) fetch(n);
  for (int bi = bgroup; bi < B; bi += step, n = n_next, n_next = length(bi + step), ++turn) {
    if (n > 0) {
      wave_fence();
#pragma unroll
      for (int i = 0; i < G::kLoads; ++i) {
        char* const o = area + (i * G::kRows + row) * G::kRow + piece;
        if (live_k) {
          *reinterpret_cast<u32x4*>(o) = in[0][i];
          *reinterpret_cast<u32x4*>(o + kRows16) = in[1][i];
        }
        if (live_v) {
          *reinterpret_cast<u32x4*>(o + 2 * kRows16) = in[2][i];
          *reinterpret_cast<u32x4*>(o + 3 * kRows16) = in[3][i];
        }
      }
      wave_fence();
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) at[x] += next[x];
    if (n_next > 0) fetch(n_next);
    f32x4 dq = zero, dk = zero, dv = zero;
    if (n != known) {
      known = n;
      back = decay.pow(max(n - 1 - c, 0));
      keep = Factor(decay, n);
    }
    f32x4 S[MT];
    if (n > 0) {
      f32x4 x1 = zero, x2 = zero, x3 = zero;
      if constexpr (MT == 1) {
        const Raw q = rows(0, 0), k = rows(1, 0), v = rows(2, 0), d = rows(3, 0);
        x1 = X::raw(v, d, x1);
        x2 = X::raw(d, v, x2);
        x3 = X::raw(q, k, x3);
      } else {
#pragma unroll
        for (int t = 0; t < MT; t += 2) {
          const Raw q0 = rows(0, t), q1 = rows(0, t + 1), k0 = rows(1, t), k1 = rows(1, t + 1), v0 = rows(2, t), v1 = rows(2, t + 1), e0 = rows(3, t), e1 = rows(3, t + 1);
          x1 = X::raw2(v0, v1, e0, e1, x1);
          x2 = X::raw2(e0, e1, v0, v1, x2);
          x3 = X::raw2(q0, q1, k0, k1, x3);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * g + e;
        x1[e] = i <= c ? x1[e] * below[e] : 0.f;
        x2[e] = i >= c && i < n ? x2[e] * above[e] : 0.f;
        x3[e] = i >= c && i < n ? x3[e] * above[e] : 0.f;
      }
      auto inter = [&](int x, f32x4 acc) {   // sum_m S[m][n] rows_x[m]
        if constexpr (MT == 1) return X::state(X::split(S[0]), X::op(rows(x, 0)), acc);
        else {
#pragma unroll
          for (int t = 0; t < MT; t += 2) acc = X::state2(X::split(S[t]), X::split(S[t + 1]), X::op(rows(x, t)), X::op(rows(x, t + 1)), acc);
          return acc;
        }
      };
      if (s0) {
        state(s0, DV, DK, 1, DV, S);
        dq = inter(3, dq) * from;
      }
      if (d1) {
        state(d1, DV, DK, 1, DV, S);
        dk = inter(2, dk) * back;
        state(d1, DK, DV, DV, 1, S);
        dv = inter(1, dv) * back;
      }
      dq = sum(cols(1, slice), x1, dq, false);
      dk = sum(cols(0, slice), x2, dk, true);
      dv = sum(cols(3, slice), x3, dv, true);
    } else if (d1) {
      state(d1, DK, DV, DV, 1, S);
    }
    if (d0) {   // g^n dS + sum_i q_i (scale g^{i+1} do_i^T)
      if (!d1)
#pragma unroll
        for (int t = 0; t < MT; ++t) S[t] = zero;
      if (n > 0) {
        f32x4 w = X::to_float(cols(3, slice));
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = 4 * g + e < n ? w[e] * into[e] : 0.f;
        const typename X::Split ws = X::split(w);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
          for (int e = 0; e < 4; ++e) S[t][e] = keep(S[t][e]);
          S[t] = X::add(X::op(cols(0, t)), ws, S[t]);
        }
      }
      if (active && slice * 16 + c < DV)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (16 * t + 4 * g + e < DK) d0[(16 * t + 4 * g + e) * DV + slice * 16 + c] = S[t][e];
    }
    bool writes = active;
    if (fold > 1) {   // (see Wave::fold)
      f32x4* const buf = sums + (turn & 1) * waves * 128;
      buf[wave * 128 + lane] = dk;
      buf[wave * 128 + 64 + lane] = dv;
      __syncthreads();
      writes = active && member == 0;
      if (writes)
        for (int k = 1; k < fold; ++k) {
          dk += buf[(wave + k) * 128 + lane];
          dv += buf[(wave + k) * 128 + 64 + lane];
        }
    }
    if (c >= n) dq = dk = dv = zero;
    wave_fence();
    auto put = [&](int x, f32x4 v) {
      char* const o = area + x * kRows16 + c * G::kCRow + 4 * g * kBytes;
      if constexpr (kBytes == 4) *reinterpret_cast<f32x4*>(o) = v;
      else *reinterpret_cast<s16x4*>(o) = X::to_out(v);
    };
    put(0, dq);
    put(1, dk);
    put(2, dv);
    wave_fence();
    auto get = [&](int x) { return *reinterpret_cast<const u32x4*>(area + x * kRows16 + row_c * G::kCRow + piece_c); };
    if (out_k && active) *reinterpret_cast<u32x4*>(oq + (unsigned)(row_c * tq + piece_c)) = get(0);
    if (out_k && writes) *reinterpret_cast<u32x4*>(ok + (unsigned)(row_c * tk + piece_c)) = get(1);
    if (out_v && writes) *reinterpret_cast<u32x4*>(ov + (unsigned)(row_c * tv + piece_c)) = get(2);
    if (DK != 16 * MT || DV != 16 * MT) {   // (the channels behind DK and DV held parts of these rows)
      wave_fence();
      for (int i = lane * 16; i < 3 * kRows16; i += 1024) *reinterpret_cast<u32x4*>(area + i) = u32x4{0, 0, 0, 0};
    }
    oq += (int64_t)step * p.T * tq;
    ok += (int64_t)step * p.T * tk;
    ov += (int64_t)step * p.T * tv;
    if (s0) s0 += next_states;
    if (d1) d1 += next_states;
    if (d0) d0 += next_states;
  }
}

// the state in front of every segment, from each segment's own (written one place further on) and the first state: in place.  A workgroup
// takes 64 elements of one state; its waves take consecutive segments each and meet through LDS
constexpr int kMaxSegments = 256;
__global__ __launch_bounds__(1024) void la_scan_kernel(LaArgs p) {
  __shared__ float total[16][64], fades[16][2];
  const Role& r = p.r[blockIdx.z];
  const int states = r.M * r.N, x = threadIdx.x & 63, z = threadIdx.x >> 6, at = blockIdx.x * 64 + x, h = blockIdx.y % p.H, bi = blockIdx.y / p.H;
  const int64_t pair = blockIdx.y;
  const int n = p.lengths ? min(max(p.lengths[bi], 0), p.T) : p.T;
  const Decay decay(p.log_decay[h]);
  const bool live = at < states;
  float* const seg = r.seg + pair * p.segments * states + at;
  const int joins = p.segments - 1, G = blockDim.x >> 6, K = (joins + G - 1) / G, s0 = min(z * K, joins), s1 = min(s0 + K, joins);   // this group's segments
  // the decay over segment s: whole, the one that holds the sequence's end, or behind it (two floats each: a rounded factor would be off the same way
  // at every joint, 256 of them by 2^-17 together)
  const int last = n / p.seg;
  const Factor over(decay, p.seg), part(decay, n - last * p.seg);
  float own[kMaxSegments / 16], run = 0.f;
#pragma unroll
  for (int k = 0; k < kMaxSegments / 16; ++k)
    if (k < K) own[k] = s0 + k < s1 && live ? seg[(int64_t)(s0 + k + 1) * states] : 0.f;
  const float first = r.s0 && live ? r.s0[pair * states + at] : 0.f;
  auto fade = [&](int s) {   // (by value, each float by itself: a choice between objects would go through memory)
    const bool whole = s < s1 && s < last, end = s < s1 && s == last;
    return Factor::of(whole ? over.hi : end ? part.hi : 1.f, whole ? over.lo : end ? part.lo : 0.f);
  };
#pragma unroll
  for (int k = 0; k < kMaxSegments / 16; ++k)
    if (k < K) run = fade(s0 + k).plus(run, own[k]);
  total[z][x] = run;
  if (x == 0) {   // (all but the last segment are whole)
    const Factor all(decay, min(max(n - s0 * p.seg, 0), (s1 - s0) * p.seg));
    fades[z][0] = all.hi;
    fades[z][1] = all.lo;
  }
  __syncthreads();
  run = first;
#pragma unroll
  for (int y = 0; y < 15; ++y)
    if (y < z) run = Factor::of(fades[y][0], fades[y][1]).plus(run, total[y][x]);
  if (!live) return;
  if (z == 0) seg[0] = first;
#pragma unroll
  for (int k = 0; k < kMaxSegments / 16; ++k)
    if (k < K && s0 + k < s1) {
      run = fade(s0 + k).plus(run, own[k]);
      seg[(int64_t)(s0 + k + 1) * states] = run;
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
  unsigned units, H;                // B H, H
  int share, M, N;
  float scale;
  int v4;                           // v's addresses are aligned to 4 elements
};

// One token.  What counts is the state: read once, written once.  LN lanes of a wave hold W floats each of a state row, so 64 / LN rows are
// in one load; NB such loads are in flight.  WS waves share a state's rows (few states: the machine would wait for a handful of waves) and
// add their parts of o through LDS.  8192 states of 64 x 64: 67 us, 268 MB at 4.0 TB/s; 2048 of 128 x 128: 97 us, 2.8 TB/s; rows that do not fill 16
// bytes go one float a lane, 8192 of 64 x 63: 155 us, 1.7 TB/s (a wave brings no state while it works on another, see la_step_small_kernel).
template <typename T, int W, int NB, int WS> __global__ __launch_bounds__(256) void la_step_kernel(StepArgs p) {
  __shared__ float part[WS == 1 ? 1 : 4][WS == 1 ? 1 : 128];
  static_assert(WS == 1 || WS == 4, "a workgroup's waves leave together");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int LN = 1;
  while (LN < 64 && LN * W < p.N) LN *= 2;
  const int ln = lane & (LN - 1), lm = lane / LN, rows = 64 / LN;
  const int share = wave & (WS - 1);
  const unsigned stride = gridDim.x * (4 / WS);
  for (unsigned u = blockIdx.x * (4 / WS) + wave / WS; u < p.units; u += stride) {
    const unsigned row = u / p.H;
    const int h = (int)(u - row * p.H);
    const int64_t bi = row;
    float* const S = p.state + (int64_t)u * p.M * p.N;
    const float log_decay = p.log_decay[h];
    const Factor decay(log_decay, expf(log_decay));
    const int64_t oq = bi * p.qb + h * p.qh, ok = bi * p.kb + h / p.share * p.kh, ov = bi * p.vb + h / p.share * p.vh;
    for (int n = ln * W; n < ((p.N + W * LN - 1) / (W * LN)) * W * LN; n += W * LN) {
      float v[W], acc[W];
      if constexpr (W == 4) {
        f32x4 t = {0.f, 0.f, 0.f, 0.f};
        if (n < p.N) t = Mat<T>::to_float(load4<T>(reinterpret_cast<const char*>(p.v) + (ov + n) * ElemTraits<T>::kBytes, p.N - n, p.v4));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = t[e];
      } else {
        v[0] = n < p.N ? load_elem<T>(p.v, ov + n) : 0.f;
      }
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] = 0.f;
      for (int m0 = share * rows * NB; m0 < p.M; m0 += WS * rows * NB) {
        float s[NB][W], q[NB], k[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const int m = m0 + i * rows + lm;
          const bool live = n < p.N && m < p.M;
          k[i] = live ? load_elem<T>(p.k, ok + m) : 0.f;
          q[i] = live ? load_elem<T>(p.q, oq + m) : 0.f;
#pragma unroll
          for (int e = 0; e < W; ++e) s[i][e] = 0.f;
          if (live) {
            if constexpr (W == 4) Vec<F32>::load(S + m * p.N + n, s[i]);
            else s[i][0] = S[m * p.N + n];
          }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const int m = m0 + i * rows + lm;
#pragma unroll
          for (int e = 0; e < W; ++e) {
            s[i][e] = decay.plus(s[i][e], k[i] * v[e]);
            acc[e] = fmaf(q[i], s[i][e], acc[e]);
          }
          if (n < p.N && m < p.M) {
            if constexpr (W == 4) Vec<F32>::store(S + m * p.N + n, s[i]);
            else S[m * p.N + n] = s[i][0];
          }
        }
      }
#pragma unroll
      for (int e = 0; e < W; ++e)
        for (int o = 32; o >= LN; o >>= 1) acc[e] += __shfl_xor(acc[e], o, 64);
      if (n < p.N && lm == 0)
#pragma unroll
        for (int e = 0; e < W; ++e) {
          if constexpr (WS == 1) store_elem<T>(p.o, (int64_t)u * p.N + n + e, acc[e] * p.scale);
          else part[wave][n + e] = acc[e];
        }
    }
    if constexpr (WS > 1) {
      __syncthreads();
      if (share == 0)
        for (int n = lane; n < p.N; n += 64) {
          float t = part[wave][n];
#pragma unroll
          for (int k = 1; k < WS; ++k) t += part[wave + k][n];
          store_elem<T>(p.o, (int64_t)u * p.N + n, t * p.scale);
        }
      __syncthreads();
    }
  }
}

// States of one load (16 x 16 floats and smaller, M <= 64 / LN): a wave walks them with the next one on its way.  (One state at a time and
// wave, however many waves, moved 3.7 TB/s: 38 us for 65536 of 16 x 16; 27 us so, 5.3 TB/s.)
template <typename T> __global__ __launch_bounds__(256) void la_step_small_kernel(StepArgs p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int LN = 1;
  while (LN * 4 < p.N) LN *= 2;
  const int n = (lane & (LN - 1)) * 4, m = lane / LN;
  const bool live = n < p.N && m < p.M;
  const int mine = m * p.N + n, states = p.M * p.N;
  struct Unit { f32x4 s, v; float q, k, decay; };
  auto fetch = [&](unsigned u) {
    Unit x{};
    const unsigned row = u / p.H;
    const int h = (int)(u - row * p.H);
    const int64_t bi = row;
    x.decay = p.log_decay[h];
    if (live) {
      x.s = *reinterpret_cast<const f32x4*>(p.state + (int64_t)u * states + mine);
      x.k = load_elem<T>(p.k, bi * p.kb + h / p.share * p.kh + m);
      x.q = load_elem<T>(p.q, bi * p.qb + h * p.qh + m);
      x.v = Mat<T>::to_float(load4<T>(reinterpret_cast<const char*>(p.v) + (bi * p.vb + h / p.share * p.vh + n) * ElemTraits<T>::kBytes, p.N - n, p.v4));
    }
    return x;
  };
  const unsigned stride = gridDim.x * 4;
  unsigned u = blockIdx.x * 4 + wave;
  if (u >= p.units) return;
  Unit x = fetch(u);
  for (;;) {
    const unsigned next = u + stride;
    Unit y = x;
    if (next < p.units) y = fetch(next);
    const Factor decay(x.decay, expf(x.decay));
    f32x4 acc;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x.s[e] = decay.plus(x.s[e], x.k * x.v[e]);
      acc[e] = x.q * x.s[e];
    }
    if (live) *reinterpret_cast<f32x4*>(p.state + (int64_t)u * states + mine) = x.s;
    for (int o = 32; o >= LN; o >>= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o, 64);
    if (live && m == 0)
#pragma unroll
      for (int e = 0; e < 4; ++e) store_elem<T>(p.o, (int64_t)u * p.N + n + e, acc[e] * p.scale);
    if (next >= p.units) return;
    x = y;
    u = next;
  }
}

inline bool known(int dtype) { return dtype == TG_F32 || dtype == TG_BF16 || dtype == TG_F16; }
inline int elem_bytes(int dtype) { return dtype == TG_F32 ? 4 : 2; }
inline bool elem_aligned(int dtype, const void* p) { return (reinterpret_cast<uintptr_t>(p) & (elem_bytes(dtype) - 1)) == 0; }
inline bool word_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

constexpr int kMaxHead = 128;
constexpr int kFold = 4;   // shared heads that are summed inside a workgroup; more: through `scratch` and la_share_kernel

inline int tiles(int m) { return m <= 16 ? 1 : m <= 32 ? 2 : m <= 64 ? 4 : 8; }

// Segments: as many as two waves per SIMD need, each of at least kMinSegment tokens.  They cost an additional pass over b and c and two launches, about
// what the whole sequence takes in 400 tokens of 16 bits or in 200 of fp32, and twice that where the machine is half full already.  Forward (gradients) of
// two sequences, 4 heads of 64, states in and out, whole and in segments: bf16 300 tokens 20 us and 17 (20 and 21), 700 tokens 36 and 20 (36 and 26); fp32
// 200 tokens 26 and 18 (26 and 20); of 20 sequences: bf16 700 tokens 37 and 42 (41 and 50), 1000 tokens 51 and 45 (54 and 61); fp32 300 tokens 35 and 40 (39 and
// 51), 520 tokens 56 and 48 (58 and 69: the gradients' three roles leave room for two segments).  Two segments never bring anything (64 sequences of 2000
// tokens, fp32: 191 us whole and 214)
constexpr int64_t kWaves = 2048;
constexpr int kMinSegment = 32;
constexpr int kCUs = 256;

// (tokens in a segment, segments) for `waves` waves per segment
void segmentation(int dtype, int T, int64_t waves, int* seg, int* segments) {
  int64_t want = waves > 0 ? kWaves / waves : 1, most = (T + kMinSegment - 1) / kMinSegment;
  if (want > most) want = most;
  if (want > kMaxSegments) want = kMaxSegments;
  const int whole = (dtype == TG_F32 ? 256 : 512) * (want < 8 ? 2 : 1);
  if (want < 3 || T < whole) { *seg = (T + 31) / 32 * 32; *segments = 1; return; }
  int64_t s = (T + want - 1) / want;
  s = (s + 31) / 32 * 32;
  *seg = (int)s;
  *segments = (int)((T + s - 1) / s);
}

// One launch.  Sequences are dealt out so that the grid fills the machine ONCE (a wave makes its decay's powers once, and no second round of
// workgroups finds the machine half empty: a third more waves than fit ran 338 us, as many as fit 274)
constexpr int kDevices = 16;
struct Resident { std::atomic<int> n[kDevices][2][kFold + 1]; };   // a kernel's workgroups on a CU, by device, folds and waves; 0: not known yet
int go(void (*kernel)(LaArgs), Resident& resident, int area, int ct, bool folds, LaArgs a, dim3 grid, int threads, hipStream_t st) {
  const int waves = threads / 64, lds = (folds ? 2 * waves * ct * 64 * 16 : 0) + waves * area;
  int dev;
  TG_CHECK_HIP(hipGetDevice(&dev));   // (a kernel's attributes are each device's own)
  int per_cu = dev < kDevices ? resident.n[dev][folds][waves].load(std::memory_order_relaxed) : 0;
  if (per_cu == 0) {
    TG_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    TG_CHECK_HIP(hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, reinterpret_cast<const void*>(kernel), threads, (size_t)lds));
    if (per_cu < 1) return TG_E_UNSUPPORTED;
    if (dev < kDevices) resident.n[dev][folds][waves].store(per_cu, std::memory_order_relaxed);
  }
  const int64_t columns = a.columns, others = columns * grid.y * grid.z, room = (int64_t)per_cu * kCUs;
  const int64_t each = (a.B * others + room - 1) / room;             // sequences of a workgroup
  a.bgroups = (int)((a.B + each - 1) / each);
  if (columns * a.bgroups > 0x7fffffff) return TG_E_UNSUPPORTED;
  grid.x = (unsigned)(columns * a.bgroups);
  kernel<<<grid, threads, lds, st>>>(a);
  return tg_launch_status();
}
template <typename T, int MT, int CT, int NS, bool STATE> int go_long(const LaArgs& a, dim3 grid, int threads, hipStream_t st) {
  static Resident resident;
  return go(la_kernel<T, MT, CT, NS, STATE>, resident, Stage<T, MT, CT, NS>::kArea, CT * NS, !STATE && a.group > 1, a, grid, threads, st);
}
template <typename T, int MT, int CT, bool STATE> int go_plain(const LaArgs& a, dim3 grid, int threads, hipStream_t st) {
  static Resident resident;
  return go(la_plain_kernel<T, MT, CT, STATE>, resident, Turn<T, MT, CT>::kArea, CT, !STATE && a.group > 1, a, grid, threads, st);
}
template <typename T, int MT> int go_short(const LaArgs& a, dim3 grid, int threads, hipStream_t st) {
  if constexpr (MT < 8) {   // (128 channels: three roles, their registers do not fit one wave)
    if (grid.y == 3 && !a.r[1].out_f32) {   // the three gradients
      static Resident resident;
      grid.y = 1;
      return go(la_short_grad_kernel<T, MT>, resident, 4 * 16 * Stage<T, MT, 1>::kRow, 2, a.group > 1, a, grid, threads, st);
    }
  }
  static Resident resident;
  return go(la_short_kernel<T, MT>, resident, Stage<T, MT, 1>::kArea, 1, a.group > 1, a, grid, threads, st);
}
// Slices of 32 columns share a chunk's scores, its rows and the columns of b between two of 16: worth it where half the waves still fill the
// machine (128 sequences of 2000 tokens, 4 bf16 heads of 64: 145 - 152 us, 177 in slices of 16; gradients 418 us, 671), not where sequences are cut
// into segments for want of waves (20 such sequences: 79 us, 59 in slices of 16; gradients 101 us, 95).  For heads wider than 16 channels beside
// operands of 17 .. 64 in 16 bits; fp32 and 128 channels do not fit the registers so
constexpr int64_t kWideWaves = 512;
inline bool can_be_wide(int dtype, int M, int N) { return dtype != TG_F32 && N > 16 && (tiles(M) == 2 || tiles(M) == 4); }
inline int slice_tiles(int dtype, int M, int N, bool wide) { return wide && can_be_wide(dtype, M, N) ? 2 : 1; }

template <typename T, int MT> int go_mt(const LaArgs& a, bool staged, bool state, int ns, dim3 grid, int threads, hipStream_t st) {
  // chunks of 32 tokens halve the work on the state per token; sequences of one chunk of 16 would waste half of them, and two tiles of 128
  // fp32 channels, or of 128 channels that every lane loads itself, do not fit the registers
  constexpr bool f32 = sizeof(typename Mat<T>::Raw) == 16;
  constexpr int CT = MT == 8 && f32 ? 1 : 2, CU = MT == 8 ? 1 : 2;
  if (staged) {
    if (!state && a.T <= 16) return go_short<T, MT>(a, grid, threads, st);
    if constexpr (!f32 && (MT == 2 || MT == 4))
      if (ns == 2) return state ? go_long<T, MT, CT, 2, true>(a, grid, threads, st) : go_long<T, MT, CT, 2, false>(a, grid, threads, st);
    return state ? go_long<T, MT, CT, 1, true>(a, grid, threads, st) : go_long<T, MT, CT, 1, false>(a, grid, threads, st);
  }
  if (state) return go_plain<T, MT, CU, true>(a, grid, threads, st);
  return a.T <= 16 ? go_plain<T, MT, 1, false>(a, grid, threads, st) : go_plain<T, MT, CU, false>(a, grid, threads, st);
}
// `roles` roles with the same number of m tiles in one launch
template <typename T> int launch(LaArgs a, int dtype, int roles, bool state, hipStream_t st) {
  int mt = 1, most = 1, ns = 2;
  bool staged = true;
  for (int i = 0; i < roles; ++i) {
    const Role& r = a.r[i];
    if (tiles(r.M) > mt) mt = tiles(r.M);
    if (r.N > most) most = r.N;
    if (slice_tiles(dtype, r.M, r.N, a.wide) < ns) ns = slice_tiles(dtype, r.M, r.N, a.wide);
    staged = staged && r.pieces;
  }
  if (!staged || (!state && a.T <= 16)) ns = 1;
  const int slices = (most + 16 * ns - 1) / (16 * ns);
  // workgroups of up to kFold waves, as few idle ones among them as possible
  const int64_t units = (int64_t)(a.H / a.group) * slices;
  if (units > 0x7fffff00) return TG_E_UNSUPPORTED;
  int per = 1;
  for (int k = 2; k <= kFold / a.group; ++k)
    if ((units + k - 1) / k * k <= (units + per - 1) / per * per) per = k;
  a.columns = (int)((units + per - 1) / per);
  const dim3 grid(1, roles, state ? a.segments - 1 : a.segments);
  const int threads = 64 * per * a.group;
  if (mt == 1) return go_mt<T, 1>(a, staged, state, ns, grid, threads, st);
  if (mt == 2) return go_mt<T, 2>(a, staged, state, ns, grid, threads, st);
  if (mt == 4) return go_mt<T, 4>(a, staged, state, ns, grid, threads, st);
  return go_mt<T, 8>(a, staged, state, ns, grid, threads, st);
}
int launch_dt(int dtype, const LaArgs& a, int roles, bool state, hipStream_t st) {
  TG_DISPATCH_DTYPE(dtype, return launch<BF16>(a, dtype, roles, state, st), return launch<F16>(a, dtype, roles, state, st),
                    return launch<F32>(a, dtype, roles, state, st));
}

struct Strided { Operand o; bool wide, pieces; };   // aligned to 4 elements, to 16 bytes: the address and all strides
Strided operand(int dtype, const void* p, const int64_t* stride, int shared) {
  auto aligned = [&](int n) {
    return (reinterpret_cast<uintptr_t>(p) & (n * elem_bytes(dtype) - 1)) == 0 && stride[0] % n == 0 && stride[1] % n == 0 && stride[2] % n == 0;
  };
  // (a chunk's rows are reached by 32-bit offsets: 32 tokens of up to 2^25 bytes)
  return {Operand{p, stride[0], stride[2], (int)stride[1], shared}, aligned(4), aligned(16 / elem_bytes(dtype)) && stride[1] * elem_bytes(dtype) <= (1 << 25)};
}

constexpr int kMost = 1 << 30;   // sequences and tokens: the kernels' steps beyond the last one stay within 32 bits
int check(int dtype, const tg_la_desc* d) {
  if (!d || !known(dtype) || d->B < 0 || d->T < 0 || d->H <= 0 || d->HK <= 0 || d->DK <= 0 || d->DV <= 0) return TG_E_BADARG;
  if (d->H % d->HK || d->DK > kMaxHead || d->DV > kMaxHead || d->B > kMost || d->T > kMost || d->H > 65536) return TG_E_UNSUPPORTED;
  for (const int64_t* s : {d->q_stride, d->k_stride, d->v_stride})
    if (s[0] < 0 || s[1] < 0 || s[2] < 0) return TG_E_BADARG;
    else if (s[1] > 0x7fffffff) return TG_E_UNSUPPORTED;
  return TG_OK;
}

inline int64_t slices_of(int dtype, int M, int N, bool wide) {
  const int n = 16 * slice_tiles(dtype, M, N, wide);
  return (N + n - 1) / n;
}
// slices and segments of the forward pass (one role) and of the backward pass (three)
void plan(int dtype, const tg_la_desc* d, bool backward, LaArgs* a) {
  auto waves = [&](bool wide) {
    const int64_t one = slices_of(dtype, d->DK, d->DV, wide);
    return (int64_t)d->B * d->H * (backward ? one + 2 * slices_of(dtype, d->DV, d->DK, wide) : one);
  };
  a->wide = waves(true) >= kWideWaves;
  segmentation(dtype, d->T, waves(a->wide), &a->seg, &a->segments);
}
inline int64_t states(const tg_la_desc* d) { return (int64_t)d->B * d->H * d->DK * d->DV; }
inline int64_t fold_floats(const tg_la_desc* d) { return d->H / d->HK > kFold ? (int64_t)d->B * d->T * d->H * (d->DK + d->DV) : 0; }

// segments' states: own ones, then joined
int join_segments(int dtype, const LaArgs& a, int roles, hipStream_t st) {
  const int rc = launch_dt(dtype, a, roles, true, st);
  if (rc != TG_OK) return rc;
  const int joins = a.segments - 1, waves = joins < 16 ? joins : 16;
  la_scan_kernel<<<dim3((a.r[0].M * a.r[0].N + 63) / 64, (unsigned)(a.B * a.H), roles), 64 * waves, 0, st>>>(a);
  return tg_launch_status();
}

// (16-byte aligned state rows go 4 floats a lane)
template <typename T> int launch_step(const StepArgs& a, bool wide, hipStream_t st) {
  auto grid = [&](int64_t units_of_wg, int64_t most) {   // units beyond `most` workgroups are walked
    const int64_t n = ((int64_t)a.units + units_of_wg - 1) / units_of_wg;
    return (int)(n < most * kCUs ? n : most * kCUs);
  };
  int LN = 1;
  while (LN * 4 < a.N) LN *= 2;
  if (!wide) la_step_kernel<T, 1, 4, 1><<<grid(4, 16), 256, 0, st>>>(a);
  else if (a.M * LN <= 64) la_step_small_kernel<T><<<grid(4, 8), 256, 0, st>>>(a);
  else if (a.units < 4 * kCUs) la_step_kernel<T, 4, 4, 4><<<grid(1, 16), 256, 0, st>>>(a);
  else la_step_kernel<T, 4, 4, 1><<<grid(4, 16), 256, 0, st>>>(a);
  return tg_launch_status();
}

}  // namespace

extern "C" int64_t tg_linear_attention_scratch_floats(int dtype, const tg_la_desc* d) {
  if (check(dtype, d) != TG_OK) return 0;
  LaArgs a;
  plan(dtype, d, false, &a);
  return a.segments > 1 ? a.segments * states(d) : 0;
}

extern "C" int tg_linear_attention(int dtype, const tg_la_desc* d, const void* q, const void* k, const void* v, const float* log_decay,
                                   const int32_t* lengths, const float* state_in, void* o, float* state_out, float* scratch, void* stream) {
  int rc = check(dtype, d);
  if (rc != TG_OK) return rc;
  if (d->B == 0) return TG_OK;
  LaArgs a{};
  plan(dtype, d, false, &a);
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
  const int piece = 16 / elem_bytes(dtype);
  const bool pieces = wide && Q.pieces && K.pieces && V.pieces && tg_aligned16(o) && d->DK % piece == 0 && d->DV % piece == 0;
  a.r[0] = Role{Q.o, K.o, V.o, o, state_in, state_out, scratch, d->DK, d->DV, d->DV, 1, d->scale, 1.f, 0, 0, 1, 0, wide, pieces};
  if (a.segments > 1 && (rc = join_segments(dtype, a, 1, st)) != TG_OK) return rc;
  return launch_dt(dtype, a, 1, false, st);
}

extern "C" int64_t tg_linear_attention_bwd_scratch_floats(int dtype, const tg_la_desc* d) {
  if (check(dtype, d) != TG_OK) return 0;
  LaArgs a;
  plan(dtype, d, true, &a);
  return fold_floats(d) + (a.segments > 1 ? 2 * a.segments * states(d) : 0);
}

extern "C" int tg_linear_attention_bwd(int dtype, const tg_la_desc* d, const void* q, const void* k, const void* v, const void* dout,
                                       const int64_t* dout_stride, const float* log_decay, const int32_t* lengths, const float* state_in,
                                       const float* dstate_out, void* dq, void* dk, void* dv, float* dstate_in, float* scratch, void* stream) {
  int rc = check(dtype, d);
  if (rc != TG_OK) return rc;
  if (d->B == 0) return TG_OK;
  LaArgs a{};
  plan(dtype, d, true, &a);
  const int G = d->H / d->HK;
  if (!log_decay || !dout_stride || (d->T > 0 && (!q || !k || !v || !dout || !dq || !dk || !dv)) || (tg_linear_attention_bwd_scratch_floats(dtype, d) && !scratch))
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
  const int piece = 16 / elem_bytes(dtype);
  const bool pieces = wide && Q.pieces && K.pieces && V.pieces && D.pieces && DK % piece == 0 && DV % piece == 0;
  if (a.segments > 1) {
    a.r[0] = Role{Q.o, K.o, V.o, nullptr, state_in, nullptr, seg_s, DK, DV, DV, 1, 0.f, 1.f, 0, 0, 1, 0, wide, pieces};
    a.r[1] = Role{K.o, Q.o, D.o, nullptr, dstate_out, nullptr, seg_d, DK, DV, DV, 1, 0.f, d->scale, 1, 1, 1, 0, wide, pieces};
    if ((rc = join_segments(dtype, a, 2, st)) != TG_OK) return rc;
  }
  const Role rq{D.o, V.o, K.o, dq, state_in, nullptr, seg_s, DV, DK, 1, DV, d->scale, 1.f, 0, 0, 1, 0, wide, pieces};
  const Role rk{V.o, D.o, Q.o, apart ? (void*)part_k : dk, dstate_out, nullptr, seg_d, DV, DK, 1, DV, 1.f, d->scale, 1, 1, fold, apart, wide, pieces};
  const Role rv{K.o, Q.o, D.o, apart ? (void*)part_v : dv, dstate_out, dstate_in, seg_d, DK, DV, DV, 1, 1.f, d->scale, 1, 1, fold, apart, wide, pieces};
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
  const Strided V = operand(dtype, v, d->v_stride, 1);
  if ((int64_t)d->B * d->H > 0x40000000) return TG_E_UNSUPPORTED;
  StepArgs a{q, k, v, o, state, log_decay, d->q_stride[0], d->q_stride[2], d->k_stride[0], d->k_stride[2], d->v_stride[0], d->v_stride[2],
             (unsigned)d->B * d->H, (unsigned)d->H, d->H / d->HK, d->DK, d->DV, d->scale, V.wide};
  const bool wide = d->DV % 4 == 0 && tg_aligned16(state);
  hipStream_t st = (hipStream_t)stream;
  TG_DISPATCH_DTYPE(dtype, return launch_step<BF16>(a, wide, st), return launch_step<F16>(a, wide, st), return launch_step<F32>(a, wide, st));
}
