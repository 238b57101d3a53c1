// Dropout from a counter-based generator: y = (residual +) keep * x / (1 - p).  The mask is never stored: element i's random word is
// word i % 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) at the counter
// (i / 4 low, i / 4 high, layer, step) under the 64-bit key `seed`, kept if word >= threshold = round(p 2^32).  Forward and backward are the
// same launch on other tensors.  (seed, step) are read from device memory, so a captured graph draws a new mask on every replay whose step
// has moved.  The mask depends on the element's index alone, not on the element type or on how a launch is cut.
// Bound by memory: 655360 x 64 bf16 elements with a residual, and the gradient, 84 us together, 420 MB at 5.0 TB/s (what a large copy reaches); eight
// elements a lane are two 16-byte pieces at most and two generator blocks.
#include "common.h"

namespace {

struct Words { unsigned w[4]; };

__device__ __forceinline__ Words philox(uint64_t block, unsigned layer, unsigned step, unsigned k0, unsigned k1) {
  unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32), c2 = layer, c3 = step;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;   // one v_mad_u64_u32 each
    c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
    c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
    c1 = (unsigned)b;
    c3 = (unsigned)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// eight elements per thread: two generator calls, 16 (32) bytes per operand
template <typename T, bool WIDE> __global__ __launch_bounds__(256) void dropout_kernel(const void* x, const void* res, void* y, int64_t n,
                                                                                       float up, unsigned threshold, const int64_t* rng, int layer) {
  const uint64_t seed = (uint64_t)rng[0];
  const unsigned step = (unsigned)rng[1];
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 256 * 8) {
    float v[8], r[8];
    const bool whole = WIDE && i + 8 <= n;
    if (whole) {
#pragma unroll
      for (int k = 0; k < 8; k += Vec<T>::N) Vec<T>::load(reinterpret_cast<const char*>(x) + (i + k) * ElemTraits<T>::kBytes, v + k);
      if (res)
#pragma unroll
        for (int k = 0; k < 8; k += Vec<T>::N) Vec<T>::load(reinterpret_cast<const char*>(res) + (i + k) * ElemTraits<T>::kBytes, r + k);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = i + k < n ? load_elem<T>(x, i + k) : 0.f;
        if (res) r[k] = i + k < n ? load_elem<T>(res, i + k) : 0.f;
      }
    }
    const Words a = philox((uint64_t)i >> 2, (unsigned)layer, step, (unsigned)seed, (unsigned)(seed >> 32));
    const Words b = philox(((uint64_t)i >> 2) + 1, (unsigned)layer, step, (unsigned)seed, (unsigned)(seed >> 32));
#pragma unroll
    for (int k = 0; k < 8; ++k) {   // a selection, not a product: a dropped infinity or NaN is gone
      v[k] = (k < 4 ? a.w[k & 3] : b.w[k & 3]) >= threshold ? v[k] * up : 0.f;
      if (res) v[k] += r[k];
    }
    if (whole) {
#pragma unroll
      for (int k = 0; k < 8; k += Vec<T>::N) Vec<T>::store(reinterpret_cast<char*>(y) + (i + k) * ElemTraits<T>::kBytes, v + k);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + k < n) store_elem<T>(y, i + k, v[k]);
    }
  }
}

template <typename T> int launch(const void* x, const void* res, void* y, int64_t n, float up, unsigned threshold, const int64_t* rng, int layer,
                                 hipStream_t st) {
  const int64_t need = (n + 2047) / 2048;
  const int grid = (int)(need < (1 << 20) ? need : (1 << 20));
  if (tg_aligned16(x) && tg_aligned16(res) && tg_aligned16(y)) dropout_kernel<T, true><<<grid, 256, 0, st>>>(x, res, y, n, up, threshold, rng, layer);
  else dropout_kernel<T, false><<<grid, 256, 0, st>>>(x, res, y, n, up, threshold, rng, layer);
  return tg_launch_status();
}

}  // namespace

extern "C" int tg_dropout(int dtype, const void* x, const void* res, void* y, int64_t n, double p, const int64_t* rng, int layer, void* stream) {
  if (dtype != TG_F32 && dtype != TG_BF16 && dtype != TG_F16) return TG_E_BADARG;
  if (n < 0 || !(p >= 0.0 && p < 1.0)) return TG_E_BADARG;
  if (n == 0) return TG_OK;
  if (!x || !y || !rng) return TG_E_BADARG;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(res) | reinterpret_cast<uintptr_t>(y);
  if ((bits & (dtype == TG_F32 ? 3 : 1)) || (reinterpret_cast<uintptr_t>(rng) & 7)) return TG_E_ALIGN;
  const double t = floor(p * 4294967296.0 + 0.5);
  const unsigned threshold = t >= 4294967295.0 ? 0xffffffffu : (unsigned)t;   // (p within 2^-33 of one)
  const float up = (float)(1.0 / (1.0 - p));
  hipStream_t st = (hipStream_t)stream;
  TG_DISPATCH_DTYPE(dtype, return launch<BF16>(x, res, y, n, up, threshold, rng, layer, st),
                    return launch<F16>(x, res, y, n, up, threshold, rng, layer, st),
                    return launch<F32>(x, res, y, n, up, threshold, rng, layer, st));
}
