// Dropout + activation with the mask drawn from a counter (gfx950): nothing is stored, the backward pass redraws it.
//
//   piece(i) = 16-bit piece i % 8 of Philox4x32-10(counter = (i / 8, offset + *step), key = seed)   (Salmon et al., SC 2011)
//   y_i = piece(i) < threshold ? 0 : act(x_i * 65536 / (65536 - threshold)),   dx_i = kept ? act'(x_i) dy_i * .. : 0
//
// Bound by HBM (x in, y out) as long as the generator stays below it: ten rounds are twenty 32 x 32 -> 64-bit products, at a
// quarter of the add rate.  A call of the generator therefore serves EIGHT elements with 16 bits each - the probability has a
// resolution of 2^-16, and the scale is that of the probability actually drawn, so the expectation is exact -: eight bf16
// elements are also one 16-byte access.  One rounding per element, at the end.
#include "common.h"
#include <type_traits>

namespace trace {

struct DropArgs {
  const void *x, *dy;   // dy: backward (then x is read only where the activation needs it)
  void* out;
  long long n;
  uint32_t threshold;
  float scale;
  uint64_t seed, offset;
  const int64_t* step;
  int act;
};

// the pieces of counter block b
__device__ __forceinline__ void drop_pieces(uint64_t b, uint64_t off, uint64_t seed, uint32_t (&w)[4]) {
  uint32_t c0 = (uint32_t)b, c1 = (uint32_t)(b >> 32), c2 = (uint32_t)off, c3 = (uint32_t)(off >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}

template <typename T> __device__ __forceinline__ float drop_get(T v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else return bf16_to_f32(v);
}
template <typename T> __device__ __forceinline__ T drop_put(float v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else return f32_to_bf16(v);
}

// a thread per counter block of eight elements; the block behind the last whole one is done element by element
template <typename T, bool BWD>
__global__ __launch_bounds__(256) void dropout_act_kernel(const DropArgs p) {
  const uint64_t off = p.offset + (p.step ? (uint64_t)*p.step : 0);
  const long long blocks = (p.n + 7) >> 3, stride = (long long)gridDim.x * 256;
  const bool need_x = !BWD || p.act;
  const float low = (p.act & TRACE_EPI_RELU) ? 0.f : (p.act & TRACE_EPI_LEAKY) ? 0.1f : 1.f;
  for (long long b = (long long)blockIdx.x * 256 + threadIdx.x; b < blocks; b += stride) {
    const long long i0 = b * 8;
    const int cnt = (int)min((long long)8, p.n - i0);
    const T *xp = static_cast<const T*>(p.x) + i0, *gp = static_cast<const T*>(p.dy) + i0;
    T* op = static_cast<T*>(p.out) + i0;
    T xv[8], gv[8], ov[8];
    if (cnt == 8) {
      if (need_x) {
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<uint4*>(xv) = *reinterpret_cast<const uint4*>(xp);
        } else {
          reinterpret_cast<uint4*>(xv)[0] = reinterpret_cast<const uint4*>(xp)[0];
          reinterpret_cast<uint4*>(xv)[1] = reinterpret_cast<const uint4*>(xp)[1];
        }
      }
      if (BWD) {
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<uint4*>(gv) = *reinterpret_cast<const uint4*>(gp);
        } else {
          reinterpret_cast<uint4*>(gv)[0] = reinterpret_cast<const uint4*>(gp)[0];
          reinterpret_cast<uint4*>(gv)[1] = reinterpret_cast<const uint4*>(gp)[1];
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (need_x && e < cnt) xv[e] = xp[e];
        if (BWD && e < cnt) gv[e] = gp[e];
      }
    }
    uint32_t w[4];
    drop_pieces((uint64_t)b, off, p.seed, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t piece = (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu;
      float v;
      if (BWD) {
        v = drop_get<T>(gv[e]) * p.scale;
        if (p.act && !(drop_get<T>(xv[e]) > 0.f)) v *= low;
      } else {
        v = drop_get<T>(xv[e]) * p.scale;
        if (p.act) v = v < 0.f ? v * low : v;   // NaN stays
      }
      ov[e] = drop_put<T>(piece < p.threshold ? 0.f : v);
    }
    if (cnt == 8) {
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(op) = *reinterpret_cast<const uint4*>(ov);
      } else {
        reinterpret_cast<uint4*>(op)[0] = reinterpret_cast<const uint4*>(ov)[0];
        reinterpret_cast<uint4*>(op)[1] = reinterpret_cast<const uint4*>(ov)[1];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < cnt) op[e] = ov[e];
    }
  }
}

template <typename T>
static int drop_call(bool backward, const T* x, const T* dy, long long n, int threshold, uint64_t seed, uint64_t offset,
                     const int64_t* step, int act, T* out, void* stream) {
  const char* what = backward ? "dropout backward" : "dropout";
  TRACE_REQUIRE(n >= 0, "%s: negative size", what);
  TRACE_REQUIRE(threshold >= 0 && threshold <= 65536, "%s: threshold %d (0 .. 65536)", what, threshold);
  TRACE_REQUIRE(act == 0 || act == TRACE_EPI_RELU || act == TRACE_EPI_LEAKY, "%s: act takes one of RELU / LEAKY", what);
  if (n == 0) return 0;
  TRACE_REQUIRE(out && (x || (backward && !act)) && (dy || !backward), "%s: null pointer", what);
  TRACE_REQUIRE((((uintptr_t)x | (uintptr_t)dy | (uintptr_t)out) & 15) == 0, "%s: operands must be 16-byte aligned", what);
  TRACE_REQUIRE(((uintptr_t)step & 7) == 0, "%s: step must be 8-byte aligned", what);
  DropArgs a = {};
  a.x = x;
  a.dy = dy;
  a.out = out;
  a.n = n;
  a.threshold = (uint32_t)threshold;
  a.scale = threshold < 65536 ? 65536.f / (float)(65536 - threshold) : 0.f;
  a.seed = seed;
  a.offset = offset;
  a.step = step;
  a.act = act;
  const long long wg = ((n + 7) / 8 + 255) / 256;
  const unsigned grid = (unsigned)(wg < 4096 ? wg : 4096);
  if (backward) dropout_act_kernel<T, true><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  else dropout_act_kernel<T, false><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  return check_launch(what);
}

}  // namespace trace

using namespace trace;

extern "C" int trace_dropout_act_bf16(const uint16_t* x, long long n, int threshold, uint64_t seed, uint64_t offset,
                                      const int64_t* step, int act, uint16_t* y, trace_stream_t stream) {
  return drop_call<uint16_t>(false, x, nullptr, n, threshold, seed, offset, step, act, y, stream);
}
extern "C" int trace_dropout_act_f32(const float* x, long long n, int threshold, uint64_t seed, uint64_t offset,
                                     const int64_t* step, int act, float* y, trace_stream_t stream) {
  return drop_call<float>(false, x, nullptr, n, threshold, seed, offset, step, act, y, stream);
}
extern "C" int trace_dropout_act_bwd_bf16(const uint16_t* x, const uint16_t* dy, long long n, int threshold, uint64_t seed,
                                          uint64_t offset, const int64_t* step, int act, uint16_t* dx, trace_stream_t stream) {
  return drop_call<uint16_t>(true, x, dy, n, threshold, seed, offset, step, act, dx, stream);
}
extern "C" int trace_dropout_act_bwd_f32(const float* x, const float* dy, long long n, int threshold, uint64_t seed,
                                         uint64_t offset, const int64_t* step, int act, float* dx, trace_stream_t stream) {
  return drop_call<float>(true, x, dy, n, threshold, seed, offset, step, act, dx, stream);
}
