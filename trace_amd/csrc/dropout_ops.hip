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

constexpr int DROP_U = 2;   // counter blocks of eight elements per thread, all loaded before the first is drawn

template <typename T> struct DropVec {   // eight elements
  uint4 w[sizeof(T) / 2];
};

// A workgroup per DROP_U x 256 counter blocks; the elements behind the last whole block are done one by one.
template <typename T, bool BWD>
__global__ __launch_bounds__(256) void dropout_act_kernel(const DropArgs p) {
  const uint64_t off = p.offset + (p.step ? (uint64_t)*p.step : 0);
  const long long whole = p.n >> 3, b0 = (long long)blockIdx.x * (DROP_U * 256) + threadIdx.x;
  const bool need_x = !BWD || p.act;
  const bool relu = p.act & TRACE_EPI_RELU;
  const DropVec<T>*xp = static_cast<const DropVec<T>*>(p.x), *gp = static_cast<const DropVec<T>*>(p.dy);
  auto one = [&](float x, float g, uint32_t piece) {
    float v;
    bool neg;
    if (BWD) {
      v = g * p.scale;
      neg = p.act && !(x > 0.f);
    } else {
      v = x * p.scale;
      neg = p.act && v < 0.f;   // NaN stays
    }
    // relu selects: the scale may have made v infinite, and 0 times that is no zero
    if (neg) v = relu ? 0.f : v * 0.1f;
    return piece < p.threshold ? 0.f : v;
  };
  DropVec<T> xv[DROP_U], gv[DROP_U];
#pragma unroll
  for (int u = 0; u < DROP_U; ++u) {
    const long long b = b0 + u * 256;
    if (b < whole) {
      if (need_x) xv[u] = xp[b];
      if (BWD) gv[u] = gp[b];
    }
  }
#pragma unroll
  for (int u = 0; u < DROP_U; ++u) {
    const long long b = b0 + u * 256;
    if (b > whole) break;
    uint32_t w[4];
    drop_pieces((uint64_t)b, off, p.seed, w);
    if (b < whole) {
      DropVec<T> o;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float x0 = 0.f, x1 = 0.f, g0 = 0.f, g1 = 0.f;
        const uint32_t *xw = &xv[u].w[0].x, *gw = &gv[u].w[0].x;
        uint32_t* ow = &o.w[0].x;
        if constexpr (sizeof(T) == 2) {
          if (need_x) x0 = __uint_as_float(xw[e / 2] << 16), x1 = __uint_as_float(xw[e / 2] & 0xffff0000u);
          if (BWD) g0 = __uint_as_float(gw[e / 2] << 16), g1 = __uint_as_float(gw[e / 2] & 0xffff0000u);
          ow[e / 2] = pack_bf16x2(one(x0, g0, w[e / 2] & 0xffffu), one(x1, g1, w[e / 2] >> 16));
        } else {
          if (need_x) x0 = __uint_as_float(xw[e]), x1 = __uint_as_float(xw[e + 1]);
          if (BWD) g0 = __uint_as_float(gw[e]), g1 = __uint_as_float(gw[e + 1]);
          ow[e] = __float_as_uint(one(x0, g0, w[e / 2] & 0xffffu));
          ow[e + 1] = __float_as_uint(one(x1, g1, w[e / 2] >> 16));
        }
      }
      static_cast<DropVec<T>*>(p.out)[b] = o;
    } else {
      const T *xt = static_cast<const T*>(p.x) + b * 8, *gt = static_cast<const T*>(p.dy) + b * 8;
      T* ot = static_cast<T*>(p.out) + b * 8;
      const int cnt = (int)(p.n - b * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < cnt)
          ot[e] = drop_put<T>(one(need_x ? drop_get<T>(xt[e]) : 0.f, BWD ? drop_get<T>(gt[e]) : 0.f,
                                  (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu));
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
  const long long wg = (n / 8 + 1 + DROP_U * 256 - 1) / (DROP_U * 256);   // a block more for what is behind the whole ones
  TRACE_REQUIRE(wg < (1ll << 31), "%s: too many elements", what);
  const unsigned grid = (unsigned)wg;
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
