// Group normalisation with an activation over channels-last maps, forward and backward (gfx950).
//
//   z = (x - mean) rstd gamma + beta,  y = act(z);  mean / var over the P * C / G elements of a (sample, group)
//   dz = act'(z) dy,  dgamma_c = sum dz xh,  dbeta_c = sum dz,  xh = (x - mean) rstd,  t = dz gamma
//   dx = rstd (t - mean_group(t) - xh mean_group(t xh))
//
// Bound by HBM: x once in, y once out (backward: x and dy in, dx out).  Two forms:
//   * one workgroup per (sample, slab of whole groups) that keeps the slab in registers between the statistics and the
//     result: everything is read once, one launch.  Taken where the slab fits (P rows of at least 64 contiguous bytes, <=
//     GN_R_FWD / GN_R_BWD 16-byte pieces per thread);
//   * larger maps in two passes over (sample, chunk of rows), a small merge of the chunks' partial results between them; the
//     second pass walks the chunks from the last to the first, so that it starts with what the caches still hold.
// Statistics are merged as (count, mean, sum of squared deviations), never as sum of squares minus squared sum: a map whose
// mean is far from zero loses nothing.  All sums in f32, in a fixed order.
#include "common.h"
#include <type_traits>

namespace trace {

constexpr int GN_BT = 512;      // threads of the one-pass form
constexpr int GN_R_FWD = 32, GN_R_BWD = 16;   // 16-byte pieces (pairs of them) that a thread of it keeps
constexpr int GN_CT = 256;      // threads of the two-pass form
constexpr int GN_MAX_C = 8192;

struct GnArgs {
  const void *x, *dy;
  const float *gamma, *beta;
  void* out;            // y or dx
  float *stats, *dgamma, *dbeta;
  float *part;          // two-pass: partial statistics / sums
  float *csum;          // backward: (N, C, 2) sums of dz and dz xh
  float *gsum;          // backward: (N, G, 2) sums of t and t xh
  int N, C, G, Cg, P, act;
  float eps;
  int slab;             // groups per workgroup of the one-pass form
  int pow2;             // its columns, and those of a group, are powers of two of whole accesses
  int rows, chunks;     // two-pass: rows per chunk
  int nt;               // two-pass: results are stored past the caches
};

// V elements of T as loaded: bf16 as 32-bit words of two (one element alone: itself), f32 as they are
template <typename T, int V> struct GnVec;
template <> struct GnVec<uint16_t, 8> { typedef __attribute__((ext_vector_type(4))) uint32_t type; };
template <> struct GnVec<uint16_t, 4> { typedef __attribute__((ext_vector_type(2))) uint32_t type; };
template <> struct GnVec<uint16_t, 2> { typedef __attribute__((ext_vector_type(1))) uint32_t type; };
template <> struct GnVec<uint16_t, 1> { typedef uint16_t type; };
template <> struct GnVec<float, 4> { typedef __attribute__((ext_vector_type(4))) float type; };
template <> struct GnVec<float, 2> { typedef __attribute__((ext_vector_type(2))) float type; };
template <> struct GnVec<float, 1> { typedef __attribute__((ext_vector_type(1))) float type; };

// bf16 pairs are taken apart by 32-bit operations where they are used: as 16-bit elements every one would hold a register
template <typename T, int V> __device__ __forceinline__ void gn_unpack(const typename GnVec<T, V>::type& r, float (&f)[V]) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = r[i];
  } else if constexpr (V == 1) {
    f[0] = bf16_to_f32(r);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      f[2 * i] = __uint_as_float(r[i] << 16);
      f[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
}
template <typename T, int V> __device__ __forceinline__ typename GnVec<T, V>::type gn_pack(const float (&f)[V]) {
  typename GnVec<T, V>::type r;
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = f[i];
  } else if constexpr (V == 1) {
    r = f32_to_bf16(f[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
  }
  return r;
}

// between the rows of an unrolled loop: the compiler would otherwise unpack all of them at once, in as many registers
__device__ __forceinline__ void gn_row_done() { __builtin_amdgcn_sched_barrier(0); }

// hardware reciprocal (1 ulp): a correctly rounded division would cost more than the rest of the element
__device__ __forceinline__ float gn_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

template <int V> __device__ __forceinline__ void gn_act(float (&z)[V], int act) {
  if (act & TRACE_EPI_RELU) {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = z[i] < 0.f ? 0.f : z[i];   // NaN stays
  } else if (act & TRACE_EPI_LEAKY) {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = z[i] < 0.f ? 0.1f * z[i] : z[i];
  } else if (act & TRACE_EPI_SILU) {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = z[i] * gn_sigmoid(z[i]);
  }
}
// dz = act'(z) dy
template <int V> __device__ __forceinline__ void gn_dact(const float (&z)[V], float (&d)[V], int act) {
  if (act & TRACE_EPI_RELU) {
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = z[i] > 0.f ? d[i] : 0.f;
  } else if (act & TRACE_EPI_LEAKY) {
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = z[i] > 0.f ? d[i] : 0.1f * d[i];
  } else if (act & TRACE_EPI_SILU) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float s = gn_sigmoid(z[i]);
      d[i] = d[i] * s * (1.f + z[i] * (1.f - s));
    }
  }
}

// a[e][s], e < len, s < nseg: sums over e, left in a[0][s].  Every thread of the workgroup calls it.
template <int BT> __device__ __forceinline__ void gn_sum_rows(float* a, int nseg, int len, int tid) {
  __syncthreads();
  int st = 1;
  while (st < len) st <<= 1;
  for (st >>= 1; st >= 1; st >>= 1) {
    const int n = min(st, len - st) * nseg;
    for (int i = tid; i < n; i += BT) a[i] += a[i + st * nseg];
    len = min(len, st);
    __syncthreads();
  }
}
// a[s][j], j < len, s < nseg: sums over j, left in a[s][0]
template <int BT> __device__ __forceinline__ void gn_sum_cols(float* a, int nseg, int len, int tid) {
  __syncthreads();
  const int pitch = len;
  int st = 1;
  while (st < len) st <<= 1;
  for (st >>= 1; st >= 1; st >>= 1) {
    const int m = min(st, len - st);
    for (int i = tid; i < m * nseg; i += BT) {
      const int s = i / m, j = i - s * m;
      a[s * pitch + j] += a[s * pitch + j + st];
    }
    len = min(len, st);
    __syncthreads();
  }
}

// Group sums of K values per thread where a slab's columns (SW, CVG of them to a group) are powers of two: butterflies over the
// lane bits that do not tell groups apart, then one exchange between the waves.  Every thread gets the sums of its own group.
template <int BT, int K> __device__ __forceinline__ void gn_group_sums(float (&v)[K], int SW, int CVG, float* red, int tid) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1)
    if (o < CVG || o >= SW) {
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], o);
    }
  // column of a thread within the slab -> its group; a slab wider than a wave has several waves per row
  const int groups = SW / CVG, g = (tid & (SW - 1)) / CVG, span = max(min(CVG, 64), 1);
  if (((tid & 63) & (span - 1)) == 0 && (SW >= 64 || (tid & 63) < SW)) {
    // one writer per (wave, group present in the wave)
#pragma unroll
    for (int k = 0; k < K; ++k) red[((tid >> 6) * groups + g) * K + k] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = 0.f;
  for (int w = 0; w < BT / 64; ++w) {
    // waves of a wide slab hold different columns: only those whose columns meet this group
    if (SW > 64) {
      const int first = (w * 64) & (SW - 1);
      if (first / CVG > g || (first + 63) / CVG < g) continue;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += red[(w * groups + g) * K + k];
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------------------------------------------
// One pass: workgroup (slab of `slab` groups, sample).  Thread = one V-wide column of the slab, rows tid / SW + i RP.
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int V, int R>
__global__ __launch_bounds__(GN_BT, 2) void gn_fwd_slab_kernel(const GnArgs p) {
  using Raw = typename GnVec<T, V>::type;
  __shared__ float red[GN_BT * V];
  __shared__ float mu[GN_BT * V], rs[GN_BT * V];   // per channel of the slab
  const int tid = threadIdx.x, n = blockIdx.y;
  const int SC = p.slab * p.Cg, SW = SC / V, RP = GN_BT / SW;   // slab channels, columns, rows per step
  const int c0 = blockIdx.x * SC;
  const int r0 = tid / SW, col = (tid - r0 * SW) * V;
  const bool on = r0 < RP;
  const T* x = static_cast<const T*>(p.x) + (long long)n * p.P * p.C + c0 + col;
  Raw raw[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = r0 + i * RP;
    if (on && row < p.P) raw[i] = *reinterpret_cast<const Raw*>(x + (long long)row * p.C);
  }
  const float inv = 1.f / ((float)p.P * (float)p.Cg);
  float mean[V], rstd[V], s[V];
#pragma unroll
  for (int v = 0; v < V; ++v) mean[v] = 0.f;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {   // the mean, then the squared deviations from it
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (on && r0 + i * RP < p.P) {
        float f[V];
        gn_unpack<T, V>(raw[i], f);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = pass ? f[v] - mean[v] : f[v];
          s[v] += pass ? d * d : d;
          asm volatile("" : "+v"(s[v]));   // one after the other: joined to wide vectors, 32 narrow rows spill
        }
      }
      gn_row_done();
    }
    if (p.pow2) {
      float t[1] = {0.f};
#pragma unroll
      for (int v = 0; v < V; ++v) t[0] += s[v];
      gn_group_sums<GN_BT, 1>(t, SW, p.Cg / V, red, tid);
      const float r = pass ? 1.f / sqrtf(t[0] * inv + p.eps) : t[0] * inv;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (pass) rstd[v] = r;
        else mean[v] = r;
      }
      continue;
    }
    if (on) {
#pragma unroll
      for (int v = 0; v < V; ++v) red[r0 * SC + col + v] = s[v];
    }
    gn_sum_rows<GN_BT>(red, SC, RP, tid);
    gn_sum_cols<GN_BT>(red, p.slab, p.Cg, tid);
    float* dst = pass ? rs : mu;
    for (int c = tid; c < SC; c += GN_BT) {
      const float t = red[c / p.Cg * p.Cg] * inv;
      dst[c] = pass ? 1.f / sqrtf(t + p.eps) : t;
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (pass) rstd[v] = on ? rs[col + v] : 0.f;
      else mean[v] = on ? mu[col + v] : 0.f;
    }
  }
  if (!on) return;
  if (r0 == 0) {   // the thread that holds a group's first channel
#pragma unroll
    for (int v = 0; v < V; ++v)
      if ((col + v) % p.Cg == 0) {
        float* st = p.stats + 2 * ((long long)n * p.G + (c0 + col + v) / p.Cg);
        st[0] = mean[v];
        st[1] = rstd[v];
      }
  }
  float ga[V], be[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    ga[v] = rstd[v] * (p.gamma ? p.gamma[c0 + col + v] : 1.f);
    be[v] = p.beta ? p.beta[c0 + col + v] : 0.f;
  }
  T* y = static_cast<T*>(p.out) + (long long)n * p.P * p.C + c0 + col;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = r0 + i * RP;
    if (row < p.P) {
      float f[V];
      gn_unpack<T, V>(raw[i], f);
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] = (f[v] - mean[v]) * ga[v] + be[v];
      gn_act<V>(f, p.act);
      *reinterpret_cast<Raw*>(y + (long long)row * p.C) = gn_pack<T, V>(f);
    }
    gn_row_done();
  }
}

// a channel's sums of dz and dz xh in one sample: the parameters' gradients themselves if there is no other sample
__device__ __forceinline__ void gn_channel_out(const GnArgs& p, int n, int c, float a, float b) {
  if (p.N > 1) {
    *reinterpret_cast<float2*>(p.csum + 2 * ((long long)n * p.C + c)) = make_float2(a, b);
  } else {
    if (p.dbeta) p.dbeta[c] = a;
    if (p.dgamma) p.dgamma[c] = b;
  }
}

template <typename T, int V, int R>
__global__ __launch_bounds__(GN_BT, 2) void gn_bwd_slab_kernel(const GnArgs p) {
  using Raw = typename GnVec<T, V>::type;
  __shared__ float ra[GN_BT * V], rb[GN_BT * V];
  const int tid = threadIdx.x, n = blockIdx.y;
  const int SC = p.slab * p.Cg, SW = SC / V, RP = GN_BT / SW;
  const int c0 = blockIdx.x * SC;
  const int r0 = tid / SW, col = (tid - r0 * SW) * V;
  const bool on = r0 < RP;
  const long long base = (long long)n * p.P * p.C + c0 + col;
  const T *x = static_cast<const T*>(p.x) + base, *dy = static_cast<const T*>(p.dy) + base;
  Raw rx[R], rd[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = r0 + i * RP;
    if (on && row < p.P) {
      rx[i] = *reinterpret_cast<const Raw*>(x + (long long)row * p.C);
      rd[i] = *reinterpret_cast<const Raw*>(dy + (long long)row * p.C);
    }
  }
  float mean[V], rstd[V], ga[V], be[V], a[V], b[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = c0 + (on ? col + v : 0);
    const float* st = p.stats + 2 * ((long long)n * p.G + c / p.Cg);
    mean[v] = st[0];
    rstd[v] = st[1];
    ga[v] = p.gamma ? p.gamma[c] : 1.f;
    be[v] = p.beta ? p.beta[c] : 0.f;
    a[v] = b[v] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (on && r0 + i * RP < p.P) {
      float f[V], d[V], z[V];
      gn_unpack<T, V>(rx[i], f);
      gn_unpack<T, V>(rd[i], d);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        f[v] = (f[v] - mean[v]) * rstd[v];
        z[v] = f[v] * ga[v] + be[v];
      }
      gn_dact<V>(z, d, p.act);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        a[v] += d[v];
        b[v] += d[v] * f[v];
      }
    }
    gn_row_done();
  }
  const float inv = 1.f / ((float)p.P * (float)p.Cg);
  if (p.pow2) {
    float t[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      t[0] += a[v] * ga[v];
      t[1] += b[v] * ga[v];
    }
    gn_group_sums<GN_BT, 2>(t, SW, p.Cg / V, ra, tid);
    // per channel: over the rows of a wave, then over the waves (of a slab as wide as a wave or wider there is nothing to add
    // within one, and the waves of one column are SW / 64 apart)
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
      if (o >= SW) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          a[v] += __shfl_xor(a[v], o);
          b[v] += __shfl_xor(b[v], o);
        }
      }
    if ((tid & 63) < SW) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        ra[(tid & 63) * V + v + (tid >> 6) * (min(SW, 64) * V)] = a[v];
        rb[(tid & 63) * V + v + (tid >> 6) * (min(SW, 64) * V)] = b[v];
      }
    }
    __syncthreads();
    const int per = min(SW, 64) * V, apart = max(SW / 64, 1);   // channels a wave holds, waves per row
    for (int c = tid; c < SC; c += GN_BT) {
      float sa = 0.f, sb = 0.f;
      for (int w = c / per; w < GN_BT / 64; w += apart) {
        sa += ra[w * per + c % per];
        sb += rb[w * per + c % per];
      }
      gn_channel_out(p, n, c0 + c, sa, sb);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      a[v] = t[0] * inv;
      b[v] = t[1] * inv;
    }
  } else {
    if (on) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        ra[r0 * SC + col + v] = a[v];
        rb[r0 * SC + col + v] = b[v];
      }
    }
    gn_sum_rows<GN_BT>(ra, SC, RP, tid);
    gn_sum_rows<GN_BT>(rb, SC, RP, tid);
    for (int c = tid; c < SC; c += GN_BT) {   // per channel: kept for dgamma / dbeta; weighted: the group's sums
      gn_channel_out(p, n, c0 + c, ra[c], rb[c]);
      const float w = p.gamma ? p.gamma[c0 + c] : 1.f;
      ra[c] *= w;
      rb[c] *= w;
    }
    gn_sum_cols<GN_BT>(ra, p.slab, p.Cg, tid);
    gn_sum_cols<GN_BT>(rb, p.slab, p.Cg, tid);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int g = on ? (col + v) / p.Cg * p.Cg : 0;
      a[v] = ra[g] * inv;
      b[v] = rb[g] * inv;
    }
  }
  if (!on) return;
  T* dx = static_cast<T*>(p.out) + base;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = r0 + i * RP;
    if (row < p.P) {
      float f[V], d[V], z[V];
      gn_unpack<T, V>(rx[i], f);
      gn_unpack<T, V>(rd[i], d);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        f[v] = (f[v] - mean[v]) * rstd[v];
        z[v] = f[v] * ga[v] + be[v];
      }
      gn_dact<V>(z, d, p.act);
#pragma unroll
      for (int v = 0; v < V; ++v) d[v] = (d[v] * ga[v] - a[v] - f[v] * b[v]) * rstd[v];
      *reinterpret_cast<Raw*>(dx + (long long)row * p.C) = gn_pack<T, V>(d);
    }
    gn_row_done();
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Two passes: workgroup (chunk of rows, sample), all channels.  Thread = V-wide columns tid % CV (+ GN_CT ..), rows of its
// own; with C / V <= GN_CT columns RP = GN_CT / CV rows go side by side.
// ---------------------------------------------------------------------------------------------------------------
// groups of the V channels from c on: one division
template <int V> __device__ __forceinline__ void gn_groups(int c, int Cg, int (&g)[V]) {
  int q = c / Cg, r = c - q * Cg;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    g[v] = q;
    if (++r == Cg) {
      r = 0;
      ++q;
    }
  }
}

struct GnMom {   // count, mean, sum of squared deviations
  float n, mean, m2;
};
__device__ __forceinline__ GnMom gn_merge(const GnMom& a, const GnMom& b) {
  const float n = a.n + b.n;
  if (n == 0.f) return a;
  const float d = b.mean - a.mean, w = b.n / n;
  return {n, a.mean + d * w, a.m2 + b.m2 + d * d * a.n * w};
}

// rows a thread loads before it uses them; in the backward kernels, where a row is two loads, half as many (8 x 25088 x 256
// without an activation: backward 109 -> 103 us; 8 rows leave registers for three waves per SIMD only)
constexpr int GN_U = 8, GN_UB = 4;

// The result of the last pass.  Maps beyond GN_NT_BYTES are stored past the caches: written lines would push out what the pass
// still has to read there (8 x 25088 x 256, SiLU: forward 77 -> 69 us, backward 123 -> 112; with the copies that write x and dy and read the
// results 315 -> 306).  Smaller maps stay for whoever reads them next (49 MB: 182 us in that chain, 186 past the caches).
constexpr long long GN_NT_BYTES = 64ll << 20;
template <typename Raw> __device__ __forceinline__ void gn_store(void* at, const Raw& v, int nt) {
  if (nt) {
    asm volatile("");   // else the compiler makes one plain store of the two
    __builtin_nontemporal_store(v, static_cast<Raw*>(at));
    asm volatile("");
  } else {
    *static_cast<Raw*>(at) = v;
  }
}

template <typename T, int V>
__global__ __launch_bounds__(GN_CT) void gn_stats_kernel(const GnArgs p) {
  using Raw = typename GnVec<T, V>::type;
  extern __shared__ float sm[];   // [RP * C] means, [RP * C] squared deviations, [RP] counts
  const int tid = threadIdx.x, n = blockIdx.y, chunk = blockIdx.x;
  const int CV = p.C / V, RP = CV < GN_CT ? GN_CT / CV : 1;
  const int row0 = chunk * p.rows, row1 = min(row0 + p.rows, p.P);
  float *me = sm, *m2 = sm + RP * p.C, *cn = sm + 2 * RP * p.C;
  const int rr = CV < GN_CT ? tid / CV : 0;
  if (rr < RP) {
    for (int cv = CV < GN_CT ? tid - rr * CV : tid; cv < CV; cv += CV < GN_CT ? CV : GN_CT) {
      const T* x = static_cast<const T*>(p.x) + (long long)n * p.P * p.C + (long long)cv * V;
      float cnt = 0.f, mean[V], dev[V];
#pragma unroll
      for (int v = 0; v < V; ++v) mean[v] = dev[v] = 0.f;
      for (int row = row0 + rr; row < row1; row += GN_U * RP) {
        Raw raw[GN_U];
        int k = 0;
#pragma unroll
        for (int i = 0; i < GN_U; ++i)
          if (row + i * RP < row1) {
            raw[i] = *reinterpret_cast<const Raw*>(x + (long long)(row + i * RP) * p.C);
            ++k;
          }
        // mean and squared deviations of these k rows, merged into the running ones
        float s[V], q[V];
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = q[v] = 0.f;
#pragma unroll
        for (int i = 0; i < GN_U; ++i)
          if (i < k) {
            float f[V];
            gn_unpack<T, V>(raw[i], f);
#pragma unroll
            for (int v = 0; v < V; ++v) s[v] += f[v];
            gn_row_done();
          }
        const float kf = (float)k, ik = 1.f / kf, tot = cnt + kf, w = kf / tot;
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] *= ik;
#pragma unroll
        for (int i = 0; i < GN_U; ++i)
          if (i < k) {
            float f[V];
            gn_unpack<T, V>(raw[i], f);
#pragma unroll
            for (int v = 0; v < V; ++v) q[v] += (f[v] - s[v]) * (f[v] - s[v]);
            gn_row_done();
          }
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = s[v] - mean[v];
          mean[v] += d * w;
          dev[v] += q[v] + d * d * cnt * w;
        }
        cnt = tot;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        me[rr * p.C + cv * V + v] = mean[v];
        m2[rr * p.C + cv * V + v] = dev[v];
      }
      cn[rr] = cnt;   // equal for all columns
    }
  }
  __syncthreads();
  // rows side by side, then the channels of each group: pairs at a time
  int len = RP, st = 1;
  while (st < len) st <<= 1;
  for (st >>= 1; st >= 1; st >>= 1) {
    const int m = min(st, len - st);
    for (int i = tid; i < m * p.C; i += GN_CT) {
      const int e = i / p.C, j = i + st * p.C;
      const GnMom r = gn_merge({cn[e], me[i], m2[i]}, {cn[e + st], me[j], m2[j]});
      me[i] = r.mean;
      m2[i] = r.m2;
    }
    __syncthreads();
    if (tid < m) cn[tid] += cn[tid + st];
    len = min(len, st);
    __syncthreads();
  }
  const float rows = (float)(row1 - row0);
  len = p.Cg;
  st = 1;
  while (st < len) st <<= 1;
  // entry j of a group holds `width(j)` channels: those j, j + st, j + 2 st .. folded so far
  for (st >>= 1; st >= 1; st >>= 1) {
    const int m = min(st, len - st);
    for (int i = tid; i < m * p.G; i += GN_CT) {
      const int g = i / m, j = i - g * m, a = g * p.Cg + j;
      // channels folded into entry e while `len` entries are left: those = e mod (the stride of the last fold)
      const int span = len == p.Cg ? p.Cg : 2 * st;
      const float na = rows * (float)((p.Cg - j + span - 1) / span), nb = rows * (float)((p.Cg - (j + st) + span - 1) / span);
      const GnMom r = gn_merge({na, me[a], m2[a]}, {nb, me[a + st], m2[a + st]});
      me[a] = r.mean;
      m2[a] = r.m2;
    }
    len = min(len, st);
    __syncthreads();
  }
  for (int g = tid; g < p.G; g += GN_CT) {
    float* o = p.part + 2 * (((long long)n * p.chunks + chunk) * p.G + g);
    o[0] = me[g * p.Cg];
    o[1] = m2[g * p.Cg];
  }
}

// workgroup per (group, sample): the chunks' moments, each thread a strided list in order, then pairs of lanes, then the waves
// -> stats
__global__ __launch_bounds__(GN_CT) void gn_merge_kernel(const GnArgs p) {
  __shared__ GnMom wm[GN_CT / 64];
  const int tid = threadIdx.x, g = blockIdx.x, n = blockIdx.y;
  GnMom m = {0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = tid; k < p.chunks; k += GN_CT) {
    const float2 o = *reinterpret_cast<const float2*>(p.part + 2 * (((long long)n * p.chunks + k) * p.G + g));
    m = gn_merge(m, {(float)min(p.rows, p.P - k * p.rows) * (float)p.Cg, o.x, o.y});
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const GnMom t = {__shfl_xor(m.n, o), __shfl_xor(m.mean, o), __shfl_xor(m.m2, o)};
    m = (tid & o) ? gn_merge(t, m) : gn_merge(m, t);   // both lanes the same way round
  }
  if ((tid & 63) == 0) wm[tid >> 6] = m;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < GN_CT / 64; ++w) m = gn_merge(m, wm[w]);
    *reinterpret_cast<float2*>(p.stats + 2 * ((long long)n * p.G + g)) = make_float2(m.mean, 1.f / sqrtf(m.m2 / m.n + p.eps));
  }
}

template <typename T, int V>
__global__ __launch_bounds__(GN_CT) void gn_apply_kernel(const GnArgs p) {
  using Raw = typename GnVec<T, V>::type;
  const int tid = threadIdx.x, n = blockIdx.y, chunk = p.chunks - 1 - blockIdx.x;
  const int CV = p.C / V, RP = CV < GN_CT ? GN_CT / CV : 1;
  const int row0 = chunk * p.rows, row1 = min(row0 + p.rows, p.P);
  const int rr = CV < GN_CT ? tid / CV : 0;
  if (rr >= RP) return;
  for (int cv = CV < GN_CT ? tid - rr * CV : tid; cv < CV; cv += CV < GN_CT ? CV : GN_CT) {
    float mean[V], ga[V], be[V];
    int grp[V];
    gn_groups<V>(cv * V, p.Cg, grp);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = cv * V + v;
      const float2 st = *reinterpret_cast<const float2*>(p.stats + 2 * ((long long)n * p.G + grp[v]));
      mean[v] = st.x;
      ga[v] = st.y * (p.gamma ? p.gamma[c] : 1.f);
      be[v] = p.beta ? p.beta[c] : 0.f;
    }
    const long long base = (long long)n * p.P * p.C + (long long)cv * V;
    const T* x = static_cast<const T*>(p.x) + base;
    T* y = static_cast<T*>(p.out) + base;
    for (int row = row0 + rr; row < row1; row += GN_U * RP) {
      Raw raw[GN_U];
#pragma unroll
      for (int i = 0; i < GN_U; ++i)
        if (row + i * RP < row1) raw[i] = *reinterpret_cast<const Raw*>(x + (long long)(row + i * RP) * p.C);
#pragma unroll
      for (int i = 0; i < GN_U; ++i)
        if (row + i * RP < row1) {
          float f[V];
          gn_unpack<T, V>(raw[i], f);
#pragma unroll
          for (int v = 0; v < V; ++v) f[v] = (f[v] - mean[v]) * ga[v] + be[v];
          gn_act<V>(f, p.act);
          gn_store<Raw>(y + (long long)(row + i * RP) * p.C, gn_pack<T, V>(f), p.nt);
          gn_row_done();
        }
    }
  }
}

// per chunk and channel: sums of dz and dz xh -> part (N, chunks, C, 2)
template <typename T, int V>
__global__ __launch_bounds__(GN_CT) void gn_bwd_sums_kernel(const GnArgs p) {
  using Raw = typename GnVec<T, V>::type;
  extern __shared__ float sm[];   // [RP * C] x 2
  const int tid = threadIdx.x, n = blockIdx.y, chunk = blockIdx.x;
  const int CV = p.C / V, RP = CV < GN_CT ? GN_CT / CV : 1;
  const int row0 = chunk * p.rows, row1 = min(row0 + p.rows, p.P);
  float *sa = sm, *sb = sm + RP * p.C;
  const int rr = CV < GN_CT ? tid / CV : 0;
  if (rr < RP) {
    for (int cv = CV < GN_CT ? tid - rr * CV : tid; cv < CV; cv += CV < GN_CT ? CV : GN_CT) {
      const long long base = (long long)n * p.P * p.C + (long long)cv * V;
      const T *x = static_cast<const T*>(p.x) + base, *dy = static_cast<const T*>(p.dy) + base;
      float mean[V], rstd[V], ga[V], be[V], a[V], b[V];
      int grp[V];
      gn_groups<V>(cv * V, p.Cg, grp);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = cv * V + v;
        const float2 st = *reinterpret_cast<const float2*>(p.stats + 2 * ((long long)n * p.G + grp[v]));
        mean[v] = st.x;
        rstd[v] = st.y;
        ga[v] = p.gamma ? p.gamma[c] : 1.f;
        be[v] = p.beta ? p.beta[c] : 0.f;
        a[v] = b[v] = 0.f;
      }
      for (int row = row0 + rr; row < row1; row += GN_UB * RP) {
        Raw rx[GN_UB], rd[GN_UB];
#pragma unroll
        for (int i = 0; i < GN_UB; ++i)
          if (row + i * RP < row1) {
            rx[i] = *reinterpret_cast<const Raw*>(x + (long long)(row + i * RP) * p.C);
            rd[i] = *reinterpret_cast<const Raw*>(dy + (long long)(row + i * RP) * p.C);
          }
#pragma unroll
        for (int i = 0; i < GN_UB; ++i)
          if (row + i * RP < row1) {
            float f[V], d[V], z[V];
            gn_unpack<T, V>(rx[i], f);
            gn_unpack<T, V>(rd[i], d);
#pragma unroll
            for (int v = 0; v < V; ++v) {
              f[v] = (f[v] - mean[v]) * rstd[v];
              z[v] = f[v] * ga[v] + be[v];
            }
            gn_dact<V>(z, d, p.act);
#pragma unroll
            for (int v = 0; v < V; ++v) {
              a[v] += d[v];
              b[v] += d[v] * f[v];
            }
            gn_row_done();
          }
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        sa[rr * p.C + cv * V + v] = a[v];
        sb[rr * p.C + cv * V + v] = b[v];
      }
    }
  }
  gn_sum_rows<GN_CT>(sa, p.C, RP, tid);
  gn_sum_rows<GN_CT>(sb, p.C, RP, tid);
  float* o = p.part + 2 * ((long long)n * p.chunks + chunk) * p.C;
  for (int c = tid; c < p.C; c += GN_CT) *reinterpret_cast<float2*>(o + 2 * c) = make_float2(sa[c], sb[c]);
}

// workgroup (group, sample): the chunks' sums -> csum (N, C, 2), weighted over the group's channels -> gsum (N, G, 2)
__global__ __launch_bounds__(GN_CT) void gn_bwd_merge_kernel(const GnArgs p) {
  __shared__ float sa[GN_CT], sb[GN_CT];
  const int tid = threadIdx.x, n = blockIdx.y, g = blockIdx.x;
  const int J = p.Cg >= GN_CT ? 1 : GN_CT / p.Cg, W = GN_CT / J;   // J threads per channel, W channels at a time
  float ta = 0.f, tb = 0.f;
  for (int c0 = 0; c0 < p.Cg; c0 += W) {
    const int j = tid / W, w = tid - j * W, c = g * p.Cg + c0 + w;
    const bool ok = j < J && c0 + w < p.Cg;
    float a = 0.f, b = 0.f;
    if (ok) {
#pragma unroll 4
      for (int k = j; k < p.chunks; k += J) {
        const float2 s = *reinterpret_cast<const float2*>(p.part + 2 * (((long long)n * p.chunks + k) * p.C + c));
        a += s.x;
        b += s.y;
      }
    }
    __syncthreads();
    sa[tid] = a;
    sb[tid] = b;
    gn_sum_rows<GN_CT>(sa, W, J, tid);
    gn_sum_rows<GN_CT>(sb, W, J, tid);
    if (ok && j == 0) {
      gn_channel_out(p, n, c, sa[w], sb[w]);
      const float ga = p.gamma ? p.gamma[c] : 1.f;
      ta += sa[w] * ga;
      tb += sb[w] * ga;
    }
  }
  __syncthreads();
  sa[tid] = ta;
  sb[tid] = tb;
  gn_sum_rows<GN_CT>(sa, 1, GN_CT, tid);
  gn_sum_rows<GN_CT>(sb, 1, GN_CT, tid);
  if (tid == 0) {
    const float inv = 1.f / ((float)p.P * (float)p.Cg);
    p.gsum[2 * ((long long)n * p.G + g)] = sa[0] * inv;
    p.gsum[2 * ((long long)n * p.G + g) + 1] = sb[0] * inv;
  }
}

// statistics of samples without positions: mean 0, variance 0
__global__ __launch_bounds__(256) void gn_empty_stats_kernel(const GnArgs p) {
  const int i = blockIdx.x * 256 + threadIdx.x;   // N G stays below 2^30: gn_check
  if (i < p.N * p.G) *reinterpret_cast<float2*>(p.stats + 2ll * i) = make_float2(0.f, 1.f / sqrtf(p.eps));
}

// The same in two launches where a thread of the merge above would add more than GN_LIST chunks one after the other, which few
// threads do if the groups are wide (one workgroup, a thread per channel, for a single group of 256 channels and more): tiles of
// eight channels with 32 lists of chunks each, then the groups.  Backward, one launch -> two: 1 x 25088 x 2048, 32 groups 129 ->
// 104 us, one group 1188 -> 108 us (lists of 392 and 1568); 4 x 25088 x 256, 4 groups 69 -> 62 (98); short lists: 8 x 25088 x 256,
// 32 groups 95 -> 98 (7), 1 x 6000 x 128, 8 groups 22 -> 32 (6).  A parameter's gradient, too, is then no row of up to 2048 terms.
constexpr int GN_LIST = 64;
__global__ __launch_bounds__(GN_CT) void gn_bwd_csum_kernel(const GnArgs p) {
  constexpr int W = 8, J = GN_CT / W;
  __shared__ float sa[GN_CT], sb[GN_CT];
  const int tid = threadIdx.x, n = blockIdx.y, w = tid % W, c = blockIdx.x * W + w;
  float a = 0.f, b = 0.f;
  if (c < p.C) {
#pragma unroll 8
    for (int k = tid / W; k < p.chunks; k += J) {
      const float2 s = *reinterpret_cast<const float2*>(p.part + 2 * (((long long)n * p.chunks + k) * p.C + c));
      a += s.x;
      b += s.y;
    }
  }
  sa[tid] = a;
  sb[tid] = b;
  gn_sum_rows<GN_CT>(sa, W, J, tid);
  gn_sum_rows<GN_CT>(sb, W, J, tid);
  if (tid < W && c < p.C) *reinterpret_cast<float2*>(p.csum + 2 * ((long long)n * p.C + c)) = make_float2(sa[w], sb[w]);
}
__global__ __launch_bounds__(GN_CT) void gn_bwd_gsum_kernel(const GnArgs p) {
  __shared__ float sa[GN_CT], sb[GN_CT];
  const int tid = threadIdx.x, n = blockIdx.y, g = blockIdx.x;
  float ta = 0.f, tb = 0.f;
  for (int i = tid; i < p.Cg; i += GN_CT) {
    const int c = g * p.Cg + i;
    const float2 s = *reinterpret_cast<const float2*>(p.csum + 2 * ((long long)n * p.C + c));
    if (p.N == 1) gn_channel_out(p, n, c, s.x, s.y);
    const float ga = p.gamma ? p.gamma[c] : 1.f;
    ta += s.x * ga;
    tb += s.y * ga;
  }
  sa[tid] = ta;
  sb[tid] = tb;
  gn_sum_rows<GN_CT>(sa, 1, GN_CT, tid);
  gn_sum_rows<GN_CT>(sb, 1, GN_CT, tid);
  if (tid == 0) {
    const float inv = 1.f / ((float)p.P * (float)p.Cg);
    *reinterpret_cast<float2*>(p.gsum + 2 * ((long long)n * p.G + g)) = make_float2(sa[0] * inv, sb[0] * inv);
  }
}

// dgamma / dbeta of channel c from the samples' sums, in sample order
__device__ __forceinline__ void gn_param_grad(const GnArgs& p, int c) {
  if (c >= p.C) return;
  float a = 0.f, b = 0.f;
  for (int n = 0; n < p.N; ++n) {
    const float2 s = *reinterpret_cast<const float2*>(p.csum + 2 * ((long long)n * p.C + c));
    a += s.x;
    b += s.y;
  }
  if (p.dbeta) p.dbeta[c] = a;
  if (p.dgamma) p.dgamma[c] = b;
}
__global__ __launch_bounds__(256) void gn_param_grad_kernel(const GnArgs p) { gn_param_grad(p, blockIdx.x * 256 + threadIdx.x); }

// dx of a chunk; the workgroups of sample 0 behind the last chunk form dgamma / dbeta
template <typename T, int V>
__global__ __launch_bounds__(GN_CT) void gn_bwd_apply_kernel(const GnArgs p) {
  using Raw = typename GnVec<T, V>::type;
  const int tid = threadIdx.x, n = blockIdx.y;
  if ((int)blockIdx.x >= p.chunks) {
    if (n == 0) gn_param_grad(p, ((int)blockIdx.x - p.chunks) * GN_CT + tid);
    return;
  }
  const int chunk = p.chunks - 1 - blockIdx.x;
  const int CV = p.C / V, RP = CV < GN_CT ? GN_CT / CV : 1;
  const int row0 = chunk * p.rows, row1 = min(row0 + p.rows, p.P);
  const int rr = CV < GN_CT ? tid / CV : 0;
  if (rr >= RP) return;
  for (int cv = CV < GN_CT ? tid - rr * CV : tid; cv < CV; cv += CV < GN_CT ? CV : GN_CT) {
    const long long base = (long long)n * p.P * p.C + (long long)cv * V;
    const T *x = static_cast<const T*>(p.x) + base, *dy = static_cast<const T*>(p.dy) + base;
    T* dx = static_cast<T*>(p.out) + base;
    float mean[V], rstd[V], ga[V], be[V], a[V], b[V];
    int grp[V];
    gn_groups<V>(cv * V, p.Cg, grp);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = cv * V + v;
      const long long at = 2 * ((long long)n * p.G + grp[v]);
      mean[v] = p.stats[at];
      rstd[v] = p.stats[at + 1];
      a[v] = p.gsum[at];
      b[v] = p.gsum[at + 1];
      ga[v] = p.gamma ? p.gamma[c] : 1.f;
      be[v] = p.beta ? p.beta[c] : 0.f;
    }
    for (int row = row0 + rr; row < row1; row += GN_UB * RP) {
      Raw rx[GN_UB], rd[GN_UB];
#pragma unroll
      for (int i = 0; i < GN_UB; ++i)
        if (row + i * RP < row1) {
          rx[i] = *reinterpret_cast<const Raw*>(x + (long long)(row + i * RP) * p.C);
          rd[i] = *reinterpret_cast<const Raw*>(dy + (long long)(row + i * RP) * p.C);
        }
#pragma unroll
      for (int i = 0; i < GN_UB; ++i)
        if (row + i * RP < row1) {
          float f[V], d[V], z[V];
          gn_unpack<T, V>(rx[i], f);
          gn_unpack<T, V>(rd[i], d);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            f[v] = (f[v] - mean[v]) * rstd[v];
            z[v] = f[v] * ga[v] + be[v];
          }
          gn_dact<V>(z, d, p.act);
#pragma unroll
          for (int v = 0; v < V; ++v) d[v] = (d[v] * ga[v] - a[v] - f[v] * b[v]) * rstd[v];
          gn_store<Raw>(dx + (long long)(row + i * RP) * p.C, gn_pack<T, V>(d), p.nt);
          gn_row_done();
        }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
struct GnPlan {
  int V;         // elements per access
  int slab, R;   // one pass: groups per workgroup (0: two passes), pieces per thread
  int rows, chunks;
};

static GnPlan gn_plan(int N, int P, int C, int G, int elem, bool backward) {
  GnPlan pl = {};
  pl.V = 16 / elem;
  while (C % pl.V) pl.V >>= 1;
  const int Cg = C / G;
  for (int k = 1; k <= G && !pl.slab; ++k) {   // the fewest whole groups that make rows of 64 bytes and whole accesses
    const long long sc = (long long)k * Cg;
    if (G % k || sc % pl.V) continue;
    if (sc * elem < 64 && k < G) continue;
    if (sc / pl.V > GN_BT) break;
    const int rp = GN_BT / (int)(sc / pl.V), pieces = ceil_div(P, rp);
    if (pieces > (backward ? GN_R_BWD : GN_R_FWD)) break;
    pl.slab = k;
    pl.R = pieces <= 4 ? 4 : pieces <= 8 ? 8 : pieces <= 16 ? 16 : 32;
  }
  // chunks of whole loads (GN_U rows of every thread): as many loads each as leave about 2048 workgroups, eight to a CU
  const int cv = C / pl.V, rp = cv < GN_CT ? GN_CT / cv : 1, unit = GN_U * rp;
  const int loads = ceil_div(ceil_div(P, unit), ceil_div(2048, N));
  pl.rows = loads * unit;
  pl.chunks = ceil_div(P, pl.rows);
  return pl;
}

static inline size_t gn_align(size_t n) { return (n + 255) & ~(size_t)255; }

// workspace: [csum][gsum][part]
static void gn_bytes(const GnPlan& pl, int N, int C, int G, bool backward, size_t* csum, size_t* gsum, size_t* part) {
  *csum = backward ? gn_align((size_t)N * C * 8) : 0;
  *gsum = backward && !pl.slab ? gn_align((size_t)N * G * 8) : 0;
  *part = pl.slab ? 0 : gn_align((size_t)N * pl.chunks * (backward ? C : G) * 8);
}

static int gn_check(int N, long long P, int C, int G, const char* what) {
  TRACE_REQUIRE(N >= 0 && P >= 0 && C > 0 && G > 0 && C % G == 0, "%s: %d channels in %d groups, %d samples", what, C, G, N);
  TRACE_REQUIRE(C <= GN_MAX_C, "%s: at most %d channels (got %d)", what, GN_MAX_C, C);
  TRACE_REQUIRE(P < (1ll << 30) && N <= 65535, "%s: sample too large (%lld positions) or too many samples (%d)", what, P, N);
  return 0;
}

template <typename T, int V> static void gn_run_slab(const GnArgs& a, const GnPlan& pl, bool backward, hipStream_t st) {
  const dim3 grid(a.G / pl.slab, a.N);
#define TRACE_GN_SLAB(RR)                                              \
  if (backward) gn_bwd_slab_kernel<T, V, RR><<<grid, GN_BT, 0, st>>>(a); \
  else gn_fwd_slab_kernel<T, V, RR><<<grid, GN_BT, 0, st>>>(a)
  if (pl.R == 4) { TRACE_GN_SLAB(4); }
  else if (pl.R == 8) { TRACE_GN_SLAB(8); }
  else if (pl.R == 16) { TRACE_GN_SLAB(16); }
  else { gn_fwd_slab_kernel<T, V, GN_R_FWD><<<grid, GN_BT, 0, st>>>(a); }
#undef TRACE_GN_SLAB
}

template <typename T, int V> static int gn_run(const GnArgs& a, const GnPlan& pl, bool backward, hipStream_t st) {
  if (pl.slab) {
    gn_run_slab<T, V>(a, pl, backward, st);
  } else {
    const int cv = a.C / V, rp = cv < GN_CT ? GN_CT / cv : 1;
    const dim3 grid(pl.chunks, a.N);
    const int lds_s = (2 * rp * a.C + rp) * 4;
    if (!backward) {
      TRACE_LDS_OPT_IN((gn_stats_kernel<T, V>), 2 * GN_MAX_C * 4 + 4096, "group_norm");
      gn_stats_kernel<T, V><<<grid, GN_CT, lds_s, st>>>(a);
      gn_merge_kernel<<<dim3(a.G, a.N), GN_CT, 0, st>>>(a);
      gn_apply_kernel<T, V><<<grid, GN_CT, 0, st>>>(a);
    } else {
      TRACE_LDS_OPT_IN((gn_bwd_sums_kernel<T, V>), 2 * GN_MAX_C * 4 + 4096, "group_norm backward");
      gn_bwd_sums_kernel<T, V><<<grid, GN_CT, lds_s, st>>>(a);
      if (pl.chunks > GN_LIST * (a.Cg >= GN_CT ? 1 : GN_CT / a.Cg)) {
        gn_bwd_csum_kernel<<<dim3(ceil_div(a.C, 8), a.N), GN_CT, 0, st>>>(a);
        gn_bwd_gsum_kernel<<<dim3(a.G, a.N), GN_CT, 0, st>>>(a);
      } else {
        gn_bwd_merge_kernel<<<dim3(a.G, a.N), GN_CT, 0, st>>>(a);
      }
      const int extra = a.N > 1 && (a.dgamma || a.dbeta) ? ceil_div(a.C, GN_CT) : 0;
      gn_bwd_apply_kernel<T, V><<<dim3(pl.chunks + extra, a.N), GN_CT, 0, st>>>(a);
    }
  }
  if (backward && pl.slab && a.N > 1 && (a.dgamma || a.dbeta)) gn_param_grad_kernel<<<ceil_div(a.C, 256), 256, 0, st>>>(a);
  return check_launch(backward ? "group_norm backward" : "group_norm");
}

template <typename T>
static int gn_call(bool backward, const T* x, const T* dy, int N, long long P, int C, int G, const float* gamma, const float* beta, float eps,
                   int act, T* out, float* stats, float* dgamma, float* dbeta, void* ws, size_t ws_bytes, void* stream) {
  const char* what = backward ? "group_norm backward" : "group_norm";
  if (int rc = gn_check(N, P, C, G, what)) return rc;
  TRACE_REQUIRE(act == 0 || act == TRACE_EPI_RELU || act == TRACE_EPI_LEAKY || act == TRACE_EPI_SILU, "%s: act takes one of RELU / LEAKY / SILU", what);
  TRACE_REQUIRE(((uintptr_t)x & 15) == 0 && ((uintptr_t)dy & 15) == 0 && ((uintptr_t)out & 15) == 0, "%s: maps must be 16-byte aligned", what);
  hipStream_t st = (hipStream_t)stream;
  GnArgs a = {};
  a.x = x;
  a.dy = dy;
  a.gamma = gamma;
  a.beta = beta;
  a.out = out;
  a.stats = stats;
  a.dgamma = dgamma;
  a.dbeta = dbeta;
  a.N = N;
  a.C = C;
  a.G = G;
  a.Cg = C / G;
  a.P = (int)P;
  a.act = act;
  a.eps = eps;
  if (N == 0 || P == 0) {   // no elements: the parameters' gradients are zero
    if (!backward && N > 0 && stats) gn_empty_stats_kernel<<<ceil_div((long long)N * G, 256), 256, 0, st>>>(a);
    a.N = 0;
    if (backward && (dgamma || dbeta)) gn_param_grad_kernel<<<ceil_div(C, 256), 256, 0, st>>>(a);
    return check_launch(what);
  }
  TRACE_REQUIRE(x && out && stats && (dy || !backward), "%s: null pointer", what);
  const GnPlan pl = gn_plan(N, (int)P, C, G, sizeof(T), backward);
  size_t csum, gsum, part;
  gn_bytes(pl, N, C, G, backward, &csum, &gsum, &part);
  TRACE_REQUIRE(ws_bytes >= csum + gsum + part && (ws || !(csum + gsum + part)), "%s: workspace of %zu bytes needed", what, csum + gsum + part);
  char* w = static_cast<char*>(ws);
  a.csum = reinterpret_cast<float*>(w);
  a.gsum = reinterpret_cast<float*>(w + csum);
  a.part = reinterpret_cast<float*>(w + csum + gsum);
  a.slab = pl.slab;
  if (pl.slab) {
    const int sw = pl.slab * a.Cg / pl.V, cvg = a.Cg % pl.V ? 0 : a.Cg / pl.V;
    a.pow2 = cvg && (sw & (sw - 1)) == 0 && (cvg & (cvg - 1)) == 0;
  }
  a.rows = pl.rows;
  a.chunks = pl.chunks;
  a.nt = (long long)N * P * C * sizeof(T) > GN_NT_BYTES;
  if constexpr (std::is_same<T, float>::value) {
    switch (pl.V) {
      case 4: return gn_run<T, 4>(a, pl, backward, st);
      case 2: return gn_run<T, 2>(a, pl, backward, st);
      default: return gn_run<T, 1>(a, pl, backward, st);
    }
  } else {
    switch (pl.V) {
      case 8: return gn_run<T, 8>(a, pl, backward, st);
      case 4: return gn_run<T, 4>(a, pl, backward, st);
      case 2: return gn_run<T, 2>(a, pl, backward, st);
      default: return gn_run<T, 1>(a, pl, backward, st);
    }
  }
}

}  // namespace trace

using namespace trace;

extern "C" size_t trace_group_norm_workspace_bytes(int N, long long P, int C, int G, int backward) {
  if (gn_check(N, P, C, G, "group_norm") || N == 0 || P == 0) return 0;
  size_t most = 0;
  for (int elem = 2; elem <= 4; elem += 2) {   // either element type
    size_t c, g, p;
    gn_bytes(gn_plan(N, (int)P, C, G, elem, backward != 0), N, C, G, backward != 0, &c, &g, &p);
    if (c + g + p > most) most = c + g + p;
  }
  return most;
}

extern "C" int trace_group_norm_act_bf16(const uint16_t* x, int N, long long P, int C, int G, const float* gamma,
                                         const float* beta, float eps, int act, uint16_t* y, float* stats, void* workspace,
                                         size_t workspace_bytes, trace_stream_t stream) {
  TRACE_REQUIRE(eps >= 0.f, "group_norm: eps must not be negative");
  return gn_call<uint16_t>(false, x, nullptr, N, P, C, G, gamma, beta, eps, act, y, stats, nullptr, nullptr, workspace, workspace_bytes, stream);
}
extern "C" int trace_group_norm_act_f32(const float* x, int N, long long P, int C, int G, const float* gamma, const float* beta,
                                        float eps, int act, float* y, float* stats, void* workspace, size_t workspace_bytes,
                                        trace_stream_t stream) {
  TRACE_REQUIRE(eps >= 0.f, "group_norm: eps must not be negative");
  return gn_call<float>(false, x, nullptr, N, P, C, G, gamma, beta, eps, act, y, stats, nullptr, nullptr, workspace, workspace_bytes, stream);
}
extern "C" int trace_group_norm_act_bwd_bf16(const uint16_t* x, const uint16_t* dy, int N, long long P, int C, int G,
                                             const float* gamma, const float* beta, const float* stats, int act, uint16_t* dx,
                                             float* dgamma, float* dbeta, void* workspace, size_t workspace_bytes,
                                             trace_stream_t stream) {
  return gn_call<uint16_t>(true, x, dy, N, P, C, G, gamma, beta, 0.f, act, dx, const_cast<float*>(stats), dgamma, dbeta,
                           workspace, workspace_bytes, stream);
}
extern "C" int trace_group_norm_act_bwd_f32(const float* x, const float* dy, int N, long long P, int C, int G,
                                            const float* gamma, const float* beta, const float* stats, int act, float* dx,
                                            float* dgamma, float* dbeta, void* workspace, size_t workspace_bytes,
                                            trace_stream_t stream) {
  return gn_call<float>(true, x, dy, N, P, C, G, gamma, beta, 0.f, act, dx, const_cast<float*>(stats), dgamma, dbeta, workspace,
                        workspace_bytes, stream);
}
