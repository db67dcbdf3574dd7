// Softmax attention with its backward pass for gfx950: bf16 operands, f32 scores, statistics and sums.
//
//   forward    s = scale q k^T over the keys a query sees, out = softmax(s) v, lse = log sum exp(s)
//   backward   P = exp(s - lse) (recomputed, never stored), delta_i = dout_i . out_i, dS = P (dout v^T - delta)
//              dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout
//
// Layout that all three kernels share.  Every product runs on v_mfma_f32_16x16x32_bf16, whose result has its column in
// the lane (lane & 15) and four consecutive rows 4 (lane >> 4) + r in the lane's registers.  The scores are formed with
// the axis that the NEXT product sums over as rows: S^T (keys x queries) in the forward and dq kernels, S (queries x
// keys) in the dk / dv kernel.  A lane then holds, for its own column, eight of the 32 summed rows of a pair of 16-row
// tiles - rows {4 g + r} and {16 + 4 g + r}, g = lane >> 4 - and these, rounded to bf16, ARE the B operand of the next
// product if its A operand lists the rows in the same order: no probability ever moves between lanes or through LDS.  The
// A operand is the staged tile read transposed (ds_read_b64_tr_b16 on rows 4 g .. 4 g + 3 and 16 + 4 g ..), so one copy of
// a tile in LDS serves both products it takes part in.  Softmax statistics belong to a column, so they live in the lane.
//
// Tiles of rows x head_dim go HBM / L2 -> LDS by 16-byte LDS-DMA, two stages deep; rows behind the sequence and columns
// behind head_dim read a zero page, so nothing behind a length is ever touched.
//
// What bounds them at full size is the matrix pipe together with the vector work between its products (an exponential, its
// scaling and its rounding per score): 2 x 4096 x 16 heads x 128 without a mask runs forward at 910 - 960 TFLOP/s, forward for a
// backward pass at 1050 - 1110 and backward at 1140 - 1200 TFLOP/s of the products it executes (calls back to back on two cards),
// where a library matmul of 8192^3 reaches 1330.  Of the cycles that its CUs are busy, the causal one of 4 key heads spends 48 % in
// the matrix pipe and 18 % in LDS reads (forward for a backward pass; dq 52 and 26 %, dk / dv 52 and 36 %), the forward pass of head
// size 256 (8 x 3136 x 784) 23 % and 25 %: neither bounds it, a workgroup of four waves alone on a CU, as half of them are, has gaps that
// nothing fills.  LDS bank conflicts: none.
// "a -> b" below are the two sides of a choice, on one card.  Choices that made the rate:
//   * every kernel is compiled for two waves per SIMD (256 registers): with more, hipcc keeps the sums in accumulation
//     registers and spends hundreds of moves per tile on them (dk / dv took twice as long), and a single spilled register
//     in the loop waits for the prefetch behind it (half as long again);
//   * 32 columns (queries, or keys) per wave where the sums fit, so a fragment from LDS feeds two products; at head_dim 256
//     and above 16 columns with the whole row in one wave beat 32 with the row shared by two, whose scores have to meet
//     in LDS (8 x 3136 x 784 x 256: 60 -> 42 us), and 32 columns with the whole row spill or leave one wave
//     per SIMD (74 - 99 us).  Only the sums of dq, dk / dv over 512 columns need the sharing;
//   * masks stand behind uniform branches, so tiles inside the sequence pay nothing for them.
#include "lds_dma.h"
#include <math.h>

namespace trace {

typedef __attribute__((ext_vector_type(8))) short at_s8;
typedef __attribute__((ext_vector_type(4))) short at_s4;
typedef __attribute__((ext_vector_type(4))) float at_f4;

__device__ __attribute__((aligned(256))) const uint4 g_at_zero[16] = {};

constexpr float AT_LOG2E = 1.4426950408889634f, AT_LN2 = 0.6931471805599453f;
constexpr int AT_CUS = 256;
constexpr int AT_MAX_SPLITS = 256;   // a thread each in attn_combine_kernel
constexpr int AT_MAX_ROWS = 0x7fffffff - 511;

struct AttnArgs {
  const uint16_t *q, *k, *v, *out, *rest, *dout;
  long long sq[3], sk[3], sv[3], sdo[3];   // elements between batches / rows / heads
  int B, Nq, Nk, H, Hk, D, causal;
  float scale;
  const int32_t *q_len, *kv_len;
  uint16_t *o, *o_rest, *dq, *dk, *dv;
  float* lse;     // written by the forward, read by the backward kernels
  float* ndelta;  // (B, H, Nq): -delta, written by the dq kernel for the dk / dv one
  float* part;    // partial results of the splits (null: one split)
  float2* part_ml;
  int pack;       // query heads whose rows share one row axis (1, or all heads of a key head)
  int units;      // heads / pack
  int tiles, splits;
};

// LDS image of a tile: rows of 2 D bytes in 16-byte chunks, chunk c of row r at position c ^ at_key(r).  The key makes both
// reads of a tile conflict-free over the 64 banks.  A fragment read (ds_read_b128) serves 16 lanes at a time: rows 0-3 and
// 12-15 of one chunk with rows 4-11 of its neighbour (chunk ^ 1), so the key leaves bit 0 alone; a transposed read
// (ds_read_b64_tr_b16) takes a 32-byte pair of chunks of 8 consecutive rows, whose keys differ in the bits above (rows of 64 /
// 128 bytes: 4 / 2 of them share a 256-byte line, only the others need different keys).
// Bits of a chunk index and of a row's offset do not overlap, so the address of any chunk is the lane's base ^ a constant.
template <int D> __device__ __forceinline__ int at_key(int r) {
  return D >= 128 ? (r & 7) << 1 : D == 64 ? ((r >> 1) & 3) << 1 : ((r >> 2) & 1) << 1;
}
template <int D> __device__ __forceinline__ int at_off(int r, int chunk) { return r * (2 * D) + ((chunk ^ at_key<D>(r)) << 4); }

template <bool NT> __device__ __forceinline__ void at_glds(const void* g, char* lds) {
  if constexpr (NT) glds16_nt(g, lds);
  else glds16(g, lds);
}

// One wave's share of the LDS-DMA of a ROWS x D tile (whole workgroup: NW waves).  Consecutive loads of a wave are STEP rows
// apart; where that is a multiple of eight rows the key repeats, and one lane offset serves them all.
template <int D, int ROWS, int NW> struct AtLoader {
  static constexpr int CPR = D / 8;
  static constexpr int INST = ROWS * CPR / 64, N = INST < NW ? 1 : INST / NW;   // loads of 1 KiB: in all, per wave
  static constexpr int STEP = 64 * NW / CPR, M = STEP % 8 == 0 ? 1 : N;
  static_assert(ROWS * CPR % 64 == 0 && (INST < NW || INST % NW == 0), "whole instructions per wave");
  uint32_t off[M];   // bytes from the tile's first row (rows x stride stay below 2^31: at_check)
  unsigned colok;    // bit j: this lane's chunk of load j lies inside head_dim
  __device__ __forceinline__ void init(long long row_stride, int d, int wave, int lane) {
    colok = 0;
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const int id = (j * NW + wave) * 64 + lane, row = id / CPR, c = (id % CPR) ^ at_key<D>(row);
      off[j] = (uint32_t)(row * row_stride * 2 + c * 16);
      if (c * 8 < d) colok |= 1u << j;
    }
  }
  // `rows` rows from `base` (uniform); further rows and the columns behind head_dim (`d` of D) read zeros
  template <bool NT = false>
  __device__ __forceinline__ void issue(char* lds, const uint16_t* base, long long row_stride, int rows, int d, int wave, int lane) const {
    if (INST < NW && wave >= INST) return;
    const char* b = reinterpret_cast<const char*>(base);
    const long long step = M == 1 ? STEP * row_stride * 2 : 0;
    if (rows >= ROWS && d == D) {
#pragma unroll
      for (int j = 0; j < N; ++j) at_glds<NT>(b + j * step + off[M == 1 ? 0 : j], lds + (j * NW + wave) * 1024);
      return;
    }
    const char* zero = reinterpret_cast<const char*>(g_at_zero);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int row = ((j * NW + wave) * 64 + lane) / CPR;
      const bool ok = ((colok >> (M == 1 ? 0 : j)) & 1u) && row < rows;
      at_glds<NT>(ok ? b + j * step + off[M == 1 ? 0 : j] : zero, lds + (j * NW + wave) * 1024);
    }
  }
};

// in a branch that every lane of the wave takes or none: keeps the compiler from running it always, with the results selected
__device__ __forceinline__ void at_keep_branch() { asm volatile(""); }

// B operand: a row of an operand as column of the product, 8 columns from 32 (kc0 + kc) + 8 g, straight from memory
template <int KC> __device__ __forceinline__ void at_load_cols(at_s8 (&f)[KC], const uint16_t* row, bool ok, int kc0, int d, int g) {
#pragma unroll
  for (int kc = 0; kc < KC; ++kc) {
    const int c = (kc0 + kc) * 32 + g * 8;
    f[kc] = (ok && c < d) ? *reinterpret_cast<const at_s8*>(row + c) : at_s8{0, 0, 0, 0, 0, 0, 0, 0};
  }
}

__device__ __forceinline__ at_s8 at_pack8(const at_f4& a, const at_f4& b) {
  union { at_s8 v; uint32_t u[4]; } o;
  o.u[0] = pack_bf16x2(a[0], a[1]);
  o.u[1] = pack_bf16x2(a[2], a[3]);
  o.u[2] = pack_bf16x2(b[0], b[1]);
  o.u[3] = pack_bf16x2(b[2], b[3]);
  return o.v;
}

// bf16 of what at_pack8 lost
__device__ __forceinline__ at_s8 at_lost8(const at_f4& a, const at_f4& b, const at_s8& packed) {
  union { at_s8 v; uint32_t u[4]; } w;
  w.v = packed;
  at_f4 x, y;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    x[r] = a[r] - __uint_as_float(r & 1 ? w.u[r >> 1] & 0xffff0000u : w.u[r >> 1] << 16);
    y[r] = b[r] - __uint_as_float(r & 1 ? w.u[2 + (r >> 1)] & 0xffff0000u : w.u[2 + (r >> 1)] << 16);
  }
  return at_pack8(x, y);
}

// Lane bases of the two kinds of reads inside a tile (bytes); the tile's own offset is added before a chunk is selected.
// rows: row lane & 15, chunk g;  selecting 32-column block kc: ^ kc << 6, rows 16 st ..: + st * 32 D
template <int D> __device__ __forceinline__ int at_row_base(int lane) { return at_off<D>(lane & 15, lane >> 4); }
// transposed: row 4 g + q, 8-byte half of the chunk pair; selecting columns 16 dt ..: ^ dt << 5, 16 rows further: + 32 D
template <int D> __device__ __forceinline__ int at_tr_base(int lane) {
  const int g = lane >> 4, q = (lane >> 2) & 3, pq = lane & 3;
  return at_off<D>(4 * g + q, pq >> 1) + (pq & 1) * 8;
}
__device__ __forceinline__ at_s8 at_row(const char* smem, int at) { return *reinterpret_cast<const at_s8*>(smem + at); }
// A operand of the summing product: rows {4 g .. 4 g + 3} and {16 + 4 g ..} from `at` on (k), 16 columns (m = lane & 15)
template <int D> __device__ __forceinline__ at_s8 at_tr(const char* smem, int at) {
  typedef __attribute__((address_space(3))) at_s4* lp;
  const at_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(smem + at));
  const at_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(smem + at + 32 * D));
  return at_s8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
}

__device__ __forceinline__ at_f4 at_mfma(const at_s8& a, const at_s8& b, const at_f4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Workgroups go to the 8 XCDs round-robin and each XCD has its own L2: XCD x gets the x-th contiguous eighth of the
// (head, split, tile) units, so the tiles that read one head's other operand share an L2.  `uneven`: under a causal mask a
// tile's work falls with its index (the caller counts from the longest); tile 0 of all heads and splits goes first then, so that
// short ones fill the end: 2 x 4096 x 16 heads x 128, forward 197 -> 176 us, backward 560 -> 448 us (4 key heads: 192 -> 159, 580 -> 470).
// `spread`: single row tiles share nothing; their splits go round all XCDs, or a long batch entry would keep one of them busy alone.
struct AtUnit {
  int tile, split, head;   // head: of all batches
};
__device__ __forceinline__ AtUnit at_unit(int lin, int tiles, int splits, int heads, bool uneven, bool spread = false) {
  const int x = lin & 7, hs = heads * splits;
  int t, h;
  if (!uneven && !spread) {
    const int total = tiles * hs, per = total >> 3, rem = total & 7, u = x * per + min(x, rem) + (lin >> 3);
    t = u % tiles;
    h = u / tiles;
  } else if ((hs & 7) == 0 && !spread) {   // neighbouring heads on one XCD
    const int hx = hs >> 3, i = lin >> 3;
    t = i / hx;
    h = x * hx + i % hx;
  } else {
    t = lin / hs;
    h = lin % hs;
  }
  return {t, h % splits, h / splits};
}
__device__ __forceinline__ int at_len(const int32_t* len, int b, int n) { return len ? min(max(len[b], 0), n) : n; }

__device__ __forceinline__ void at_store4(uint16_t* dst, float a, float b, float c, float d) {
  uint2 o;
  o.x = pack_bf16x2(a, b);
  o.y = pack_bf16x2(c, d);
  *reinterpret_cast<uint2*>(dst) = o;
}

// the result, and what its rounding lost
template <bool FINE> __device__ __forceinline__ void at_store_out(const AttnArgs& p, long long at, const at_f4& v) {
  uint2 o;
  o.x = pack_bf16x2(v[0], v[1]);
  o.y = pack_bf16x2(v[2], v[3]);
  *reinterpret_cast<uint2*>(p.o + at) = o;
  if constexpr (FINE)
    at_store4(p.o_rest + at, v[0] - bf16_to_f32((uint16_t)o.x), v[1] - bf16_to_f32((uint16_t)(o.x >> 16)),
              v[2] - bf16_to_f32((uint16_t)o.y), v[3] - bf16_to_f32((uint16_t)(o.y >> 16)));
}

// Fragments are read AT_AHEAD ahead of the products that take them: an LDS read takes longer than the NT products of one
// fragment, and left alone hipcc reads each one right in front of its use (one ahead -> four: 2 x 4096 x 16 heads x 128 forward
// 295 -> 285 us, backward 821 -> 802, 8 x 3136 x 784 x 256 46 -> 42; two or six ahead within 2 % of four).
constexpr int AT_AHEAD = 4;
__device__ __forceinline__ void at_order() { __builtin_amdgcn_sched_barrier(0); }

// s[st][nt] (16-row tiles of a staged tile x 16 columns) += rows . columns over the wave's KC 32-column blocks
template <int D, int ST, int NT, int KC>
__device__ __forceinline__ void at_score(const char* smem, int at, const at_s8 (&f)[NT][KC], at_f4 (&s)[ST][NT]) {
  constexpr int F = KC * ST, A = F < AT_AHEAD ? F : AT_AHEAD;
  at_s8 a[A];
#pragma unroll
  for (int i = 0; i < A; ++i) a[i] = at_row(smem, (at ^ ((i / ST) << 6)) + (i % ST) * 32 * D);
#pragma unroll
  for (int i = 0; i < F; ++i) {
    const int kc = i / ST, st = i % ST, j = i + A;
    const at_s8 x = a[i % A];
    if (j < F) a[i % A] = at_row(smem, (at ^ ((j / ST) << 6)) + (j % ST) * 32 * D);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[st][nt] = at_mfma(x, f[nt][kc], s[st][nt]);
    at_order();
  }
}

// Transposed fragments of a tile in the order of a summing product: column blocks of 16, KK row blocks of 32 each
template <int D, int DT, int KK> struct AtTrAhead {
  static constexpr int F = DT * KK, A = F < AT_AHEAD ? F : AT_AHEAD;
  at_s8 a[A];
  __device__ __forceinline__ static at_s8 load(const char* smem, int at, int i) { return at_tr<D>(smem, (at ^ ((i / KK) << 5)) + (i % KK) * 64 * D); }
  __device__ __forceinline__ void start(const char* smem, int at) {
#pragma unroll
    for (int i = 0; i < A; ++i) a[i] = load(smem, at, i);
    at_order();
  }
  // fragment i, whose place the one A behind it takes
  __device__ __forceinline__ at_s8 take(const char* smem, int at, int i) {
    const at_s8 x = a[i % A];
    if (i + A < F) a[i % A] = load(smem, at, i + A);
    return x;
  }
};

// DW waves of a row group hold partial scores over their share of head_dim: every one gets the sum, added in wave order
// (equal bits in all of them).  Each wave's scores pass through its own part of the exchange buffer; the caller has a barrier
// between the last reads of one exchange and the next.
template <int ST, int NT, int DW>
__device__ __forceinline__ void at_exchange(char* xbuf, int wave, int lane, at_f4 (&s)[ST][NT]) {
  constexpr int REG = ST * NT * 1024;
  char* mine = xbuf + wave * REG + lane * 16;
#pragma unroll
  for (int st = 0; st < ST; ++st)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) *reinterpret_cast<at_f4*>(mine + (st * NT + nt) * 1024) = s[st][nt];
  ring_barrier();
  const int wd = wave % DW;
  const char* group = xbuf + (wave - wd) * REG + lane * 16;
#pragma unroll
  for (int st = 0; st < ST; ++st)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      at_f4 t = *reinterpret_cast<const at_f4*>(group + (st * NT + nt) * 1024);
#pragma unroll
      for (int o = 1; o < DW; ++o) t += *reinterpret_cast<const at_f4*>(group + o * REG + (st * NT + nt) * 1024);
      s[st][nt] = t;
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Forward.  A row group of DW waves owns NT * 16 query rows of one (batch, head), each wave D / DW columns of head_dim; a
// workgroup is NW / DW groups.  With few query rows the rows of all heads that share a key head form one row axis (`pack`), so
// the keys are read once for them.  Key tiles of BN rows; `splits` workgroups share the keys of a row tile and leave (max, sum,
// unnormalised out) for attn_combine_kernel.
// The probabilities are rounded to bf16 for the product (2^-9 each on average, averaged over a row), which is as much as the
// result's own rounding.  FINE (a forward pass that a backward pass follows): a second product adds what that rounding lost, and
// what rounding the result loses is written as well.  delta = dout . out enters every dS = P (dout v^T - delta): with the
// plain out, half of the error of dq and dk came from it (relative 2.6 - 3.1e-3 against 2.3e-3).
// A tile's scores are formed right in front of its softmax: the two waves of a SIMD fill each other's gaps, and forming the next
// tile's scores beside the softmax, interleaved or not, was 0 - 10 % slower (8 x 3136 x 784 x 256: 42 -> 46 us).
// ---------------------------------------------------------------------------------------------------------------
template <int D, int NT, int NW, int DW, int BN, bool FINE>
__global__ __launch_bounds__(64 * NW, 2) void attn_fwd_kernel(const AttnArgs p) {
  constexpr int TR = NW / DW * NT * 16, KC = D / 32 / DW, DT = D / 16 / DW, ST = BN / 16;
  constexpr int TILE = BN * D * 2;
  constexpr bool SMALL = TR == 16;   // one row tile: its keys are read once, past the caches
  extern __shared__ __attribute__((aligned(16))) char smem[];   // two stages of [K tile][V tile], exchange buffer
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wd = wave % DW, wr = wave / DW;
  const AtUnit u = at_unit(blockIdx.x, p.tiles, p.splits, p.units * p.B, p.causal, SMALL);
  const int tile = p.causal ? p.tiles - 1 - u.tile : u.tile;
  const int unit = u.head % p.units, b = u.head / p.units;
  const int G = p.H / p.Hk, hk = unit * p.pack / G;
  const int qlen = at_len(p.q_len, b, p.Nq), kvlen = at_len(p.kv_len, b, p.Nk), diff = kvlen - qlen;
  const int nrows = p.pack * p.Nq;

  int row_i[NT], row_h[NT], lim[NT];   // query, head and number of keys seen, of this lane's columns
  at_s8 qf[NT][KC];
  int wmin = 0x7fffffff, wmax = 0;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = tile * TR + (wr * NT + nt) * 16 + (lane & 15);
    const int hh = p.pack > 1 ? r / p.Nq : 0;
    row_h[nt] = unit * p.pack + hh;
    row_i[nt] = r < nrows ? r - hh * p.Nq : -1;
    const bool ok = row_i[nt] >= 0 && row_i[nt] < qlen;
    lim[nt] = !ok ? 0 : p.causal ? min(max(row_i[nt] + diff + 1, 0), kvlen) : kvlen;
    if (lim[nt] > 0) wmin = min(wmin, lim[nt]);
    wmax = max(wmax, lim[nt]);
    at_load_cols<KC>(qf[nt], p.q + b * p.sq[0] + (ok ? row_i[nt] : 0) * p.sq[1] + (ok ? row_h[nt] : 0) * p.sq[2], ok, wd * KC, p.D, g);
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    wmin = min(wmin, __shfl_xor(wmin, o));
    wmax = max(wmax, __shfl_xor(wmax, o));
  }
  wmin = __builtin_amdgcn_readfirstlane(wmin);
  wmax = __builtin_amdgcn_readfirstlane(wmax);

  int kend = 0;   // keys that some row of the workgroup sees
  if (p.pack > 1) {
    kend = qlen > 0 ? kvlen : 0;
  } else {
    const int last = min((tile + 1) * TR, qlen) - 1;
    if (last >= tile * TR) kend = p.causal ? min(max(last + diff + 1, 0), kvlen) : kvlen;
  }
  // a split's share: of the keys in sight, or, for single row tiles, of the longest batch entry's keys, so that entries of
  // different lengths make shares of one size
  const int ntile = (kend + BN - 1) / BN, per = ((SMALL ? (p.Nk + BN - 1) / BN : ntile) + p.splits - 1) / p.splits;
  const int t0 = min(u.split * per, ntile), t1 = min(t0 + per, ntile);

  AtLoader<D, BN, NW> lk, lv;
  lk.init(p.sk[1], p.D, wave, lane);
  lv.init(p.sv[1], p.D, wave, lane);
  const uint16_t* kb = p.k + b * p.sk[0] + hk * p.sk[2];
  const uint16_t* vb = p.v + b * p.sv[0] + hk * p.sv[2];
  auto issue = [&](int t) {
    const int st = ((t - t0) & 1) * (2 * TILE), k0 = t * BN;
    lk.template issue<SMALL>(smem + st, kb + k0 * p.sk[1], p.sk[1], kend - k0, p.D, wave, lane);
    lv.template issue<SMALL>(smem + st + TILE, vb + k0 * p.sv[1], p.sv[1], kend - k0, p.D, wave, lane);
  };
  const int row_at = at_row_base<D>(lane) ^ (wd * KC << 6), tr_at = (at_tr_base<D>(lane) ^ (wd * DT << 5)) + TILE;

  const float c = p.scale * AT_LOG2E;
  at_f4 acc[DT][NT];
  float m[NT], l[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -INFINITY;
    l[nt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt][nt] = at_f4{0.f, 0.f, 0.f, 0.f};
  }
  if (t0 < t1) issue(t0);
  for (int t = t0; t < t1; ++t) {
    wait_vmcnt<0>();
    ring_barrier();   // tile t landed for every wave; every wave is done reading the other stage
    const int stage = ((t - t0) & 1) * (2 * TILE), key0 = t * BN;
    if (t + 1 < t1) issue(t + 1);
    if (DW == 1 && key0 >= wmax) continue;   // no row of this wave sees these keys
    at_f4 s[ST][NT];
#pragma unroll
    for (int st = 0; st < ST; ++st)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[st][nt] = at_f4{0.f, 0.f, 0.f, 0.f};
    at_score<D>(smem, row_at + stage, qf, s);
    if constexpr (DW > 1) at_exchange<ST, NT, DW>(smem + 4 * TILE, wave, lane, s);
    if (key0 + BN > wmin) {
      at_keep_branch();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int st = 0; st < ST; ++st)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key0 + st * 16 + 4 * g + r >= lim[nt]) s[st][nt][r] = -INFINITY;
    }
    AtTrAhead<D, DT, BN / 32> va;
    va.start(smem, tr_at + stage);
    at_s8 pf[BN / 32][NT], pl[BN / 32][NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mx = m[nt];
#pragma unroll
      for (int st = 0; st < ST; ++st)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[st][nt][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float base = mx == -INFINITY ? 0.f : mx * c;   // rows that saw nothing yet: exp2(-inf) = 0 below
      const float alpha = __builtin_amdgcn_exp2f(m[nt] * c - base);
      m[nt] = mx;
      float sum = 0.f;
#pragma unroll
      for (int st = 0; st < ST; ++st)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[st][nt][r] = __builtin_amdgcn_exp2f(s[st][nt][r] * c - base);
          sum += s[st][nt][r];
        }
      l[nt] = l[nt] * alpha + sum;
      if (__any(alpha != 1.f)) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt][nt] *= alpha;
      }
#pragma unroll
      for (int kk = 0; kk < BN / 32; ++kk) {   // the sum above is not rounded
        pf[kk][nt] = at_pack8(s[2 * kk][nt], s[2 * kk + 1][nt]);
        if constexpr (FINE) pl[kk][nt] = at_lost8(s[2 * kk][nt], s[2 * kk + 1][nt], pf[kk][nt]);
      }
    }
#pragma unroll
    for (int i = 0; i < DT * (BN / 32); ++i) {
      const int dt = i / (BN / 32), kk = i % (BN / 32);
      const at_s8 a = va.take(smem, tr_at + stage, i);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[dt][nt] = at_mfma(a, pf[kk][nt], acc[dt][nt]);
      if constexpr (FINE) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[dt][nt] = at_mfma(a, pl[kk][nt], acc[dt][nt]);
      }
      at_order();
    }
  }
  const bool split = p.splits > 1;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float sum = l[nt];
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (row_i[nt] < 0) continue;
    const bool any = lim[nt] > 0 && !(split && sum == 0.f);   // a split may hold none of the keys that the row sees; NaN counts
    const long long row = ((long long)b * p.H + row_h[nt]) * p.Nq + row_i[nt];
    if (split) {
      const long long rows = (long long)p.B * p.H * p.Nq, at = u.split * rows + row;
      if (g == 0 && wd == 0) p.part_ml[at] = any ? make_float2(m[nt] * c, sum) : make_float2(-INFINITY, 0.f);
      if (!any) continue;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const int d = 16 * (wd * DT + dt) + 4 * g;
        if (d < p.D) *reinterpret_cast<at_f4*>(p.part + at * p.D + d) = acc[dt][nt];
      }
      continue;
    }
    if (g == 0 && wd == 0 && p.lse) p.lse[row] = any ? (m[nt] * c + __builtin_amdgcn_logf(sum)) * AT_LN2 : -INFINITY;
    const float inv = any ? 1.f / sum : 0.f;
    const long long o = (((long long)b * p.Nq + row_i[nt]) * p.H + row_h[nt]) * p.D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int d = 16 * (wd * DT + dt) + 4 * g;
      if (d < p.D) at_store_out<FINE>(p, o + d, any ? acc[dt][nt] * inv : at_f4{0.f, 0.f, 0.f, 0.f});
    }
  }
}

// out / lse of a row from its splits' (max, sum, unnormalised out).  A workgroup per row: a thread per split (AT_MAX_SPLITS at
// most) turns the statistics into weights, then groups of D / 4 threads add strided lists of splits, and the first group adds the
// groups.
template <bool FINE> __global__ __launch_bounds__(256) void attn_combine_kernel(const AttnArgs p) {
  __shared__ float weight[AT_MAX_SPLITS], part[2][4];
  __shared__ at_f4 red[256];
  const int tid = threadIdx.x, wave = tid >> 6, dq = p.D >> 2, groups = min(256 / dq, p.splits);
  const long long rows = (long long)p.B * p.H * p.Nq, row = blockIdx.x;
  {
    const float2 ml = tid < p.splits ? p.part_ml[tid * rows + row] : make_float2(-INFINITY, 0.f);
    float mx = ml.x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    if ((tid & 63) == 0) part[0][wave] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(part[0][0], part[0][1]), fmaxf(part[0][2], part[0][3]));
    const float w = ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - mx);
    float sum = w * ml.y;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
    if ((tid & 63) == 0) part[1][wave] = sum;
    __syncthreads();
    sum = (part[1][0] + part[1][1]) + (part[1][2] + part[1][3]);
    weight[tid] = sum == 0.f ? 0.f : w / sum;
    if (tid == 0 && p.lse) p.lse[row] = sum == 0.f ? -INFINITY : (mx + __builtin_amdgcn_logf(sum)) * AT_LN2;
  }
  __syncthreads();
  const int grp = tid / dq, d = (tid - grp * dq) * 4;
  if (grp < groups) {
    at_f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = grp; s < p.splits; s += groups)
      if (weight[s] != 0.f) o += weight[s] * *reinterpret_cast<const at_f4*>(p.part + (s * rows + row) * p.D + d);   // else: never written
    red[tid] = o;
  }
  __syncthreads();
  if (grp == 0) {
    at_f4 o = red[tid];
    for (int k = 1; k < groups; ++k) o += red[k * dq + tid];
    const int i = (int)(row % p.Nq), h = (int)(row / p.Nq % p.H);
    const long long b = row / p.Nq / p.H;
    at_store_out<FINE>(p, ((b * p.Nq + i) * p.H + h) * p.D + d, o);
  }
}

// The same for at most AT_FEW splits: a thread per four columns of a row.  Thousands of rows come in few splits, and a workgroup
// each would cost them more than the sums.
constexpr int AT_FEW = 8;
template <bool FINE> __global__ __launch_bounds__(256) void attn_combine_few_kernel(const AttnArgs p) {
  const int dq = p.D >> 2, sub = threadIdx.x / dq, d = ((int)threadIdx.x - sub * dq) * 4;
  const int rows = p.B * p.H * p.Nq, row = blockIdx.x * (256 / dq) + sub;   // rows stay below 2^31: at_check
  if (sub >= 256 / dq || row >= rows) return;
  const float* src = p.part + (long long)row * p.D + d;
  const long long step = (long long)rows * p.D;
  float mx = -INFINITY, w[AT_FEW];
  float2 ml[AT_FEW];
#pragma unroll
  for (int s = 0; s < AT_FEW; ++s)
    if (s < p.splits) ml[s] = p.part_ml[(long long)s * rows + row];
#pragma unroll
  for (int s = 0; s < AT_FEW; ++s)
    if (s < p.splits) mx = fmaxf(mx, ml[s].x);
  float sum = 0.f;
#pragma unroll
  for (int s = 0; s < AT_FEW; ++s) {
    w[s] = s >= p.splits || ml[s].y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[s].x - mx);
    if (s < p.splits) sum += w[s] * ml[s].y;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  at_f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < AT_FEW; ++s)
    if (w[s] != 0.f) o += (w[s] * inv) * *reinterpret_cast<const at_f4*>(src + s * step);   // else: never written
  const int i = row % p.Nq, bh = row / p.Nq, h = bh % p.H, b = bh / p.H;
  at_store_out<FINE>(p, (((long long)b * p.Nq + i) * p.H + h) * p.D + d, o);
  if (d == 0 && p.lse) p.lse[row] = sum == 0.f ? -INFINITY : (mx + __builtin_amdgcn_logf(sum)) * AT_LN2;
}

// ---------------------------------------------------------------------------------------------------------------
// dq (and delta).  The same walk as the forward's over key tiles of 32, with two scoring products (q k^T and dout v^T); the
// second one starts from -delta instead of zero.  dS is rounded to bf16 for the product, as P is in the forward kernel.  dq and
// dk / dv each form P and dS for themselves: seven products instead of the five of one pass, whose dq (or dk, dv) would have to
// be added up by atomics in whatever order workgroups come.  2 x 4096 x 16 / 4 heads x 128, causal (kernel times): 201 us, dk / dv 267 us
// and 23 us for joining its splits.
// The rows of dS sum to zero, so dq only has what the keys differ by, but the rounding of dS goes with all of a key: with few
// columns the weighted mean of the keys is a good part of them (|k|^2 of D + 4 against D + 1 for unit normal q, k), and dq is
// less exact than its own rounding explains.  Up to 32 columns a second product therefore adds what that rounding lost
// (relative error at 8 columns 2.56e-3 -> 1.65e-3, at 16 2.48e-3 -> 1.67e-3; 4 x 2048 x 16 heads x 32: backward 155 -> 178 us).
// ---------------------------------------------------------------------------------------------------------------
template <int D, int NT, int NW, int DW>
__global__ __launch_bounds__(64 * NW, 2) void attn_bwd_q_kernel(const AttnArgs p) {
  constexpr int BN = 32, TR = NW / DW * NT * 16, KC = D / 32 / DW, DT = D / 16 / DW;
  constexpr int TILE = BN * D * 2;
  constexpr bool FINE = D <= 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wd = wave % DW, wr = wave / DW;
  char* xbuf = smem + 4 * TILE;
  const AtUnit u = at_unit(blockIdx.x, p.tiles, p.splits, p.H * p.B, p.causal);
  const int tile = p.causal ? p.tiles - 1 - u.tile : u.tile, h = u.head % p.H, b = u.head / p.H;
  const int hk = h / (p.H / p.Hk);
  const int qlen = at_len(p.q_len, b, p.Nq), kvlen = at_len(p.kv_len, b, p.Nk), diff = kvlen - qlen;

  int row_i[NT], lim[NT];
  float lse2[NT], ndelta[NT];
  at_s8 qf[NT][KC], df[NT][KC];
  int wmin = 0x7fffffff, wmax = 0;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int i = tile * TR + (wr * NT + nt) * 16 + (lane & 15);
    row_i[nt] = i;
    const bool ok = i < qlen;
    lim[nt] = !ok ? 0 : p.causal ? min(max(i + diff + 1, 0), kvlen) : kvlen;
    if (lim[nt] > 0) wmin = min(wmin, lim[nt]);
    wmax = max(wmax, lim[nt]);
    const int ii = ok ? i : 0;
    at_load_cols<KC>(qf[nt], p.q + b * p.sq[0] + ii * p.sq[1] + h * p.sq[2], ok, wd * KC, p.D, g);
    at_load_cols<KC>(df[nt], p.dout + b * p.sdo[0] + ii * p.sdo[1] + h * p.sdo[2], ok, wd * KC, p.D, g);
    const long long orow = (((long long)b * p.Nq + ii) * p.H + h) * p.D;
    float sum = 0.f;
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      const int cc = (wd * KC + kc) * 32 + g * 8;
      if (ok && cc < p.D) {
        const at_s8 ov = *reinterpret_cast<const at_s8*>(p.out + orow + cc), rv = *reinterpret_cast<const at_s8*>(p.rest + orow + cc);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          sum += (bf16_to_f32((uint16_t)ov[e]) + bf16_to_f32((uint16_t)rv[e])) * bf16_to_f32((uint16_t)df[nt][kc][e]);
      }
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    ndelta[nt] = -sum;
    lse2[nt] = ok ? p.lse[((long long)b * p.H + h) * p.Nq + ii] * AT_LOG2E : 0.f;
  }
  if constexpr (DW > 1) {   // the waves' shares of head_dim
    float* xs = reinterpret_cast<float*>(xbuf);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) xs[(wave * NT + nt) * 64 + lane] = ndelta[nt];
    ring_barrier();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float sum = 0.f;
#pragma unroll
      for (int o = 0; o < DW; ++o) sum += xs[((wave - wd + o) * NT + nt) * 64 + lane];
      ndelta[nt] = sum;
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
    if (row_i[nt] < qlen && g == 0 && wd == 0 && u.split == 0) p.ndelta[((long long)b * p.H + h) * p.Nq + row_i[nt]] = ndelta[nt];
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    wmin = min(wmin, __shfl_xor(wmin, o));
    wmax = max(wmax, __shfl_xor(wmax, o));
  }
  wmin = __builtin_amdgcn_readfirstlane(wmin);
  wmax = __builtin_amdgcn_readfirstlane(wmax);

  int kend = 0;
  const int last = min((tile + 1) * TR, qlen) - 1;
  if (last >= tile * TR) kend = p.causal ? min(max(last + diff + 1, 0), kvlen) : kvlen;
  const int ntile = (kend + BN - 1) / BN, per = (ntile + p.splits - 1) / p.splits;
  const int t0 = min(u.split * per, ntile), t1 = min(t0 + per, ntile);

  AtLoader<D, BN, NW> lk, lv;
  lk.init(p.sk[1], p.D, wave, lane);
  lv.init(p.sv[1], p.D, wave, lane);
  const uint16_t* kb = p.k + b * p.sk[0] + hk * p.sk[2];
  const uint16_t* vb = p.v + b * p.sv[0] + hk * p.sv[2];
  auto issue = [&](int t) {
    const int st = ((t - t0) & 1) * (2 * TILE), k0 = t * BN;
    lk.issue(smem + st, kb + k0 * p.sk[1], p.sk[1], kend - k0, p.D, wave, lane);
    lv.issue(smem + st + TILE, vb + k0 * p.sv[1], p.sv[1], kend - k0, p.D, wave, lane);
  };
  const int row_at = at_row_base<D>(lane) ^ (wd * KC << 6), tr_at = at_tr_base<D>(lane) ^ (wd * DT << 5);
  const float c = p.scale * AT_LOG2E;
  at_f4 acc[DT][NT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[dt][nt] = at_f4{0.f, 0.f, 0.f, 0.f};
  if (t0 < t1) issue(t0);
  for (int t = t0; t < t1; ++t) {
    wait_vmcnt<0>();
    ring_barrier();
    const int stage = ((t - t0) & 1) * (2 * TILE), key0 = t * BN;
    if (t + 1 < t1) issue(t + 1);
    if (DW == 1 && key0 >= wmax) continue;
    at_f4 s[2][NT], dp[2][NT];
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float d0 = DW == 1 || wd == 0 ? ndelta[nt] : 0.f;
        s[st][nt] = at_f4{0.f, 0.f, 0.f, 0.f};
        dp[st][nt] = at_f4{d0, d0, d0, d0};
      }
    at_score<D>(smem, row_at + stage, qf, s);
    at_score<D>(smem, row_at + stage + TILE, df, dp);
    if constexpr (DW > 1) {
      at_exchange<2, NT, DW>(xbuf, wave, lane, s);
      ring_barrier();
      at_exchange<2, NT, DW>(xbuf, wave, lane, dp);
    }
    AtTrAhead<D, DT, 1> ka;
    ka.start(smem, tr_at + stage);
    const bool mask = key0 + BN > wmin;
    at_s8 ds[NT], dl[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[st][nt][r] = __builtin_amdgcn_exp2f(s[st][nt][r] * c - lse2[nt]);
    }
    if (mask) {
      at_keep_branch();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key0 + st * 16 + 4 * g + r >= lim[nt]) s[st][nt][r] = 0.f;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const at_f4 lo = s[0][nt] * dp[0][nt], hi = s[1][nt] * dp[1][nt];
      ds[nt] = at_pack8(lo, hi);
      if constexpr (FINE) dl[nt] = at_lost8(lo, hi, ds[nt]);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const at_s8 a = ka.take(smem, tr_at + stage, dt);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[dt][nt] = at_mfma(a, ds[nt], acc[dt][nt]);
      if constexpr (FINE) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[dt][nt] = at_mfma(a, dl[nt], acc[dt][nt]);
      }
      at_order();
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (row_i[nt] >= p.Nq) continue;
    const bool any = lim[nt] > 0;
    const long long at = (((long long)b * p.Nq + row_i[nt]) * p.H + h) * p.D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int d = 16 * (wd * DT + dt) + 4 * g;
      if (d >= p.D) continue;
      const at_f4 a = any ? acc[dt][nt] : at_f4{0.f, 0.f, 0.f, 0.f};
      if (p.splits > 1)
        *reinterpret_cast<at_f4*>(p.part + u.split * ((long long)p.B * p.Nq * p.H * p.D) + at + d) = a;
      else
        at_store4(p.dq + at + d, a[0] * p.scale, a[1] * p.scale, a[2] * p.scale, a[3] * p.scale);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// dk and dv.  A workgroup owns NW / DW * NT * 16 keys of one (batch, key head) - in registers as B operands - and walks the
// 32-row tiles of q and dout of every query head that reads it, so the gradients of shared heads are summed in a fixed order.
// P and dS are rounded to bf16 for their products, at every head size: each is as much as the result's own rounding, so that dk and
// dv are off by sqrt(2) of that (relative 2.34e-3, 1.66e-3 for the correctly rounded result; dq above 32 columns likewise).  What the
// rounding loses would take two products more, nine for seven of the backward pass.
// ---------------------------------------------------------------------------------------------------------------
template <int D, int NT, int NW, int DW>
__global__ __launch_bounds__(64 * NW, 2) void attn_bwd_kv_kernel(const AttnArgs p) {
  constexpr int BQ = 32, TK = NW / DW * NT * 16, KC = D / 32 / DW, DT = D / 16 / DW;
  constexpr int TILE = BQ * D * 2;
  constexpr bool VL = DW == 1;   // the values as a tile in LDS instead of registers, which the sums need
  extern __shared__ __attribute__((aligned(16))) char smem[];   // two stages of [q][dout], [v], two of [32 lse, 32 -delta], exchange
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wd = wave % DW, wr = wave / DW;
  constexpr int V_AT = 4 * TILE;
  char* stats = smem + V_AT + (VL ? TK * D * 2 : 0);
  char* xbuf = stats + 512;
  const AtUnit u = at_unit(blockIdx.x, p.tiles, p.splits, p.Hk * p.B, p.causal);
  const int tile = u.tile, hk = u.head % p.Hk, b = u.head / p.Hk;   // under a causal mask the first keys have the most queries
  const int G = p.H / p.Hk;
  const int qlen = at_len(p.q_len, b, p.Nq), kvlen = at_len(p.kv_len, b, p.Nk), diff = kvlen - qlen;
  const int key_first = tile * TK, wkey = key_first + wr * NT * 16;

  int key[NT];
  at_s8 kf[NT][KC], vf[VL ? 1 : NT][KC];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    key[nt] = wkey + nt * 16 + (lane & 15);
    const bool ok = key[nt] < kvlen;
    const int kk = ok ? key[nt] : 0;
    at_load_cols<KC>(kf[nt], p.k + b * p.sk[0] + kk * p.sk[1] + hk * p.sk[2], ok, wd * KC, p.D, g);
    if constexpr (!VL) at_load_cols<KC>(vf[nt], p.v + b * p.sv[0] + kk * p.sv[1] + hk * p.sv[2], ok, wd * KC, p.D, g);
  }
  at_f4 ak[DT][NT], av[DT][NT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) ak[dt][nt] = av[dt][nt] = at_f4{0.f, 0.f, 0.f, 0.f};

  // query tiles qt0 .. nq - 1 of each of the G heads, as one list of which this split takes a part
  const int nq = key_first < kvlen ? (qlen + BQ - 1) / BQ : 0;
  const int qt0 = p.causal ? min(max(key_first - diff, 0) / BQ, nq) : 0;
  const int per_head = nq - qt0, n_it = per_head * G, per = (n_it + p.splits - 1) / p.splits;
  const int it0 = min(u.split * per, n_it), it1 = min(it0 + per, n_it);

  AtLoader<D, BQ, NW> lq, ld;
  lq.init(p.sq[1], p.D, wave, lane);
  ld.init(p.sdo[1], p.D, wave, lane);
  const uint16_t* qb = p.q + b * p.sq[0] + (long long)hk * G * p.sq[2];
  const uint16_t* db = p.dout + b * p.sdo[0] + (long long)hk * G * p.sdo[2];
  const float* stat = (lane < 32 ? p.lse : p.ndelta) + ((long long)b * p.H + (long long)hk * G) * p.Nq;

  int head = 0, qt = 0;          // of the tile issued last
  auto issue = [&](int it) {
    const int par = (it - it0) & 1, q0 = qt * BQ;
    lq.issue(smem + par * (2 * TILE), qb + head * p.sq[2] + q0 * p.sq[1], p.sq[1], qlen - q0, p.D, wave, lane);
    ld.issue(smem + par * (2 * TILE) + TILE, db + head * p.sdo[2] + q0 * p.sdo[1], p.sdo[1], qlen - q0, p.D, wave, lane);
    if (wave == 0) {
      const int i = q0 + (lane & 31);
      const float* src = i < qlen ? stat + (long long)head * p.Nq + i : reinterpret_cast<const float*>(g_at_zero);
      __builtin_amdgcn_global_load_lds((gptr_t)src, (lptr_t)(stats + par * 256), 4, 0, 0);
    }
  };
  const int row_at = at_row_base<D>(lane) ^ (wd * KC << 6), tr_at = at_tr_base<D>(lane) ^ (wd * DT << 5);
  const float c = p.scale * AT_LOG2E;
  if (it0 < it1) {
    if constexpr (VL) {
      AtLoader<D, TK, NW> lv;
      lv.init(p.sv[1], p.D, wave, lane);
      lv.issue(smem + V_AT, p.v + b * p.sv[0] + hk * p.sv[2] + key_first * p.sv[1], p.sv[1], kvlen - key_first, p.D, wave, lane);
    }
    head = it0 / per_head;
    qt = qt0 + it0 - head * per_head;
    issue(it0);
  }
  for (int it = it0; it < it1; ++it) {
    wait_vmcnt<0>();
    ring_barrier();
    const int par = (it - it0) & 1, stage = par * (2 * TILE), q0 = qt * BQ;
    if (++qt == nq) {
      qt = qt0;
      ++head;
    }
    if (it + 1 < it1) issue(it + 1);
    if (DW == 1 && p.causal && wkey > q0 + BQ - 1 + diff) continue;   // no key of this wave is seen
    at_f4 s[2][NT], dp[2][NT];
    const float* sp = reinterpret_cast<const float*>(stats + par * 256) + 4 * g;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const at_f4 nd = *reinterpret_cast<const at_f4*>(sp + 32 + st * 16);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        s[st][nt] = at_f4{0.f, 0.f, 0.f, 0.f};
        dp[st][nt] = DW == 1 || wd == 0 ? nd : at_f4{0.f, 0.f, 0.f, 0.f};
      }
    }
    at_score<D>(smem, row_at + stage, kf, s);
    if constexpr (VL) {
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) {
        at_s8 bv[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) bv[nt] = at_row(smem, V_AT + (row_at ^ (kc << 6)) + (wr * NT + nt) * 32 * D);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const at_s8 a = at_row(smem, ((row_at + stage + TILE) ^ (kc << 6)) + st * 32 * D);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) dp[st][nt] = at_mfma(a, bv[nt], dp[st][nt]);
        }
      }
    } else {
      at_score<D>(smem, row_at + stage + TILE, vf, dp);
    }
    if constexpr (DW > 1) {
      at_exchange<2, NT, DW>(xbuf, wave, lane, s);
      ring_barrier();
      at_exchange<2, NT, DW>(xbuf, wave, lane, dp);
    }
    at_f4 lse2[2];
#pragma unroll
    for (int st = 0; st < 2; ++st) lse2[st] = *reinterpret_cast<const at_f4*>(sp + st * 16) * AT_LOG2E;
    const bool mask = q0 + BQ > qlen || wkey + NT * 16 > kvlen || (p.causal && wkey + NT * 16 - 1 > q0 + diff);
    at_s8 pf[NT], ds[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[st][nt][r] = __builtin_amdgcn_exp2f(s[st][nt][r] * c - lse2[st][r]);
    }
    if (mask) {
      at_keep_branch();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // queries from `first` on see this key
        const int first = key[nt] >= kvlen ? 0x7fffffff : p.causal ? key[nt] - diff : 0;
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = q0 + st * 16 + 4 * g + r;
            if (i >= qlen || i < first) s[st][nt][r] = 0.f;
          }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      pf[nt] = at_pack8(s[0][nt], s[1][nt]);
      ds[nt] = at_pack8(s[0][nt] * dp[0][nt], s[1][nt] * dp[1][nt]);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const at_s8 ad = at_tr<D>(smem, (tr_at + stage + TILE) ^ (dt << 5)), aq = at_tr<D>(smem, (tr_at + stage) ^ (dt << 5));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        av[dt][nt] = at_mfma(ad, pf[nt], av[dt][nt]);
        ak[dt][nt] = at_mfma(aq, ds[nt], ak[dt][nt]);
      }
    }
  }
  const long long n_all = (long long)p.B * p.Nk * p.Hk * p.D;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (key[nt] >= p.Nk) continue;
    const long long at = (((long long)b * p.Nk + key[nt]) * p.Hk + hk) * p.D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int d = 16 * (wd * DT + dt) + 4 * g;
      if (d >= p.D) continue;
      const at_f4 a = ak[dt][nt], w = av[dt][nt];
      if (p.splits > 1) {
        float* dst = p.part + (long long)u.split * 2 * n_all + at + d;
        *reinterpret_cast<at_f4*>(dst) = a;
        *reinterpret_cast<at_f4*>(dst + n_all) = w;
      } else {
        at_store4(p.dk + at + d, a[0] * p.scale, a[1] * p.scale, a[2] * p.scale, a[3] * p.scale);
        at_store4(p.dv + at + d, w[0], w[1], w[2], w[3]);
      }
    }
  }
}

// dst = bf16(mul * sum over splits), in split order; four elements per thread, n % 8 == 0.  The first n of a split's part go
// to dst0 with mul0, the n behind them (blockIdx.y = 1) to dst1 with mul1.
__global__ __launch_bounds__(256) void attn_reduce_kernel(const float* __restrict__ part, long long split_stride, int splits,
                                                          long long n, float mul0, uint16_t* __restrict__ dst0, float mul1,
                                                          uint16_t* __restrict__ dst1) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const float* src = part + (blockIdx.y ? n : 0) + i;
  at_f4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) a += *reinterpret_cast<const at_f4*>(src + s * split_stride);
  const float mul = blockIdx.y ? mul1 : mul0;
  at_store4((blockIdx.y ? dst1 : dst0) + i, a[0] * mul, a[1] * mul, a[2] * mul, a[3] * mul);
}

// ---------------------------------------------------------------------------------------------------------------
// Host: one rule for a call's tiles and splits, used for the workspace size and for the launch.
// ---------------------------------------------------------------------------------------------------------------
struct AttnPlan {
  int D;                                   // head_dim rounded up to a built size
  int pack, units, tile_rows, tiles, splits;   // forward
  int q_rows, q_tiles, q_splits;           // dq
  int k_rows, k_tiles, k_splits;           // dk / dv
};

static inline size_t at_align(size_t n) { return (n + 255) & ~(size_t)255; }

// Splits so that about `per_cu` workgroups per CU exist, each with at least `min_iters` iterations of its loop (32 rows): the
// partial results cost a pass over f32 copies of the output and a launch.  4 x 500 x 4 heads x 128: forward 17.5 us with at least
// 8, 20.6 with 4; backward 43 with 4, 8 % more with 8, 24 % more with 2.  At most `per_cu` each, or a few of them would run
// alone at the end (1 x 3136 x 784 x 512, backward: 13 key tiles in 20 shares 122 us, in 17 78 us), and no empty shares.
static int at_splits(long long groups, int iters, int min_iters, int per_cu) {
  if (groups <= 0 || iters <= 0) return 1;
  long long s = per_cu * AT_CUS / groups;
  const long long most = iters / min_iters;
  if (s > most) s = most;
  if (s > AT_MAX_SPLITS) s = AT_MAX_SPLITS;
  if (s <= 1) return 1;
  const int per = ceil_div(iters, s);
  return ceil_div(iters, per);
}

// Whether half a tile of rows serves a call better than a whole one: where whole tiles would have to be split to fill the card and
// their shares stay short (`most` iterations), the joining of the shares costs more than half tiles, whose fragments from LDS feed
// half the products.  Forward / backward, whole -> half: 128 x 8 heads causal, 8 x 1024: 54 -> 34 us / 152 -> 90, 16 x 512: 45 ->
// 23 / 130 -> 63; 4 x 1024: 39 -> 33 / 117 -> 80; 8 x 500 x 4 heads x 256: backward 80 -> 61.  Longer
// shares (1 x 4096 x 8 heads x 128: 64 iterations): 103 -> 112 / 251 -> 296; full grids (8 x 1024): 46 -> 54 / 129 -> 157.
static bool at_short(long long groups, int iters, int min_iters, int per_cu, int most) {
  return 2 * groups <= per_cu * AT_CUS && ceil_div(iters, at_splits(groups, iters, min_iters, per_cu)) <= most;
}

static AttnPlan at_plan(const trace_attention_desc* d) {
  AttnPlan pl;
  const int hd = d->head_dim;
  pl.D = hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : hd <= 256 ? 256 : 512;
  const int G = d->heads / d->kv_heads, uneven = d->causal ? 2 : 1;   // uneven work: more, shorter workgroups
  const long long qh = (long long)d->heads * d->batch, kh = (long long)d->kv_heads * d->batch;
  const int k_iters = ceil_div(d->k_rows, 32), q_iters = ceil_div(d->q_rows, 32) * G;
  const auto q_groups = [&](int rows) { return ceil_div(d->q_rows, rows) * qh; };
  // head_dim 512: 32 rows with four waves where 64-row tiles with their splits reach half of the CUs at most (too few keys to split):
  // 8 x 784 rows over 196 keys, forward for a backward pass 28 -> 21 us, dq 29 -> 23; where they can be split, whole tiles are
  // ahead (2 x 2048 x 2048 50 against 65 us)
  const auto half512 = [&](int min_iters) {
    return q_groups(64) * at_splits(q_groups(64), k_iters, min_iters, uneven) <= AT_CUS / 2;
  };

  // few query rows: all heads of a key head on one row axis, 16 rows per workgroup (its one row group streams the keys)
  const bool small = (long long)d->q_rows * G <= 16;
  pl.pack = small ? G : 1;
  pl.units = d->heads / pl.pack;
  const int held = (small ? (pl.D <= 128 ? 5 : pl.D == 256 ? 2 : 1) : (pl.D <= 256 ? 2 : 1) * uneven);   // workgroups that a CU holds, by their LDS
  if (small) pl.tile_rows = 16;
  else if (pl.D <= 128) pl.tile_rows = at_short(q_groups(128), k_iters, 8, held, 16) ? 64 : 128;
  else if (pl.D == 256) pl.tile_rows = 64;
  // one workgroup of eight waves per CU: 128 rows with each wave on a whole row where that fills the card (4 x 4 x 2048 rows: 111
  // against 133 us), else 64 rows with two waves on each (8 x 784 rows over 196 keys: 22 against 28 us), or half of that
  else pl.tile_rows = q_groups(128) >= AT_CUS ? 128 : half512(8) ? 32 : 64;
  pl.tiles = ceil_div((long long)pl.pack * d->q_rows, pl.tile_rows);
  pl.splits = at_splits((long long)pl.tiles * pl.units * d->batch, k_iters, small ? 4 : 8, held);

  const int per_cu = (pl.D <= 128 ? 2 : 1) * uneven;   // workgroups that a CU holds, by their LDS
  pl.q_rows = pl.D <= 256 ? (at_short(q_groups(128), k_iters, 4, per_cu, 16) ? 64 : 128) : half512(4) ? 32 : 64;
  pl.q_tiles = ceil_div(d->q_rows, pl.q_rows);
  pl.q_splits = at_splits(pl.q_tiles * qh, k_iters, 4, per_cu);
  // head_dim 512: 64 keys with two waves on each row or 32 with four (8 x 784 rows over 196 keys with the reduction of the splits 35 ->
  // 31 us; 4 x 3136 over 784, whose shares are long, backward 155 against 181)
  pl.k_rows = pl.D <= 256 ? 128 : 64;
  if (at_short(ceil_div(d->k_rows, pl.k_rows) * kh, q_iters, 4, per_cu, pl.D <= 256 ? 16 : 8)) pl.k_rows /= 2;
  pl.k_tiles = ceil_div(d->k_rows, pl.k_rows);
  pl.k_splits = at_splits(pl.k_tiles * kh, q_iters, 4, per_cu);
  return pl;
}

static int at_check(const trace_attention_desc* d, const char* what) {
  TRACE_REQUIRE(d, "%s: null descriptor", what);
  TRACE_REQUIRE(d->batch >= 0 && d->q_rows >= 0 && d->k_rows >= 0 && d->heads > 0 && d->kv_heads > 0, "%s: bad sizes", what);
  TRACE_REQUIRE(d->heads % d->kv_heads == 0, "%s: heads (%d) must be a multiple of kv_heads (%d)", what, d->heads, d->kv_heads);
  TRACE_REQUIRE(d->head_dim >= 8 && d->head_dim <= 512 && d->head_dim % 8 == 0, "%s: head_dim %d (8 .. 512, multiple of 8)",
                what, d->head_dim);
  TRACE_REQUIRE(d->scale > 0.f && d->scale <= 3.0e38f, "%s: scale must be positive and finite", what);
  // rows are counted in 32 bits to the end of the last tile (at most 128 rows) and one tile further
  TRACE_REQUIRE(d->q_rows <= AT_MAX_ROWS && d->k_rows <= AT_MAX_ROWS, "%s: too many rows (at most 2^31 - 512)", what);
  // tiles x heads x batch are grid indices, of query heads over query rows (rows x heads of a packed call are row indices too) and
  // of key heads over key rows
  const long long qr = (long long)d->batch * d->heads * (d->q_rows + 2), kr = (long long)d->batch * d->kv_heads * (d->k_rows + 2);
  TRACE_REQUIRE(qr < (1ll << 31) - 1 && kr < (1ll << 31) - 1, "%s: too many rows (batch x heads x rows of queries or keys)", what);
  for (int i = 0; i < 3; ++i)
    TRACE_REQUIRE(((d->stride_q[i] | d->stride_k[i] | d->stride_v[i]) & 7) == 0, "%s: strides must be multiples of 8 elements", what);
  for (long long st : {d->stride_q[1], d->stride_k[1], d->stride_v[1], d->stride_do[1]})   // 64-row tiles: 32-bit byte offsets
    TRACE_REQUIRE(st >= 0 && st < (1ll << 24), "%s: row strides must be below 2^24 elements", what);
  return 0;
}

static AttnArgs at_args(const trace_attention_desc* d, const uint16_t* q, const uint16_t* k, const uint16_t* v) {
  AttnArgs a = {};
  a.q = q;
  a.k = k;
  a.v = v;
  for (int i = 0; i < 3; ++i) {
    a.sq[i] = d->stride_q[i];
    a.sk[i] = d->stride_k[i];
    a.sv[i] = d->stride_v[i];
    a.sdo[i] = d->stride_do[i];
  }
  a.B = d->batch;
  a.Nq = d->q_rows;
  a.Nk = d->k_rows;
  a.H = d->heads;
  a.Hk = d->kv_heads;
  a.D = d->head_dim;
  a.causal = d->causal ? 1 : 0;
  a.scale = d->scale;
  a.q_len = d->q_len;
  a.kv_len = d->kv_len;
  return a;
}

static bool at_aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int D, int NT, int NW, int DW, int BN> static int at_launch_fwd(const AttnArgs& a, hipStream_t st) {
  const int lds = 4 * BN * D * 2 + (DW > 1 ? NW * (BN / 16) * NT * 1024 : 0);
  const unsigned grid = (unsigned)a.tiles * a.units * a.B * a.splits;
  if (a.o_rest) {
    TRACE_LDS_OPT_IN((attn_fwd_kernel<D, NT, NW, DW, BN, true>), lds, "attention");
    attn_fwd_kernel<D, NT, NW, DW, BN, true><<<grid, 64 * NW, lds, st>>>(a);
  } else {
    TRACE_LDS_OPT_IN((attn_fwd_kernel<D, NT, NW, DW, BN, false>), lds, "attention");
    attn_fwd_kernel<D, NT, NW, DW, BN, false><<<grid, 64 * NW, lds, st>>>(a);
  }
  return 0;
}
template <int D, int NT, int NW, int DW> static int at_launch_q(const AttnArgs& a, hipStream_t st) {
  const int lds = 4 * 32 * D * 2 + (DW > 1 ? NW * 2 * NT * 1024 : 0);
  TRACE_LDS_OPT_IN((attn_bwd_q_kernel<D, NT, NW, DW>), lds, "attention backward");
  attn_bwd_q_kernel<D, NT, NW, DW><<<(unsigned)a.tiles * a.H * a.B * a.splits, 64 * NW, lds, st>>>(a);
  return 0;
}
template <int D, int NT, int NW, int DW> static int at_launch_kv(const AttnArgs& a, hipStream_t st) {
  const int lds = 4 * 32 * D * 2 + 512 + (DW > 1 ? NW * 2 * NT * 1024 : NW * NT * 16 * D * 2);
  TRACE_LDS_OPT_IN((attn_bwd_kv_kernel<D, NT, NW, DW>), lds, "attention backward");
  attn_bwd_kv_kernel<D, NT, NW, DW><<<(unsigned)a.tiles * a.Hk * a.B * a.splits, 64 * NW, lds, st>>>(a);
  return 0;
}

}  // namespace trace

using namespace trace;

static size_t at_fwd_bytes(const trace_attention_desc* d, const AttnPlan& pl) {
  if (pl.splits <= 1) return 0;
  const size_t rows = (size_t)d->batch * d->heads * d->q_rows;
  return at_align(pl.splits * rows * sizeof(float2)) + at_align(pl.splits * rows * d->head_dim * sizeof(float));
}

extern "C" size_t trace_attention_fwd_workspace_bytes(const trace_attention_desc* d) {
  if (at_check(d, "attention")) return 0;
  return at_fwd_bytes(d, at_plan(d));
}

extern "C" int trace_attention_fwd_bf16(const trace_attention_desc* d, const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                        uint16_t* out, float* lse, uint16_t* out_rest, void* workspace,
                                        size_t workspace_bytes, trace_stream_t stream) {
  if (int rc = at_check(d, "attention")) return rc;
  if (d->batch == 0 || d->q_rows == 0) return 0;
  TRACE_REQUIRE(q && out && (d->k_rows == 0 || (k && v)), "attention: null pointer");
  TRACE_REQUIRE(at_aligned(q) && at_aligned(k) && at_aligned(v) && at_aligned(out) && at_aligned(out_rest),
                "attention: operands must be 16-byte aligned");
  const AttnPlan pl = at_plan(d);
  const size_t need = at_fwd_bytes(d, pl);
  TRACE_REQUIRE(workspace_bytes >= need && (!need || workspace), "attention: workspace of %zu bytes needed", need);
  AttnArgs a = at_args(d, q, k, v);
  a.o = out;
  a.o_rest = out_rest;
  a.lse = lse;
  a.pack = pl.pack;
  a.units = pl.units;
  a.tiles = pl.tiles;
  a.splits = pl.splits;
  const long long rows = (long long)d->batch * d->heads * d->q_rows;
  if (pl.splits > 1) {
    a.part_ml = reinterpret_cast<float2*>(workspace);
    a.part = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + at_align(pl.splits * rows * sizeof(float2)));
  }
  hipStream_t st = (hipStream_t)stream;
  int rc = 0;
  if (pl.tile_rows == 16) {
    switch (pl.D) {
      case 32: rc = at_launch_fwd<32, 1, 1, 1, 32>(a, st); break;
      case 64: rc = at_launch_fwd<64, 1, 1, 1, 32>(a, st); break;
      case 128: rc = at_launch_fwd<128, 1, 1, 1, 32>(a, st); break;
      case 256: rc = at_launch_fwd<256, 1, 2, 2, 32>(a, st); break;
      default: rc = at_launch_fwd<512, 1, 4, 4, 32>(a, st); break;
    }
  } else {
    const bool whole = pl.tile_rows == 128;
    switch (pl.D) {
      case 32: rc = whole ? at_launch_fwd<32, 2, 4, 1, 64>(a, st) : at_launch_fwd<32, 1, 4, 1, 64>(a, st); break;
      case 64: rc = whole ? at_launch_fwd<64, 2, 4, 1, 64>(a, st) : at_launch_fwd<64, 1, 4, 1, 64>(a, st); break;
      case 128: rc = whole ? at_launch_fwd<128, 2, 4, 1, 64>(a, st) : at_launch_fwd<128, 1, 4, 1, 64>(a, st); break;
      case 256: rc = at_launch_fwd<256, 1, 4, 1, 32>(a, st); break;
      default:
        rc = whole ? at_launch_fwd<512, 1, 8, 1, 32>(a, st)
             : pl.tile_rows == 64 ? at_launch_fwd<512, 1, 8, 2, 32>(a, st) : at_launch_fwd<512, 1, 4, 2, 32>(a, st);
        break;
    }
  }
  if (rc) return rc;
  if (int e = check_launch("attention")) return e;
  if (pl.splits > 1) {
    if (pl.splits <= AT_FEW) {
      const int grid = ceil_div(rows, 256 / (d->head_dim / 4));
      if (out_rest) attn_combine_few_kernel<true><<<grid, 256, 0, st>>>(a);
      else attn_combine_few_kernel<false><<<grid, 256, 0, st>>>(a);
    } else if (out_rest) {
      attn_combine_kernel<true><<<(unsigned)rows, 256, 0, st>>>(a);
    } else {
      attn_combine_kernel<false><<<(unsigned)rows, 256, 0, st>>>(a);
    }
    return check_launch("attention combine");
  }
  return 0;
}

struct AttnBwdBytes {
  size_t delta, q, kv;
};
static AttnBwdBytes at_bwd_bytes(const trace_attention_desc* d, const AttnPlan& pl) {
  AttnBwdBytes s;
  s.delta = at_align((size_t)d->batch * d->heads * d->q_rows * sizeof(float));
  s.q = pl.q_splits > 1 ? at_align((size_t)pl.q_splits * d->batch * d->q_rows * d->heads * d->head_dim * sizeof(float)) : 0;
  s.kv = pl.k_splits > 1 ? at_align((size_t)pl.k_splits * 2 * d->batch * d->k_rows * d->kv_heads * d->head_dim * sizeof(float)) : 0;
  return s;
}

extern "C" size_t trace_attention_bwd_workspace_bytes(const trace_attention_desc* d) {
  if (at_check(d, "attention backward")) return 0;
  const AttnBwdBytes s = at_bwd_bytes(d, at_plan(d));
  return s.delta + (s.q > s.kv ? s.q : s.kv);   // the splits of dq are reduced before those of dk / dv are written
}

extern "C" int trace_attention_bwd_bf16(const trace_attention_desc* d, const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                        const uint16_t* out, const float* lse, const uint16_t* out_rest,
                                        const uint16_t* dout, uint16_t* dq, uint16_t* dk, uint16_t* dv, void* workspace,
                                        size_t workspace_bytes, trace_stream_t stream) {
  if (int rc = at_check(d, "attention backward")) return rc;
  for (int i = 0; i < 3; ++i)
    TRACE_REQUIRE((d->stride_do[i] & 7) == 0, "attention backward: strides must be multiples of 8 elements");
  if (d->batch == 0) return 0;
  TRACE_REQUIRE(d->q_rows == 0 || (q && out && lse && out_rest && dout && dq), "attention backward: null pointer");
  TRACE_REQUIRE(d->k_rows == 0 || (k && v && dk && dv), "attention backward: null pointer");
  TRACE_REQUIRE(at_aligned(q) && at_aligned(k) && at_aligned(v) && at_aligned(out) && at_aligned(out_rest) && at_aligned(dout) && at_aligned(dq) &&
                    at_aligned(dk) && at_aligned(dv),
                "attention backward: operands must be 16-byte aligned");
  const AttnPlan pl = at_plan(d);
  const AttnBwdBytes s = at_bwd_bytes(d, pl);
  const size_t need = s.delta + (s.q > s.kv ? s.q : s.kv);
  TRACE_REQUIRE(workspace_bytes >= need && (!need || workspace), "attention backward: workspace of %zu bytes needed", need);
  AttnArgs a = at_args(d, q, k, v);
  a.out = out;
  a.rest = out_rest;
  a.dout = dout;
  a.lse = const_cast<float*>(lse);
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.ndelta = reinterpret_cast<float*>(workspace);
  a.part = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + s.delta);
  hipStream_t st = (hipStream_t)stream;
  int rc = 0;
  if (d->q_rows > 0) {
    a.tiles = pl.q_tiles;
    a.splits = pl.q_splits;
    const bool whole = pl.q_rows == (pl.D <= 256 ? 128 : 64);
    switch (pl.D) {
      case 32: rc = whole ? at_launch_q<32, 2, 4, 1>(a, st) : at_launch_q<32, 1, 4, 1>(a, st); break;
      case 64: rc = whole ? at_launch_q<64, 2, 4, 1>(a, st) : at_launch_q<64, 1, 4, 1>(a, st); break;
      case 128: rc = whole ? at_launch_q<128, 2, 4, 1>(a, st) : at_launch_q<128, 1, 4, 1>(a, st); break;
      case 256: rc = whole ? at_launch_q<256, 1, 8, 1>(a, st) : at_launch_q<256, 1, 4, 1>(a, st); break;
      default: rc = whole ? at_launch_q<512, 1, 8, 2>(a, st) : at_launch_q<512, 1, 4, 2>(a, st); break;
    }
    if (rc) return rc;
    if (int e = check_launch("attention backward (dq)")) return e;
    if (pl.q_splits > 1) {
      const long long n = (long long)d->batch * d->q_rows * d->heads * d->head_dim;
      attn_reduce_kernel<<<ceil_div(n, 1024), 256, 0, st>>>(a.part, n, pl.q_splits, n, d->scale, dq, 0.f, nullptr);
      if (int e = check_launch("attention backward (dq splits)")) return e;
    }
  }
  if (d->k_rows > 0) {
    a.tiles = pl.k_tiles;
    a.splits = pl.k_splits;
    const bool whole = pl.k_rows == (pl.D <= 256 ? 128 : 64);
    switch (pl.D) {
      case 32: rc = whole ? at_launch_kv<32, 2, 4, 1>(a, st) : at_launch_kv<32, 1, 4, 1>(a, st); break;
      case 64: rc = whole ? at_launch_kv<64, 2, 4, 1>(a, st) : at_launch_kv<64, 1, 4, 1>(a, st); break;
      case 128: rc = whole ? at_launch_kv<128, 2, 4, 1>(a, st) : at_launch_kv<128, 1, 4, 1>(a, st); break;
      case 256: rc = whole ? at_launch_kv<256, 1, 8, 1>(a, st) : at_launch_kv<256, 1, 4, 1>(a, st); break;
      default: rc = whole ? at_launch_kv<512, 1, 8, 2>(a, st) : at_launch_kv<512, 1, 8, 4>(a, st); break;
    }
    if (rc) return rc;
    if (int e = check_launch("attention backward (dk, dv)")) return e;
    if (pl.k_splits > 1) {
      const long long n = (long long)d->batch * d->k_rows * d->kv_heads * d->head_dim;
      attn_reduce_kernel<<<dim3(ceil_div(n, 1024), 2), 256, 0, st>>>(a.part, 2 * n, pl.k_splits, n, d->scale, dk, 1.0f, dv);
      if (int e = check_launch("attention backward (dk, dv splits)")) return e;
    }
  }
  return 0;
}
