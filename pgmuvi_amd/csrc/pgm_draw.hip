// pgm_draw.hip -- draws from rows of log-weights (the frequency posterior of a periodogram), with tempering and truncation.
//
// Row l of `cols` log-weights, best value m:   z_i = (l_i - m) / T,   w_i = exp z_i  (one for the best, zero for -inf and NaN).
// In the order (l descending, i ascending):    A = the first top_k entries,   P = the shortest beginning of A that holds at least
// top_p of A's weight,   kept = the entries of P with w_i >= min_p.   Z = sum of the kept weights, and a number u in [0, 1) draws
// the first kept i, in the order of i, whose running sum F(i) exceeds u Z.  log p = z_i - log Z.
//
// All three truncations keep a beginning of ONE order, so the kept set is "everything before a cut (value, index)" and w >= min_p.
// The cut is found by histograms over the values' ordered bit patterns ("keys"), 2048 bins per pass over the range that still
// matters: counts for top_k; weights for top_p, held in two integer words (2^-40 and 2^-80 steps: sums of integers do not
// depend on the order of the LDS atomics, and 80 bits are more than the fp64 sums they are compared with).  Equal values are
// split by index the same way.  The running sums are fp64, formed cell by cell (64 E neighbouring entries) in a fixed order: the
// same call gives the same draws.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>
#include <algorithm>
#include "../../include/pgmuvi_hip.h"
#include "pgm_exp.h"

namespace {

typedef unsigned long long u64;
constexpr int LOAD = 16, BATCH = 4;                             // bytes of a lane's load; loads of a wavefront in flight
constexpr int MAX_CELLS = 2048;                                 // of a row (wider cells beyond: `units` loads per lane each)
constexpr int64_t MAX_COLS = 1 << 24;                             // (2^24 weights of at most one, in steps of 2^-40, fit 64 bits)
constexpr int64_t EVERY = INT64_MAX;

// ---- values and their keys: unsigned integers in the same order; -0 is +0, NaN is -inf.  `wide`: what maxima are formed in -----
__device__ __forceinline__ u64 key_of_bits(u64 b) { return (b >> 63) ? ~b : b | (1ull << 63); }
__device__ __forceinline__ uint32_t key_of_bits(uint32_t b) { return (b >> 31) ? ~b : b | (1u << 31); }
struct F64 {
  typedef double raw, wide; typedef u64 key;
  static constexpr raw absent() { return -__builtin_inf(); }
  static __device__ __forceinline__ wide widen(raw x) { return x; }
  static __device__ __forceinline__ wide larger(wide a, wide b) { return __builtin_fmax(a, b); }        // (a NaN loses)
  static __device__ __forceinline__ key to_key(raw x) { return key_of_bits((u64)__double_as_longlong(x != x ? absent() : x + 0.0)); }
  static __device__ __forceinline__ key key_of_wide(wide x) { return to_key(x); }
  static __device__ __forceinline__ double of_key(key k) { return __longlong_as_double((long long)((k >> 63) ? k & ~(1ull << 63) : ~k)); }
};
struct F32 {
  typedef float raw, wide; typedef uint32_t key;
  static constexpr raw absent() { return -__builtin_inff(); }
  static __device__ __forceinline__ wide widen(raw x) { return x; }
  static __device__ __forceinline__ wide larger(wide a, wide b) { return __builtin_fmaxf(a, b); }
  static __device__ __forceinline__ key to_key(raw x) { return key_of_bits(__float_as_uint(x != x ? absent() : x + 0.0f)); }
  static __device__ __forceinline__ key key_of_wide(wide x) { return to_key(x); }
  static __device__ __forceinline__ double of_key(key k) { return (double)__uint_as_float((k >> 31) ? k & ~(1u << 31) : ~k); }
};
template <int F16BIT> struct Half {                              // bf16 (0) and fp16 (1): the 16-bit patterns are ordered the same way
  typedef uint16_t raw; typedef float wide; typedef uint32_t key;
  static constexpr uint32_t INF = F16BIT ? 0x7c00u : 0x7f80u;
  static constexpr raw absent() { return (raw)(0x8000u | INF); }
  static __device__ __forceinline__ wide widen(raw b) {
    if constexpr (F16BIT) { __half_raw r; r.x = b; return __half2float(__half(r)); }
    else return __uint_as_float((uint32_t)b << 16);
  }
  static __device__ __forceinline__ wide larger(wide a, wide b) { return __builtin_fmaxf(a, b); }
  static __device__ __forceinline__ key to_key(raw b) {
    const uint32_t mag = b & 0x7fffu;
    if (mag > INF) return 0xffffu - (0x8000u | INF);
    if (mag == 0) return 0x8000u;
    return (b >> 15) ? 0xffffu - b : b | 0x8000u;
  }
  static __device__ __forceinline__ key key_of_wide(wide x) {     // (x is one of the type's values)
    if constexpr (F16BIT) { const __half h = __float2half(x); return to_key(static_cast<__half_raw>(h).x); }
    else return to_key((raw)(__float_as_uint(x) >> 16));
  }
  static __device__ __forceinline__ double of_key(key k) { return (double)widen((raw)((k & 0x8000u) ? k & 0x7fffu : 0xffffu - k)); }
};

struct Param { double v; const double* p; };                    // one number for every row, or one per row
struct ParamI { int64_t v; const int64_t* p; };
constexpr int STATE = 2;                                        // per row in memory: the cut's key and index
struct DrawArgs {
  const void* logits; int64_t row_stride, col_stride, cols;
  const int64_t* lengths;                                       // entries of each row, or null: cols
  const double* u; int64_t draws;
  Param temperature, top_p, min_p; ParamI top_k;
  int64_t* index; double* logp;
  int units, max_cells;                                         // loads per lane and cell, cells of a full row
  u64* keys; double* sums; u64* lows; u64* state;               // rows whose passes are launches of their own: [row][max_cells], [row][groups], [row][STATE]
};

template <class K> struct Cut { K key; int64_t idx; };          // kept: key above, or equal and index not above
template <class K> __device__ __forceinline__ bool before(const Cut<K>& c, K key, int64_t i) { return key > c.key || (key == c.key && i <= c.idx); }

// ---- wavefront reductions -------------------------------------------------------------------------------------------------
// (within rows of 16 lanes by data-parallel moves -- a shuffle goes through the LDS, ~100 cycles a step --, the four rows by lane reads)
template <int CTRL> __device__ __forceinline__ double moved(double v) {
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, true), __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL> __device__ __forceinline__ float moved(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true)); }
__device__ __forceinline__ double of_lane(double v, int l) { return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l), __builtin_amdgcn_readlane(__double2loint(v), l)); }
__device__ __forceinline__ float of_lane(float v, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); }
template <class V, class Op> __device__ __forceinline__ V wave_join(V v, Op op) {
  v = op(v, moved<0xB1>(v));                                    // neighbours, pairs, halves of a row, the row
  v = op(v, moved<0x4E>(v));
  v = op(v, moved<0x141>(v));
  v = op(v, moved<0x140>(v));
  return op(op(of_lane(v, 0), of_lane(v, 16)), op(of_lane(v, 32), of_lane(v, 48)));
}
__device__ __forceinline__ double wave_sum(double v) { return wave_join(v, [](double a, double b) { return a + b; }); }
__device__ __forceinline__ float wave_max(float v) { return wave_join(v, [](float a, float b) { return __builtin_fmaxf(a, b); }); }
__device__ __forceinline__ double wave_max(double v) { return wave_join(v, [](double a, double b) { return __builtin_fmax(a, b); }); }
__device__ __forceinline__ u64 wave_max(u64 v) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) { const u64 o = __shfl_xor(v, s); v = o > v ? o : v; }
  return v;
}
template <class V> __device__ __forceinline__ V wave_scan(V v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) { const V o = __shfl_up(v, s); if (lane >= s) v += o; }
  return v;
}
__device__ __forceinline__ double mass_of(u64 hi, u64 lo) { return (double)hi * 0x1p-40 + (double)lo * 0x1p-80; }

// ---- one row ----------------------------------------------------------------------------------------------------------------
template <class F> struct Row {
  typedef typename F::raw raw; typedef typename F::key K;
  static constexpr int VEC = LOAD / (int)sizeof(raw), UNIT = 64 * VEC;       // entries of one load of a lane, of a wavefront
  const raw* x; int64_t stride, n;
  int units, cells;
  double best, t, per_t;                                        // highest value, temperature, 1 / temperature
  __device__ __forceinline__ int64_t width() const { return (int64_t)units * UNIT; }
  __device__ __forceinline__ K key(int64_t i) const { return F::to_key(x[i * stride]); }
  __device__ __forceinline__ double z(K k) const { const double l = F::of_key(k); return l == best ? 0.0 : (l - best) / t; }
  __device__ __forceinline__ double weight_of(double l) const { return l == best ? 1.0 : exp_neg((l - best) * per_t); }      // (l above -inf)
  __device__ __forceinline__ double weight(K k) const { return weight_of(F::of_key(k)); }
  // this lane's entries of unit j: VEC neighbours from at(j) on; behind the end -inf
  __device__ __forceinline__ int64_t at(int64_t j) const { return j * UNIT + (threadIdx.x & 63) * VEC; }
  __device__ __forceinline__ bool whole(int64_t j) const { return stride == 1 && (j + 1) * UNIT <= n; }
  __device__ __forceinline__ void load_whole(int64_t j, raw (&r)[VEC]) const { __builtin_memcpy(r, x + at(j), LOAD); }
  __device__ __forceinline__ void load(int64_t j, raw (&r)[VEC]) const {
    const int64_t i = at(j);
    if (whole(j)) { load_whole(j, r); return; }
#pragma unroll
    for (int e = 0; e < VEC; ++e) r[e] = i + e < n ? x[(i + e) * stride] : F::absent();
  }
};
template <class F> __device__ __forceinline__ typename F::key neg_key() {                     // the key of -inf (and NaN)
  return F::to_key(F::absent());
}
// a key above that of -inf and not above any whose value is at least v
template <class F> __device__ __forceinline__ typename F::key key_below(double v) {
  typedef typename F::key K;
  const K neg = neg_key<F>();
  K k;
  if constexpr (sizeof(typename F::raw) == 8) k = F::to_key(v);
  else if constexpr (sizeof(typename F::raw) == 4) k = F::to_key((float)v);
  else {                                                        // (halves: by bisection of their ordered patterns, up to +inf)
    K a = neg, b = 0xffffu - neg;
    while (a + 1 < b) { const K m = (a + b) >> 1; if (F::of_key(m) >= v) b = m; else a = m; }
    k = b;
  }
  return k <= neg + 1 ? neg + 1 : k - 1;
}

// Two builds of a row's code: 8 wavefronts for long rows, 4 for short ones and for the launches that share a row among workgroups
struct Long { static constexpr int NT = 512, BITS = 11, CELLS = MAX_CELLS, LIST = 512; };
struct Short { static constexpr int NT = 256, BITS = 9, CELLS = 64, LIST = 256; };

template <class C> struct Shared {
  static constexpr int BINS = 1 << C::BITS, NW = C::NT / 64;
  union {
    struct { uint32_t count[BINS]; u64 hi[BINS], lo[BINS]; } bins;
    double cells[C::CELLS];                                     // weights of the cells, then their running sums
  };
  u64 best[C::CELLS];                                           // highest key of every cell, 0: nothing above -inf
  u64 list_key[C::LIST]; uint32_t list_idx[C::LIST];
  u64 red[NW], part[3][NW], found[7];
  double sums[NW];
  int listed;
};

template <class C> __device__ __forceinline__ u64 block_max(u64 (&red)[C::NT / 64], u64 v) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < C::NT / 64; ++w) v = red[w] > v ? red[w] : v;
  return v;
}
// running sum over the workgroup's threads, in thread order
template <class C> __device__ __forceinline__ double block_scan(double (&sums)[C::NT / 64], double v) {
  const double inc = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sums[threadIdx.x >> 6] = inc;
  __syncthreads();
  double base = 0.0;
  for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) base += sums[w];
  return base + inc;
}

// f(cell, this lane's entries of one unit, first index, last unit of the cell?) for the cells c0 <= c < c1 -- with SEEN only those
// whose highest key is at least `lo`: a wavefront per cell.  The next BATCH cells' loads are in flight while the present ones are
// worked on.
template <bool SEEN, int THREADS, bool HEAVY = true, class F, class Fn> __device__ __forceinline__ void for_cells(const Row<F>& R, const u64* best, int c0, int c1, u64 lo, Fn f) {
  typedef typename F::raw raw;
  constexpr int NW = THREADS / 64, VEC = Row<F>::VEC, STEP = NW * BATCH;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int full = c0;                                                // the cells up to here are one whole load per lane
  if (R.units == 1 && R.stride == 1) {
    const int whole = (int)(R.n / Row<F>::UNIT);
    full = whole < c1 ? whole : c1;
    raw next[BATCH][VEC];
    auto wanted = [&](int cc) { return cc < full && (!SEEN || best[cc] >= lo); };
    auto fetch = [&](int c) {
#pragma unroll
      for (int s = 0; s < BATCH; ++s) if (wanted(c + s * NW)) R.load_whole(c + s * NW, next[s]);
    };
    int c = c0 + wave;
    if (c < full) fetch(c);
    for (; c < full; c += STEP) {
      raw r[BATCH][VEC];
      __builtin_memcpy(r, next, sizeof(r));
      if (c + STEP < full) fetch(c + STEP);
#pragma unroll
      for (int s = 0; s < BATCH; ++s) {
        if (wanted(c + s * NW)) f(c + s * NW, r[s], R.at(c + s * NW), true);
        if (HEAVY) __builtin_amdgcn_sched_barrier(0);           // (one unit's exponentials at a time: interleaved, four units' do not fit the registers)
      }
    }
    full = full > c0 ? full : c0;
  }
  for (int c = full + wave; c < c1; c += NW) {                  // the row's end; strided rows; very long ones
    if (SEEN && best[c] < lo) continue;
    for (int j = 0; j < R.units; ++j) {
      raw r[VEC];
      const int64_t u = (int64_t)c * R.units + j;
      R.load(u, r);
      f(c, r, R.at(u), j == R.units - 1);
    }
  }
}

// ---- the cut -------------------------------------------------------------------------------------------------------------------
// The bin that holds it: `want` entries, or (WEIGHTED) `target` of weight -- `share` of all that the bins hold on the first pass,
// where target < 0 asks for it.  found: bin, entries before it, in it, hi / lo before it, target, entries in all bins
template <bool WEIGHTED, class C> __device__ __forceinline__ void find_bin(Shared<C>& S, u64 before_n, u64 before_hi, u64 before_lo, u64 want, double share, double target) {
  constexpr int PER = Shared<C>::BINS / C::NT, NW = C::NT / 64;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, b0 = t * PER;
  __syncthreads();
  u64 n = 0, hi = 0, lo = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) { n += S.bins.count[b0 + k]; if (WEIGHTED) { hi += S.bins.hi[b0 + k]; lo += S.bins.lo[b0 + k]; } }
  u64 sn = wave_scan(n), shi = WEIGHTED ? wave_scan(hi) : 0, slo = WEIGHTED ? wave_scan(lo) : 0;
  if (lane == 63) { S.part[0][wave] = sn; S.part[1][wave] = shi; S.part[2][wave] = slo; }
  __syncthreads();
  u64 all = 0, all_hi = 0, all_lo = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w == wave) { sn += all; shi += all_hi; slo += all_lo; }
    all += S.part[0][w]; all_hi += S.part[1][w]; all_lo += S.part[2][w];
  }
  if (WEIGHTED) {
    if (target < 0.0) target = share * mass_of(all_hi, all_lo);
    const double most = mass_of(before_hi + all_hi, before_lo + all_lo);
    target = target < most ? target : most;                     // (a rounding of the product must not put it behind the end)
  } else if (want > before_n + all) want = before_n + all;
  auto reached = [&](u64 an, u64 ahi, u64 alo) { return WEIGHTED ? mass_of(before_hi + ahi, before_lo + alo) >= target : before_n + an >= want; };
  u64 an = sn - n, ahi = shi - hi, alo = slo - lo;
  if (n && !reached(an, ahi, alo) && reached(sn, shi, slo)) {
    int b = b0;
#pragma unroll
    for (int k = 0; k < PER - 1; ++k) {
      if (b != b0 + k) continue;
      const u64 c = S.bins.count[b], h = WEIGHTED ? S.bins.hi[b] : 0, l = WEIGHTED ? S.bins.lo[b] : 0;
      if (c && reached(an + c, ahi + h, alo + l)) continue;     // (this one)
      an += c; ahi += h; alo += l; ++b;
    }
    S.found[0] = (u64)b; S.found[1] = before_n + an; S.found[2] = S.bins.count[b]; S.found[3] = before_hi + ahi; S.found[4] = before_lo + alo;
    S.found[5] = (u64)__double_as_longlong(target); S.found[6] = all;
  }
  __syncthreads();
}
template <bool WEIGHTED, class C> __device__ __forceinline__ void clear_bins(Shared<C>& S) {
  __syncthreads();
  for (int b = threadIdx.x; b < Shared<C>::BINS; b += C::NT) { S.bins.count[b] = 0; if (WEIGHTED) { S.bins.hi[b] = 0; S.bins.lo[b] = 0; } }
  if (threadIdx.x == 0) S.listed = 0;
  __syncthreads();
}
template <class C> __device__ __forceinline__ int shift_of(u64 span) { return span < (u64)Shared<C>::BINS ? 0 : 64 - __clzll(span) - C::BITS; }

// The list in the order of the cut: every thread counts what is ahead of its entry (broadcast reads, two barriers; a sort by
// exchanges takes 45 of them for 512 entries)
template <class C> __device__ __forceinline__ void sort_list(Shared<C>& S, int count) {
  const int t = threadIdx.x;
  __syncthreads();
  u64 key = 0; uint32_t idx = 0; int rank = 0, ties = 0;
  if (t < count) { key = S.list_key[t]; idx = S.list_idx[t]; }
  if (t - (t & 63) < count) {
    for (int j = 0; j < count; ++j) { const u64 k = S.list_key[j]; rank += k > key; ties += k == key; }
    if (__any(t < count && ties > 1))
      for (int j = 0; j < count; ++j) rank += S.list_key[j] == key && S.list_idx[j] < idx;
  }
  __syncthreads();
  if (t < count) { S.list_key[rank] = key; S.list_idx[rank] = idx; }
  __syncthreads();
}

// adds a weight to a bin: 2^-40 steps in one word, 2^-80 steps in the other (the magic number 2^52 leaves the rounded integer in the
// low bits of a sum)
template <class C> __device__ __forceinline__ void add_weight(Shared<C>& S, int b, double w) {
  const double x = w * 0x1p40, magic = 0x1p52, h = __builtin_floor(x), l = (x - h) * 0x1p40;
  const u64 hi = (u64)__double_as_longlong(h + magic) & ((1ull << 52) - 1), lo = (u64)__double_as_longlong(l + magic) & ((1ull << 52) - 1);
  if (hi) atomicAdd(&S.bins.hi[b], hi);
  if (lo) atomicAdd(&S.bins.lo[b], lo);
}

// The cut behind the first `want` entries of what `have` keeps (WEIGHTED: behind the shortest beginning with `share` of its weight).
// lo / hi: range of keys that can matter; S.best: the cells' highest keys.  The first bins divide the range of values evenly,
// the later ones (where a bin held too many to sort) the range of the bin's keys.
template <bool WEIGHTED, class C, class F> __device__ Cut<typename F::key> select(const Row<F>& R, Shared<C>& S, typename F::key lo, typename F::key hi,
                                                                                  Cut<typename F::key> have, u64 want, double share) {
  typedef typename F::key K;
  typedef typename F::raw raw;
  constexpr int VEC = Row<F>::VEC, BINS = Shared<C>::BINS;
  u64 bn = 0, bhi = 0, blo = 0;
  double target = -1.0;
  bool first = true;
  const double range = F::of_key(hi) - F::of_key(lo), scale = BINS / range;
  bool even = range > 0.0 && range < 1e300 && scale < 1e300;
  const double best = R.best;
  auto even_bin = [&](double l) { const int b = (int)((best - l) * scale); return b < BINS ? b : BINS - 1; };
  for (;;) {
    const int shift = shift_of<C>((u64)(hi - lo));
    clear_bins<WEIGHTED>(S);
    for_cells<true, C::NT>(R, S.best, 0, R.cells, lo, [&](int, const raw (&r)[VEC], int64_t i, bool) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const K k = F::to_key(r[e]);
        if (k < lo || k > hi || !before(have, k, i + e)) continue;
        const double l = (double)F::widen(r[e]);
        const int b = even ? even_bin(l) : (int)((u64)(hi - k) >> shift);
        atomicAdd(&S.bins.count[b], 1u);
        if (WEIGHTED) { add_weight(S, b, R.weight_of(l)); __builtin_amdgcn_sched_barrier(0); }
      }
    });
    find_bin<WEIGHTED>(S, bn, bhi, blo, want, share, target);
    if (!WEIGHTED && first && S.found[6] <= want) return Cut<K>{lo, EVERY};       // (all of them)
    first = false;
    const u64 bin = S.found[0], in_bin = S.found[2];
    bn = S.found[1]; bhi = S.found[3]; blo = S.found[4]; target = __longlong_as_double((long long)S.found[5]);
    K top = hi, bottom = lo;
    if (!even) {
      top = (K)(hi - (K)(bin << shift));
      const u64 width = (1ull << shift) - 1;
      bottom = (u64)(top - lo) <= width ? lo : (K)(top - (K)width);
    }
    auto in_it = [&](K k, raw r) { return k >= bottom && k <= top && (!even || even_bin((double)F::widen(r)) == (int)bin); };
    if (in_bin <= (u64)C::LIST) {
      // few enough to sort: the bin's entries by (key, index), then the first that reaches the target
      for_cells<true, C::NT>(R, S.best, 0, R.cells, bottom, [&](int, const raw (&r)[VEC], int64_t i, bool) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const K k = F::to_key(r[e]);
          if (!in_it(k, r[e]) || !before(have, k, i + e)) continue;
          const int at = atomicAdd(&S.listed, 1);
          S.list_key[at] = k; S.list_idx[at] = (uint32_t)(i + e);
        }
      });
      const int count = (int)in_bin, t = threadIdx.x;
      sort_list(S, count);
      int at = (int)(want - bn) - 1;
      if (WEIGHTED) {
        const double sum = block_scan<C>(S.sums, t < count ? R.weight((K)S.list_key[t]) : 0.0);
        const bool yes = t < count && mass_of(bhi, blo) + sum >= target;
        at = count - 1 - (int)block_max<C>(S.red, yes ? (u64)(count - 1 - t) : 0);
      }
      return Cut<K>{(K)S.list_key[at], (int64_t)S.list_idx[at]};
    }
    if (even) {                                                 // the keys of the bin's entries
      u64 high = 0, low = ~0ull;
      for_cells<true, C::NT>(R, S.best, 0, R.cells, lo, [&](int, const raw (&r)[VEC], int64_t i, bool) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const K k = F::to_key(r[e]);
          if (!in_it(k, r[e]) || !before(have, k, i + e)) continue;
          high = (u64)k > high ? (u64)k : high; low = (u64)k < low ? (u64)k : low;
        }
      });
      hi = (K)block_max<C>(S.red, high); lo = (K)~block_max<C>(S.red, ~low);
      even = false;
      if (!WEIGHTED && bn + in_bin == want) return Cut<K>{lo, EVERY};
      continue;
    }
    if (!WEIGHTED && bn + in_bin == want) return Cut<K>{bottom, EVERY};
    if (shift == 0) {                                           // many equal values: the first m of them by index
      u64 m = WEIGHTED ? 1 : want - bn;
      if (WEIGHTED) {
        const double w = R.weight(top), above = mass_of(bhi, blo);
        const double guess = ceil((target - above) / w);
        m = guess >= (double)in_bin ? in_bin : guess < 1.0 ? 1 : (u64)guess;
        while (m > 1 && above + (double)(m - 1) * w >= target) --m;
        while (m < in_bin && above + (double)m * w < target) ++m;
      }
      if (m >= in_bin) return Cut<K>{bottom, EVERY};
      int64_t i0 = 0, i1 = R.n - 1;
      u64 passed = 0;
      for (;;) {
        const int ishift = shift_of<C>((u64)(i1 - i0));
        clear_bins<false>(S);
        for_cells<true, C::NT>(R, S.best, (int)(i0 / R.width()), (int)(i1 / R.width()) + 1, top, [&](int, const raw (&r)[VEC], int64_t i, bool) {
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (F::to_key(r[e]) == top && i + e >= i0 && i + e <= i1 && before(have, top, i + e)) atomicAdd(&S.bins.count[(u64)(i + e - i0) >> ishift], 1u);
        });
        find_bin<false>(S, passed, 0, 0, m, 0.0, 0.0);
        const int64_t from = i0 + (int64_t)(S.found[0] << ishift), to = from + (int64_t)((1ull << ishift) - 1);
        passed = S.found[1];
        const u64 here = S.found[2];
        i0 = from;
        i1 = to < i1 ? to : i1;
        if (ishift == 0 || passed + here == m) return Cut<K>{top, i1};
      }
    }
    hi = top; lo = bottom;
  }
}
template <class K> __device__ __forceinline__ Cut<K> tighter(const Cut<K>& a, const Cut<K>& b) {
  if (a.key != b.key) return a.key > b.key ? a : b;
  return a.idx < b.idx ? a : b;
}

// ---- a row's settings -------------------------------------------------------------------------------------------------------------
struct Settings { double t, top_p, min_p; int64_t top_k; bool plain; };
__device__ __forceinline__ Settings settings_of(const DrawArgs& A, int64_t row) {
  Settings s;
  const double temp = A.temperature.p ? A.temperature.p[row] : A.temperature.v;
  s.top_p = A.top_p.p ? A.top_p.p[row] : A.top_p.v;
  s.min_p = A.min_p.p ? A.min_p.p[row] : A.min_p.v;
  s.top_k = A.top_k.p ? A.top_k.p[row] : A.top_k.v;
  if (s.top_p <= 0.0 || !(temp > 0.0)) s.top_k = 1;            // the best entry alone (the first of equal ones)
  s.t = temp > 0.0 ? (temp < 1e300 ? temp : 1e300) : 1.0;
  if (!(s.top_p > 0.0 && s.top_p < 1.0)) s.top_p = 1.0;
  s.min_p = s.min_p > 0.0 ? (s.min_p < 1.0 ? s.min_p : 1.0) : 0.0;
  s.top_k = s.top_k > 0 ? s.top_k : 0;
  s.plain = s.top_k == 0 && s.top_p == 1.0 && s.min_p == 0.0;
  return s;
}
template <class F> __device__ __forceinline__ Row<F> row_of(const DrawArgs& A, int64_t row, double t) {
  Row<F> R;
  int64_t n = A.cols;
  if (A.lengths) { n = A.lengths[row]; n = n < 0 ? 0 : n > A.cols ? A.cols : n; }
  R.x = static_cast<const typename F::raw*>(A.logits) + row * A.row_stride; R.stride = A.col_stride; R.n = n;
  R.units = A.units;
  R.cells = (int)((n + R.width() - 1) / R.width());
  R.best = 0.0; R.t = t; R.per_t = 1.0 / t;
  return R;
}

// does the cut need the lowest key of the row (as the end of the bins' range)?
__device__ __forceinline__ bool wants_lowest(const Settings& p, int cells) { return p.top_k >= cells || (p.top_k == 0 && p.top_p < 1.0); }

// ---- the passes over a row ----------------------------------------------------------------------------------------------------------
// highest key of the cells [c0, c1) -> keys[c]; where nothing is truncated (SUMS) also their weight relative to it.
// Returns, where `lowest` asks for it, this lane's lowest value above -inf (else +inf)
template <int THREADS, bool SUMS, class F> __device__ __forceinline__ typename F::wide pass_best(Row<F> R, int c0, int c1, u64* keys, double* sums, bool lowest) {
  typedef typename F::raw raw;
  typedef typename F::wide wide;
  constexpr int VEC = Row<F>::VEC;
  const wide none = (wide)-__builtin_inf();
  wide run = none, low = -none;
  for_cells<false, THREADS, SUMS>(R, (const u64*)nullptr, c0, c1, 0, [&](int c, const raw (&r)[VEC], int64_t, bool last) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) run = F::larger(run, F::widen(r[e]));
    if (lowest) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) { const wide v = F::widen(r[e]); low = v > none && v < low ? v : low; }
    }
    if (!last) return;
    const wide top = wave_max(run);
    run = none;
    if ((threadIdx.x & 63) == 0) keys[c] = top > none ? (u64)F::key_of_wide(top) : 0;
    if constexpr (!SUMS) return;
    double s = 0.0;
    if (top > none) {
      R.best = (double)top;
      auto add = [&](raw x) { const wide v = F::widen(x); s += v > none ? R.weight_of((double)v) : 0.0; };
      if (R.units == 1) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) { add(r[e]); if (e & 1) __builtin_amdgcn_sched_barrier(0); }
      } else {
        for (int j = 0; j < R.units; ++j) {
          raw q[VEC];
          R.load((int64_t)c * R.units + j, q);
#pragma unroll
          for (int e = 0; e < VEC; ++e) { add(q[e]); if (e & 1) __builtin_amdgcn_sched_barrier(0); }
        }
      }
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sums[c] = s;
  });
  return low;
}
// kept weight of the cells [c0, c1) -> sums[c]
template <int THREADS, class F> __device__ __forceinline__ void pass_weights(const Row<F>& R, const u64* best, int c0, int c1, const Cut<typename F::key>& cut, double min_p, double* sums) {
  typedef typename F::key K;
  constexpr int VEC = Row<F>::VEC;
  const K neg = neg_key<F>();
  K lo = cut.key > neg ? cut.key : neg + 1;
  if (min_p > 0.0) {                                            // (no cell below this, with room for the roundings, has an entry of that weight)
    double v = R.best + R.t * log(min_p);
    v -= 1e-12 * (fabs(v) + fabs(R.best)) + 1e-9 * R.t;
    const K m = key_below<F>(v);
    lo = m > lo ? m : lo;
  }
  for (int c = c0 + (int)threadIdx.x; c < c1; c += THREADS) if (best[c] < (u64)lo) sums[c] = 0.0;
  double s = 0.0;
  for_cells<true, THREADS>(R, best, c0, c1, (u64)lo, [&](int c, const typename F::raw (&r)[VEC], int64_t i, bool last) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const K k = F::to_key(r[e]);
      if (k >= lo && before(cut, k, i + e)) { const double w = R.weight_of((double)F::widen(r[e])); s += w < min_p ? 0.0 : w; }
      if (e & 1) __builtin_amdgcn_sched_barrier(0);
    }
    if (!last) return;
    const double total = wave_sum(s);
    s = 0.0;
    if ((threadIdx.x & 63) == 0) sums[c] = total;
  });
}
// running sums over S.cells
template <class C> __device__ __forceinline__ void scan_cells(Shared<C>& S, int cells) {
  constexpr int PER = (C::CELLS + C::NT - 1) / C::NT;
  double v[PER], s = 0.0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PER; ++k) { const int c = threadIdx.x * PER + k; s += c < cells ? S.cells[c] : 0.0; v[k] = s; }
  const double base = block_scan<C>(S.sums, s) - s;
#pragma unroll
  for (int k = 0; k < PER; ++k) { const int c = threadIdx.x * PER + k; if (c < cells) S.cells[c] = base + v[k]; }
  __syncthreads();
}
// the draws [s0, s1) of a row from its running sums, one wavefront each
template <class C, class F> __device__ __forceinline__ void draw(const DrawArgs& A, const Row<F>& R, const Shared<C>& S, int64_t row, int64_t s0, int64_t s1,
                                                                 const Cut<typename F::key>& cut, double min_p) {
  typedef typename F::key K;
  const K neg = neg_key<F>();
  const int lane = threadIdx.x & 63;
  const double Z = S.cells[R.cells - 1], log_z = log(Z);
  for (int64_t s = s0 + (threadIdx.x >> 6); s < s1; s += Shared<C>::NW) {
    double target = A.u[row * A.draws + s] * Z;
    target = target > 0.0 ? target : target == target ? 0.0 : Z;   // (u outside [0, 1): the first or the last kept entry)
    auto first_above = [&](double x, bool or_equal) {
      int a = 0, b = R.cells;
      while (a < b) { const int m = (a + b) >> 1; const double f = S.cells[m]; if (f > x || (or_equal && f >= x)) b = m; else a = m + 1; }
      return a;
    };
    int c = first_above(target, false);
    if (c == R.cells) { c = first_above(Z, true); target = __builtin_inf(); }
    double base = c ? S.cells[c - 1] : 0.0;
    const int64_t i0 = c * R.width();
    int64_t found = -1, last = -1;
    const int steps = R.units * Row<F>::VEC;
    for (int j = 0; j < steps && found < 0; ++j) {
      const int64_t i = i0 + 64 * (int64_t)j + lane;
      double w = 0.0;
      if (i < R.n) {
        const K k = R.key(i);
        if (k > neg && before(cut, k, i)) { w = R.weight(k); w = w < min_p ? 0.0 : w; }
      }
      const double inc = wave_scan(w);
      const u64 hit = __ballot(w > 0.0 && base + inc > target), some = __ballot(w > 0.0);
      if (hit) found = i0 + 64 * (int64_t)j + __ffsll(hit) - 1;
      if (some) last = i0 + 64 * (int64_t)j + 63 - __clzll(some);
      base += __shfl(inc, 63);
    }
    if (found < 0) found = last;                                // (the cell's own sum and this one differ by a rounding)
    if (lane == 0) {
      A.index[row * A.draws + s] = found;
      if (A.logp) A.logp[row * A.draws + s] = R.z(R.key(found)) - log_z;
    }
  }
}
__device__ __forceinline__ void draw_nothing(const DrawArgs& A, int64_t row, int64_t s0, int64_t s1, int threads) {
  for (int64_t s = s0 + threadIdx.x; s < s1; s += threads) {
    A.index[row * A.draws + s] = -1;
    if (A.logp) A.logp[row * A.draws + s] = -__builtin_inf();
  }
}
// All truncations on a list that holds the row's first top_k entries: sorts it and returns how many are kept (the first ones)
template <class C, class F> __device__ __forceinline__ int keep_list(const Row<F>& R, Shared<C>& S, const Settings& p, int count) {
  typedef typename F::key K;
  const int t = threadIdx.x;
  sort_list(S, count);
  int n = p.top_k < count ? (int)p.top_k : count;
  const double w = t < n ? R.weight((K)S.list_key[t]) : 0.0;
  const double sum = block_scan<C>(S.sums, w);
  if (p.top_p < 1.0) {
    __syncthreads();
    if (t == n - 1) S.sums[0] = sum;
    __syncthreads();
    const bool yes = t < n && sum >= p.top_p * S.sums[0];
    n -= (int)block_max<C>(S.red, yes ? (u64)(n - 1 - t) : 0);
  }
  const int heavy = (int)block_max<C>(S.red, t < n && w >= p.min_p ? (u64)(t + 1) : 0);      // (the best one always is)
  return heavy;
}
// the draws from the first n entries of a sorted list: by index, running sums in S.cells, one thread per draw
template <class C, class F> __device__ __forceinline__ void draw_list(const DrawArgs& A, const Row<F>& R, Shared<C>& S, int64_t row, int n) {
  typedef typename F::key K;
  static_assert(C::LIST <= C::CELLS || C::LIST <= Shared<C>::BINS, "running sums of the list");
  const int t = threadIdx.x;
  u64 key = 0; uint32_t idx = 0; int rank = 0;
  if (t < n) { key = S.list_key[t]; idx = S.list_idx[t]; }
  if (t - (t & 63) < n) for (int j = 0; j < n; ++j) rank += S.list_idx[j] < idx;
  __syncthreads();
  if (t < n) { S.list_key[rank] = key; S.list_idx[rank] = idx; }
  __syncthreads();
  const double sum = block_scan<C>(S.sums, t < n ? R.weight((K)S.list_key[t]) : 0.0);
  double* run = reinterpret_cast<double*>(S.bins.hi);
  if (t < n) run[t] = sum;
  __syncthreads();
  const double Z = run[n - 1], log_z = log(Z);
  for (int64_t s = t; s < A.draws; s += C::NT) {
    double target = A.u[row * A.draws + s] * Z;
    target = target > 0.0 ? target : target == target ? 0.0 : Z;
    auto first_above = [&](double x, bool or_equal) {
      int a = 0, b = n;
      while (a < b) { const int m = (a + b) >> 1; const double f = run[m]; if (f > x || (or_equal && f >= x)) b = m; else a = m + 1; }
      return a;
    };
    int j = first_above(target, false);
    if (j == n) j = first_above(Z, true);
    A.index[row * A.draws + s] = (int64_t)S.list_idx[j];
    if (A.logp) A.logp[row * A.draws + s] = R.z((K)S.list_key[j]) - log_z;
  }
}
// The cut of a row whose cells' highest keys are in S.best; R.best is set.  listed > 0: the list holds exactly the kept entries
template <class C, class F> __device__ Cut<typename F::key> cut_of(const Row<F>& R, Shared<C>& S, const Settings& p, u64 kmin, u64 kmax, int& listed) {
  typedef typename F::key K;
  constexpr int VEC = Row<F>::VEC;
  Cut<K> cut{neg_key<F>(), -1};
  listed = 0;
  if (p.top_k > 0) {
    // The top_k-th highest of the cells' best is a lower bound of the cut: only cells that reach it are looked at again.  (kmin: the
    // lowest key of the row where wants_lowest asked for it, else the lowest there can be)
    K lo = (K)kmin;
    clear_bins<false>(S);
    if (p.top_k < R.cells) {
      u64 low = ~0ull;
      for (int c = threadIdx.x; c < R.cells; c += C::NT) { const u64 k = S.best[c]; low = k && k < low ? k : low; }
      low = ~block_max<C>(S.red, ~low);
      const int shift = shift_of<C>(kmax - low);
      for (int c = threadIdx.x; c < R.cells; c += C::NT) if (S.best[c]) atomicAdd(&S.bins.count[(kmax - S.best[c]) >> shift], 1u);
      find_bin<false>(S, 0, 0, 0, (u64)p.top_k, 0.0, 0.0);
      if (S.found[6] >= (u64)p.top_k) {
        const u64 drop = ((S.found[0] + 1) << shift) - 1;       // (to the lowest key of the bin)
        lo = (K)(drop < kmax - low ? kmax - drop : low);
      }
    }
    if (p.top_k <= C::LIST && (lo > (K)kmin || R.n <= C::LIST)) {
      // few: all entries that reach it, if they fit the list -- everything else happens there
      for_cells<true, C::NT>(R, S.best, 0, R.cells, lo, [&](int, const typename F::raw (&r)[VEC], int64_t i, bool) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const K k = F::to_key(r[e]);
          if (k < lo) continue;
          const int at = atomicAdd(&S.listed, 1);
          if (at < C::LIST) { S.list_key[at] = k; S.list_idx[at] = (uint32_t)(i + e); }
        }
      });
      __syncthreads();
      const int count = S.listed;
      if (count <= C::LIST) {
        listed = keep_list<C, F>(R, S, p, count);
        return Cut<K>{(K)S.list_key[listed - 1], (int64_t)S.list_idx[listed - 1]};
      }
    }
    cut = tighter(cut, select<false, C, F>(R, S, lo, (K)kmax, cut, (u64)p.top_k, 0.0));
  }
  if (p.top_p < 1.0) {
    // entries below exp(-56) < 2^-80 of the best one weigh nothing in the bins
    const K floor = key_below<F>(R.best - 56.0 * R.t);
    const K least = cut.key > (K)kmin ? cut.key : (K)kmin;
    cut = tighter(cut, select<true, C, F>(R, S, floor > least ? floor : least, (K)kmax, cut, 0, p.top_p));
  }
  return cut;
}

// ---- kernels --------------------------------------------------------------------------------------------------------------------------
// One workgroup per row: everything, or (draws_here 0: many draws per row) all but the draws, which k_draws makes from memory
template <class C, class F> __global__ __launch_bounds__(C::NT) __attribute__((amdgpu_waves_per_eu(4))) void k_row(DrawArgs A, int draws_here) {
  typedef typename F::key K;
  __shared__ Shared<C> S;
  const int64_t row = blockIdx.x;
  const Settings p = settings_of(A, row);
  Row<F> R = row_of<F>(A, row, p.t);
  const bool lowest = wants_lowest(p, R.cells);
  const typename F::wide low = p.plain ? pass_best<C::NT, true, F>(R, 0, R.cells, S.best, S.cells, false)
                                        : pass_best<C::NT, false, F>(R, 0, R.cells, S.best, nullptr, lowest);
  __syncthreads();
  u64 top = 0;
  for (int c = threadIdx.x; c < R.cells; c += C::NT) top = S.best[c] > top ? S.best[c] : top;
  const u64 kmax = block_max<C>(S.red, top);
  Cut<K> cut{neg_key<F>(), -1};
  if (kmax != 0) {
    R.best = F::of_key((K)kmax);
    if (!p.plain) {
      const u64 kmin = lowest ? ~block_max<C>(S.red, ~(u64)F::key_of_wide(low)) : (u64)neg_key<F>() + 1;
      int listed;
      cut = cut_of<C, F>(R, S, p, kmin, kmax, listed);
      if (listed && draws_here) { draw_list<C, F>(A, R, S, row, listed); return; }
      __syncthreads();                                          // (the cells take the bins' place)
      pass_weights<C::NT, F>(R, S.best, 0, R.cells, cut, p.min_p, S.cells);
    } else if (draws_here) {
      for (int c = threadIdx.x; c < R.cells; c += C::NT) S.cells[c] *= S.best[c] ? R.weight((K)S.best[c]) : 0.0;
    }
  }
  if (draws_here) {
    if (kmax == 0) { draw_nothing(A, row, 0, A.draws, C::NT); return; }
    scan_cells(S, R.cells);
    draw<C, F>(A, R, S, row, 0, A.draws, cut, p.min_p);
    return;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < R.cells; c += C::NT) { A.keys[row * A.max_cells + c] = S.best[c]; A.sums[row * A.max_cells + c] = S.cells[c]; }
  if (threadIdx.x == 0) { A.state[row * STATE] = (u64)cut.key; A.state[row * STATE + 1] = (u64)cut.idx; }
}

// The same over several launches, for a few long rows whose cells are dealt to `groups` workgroups each.  First: the cells' highest
// keys, the lowest key of each group, and -- nothing truncated -- the cells' weights
template <class F> __global__ __launch_bounds__(256) void k_best(DrawArgs A, int groups) {
  __shared__ u64 red[4];
  const int64_t row = blockIdx.x / groups;
  const int g = blockIdx.x % groups;
  const Settings p = settings_of(A, row);
  const Row<F> R = row_of<F>(A, row, p.t);
  const int c0 = (int)((int64_t)R.cells * g / groups), c1 = (int)((int64_t)R.cells * (g + 1) / groups);
  const bool lowest = wants_lowest(p, R.cells);
  u64* keys = A.keys + row * A.max_cells;
  const typename F::wide low = p.plain ? pass_best<256, true, F>(R, c0, c1, keys, A.sums + row * A.max_cells, false)
                                        : pass_best<256, false, F>(R, c0, c1, keys, nullptr, lowest);
  const u64 kmin = lowest ? ~block_max<Short>(red, ~(u64)F::key_of_wide(low)) : (u64)neg_key<F>() + 1;
  if (threadIdx.x == 0) {
    A.lows[row * groups + g] = kmin;
    if (g == 0) { A.state[row * STATE] = (u64)neg_key<F>(); A.state[row * STATE + 1] = (u64)-1; }
  }
}
// ... the cut (only where one may be asked for)
template <class F> __global__ __launch_bounds__(Long::NT) __attribute__((amdgpu_waves_per_eu(4))) void k_cut(DrawArgs A, int groups) {
  typedef typename F::key K;
  __shared__ Shared<Long> S;
  const int64_t row = blockIdx.x;
  const Settings p = settings_of(A, row);
  Row<F> R = row_of<F>(A, row, p.t);
  u64 top = 0, low = ~0ull;
  for (int c = threadIdx.x; c < R.cells; c += Long::NT) { const u64 k = A.keys[row * A.max_cells + c]; S.best[c] = k; top = k > top ? k : top; }
  for (int g = threadIdx.x; g < groups; g += Long::NT) { const u64 k = A.lows[row * groups + g]; low = k < low ? k : low; }
  const u64 kmax = block_max<Long>(S.red, top), kmin = ~block_max<Long>(S.red, ~low);
  if (kmax == 0) return;
  R.best = F::of_key((K)kmax);
  int listed;
  const Cut<K> cut = cut_of<Long, F>(R, S, p, kmin, kmax, listed);
  if (threadIdx.x == 0) { A.state[row * STATE] = (u64)cut.key; A.state[row * STATE + 1] = (u64)cut.idx; }
}
template <int THREADS> __device__ __forceinline__ u64 best_of_row(const DrawArgs& A, int64_t row, int cells, u64 (&red)[THREADS / 64]) {
  u64 top = 0;
  for (int c = threadIdx.x; c < cells; c += THREADS) { const u64 k = A.keys[row * A.max_cells + c]; top = k > top ? k : top; }
  if constexpr (THREADS == Short::NT) return block_max<Short>(red, top); else return block_max<Long>(red, top);
}
// ... the cells' kept weights
template <class F> __global__ __launch_bounds__(256) void k_weights(DrawArgs A, int groups) {
  typedef typename F::key K;
  __shared__ u64 red[4];
  const int64_t row = blockIdx.x / groups;
  const int g = blockIdx.x % groups;
  const Settings p = settings_of(A, row);
  Row<F> R = row_of<F>(A, row, p.t);
  const u64 kmax = best_of_row<256>(A, row, R.cells, red);
  if (p.plain || kmax == 0) return;
  R.best = F::of_key((K)kmax);
  const Cut<K> cut{(K)A.state[row * STATE], (int64_t)A.state[row * STATE + 1]};
  const int c0 = (int)((int64_t)R.cells * g / groups), c1 = (int)((int64_t)R.cells * (g + 1) / groups);
  pass_weights<256, F>(R, A.keys + row * A.max_cells, c0, c1, cut, p.min_p, A.sums + row * A.max_cells);
}
// ... and the draws, `per` of a row in every workgroup
template <class F> __global__ __launch_bounds__(Long::NT) void k_draws(DrawArgs A, int blocks, int per) {
  typedef typename F::key K;
  __shared__ Shared<Long> S;
  const int64_t row = blockIdx.x / blocks;
  const int64_t s0 = (int64_t)(blockIdx.x % blocks) * per, s1 = s0 + per < A.draws ? s0 + per : A.draws;
  const Settings p = settings_of(A, row);
  Row<F> R = row_of<F>(A, row, p.t);
  const u64 kmax = best_of_row<Long::NT>(A, row, R.cells, S.red);
  if (kmax == 0) { draw_nothing(A, row, s0, s1, Long::NT); return; }
  R.best = F::of_key((K)kmax);
  const Cut<K> cut{(K)A.state[row * STATE], (int64_t)A.state[row * STATE + 1]};
  for (int c = threadIdx.x; c < R.cells; c += Long::NT) {
    double w = A.sums[row * A.max_cells + c];
    if (p.plain) { const u64 k = A.keys[row * A.max_cells + c]; w *= k ? R.weight((K)k) : 0.0; }
    S.cells[c] = w;
  }
  scan_cells(S, R.cells);
  draw<Long, F>(A, R, S, row, s0, s1, cut, p.min_p);
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------
// How a call runs: cells of a row, workgroups per row (0: one workgroup does a whole row), draws apart from the rest or not
struct Plan { int units, max_cells, groups; bool short_rows, draws_here; };
Plan plan_of(int type, int64_t rows, int64_t cols, int64_t draws) {
  Plan p;
  const int64_t unit = 64 * (type == 0 ? 2 : type == 1 ? 4 : 8);
  p.units = (int)((cols + unit * MAX_CELLS - 1) / (unit * MAX_CELLS));
  p.max_cells = (int)((cols + unit * p.units - 1) / (unit * p.units));
  p.short_rows = p.max_cells <= (rows >= 512 ? 64 : 16);
  p.groups = (!p.short_rows && p.max_cells >= 64 && rows <= 64) ? (int)std::min<int64_t>(p.max_cells / 16, std::max<int64_t>(1, 512 / rows)) : 0;
  p.draws_here = p.groups == 0 && draws <= 64;
  return p;
}
int64_t scratch_of(const Plan& p, int64_t rows) { return p.draws_here ? 0 : rows * (2 * (int64_t)p.max_cells + p.groups + STATE); }

template <class F> void launch(DrawArgs& A, const Plan& p, int64_t rows, hipStream_t st) {
  if (p.groups == 0) {
    if (p.short_rows) hipLaunchKernelGGL((k_row<Short, F>), dim3((unsigned)rows), dim3(Short::NT), 0, st, A, p.draws_here ? 1 : 0);
    else hipLaunchKernelGGL((k_row<Long, F>), dim3((unsigned)rows), dim3(Long::NT), 0, st, A, p.draws_here ? 1 : 0);
    if (p.draws_here) return;
  } else {
    const dim3 grid((unsigned)(rows * p.groups));
    hipLaunchKernelGGL(k_best<F>, grid, dim3(256), 0, st, A, p.groups);
    const bool cuts = A.temperature.p || A.temperature.v == 0.0 || A.top_k.p || A.top_k.v > 0 || A.top_p.p || A.top_p.v < 1.0;
    if (cuts) hipLaunchKernelGGL(k_cut<F>, dim3((unsigned)rows), dim3(Long::NT), 0, st, A, p.groups);
    if (cuts || A.min_p.p || A.min_p.v > 0.0) hipLaunchKernelGGL(k_weights<F>, grid, dim3(256), 0, st, A, p.groups);
  }
  // a wavefront makes one draw at a time: two each, more where that fills the chip anyway
  const int per = (int)std::max<int64_t>(16, (A.draws * rows / 1024 + 15) / 16 * 16);
  const int blocks = (int)((A.draws + per - 1) / per);
  hipLaunchKernelGGL(k_draws<F>, dim3((unsigned)(rows * blocks)), dim3(Long::NT), 0, st, A, blocks, per);
}
}  // namespace

extern "C" int64_t pgm_draw_scratch_doubles(int type, int64_t rows, int64_t cols, int64_t draws) {
  if (type < 0 || type > 3 || rows < 1 || cols < 1 || cols >= MAX_COLS || draws < 1) return 0;
  return scratch_of(plan_of(type, rows, cols, draws), rows);
}

extern "C" int pgm_draw_indices(const void* logits, int type, int64_t rows, int64_t cols, int64_t row_stride, int64_t col_stride,
                                const int64_t* lengths, const double* u, int64_t draws,
                                double temperature, const double* temperature_row, int64_t top_k, const int64_t* top_k_row,
                                double top_p, const double* top_p_row, double min_p, const double* min_p_row,
                                int64_t* index, double* logp, double* scratch, int64_t scratch_doubles, void* stream) {
  if (!logits) return -1;
  if (type < 0 || type > 3) return -2;
  if (rows < 1 || rows > 0x7fffffff) return -3;
  if (cols < 1 || cols >= MAX_COLS) return -4;
  if (row_stride < 0) return -5;
  if (col_stride < 0) return -6;
  if (!u) return -8;
  if (draws < 1) return -9;
  if (!temperature_row && !(temperature >= 0.0 && temperature <= 1e300)) return -10;
  if (!top_k_row && top_k < 0) return -12;
  if (!top_p_row && !(top_p >= 0.0 && top_p <= 1.0)) return -14;
  if (!min_p_row && !(min_p >= 0.0 && min_p <= 1.0)) return -16;
  if (!index) return -18;
  if (draws > 0x7fffffff || rows * draws > ((int64_t)1 << 40)) return -9;
  const Plan p = plan_of(type, rows, cols, draws);
  const int64_t need = scratch_of(p, rows);
  if (need > 0 && !scratch) return -20;
  if (need > scratch_doubles) return -21;
  DrawArgs A{logits, row_stride, col_stride, cols, lengths, u, draws, {temperature, temperature_row}, {top_p, top_p_row}, {min_p, min_p_row},
             {top_k, top_k_row}, index, logp, p.units, p.max_cells, nullptr, nullptr, nullptr, nullptr};
  if (need > 0) {
    A.keys = reinterpret_cast<u64*>(scratch);
    A.sums = scratch + rows * p.max_cells;
    A.lows = reinterpret_cast<u64*>(scratch + 2 * rows * p.max_cells);
    A.state = A.lows + rows * p.groups;
  }
  hipStream_t st = (hipStream_t)stream;
  if (type == 0) launch<F64>(A, p, rows, st);
  else if (type == 1) launch<F32>(A, p, rows, st);
  else if (type == 2) launch<Half<0>>(A, p, rows, st);
  else launch<Half<1>>(A, p, rows, st);
  return hipGetLastError() == hipSuccess ? 0 : -99;
}
