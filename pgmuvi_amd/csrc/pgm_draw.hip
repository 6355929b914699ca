// pgm_draw.hip -- draws from rows of log-weights (the frequency posterior of a periodogram), with tempering and truncation.
//
// Row l of `cols` log-weights, best value m:   z_i = (l_i - m) / T,   w_i = exp z_i  (one for the best, zero for -inf and NaN).
// In the order (l descending, i ascending):    A = the first top_k entries,   P = the shortest beginning of A that holds at least
// top_p of A's weight,   kept = the entries of P with w_i >= min_p.   Z = sum of the kept weights, and a number u in [0, 1) draws
// the first kept i, in the order of i, whose running sum F(i) exceeds u Z.  log p = z_i - log Z.
//
// All three truncations keep a beginning of ONE order, so the kept set is "everything before a cut (value, index)" and w >= min_p.
// The first pass finds the highest value of every cell of 256 or 512 neighbouring entries; every later pass looks only at the cells
// that reach what it looks for.  The cut is found by histograms, 512 to 2048 bins per pass over the range of values that still
// matters, until a bin is small enough to sort: counts for top_k; weights for top_p, held in two integer words (2^-40 and 2^-80
// steps: sums of integers do not depend on the order of the LDS atomics, and 80 bits are more than the fp64 sums they are compared
// with).  Equal values are split by index the same way.  The running sums are fp64, cell by cell in a fixed order: the same call
// gives the same draws.
//
// What bounds it (MI355X; a copy moves 4.9 TB/s, so that reading a row once is the floor of all but the smallest calls).
//   4096 x 51200 fp32, top_k 50 and top_p 0.9, one draw: 206 us, 4.1 TB/s of the one pass that reads everything (171 us at the
//     copy's rate); the list and the draw overlap with other rows' loads.  Not truncated: 280 us, the exponentials of 2.1e8 entries.
//   512 x 25600 fp64, top_p 0.95, four draws: 91 us against 21 for the bytes.  A row is one workgroup and all of them are on the chip at
//     once, two to a CU, so that the call takes as long as its slowest row.  Stamped (which adds 5 us), a row takes 46 us where a few
//     peaks hold the 0.95 and 95 where noise does, 67 in the mean: highest values 13 us, waiting for each other and clearing the bins 4,
//     bins 23 (exponential and three LDS atomics an entry: count and two words) and 5 of waiting, the bin 3, the cut's entries and the
//     cells' weights 9 and 2 of waiting, the sort 1, joining the list to the cells 3, scan and draws 4.  min_p or nothing instead of
//     top_p: 32 us.
//   1 x 204800 fp64, min_p 0.02, 1000 draws: 15 us on the GPU (calls back to back in a graph), three launches one after the other; their
//     bytes take 0.3.
//   Short calls (1 x 1113 fp64, 8 draws): 8 us, one launch whose phases wait for each other.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>
#include <algorithm>
#include "../../include/pgmuvi_hip.h"
#include "pgm_exp.h"

namespace {

typedef unsigned long long u64;
constexpr int LOAD = 16, CB = 2;                                // bytes of a lane's load; cells a wavefront works on at a time
constexpr int MAX_CELLS = 1024;                                 // of a row (longer rows: wider cells)
constexpr int64_t MAX_COLS = 1 << 24;                           // 2^24 weights of at most one, in steps of 2^-40, fit 64 bits
constexpr int64_t MAX_ROWS = 1 << 23;                           // 512 threads a row: less than 2^32 of a launch
constexpr int64_t EVERY = INT64_MAX;
constexpr double INF = __builtin_inf();

// ---- types of the log-weights.  `wide`: what maxima are formed in; U: loads of a lane that make up a cell (the wavefront's reduction
// for a cell costs ~35 instructions: over two loads of two fp64 or four fp32 entries each, over one of eight 16-bit ones)
// (larger: a is never a signalling NaN, b may be one, which the hardware's maximum would return quiet instead of the other operand --
// compiled with b made quiet in the form of two operands, but not in that of three, hence the canonical b of fp32 and bf16, whose
// bits are loaded as they are: a quiet NaN loses)
struct F64 {
  typedef double raw, wide;
  static constexpr int U = 2;
  static constexpr raw absent() { return -__builtin_inf(); }
  static __device__ __forceinline__ wide widen(raw x) { return x; }
  static __device__ __forceinline__ wide larger(wide a, wide b) { return __builtin_fmax(a, b); }
};
struct F32 {
  typedef float raw, wide;
  static constexpr int U = 2;
  static constexpr raw absent() { return -__builtin_inff(); }
  static __device__ __forceinline__ wide widen(raw x) { return x; }
  static __device__ __forceinline__ wide larger(wide a, wide b) { return __builtin_fmaxf(a, __builtin_canonicalizef(b)); }
};
template <int F16BIT> struct Half {                              // bf16 (0) and fp16 (1)
  typedef uint16_t raw; typedef float wide;
  static constexpr int U = 1;
  static constexpr raw absent() { return F16BIT ? 0xfc00u : 0xff80u; }
  static __device__ __forceinline__ wide widen(raw b) {
    if constexpr (F16BIT) { __half_raw r; r.x = b; return __half2float(__half(r)); }
    else return __uint_as_float((uint32_t)b << 16);
  }
  static __device__ __forceinline__ wide larger(wide a, wide b) { return __builtin_fmaxf(a, F16BIT ? b : __builtin_canonicalizef(b)); }
};
// a bound not above v, in the type comparisons are cheap in
__device__ __forceinline__ void bound_below(double v, double& w) { w = v; }
__device__ __forceinline__ void bound_below(double v, float& w) { w = (float)v; w -= fabsf(w) * 2.4e-7f + 1e-37f; }
// ordered bit patterns of the values (-0 as +0)
__device__ __forceinline__ u64 key_of(double x) { const u64 b = (u64)__double_as_longlong(x + 0.0); return (b >> 63) ? ~b : b | (1ull << 63); }
__device__ __forceinline__ double of_key(u64 k) { return __longlong_as_double((long long)((k >> 63) ? k & ~(1ull << 63) : ~k)); }

struct Param { double v; const double* p; };                    // one number for every row, or one per row
struct ParamI { int64_t v; const int64_t* p; };
struct CutState { double value; int64_t idx; };
constexpr int64_t DRAWN = -2;                                   // (a cut's idx: the row's draws have been made)
constexpr int TABLE_BINS = 4096, TABLE_LIST = 1024;             // (those of the build All below)
struct Table { u64 hi[TABLE_BINS], lo[TABLE_BINS]; double value[TABLE_LIST]; uint32_t count[TABLE_BINS], idx[TABLE_LIST]; int listed, pad; };
struct DrawArgs {
  const void* logits; int64_t row_stride, col_stride, cols;
  const int64_t* lengths;                                       // entries of each row, or null: cols
  const double* u; int64_t draws;
  Param temperature, top_p, min_p; ParamI top_k;
  int64_t* index; double* logp;
  int mult, max_cells;                                          // loads per lane and cell over U, cells of a full row
  double *best, *sums, *lows; CutState* cut; Table* tables;     // rows whose passes are launches of their own: [row][max_cells] twice, [row][groups], [row], [row][2]
  double* lots;                                                 // [row][64 mult max_cells], where many draws share them
};

// kept: values above the cut's, and equal ones up to its index
struct Cut {
  double value; int64_t idx;
  __device__ __forceinline__ bool keeps(double l, int64_t i) const { return l > value || (l == value && i <= idx); }
};
__device__ __forceinline__ Cut tighter(const Cut& a, const Cut& b) {
  if (a.value != b.value) return a.value > b.value ? a : b;
  return a.idx < b.idx ? a : b;
}

// ---- wavefront and workgroup reductions --------------------------------------------------------------------------------------
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
template <class V> __device__ __forceinline__ V wave_scan(V v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) { const V o = __shfl_up(v, s); if (lane >= s) v += o; }
  return v;
}
template <int THREADS> __device__ __forceinline__ double block_max(double* red, double v) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) v = __builtin_fmax(v, red[w]);
  return v;
}
template <int THREADS> __device__ __forceinline__ double block_min(double* red, double v) { return -block_max<THREADS>(red, -v); }
// running sum over the workgroup's threads, in thread order
template <int THREADS> __device__ __forceinline__ double block_scan(double* red, double v) {
  const double inc = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = inc;
  __syncthreads();
  double base = 0.0;
  for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) base += red[w];
  return base + inc;
}
__device__ __forceinline__ double mass_of(u64 hi, u64 lo) { return (double)hi * 0x1p-40 + (double)lo * 0x1p-80; }

// ---- one row ----------------------------------------------------------------------------------------------------------------
template <class F> struct Row {
  typedef typename F::raw raw;
  static constexpr int U = F::U, VEC = LOAD / (int)sizeof(raw), UNIT = 64 * VEC;       // entries of one load of a lane, of a wavefront
  // (global memory by type: through a generic pointer the loads would count as LDS accesses as well, and every wait for the LDS would
  // hold up the loads in flight)
  typedef const __attribute__((address_space(1))) raw* Global;
  typedef raw Lot __attribute__((ext_vector_type(VEC), aligned(sizeof(raw))));
  Global x; int64_t stride, n;
  int mult, cells;
  double best, t, per_t;                                        // highest value, temperature, 1 / temperature
  __device__ __forceinline__ int64_t width() const { return (int64_t)mult * (U * UNIT); }
  __device__ __forceinline__ double value(int64_t i) const { return (double)F::widen(x[i * stride]); }
  __device__ __forceinline__ double z(double l) const { return l == best ? 0.0 : (l - best) / t; }
  // (the product with 1 / T, one instruction against the ten or so of z's quotient: one rounding more, 2^-53 |z| relative to the weight.
  // The log-probabilities are z's.  Where the best value is infinite only infinite ones are kept: their difference, a NaN, is clamped
  // to zero here)
  __device__ __forceinline__ double weight(double l) const { return exp_neg(__builtin_fmin((l - best) * per_t, 0.0)); }
  // this lane's entries of the group of U loads number g: load q's entry e is number first(g) + q UNIT + e; behind the end -inf
  __device__ __forceinline__ int64_t first(int64_t g) const { return g * (U * UNIT) + (threadIdx.x & 63) * VEC; }
  __device__ __forceinline__ void load_whole(int64_t g, raw (&r)[U][VEC]) const {
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const Lot v = *reinterpret_cast<const __attribute__((address_space(1))) Lot*>(x + first(g) + q * UNIT);
#pragma unroll
      for (int e = 0; e < VEC; ++e) r[q][e] = v[e];
    }
  }
  __device__ __forceinline__ void load_part(int64_t g, raw (&r)[U][VEC]) const {
#pragma unroll
    for (int q = 0; q < U; ++q)
#pragma unroll
      for (int e = 0; e < VEC; ++e) { const int64_t i = first(g) + q * UNIT + e; r[q][e] = i < n ? x[i * stride] : F::absent(); }
  }
};

// Builds of a row's code: 8 wavefronts for a row, 4 where there are rows enough to fill the chip with such workgroups (their phases
// overlap better), one with small tables for very short rows (no barriers); All: the launches that share a long row's cut
struct Long { static constexpr int NT = 512, BITS = 11, CELLS = MAX_CELLS, LIST = 512; };
struct Many { static constexpr int NT = 256, BITS = 10, CELLS = MAX_CELLS, LIST = 256; };
struct Tiny { static constexpr int NT = 64, BITS = 8, CELLS = 8, LIST = 64; };
struct All { static constexpr int NT = 1024, BITS = 12, CELLS = MAX_CELLS, LIST = 1024; };

template <class C> struct Shared {
  static constexpr int BINS = 1 << C::BITS, NW = C::NT / 64;
  union {
    struct { uint32_t count[BINS]; u64 hi[BINS], lo[BINS]; } bins;
    double cells[C::CELLS];                                     // weights of the cells, then their running sums
  };
  double best[C::CELLS];                                        // highest value of every cell
  double list_value[C::LIST]; uint32_t list_idx[C::LIST];
  double red[NW];
  u64 part[3][NW], found[7];
  int listed;
};

// f(cell, this lane's entries, number of its first one, last group of the cell?) for the cells c0 <= c < c1 -- with SEEN only those
// whose highest value is at least `lo`: a wavefront per cell.  The next CB cells' loads are in flight while the present ones are
// worked on; the row's end, strided rows and very long ones go one group of loads after the other.
template <bool SEEN, int THREADS, class F, class Fn> __device__ __forceinline__ void for_cells(const Row<F>& R, const double* best, int c0, int c1, double lo, Fn f) {
  typedef typename F::raw raw;
  constexpr int NW = THREADS / 64, VEC = Row<F>::VEC, U = F::U, STEP = NW * CB;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int full = c0;                                                // the cells up to here are one whole group of loads
  if (R.mult == 1 && R.stride == 1) {
    const int whole = (int)(R.n / (U * Row<F>::UNIT));
    full = whole < c1 ? whole : c1;
    full = full > c0 ? full : c0;
  }
  raw next[CB][U][VEC];
  auto wanted = [&](int cc) { return !SEEN || best[cc] >= lo; };
  auto fetch = [&](int c) {
#pragma unroll
    for (int s = 0; s < CB; ++s) if (c + s * NW < full && wanted(c + s * NW)) R.load_whole(c + s * NW, next[s]);
  };
  // (two loops: in one, the compiler's wait for the loads of the slow kind would hold up those in flight as well)
  int c = c0 + wave;
  if (c < full) fetch(c);
  for (; c < full; c += STEP) {
    raw r[CB][U][VEC];
    __builtin_memcpy(r, next, sizeof(r));
    if (c + STEP < full) fetch(c + STEP);
#pragma unroll
    for (int s = 0; s < CB; ++s)
      if (c + s * NW < full && wanted(c + s * NW)) f(c + s * NW, r[s], R.first(c + s * NW), true);
  }
  for (c = full + wave; c < c1; c += NW) {
    if (!wanted(c)) continue;
    for (int j = 0; j < R.mult; ++j) {
      raw r[U][VEC];
      const int64_t g = (int64_t)c * R.mult + j;
      if (R.stride == 1 && (g + 1) * (U * Row<F>::UNIT) <= R.n) R.load_whole(g, r); else R.load_part(g, r);
      f(c, r, R.first(g), j == R.mult - 1);
    }
  }
}
// g(value, number) for this lane's entries of a group, two at a time in a loop (unrolled, the exponentials of all of them fill the
// registers several times over)
template <class F, class Fn> __device__ __forceinline__ void each(const typename F::raw (&r)[F::U][Row<F>::VEC], int64_t i0, Fn g) {
  constexpr int VEC = Row<F>::VEC, M = F::U * VEC;
  typename F::wide v[M];
#pragma unroll
  for (int m = 0; m < M; ++m) v[m] = F::widen(r[m / VEC][m % VEC]);
#pragma unroll 1
  for (int m = 0; m < M; m += 2) {
    const int64_t i = i0 + (m / VEC) * Row<F>::UNIT + m % VEC;
    g(v[0], i);
    g(v[1], i + 1);
#pragma unroll
    for (int k = 0; k + 2 < M; ++k) v[k] = v[k + 2];
  }
}

// ---- the cut -------------------------------------------------------------------------------------------------------------------
// The bin that holds it: `want` entries, or (WEIGHTED) `target` of weight -- `share` of all that the bins hold on the first pass,
// where target < 0 asks for it.  found: bin, entries before it, in it, hi / lo before it, target, entries in all bins.  There is
// always exactly one: the goal is at most what the bins hold, and the running sums of integers never decrease
template <bool WEIGHTED, class C> __device__ __forceinline__ void find_bin(Shared<C>& S, u64 before_n, u64 before_hi, u64 before_lo, u64 want, double share, double target) {
  constexpr int PER = Shared<C>::BINS / C::NT, NW = C::NT / 64;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, b0 = t * PER;
  __syncthreads();
  u64 n = 0, hi = 0, lo = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) { n += S.bins.count[b0 + k]; if (WEIGHTED) { hi += S.bins.hi[b0 + k]; lo += S.bins.lo[b0 + k]; } }
  u64 sn = wave_scan((uint32_t)n), shi = WEIGHTED ? wave_scan(hi) : 0, slo = WEIGHTED ? wave_scan(lo) : 0;
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
    target = target < most ? target : most;
  } else if (want > before_n + all) want = before_n + all;
  auto reached = [&](u64 an, u64 ahi, u64 alo) { return WEIGHTED ? mass_of(before_hi + ahi, before_lo + alo) >= target : before_n + an >= want; };
  u64 an = sn - n, ahi = shi - hi, alo = slo - lo;
  if (n && !reached(an, ahi, alo) && reached(sn, shi, slo)) {
    int b = b0;
    for (; b < b0 + PER - 1; ++b) {
      const u64 c = S.bins.count[b], h = WEIGHTED ? S.bins.hi[b] : 0, l = WEIGHTED ? S.bins.lo[b] : 0;
      if (c && reached(an + c, ahi + h, alo + l)) break;
      an += c; ahi += h; alo += l;
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
  double value = 0.0; uint32_t idx = 0; int rank = 0, ties = 0;
  if (t < count) { value = S.list_value[t]; idx = S.list_idx[t]; }
  if (t - (t & 63) < count) {
    for (int j = 0; j < count; ++j) { const double v = S.list_value[j]; rank += v > value; ties += v == value; }
    if (__any(t < count && ties > 1))
      for (int j = 0; j < count; ++j) rank += S.list_value[j] == value && S.list_idx[j] < idx;
  }
  __syncthreads();
  if (t < count) { S.list_value[rank] = value; S.list_idx[rank] = idx; }
  __syncthreads();
}
// The same where the bins hold the counts of the listed entries (bin(value) of theirs): by bins first, then each entry counts what is
// ahead of it in its own bin (512 entries of a 16-bit type, many of them equal: 21 -> 4 us)
template <class C, class Bin> __device__ __forceinline__ void sort_list_by_bins(Shared<C>& S, int count, Bin bin) {
  constexpr int PER = Shared<C>::BINS / C::NT;
  uint32_t* start = reinterpret_cast<uint32_t*>(S.bins.hi);      // entries before each bin
  uint32_t* taken = reinterpret_cast<uint32_t*>(S.bins.lo);
  const int t = threadIdx.x, b0 = t * PER;
  __syncthreads();
  uint32_t n = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) n += S.bins.count[b0 + k];
  uint32_t before = (uint32_t)block_scan<C::NT>(S.red, (double)n) - n;
#pragma unroll
  for (int k = 0; k < PER; ++k) { start[b0 + k] = before; taken[b0 + k] = 0; before += S.bins.count[b0 + k]; }
  double value = 0.0; uint32_t idx = 0; int b = 0;
  if (t < count) { value = S.list_value[t]; idx = S.list_idx[t]; b = bin(value); }
  __syncthreads();
  if (t < count) { const uint32_t at = start[b] + atomicAdd(&taken[b], 1u); S.list_value[at] = value; S.list_idx[at] = idx; }
  __syncthreads();
  int rank = 0;
  if (t < count) {                                              // (the entry that came to place t)
    value = S.list_value[t]; idx = S.list_idx[t]; b = bin(value);
    const int from = (int)start[b], to = from + (int)S.bins.count[b];
    rank = from;
    for (int j = from; j < to; ++j) { const double v = S.list_value[j]; rank += v > value || (v == value && S.list_idx[j] < idx); }
  }
  __syncthreads();
  if (t < count) { S.list_value[rank] = value; S.list_idx[rank] = idx; }
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

struct Even {                                                   // the first bins: the range of values in equal parts
  double best, scale; bool good; int bins;
  __device__ __forceinline__ Even(double best_, double lo, int bins_) : best(best_), scale(bins_ / (best_ - lo)), bins(bins_) { good = best - lo > 0.0 && best - lo < 1e300 && scale < 1e300; }
  __device__ __forceinline__ int bin(double l) const { const int b = (int)((best - l) * scale); return b < bins ? b : bins - 1; }
};
// The cut behind the first `want` entries of what `have` keeps (WEIGHTED: behind the shortest beginning with `share` of its weight);
// lo <= every value that can matter.  The first bins divide the range of values evenly, the later ones (where a bin held too many
// to sort) the range of the ordered bit patterns of the bin's values, at least a factor BINS / 2 narrower each time.
// SEEDED: the first bins, and the list of their bin's entries if it is short enough, have been made by other launches
// `summed` (WEIGHTED; may be null): where the first bin is short enough, the pass that collects its entries also forms the cells' kept
// weights (S.cells; of entries with a weight of at least min_p), and says so
template <bool WEIGHTED, bool SEEDED, class C, class F> __device__ __forceinline__ Cut select(const Row<F>& R, Shared<C>& S, double lo, Cut have, u64 want, double share,
                                                                             double min_p = 0.0, bool* summed = nullptr) {
  typedef typename F::raw raw;
  typedef typename F::wide wide;
  constexpr int VEC = Row<F>::VEC, U = F::U, BINS = Shared<C>::BINS;
  u64 bn = 0, bhi = 0, blo = 0;
  double target = -1.0;
  bool first = true;
  lo = lo > have.value ? lo : have.value;
  const Even parts(R.best, lo, BINS);
  bool even = parts.good;
  u64 khi = key_of(R.best), klo = key_of(lo);                   // the later bins' range
  for (;;) {
    const int shift = shift_of<C>(khi - klo);
    wide quick; bound_below(lo, quick);
    // all the entries in the range, f(value, index, bin)
    auto entries = [&](auto f) {
      for_cells<true, C::NT>(R, S.best, 0, R.cells, lo, [&](int, const raw (&r)[U][VEC], int64_t i0, bool) {
        each<F>(r, i0, [&](wide v, int64_t i) {
          const double l = (double)v;
          if (v < quick || !(l >= lo) || !have.keeps(l, i)) return;
          if (even) f(l, i, parts.bin(l));
          else { const u64 k = key_of(l); if (k <= khi) f(l, i, (int)((khi - k) >> shift)); }
        });
      });
    };
    const bool seeded = SEEDED && first && even;
    if (!seeded) {
      clear_bins<WEIGHTED>(S);
      entries([&](double l, int64_t, int b) {
        atomicAdd(&S.bins.count[b], 1u);
        if (WEIGHTED) add_weight(S, b, R.weight(l));
      });
    }
    find_bin<WEIGHTED>(S, bn, bhi, blo, want, share, target);
    if (!WEIGHTED && first && S.found[6] <= want) return Cut{lo, EVERY};          // (all of them)
    first = false;
    const int bin = (int)S.found[0];
    const u64 in_bin = S.found[2];
    bn = S.found[1]; bhi = S.found[3]; blo = S.found[4]; target = __longlong_as_double((long long)S.found[5]);
    if (in_bin <= (u64)C::LIST) {
      // few enough to sort: the bin's entries in the cut's order, then the first that reaches the goal
      const bool sums = WEIGHTED && !SEEDED && summed && even;
      if (sums) {
        // (no entry of this bin or a higher one is below this; the bins' place is free)
        const double least = bin + 1 < BINS ? R.best - (bin + 1.001) / parts.scale : lo;
        for (int c = threadIdx.x; c < R.cells; c += C::NT) if (!(S.best[c] >= least)) S.cells[c] = 0.0;
        double w = 0.0;
        for_cells<true, C::NT>(R, S.best, 0, R.cells, least, [&](int c, const raw (&r)[U][VEC], int64_t i0, bool last) {
          each<F>(r, i0, [&](wide v, int64_t i) {
            const double l = (double)v;
            if (!(l >= lo) || !have.keeps(l, i)) return;
            const int b = parts.bin(l);
            if (b < bin) { const double x = R.weight(l); w += x < min_p ? 0.0 : x; }
            if (b == bin) { const int at = atomicAdd(&S.listed, 1); S.list_value[at] = l; S.list_idx[at] = (uint32_t)i; }
          });
          if (!last) return;
          const double total = wave_sum(w);
          w = 0.0;
          if ((threadIdx.x & 63) == 0) S.cells[c] = total;
        });
      } else if (!seeded)
        entries([&](double l, int64_t i, int b) {
          if (b != bin) return;
          const int at = atomicAdd(&S.listed, 1);
          S.list_value[at] = l; S.list_idx[at] = (uint32_t)i;
        });
      const int count = (int)in_bin, t = threadIdx.x;
      sort_list(S, count);
      int at = (int)(want - bn) - 1;
      if (WEIGHTED) {
        const double sum = block_scan<C::NT>(S.red, t < count ? R.weight(S.list_value[t]) : 0.0);
        at = (int)block_min<C::NT>(S.red, t < count && mass_of(bhi, blo) + sum >= target ? (double)t : (double)(count - 1));
      }
      const Cut cut{S.list_value[at], (int64_t)S.list_idx[at]};
      if (sums) {
        // the kept entries of the bin join their cells, one thread per cell and in the list's order
        __syncthreads();
        if (t < count) {
          const double w = R.weight(S.list_value[t]);
          S.list_value[t] = t <= at && w >= min_p ? w : 0.0;
          S.list_idx[t] = (uint32_t)((int64_t)S.list_idx[t] / R.width());
        }
        __syncthreads();
        for (int c = t; c < R.cells; c += C::NT) {
          double w = S.cells[c];
          for (int j = 0; j <= at; ++j) w += S.list_idx[j] == (uint32_t)c ? S.list_value[j] : 0.0;
          S.cells[c] = w;
        }
        *summed = true;
      }
      return cut;
    }
    double high = -INF, low = INF;                              // the range of the bin's values
    entries([&](double l, int64_t, int b) { if (b == bin) { high = l > high ? l : high; low = l < low ? l : low; } });
    high = block_max<C::NT>(S.red, high); low = block_min<C::NT>(S.red, low);
    if (!WEIGHTED && bn + in_bin == want) return Cut{low, EVERY};
    if (high == low) {                                          // many equal values: the first m of them by index
      u64 m = WEIGHTED ? 1 : want - bn;
      if (WEIGHTED) {
        const double w = R.weight(low), above = mass_of(bhi, blo);
        const double guess = ceil((target - above) / w);
        m = guess >= (double)in_bin ? in_bin : guess < 1.0 ? 1 : (u64)guess;
        while (m > 1 && above + (double)(m - 1) * w >= target) --m;
        while (m < in_bin && above + (double)m * w < target) ++m;
      }
      if (m >= in_bin) return Cut{low, EVERY};
      int64_t i0 = 0, i1 = R.n - 1;
      u64 passed = 0;
      for (;;) {
        const int ishift = shift_of<C>((u64)(i1 - i0));
        clear_bins<false>(S);
        for_cells<true, C::NT>(R, S.best, (int)(i0 / R.width()), (int)(i1 / R.width()) + 1, low, [&](int, const raw (&r)[U][VEC], int64_t at, bool) {
          each<F>(r, at, [&](wide v, int64_t i) {
            if ((double)v == low && i >= i0 && i <= i1 && have.keeps(low, i)) atomicAdd(&S.bins.count[(u64)(i - i0) >> ishift], 1u);
          });
        });
        find_bin<false>(S, passed, 0, 0, m, 0.0, 0.0);
        const int64_t from = i0 + (int64_t)(S.found[0] << ishift), to = from + (int64_t)((1ull << ishift) - 1);
        passed = S.found[1];
        const u64 here = S.found[2];
        i0 = from;
        i1 = to < i1 ? to : i1;
        if (ishift == 0 || passed + here == m) return Cut{low, i1};
      }
    }
    even = false;
    khi = key_of(high); klo = key_of(low); lo = low;
  }
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
  R.x = (typename Row<F>::Global)static_cast<const typename F::raw*>(A.logits) + row * A.row_stride; R.stride = A.col_stride; R.n = n;
  R.mult = A.mult;
  R.cells = (int)((n + R.width() - 1) / R.width());
  R.best = 0.0; R.t = t; R.per_t = 1.0 / t;
  return R;
}
// does the cut need the lowest value of the row (as the end of the bins' range)?
__device__ __forceinline__ bool wants_lowest(const Settings& p, int cells) { return p.top_k >= cells || (p.top_k == 0 && p.top_p < 1.0); }
// what is kept before any truncation: everything above -inf, but only the infinite entries where there are any
__device__ __forceinline__ Cut everything(double best) { return best == INF ? Cut{INF, EVERY} : Cut{-INF, -1}; }

// ---- the passes over a row ----------------------------------------------------------------------------------------------------------
// highest value of the cells [c0, c1) -> best[c]; where nothing is truncated (SUMS) also their weight relative to it -> sums[c].
// Returns, where `lowest` asks for it, this lane's lowest value above -inf (else +inf)
template <int THREADS, bool SUMS, class F> __device__ __forceinline__ double pass_best(Row<F> R, int c0, int c1, double* best, double* sums, bool lowest) {
  typedef typename F::raw raw;
  typedef typename F::wide wide;
  constexpr int VEC = Row<F>::VEC, U = F::U;
  const wide none = (wide)-INF;
  wide run = none, low = -none;
  for_cells<false, THREADS>(R, (const double*)nullptr, c0, c1, 0.0, [&](int c, const raw (&r)[U][VEC], int64_t, bool last) {
#pragma unroll
    for (int q = 0; q < U; ++q)
#pragma unroll
      for (int e = 0; e < VEC; ++e) run = F::larger(run, F::widen(r[q][e]));
    if (lowest) {
#pragma unroll
      for (int q = 0; q < U; ++q)
#pragma unroll
        for (int e = 0; e < VEC; ++e) { const wide v = F::widen(r[q][e]); low = v > none && v < low ? v : low; }
    }
    if (!last) return;
    const wide top = wave_max(run);
    run = none;
    if ((threadIdx.x & 63) == 0) best[c] = (double)top;
    if constexpr (!SUMS) return;
    double s = 0.0;
    if (top > none) {
      R.best = (double)top;
      const bool certain = top == -none;                        // (an infinite entry: the finite ones beside it weigh nothing)
      auto add = [&](const raw (&x)[U][VEC]) {
        each<F>(x, 0, [&](wide v, int64_t) {
          const double w = R.weight((double)v);
          s += v > none && (!certain || v == top) ? w : 0.0;
        });
      };
      if (R.mult == 1) add(r);
      else for (int j = 0; j < R.mult; ++j) {
        raw x[U][VEC];
        const int64_t g = (int64_t)c * R.mult + j;
        if (R.stride == 1 && (g + 1) * (U * Row<F>::UNIT) <= R.n) R.load_whole(g, x); else R.load_part(g, x);
        add(x);
      }
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sums[c] = s;
  });
  return (double)low;
}
// the factor of a cell's weight relative to its own best value
template <class F> __device__ __forceinline__ double cell_factor(const Row<F>& R, double top) {
  if (!(top > -INF) || (R.best == INF && top < INF)) return 0.0;
  return R.weight(top);
}
// kept weight of the cells [c0, c1) -> sums[c]
template <int THREADS, class F> __device__ __forceinline__ void pass_weights(const Row<F>& R, const double* best, int c0, int c1, const Cut& cut, double min_p, double* sums) {
  typedef typename F::raw raw;
  typedef typename F::wide wide;
  constexpr int VEC = Row<F>::VEC, U = F::U;
  double lo = cut.value > -1.7976931348623157e308 ? cut.value : -1.7976931348623157e308;
  if (min_p > 0.0 && R.best < INF) {                            // (no entry below this, with room for the roundings, has that weight)
    double v = R.best + R.t * log(min_p);
    v -= 1e-12 * (fabs(v) + fabs(R.best)) + 1e-9 * R.t;
    lo = v > lo ? v : lo;
  }
  wide quick; bound_below(lo, quick);
  for (int c = c0 + (int)threadIdx.x; c < c1; c += THREADS) if (!(best[c] >= lo)) sums[c] = 0.0;
  double s = 0.0;
  for_cells<true, THREADS>(R, best, c0, c1, lo, [&](int c, const raw (&r)[U][VEC], int64_t i0, bool last) {
    each<F>(r, i0, [&](wide v, int64_t i) {
      const double l = (double)v;
      if (v < quick || !(l >= lo) || !cut.keeps(l, i)) return;
      const double w = R.weight(l);
      s += w < min_p ? 0.0 : w;
    });
    if (!last) return;
    const double total = wave_sum(s);
    s = 0.0;
    if ((threadIdx.x & 63) == 0) sums[c] = total;
  });
}
// running sums over the cells, in place
template <class C> __device__ __forceinline__ void scan_cells(double* sums, double* red, int cells) {
  constexpr int PER = (C::CELLS + C::NT - 1) / C::NT;
  double v[PER], s = 0.0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PER; ++k) { const int c = threadIdx.x * PER + k; s += c < cells ? sums[c] : 0.0; v[k] = s; }
  const double base = block_scan<C::NT>(red, s) - s;
#pragma unroll
  for (int k = 0; k < PER; ++k) { const int c = threadIdx.x * PER + k; if (c < cells) sums[c] = base + v[k]; }
  __syncthreads();
}
// first of n running sums above x (or equal to it)
template <class Run> __device__ __forceinline__ int first_above(Run run, int n, double x, bool or_equal) {
  int a = 0, b = n;
  while (a < b) { const int m = (a + b) >> 1; const double f = run[m]; if (f > x || (or_equal && f >= x)) b = m; else a = m + 1; }
  return a;
}
__device__ __forceinline__ double target_of(double u, double Z) {                            // (u outside [0, 1): the first or the last kept entry)
  const double x = u * Z;
  return x > 0.0 ? x : x == x ? 0.0 : Z;
}
__device__ __forceinline__ void put_draw(const DrawArgs& A, int64_t at, int64_t found, double logp) {
  A.index[at] = found;
  if (A.logp) A.logp[at] = logp;
}
// (Running sums of two threads are rounded differently, so that one may grow by a rounding over entries that weigh nothing.  A draw
// that falls into such a gap takes the nearest kept entry behind it, or before it where there is none.)
// The draws [s0, s1) of a row from the running sums of its cells, one wavefront each
template <int THREADS, class F> __device__ __forceinline__ void draw(const DrawArgs& A, const Row<F>& R, const double* cells, int64_t row, int64_t s0, int64_t s1, const Cut& cut, double min_p) {
  const int lane = threadIdx.x & 63;
  const double Z = cells[R.cells - 1], log_z = log(Z);
  for (int64_t s = s0 + (threadIdx.x >> 6); s < s1; s += THREADS / 64) {
    double target = target_of(A.u[row * A.draws + s], Z);
    int c = first_above(cells, R.cells, target, false);
    if (c == R.cells) { c = first_above(cells, R.cells, Z, true); target = INF; }
    // the cell's running weight: every lane sums PER neighbouring entries, one scan over the lanes, and the lane that reaches the
    // target looks through its own
    constexpr int PER = F::U * Row<F>::VEC;
    int64_t found = -1;
    for (int step = 1, start = c; found < 0 && c >= 0;) {
      int64_t last = -1;
      double base = c ? cells[c - 1] : 0.0;
      for (int j = 0; j < R.mult && found < 0; ++j) {
        const int64_t i0 = c * R.width() + (int64_t)j * 64 * PER + lane * PER;
        double w[PER], sum = 0.0;
        int some = -1;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          w[e] = 0.0;
          if (i0 + e < R.n) {
            const double l = R.value(i0 + e);
            if (l > -INF && cut.keeps(l, i0 + e)) { const double x = R.weight(l); w[e] = x < min_p ? 0.0 : x; }
          }
          sum += w[e];
          some = w[e] > 0.0 ? e : some;
        }
        const double inc = wave_scan(sum);
        const u64 hit = __ballot(sum > 0.0 && base + inc > target), any = __ballot(sum > 0.0);
        if (any) { const int l = 63 - __clzll(any); last = i0 - lane * PER + l * PER + __shfl(some, l); }
        if (hit) {
          const int l = __ffsll(hit) - 1;
          double run = base + (inc - sum);
          int e = some;                                         // (its last kept one, should the sums differ by a rounding)
#pragma unroll
          for (int k = PER - 1; k >= 0; --k) {                  // run before entry k, from the back: the first that passes the target stays
            double r = run;
#pragma unroll
            for (int m = 0; m <= k; ++m) r += w[m];
            if (w[k] > 0.0 && r > target) e = k;
          }
          found = i0 - lane * PER + l * PER + __shfl(e, l);
        }
        base += __shfl(inc, 63);
      }
      if (found < 0) found = last;                              // (the cell's own sum and this one differ by a rounding)
      if (found < 0) {                                          // (nothing kept in this cell)
        c += step;
        if (c == R.cells) { step = -1; c = start - 1; }
      }
    }
    if (lane == 0) put_draw(A, row * A.draws + s, found, found < 0 ? -INF : R.z(R.value(found)) - log_z);
  }
}
template <class F> __device__ __forceinline__ double kept_weight(const Row<F>& R, const Cut& cut, double min_p, int64_t i) {
  if (i >= R.n) return 0.0;
  const double l = R.value(i);
  if (!(l > -INF) || !cut.keeps(l, i)) return 0.0;
  const double w = R.weight(l);
  return w < min_p ? 0.0 : w;
}
// The entry of lot j (PER neighbouring entries; run: running sums of the lots) where the running sum passes `target`
template <class F, class Run> __device__ __forceinline__ int64_t entry_of_lot(const Row<F>& R, Run run, int lots, int j, double target, const Cut& cut, double min_p) {
  constexpr int PER = F::U * Row<F>::VEC;
  double r = j ? run[j - 1] : 0.0;
  int64_t found = -1;
#pragma unroll 1
  for (int k = j, step = 1; found < 0 && k >= 0;) {
#pragma unroll 1
    for (int e = 0; e < PER; ++e) {
      const int64_t i = (int64_t)k * PER + e;
      const double w = kept_weight(R, cut, min_p, i);
      r += w;
      // (else its last kept one: the sums differ by a rounding.  So too on the way back, where the lots behind weigh nothing)
      if (w > 0.0) { found = i; if (step > 0 && r > target) break; }
    }
    k += step;                                                  // (nothing kept in this lot)
    if (k == lots) { step = -1; k = j - 1; }
  }
  return found;
}
__device__ __forceinline__ void draw_nothing(const DrawArgs& A, int64_t row, int64_t s0, int64_t s1, int threads) {
  for (int64_t s = s0 + threadIdx.x; s < s1; s += threads) {
    A.index[row * A.draws + s] = -1;
    if (A.logp) A.logp[row * A.draws + s] = -INF;
  }
}
// All truncations on a sorted list that holds the row's first top_k entries: how many are kept (the first ones)
template <class C, class F> __device__ __forceinline__ int keep_list(const Row<F>& R, Shared<C>& S, const Settings& p, int count) {
  const int t = threadIdx.x;
  int n = p.top_k < count ? (int)p.top_k : count;
  const double w = t < n ? R.weight(S.list_value[t]) : 0.0;
  const double sum = block_scan<C::NT>(S.red, w);
  if (p.top_p < 1.0) {
    __syncthreads();
    if (t == n - 1) S.red[0] = sum;
    __syncthreads();
    const double goal = p.top_p * S.red[0];
    n = 1 + (int)block_min<C::NT>(S.red, t < n && sum >= goal ? (double)t : (double)(n - 1));
  }
  return (int)block_max<C::NT>(S.red, t < n && w >= p.min_p ? (double)(t + 1) : 1.0);        // (the best one always is)
}
// the draws from the first n entries of a sorted list: by index, running sums in LDS, one thread per draw
template <class C, class F> __device__ __forceinline__ void draw_list(const DrawArgs& A, const Row<F>& R, Shared<C>& S, int64_t row, int n) {
  static_assert(C::LIST <= Shared<C>::BINS, "running sums of the list in the bins' place");
  const int t = threadIdx.x;
  double value = 0.0; uint32_t idx = 0; int rank = 0;
  if (t < n) { value = S.list_value[t]; idx = S.list_idx[t]; }
  if (t - (t & 63) < n) for (int j = 0; j < n; ++j) rank += S.list_idx[j] < idx;
  __syncthreads();
  if (t < n) { S.list_value[rank] = value; S.list_idx[rank] = idx; }
  __syncthreads();
  const double sum = block_scan<C::NT>(S.red, t < n ? R.weight(S.list_value[t]) : 0.0);
  double* run = reinterpret_cast<double*>(S.bins.hi);
  if (t < n) run[t] = sum;
  __syncthreads();
  const double Z = run[n - 1], log_z = log(Z);
  for (int64_t s = t; s < A.draws; s += C::NT) {
    int j = first_above(run, n, target_of(A.u[row * A.draws + s], Z), false);
    if (j == n) j = first_above(run, n, Z, true);
    const int start = j;
    while (j < n && !(R.weight(S.list_value[j]) > 0.0)) ++j;     // (see draw)
    if (j == n) for (j = start; j > 0 && !(R.weight(S.list_value[j]) > 0.0);) --j;
    put_draw(A, row * A.draws + s, (int64_t)S.list_idx[j], R.z(S.list_value[j]) - log_z);
  }
}
// A lower bound of the top_k-th value: the top_k-th highest of the cells' best values, from bins over them (S.best); `lowest` if there
// are no more cells than that, or none with anything in them, and the bins are empty then (bounded: false: cut_of counts the row's
// entries in them).  Only cells that reach the bound are looked at again
template <class C, class F> __device__ __forceinline__ double bound_of_top_k(const Row<F>& R, Shared<C>& S, int64_t top_k, double lowest, bool& bounded) {
  bounded = false;
  clear_bins<false>(S);
  if (top_k >= R.cells) return lowest;
  double least = INF;
  for (int c = threadIdx.x; c < R.cells; c += C::NT) { const double v = S.best[c]; least = v > -INF && v < least ? v : least; }
  const u64 top = key_of(R.best), low = key_of(block_min<C::NT>(S.red, least));
  const int shift = shift_of<C>(top - low);
  for (int c = threadIdx.x; c < R.cells; c += C::NT) if (S.best[c] > -INF) atomicAdd(&S.bins.count[(top - key_of(S.best[c])) >> shift], 1u);
  find_bin<false>(S, 0, 0, 0, (u64)top_k, 0.0, 0.0);
  if (S.found[6] < (u64)top_k) { clear_bins<false>(S); return lowest; }
  const u64 drop = ((S.found[0] + 1) << shift) - 1;             // (to the lowest pattern of the bin)
  bounded = true;
  return of_key(drop < top - low ? top - drop : low);
}
// ... of what top_p keeps: entries below exp(-56) < 2^-80 of the best one weigh nothing in the bins
template <class F> __device__ __forceinline__ double bound_of_top_p(const Row<F>& R, double lowest, const Cut& cut) {
  double lo = R.best < INF ? R.best - 56.0 * R.t : INF;
  lo = lo > lowest ? lo : lowest;
  return lo > cut.value ? lo : cut.value;
}
__device__ __forceinline__ double finite_lowest(double v) { return v > -1.7976931348623157e308 ? v : -1.7976931348623157e308; }
// The cut of a row whose cells' highest values are in S.best; R.best is set; `lowest` of the row where wants_lowest asked for it, else
// -inf.  listed > 0: the list holds exactly the kept entries; summed: S.cells the cells' kept weights
template <class C, class F> __device__ __forceinline__ Cut cut_of(const Row<F>& R, Shared<C>& S, const Settings& p, double lowest, int& listed, bool& summed) {
  typedef typename F::raw raw;
  typedef typename F::wide wide;
  constexpr int VEC = Row<F>::VEC, U = F::U;
  Cut cut = everything(R.best);
  listed = 0;
  summed = false;
  lowest = finite_lowest(lowest);
  if (p.top_k > 0) {
    bool bounded;
    const double lo = bound_of_top_k<C, F>(R, S, p.top_k, lowest, bounded);
    __syncthreads();
    int upto = -1;                                              // (bins the list takes; -1: everything from the bound on)
    const Even parts(R.best, lo > cut.value ? lo : cut.value, Shared<C>::BINS);
    if (p.top_k <= C::LIST && !bounded && R.n > 64 && parts.good) {
      // no bound from the cells: from bins over all entries
      const double floor = lo > cut.value ? lo : cut.value;
      for_cells<true, C::NT>(R, S.best, 0, R.cells, floor, [&](int, const raw (&r)[U][VEC], int64_t i0, bool) {
        each<F>(r, i0, [&](wide v, int64_t) { const double l = (double)v; if (l >= floor) atomicAdd(&S.bins.count[parts.bin(l)], 1u); });
      });
      find_bin<false>(S, 0, 0, 0, (u64)p.top_k, 0.0, 0.0);
      if (S.found[1] + S.found[2] <= (u64)C::LIST) { upto = (int)S.found[0]; bounded = true; }
    }
    if (p.top_k <= C::LIST && (bounded || R.n <= C::LIST)) {
      // few: all entries that reach it, if they fit the list -- everything else happens there
      wide quick; bound_below(lo, quick);
      const double floor = lo > cut.value ? lo : cut.value;
      for_cells<true, C::NT>(R, S.best, 0, R.cells, lo, [&](int, const raw (&r)[U][VEC], int64_t i0, bool) {
        each<F>(r, i0, [&](wide v, int64_t i) {
          const double l = (double)v;
          if (v < quick || !(l >= floor) || !(l > -INF)) return;
          if (upto >= 0 && parts.bin(l) > upto) return;
          const int at = atomicAdd(&S.listed, 1);
          if (at < C::LIST) { S.list_value[at] = l; S.list_idx[at] = (uint32_t)i; }
        });
      });
      __syncthreads();
      const int count = S.listed;
      if (count <= C::LIST) {
        if (upto >= 0) sort_list_by_bins(S, count, [&](double l) { return parts.bin(l); }); else sort_list(S, count);
        listed = keep_list<C, F>(R, S, p, count);
        return Cut{S.list_value[listed - 1], (int64_t)S.list_idx[listed - 1]};
      }
    }
    cut = tighter(cut, select<false, false, C, F>(R, S, lo, cut, (u64)p.top_k, 0.0));
  }
  if (p.top_p < 1.0) cut = tighter(cut, select<true, false, C, F>(R, S, bound_of_top_p(R, lowest, cut), cut, 0, p.top_p, p.min_p, &summed));
  return cut;
}

// A row of one wavefront's build: running sums lane by lane (PER neighbouring entries each) in LDS, then one lane per draw
template <class C, class F> __device__ __forceinline__ void draw_tiny(const DrawArgs& A, const Row<F>& R, Shared<C>& S, int64_t row, const Cut& cut, double min_p) {
  constexpr int PER = F::U * Row<F>::VEC;
  static_assert(C::NT == 64 && C::CELLS * 64 <= 2 * Shared<C>::BINS, "running sums in the bins' place");
  double* run = reinterpret_cast<double*>(S.bins.hi);            // (hi and lo)
  const int lane = threadIdx.x;
  const int lots = (int)((R.n + PER - 1) / PER), rounds = (lots + 63) / 64;
  double base = 0.0;
  __syncthreads();
  for (int c = 0; c < rounds; ++c) {
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < PER; ++e) sum += kept_weight(R, cut, min_p, (int64_t)(c * 64 + lane) * PER + e);
    const double inc = wave_scan(sum);
    run[c * 64 + lane] = base + inc;
    base += __shfl(inc, 63);
  }
  __syncthreads();
  const double Z = run[lots - 1], log_z = log(Z);
  for (int64_t s = lane; s < A.draws; s += 64) {
    double target = target_of(A.u[row * A.draws + s], Z);
    int j = first_above(run, lots, target, false);
    if (j == lots) { j = first_above(run, lots, Z, true); target = INF; }
    const int64_t found = entry_of_lot(R, run, lots, j, target, cut, min_p);
    put_draw(A, row * A.draws + s, found, found < 0 ? -INF : R.z(R.value(found)) - log_z);
  }
}

// ---- kernels --------------------------------------------------------------------------------------------------------------------------
// One workgroup per row: everything, or (draws_here 0: many draws per row) all but the draws of rows whose kept entries are not in a
// list, which k_draws makes from memory
template <class C, class F> __global__ __launch_bounds__(C::NT) __attribute__((amdgpu_waves_per_eu(4))) void k_row(DrawArgs A, int draws_here) {
  __shared__ Shared<C> S;
  const int64_t row = blockIdx.x;
  const Settings p = settings_of(A, row);
  Row<F> R = row_of<F>(A, row, p.t);
  const bool lowest = wants_lowest(p, R.cells);
  constexpr bool TINY = C::NT == 64;                            // (makes its own draws always)
  const bool plain = p.plain && !TINY;
  const double low = plain ? pass_best<C::NT, true, F>(R, 0, R.cells, S.best, S.cells, false)
                           : pass_best<C::NT, false, F>(R, 0, R.cells, S.best, nullptr, lowest);
  __syncthreads();
  double top = -INF;
  for (int c = threadIdx.x; c < R.cells; c += C::NT) top = S.best[c] > top ? S.best[c] : top;
  R.best = block_max<C::NT>(S.red, top);
  Cut cut = everything(R.best);
  if (R.best > -INF) {
    if (!p.plain) {
      int listed;
      bool summed;
      cut = cut_of<C, F>(R, S, p, lowest ? block_min<C::NT>(S.red, low) : -INF, listed, summed);
      if (listed) {
        draw_list<C, F>(A, R, S, row, listed);
        if (!TINY && !draws_here && threadIdx.x == 0) A.cut[row] = CutState{0.0, DRAWN};
        return;
      }
      if constexpr (TINY) { draw_tiny<C, F>(A, R, S, row, cut, p.min_p); return; }
      __syncthreads();                                          // (the cells take the bins' place)
      if (!summed) pass_weights<C::NT, F>(R, S.best, 0, R.cells, cut, p.min_p, S.cells);
    } else if constexpr (TINY) {
      draw_tiny<C, F>(A, R, S, row, cut, 0.0);
      return;
    } else if (draws_here) {
      for (int c = threadIdx.x; c < R.cells; c += C::NT) S.cells[c] *= cell_factor(R, S.best[c]);
    }
  }
  if (TINY || draws_here) {
    if (!(R.best > -INF)) { draw_nothing(A, row, 0, A.draws, C::NT); return; }
    scan_cells<C>(S.cells, S.red, R.cells);
    draw<C::NT, F>(A, R, S.cells, row, 0, A.draws, cut, p.min_p);
    return;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < R.cells; c += C::NT) { A.best[row * A.max_cells + c] = S.best[c]; A.sums[row * A.max_cells + c] = S.cells[c]; }
  if (threadIdx.x == 0) A.cut[row] = CutState{cut.value, cut.idx};
}

// The same over several launches, for a few long rows whose cells are dealt to `groups` workgroups each.  First: the cells' highest
// values, the lowest value of each group, and -- nothing truncated -- the cells' weights.  The bins and lists of the launches
// behind it start empty
template <class F> __global__ __launch_bounds__(256) void k_best(DrawArgs A, int groups, int stages) {
  __shared__ double red[4];
  const int64_t row = blockIdx.x / groups;
  const int g = blockIdx.x % groups;
  const Settings p = settings_of(A, row);
  const Row<F> R = row_of<F>(A, row, p.t);
  const int c0 = (int)((int64_t)R.cells * g / groups), c1 = (int)((int64_t)R.cells * (g + 1) / groups);
  const bool lowest = wants_lowest(p, R.cells);
  double* best = A.best + row * A.max_cells;
  const double low = p.plain ? pass_best<256, true, F>(R, c0, c1, best, A.sums + row * A.max_cells, false)
                             : pass_best<256, false, F>(R, c0, c1, best, nullptr, lowest);
  const double least = lowest ? block_min<256>(red, low) : -INF;
  if (threadIdx.x == 0) A.lows[row * groups + g] = least;
  for (int k = 0; k < stages; ++k) {
    Table& T = A.tables[row * 2 + k];
    for (int b = g * 256 + threadIdx.x; b < TABLE_BINS; b += groups * 256) { T.count[b] = 0; T.hi[b] = 0; T.lo[b] = 0; }
    if (g == 0 && threadIdx.x == 0) { T.listed = 0; if (k == 0) { const Cut c = Cut{-INF, -1}; A.cut[row] = CutState{c.value, c.idx}; } }
  }
}
// What the launches of a stage (0: top_k, 1: top_p) start from; false: the row has no such truncation
template <class F> __device__ __forceinline__ bool start_stage(const DrawArgs& A, int64_t row, int groups, int stage, Shared<All>& S, Settings& p, Row<F>& R, Cut& have, double& lo) {
  p = settings_of(A, row);
  if (stage == 0 ? p.top_k == 0 : p.top_p == 1.0) return false;
  R = row_of<F>(A, row, p.t);
  double top = -INF, low = INF;
  for (int c = threadIdx.x; c < R.cells; c += All::NT) { const double v = A.best[row * A.max_cells + c]; S.best[c] = v; top = v > top ? v : top; }
  for (int g = threadIdx.x; g < groups; g += All::NT) { const double v = A.lows[row * groups + g]; low = v < low ? v : low; }
  R.best = block_max<All::NT>(S.red, top);
  low = finite_lowest(block_min<All::NT>(S.red, low));
  if (!(R.best > -INF)) return false;
  have = everything(R.best);
  if (stage == 1) have = tighter(have, Cut{A.cut[row].value, A.cut[row].idx});
  bool bounded;
  lo = stage == 0 ? bound_of_top_k<All, F>(R, S, p.top_k, low, bounded) : bound_of_top_p(R, low, have);
  lo = lo > have.value ? lo : have.value;
  return true;
}
// ... the first bins of a stage
template <bool WEIGHTED, class F> __global__ __launch_bounds__(All::NT) void k_bins(DrawArgs A, int groups, int shares) {
  typedef typename F::raw raw;
  typedef typename F::wide wide;
  constexpr int VEC = Row<F>::VEC, U = F::U;
  __shared__ Shared<All> S;
  const int64_t row = blockIdx.x / shares;
  const int g = blockIdx.x % shares;
  Settings p; Row<F> R; Cut have; double lo;
  if (!start_stage<F>(A, row, groups, WEIGHTED ? 1 : 0, S, p, R, have, lo)) return;
  const Even parts(R.best, lo, Shared<All>::BINS);
  if (!parts.good) return;
  clear_bins<WEIGHTED>(S);
  wide quick; bound_below(lo, quick);
  const int c0 = (int)((int64_t)R.cells * g / shares), c1 = (int)((int64_t)R.cells * (g + 1) / shares);
  for_cells<true, All::NT>(R, S.best, c0, c1, lo, [&](int, const raw (&r)[U][VEC], int64_t i0, bool) {
    each<F>(r, i0, [&](wide v, int64_t i) {
      const double l = (double)v;
      if (v < quick || !(l >= lo) || !have.keeps(l, i)) return;
      const int b = parts.bin(l);
      atomicAdd(&S.bins.count[b], 1u);
      if (WEIGHTED) add_weight(S, b, R.weight(l));
    });
  });
  __syncthreads();
  Table& T = A.tables[row * 2 + (WEIGHTED ? 1 : 0)];
  for (int b = threadIdx.x; b < TABLE_BINS; b += All::NT) {     // (sums of integers: the order of the workgroups does not matter)
    if (!S.bins.count[b]) continue;
    atomicAdd(&T.count[b], S.bins.count[b]);
    if (WEIGHTED) { if (S.bins.hi[b]) atomicAdd(&T.hi[b], S.bins.hi[b]); if (S.bins.lo[b]) atomicAdd(&T.lo[b], S.bins.lo[b]); }
  }
}
template <bool WEIGHTED> __device__ __forceinline__ void load_bins(Shared<All>& S, const Table& T) {
  __syncthreads();
  for (int b = threadIdx.x; b < TABLE_BINS; b += All::NT) { S.bins.count[b] = T.count[b]; if (WEIGHTED) { S.bins.hi[b] = T.hi[b]; S.bins.lo[b] = T.lo[b]; } }
  if (threadIdx.x == 0) S.listed = 0;
}
// ... the entries of the bin that holds the cut
template <bool WEIGHTED, class F> __global__ __launch_bounds__(All::NT) void k_list(DrawArgs A, int groups, int shares) {
  typedef typename F::raw raw;
  typedef typename F::wide wide;
  constexpr int VEC = Row<F>::VEC, U = F::U;
  __shared__ Shared<All> S;
  const int64_t row = blockIdx.x / shares;
  const int g = blockIdx.x % shares;
  Settings p; Row<F> R; Cut have; double lo;
  if (!start_stage<F>(A, row, groups, WEIGHTED ? 1 : 0, S, p, R, have, lo)) return;
  const Even parts(R.best, lo, Shared<All>::BINS);
  if (!parts.good) return;
  Table& T = A.tables[row * 2 + (WEIGHTED ? 1 : 0)];
  load_bins<WEIGHTED>(S, T);
  find_bin<WEIGHTED>(S, 0, 0, 0, (u64)p.top_k, p.top_p, -1.0);
  if (S.found[2] > (u64)All::LIST) return;
  const int bin = (int)S.found[0];
  wide quick; bound_below(lo, quick);
  const int c0 = (int)((int64_t)R.cells * g / shares), c1 = (int)((int64_t)R.cells * (g + 1) / shares);
  for_cells<true, All::NT>(R, S.best, c0, c1, lo, [&](int, const raw (&r)[U][VEC], int64_t i0, bool) {
    each<F>(r, i0, [&](wide v, int64_t i) {
      const double l = (double)v;
      if (v < quick || !(l >= lo) || parts.bin(l) != bin || !have.keeps(l, i)) return;
      const int at = atomicAdd(&T.listed, 1);
      T.value[at] = l; T.idx[at] = (uint32_t)i;
    });
  });
}
// ... and the cut of the stage
template <bool WEIGHTED, class F> __global__ __launch_bounds__(All::NT) void k_cut(DrawArgs A, int groups) {
  __shared__ Shared<All> S;
  const int64_t row = blockIdx.x;
  Settings p; Row<F> R; Cut have; double lo;
  if (!start_stage<F>(A, row, groups, WEIGHTED ? 1 : 0, S, p, R, have, lo)) return;
  const Table& T = A.tables[row * 2 + (WEIGHTED ? 1 : 0)];
  load_bins<WEIGHTED>(S, T);
  for (int t = threadIdx.x; t < T.listed; t += All::NT) { S.list_value[t] = T.value[t]; S.list_idx[t] = T.idx[t]; }
  const Cut cut = tighter(have, select<WEIGHTED, true, All, F>(R, S, lo, have, (u64)p.top_k, p.top_p));
  if (threadIdx.x == 0) A.cut[row] = CutState{cut.value, cut.idx};
}
template <int THREADS> __device__ __forceinline__ double best_of_row(const DrawArgs& A, int64_t row, int cells, double* red) {
  double top = -INF;
  for (int c = threadIdx.x; c < cells; c += THREADS) { const double v = A.best[row * A.max_cells + c]; top = v > top ? v : top; }
  return block_max<THREADS>(red, top);
}
// ... the cells' kept weights (cuts 0: no launch of k_cut came before)
template <class F> __global__ __launch_bounds__(256) void k_weights(DrawArgs A, int groups, int cuts) {
  __shared__ double red[4];
  const int64_t row = blockIdx.x / groups;
  const int g = blockIdx.x % groups;
  const Settings p = settings_of(A, row);
  Row<F> R = row_of<F>(A, row, p.t);
  R.best = best_of_row<256>(A, row, R.cells, red);
  if (p.plain || !(R.best > -INF)) return;
  const Cut cut = cuts ? tighter(everything(R.best), Cut{A.cut[row].value, A.cut[row].idx}) : everything(R.best);
  const int c0 = (int)((int64_t)R.cells * g / groups), c1 = (int)((int64_t)R.cells * (g + 1) / groups);
  pass_weights<256, F>(R, A.best + row * A.max_cells, c0, c1, cut, p.min_p, A.sums + row * A.max_cells);
}
// The running sums of a row's cells from memory; false: nothing to draw from them
struct Sums { double cells[MAX_CELLS], red[Long::NT / 64]; };
template <class F> __device__ __forceinline__ bool load_sums(const DrawArgs& A, Sums& S, Row<F>& R, const Settings& p, int64_t row, int cuts, Cut& cut) {
  R.best = best_of_row<Long::NT>(A, row, R.cells, S.red);
  if (!(R.best > -INF)) return false;
  cut = cuts ? tighter(everything(R.best), Cut{A.cut[row].value, A.cut[row].idx}) : everything(R.best);
  for (int c = threadIdx.x; c < R.cells; c += Long::NT) {
    const double w = A.sums[row * A.max_cells + c];
    S.cells[c] = p.plain ? w * cell_factor(R, A.best[row * A.max_cells + c]) : w;
  }
  scan_cells<Long>(S.cells, S.red, R.cells);
  return true;
}
typedef __attribute__((address_space(1))) double* Lots;
// ... the running sums of the cells' lots (PER neighbouring entries, a lane's share of draw), for rows with many draws
__device__ __forceinline__ bool drawn(const DrawArgs& A, int64_t row, int cuts) { return cuts && A.cut[row].idx == DRAWN; }
template <class F> __global__ __launch_bounds__(Long::NT) void k_lots(DrawArgs A, int shares, int cuts) {
  __shared__ Sums S;
  constexpr int PER = F::U * Row<F>::VEC;
  const int64_t row = blockIdx.x / shares;
  const int g = blockIdx.x % shares, lane = threadIdx.x & 63;
  if (drawn(A, row, cuts)) return;
  const Settings p = settings_of(A, row);
  Row<F> R = row_of<F>(A, row, p.t);
  Cut cut;
  if (!load_sums(A, S, R, p, row, cuts, cut)) return;
  const Lots lots = (Lots)A.lots + row * ((int64_t)A.max_cells * A.mult * 64);
  const int c0 = (int)((int64_t)R.cells * g / shares), c1 = (int)((int64_t)R.cells * (g + 1) / shares);
  for (int c = c0 + (int)(threadIdx.x >> 6); c < c1; c += Long::NT / 64) {
    double base = c ? S.cells[c - 1] : 0.0;
    const bool some = A.best[row * A.max_cells + c] >= cut.value;
    for (int j = 0; j < R.mult; ++j) {
      const int64_t lot = ((int64_t)c * R.mult + j) * 64 + lane;
      double sum = 0.0;
      if (some) {
#pragma unroll
        for (int e = 0; e < PER; ++e) sum += kept_weight(R, cut, p.min_p, lot * PER + e);
      }
      const double inc = wave_scan(sum);
      lots[lot] = base + inc;
      base += __shfl(inc, 63);
    }
  }
}
// ... and the draws, `per` of a row in every workgroup: a wavefront for each, or (LOTS) a lane
template <class F, bool LOTS> __global__ __launch_bounds__(Long::NT) void k_draws(DrawArgs A, int blocks, int per, int cuts) {
  __shared__ Sums S;
  const int64_t row = blockIdx.x / blocks;
  const int64_t s0 = (int64_t)(blockIdx.x % blocks) * per, s1 = s0 + per < A.draws ? s0 + per : A.draws;
  if (drawn(A, row, cuts)) return;
  const Settings p = settings_of(A, row);
  Row<F> R = row_of<F>(A, row, p.t);
  Cut cut;
  if (!load_sums(A, S, R, p, row, cuts, cut)) { draw_nothing(A, row, s0, s1, Long::NT); return; }
  if constexpr (!LOTS) {
    draw<Long::NT, F>(A, R, S.cells, row, s0, s1, cut, p.min_p);
  } else {
    constexpr int PER = F::U * Row<F>::VEC;
    const Lots run = (Lots)A.lots + row * ((int64_t)A.max_cells * A.mult * 64);
    const int all = (int)((R.n + PER - 1) / PER), each_cell = 64 * R.mult;
    const double Z = S.cells[R.cells - 1], log_z = log(Z);
    for (int64_t s = s0 + threadIdx.x; s < s1; s += Long::NT) {
      double target = target_of(A.u[row * A.draws + s], Z);
      int c = first_above(S.cells, R.cells, target, false);
      if (c == R.cells) { c = first_above(S.cells, R.cells, Z, true); target = INF; }
      const int from = c * each_cell, n = all - from < each_cell ? all - from : each_cell;
      int j = first_above(run + from, n, target, false);
      if (j == n) { j = first_above(run + from, n, run[from + n - 1], true); target = INF; }
      const int64_t found = entry_of_lot(R, run, all, from + j, target, cut, p.min_p);
      put_draw(A, row * A.draws + s, found, found < 0 ? -INF : R.z(R.value(found)) - log_z);
    }
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------
// How a call runs: cells of a row, workgroups per row (0: one workgroup does a whole row), which build of it (0 Long, 1 Many, 2 Tiny),
// draws made by the row's own workgroup, and from lots where not
struct Plan { int mult, max_cells, groups, shares, build; bool draws_here, lots; };
static_assert(Shared<All>::BINS == TABLE_BINS && All::LIST == TABLE_LIST, "tables in memory");
enum Cuts { NO_CUT = 0, CUT = 1, FEW = 2 };                     // truncated?  FEW: to no more entries than a list takes
Plan plan_of(int type, int64_t rows, int64_t cols, int64_t draws, Cuts cuts) {
  Plan p;
  const int64_t group = type == 0 ? 2 * 128 : type == 1 ? 2 * 256 : 512;
  p.mult = (int)((cols + group * MAX_CELLS - 1) / (group * MAX_CELLS));
  p.max_cells = (int)((cols + group * p.mult - 1) / (group * p.mult));
  // One wavefront per row: many short rows (4096 x 1113 fp64, top_p, 8 draws: 54 us against 67 with four; 1000 of them: 29 against 22,
  // hence the 1024), and the shortest while it can make the draws (300 x 161, top_p, 8 draws: 16 against 23; 256 draws: 25 against 32;
  // 1000 draws: 54 against 30).  Four wavefronts where rows fill the chip (two such workgroups' phases overlap better than one of
  // eight: 4096 x 51200 fp32, top_k 50, 208 us against 227); eight else
  p.build = (p.max_cells <= Tiny::CELLS && rows >= 1024) || (p.max_cells <= 2 && draws <= 256) ? 2 : rows > 512 ? 1 : 0;
  // A few long rows are cut into pieces, so that more of the chip works on them, at the price of one launch more, with a cut of four or
  // seven (fp64, plain, one workgroup against pieces: 1 x 25600 19 and 13 us, 1 x 204800 93 and 14, 64 x 204800 97 and 41, 256 x 204800
  // 111 and 124;  top_p: 1 x 25600 37 and 49, 1 x 51200 61 and 50, 64 x 51200 67 and 82, 64 x 102400 110 and 99, 128 x 204800 200 and
  // 195;  top_k 20, which a row's own workgroup makes from a list: 1 x 204800 47 and 47, 64 x 204800 49 and 78)
  const int64_t loads = (int64_t)p.max_cells * p.mult, least = cuts == NO_CUT ? 48 : cuts == CUT ? 160 + 2 * rows : 800 + 3 * rows;
  p.groups = (p.build == 0 && loads >= least && rows <= 128) ? (int)std::min<int64_t>(p.max_cells / 8, std::max<int64_t>(1, 512 / rows)) : 0;
  p.shares = (int)std::max<int64_t>(1, std::min<int64_t>(p.max_cells / 16, 256 / rows));      // (of the launches with 16 wavefronts and tables to merge)
  // A wavefront takes 3 us for a draw, a launch more 4: four rounds of them in place (300 x 1113, 17 draws: 16 us against 24; 64: 35
  // against 20).  One wavefront's rows have lanes make them
  p.draws_here = p.groups == 0 && (p.build == 2 || draws <= (p.build == 1 ? 16 : 32));
  // Lots: each cell's weights once for all draws of the row, then a lane per draw instead of a wavefront.  Worth it where a row has as
  // many draws as cells and the chip has more draws than wavefronts (600 x 50000 fp32, 300 draws: 174 us against 388; 65 draws on
  // those 98 cells: 158 without; 32 x 161, 168 draws: 24 both)
  p.lots = !p.draws_here && draws >= p.max_cells && draws * rows >= 8192;
  return p;
}
int64_t lots_of(const Plan& p) { return p.lots ? (int64_t)p.max_cells * p.mult * 64 : 0; }
int64_t scratch_of(const Plan& p, int64_t rows) {
  if (p.draws_here) return 0;
  return rows * (2 * (int64_t)p.max_cells + p.groups + 2 + lots_of(p) + (p.groups ? 2 * (int64_t)(sizeof(Table) / sizeof(double)) : 0));
}
static_assert(sizeof(Table) % sizeof(double) == 0, "scratch in doubles");
Cuts cuts_of(const DrawArgs& A) {
  if (!A.temperature.p && A.temperature.v == 0.0) return FEW;
  if (!A.top_p.p && A.top_p.v == 0.0) return FEW;
  if (!A.top_k.p && A.top_k.v > 0 && A.top_k.v <= Long::LIST) return FEW;
  return A.temperature.p || A.top_k.p || A.top_k.v > 0 || A.top_p.p || A.top_p.v < 1.0 ? CUT : NO_CUT;
}

template <class F> void launch(DrawArgs& A, const Plan& p, int64_t rows, hipStream_t st) {
  int cuts = 1;
  if (p.groups == 0) {
    const dim3 grid((unsigned)rows);
    // (where a list of few entries is likely, its draws are cheap: 300 x 1113 rows of 64 draws, top_k 20: 16 us, with launches for the
    // draws of other rows 21)
    const bool here = p.draws_here || (A.draws <= 64 && !A.top_k.p && A.top_k.v > 0 && A.top_k.v <= 64);
    if (p.build == 2) hipLaunchKernelGGL((k_row<Tiny, F>), grid, dim3(Tiny::NT), 0, st, A, here ? 1 : 0);
    else if (p.build == 1) hipLaunchKernelGGL((k_row<Many, F>), grid, dim3(Many::NT), 0, st, A, here ? 1 : 0);
    else hipLaunchKernelGGL((k_row<Long, F>), grid, dim3(Long::NT), 0, st, A, here ? 1 : 0);
    if (here) return;
  } else {
    const dim3 grid((unsigned)(rows * p.groups));
    const bool ks = A.temperature.p || A.temperature.v == 0.0 || A.top_k.p || A.top_k.v > 0 || A.top_p.p || A.top_p.v == 0.0;
    const bool ps = A.top_p.p || (A.top_p.v < 1.0 && A.top_p.v > 0.0);
    cuts = ks || ps;
    hipLaunchKernelGGL(k_best<F>, grid, dim3(256), 0, st, A, p.groups, ks || ps ? 2 : 0);
    const dim3 shared((unsigned)(rows * p.shares)), one((unsigned)rows), all(All::NT);
    if (ks) {
      hipLaunchKernelGGL((k_bins<false, F>), shared, all, 0, st, A, p.groups, p.shares);
      hipLaunchKernelGGL((k_list<false, F>), shared, all, 0, st, A, p.groups, p.shares);
      hipLaunchKernelGGL((k_cut<false, F>), one, all, 0, st, A, p.groups);
    }
    if (ps) {
      hipLaunchKernelGGL((k_bins<true, F>), shared, all, 0, st, A, p.groups, p.shares);
      hipLaunchKernelGGL((k_list<true, F>), shared, all, 0, st, A, p.groups, p.shares);
      hipLaunchKernelGGL((k_cut<true, F>), one, all, 0, st, A, p.groups);
    }
    if (cuts || A.min_p.p || A.min_p.v > 0.0) hipLaunchKernelGGL(k_weights<F>, grid, dim3(256), 0, st, A, p.groups, cuts);
  }
  if (p.lots) {
    const int shares = (int)std::max<int64_t>(1, std::min<int64_t>(p.max_cells / 8, 1024 / rows));
    hipLaunchKernelGGL(k_lots<F>, dim3((unsigned)(rows * shares)), dim3(Long::NT), 0, st, A, shares, cuts);
  }
  // a wavefront makes one draw at a time (with lots: 64): one each while that leaves the chip room (calls back to back in a graph,
  // 1 x 204800, 1000 draws: 15 us against 18 with two; 100 x 20000, 40: 17 against 21), else two, or more where that fills it anyway
  const int at_once = p.lots ? Long::NT : A.draws * rows <= 4096 ? 8 : 16;
  const int per = (int)std::max<int64_t>(at_once, (A.draws * rows / 1024 + at_once - 1) / at_once * at_once);
  const int blocks = (int)((A.draws + per - 1) / per);
  const dim3 grid((unsigned)(rows * blocks));
  if (p.lots) hipLaunchKernelGGL((k_draws<F, true>), grid, dim3(Long::NT), 0, st, A, blocks, per, cuts);
  else hipLaunchKernelGGL((k_draws<F, false>), grid, dim3(Long::NT), 0, st, A, blocks, per, cuts);
}
}  // namespace

extern "C" int64_t pgm_draw_scratch_doubles(int type, int64_t rows, int64_t cols, int64_t draws) {
  if (type < 0 || type > 3 || rows < 1 || rows >= MAX_ROWS || cols < 1 || cols >= MAX_COLS || draws < 1) return 0;
  int64_t most = 0;                                             // (whatever the truncation)
  for (const Cuts cuts : {NO_CUT, CUT, FEW}) most = std::max(most, scratch_of(plan_of(type, rows, cols, draws, cuts), rows));
  return most;
}

extern "C" int pgm_draw_indices(const void* logits, int type, int64_t rows, int64_t cols, int64_t row_stride, int64_t col_stride,
                                const int64_t* lengths, const double* u, int64_t draws,
                                double temperature, const double* temperature_row, int64_t top_k, const int64_t* top_k_row,
                                double top_p, const double* top_p_row, double min_p, const double* min_p_row,
                                int64_t* index, double* logp, double* scratch, int64_t scratch_doubles, void* stream) {
  if (!logits) return -1;
  if (type < 0 || type > 3) return -2;
  if (rows < 1 || rows >= MAX_ROWS) return -3;
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
  DrawArgs A{logits, row_stride, col_stride, cols, lengths, u, draws, {temperature, temperature_row}, {top_p, top_p_row}, {min_p, min_p_row},
             {top_k, top_k_row}, index, logp, 0, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
  const Plan p = plan_of(type, rows, cols, draws, cuts_of(A));
  const int64_t need = scratch_of(p, rows);
  if (need > 0 && !scratch) return -20;
  if (need > scratch_doubles) return -21;
  A.mult = p.mult; A.max_cells = p.max_cells;
  if (need > 0) {
    A.best = scratch;
    A.sums = scratch + rows * p.max_cells;
    A.lows = scratch + 2 * rows * p.max_cells;
    A.cut = reinterpret_cast<CutState*>(A.lows + rows * p.groups);
    A.tables = reinterpret_cast<Table*>(A.cut + rows);
    A.lots = scratch + need - rows * lots_of(p);
  }
  hipStream_t st = (hipStream_t)stream;
  if (type == 0) launch<F64>(A, p, rows, st);
  else if (type == 1) launch<F32>(A, p, rows, st);
  else if (type == 2) launch<Half<0>>(A, p, rows, st);
  else launch<Half<1>>(A, p, rows, st);
  return hipGetLastError() == hipSuccess ? 0 : -99;
}
