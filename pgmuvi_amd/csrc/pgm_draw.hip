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
#include "../../include/pgmuvi_hip.h"

namespace {

typedef unsigned long long u64;
constexpr int NT = 1024, NW = NT / 64, BINS = 2048, MAX_CELLS = 4096;
constexpr int64_t MAX_COLS = 1 << 24;                             // (2^24 weights of at most one, in steps of 2^-40, fit 64 bits)
constexpr int64_t EVERY = INT64_MAX;

// ---- values and their keys: unsigned integers in the same order; -0 is +0, NaN is -inf ------------------------------------
struct F64 {
  typedef double raw; typedef u64 key;
  static __device__ __forceinline__ double value(raw x) { return x; }
  static __device__ __forceinline__ key to_key(raw x) {
    x = x != x ? -__builtin_inf() : x + 0.0;
    const u64 b = (u64)__double_as_longlong(x);
    return (b >> 63) ? ~b : b | (1ull << 63);
  }
  static __device__ __forceinline__ double of_key(key k) { return __longlong_as_double((long long)((k >> 63) ? k & ~(1ull << 63) : ~k)); }
};
struct F32 {
  typedef float raw; typedef uint32_t key;
  static __device__ __forceinline__ key to_key(float x) {
    x = x != x ? -__builtin_inff() : x + 0.0f;
    const uint32_t b = __float_as_uint(x);
    return (b >> 31) ? ~b : b | (1u << 31);
  }
  static __device__ __forceinline__ double of_key(key k) { return (double)__uint_as_float((k >> 31) ? k & ~(1u << 31) : ~k); }
};
template <int F16BIT> struct Half {                              // bf16 (0) and fp16 (1): the 16-bit patterns are ordered the same way
  typedef uint16_t raw; typedef uint32_t key;
  static __device__ __forceinline__ key to_key(uint16_t b) {
    const uint32_t inf = F16BIT ? 0x7c00u : 0x7f80u, mag = b & 0x7fffu;
    if (mag > inf) return 0xffffu - (0x8000u | inf);
    if (mag == 0) return 0x8000u;
    return (b >> 15) ? 0xffffu - b : b | 0x8000u;
  }
  static __device__ __forceinline__ double of_key(key k) {
    const uint16_t b = (uint16_t)((k & 0x8000u) ? k & 0x7fffu : 0xffffu - k);
    if constexpr (F16BIT) { __half_raw r; r.x = b; return (double)__half2float(__half(r)); }
    else return (double)__uint_as_float((uint32_t)b << 16);
  }
};

struct Param { double v; const double* p; };                    // one number for every row, or one per row
struct ParamI { int64_t v; const int64_t* p; };
struct DrawArgs {
  const void* logits; int64_t row_stride, col_stride, cols;
  const int64_t* lengths;                                       // entries of each row, or null: cols
  const double* u; int64_t draws;
  Param temperature, top_p, min_p; ParamI top_k;
  int64_t* index; double* logp;
};

template <class K> struct Cut { K key; int64_t idx; };          // kept: key above, or equal and index not above
template <class K> __device__ __forceinline__ bool before(const Cut<K>& c, K key, int64_t i) { return key > c.key || (key == c.key && i <= c.idx); }

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s);
  return v;
}
template <class V> __device__ __forceinline__ V wave_scan(V v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) { const V o = __shfl_up(v, s); if (lane >= s) v += o; }
  return v;
}

struct Bins { uint32_t count[BINS]; u64 hi[BINS], lo[BINS]; };
struct Shared {
  union { Bins bins; double cells[MAX_CELLS]; };
  u64 red[NW][3];
  u64 found[6];
  double sums[NW];
};

__device__ __forceinline__ double mass_of(u64 hi, u64 lo) { return (double)hi * 0x1p-40 + (double)lo * 0x1p-80; }

template <class F> struct Row {
  typedef typename F::key K;
  const typename F::raw* x; int64_t stride, n;
  double best, t;
  __device__ __forceinline__ K key(int64_t i) const { return F::to_key(x[i * stride]); }
  __device__ __forceinline__ double z(K k) const { const double l = F::of_key(k); return l == best ? 0.0 : (l - best) / t; }
  __device__ __forceinline__ double weight(K k) const { return exp(z(k)); }
};

// The bin that holds the cut, by wavefront 0: `want` entries (counts), or `share` of the weight (bins hold everything that
// counts on the first pass: total < 0 asks for it).  found = bin, entries before it, entries in it, hi / lo before it.
template <bool WEIGHTED> __device__ __forceinline__ void find_bin(Shared& S, u64 before_n, u64 before_hi, u64 before_lo, u64 want, double share, double& target) {
  __syncthreads();
  if (threadIdx.x < 64) {
    constexpr int PER = BINS / 64;
    const int lane = threadIdx.x, b0 = lane * PER;
    u64 n = 0, hi = 0, lo = 0;
    for (int k = 0; k < PER; ++k) { n += S.bins.count[b0 + k]; if (WEIGHTED) { hi += S.bins.hi[b0 + k]; lo += S.bins.lo[b0 + k]; } }
    const u64 sn = wave_scan(n), shi = WEIGHTED ? wave_scan(hi) : 0, slo = WEIGHTED ? wave_scan(lo) : 0;
    if (WEIGHTED && target < 0.0) target = share * mass_of(__shfl(shi, 63), __shfl(slo, 63));
    auto reached = [&](u64 an, u64 ahi, u64 alo) { return WEIGHTED ? mass_of(before_hi + ahi, before_lo + alo) >= target : before_n + an >= want; };
    const u64 mask = __ballot(reached(sn, shi, slo));
    const int owner = mask ? __ffsll(mask) - 1 : 63 - __clzll(__ballot(n > 0) | 1ull);       // (always reached, but for a rounding of the target)
    if (lane == owner) {
      u64 an = sn - n, ahi = shi - hi, alo = slo - lo;
      int b = b0;
      for (int k = 0; k < PER; ++k) {
        const u64 c = S.bins.count[b0 + k];
        if (c == 0) continue;
        b = b0 + k;
        if (k + 1 == PER || reached(an + c, ahi + (WEIGHTED ? S.bins.hi[b] : 0), alo + (WEIGHTED ? S.bins.lo[b] : 0))) break;
        bool more = false;                                      // (the last bin with entries ends the search whatever the comparison says)
        for (int j = k + 1; j < PER; ++j) more = more || S.bins.count[b0 + j] != 0;
        if (!more) break;
        an += c;
        if (WEIGHTED) { ahi += S.bins.hi[b]; alo += S.bins.lo[b]; }
      }
      S.found[0] = (u64)b; S.found[1] = before_n + an; S.found[2] = S.bins.count[b]; S.found[3] = before_hi + ahi; S.found[4] = before_lo + alo;
      S.found[5] = (u64)__double_as_longlong(target);
    }
  }
  __syncthreads();
}
__device__ __forceinline__ void clear_bins(Shared& S) {
  __syncthreads();
  for (int b = threadIdx.x; b < BINS; b += NT) { S.bins.count[b] = 0; S.bins.hi[b] = 0; S.bins.lo[b] = 0; }
  __syncthreads();
}

// the cut behind the first `want` entries of what `have` keeps (WEIGHTED: behind the shortest beginning with `share` of its weight)
template <bool WEIGHTED, class F> __device__ Cut<typename F::key> select(const Row<F>& R, Shared& S, typename F::key kmin, typename F::key kmax,
                                                                         Cut<typename F::key> have, u64 want, double share) {
  typedef typename F::key K;
  K hi = kmax, lo = kmin;
  u64 bn = 0, bhi = 0, blo = 0;
  double target = -1.0;
  for (;;) {
    const u64 span = (u64)(hi - lo);
    const int shift = span < BINS ? 0 : 64 - __clzll(span) - 11;
    clear_bins(S);
    for (int64_t i = threadIdx.x; i < R.n; i += NT) {
      const K k = R.key(i);
      if (k < lo || k > hi || !before(have, k, i)) continue;
      const int b = (int)((u64)(hi - k) >> shift);
      atomicAdd(&S.bins.count[b], 1u);
      if (WEIGHTED) {
        const double w = R.weight(k) * 0x1p40;
        const u64 whi = (u64)w, wlo = (u64)((w - (double)whi) * 0x1p40);
        if (whi) atomicAdd(&S.bins.hi[b], whi);
        if (wlo) atomicAdd(&S.bins.lo[b], wlo);
      }
    }
    find_bin<WEIGHTED>(S, bn, bhi, blo, want, share, target);
    const u64 bin = S.found[0], in_bin = S.found[2];
    bn = S.found[1]; bhi = S.found[3]; blo = S.found[4]; target = __longlong_as_double((long long)S.found[5]);
    const K top = (K)(hi - (K)(bin << shift));
    const u64 width = (1ull << shift) - 1;
    const K bottom = (u64)(top - lo) <= width ? lo : (K)(top - (K)width);
    Cut<K> cut{bottom, EVERY};
    if (in_bin == 1 || (!WEIGHTED && bn + in_bin == want)) return cut;
    if (shift == 0) {                                           // equal values: the first m of them by index
      u64 m = WEIGHTED ? 1 : want - bn;
      if (WEIGHTED) {
        const double w = R.weight(top), above = mass_of(bhi, blo);
        const double guess = ceil((target - above) / w);
        m = guess >= (double)in_bin ? in_bin : guess < 1.0 ? 1 : (u64)guess;
        while (m > 1 && above + (double)(m - 1) * w >= target) --m;
        while (m < in_bin && above + (double)m * w < target) ++m;
      }
      if (m >= in_bin) return cut;
      int64_t i0 = 0, i1 = R.n - 1;
      u64 passed = 0;
      for (;;) {
        const u64 ispan = (u64)(i1 - i0);
        const int ishift = ispan < BINS ? 0 : 64 - __clzll(ispan) - 11;
        clear_bins(S);
        for (int64_t i = i0 + threadIdx.x; i <= i1; i += NT)
          if (R.key(i) == top && before(have, top, i)) atomicAdd(&S.bins.count[(u64)(i - i0) >> ishift], 1u);
        double none = 0.0;
        find_bin<false>(S, passed, 0, 0, m, 0.0, none);
        const int64_t first = i0 + (int64_t)(S.found[0] << ishift), last = first + (int64_t)((1ull << ishift) - 1);
        passed = S.found[1];
        const u64 here = S.found[2];
        i0 = first;
        i1 = last < i1 ? last : i1;
        if (ishift == 0 || passed + here == m) { cut.key = top; cut.idx = i1; return cut; }
        __syncthreads();
      }
    }
    hi = top; lo = bottom;
    __syncthreads();                                            // (found has been read by everybody)
  }
}
template <class K> __device__ __forceinline__ Cut<K> tighter(const Cut<K>& a, const Cut<K>& b) {
  if (a.key != b.key) return a.key > b.key ? a : b;
  return a.idx < b.idx ? a : b;
}

template <class F> __global__ __launch_bounds__(NT) void k_draw(DrawArgs A) {
  typedef typename F::key K;
  __shared__ Shared S;
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  int64_t n = A.cols;
  if (A.lengths) { n = A.lengths[row]; n = n < 0 ? 0 : n > A.cols ? A.cols : n; }
  Row<F> R;
  R.x = static_cast<const typename F::raw*>(A.logits) + row * A.row_stride; R.stride = A.col_stride; R.n = n;

  // the best and the lowest key above -inf, and how many there are
  K neg;
  if constexpr (sizeof(typename F::raw) == 2) neg = F::to_key((typename F::raw)0xffffu);      // (a NaN: the key of -inf)
  else neg = F::to_key((typename F::raw)(-__builtin_inf()));
  u64 kmax = 0, kmin = ~0ull, valid = 0;
  for (int64_t i = t; i < n; i += NT) {
    const K k = R.key(i);
    if (k <= neg) continue;
    kmax = kmax > (u64)k ? kmax : (u64)k; kmin = kmin < (u64)k ? kmin : (u64)k; ++valid;
  }
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) {
    const u64 a = __shfl_xor(kmax, s), b = __shfl_xor(kmin, s);
    kmax = kmax > a ? kmax : a; kmin = kmin < b ? kmin : b; valid += __shfl_xor(valid, s);
  }
  if (lane == 0) { S.red[wave][0] = kmax; S.red[wave][1] = kmin; S.red[wave][2] = valid; }
  __syncthreads();
  kmax = 0; kmin = ~0ull; valid = 0;
  for (int w = 0; w < NW; ++w) {
    kmax = kmax > S.red[w][0] ? kmax : S.red[w][0]; kmin = kmin < S.red[w][1] ? kmin : S.red[w][1]; valid += S.red[w][2];
  }
  int64_t* index = A.index + row * A.draws;
  double* logp = A.logp ? A.logp + row * A.draws : nullptr;
  if (valid == 0) {                                             // nothing to draw from
    for (int64_t s = t; s < A.draws; s += NT) { index[s] = -1; if (logp) logp[s] = -__builtin_inf(); }
    return;
  }
  R.best = F::of_key((K)kmax);
  const double temp = A.temperature.p ? A.temperature.p[row] : A.temperature.v;
  R.t = temp < 1e300 ? temp : 1e300;
  const double top_p = A.top_p.p ? A.top_p.p[row] : A.top_p.v;
  double min_p = A.min_p.p ? A.min_p.p[row] : A.min_p.v;
  min_p = min_p > 1.0 ? 1.0 : min_p;
  int64_t top_k = A.top_k.p ? A.top_k.p[row] : A.top_k.v;
  if (!(temp > 0.0) || top_p <= 0.0) top_k = 1;                 // the best entry alone (the first of equal ones)
  if (!(temp > 0.0)) R.t = 1.0;

  Cut<K> cut{neg, -1};
  if (top_k > 0 && (u64)top_k < valid) cut = tighter(cut, select<false, F>(R, S, (K)kmin, (K)kmax, cut, (u64)top_k, 0.0));
  if (top_p > 0.0 && top_p < 1.0) cut = tighter(cut, select<true, F>(R, S, (K)kmin, (K)kmax, cut, 0, top_p));
  __syncthreads();                                              // (the cells take the bins' place)

  auto kept = [&](int64_t i) -> double {                        // the weight of entry i, zero if it is not kept
    const K k = R.key(i);
    if (k <= neg || !before(cut, k, i)) return 0.0;
    const double w = R.weight(k);
    return w < min_p ? 0.0 : w;
  };
  int64_t steps = (n + 64 * (int64_t)MAX_CELLS - 1) / (64 * (int64_t)MAX_CELLS);
  steps = steps < 4 ? 4 : steps;
  const int64_t width = 64 * steps;
  const int cells = (int)((n + width - 1) / width);
  for (int c = wave; c < cells; c += NW) {
    const int64_t i0 = c * width + lane;
    double s = 0.0;
    for (int64_t j = 0; j < steps; ++j) { const int64_t i = i0 + 64 * j; if (i < n) s += kept(i); }
    s = wave_sum(s);
    if (lane == 0) S.cells[c] = s;
  }
  __syncthreads();
  {                                                             // running sums over the cells: four per thread, wavefronts, workgroup
    constexpr int PER = MAX_CELLS / NT;
    double v[PER], s = 0.0;
#pragma unroll
    for (int k = 0; k < PER; ++k) { const int c = t * PER + k; s += c < cells ? S.cells[c] : 0.0; v[k] = s; }
    const double inc = wave_scan(s);
    if (lane == 63) S.sums[wave] = inc;
    __syncthreads();
    double base = inc - s;
    for (int w = 0; w < wave; ++w) base += S.sums[w];
#pragma unroll
    for (int k = 0; k < PER; ++k) { const int c = t * PER + k; if (c < cells) S.cells[c] = base + v[k]; }
    __syncthreads();
  }
  const double Z = S.cells[cells - 1], log_z = log(Z);
  for (int64_t s = wave; s < A.draws; s += NW) {                // one wavefront per draw
    double target = A.u[row * A.draws + s] * Z;
    target = target > 0.0 ? target : target == target ? 0.0 : Z;   // (u outside [0, 1): the first or the last kept entry)
    auto first_above = [&](double x, bool or_equal) {
      int a = 0, b = cells;
      while (a < b) { const int m = (a + b) >> 1; const double f = S.cells[m]; if (f > x || (or_equal && f >= x)) b = m; else a = m + 1; }
      return a;
    };
    int c = first_above(target, false);
    if (c == cells) { c = first_above(Z, true); target = __builtin_inf(); }
    double base = c ? S.cells[c - 1] : 0.0;
    int64_t found = -1, last = -1;
    for (int64_t j = 0; j < steps && found < 0; ++j) {
      const int64_t i = c * width + 64 * j + lane;
      const double w = i < n ? kept(i) : 0.0, inc = wave_scan(w);
      const u64 hit = __ballot(w > 0.0 && base + inc > target), some = __ballot(w > 0.0);
      if (hit) found = c * width + 64 * j + __ffsll(hit) - 1;
      if (some) last = c * width + 64 * j + 63 - __clzll(some);
      base += __shfl(inc, 63);
    }
    if (found < 0) found = last;                                // (the cell's own sum and this one differ by a rounding)
    if (lane == 0) {
      index[s] = found;
      if (logp) logp[s] = R.z(R.key(found)) - log_z;
    }
  }
}

}  // namespace

extern "C" int pgm_draw_indices(const void* logits, int type, int64_t rows, int64_t cols, int64_t row_stride, int64_t col_stride,
                                const int64_t* lengths, const double* u, int64_t draws,
                                double temperature, const double* temperature_row, int64_t top_k, const int64_t* top_k_row,
                                double top_p, const double* top_p_row, double min_p, const double* min_p_row,
                                int64_t* index, double* logp, void* stream) {
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
  DrawArgs A{logits, row_stride, col_stride, cols, lengths, u, draws, {temperature, temperature_row}, {top_p, top_p_row}, {min_p, min_p_row},
             {top_k, top_k_row}, index, logp};
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)rows);
  if (type == 0) hipLaunchKernelGGL(k_draw<F64>, grid, dim3(NT), 0, st, A);
  else if (type == 1) hipLaunchKernelGGL(k_draw<F32>, grid, dim3(NT), 0, st, A);
  else if (type == 2) hipLaunchKernelGGL(k_draw<Half<0>>, grid, dim3(NT), 0, st, A);
  else hipLaunchKernelGGL(k_draw<Half<1>>, grid, dim3(NT), 0, st, A);
  return hipGetLastError() == hipSuccess ? 0 : -99;
}
