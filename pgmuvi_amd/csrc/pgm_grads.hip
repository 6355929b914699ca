// pgm_grads.hip -- the norm of a set of gradients and its clipping, over many tensors in few launches.
//
//   n = (sum_t sum_i |g_ti|^p)^(1/p)   (p = 1, 2, inf),     c = min(1, max_norm / (n + 1e-6)),     g' = c g
// over everything (one model's gradients), or for every index b of a leading "member" axis by itself (a batch of fits that
// advance together: each light curve has its own norm and factor).
//
// Launches.  The tensors' addresses travel as kernel arguments (TABLE entries per launch: no table in device memory, nothing to
// upload, and a captured graph holds them like any other kernel's arguments).  Large sets: k_norm_part (partial sums of
// contiguous ranges, at most PARTS workgroups) and then k_scale, whose every workgroup adds the partial sums up again in the
// same fixed order -- or k_norm_final, one workgroup, where only the norm is asked for.  Small sets and batches of members:
// k_member_kept (entries in registers between norm and scaling) or k_member, one workgroup per member, norm and scaling in one
// launch.  No atomics: every result is reproducible bit for bit.
//
// What bounds it: memory, at a copy's rate of 4.9 TB/s on this card (reading alone goes faster).  The norm of 2.1 GB fp64: 358 us,
// 6.0 TB/s.  Clipping 1.07 GB bf16 into other tensors: k_norm_part 221 us (4.9 TB/s) + k_scale 419 (5.1 TB/s of reading and writing);
// in place 617 together, and 227 where nothing exceeds the limit.  The second read is needed, the set does not fit the caches.  The
// norm of 64 MB in 61 fp32 tensors: 16 + 4 us on the GPU, 35 with the host's description of them.  4096 members of 64 KB fp64: 105 us,
// 5.1 TB/s, each read once.
// Small sets are one launch (the five tensors of a fit, 14 numbers: 6 us on the GPU, 17 with the host).
//
// Arithmetic.  All sums are fp64 whatever the tensors' type.  An fp64 square overflows from 1e154 on and vanishes below
// 1e-162: fp64 entries go to one of three accumulators by magnitude (above 2^480, below 2^-480, between), the outer two
// scaled by powers of two, so that the norm is right over the whole range (a diverging fit is where clipping matters).  The
// other types' squares fit fp64 as they are.  The product c g is formed in fp64 and rounded once to the tensor's type (through
// fp32 for the 16-bit types: 2^-24 against their own 2^-8 / 2^-11).
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>
#include <algorithm>
#include <vector>
#include "../../include/pgmuvi_hip.h"

namespace {

constexpr int TABLE = 64;             // tensors per launch (kernel arguments stay below 4 KB)
constexpr int STRIDED_TABLE = 24;     // tensors whose entries are not one contiguous run (136 bytes each)
constexpr int PARTS = 2048;           // partial sums per pass of a large set: 8 workgroups per CU, all resident at once
constexpr int NT = 256;
constexpr int MAX_MEMBERS = 1 << 22;  // 1024 threads each: less than 2^32 of a launch
constexpr int CHUNK = 16384;          // bytes of one tensor a workgroup takes at a time: four 16-byte loads per thread in flight

enum { T_F64 = 0, T_F32 = 1, T_BF16 = 2, T_F16 = 3 };
__host__ __device__ constexpr int type_bytes(int t) { return t == T_F64 ? 8 : t == T_F32 ? 4 : 2; }

struct Entry { const char* in; char* out; int64_t n, in_stride, out_stride; int chunk0; int type; };   // n entries per member; member strides in entries
struct Table { int count, chunks, p, pad; Entry e[TABLE]; };
static_assert(sizeof(Table) <= 3600, "kernel arguments");
struct StridedEntry { const char* in; char* out; int64_t in_member, out_member, size[4], in_stride[4], out_stride[4]; int type, pad; };
struct StridedTable { int count, chunks, p, pad; StridedEntry e[STRIDED_TABLE]; };
static_assert(sizeof(StridedTable) <= 3600, "kernel arguments");

// ---- accumulation --------------------------------------------------------------------------------------------------
struct Acc { double mid, big, small; };

constexpr double BIG = 0x1p480, SMALL = 0x1p-480, UP = 0x1p600, DOWN = 0x1p-600;

template <int TYPE, int P> __device__ __forceinline__ void take(Acc& a, double x) {
  if constexpr (P == 2) {
    if constexpr (TYPE == T_F64) {
      const double m = fabs(x);
      const bool b = m > BIG, s = m < SMALL;
      const double y = x * (b ? DOWN : s ? UP : 1.0), q = y * y;
      a.mid += (b || s) ? 0.0 : q;                              // (a NaN is neither: it lands here)
      a.big += b ? q : 0.0;
      a.small += s ? q : 0.0;
    } else {
      a.mid = __builtin_fma(x, x, a.mid);
    }
  } else if constexpr (P == 1) {
    a.mid += fabs(x);
  } else {
    const double m = fabs(x);
    a.mid = (m > a.mid || m != m) ? m : a.mid;                  // (the comparison fails once a.mid is a NaN: it stays)
  }
}
__device__ __forceinline__ void join(Acc& a, const Acc& b, int p) {
  if (p != 0) { a.mid += b.mid; a.big += b.big; a.small += b.small; }
  else a.mid = (b.mid > a.mid || b.mid != b.mid) ? b.mid : a.mid;
}
__device__ __forceinline__ double norm_of(const Acc& a, int p) {
  if (p != 2) return a.mid;
  if (a.big > 0.0) return sqrt(a.big + a.mid * DOWN * DOWN) * UP;    // (the small ones are below 2^-960 of these)
  if (a.mid == 0.0) return sqrt(a.small) * DOWN;
  return sqrt(a.mid + a.small * DOWN * DOWN);
}
__device__ __forceinline__ double factor_of(double norm, double max_norm) {
  if (max_norm > 1.7976931348623157e308) return 1.0;
  const double c = max_norm / (norm + 1e-6);
  return c > 1.0 ? 1.0 : c;                                     // (a NaN norm gives a NaN factor, an infinite one zero)
}

// sum over the workgroup in a fixed order; every thread gets the result.  red: one Acc per wavefront
template <int THREADS> __device__ __forceinline__ Acc block_join(Acc a, int p, Acc* red) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) {
    Acc o{__shfl_xor(a.mid, s), __shfl_xor(a.big, s), __shfl_xor(a.small, s)};
    join(a, o, p);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  Acc r = red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) join(r, red[w], p);
  return r;
}

// ---- entries of a tensor ----------------------------------------------------------------------------------------------
template <int TYPE> struct Vec;       // 16 bytes of a tensor, aligned to its entries only (gfx950 loads and stores those as one dwordx4)
template <> struct Vec<T_F64> { static constexpr int N = 2; double v[2]; __device__ double get(int i) const { return v[i]; } __device__ void set(int i, double x) { v[i] = x; } };
template <> struct Vec<T_F32> { static constexpr int N = 4; float v[4]; __device__ double get(int i) const { return v[i]; } __device__ void set(int i, double x) { v[i] = (float)x; } };
template <> struct Vec<T_BF16> { static constexpr int N = 8; __hip_bfloat16 v[8]; __device__ double get(int i) const { return (double)__bfloat162float(v[i]); } __device__ void set(int i, double x) { v[i] = __float2bfloat16((float)x); } };
template <> struct Vec<T_F16> { static constexpr int N = 8; __half v[8]; __device__ double get(int i) const { return (double)__half2float(v[i]); } __device__ void set(int i, double x) { v[i] = __float2half((float)x); } };

template <int TYPE> __device__ __forceinline__ double load1(const char* p, int64_t i) {
  if constexpr (TYPE == T_F64) return reinterpret_cast<const double*>(p)[i];
  else if constexpr (TYPE == T_F32) return reinterpret_cast<const float*>(p)[i];
  else if constexpr (TYPE == T_BF16) return (double)__bfloat162float(reinterpret_cast<const __hip_bfloat16*>(p)[i]);
  else return (double)__half2float(reinterpret_cast<const __half*>(p)[i]);
}
template <int TYPE> __device__ __forceinline__ void store1(char* p, int64_t i, double x) {
  if constexpr (TYPE == T_F64) reinterpret_cast<double*>(p)[i] = x;
  else if constexpr (TYPE == T_F32) reinterpret_cast<float*>(p)[i] = (float)x;
  else if constexpr (TYPE == T_BF16) reinterpret_cast<__hip_bfloat16*>(p)[i] = __float2bfloat16((float)x);
  else reinterpret_cast<__half*>(p)[i] = __float2half((float)x);
}

// entries [lo, hi) of one contiguous run, by the whole workgroup
template <int TYPE, int THREADS, int P> __device__ __forceinline__ void run_norm_p(Acc& a, const char* in, int64_t lo, int64_t hi) {
  using V = Vec<TYPE>;
  constexpr int N = V::N, S = type_bytes(TYPE);
  int64_t i = lo + (int64_t)threadIdx.x * N;
  for (; i + 3 * THREADS * N + N <= hi; i += 4 * THREADS * N) {
    V v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) __builtin_memcpy(&v[k], in + (i + k * THREADS * N) * S, 16);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < N; ++j) take<TYPE, P>(a, v[k].get(j));
  }
  for (; i + N <= hi; i += THREADS * N) {
    V v;
    __builtin_memcpy(&v, in + i * S, 16);
#pragma unroll
    for (int j = 0; j < N; ++j) take<TYPE, P>(a, v.get(j));
  }
  for (int64_t k = i; k < hi && k < i + N; ++k) take<TYPE, P>(a, load1<TYPE>(in, k));    // (the one thread whose vector ends past hi)
}
template <int TYPE, int THREADS> __device__ __forceinline__ void run_norm(Acc& a, const char* in, int64_t lo, int64_t hi, int p) {
  if (p == 2) run_norm_p<TYPE, THREADS, 2>(a, in, lo, hi);
  else if (p == 1) run_norm_p<TYPE, THREADS, 1>(a, in, lo, hi);
  else run_norm_p<TYPE, THREADS, 0>(a, in, lo, hi);
}
template <int TYPE> __device__ __forceinline__ void take_p(Acc& a, double x, int p) {
  if (p == 2) take<TYPE, 2>(a, x); else if (p == 1) take<TYPE, 1>(a, x); else take<TYPE, 0>(a, x);
}
template <int TYPE, int THREADS> __device__ __forceinline__ void run_scale(const char* in, char* out, int64_t lo, int64_t hi, double c) {
  using V = Vec<TYPE>;
  constexpr int N = V::N, S = type_bytes(TYPE);
  int64_t i = lo + (int64_t)threadIdx.x * N;
  for (; i + 3 * THREADS * N + N <= hi; i += 4 * THREADS * N) {
    V v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) __builtin_memcpy(&v[k], in + (i + k * THREADS * N) * S, 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[k].set(j, v[k].get(j) * c);
      __builtin_memcpy(out + (i + k * THREADS * N) * S, &v[k], 16);
    }
  }
  for (; i + N <= hi; i += THREADS * N) {
    V v;
    __builtin_memcpy(&v, in + i * S, 16);
#pragma unroll
    for (int j = 0; j < N; ++j) v.set(j, v.get(j) * c);
    __builtin_memcpy(out + i * S, &v, 16);
  }
  for (int64_t k = i; k < hi && k < i + N; ++k) store1<TYPE>(out, k, load1<TYPE>(in, k) * c);
}
#define PGM_BY_TYPE(TYPE, CALL)                  \
  switch (TYPE) {                                \
    case T_F64: CALL(T_F64); break;              \
    case T_F32: CALL(T_F32); break;              \
    case T_BF16: CALL(T_BF16); break;            \
    default: CALL(T_F16); break;                 \
  }

// the chunks [c0, c1) of the table's tensors, one contiguous piece of one tensor at a time: f(entry, first, last)
template <class F> __device__ __forceinline__ void for_pieces(const Table& T, int c0, int c1, F f) {
  if (c0 >= c1) return;
  int lo = 0, hi = T.count - 1;
  while (lo < hi) { const int m = (lo + hi + 1) >> 1; if (T.e[m].chunk0 <= c0) lo = m; else hi = m - 1; }
  for (int t = lo; t < T.count && c0 < c1; ++t) {
    const Entry& e = T.e[t];
    const int end = (t + 1 < T.count) ? T.e[t + 1].chunk0 : T.chunks;
    const int stop = end < c1 ? end : c1;
    const int64_t per = CHUNK / type_bytes(e.type);
    const int64_t first = (int64_t)(c0 - e.chunk0) * per, last = (int64_t)(stop - e.chunk0) * per;
    f(e, first, last < e.n ? last : e.n);
    c0 = stop;
  }
}

// ---- kernels ------------------------------------------------------------------------------------------------------------
// grid: (workgroups per member) x members; partial of workgroup g of member b at part[b * slots + slot0 + g]
__global__ __launch_bounds__(NT) void k_norm_part(Table T, int groups, Acc* __restrict__ part, int64_t slots, int64_t slot0) {
  __shared__ Acc red[NT / 64];
  const int64_t b = blockIdx.x / groups;
  const int g = blockIdx.x % groups;
  const int c0 = (int)((int64_t)T.chunks * g / groups), c1 = (int)((int64_t)T.chunks * (g + 1) / groups);
  Acc a{0.0, 0.0, 0.0};
  for_pieces(T, c0, c1, [&](const Entry& e, int64_t first, int64_t last) {
    const char* in = e.in + b * e.in_stride * type_bytes(e.type);
#define PGM_CALL(TY) run_norm<TY, NT>(a, in, first, last, T.p)
    PGM_BY_TYPE(e.type, PGM_CALL)
#undef PGM_CALL
  });
  a = block_join<NT>(a, T.p, red);
  if (threadIdx.x == 0) part[b * slots + slot0 + g] = a;
}

template <int THREADS> __device__ __forceinline__ Acc join_parts(const Acc* part, int64_t slots, int p, Acc* red) {
  Acc a{0.0, 0.0, 0.0};
  for (int64_t i = threadIdx.x; i < slots; i += THREADS) join(a, part[i], p);
  return block_join<THREADS>(a, p, red);
}
__device__ __forceinline__ void store_norm(void* norm, int norm_f64, int64_t b, double n) {
  if (norm_f64) static_cast<double*>(norm)[b] = n; else static_cast<float*>(norm)[b] = (float)n;
}

__global__ __launch_bounds__(1024) void k_norm_final(const Acc* __restrict__ part, int64_t slots, int p, void* norm, int norm_f64) {
  __shared__ Acc red[16];
  const int64_t b = blockIdx.x;
  const Acc a = join_parts<1024>(part + b * slots, slots, p, red);
  if (threadIdx.x == 0) store_norm(norm, norm_f64, b, norm_of(a, p));
}

__global__ __launch_bounds__(NT) void k_scale(Table T, int groups, const Acc* __restrict__ part, int64_t slots, double max_norm,
                                              void* norm, int norm_f64) {
  __shared__ Acc red[NT / 64];
  const int64_t b = blockIdx.x / groups;
  const int g = blockIdx.x % groups;
  const double n = norm_of(join_parts<NT>(part + b * slots, slots, T.p, red), T.p);
  if (norm && g == 0 && threadIdx.x == 0) store_norm(norm, norm_f64, b, n);
  const double c = factor_of(n, max_norm);
  const int c0 = (int)((int64_t)T.chunks * g / groups), c1 = (int)((int64_t)T.chunks * (g + 1) / groups);
  for_pieces(T, c0, c1, [&](const Entry& e, int64_t first, int64_t last) {
    const int s = type_bytes(e.type);
    const char* in = e.in + b * e.in_stride * s;
    char* out = e.out + b * e.out_stride * s;
    if (c == 1.0 && in == out) return;                          // (nothing to change: times one)
#define PGM_CALL(TY) run_scale<TY, NT>(in, out, first, last, c)
    PGM_BY_TYPE(e.type, PGM_CALL)
#undef PGM_CALL
  });
}

// one workgroup per member: norm and, with `scale`, the scaling behind it
template <int THREADS> __global__ __launch_bounds__(THREADS) void k_member(Table T, int scale, double max_norm, void* norm, int norm_f64) {
  __shared__ Acc red[THREADS / 64];
  const int64_t b = blockIdx.x;
  Acc a{0.0, 0.0, 0.0};
  for (int t = 0; t < T.count; ++t) {
    const Entry& e = T.e[t];
    const char* in = e.in + b * e.in_stride * type_bytes(e.type);
#define PGM_CALL(TY) run_norm<TY, THREADS>(a, in, 0, e.n, T.p)
    PGM_BY_TYPE(e.type, PGM_CALL)
#undef PGM_CALL
  }
  const double n = norm_of(block_join<THREADS>(a, T.p, red), T.p);
  if (threadIdx.x == 0) store_norm(norm, norm_f64, b, n);
  if (!scale) return;
  const double c = factor_of(n, max_norm);
  for (int t = 0; t < T.count; ++t) {
    const Entry& e = T.e[t];
    const int s = type_bytes(e.type);
    const char* in = e.in + b * e.in_stride * s;
    char* out = e.out + b * e.out_stride * s;
    if (c == 1.0 && in == out) continue;
#define PGM_CALL(TY) run_scale<TY, THREADS>(in, out, 0, e.n, c)
    PGM_BY_TYPE(e.type, PGM_CALL)
#undef PGM_CALL
  }
}

// The same for members of one type that fit the workgroup's registers: KEEP slots of one 16-byte vector per thread, each slot a stretch
// of one tensor.  The entries stay there between the norm and the scaling, so that every gradient is read once (4096 members of
// 64 KB: 188 us with a second pass through the cache).  Which tensor a slot belongs to is the host's arithmetic: a lookup per vector
// in the table of tensors held up the loads (175 us)
constexpr int SLOTS = 12;
struct Slot { const char* in; char* out; int64_t n, in_stride, out_stride, first; };
struct SlotTable { int count, p; Slot s[SLOTS]; };
template <int TYPE, int THREADS, int KEEP> __global__ __launch_bounds__(THREADS) void k_member_kept(SlotTable V, int scale, double max_norm, void* norm, int norm_f64) {
  typedef Vec<TYPE> Reg;
  constexpr int N = Reg::N, S = type_bytes(TYPE);
  static_assert(KEEP <= SLOTS, "slots");
  __shared__ Acc red[THREADS / 64];
  const int64_t b = blockIdx.x;
  Reg v[KEEP];
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[k].set(j, 0.0);
    if (k >= V.count) continue;
    const Slot& e = V.s[k];
    const int64_t i = e.first + (int64_t)threadIdx.x * N;
    const char* in = e.in + (b * e.in_stride + i) * S;
    if (i + N <= e.n) __builtin_memcpy(&v[k], in, 16);
    else
#pragma unroll
      for (int j = 0; j < N; ++j) if (i + j < e.n) v[k].v[j] = reinterpret_cast<const Reg*>(in)->v[j];
  }
  Acc a{0.0, 0.0, 0.0};
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
#pragma unroll
    for (int j = 0; j < N; ++j) take_p<TYPE>(a, v[k].get(j), V.p);                            // (zeros add nothing)
    __builtin_amdgcn_sched_barrier(0);                          // (one vector's conversions at a time: all of them do not fit the registers)
  }
  const double n = norm_of(block_join<THREADS>(a, V.p, red), V.p);
  if (threadIdx.x == 0) store_norm(norm, norm_f64, b, n);
  if (!scale) return;
  const double c = factor_of(n, max_norm);
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    if (k >= V.count) continue;
    const Slot& e = V.s[k];
    const int64_t i = e.first + (int64_t)threadIdx.x * N;
    char* out = e.out + (b * e.out_stride + i) * S;
    if (c == 1.0 && out == e.in + (b * e.in_stride + i) * S) continue;                        // (nothing to change: times one)
#pragma unroll
    for (int j = 0; j < N; ++j) v[k].set(j, v[k].get(j) * c);
    if (i + N <= e.n) __builtin_memcpy(out, &v[k], 16);
    else
#pragma unroll
      for (int j = 0; j < N; ++j) if (i + j < e.n) reinterpret_cast<Reg*>(out)->v[j] = v[k].v[j];
    __builtin_amdgcn_sched_barrier(0);
  }
}

// ---- tensors whose entries are not one run: one entry per thread and step, its address from the four sizes -----------------
template <class F> __device__ __forceinline__ void for_strided(const StridedTable& T, int64_t b, int g, int groups, F f) {
  for (int t = 0; t < T.count; ++t) {
    const StridedEntry& e = T.e[t];
    const int64_t n = e.size[0] * e.size[1] * e.size[2] * e.size[3];
    for (int64_t i = (int64_t)g * NT + threadIdx.x; i < n; i += (int64_t)groups * NT) {
      int64_t r = i, in = b * e.in_member, out = b * e.out_member;
#pragma unroll
      for (int d = 3; d >= 0; --d) {
        const int64_t q = r / e.size[d], k = r - q * e.size[d];
        in += k * e.in_stride[d]; out += k * e.out_stride[d];
        r = q;
      }
      f(e, in, out);
    }
  }
}
__global__ __launch_bounds__(NT) void k_norm_part_strided(StridedTable T, int groups, Acc* __restrict__ part, int64_t slots, int64_t slot0) {
  __shared__ Acc red[NT / 64];
  const int64_t b = blockIdx.x / groups;
  const int g = blockIdx.x % groups;
  Acc a{0.0, 0.0, 0.0};
  for_strided(T, b, g, groups, [&](const StridedEntry& e, int64_t in, int64_t) {
#define PGM_CALL(TY) take_p<TY>(a, load1<TY>(e.in, in), T.p)
    PGM_BY_TYPE(e.type, PGM_CALL)
#undef PGM_CALL
  });
  a = block_join<NT>(a, T.p, red);
  if (threadIdx.x == 0) part[b * slots + slot0 + g] = a;
}
__global__ __launch_bounds__(NT) void k_scale_strided(StridedTable T, int groups, const Acc* __restrict__ part, int64_t slots, double max_norm,
                                                      void* norm, int norm_f64) {
  __shared__ Acc red[NT / 64];
  const int64_t b = blockIdx.x / groups;
  const int g = blockIdx.x % groups;
  const double n = norm_of(join_parts<NT>(part + b * slots, slots, T.p, red), T.p);
  if (norm && g == 0 && threadIdx.x == 0) store_norm(norm, norm_f64, b, n);
  const double c = factor_of(n, max_norm);
  for_strided(T, b, g, groups, [&](const StridedEntry& e, int64_t in, int64_t out) {
#define PGM_CALL(TY) store1<TY>(e.out, out, load1<TY>(e.in, in) * c)
    PGM_BY_TYPE(e.type, PGM_CALL)
#undef PGM_CALL
  });
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// May two of the arrays a clipping call touches share memory where one of them is written?  An array is runs of `run` bytes at every
// combination of up to five steps (the member axis and a layout's four dimensions; bytes, largest step first): [lo, lo + reach) holds it.
struct Axis { uint64_t size, step; };
struct Box { Axis a[5]; int n; uint64_t run; };

uint64_t reach_of(const Box& b, int from) {
  uint64_t r = b.run;
  for (int d = from; d < b.n; ++d) r += (b.a[d].size - 1) * b.a[d].step;
  return r;
}
// entries at the same address?  (No for sure where every step clears all the smaller ones)
bool meets_itself(const Box& b) {
  for (int d = 0; d < b.n; ++d) if (b.a[d].step < reach_of(b, d + 1)) return true;
  return false;
}
// Disjoint for sure?  `a` from its axis i on, at zero, and `b` from its axis j on, `at` bytes behind (or, negative, in front).  Over the
// largest step both are laid out in, each lies within one period of it or may reach into the next one: the rests are compared within
// the period they share, and one further.  (Columns of a matrix, blocks of a grid, members' rows in one buffer.)
bool apart(const Box& a, int i, const Box& b, int j, int64_t at) {
  const int64_t ra = (int64_t)reach_of(a, i), rb = (int64_t)reach_of(b, j);
  if (at >= ra || -at >= rb) return true;
  const uint64_t sa = i < a.n ? a.a[i].step : 0, sb = j < b.n ? b.a[j].step : 0;
  const int64_t step = (int64_t)(sa > sb ? sa : sb);
  if (step == 0) return false;                                  // (two runs that meet)
  const int i2 = sa == (uint64_t)step ? i + 1 : i, j2 = sb == (uint64_t)step ? j + 1 : j;
  if ((int64_t)reach_of(a, i2) > step || (int64_t)reach_of(b, j2) > step) return false;       // (interleaved otherwise: not decided here)
  const int64_t d = ((at % step) + step) % step;
  return apart(a, i2, b, j2, d) && apart(a, i2, b, j2, d - step);
}
struct Item { int type; int64_t n; const char* in; char* out; int64_t in_member, out_member; const int64_t* layout; int64_t bytes, chunks; };
Box box_of(const Item& it, int batch, bool write) {
  const int s = type_bytes(it.type), o = write ? 8 : 4;
  Box b{{}, 0, (uint64_t)(it.layout ? s : it.bytes)};
  auto axis = [&](int64_t size, int64_t step) { if (size > 1) b.a[b.n++] = Axis{(uint64_t)size, (uint64_t)step * s}; };
  axis(batch, write ? it.out_member : it.in_member);
  if (it.layout) for (int d = 0; d < 4; ++d) axis(it.layout[d], it.layout[o + d]);
  std::sort(b.a, b.a + b.n, [](const Axis& x, const Axis& y) { return x.step > y.step; });
  return b;
}
struct Span { uint64_t lo, hi; const Item* it; bool write; };
bool any_clash(std::vector<Span>& v, int batch) {
  std::sort(v.begin(), v.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
  for (size_t i = 0; i < v.size(); ++i)
    for (size_t j = i + 1; j < v.size() && v[j].lo < v[i].hi; ++j)
      if ((v[i].write || v[j].write) &&
          !apart(box_of(*v[i].it, batch, v[i].write), 0, box_of(*v[j].it, batch, v[j].write), 0, (int64_t)(v[j].lo - v[i].lo))) return true;
  return false;
}

// One workgroup per member, in one launch: few tensors (one after the other, more take longer than two launches) of no more bytes
// than a CU streams in the time a second launch takes, or, with members for half the chip, than its registers hold.  GPU times in
// fp64, one launch against two: 1 member, 5 tensors, 112 B 6.2 and 7.0 us, 16 KB 6.4 and 7.2, 64 KB 8.6 and 8.1 (a launch less for
// the host), 256 KB 12.5 and 7.4; 16 tensors, 4 KB 10.6 and 7.5;  512 members, 5 tensors, 64 KB 12.2 and 24.6, 320 KB 42 and 39;
// 20 tensors, 64 KB 48 and 29
bool one_launch(int batch, int64_t count, int64_t bytes, bool strided) {
  return !strided && count <= 8 && bytes <= (batch < 128 ? 65536 : 98304);
}

int run_clip(int batch, int count, const uint64_t* in, const uint64_t* out, const int64_t* numel, const unsigned char* type,
             const int64_t* member, const int64_t* layout, int p, double max_norm, void* norm, int norm_f64, double* scratch,
             int64_t scratch_doubles, hipStream_t st) {
  std::vector<Item> flat, loose;
  int64_t per_member = 0, flat_chunks = 0, loose_chunks = 0;
  for (int t = 0; t < count; ++t) {
    if (numel[t] < 0) return -5;
    if (type[t] > T_F16) return -6;
    if (numel[t] == 0) continue;
    if (!in[t]) return -3;
    if (out && !out[t]) return -4;
    const int s = type_bytes(type[t]);
    Item it{type[t], numel[t], (const char*)in[t], out ? (char*)out[t] : nullptr, 0, 0, nullptr, numel[t] * s, 0};
    if (batch > 1) {
      if (!member || member[2 * t] < 0 || member[2 * t + 1] < 0) return -7;
      it.in_member = member[2 * t]; it.out_member = member[2 * t + 1];
    }
    const int64_t* L = layout ? layout + 12 * t : nullptr;
    if (L && L[0] > 0) {
      int64_t n = 1;
      for (int d = 0; d < 4; ++d) { if (L[d] < 1 || L[4 + d] < 0 || L[8 + d] < 0) return -8; n *= L[d]; }
      if (n != numel[t]) return -8;
      it.layout = L; it.chunks = (it.n + 4 * NT - 1) / (4 * NT);
      loose.push_back(it); loose_chunks += it.chunks;
    } else {
      it.chunks = (it.bytes + CHUNK - 1) / CHUNK;
      flat.push_back(it); flat_chunks += it.chunks;
    }
    per_member += it.bytes;
  }
  if (out) {
    std::vector<Span> spans;
    spans.reserve(2 * (flat.size() + loose.size()));
    for (const std::vector<Item>* items : {&flat, &loose})
      for (const Item& it : *items) {
        const Box to = box_of(it, batch, true);
        if (meets_itself(to)) return -12;                        // (entries, or members, written over each other)
        bool same = it.in == it.out && (batch == 1 || it.in_member == it.out_member);
        if (it.layout) for (int d = 0; d < 4; ++d) same = same && (it.layout[d] == 1 || it.layout[4 + d] == it.layout[8 + d]);
        if (!same) spans.push_back(Span{(uint64_t)it.in, (uint64_t)it.in + reach_of(box_of(it, batch, false), 0), &it, false});
        spans.push_back(Span{(uint64_t)it.out, (uint64_t)it.out + reach_of(to, 0), &it, true});
      }
    if (any_clash(spans, batch)) return -12;
  }
  if (flat_chunks > (1 << 30) || loose_chunks > (1 << 30)) return -5;
  const int scale = out ? 1 : 0;

  auto fill = [&](Table& T, size_t i0, size_t i1) {
    T.count = (int)(i1 - i0); T.p = p; T.pad = 0;
    int64_t c = 0;
    for (size_t i = i0; i < i1; ++i) {
      T.e[i - i0] = Entry{flat[i].in, flat[i].out, flat[i].n, flat[i].in_member, flat[i].out_member, (int)c, flat[i].type};
      c += flat[i].chunks;
    }
    T.chunks = (int)c;
  };
  if (one_launch(batch, count, per_member, layout != nullptr)) {
    // slots of 256 threads while eight of them cover the member (8 members share a CU), else of 512 while twelve do
    constexpr int SMALL = 256, FEW = 8, LARGE = 512;
    auto slots = [&](int threads) {
      int64_t n = 0;
      for (const Item& it : flat) n += (it.bytes + 16 * threads - 1) / (16 * threads);
      return n;
    };
    bool same = true;
    for (const Item& it : flat) same = same && it.type == flat[0].type;
    const int threads = slots(SMALL) <= FEW ? SMALL : slots(LARGE) <= SLOTS ? LARGE : 0;
    if (!flat.empty() && same && threads) {
      SlotTable V;
      V.count = 0; V.p = p;
      for (const Item& it : flat)
        for (int64_t i = 0; i < it.n; i += (int64_t)threads * (16 / type_bytes(it.type)))
          V.s[V.count++] = Slot{it.in, it.out, it.n, it.in_member, it.out_member, i};
#define PGM_CALL(TY) do { if (threads == SMALL) hipLaunchKernelGGL((k_member_kept<TY, SMALL, FEW>), dim3(batch), dim3(SMALL), 0, st, V, scale, max_norm, norm, norm_f64); \
                          else hipLaunchKernelGGL((k_member_kept<TY, LARGE, SLOTS>), dim3(batch), dim3(LARGE), 0, st, V, scale, max_norm, norm, norm_f64); } while (0)
      PGM_BY_TYPE(flat[0].type, PGM_CALL)
#undef PGM_CALL
    } else {
      Table T;
      fill(T, 0, flat.size());
      if (per_member <= 8192) hipLaunchKernelGGL(k_member<NT>, dim3(batch), dim3(NT), 0, st, T, scale, max_norm, norm, norm_f64);
      else hipLaunchKernelGGL(k_member<1024>, dim3(batch), dim3(1024), 0, st, T, scale, max_norm, norm, norm_f64);
    }
    return hipGetLastError() == hipSuccess ? 0 : -99;
  }
  if (!scratch) return -13;
  struct Launch { size_t i0, i1; int64_t chunks; int groups; bool strided; int64_t slot0; };
  std::vector<Launch> launches;
  auto plan = [&](const std::vector<Item>& items, size_t width, bool strided) {
    for (size_t i0 = 0; i0 < items.size(); i0 += width) {
      Launch l{i0, std::min(items.size(), i0 + width), 0, 0, strided, 0};
      for (size_t i = l.i0; i < l.i1; ++i) l.chunks += items[i].chunks;
      launches.push_back(l);
    }
  };
  plan(flat, TABLE, false);
  plan(loose, STRIDED_TABLE, true);
  const int64_t all = flat_chunks + loose_chunks;
  int64_t slots = 0;
  for (auto& l : launches) {
    const double share = (double)PARTS / batch * l.chunks / all;
    l.groups = (int)std::max<int64_t>(1, std::min<int64_t>(l.chunks, (int64_t)share));
    l.slot0 = slots;
    slots += l.groups;
  }
  if (slots * batch * 3 > scratch_doubles) return -14;
  Acc* part = reinterpret_cast<Acc*>(scratch);
  for (int pass = 0; pass <= scale; ++pass) {
    for (size_t k = 0; k < launches.size(); ++k) {
      const Launch& l = launches[k];
      const dim3 grid((unsigned)((int64_t)l.groups * batch));
      void* write = k == 0 ? norm : nullptr;
      if (!l.strided) {
        Table T;
        fill(T, l.i0, l.i1);
        if (pass == 0) hipLaunchKernelGGL(k_norm_part, grid, dim3(NT), 0, st, T, l.groups, part, slots, l.slot0);
        else hipLaunchKernelGGL(k_scale, grid, dim3(NT), 0, st, T, l.groups, part, slots, max_norm, write, norm_f64);
      } else {
        StridedTable T;
        T.count = (int)(l.i1 - l.i0); T.chunks = (int)l.chunks; T.p = p; T.pad = 0;
        for (size_t i = l.i0; i < l.i1; ++i) {
          StridedEntry& e = T.e[i - l.i0];
          const Item& it = loose[i];
          e.in = it.in; e.out = it.out; e.in_member = it.in_member; e.out_member = it.out_member; e.type = it.type; e.pad = 0;
          for (int d = 0; d < 4; ++d) { e.size[d] = it.layout[d]; e.in_stride[d] = it.layout[4 + d]; e.out_stride[d] = it.layout[8 + d]; }
        }
        if (pass == 0) hipLaunchKernelGGL(k_norm_part_strided, grid, dim3(NT), 0, st, T, l.groups, part, slots, l.slot0);
        else hipLaunchKernelGGL(k_scale_strided, grid, dim3(NT), 0, st, T, l.groups, part, slots, max_norm, write, norm_f64);
      }
    }
    if (pass == 0 && (!scale || launches.empty()))
      hipLaunchKernelGGL(k_norm_final, dim3(batch), dim3(1024), 0, st, part, slots, p, norm, norm_f64);
  }
  return hipGetLastError() == hipSuccess ? 0 : -99;
}

}  // namespace

extern "C" int64_t pgm_grad_scratch_doubles(int batch, int count, int64_t bytes, int strided) {
  if (batch < 1 || count < 0 || bytes < 0) return 0;
  if (one_launch(batch, count, bytes, strided != 0)) return 0;
  // one partial sum of three doubles per workgroup: PARTS of them, and at most one more per launch and member
  const int64_t launches = (int64_t)count / TABLE + 1 + (int64_t)count / STRIDED_TABLE + 1;
  return 3 * ((int64_t)PARTS + launches * batch);
}

extern "C" int pgm_grad_clip(int batch, int count, const uint64_t* in_host, const uint64_t* out_host, const int64_t* numel_host,
                             const unsigned char* type_host, const int64_t* member_host, const int64_t* layout_host, int p,
                             double max_norm, void* norm, int norm_f64, double* scratch, int64_t scratch_doubles, void* stream) {
  if (batch < 1 || batch >= MAX_MEMBERS) return -1;
  if (count < 0) return -2;
  if (count > 0 && !in_host) return -3;
  if (count > 0 && !numel_host) return -5;
  if (count > 0 && !type_host) return -6;
  if (p < 0 || p > 2) return -9;
  if (out_host && !(max_norm >= 0.0)) return -10;
  if (!norm) return -11;
  try {
    return run_clip(batch, count, in_host, out_host, numel_host, type_host, member_host, layout_host, p, max_norm, norm, norm_f64,
                    scratch, scratch_doubles, (hipStream_t)stream);
  } catch (...) {                                               // (out of host memory)
    return -98;
  }
}
