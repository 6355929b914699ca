// pgm_kernels.hip -- device kernels of the exact-GP hot path (gfx950 only).
//
// One evaluation = SM kernel build -> blocked factorisation sweep (Cholesky + the
// inverse factor in the same sweep) -> A^-1 tiles with the gradient contraction
// fused into their epilogue -> a tiny finalise.  See DESIGN.md for the algorithm
// and data layout; reference call sites are cited in include/pgmuvi_hip.h.
#include "pgm_internal.h"
#include "pgm_exp.h"

namespace {

constexpr double PI = 3.14159265358979323846;
constexpr double TWO_PI_SQ = 2.0 * PI * PI;
// The per-point factor x_i v_qd is staged as x_i v_qd pi sqrt(2): the Gaussian envelope exp(-2 pi^2 (x_i v - x_j v)^2) is then
// exp(-(difference of the staged values)^2) -- the same scale-then-subtract form as GPyTorch's, one multiplication less per pair.
constexpr double PI_SQRT2 = 4.44288293815836624702;

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// The same sum without the LDS crossbar (wave_sum's __shfl_xor is ds_bpermute_b32, ~100 cycles of latency per step and two per
// double): four DPP steps inside each row of 16 lanes -- quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror, row_mirror -- then the
// four row totals by v_readlane.  Every lane returns the total.  A different association than wave_sum's butterfly: used where
// sums are compared to rounding (the gradient partial sums of k_small), never where bits are (the value's sums).
__device__ __forceinline__ double wave_sum_dpp(double v) {
#define PGM_DPP_STEP(CTRL) do { \
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, true); \
    const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, true); \
    v += __hiloint2double(hi, lo); } while (0)
  PGM_DPP_STEP(0xB1);
  PGM_DPP_STEP(0x4E);
  PGM_DPP_STEP(0x141);
  PGM_DPP_STEP(0x140);
#undef PGM_DPP_STEP
  auto rl = [](double x, int l) { return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), l), __builtin_amdgcn_readlane(__double2loint(x), l)); };
  return (rl(v, 0) + rl(v, 16)) + (rl(v, 32) + rl(v, 48));
}

// idx -> (i <= j) of the column-major enumeration of an upper triangle
__device__ __forceinline__ void tri_decode(int idx, int& i, int& j) {
  int jj = (int)((sqrt(8.0 * (double)idx + 1.0) - 1.0) * 0.5);
  while ((jj + 1) * (jj + 2) / 2 <= idx) ++jj;
  while (jj * (jj + 1) / 2 > idx) --jj;
  j = jj;
  i = idx - jj * (jj + 1) / 2;
}

// Batches: which (tile, light curve) a workgroup takes.  The dispatcher deals workgroups round-robin over the 8 XCDs in
// launch order (x fastest, then z), each XCD with an L2 of its own: with the plain (blockIdx.x, blockIdx.z) = (tile, light
// curve) reading, the tiles of one light curve -- which share their operand panels -- are spread over all eight L2s and every
// panel is fetched from the memory side up to eight times (measured, 64 x N=2048: 25 % L2 hit rate in the trailing update,
// 3.9 TB/s at the fabric).  Remapped, the workgroups that share an XCD (equal launch index mod 8) work through the light
// curves  g, g+8, g+16, ...  one after the other, all tiles of one before the next.  A pure relabelling (bijective whenever
// the batch is a multiple of 8, identity otherwise): placement is a speed matter only, every tile is still computed once.
__device__ __forceinline__ void xcd_batch_remap(int& x, int& b) {
  const int X = (int)gridDim.x, Z = (int)gridDim.z;
  if (Z & 7) return;
  const int L = x + X * b;
  const int g = L & 7, s = L >> 3;
  const int ci = s / X;
  b = __builtin_amdgcn_readfirstlane(g + 8 * ci);
  x = __builtin_amdgcn_readfirstlane(s - ci * X);
}

// ---------------------------------------------------------------------------
// Per-point factors.  GPyTorch evaluates cos(2 pi (x_i mu - x_j mu)); the angle
// difference is expanded (cos a cos b + sin a sin b) so the N^2 pass needs no
// trigonometry, only the N*Q*d sincospi here.
// The caller's output pointers of this evaluation go to device memory: k_precompute is launched with them as arguments,
// k_finalize is replayed from a graph captured once per problem shape and reads them from there.
// points of light curve b / its index in the caller's arrays (ragged batches: pgm_internal.h)
__device__ __forceinline__ int pts(const PgmDev& P, int b) { return P.nvec ? P.nvec[b] : P.n; }
__device__ __forceinline__ int caller_slot(const PgmDev& P, int b) { return P.cmap ? P.cmap[b] : b; }
// block rows light curve b really has (a trimmed ragged launch set, pgm_internal.h) -- otherwise the set's
__device__ __forceinline__ int own_rows(const PgmDev& P, int b) { return P.trim ? (P.nvec[b] + NB - 1) / NB : P.nb; }
// Workgroup -> (member b, index x among the member's own workgroups, the member's block rows) in the 1-D grid of a trimmed
// ragged set (RagClasses, pgm_internal.h); false: a workgroup past the end of its XCD's list (the lists differ by a member
// per class at most).
__device__ __forceinline__ bool rag_decode(const RagClasses& rc, int& x, int& b, int& rows) {
  const int g = (int)blockIdx.x & 7;
  int s = (int)blockIdx.x >> 3;
  for (int c = 0; c < rc.n; ++c) {
    const int z0 = (int)rc.z0[c], z1 = (int)rc.z0[c + 1], X = rc.x[c];
    const int first = z0 + ((g - z0) & 7);                       // the class's first member that is this XCD's
    const int cnt = first < z1 ? (z1 - first + 7) >> 3 : 0;
    if (s < cnt * X) {
      const int i = s / X;
      x = __builtin_amdgcn_readfirstlane(s - i * X);
      b = __builtin_amdgcn_readfirstlane(first + 8 * i);
      rows = __builtin_amdgcn_readfirstlane((int)rc.nb[c]);
      return true;
    }
    s -= cnt * X;
  }
  return false;
}

__device__ __forceinline__ void publish_output_pointers(const PgmDev& P) {
  if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 64 && P.outp) {
    P.outp[0] = (unsigned long long)P.mll; P.outp[1] = (unsigned long long)P.g_w; P.outp[2] = (unsigned long long)P.g_mu;
    P.outp[3] = (unsigned long long)P.g_v; P.outp[4] = (unsigned long long)P.g_noise; P.outp[5] = (unsigned long long)P.g_mean;
    P.outp[6] = (unsigned long long)P.info_out;
    P.outp[7] = (unsigned long long)P.seq;                   // (the evaluation's number: the last diagonal block stamps the status with it)
    P.outp[8] = (unsigned long long)P.cstride;
  }
}

// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_precompute(PgmDev P) {
  const int b = blockIdx.z;
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int cb = caller_slot(P, b), n = pts(P, b);           // (the caller's arrays: slot cb, P.cstride points apart)
  if (blockIdx.x == 0 && threadIdx.x == 0) P.info[b] = 0;
  publish_output_pointers(P);
  if (blockIdx.x == 0 && threadIdx.x < P.q + 2 * P.qd) {
    const int s = threadIdx.x;
    double val;
    if (s < P.q) val = P.w[(int64_t)cb * P.q + s];
    else if (s < P.q + P.qd) val = P.mu[(int64_t)cb * P.qd + (s - P.q)];
    else val = P.v[(int64_t)cb * P.qd + (s - P.q - P.qd)];
    P.hyp[(int64_t)b * (PGM_MAX_QD * 3) + s] = val;
  }
  if (i >= P.np) return;
  double* pre = P.pre + b * P.sPre;
  const bool valid = i < n;
  const int64_t ci = (int64_t)cb * P.cstride + i;
  for (int dd = 0; dd < P.d; ++dd) {
    const double xi = valid ? P.x[ci * P.d + dd] : 0.0;
    pre[(int64_t)(3 * P.qd + dd) * P.np + i] = xi;
    for (int q = 0; q < P.q; ++q) {
      const int qd = q * P.d + dd;
      const double mu = P.mu[(int64_t)cb * P.qd + qd], v = P.v[(int64_t)cb * P.qd + qd];
      double s, c;
      sincospi(2.0 * (xi * mu), &s, &c);
      pre[(int64_t)(qd * 3 + 0) * P.np + i] = c;
      pre[(int64_t)(qd * 3 + 1) * P.np + i] = s;
      pre[(int64_t)(qd * 3 + 2) * P.np + i] = xi * v * PI_SQRT2;
    }
  }
  const int64_t vi = (int64_t)b * P.sVec + i;
  P.r[vi] = valid ? (P.y[ci] - P.mean[ci]) : 0.0;
  // everything added to the diagonal: fixed noise + scalar noise + jitter (identity on the padding)
  P.diagadd[vi] = valid ? ((P.noise ? P.noise[ci] : 0.0) + P.noise_scalar + (P.noise_scalar_dev ? P.noise_scalar_dev[cb] : 0.0) + P.jitter) : 0.0;
}

// stage the per-point factor slices of block row `ib` and block column `jb` in LDS
__device__ __forceinline__ void stage_factors(const PgmDev& P, const double* pre, int ib, int jb,
                                              double* rowd, double* cold) {
  const int total = P.pre_slots * NB;
  for (int e = threadIdx.x; e < total; e += NTHREADS) {
    const int slot = e / NB, m = e % NB;
    rowd[e] = pre[(int64_t)slot * P.np + ib * NB + m];
    cold[e] = pre[(int64_t)slot * P.np + jb * NB + m];
  }
}

// k(x_m, x_n) from staged factors (m, n tile-local)
template <int D, int ORDER>
__device__ __forceinline__ double sm_pair(const double* rowd, const double* cold, const double* wl,
                                          int Q, int m, int n) {
  double S[D];
#pragma unroll
  for (int dd = 0; dd < D; ++dd) S[dd] = 0.0;
  double K1 = 0.0;
  for (int q = 0; q < Q; ++q) {
    double prod = 1.0;
#pragma unroll
    for (int dd = 0; dd < D; ++dd) {
      const int qd = q * D + dd;
      const double ds = rowd[(qd * 3 + 2) * NB + m] - cold[(qd * 3 + 2) * NB + n];
      const double e = exp_neg(-(ds * ds));
      const double cc = rowd[(qd * 3 + 0) * NB + m] * cold[(qd * 3 + 0) * NB + n] +
                        rowd[(qd * 3 + 1) * NB + m] * cold[(qd * 3 + 1) * NB + n];
      if (ORDER == 0) S[dd] += wl[q] * e * cc; else prod *= e * cc;
    }
    if (ORDER != 0) K1 += wl[q] * prod;
  }
  if (ORDER != 0) return K1;
  double K = 1.0;
#pragma unroll
  for (int dd = 0; dd < D; ++dd) K *= S[dd];
  return K;
}

// ---------------------------------------------------------------------------
// A = K + diag(noise + noise_scalar + jitter), upper block triangle only, padded
// with the identity.  One workgroup per 128x128 tile; a wave stores one full row
// (1 KiB) per instruction.
// ---------------------------------------------------------------------------
constexpr int BUILD_SPLIT_1D = 4, BUILD_SPLIT_SMALL = 16, BUILD_SPLIT_BIG = 2;
// 1-D kernel matrix: 1/SPLIT of the tile (ib, jb) -- rows part*NB/SPLIT ... -- by 256 threads (tid), factors staged in LDS.
// Shared by k_build and by the build workers beside diagonal block 0 (k_diag).
template <int SPLIT>
__device__ __forceinline__ void build_part_1d(const PgmDev& P, const double* rowd, const double* cold, const double* wl,
                                              int b, int ib, int jb, int part, int tid, const double* dadd = nullptr) {
  double* A = P.A + b * P.sA;
  const int n = pts(P, b);
  const int c2 = (tid & 63) * 2, rg = tid >> 6;
    // 1-D: mixtures outermost, the thread's two column factors in registers, its 32 x 2 entries accumulated in
    // registers: three LDS reads (the row's factors, broadcast) per two entries and mixture instead of nine
    constexpr int RR = NB / 4 / SPLIT;                     // rows per thread
    const int row0 = part * (NB / SPLIT);
    double acc[RR][2];
#pragma unroll
    for (int rr = 0; rr < RR; ++rr) { acc[rr][0] = 0.0; acc[rr][1] = 0.0; }
    for (int q = 0; q < P.q; ++q) {
      const double wq = wl[q];
      const double* cq = cold + q * 3 * NB;
      const double* rq = rowd + q * 3 * NB;
      // (the mixture weight rides on the thread's column factors: 4 multiplications per mixture instead of one per pair.
      //  24 fp64 instructions per pair and mixture are left -- the difference, its square, 19 for the exponential, 3 for the
      //  weighted cosine of the angle difference and its accumulation)
      const double cc0 = wq * cq[c2], cc1 = wq * cq[c2 + 1], cs0 = wq * cq[NB + c2], cs1 = wq * cq[NB + c2 + 1];
      const double cv0 = cq[2 * NB + c2], cv1 = cq[2 * NB + c2 + 1];
#pragma unroll
      for (int rr = 0; rr < RR; ++rr) {
        const int m = row0 + rg + 4 * rr;
        const double rc = rq[m], rs = rq[NB + m], rv = rq[2 * NB + m];
        const double d0 = rv - cv0, d1 = rv - cv1;
        acc[rr][0] = __builtin_fma(exp_neg_fast(-(d0 * d0)), __builtin_fma(rc, cc0, rs * cs0), acc[rr][0]);
        acc[rr][1] = __builtin_fma(exp_neg_fast(-(d1 * d1)), __builtin_fma(rc, cc1, rs * cs1), acc[rr][1]);
      }
    }
#pragma unroll
    for (int rr = 0; rr < RR; ++rr) {
      const int gi = ib * NB + row0 + rg + 4 * rr;
      v2d out;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int gj = jb * NB + c2 + u;
        double val = acc[rr][u];
        if (gi < n && gj < n) { if (gi == gj) val += dadd ? dadd[gi - ib * NB] : P.diagadd[b * P.sVec + gi]; }
        else val = (gi == gj) ? 1.0 : 0.0;
        out[u] = val;
      }
      *reinterpret_cast<v2d*>(A + (int64_t)gi * P.ld + jb * NB + c2) = out;
    }
}

// ---------------------------------------------------------------------------
// Device-resident fit: one optimiser iteration of pgmuvi/trainers.py:177-195 --
// constraint transforms, the evaluation above, the chain rule back to the raw parameters, the SGD / Adam / AdamW
// update, the loss and parameter log -- is two small kernels around the evaluation's launch sequence, all of it one
// hipGraph replayed per iteration with no host work in between.  Raw parameter vector (P entries):
//   [ mean: constant, or d weights + bias (linear) | w (Q) | mu (Q d) | v (Q d) | (learned scalar noise) ].
// ---------------------------------------------------------------------------
struct FitDev {
  int P, n, d, q, qd, nmean, has_noise, optimizer, max_iter;      // nmean: 1 (constant mean) or d+1 (linear); optimizer: 0 SGD, 1 Adam, 2 AdamW
  const double* x;      // [n][d] (linear mean)
  double lr, beta1, beta2, eps, weight_decay;
  double* raw;          // [P] in/out
  const int* ckind;     // [P] 0 none, 1 softplus + lb, 2 ub - softplus(-raw), 3 lb + span sigmoid(raw)
  const double* ca;     // [P] lb (kinds 1, 3) or ub (kind 2)
  const double* cb;     // [P] span (kind 3)
  double* theta;        // [P] constrained values of this iteration
  double* mean_vec;     // [n]
  double* noise_scalar; // [1]
  double* m1;           // [P] Adam first moment
  double* m2;           // [P] Adam second moment
  int* it;              // [1] iterations done so far
  int* it_host;         // host-mapped copy of it (+ [1]: the evaluation's status, written by the evaluation itself): the host reads the log without a device copy
  double* loss_hist;    // [max_iter]
  double* raw_hist;     // [max_iter][P] raw parameters after each step
  // priors on the constrained parameters (MAP): the reference's ExactMarginalLogLikelihood adds sum log p(theta) before the
  // division by N (pgmuvi/lightcurve.py:3273-3322 registers Normal and LogNormal priors)
  const int* pkind;     // [P] 0 none, 1 Normal(loc, scale), 2 LogNormal(loc, scale)
  const double* ploc;   // [P]
  const double* pscale; // [P]
  const double* clip;   // [1] largest norm of the gradient with respect to the raw vector a step takes, or -1: no limit
};

__device__ __forceinline__ double softplus_d(double x) { return x > 20.0 ? x : log1p(exp(x)); }
__device__ __forceinline__ double sigmoid_d(double x) { return 1.0 / (1.0 + exp(-x)); }

__device__ __forceinline__ double fit_theta(const FitDev& F, int p) {
  const double r = F.raw[p];
  if (F.ckind[p] == 1) return softplus_d(r) + F.ca[p];
  if (F.ckind[p] == 2) return F.ca[p] - softplus_d(-r);
  if (F.ckind[p] == 3) return sigmoid_d(r) * F.cb[p] + F.ca[p];
  return r;
}

// Short light curves (one of at most 55 tiles; round 6: also with two input dimensions): per-point factors and kernel matrix in ONE launch in front of the graph --
// an evaluation of N = 89 points is five dependent launches of which the first two do microseconds of work.  A workgroup
// computes the factors of its tile's 128 rows and 128 columns itself, straight from the caller's arrays into LDS (4 sincospi per
// thread at Q = 4) and builds its sixteenth of the tile from them (build_part_1d, the code of k_build); the workgroups of the
// diagonal tiles also leave their block row's factors, residual and diagonal addend in the workspace, where the later
// kernels expect what k_precompute writes -- the same expressions, hence the same bits.
// FIT (pgm_fit_*: the device-resident optimiser loop): the constrained parameters come from the raw vector -- every workgroup
// transforms the (at most 51) parameters for itself, workgroup 0 leaves them in F.theta for the step at the end of the iteration --
// and the mean is the constant (or linear) mean module's: k_fit_pre, k_precompute and k_build in one launch.
template <bool FIT, int D = 1, int ORDER = 0>
__global__ __launch_bounds__(256) void k_prebuild(PgmDev P, FitDev F) {
  constexpr int SPLIT = BUILD_SPLIT_SMALL;
  const int b = blockIdx.z, t = threadIdx.x;
  const int part = blockIdx.x % SPLIT;
  int ib, jb;
  tri_decode(blockIdx.x / SPLIT, ib, jb);
  extern __shared__ __attribute__((aligned(16))) double sm[];      // 2*pre_slots*NB + PGM_MAX_QD + NB (+ 64: FIT) doubles
  double* rowd = sm;
  double* cold = sm + P.pre_slots * NB;
  double* wl = cold + P.pre_slots * NB;
  double* dloc = wl + PGM_MAX_QD;
  double* thl = dloc + NB;                                      // [64] (FIT) constrained parameters
  const int cb = caller_slot(P, b), n = pts(P, b);
  const int Q = P.q, QD = Q * D;
  if (blockIdx.x == 0 && t == 0) P.info[b] = 0;
  publish_output_pointers(P);
  if (FIT) {
    if (t < F.P) {
      const double th = fit_theta(F, t);
      thl[t] = th;
      if (blockIdx.x == 0) { F.theta[t] = th; if (F.has_noise && t == F.P - 1) F.noise_scalar[0] = th; }
    }
    __syncthreads();
  }
  // parameter s of [w (Q) | mu (Q D) | v (Q D)]
  auto hyper = [&](int s3) -> double {
    if (FIT) return thl[F.nmean + s3];
    if (s3 < Q) return P.w[(int64_t)cb * Q + s3];
    if (s3 < Q + QD) return P.mu[(int64_t)cb * QD + (s3 - Q)];
    return P.v[(int64_t)cb * QD + (s3 - Q - QD)];
  };
  const double nscal = FIT ? (F.has_noise ? thl[F.P - 1] : 0.0) : P.noise_scalar + (P.noise_scalar_dev ? P.noise_scalar_dev[cb] : 0.0);
  if (blockIdx.x == 0 && t < Q + 2 * QD) P.hyp[(int64_t)b * (PGM_MAX_QD * 3) + t] = hyper(t);
  if (t < Q) wl[t] = hyper(t);
  const bool writer = (ib == jb) && part == 0;                  // (uniform) this workgroup leaves block row ib's per-point values behind
  double* pre = P.pre + b * P.sPre;
  // points of the row block (side 0) and of the column block (side 1): one (point, side) per thread and round
  for (int e = t; e < 2 * NB; e += 256) {
    const int side = e >> 7, m = e & (NB - 1);
    const int i = (side ? jb : ib) * NB + m;
    const bool valid = i < n;
    const int64_t ci = (int64_t)cb * P.cstride + i;
    double* fac = side ? cold : rowd;
    double xd[D];
#pragma unroll
    for (int dd = 0; dd < D; ++dd) {
      xd[dd] = valid ? P.x[ci * D + dd] : 0.0;
      fac[(3 * QD + dd) * NB + m] = xd[dd];
    }
    for (int qd = 0; qd < QD; ++qd) {
      const double xi = xd[D == 1 ? 0 : qd % D];
      const double mu = hyper(Q + qd), v = hyper(Q + QD + qd);
      double sn, cs;
      sincospi(2.0 * (xi * mu), &sn, &cs);
      fac[(qd * 3 + 0) * NB + m] = cs;
      fac[(qd * 3 + 1) * NB + m] = sn;
      fac[(qd * 3 + 2) * NB + m] = xi * v * PI_SQRT2;
      if (writer && side == 0) {
        pre[(int64_t)(qd * 3 + 0) * P.np + i] = cs;
        pre[(int64_t)(qd * 3 + 1) * P.np + i] = sn;
        pre[(int64_t)(qd * 3 + 2) * P.np + i] = xi * v * PI_SQRT2;
      }
    }
    if (side == 0) {
      const double da = valid ? ((P.noise ? P.noise[ci] : 0.0) + nscal + P.jitter) : 0.0;
      dloc[m] = da;
      if (writer) {
        const int64_t vi = (int64_t)b * P.sVec + i;
#pragma unroll
        for (int dd = 0; dd < D; ++dd) pre[(int64_t)(3 * QD + dd) * P.np + i] = xd[dd];
        double mean_i;
        if (FIT) {
          mean_i = thl[F.nmean - 1];                             // the constant, or the bias of a linear mean (its d weights first)
          if (F.nmean > 1) for (int dd = 0; dd < D; ++dd) mean_i += xd[dd] * thl[dd];
        } else mean_i = valid ? P.mean[ci] : 0.0;
        P.r[vi] = valid ? (P.y[ci] - mean_i) : 0.0;
        P.diagadd[vi] = da;
      }
    }
  }
  __syncthreads();
  if constexpr (D == 1) {
    build_part_1d<SPLIT>(P, rowd, cold, wl, b, ib, jb, part, t, dloc);
  } else {                                                      // (k_build<2, ORDER>'s loop on this workgroup's sixteenth of the tile)
    double* A = P.A + b * P.sA;
    const int c2 = (t & 63) * 2, rg = t >> 6;
    constexpr int RR = NB / 4 / SPLIT;
    for (int rr = part * RR; rr < (part + 1) * RR; ++rr) {
      const int m = rg + 4 * rr;
      const int gi = ib * NB + m;
      v2d out;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int nloc = c2 + u, gj = jb * NB + nloc;
        double val;
        if (gi < n && gj < n) {
          val = sm_pair<D, ORDER>(rowd, cold, wl, Q, m, nloc);
          if (gi == gj) val += dloc[m];
        } else {
          val = (gi == gj) ? 1.0 : 0.0;
        }
        out[u] = val;
      }
      *reinterpret_cast<v2d*>(A + (int64_t)gi * P.ld + jb * NB + c2) = out;
    }
  }
}


template <int D, int ORDER, int SPLIT1 = (D == 1 ? BUILD_SPLIT_1D : 1)>
__global__ __launch_bounds__(256) void k_build(PgmDev P) {
  const int b = blockIdx.z;
  int ib, jb;
  // (1-D: a workgroup builds a quarter of a tile, 32 rows: 2112 workgroups even out over the 256 CUs where 528 did not;
  //  a sixteenth, 8 rows, when the whole call has only a few tiles -- short light curves: 9 -> 5 us at N=128.
  //  2-D: whole tiles, or sixteenths when the call has few tiles -- the reference's 2-D examples have 225 and 250 points, three
  //  tiles: one workgroup per tile took 48 of the evaluation's 152 us, round 6)
  constexpr int SPLIT = SPLIT1;
  const int part = blockIdx.x % SPLIT;
  if (P.build_beside) { ib = 0; jb = blockIdx.x / SPLIT; }      // block row 0 only: the rest is built beside diagonal block 0 (k_diag)
  else tri_decode(blockIdx.x / SPLIT, ib, jb);
  if (jb >= own_rows(P, b)) return;                              // (trimmed ragged set: a tile the light curve does not have; ib <= jb)
  extern __shared__ __attribute__((aligned(16))) double sm[];      // 2*pre_slots*NB + PGM_MAX_QD doubles
  double* rowd = sm;
  double* cold = sm + P.pre_slots * NB;
  double* wl = cold + P.pre_slots * NB;
  const double* pre = P.pre + b * P.sPre;
  stage_factors(P, pre, ib, jb, rowd, cold);
  if (threadIdx.x < P.q) wl[threadIdx.x] = P.hyp[(int64_t)b * (PGM_MAX_QD * 3) + threadIdx.x];
  __syncthreads();
  double* A = P.A + b * P.sA;
  const int c2 = (threadIdx.x & 63) * 2, rg = threadIdx.x >> 6;
  if (D == 1) {
    build_part_1d<SPLIT>(P, rowd, cold, wl, b, ib, jb, part, threadIdx.x);
    return;
  }
  const int n = pts(P, b);
  constexpr int RR = NB / 4 / SPLIT;                             // rows per thread
  for (int rr = part * RR; rr < (part + 1) * RR; ++rr) {
    const int m = rg + 4 * rr;
    const int gi = ib * NB + m;
    v2d out;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int nloc = c2 + u, gj = jb * NB + nloc;
      double val;
      if (gi < n && gj < n) {
        val = sm_pair<D, ORDER>(rowd, cold, wl, P.q, m, nloc);
        if (gi == gj) val += P.diagadd[b * P.sVec + gi];
      } else {
        val = (gi == gj) ? 1.0 : 0.0;
      }
      out[u] = val;
    }
    *reinterpret_cast<v2d*>(A + (int64_t)gi * P.ld + jb * NB + c2) = out;
  }
}

// ---------------------------------------------------------------------------
// Diagonal block k (128x128, on the critical path of every step):
//   U_kk = chol_upper(A_kk),  V_kk = U_kk^-T (both orientations, for the row solve),
//   the block's share of log det,  z_k = V_kk r_k  and  alpha_k = V_kk^T z_k.
// The block lives in LDS and is processed as 8x8 sub-blocks of 16x16 -- the same
// right-looking sweep as the outer algorithm, one level down:
//   (a) one wavefront factors the 16x16 diagonal sub-block in registers (a column per
//       lane; lanes 16-31 carry the identity so the same instruction stream yields the
//       inverse factor), pivots broadcast with v_readlane;
//   (b) the other sub-blocks of block row s are multiplied by that inverse (MFMA);
//   (c) trailing sub-blocks T_ij -= U_si^T U_sj and R_ij -= U_si^T V_sj (MFMA), while
//       wave 0 already factors the next diagonal sub-block (look-ahead).
// T (upper) and the evolving inverse factor (strictly lower) share one LDS image.
// ---------------------------------------------------------------------------
constexpr int DB = 16;
constexpr int PM = NB + 16;
constexpr int DIAG_THREADS = 1024;        // 16 wavefronts: the chain wave, 14 workers, one bookkeeper


__device__ __forceinline__ double readlane_d(double x, int l) {
  int lo = __double2loint(x), hi = __double2hiint(x);
  lo = __builtin_amdgcn_readlane(lo, l);
  hi = __builtin_amdgcn_readlane(hi, l);
  return __hiloint2double(hi, lo);
}

// 1/sqrt(d): hardware seed + one Newton step (relative error ~1e-15)
__device__ __forceinline__ double rsqrt_nr(double d) {
  const double y = __builtin_amdgcn_rsq(d);
  const double e = __builtin_fma(-d * y, y, 1.0);
  return __builtin_fma(0.5 * y, e, y);
}

// The diagonal block on ONE workgroup of 16 wavefronts (round 3 form).  The 128x128 block is 8x8 sub-blocks of 16x16; step s
// factors sub-block (s, s) on the chain wave, solves block row s and applies it to everything behind it -- the same sweep one
// level down.  Every sub-block lives in the REGISTERS of one worker wavefront for the whole kernel, in the f64 MFMA C layout
// (lane (g, n): rows g + 4r of column n) -- which is also the A- and the B-fragment layout of the products it enters later,
// so a block is read from memory once, its accumulator never travels, and only FINISHED block rows go through LDS (as the
// operands of the others).  Before: all sub-blocks in LDS, read and written by every update (270 KB of LDS traffic per step).
//   wave 0            the chain: potrf of (s+1, s+1) while the workers apply block row s; it also solves its own copy of
//                     (s, s+1) and applies it to (s+1, s+1), so that it never waits for more than the two barriers of a step
//   waves 4, 8, 12    its SIMD-mates (a wavefront w runs on SIMD w % 4) keep the books / store V_ss: no MFMA on the chain's SIMD
//   the other twelve  workers; sub-block (i, j) belongs to DIAG_OWN[worker][slot] -- found by search: the 7 blocks of a row on
//                     7 different workers, and per step at most 3, 3, 3, 3, 2, 2, 1 active blocks per worker (the lower bound)
// The arithmetic per sub-block is what it always was (4 chained MFMAs per update or solve, steps in order): results are bit
// for bit those of rounds 1-2.
constexpr int DIAG_WORKERS = 12, DIAG_SLOTS = 6;
alignas(8) __constant__ unsigned char DIAG_OWN[DIAG_WORKERS][8] = {   // (a worker reads its row as one 64-bit scalar load)
       // (i << 4) | j, 0xff: none
  {0x02, 0x36, 0x43, 0x44, 0x55, 0x64, 0xff, 0xff}, {0x03, 0x13, 0x34, 0x51, 0x65, 0x66, 0xff, 0xff},
  {0x04, 0x16, 0x24, 0x31, 0x56, 0x62, 0xff, 0xff}, {0x20, 0x35, 0x42, 0x52, 0x74, 0xff, 0xff, 0xff},
  {0x17, 0x27, 0x60, 0x71, 0xff, 0xff, 0xff, 0xff}, {0x05, 0x15, 0x37, 0x41, 0x50, 0x75, 0xff, 0xff},
  {0x07, 0x33, 0x47, 0x67, 0x76, 0xff, 0xff, 0xff}, {0x22, 0x23, 0x32, 0x57, 0x73, 0xff, 0xff, 0xff},
  {0x14, 0x25, 0x40, 0x63, 0x72, 0xff, 0xff, 0xff}, {0x01, 0x26, 0x45, 0x54, 0x70, 0xff, 0xff, 0xff},
  {0x06, 0x10, 0x46, 0x61, 0xff, 0xff, 0xff, 0xff}, {0x12, 0x21, 0x30, 0x53, 0x77, 0xff, 0xff, 0xff}};

struct DiagCtx {
  double* prow;     // LDS [2][8][256]: the solved block row of step s (parity s & 1), sub-block j row-major = fragment r at [64 r + lane]
  double* dg;       // LDS [8][256]: diagonal sub-block i with the steps < i-1 applied (its owner's last word; the chain applies step i-1)
  double* sup;      // LDS [8][256]: sub-block (i, i+1) with the steps < i applied, unsolved (the chain solves its own copy)
  double* uiS;      // uiS[k*16+m] = V_ss[m][k]
  double* udg;      // U_pp (square roots of the pivots)
  double* Akk;      // global diagonal block of the matrix
  int64_t ld;
  double* Dinv0;    // global Uinv  [p][m]
  double* Dinv1;    // global Uinv^T = V [k][n]
  double* dump;     // LDS scratch (one slot per lane) that absorbs predicated-off stores
};

// LDS-only barrier: global stores issued earlier keep draining in the background
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ v4d diag_load_block(const DiagCtx& c, int i, int j, int lane) {
  const int g = lane >> 4, n = lane & 15;
  v4d v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = c.Akk[(int64_t)(i * DB + g + 4 * r) * c.ld + j * DB + n];
  return v;
}

// (a) one wavefront: Cholesky of the 16x16 sub-block s (`ua`, C layout) plus its inverse factor.
// The block and an identity (whose image under the same row operations is V = u^-T)
// are held in the f64 MFMA C layout (lane (g, n) = rows g+4r of column n).  Pivots go
// in mini-panels of 4 rows: the panel is exchanged through LDS so that every lane
// holds the 4 panel rows of its column, is factored with uniform multipliers
// (v_readlane), and the rank-4 trailing update of both images is one MFMA each:
//   acc -= P^T P  ==  mfma(-row, row, acc)   (the panel row IS the A and B fragment).
// Leaves V_ss in block s of the block row's LDS image (zero above its diagonal by construction: the identity's image
// only ever takes multiples of earlier rows), its transpose in uiS, the pivots' square roots in udg.
// Every lane gets the value its column holds in each of the wavefront's four 16-lane rows: p[q] = x of lane (q, n).  Three
// gfx950 lane swaps per 32-bit half (v_permlane32_swap: [x0 x1 x0 x1], [x2 x3 x2 x3]; v_permlane16_swap of each with itself),
// no LDS (the exchange through a 1-KB LDS buffer, rounds 1-2, waited behind the workers' LDS traffic; N=1000 0.308 -> 0.307 ms).
typedef unsigned v2u_sw __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void rows_to_all(double x, double (&p)[4]) {
  unsigned h[2] = {(unsigned)__double2loint(x), (unsigned)__double2hiint(x)};
  unsigned o[4][2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const v2u_sw r = __builtin_amdgcn_permlane32_swap(h[w], h[w], false, false);
    const v2u_sw lo = __builtin_amdgcn_permlane16_swap(r[0], r[0], false, false);
    const v2u_sw hi = __builtin_amdgcn_permlane16_swap(r[1], r[1], false, false);
    o[0][w] = lo[0]; o[1][w] = lo[1]; o[2][w] = hi[0]; o[3][w] = hi[1];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) p[q] = __hiloint2double((int)o[q][1], (int)o[q][0]);
}

__device__ __forceinline__ void diag_potrf16(const DiagCtx& c, int s, int lane, v4d ua, bool barrier) {
  const int g = lane >> 4, n = lane & 15;
  v4d va;                                     // identity image (C layout)
#pragma unroll
  for (int r = 0; r < 4; ++r) va[r] = (g + 4 * r == n) ? 1.0 : 0.0;
  double fa[4], fb[4];
  // No test inside the pivot chain: a non-positive pivot turns into NaN (rsq of a negative) or
  // inf and poisons everything after it; the first bad diagonal entry is located once, after
  // the block is finished (bookkeeping wave), which keeps ~5 instructions per pivot off the chain.
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    double pa[4], pb[4];
    rows_to_all(ua[m], pa);
    rows_to_all(va[m], pb);
#pragma unroll
    for (int pl = 0; pl < 4; ++pl) {
      const double dp = readlane_d(pa[pl], 4 * m + pl);
      const double rs = rsqrt_nr(dp);
      pa[pl] *= rs;
      pb[pl] *= rs;
#pragma unroll
      for (int ql = pl + 1; ql < 4; ++ql) {
        const double mult = readlane_d(pa[pl], 4 * m + ql);
        pa[ql] = __builtin_fma(-mult, pa[pl], pa[ql]);
        pb[ql] = __builtin_fma(-mult, pb[pl], pb[ql]);
      }
    }
    const double ra = (g == 0) ? pa[0] : (g == 1) ? pa[1] : (g == 2) ? pa[2] : pa[3];
    const double rb = (g == 0) ? pb[0] : (g == 1) ? pb[1] : (g == 2) ? pb[2] : pb[3];
    fa[m] = ra;
    fb[m] = rb;
    if (m < 3) {
      ua = __builtin_amdgcn_mfma_f64_16x16x4f64(-ra, ra, ua, 0, 0, 0);
      va = __builtin_amdgcn_mfma_f64_16x16x4f64(-ra, rb, va, 0, 0, 0);
    }
    // The second barrier of the previous step ("block row s-1 is in LDS") is nothing this wavefront waits for -- it only has to
    // be counted: met here, one mini-panel into the factorisation, the workers' row solves are over and the chain never idles at it.
    if (barrier && m == 0) lds_barrier();                     // (wave-uniform)
  }
  double* mydump = c.dump + lane;
  double* vss = c.prow + (s & 1) * (NB / DB) * DB * DB + s * DB * DB + lane;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = g + 4 * r;
    vss[64 * r] = fb[r];                           // V_ss, row-major (U_ss above its diagonal is needed by nobody)
    c.uiS[n * DB + i] = fb[r];                     // uiS[k*16+m] = V[m][k]
    double* dst = (n == i) ? (c.udg + s * DB + i) : mydump;
    *dst = fa[r];                                  // U_ii = sqrt(pivot)
  }
}

// (b) X <- V_ss X for a sub-block of block row s held in the C layout (= the B-fragment layout: k-step r is x[r])
__device__ __forceinline__ v4d diag_solve(const DiagCtx& c, const v4d& x, int lane) {
  const int kq = lane >> 4, n = lane & 15;
  double a[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) a[r] = c.uiS[(4 * r + kq) * DB + n];
  v4d acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(a[r], x[r], acc, 0, 0, 0);
  return acc;
}

__device__ __forceinline__ void diag_put(double* dst, const v4d& v, int lane) {      // one sub-block into an LDS image
#pragma unroll
  for (int r = 0; r < 4; ++r) dst[64 * r + lane] = v[r];
}
__device__ __forceinline__ v4d diag_get(const double* src, int lane) {
  v4d v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = src[64 * r + lane];
  return v;
}

// finished block (s, j), j <= s, of V = U^-T: to both inverse images, straight from the registers.  A CU retires only ~10 B/clk
// of stores: they are issued right behind the step that finished the block and drain beside the arithmetic of the next ones.
// (The transposed image leaves as 32-byte pieces.  Measured and not kept, both no faster: whole 128-byte row segments from a
//  transposed read of the block row's LDS image, and from X^T made by four MFMAs against an identity -- the write path counts
//  bytes, and the workers' matrix pipes are what the early steps run out of.)
// which: 1 = the row-major image, 2 = the transposed one, 3 = both.  (The zero triangles are cleared once, at workspace creation.)
__device__ __forceinline__ void diag_store_v(const DiagCtx& c, int s, int j, const v4d& v, int lane, int which = 3) {
  const int kq = lane >> 4, n = lane & 15;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = kq + 4 * r;
    if (j < s || n <= i) {
      if (which & 1) c.Dinv1[(s * DB + i) * NB + j * DB + n] = v[r];
      if (which & 2) c.Dinv0[(j * DB + n) * NB + s * DB + i] = v[r];
    }
  }
}

// Where the diagonal block's sub-blocks come from: the matrix in memory (k_diag), or straight from the per-point factors of a
// short light curve staged in LDS (k_small, below: the block is never written to memory).
struct LoadFromMatrix {
  __device__ __forceinline__ v4d operator()(const DiagCtx& c, int i, int j, int lane) const { return diag_load_block(c, i, j, lane); }
};
// What a worker does with the finished block row of step s (LDS image `row`) besides its updates: nothing (k_diag), or its share of
// the products A^-1 (i, j) += V(s, i)^T V(s, j) (k_small: the inverse accumulates while the chain factors the next sub-block).
struct NoRowHook {
  __device__ __forceinline__ void operator()(int, const double*, int) const {}
};

// a worker wavefront: its sub-blocks through all steps.  (The slot table stays packed in one scalar register pair and is
// decoded where it is used: two dozen wave-uniform integers kept live across the loop made the compiler spill scalars.)
// PAD_STORES false / SKIP_PAD true (k_small): the sub-blocks of the identity padding -- rows and columns beyond the light curve's
// last sub-block row, zero or identity for good -- are neither solved, published, updated nor stored (k_diag runs their
// arithmetic on zeros and stores them: the block row's image and the inverse images are read whole by the kernels behind it).
template <class Load = LoadFromMatrix, class Hook = NoRowHook, bool PAD_STORES = true, bool SKIP_PAD = false>
__device__ __forceinline__ void diag_worker(const DiagCtx& c, int q, int lane, int nse, const Load load = Load(), Hook&& hook = Hook()) {
  constexpr int NS = NB / DB;
  const unsigned long long pack = *reinterpret_cast<const unsigned long long*>(DIAG_OWN[q]);
#define SLOT_E(t) ((int)((pack >> (8 * (t))) & 0xffull))
  v4d acc[DIAG_SLOTS];
#pragma unroll
  for (int t = 0; t < DIAG_SLOTS; ++t) {
    const int e = SLOT_E(t), i = e >> 4, j = e & 15;
    if (e != 0xff && i <= j) acc[t] = load(c, i, j, lane);
    else acc[t] = v4d{0.0, 0.0, 0.0, 0.0};
  }
  for (int s = 0; s < nse; ++s) {
    double* row = c.prow + (s & 1) * NS * DB * DB;
    lds_barrier();                                             // V_ss of this step is in LDS
#pragma unroll
    for (int t = 0; t < DIAG_SLOTS; ++t) {
      const int e = SLOT_E(t), i = e >> 4, j = e & 15;
      if (i == s && j != s && (!SKIP_PAD || j < nse)) {        // my block of block row s: solve, publish
        acc[t] = diag_solve(c, acc[t], lane);
        diag_put(row + j * DB * DB, acc[t], lane);
      }
    }
    lds_barrier();                                             // block row s is in LDS
#pragma unroll
    for (int t = 0; t < DIAG_SLOTS; ++t) {
      const int e = SLOT_E(t), i = e >> 4, j = e & 15;
      // steps whose block row is applied to this block: U (i < j): 0 .. i-1;  V (i > j): j .. i-1 (it is zero before);
      // diagonal: 0 .. i-2 (the chain applies i-1 itself);  none: never
      const int lo = (i > j) ? j : 0, hi = (e == 0xff) ? 0 : (i == j) ? i - 1 : i;
      if (s >= lo && s < hi && (!SKIP_PAD || (i < nse && j < nse))) {     // C(i,j) -= U(s,i)^T B(s,j);  B is U(s,j) (j>s), V(s,j) (j<s) or V_ss
        const double* pa = row + i * DB * DB + lane;
        const double* pb = row + j * DB * DB + lane;
        double a[4], b[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) { a[r] = -pa[64 * r]; b[r] = pb[64 * r]; }
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t] = __builtin_amdgcn_mfma_f64_16x16x4f64(a[r], b[r], acc[t], 0, 0, 0);
        if (i == j && s == i - 2) diag_put(c.dg + i * DB * DB, acc[t], lane);              // over to the chain
        if (j == i + 1 && s == i - 1) diag_put(c.sup + i * DB * DB, acc[t], lane);
      }
    }
#pragma unroll
    for (int t = 0; t < DIAG_SLOTS; ++t) {
      const int e = SLOT_E(t), i = e >> 4, j = e & 15;
      if (i == s && j < s) diag_store_v(c, s, j, acc[t], lane);
    }
    // (the hook's work on block row s goes behind the step's updates: early steps have many updates and few products of the
    //  inverse, late steps the other way round.  Between the step's two barriers instead -- on block row s-1, whose image stays
    //  until row s+1 is published -- it held the chain up at the second barrier: same-box A/B in k_small, N=89 52.7k against
    //  50.0k clock ticks to the end of the chain, 74.6k / 73.9k for the kernel; N=128 108.0k / 107.0k)
    hook(s, row, lane);
  }
  // block rows of identity padding (the last diagonal block of a light curve whose length is no multiple of 128): zero blocks
  // (PAD_STORES false, k_small: prediction, the only reader of a single block's inverse images, completes them itself)
  if constexpr (PAD_STORES) {
#pragma unroll
    for (int t = 0; t < DIAG_SLOTS; ++t) {
      const int e = SLOT_E(t), i = e >> 4, j = e & 15;
      if (i >= nse && i < NS && j < i) diag_store_v(c, i, j, acc[t], lane);
    }
  }
#undef SLOT_E
}

// the chain wavefront
template <class Load = LoadFromMatrix>
__device__ __forceinline__ void diag_chain(const DiagCtx& c, int lane, int nse, const Load load = Load()) {
#ifdef PGM_DIAG_STAMPS
  long long st_[40]; int sn_ = 0;
#define STAMP() do { if (sn_ < 40) st_[sn_++] = __builtin_amdgcn_s_memtime(); } while (0)
#else
#define STAMP() do {} while (0)
#endif
  STAMP();
  __builtin_amdgcn_s_setprio(3);
  v4d d = load(c, 0, 0, lane);
  v4d x = load(c, 0, 1, lane);                                // what step 0 needs beyond (0, 0) comes straight from memory
  v4d dn = load(c, 1, 1, lane);
  // pass s: the first barrier of step s, the chain's own solve and update, then the factorisation of sub-block s+1 (the
  // factorisation is a long piece of straight-line code: ONE copy of it, pass -1 is sub-block 0 -- the workgroup's
  // neighbour CU shares the instruction cache with it and runs filler tiles)
#pragma clang loop unroll(disable)
  for (int s = -1; s < nse; ++s) {
    if (s >= 0) {
      lds_barrier();
      STAMP();
      if (s + 1 < nse) {
        if (s > 0) { x = diag_get(c.sup + s * DB * DB, lane); dn = diag_get(c.dg + (s + 1) * DB * DB, lane); }
        const v4d u = diag_solve(c, x, lane);                  // U(s, s+1): the chain's own copy, the bits of its owner's
        d = dn;
#pragma unroll
        for (int r = 0; r < 4; ++r) d = __builtin_amdgcn_mfma_f64_16x16x4f64(-u[r], u[r], d, 0, 0, 0);
      }
      STAMP();
    }
    if (s + 1 < nse) diag_potrf16(c, s + 1, lane, d, __builtin_amdgcn_readfirstlane(s) >= 0);
    else if (s >= 0) lds_barrier();                            // (nse = 0, a block of padding: no step, no barrier)
    STAMP();
  }
#ifdef PGM_DIAG_STAMPS
  if (lane == 0 && blockIdx.z == 0) {      // clock ticks: start, potrf(0), then per step: barrier A, solve + update, potrf(s+1) with barrier B inside
    printf("chain: ");
    for (int q = 1; q < sn_; ++q) printf("%d ", (int)(st_[q] - st_[0]));
    printf("\n");
  }
#endif
#undef STAMP
}

// Filler role of the fused diagonal-block launch.  While workgroup 0 factors block k on one CU
// (a ~26 us latency-bound chain) the other 255 CUs would idle; instead the same launch carries
// trailing-update tiles of later block rows (the rows and sources the host's plan selects, below) --
// work that neither this diagonal block nor the following row solve depends on.  A filler
// workgroup is the same 16 wavefronts as the factoring one and multiplies one 128x128 tile at a
// time, a 32x32 sub-tile per wavefront.
// (direct form of the multiply loop, pgm_gemm.h: fragments straight from memory, four k-steps in flight per wavefront;
//  the staged LDS form of rounds 1-2 -- 45.2 us for a 256-deep filler tile against 41 -- is gone)
using CfgFill = TileCfg<128, 128, 32, 32, 4, DIAG_THREADS, KB, true>;
static_assert(CfgFill::LDS_DOUBLES <= NB * PM, "the filler's LDS stages must fit the diagonal block image");

// (A persistent variant -- one filler workgroup per CU looping over tiles with the next tile's C
//  values and first operand chunk prefetched -- was measured and rejected: at 1024 threads the
//  128-VGPR cap makes the extra 32 registers spill into the multiply loop.)
//
// Which finished block rows ("sources") a filler tile of block row r applies is the host's choice,
// per launch: the last one or two sources before k_end, or none (the row sits this launch out).  One source per
// launch for every row is the plain schedule; when that makes more tiles than CUs (two rounds of
// ~23 us each against a 28 us diagonal block) every other row waits one launch and then applies two
// sources in one pass (k-depth 256: the C tile is read and written once for twice the flops, and
// the launch needs one round).
// The plan travels as two bit masks over the block rows (kernel arguments = scalar registers: decoding the
// tile index must not touch memory): skip bit set = the row sits the launch out, two bit set = it applies
// sources k_end-2 and k_end-1, else k_end-1 only.
// Look-ahead (run_sweep): `own` >= 0 names the block row whose diagonal block is being factored by this very launch (its
// other tiles take their last sources here, the (own, own) tile is left out) -- the tile next to the diagonal, (own, own+1),
// is also copied to P.crit, where the following row-solve launch's diagonal-tile workgroups read it while the row solve
// overwrites it in place; own_zero: the row has nothing pending, only that copy is made.
// `dg` >= 0: one more tile after the planned rows', the diagonal tile of block row dg alone (one source, or two with dg_two):
// the look-ahead of the coming row solve needs that tile up to date, the rest of its row may stay behind (run_sweep).
constexpr bool FILL_NT = true;                 // the fused sweep's tiles read and write their C tile with the non-temporal hint (pgm_gemm.h)
constexpr int FILL_MAX_NB = 48;
struct FillPlan { unsigned long long skip, two; int own, own_zero, dg, dg_two; };
// Which planned tile a filler workgroup of k_diag takes (one light curve): the dispatcher deals workgroups round-robin over the
// 8 XCDs, each with an L2 of its own, so with the plain index every XCD works on every 8th tile of every row and fetches nearly
// all of the launch's operand tiles (~40 per source) from the memory side; the host's map gives the workgroups of one XCD a
// block of about 4 rows x 8 columns of tiles (12 operand tiles).  Placement only: every tile is still computed once.
// (Kernel argument = scalar loads issued with the other arguments: no dependent memory access in front of the tile.)
struct FillMap { int on; unsigned idx[128]; };   // (two 16-bit entries per word: scalar loads are 32 bits wide)

// One planned trailing-update tile (or BM x BN sub-tile of it): workgroup index widx counts the sub-tiles of
// the planned rows >= r_from in row order.  Used by the filler workgroups of k_diag (128x128, 16 wavefronts)
// and, with 64x64 sub-tiles on 8 wavefronts, by the chain's two small launches (k_update_rows, the tail of
// k_trsm's grid), whose idle CUs take part of the trailing update as well.
template <class C>
__device__ __forceinline__ void plan_tile(const PgmDev& P, double* lds, const FillPlan& plan, int k_end, int r_from, int widx) {
  constexpr int SUBM = NB / C::BM, SUBN = NB / C::BN;
  const int b = blockIdx.z;
  const int nR = P.need_grad ? k_end : 0;                    // inverse-factor tiles (r, j), j < k_end
  const int sub = widx % (SUBM * SUBN);
  int tile = widx / (SUBM * SUBN);
  const int si = sub / SUBN, sj = sub % SUBN;
  int r = r_from;
  for (; r < P.nb; ++r) {
    const int cnt = ((plan.skip >> r) & 1ull) ? 0 : (r == plan.own ? (plan.own_zero ? 1 : (P.nb - r - 1) + nR) : (P.nb - r) + nR);
    if (tile < cnt) break;
    tile -= cnt;
  }
  bool dgt = false;
  if (r >= P.nb) {                                           // (uniform for the workgroup)
    if (plan.dg < 0 || tile != 0) return;
    r = plan.dg; dgt = true;                                 // tile 0 of a row that is not `own` = its diagonal tile
  }
  r = __builtin_amdgcn_readfirstlane(r);
  tile = __builtin_amdgcn_readfirstlane(tile);
  const int own = (!dgt && r == plan.own) ? 1 : 0;
  const bool copy_only = own && plan.own_zero;
  const int lo = copy_only ? k_end : k_end - 1 - (dgt ? plan.dg_two : (int)((plan.two >> r) & 1ull));
  const bool syrk = tile < P.nb - r - own;
  const int j = syrk ? r + own + tile : tile - (P.nb - r - own);
  const int pstart = (!syrk && j > lo) ? j : lo;             // V_pj vanishes for p < j
  const bool assign = !syrk && j >= lo;                      // first contribution to this tile of R
  double* A = P.A + b * P.sA;
  const double* Dv = P.Dinv + b * P.sDinv;
  const int64_t ld = P.ld;
  double* Cp = A + ((int64_t)r * NB + si * C::BM) * ld + j * NB + sj * C::BN;
  // operand pointers of the (at most two, see run_sweep) k-blocks, fixed before the loop: the multiply
  // loop of a 16-wave workgroup is short of instruction issue slots, not of MFMA
  const int nkb = k_end - pstart;
  const double* pa0 = A + (int64_t)pstart * NB * ld + r * NB + si * C::BM;
  const double* pb0 = (assign ? Dv + ((int64_t)j * 2 + 1) * NB * NB : A + (int64_t)pstart * NB * ld + j * NB) + sj * C::BN;
  const int64_t ldb0 = assign ? NB : ld;
  const double* pa1 = pa0 + NB * ld;
  const double* pb1 = A + (int64_t)(pstart + 1) * NB * ld + j * NB + sj * C::BN;
  v4d acc[C::TM][C::TN];
  if (assign) acc_zero<C>(acc); else acc_load_raw<C, FILL_NT>(Cp, ld, acc);   // (negated inside gemm_tn: see negate_late there)
  if (nkb == 1) {
    gemm_tn<C>(lds, 1, [&](int, const double*& pa, int64_t& lda, const double*& pb, int64_t& ldb) {
      pa = pa0; lda = ld; pb = pb0; ldb = ldb0;
    }, acc, 0, !assign);
  } else if (nkb == 2) {                                     // two sources (the host never plans more)
    gemm_tn<C>(lds, 2, [&](int kb, const double*& pa, int64_t& lda, const double*& pb, int64_t& ldb) {
      pa = kb ? pa1 : pa0; lda = ld; pb = kb ? pb1 : pb0; ldb = kb ? ld : ldb0;
    }, acc, 0, !assign);
  } else if (!assign) {                                      // (copy only)
    acc_negate<C>(acc);
  }
  if (!copy_only) acc_store<C, FILL_NT>(Cp, ld, acc, -1.0);
  if (own && syrk && tile == 0)                              // (uniform) the tile the coming row solve's look-ahead reads
    acc_store<C>(P.crit + (int64_t)b * NB * NB + (int64_t)si * C::BM * NB + sj * C::BN, NB, acc, -1.0);
}

// Second filler role of the late diagonal-block launches (one light curve): when the plan leaves CUs without an update
// tile, they start on the inverse pass -- one product  R_ij += V_pi^T V_pj  of a block row p that is already final, kept
// negated in R (acc_load_neg reads it back); k_lauum_grad later continues from R instead of from zero.
constexpr int LAUUM_LOAD = 1 << 16;
template <class C>
__device__ __forceinline__ void early_inverse_tile(const PgmDev& P, double* lds, const int4 task, int sub = 0) {
  constexpr int SUBN = NB / C::BN;
  const int si = sub / SUBN, sj = sub % SUBN;                  // (64x64 sub-tiles when the task rides a row-solve launch)
  const int i = task.x, j = task.y, p = task.z;
  const int64_t ld = P.ld;
  double* Rp = P.R + ((int64_t)i * NB + si * C::BM) * ld + j * NB + sj * C::BN;
  const double* pa0 = ((p > i) ? P.A + (int64_t)p * NB * ld + i * NB : P.Dinv + ((int64_t)i * 2 + 1) * NB * NB) + si * C::BM;
  const double* pb0 = ((p > j) ? P.A + (int64_t)p * NB * ld + j * NB : P.Dinv + ((int64_t)j * 2 + 1) * NB * NB) + sj * C::BN;
  const int64_t lda0 = (p > i) ? ld : NB, ldb0 = (p > j) ? ld : NB;
  v4d acc[C::TM][C::TN];
  const bool cont = (task.w & LAUUM_LOAD) != 0;
  if (cont) acc_load_raw<C, FILL_NT>(Rp, ld, acc); else acc_zero<C>(acc);
  gemm_tn<C>(lds, 1, [&](int, const double*& pa, int64_t& lda, const double*& pb, int64_t& ldb) {
    pa = pa0; lda = lda0; pb = pb0; ldb = ldb0;
  }, acc, 0, cont);
  acc_store<C, FILL_NT>(Rp, ld, acc, -1.0);
}

// Third filler role, diagonal block 0 only (one light curve, 1-D spectral mixture): while the first diagonal block is factored
// nothing else of the sweep can run yet -- no block row is finished -- so the launch's other workgroups build the kernel matrix
// below block row 0 (k_build built that row alone: all diagonal block 0 and row solve 0 need).  A workgroup takes whole tiles
// (i, j), 1 <= i <= j, a quarter per 256 threads: the very code of k_build (build_part_1d), so the matrix has the same bits.
__device__ __forceinline__ void build_beside_diag(const PgmDev& P, double* lds, int widx, int nworkers, int ntile) {
  const int b = blockIdx.z;
  double* rowd = lds;
  double* cold = lds + P.pre_slots * NB;
  double* wl = cold + P.pre_slots * NB;
  const double* pre = P.pre + b * P.sPre;
  if (threadIdx.x < P.q) wl[threadIdx.x] = P.hyp[(int64_t)b * (PGM_MAX_QD * 3) + threadIdx.x];
  const int total = P.pre_slots * NB;
  for (int t = widx; t < ntile; t += nworkers) {
    int i, j;
    tri_decode(t, i, j);                                       // (triangle of the block rows 1 .. nb-1)
    i += 1; j += 1;
    for (int e = threadIdx.x; e < total; e += DIAG_THREADS) {
      const int slot = e / NB, m = e % NB;
      rowd[e] = pre[(int64_t)slot * P.np + i * NB + m];
      cold[e] = pre[(int64_t)slot * P.np + j * NB + m];
    }
    __syncthreads();
    build_part_1d<4>(P, rowd, cold, wl, b, i, j, (int)(threadIdx.x >> 8), (int)(threadIdx.x & 255));
    __syncthreads();
  }
}

__global__ __launch_bounds__(DIAG_THREADS, 4) void k_diag(PgmDev P, int k, int fill_end, int fill_lo, FillPlan plan, int nfill, int task_lo, int build_tiles, FillMap map) {
  const int b = blockIdx.z;
  // (no early exit on P.info here or in k_trsm / k_update: after a failed pivot the chain kernels just
  //  carry NaNs -- no address depends on data -- and a dependent scalar load in front of every one of the
  //  ~65 chained launches costs 0.4 us each, 1 % of an evaluation)
  __shared__ __attribute__((aligned(16))) double M[NB * PM];
  __shared__ double uiS[DB * DB];
  __shared__ double rsv[NB], zsv[NB], alv[NB], udg[NB], dump[64];
  if (blockIdx.x > 0) {
    const int widx = (int)blockIdx.x - 1;
    const int slot = map.on ? (int)((map.idx[widx >> 1] >> (16 * (widx & 1))) & 0xffffu) : widx;   // (map: tiles and early tasks of the launch alike)
    if (map.on ? slot < nfill : widx < nfill) plan_tile<CfgFill>(P, M, plan, fill_end, fill_lo, slot);
    else if (build_tiles > 0) build_beside_diag(P, M, widx - nfill, (int)gridDim.x - 1 - nfill, build_tiles);   // (diagonal block 0 only)
    else early_inverse_tile<CfgFill>(P, M, P.tasks[task_lo + slot - nfill]);
    return;
  }
#ifdef PGM_DIAG_STAMPS
  const long long entry_ = __builtin_amdgcn_s_memtime();
#endif
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);     // wave-uniform: index math goes to the scalar unit
  constexpr int NS = NB / DB;
  DiagCtx c;
  c.prow = M; c.dg = M + 2 * NS * DB * DB; c.sup = c.dg + NS * DB * DB;
  c.uiS = uiS; c.udg = udg; c.dump = dump;
  c.Akk = P.A + b * P.sA + (int64_t)k * NB * P.ld + k * NB;
  c.ld = P.ld;
  c.Dinv0 = P.Dinv + b * P.sDinv + (int64_t)k * 2 * NB * NB;
  c.Dinv1 = c.Dinv0 + NB * NB;
  // The last block of a light curve whose length is no multiple of 128 ends in identity padding, decoupled from the data:
  // the sub-block steps that would "factor" it are left out (N=89: 6 of 8 steps), its inverse images are zero blocks and identities.
  // (A light curve of a ragged batch that is shorter than its launch set's block rows has whole blocks of padding: nse = 0,
  //  nothing is factored, the block's z, alpha and log det are zero and its inverse images the identity.)
  const int left = pts(P, b) - k * NB;
  const int valid = left < 0 ? 0 : (left < NB ? left : NB);
  const int nse = __builtin_amdgcn_readfirstlane((valid + DB - 1) / DB);
  // Every wavefront meets the same two barriers per step: V_ss in LDS / block row s in LDS.
  if (wave == 0) {
    diag_chain(c, lane, nse);
  } else if ((wave & 3) != 0) {
    diag_worker(c, wave - 1 - (wave >> 2), lane, nse);
  } else if (wave == 4) {
    // bookkeeping: z_k = V_kk r_k by forward substitution beside the factorisation, alpha_k, log det, the pivot check
    int* info = P.info + b;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      rsv[lane + 64 * u] = P.r[b * P.sVec + k * NB + lane + 64 * u];
      alv[lane + 64 * u] = 0.0;
      zsv[lane + 64 * u] = 0.0;
    }
    double lgsum = 0.0;
    int firstbad = -1;
    for (int s = 0; s < nse; ++s) {
      const double* row = c.prow + (s & 1) * NS * DB * DB;
      lds_barrier();
      if (lane < DB) {                                           // z_s = V_ss r_s (r_s is final since step s-1)
        double acc = 0.0;
#pragma unroll
        for (int kk = 0; kk < DB; ++kk) acc += uiS[kk * DB + lane] * rsv[s * DB + kk];
        zsv[s * DB + lane] = acc;
      }
      lds_barrier();
      // forward substitution / alpha updates with block row s (2 columns per lane)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int colg = lane + 64 * u, jb = colg / DB;
        double acc = 0.0;
#pragma unroll
        for (int m = 0; m < DB; ++m) acc += row[jb * DB * DB + m * DB + (colg - jb * DB)] * zsv[s * DB + m];   // (V_ss is zero above its diagonal)
        if (jb > s) rsv[colg] -= acc; else alv[colg] += acc;
      }
      // ... and the block's share of log det A and the pivot check, one 16x16 sub-block per step, so that nothing is left after the last
      {
        const double u = udg[s * DB + (lane & 15)];
        const unsigned long long badm = __ballot(!(u > 0.0 && u < 1e300)) & 0xffffull;
        if (badm && firstbad < 0) firstbad = s * DB + (int)__builtin_ctzll(badm);
        if (lane < DB) lgsum += 2.0 * log(u);
      }
      if (s == nse - 1) {                                 // z_k, alpha_k, log det, info: final now
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          P.z[b * P.sVec + k * NB + lane + 64 * u] = zsv[lane + 64 * u];
          P.alpha[b * P.sVec + k * NB + lane + 64 * u] = alv[lane + 64 * u];
        }
        const double tot = wave_sum(lgsum);
        if (lane == 0) {
          P.logdet[b * P.sLogdet + k] = tot;
          // first pivot that was not positive: U_pp is then NaN/inf (or 0), and so is everything after it
          if (firstbad >= 0 && *info == 0) *info = k * NB + 1 + firstbad;
          // the status is final with the last diagonal block: the host's copy (pgm_factorisation_status) is written here
          // (then the evaluation's number, at system scope: a host that finds the number knows the status beside it is this evaluation's)
          if (k == P.nb - 1 && P.info_host) {
            P.info_host[b] = *info;
            __threadfence_system();
            P.seq_host[b] = (long long)P.outp[7];
          }
        }
      }
    }
    if (nse == 0) {                                       // a block of padding (ragged batches): zeros, and the status if it is the last
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        P.z[b * P.sVec + k * NB + lane + 64 * u] = 0.0;
        P.alpha[b * P.sVec + k * NB + lane + 64 * u] = 0.0;
      }
      if (lane == 0) {
        P.logdet[b * P.sLogdet + k] = 0.0;
        if (k == P.nb - 1 && P.info_host) {
          P.info_host[b] = *info;
          __threadfence_system();
          P.seq_host[b] = (long long)P.outp[7];
        }
      }
    }
  } else {
    // waves 8 and 12: V_ss leaves for the two inverse images (one each)
    const int kq = lane >> 4, n = lane & 15;
    for (int s = 0; s < NS; ++s) {
      v4d v;
      if (s < nse) {
        lds_barrier();
        v = diag_get(c.prow + (s & 1) * NS * DB * DB + s * DB * DB, lane);
        lds_barrier();
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = (kq + 4 * r == n) ? 1.0 : 0.0;
      }
      diag_store_v(c, s, s, v, lane, wave == 8 ? 1 : 2);
    }
  }
#ifdef PGM_DIAG_STAMPS
  {   // when every wavefront of the factoring workgroup entered and left, when its stores had drained (ticks after the first entry)
    __shared__ long long wt_[DIAG_THREADS / 64][3];
    const long long t1_ = __builtin_amdgcn_s_memtime();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const long long t2_ = __builtin_amdgcn_s_memtime();
    if (lane == 0) { wt_[wave][0] = entry_; wt_[wave][1] = t1_; wt_[wave][2] = t2_; }
    __syncthreads();
    if (t == 0 && blockIdx.z == 0) {
      long long t0_ = wt_[0][0];
      for (int w = 1; w < DIAG_THREADS / 64; ++w) if (wt_[w][0] < t0_) t0_ = wt_[w][0];
      printf("waves (entry, done, drained): ");
      for (int w = 0; w < DIAG_THREADS / 64; ++w) printf("%d:%d,%d,%d ", w, (int)(wt_[w][0] - t0_), (int)(wt_[w][1] - t0_), (int)(wt_[w][2] - t0_));
      printf("\n");
    }
  }
#endif
}

// ---------------------------------------------------------------------------
// Block row k after its diagonal block:  C <- Uinv_kk^T C for every other block of
// the row (U_kj for j > k, V_kj for j < k), 128 x 32 column slabs, in place.
// Epilogue: the forward substitution rides along,  r_j -= U_kj^T z_k  (j > k), and
// so does alpha,  alpha_j += V_kj^T z_k  (j < k).
// ---------------------------------------------------------------------------
using CfgTrsm = TileCfg<128, 32, 32, 32, 4>;               // (prediction right-hand sides)
// 8 wavefronts, a 32x16 sub-tile each: the launch sits on the chain and is bound by its own latency, so the
// multiply body is cut to 64 MFMAs per wavefront (2 us) rather than sized for operand reuse
// (16-column slabs -- twice the workgroups, half the MFMAs each -- were measured in round 2 and lost: 2.169 -> 2.178 ms)
using CfgTrsmChain = TileCfg<128, 32, 32, 16, 4, 512>;
using CfgLook = TileCfg<128, 32, 32, 16, 4, 512>;          // the look-ahead workgroups: two 16-column slabs each
constexpr int TRSM_SLABS = NB / CfgTrsmChain::BN;
using CfgHead = TileCfg<64, 64, 32, 16, 4, 512>;           // the chain's update tiles: 64x64 sub-tiles, same reasoning
constexpr int CHAIN_LDS = CfgLook::LDS_DOUBLES > CfgHead::LDS_DOUBLES ? CfgLook::LDS_DOUBLES : CfgHead::LDS_DOUBLES;
static_assert(CfgTrsmChain::LDS_DOUBLES <= CHAIN_LDS, "row-solve staging");

// planned trailing-update tiles as their own launch (the fused sweep's head update of block row k, plus
// whatever else the host's plan puts on this launch's idle CUs)
__global__ __launch_bounds__(CfgHead::NT, 2) void k_update_rows(PgmDev P, int k_end, int r_from, FillPlan plan) {
  __shared__ __attribute__((aligned(16))) double lds[CfgHead::LDS_DOUBLES];
  plan_tile<CfgHead>(P, lds, plan, k_end, r_from, (int)blockIdx.x);
}

// one column slab (C::BN columns, slab number `slab`) of block (k, jb) of block row k:  C <- Uinv_kk^T C, in place, and the
// slab's share of the forward substitution / alpha update
template <class C>
__device__ __forceinline__ void trsm_slab(const PgmDev& P, double* lds, double* zs, double (*red)[C::WN], int b, int k, int jb, int slab) {
  double* A = P.A + b * P.sA;
  double* Cb = A + (int64_t)k * NB * P.ld + jb * NB + slab * C::BN;
  const double* Uinv = P.Dinv + b * P.sDinv + (int64_t)k * 2 * NB * NB;
  if (threadIdx.x < NB) zs[threadIdx.x] = P.z[b * P.sVec + k * NB + threadIdx.x];
  v4d acc[C::TM][C::TN];
  acc_zero<C>(acc);
  const int64_t ld = P.ld;
  gemm_tn<C>(lds, 1, [&](int, const double*& pa, int64_t& lda, const double*& pb, int64_t& ldb) {
    pa = Uinv; lda = NB; pb = Cb; ldb = ld;
  }, acc);
  acc_store<C>(Cb, ld, acc, 1.0);
  const WavePos wp = wave_pos<C>();
#pragma unroll
  for (int tj = 0; tj < C::TN; ++tj) {
    double s = 0.0;
#pragma unroll
    for (int ti = 0; ti < C::TM; ++ti)
#pragma unroll
      for (int r = 0; r < 4; ++r) s = __builtin_fma(acc[ti][tj][r], zs[acc_row<C>(wp, ti, r)], s);
    s += __shfl_xor(s, 16, 64);
    s += __shfl_xor(s, 32, 64);
    if (wp.lane < 16) red[wp.wave][tj * 16 + wp.lane] = s;
  }
  __syncthreads();
  if (threadIdx.x < C::BN) {
    // column c: the wavefronts of its column group, top to bottom (fixed order)
    const int c = threadIdx.x, nw = c / C::WN, cc = c % C::WN;
    double tot = 0.0;
#pragma unroll
    for (int mw = 0; mw < C::BM / C::WM; ++mw) tot += red[mw * C::WAVES_N + nw][cc];
    const int64_t g = b * P.sVec + jb * NB + slab * C::BN + c;
    if (jb > k) P.r[g] -= tot; else P.alpha[g] += tot;
  }
}

// Look-ahead of the fused sweep: the diagonal tile of the NEXT block row, A_{k+1,k+1} -= U_{k,k+1}^T U_{k,k+1}, inside the row
// solve's own launch, so that diagonal block k+1 can start right behind it (the rest of row k+1 takes source k beside that
// diagonal block, as filler tiles).  No workgroup of the launch may wait for another, so each of the 36 workgroups -- one per
// pair (s1 <= s2) of 16-column slabs -- solves its two slabs of U_{k,k+1} again for itself from the copy of the unsolved
// tile in P.crit (the row solve proper overwrites the tile in place meanwhile), keeps them in LDS and multiplies the 16x16
// block (s1, s2).
constexpr int LOOK_SLAB = 16, LOOK_NS = NB / LOOK_SLAB, LOOK_PAIRS = LOOK_NS * (LOOK_NS + 1) / 2;
template <class C>
__device__ __forceinline__ void lookahead_diag_tile(const PgmDev& P, double* lds, int b, int k, int pair) {
  static_assert(C::BM == NB && C::BN == 2 * LOOK_SLAB && C::TN == 1 && C::NT == 512, "two 16-column slabs per workgroup");
  int s1, s2;
  tri_decode(pair, s1, s2);
  const double* Uinv = P.Dinv + b * P.sDinv + (int64_t)k * 2 * NB * NB;
  const double* Bp = P.crit + (int64_t)b * NB * NB + s1 * LOOK_SLAB;
  const WavePos wp = wave_pos<C>();
  // the 16x16 block this workgroup updates is asked for now, in the shadow of the solve (it is final since the launch before:
  // asked for behind the solve, as in rounds 2-3, its round trip sat on the chain once per block row)
  double* Cd = P.A + b * P.sA + ((int64_t)(k + 1) * NB + s1 * LOOK_SLAB + (wp.lane >> 4)) * P.ld + (k + 1) * NB + s2 * LOOK_SLAB + (wp.lane & 15);
  v4d d = {0.0, 0.0, 0.0, 0.0};
  if (wp.wave == 0) {
#pragma unroll
    for (int r = 0; r < 4; ++r) d[r] = Cd[(int64_t)4 * r * P.ld];
  }
  v4d acc[C::TM][C::TN];
  acc_zero<C>(acc);
  gemm_tn<C>(lds, 1, [&](int, const double*& pa, int64_t& lda, const double*& pb, int64_t& ldb) {
    pa = Uinv; lda = NB; pb = Bp; ldb = NB;
  }, acc, (s2 - s1) * LOOK_SLAB - LOOK_SLAB);
  // (gemm_tn ends on a barrier: the staging area is free) the two solved slabs as one [k][32] image
  constexpr int PX = 2 * LOOK_SLAB + 16;
#pragma unroll
  for (int ti = 0; ti < C::TM; ++ti)
#pragma unroll
    for (int r = 0; r < 4; ++r) lds[acc_row<C>(wp, ti, r) * PX + acc_col<C>(wp, 0)] = acc[ti][0][r];
  __syncthreads();
  // one wavefront, the 32 k-steps in order, starting from -C: the very sequence of operations a trailing-update tile
  // applies to this block (acc_load_neg, MFMAs with k ascending, store of -acc), so the factor -- and with it the value --
  // is bit for bit what the schedules without look-ahead produce
  if (wp.wave == 0) {
    d = -d;
#pragma unroll 8
    for (int kk = 0; kk < NB / 4; ++kk) {
      const int krow = kk * 4 + (wp.lane >> 4);
      d = __builtin_amdgcn_mfma_f64_16x16x4f64(lds[krow * PX + (wp.lane & 15)], lds[krow * PX + LOOK_SLAB + (wp.lane & 15)], d, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) Cd[(int64_t)4 * r * P.ld] = -d[r];
  }
}

// workgroups [nlook, nlook + nslabs) are the row solve; the first nlook (0 or 36) form the next diagonal tile (look-ahead);
// workgroups beyond are planned trailing-update tiles riding on this launch's idle CUs, then early inverse-pass products
// (64x64 sub-tiles of the tasks P.tasks[task_lo ...], four workgroups per task)
__global__ __launch_bounds__(CfgTrsmChain::NT, 2) void k_trsm(PgmDev P, int k, int nslabs, int k_end, int r_from, FillPlan plan, int nlook, int nextra, int task_lo) {
  using C = CfgTrsmChain;
  __shared__ __attribute__((aligned(16))) double lds[CHAIN_LDS];
  __shared__ double zs[NB];
  __shared__ double red[C::NT / 64][C::WN];
  if ((int)blockIdx.x < nlook) { lookahead_diag_tile<CfgLook>(P, lds, blockIdx.z, k, (int)blockIdx.x); return; }
  const int bx0 = (int)blockIdx.x - nlook;
  if (bx0 >= nslabs + nextra) {                                  // early inverse-pass products on CUs the launch leaves idle (run_sweep)
    const int e = bx0 - nslabs - nextra;
    early_inverse_tile<CfgHead>(P, lds, P.tasks[task_lo + e / 4], e % 4);
    return;
  }
  if (bx0 >= nslabs) { plan_tile<CfgHead>(P, lds, plan, k_end, r_from, bx0 - nslabs); return; }
  int b = blockIdx.z, bx = bx0;
  if ((int)gridDim.x == nslabs) xcd_batch_remap(bx, b);          // (no planned tiles in the grid: batches, panel sweep)
  const int slab = bx % TRSM_SLABS;
  int jb = bx / TRSM_SLABS;
  if (P.need_grad) { if (jb >= k) jb += 1; } else { jb += k + 1; }
  trsm_slab<C>(P, lds, zs, red, b, k, jb, slab);
}

// ---------------------------------------------------------------------------
// The chain's row solve, round 4: the same launch -- look-ahead workgroups, slab workgroups, update sub-tiles and early
// inverse-pass products in the grid's tail -- on workgroups of 16 wavefronts that go through memory ONCE.
// k_trsm stages U_kk^-1 and its slab through LDS in eight 16-row chunks, one barrier and an LDS round trip per chunk, the
// second half of the chunks requested when the first has been consumed: stamps (s_memtime) put a look-ahead workgroup at
// 5.5 us for the solve + 1.8 us for its 32-step product and a slab workgroup at 6.5 us, of which the MFMA work is 0.4 us --
// the rest is two memory round trips and eight chunk latencies in sequence, once per block row on the chain.
// Here every global load of the workgroup is issued in its first instructions: the upper triangle of U_kk^-1 (72 KB, all threads
// together, to LDS) and each wavefront's B fragments straight into registers (wavefront (rb, h) owns the 16 x 16 block of rows
// 16 rb .. of column half h and needs the rows p < 16 (rb + 1) only: U_kk^-1 is upper triangular) -- one round trip; then one
// barrier, and every wavefront runs its own chain of 4 (rb + 1) MFMAs with A fragments from LDS.  The MFMAs that are left out
// would add exact zeros and the others run in k order from a zero accumulator, the forward-substitution sums are formed from
// an LDS image of the solved slab in the slab kernel's order, and the look-ahead block takes its 32 k-steps in order from -C:
// same bits as k_trsm (PGM_TRSM16=0; tests compare).
// ---------------------------------------------------------------------------
using CfgSmall = TileCfg<64, 64, 32, 32, 8, 256, KB, true>;   // 64x64 tiles on 4 wavefronts, direct form (also: deep updates with few tiles, quarter tiles of the inverse pass)
constexpr int T16_THREADS = 1024;
// LDS of a workgroup: U_kk^-1 as eight column panels -- panel rb holds the rows p < 16 (rb + 1) of the columns 16 rb .. 16 rb + 15,
// all a wavefront of row block rb ever reads, 72 KB for the upper triangle instead of 147 KB for the padded square -- then per
// 16-column half of the slab an image of the unsolved and one of the solved values, [row][16].  (Pitch 16 doubles: the rows
// 4 kk + g, g = 0 .. 3, of one fragment read fall on disjoint bank halves.)
constexpr int T16_PANEL = 16 * NB / 2 * 9;                     // sum over rb of 16 (rb + 1) rows x 16 columns
constexpr int T16_HALF = NB * 16;
constexpr int T16_LDS = T16_PANEL + 4 * T16_HALF;              // 139 KB
static_assert(T16_LDS <= NB * PM, "as large as the diagonal block's image at most");
__device__ __forceinline__ int t16_panel(int rb) { return 128 * rb * (rb + 1); }     // first double of panel rb
// the tail's 64x64 sub-tiles: one per workgroup on all 16 wavefronts (a 16x16 block each), staged through LDS in chunks of 32
// rows -- as many 16-byte pieces per chunk as threads, no predicated loads.  (Measured against it: the direct form of the loop on
// 16x16 blocks, and two sub-tiles side by side on eight wavefronts each -- both bound by the L1: a block that small re-fetches
// its operands per wavefront; N=4096 1.87 -> 1.96 ms with them, 1.87 -> 1.85 with this one.)
using CfgTail16 = TileCfg<64, 64, 16, 16, 2, 1024, 32>;
static_assert(CfgTail16::LDS_DOUBLES <= T16_LDS, "staging inside the workgroup's LDS");
// wavefront <-> (row block, column half): row blocks rb and 7 - rb on one SIMD -- a wavefront w runs on SIMD w % 4 --, so that
// every SIMD has 4 (rb + 1) + 4 (8 - rb) = 36 MFMAs per half (with rb = w % 8 SIMD 3 had 48 and the launch waited for it)
__device__ __forceinline__ int t16_rb(int wave) { return (wave & 4) ? 7 - (wave & 3) : (wave & 3); }
__device__ __forceinline__ int t16_wave(int rb, int h) { return (rb < 4 ? rb : 11 - rb) + 8 * h; }

// U = Uinv_kk^T C for the 128 x 32 slab at Cs (pitch ldc; its right half hsplit doubles further along: two 16-column slabs of
// the look-ahead copy, or 16 for one slab of 32): every wavefront (rb, h) leaves its 16 x 16 block in the solved image of its
// half (lds + T16_PANEL + (2 + h) T16_HALF), in place when `store`, and then raises done[wave].  `halves` = 1: only the left 16
// columns (wavefronts 8 .. 15 idle).  No barrier after the one that publishes the operands: whoever needs solved blocks waits
// for their flags (the look-ahead's product, which walks down the rows as they are finished) or for the workgroup's next
// barrier (the slab's forward substitution).  Compact code on purpose: a workgroup runs it once, behind a diagonal-block
// launch that has evicted it from the instruction cache -- the first version, with the 32 k-steps and the 32 fragment loads of a
// wavefront unrolled and guarded one by one, spent more time fetching instructions than multiplying (3.1 us for a 32-step chain).
__device__ __forceinline__ void solve_slab16(const double* __restrict__ Uinv, double* __restrict__ Cs, int64_t ldc, int hsplit,
                                             int halves, bool store, double* lds, volatile int* done) {
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int rb = t16_rb(wave), h = wave >> 3;
  const int g = lane >> 4, n = lane & 15;
  double* pan = lds;
  double* Bs = lds + T16_PANEL;                               // unsolved halves, then the solved ones
  {  // every global load of the workgroup, at once: the slab (two 16-byte pieces per thread), then the panels of U_kk^-1
    v2d bt[2], ut[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int e = t + u * T16_THREADS, row = e >> 4, c2 = (e & 15) * 2;
      if (c2 < 16 * halves) bt[u] = *reinterpret_cast<const v2d*>(Cs + (int64_t)row * ldc + (c2 < 16 ? c2 : hsplit + c2 - 16));
    }
    const int prow = t >> 3, pc2 = (t & 7) * 2;               // panel q: thread t < 128 (q + 1) takes piece (row t / 8, columns 2 (t % 8) ..)
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (t < 128 * (q + 1)) ut[q] = *reinterpret_cast<const v2d*>(Uinv + prow * NB + 16 * q + pc2);
    if (t < 16) done[t] = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int e = t + u * T16_THREADS, row = e >> 4, c2 = (e & 15) * 2;
      if (c2 < 16 * halves) *reinterpret_cast<v2d*>(Bs + (c2 >> 4) * T16_HALF + row * 16 + (c2 & 15)) = bt[u];
    }
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (t < 128 * (q + 1)) *reinterpret_cast<v2d*>(pan + t16_panel(q) + prow * 16 + pc2) = ut[q];
  }
  __syncthreads();
  if (h < halves) {                                           // (uniform) 4 (rb + 1) k-steps in order, fragments one group of four ahead
    v4d acc = {0.0, 0.0, 0.0, 0.0};
#ifdef PGM_RELAX_TRSM          // (lab build, DESIGN section 12: the k-steps of a block dealt to two accumulators -- other bits, half the dependent chain)
    v4d acc2 = {0.0, 0.0, 0.0, 0.0};
#endif
    const double* pa = pan + t16_panel(rb) + g * 16 + n;
    const double* pb = Bs + h * T16_HALF + g * 16 + n;
    double a[4], bq[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) { a[u] = pa[u * 64]; bq[u] = pb[u * 64]; }
#pragma clang loop unroll(disable)
    for (int gq = 0; gq <= rb; ++gq) {
      double an[4], bn[4];
      const int nx = (gq < rb) ? gq + 1 : gq;                  // (the last group reads its own fragments again: no branch in the loop)
#pragma unroll
      for (int u = 0; u < 4; ++u) { an[u] = pa[(4 * nx + u) * 64]; bn[u] = pb[(4 * nx + u) * 64]; }
#ifdef PGM_RELAX_TRSM
#pragma unroll
      for (int u = 0; u < 4; u += 2) {
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64(a[u], bq[u], acc, 0, 0, 0);
        acc2 = __builtin_amdgcn_mfma_f64_16x16x4f64(a[u + 1], bq[u + 1], acc2, 0, 0, 0);
      }
#else
#pragma unroll
      for (int u = 0; u < 4; ++u) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(a[u], bq[u], acc, 0, 0, 0);
#endif
#pragma unroll
      for (int u = 0; u < 4; ++u) { a[u] = an[u]; bq[u] = bn[u]; }
    }
#ifdef PGM_RELAX_TRSM
    acc += acc2;
#endif
    double* Us = Bs + (2 + h) * T16_HALF;
    double* Ch = Cs + (h ? hsplit : 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * rb + g + 4 * r;
      Us[row * 16 + n] = acc[r];
      if (store) Ch[(int64_t)row * ldc + n] = acc[r];          // (in place: every thread's loads of the slab were over before the barrier)
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");         // the block is in LDS: raise the flag
    if (lane == 0) done[wave] = 1;
  }
}

__global__ __launch_bounds__(T16_THREADS) void k_trsm16(PgmDev P, int k, int nslabs, int k_end, int r_from, FillPlan plan, int nlook, int nextra, int task_lo) {
  __shared__ __attribute__((aligned(16))) double pan[T16_LDS];
  __shared__ double zs[NB];
  __shared__ double red[8][16];
  __shared__ int done[16];
  double* Us = pan + T16_PANEL + 2 * T16_HALF;                // solved image of half h at Us + h T16_HALF: [row][16]
  const int b = blockIdx.z, t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int g = lane >> 4, n = lane & 15;
  const double* Uinv = P.Dinv + b * P.sDinv + (int64_t)k * 2 * NB * NB;
  if ((int)blockIdx.x < nlook) {
    // look-ahead: the 16 x 16 block (s1, s2) of the next diagonal tile, A_{k+1,k+1} -= U[:, s1]^T U[:, s2], from this
    // workgroup's own solve of the two slabs (the copy of the unsolved tile in P.crit).  The product's 32 k-steps run in order
    // from -C on wavefront 0 -- whose own row block, the first, is solved after four MFMAs -- and follow the other wavefronts
    // down the rows: k-step kk needs row block kk / 4, which is finished 4 (kk / 4 + 1) MFMAs into the solve.
    int s1, s2;
    tri_decode((int)blockIdx.x, s1, s2);
    double* Cd = P.A + b * P.sA + ((int64_t)(k + 1) * NB + s1 * LOOK_SLAB + g) * P.ld + (k + 1) * NB + s2 * LOOK_SLAB + n;
    v4d d = {0.0, 0.0, 0.0, 0.0};
    if (wave == 0) {                                          // (final since the launch before: its round trip rides with the others)
#pragma unroll
      for (int r = 0; r < 4; ++r) d[r] = Cd[(int64_t)4 * r * P.ld];
    }
    const int halves = (s1 == s2) ? 1 : 2;
    solve_slab16(Uinv, P.crit + (int64_t)b * NB * NB + s1 * LOOK_SLAB, NB, (s2 - s1) * LOOK_SLAB, halves, false, pan, done);
    if (wave == 0) {
      const double* u1 = Us + g * 16 + n;
      const double* u2 = Us + (halves - 1) * T16_HALF + g * 16 + n;
      d = -d;
#ifdef PGM_RELAX_TRSM          // (lab build: the four k-steps of a row block on four accumulators, summed at the end)
      v4d dx[3] = {v4d{0.0, 0.0, 0.0, 0.0}, v4d{0.0, 0.0, 0.0, 0.0}, v4d{0.0, 0.0, 0.0, 0.0}};
#endif
#pragma clang loop unroll(disable)
      for (int rbn = 0; rbn < NB / 16; ++rbn) {
        // (bounded: a flag that never comes -- it cannot, the wavefronts of a workgroup are resident together -- ends in a wrong
        //  block and a failed factorisation, not in a hang)
        for (int spin = 0; spin < (1 << 22) && (done[t16_wave(rbn, 0)] == 0 || done[t16_wave(rbn, halves - 1)] == 0); ++spin) __builtin_amdgcn_s_sleep(1);
#ifdef PGM_RELAX_TRSM
        d = __builtin_amdgcn_mfma_f64_16x16x4f64(u1[(4 * rbn) * 64], u2[(4 * rbn) * 64], d, 0, 0, 0);
#pragma unroll
        for (int u = 1; u < 4; ++u) dx[u - 1] = __builtin_amdgcn_mfma_f64_16x16x4f64(u1[(4 * rbn + u) * 64], u2[(4 * rbn + u) * 64], dx[u - 1], 0, 0, 0);
#else
#pragma unroll
        for (int u = 0; u < 4; ++u) d = __builtin_amdgcn_mfma_f64_16x16x4f64(u1[(4 * rbn + u) * 64], u2[(4 * rbn + u) * 64], d, 0, 0, 0);
#endif
      }
#ifdef PGM_RELAX_TRSM
      d = (d + dx[0]) + (dx[1] + dx[2]);
#endif
#pragma unroll
      for (int r = 0; r < 4; ++r) Cd[(int64_t)4 * r * P.ld] = -d[r];
    }
    return;
  }
  const int bx0 = (int)blockIdx.x - nlook;
  if (bx0 >= nslabs + nextra) {                                  // early inverse-pass products on CUs the launch leaves idle
    const int e = bx0 - nslabs - nextra;
    early_inverse_tile<CfgTail16>(P, pan, P.tasks[task_lo + e / 4], e % 4);
    return;
  }
  if (bx0 >= nslabs) { plan_tile<CfgTail16>(P, pan, plan, k_end, r_from, bx0 - nslabs); return; }
  // one 32-column slab of block (k, jb): solved in place, then its share of the forward substitution / alpha update
  const int slab = bx0 % TRSM_SLABS;
  int jb = bx0 / TRSM_SLABS;
  if (P.need_grad) { if (jb >= k) jb += 1; } else { jb += k + 1; }
  if (t < NB) zs[t] = P.z[b * P.sVec + k * NB + t];
  double* Cb = P.A + b * P.sA + (int64_t)k * NB * P.ld + jb * NB + slab * CfgTrsmChain::BN;
  solve_slab16(Uinv, Cb, P.ld, 16, 2, true, pan, done);
  __syncthreads();                                            // every block of the slab is solved
  if (wave < 8) {                                             // the sums of trsm_slab, in its order: wavefront (mw, nw) = 32 rows x 16 columns
    const int mw = wave >> 1, nw = wave & 1;
    double sp = 0.0;
#pragma unroll
    for (int ti = 0; ti < 2; ++ti)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 32 * mw + 16 * ti + g + 4 * r;
        sp = __builtin_fma(Us[nw * T16_HALF + row * 16 + n], zs[row], sp);
      }
    sp += __shfl_xor(sp, 16, 64);
    sp += __shfl_xor(sp, 32, 64);
    if (lane < 16) red[wave][lane] = sp;
  }
  __syncthreads();
  if (t < CfgTrsmChain::BN) {
    const int nw = t / 16, cc = t % 16;
    double tot = 0.0;
#pragma unroll
    for (int mw = 0; mw < 4; ++mw) tot += red[mw * 2 + nw][cc];
    const int64_t gi = b * P.sVec + jb * NB + slab * CfgTrsmChain::BN + t;
    if (jb > k) P.r[gi] -= tot; else P.alpha[gi] += tot;
  }
}

// ---------------------------------------------------------------------------
// The chain's row solve for a HANDFUL of light curves in the fused sweep (round 5; config 5's tick: 8 chains x N=2048).
// k_trsm16 gives every 128 x 32 slab a workgroup that holds a whole CU: with eight light curves a block row is 8 x (60 slabs +
// 36 look-ahead pairs) = 768 of them, three rounds -- and the staged slab kernel (k_trsm, two per CU) pays its eight chunk
// latencies in 1.5 rounds: 24 us per block row either way, on a chain of 16 (`profiles/r04_timeline_cfg5_tick_8x2048.txt`).
// Here a workgroup takes a 128 x 64 slab -- or, `npass` = 2, the two slabs of a block one after the other, the triangle of
// U_kk^-1 staying in LDS and the second slab's values already on their way while the first is solved -- and every wavefront
// (rb, h) runs TWO 16 x 16 blocks side by side: the dependent v_mfma_f64_16x16x4 chain of k_trsm16 advances a step per ~135
// cycles where the pipe issues one per 64, so the second block rides in the shadow of the first.  The look-ahead, 36 workgroups
// per light curve there, is 6 here: two for the diagonal quadrants of the next diagonal tile (the 64 columns of its half
// solved from the copy in P.crit, then the quadrant's upper 16 x 16 blocks, one per wavefront, 32 k-steps in order from -C) and
// four for the quadrant above the diagonal (32 columns of either half, 2 x 2 blocks each).  8 x N=2048: 8 x (15 + 6) = 168
// workgroups, one round.  Every 16 x 16 block of the solve still receives its k-steps in ascending order from zero, every
// block of the next diagonal tile its 32 from -C, and the forward-substitution sums are formed in the slab kernel's order:
// the bits of k_trsm and k_trsm16 (PGM_TRSM64=0; tests compare).  The update sub-tiles that k_trsm carries in its grid's tail
// do not ride here (every workgroup of this kernel holds a CU): the host launches them behind it (k_update_rows).
// ---------------------------------------------------------------------------
constexpr int T64_LOOK = 6;                                    // look-ahead workgroups per light curve
constexpr int T64_B = 4 * T16_HALF;                            // the slab's image: four 16-column blocks [row][16], unsolved, then solved in place
static_assert(T16_PANEL + T64_B == T16_LDS, "k_trsm16's LDS budget");

// the 128 x 64 slab whose two 32-column groups start at columns co0 / co1 of Cs: 16-byte pieces, four per thread
__device__ __forceinline__ void slab64_load(const double* __restrict__ Cs, int64_t ldc, int co0, int co1, v2d (&bt)[4]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int e = (int)threadIdx.x + u * T16_THREADS, row = e >> 5, c2 = (e & 31) * 2;
    bt[u] = *reinterpret_cast<const v2d*>(Cs + (int64_t)row * ldc + (c2 < 32 ? co0 + c2 : co1 + c2 - 32));
  }
}
__device__ __forceinline__ void slab64_put(double* __restrict__ Bs, const v2d (&bt)[4]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int e = (int)threadIdx.x + u * T16_THREADS, row = e >> 5, c2 = (e & 31) * 2;
    *reinterpret_cast<v2d*>(Bs + (c2 >> 4) * T16_HALF + row * 16 + (c2 & 15)) = bt[u];
  }
}
// wavefront (rb, h): the two 16 x 16 blocks of rows 16 rb .. of column blocks 2 h and 2 h + 1, 4 (rb + 1) k-steps each in order
// from zero (A fragments: panel rb of U_kk^-1; B fragments: the unsolved image), fragments one group of four ahead
__device__ __forceinline__ void solve64_blocks(const double* __restrict__ pan, const double* __restrict__ Bs, int rb, int h, int g, int n,
                                               v4d& acc0, v4d& acc1) {
  acc0 = v4d{0.0, 0.0, 0.0, 0.0}; acc1 = acc0;
  const double* pa = pan + t16_panel(rb) + g * 16 + n;
  const double* pb = Bs + 2 * h * T16_HALF + g * 16 + n;
  double a[4], b0[4], b1[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) { a[u] = pa[u * 64]; b0[u] = pb[u * 64]; b1[u] = pb[T16_HALF + u * 64]; }
#pragma clang loop unroll(disable)
  for (int gq = 0; gq <= rb; ++gq) {
    double an[4], bn0[4], bn1[4];
    const int nx = (gq < rb) ? gq + 1 : gq;                    // (the last group reads its own fragments again: no branch in the loop)
#pragma unroll
    for (int u = 0; u < 4; ++u) { an[u] = pa[(4 * nx + u) * 64]; bn0[u] = pb[(4 * nx + u) * 64]; bn1[u] = pb[T16_HALF + (4 * nx + u) * 64]; }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      acc0 = __builtin_amdgcn_mfma_f64_16x16x4f64(a[u], b0[u], acc0, 0, 0, 0);
      acc1 = __builtin_amdgcn_mfma_f64_16x16x4f64(a[u], b1[u], acc1, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) { a[u] = an[u]; b0[u] = bn0[u]; b1[u] = bn1[u]; }
  }
}

__global__ __launch_bounds__(T16_THREADS) void k_trsm64(PgmDev P, int k, int nitems, int npass, int nlook) {
  __shared__ __attribute__((aligned(16))) double pan[T16_LDS];
  __shared__ double zs[NB];
  __shared__ double red[4][64];
  double* Bs = pan + T16_PANEL;
  const int b = blockIdx.z, t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int rb = t16_rb(wave), h = wave >> 3;
  const int g = lane >> 4, n = lane & 15;
  const double* Uinv = P.Dinv + b * P.sDinv + (int64_t)k * 2 * NB * NB;
  const bool look = (int)blockIdx.x < nlook;                   // (uniform)
  // ---- what this workgroup solves: `passes` slabs of 64 columns, the first one's two 32-column groups at co0 / co1 of Cs
  const double* Cs; int64_t ldc; int co0, co1, passes = 1, jb = 0, half0 = 0;
  int role = 0;
  if (look) {
    role = (int)blockIdx.x;                                    // 0, 1: diagonal quadrants; 2 .. 5: the quadrant above the diagonal, 32 x 32 columns each
    Cs = P.crit + (int64_t)b * NB * NB; ldc = NB;
    if (role < 2) { co0 = 64 * role; co1 = co0 + 32; }
    else { co0 = 32 * ((role - 2) >> 1); co1 = 64 + 32 * ((role - 2) & 1); }
  } else {
    const int item = (int)blockIdx.x - nlook;
    if (item >= nitems) return;
    int jbi = (npass == 2) ? item : item >> 1;
    half0 = (npass == 2) ? 0 : (item & 1);
    passes = npass;
    if (P.need_grad) { if (jbi >= k) jbi += 1; } else { jbi += k + 1; }
    jb = jbi;
    Cs = P.A + b * P.sA + (int64_t)k * NB * P.ld + jb * NB; ldc = P.ld;
    co0 = 64 * half0; co1 = co0 + 32;
    if (t < NB) zs[t] = P.z[b * P.sVec + k * NB + t];
  }
  // ---- every global load of the workgroup at once: the slab, the panels of U_kk^-1 (and, look-ahead, the blocks it will update)
  v2d bt[4];
  slab64_load(Cs, ldc, co0, co1, bt);
  {
    v2d ut[8];
    const int prow = t >> 3, pc2 = (t & 7) * 2;               // panel q: thread t < 128 (q + 1) takes piece (row t / 8, columns 2 (t % 8) ..)
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (t < 128 * (q + 1)) ut[q] = *reinterpret_cast<const v2d*>(Uinv + prow * NB + 16 * q + pc2);
    slab64_put(Bs, bt);
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (t < 128 * (q + 1)) *reinterpret_cast<v2d*>(pan + t16_panel(q) + prow * 16 + pc2) = ut[q];
  }
  // look-ahead: wavefront w owns block (bi, bj) of its quadrant -- global 16-column block indices (gi, gj) of the next diagonal tile
  int bi = 0, bj = 0, gi = 0, gj = 0;
  bool mine = false;
  v4d d = {0.0, 0.0, 0.0, 0.0};
  double* Cd = nullptr;
  if (look) {
    if (role < 2) { bi = wave >> 2; bj = wave & 3; mine = bi <= bj; gi = 4 * role + bi; gj = 4 * role + bj; }
    else { bi = wave >> 1; bj = 2 + (wave & 1); mine = wave < 4; gi = 2 * ((role - 2) >> 1) + bi; gj = 4 + 2 * ((role - 2) & 1) + (bj - 2); }
    if (mine) {                                                // (final since the launch before: its round trip rides with the others)
      Cd = P.A + b * P.sA + ((int64_t)(k + 1) * NB + gi * 16 + g) * P.ld + (k + 1) * NB + gj * 16 + n;
#pragma unroll
      for (int r = 0; r < 4; ++r) d[r] = Cd[(int64_t)4 * r * P.ld];
    }
  }
  for (int pass = 0; pass < passes; ++pass) {
    __syncthreads();                                            // the operands are in LDS
    const bool more = pass + 1 < passes;                        // (uniform) the next slab's values: asked for now, stored when this one is done with the image
    if (more) slab64_load(Cs, ldc, co0 + 64, co1 + 64, bt);
    v4d acc0, acc1;
    solve64_blocks(pan, Bs, rb, h, g, n, acc0, acc1);
    __syncthreads();                                            // every wavefront has read what it needs of the unsolved image
    {
      double* U0 = Bs + 2 * h * T16_HALF;
      double* G0 = look ? nullptr : const_cast<double*>(Cs) + (h ? co1 : co0) + 64 * pass;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * rb + g + 4 * r;
        U0[row * 16 + n] = acc0[r]; U0[T16_HALF + row * 16 + n] = acc1[r];
        if (!look) { G0[(int64_t)row * ldc + n] = acc0[r]; G0[(int64_t)row * ldc + 16 + n] = acc1[r]; }   // (in place)
      }
    }
    __syncthreads();                                            // the solved image is complete
    if (look) break;
    // the slab's share of the forward substitution / alpha update, in trsm_slab's order: wavefront (mw, cb) = 32 rows of column block cb
    {
      const int mw = wave >> 2, cb = wave & 3;
      double sp = 0.0;
#pragma unroll
      for (int ti = 0; ti < 2; ++ti)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 32 * mw + 16 * ti + g + 4 * r;
          sp = __builtin_fma(Bs[cb * T16_HALF + row * 16 + n], zs[row], sp);
        }
      sp += __shfl_xor(sp, 16, 64);
      sp += __shfl_xor(sp, 32, 64);
      if (lane < 16) red[mw][cb * 16 + lane] = sp;
    }
    __syncthreads();
    if (t < 64) {
      double tot = 0.0;
#pragma unroll
      for (int mw = 0; mw < 4; ++mw) tot += red[mw][t];
      const int64_t gidx = b * P.sVec + jb * NB + 64 * (half0 + pass) + t;
      if (jb > k) P.r[gidx] -= tot; else P.alpha[gidx] += tot;
    }
    if (more) slab64_put(Bs, bt);                               // (the image is free: every wavefront read its share for the sums before the last barrier)
  }
  if (look && mine) {
    // the block's 32 k-steps in order from -C -- the very sequence of a trailing-update tile: same bits as every other schedule
    const double* u1 = Bs + bi * T16_HALF + g * 16 + n;
    const double* u2 = Bs + bj * T16_HALF + g * 16 + n;
    d = -d;
#pragma clang loop unroll(disable)
    for (int q4 = 0; q4 < NB / 16; ++q4) {
#pragma unroll
      for (int u = 0; u < 4; ++u) d = __builtin_amdgcn_mfma_f64_16x16x4f64(u1[(4 * q4 + u) * 64], u2[(4 * q4 + u) * 64], d, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) Cd[(int64_t)4 * r * P.ld] = -d[r];
  }
}

// ---------------------------------------------------------------------------
// The row solve of batches (panel / left-looking sweeps, where the launch is throughput work, not a link of a latency chain).
// The slab kernel above runs one 128-deep product per workgroup behind a fresh copy of U_kk^-1: 160 KB fetched for 2 us of
// MFMA, the launch bound by prologues (64 x N=2048: 97 us per block row at a quarter of the matrix pipe).  Here a workgroup
// keeps U_kk^-1 in LDS for its whole life (147 KB: one workgroup per CU) and its 8 wavefronts stream 16-column strips of
// the block row through it, each on its own: the strip's 128 x 16 values go straight from memory into MFMA B fragments
// (32 eight-byte loads per lane, all in flight at once), the A fragments come from the LDS image -- no staging stores, no
// barrier after the prologue.  U_kk^-1 is upper triangular ([p][m], zero for p > m), so k-step kk only reaches the 16-row
// output tiles ti >= kk / 4: 144 MFMAs per strip instead of 256, every wavefront the same number.  The MFMAs that are left
// out would add exact zeros, the others run in the slab kernel's order (k ascending from a zero accumulator), and the
// forward-substitution sums are formed in the slab kernel's order too (pairs of 16-row tiles, butterfly over the row
// groups, the four 32-row groups top to bottom): same bits as k_trsm.
// ---------------------------------------------------------------------------
constexpr int STRIP_THREADS = 512, STRIP_W = 16;
// (TRIM: a trimmed ragged launch set -- a kernel of its own, so that the equal-length path keeps its code to the instruction)
template <bool TRIM>
__global__ __launch_bounds__(STRIP_THREADS, 2) void k_trsm_strips(PgmDev P, int k, int nblocks) {
  __shared__ __attribute__((aligned(16))) double Ui[NB * PM];
  __shared__ double zs[NB];
  const int b = blockIdx.z, t = threadIdx.x, lane = t & 63;
  if constexpr (TRIM) {   // (the light curve's own block columns only -- they are the first ones of the strip order)
    const int own = own_rows(P, b);
    if (k >= own) return;
    nblocks -= P.nb - own;
  }
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const double* Uinv = P.Dinv + b * P.sDinv + (int64_t)k * 2 * NB * NB;
  {  // U_kk^-1 -> LDS (16 x 16-B loads per thread, all in flight)
    constexpr int NV = NB * NB / 2 / STRIP_THREADS;
    v2d tmp[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int e = t + u * STRIP_THREADS, row = e / (NB / 2), c2 = (e % (NB / 2)) * 2;
      tmp[u] = *reinterpret_cast<const v2d*>(Uinv + row * NB + c2);
    }
    if (t < NB) zs[t] = P.z[b * P.sVec + k * NB + t];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int e = t + u * STRIP_THREADS, row = e / (NB / 2), c2 = (e % (NB / 2)) * 2;
      *reinterpret_cast<v2d*>(Ui + row * PM + c2) = tmp[u];
    }
  }
  __syncthreads();
  double* A = P.A + b * P.sA;
  const int64_t ld = P.ld;
  const int g = lane >> 4, n = lane & 15;
  constexpr int SPB = NB / STRIP_W;                           // strips per block
  const int nstrips = nblocks * SPB;
  const int stride = (int)gridDim.x * (STRIP_THREADS / 64);
  typedef unsigned v2u __attribute__((ext_vector_type(2)));
  // (buffer addressing: a uniform descriptor per strip, the row as a scalar offset and ONE 32-bit lane offset -- the 32 loads
  //  and 32 stores of a strip share a single address register instead of 64 address pairs)
  const int voff = (g * (int)ld + n) * 8, rowb = (int)ld * 8;
  auto strip_block = [&](int sidx) { int jb = sidx / SPB; if (P.need_grad) { if (jb >= k) jb += 1; } else { jb += k + 1; } return jb; };
  auto strip_desc = [&](int sidx) {
    double* Cs = A + (int64_t)k * NB * ld + strip_block(sidx) * NB + (sidx % SPB) * STRIP_W;     // uniform
    return __builtin_amdgcn_make_buffer_rsrc(Cs, 0, 0x7fffffff, 0x00027000);
  };
  int sidx = (int)blockIdx.x * (STRIP_THREADS / 64) + wave;
  if (sidx >= nstrips) return;
  __amdgpu_buffer_rsrc_t rs = strip_desc(sidx);
  double bf[NB / 4];
#pragma unroll
  for (int kk = 0; kk < NB / 4; ++kk) bf[kk] = __builtin_bit_cast(double, __builtin_amdgcn_raw_buffer_load_b64(rs, voff, 4 * kk * rowb, 0));
  const double* arow0 = Ui + g * PM + n;
  for (;;) {
    // the NEXT strip's values are requested while this one is multiplied, half a strip at a time into the fragment
    // registers the MFMAs have just released: the wavefront never sits out a memory round trip between two strips
    const int nxt = sidx + stride;
    const bool more = nxt < nstrips;                             // (uniform)
    const __amdgpu_buffer_rsrc_t rn = strip_desc(more ? nxt : sidx);
    v4d acc[NB / 16];
#pragma unroll
    for (int ti = 0; ti < NB / 16; ++ti) acc[ti] = v4d{0.0, 0.0, 0.0, 0.0};
    // A fragments one k-step ahead of the MFMAs that use them (the fence keeps the compiler from hoisting all 144 LDS reads
    // to the top, which spills)
    double af[2][NB / 16];
#pragma unroll
    for (int ti = 0; ti < NB / 16; ++ti) af[0][ti] = arow0[16 * ti];
#pragma unroll
    for (int kk = 0; kk < NB / 4; ++kk) {
      if (kk + 1 < NB / 4) {
        const double* arow = arow0 + 4 * (kk + 1) * PM;
#pragma unroll
        for (int ti = (kk + 1) / 4; ti < NB / 16; ++ti) af[(kk + 1) & 1][ti] = arow[16 * ti];
      }
      asm volatile("" ::: "memory");
#pragma unroll
      for (int ti = kk / 4; ti < NB / 16; ++ti)
        acc[ti] = __builtin_amdgcn_mfma_f64_16x16x4f64(af[kk & 1][ti], bf[kk], acc[ti], 0, 0, 0);
      if ((kk == NB / 8 - 1 || kk == NB / 4 - 1) && more) {      // the half just consumed: refill it for the next strip
#pragma unroll
        for (int q = kk + 1 - NB / 8; q <= kk; ++q) bf[q] = __builtin_bit_cast(double, __builtin_amdgcn_raw_buffer_load_b64(rn, voff, 4 * q * rowb, 0));
      }
    }
#pragma unroll
    for (int ti = 0; ti < NB / 16; ++ti)
#pragma unroll
      for (int r = 0; r < 4; ++r) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(v2u, (double)acc[ti][r]), rs, voff, (16 * ti + 4 * r) * rowb, 0);
    // forward substitution / alpha update of the strip's 16 columns (the summation order of trsm_slab)
    double tot = 0.0;
#pragma unroll
    for (int mw = 0; mw < 4; ++mw) {
      double sp = 0.0;
#pragma unroll
      for (int ti = 2 * mw; ti < 2 * mw + 2; ++ti)
#pragma unroll
        for (int r = 0; r < 4; ++r) sp = __builtin_fma(acc[ti][r], zs[16 * ti + g + 4 * r], sp);
      sp += __shfl_xor(sp, 16, 64);
      sp += __shfl_xor(sp, 32, 64);
      tot += sp;
    }
    if (lane < STRIP_W) {
      const int jb = strip_block(sidx);
      const int64_t gi = b * P.sVec + jb * NB + (sidx % SPB) * STRIP_W + lane;
      if (jb > k) P.r[gi] -= tot; else P.alpha[gi] += tot;
    }
    if (!more) break;
    sidx = nxt; rs = rn;
  }
}

// ---------------------------------------------------------------------------
// Trailing update with a panel of `dp` finished block rows k0..k0+dp-1 (the dominant
// kernel), applied to block rows r_lo..r_hi-1:
//   A_rj -= sum_p U_pr^T U_pj        r <= j            (Cholesky trailing update)
//   R_rj -= sum_p U_pr^T V_pj        j <= k0+dp-1      (inverse factor, same sweep; p >= j)
// Delaying the update until dp rows are finished multiplies the k-depth of every visit
// of a C tile by dp, i.e. divides the read-modify-write traffic of the trailing matrix --
// which, not MFMA issue, bounds a K=128 update on this machine.
// The same kernel with dp=1 and a short row range is the in-panel update.
// ---------------------------------------------------------------------------
// RAG: a trimmed ragged launch set (`rc`) -- an instantiation of its own, so that the equal-length path keeps its code to the
// instruction (with the class table as an argument of the one kernel, its workgroups waited for two kernel-argument round trips
// instead of one: 512 x N=2048 +0.85 % in this kernel)
struct NoClasses {};
template <class C, bool RAG>
__global__ __launch_bounds__(C::NT, 2) void k_update(PgmDev P, int k0, int dp, int r_lo, int r_hi, std::conditional_t<RAG, RagClasses, NoClasses> rc) {
  int b = blockIdx.z, bx = blockIdx.x, nbr = P.nb;              // nbr: the block rows the tiles are counted for
  bool classes = false;
  if constexpr (RAG) {
    classes = rc.n != 0;
    if (classes) { if (!rag_decode(rc, bx, b, nbr)) return; if (r_hi > nbr) r_hi = nbr; }      // (the member's own tiles, all of them real)
  }
  if (!classes) xcd_batch_remap(bx, b);
  constexpr int SUB = NB / C::BM;
  static_assert(C::BM == C::BN, "square tiles");
  // (Single light curve: an XCD-aware 8x8 super-block order of the tiles was measured and rejected at N=4096: a whole
  //  trailing update is only 1-2 co-resident sets of tiles, so the empty tiles of the trapezoid unbalance the XCDs more
  //  than the L2 reuse returns -- and the matrix sits in the Infinity Cache anyway.)
  const int sub = bx % (SUB * SUB);
  int tile = bx / (SUB * SUB);
  const int si = sub / SUB, sj = sub % SUB;
  const int kend = k0 + dp - 1;
  const int nR = P.need_grad ? kend + 1 : 0;              // inverse-factor tiles per block row
  int r = r_lo;
  for (; r < r_hi; ++r) {                                   // rows are few: linear decode
    const int cnt = (nbr - r) + nR;
    if (tile < cnt) break;
    tile -= cnt;
  }
  const bool syrk = tile < nbr - r;
  const int j = syrk ? r + tile : tile - (nbr - r);
  if constexpr (RAG) {
    if (P.trim && !classes) { const int own = own_rows(P, b); if (r >= own || (syrk && j >= own)) return; }   // (the box of a trimmed set: a tile the light curve does not have)
  }
  const int pstart = (!syrk && j > k0) ? j : k0;            // V_pj vanishes for p < j
  const bool assign = !syrk && j >= k0;                      // first contribution to this R tile
  double* A = P.A + b * P.sA;
  const double* Dv = P.Dinv + b * P.sDinv;
  const int64_t ld = P.ld;
  double* Cp = A + ((int64_t)r * NB + si * C::BM) * ld + j * NB + sj * C::BN;
  __shared__ __attribute__((aligned(16))) double lds[C::LDS_DOUBLES];
  v4d acc[C::TM][C::TN];
  if constexpr (RAG) {
    // A light curve's last block ends in identity padding (n is no multiple of 128): a wavefront whose whole sub-tile lies in the
    // padded rows of block row r or the padded columns of block column j would subtract exact zeros -- it leaves at once (the
    // first visit of a tile of the inverse factor stores its zeros); the direct loop has no barrier, the wavefronts of a tile do
    // not wait for one another.  512 x N ~ U{1024..2048}: 5.4 % of this kernel's products.
    static_assert(C::DIRECT, "wavefronts leave on their own: no barrier in the multiply loop");
    if (P.trim) {
      const int own = classes ? nbr : own_rows(P, b);
      const int rem = P.nvec[b] - (own - 1) * NB;               // points in the last block
      if (rem < NB && (r == own - 1 || j == own - 1)) {
        const WavePos wq = wave_pos<C>();
        if ((r == own - 1 && si * C::BM + wq.m0 >= rem) || (j == own - 1 && sj * C::BN + wq.n0 >= rem)) {
          if (assign) { acc_zero<C>(acc); acc_store<C>(Cp, ld, acc, -1.0); }
          return;
        }
      }
    }
  }
  if (assign) acc_zero<C>(acc); else acc_load_raw<C>(Cp, ld, acc);   // (negated inside gemm_tn: see negate_late there)
  gemm_tn<C>(lds, kend - pstart + 1, [&](int kb, const double*& pa, int64_t& lda, const double*& pb, int64_t& ldb) {
    const int p = pstart + kb;
    pa = A + (int64_t)p * NB * ld + r * NB + si * C::BM; lda = ld;
    if (!syrk && p == j) { pb = Dv + ((int64_t)j * 2 + 1) * NB * NB + sj * C::BN; ldb = NB; }
    else { pb = A + (int64_t)p * NB * ld + j * NB + sj * C::BN; ldb = ld; }
  }, acc, 0, !assign);
  acc_store<C>(Cp, ld, acc, -1.0);
}

// ---------------------------------------------------------------------------
// A^-1 tile (i <= j) = sum_{p >= j} V_pi^T V_pj, never written to memory: the
// epilogue forms G = alpha alpha^T - A^-1 and contracts it with dK/d(w, mu, v)
// recomputed from the per-point factors, leaving one partial sum per hyper-
// parameter and tile (summed in fixed order by k_finalize: bitwise reproducible).
// ---------------------------------------------------------------------------
// the staged form keeps the name CfgBigLds: its LDS budget is what the gradient epilogues stage their factors in
using CfgBigLds = TileCfg<128, 128, 64, 64, 2>;
struct CfgBig : TileCfg<128, 128, 64, 64, 4, 256, KB, true> { static constexpr int LDS_DOUBLES = CfgBigLds::LDS_DOUBLES; };
using CfgUpd = CfgBig;                                       // (8 wavefronts per 128x128 tile: measured in round 2, -0.7 %, not kept)
#ifndef PGM_SUB_PF
#define PGM_SUB_PF 8
#endif
using CfgSub = TileCfg<64, 64, 32, 32, PGM_SUB_PF, 256, KB, true>;   // quarter tiles of the inverse/gradient pass of short light curves (CfgSmall's shape)
// Sixteenth tiles (round 6) for light curves of a few block rows, where the launch is a handful of work items on an otherwise
// idle chip and its length is set by latencies, not by arithmetic (N=256, quarter tiles, ticks of the longest item: multiply
// 14.5 us -- 64 k-steps with 8 in flight, a memory round trip per 8 --, staging 2.8, epilogue 6.8 of the launch's 25): a 32x32
// sub-tile per workgroup, one 16x16 MFMA tile per wavefront with PGM_SUB16_PF k-steps in flight (two 8-byte fragments each),
// 4 pairs per lane in the epilogue.
#ifndef PGM_SUB16_PF
#define PGM_SUB16_PF 16
#endif
using CfgSub16 = TileCfg<32, 32, 16, 16, PGM_SUB16_PF, 256, KB, true>;
// The epilogue reuses the GEMM's LDS: per-point factors of the tile's rows and columns for
// a chunk of mixtures at a time (all of them when Q*d is small, the usual case).
constexpr int EPI_FIXED = 2 * NB + PGM_MAX_QD + 4 * (3 * PGM_MAX_QD + 1);          // alpha slices, weights, wave partials
constexpr int EPI_SLOTS = (CfgBig::LDS_DOUBLES - EPI_FIXED) / (2 * NB);             // staged factor rows (of 128) per side
static_assert(EPI_SLOTS >= 3 * 2 + 2, "epilogue staging needs room for one 2-D mixture");

// ---------------------------------------------------------------------------
// diag(A^-1)_c = sum_k V[k][c]^2 (column sums of squares of the inverse factor), needed
// for d mll / d noise_c = (alpha_c^2 - (A^-1)_cc) / 2N.  Memory-bound (reads V once).
// Work item (jb, sp): column block x row split; partial sums reduced by k_finalize.  The items run as the last
// nb * AINV_SPLITS workgroups of the k_lauum_grad launch (they are independent of it, and short).
// ---------------------------------------------------------------------------
constexpr int AINV_SPLITS = 32;
__device__ __forceinline__ void ainv_diag_item(const PgmDev& P, int jb, int sp, double* red, int b) {
  const double* A = P.A + b * P.sA;
  const double* Vjj = P.Dinv + b * P.sDinv + ((int64_t)jb * 2 + 1) * NB * NB;
  const int c = threadIdx.x & 127, half = threadIdx.x >> 7;
  const int own = own_rows(P, b);
  if (jb >= own) return;                                   // (uniform; trimmed ragged set: nobody reads these columns' sums)
  const int nrows = (own - jb) * NB;                       // rows jb*NB .. the light curve's last
  const int per = ((nrows + AINV_SPLITS - 1) / AINV_SPLITS + 7) / 8 * 8;
  const int r0 = sp * per, r1 = min(nrows, r0 + per);
  auto ld = [&](int rr) -> double {
    return (rr < NB) ? Vjj[rr * NB + c] : A[(int64_t)(jb * NB + rr) * P.ld + jb * NB + c];
  };
  double s0 = 0.0, s1 = 0.0, s2 = 0.0, s3 = 0.0;
  int rr = r0 + half;
  for (; rr + 6 < r1; rr += 8) {                           // four independent loads in flight per lane
    const double v0 = ld(rr), v1 = ld(rr + 2), v2 = ld(rr + 4), v3 = ld(rr + 6);
    s0 += v0 * v0; s1 += v1 * v1; s2 += v2 * v2; s3 += v3 * v3;
  }
  for (; rr < r1; rr += 2) { const double v0 = ld(rr); s0 += v0 * v0; }
  const double s = (s0 + s1) + (s2 + s3);
  if (half == 1) red[c] = s;
  __syncthreads();
  if (half == 0) P.dpart[b * P.sDpart + (int64_t)sp * P.np + jb * NB + c] = s + red[c];
}

// diag(A^-1) straight from the work items of the (j, j) tiles of A^-1: the lanes that hold diagonal elements write this item's
// share to its row of dpart (item number = k-blocks before it / k-blocks per item); k_finalize sums the rows the tile has
template <class C>
__device__ __forceinline__ void ainv_diag_from_tile(const PgmDev& P, int b, int j, int p0, const v4d (&acc)[C::TM][C::TN], const WavePos wp) {
  if (wp.m0 != wp.n0) return;
#pragma unroll
  for (int ti = 0; ti < C::TM; ++ti)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if ((wp.lane >> 4) + 4 * r == (wp.lane & 15))
        P.dpart[b * P.sDpart + (int64_t)((p0 - j) / P.ainv_from_tiles) * P.np + j * NB + acc_col<C>(wp, ti)] = acc[ti][ti][r];
}

// The same items as a launch of their own: big batches of small problems have tens of thousands of them, and inside the
// inverse/gradient launch they would run at its occupancy (two workgroups per CU, 64 KB of LDS each).
__global__ __launch_bounds__(256) void k_ainv_diag(PgmDev P) {
  __shared__ double red[NB];
  if (P.info[blockIdx.z] != 0) return;
  ainv_diag_item(P, (int)blockIdx.x, (int)blockIdx.y, red, (int)blockIdx.z);
}

// C = CfgBig: one workgroup per work item, the whole 128x128 tile.  C = CfgSub (few work items: short light curves, where one
// workgroup per tile would leave most CUs idle behind a 40 us gradient epilogue): four workgroups per work item, a 64x64
// sub-tile each -- launch index 4 * item + sub-tile, one row of partial sums per workgroup (P.nitems counts workgroups).
template <int D, int ORDER, class C>
__device__ __forceinline__ void lauum_grad_item(const PgmDev& P, double* lds, int b, int bx, int rows = -1) {
  constexpr int SUB = NB / C::BM;                              // sub-tiles per side (1 or 2)
  static_assert(C::BM == C::BN && C::NT == NTHREADS && (SUB == 1 || SUB == 2 || SUB == 4), "whole, quarter or sixteenth tiles");
  if (P.info[b] != 0) return;
#ifdef PGM_LAUUM_STAMPS       // (lab build: clock ticks of the phases of the launch's first work items, printed by their thread 0)
  long long lst_[8]; int lsn_ = 0;
#define LSTAMP() do { if (lsn_ < 8) lst_[lsn_++] = __builtin_amdgcn_s_memtime(); } while (0)
#else
#define LSTAMP() do {} while (0)
#endif
  LSTAMP();
  // the diag(A^-1) items ride at the end of the grid (placed first they delay the long inverse tiles: +0.04 ms)
  if (bx >= P.nitems) { const int a = bx - P.nitems; ainv_diag_item(P, a % P.nb, a / P.nb, lds, b); return; }
  // work item = (tile i <= j, k-blocks [p0, p0+len)): long inverse tiles are split along k so
  // that no single workgroup sets the makespan; the contraction below is linear in the tile
  const int lb = bx;
  // (rows >= 0, the 1-D grid of a trimmed ragged set with one work item per tile: the member's own tiles in triangular order)
  int4 item;
  if (rows >= 0) { int ti, tj; tri_decode(lb / (SUB * SUB), ti, tj); item = make_int4(ti, tj, tj, rows - tj); }
  else item = P.items[lb / (SUB * SUB)];
  const int i = item.x, j = item.y, p0 = item.z;
  int plen = item.w & 0xffff;
  const int own = rows >= 0 ? rows : own_rows(P, b);
  if (P.trim && rows < 0) {                                    // (the box of a trimmed ragged set: block rows p0 .. of the light curve's own)
    if (p0 >= own) {                                           // none (uniform): the item counts nothing, k_finalize sums a zero
      double* part0 = P.partials + b * P.sPart + (int64_t)lb * P.nslot;
      for (int s = threadIdx.x; s < P.nslot; s += NTHREADS) part0[s] = 0.0;
      return;
    }
    if (plen > own - p0) plen = own - p0;
  }
  const int mo = ((lb % (SUB * SUB)) / SUB) * C::BM, no = ((lb % (SUB * SUB)) % SUB) * C::BN;      // the sub-tile's place in the tile
  double* A = P.A + b * P.sA;
  const double* Dv = P.Dinv + b * P.sDinv;
  const int64_t ld = P.ld;
  v4d acc[C::TM][C::TN];
  // A diagonal tile (i == j) is symmetric: its four wavefronts compute the upper MFMA tiles of the two diagonal quadrants and
  // half of quadrant (0, 64) each, nobody quadrant (64, 0) (pgm_gemm.h, "Symmetric tiles"): 0.625 of a full tile's time, for
  // the multiply loop and for the gradient epilogue behind it.  (Whole tiles only: the quarter-tile form of short light curves
  // keeps full tiles.)
  WavePos wp = wave_pos<C>();
  int shape = SH_FULL;
  if constexpr (SUB == 1 && C::DIRECT) {
    if (i == j) {
      shape = (wp.wave == 0 || wp.wave == 3) ? SH_UPPER : (wp.wave == 1 ? SH_ROWS_LO : SH_ROWS_HI);
      if (wp.wave == 2) { wp.m0 = 0; wp.n0 = C::WN; }
    }
    shape = __builtin_amdgcn_readfirstlane(shape);
  }
  // (the sum over the block rows before p0 was left in R, negated, by the sweep's spare filler workgroups)
  const bool cont = (item.w & LAUUM_LOAD) != 0;
  const double* Rt = cont ? P.R + ((int64_t)i * NB + mo) * ld + j * NB + no : nullptr;
  auto operands = [&](int kb, const double*& pa, int64_t& lda, const double*& pb, int64_t& ldb) {
    const int p = p0 + kb;
#ifdef PGM_LAUUM_HOT            // (lab build, timing only: every work item multiplies the same two tiles -- what would perfect L2 locality be worth?)
    pa = A + (int64_t)(P.nb - 1) * NB * ld + mo; lda = ld; pb = A + (int64_t)(P.nb - 1) * NB * ld + NB + no; ldb = ld;
    return;
#endif
    if (p > i) { pa = A + (int64_t)p * NB * ld + i * NB + mo; lda = ld; }
    else { pa = Dv + ((int64_t)i * 2 + 1) * NB * NB + mo; lda = NB; }
    if (p > j) { pb = A + (int64_t)p * NB * ld + j * NB + no; ldb = ld; }
    else { pb = Dv + ((int64_t)j * 2 + 1) * NB * NB + no; ldb = NB; }
  };
  // (a member of a trimmed ragged set whose last block ends in padding: the rows of V beyond its last point are zero, whole
  //  groups of 16 of them are left out of the item's last k-block -- 512 x N ~ U{1024..2048}: 8 % of the pass's products)
  int skip_ks = 0;
  if (rows >= 0 && p0 + plen == own) skip_ks = ((own * NB - pts(P, b)) / 16) * 4;
  auto full_tile = [&]() {
    if (cont) acc_load_raw<C>(Rt, ld, acc, wp); else acc_zero<C>(acc);      // (negated inside gemm_tn)
    gemm_tn<C>(lds, plen, operands, acc, 0, cont, skip_ks);
  };
  if constexpr (SUB == 1 && C::DIRECT) {
    if (shape == SH_FULL) full_tile();
    else if (shape == SH_UPPER) { acc_init_shaped<C, SH_UPPER>(Rt, ld, acc, wp); gemm_direct_shaped<C, SH_UPPER>(wp, plen, operands, acc, cont, skip_ks); acc_clear_outside<C, SH_UPPER>(acc); }
    else if (shape == SH_ROWS_LO) { acc_init_shaped<C, SH_ROWS_LO>(Rt, ld, acc, wp); gemm_direct_shaped<C, SH_ROWS_LO>(wp, plen, operands, acc, cont, skip_ks); acc_clear_outside<C, SH_ROWS_LO>(acc); }
    else { acc_init_shaped<C, SH_ROWS_HI>(Rt, ld, acc, wp); gemm_direct_shaped<C, SH_ROWS_HI>(wp, plen, operands, acc, cont, skip_ks); acc_clear_outside<C, SH_ROWS_HI>(acc); }
  } else {
    full_tile();
  }

  LSTAMP();
  if constexpr (SUB == 1) { if (P.ainv_from_tiles && i == j) ainv_diag_from_tile<C>(P, b, j, p0, acc, wp); }
  // ---- epilogue: LDS is free again (gemm_tn ends on a barrier)
  const int Q = P.q;
  constexpr int QC = (EPI_SLOTS - D) / (3 * D);          // mixtures staged at once
  const int nchunks = (Q + QC - 1) / QC;
  double* arow = lds;
  double* acol = arow + NB;
  double* wl = acol + NB;
  double* wpart = wl + PGM_MAX_QD;                       // [4][nslot]
  double* rowd = lds + EPI_FIXED;                        // [3*qc*D + D][NB]: cos, sin, x*v per (q,d) then raw x per d
  double* cold = rowd + EPI_SLOTS * NB;
  const double* pre = P.pre + b * P.sPre;
  auto stage = [&](int q0, int qc) {                      // uniform across the workgroup
    __syncthreads();
    const int nfac = 3 * qc * D;
    for (int e = threadIdx.x; e < (nfac + D) * NB; e += NTHREADS) {
      const int slot = e / NB, m = e % NB;
      const int src = (slot < nfac) ? (3 * q0 * D + slot) : (3 * P.qd + (slot - nfac));
      rowd[e] = pre[(int64_t)src * P.np + i * NB + m];
      cold[e] = pre[(int64_t)src * P.np + j * NB + m];
    }
    __syncthreads();
  };
  if (threadIdx.x < NB) {
    arow[threadIdx.x] = P.alpha[b * P.sVec + i * NB + threadIdx.x];
    acol[threadIdx.x] = P.alpha[b * P.sVec + j * NB + threadIdx.x];
  }
  if (threadIdx.x < Q) wl[threadIdx.x] = P.hyp[(int64_t)b * (PGM_MAX_QD * 3) + threadIdx.x];
  for (int e = threadIdx.x; e < 4 * P.nslot; e += NTHREADS) wpart[e] = 0.0;
  if (nchunks == 1) stage(0, Q); else __syncthreads();
  LSTAMP();

  const double sym = (i == j) ? 1.0 : 2.0;
  const int npts = pts(P, b);
  double* mypart = wpart + wp.wave * P.nslot;
  // acc <- sym * G = sym * (alpha alpha^T - A^-1), in place; the diagonal of G is the noise gradient
#pragma unroll
  for (int ti = 0; ti < C::TM; ++ti)
#pragma unroll
    for (int tj = 0; tj < C::TN; ++tj)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = mo + acc_row<C>(wp, ti, r), n = no + acc_col<C>(wp, tj);
        const int gi = i * NB + m, gj = j * NB + n;
        const bool valid = (gi < npts) && (gj < npts);
        const double aa = (p0 + plen == own) ? arow[m] * acol[n] : 0.0;     // alpha alpha^T enters once per tile: with its last block row
        // (shaped diagonal tile: an MFMA tile above the diagonal stands for its mirror image too, the ones that were not computed count nothing)
        const double wt = shape == SH_FULL ? sym : (tj < shape_tj_lo(shape, ti) ? 0.0 : (shape == SH_UPPER && ti == tj) ? 1.0 : 2.0);
        acc[ti][tj][r] = (valid && wt != 0.0) ? wt * (aa - acc[ti][tj][r]) : 0.0;
      }
  LSTAMP();
  // One input dimension, every mixture staged at once (the usual case): mixtures outermost and the whole sub-tile unrolled
  // inside -- accumulator elements are addressed statically (no copy of a row of G per step), the three sums are reduced
  // across the wavefront once per mixture instead of once per mixture and MFMA-tile row, the time difference and the row's
  // factors are read once per (row, mixture).  31 fp64 instructions per pair and mixture (45 in the general loop below):
  // difference, its square, 19 for the exponential, 4 for cosine and sine of the angle difference, 5 for the three sums.
  bool done = false;
  if constexpr (D == 1) {
    if (nchunks == 1) {
      done = true;
      const double* rowx = rowd + 3 * Q * NB;
      const double* colx = cold + 3 * Q * NB;
#pragma unroll 1
      for (int q = 0; q < Q; ++q) {
        const double* rq = rowd + q * 3 * NB;
        const double* cq = cold + q * 3 * NB;
        double gw = 0.0, gmu = 0.0, gv = 0.0;
#pragma unroll
        for (int ti = 0; ti < C::TM; ++ti) {
          const int tj_lo = shape_tj_lo(shape, ti);          // (uniform) the MFMA tiles of this row that count: tj_lo .. TN-1
          if (tj_lo >= C::TN) continue;
          double rc[4], rs[4], rv[4], rx[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int m = mo + acc_row<C>(wp, ti, r);
            rc[r] = rq[m]; rs[r] = rq[NB + m]; rv[r] = rq[2 * NB + m]; rx[r] = rowx[m];
          }
#pragma unroll
          for (int tj = 0; tj < C::TN; ++tj) {
            if (tj < tj_lo) continue;
            const int n = no + acc_col<C>(wp, tj);
            const double cc_ = cq[n], cs_ = cq[NB + n], cv = cq[2 * NB + n], cx = colx[n];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const double ds = rv[r] - cv;
              const double GE = acc[ti][tj][r] * exp_neg_fast(-(ds * ds));
              const double CC = __builtin_fma(rc[r], cc_, rs[r] * cs_);
              const double SN = __builtin_fma(rs[r], cc_, -(rc[r] * cs_));
              const double tau = rx[r] - cx;
              const double t = GE * tau;
              gw = __builtin_fma(GE, CC, gw);
              gmu = __builtin_fma(t, SN, gmu);
              gv = __builtin_fma(t, CC * tau, gv);
            }
          }
        }
        // (DPP row reductions here instead of the LDS-crossbar butterfly, wave_sum_dpp: N=4096 1.869 -> 1.863 ms, N=2048 0.552 -> 0.550,
        //  64 x N=2048 within the noise -- round 6, same-box A/B; not worth other gradient bits)
        gw = wave_sum(gw); gmu = wave_sum(gmu); gv = wave_sum(gv);
        if (wp.lane == 0) { mypart[q] += gw; mypart[Q + q] += gmu; mypart[2 * Q + q] += gv; }
      }
    }
  }
#pragma unroll 1
  for (int ti = 0; ti < C::TM && !done; ++ti) {
    const int tj_lo = shape_tj_lo(shape, ti);               // (uniform) the MFMA tiles of this row that count: tj_lo .. TN-1
    if (tj_lo >= C::TN) continue;
    double Sd[D][C::TN][4];
    v4d Gw[C::TN];                 // this ti's row of G tiles (runtime ti: select statically)
#pragma unroll
    for (int tt = 0; tt < C::TM; ++tt)
      if (tt == ti) {
#pragma unroll
        for (int tj = 0; tj < C::TN; ++tj) Gw[tj] = acc[tt][tj];
      }
    if (D == 2 && ORDER == 0) {
#pragma unroll
      for (int dd = 0; dd < D; ++dd)
#pragma unroll
        for (int tj = 0; tj < C::TN; ++tj)
#pragma unroll
          for (int r = 0; r < 4; ++r) Sd[dd][tj][r] = 0.0;
      for (int ch = 0; ch < nchunks; ++ch) {
        const int q0 = ch * QC, qc = min(QC, Q - q0);
        if (nchunks > 1) stage(q0, qc);
        for (int ql = 0; ql < qc; ++ql) {
#pragma unroll
          for (int dd = 0; dd < D; ++dd) {
            const int qd = ql * D + dd;
#pragma unroll
            for (int tj = 0; tj < C::TN; ++tj) {
              if (tj < tj_lo) continue;
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int m = mo + acc_row<C>(wp, ti, r), n = no + acc_col<C>(wp, tj);
                const double ds = rowd[(qd * 3 + 2) * NB + m] - cold[(qd * 3 + 2) * NB + n];
                const double e = exp_neg(-(ds * ds));
                const double cc = rowd[(qd * 3 + 0) * NB + m] * cold[(qd * 3 + 0) * NB + n] +
                                  rowd[(qd * 3 + 1) * NB + m] * cold[(qd * 3 + 1) * NB + n];
                Sd[dd][tj][r] += wl[q0 + ql] * e * cc;
              }
            }
          }
        }
      }
    }
    for (int ch = 0; ch < nchunks; ++ch) {
      const int q0 = ch * QC, qc = min(QC, Q - q0);
      if (nchunks > 1) stage(q0, qc);
      const double* rowx = rowd + 3 * qc * D * NB;
      const double* colx = cold + 3 * qc * D * NB;
      for (int ql = 0; ql < qc; ++ql) {
        const int q = q0 + ql;
        double gw = 0.0, gmu[D], gv[D];
#pragma unroll
        for (int dd = 0; dd < D; ++dd) { gmu[dd] = 0.0; gv[dd] = 0.0; }
#pragma unroll
        for (int tj = 0; tj < C::TN; ++tj) {
          if (tj < tj_lo) continue;                            // (a row of a shaped diagonal tile: only the tiles that were computed)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int m = mo + acc_row<C>(wp, ti, r), n = no + acc_col<C>(wp, tj);
            double E[D], CC[D], SN[D], TAU[D];
#pragma unroll
            for (int dd = 0; dd < D; ++dd) {
              const int qd = ql * D + dd;
              const double rc = rowd[(qd * 3 + 0) * NB + m], rsn = rowd[(qd * 3 + 1) * NB + m];
              const double cc_ = cold[(qd * 3 + 0) * NB + n], cs_ = cold[(qd * 3 + 1) * NB + n];
              const double ds = rowd[(qd * 3 + 2) * NB + m] - cold[(qd * 3 + 2) * NB + n];
              E[dd] = exp_neg(-(ds * ds));
              CC[dd] = rc * cc_ + rsn * cs_;
              SN[dd] = rsn * cc_ - rc * cs_;
              TAU[dd] = rowx[dd * NB + m] - colx[dd * NB + n];
            }
            const double G = Gw[tj][r];
            if (D == 1) {
              const double GE = G * E[0];
              gw += GE * CC[0];
              gmu[0] += GE * SN[0] * TAU[0];
              gv[0] += GE * CC[0] * TAU[0] * TAU[0];
            } else {
#pragma unroll
              for (int dd = 0; dd < D; ++dd) {
                const int o = (D == 2) ? 1 - dd : 0;
                const double oth = (ORDER == 0) ? Sd[o][tj][r] : E[o] * CC[o];
                const double GE = G * oth * E[dd];
                if (ORDER == 0) gw += GE * CC[dd];
                gmu[dd] += GE * SN[dd] * TAU[dd];
                gv[dd] += GE * CC[dd] * TAU[dd] * TAU[dd];
              }
              if (ORDER != 0) gw += G * E[0] * CC[0] * E[1 % D] * CC[1 % D];
            }
          }
        }
        gw = wave_sum(gw);
#pragma unroll
        for (int dd = 0; dd < D; ++dd) { gmu[dd] = wave_sum(gmu[dd]); gv[dd] = wave_sum(gv[dd]); }
        if (wp.lane == 0) {
          mypart[q] += gw;
#pragma unroll
          for (int dd = 0; dd < D; ++dd) {
            mypart[Q + q * D + dd] += gmu[dd];
            mypart[Q + Q * D + q * D + dd] += gv[dd];
          }
        }
      }
    }
  }
  LSTAMP();
  __syncthreads();
  double* part = P.partials + b * P.sPart + (int64_t)lb * P.nslot;
  for (int s = threadIdx.x; s < P.nslot; s += NTHREADS)
    part[s] = wpart[s] + wpart[P.nslot + s] + wpart[2 * P.nslot + s] + wpart[3 * P.nslot + s];
#ifdef PGM_LAUUM_STAMPS
  LSTAMP();
  if (threadIdx.x == 0 && b == 0 && (lb < 12 || lb == P.nitems - 1))
    printf("lauum item %d (i=%d j=%d p0=%d plen=%d cont=%d) ticks: multiply %d stage %d G %d epilogue %d all waves %d  start %lld\n", lb, i, j, p0, plen, (int)cont,
           (int)(lst_[1] - lst_[0]), (int)(lst_[2] - lst_[0]), (int)(lst_[3] - lst_[0]), (int)(lst_[4] - lst_[0]), (int)(lst_[5] - lst_[0]), lst_[0]);
#endif
#undef LSTAMP
}

// ---------------------------------------------------------------------------
// mll = -(||z||^2 + log det A + n log 2 pi) / 2n ;  gradients from the partials.
// ---------------------------------------------------------------------------
// One role of the finalise step on FIN_THREADS threads: role 0 = the scalars (mll, hyper-parameter gradients), role r >= 1 = the
// per-point gradients of points (r - 1) FIN_THREADS ...  (Round 4, measured and not kept: for short light curves the LAST workgroup
// of the inverse/gradient launch running these roles -- a ticket per workgroup behind a device-scope fence -- instead of a launch
// of its own: N=89 0.052 -> 0.057 ms, N=1000 0.278 -> 0.315; the fences cost more than the launch, as with round 3's combine mode.)
template <int FIN_THREADS>
__device__ __forceinline__ void finalize_role(const PgmDev& P, int b, int role, double* red) {
  const int t = threadIdx.x;
  const int bad = P.info[b];
  const int n = pts(P, b), cb = caller_slot(P, b);           // (ragged batches: this light curve's length and its place in the caller's arrays)
  // workgroup 0: the scalars (mll, hyper-parameter gradients); workgroups 1..: the per-point gradients
  // (mean and noise), FIN_THREADS points each -- side by side instead of one after the other
  // (a failed factorisation leaves NaN in every output, so that no caller steps on the previous evaluation's gradients)
  const double qnan = __longlong_as_double(0x7ff8000000000000LL);
  // results go to the workspace (the dense back-end and prediction read them there) and, where this evaluation's caller left
  // its output pointers (P.outp, written by k_precompute), straight to the caller's arrays
  double* c_mll = nullptr; double* c_gw = nullptr; double* c_gmu = nullptr; double* c_gv = nullptr;
  double* c_gnoise = nullptr; double* c_gmean = nullptr; int* c_info = nullptr;
  if (P.outp) {
    c_mll = (double*)P.outp[0]; c_gw = (double*)P.outp[1]; c_gmu = (double*)P.outp[2]; c_gv = (double*)P.outp[3];
    c_gnoise = (double*)P.outp[4]; c_gmean = (double*)P.outp[5]; c_info = (int*)P.outp[6];
  }
  const int64_t cs = P.outp ? (int64_t)P.outp[8] : P.cstride;   // points per light curve slot in the caller's arrays
  if (role > 0) {
    if (!P.need_grad) return;
    const double half_n = 0.5 / (double)n;
    const int i = (role - 1) * FIN_THREADS + t;
    if (bad) {
      if (i < n) {
        P.out_gmean[b * P.sVec + i] = qnan; P.out_gnoise[b * P.sVec + i] = qnan;
        if (c_gmean) c_gmean[(int64_t)cb * cs + i] = qnan;
        if (c_gnoise) c_gnoise[(int64_t)cb * cs + i] = qnan;
      }
      return;
    }
    if (i < n) {
      const double al = P.alpha[b * P.sVec + i];
      P.out_gmean[b * P.sVec + i] = al / (double)n;
      if (c_gmean) c_gmean[(int64_t)cb * cs + i] = al / (double)n;
      double dsum = 0.0;
      if (P.ainv_from_tiles) {
        const int cnt = (own_rows(P, b) - i / NB + P.ainv_from_tiles - 1) / P.ainv_from_tiles;      // work items of tile (jb, jb) that have block rows
        for (int sp = 0; sp < cnt; ++sp) dsum += P.dpart[b * P.sDpart + (int64_t)sp * P.np + i];
      } else {
#pragma unroll
        for (int sp = 0; sp < AINV_SPLITS; ++sp) dsum += P.dpart[b * P.sDpart + (int64_t)sp * P.np + i];
      }
      P.out_gnoise[b * P.sVec + i] = half_n * (al * al - dsum);
      if (c_gnoise) c_gnoise[(int64_t)cb * cs + i] = half_n * (al * al - dsum);
    }
    return;
  }
  // (a member of a trimmed ragged set: its own block rows -- nothing was written beyond them -- and, with one work item per
  //  tile, the partial sums of its own tiles)
  const int own = own_rows(P, b), own_items = P.trim_tri ? own * (own + 1) / 2 : P.nitems;
  double s = 0.0;
  for (int i = t; i < own * NB; i += FIN_THREADS) { const double zi = P.z[b * P.sVec + i]; s += zi * zi; }
  for (int kk = t; kk < own; kk += FIN_THREADS) s += P.logdet[b * P.sLogdet + kk];
  s = wave_sum(s);
  if ((t & 63) == 0) red[t >> 6] = s;
  __syncthreads();
  if (t == 0) {
    double tot = 0.0;
    for (int wv = 0; wv < FIN_THREADS / 64; ++wv) tot += red[wv];
    const double val = bad ? qnan : -0.5 * (tot + (double)n * log(2.0 * PI)) / (double)n;
    P.out_small[b * P.sOut + 0] = val;
    if (c_mll) c_mll[cb] = val;
    if (c_info) c_info[cb] = bad;
  }
  if (!P.need_grad) return;
  // slot s of the hyper-parameter gradients in the caller's arrays: w (q), mu (q*d), v (q*d)
  auto c_slot = [&](int s, double val) {
    if (s < P.q) { if (c_gw) c_gw[(int64_t)cb * P.q + s] = val; }
    else if (s < P.q + P.qd) { if (c_gmu) c_gmu[(int64_t)cb * P.qd + (s - P.q)] = val; }
    else if (s < P.q + 2 * P.qd) { if (c_gv) c_gv[(int64_t)cb * P.qd + (s - P.q - P.qd)] = val; }
  };
  if (bad) {
    if (t >= 1 && t < 1 + P.q + 2 * P.qd) { P.out_small[b * P.sOut + t] = qnan; c_slot(t - 1, qnan); }
    return;
  }
  const double half_n = 0.5 / (double)n;
  const int Q = P.q, QD = P.qd;
  const double* hyp = P.hyp + (int64_t)b * (PGM_MAX_QD * 3);
  const int wave = t >> 6, lane = t & 63;
  for (int sidx = wave; sidx < P.nslot; sidx += FIN_THREADS / 64) {
    const double* part = P.partials + b * P.sPart + sidx;
    double a0 = 0.0, a1 = 0.0, a2 = 0.0, a3 = 0.0;
    int tile = lane;
    for (; tile + 192 < own_items; tile += 256) {
      a0 += part[(int64_t)tile * P.nslot]; a1 += part[(int64_t)(tile + 64) * P.nslot];
      a2 += part[(int64_t)(tile + 128) * P.nslot]; a3 += part[(int64_t)(tile + 192) * P.nslot];
    }
    for (; tile < own_items; tile += 64) a0 += part[(int64_t)tile * P.nslot];
    double acc = wave_sum((a0 + a1) + (a2 + a3));   // fixed summation order: reproducible
    if (lane != 0) continue;
    double val = 0.0;
    if (sidx < Q) {
      val = half_n * acc;
    } else if (sidx < Q + QD) {
      const int qd = sidx - Q, q = qd / P.d;
      val = half_n * (-2.0 * PI) * hyp[q] * acc;
    } else if (sidx < Q + 2 * QD) {
      const int qd = sidx - Q - QD, q = qd / P.d;
      val = half_n * (-2.0 * TWO_PI_SQ) * hyp[Q + QD + qd] * hyp[q] * acc;
    }
    if (sidx < Q + 2 * QD) { P.out_small[b * P.sOut + 1 + sidx] = val; c_slot(sidx, val); }
    // the last slot (sum of the diagonal of G) is only needed for a scalar noise: the
    // caller sums g_noise instead, so nothing to do here.
  }
}

constexpr int FIN_THREADS_K = 1024;
__global__ __launch_bounds__(FIN_THREADS_K) void k_finalize(PgmDev P) {
  __shared__ double red[FIN_THREADS_K / 64];
  finalize_role<FIN_THREADS_K>(P, (int)blockIdx.z, (int)blockIdx.x, red);
}

template <int D, int ORDER, class C>
__global__ __launch_bounds__(256, 2) void k_lauum_grad(PgmDev P) {
  int b = blockIdx.z, bx = blockIdx.x;
  xcd_batch_remap(bx, b);
  __shared__ __attribute__((aligned(16))) double lds[CfgBig::LDS_DOUBLES];
  lauum_grad_item<D, ORDER, C>(P, lds, b, bx);
}
// ... of a trimmed ragged launch set with one work item per tile: the 1-D grid of the members' own tiles (RagClasses)
template <int D, int ORDER, class C>
__global__ __launch_bounds__(256, 2) void k_lauum_grad_rag(PgmDev P, RagClasses rc) {
  int b = 0, bx = 0, rows = -1;
  if (!rag_decode(rc, bx, b, rows)) return;
  __shared__ __attribute__((aligned(16))) double lds[CfgBig::LDS_DOUBLES];
  lauum_grad_item<D, ORDER, C>(P, lds, b, bx, rows);
}

// ---------------------------------------------------------------------------
// Generic dense K(x1, x2) for to_dense() / cross-covariances (not on the MLL path).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_sm_dense(const double* x1, int64_t n1, const double* x2, int64_t n2, int d,
                                                  const double* w, const double* mu, const double* v, int q,
                                                  const double* noise, double noise_scalar, int dim_order,
                                                  double* K, int64_t ldk) {
  const int64_t j = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const int64_t i = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6);
  if (i >= n1 || j >= n2) return;
  double S[PGM_MAX_D] = {0.0, 0.0};
  double K1 = 0.0;
  for (int qq = 0; qq < q; ++qq) {
    double prod = 1.0;
    for (int dd = 0; dd < d; ++dd) {
      const double a = x1[i * d + dd], c = x2[j * d + dd];
      const double m = mu[qq * d + dd], s = v[qq * d + dd];
      const double ds = a * s - c * s;
      const double e = exp_neg(-TWO_PI_SQ * ds * ds) * cospi(2.0 * (a * m - c * m));
      if (dim_order == 0) S[dd] += w[qq] * e; else prod *= e;
    }
    if (dim_order != 0) K1 += w[qq] * prod;
  }
  double val = K1;
  if (dim_order == 0) { val = 1.0; for (int dd = 0; dd < d; ++dd) val *= S[dd]; }
  if (i == j && x1 == x2) val += noise_scalar + (noise ? noise[i] : 0.0);
  K[i * ldk + j] = val;
}

// ---------------------------------------------------------------------------
// Posterior prediction.  Ks[p][m] = k(x_p, x*_m) is
// built tile-wise, then B = U^-T Ks by the same block forward substitution as the
// factorisation sweep (row solve + trailing update on the right-hand sides), and
//   mean*_m = m*_m + sum_p B[p][m] z_p ,   var*_m = k(x*,x*) - sum_p B[p][m]^2 .
// ---------------------------------------------------------------------------
template <int D, int ORDER>
__global__ __launch_bounds__(256) void k_pred_cross(PgmDev P, const double* __restrict__ xt, int64_t M, int64_t Mp,
                                                    double* __restrict__ Ks) {
  const int jb = blockIdx.x, ib = blockIdx.y;
  extern __shared__ __attribute__((aligned(16))) double sm[];
  double* rowd = sm;
  double* cold = sm + P.pre_slots * NB;
  double* wl = cold + P.pre_slots * NB;
  const double* pre = P.pre;
  const double* hyp = P.hyp;
  for (int e = threadIdx.x; e < P.pre_slots * NB; e += NTHREADS) {
    const int slot = e / NB, m = e % NB;
    rowd[e] = pre[(int64_t)slot * P.np + ib * NB + m];
  }
  for (int e = threadIdx.x; e < P.qd * NB; e += NTHREADS) {
    const int qd = e / NB, c = e % NB, dd = qd % P.d;
    const int64_t gj = (int64_t)jb * NB + c;
    const double xj = (gj < M) ? xt[gj * P.d + dd] : 0.0;
    double s, co;
    sincospi(2.0 * (xj * hyp[P.q + qd]), &s, &co);
    cold[(qd * 3 + 0) * NB + c] = co;
    cold[(qd * 3 + 1) * NB + c] = s;
    cold[(qd * 3 + 2) * NB + c] = xj * hyp[P.q + P.qd + qd] * PI_SQRT2;      // (the scaling of k_precompute's staged factors)
  }
  if (threadIdx.x < P.q) wl[threadIdx.x] = hyp[threadIdx.x];
  __syncthreads();
  const int c2 = (threadIdx.x & 63) * 2, rg = threadIdx.x >> 6;
  for (int rr = 0; rr < NB / 4; ++rr) {
    const int m = rg + 4 * rr;
    const int gi = ib * NB + m;
    v2d out;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t gj = (int64_t)jb * NB + c2 + u;
      out[u] = (gi < P.n && gj < M) ? sm_pair<D, ORDER>(rowd, cold, wl, P.q, m, c2 + u) : 0.0;
    }
    *reinterpret_cast<v2d*>(Ks + (int64_t)gi * Mp + (int64_t)jb * NB + c2) = out;
  }
}

__global__ __launch_bounds__(256, 2) void k_pred_trsm(PgmDev P, int k, double* Ks, int64_t Mp) {
  using C = CfgTrsm;
  double* Cb = Ks + (int64_t)k * NB * Mp + (int64_t)blockIdx.x * C::BN;
  const double* Uinv = P.Dinv + (int64_t)k * 2 * NB * NB;
  __shared__ __attribute__((aligned(16))) double lds[C::LDS_DOUBLES];
  v4d acc[C::TM][C::TN];
  acc_zero<C>(acc);
  gemm_tn<C>(lds, 1, [&](int, const double*& pa, int64_t& lda, const double*& pb, int64_t& ldb) {
    pa = Uinv; lda = NB; pb = Cb; ldb = Mp;
  }, acc);
  acc_store<C>(Cb, Mp, acc, 1.0);
}

__global__ __launch_bounds__(256, 2) void k_pred_update(PgmDev P, int k, double* Ks, int64_t Mp) {
  using C = CfgBig;
  const int i = k + 1 + blockIdx.y;
  const double* pa0 = P.A + (int64_t)k * NB * P.ld + i * NB;
  const double* pb0 = Ks + (int64_t)k * NB * Mp + (int64_t)blockIdx.x * NB;
  double* Cp = Ks + (int64_t)i * NB * Mp + (int64_t)blockIdx.x * NB;
  const int64_t ld = P.ld;
  __shared__ __attribute__((aligned(16))) double lds[C::LDS_DOUBLES];
  v4d acc[C::TM][C::TN];
  acc_load_neg<C>(Cp, Mp, acc);
  gemm_tn<C>(lds, 1, [&](int, const double*& pa, int64_t& lda, const double*& pb, int64_t& ldb) {
    pa = pa0; lda = ld; pb = pb0; ldb = Mp;
  }, acc);
  acc_store<C>(Cp, Mp, acc, -1.0);
}

__global__ __launch_bounds__(256) void k_pred_reduce(PgmDev P, const double* __restrict__ Ks, int64_t M, int64_t Mp,
                                                     const double* __restrict__ mean_test, double* __restrict__ mean_out,
                                                     double* __restrict__ var_out, const double* __restrict__ kss_in) {
  const int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (m >= M) return;
  double s1 = 0.0, s2 = 0.0;
  for (int row = 0; row < P.np; ++row) {
    const double bv = Ks[(int64_t)row * Mp + m];
    s1 += bv * P.z[row];
    s2 += bv * bv;
  }
  double wsum = 0.0;
  for (int q = 0; q < P.q; ++q) wsum += P.hyp[q];
  double kss = wsum;
  if (P.dim_order == 0) for (int dd = 1; dd < P.d; ++dd) kss *= wsum;
  if (mean_out) mean_out[m] = (mean_test ? mean_test[m] : 0.0) + s1;
  if (kss_in) kss = kss_in[m];                     // dense back-end: prior variances supplied by the caller
  if (var_out) var_out[m] = kss - s2;
}

// back-to-back fp64 MFMA issue probe: accumulators pinned to VGPRs (the AGPR form of
// v_mfma_f64_16x16x4_f64 issues at half rate on gfx950)
__global__ __launch_bounds__(256) void k_probe_mfma(double* out, int iters) {
  v4d acc[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) acc[u] = v4d{0.0, 0.0, 0.0, 0.0};
  double a = 1.0 + threadIdx.x * 1e-9, bb = 1.0 - threadIdx.x * 1e-9;
  if (iters < 0) {                                             // (tools: operands with busy mantissas, |iters| iterations)
    iters = -iters;
    a = __longlong_as_double(0x3ff0000000000000LL | ((0x9e3779b97f4a7c15ULL * (threadIdx.x + 1) + blockIdx.x) >> 12));
    bb = __longlong_as_double(0x3fe0000000000000LL | ((0xc2b2ae3d27d4eb4fULL * (threadIdx.x + 7) + blockIdx.x) >> 12)) - 1.25;
  }
  for (int it = 0; it < iters; ++it) {
#pragma unroll
    for (int u = 0; u < 8; ++u) asm volatile("v_mfma_f64_16x16x4_f64 %0, %1, %2, %0" : "+v"(acc[u]) : "v"(a), "v"(bb));
  }
  double s = 0.0;
#pragma unroll
  for (int u = 0; u < 8; ++u) s += acc[u][0] + acc[u][1] + acc[u][2] + acc[u][3];
  if (s == 12345.678) out[0] = s;
}

// GEMM-core efficiency probe (tools only): every workgroup multiplies `nkb` k-blocks of operand
// strips; `spread` strips apart so that the operands either stay in L2 (spread = 0) or stream
template <class C>
__global__ __launch_bounds__(256, 2) void k_gemm_probe(const double* A, int64_t ld, int nkb, int spread, double* out) {
  __shared__ __attribute__((aligned(16))) double lds[C::LDS_DOUBLES];
  v4d acc[C::TM][C::TN];
  acc_zero<C>(acc);
  const int64_t off = (int64_t)(blockIdx.x % 16) * spread * C::BM;
  gemm_tn<C>(lds, nkb, [&](int kb, const double*& pa, int64_t& lda, const double*& pb, int64_t& ldb) {
    pa = A + (int64_t)kb * NB * ld + off; lda = ld; pb = A + (int64_t)kb * NB * ld + off + C::BM; ldb = ld;
  }, acc);
  double s = 0.0;
#pragma unroll
  for (int ti = 0; ti < C::TM; ++ti)
#pragma unroll
    for (int tj = 0; tj < C::TN; ++tj) s += acc[ti][tj][0] + acc[ti][tj][3];
  if (s == 1.2345) out[0] = s;
}

// Tile-product probe (tools only): workgroup t does what a trailing-update tile does -- reads its C tile, multiplies `nkb`
// k-blocks of two operand panels, writes the tile back -- on a synthetic 24-column arrangement of distinct tiles.
// MODE bit 0: the C tile is not read (accumulation from zero), bit 1: it is not written, bit 2: it is read
// unnegated and negated only after the first operand chunks were requested (one memory round trip instead of two).
template <class C, int WPS, int MODE = 0>
__global__ __launch_bounds__(C::NT, WPS) void k_tile_probe(double* A, int64_t ld, int nkb) {
  __shared__ __attribute__((aligned(16))) double lds[C::LDS_DOUBLES];
  constexpr int SUBM = NB / C::BM, SUBN = NB / C::BN;
  const int sub = blockIdx.x % (SUBM * SUBN), t = blockIdx.x / (SUBM * SUBN);
  const int r = 8 + t / 24, j = t % 24, si = sub / SUBN, sj = sub % SUBN;
  double* Cp = A + ((int64_t)r * NB + si * C::BM) * ld + j * NB + sj * C::BN;
  v4d acc[C::TM][C::TN];
  if (MODE & 4) acc_load_raw<C>(Cp, ld, acc);
  else if (MODE & 1) acc_zero<C>(acc); else acc_load_neg<C>(Cp, ld, acc);
  const double* pa0 = A + (int64_t)(r - 8) * NB + si * C::BM;
  const double* pb0 = A + (int64_t)j * NB + sj * C::BN;
  gemm_tn<C>(lds, nkb, [&](int kb, const double*& pa, int64_t& lda, const double*& pb, int64_t& ldb) {
    pa = pa0 + (int64_t)kb * NB * ld; lda = ld; pb = pb0 + (int64_t)kb * NB * ld; ldb = ld;
  }, acc, 0, (MODE & 4) != 0);
  if (MODE & 2) { if (acc[0][0][0] == 1.2345e300) Cp[0] = 0.0; } else acc_store<C>(Cp, ld, acc, -1.0);
}

// ---------------------------------------------------------------------------
// Dense back-end: the caller supplies A = K + noise as a dense symmetric matrix
// (any kernel: the shim's RBF / Matern / periodic / RQ / products / sums build it with torch), the same sweep
// factors it, and the gradient leaves as the dense matrix dmll/dA = (alpha alpha^T - A^-1) / 2N for torch's
// autograd to pull back through whatever built A.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_dense_in(PgmDev P, const double* __restrict__ Ain, int64_t lda,
                                                  const double* __restrict__ rin) {
  const int b = blockIdx.z;
  int ib, jb;
  tri_decode(blockIdx.x, ib, jb);
  if (blockIdx.x == 0 && threadIdx.x == 0) P.info[b] = 0;
  const double* Ab = Ain + (int64_t)b * P.n * lda;
  double* A = P.A + b * P.sA;
  const int c2 = (threadIdx.x & 63) * 2, rg = threadIdx.x >> 6;
  for (int rr = 0; rr < NB / 4; ++rr) {
    const int m = rg + 4 * rr;
    const int gi = ib * NB + m;
    v2d out;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int gj = jb * NB + c2 + u;
      double val;
      if (gi < P.n && gj < P.n) { val = Ab[(int64_t)gi * lda + gj]; if (gi == gj) val += P.jitter; }
      else val = (gi == gj) ? 1.0 : 0.0;
      out[u] = val;
    }
    *reinterpret_cast<v2d*>(A + (int64_t)gi * P.ld + jb * NB + c2) = out;
  }
  if (ib == jb && threadIdx.x < NB) {
    const int gi = ib * NB + threadIdx.x;
    P.r[b * P.sVec + gi] = (gi < P.n) ? rin[(int64_t)b * P.n + gi] : 0.0;
  }
}

// Upper-triangle tiles of G = scale * (alpha alpha^T - A^-1), accumulated over the k-split work items of a tile
// with fp64 atomics (G zeroed beforehand): reproducible to round-off only, unlike the fused SM path.
__global__ __launch_bounds__(256, 2) void k_lauum_dense(PgmDev P, double* __restrict__ G, int64_t ldg, double scale) {
  using C = CfgBig;
  const int b = blockIdx.z;
  if (P.info[b] != 0) return;
  const int4 item = P.items[blockIdx.x];
  const int i = item.x, j = item.y, p0 = item.z, plen = item.w;
  double* A = P.A + b * P.sA;
  const double* Dv = P.Dinv + b * P.sDinv;
  const int64_t ld = P.ld;
  __shared__ __attribute__((aligned(16))) double lds[C::LDS_DOUBLES];
  v4d acc[C::TM][C::TN];
  acc_zero<C>(acc);
  gemm_tn<C>(lds, plen, [&](int kb, const double*& pa, int64_t& lda, const double*& pb, int64_t& ldb) {
    const int p = p0 + kb;
    if (p > i) { pa = A + (int64_t)p * NB * ld + i * NB; lda = ld; }
    else { pa = Dv + ((int64_t)i * 2 + 1) * NB * NB; lda = NB; }
    if (p > j) { pb = A + (int64_t)p * NB * ld + j * NB; ldb = ld; }
    else { pb = Dv + ((int64_t)j * 2 + 1) * NB * NB; ldb = NB; }
  }, acc);
  double* arow = lds;
  double* acol = lds + NB;
  if (threadIdx.x < NB) {
    arow[threadIdx.x] = P.alpha[b * P.sVec + i * NB + threadIdx.x];
    acol[threadIdx.x] = P.alpha[b * P.sVec + j * NB + threadIdx.x];
  }
  __syncthreads();
  const WavePos wp = wave_pos<C>();
  double* Gb = G + (int64_t)b * P.n * ldg;
#pragma unroll
  for (int ti = 0; ti < C::TM; ++ti)
#pragma unroll
    for (int tj = 0; tj < C::TN; ++tj)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = acc_row<C>(wp, ti, r), n = acc_col<C>(wp, tj);
        const int gi = i * NB + m, gj = j * NB + n;
        if (gi < P.n && gj < P.n) {
          const double aa = (p0 == j) ? arow[m] * acol[n] : 0.0;
          unsafeAtomicAdd(Gb + (int64_t)gi * ldg + gj, scale * (aa - acc[ti][tj][r]));
        }
      }
}

// lower triangle of G <- transpose of the upper one (32x32 blocks through LDS)
__global__ __launch_bounds__(256) void k_dense_sym(double* __restrict__ G, int64_t ldg, int64_t n) {
  __shared__ double tile[32][33];
  const int b = blockIdx.z;
  const int bi = blockIdx.y, bj = blockIdx.x;           // block (bi, bj) of the LOWER triangle: bi > bj
  if (bi <= bj) return;
  double* Gb = G + (int64_t)b * n * ldg;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int rr = ty; rr < 32; rr += 8) {
    const int64_t gi = (int64_t)bj * 32 + rr, gj = (int64_t)bi * 32 + tx;      // upper block (bj, bi)
    tile[rr][tx] = (gi < n && gj < n) ? Gb[gi * ldg + gj] : 0.0;
  }
  __syncthreads();
  for (int rr = ty; rr < 32; rr += 8) {
    const int64_t gi = (int64_t)bi * 32 + rr, gj = (int64_t)bj * 32 + tx;
    if (gi < n && gj < n) Gb[gi * ldg + gj] = tile[tx][rr];
  }
}

__global__ __launch_bounds__(256) void k_dense_out(PgmDev P, double* __restrict__ mll, double* __restrict__ g_r, int* __restrict__ info) {
  const int b = blockIdx.z;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (blockIdx.x == 0 && threadIdx.x == 0) { mll[b] = P.out_small[b * P.sOut]; if (info) info[b] = P.info[b]; }
  if (g_r && i < P.n) g_r[(int64_t)b * P.n + i] = -P.alpha[b * P.sVec + i] / (double)P.n;
}

// right-hand sides of the dense prediction: the caller's K(x_train, x_test), zero padded
__global__ __launch_bounds__(256) void k_pred_in(PgmDev P, const double* __restrict__ Kin, int64_t ldk, int64_t M, int64_t Mp,
                                                 double* __restrict__ Ks) {
  const int64_t gj = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int gi = blockIdx.y;
  if (gj >= Mp) return;
  Ks[(int64_t)gi * Mp + gj] = (gi < P.n && gj < M) ? Kin[(int64_t)gi * ldk + gj] : 0.0;
}

__global__ __launch_bounds__(256) void k_fit_pre(FitDev F) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  __shared__ double mpar[PGM_MAX_D + 1];
  if (threadIdx.x < F.P && blockIdx.x == 0) {
    const int p = threadIdx.x;
    const double th = fit_theta(F, p);
    F.theta[p] = th;
    if (F.has_noise && p == F.P - 1) F.noise_scalar[0] = th;
  }
  // every workgroup needs the mean's parameters: recomputed locally instead of waiting for workgroup 0
  if (threadIdx.x < F.nmean) mpar[threadIdx.x] = fit_theta(F, threadIdx.x);
  __syncthreads();
  if (i < F.n) {
    double m = mpar[F.nmean - 1];                           // the constant, or the bias of a linear mean
    if (F.nmean > 1) for (int dd = 0; dd < F.d; ++dd) m += F.x[(int64_t)i * F.d + dd] * mpar[dd];
    F.mean_vec[i] = m;
  }
}

// after the evaluation: loss, gradients w.r.t. the raw parameters, optimiser step, log.  One workgroup of NT >= 256 threads, of
// which the first 256 work (k_fit_post: NT = 256; k_small, the one-launch evaluation of a short light curve: 1024) -- the same
// sums in the same order either way.  The evaluation's results may live in memory or in LDS (generic pointers).
// What one parameter's thread reads from memory for the step: loaded where the kernel starts (k_small: the loads complete behind
// the whole evaluation instead of in front of the step).
struct FitLoads {
  double raw, ca, cb, ploc, pscale, m1, m2, clip;
  int ckind, pkind, it;
};
__device__ __forceinline__ FitLoads fit_loads(const FitDev& F) {
  FitLoads L;
  const int t = threadIdx.x;
  L.it = F.it[0];
  L.clip = F.clip[0];
  L.raw = L.ca = L.cb = L.ploc = L.pscale = L.m1 = L.m2 = 0.0; L.ckind = L.pkind = 0;
  if (t < F.P) {
    L.raw = F.raw[t]; L.ckind = F.ckind[t]; L.ca = F.ca[t]; L.cb = F.cb[t];
    L.pkind = F.pkind[t]; L.ploc = F.ploc[t]; L.pscale = F.pscale[t]; L.m1 = F.m1[t]; L.m2 = F.m2[t];
  }
  return L;
}
__device__ __forceinline__ double fit_theta_of(const FitLoads& L) {
  if (L.ckind == 1) return softplus_d(L.raw) + L.ca;
  if (L.ckind == 2) return L.ca - softplus_d(-L.raw);
  if (L.ckind == 3) return sigmoid_d(L.raw) * L.cb + L.ca;
  return L.raw;
}

template <int NT>
__device__ __forceinline__ void fit_post_body(const FitDev& F, const FitLoads& L, const double* mll, const double* g_w, const double* g_mu, const double* g_v,
                                              const double* g_noise, const double* g_mean, double* red /*[256]*/, double* sums /*[PGM_MAX_D + 2]*/) {
  static_assert(NT >= 256, "the first 256 threads do the work");
  const int t = threadIdx.x;
  // sums of dmll/dmean_i (times x_i,dd for the weights of a linear mean) and, last, of dmll/dnoise_i
  if constexpr (NT > 256) {
    // (k_small: at most 128 points, the evaluation's results in LDS: one wavefront per sum, one barrier)
    const int wave = t >> 6, lane = t & 63;
    if (wave <= F.nmean) {
      const int which = wave;
      double s = 0.0;
      if (which == F.nmean) { if (F.has_noise) for (int i = lane; i < F.n; i += 64) s += g_noise[i]; }
      else if (which == F.nmean - 1) { for (int i = lane; i < F.n; i += 64) s += g_mean[i]; }
      else { for (int i = lane; i < F.n; i += 64) s += g_mean[i] * F.x[(int64_t)i * F.d + which]; }
      s = wave_sum_dpp(s);
      if (lane == 0) sums[which] = s;
    }
    __syncthreads();
  } else {
    for (int which = 0; which <= F.nmean; ++which) {
      double s = 0.0;
      if (which == F.nmean) { if (F.has_noise) for (int i = t; i < F.n; i += 256) s += g_noise[i]; }
      else if (which == F.nmean - 1) { for (int i = t; i < F.n; i += 256) s += g_mean[i]; }
      else { for (int i = t; i < F.n; i += 256) s += g_mean[i] * F.x[(int64_t)i * F.d + which]; }
      red[t] = s;
      __syncthreads();
      for (int h = 128; h > 0; h >>= 1) { if (t < h) red[t] += red[t + h]; __syncthreads(); }
      if (t == 0) sums[which] = red[0];
      __syncthreads();
    }
  }
  const int it = L.it;
  // log prior of every parameter and its derivative w.r.t. the constrained value
  double lp = 0.0, dlp = 0.0;
  if (t < F.P && L.pkind != 0) {
    const double th = fit_theta_of(L), mu = L.ploc, sg = L.pscale;
    constexpr double HALF_LOG_2PI = 0.91893853320467274178;
    if (L.pkind == 1) {
      const double zz = (th - mu) / sg;
      lp = -0.5 * zz * zz - log(sg) - HALF_LOG_2PI;
      dlp = -zz / sg;
    } else {
      const double lt = log(th), zz = (lt - mu) / sg;
      lp = -0.5 * zz * zz - log(sg) - HALF_LOG_2PI - lt;
      dlp = -(1.0 + zz / sg) / th;
    }
  }
  double lp_sum;
  if constexpr (NT > 256) {
    lp_sum = t < 64 ? wave_sum_dpp(lp) : 0.0;                  // (P <= 51 parameters: all of them in wavefront 0, and so is thread 0, the only reader)
  } else {
    red[t] = lp;
    __syncthreads();
    for (int h = 128; h > 0; h >>= 1) { if (t < h) red[t] += red[t + h]; __syncthreads(); }
    lp_sum = red[0];
  }
  // a failed factorisation (NaN value and gradients): the step is skipped -- parameters and moments stay as they are, the
  // log holds the NaN loss for the host to find at its next read
  const bool ok = isfinite(mll[0]);
  if (t < F.P && it < F.max_iter && !ok) F.raw_hist[(int64_t)it * F.P + t] = L.raw;
  double g = 0.0;                                           // d(-mll)/d raw_p
  if (t < F.P && it < F.max_iter && ok) {
    const int p = t, o = F.nmean;
    double gth;                                             // d(-mll)/d theta_p
    if (p < o) gth = -sums[p];
    else if (p < o + F.q) gth = -g_w[p - o];
    else if (p < o + F.q + F.qd) gth = -g_mu[p - o - F.q];
    else if (p < o + F.q + 2 * F.qd) gth = -g_v[p - o - F.q - F.qd];
    else gth = -sums[F.nmean];
    gth -= dlp / (double)F.n;
    const double r = L.raw;
    double dth = 1.0;                                       // d theta / d raw
    if (L.ckind == 1) dth = sigmoid_d(r);
    else if (L.ckind == 2) dth = sigmoid_d(-r);
    else if (L.ckind == 3) { const double sg = sigmoid_d(r); dth = L.cb * sg * (1.0 - sg); }
    g = gth * dth;
  }
  if (L.clip >= 0.0 && t < 64) {
    // the gradient's norm (P <= 52 entries: wavefront 0 holds them all), scaled by the largest entry so that no square overflows.  Zero,
    // an infinity or a NaN as the largest entry is the norm itself (inf / inf would make a NaN of it: a factor of zero is due there)
    double top = fabs(g);
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) { const double v = __shfl_xor(top, s); top = (v > top || v != v) ? v : top; }
    const bool scaled = top > 0.0 && top <= 1.7976931348623157e308;
    const double q = scaled ? g / top : 0.0;
    const double norm = scaled ? top * sqrt(wave_sum_dpp(q * q)) : top;
    const double c = L.clip / (norm + 1e-6);
    if (!(c >= 1.0)) g *= c;
  }
  if (t < F.P && it < F.max_iter && ok) {
    const int p = t;
    const double r = L.raw;
    double x = r;
    if (F.optimizer == 0) {
      x = r - F.lr * g;
    } else {
      if (F.optimizer == 2) x = r * (1.0 - F.lr * F.weight_decay);
      const double a = F.beta1 * L.m1 + (1.0 - F.beta1) * g;
      const double v2 = F.beta2 * L.m2 + (1.0 - F.beta2) * g * g;
      F.m1[p] = a; F.m2[p] = v2;
      const double step = (double)(it + 1);
      const double bc1 = 1.0 - pow(F.beta1, step), bc2 = 1.0 - pow(F.beta2, step);
      x -= (F.lr / bc1) * a / (sqrt(v2) / sqrt(bc2) + F.eps);
    }
    F.raw[p] = x;
    F.raw_hist[(int64_t)it * F.P + p] = x;
  }
  if (t == 0 && it < F.max_iter) F.loss_hist[it] = -(mll[0] + lp_sum / (double)F.n);
  if (t == 0) {                                             // (every thread read the counter when the kernel started)
    F.it[0] = it + 1;
    if (F.it_host) { __threadfence_system(); F.it_host[0] = it + 1; }       // (behind this iteration's log entries)
  }
}

__global__ __launch_bounds__(256) void k_fit_post(FitDev F, const double* __restrict__ mll, const double* __restrict__ g_w,
                                                  const double* __restrict__ g_mu, const double* __restrict__ g_v,
                                                  const double* __restrict__ g_noise, const double* __restrict__ g_mean) {
  __shared__ double red[256], sums[PGM_MAX_D + 2];
  const FitLoads L = fit_loads(F);
  fit_post_body<256>(F, L, mll, g_w, g_mu, g_v, g_noise, g_mean, red, sums);
}

// k_finalize and k_fit_post in one launch (one light curve of at most FIN_THREADS_K = 1024 points: the scalars and the per-point
// gradients are ONE workgroup's work, and the optimiser step needs nothing from anybody else): the iteration of pgm_fit_* loses a launch.
__global__ __launch_bounds__(FIN_THREADS_K) void k_finalize_fit(PgmDev P, FitDev F) {
  __shared__ double red[256], sums[PGM_MAX_D + 2];
  const FitLoads L = fit_loads(F);
  finalize_role<FIN_THREADS_K>(P, 0, 0, red);
  finalize_role<FIN_THREADS_K>(P, 0, 1, red);
  __syncthreads();                                              // (the results are in the caller's arrays: this workgroup's own stores, complete)
  const double* mll = (const double*)P.outp[0];
  fit_post_body<FIN_THREADS_K>(F, L, mll, (const double*)P.outp[1], (const double*)P.outp[2], (const double*)P.outp[3],
                               (const double*)P.outp[4], (const double*)P.outp[5], red, sums);
}

// ---------------------------------------------------------------------------
// ONE LAUNCH for a light curve of at most 128 points (round 6; spectral mixture, one or two input dimensions).  The reference's one published workload is
// N = 89 (/root/reference/paper/paper.md:113): a single diagonal block, for which an evaluation used to be k_prebuild -> k_diag ->
// k_lauum_grad -> k_finalize -- four dependent launches of which only the second does more than a few microseconds of work -- and a
// training iteration seven (k_fit_pre, k_precompute, k_build, k_diag, k_lauum_grad, k_finalize, k_fit_post).  Here one workgroup of
// 16 wavefronts per light curve does all of it, and nothing but results and the state prediction reads later touches memory:
//   A  (FIT) raw -> constrained parameters; the mixture's parameters to LDS
//   B  per-point factors cos / sin(2 pi x mu_q), x v_q pi sqrt 2, residual and diagonal addend: LDS (and the workspace, for prediction)
//   C  the diagonal block's factorisation exactly as k_diag runs it (diag_chain / diag_worker / the bookkeeping wavefront) -- but a
//      wavefront BUILDS the 16x16 sub-blocks it owns straight from the factors in LDS, in the MFMA C layout they are factored in:
//      the kernel matrix is never written to memory (same expressions as build_part_1d, hence the same matrix bits)
//   D  V = U^-T back from the inverse image just written (L2) into LDS as 16x16 fragments; A^-1 = V^T V sub-block by sub-block over
//      the upper triangle (4 MFMAs per sub-block row), the sub-blocks dealt to the 16 wavefronts
//   E  G = alpha alpha^T - A^-1 contracted with dK/d(w, mu, v) in registers (the 1-D epilogue of lauum_grad_item), diag(A^-1) -> noise gradient
//   F  mll, gradients, status -> the caller's arrays and the workspace;  (FIT) the optimiser step of k_fit_post
// The batch rides on gridDim.z (any number of short light curves per call, each with its own length: pts()).
// ---------------------------------------------------------------------------
template <int D, int ORDER>
struct LoadFromFactors {
  const double* fac;    // LDS [(3 qd + k) * NB + m]: cos, sin, x v pi sqrt2 per (mixture, dimension); then raw x per dimension
  const double* wl;     // LDS [Q] mixture weights
  const double* dadd;   // LDS [NB] diagonal addend
  int Q, n;
  __device__ __forceinline__ v4d operator()(const DiagCtx&, int i, int j, int lane) const {
    const int g = lane >> 4, col = j * DB + (lane & 15);
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    if constexpr (D == 1) {                                     // (the expressions of build_part_1d)
      for (int q = 0; q < Q; ++q) {
        const double wq = wl[q];
        const double* cq = fac + q * 3 * NB;
        const double cc0 = wq * cq[col], cs0 = wq * cq[NB + col], cv0 = cq[2 * NB + col];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int m = i * DB + g + 4 * r;
          const double rc = cq[m], rs = cq[NB + m], rv = cq[2 * NB + m];
          const double d0 = rv - cv0;
          acc[r] = __builtin_fma(exp_neg_fast(-(d0 * d0)), __builtin_fma(rc, cc0, rs * cs0), acc[r]);
        }
      }
    } else {                                                    // (k_build<2, ORDER>: sm_pair on the staged factors)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] = sm_pair<D, ORDER>(fac, fac, wl, Q, i * DB + g + 4 * r, col);
    }
    v4d out;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int gi = i * DB + g + 4 * r;
      double val = acc[r];
      if (gi < n && col < n) { if (gi == col) val += dadd[gi]; }
      else val = (gi == col) ? 1.0 : 0.0;
      out[r] = val;
    }
    return out;
  }
};

constexpr int SMALL_MAXT = 3;                                  // sub-blocks of the upper triangle per wavefront: ceil(36 / 16)
constexpr int SMALL_VIMG = (NB / DB) * (NB / DB + 1) / 2 * DB * DB;   // 36 sub-blocks of 256
// doubles of dynamic LDS
__host__ __device__ constexpr int small_lds_doubles(int q, int d = 1) {
  return SMALL_VIMG + (3 * q * d + d) * NB + DB * DB + 8 * NB + 64 + 64 + 3 * PGM_MAX_QD + 64 + 8 + 16 * (3 * PGM_MAX_QD + 1) + 256 + 8 + 10 * 64;
}

template <bool FIT, int D = 1, int ORDER = 0>
__global__ __launch_bounds__(DIAG_THREADS) void k_small(PgmDev P, FitDev F) {
  extern __shared__ __attribute__((aligned(16))) double sm[];
  constexpr int NS = NB / DB;
  const int b = blockIdx.z, t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int Q = P.q, QD = Q * D, nslot = Q + 2 * QD + 1;
  double* M = sm;                                   // factorisation: prow [2][8][256] | dg [8][256] | sup [8][256]; then the V image [36][256]
  double* fac = M + SMALL_VIMG;                     // [(3 Q D + D)][NB]
  double* uiS = fac + (3 * QD + D) * NB;            // [256]
  double* rsv = uiS + DB * DB;                      // residual (consumed by the forward substitution)
  double* zsv = rsv + NB;                           // z = V r
  double* alv = zsv + NB;                           // alpha = A^-1 r
  double* udg = alv + NB;                           // sqrt of the pivots
  double* dadd = udg + NB;                          // diagonal addend
  double* dvec = dadd + NB;                         // diag(A^-1)
  double* gme = dvec + NB;                          // dmll/dmean
  double* gno = gme + NB;                           // dmll/dnoise
  double* dump = gno + NB;                          // [64]
  double* thl = dump + 64;                          // [64] (FIT) constrained parameters
  double* hypl = thl + 64;                          // [3 * PGM_MAX_QD] w | mu | v
  double* outs = hypl + 3 * PGM_MAX_QD;             // [64] mll, g_w, g_mu, g_v
  double* misc = outs + 64;                         // [8] 0: log det, 1: status
  double* wpart = misc + 8;                         // [16][nslot]
  double* red = wpart + 16 * (3 * PGM_MAX_QD + 1);  // [256] (FIT)
  double* sums = red + 256;                         // [8]   (FIT) [7]: the gradient's limit
  double* fitl = sums + 8;                          // [10][64] (FIT) what the optimiser step reads from memory, parked here meanwhile
  const int cb = caller_slot(P, b), n = pts(P, b);
  const int nse = __builtin_amdgcn_readfirstlane((n + DB - 1) / DB);
  double* pre = P.pre + b * P.sPre;
#ifdef PGM_SMALL_STAMPS       // (lab build: clock ticks of the phases, wavefront 0 / a worker / the bookkeeper; printed by thread 0 of light curve 0)
  __shared__ long long stw_[16][4];
  long long sst_[12]; int ssn_ = 0;
#define SSTAMP() do { if (ssn_ < 12) sst_[ssn_++] = __builtin_amdgcn_s_memtime(); } while (0)
#else
#define SSTAMP() do {} while (0)
#endif
  SSTAMP();
  // (The inverse images' identity padding -- rows of sub-blocks the light curve does not have -- is NOT written here: only
  //  prediction multiplies with whole 128 x 128 images, and it completes them first, k_small_pad: up to 100 KB of stores per
  //  evaluation of a short light curve otherwise.  No barrier of this kernel waits for memory: lds_barrier.)

  // (the observation time this thread needs in phase B, requested now: its round trip overlaps that of the parameters)
  // (dimension (t >> 7) % D of point t & 127: what this thread needs in every round of the factor loop below)
  const double x_pre = ((t & (NB - 1)) < n) ? P.x[((int64_t)cb * P.cstride + (t & (NB - 1))) * D + ((t >> 7) % D)] : 0.0;
  double y_pre = 0.0, nz_pre = 0.0, mean_pre = 0.0;
  if (t < NB && t < n) {
    const int64_t ci = (int64_t)cb * P.cstride + t;
    y_pre = P.y[ci];
    nz_pre = P.noise ? P.noise[ci] : 0.0;
    if (!FIT) mean_pre = P.mean[ci];
  }
  // ---- A: the mixture's parameters
  if (FIT) {
    // (everything the optimiser step at the end reads from memory is requested now and parked in LDS: twenty registers per lane
    //  held across the whole kernel made the compiler spill)
    const FitLoads L = fit_loads(F);
    if (t < 64) {
      fitl[0 * 64 + t] = L.raw; fitl[1 * 64 + t] = L.ca; fitl[2 * 64 + t] = L.cb; fitl[3 * 64 + t] = L.ploc; fitl[4 * 64 + t] = L.pscale;
      fitl[5 * 64 + t] = L.m1; fitl[6 * 64 + t] = L.m2; fitl[7 * 64 + t] = (double)L.ckind; fitl[8 * 64 + t] = (double)L.pkind; fitl[9 * 64 + t] = (double)L.it;
      if (t == 0) sums[7] = L.clip;                             // (the sums take the first PGM_MAX_D + 2 places)
    }
    if (t < F.P) { const double th = fit_theta_of(L); thl[t] = th; F.theta[t] = th; if (F.has_noise && t == F.P - 1) F.noise_scalar[0] = th; }
    lds_barrier();
  }
  if (t < Q + 2 * QD) {                                          // [w (Q) | mu (Q D) | v (Q D)]
    double val;
    if (FIT) val = thl[F.nmean + t];
    else if (t < Q) val = P.w[(int64_t)cb * Q + t];
    else if (t < Q + QD) val = P.mu[(int64_t)cb * QD + (t - Q)];
    else val = P.v[(int64_t)cb * QD + (t - Q - QD)];
    hypl[t] = val;
    P.hyp[(int64_t)b * (PGM_MAX_QD * 3) + t] = val;
  }
  lds_barrier();
  SSTAMP();
  // ---- B: per-point factors
  const double nscal = FIT ? (F.has_noise ? thl[F.P - 1] : 0.0)
                           : P.noise_scalar + (P.noise_scalar_dev ? P.noise_scalar_dev[cb] : 0.0);
  for (int e = t; e < NB * QD; e += DIAG_THREADS) {
    const int m = e & (NB - 1), qd = e >> 7;                    // qd = q D + dd
    const double xi = x_pre;                                    // (m == t & 127 and dd == (t >> 7) % D in every round: 8 rows of 128 threads)
    const double mu = hypl[Q + qd], v = hypl[Q + QD + qd];
    double sn, cs;
    sincospi(2.0 * (xi * mu), &sn, &cs);
    const double xv = xi * v * PI_SQRT2;
    fac[(qd * 3 + 0) * NB + m] = cs; fac[(qd * 3 + 1) * NB + m] = sn; fac[(qd * 3 + 2) * NB + m] = xv;
    pre[(int64_t)(qd * 3 + 0) * P.np + m] = cs; pre[(int64_t)(qd * 3 + 1) * P.np + m] = sn; pre[(int64_t)(qd * 3 + 2) * P.np + m] = xv;
  }
  if (t < NB) {
    const int m = t;
    const bool valid = m < n;
    double xd[D];
    xd[0] = x_pre;                                             // (t < 128: dimension 0)
#pragma unroll
    for (int dd = 1; dd < D; ++dd) xd[dd] = valid ? P.x[((int64_t)cb * P.cstride + m) * D + dd] : 0.0;
#pragma unroll
    for (int dd = 0; dd < D; ++dd) { fac[(3 * QD + dd) * NB + m] = xd[dd]; pre[(int64_t)(3 * QD + dd) * P.np + m] = xd[dd]; }
    double mean_i;
    if (FIT) {
      mean_i = thl[F.nmean - 1];                               // the constant, or the bias of a linear mean (its d weights first)
      if (F.nmean > 1) for (int dd = 0; dd < D; ++dd) mean_i += xd[dd] * thl[dd];
      if (valid) F.mean_vec[m] = mean_i;
    } else mean_i = mean_pre;
    const double rr = valid ? (y_pre - mean_i) : 0.0;
    const double da = valid ? (nz_pre + nscal + P.jitter) : 0.0;
    rsv[m] = rr; zsv[m] = 0.0; alv[m] = 0.0; dadd[m] = da; dvec[m] = 0.0;
    const int64_t vi = (int64_t)b * P.sVec + m;
    P.r[vi] = rr; P.diagadd[vi] = da;
  }
  if (t == 0) { misc[0] = 0.0; misc[1] = 0.0; }
  lds_barrier();
  SSTAMP();

  // ---- C0: the sub-blocks of the upper triangle the light curve has, built by ALL 16 wavefronts into the (still unused) block image:
  // block (i, j), i <= j < nse, at j (j + 1) / 2 + i, row-major 16 x 16 -- the MFMA C layout's LDS form (diag_put / diag_get).
  // (The exp of the build is VALU work; the factorisation's workers sit on three of the four SIMDs and would spend 13 us on it.
  //  Measured and not kept: the chain factoring sub-block (0, 0) beside the build instead of behind it -- the build's wavefronts on
  //  the chain's SIMD slow that factorisation down by more than it gains: N=89 75.0k against 74.3k clock ticks, N=128, Q=4 131.3k / 128.7k.)
  {
    const LoadFromFactors<D, ORDER> build{fac, hypl, dadd, Q, n};
    const int T = nse * (nse + 1) / 2;
    for (int u = wave; u < T; u += 16) {
      int i, j;
      tri_decode(u, i, j);
      i = __builtin_amdgcn_readfirstlane(i); j = __builtin_amdgcn_readfirstlane(j);
      diag_put(M + u * DB * DB, build(DiagCtx{}, i, j, lane), lane);
    }
  }
  lds_barrier();
  SSTAMP();

  // ---- C: the factorisation (the roles of k_diag's workgroup 0); D: the inverse accumulates beside it
  DiagCtx c;
  c.prow = M; c.dg = M + 2 * NS * DB * DB; c.sup = c.dg + NS * DB * DB;
  c.uiS = uiS; c.udg = udg; c.dump = dump;
  c.Akk = nullptr; c.ld = 0;
  c.Dinv0 = P.Dinv + b * P.sDinv;
  c.Dinv1 = c.Dinv0 + NB * NB;
  // sub-block (i, j) from the image, or what the identity padding holds beyond the light curve's last sub-block row.
  // (Nothing writes the image before every wavefront has taken its blocks: the chain's first LDS write is V_00 over image block
  //  (0, 0), which only the chain reads; the workers publish block row 0 behind the step's first barrier, which they reach with
  //  their blocks in registers.)
  auto load = [&](const DiagCtx&, int i, int j, int ln) -> v4d {
    if (j < nse) return diag_get(M + (j * (j + 1) / 2 + i) * DB * DB, ln);      // (i <= j)
    v4d o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = (i == j && (ln >> 4) + 4 * r == (ln & 15)) ? 1.0 : 0.0;
    return o;
  };
  // A^-1 sub-block (i, j), i <= j, = sum over s >= j of V(s, i)^T V(s, j): sub-block number u = j (j + 1) / 2 + i belongs to worker
  // u mod 12 (at every step the blocks that receive a product, j <= s, are a prefix of that order: evenly dealt), at most 3 each
  v4d G[SMALL_MAXT];
#pragma unroll
  for (int k = 0; k < SMALL_MAXT; ++k) G[k] = v4d{0.0, 0.0, 0.0, 0.0};
  const int widx = wave - 1 - (wave >> 2);                      // worker number 0 .. 11 (workers only)
  int ti[SMALL_MAXT], tj[SMALL_MAXT];
#pragma unroll
  for (int k = 0; k < SMALL_MAXT; ++k) {
    int i = 0, j = NS;                                         // (j = NS: no such sub-block)
    const int u = widx + DIAG_WORKERS * k;
    if ((wave & 3) != 0 && u < NS * (NS + 1) / 2) tri_decode(u, i, j);
    ti[k] = __builtin_amdgcn_readfirstlane(i); tj[k] = __builtin_amdgcn_readfirstlane(j);
  }
  auto inverse_products = [&](int s, const double* row, int ln) {
    if (!P.need_grad) return;
#pragma unroll
    for (int k = 0; k < SMALL_MAXT; ++k) {
      if (tj[k] > s) continue;                                  // (uniform)
      const double* pa = row + ti[k] * DB * DB + ln;
      const double* pb = row + tj[k] * DB * DB + ln;
#pragma unroll
      for (int r = 0; r < 4; ++r) G[k] = __builtin_amdgcn_mfma_f64_16x16x4f64(pa[64 * r], pb[64 * r], G[k], 0, 0, 0);
    }
  };
  if (wave == 0) {
    diag_chain(c, lane, nse, load);
  } else if ((wave & 3) != 0) {
    diag_worker<decltype(load), decltype(inverse_products)&, false, true>(c, widx, lane, nse, load, inverse_products);
  } else if (wave == 4) {
    double lgsum = 0.0;
    int firstbad = -1;
    for (int s = 0; s < nse; ++s) {
      const double* row = c.prow + (s & 1) * NS * DB * DB;
      lds_barrier();
      if (lane < DB) {                                           // z_s = V_ss r_s (r_s is final since step s-1)
        double acc = 0.0;
#pragma unroll
        for (int kk = 0; kk < DB; ++kk) acc += uiS[kk * DB + lane] * rsv[s * DB + kk];
        zsv[s * DB + lane] = acc;
      }
      lds_barrier();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int colg = lane + 64 * u, jb = colg / DB;
        if (jb >= nse) continue;                                 // (columns of the identity padding: their blocks are not published)
        double acc = 0.0;
#pragma unroll
        for (int m = 0; m < DB; ++m) acc += row[jb * DB * DB + m * DB + (colg - jb * DB)] * zsv[s * DB + m];
        if (jb > s) rsv[colg] -= acc; else alv[colg] += acc;
      }
      {
        const double u = udg[s * DB + (lane & 15)];
        const unsigned long long badm = __ballot(!(u > 0.0 && u < 1e300)) & 0xffffull;
        if (badm && firstbad < 0) firstbad = s * DB + (int)__builtin_ctzll(badm);
        if (lane < DB) lgsum += 2.0 * log(u);
      }
    }
    const double tot = wave_sum(lgsum);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      P.z[b * P.sVec + lane + 64 * u] = zsv[lane + 64 * u];
      P.alpha[b * P.sVec + lane + 64 * u] = alv[lane + 64 * u];
    }
    if (lane == 0) {
      P.logdet[b * P.sLogdet] = tot;
      misc[0] = tot;
      const int info = firstbad >= 0 ? 1 + firstbad : 0;
      misc[1] = (double)info;
      // the status is final here: to the workspace and the caller; the host's copy follows right behind the barrier (below)
      P.info[b] = info;
      if (P.info_out) P.info_out[cb] = info;
    }
  } else {
    // waves 8 and 12: V_ss leaves for the two inverse images (one each)
    const int which = wave == 8 ? 1 : 2;
    for (int s = 0; s < nse; ++s) {
      lds_barrier();
      const v4d v = diag_get(c.prow + (s & 1) * NS * DB * DB + s * DB * DB, lane);
      lds_barrier();
      diag_store_v(c, s, s, v, lane, which);
    }
  }
#ifdef PGM_SMALL_STAMPS
  if (lane == 0) stw_[wave][0] = __builtin_amdgcn_s_memtime();
#endif
  SSTAMP();
  for (int e = t; e < 16 * nslot; e += DIAG_THREADS) wpart[e] = 0.0;
  lds_barrier();                                                // (LDS only: alpha, the status; the inverse images drain in the background)
  SSTAMP();
  const int bad = (int)misc[1];
  // the host may be polling for the status (the Python surface's psd_safe_cholesky-style check): it gets it before the gradient
  // epilogue, not behind it -- from the wavefront with the fewest sub-blocks to contract, and not in front of the barrier above
  // (a system-scope fence waits for the wavefront's earlier stores: on the bookkeeper it held every wavefront up for ~2 us)
  if (t == DIAG_THREADS - 64 && P.info_host) {
    P.info_host[b] = bad;
    __threadfence_system();
    P.seq_host[b] = P.seq;
  }
  const double qnan = __longlong_as_double(0x7ff8000000000000LL);
  const double half_n = 0.5 / (double)n;
  const bool grad = P.need_grad && !bad;
  // The gradient epilogue is VALU work (one exp per pair and mixture): the A^-1 sub-blocks go from the twelve workers, which sit on
  // three of the four SIMDs, through the block image (free again) to all sixteen wavefronts
  const int T = nse * (nse + 1) / 2;
  if (grad && (wave & 3) != 0) {
#pragma unroll
    for (int k = 0; k < SMALL_MAXT; ++k)
      if (tj[k] < nse) diag_put(M + (widx + DIAG_WORKERS * k) * DB * DB, G[k], lane);
  }
  lds_barrier();
  if (grad) {
    // ---- E: G = weight * (alpha alpha^T - A^-1) on the valid pairs, the diagonal of A^-1 for the noise gradient, and the contraction
    // with dK/d(w, mu, v) (the 1-D epilogue of lauum_grad_item on 16 x 16 sub-blocks)
    int nt = 0;
#pragma unroll
    for (int k = 0; k < SMALL_MAXT; ++k) {
      const int u = wave + 16 * k;
      int i = 0, j = NS;
      if (u < T) tri_decode(u, i, j);
      ti[k] = __builtin_amdgcn_readfirstlane(i); tj[k] = __builtin_amdgcn_readfirstlane(j);
      if (u >= T) continue;
      nt = k + 1;
      G[k] = diag_get(M + u * DB * DB, lane);
      const int g = lane >> 4, col = tj[k] * DB + (lane & 15);
      const double wt = (ti[k] == tj[k]) ? 1.0 : 2.0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = ti[k] * DB + g + 4 * r;
        if (ti[k] == tj[k] && m == col) dvec[m] = G[k][r];
        G[k][r] = (m < n && col < n) ? wt * (alv[m] * alv[col] - G[k][r]) : 0.0;
      }
    }
    const double* xs = fac + 3 * QD * NB;                       // raw x per dimension
    double* mypart = wpart + wave * nslot;
    if constexpr (D == 1) {
#pragma unroll 1
      for (int q = 0; q < Q; ++q) {
        const double* rq = fac + q * 3 * NB;
        double gw = 0.0, gmu = 0.0, gv = 0.0;
#pragma unroll
        for (int k = 0; k < SMALL_MAXT; ++k) {
          if (k >= nt || tj[k] >= nse) continue;
          const int g = lane >> 4, col = tj[k] * DB + (lane & 15);
          const double cc_ = rq[col], cs_ = rq[NB + col], cv = rq[2 * NB + col], cx = xs[col];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int m = ti[k] * DB + g + 4 * r;
            const double rc = rq[m], rs = rq[NB + m], rv = rq[2 * NB + m], rx = xs[m];
            const double ds = rv - cv;
            const double GE = G[k][r] * exp_neg_fast(-(ds * ds));
            const double CC = __builtin_fma(rc, cc_, rs * cs_);
            const double SN = __builtin_fma(rs, cc_, -(rc * cs_));
            const double tau = rx - cx;
            const double tt = GE * tau;
            gw = __builtin_fma(GE, CC, gw);
            gmu = __builtin_fma(tt, SN, gmu);
            gv = __builtin_fma(tt, CC * tau, gv);
          }
        }
        gw = wave_sum_dpp(gw); gmu = wave_sum_dpp(gmu); gv = wave_sum_dpp(gv);
        if (lane == 0) { mypart[q] = gw; mypart[Q + q] = gmu; mypart[2 * Q + q] = gv; }
      }
    } else {
      // two input dimensions (the general loop of lauum_grad_item on 16 x 16 sub-blocks): K = prod_d sum_q (ORDER 0) or sum_q prod_d
      auto pair_terms = [&](int qd, int m, int col, int dd, double& E, double& CC, double& SN, double& TAU) {
        const double* rq = fac + qd * 3 * NB;
        const double rc = rq[m], rsn = rq[NB + m], cc_ = rq[col], cs_ = rq[NB + col];
        const double ds = rq[2 * NB + m] - rq[2 * NB + col];
        E = exp_neg(-(ds * ds));
        CC = rc * cc_ + rsn * cs_;
        SN = rsn * cc_ - rc * cs_;
        TAU = xs[dd * NB + m] - xs[dd * NB + col];
      };
      double Sd[SMALL_MAXT][D][4];                               // ORDER 0: sum_q w_q E CC per dimension and pair
      if (ORDER == 0) {
#pragma unroll
        for (int k = 0; k < SMALL_MAXT; ++k)
#pragma unroll
          for (int dd = 0; dd < D; ++dd)
#pragma unroll
            for (int r = 0; r < 4; ++r) Sd[k][dd][r] = 0.0;
#pragma unroll 1
        for (int q = 0; q < Q; ++q) {
#pragma unroll
          for (int k = 0; k < SMALL_MAXT; ++k) {
            if (k >= nt || tj[k] >= nse) continue;
            const int g = lane >> 4, col = tj[k] * DB + (lane & 15);
#pragma unroll
            for (int dd = 0; dd < D; ++dd)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                double E, CC, SN, TAU;
                pair_terms(q * D + dd, ti[k] * DB + g + 4 * r, col, dd, E, CC, SN, TAU);
                Sd[k][dd][r] += hypl[q] * E * CC;
              }
          }
        }
      }
#pragma unroll 1
      for (int q = 0; q < Q; ++q) {
        double gw = 0.0, gmu[D], gv[D];
#pragma unroll
        for (int dd = 0; dd < D; ++dd) { gmu[dd] = 0.0; gv[dd] = 0.0; }
#pragma unroll
        for (int k = 0; k < SMALL_MAXT; ++k) {
          if (k >= nt || tj[k] >= nse) continue;
          const int g = lane >> 4, col = tj[k] * DB + (lane & 15);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int m = ti[k] * DB + g + 4 * r;
            double E[D], CC[D], SN[D], TAU[D];
#pragma unroll
            for (int dd = 0; dd < D; ++dd) pair_terms(q * D + dd, m, col, dd, E[dd], CC[dd], SN[dd], TAU[dd]);
            const double Gv = G[k][r];
#pragma unroll
            for (int dd = 0; dd < D; ++dd) {
              const int o = 1 - dd;
              const double oth = (ORDER == 0) ? Sd[k][o][r] : E[o] * CC[o];
              const double GE = Gv * oth * E[dd];
              if (ORDER == 0) gw += GE * CC[dd];
              gmu[dd] += GE * SN[dd] * TAU[dd];
              gv[dd] += GE * CC[dd] * TAU[dd] * TAU[dd];
            }
            if (ORDER != 0) gw += Gv * E[0] * CC[0] * E[1] * CC[1];
          }
        }
        gw = wave_sum_dpp(gw);
#pragma unroll
        for (int dd = 0; dd < D; ++dd) { gmu[dd] = wave_sum_dpp(gmu[dd]); gv[dd] = wave_sum_dpp(gv[dd]); }
        if (lane == 0) {
          mypart[q] = gw;
#pragma unroll
          for (int dd = 0; dd < D; ++dd) { mypart[Q + q * D + dd] = gmu[dd]; mypart[Q + QD + q * D + dd] = gv[dd]; }
        }
      }
    }
  }
  SSTAMP();
  lds_barrier();
  SSTAMP();

  // ---- F: results.  (A failed factorisation leaves NaN in every output, as k_finalize does.)
  if (wave == 0) {
    // (the order of k_finalize's sums, so that a light curve has the same value bit for bit whichever path evaluates it -- alone
    //  here, or as a member of a ragged launch set through the launch sequence: thread i holds z_i^2, thread 0 also the log det,
    //  one wavefront sum per 64 points, the two added in order)
    double s_lo = zsv[lane] * zsv[lane], s_hi = zsv[lane + 64] * zsv[lane + 64];
    // (k_finalize's products are rounded before anything is added to them -- there each is an fma onto 0.0 in a loop of its own.
    //  Here the compiler contracted the product into the first add behind it -- the log det on lane 0, the butterfly's first step on
    //  every lane: fma(z, z, neighbour) -- and the two paths differed in the value's last bit once in several hundred light curves;
    //  the ragged fuzz at 120 calls x ~40 members found one (`tools/lab/ragged_repro.py 31 17 13`).  The empty asm statements keep
    //  the products apart from the sums.)
    asm volatile("" : "+v"(s_lo));
    asm volatile("" : "+v"(s_hi));
    if (lane == 0) s_lo += misc[0];
    s_lo = wave_sum(s_lo); s_hi = wave_sum(s_hi);
    if (lane == 0) {
      double tot = 0.0;
      tot += s_lo; tot += s_hi;
      const double val = bad ? qnan : -0.5 * (tot + (double)n * log(2.0 * PI)) / (double)n;
#ifdef PGM_SMALL_PEEK
      P.partials[0] = s_lo; P.partials[1] = s_hi; P.partials[2] = tot; P.partials[3] = misc[0]; P.partials[4] = zsv[0]; P.partials[5] = val; P.partials[6] = (double)n;
#endif
      outs[0] = val;
      P.out_small[b * P.sOut] = val;
      if (P.mll) P.mll[cb] = val;
    }
  }
  if (P.need_grad) {
    if (t >= 64 && t < 64 + Q + 2 * QD) {                        // slot s of the hyper-parameter gradients: w (Q), mu (Q D), v (Q D)
      const int s3 = t - 64;
      double acc = 0.0;
      for (int wv = 0; wv < 16; ++wv) acc += wpart[wv * nslot + s3];     // fixed order
      double val;
      if (s3 < Q) val = half_n * acc;
      else if (s3 < Q + QD) val = half_n * (-2.0 * PI) * hypl[(s3 - Q) / D] * acc;
      else val = half_n * (-2.0 * TWO_PI_SQ) * hypl[s3] * hypl[(s3 - Q - QD) / D] * acc;
      if (bad) val = qnan;
      outs[1 + s3] = val;
      P.out_small[b * P.sOut + 1 + s3] = val;
      if (s3 < Q) { if (P.g_w) P.g_w[(int64_t)cb * Q + s3] = val; }
      else if (s3 < Q + QD) { if (P.g_mu) P.g_mu[(int64_t)cb * QD + (s3 - Q)] = val; }
      else { if (P.g_v) P.g_v[(int64_t)cb * QD + (s3 - Q - QD)] = val; }
    }
    if (t >= 128 && t < 128 + NB) {
      const int m = t - 128;
      const double al = alv[m];
      const double gm = bad ? qnan : al / (double)n, gn = bad ? qnan : half_n * (al * al - dvec[m]);
      gme[m] = (m < n) ? gm : 0.0; gno[m] = (m < n) ? gn : 0.0;
      if (m < n) {
        P.out_gmean[b * P.sVec + m] = gm; P.out_gnoise[b * P.sVec + m] = gn;
        if (P.g_mean) P.g_mean[(int64_t)cb * P.cstride + m] = gm;
        if (P.g_noise) P.g_noise[(int64_t)cb * P.cstride + m] = gn;
      }
    }
  }
  SSTAMP();
  if (FIT) {
    lds_barrier();
    FitLoads L;
    const int tl = t & 63;                                      // (P <= 51 parameters: wavefront 0 holds them; the others only need `it`)
    L.raw = fitl[0 * 64 + tl]; L.ca = fitl[1 * 64 + tl]; L.cb = fitl[2 * 64 + tl]; L.ploc = fitl[3 * 64 + tl]; L.pscale = fitl[4 * 64 + tl];
    L.m1 = fitl[5 * 64 + tl]; L.m2 = fitl[6 * 64 + tl]; L.ckind = (int)fitl[7 * 64 + tl]; L.pkind = (int)fitl[8 * 64 + tl]; L.it = (int)fitl[9 * 64 + tl];
    L.clip = sums[7];
    fit_post_body<DIAG_THREADS>(F, L, outs, outs + 1, outs + 1 + Q, outs + 1 + Q + QD, gno, gme, red, sums);
  }
  SSTAMP();
#ifdef PGM_SMALL_STAMPS
  __syncthreads();
  if (t == 0 && b == 0) {
    printf("k_small n=%d nse=%d q=%d ticks: ", n, nse, Q);
    for (int k = 1; k < ssn_; ++k) printf("%d ", (int)(sst_[k] - sst_[0]));
    printf("| role done (wave:ticks): ");
    for (int w = 0; w < 16; ++w) printf("%d:%d ", w, (int)(stw_[w][0] - sst_[0]));
    printf("\n");
  }
#endif
#undef SSTAMP
}

// The identity padding of the inverse images of a light curve k_small evaluated (workspace slot 0): rows / columns of the
// sub-blocks beyond its last one.  Launched by pgm_predict_f64 in front of its right-hand-side solve.
__global__ __launch_bounds__(256) void k_small_pad(PgmDev P) {
  const int nse = (P.n + DB - 1) / DB, first = nse * DB;
  double* inv0 = P.Dinv;                // [p][m] = V[m][p]
  double* inv1 = P.Dinv + NB * NB;      // [k][n] = V[k][n]
  for (int e = blockIdx.x * 256 + threadIdx.x; e < (NB - first) * NB; e += gridDim.x * 256) {
    const int k = first + e / NB, c = e % NB;          // row k >= first of V: zero but for the diagonal
    const double val = (k == c) ? 1.0 : 0.0;
    inv1[k * NB + c] = val;
    inv0[c * NB + k] = val;
  }
}

// ---------------------------------------------------------------------------
// The NUTS / HMC potential of config 5 on the device (pgm_pot_*, round 5): per chain b the unconstrained vector
//   z = [c, log w (q), log mu (q d), log v (q d) (, log sigma^2)]
// -> theta (k_pot_pre: exp for every site but the mean constant; the mean vector, the mixture arrays and the noise variance the
// evaluation reads), the fused evaluation, and (k_pot_post)
//   U(z) = -[ N mll(theta) + sum_p log Normal(z_p; loc_p, scale_p) ],   dU/dz_p = -[ N dmll/dtheta_p * dtheta_p/dz_p - (z_p - loc_p) / scale_p^2 ]
// (for a log site, LogNormal(loc, scale) on theta plus the Jacobian z is exactly the Normal(loc, scale) density of z: the
// reference's default priors, /root/reference/pgmuvi/lightcurve.py:3235-3330, in the coordinates pyro samples).  z comes from
// and U, dU/dz go to host-mapped memory: one graph replay per leapfrog step, no copy launches, no stream synchronisation
// (the host polls the stamp k_pot_post leaves behind its results).
// ---------------------------------------------------------------------------
struct PotDev {
  int B, P, n, q, qd, has_noise;
  const double* z;        // [B][P] host-mapped: this tick's positions
  const double* loc;      // [B][P]
  const double* scale;    // [B][P]
  double* theta;          // [B][P]
  double* mean_vec;       // [B][n]
  double* w;              // [B][q]
  double* mu;             // [B][qd]
  double* v;              // [B][qd]
  double* noise_scalar;   // [B]
  double* res;            // [B][1 + P] host-mapped: U, dU/dz
  int* res_info;          // [B] host-mapped
  long long* res_seq;     // [B] host-mapped: the tick number behind res (written last, system scope)
  const long long* tick;  // [1] host-mapped: this tick's number
};

__global__ __launch_bounds__(256) void k_pot_pre(PotDev F) {
  const int b = blockIdx.z, i = blockIdx.x * 256 + threadIdx.x;
  const double* z = F.z + (int64_t)b * F.P;
  if (blockIdx.x == 0 && threadIdx.x < F.P) {
    const int p = threadIdx.x;
    const double th = p == 0 ? z[0] : exp(z[p]);
    F.theta[(int64_t)b * F.P + p] = th;
    if (p >= 1 && p < 1 + F.q) F.w[(int64_t)b * F.q + p - 1] = th;
    else if (p >= 1 + F.q && p < 1 + F.q + F.qd) F.mu[(int64_t)b * F.qd + p - 1 - F.q] = th;
    else if (p >= 1 + F.q + F.qd && p < 1 + F.q + 2 * F.qd) F.v[(int64_t)b * F.qd + p - 1 - F.q - F.qd] = th;
    else if (p >= 1) F.noise_scalar[b] = th;
  }
  if (i < F.n) F.mean_vec[(int64_t)b * F.n + i] = z[0];
}

// one workgroup per chain
__global__ __launch_bounds__(256) void k_pot_post(PotDev F, const double* __restrict__ mll, const double* __restrict__ g_w,
                                                  const double* __restrict__ g_mu, const double* __restrict__ g_v,
                                                  const double* __restrict__ g_noise, const double* __restrict__ g_mean,
                                                  const int* __restrict__ info) {
  __shared__ double red[256], sums[2], lpsum;
  const int b = blockIdx.x, t = threadIdx.x;
  for (int which = 0; which < 2; ++which) {                   // sum of dmll/dmean_i; of dmll/dnoise_i (a learned noise variance)
    double s = 0.0;
    if (which == 0) for (int i = t; i < F.n; i += 256) s += g_mean[(int64_t)b * F.n + i];
    else if (F.has_noise) for (int i = t; i < F.n; i += 256) s += g_noise[(int64_t)b * F.n + i];
    red[t] = s;
    __syncthreads();
    for (int h = 128; h > 0; h >>= 1) { if (t < h) red[t] += red[t + h]; __syncthreads(); }
    if (t == 0) sums[which] = red[0];
    __syncthreads();
  }
  constexpr double HALF_LOG_2PI = 0.91893853320467274178;
  double lp = 0.0, g = 0.0;
  const int64_t o = (int64_t)b * F.P;
  if (t < F.P) {
    const int p = t;
    const double zz = (F.z[o + p] - F.loc[o + p]) / F.scale[o + p];
    lp = -0.5 * zz * zz - log(F.scale[o + p]) - HALF_LOG_2PI;
    double gth;                                               // dmll / dtheta_p
    if (p == 0) gth = sums[0];
    else if (p < 1 + F.q) gth = g_w[(int64_t)b * F.q + p - 1];
    else if (p < 1 + F.q + F.qd) gth = g_mu[(int64_t)b * F.qd + p - 1 - F.q];
    else if (p < 1 + F.q + 2 * F.qd) gth = g_v[(int64_t)b * F.qd + p - 1 - F.q - F.qd];
    else gth = sums[1];
    const double gl = p == 0 ? gth : gth * F.theta[o + p];      // d/dz = theta d/dtheta for the log sites
    g = -((double)F.n * gl - zz / F.scale[o + p]);
  }
  red[t] = lp;
  __syncthreads();
  for (int h = 128; h > 0; h >>= 1) { if (t < h) red[t] += red[t + h]; __syncthreads(); }
  if (t == 0) lpsum = red[0];
  __syncthreads();
  const double U = -((double)F.n * mll[b] + lpsum);
  const bool bad = info[b] != 0 || !isfinite(U);
  double* res = F.res + (int64_t)b * (1 + F.P);
  if (t == 0) { res[0] = bad ? __builtin_huge_val() : U; F.res_info[b] = info[b]; }
  if (t < F.P) res[1 + t] = bad ? 0.0 : g;
  __threadfence_system();
  __syncthreads();
  if (t == 0) F.res_seq[b] = F.tick[0];
}

#include "pgm_generic.inc"

}  // namespace

// ===========================================================================
// host side
// ===========================================================================
#include "pgm_host.inc"
