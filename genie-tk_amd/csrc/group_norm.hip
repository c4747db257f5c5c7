// Group norm with an activation over channels-last tensors, for gfx950.
//
// Over the m values of a sample's group that count (mask not 0): mean, var =
// mean(d^2) with d = x - mean, r = 1 / sqrt(var + eps), h = d r, z = h w + b and
// y = act(z).  Backward, with dz = dy act'(z) and g = dz w:
//   dx = r (g - mean(g) - h mean(g h)),  dw = sum dz h,  db = sum dz
// The statistics are sums of x - x0 and (x - x0)^2 in 64 bits around a value x0 that a
// thread has itself; threads and chunks are joined by their means and their sums of
// squares around them.  So the variance is off by 2^-53 of its root times the values'
// distance from zero, where sums of x^2 lose the square of that distance.  The mean is
// kept as a sum of two floats, so that d is off by its own rounding only.
//
// Memory bounds it: some 15 to 40 operations a value of 2 or 4 bytes.  A sample's
// group has to be read whole before its first result.  Where a slice of a sample
// (all its positions, some whole groups) fits the registers of one block, a block
// holds it from its one load to its one store.  Larger samples are streamed twice:
// one launch sums, the next one applies, in the opposite order, so that what was read
// last, and is still in the caches, comes first.
// On MI355X, inputs in rotation, forward and backward with both parameters: 4096 rows of
// 512 bf16 channels 8 + 19 us, of which a launch by itself is 3.4 (two block barriers a
// row, the backward pass' partial sums); 16 x 256 x 320 fp32 8 + 14; 8 x 4096 x 256 bf16
// 17 + 24; 2^18 x 128 bf16, 36 % of the positions masked, 41 + 61; 2^20 x 128 bf16 with
// gelu 161 + 274, without an activation 138 + 219, memory's time (each tensor of 268 MB
// twice, at 5.1 to 6.6 TB/s).
#include <math.h>

#include <algorithm>

#include "capi_util.hpp"
#include "column_sums.hpp"
#include "common.hpp"
#include "pack.hpp"
#include "row_vec.hpp"

namespace gtk {

// One sample's group, as gtk_group_norm_forward writes it.
struct GroupStats {
  float mean, low, rstd, inv;
};

// Some of a group's values: their mean x, and the sum y of their squared distances from it.
typedef double2 Moments;

// Of n values, from the sums of their distances from x0 and of those squared; inv = 1 / n,
// or 0 without.
__device__ __forceinline__ Moments around(double x0, double s, double q, double inv) {
  const double d = s * inv;
  return {x0 + d, fma(-d, s, q)};
}

// inv: as there.  v_rsq_f64 has 24 bits or more, what the result keeps.
__device__ __forceinline__ GroupStats close_stats(const Moments& m, double inv, float eps) {
  GroupStats g{0.f, 0.f, 0.f, 0.f};
  if (inv > 0) {
    const double var = m.y * inv;
    g.mean = (float)m.x;
    g.low = (float)(m.x - (double)g.mean);
    // a NaN stays one (fmax would drop it)
    g.rstd = (float)__builtin_amdgcn_rsq((var < 0 ? 0.0 : var) + (double)eps);
    g.inv = (float)inv;
  }
  return g;
}

// ---------------------------------------------------------------------------
// Activations.  The quotients are v_rcp_f32 (1 ulp); a division would take ten
// instructions.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float logistic(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

// The standard normal distribution's function below -|z| is e^(-z^2/2) t P(t) with t =
// 1 / (1 + 0.3 |z|), which keeps its relative accuracy to the end; P was fitted to
// erfcx (weighted least squares on |z| <= 14, iterated towards equal errors): 1.5e-7 of
// the value, 4.4e-7 with fp32's roundings.  Inputs of bf16 take the same: the
// parameters' gradients may be fp32 beside them.
struct Tail {
  float e, tp;  // e^(-z^2/2), t P(t)
  static constexpr float k = 0.3f;
  // k |z|, and -z^2 log2(e) / 2
  __device__ __forceinline__ Tail(float size, float power) {
    e = __builtin_amdgcn_exp2f(power);
    const float t = __builtin_amdgcn_rcpf(size + 1.f);
    float p = 0.03567477342812997f;
    p = fmaf(p, t, -0.1572030800704706f);
    p = fmaf(p, t, 0.20635350232969402f);
    p = fmaf(p, t, -0.05368364104385134f);
    p = fmaf(p, t, 0.1285616251824942f);
    p = fmaf(p, t, 0.09991349247240931f);
    p = fmaf(p, t, 0.12075395598321578f);
    p = fmaf(p, t, 0.11962929883230777f);
    tp = t * p;
  }
};

constexpr float kLargest = 3.402823466e38f;

// silu(z) = z s(z); gelu(z) = z Phi(z) = max(z, 0) - |z| Phi(-|z|), whose last product is 0
// at an infinite z too
template <int ACT> __device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == GTK_ACT_SILU) return z * logistic(z);
  if constexpr (ACT == GTK_ACT_GELU) {
    const Tail a(Tail::k * fabsf(z), z * z * -0.7213475204f);
    return fmaf(-fminf(fabsf(z), kLargest), a.e * a.tp, fmaxf(z, 0.f));
  }
  return z;
}
// silu' = s + z s (1 - s); gelu' = Phi(z) + z phi(z), 1 - that of -z.  The argument is
// kScale z, which the coefficients of z carry: one product less a value.  Of SiLU's it may
// be infinite where z is not.
template <int ACT> struct Slope {
  static constexpr float kScale =
      ACT == GTK_ACT_SILU ? 1.4426950409f : ACT == GTK_ACT_GELU ? 0.8493218003f : 1.f;  // log2(e); sqrt(log2(e) / 2)
};
template <int ACT> __device__ __forceinline__ float activate_slope(float u) {
  if constexpr (ACT == GTK_ACT_SILU) {
    constexpr float ln2 = 0.6931471806f;
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-u));
    return s * fmaf(__builtin_amdgcn_fmed3f(u, -kLargest, kLargest), fmaf(-s, ln2, ln2), 1.f);
  }
  if constexpr (ACT == GTK_ACT_GELU) {
    constexpr float back = 1.f / Slope<ACT>::kScale;
    const Tail a(Tail::k * back * fabsf(u), -(u * u));
    const float below = a.e * fmaf(-fabsf(u), 0.3989422804f * back, a.tp);
    return u < 0.f ? below : 1.f - below;
  }
  return 1.f;
}

// ---------------------------------------------------------------------------
// Threads over positions and channels.  A team of `threads` has `across` vectors of
// VE channels side by side and `rows` positions at once.  A vector's channels fall
// into SL slots, each within one group.  Where the width is no multiple of VE the
// last vector is moved back to end with it, and its first `skip` channels count for
// nothing in sums (both threads store the same results there).
// ---------------------------------------------------------------------------
template <typename T_, int VE_, int SL_> struct Form {
  typedef T_ T;
  static constexpr int VE = VE_, SL = SL_, CPS = VE / SL;  // channels a slot
};

struct Team {
  int threads, across, rows;
  int pitch;  // of a slot's (channel's) partial sums in LDS
  int lanes;  // that share one group's sum, a power of two
  int channel_lanes;
};

struct Shape {
  int64_t B, P;
  int C, G, cg;
  double inv;  // 1 / the values of a group

  static Shape of(int64_t B, int64_t P, int64_t C, int64_t G) {
    return {B, P, (int)C, (int)G, (int)(C / G), 1.0 / ((double)P * (double)(C / G))};
  }
  __device__ __forceinline__ double inverse(int64_t positions) const {
    return positions ? 1.0 / ((double)positions * (double)cg) : 0.0;
  }
};

template <typename F> struct Place {
  int at, row, skip;  // first channel within the slice
  bool on, first;     // threads past the last whole row repeat that one, and are off
  __device__ __forceinline__ Place(int t, const Team& g, int width) {
    row = t / g.across;
    const int nominal = (t - row * g.across) * F::VE;
    on = row < g.rows;
    if (!on) row = g.rows - 1;
    first = nominal == 0;
    at = nominal + F::VE <= width ? nominal : width - F::VE;
    skip = nominal - at;
  }
};

// Partial sums of N runs of channels each, [run][row of the team].
template <int N, int VE, typename S>
__device__ __forceinline__ void put_sums(S* sums, const S (&v)[N], int at, int skip, int row, bool on, const Team& g) {
  if (!on) return;
  constexpr int RUN = VE / N;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (j * RUN < skip) continue;
    S* to = sums + (at / RUN + j) * g.pitch;
    to[row] = v[j];
    if (row == g.rows - 1 && g.pitch > g.rows) to[g.rows] = S{0, 0};
  }
}

// The positions that a row of the team counts: its first thread's.
template <typename P> __device__ __forceinline__ void put_count(int* counts, int n, const P& at, const Team& g) {
  if (!at.first || !at.on) return;
  counts[at.row] = n;
  if (at.row == g.rows - 1 && g.pitch > g.rows) counts[g.rows] = 0;
}

template <typename S> __device__ __forceinline__ S lanes_sum(S a, int lanes) {
  for (int off = lanes / 2; off; off /= 2) {
    a.x += __shfl_xor(a.x, off, 64);
    a.y += __shfl_xor(a.y, off, 64);
  }
  return a;
}

// f(o, sum of the o-th `len` entries) for o < outs, by one lane of each `lanes`; U
// loads in flight.
template <int U = 4, typename S, typename Fn>
__device__ __forceinline__ void sum_runs(const S* sums, int outs, int len, int t, int threads, int lanes, Fn f) {
  const int l = t & (lanes - 1);
  for (int o = t / lanes; o < outs; o += threads / lanes) {
    const S* from = sums + (int64_t)o * len;
    S a{0, 0};
#pragma unroll U
    for (int e = l; e < len; e += lanes) {
      a.x += from[e].x;
      a.y += from[e].y;
    }
    a = lanes_sum(a, lanes);
    if (l == 0) f(o, a);
  }
}

// How many positions n entries count, and the first entry that counts any (0 without).
struct Counted {
  int64_t positions;
  int first;
  // the same in each lane
  static __device__ __forceinline__ Counted of(const int* counts, int n, int t, int lanes) {
    Counted a{0, n};
    for (int e = t & (lanes - 1); e < n; e += lanes) {
      const int here = counts[e];
      a.positions += here;
      if (here && e < a.first) a.first = e;
    }
    for (int off = lanes / 2; off; off /= 2) {
      a.positions += __shfl_xor(a.positions, off, 64);
      a.first = min(a.first, __shfl_xor(a.first, off, 64));
    }
    if (a.first == n) a.first = 0;
    return a;
  }
};

// f(o, the o-th `len` entries joined) for o < outs, as sum_runs, around the mean of entry
// `first`, which has values (if any has).  of(e): the number of them in entry e.
template <int U = 4, typename Of, typename Fn>
__device__ __forceinline__ void join_runs(const Moments* entries, int outs, int len, int first, double inv, int t,
                                          int threads, int lanes, Of of, Fn f) {
  const int l = t & (lanes - 1);
  for (int o = t / lanes; o < outs; o += threads / lanes) {
    const Moments* from = entries + (int64_t)o * len;
    const double x0 = from[first].x;
    double2 a{0, 0};
#pragma unroll U
    for (int e = l; e < len; e += lanes) {
      const Moments m = from[e];
      const double d = m.x - x0, nd = of(e) * d;
      a.x += nd;
      a.y += fma(nd, d, m.y);
    }
    a = lanes_sum(a, lanes);
    if (l == 0) f(o, around(x0, a.x, a.y, inv));
  }
}

template <typename F> __device__ __forceinline__ void load_params(float* f, const ParamVec& p, int c, float none) {
  if (p.p) {
    load_run<F::VE>(f, p, c);
  } else {
#pragma unroll
    for (int e = 0; e < F::VE; ++e) f[e] = none;
  }
}

// A thread's values, slot by slot, around the first one of each.
template <typename F> struct Running {
  float x0[F::SL];
  double2 sum[F::SL];
  int n;  // vectors
  __device__ __forceinline__ Running() : n(0) {
#pragma unroll
    for (int j = 0; j < F::SL; ++j) {
      x0[j] = 0.f;
      sum[j] = double2{0, 0};
    }
  }
  __device__ __forceinline__ void add(const float* f) {
#pragma unroll
    for (int j = 0; j < F::SL; ++j) x0[j] = n ? x0[j] : f[j * F::CPS];
#pragma unroll
    for (int e = 0; e < F::VE; ++e) {
      double2& s = sum[e / F::CPS];
      const double v = (double)f[e] - (double)x0[e / F::CPS];
      s.x += v;
      s.y = fma(v, v, s.y);
    }
    ++n;
  }
  __device__ __forceinline__ void close(Moments (&m)[F::SL]) const {
    const double inv = n ? 1.0 / ((double)n * F::CPS) : 0.0;
#pragma unroll
    for (int j = 0; j < F::SL; ++j) m[j] = around(x0[j], sum[j].x, sum[j].y, inv);
  }
};

// What a thread needs of its groups and channels.  With d = x - mean, exact where x
// is near the mean: z = d (r w) + (b - low r w), and in the backward pass h = d r -
// low r, z = h w + b.
template <typename F> struct Params {
  float w[F::VE], b[F::VE];
  Params() = default;
  __device__ __forceinline__ Params(const ParamVec& wp, const ParamVec& bp, int c) { load(wp, bp, c); }
  __device__ __forceinline__ void load(const ParamVec& wp, const ParamVec& bp, int c) {
    load_params<F>(w, wp, c, 1.f);
    load_params<F>(b, bp, c, 0.f);
  }
};
template <typename F> struct ForwardCoefs {
  float mean[F::SL], a[F::VE], b[F::VE];
  __device__ __forceinline__ void set(const GroupStats* stats, const Params<F>& p, int at, int cg) {
#pragma unroll
    for (int j = 0; j < F::SL; ++j) {
      const GroupStats g = stats[(at + j * F::CPS) / cg];
      mean[j] = g.mean;
#pragma unroll
      for (int e = j * F::CPS; e < (j + 1) * F::CPS; ++e) {
        a[e] = g.rstd * p.w[e];
        b[e] = fmaf(-g.low, a[e], p.b[e]);
      }
    }
  }
  template <int ACT> __device__ __forceinline__ void apply(float* f) const {
#pragma unroll
    for (int e = 0; e < F::VE; ++e) f[e] = activate<ACT>(fmaf(f[e] - mean[e / F::CPS], a[e], b[e]));
  }
};
template <typename F, int ACT> struct BackwardCoefs {
  float mean[F::SL], rstd[F::SL], shift[F::SL], w[F::VE], a[F::VE], b[F::VE];
  __device__ __forceinline__ void set(const GroupStats* stats, const Params<F>& p, int at, int cg) {
#pragma unroll
    for (int j = 0; j < F::SL; ++j) {
      const GroupStats g = stats[(at + j * F::CPS) / cg];
      mean[j] = g.mean;
      rstd[j] = g.rstd;
      shift[j] = -g.low * g.rstd;
    }
#pragma unroll
    for (int e = 0; e < F::VE; ++e) {
      w[e] = p.w[e];
      a[e] = p.w[e] * Slope<ACT>::kScale;
      b[e] = p.b[e] * Slope<ACT>::kScale;
    }
  }
  // f = h, g = dL/dz
  __device__ __forceinline__ void apply(float* f, float* g) const {
#pragma unroll
    for (int e = 0; e < F::VE; ++e) {
      const int j = e / F::CPS;
      f[e] = fmaf(f[e] - mean[j], rstd[j], shift[j]);
      g[e] *= activate_slope<ACT>(fmaf(f[e], a[e], b[e]));
    }
  }
  // f = dL/dx of h = f and dz = g; means: of g w and g w h over the group
  __device__ __forceinline__ void finish(float* f, const float* g, const float2 (&means)[F::SL]) const {
#pragma unroll
    for (int e = 0; e < F::VE; ++e) {
      const int j = e / F::CPS;
      f[e] = fmaf(-f[e], means[j].y, fmaf(g[e], w[e], -means[j].x)) * rstd[j];
    }
  }
};

struct Inputs {
  const void* x;
  int64_t xs;
  const float* mask;
  ParamVec w, b;
};

// ---------------------------------------------------------------------------
// Resident: a team a slice of `groups` whole groups of one sample.
// ---------------------------------------------------------------------------
struct ResidentPlan {
  Team team;
  int held;    // vectors a thread
  int groups;  // a slice
  int slices;
  size_t lds;  // of a team
  // backward: blocks of a slice (each team takes several samples), and the block's
  // partial sums of a channel in LDS
  int teams, blocks, pitch, lanes;
};

constexpr int kThreads = 512;  // of a block, at most: 256 registers a thread

template <typename F, int NV, int ACT>
__global__ __launch_bounds__(kThreads) void gn_resident_forward_kernel(Inputs in, typename F::T* __restrict__ y,
                                                                       GroupStats* __restrict__ stats, Shape s,
                                                                       ResidentPlan p, float eps) {
  typedef typename F::T T;
  extern __shared__ double2 gn_lds[];
  const Team& g = p.team;
  const int t = threadIdx.x % g.threads, team = threadIdx.x / g.threads, teams = p.teams;
  const int width = p.groups * s.cg;
  const Place<F> at(t, g, width);
  char* lds = (char*)gn_lds + team * p.lds;
  Moments* sums = (Moments*)lds;
  GroupStats* mine = (GroupStats*)(sums + (int64_t)width / F::CPS * g.pitch);
  int* row_counts = (int*)(mine + p.groups);
  const int64_t units = s.B * p.slices, steps = (units + teams - 1) / teams;
  for (int64_t step = blockIdx.x; step < steps; step += gridDim.x) {
    // slices of a sample share lines of memory: on one die
    const int64_t unit = xcd_remap_any(step, steps) * teams + team;
    const bool any = unit < units;
    const int64_t u = any ? unit : units - 1, b = u / p.slices;
    const int slice = (int)(u - b * p.slices), c = slice * width + at.at;
    const int P = (int)s.P;
    Vec<T, F::VE> x[NV];
    bool live[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {  // past the last position that one again
      const int pos = at.row + k * g.rows;
      const int64_t row = b * P + (pos < P ? pos : P - 1);
      x[k].load((const T*)in.x + row * in.xs + c);
      live[k] = at.on && pos < P && (!in.mask || in.mask[row] != 0.f);
    }
    constexpr bool LATE = F::SL > 4 && NV > 8;  // 256 registers do not hold them beside the sums
    Params<F> params;
    if (!LATE) params.load(in.w, in.b, c);
    Running<F> sum;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float f[F::VE];
      x[k].get(f);
      if (live[k]) sum.add(f);
    }
    Moments own[F::SL];
    sum.close(own);
    put_sums<F::SL, F::VE>(sums, own, at.at, at.skip, at.row, at.on, g);
    put_count(row_counts, sum.n, at, g);
    __syncthreads();
    Counted counted{P, 0};
    if (in.mask) counted = Counted::of(row_counts, g.rows, t, g.lanes);
    const double inv = in.mask ? s.inverse(counted.positions) : s.inv;
    join_runs(sums, p.groups, s.cg / F::CPS * g.pitch, counted.first, inv, t, g.threads, g.lanes,
              [&](int e) { return (double)row_counts[(unsigned)e % (unsigned)g.pitch] * F::CPS; },
              [&](int o, const Moments& m) {
                mine[o] = close_stats(m, inv, eps);
                if (any) stats[b * s.G + slice * p.groups + o] = mine[o];
              });
    __syncthreads();
    if (LATE) params.load(in.w, in.b, c);
    ForwardCoefs<F> co;
    co.set(mine, params, at.at, s.cg);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int pos = at.row + k * g.rows;
      float f[F::VE] = {};
      x[k].forget_unpacked();
      if (live[k]) {
        x[k].get(f);
        co.template apply<ACT>(f);
      }
      x[k].set(f);
      if (any && at.on && pos < P) x[k].store(y + (b * P + pos) * s.C + c);
    }
  }
}

// dx, and the block's sums of dz h and dz over its samples, part[block of the
// slice][0 and 1][c].
template <typename F, int NV, int ACT>
__global__ __launch_bounds__(kThreads) void gn_resident_backward_kernel(
    Inputs in, const typename F::T* __restrict__ dy, int64_t ds, const GroupStats* __restrict__ stats,
    typename F::T* __restrict__ dx, float* __restrict__ part, Shape s, ResidentPlan p) {
  typedef typename F::T T;
  extern __shared__ double2 gn_lds[];
  const Team& g = p.team;
  const int t = threadIdx.x % g.threads, team = threadIdx.x / g.threads;
  const int width = p.groups * s.cg;
  const Place<F> at(t, g, width);
  float2* means = (float2*)((char*)gn_lds + team * p.lds);
  float2* sums = means + p.groups;
  // slices of a sample share lines of memory: on one die
  const int id = (int)xcd_remap_any(blockIdx.x, gridDim.x), index = id / p.slices;
  const int slice = id - index * p.slices, c = slice * width + at.at;
  float2 channel[F::VE];
#pragma unroll
  for (int e = 0; e < F::VE; ++e) channel[e] = float2{0.f, 0.f};
  for (int64_t b0 = (int64_t)index * p.teams; b0 < s.B; b0 += (int64_t)p.blocks * p.teams) {
    const bool any = b0 + team < s.B;
    const int64_t b = any ? b0 + team : s.B - 1;
    const int P = (int)s.P;
    Vec<T, F::VE> x[NV], d[NV];
    bool live[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {  // past the last position that one again
      const int pos = at.row + k * g.rows;
      const int64_t row = b * P + (pos < P ? pos : P - 1);
      x[k].load((const T*)in.x + row * in.xs + c);
      d[k].load(dy + row * ds + c);
      live[k] = any && at.on && pos < P && (!in.mask || in.mask[row] != 0.f);
    }
    const GroupStats* of = stats + b * s.G + slice * p.groups;
    BackwardCoefs<F, ACT> co;
    co.set(of, Params<F>(in.w, in.b, c), at.at, s.cg);
    float2 sum[F::SL];
#pragma unroll
    for (int j = 0; j < F::SL; ++j) sum[j] = float2{0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (!live[k]) continue;
      float f[F::VE], dz[F::VE];
      x[k].get(f);
      d[k].get(dz);
      co.apply(f, dz);
#pragma unroll
      for (int e = 0; e < F::VE; ++e) {
        const float gw = dz[e] * co.w[e];
        sum[e / F::CPS].x += gw;
        sum[e / F::CPS].y = fmaf(gw, f[e], sum[e / F::CPS].y);
        channel[e].x = fmaf(dz[e], f[e], channel[e].x);
        channel[e].y += dz[e];
      }
    }
    if (!dx) continue;
    put_sums<F::SL, F::VE>(sums, sum, at.at, at.skip, at.row, at.on, g);
    __syncthreads();
    sum_runs(sums, p.groups, s.cg / F::CPS * g.pitch, t, g.threads, g.lanes, [&](int o, float2 a) {
      const float inv = of[o].inv;
      means[o] = float2{a.x * inv, a.y * inv};
    });
    __syncthreads();
    float2 mean[F::SL];
#pragma unroll
    for (int j = 0; j < F::SL; ++j) mean[j] = means[(at.at + j * F::CPS) / s.cg];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int pos = at.row + k * g.rows;
      float f[F::VE] = {};
      x[k].forget_unpacked();
      d[k].forget_unpacked();
      if (live[k]) {
        float dz[F::VE];
        x[k].get(f);
        d[k].get(dz);
        co.apply(f, dz);
        co.finish(f, dz, mean);
      }
      x[k].set(f);
      if (any && at.on && pos < P) x[k].store(dx + (b * P + pos) * s.C + c);
    }
  }
  if (!part) return;
  // the rows of all teams
  float2* channels = (float2*)gn_lds;
  const Team block{0, 0, g.rows * p.teams, p.pitch, 0, 0};
  __syncthreads();
  put_sums<F::VE, F::VE>(channels, channel, at.at, at.skip, team * g.rows + at.row, at.on, block);
  __syncthreads();
  float* dst = part + (int64_t)index * 2 * s.C + slice * width;
  sum_runs(channels, width, p.pitch, threadIdx.x, blockDim.x, p.lanes, [&](int o, float2 a) {
    dst[o] = a.x;
    dst[s.C + o] = a.y;
  });
}

// ---------------------------------------------------------------------------
// Streamed: a team is a block, and has a chunk of a sample's positions (`steps` times
// the team's rows) in a slice of `groups` whole groups: all of them, unless they are
// more than 512 vectors wide.
// ---------------------------------------------------------------------------
struct StreamPlan {
  Team team;
  int groups, slices;
  int chunks, parts;          // of this launch; of the one that summed
  int64_t steps, all, whole;  // of a chunk; of a sample; those of them that have all their rows
};

// A block's chunk: steps [first, last) of sample b, of which those before `whole` have
// all their rows, in the slice that starts at group g0.
struct Chunk {
  int64_t index, b, first, last, whole;  // index: of (sample, chunk)
  int chunk, g0;
  __device__ __forceinline__ Chunk(int64_t item, const StreamPlan& p) {
    index = p.slices == 1 ? item : item / p.slices;
    g0 = (int)(item - index * p.slices) * p.groups;
    b = index / p.chunks;
    chunk = (int)(index - b * p.chunks);
    first = chunk * p.steps;
    last = first + p.steps < p.all ? first + p.steps : p.all;
    whole = last < p.whole ? last : p.whole;
  }
};

// A thread's vectors of one tensor or two, and whether their positions count.
template <typename F, int U, bool TWO> struct Held {
  Vec<typename F::T, F::VE> x[U], d[TWO ? U : 1];
  bool live[U];
};

// A thread's place in the tensors, at a step of its chunk's sample.  KEEP: a second
// launch reads the values again.
template <typename F, bool TWO, bool KEEP, bool MASKED> struct Cursor {
  typedef typename F::T T;
  const T *x, *d;
  const float* mask;
  int64_t x_step, d_step;
  int rows, row;
  int64_t left;  // positions behind the sample's first one
  __device__ __forceinline__ Cursor(const Inputs& in, const T* dy, int64_t ds, const Shape& s, const Team& g, int64_t b,
                                    int c, const Place<F>& at)
      : x_step(g.rows * in.xs), d_step(g.rows * ds), rows(g.rows), row(at.row), left(s.P) {
    x = (const T*)in.x + (b * s.P + at.row) * in.xs + c;
    d = TWO ? dy + (b * s.P + at.row) * ds + c : nullptr;
    mask = MASKED ? in.mask + b * s.P + at.row : nullptr;
  }
  template <int U> __device__ __forceinline__ void load_live(Held<F, U, TWO>& v, int64_t step) const {
#pragma unroll
    for (int j = 0; j < U; ++j) v.live[j] = !MASKED || mask[(step + j) * rows] != 0.f;
  }
  // what does not count is not read
  template <int U> __device__ __forceinline__ void load(Held<F, U, TWO>& v, int64_t step) const {
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (v.live[j]) get(v, j, step + j);
  }
  // One step, which not all threads may have a position in.
  __device__ __forceinline__ void load_one(Held<F, 1, TWO>& v, int64_t step) const {
    v.live[0] = inside(step) && (!MASKED || mask[step * rows] != 0.f);
    if (v.live[0]) get(v, 0, step);
  }
  __device__ __forceinline__ bool inside(int64_t step) const { return step * rows + row < left; }

 private:
  template <int U> __device__ __forceinline__ void get(Held<F, U, TWO>& v, int j, int64_t step) const {
    if constexpr (KEEP) {
      v.x[j].load_plain(x + step * x_step);
      if constexpr (TWO) v.d[j].load_plain(d + step * d_step);
    } else {
      v.x[j].load(x + step * x_step);
      if constexpr (TWO) v.d[j].load(d + step * d_step);
    }
  }
};

// Calls use(held, j, step) for the chunk's steps, forwards or backwards, U whole ones at
// a time while the next U are on their way, and the mask of those behind them;
// start() runs behind the first loads.
template <int U, bool BACK, typename F, bool TWO, bool KEEP, bool MASKED, typename Start, typename Use>
__device__ __forceinline__ void for_steps(const Cursor<F, TWO, KEEP, MASKED>& at, const Chunk& k, Start start,
                                          Use use) {
  const int64_t whole = k.whole > k.first ? k.whole - k.first : 0, sets = whole / U;
  Held<F, U, TWO> now, next;
  auto step_of = [&](int64_t i) { return k.first + (BACK ? sets - 1 - i : i) * U; };
  if (sets) {
    at.load_live(now, step_of(0));
    if (sets > 1) at.load_live(next, step_of(1));
    at.load(now, step_of(0));
  }
  start();
  auto rest = [&]() {
    for (int64_t step = k.first + sets * U; step < k.last; ++step) {
      Held<F, 1, TWO> one;
      at.load_one(one, step);
      use(one, 0, step);
    }
  };
  if (BACK) rest();
  for (int64_t i = 0; i < sets; ++i) {
    Held<F, U, TWO> ahead;
    if (i + 1 < sets) at.load(next, step_of(i + 1));
    if (i + 2 < sets) at.load_live(ahead, step_of(i + 2));
#pragma unroll
    for (int j = 0; j < U; ++j) use(now, j, step_of(i) + j);
    now = next;
#pragma unroll
    for (int j = 0; j < U; ++j) next.live[j] = ahead.live[j];
  }
  if (!BACK) rest();
}

// part[b][group][chunk], counts[b][chunk]
template <typename F, bool MASKED>
__global__ __launch_bounds__(kThreads) void gn_stats_kernel(Inputs in, Moments* __restrict__ part,
                                                            int* __restrict__ chunk_counts, Shape s, StreamPlan p) {
  extern __shared__ double2 gn_lds[];
  __shared__ int row_counts[kThreads + 1];
  const Team& g = p.team;
  const int t = threadIdx.x;
  const int width = p.groups * s.cg;
  const Place<F> at(t, g, width);
  for (int64_t item = blockIdx.x; item < s.B * p.chunks * p.slices; item += gridDim.x) {
    const Chunk k(item, p);
    const int c = k.g0 * s.cg + at.at;
    Running<F> sum;
    const Cursor<F, false, true, MASKED> from(in, nullptr, 0, s, g, k.b, c, at);
    for_steps<4, false>(from, k, [] {}, [&](auto& v, int j, int64_t) {
      if (!v.live[j]) return;
      float f[F::VE];
      v.x[j].get(f);
      sum.add(f);
    });
    Moments own[F::SL];
    sum.close(own);
    put_sums<F::SL, F::VE>(gn_lds, own, at.at, at.skip, at.row, at.on, g);
    put_count(row_counts, sum.n, at, g);
    __syncthreads();
    const Counted counted = Counted::of(row_counts, g.rows, t, g.lanes);
    join_runs(gn_lds, p.groups, s.cg / F::CPS * g.pitch, counted.first, s.inverse(counted.positions), t, kThreads,
              g.lanes, [&](int e) { return (double)row_counts[(unsigned)e % (unsigned)g.pitch] * F::CPS; },
              [&](int o, const Moments& m) { part[(k.b * s.G + k.g0 + o) * p.chunks + k.chunk] = m; });
    if (t == 0 && k.g0 == 0) chunk_counts[k.index] = (int)counted.positions;
    __syncthreads();
  }
}

template <typename F, int ACT, bool MASKED>
__global__ __launch_bounds__(kThreads) void gn_apply_kernel(Inputs in, const Moments* __restrict__ part,
                                                            const int* __restrict__ chunk_counts,
                                                            typename F::T* __restrict__ y,
                                                            GroupStats* __restrict__ stats, Shape s, StreamPlan p,
                                                            float eps) {
  typedef typename F::T T;
  extern __shared__ double2 gn_lds[];
  GroupStats* mine = (GroupStats*)gn_lds;
  const Team& g = p.team;
  const int t = threadIdx.x;
  const int width = p.groups * s.cg;
  const Place<F> at(t, g, width);
  for (int64_t item = blockIdx.x; item < s.B * p.chunks * p.slices; item += gridDim.x) {
    const Chunk k(item, p);
    const int c = k.g0 * s.cg + at.at;
    const Cursor<F, false, false, MASKED> from(in, nullptr, 0, s, g, k.b, c, at);
    T* to = y + (k.b * s.P + at.row) * s.C + c;
    const int64_t y_step = (int64_t)g.rows * s.C;
    ForwardCoefs<F> co;
    auto start = [&]() {
      const Params<F> params(in.w, in.b, c);
      const int* counts = chunk_counts + k.b * p.parts;
      Counted counted{s.P, 0};
      if (MASKED) counted = Counted::of(counts, p.parts, t, g.lanes);
      const double inv = MASKED ? s.inverse(counted.positions) : s.inv;
      join_runs<8>(part + (k.b * s.G + k.g0) * p.parts, p.groups, p.parts, counted.first, inv, t, kThreads, g.lanes,
                   [&](int e) { return (double)counts[e] * s.cg; },
                   [&](int o, const Moments& m) {
                     mine[o] = close_stats(m, inv, eps);
                     if (k.chunk == 0) stats[k.b * s.G + k.g0 + o] = mine[o];
                   });
      __syncthreads();
      co.set(mine, params, at.at, s.cg);
    };
    for_steps<4, true>(from, k, start, [&](auto& v, int j, int64_t step) {
      Vec<T, F::VE> o;
      o.zero();
      if (v.live[j]) {
        float f[F::VE];
        v.x[j].get(f);
        co.template apply<ACT>(f);
        o.set(f);
      }
      if (at.on && from.inside(step)) o.store(to + step * y_step);
    });
    __syncthreads();
  }
}

// The chunk's sums of dz h and dz, channels[b][chunk][0 and 1][c], and of g and g h,
// part[b][group][chunk].
template <typename F, int ACT, bool MASKED>
__global__ __launch_bounds__(kThreads) void gn_backward_sums_kernel(Inputs in, const typename F::T* __restrict__ dy,
                                                                    int64_t ds, const GroupStats* __restrict__ stats,
                                                                    float2* __restrict__ part,
                                                                    float* __restrict__ channels, Shape s,
                                                                    StreamPlan p) {
  extern __shared__ double2 gn_lds[];
  float2* weighted = (float2*)gn_lds;  // [width]: a channel's part of its group's sums
  const int width = p.groups * s.cg;
  float2* sums = weighted + width;
  float* weight = (float*)(sums + (int64_t)width * p.team.pitch);
  const Team& g = p.team;
  const int t = threadIdx.x;
  const Place<F> at(t, g, width);
  for (int64_t item = blockIdx.x; item < s.B * p.chunks * p.slices; item += gridDim.x) {
    const Chunk k(item, p);
    const int c = k.g0 * s.cg + at.at;
    BackwardCoefs<F, ACT> co;
    float2 sum[F::VE];
#pragma unroll
    for (int e = 0; e < F::VE; ++e) sum[e] = float2{0.f, 0.f};
    auto start = [&]() {
      const Params<F> params(in.w, in.b, c);
      co.set(stats + k.b * s.G + k.g0, params, at.at, s.cg);
#pragma unroll
      for (int e = 0; e < F::VE; ++e)
        if (at.row == 0) weight[at.at + e] = params.w[e];
    };
    const Cursor<F, true, true, MASKED> from(in, dy, ds, s, g, k.b, c, at);
    for_steps<2, false>(from, k, start, [&](auto& v, int j, int64_t) {
      if (!v.live[j]) return;
      float f[F::VE], dz[F::VE];
      v.x[j].get(f);
      v.d[j].get(dz);
      co.apply(f, dz);
#pragma unroll
      for (int e = 0; e < F::VE; ++e) {
        sum[e].x = fmaf(dz[e], f[e], sum[e].x);
        sum[e].y += dz[e];
      }
    });
    put_sums<F::VE, F::VE>(sums, sum, at.at, at.skip, at.row, at.on, g);
    __syncthreads();
    float* to = channels ? channels + k.index * 2 * s.C + k.g0 * s.cg : nullptr;
    sum_runs(sums, width, g.pitch, t, kThreads, g.channel_lanes, [&](int o, float2 a) {
      if (to) {
        to[o] = a.x;
        to[s.C + o] = a.y;
      }
      const float w = weight[o];
      weighted[o] = float2{a.y * w, a.x * w};
    });
    __syncthreads();
    if (part)
      sum_runs(weighted, p.groups, s.cg, t, kThreads, g.lanes,
               [&](int o, float2 a) { part[(k.b * s.G + k.g0 + o) * p.chunks + k.chunk] = a; });
    __syncthreads();
  }
}

template <typename F, int ACT, bool MASKED>
__global__ __launch_bounds__(kThreads) void gn_backward_apply_kernel(
    Inputs in, const typename F::T* __restrict__ dy, int64_t ds, const GroupStats* __restrict__ stats,
    const float2* __restrict__ part, typename F::T* __restrict__ dx, ColumnSums close, int blocks, Shape s,
    StreamPlan p) {
  typedef typename F::T T;
  extern __shared__ double2 gn_lds[];
  if ((int)blockIdx.x >= blocks) {  // the parameters' gradients
    close_columns<16, kThreads / 16>(close, (int)blockIdx.x - blocks, (float*)gn_lds);
    return;
  }
  float2* means = (float2*)gn_lds;
  const Team& g = p.team;
  const int t = threadIdx.x;
  const int width = p.groups * s.cg;
  const Place<F> at(t, g, width);
  for (int64_t item = blockIdx.x; item < s.B * p.chunks * p.slices; item += blocks) {
    const Chunk k(item, p);
    const int c = k.g0 * s.cg + at.at;
    const Cursor<F, true, false, MASKED> from(in, dy, ds, s, g, k.b, c, at);
    T* to = dx + (k.b * s.P + at.row) * s.C + c;
    const int64_t dx_step = (int64_t)g.rows * s.C;
    BackwardCoefs<F, ACT> co;
    float2 mean[F::SL];
    auto start = [&]() {
      const GroupStats* of = stats + k.b * s.G + k.g0;
      co.set(of, Params<F>(in.w, in.b, c), at.at, s.cg);
      const float2* sums = part + (k.b * s.G + k.g0) * p.parts;
      sum_runs<8>(sums, p.groups, p.parts, t, kThreads, g.lanes, [&](int o, float2 a) {
        const float inv = of[o].inv;
        means[o] = float2{a.x * inv, a.y * inv};
      });
      __syncthreads();
#pragma unroll
      for (int j = 0; j < F::SL; ++j) mean[j] = means[(at.at + j * F::CPS) / s.cg];
    };
    for_steps<2, true>(from, k, start, [&](auto& v, int j, int64_t step) {
      Vec<T, F::VE> o;
      o.zero();
      if (v.live[j]) {
        float f[F::VE], dz[F::VE];
        v.x[j].get(f);
        v.d[j].get(dz);
        co.apply(f, dz);
        co.finish(f, dz, mean);
        o.set(f);
      }
      if (at.on && from.inside(step)) o.store(to + step * dx_step);
    });
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Swept: groups that are wider than a block's threads span.  A block a sample's group,
// and for the parameters a block a channel.
// ---------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void block_add(T (&v)[3], T (*red)[4]) {
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    for (int off = 32; off; off >>= 1) v[k] += __shfl_xor(v[k], off, 64);
    if ((threadIdx.x & 63) == 0) red[k][threadIdx.x >> 6] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) v[k] = red[k][0] + red[k][1] + red[k][2] + red[k][3];
}

// Calls f(position, channel) for this thread's values of a group that starts at
// channel c0.
template <typename Fn> __device__ __forceinline__ void for_values(const Shape& s, int c0, Fn f) {
  for (int64_t pos = 0; pos < s.P; ++pos)
    for (int k = threadIdx.x; k < s.cg; k += 256) f(pos, c0 + k);
}

template <typename T, int ACT>
__global__ __launch_bounds__(256) void gn_swept_forward_kernel(Inputs in, T* __restrict__ y,
                                                               GroupStats* __restrict__ stats, Shape s, float eps) {
  __shared__ double red[3][4];
  const T* x = (const T*)in.x;
  for (int64_t bg = blockIdx.x; bg < s.B * s.G; bg += gridDim.x) {
    const int64_t first = bg / s.G * s.P;
    const int c0 = (int)(bg % s.G) * s.cg;
    double v[3] = {0, 0, 0};
    float x0 = 0.f;  // the first channel's value at the first position that counts
    for_values(s, c0, [&](int64_t pos, int c) {
      if (in.mask && in.mask[first + pos] == 0.f) return;
      const T* row = x + (first + pos) * in.xs;
      if (v[2] == 0) x0 = to_f32(row[c0]);
      const double d = (double)to_f32(row[c]) - (double)x0;
      v[0] += d;
      v[1] = fma(d, d, v[1]);
      v[2] += 1;
    });
    block_add(v, red);
    const double inv = v[2] > 0 ? 1.0 / v[2] : 0.0;
    // threads without a channel have no x0, nor a use for it
    const GroupStats g = close_stats(around(x0, v[0], v[1], inv), inv, eps);
    if (threadIdx.x == 0) stats[bg] = g;
    for_values(s, c0, [&](int64_t pos, int c) {
      const bool live = !in.mask || in.mask[first + pos] != 0.f;
      const float h = ((to_f32(x[(first + pos) * in.xs + c]) - g.mean) - g.low) * g.rstd;
      const float z = fmaf(h, in.w.get(c, 1.f), in.b.get(c, 0.f));
      y[(first + pos) * s.C + c] = cvt<T>(live ? activate<ACT>(z) : 0.f);
    });
  }
}

// h and dz of a value; false where it does not count.
template <int ACT, typename T>
__device__ __forceinline__ bool swept_backward(const Inputs& in, const T* dy, int64_t ds, const GroupStats& g,
                                               int64_t row, int c, float& h, float& dz) {
  h = dz = 0.f;
  if (in.mask && in.mask[row] == 0.f) return false;
  h = ((to_f32(((const T*)in.x)[row * in.xs + c]) - g.mean) - g.low) * g.rstd;
  const float z = fmaf(h, in.w.get(c, 1.f), in.b.get(c, 0.f));
  dz = to_f32(dy[row * ds + c]) * activate_slope<ACT>(Slope<ACT>::kScale * z);
  return true;
}

template <typename T, int ACT>
__global__ __launch_bounds__(256) void gn_swept_backward_kernel(Inputs in, const T* __restrict__ dy, int64_t ds,
                                                                const GroupStats* __restrict__ stats,
                                                                T* __restrict__ dx, Shape s) {
  __shared__ double red[3][4];
  for (int64_t bg = blockIdx.x; bg < s.B * s.G; bg += gridDim.x) {
    const int64_t first = bg / s.G * s.P;
    const int c0 = (int)(bg % s.G) * s.cg;
    const GroupStats g = stats[bg];
    float h, dz;
    double v[3] = {0, 0, 0};
    for_values(s, c0, [&](int64_t pos, int c) {
      swept_backward<ACT>(in, dy, ds, g, first + pos, c, h, dz);
      const float gw = dz * in.w.get(c, 1.f);
      v[0] += gw;
      v[1] += (double)gw * h;
    });
    block_add(v, red);
    const float c1 = (float)(v[0] * g.inv), c2 = (float)(v[1] * g.inv);
    for_values(s, c0, [&](int64_t pos, int c) {
      const bool live = swept_backward<ACT>(in, dy, ds, g, first + pos, c, h, dz);
      dx[(first + pos) * s.C + c] = cvt<T>(live ? (dz * in.w.get(c, 1.f) - c1 - h * c2) * g.rstd : 0.f);
    });
  }
}

template <typename T, int ACT>
__global__ __launch_bounds__(256) void gn_swept_params_kernel(Inputs in, const T* __restrict__ dy, int64_t ds,
                                                              const GroupStats* __restrict__ stats,
                                                              void* __restrict__ dw, void* __restrict__ db, int dst_bf,
                                                              Shape s) {
  __shared__ double red[3][4];
  for (int c = blockIdx.x; c < s.C; c += gridDim.x) {
    double v[3] = {0, 0, 0};
    for (int64_t row = threadIdx.x; row < s.B * s.P; row += 256) {
      float h, dz;
      swept_backward<ACT>(in, dy, ds, stats[row / s.P * s.G + c / s.cg], row, c, h, dz);
      v[0] += (double)dz * h;
      v[1] += dz;
    }
    block_add(v, red);
    if (threadIdx.x) continue;
    for (int k = 0; k < 2; ++k) {
      void* dst = k ? db : dw;
      if (!dst) continue;
      if (dst_bf)
        ((bf16*)dst)[c] = (bf16)(float)v[k];
      else
        ((float*)dst)[c] = (float)v[k];
    }
  }
}

// ---------------------------------------------------------------------------
// Plans
// ---------------------------------------------------------------------------
constexpr size_t kMostLds = 156 * 1024;
constexpr int kMostBlocks = 1 << 20;  // the kernels loop past that

static int pow2_up(int64_t v) {
  int p = 1;
  while (p < v) p *= 2;
  return p;
}
// A power of two of lanes for each of `outs` sums.
static int lanes_for(int threads, int64_t outs) {
  int l = 64;
  while (l > 1 && (l > threads || l * outs > threads)) l /= 2;
  return l;
}
static Team make_team(int threads, int across, int64_t groups, int64_t channels) {
  Team t;
  t.threads = threads;
  t.across = across;
  t.rows = threads / across;
  // an odd pitch, or neighbouring slots' sums would lie in the same banks
  t.pitch = t.rows >= 8 ? t.rows | 1 : t.rows;
  t.lanes = lanes_for(threads, groups);
  t.channel_lanes = lanes_for(threads, channels);
  return t;
}

// Vectors a thread holds at most: what 256 registers take.
template <typename F> constexpr int most_held(bool backward) { return !backward ? 16 : F::SL > 2 ? 4 : 8; }

static size_t block_lds(const ResidentPlan& p, int64_t width, bool backward) {
  const size_t sums = p.lds * p.teams;
  return backward ? std::max(sums, (size_t)width * p.pitch * sizeof(float2)) : sums;
}

// Slices whose rows fill 64-byte pieces of memory (8 samples of 4096 positions and 256
// bf16 channels forward in 16-byte pieces: 33 us, streamed 17), wider ones as long as
// they leave four teams a CU.
template <typename F> static bool plan_resident(const Shape& s, bool backward, ResidentPlan* plan) {
  const int most = most_held<F>(backward), cus = device_cus();
  if (s.P > (int64_t)kThreads * most) return false;
  bool found = false;
  // the most groups that a block's threads span
  const int64_t span = std::min<int64_t>(s.G, (int64_t)kThreads * F::VE / s.cg);
  for (int groups = 1; groups <= span; ++groups) {
    const int64_t width = (int64_t)groups * s.cg;
    if (s.G % groups || width < F::VE || (groups < s.G && width * (int64_t)sizeof(typename F::T) < 64)) continue;
    const int64_t across = (width + F::VE - 1) / F::VE, units = s.B * (s.G / groups);
    if (found && units < 4 * (int64_t)cus) break;
    int threads = pow2_up(across);
    auto held = [&](int n) { return (s.P + n / across - 1) / (n / across); };
    while (threads < kThreads && held(threads) > most) threads *= 2;
    if (held(threads) > most) break;
    // A CU takes some 0.15 ns a value (backward 0.4): few teams of many values are slower
    // than two launches over all CUs.  128 bf16 channels in four teams, backward with the
    // closing launch: 256 positions 11.4 us, streamed 12.7; 400 positions 13.7, 12.9; 1024
    // positions 18.7, 12.8, and forward 10.2, 10.6.
    if (units < 2 * (int64_t)cus && s.P * width > (backward ? 8192 : 32768)) break;
    // more threads where there are few teams
    while (threads < kThreads && held(threads) > 1 && units * threads < 512 * (int64_t)cus) threads *= 2;
    ResidentPlan p;
    p.team = make_team(threads, (int)across, groups, width);
    p.held = (int)held(threads);
    p.groups = groups;
    p.slices = s.G / groups;
    p.lds = backward ? (groups + width / F::CPS * p.team.pitch) * sizeof(float2)
                     : width / F::CPS * p.team.pitch * sizeof(Moments) + groups * sizeof(GroupStats) +
                           p.team.pitch * sizeof(int);
    p.lds = (p.lds + 15) & ~size_t(15);
    p.teams = (backward ? kThreads : std::max(256, threads)) / threads;
    // two blocks a CU: each leaves 2 C partial sums
    p.blocks = (int)std::min<int64_t>((s.B + p.teams - 1) / p.teams, std::max(1, 2 * cus / p.slices));
    p.pitch = p.team.rows * p.teams | 1;
    p.lanes = lanes_for(kThreads, width);
    if (block_lds(p, width, backward) > kMostLds) break;
    *plan = p;
    found = true;
  }
  return found;
}

// The launch that sums has a chunk a CU, the one that applies two of them where they are
// long: each of its blocks adds its sample's partial sums up (2^20 positions of 128 bf16
// channels without an activation 85 + 123 us, with one chunk 81 + 131; 2^18 of them with
// silu 24 + 36, with two 25 + 38).
template <typename F> static bool plan_streamed(const Shape& s, bool backward, StreamPlan* p, StreamPlan* apply) {
  // the most groups that a block's threads span
  int64_t groups = std::min<int64_t>(s.G, (int64_t)kThreads * F::VE / s.cg);
  while (groups > 1 && s.G % groups) --groups;
  const int64_t width = groups * s.cg;
  if (groups < 1 || width < F::VE) return false;
  const int slices = (int)(s.G / groups);
  p->slices = slices;
  p->groups = (int)groups;
  p->team = make_team(kThreads, (int)((width + F::VE - 1) / F::VE), p->groups, width);
  p->all = (s.P + p->team.rows - 1) / p->team.rows;
  p->whole = s.P / p->team.rows;
  const int64_t cus = device_cus();
  const int64_t samples = s.B * slices;
  auto split = [&](StreamPlan* p, int64_t blocks) {
    const int64_t want = std::max<int64_t>(1, blocks / samples);
    p->steps = (p->all + want - 1) / want;
    // whole sets of the kernels' steps, the rest is read step by step: more steps, not
    // fewer, or some CUs would have a chunk more (640 x 640 positions of 128 bf16
    // channels forward, 52 steps a chunk: 60 us in two launches; 48 steps: 80)
    const int64_t set = backward ? 2 : 4;
    if (p->steps >= 12) p->steps = (p->steps + set - 1) / set * set;
    p->chunks = (int)((p->all + p->steps - 1) / p->steps);
  };
  split(p, cus);
  p->parts = p->chunks;
  *apply = *p;
  if (p->all * samples >= 64 * cus) split(apply, 2 * cus);
  return true;
}

template <typename F> struct Plan {
  bool resident, streamed;
  ResidentPlan r;
  StreamPlan t, apply;
  Plan(const Shape& s, bool backward) {
    resident = plan_resident<F>(s, backward, &r);
    streamed = !resident && plan_streamed<F>(s, backward, &t, &apply);
  }
  int64_t parts(const Shape& s) const { return resident ? r.blocks : streamed ? s.B * t.chunks : 0; }
};

// Calls run(Form) for the types and the width of a slot.
template <typename T, typename Fn> static auto for_form(const Shape& s, Fn run) {
  constexpr int VE = 16 / sizeof(T);
  if (s.C < VE) return run(Form<T, 1, 1>());
  if (s.cg % VE == 0) return run(Form<T, VE, 1>());
  if (s.cg % (VE / 2) == 0) return run(Form<T, VE, 2>());
  return run(Form<T, VE, VE>());
}
// Calls run(number) for the smallest number of held vectors that is enough.
template <int MOST, typename Fn> static void for_held(int held, Fn run) {
  if constexpr (MOST > 8)
    if (held > 8) return run(std::integral_constant<int, 16>());
  if constexpr (MOST > 4)
    if (held > 4) return run(std::integral_constant<int, 8>());
  if (held > 2) return run(std::integral_constant<int, 4>());
  if (held > 1) return run(std::integral_constant<int, 2>());
  run(std::integral_constant<int, 1>());
}

template <typename Fn> static void for_mask(const Inputs& in, Fn run) {
  if (in.mask) return run(std::true_type());
  run(std::false_type());
}

template <typename Fn> static void for_activation(int act, Fn run) {
  if (act == GTK_ACT_SILU) return run(std::integral_constant<int, GTK_ACT_SILU>());
  if (act == GTK_ACT_GELU) return run(std::integral_constant<int, GTK_ACT_GELU>());
  run(std::integral_constant<int, GTK_ACT_NONE>());
}

static unsigned blocks_for(int64_t items) { return (unsigned)std::min<int64_t>(items, kMostBlocks); }

template <typename F> struct ForwardWork {
  Moments* part;
  int* counts;
  ForwardWork(Carve& cv, const Shape& s, const Plan<F>& p) {
    part = cv.take<Moments>(p.streamed ? s.B * s.G * p.t.chunks : 0);
    counts = cv.take<int>(p.streamed ? s.B * p.t.chunks : 0);
  }
};
template <typename F> struct BackwardWork {
  float2* part;
  float* channels;
  BackwardWork(Carve& cv, const Shape& s, const Plan<F>& p) {
    part = cv.take<float2>(p.streamed ? s.B * s.G * p.t.chunks : 0);
    channels = cv.take<float>(2 * (int64_t)s.C * p.parts(s));
  }
};

template <typename F>
static int launch_gn_forward(const Inputs& in, void* yp, GroupStats* stats, const Shape& s, float eps, int act,
                             void* ws, size_t ws_bytes, hipStream_t st) {
  typedef typename F::T T;
  T* y = (T*)yp;
  const Plan<F> p(s, false);
  if (p.resident) {
    StageTimer timer("group_norm_forward", st);
    const unsigned blocks = blocks_for((s.B * p.r.slices + p.r.teams - 1) / p.r.teams);
    for_activation(act, [&](auto a) {
      for_held<most_held<F>(false)>(p.r.held, [&](auto nv) {
        gn_resident_forward_kernel<F, decltype(nv)::value, decltype(a)::value>
            <<<blocks, p.r.teams * p.r.team.threads, block_lds(p.r, p.r.groups * s.cg, false), st>>>(in, y, stats, s,
                                                                                                     p.r, eps);
      });
    });
  } else if (p.streamed) {
    Carve cv(ws, ws_bytes);
    const ForwardWork<F> work(cv, s, p);
    const unsigned blocks = blocks_for(s.B * p.t.chunks * p.t.slices);
    {
      StageTimer timer("group_norm_stats", st);
      const size_t lds = (size_t)(p.t.groups * s.cg / F::CPS) * p.t.team.pitch * sizeof(Moments);
      for_mask(in, [&](auto m) {
        gn_stats_kernel<F, decltype(m)::value><<<blocks, kThreads, lds, st>>>(in, work.part, work.counts, s, p.t);
      });
      GTK_LAUNCH_CHECK();
    }
    StageTimer timer("group_norm_apply", st);
    const unsigned behind = blocks_for(s.B * p.apply.chunks * p.apply.slices);
    for_activation(act, [&](auto a) {
      for_mask(in, [&](auto m) {
        gn_apply_kernel<F, decltype(a)::value, decltype(m)::value>
            <<<behind, kThreads, p.t.groups * sizeof(GroupStats), st>>>(in, work.part, work.counts, y, stats, s,
                                                                        p.apply, eps);
      });
    });
  } else {
    StageTimer timer("group_norm_forward", st);
    for_activation(act, [&](auto a) {
      gn_swept_forward_kernel<T, decltype(a)::value><<<blocks_for(s.B * s.G), 256, 0, st>>>(in, y, stats, s, eps);
    });
  }
  GTK_LAUNCH_CHECK();
  return GTK_OK;
}

template <typename F>
static int launch_gn_backward(const Inputs& in, const void* dyp, int64_t ds, const GroupStats* stats, void* dxp,
                              void* dw, void* db, int dst_bf, const Shape& s, int act, void* ws, size_t ws_bytes,
                              hipStream_t st) {
  typedef typename F::T T;
  const T* dy = (const T*)dyp;
  T* dx = (T*)dxp;
  const Plan<F> p(s, true);
  Carve cv(ws, ws_bytes);
  const BackwardWork<F> work(cv, s, p);
  const bool sums = dw || db;
  if (p.resident) {
    StageTimer timer("group_norm_backward", st);
    for_activation(act, [&](auto a) {
      for_held<most_held<F>(true)>(p.r.held, [&](auto nv) {
        gn_resident_backward_kernel<F, decltype(nv)::value, decltype(a)::value>
            <<<(unsigned)p.r.blocks * p.r.slices, kThreads, block_lds(p.r, p.r.groups * s.cg, true), st>>>(
                in, dy, ds, stats, dx, sums ? work.channels : nullptr, s, p.r);
      });
    });
    GTK_LAUNCH_CHECK();
  } else if (p.streamed) {
    const unsigned blocks = blocks_for(s.B * p.t.chunks * p.t.slices);
    {
      StageTimer timer("group_norm_backward_sums", st);
      const size_t lds = (size_t)p.t.groups * s.cg * ((1 + p.t.team.pitch) * sizeof(float2) + sizeof(float));
      for_activation(act, [&](auto a) {
        for_mask(in, [&](auto m) {
          gn_backward_sums_kernel<F, decltype(a)::value, decltype(m)::value><<<blocks, kThreads, lds, st>>>(
              in, dy, ds, stats, dx ? work.part : nullptr, sums ? work.channels : nullptr, s, p.t);
        });
      });
      GTK_LAUNCH_CHECK();
    }
    const ColumnSums close{work.channels, (int)p.parts(s), s.C, dw, db, dst_bf};
    const unsigned more = sums ? (2 * s.C + 15) / 16 : 0;
    if (dx) {
      StageTimer timer("group_norm_backward_apply", st);
      const unsigned behind = blocks_for(s.B * p.apply.chunks * p.apply.slices);
      const size_t lds = std::max(p.t.groups * sizeof(float2), sums ? kThreads * sizeof(float) : 0);
      for_activation(act, [&](auto a) {
        for_mask(in, [&](auto m) {
          gn_backward_apply_kernel<F, decltype(a)::value, decltype(m)::value><<<behind + more, kThreads, lds, st>>>(
              in, dy, ds, stats, work.part, dx, close, (int)behind, s, p.apply);
        });
      });
    } else {  // in the same order
      StageTimer timer("group_norm_close", st);
      column_close_kernel<16, kThreads / 16><<<more, kThreads, 0, st>>>(close);
    }
    GTK_LAUNCH_CHECK();
    return GTK_OK;
  } else {
    if (dx) {
      StageTimer timer("group_norm_backward", st);
      for_activation(act, [&](auto a) {
        gn_swept_backward_kernel<T, decltype(a)::value>
            <<<blocks_for(s.B * s.G), 256, 0, st>>>(in, dy, ds, stats, dx, s);
      });
      GTK_LAUNCH_CHECK();
    }
    if (sums) {
      StageTimer timer("group_norm_params", st);
      for_activation(act, [&](auto a) {
        gn_swept_params_kernel<T, decltype(a)::value>
            <<<blocks_for(s.C), 256, 0, st>>>(in, dy, ds, stats, dw, db, dst_bf, s);
      });
      GTK_LAUNCH_CHECK();
    }
    return GTK_OK;
  }
  if (!sums) return GTK_OK;
  return launch_column_close("group_norm_close", work.channels, (int)p.parts(s), s.C, dw, db, dst_bf, st);
}

static bool gn_shape_ok(int64_t B, int64_t P, int64_t C, int64_t G, int dtype) {
  const int64_t most = (int64_t)1 << 48;
  return B >= 0 && P >= 1 && C >= 1 && C <= 1 << 24 && G >= 1 && G <= C && C % G == 0 && P <= most / C &&
         B <= most / (P * C) && (dtype == GTK_F32 || dtype == GTK_BF16);
}

template <template <typename> class Work> static size_t work_size(const Shape& s, int dtype, bool backward) {
  auto size = [&](auto form) {
    typedef decltype(form) F;
    Carve cv(nullptr, SIZE_MAX);
    const Plan<F> p(s, backward);
    const Work<F> work(cv, s, p);
    return cv.off;
  };
  return dtype == GTK_F32 ? for_form<float>(s, size) : for_form<bf16>(s, size);
}

}  // namespace gtk

using namespace gtk;

#define GTK_GN_CHECK(name)                                                                                        \
  GTK_REQUIRE(gn_shape_ok(B, positions, c, groups, dtype), GTK_EINVAL,                                            \
              name ": bad shape [%lld][%lld][%lld] in %lld groups, dtype %d", (long long)B, (long long)positions, \
              (long long)c, (long long)groups, dtype);                                                            \
  GTK_REQUIRE(param_dtype == GTK_F32 || param_dtype == GTK_BF16, GTK_EINVAL, name ": bad parameter dtype %d",     \
              param_dtype);                                                                                       \
  GTK_REQUIRE(activation >= GTK_ACT_NONE && activation <= GTK_ACT_GELU, GTK_EINVAL, name ": bad activation %d",   \
              activation);                                                                                        \
  GTK_REQUIRE(x_stride >= 0, GTK_EINVAL, name ": negative stride")

extern "C" size_t gtk_group_norm_workspace_size(int64_t B, int64_t positions, int64_t c, int64_t groups, int dtype) {
  if (!gn_shape_ok(B, positions, c, groups, dtype) || B == 0) return 0;
  return work_size<ForwardWork>(Shape::of(B, positions, c, groups), dtype, false);
}

extern "C" int gtk_group_norm_forward(const void* x, int64_t x_stride, const float* mask, void* y, float* stats,
                                      const void* weight, const void* bias, int param_dtype, int64_t B,
                                      int64_t positions, int64_t c, int64_t groups, float eps, int activation,
                                      int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  GTK_GN_CHECK("gtk_group_norm_forward");
  if (B == 0) return GTK_OK;
  GTK_REQUIRE(x && y && stats, GTK_EINVAL, "gtk_group_norm_forward: null pointer");
  const size_t need = gtk_group_norm_workspace_size(B, positions, c, groups, dtype);
  GTK_REQUIRE(workspace_bytes >= need && (workspace || !need), GTK_EWORKSPACE,
              "gtk_group_norm_forward: workspace %zu < %zu bytes", workspace ? workspace_bytes : 0, need);
  const int pbf = param_dtype == GTK_BF16;
  const Inputs in{x, x_stride, mask, {weight, pbf}, {bias, pbf}};
  const Shape s = Shape::of(B, positions, c, groups);
  auto run = [&](auto form) {
    return launch_gn_forward<decltype(form)>(in, y, (GroupStats*)stats, s, eps, activation, workspace, workspace_bytes,
                                             (hipStream_t)stream);
  };
  return dtype == GTK_F32 ? for_form<float>(s, run) : for_form<bf16>(s, run);
}

extern "C" size_t gtk_group_norm_backward_workspace_size(int64_t B, int64_t positions, int64_t c, int64_t groups,
                                                         int dtype) {
  if (!gn_shape_ok(B, positions, c, groups, dtype) || B == 0) return 0;
  return work_size<BackwardWork>(Shape::of(B, positions, c, groups), dtype, true);
}

extern "C" int gtk_group_norm_backward(const void* x, int64_t x_stride, const float* mask, const void* dy,
                                       int64_t dy_stride, const float* stats, const void* weight, const void* bias,
                                       int param_dtype, void* dx, void* dweight, void* dbias, int64_t B,
                                       int64_t positions, int64_t c, int64_t groups, int activation, int dtype,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  GTK_GN_CHECK("gtk_group_norm_backward");
  GTK_REQUIRE(dy_stride >= 0, GTK_EINVAL, "gtk_group_norm_backward: negative stride");
  if (!dx && !dweight && !dbias) return GTK_OK;
  GTK_REQUIRE(B == 0 || (x && dy && stats), GTK_EINVAL, "gtk_group_norm_backward: null pointer");
  const size_t need = gtk_group_norm_backward_workspace_size(B, positions, c, groups, dtype);
  GTK_REQUIRE(workspace_bytes >= need && (workspace || !need), GTK_EWORKSPACE,
              "gtk_group_norm_backward: workspace %zu < %zu bytes", workspace ? workspace_bytes : 0, need);
  const int pbf = param_dtype == GTK_BF16;
  if (B == 0)  // no samples: the sums are zero
    return dweight || dbias
               ? launch_column_close("group_norm_close", nullptr, 0, (int)c, dweight, dbias, pbf, (hipStream_t)stream)
               : GTK_OK;
  const Inputs in{x, x_stride, mask, {weight, pbf}, {bias, pbf}};
  const Shape s = Shape::of(B, positions, c, groups);
  auto run = [&](auto form) {
    return launch_gn_backward<decltype(form)>(in, dy, dy_stride, (const GroupStats*)stats, dx, dweight, dbias, pbf, s,
                                              activation, workspace, workspace_bytes, (hipStream_t)stream);
  };
  return dtype == GTK_F32 ? for_form<float>(s, run) : for_form<bf16>(s, run);
}
