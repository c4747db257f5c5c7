// LayerNorm as training uses it, for gfx950: rows at any stride, the affine
// optional and in either parameter type, and the backward pass with the
// reduction of the weight's and the bias' gradient.
//
// With d = x - mean, r = 1 / sqrt(mean(d^2) + eps), h = d r and g = dy w, a row
// of D values has
//   y  = h w + b
//   dx = r (g - mean(g) - h mean(g h))
// and over all rows dw = sum dy h, db = sum dy.  Mean and r are computed again
// from x in the backward pass, which has to read x anyway: nothing but x is
// kept from the forward pass.
//
// The sums of a row are taken of x - x_0, x_0 its first value: where the row
// lies far from zero and close together that difference is exact, and in any
// row |x - x_0| is at most twice the largest |d|, so what 32 bits lose follows
// the row's spread and not its offset.  (77 values of 1000.1 summed as they are
// give a mean 6e-5 away, which with eps = 1e-5 makes h 0.02 instead of 0.  The
// subtraction costs 1 to 2 %: 2^20 bf16 rows of 128, both passes, 226 us against
// 224; 3000 of 16384, 122 against 120.)  Each difference is divided by D before
// it is added, so that a row with the type's lowest value in it, in a masked
// place, has a finite mean; its variance is infinite in 32 bits, r and h are 0.
//
// Some twenty operations a value of 2 or 4 bytes: memory bounds both passes.  A
// row of up to kWidestInRegisters values therefore stays in the registers of its
// threads from its one load to its one store; wider ones are swept several times.
// On MI355X, inputs in rotation: 2^20 bf16 rows of 128 take 86 us forward (6.3
// TB/s) and 145 us backward (5.6 TB/s), 2^18 take 24 and 41 us, 4096 of 4096 17
// and 31 us, 10007 fp32 rows of 1023 17 and 31 us (backward: both launches); a
// copy beyond the caches runs at 6.3 TB/s.  Short launches are bound by their
// latency: 4096 fp32 rows of 128 take 3 us forward and 5 + 3 us backward.
#include <algorithm>

#include "capi_util.hpp"
#include "common.hpp"
#include "pack.hpp"

namespace gtk {

// A parameter vector of either type, or none.
struct ParamVec {
  const void* p = nullptr;
  int bf = 0;
  __device__ __forceinline__ float get(int c, float none) const {
    if (!p) return none;
    return bf ? to_f32(((const bf16*)p)[c]) : ((const float*)p)[c];
  }
};

// ---------------------------------------------------------------------------
// Rows in registers.  W waves share a row, or W = 1 and L <= 64 lanes of a wave
// do; lane t of a row's L * W lanes holds vectors of VE values (16 bytes), NV of
// them, vector j at column (j * L * W + t) * VE.  A width that is no multiple
// of VE ends with a vector that is moved back to end at column D: its first
// `skip` values belong to the vector before it and count for nothing in the
// row's sums (both lanes compute and store the same values there).  Rows of
// any alignment are read with 16-byte accesses, which gfx950 does at any
// address of the element's alignment.  VE = 1 is for rows shorter than one
// vector.  Loads and stores are non-temporal: each value is used once (2^20
// bf16 rows of 128, plain stores 86 and 155 us, non-temporal ones 84 and 147).
// ---------------------------------------------------------------------------
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

template <typename T, int VE> struct Vec {
  u32x4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = __builtin_nontemporal_load((const u32x4_any*)p); }
  __device__ __forceinline__ void store(T* p) const { __builtin_nontemporal_store(raw, (u32x4_any*)p); }
  __device__ __forceinline__ void get(float* f) const {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(raw[i] << 16);
        f[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(raw[i]);
    }
  }
  __device__ __forceinline__ void set(const float* f) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = __float_as_uint(f[i]);
    }
  }
};
template <typename T> struct Vec<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ void get(float* f) const { f[0] = to_f32(v); }
  __device__ __forceinline__ void set(const float* f) { v = cvt<T>(f[0]); }
};

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
// Sum over groups of L neighbouring lanes, the same bits in each of them.
template <int L> __device__ __forceinline__ float lane_sum(float v) {
  if (L >= 2) v += dpp<0xB1>(v);    // lane ^ 1
  if (L >= 4) v += dpp<0x4E>(v);    // lane ^ 2
  if (L >= 8) v += dpp<0x141>(v);   // the other four of eight
  if (L >= 16) v += dpp<0x140>(v);  // the other eight of sixteen
  if (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (L >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// The value of the first of L neighbouring lanes in each of them.
template <int L> __device__ __forceinline__ float first_lane(float v) {
  if constexpr (L == 64)
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
  else  // from lane & ~(L - 1) of each half wave
    return __uint_as_float(__builtin_amdgcn_ds_swizzle(__float_as_uint(v), 32 - L));
}

// The launch shape of one kernel: see above; BT threads a block, U rows a lane
// group at once, EXACT: D = L * W * NV * VE.
template <typename T_, int VE_, int NV_, int L_, int W_, int BT_, int U_, bool EXACT_> struct Shape {
  typedef T_ T;
  static constexpr int VE = VE_, NV = NV_, L = L_, W = W_, BT = BT_, U = U_;
  static constexpr bool EXACT = EXACT_;
  static constexpr int GROUPS = BT / (L * W);  // rows a block has in hand, times U
  static constexpr int ROWS = GROUPS * U;      // rows a block step
  static_assert(W == 1 || L == 64, "a row over several waves takes whole waves");
};

template <typename S> struct Columns {
  int c[S::NV], skip[S::NV];
  __device__ __forceinline__ Columns(int t, int D) {
#pragma unroll
    for (int j = 0; j < S::NV; ++j) {
      const int nominal = (j * S::L * S::W + t) * S::VE;
      c[j] = S::EXACT || nominal + S::VE <= D ? nominal : D - S::VE;
      skip[j] = S::EXACT || nominal < D ? nominal - c[j] : S::VE;  // VE: no column
    }
  }
};

// Sums of K values a lane over the row's lanes; red: K * (waves of a block)
// floats that no other call uses before the next barrier of this kernel.
template <typename S, int K> __device__ __forceinline__ void row_sums(float (&v)[K], float* red) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = lane_sum<S::L>(v[k]);
  if constexpr (S::W > 1) {
    const int wave = wave_id(), first = wave / S::W * S::W;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[k * (S::BT / 64) + wave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < S::W; ++w) v[k] += red[k * (S::BT / 64) + first + w];
    }
  }
}

// x_0 of a row: its lanes have it, where they are one wave's or fewer (rows of
// several waves load it with the row: no barrier for it).
template <typename S> struct Origin {
  typename S::T v;
  __device__ __forceinline__ void load(const typename S::T* row) {
    if constexpr (S::W > 1) v = *row;
  }
  // first: the lane's first value; column 0 is the first lane's
  __device__ __forceinline__ float get(float first) const {
    if constexpr (S::W > 1)
      return to_f32(v);
    else
      return first_lane<S::L>(first);
  }
};

// N consecutive values of a parameter vector (the branches are uniform).
template <int N> __device__ __forceinline__ void load_run(float* f, const ParamVec& p, int c) {
  if constexpr (N == 1) {
    f[0] = p.get(c, 0.f);
  } else if (p.bf) {
    uint32_t raw[N / 2];
    __builtin_memcpy(raw, (const bf16*)p.p + c, sizeof(raw));
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      f[2 * i] = __uint_as_float(raw[i] << 16);
      f[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
    }
  } else {
    __builtin_memcpy(f, (const float*)p.p + c, N * sizeof(float));
  }
}
template <typename S> __device__ __forceinline__ void load_param(float* f, const ParamVec& p, const Columns<S>& C, float none) {
  if (p.p) {
#pragma unroll
    for (int j = 0; j < S::NV; ++j) load_run<S::VE>(f + j * S::VE, p, C.c[j]);
  } else {
#pragma unroll
    for (int i = 0; i < S::NV * S::VE; ++i) f[i] = none;
  }
}

template <typename S>
__global__ __launch_bounds__(S::BT) void ln_forward_kernel(const typename S::T* __restrict__ x, int64_t xs,
                                                           typename S::T* __restrict__ y, ParamVec w, ParamVec b,
                                                           int64_t rows, int D, float eps) {
  typedef typename S::T T;
  constexpr int U = S::U, NV = S::NV, VE = S::VE, N = NV * VE;
  __shared__ float red[2][U * S::BT / 64];
  const int t = threadIdx.x % (S::L * S::W), group = threadIdx.x / (S::L * S::W);
  const Columns<S> C(t, D);
  const float inv = 1.0f / (float)D;
  float wf[N], bf[N];
  bool first = true;
  for (int64_t r0 = (int64_t)blockIdx.x * S::ROWS; r0 < rows; r0 += (int64_t)gridDim.x * S::ROWS) {
    Vec<T, VE> in[U][NV];
    Origin<S> origin[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // rows past the last one read the last one and are not stored
      const int64_t r = r0 + u * S::GROUPS + group, rc = r < rows ? r : rows - 1;
      origin[u].load(x + rc * xs);
#pragma unroll
      for (int j = 0; j < NV; ++j) in[u][j].load(x + rc * xs + C.c[j]);
    }
    if (first) {  // behind the first rows' loads
      load_param<S>(wf, w, C, 1.f);
      load_param<S>(bf, b, C, 0.f);
      first = false;
    }
    float s[U], q[U], f[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) in[u][j].get(&f[u][j * VE]);
      const float x0 = origin[u].get(f[u][0]);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        f[u][i] -= x0;
        s[u] += (S::EXACT || i % VE >= C.skip[i / VE] ? f[u][i] : 0.f) * inv;
      }
    }
    row_sums<S>(s, red[0]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      q[u] = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float d = f[u][j * VE + e] - s[u];
          f[u][j * VE + e] = d;
          q[u] += S::EXACT || e >= C.skip[j] ? d * d : 0.f;
        }
    }
    row_sums<S>(q, red[1]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float rstd = 1.0f / sqrtf(q[u] * inv + eps);
      const int64_t r = r0 + u * S::GROUPS + group;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float o[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) o[e] = f[u][j * VE + e] * rstd * wf[j * VE + e] + bf[j * VE + e];
        Vec<T, VE> out;
        out.set(o);
        if (r < rows && (S::EXACT || C.skip[j] < VE)) out.store(y + r * D + C.c[j]);
      }
    }
  }
}

// dx of every row, and this block's sums of dy h and dy over its rows:
// part[block][0][c], part[block][1][c].  The second reduction takes three sums
// at once: with q = sum d^2 and s2 = sum g d, mean(g h) = r s2 / D.  A thread
// keeps its columns over all its rows, so the column sums cost two registers a
// value and no traffic until the end; blocks are few and long-lived for that.
// With one vector a thread (NV = 1) the next step's rows are on their way while
// this one is reduced; with more the registers hold one step's only.
template <typename S>
__global__ __launch_bounds__(S::BT) void ln_backward_kernel(const typename S::T* __restrict__ x, int64_t xs,
                                                            const typename S::T* __restrict__ dy, int64_t ds,
                                                            typename S::T* __restrict__ dx, ParamVec w,
                                                            float* __restrict__ part, int64_t rows, int D, float eps) {
  typedef typename S::T T;
  constexpr int U = S::U, NV = S::NV, VE = S::VE, N = NV * VE;
  __shared__ float red0[U * S::BT / 64], red1[3 * U * S::BT / 64];
  extern __shared__ float sums[];  // [2][D], where a block has several groups
  // the widest rows read the weight again for each row: their registers hold no more
  constexpr bool KEEP = NV == 1;
  const int t = threadIdx.x % (S::L * S::W), group = threadIdx.x / (S::L * S::W);
  const Columns<S> C(t, D);
  const float inv = 1.0f / (float)D;
  float wf[N], aw[N], ab[N];
#pragma unroll
  for (int i = 0; i < N; ++i) aw[i] = ab[i] = 0.f;
  Vec<T, VE> xv[U][NV], gv[U][NV];
  Origin<S> origin[U];
  // past the end the last row again
  auto load_rows = [&](int64_t r0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * S::GROUPS + group, rc = r < rows ? r : rows - 1;
      origin[u].load(x + rc * xs);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        xv[u][j].load(x + rc * xs + C.c[j]);
        gv[u][j].load(dy + rc * ds + C.c[j]);
      }
    }
  };
  const int64_t stride = (int64_t)gridDim.x * S::ROWS;
  int64_t r0 = (int64_t)blockIdx.x * S::ROWS;
  load_rows(r0);
  if constexpr (KEEP) load_param<S>(wf, w, C, 1.f);
  for (; r0 < rows; r0 += stride) {
    float f[U][N], g[U][N], s[U], m[3 * U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        xv[u][j].get(&f[u][j * VE]);
        gv[u][j].get(&g[u][j * VE]);
      }
      const float x0 = origin[u].get(f[u][0]);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        f[u][i] -= x0;
        s[u] += (S::EXACT || i % VE >= C.skip[i / VE] ? f[u][i] : 0.f) * inv;
      }
    }
    if constexpr (KEEP)
      load_rows(r0 + stride);  // the next step's
    else
      load_param<S>(wf, w, C, 1.f);
    row_sums<S>(s, red0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float q = 0.f, s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = f[u][i] - s[u];
        const bool counts = S::EXACT || i % VE >= C.skip[i / VE];
        const float gw = counts ? g[u][i] * wf[i] : 0.f;
        f[u][i] = d;
        q += counts ? d * d : 0.f;
        s1 += gw;
        s2 += gw * d;
      }
      m[3 * u] = q;
      m[3 * u + 1] = s1;
      m[3 * u + 2] = s2;
    }
    row_sums<S>(m, red1);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float rstd = 1.0f / sqrtf(m[3 * u] * inv + eps);
      const float c1 = m[3 * u + 1] * inv, c2 = m[3 * u + 2] * inv * rstd;
      const int64_t r = r0 + u * S::GROUPS + group;
      const bool live = r < rows;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float o[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const int i = j * VE + e;
          const float h = f[u][i] * rstd;
          o[e] = (g[u][i] * wf[i] - c1 - h * c2) * rstd;
          if (live) {
            aw[i] += g[u][i] * h;
            ab[i] += g[u][i];
          }
        }
        Vec<T, VE> out;
        out.set(o);
        if (dx && live && (S::EXACT || C.skip[j] < VE)) out.store(dx + r * D + C.c[j]);
      }
    }
    if constexpr (!KEEP) load_rows(r0 + stride);
  }
  if (!part) return;
  // the groups' sums: first those of a wave, then wave after wave in LDS, as
  // whole vectors (value by value: 4096 rows of 4096 32.7 us, so 28.5)
  if constexpr (S::W == 1) {
#pragma unroll
    for (int off = S::L; off < 64; off <<= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        aw[i] += __shfl_xor(aw[i], off, 64);
        ab[i] += __shfl_xor(ab[i], off, 64);
      }
  }
  constexpr int TURNS = S::W == 1 ? S::BT / 64 : S::GROUPS;
  const int turn = S::W == 1 ? wave_id() : group;
  const bool holds = S::W > 1 || (threadIdx.x & 63) < S::L;
  float* dst = part + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {
    if (turn == k && holds) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = C.c[j];
        float *a = aw + j * VE, *b = ab + j * VE;
        if (S::EXACT || C.skip[j] == 0) {  // whole vectors
          if (k > 0) {
            float v[2][VE];
            __builtin_memcpy(v[0], sums + c, sizeof(v[0]));
            __builtin_memcpy(v[1], sums + D + c, sizeof(v[1]));
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              a[e] += v[0][e];
              b[e] += v[1][e];
            }
          }
          float* to = k == TURNS - 1 ? dst : sums;
          __builtin_memcpy(to + c, a, VE * sizeof(float));
          __builtin_memcpy(to + D + c, b, VE * sizeof(float));
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            if (e < C.skip[j]) continue;
            const float vw = k == 0 ? a[e] : sums[c + e] + a[e], vb = k == 0 ? b[e] : sums[D + c + e] + b[e];
            (k == TURNS - 1 ? dst : sums)[c + e] = vw;
            (k == TURNS - 1 ? dst : sums)[D + c + e] = vb;
          }
        }
      }
    }
    if (k < TURNS - 1) __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Rows that registers do not hold: a block a row, several sweeps.
// ---------------------------------------------------------------------------
constexpr int kWideThreads = 1024;
template <int K> __device__ __forceinline__ void block_sums(float (&v)[K], float* red) {
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = lane_sum<64>(v[k]);
    if ((threadIdx.x & 63) == 0) red[k * 16 + wave_id()] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = 0.f;
#pragma unroll
    for (int w = 0; w < kWideThreads / 64; ++w) v[k] += red[k * 16 + w];
  }
}

// Calls f(c, skip) for this thread's vectors of a row: at column c, of which
// the first `skip` values belong to another thread's vector (the last one ends
// at the row's end).
template <typename T, typename F> __device__ __forceinline__ void for_vectors(int D, F f) {
  constexpr int VE = 16 / sizeof(T);
#pragma unroll 4
  for (int c = threadIdx.x * VE; c < D; c += kWideThreads * VE) {
    const int at = c + VE <= D ? c : D - VE;
    f(at, c - at);
  }
}

template <typename T>
__global__ __launch_bounds__(kWideThreads) void ln_forward_wide_kernel(const T* __restrict__ x, int64_t xs,
                                                                       T* __restrict__ y, ParamVec w, ParamVec b,
                                                                       int64_t rows, int D, float eps) {
  constexpr int VE = 16 / sizeof(T);
  __shared__ float red[16];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    const float inv = 1.0f / (float)D;
    const float x0 = to_f32(xr[0]);
    float s[1] = {0.f}, q[1] = {0.f};
    for_vectors<T>(D, [&](int c, int skip) {
      Vec<T, VE> v;
      float f[VE];
      v.load(xr + c);
      v.get(f);
#pragma unroll
      for (int e = 0; e < VE; ++e) s[0] += (e >= skip ? f[e] - x0 : 0.f) * inv;
    });
    block_sums(s, red);
    const float mean = s[0];  // of x - x_0
    for_vectors<T>(D, [&](int c, int skip) {
      Vec<T, VE> v;
      float f[VE];
      v.load(xr + c);
      v.get(f);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float d = (f[e] - x0) - mean;
        q[0] += e >= skip ? d * d : 0.f;
      }
    });
    block_sums(q, red);
    const float rstd = 1.0f / sqrtf(q[0] * inv + eps);
    for_vectors<T>(D, [&](int c, int) {
      Vec<T, VE> v;
      float f[VE], wf[VE], bf[VE];
      v.load(xr + c);
      v.get(f);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        wf[e] = 1.f;
        bf[e] = 0.f;
      }
      if (w.p) load_run<VE>(wf, w, c);
      if (b.p) load_run<VE>(bf, b, c);
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = ((f[e] - x0) - mean) * rstd * wf[e] + bf[e];
      v.set(f);
      v.store(y + r * D + c);
    });
  }
}

// dx, and the mean of the row's x - x_0 and its rstd for the column sums.
template <typename T>
__global__ __launch_bounds__(kWideThreads) void ln_backward_wide_kernel(const T* __restrict__ x, int64_t xs,
                                                                        const T* __restrict__ dy, int64_t ds,
                                                                        T* __restrict__ dx, ParamVec w,
                                                                        float2* __restrict__ stats, int64_t rows, int D,
                                                                        float eps) {
  constexpr int VE = 16 / sizeof(T);
  __shared__ float red[48];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    const T* dr = dy + r * ds;
    const float inv = 1.0f / (float)D;
    const float x0 = to_f32(xr[0]);
    float s[1] = {0.f}, m[3] = {0.f, 0.f, 0.f};
    for_vectors<T>(D, [&](int c, int skip) {
      Vec<T, VE> v;
      float f[VE];
      v.load(xr + c);
      v.get(f);
#pragma unroll
      for (int e = 0; e < VE; ++e) s[0] += (e >= skip ? f[e] - x0 : 0.f) * inv;
    });
    block_sums(s, red);
    const float mean = s[0];  // of x - x_0
    // d and g at column c
    auto load = [&](int c, float* d, float* g) {
      Vec<T, VE> xv, gv;
      float wf[VE];
      xv.load(xr + c);
      gv.load(dr + c);
      xv.get(d);
      gv.get(g);
      if (w.p) {
        load_run<VE>(wf, w, c);
#pragma unroll
        for (int e = 0; e < VE; ++e) g[e] *= wf[e];
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) d[e] = (d[e] - x0) - mean;
    };
    for_vectors<T>(D, [&](int c, int skip) {
      float d[VE], g[VE];
      load(c, d, g);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float dm = e >= skip ? d[e] : 0.f, gm = e >= skip ? g[e] : 0.f;
        m[0] += dm * dm;
        m[1] += gm;
        m[2] += gm * dm;
      }
    });
    block_sums(m, red);
    const float rstd = 1.0f / sqrtf(m[0] * inv + eps);
    const float c1 = m[1] * inv, c2 = m[2] * inv * rstd;
    if (dx)
      for_vectors<T>(D, [&](int c, int) {
        float d[VE], g[VE];
        load(c, d, g);
#pragma unroll
        for (int e = 0; e < VE; ++e) d[e] = (g[e] - c1 - d[e] * rstd * c2) * rstd;
        Vec<T, VE> v;
        v.set(d);
        v.store(dx + r * D + c);
      });
    if (threadIdx.x == 0) stats[r] = float2{mean, rstd};
  }
}

// Column sums of dy h and dy over the rows of split blockIdx.y, 64 columns a
// block: part[split][0][c], part[split][1][c].
template <typename T>
__global__ __launch_bounds__(256) void ln_columns_kernel(const T* __restrict__ x, int64_t xs, const T* __restrict__ dy,
                                                         int64_t ds, const float2* __restrict__ stats,
                                                         float* __restrict__ part, int64_t rows, int D) {
  __shared__ float red[2][4][64];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int c = blockIdx.x * 64 + lane;
  float aw = 0.f, ab = 0.f;
  if (c < D)
    for (int64_t r = (int64_t)blockIdx.y * 4 + wave; r < rows; r += (int64_t)gridDim.y * 4) {
      const float2 st = stats[r];
      const float g = to_f32(dy[r * ds + c]);
      aw += g * (((to_f32(x[r * xs + c]) - to_f32(x[r * xs])) - st.x) * st.y);
      ab += g;
    }
  red[0][wave][lane] = aw;
  red[1][wave][lane] = ab;
  __syncthreads();
  if (wave < 2 && c < D)
    part[((int64_t)blockIdx.y * 2 + wave) * D + c] =
        (red[wave][0][lane] + red[wave][1][lane]) + (red[wave][2][lane] + red[wave][3][lane]);
}

// dst[c] = sum over the partials (c < D: the weight's, else the bias'): OUTS of
// the 2 D sums a block, CHUNKS threads each, eight loads in flight.
template <int OUTS, int CHUNKS>
__global__ __launch_bounds__(OUTS * CHUNKS) void ln_close_kernel(const float* __restrict__ part, int parts, int D,
                                                                 void* __restrict__ dw, void* __restrict__ db,
                                                                 int dst_bf) {
  __shared__ float red[CHUNKS][OUTS];
  const int o = threadIdx.x % OUTS, ch = threadIdx.x / OUTS;
  const int64_t i = (int64_t)blockIdx.x * OUTS + o, n = 2 * (int64_t)D;
  void* dst = i < D ? dw : db;
  const bool live = i < n && dst;
  float a[8] = {};
  if (live)
    for (int k = ch; k < parts; k += 8 * CHUNKS)
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int ku = k + u * CHUNKS;
        const float v = part[(ku < parts ? ku : parts - 1) * n + i];
        a[u] += ku < parts ? v : 0.f;
      }
  red[ch][o] = ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
  // in pairs
#pragma unroll
  for (int w = CHUNKS / 2; w > 0; w /= 2) {
    __syncthreads();
    if (ch < w) red[ch][o] += red[ch + w][o];
  }
  if (ch != 0 || !live) return;
  const float s = red[0][o];
  const int c = (int)(i < D ? i : i - D);
  if (dst_bf)
    ((bf16*)dst)[c] = cvt<bf16>(s);
  else
    ((float*)dst)[c] = s;
}

static int launch_ln_close(const float* part, int parts, int D, void* dw, void* db, int dst_bf, hipStream_t st) {
  StageTimer timer("layer_norm_close", st);
  // narrow rows leave few sums, and many partials of each: more threads a sum
  // (backward, 2^18 rows of 128: 40.5 us against 44.2 with 32 x 32; 2048 rows of
  // 8192: 34.0 against 31.4)
  if (D <= 512)
    ln_close_kernel<16, 64><<<(2 * D + 15) / 16, 1024, 0, st>>>(part, parts, D, dw, db, dst_bf);
  else
    ln_close_kernel<32, 32><<<(2 * D + 31) / 32, 1024, 0, st>>>(part, parts, D, dw, db, dst_bf);
  GTK_LAUNCH_CHECK();
  return GTK_OK;
}

// ---------------------------------------------------------------------------
// Shapes by width
// ---------------------------------------------------------------------------
// Calls run(Shape) for the narrowest shape that holds D: U rows a lane group at
// once where the shape is filled, UM where it is not.
template <typename T, int VE, int NV, int L, int W, int BT, int U, int UM, typename F>
static int with_shape(int D, F& run) {
  if (D == VE * NV * L * W) return run(Shape<T, VE, NV, L, W, BT, U, true>());
  return run(Shape<T, VE, NV, L, W, BT, UM, false>());
}

template <typename T, bool BACKWARD, typename F> static int for_shape(int D, F run) {
  constexpr int VE = 16 / sizeof(T);
  // A wave or less a row.  Backward blocks of 512 threads, two a CU: 2^20 bf16
  // rows of 128 in 154 us, of 256 threads 159, of 1024 163.  Two rows a group
  // keep more loads in flight (147 us with one, 140 with two); where the shape
  // is not filled the masks take their registers (10^5 rows of 384: 53 and 57).
  constexpr int B = BACKWARD ? 512 : 256, UM = BACKWARD ? 1 : 2;
  if (D < VE) return run(Shape<T, 1, 1, VE, 1, B, UM, false>());
  if (D <= 2 * VE) return with_shape<T, VE, 1, 2, 1, B, 2, UM>(D, run);
  if (D <= 4 * VE) return with_shape<T, VE, 1, 4, 1, B, 2, UM>(D, run);
  if (D <= 8 * VE) return with_shape<T, VE, 1, 8, 1, B, 2, UM>(D, run);
  if (D <= 16 * VE) return with_shape<T, VE, 1, 16, 1, B, 2, UM>(D, run);
  if (D <= 32 * VE) return with_shape<T, VE, 1, 32, 1, B, 2, UM>(D, run);
  if (D <= 64 * VE) return with_shape<T, VE, 1, 64, 1, B, 2, UM>(D, run);
  // Several waves: forward, two rows a group wait for each barrier once (4096
  // rows of 4096: 16.4 us, with one 18.2).  The backward's one block a CU leaves
  // the fewest partial sums; 512 threads hold enough loads in flight (16384 rows
  // of 1024: 25 us, of 1024 threads 27; two rows a group 27.5).
  constexpr int U = BACKWARD ? 1 : 2, BW = BACKWARD ? 512 : 256;
  if (D <= 128 * VE) return with_shape<T, VE, 1, 64, 2, BW, U, U>(D, run);
  if (D <= 256 * VE) return with_shape<T, VE, 1, 64, 4, BW, U, U>(D, run);
  if (D <= 512 * VE) return with_shape<T, VE, 1, 64, 8, 512, U, U>(D, run);
  if (D <= 1024 * VE) return with_shape<T, VE, 1, 64, 16, 1024, U, U>(D, run);
  if constexpr (sizeof(T) == 4)
    if (D > 2048 * VE) return with_shape<T, VE, 4, 64, 16, 1024, 1, 1>(D, run);
  return with_shape<T, VE, 2, 64, 16, 1024, U, U>(D, run);
}
// 3000 fp32 rows of 16384: backward 131 us in registers, 293 by sweeps.
constexpr int kWidestInRegisters = 16384;

// Blocks of the backward kernel: each leaves 2 D partial sums, so few.
static int backward_blocks(int64_t rows, int rows_a_step, int blocks_a_cu) {
  const int64_t steps = (rows + rows_a_step - 1) / rows_a_step;
  return (int)std::min<int64_t>(steps, (int64_t)device_cus() * blocks_a_cu);
}

static int column_splits(int64_t rows) { return (int)std::min<int64_t>(256, std::max<int64_t>(1, (rows + 15) / 16)); }

// Partial sums that the backward pass leaves for its last launch.
template <typename T> static int backward_parts(int64_t rows, int D) {
  if (D > kWidestInRegisters) return column_splits(rows);
  return for_shape<T, true>(D, [&](auto shape) {
    typedef decltype(shape) S;
    return backward_blocks(rows, S::ROWS, S::W == 1 ? 2 : 1);
  });
}

template <typename T> static void carve_ln_backward(Carve& cv, int64_t rows, int64_t d, float2** stats, float** part) {
  *stats = cv.take<float2>(d > kWidestInRegisters ? rows : 0);
  *part = cv.take<float>(2 * d * backward_parts<T>(rows, (int)d));
}

template <typename T>
static int launch_ln_forward(const T* x, int64_t xs, T* y, ParamVec w, ParamVec b, int64_t rows, int D, float eps,
                             hipStream_t st) {
  StageTimer timer("layer_norm_forward", st);
  if (D > kWidestInRegisters)
    ln_forward_wide_kernel<T><<<(unsigned)std::min<int64_t>(rows, 1 << 20), kWideThreads, 0, st>>>(x, xs, y, w, b, rows, D, eps);
  else
    for_shape<T, false>(D, [&](auto shape) {
      typedef decltype(shape) S;
      const unsigned grid = (unsigned)std::min<int64_t>((rows + S::ROWS - 1) / S::ROWS, 1 << 20);
      ln_forward_kernel<S><<<grid, S::BT, 0, st>>>(x, xs, y, w, b, rows, D, eps);
      return 0;
    });
  GTK_LAUNCH_CHECK();
  return GTK_OK;
}

template <typename T>
static int launch_ln_backward(const T* x, int64_t xs, const T* dy, int64_t ds, T* dx, ParamVec w, void* dw, void* db,
                              int dst_bf, int64_t rows, int D, float eps, void* ws, size_t ws_bytes, hipStream_t st) {
  Carve cv(ws, ws_bytes);
  float2* stats;
  float* part;
  carve_ln_backward<T>(cv, rows, D, &stats, &part);
  const bool sums = dw || db;
  const int parts = backward_parts<T>(rows, D);
  if (D > kWidestInRegisters) {
    {
      StageTimer timer("layer_norm_backward", st);
      ln_backward_wide_kernel<T><<<(unsigned)std::min<int64_t>(rows, 1 << 20), kWideThreads, 0, st>>>(
          x, xs, dy, ds, dx, w, stats, rows, D, eps);
      GTK_LAUNCH_CHECK();
    }
    if (sums) {
      StageTimer timer("layer_norm_columns", st);
      ln_columns_kernel<T><<<dim3((D + 63) / 64, parts), 256, 0, st>>>(x, xs, dy, ds, stats, part, rows, D);
      GTK_LAUNCH_CHECK();
    }
  } else {
    StageTimer timer("layer_norm_backward", st);
    for_shape<T, true>(D, [&](auto shape) {
      typedef decltype(shape) S;
      const size_t lds = S::BT / 64 > S::W ? 2 * (size_t)D * sizeof(float) : 0;
      ln_backward_kernel<S><<<(unsigned)parts, S::BT, lds, st>>>(x, xs, dy, ds, dx, w, sums ? part : nullptr, rows, D, eps);
      return 0;
    });
    GTK_LAUNCH_CHECK();
  }
  return sums ? launch_ln_close(part, parts, D, dw, db, dst_bf, st) : GTK_OK;
}

}  // namespace gtk

using namespace gtk;

#define GTK_LN_CHECK_SHAPE(name)                                                                             \
  GTK_REQUIRE(rows >= 0 && rows <= (int64_t)1 << 40, GTK_EINVAL, name ": bad row count %lld", (long long)rows); \
  GTK_REQUIRE(d >= 1 && d <= 1 << 24, GTK_EINVAL, name ": d=%lld not in [1, 2^24]", (long long)d);           \
  GTK_REQUIRE(dtype == GTK_F32 || dtype == GTK_BF16, GTK_EINVAL, name ": bad dtype %d", dtype);              \
  GTK_REQUIRE(param_dtype == GTK_F32 || param_dtype == GTK_BF16, GTK_EINVAL, name ": bad parameter dtype %d", \
              param_dtype);                                                                                  \
  GTK_REQUIRE(x_stride >= 0, GTK_EINVAL, name ": negative row stride")

extern "C" int gtk_layer_norm_forward(const void* x, int64_t x_stride, void* y, const void* weight, const void* bias,
                                      int param_dtype, int64_t rows, int64_t d, float eps, int dtype, void* stream) {
  GTK_LN_CHECK_SHAPE("gtk_layer_norm_forward");
  if (rows == 0) return GTK_OK;
  GTK_REQUIRE(x && y, GTK_EINVAL, "gtk_layer_norm_forward: null pointer");
  hipStream_t st = (hipStream_t)stream;
  const ParamVec w{weight, param_dtype == GTK_BF16}, b{bias, param_dtype == GTK_BF16};
  if (dtype == GTK_F32) return launch_ln_forward<float>((const float*)x, x_stride, (float*)y, w, b, rows, (int)d, eps, st);
  return launch_ln_forward<bf16>((const bf16*)x, x_stride, (bf16*)y, w, b, rows, (int)d, eps, st);
}

extern "C" size_t gtk_layer_norm_backward_workspace_size(int64_t rows, int64_t d, int dtype) {
  if (rows < 0 || rows > (int64_t)1 << 40 || d < 1 || d > 1 << 24 || (dtype != GTK_F32 && dtype != GTK_BF16)) return 0;
  Carve cv(nullptr, SIZE_MAX);
  float2* stats;
  float* part;
  if (dtype == GTK_F32)
    carve_ln_backward<float>(cv, rows, d, &stats, &part);
  else
    carve_ln_backward<bf16>(cv, rows, d, &stats, &part);
  return cv.off;
}

extern "C" int gtk_layer_norm_backward(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride,
                                       const void* weight, int param_dtype, void* dx, void* dweight, void* dbias,
                                       int64_t rows, int64_t d, float eps, int dtype, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  GTK_LN_CHECK_SHAPE("gtk_layer_norm_backward");
  GTK_REQUIRE(dy_stride >= 0, GTK_EINVAL, "gtk_layer_norm_backward: negative row stride");
  if (!dx && !dweight && !dbias) return GTK_OK;
  hipStream_t st = (hipStream_t)stream;
  const int pbf = param_dtype == GTK_BF16;
  if (rows == 0)  // no rows: the sums are zero
    return dweight || dbias ? launch_ln_close(nullptr, 0, (int)d, dweight, dbias, pbf, st) : GTK_OK;
  GTK_REQUIRE(x && dy && workspace, GTK_EINVAL, "gtk_layer_norm_backward: null pointer");
  const size_t need = gtk_layer_norm_backward_workspace_size(rows, d, dtype);
  GTK_REQUIRE(workspace_bytes >= need, GTK_EWORKSPACE, "gtk_layer_norm_backward: workspace %zu < %zu bytes",
              workspace_bytes, need);
  const ParamVec w{weight, pbf};
  if (dtype == GTK_F32)
    return launch_ln_backward<float>((const float*)x, x_stride, (const float*)dy, dy_stride, (float*)dx, w, dweight,
                                     dbias, pbf, rows, (int)d, eps, workspace, workspace_bytes, st);
  return launch_ln_backward<bf16>((const bf16*)x, x_stride, (const bf16*)dy, dy_stride, (bf16*)dx, w, dweight, dbias,
                                  pbf, rows, (int)d, eps, workspace, workspace_bytes, st);
}
