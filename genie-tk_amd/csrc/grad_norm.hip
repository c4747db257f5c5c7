// The global norm of a set of gradients, and clipping by it, for gfx950.
//
//   n = (sum |g|^p)^(1/p) over every value of every tensor, p in {1, 2, inf}
//   k = min(1, max_norm / (n + 1e-6)),  out = k g
//
// The values' squares and their sums are 64-bit: the square of a 32-bit float
// fits a 64-bit one exactly, so neither gradients above 1.8e19 overflow nor
// ones below 1e-23 vanish.  The tensors' addresses and sizes travel in the
// kernel arguments, 248 runs of memory a launch (165 with outputs): no table is
// copied to the GPU, and a captured launch keeps them.  A block takes one chunk
// of one run and leaves one partial sum; one block adds those in a fixed order,
// so equal inputs in equal places give equal bits.
//
// The norm reads every value once, the product reads and writes it once more:
// memory, or for small sets the launches.  On MI355X 4e8 bf16 values take 123 us
// (6.5 TB/s, reading alone reaches 7.0; conversion to 64 bits and the product-sum
// are hidden), in norms of order 1 and inf too.  1.5e8 fp32 values clipped into
// fp32 masters take 309 us (1.8 GB moved, 5.8 TB/s; a copy reaches 6.3), in place
// 321 us, and bf16 ones in place 167 us (5.6 and 5.4 TB/s).  The 464 gradients of
// an 8-layer net, as its backward pass leaves them: 33 us in place, 44 into
// masters, of which the GPU works 16; the 1392 of 24 layers 71 to 80 and 106 to
// 120.  Those are the host's: it touches every tensor.
// Reading the values in reverse for the product, to find the last of them still
// in the Infinity Cache, gained nothing (432 us forwards, 451 backwards).
#include <algorithm>
#include <memory>
#include <new>
#include <type_traits>

#include "capi_util.hpp"
#include "common.hpp"
#include "pack.hpp"

namespace gtk {

// One launch's tensors (or parts of one): src[k] of n[k] values, whose blocks
// start at first[k].  The types are the two top bits of n.
constexpr uint32_t kSrcBf = 1u << 31, kDstBf = 1u << 30, kCountMask = kDstBf - 1;
constexpr int64_t kMaxPart = (int64_t)1 << 29;  // values an entry; a multiple of every chunk
template <int MAX, bool OUT> struct Jobs {
  static constexpr int kMax = MAX;
  static constexpr bool kOut = OUT;
  uint64_t src[MAX];
  uint64_t dst[OUT ? MAX : 1];
  uint32_t n[MAX];
  uint32_t first[MAX];
  uint32_t count, chunk;  // chunk: values a block
};
typedef Jobs<248, false> JobsIn;     // in place, or read alone
typedef Jobs<165, true> JobsInOut;
static_assert(sizeof(JobsIn) <= 4000 && sizeof(JobsInOut) <= 4000, "kernel arguments");

// The entry that block blockIdx.x works on: every wave counts the entries that
// start at or before it, 64 at a time.
template <typename J> __device__ __forceinline__ int find_entry(const J& jobs) {
  const uint32_t lane = threadIdx.x & 63;
  int k = 0;
#pragma unroll
  for (uint32_t i = 0; i < (uint32_t)J::kMax; i += 64) {
    const uint32_t at = i + lane;
    const bool before = at < jobs.count && jobs.first[at < (uint32_t)J::kMax ? at : 0] <= blockIdx.x;
    k += __popcll(__ballot(before));
  }
  return __builtin_amdgcn_readfirstlane(k - 1);
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));  // 16 bytes at any address of the element's alignment
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));

constexpr int kThreads = 256;

// The largest |g| is found on the bits: the order of non-negative floats is
// that of their bits, infinity and NaN (the largest) included.
template <int KIND> struct Sum {
  double v = 0.0;
  uint32_t m = 0;
  __device__ __forceinline__ void add(float x) {
    if (KIND == GTK_NORM_2) v = __builtin_fma((double)x, (double)x, v);
    if (KIND == GTK_NORM_1) v += (double)fabsf(x);
    if (KIND == GTK_NORM_INF) {
      const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
      m = a > m ? a : m;
    }
  }
  __device__ __forceinline__ void join(const Sum& o) {
    v += o.v;
    m = o.m > m ? o.m : m;
  }
  // as 64 bits in memory
  __device__ __forceinline__ void put(double* p) const {
    *p = KIND == GTK_NORM_INF ? __builtin_bit_cast(double, (uint64_t)m) : v;
  }
  __device__ __forceinline__ static Sum of(double d) {
    Sum s;
    if (KIND == GTK_NORM_INF)
      s.m = (uint32_t)__builtin_bit_cast(uint64_t, d);
    else
      s.v = d;
    return s;
  }
};

template <int KIND, int WAVES> __device__ __forceinline__ Sum<KIND> block_join(Sum<KIND> s, double* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    Sum<KIND> o;
    o.v = __shfl_xor(s.v, off, 64);
    o.m = __shfl_xor(s.m, off, 64);
    s.join(o);
  }
  if ((threadIdx.x & 63) == 0) s.put(red + (threadIdx.x >> 6));
  __syncthreads();
  s = Sum<KIND>::of(red[0]);
#pragma unroll
  for (int w = 1; w < WAVES; ++w) s.join(Sum<KIND>::of(red[w]));
  return s;
}

// 16 bytes of values as floats.
template <bool BF> __device__ __forceinline__ void widen(u32x4 raw, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (BF) {
      f[2 * i] = __uint_as_float(raw[i] << 16);
      f[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
    } else {
      f[i] = __uint_as_float(raw[i]);
    }
  }
}

// The sum over p[0 .. n): U vectors of 16 bytes in flight a thread, then the
// last n % VE values one a thread.
template <int KIND, bool BF> __device__ __forceinline__ Sum<KIND> sum_run(const void* base, int64_t begin, uint32_t n) {
  typedef typename std::conditional<BF, bf16, float>::type T;
  constexpr uint32_t VE = BF ? 8 : 4, U = 4;
  const T* p = (const T*)base + begin;
  Sum<KIND> s[2];
  const uint32_t vecs = n / VE;
  uint32_t v = threadIdx.x;
  for (; v + (U - 1) * kThreads < vecs; v += U * kThreads) {
    u32x4 raw[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
      raw[u] = __builtin_nontemporal_load((const u32x4_any*)(p + (uint64_t)(v + u * kThreads) * VE));
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      float f[VE];
      widen<BF>(raw[u], f);
#pragma unroll
      for (uint32_t e = 0; e < VE; ++e) s[e & 1].add(f[e]);
    }
  }
  for (; v < vecs; v += kThreads) {
    float f[VE];
    widen<BF>(*(const u32x4_any*)(p + (uint64_t)v * VE), f);
#pragma unroll
    for (uint32_t e = 0; e < VE; ++e) s[e & 1].add(f[e]);
  }
  if (threadIdx.x < n % VE) s[0].add(to_f32(p[(uint64_t)vecs * VE + threadIdx.x]));
  s[0].join(s[1]);
  return s[0];
}

template <int KIND>
__global__ __launch_bounds__(kThreads) void grad_partials_kernel(JobsIn J, double* __restrict__ part) {
  __shared__ double red[kThreads / 64];
  const int k = find_entry(J);
  const uint32_t count = J.n[k] & kCountMask, block = blockIdx.x - J.first[k];
  const int64_t begin = (int64_t)block * J.chunk;
  const uint32_t n = (uint32_t)(begin + J.chunk < count ? J.chunk : count - begin);
  const void* p = (const void*)J.src[k];
  Sum<KIND> s = J.n[k] & kSrcBf ? sum_run<KIND, true>(p, begin, n) : sum_run<KIND, false>(p, begin, n);
  s = block_join<KIND, kThreads / 64>(s, red);
  if (threadIdx.x == 0) s.put(part + blockIdx.x);
}

constexpr int kCloseThreads = 1024;
template <int KIND>
__global__ __launch_bounds__(kCloseThreads) void grad_norm_close_kernel(const double* __restrict__ part, int64_t parts,
                                                                        float* __restrict__ norm) {
  __shared__ double red[kCloseThreads / 64];
  constexpr int U = 8;
  Sum<KIND> s;
  for (int64_t i = threadIdx.x; i < parts; i += U * kCloseThreads) {
    double d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = i + u * kCloseThreads;
      d[u] = part[at < parts ? at : parts - 1];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kCloseThreads < parts) s.join(Sum<KIND>::of(d[u]));
  }
  s = block_join<KIND, kCloseThreads / 64>(s, red);
  if (threadIdx.x == 0) *norm = KIND == GTK_NORM_INF ? __uint_as_float(s.m) : (float)(KIND == GTK_NORM_2 ? sqrt(s.v) : s.v);
}

// The factor of the clipping, one rounding to 32 bits.  A norm of NaN makes it
// NaN, an infinite one 0.
__device__ __forceinline__ float clip_factor(float norm, double max_norm) {
  const double f = max_norm / ((double)norm + 1e-6);
  return f > 1.0 ? 1.f : (float)f;
}

template <bool SRC_BF, bool DST_BF> __device__ __forceinline__ void put_vec(void* dst, const float* f) {
  if constexpr (DST_BF) {
    if constexpr (SRC_BF)
      *(u32x4_any*)dst = u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                               pack_bf16x2(f[6], f[7])};
    else
      *(u32x2_any*)dst = u32x2{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])};
  } else {
#pragma unroll
    for (int h = 0; h < (SRC_BF ? 2 : 1); ++h)
      ((u32x4_any*)dst)[h] = u32x4{__float_as_uint(f[4 * h]), __float_as_uint(f[4 * h + 1]),
                                   __float_as_uint(f[4 * h + 2]), __float_as_uint(f[4 * h + 3])};
  }
}

// dst[i] = src[i] * k for i in [begin, begin + n).  No thread writes what another
// reads, so dst may be src.
template <bool SRC_BF, bool DST_BF>
__device__ __forceinline__ void scale_run(const void* src, void* dst, int64_t begin, uint32_t n, float k) {
  typedef typename std::conditional<SRC_BF, bf16, float>::type S;
  typedef typename std::conditional<DST_BF, bf16, float>::type D;
  constexpr uint32_t VE = SRC_BF ? 8 : 4, U = 4;
  const S* p = (const S*)src + begin;
  D* q = (D*)dst + begin;
  const uint32_t vecs = n / VE;
  uint32_t v = threadIdx.x;
  for (; v + (U - 1) * kThreads < vecs; v += U * kThreads) {
    u32x4 raw[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) raw[u] = *(const u32x4_any*)(p + (uint64_t)(v + u * kThreads) * VE);
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      float f[VE];
      widen<SRC_BF>(raw[u], f);
#pragma unroll
      for (uint32_t e = 0; e < VE; ++e) f[e] *= k;
      put_vec<SRC_BF, DST_BF>(q + (uint64_t)(v + u * kThreads) * VE, f);
    }
  }
  for (; v < vecs; v += kThreads) {
    float f[VE];
    widen<SRC_BF>(*(const u32x4_any*)(p + (uint64_t)v * VE), f);
#pragma unroll
    for (uint32_t e = 0; e < VE; ++e) f[e] *= k;
    put_vec<SRC_BF, DST_BF>(q + (uint64_t)v * VE, f);
  }
  if (threadIdx.x < n % VE) {
    const uint64_t i = (uint64_t)vecs * VE + threadIdx.x;
    q[i] = cvt<D>(to_f32(p[i]) * k);
  }
}

template <typename J>
__global__ __launch_bounds__(kThreads) void grad_scale_kernel(J jobs, const float* __restrict__ norm, double max_norm) {
  const float f = clip_factor(*norm, max_norm);
  if (!J::kOut && f == 1.f) return;  // the product would leave every value's bits
  const int k = find_entry(jobs);
  const uint32_t flags = jobs.n[k], count = flags & kCountMask, block = blockIdx.x - jobs.first[k];
  const int64_t begin = (int64_t)block * jobs.chunk;
  const uint32_t n = (uint32_t)(begin + jobs.chunk < count ? jobs.chunk : count - begin);
  const void* src = (const void*)jobs.src[k];
  void* dst = J::kOut ? (void*)jobs.dst[J::kOut ? k : 0] : (void*)src;
  if (flags & kSrcBf) {
    if (flags & kDstBf)
      scale_run<true, true>(src, dst, begin, n, f);
    else if (J::kOut)
      scale_run<true, false>(src, dst, begin, n, f);
  } else {
    if (!(flags & kDstBf))
      scale_run<false, false>(src, dst, begin, n, f);
    else if (J::kOut)
      scale_run<false, true>(src, dst, begin, n, f);
  }
}

// Values a block, the same for a whole pass: at least kMinChunk, and doubled up
// to `most` while the pass has more than 16 blocks a CU.  The norm takes blocks
// of up to kNormChunk values (a block pays for finding its tensor and for
// joining its sums: 4e8 bf16 values in 142 us with blocks of 131072 values, 126
// with 16384, 136 with 8192), the product kScaleChunk (it has no sums to join:
// 1.5e8 fp32 values clipped to masters in 352, 334, 317 us).  Past 65536 blocks
// they grow again, so that the partial sums stay few.
constexpr int64_t kMinChunk = 4096, kNormChunk = 16384, kScaleChunk = 8192;
static int64_t chunk_of(const gtk_tensor_list* g, int64_t most) {
  int64_t total = 0;
  for (int64_t i = 0; i < g->count; ++i) total += g->numel[i];
  int64_t chunk = kMinChunk;
  while (chunk < kMaxPart && total / chunk > (chunk < most ? 16 * 256 : 65536)) chunk *= 2;
  return chunk;
}

// Most blocks that the list takes: runs that are joined take fewer.
static int64_t most_blocks(const gtk_tensor_list* g, int64_t chunk) {
  int64_t b = 0;
  for (int64_t i = 0; i < g->count; ++i) b += (g->numel[i] + chunk - 1) / chunk;
  return b;
}

// Calls launch(jobs, blocks, first partial) for every J::kMax entries.
// Tensors that lie one behind the other in memory are one run, and so one entry.
// An operator's backward pass leaves its gradients in one buffer, but partly in
// another order than the module's parameters: a pair-stack layer's 58 gradients
// are 15 runs, the 1392 of 24 layers 360, two launches a pass (apart: six; in one
// buffer in the list's order: one.  In place 71, 89 and 63 us).
template <typename J, typename F>
static int for_each_launch(const gtk_tensor_list* g, const gtk_tensor_list* out, int64_t chunk, F launch) {
  J jobs;
  jobs.chunk = (uint32_t)chunk;
  jobs.count = 0;
  uint32_t blocks = 0;
  int64_t base = 0;
  const gtk_tensor_list* o = out ? out : g;
  for (int64_t i = 0; i < g->count;) {
    const int64_t i0 = i;
    const bool sbf = g->dtype[i] == GTK_BF16, dbf = o->dtype[i] == GTK_BF16;
    const uint32_t flags = (sbf ? kSrcBf : 0) | (dbf ? kDstBf : 0);
    const char* src = (const char*)g->data[i];
    char* dst = (char*)o->data[i];
    int64_t run = g->numel[i];
    const int64_t se = sbf ? 2 : 4, de = dbf ? 2 : 4;
    for (++i; i < g->count; ++i) {
      if (g->numel[i] == 0) continue;
      if (run == 0 || g->data[i] != src + run * se || g->dtype[i] != g->dtype[i0] || o->data[i] != dst + run * de ||
          o->dtype[i] != o->dtype[i0])
        break;
      run += g->numel[i];
    }
    for (int64_t at = 0; at < run; at += kMaxPart) {
      const int64_t n = std::min(run - at, kMaxPart);
      const uint32_t k = jobs.count++;
      jobs.src[k] = (uint64_t)(uintptr_t)(src + at * se);
      if (J::kOut) jobs.dst[J::kOut ? k : 0] = (uint64_t)(uintptr_t)(dst + at * de);
      jobs.n[k] = (uint32_t)n | flags;
      jobs.first[k] = blocks;
      blocks += (uint32_t)((n + chunk - 1) / chunk);
      if (jobs.count == (uint32_t)J::kMax || blocks >= 1u << 22) {
        const int rc = launch(jobs, blocks, base);
        if (rc) return rc;
        base += blocks;
        jobs.count = blocks = 0;
      }
    }
  }
  return jobs.count ? launch(jobs, blocks, base) : GTK_OK;
}

static int check_list(const gtk_tensor_list* g, const char* name) {
  GTK_REQUIRE(g && g->count >= 0, GTK_EINVAL, "%s: bad tensor list", name);
  GTK_REQUIRE(g->count == 0 || (g->data && g->numel && g->dtype), GTK_EINVAL, "%s: null pointer", name);
  for (int64_t i = 0; i < g->count; ++i) {
    GTK_REQUIRE(g->numel[i] >= 0 && g->numel[i] <= (int64_t)1 << 40, GTK_EINVAL, "%s: tensor %lld: bad size %lld", name,
                (long long)i, (long long)g->numel[i]);
    GTK_REQUIRE(g->dtype[i] == GTK_F32 || g->dtype[i] == GTK_BF16, GTK_EINVAL, "%s: tensor %lld: bad dtype %d", name,
                (long long)i, g->dtype[i]);
    GTK_REQUIRE(g->numel[i] == 0 || g->data[i], GTK_EINVAL, "%s: tensor %lld: null pointer", name, (long long)i);
  }
  return GTK_OK;
}

struct Span {
  const char *begin, *end;
};

// The memory of a list's tensors, in ascending order.
struct Spans {
  std::unique_ptr<Span[]> v;
  int64_t n = 0;
  bool sorted = true;
  explicit Spans(int64_t most) : v(new (std::nothrow) Span[(size_t)most + 1]) {}
  void add(const gtk_tensor_list* l, int64_t i) {
    if (l->numel[i] == 0) return;
    const char* p = (const char*)l->data[i];
    if (n && p < v[n - 1].begin) sorted = false;
    v[n++] = {p, p + l->numel[i] * (int64_t)dtype_size(l->dtype[i])};
  }
  void sort() {
    if (!sorted) std::sort(v.get(), v.get() + n, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  }
};

// Nothing that is written is written twice or read by another tensor's block:
// blocks run in any order.
static int check_overlap(const gtk_tensor_list* g, const gtk_tensor_list* out, const char* name) {
  Spans w(g->count), r(out ? g->count : 0);
  GTK_REQUIRE(w.v && r.v, GTK_EINVAL, "%s: out of host memory", name);
  for (int64_t i = 0; i < g->count; ++i) {
    w.add(out ? out : g, i);
    // a tensor clipped onto itself is read and written by the same thread
    if (out && !(out->data[i] == g->data[i] && out->dtype[i] == g->dtype[i])) r.add(g, i);
  }
  w.sort();
  r.sort();
  const char *any = nullptr, *written = nullptr;  // the furthest ends so far
  for (int64_t i = 0, j = 0; i < w.n || j < r.n;) {
    const bool write = j == r.n || (i < w.n && w.v[i].begin <= r.v[j].begin);
    const Span& s = write ? w.v[i++] : r.v[j++];
    GTK_REQUIRE(s.begin >= (write ? any : written), GTK_EINVAL,
                "%s: a tensor that is written overlaps another (or is given twice)", name);
    any = std::max(any, s.end);
    if (write) written = std::max(written, s.end);
  }
  return GTK_OK;
}

template <int KIND>
static int launch_norm(const gtk_tensor_list* g, float* norm, double* part, hipStream_t st) {
  int64_t parts = 0;
  {
    StageTimer timer("grad_partials", st);
    const int rc = for_each_launch<JobsIn>(g, nullptr, chunk_of(g, kNormChunk), [&](const JobsIn& J, unsigned blocks, int64_t base) -> int {
      grad_partials_kernel<KIND><<<blocks, kThreads, 0, st>>>(J, part + base);
      GTK_LAUNCH_CHECK();
      parts = base + blocks;
      return GTK_OK;
    });
    if (rc) return rc;
  }
  StageTimer timer("grad_norm_close", st);
  grad_norm_close_kernel<KIND><<<1, kCloseThreads, 0, st>>>(part, parts, norm);
  GTK_LAUNCH_CHECK();
  return GTK_OK;
}

static int launch_norm(int kind, const gtk_tensor_list* g, float* norm, double* part, hipStream_t st) {
  switch (kind) {
    case GTK_NORM_2: return launch_norm<GTK_NORM_2>(g, norm, part, st);
    case GTK_NORM_1: return launch_norm<GTK_NORM_1>(g, norm, part, st);
    default: return launch_norm<GTK_NORM_INF>(g, norm, part, st);
  }
}

template <typename J>
static int launch_scale(const gtk_tensor_list* g, const gtk_tensor_list* out, double max_norm, const float* norm,
                        hipStream_t st) {
  StageTimer timer("grad_scale", st);
  return for_each_launch<J>(g, out, chunk_of(g, kScaleChunk), [&](const J& jobs, unsigned blocks, int64_t) -> int {
    grad_scale_kernel<J><<<blocks, kThreads, 0, st>>>(jobs, norm, max_norm);
    GTK_LAUNCH_CHECK();
    return GTK_OK;
  });
}

static int launch_scale(const gtk_tensor_list* g, const gtk_tensor_list* out, double max_norm, const float* norm,
                        hipStream_t st) {
  return out ? launch_scale<JobsInOut>(g, out, max_norm, norm, st) : launch_scale<JobsIn>(g, out, max_norm, norm, st);
}

static int check_out(const gtk_tensor_list* g, const gtk_tensor_list* out, const char* name) {
  int rc;
  if (out) {
    if ((rc = check_list(out, name))) return rc;
    GTK_REQUIRE(out->count == g->count, GTK_EINVAL, "%s: %lld outputs for %lld gradients", name, (long long)out->count,
                (long long)g->count);
    for (int64_t i = 0; i < g->count; ++i)
      GTK_REQUIRE(out->numel[i] == g->numel[i], GTK_EINVAL, "%s: output %lld has another size", name, (long long)i);
  }
  return check_overlap(g, out, name);
}

}  // namespace gtk

using namespace gtk;

#define GTK_NORM_CHECK(name)                                                                                        \
  int rc;                                                                                                           \
  if ((rc = check_list(grads, name))) return rc;                                                                    \
  GTK_REQUIRE(kind == GTK_NORM_2 || kind == GTK_NORM_1 || kind == GTK_NORM_INF, GTK_EINVAL, name ": bad norm %d",   \
              kind);                                                                                                \
  GTK_REQUIRE(norm && workspace, GTK_EINVAL, name ": null pointer");                                                \
  const size_t need = gtk_grad_norm_workspace_size(grads);                                                          \
  GTK_REQUIRE(workspace_bytes >= need, GTK_EWORKSPACE, name ": workspace %zu < %zu bytes", workspace_bytes, need);  \
  GTK_REQUIRE(((uintptr_t)workspace & 7) == 0, GTK_EINVAL, name ": workspace not aligned to 8 bytes");              \
  hipStream_t st = (hipStream_t)stream

extern "C" size_t gtk_grad_norm_workspace_size(const gtk_tensor_list* grads) {
  if (check_list(grads, "gtk_grad_norm_workspace_size")) return 0;
  return sizeof(double) * (size_t)std::max<int64_t>(1, most_blocks(grads, chunk_of(grads, kNormChunk)));
}

extern "C" int gtk_grad_norm(const gtk_tensor_list* grads, int kind, float* norm, void* workspace,
                             size_t workspace_bytes, void* stream) {
  GTK_NORM_CHECK("gtk_grad_norm");
  return launch_norm(kind, grads, norm, (double*)workspace, st);
}

extern "C" int gtk_grad_clip(const gtk_tensor_list* grads, const gtk_tensor_list* out, int kind, double max_norm,
                             float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  GTK_NORM_CHECK("gtk_grad_clip");
  GTK_REQUIRE(max_norm >= 0.0, GTK_EINVAL, "gtk_grad_clip: max_norm %g is negative or not a number", max_norm);
  if ((rc = check_out(grads, out, "gtk_grad_clip"))) return rc;
  if ((rc = launch_norm(kind, grads, norm, (double*)workspace, st))) return rc;
  return launch_scale(grads, out, max_norm, norm, st);
}

extern "C" int gtk_grad_clip_with_norm(const gtk_tensor_list* grads, const gtk_tensor_list* out, double max_norm,
                                       const float* norm, void* stream) {
  int rc;
  if ((rc = check_list(grads, "gtk_grad_clip_with_norm"))) return rc;
  GTK_REQUIRE(norm, GTK_EINVAL, "gtk_grad_clip_with_norm: null pointer");
  GTK_REQUIRE(max_norm >= 0.0, GTK_EINVAL, "gtk_grad_clip_with_norm: max_norm %g is negative or not a number", max_norm);
  if ((rc = check_out(grads, out, "gtk_grad_clip_with_norm"))) return rc;
  return launch_scale(grads, out, max_norm, norm, (hipStream_t)stream);
}
