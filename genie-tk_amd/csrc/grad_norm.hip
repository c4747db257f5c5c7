// The global norm of a set of gradients, and clipping by it, for gfx950.
//
//   n = (sum |g|^p)^(1/p) over every value of every tensor, p in {1, 2, inf}
//   k = min(1, max_norm / (n + 1e-6)),  out = k g
//
// The values' squares and their sums are 64-bit: the square of a 32-bit float
// fits a 64-bit one exactly, so neither gradients above 1.8e19 overflow nor
// ones below 1e-23 vanish.  The tensors' addresses and sizes travel in the
// kernel arguments, kMaxTensors a launch: no table is copied to the GPU, and a
// captured launch keeps them.  Every block writes one partial sum and one
// block adds them in a fixed order, so equal inputs give equal bits.
#include <algorithm>
#include <memory>
#include <new>

#include "capi_util.hpp"
#include "common.hpp"
#include "pack.hpp"

namespace gtk {

constexpr int kMaxTensors = 100;
struct NormJobs {
  const void* src[kMaxTensors];
  void* dst[kMaxTensors];
  int64_t n[kMaxTensors];
  int first[kMaxTensors + 1];  // first block of each tensor
  uint8_t src_bf[kMaxTensors], dst_bf[kMaxTensors];
  int count;
  int64_t chunk;  // values a block
};
static_assert(sizeof(NormJobs) <= 4000, "kernel arguments");

__device__ __forceinline__ float grad_at(const void* p, int bf, int64_t i) {
  return bf ? to_f32(((const bf16*)p)[i]) : ((const float*)p)[i];
}

// The tensor of this block, and its range of values.
__device__ __forceinline__ int find_job(const NormJobs& J, int64_t& begin, int64_t& end) {
  int k = 0;
  while (k + 1 < J.count && (int)blockIdx.x >= J.first[k + 1]) ++k;
  begin = (int64_t)((int)blockIdx.x - J.first[k]) * J.chunk;
  end = begin + J.chunk < J.n[k] ? begin + J.chunk : J.n[k];
  return k;
}

// The largest |g| is found on the bits: the order of non-negative floats is
// that of their bits, infinity and NaN (the largest) included.
template <int KIND>
__device__ __forceinline__ double block_join(double s, double* red) {
  const int waves = blockDim.x >> 6;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const double o = __shfl_xor(s, off, 64);
    if (KIND == GTK_NORM_INF) {
      const uint64_t a = __builtin_bit_cast(uint64_t, s), b = __builtin_bit_cast(uint64_t, o);
      s = __builtin_bit_cast(double, a > b ? a : b);
    } else {
      s += o;
    }
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  s = red[0];
  for (int w = 1; w < waves; ++w) {
    if (KIND == GTK_NORM_INF) {
      const uint64_t a = __builtin_bit_cast(uint64_t, s), b = __builtin_bit_cast(uint64_t, red[w]);
      s = __builtin_bit_cast(double, a > b ? a : b);
    } else {
      s += red[w];
    }
  }
  return s;
}

template <int KIND>
__global__ __launch_bounds__(256) void grad_partials_kernel(NormJobs J, double* __restrict__ part) {
  __shared__ double red[4];
  int64_t begin, end;
  const int k = find_job(J, begin, end);
  double s = 0.0;
  uint32_t m = 0;
  for (int64_t i = begin + threadIdx.x; i < end; i += 256) {
    const float v = grad_at(J.src[k], J.src_bf[k], i);
    if (KIND == GTK_NORM_2) s += (double)v * (double)v;
    if (KIND == GTK_NORM_1) s += (double)fabsf(v);
    if (KIND == GTK_NORM_INF) {
      const uint32_t a = __float_as_uint(v) & 0x7fffffffu;
      m = a > m ? a : m;
    }
  }
  if (KIND == GTK_NORM_INF) s = __builtin_bit_cast(double, (uint64_t)m);
  s = block_join<KIND>(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <int KIND>
__global__ __launch_bounds__(1024) void grad_norm_close_kernel(const double* __restrict__ part, int64_t parts,
                                                               float* __restrict__ norm) {
  __shared__ double red[16];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < parts; i += 1024) {
    if (KIND == GTK_NORM_INF) {
      const uint64_t a = __builtin_bit_cast(uint64_t, s), b = __builtin_bit_cast(uint64_t, part[i]);
      s = __builtin_bit_cast(double, a > b ? a : b);
    } else {
      s += part[i];
    }
  }
  s = block_join<KIND>(s, red);
  if (threadIdx.x == 0) {
    if (KIND == GTK_NORM_2) s = sqrt(s);
    *norm = KIND == GTK_NORM_INF ? __uint_as_float((uint32_t)__builtin_bit_cast(uint64_t, s)) : (float)s;
  }
}

// The factor of the clipping, one rounding to 32 bits.  A norm of NaN makes it
// NaN, an infinite one 0.
__device__ __forceinline__ float clip_factor(float norm, double max_norm) {
  const double f = max_norm / ((double)norm + 1e-6);
  return f > 1.0 ? 1.f : (float)f;
}

__global__ __launch_bounds__(256) void grad_scale_kernel(NormJobs J, const float* __restrict__ norm, double max_norm) {
  int64_t begin, end;
  const int k = find_job(J, begin, end);
  const float f = clip_factor(*norm, max_norm);
  for (int64_t i = begin + threadIdx.x; i < end; i += 256) {
    const float v = grad_at(J.src[k], J.src_bf[k], i) * f;
    if (J.dst_bf[k])
      ((bf16*)J.dst[k])[i] = cvt<bf16>(v);
    else
      ((float*)J.dst[k])[i] = v;
  }
}

constexpr int64_t kChunk = 8192;

static int64_t total_blocks(const gtk_tensor_list* g) {
  int64_t b = 0;
  for (int64_t i = 0; i < g->count; ++i) b += (g->numel[i] + kChunk - 1) / kChunk;
  return b;
}

// Calls launch(jobs, blocks, first partial) for every kMaxTensors tensors.
template <typename F>
static int for_each_launch(const gtk_tensor_list* g, const gtk_tensor_list* out, F launch) {
  NormJobs J;
  J.chunk = kChunk;
  J.count = 0;
  J.first[0] = 0;
  int64_t base = 0;
  auto flush = [&]() -> int {
    if (J.count == 0) return GTK_OK;
    const int rc = launch(J, (unsigned)J.first[J.count], base);
    base += J.first[J.count];
    J.count = 0;
    return rc;
  };
  for (int64_t i = 0; i < g->count; ++i) {
    // a large tensor takes several entries: block counts stay in 32 bits
    for (int64_t at = 0; at < g->numel[i];) {
      const int64_t n = std::min<int64_t>(g->numel[i] - at, kChunk << 16);
      const int k = J.count++;
      const int64_t sb = g->dtype[i] == GTK_BF16 ? 2 : 4;
      J.src[k] = (const char*)g->data[i] + at * sb;
      J.src_bf[k] = g->dtype[i] == GTK_BF16;
      const gtk_tensor_list* o = out ? out : g;
      J.dst[k] = (char*)o->data[i] + at * (o->dtype[i] == GTK_BF16 ? 2 : 4);
      J.dst_bf[k] = o->dtype[i] == GTK_BF16;
      J.n[k] = n;
      J.first[k + 1] = J.first[k] + (int)((n + kChunk - 1) / kChunk);
      at += n;
      if (J.count == kMaxTensors) {
        const int rc = flush();
        if (rc) return rc;
      }
    }
  }
  return flush();
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
  bool written;
};

// Nothing that is written is written twice or read by another tensor's block:
// blocks run in any order.
static int check_overlap(const gtk_tensor_list* g, const gtk_tensor_list* out, const char* name) {
  const gtk_tensor_list* o = out ? out : g;
  const std::unique_ptr<Span[]> v(new (std::nothrow) Span[2 * (size_t)g->count + 1]);
  GTK_REQUIRE(v, GTK_EINVAL, "%s: out of host memory", name);
  int64_t spans = 0;
  bool sorted = true;
  auto add = [&](const gtk_tensor_list* l, int64_t i, bool written) {
    if (l->numel[i] == 0) return;
    const char* p = (const char*)l->data[i];
    if (spans && p < v[spans - 1].begin) sorted = false;
    v[spans++] = {p, p + l->numel[i] * (int64_t)dtype_size(l->dtype[i]), written};
  };
  for (int64_t i = 0; i < g->count; ++i) add(o, i, true);
  for (int64_t i = 0; out && i < g->count; ++i)
    // a tensor clipped onto itself is read and written by the same thread
    if (!(out->data[i] == g->data[i] && out->dtype[i] == g->dtype[i])) add(g, i, false);
  if (!sorted) std::sort(v.get(), v.get() + spans, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  const char *any = nullptr, *written = nullptr;  // the furthest ends so far
  for (int64_t i = 0; i < spans; ++i) {
    const Span& s = v[i];
    GTK_REQUIRE(s.begin >= written && (!s.written || s.begin >= any), GTK_EINVAL,
                "%s: a tensor that is written overlaps another (or is given twice)", name);
    any = std::max(any, s.end);
    if (s.written) written = std::max(written, s.end);
  }
  return GTK_OK;
}

template <int KIND>
static int launch_norm(const gtk_tensor_list* g, float* norm, double* part, hipStream_t st) {
  {
    StageTimer timer("grad_partials", st);
    const int rc = for_each_launch(g, nullptr, [&](const NormJobs& J, unsigned blocks, int64_t base) -> int {
      grad_partials_kernel<KIND><<<blocks, 256, 0, st>>>(J, part + base);
      GTK_LAUNCH_CHECK();
      return GTK_OK;
    });
    if (rc) return rc;
  }
  StageTimer timer("grad_norm_close", st);
  grad_norm_close_kernel<KIND><<<1, 1024, 0, st>>>(part, total_blocks(g), norm);
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

static int launch_scale(const gtk_tensor_list* g, const gtk_tensor_list* out, double max_norm, const float* norm,
                        hipStream_t st) {
  StageTimer timer("grad_scale", st);
  return for_each_launch(g, out, [&](const NormJobs& J, unsigned blocks, int64_t) -> int {
    grad_scale_kernel<<<blocks, 256, 0, st>>>(J, norm, max_norm);
    GTK_LAUNCH_CHECK();
    return GTK_OK;
  });
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
  return sizeof(double) * (size_t)std::max<int64_t>(1, total_blocks(grads));
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
