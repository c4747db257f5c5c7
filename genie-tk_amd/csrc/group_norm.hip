// Group norm with an activation over channels-last tensors, for gfx950.
//
// Over the m values of a sample's group that count (mask not 0): mean, var =
// mean(d^2) with d = x - mean, r = 1 / sqrt(var + eps), h = d r, z = h w + b and
// y = act(z).  Backward, with dz = dy act'(z) and g = dz w:
//   dx = r (g - mean(g) - h mean(g h)),  dw = sum dz h,  db = sum dz
// The statistics are sums of x and x^2 in 64 bits: a product of two 32-bit values
// is exact there, so far from zero as a value lies, the variance loses nothing
// that matters.  The mean is kept as a sum of two floats, so that d is off by its
// own rounding only.
#include <math.h>

#include <algorithm>

#include "capi_util.hpp"
#include "common.hpp"
#include "pack.hpp"

namespace gtk {

// One sample's group, as gtk_group_norm_forward writes it.
struct GroupStats {
  float mean, low, rstd, inv;
};

__device__ __forceinline__ GroupStats close_stats(double s, double q, double count, float eps) {
  GroupStats g{0.f, 0.f, 0.f, 0.f};
  if (count > 0) {
    const double mean = s / count, var = fmax(q / count - mean * mean, 0.0);
    g.mean = (float)mean;
    g.low = (float)(mean - (double)g.mean);
    g.rstd = (float)(1.0 / sqrt(var + (double)eps));
    g.inv = (float)(1.0 / count);
  }
  return g;
}

// The value of the standard normal distribution's function and density at z.
__device__ __forceinline__ float normal_below(float z, float& density) {
  density = 0.3989422804f * expf(-0.5f * z * z);
  return 0.5f * erfcf(-0.70710678f * z);
}

__device__ __forceinline__ float activate(float z, int act) {
  float density;
  if (act == GTK_ACT_SILU) return z * sigmoidf_(z);
  if (act == GTK_ACT_GELU) return z * normal_below(z, density);
  return z;
}
__device__ __forceinline__ float activate_slope(float z, int act) {
  if (act == GTK_ACT_SILU) {
    const float s = sigmoidf_(z);
    return s * (1.f + z * (1.f - s));
  }
  if (act == GTK_ACT_GELU) {
    float density;
    const float below = normal_below(z, density);
    return below + z * density;
  }
  return 1.f;
}

struct ParamVector {
  const void* p;
  int bf;
  __device__ __forceinline__ float get(int64_t c, float none) const {
    if (!p) return none;
    return bf ? to_f32(((const bf16*)p)[c]) : ((const float*)p)[c];
  }
};

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

// A block a sample's group.
template <typename T>
__global__ __launch_bounds__(256) void gn_forward_kernel(const T* __restrict__ x, int64_t xs,
                                                         const float* __restrict__ mask, T* __restrict__ y,
                                                         GroupStats* __restrict__ stats, ParamVector w, ParamVector b,
                                                         int64_t P, int64_t C, int64_t G, float eps, int act) {
  __shared__ double red[3][4];
  const int64_t bg = blockIdx.x, n = bg / G, cg = C / G, c0 = bg % G * cg;
  double v[3] = {0, 0, 0};
  for (int64_t i = threadIdx.x; i < P * cg; i += 256) {
    const int64_t row = n * P + i / cg;
    if (mask && mask[row] == 0.f) continue;
    const double f = to_f32(x[row * xs + c0 + i % cg]);
    v[0] += f;
    v[1] += f * f;
    v[2] += 1;
  }
  block_add(v, red);
  const GroupStats g = close_stats(v[0], v[1], v[2], eps);
  if (threadIdx.x == 0) stats[bg] = g;
  for (int64_t i = threadIdx.x; i < P * cg; i += 256) {
    const int64_t row = n * P + i / cg, c = c0 + i % cg;
    const bool live = !mask || mask[row] != 0.f;
    const float h = ((to_f32(x[row * xs + c]) - g.mean) - g.low) * g.rstd;
    y[row * C + c] = cvt<T>(live ? activate(h * w.get(c, 1.f) + b.get(c, 0.f), act) : 0.f);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void gn_backward_kernel(const T* __restrict__ x, int64_t xs,
                                                          const float* __restrict__ mask, const T* __restrict__ dy,
                                                          int64_t ds, const GroupStats* __restrict__ stats,
                                                          ParamVector w, ParamVector b, T* __restrict__ dx, int64_t P,
                                                          int64_t C, int64_t G, int act) {
  __shared__ double red[3][4];
  const int64_t bg = blockIdx.x, n = bg / G, cg = C / G, c0 = bg % G * cg;
  const GroupStats st = stats[bg];
  auto at = [&](int64_t i, float& h, float& g) {
    const int64_t row = n * P + i / cg, c = c0 + i % cg;
    h = g = 0.f;
    if (mask && mask[row] == 0.f) return false;
    h = ((to_f32(x[row * xs + c]) - st.mean) - st.low) * st.rstd;
    g = to_f32(dy[row * ds + c]) * activate_slope(h * w.get(c, 1.f) + b.get(c, 0.f), act) * w.get(c, 1.f);
    return true;
  };
  double v[3] = {0, 0, 0};
  float h, g;
  for (int64_t i = threadIdx.x; i < P * cg; i += 256) {
    at(i, h, g);
    v[0] += g;
    v[1] += (double)g * h;
  }
  block_add(v, red);
  const float c1 = (float)(v[0] * st.inv), c2 = (float)(v[1] * st.inv);
  for (int64_t i = threadIdx.x; i < P * cg; i += 256) {
    const bool live = at(i, h, g);
    dx[(n * P + i / cg) * C + c0 + i % cg] = cvt<T>(live ? (g - c1 - h * c2) * st.rstd : 0.f);
  }
}

// A block a channel.
template <typename T>
__global__ __launch_bounds__(256) void gn_params_kernel(const T* __restrict__ x, int64_t xs,
                                                        const float* __restrict__ mask, const T* __restrict__ dy,
                                                        int64_t ds, const GroupStats* __restrict__ stats, ParamVector w,
                                                        ParamVector b, void* __restrict__ dw, void* __restrict__ db,
                                                        int dst_bf, int64_t B, int64_t P, int64_t C, int64_t G,
                                                        int act) {
  __shared__ double red[3][4];
  const int64_t c = blockIdx.x;
  double v[3] = {0, 0, 0};
  for (int64_t row = threadIdx.x; row < B * P; row += 256) {
    if (mask && mask[row] == 0.f) continue;
    const GroupStats st = stats[row / P * G + c / (C / G)];
    const float h = ((to_f32(x[row * xs + c]) - st.mean) - st.low) * st.rstd;
    const float dz = to_f32(dy[row * ds + c]) * activate_slope(h * w.get(c, 1.f) + b.get(c, 0.f), act);
    v[0] += (double)dz * h;
    v[1] += dz;
  }
  block_add(v, red);
  if (threadIdx.x) return;
  for (int k = 0; k < 2; ++k) {
    void* dst = k ? db : dw;
    if (!dst) continue;
    if (dst_bf)
      ((bf16*)dst)[c] = (bf16)(float)v[k];
    else
      ((float*)dst)[c] = (float)v[k];
  }
}

static bool gn_shape_ok(int64_t B, int64_t P, int64_t C, int64_t G, int dtype) {
  const int64_t most = (int64_t)1 << 48;
  return B >= 0 && P >= 1 && C >= 1 && C <= 1 << 24 && G >= 1 && G <= C && C % G == 0 && P <= most / C &&
         B <= most / (P * C) && (dtype == GTK_F32 || dtype == GTK_BF16);
}

template <typename T>
static int launch_gn_forward(const void* x, int64_t xs, const float* mask, void* y, float* stats, ParamVector w,
                             ParamVector b, int64_t B, int64_t P, int64_t C, int64_t G, float eps, int act,
                             hipStream_t st) {
  StageTimer timer("group_norm_forward", st);
  gn_forward_kernel<T><<<(unsigned)(B * G), 256, 0, st>>>((const T*)x, xs, mask, (T*)y, (GroupStats*)stats, w, b, P, C,
                                                          G, eps, act);
  GTK_LAUNCH_CHECK();
  return GTK_OK;
}

template <typename T>
static int launch_gn_backward(const void* x, int64_t xs, const float* mask, const void* dy, int64_t ds,
                              const float* stats, ParamVector w, ParamVector b, void* dx, void* dw, void* db, int pbf,
                              int64_t B, int64_t P, int64_t C, int64_t G, int act, hipStream_t st) {
  if (dx && B) {
    StageTimer timer("group_norm_backward", st);
    gn_backward_kernel<T><<<(unsigned)(B * G), 256, 0, st>>>((const T*)x, xs, mask, (const T*)dy, ds,
                                                             (const GroupStats*)stats, w, b, (T*)dx, P, C, G, act);
    GTK_LAUNCH_CHECK();
  }
  if (dw || db) {
    StageTimer timer("group_norm_params", st);
    gn_params_kernel<T><<<(unsigned)C, 256, 0, st>>>((const T*)x, xs, mask, (const T*)dy, ds, (const GroupStats*)stats,
                                                     w, b, dw, db, pbf, B, P, C, G, act);
    GTK_LAUNCH_CHECK();
  }
  return GTK_OK;
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
  return 0;
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
  const ParamVector w{weight, param_dtype == GTK_BF16}, b{bias, param_dtype == GTK_BF16};
  return (dtype == GTK_F32 ? launch_gn_forward<float> : launch_gn_forward<bf16>)(
      x, x_stride, mask, y, stats, w, b, B, positions, c, groups, eps, activation, (hipStream_t)stream);
}

extern "C" size_t gtk_group_norm_backward_workspace_size(int64_t B, int64_t positions, int64_t c, int64_t groups,
                                                         int dtype) {
  return 0;
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
  const ParamVector w{weight, param_dtype == GTK_BF16}, b{bias, param_dtype == GTK_BF16};
  return (dtype == GTK_F32 ? launch_gn_backward<float> : launch_gn_backward<bf16>)(
      x, x_stride, mask, dy, dy_stride, stats, w, b, dx, dweight, dbias, param_dtype == GTK_BF16, B, positions, c,
      groups, activation, (hipStream_t)stream);
}
