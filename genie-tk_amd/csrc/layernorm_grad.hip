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

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// One wave per row, three sweeps.
template <typename T>
__global__ __launch_bounds__(256) void ln_forward_kernel(const T* __restrict__ x, int64_t xs, T* __restrict__ y,
                                                         ParamVec w, ParamVec b, int64_t rows, int D, float eps) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + wave_id(); r < rows; r += (int64_t)gridDim.x * 4) {
    const T* xr = x + r * xs;
    float s = 0.f, q = 0.f;
    for (int c = lane; c < D; c += 64) s += to_f32(xr[c]);
    const float mean = wave_sum(s) / (float)D;
    for (int c = lane; c < D; c += 64) {
      const float d = to_f32(xr[c]) - mean;
      q += d * d;
    }
    const float rstd = 1.0f / sqrtf(wave_sum(q) / (float)D + eps);
    for (int c = lane; c < D; c += 64)
      y[r * D + c] = cvt<T>((to_f32(xr[c]) - mean) * rstd * w.get(c, 1.f) + b.get(c, 0.f));
  }
}

// One wave per row: dx, and the row's mean and rstd for the column sums.
template <typename T>
__global__ __launch_bounds__(256) void ln_backward_rows_kernel(const T* __restrict__ x, int64_t xs,
                                                               const T* __restrict__ dy, int64_t ds,
                                                               T* __restrict__ dx, ParamVec w, float2* __restrict__ stats,
                                                               int64_t rows, int D, float eps) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + wave_id(); r < rows; r += (int64_t)gridDim.x * 4) {
    const T* xr = x + r * xs;
    const T* dr = dy + r * ds;
    float s = 0.f, q = 0.f, s1 = 0.f, s2 = 0.f;
    for (int c = lane; c < D; c += 64) s += to_f32(xr[c]);
    const float mean = wave_sum(s) / (float)D;
    for (int c = lane; c < D; c += 64) {
      const float d = to_f32(xr[c]) - mean;
      const float g = to_f32(dr[c]) * w.get(c, 1.f);
      q += d * d;
      s1 += g;
      s2 += g * d;
    }
    const float rstd = 1.0f / sqrtf(wave_sum(q) / (float)D + eps);
    const float c1 = wave_sum(s1) / (float)D, c2 = wave_sum(s2) / (float)D * rstd;
    if (dx)
      for (int c = lane; c < D; c += 64) {
        const float h = (to_f32(xr[c]) - mean) * rstd;
        dx[r * D + c] = cvt<T>((to_f32(dr[c]) * w.get(c, 1.f) - c1 - h * c2) * rstd);
      }
    if (stats && lane == 0) stats[r] = float2{mean, rstd};
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
      aw += g * ((to_f32(x[r * xs + c]) - st.x) * st.y);
      ab += g;
    }
  red[0][wave][lane] = aw;
  red[1][wave][lane] = ab;
  __syncthreads();
  if (wave < 2 && c < D)
    part[((int64_t)blockIdx.y * 2 + wave) * D + c] =
        (red[wave][0][lane] + red[wave][1][lane]) + (red[wave][2][lane] + red[wave][3][lane]);
}

// dst[c] = sum of the splits' partials (blockIdx.y: 0 the weight's, 1 the bias').
__global__ __launch_bounds__(256) void ln_close_kernel(const float* __restrict__ part, int splits, int D,
                                                       void* __restrict__ dw, void* __restrict__ db, int dst_bf) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  void* dst = blockIdx.y ? db : dw;
  if (c >= D || !dst) return;
  float s = 0.f;
  for (int k = 0; k < splits; ++k) s += part[((int64_t)k * 2 + blockIdx.y) * D + c];
  if (dst_bf)
    ((bf16*)dst)[c] = cvt<bf16>(s);
  else
    ((float*)dst)[c] = s;
}

static int column_splits(int64_t rows) { return (int)std::min<int64_t>(256, std::max<int64_t>(1, (rows + 15) / 16)); }

static unsigned row_blocks(int64_t rows) { return (unsigned)std::min<int64_t>((rows + 3) / 4, 1 << 16); }

static int launch_ln_close(const float* part, int splits, int D, void* dw, void* db, int dst_bf, hipStream_t st) {
  StageTimer timer("layer_norm_close", st);
  ln_close_kernel<<<dim3((D + 255) / 256, 2), 256, 0, st>>>(part, splits, D, dw, db, dst_bf);
  GTK_LAUNCH_CHECK();
  return GTK_OK;
}

template <typename T>
static int launch_ln_backward(const T* x, int64_t xs, const T* dy, int64_t ds, T* dx, ParamVec w, void* dw, void* db,
                              int dst_bf, int64_t rows, int D, float eps, float2* stats, float* part, hipStream_t st) {
  {
    StageTimer timer("layer_norm_backward", st);
    ln_backward_rows_kernel<T><<<row_blocks(rows), 256, 0, st>>>(x, xs, dy, ds, dx, w, stats, rows, D, eps);
    GTK_LAUNCH_CHECK();
  }
  if (!dw && !db) return GTK_OK;
  const int splits = column_splits(rows);
  {
    StageTimer timer("layer_norm_columns", st);
    ln_columns_kernel<T><<<dim3((D + 63) / 64, splits), 256, 0, st>>>(x, xs, dy, ds, stats, part, rows, D);
    GTK_LAUNCH_CHECK();
  }
  return launch_ln_close(part, splits, D, dw, db, dst_bf, st);
}

static void carve_ln_backward(Carve& cv, int64_t rows, int64_t d, float2** stats, float** part) {
  *stats = cv.take<float2>(rows);
  *part = cv.take<float>(2 * d * column_splits(rows));
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
  StageTimer timer("layer_norm_forward", st);
  if (dtype == GTK_F32)
    ln_forward_kernel<float><<<row_blocks(rows), 256, 0, st>>>((const float*)x, x_stride, (float*)y, w, b, rows, (int)d, eps);
  else
    ln_forward_kernel<bf16><<<row_blocks(rows), 256, 0, st>>>((const bf16*)x, x_stride, (bf16*)y, w, b, rows, (int)d, eps);
  GTK_LAUNCH_CHECK();
  return GTK_OK;
}

extern "C" size_t gtk_layer_norm_backward_workspace_size(int64_t rows, int64_t d, int dtype) {
  if (rows < 0 || rows > (int64_t)1 << 40 || d < 1 || d > 1 << 24 || (dtype != GTK_F32 && dtype != GTK_BF16)) return 0;
  Carve cv(nullptr, SIZE_MAX);
  float2* stats;
  float* part;
  carve_ln_backward(cv, rows, d, &stats, &part);
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
  Carve cv(workspace, workspace_bytes);
  float2* stats;
  float* part;
  carve_ln_backward(cv, rows, d, &stats, &part);
  if (dtype == GTK_F32)
    return launch_ln_backward<float>((const float*)x, x_stride, (const float*)dy, dy_stride, (float*)dx, w, dweight,
                                     dbias, pbf, rows, (int)d, eps, stats, part, st);
  return launch_ln_backward<bf16>((const bf16*)x, x_stride, (const bf16*)dy, dy_stride, (bf16*)dx, w, dweight, dbias,
                                  pbf, rows, (int)d, eps, stats, part, st);
}
