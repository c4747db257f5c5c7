// The closing launch of a normalisation's parameter gradients: column sums over the
// partial sums that the backward pass' blocks leave, part[block][weight, bias][D].
#pragma once
#include "capi_util.hpp"
#include "common.hpp"

namespace gtk {

struct ColumnSums {
  const float* part;
  int parts, D;
  void *dw, *db;
  int dst_bf;
};

// dst[c] = sum over the partials (c < D: the weight's, else the bias'): the block'th
// OUTS of the 2 D sums, by CHUNKS threads each, eight loads in flight; red:
// OUTS * CHUNKS floats.
template <int OUTS, int CHUNKS>
__device__ __forceinline__ void close_columns(const ColumnSums& s, int block, float* red) {
  const int o = threadIdx.x % OUTS, ch = threadIdx.x / OUTS;
  const int64_t i = (int64_t)block * OUTS + o, n = 2 * (int64_t)s.D;
  void* dst = i < s.D ? s.dw : s.db;
  const bool live = i < n && dst;
  float a[8] = {};
  if (live)
    for (int k = ch; k < s.parts; k += 8 * CHUNKS)
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int ku = k + u * CHUNKS;
        const float v = s.part[(ku < s.parts ? ku : s.parts - 1) * n + i];
        a[u] += ku < s.parts ? v : 0.f;
      }
  red[ch * OUTS + o] = ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
  // in pairs
#pragma unroll
  for (int w = CHUNKS / 2; w > 0; w /= 2) {
    __syncthreads();
    if (ch < w) red[ch * OUTS + o] += red[(ch + w) * OUTS + o];
  }
  if (ch != 0 || !live) return;
  const int c = (int)(i < s.D ? i : i - s.D);
  if (s.dst_bf)
    ((bf16*)dst)[c] = cvt<bf16>(red[o]);
  else
    ((float*)dst)[c] = red[o];
}

template <int OUTS, int CHUNKS> __global__ __launch_bounds__(OUTS * CHUNKS) void column_close_kernel(ColumnSums s) {
  __shared__ float red[OUTS * CHUNKS];
  close_columns<OUTS, CHUNKS>(s, blockIdx.x, red);
}

inline int launch_column_close(const char* name, const float* part, int parts, int D, void* dw, void* db, int dst_bf,
                               hipStream_t st) {
  StageTimer timer(name, st);
  // narrow rows leave few sums, and many partials of each: more threads a sum
  // (LayerNorm's backward, 2^18 rows of 128: 40.5 us against 44.2 with 32 x 32; 2048
  // rows of 8192: 34.0 against 31.4)
  if (D <= 512)
    column_close_kernel<16, 64><<<(2 * D + 15) / 16, 1024, 0, st>>>(ColumnSums{part, parts, D, dw, db, dst_bf});
  else
    column_close_kernel<32, 32><<<(2 * D + 31) / 32, 1024, 0, st>>>(ColumnSums{part, parts, D, dw, db, dst_bf});
  GTK_LAUNCH_CHECK();
  return GTK_OK;
}

}  // namespace gtk
