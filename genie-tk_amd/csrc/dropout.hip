// Dropout with a counter-based generator, for gfx950: the mask is a function of
// (seed, offset, place), computed where it is used, in the backward pass again.
#include <math.h>

#include "capi_util.hpp"
#include "common.hpp"

namespace gtk {

// Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers:
// as easy as 1, 2, 3", SC 2011): ten rounds of two 32 x 32 -> 64 bit products over
// a 128-bit counter, under a 64-bit key that a Weyl sequence changes each round.
struct Philox {
  uint32_t w[4];
  __device__ __forceinline__ Philox(uint64_t at, uint64_t offset, uint64_t key) {
    uint32_t c0 = (uint32_t)at, c1 = (uint32_t)(at >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
      c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
      c1 = (uint32_t)p1;
      c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
      c3 = (uint32_t)p0;
      k0 += 0x9E3779B9u;
      k1 += 0xBB67AE85u;
    }
    w[0] = c0;
    w[1] = c1;
    w[2] = c2;
    w[3] = c3;
  }
};

template <typename TX, typename TR, typename TO>
__global__ __launch_bounds__(256) void dropout_kernel(const TX* __restrict__ x, const TR* __restrict__ residual,
                                                      TO* __restrict__ out, int64_t shared, int64_t inner, int64_t n,
                                                      uint32_t t, float scale, uint64_t seed,
                                                      const uint64_t* __restrict__ seed_device, uint64_t offset) {
  const uint64_t key = seed_device ? *seed_device : seed;
  const int64_t blocks = (inner + 7) / 8;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i % inner, o = i / inner / shared;
    const Philox ph(o * blocks + r / 8, offset, key);
    const uint32_t bits = ph.w[r % 8 / 2] >> (r % 2 * 16) & 0xffff;
    const float base = residual ? to_f32(residual[i]) : 0.f;
    out[i] = cvt<TO>(bits >= t ? fmaf(to_f32(x[i]), scale, base) : base);
  }
}

template <typename TX, typename TR, typename TO>
static int launch_dropout(const void* x, const void* residual, void* out, int64_t outer, int64_t shared, int64_t inner,
                          uint32_t t, float scale, uint64_t seed, const uint64_t* seed_device, uint64_t offset,
                          hipStream_t st) {
  StageTimer timer("dropout", st);
  const int64_t n = outer * shared * inner;
  dropout_kernel<TX, TR, TO><<<(unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20), 256, 0, st>>>(
      (const TX*)x, (const TR*)residual, (TO*)out, shared, inner, n, t, scale, seed, seed_device, offset);
  GTK_LAUNCH_CHECK();
  return GTK_OK;
}

}  // namespace gtk

using namespace gtk;

// a * b for a, b >= 0, or -1 past 2^48.
static int64_t times(int64_t a, int64_t b) {
  return a < 0 || b < 0 || (b && a > ((int64_t)1 << 48) / b) ? -1 : a * b;
}

extern "C" int gtk_dropout(const void* x, int dtype, const void* residual, int residual_dtype, void* out, int out_dtype,
                           int64_t outer, int64_t shared, int64_t inner, double p, uint64_t seed,
                           const uint64_t* seed_device, uint64_t offset, void* stream) {
  auto known = [](int d) { return d == GTK_F32 || d == GTK_BF16; };
  GTK_REQUIRE(known(dtype) && known(out_dtype), GTK_EINVAL, "gtk_dropout: bad dtype %d -> %d", dtype, out_dtype);
  GTK_REQUIRE(!residual || (residual_dtype == out_dtype && (dtype == out_dtype || dtype == GTK_BF16)), GTK_EINVAL,
              "gtk_dropout: types (%d, %d) -> %d", dtype, residual_dtype, out_dtype);
  GTK_REQUIRE(p >= 0.0 && p <= 1.0, GTK_EINVAL, "gtk_dropout: p=%g not in [0, 1]", p);
  GTK_REQUIRE(outer >= 0 && shared >= 0 && inner >= 0 && inner <= (int64_t)1 << 48 &&
                  times(times(outer, shared), inner) >= 0 && times(outer, (inner + 7) / 8 * 8) >= 0,
              GTK_EINVAL, "gtk_dropout: bad shape [%lld][%lld][%lld]", (long long)outer, (long long)shared,
              (long long)inner);
  if (outer == 0 || shared == 0 || inner == 0) return GTK_OK;
  GTK_REQUIRE(x && out, GTK_EINVAL, "gtk_dropout: null pointer");
  const uint32_t t = (uint32_t)nearbyint(65536.0 * p);
  const float scale = t < 65536 ? 65536.0f / (float)(65536 - t) : 0.f;
  hipStream_t st = (hipStream_t)stream;
  auto run = [&](auto tx, auto tr, auto to) {
    return launch_dropout<decltype(tx), decltype(tr), decltype(to)>(x, residual, out, outer, shared, inner, t, scale,
                                                                    seed, seed_device, offset, st);
  };
  if (out_dtype == GTK_BF16) return dtype == GTK_BF16 ? run(bf16(), bf16(), bf16()) : run(float(), bf16(), bf16());
  return dtype == GTK_BF16 ? run(bf16(), float(), float()) : run(float(), float(), float());
}
