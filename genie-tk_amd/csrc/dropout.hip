// Dropout with a counter-based generator, for gfx950: the mask is a function of
// (seed, offset, place), computed where it is used, and in the backward pass again.
//
// One evaluation of the generator decides eight values (16 bits each, one unit);
// it is some 130 instructions, 20 of them wide products at a quarter of the rate.
// A value of its own mask therefore costs some 25 issue slots, and a bf16 one moves
// 4 bytes: at 6 TB/s the arithmetic takes about as long as the memory, and both
// overlap as long as loads are on their way while a unit is drawn.  Under a mask
// that is shared along a dimension each thread draws its unit once and walks that
// dimension: memory bounds it.
#include <math.h>

#include "capi_util.hpp"
#include "common.hpp"
#include "row_vec.hpp"

namespace gtk {

struct Key {
  uint64_t seed, offset;
  uint32_t below, live;  // a value is kept if its 16 bits, as the upper half of a word, are not below

  // t of 65536 are dropped
  static Key of(uint64_t seed, uint64_t offset, uint32_t t) {
    return t < 65536 ? Key{seed, offset, t << 16, ~0u} : Key{seed, offset, 1u, 0u};
  }
};

// Which of a unit's eight values are kept.
struct Keep {
  bool k[8];

  // Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers:
  // as easy as 1, 2, 3", SC 2011): ten rounds of two 32 x 32 -> 64 bit products over
  // a 128-bit counter, under a 64-bit key that a Weyl sequence changes each round.
  __device__ __forceinline__ void draw(uint64_t unit, const Key& key) {
    uint32_t c[4] = {(uint32_t)unit, (uint32_t)(unit >> 32), (uint32_t)key.offset, (uint32_t)(key.offset >> 32)};
    uint32_t k0 = (uint32_t)key.seed, k1 = (uint32_t)(key.seed >> 32);
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const uint64_t p0 = (uint64_t)0xD2511F53u * c[0], p1 = (uint64_t)0xCD9E8D57u * c[2];
      c[0] = xor3((uint32_t)(p1 >> 32), c[1], k0);
      c[1] = (uint32_t)p1;
      c[2] = xor3((uint32_t)(p0 >> 32), c[3], k1);
      c[3] = (uint32_t)p0;
      k0 += 0x9E3779B9u;
      k1 += 0xBB67AE85u;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = c[i] & key.live;
      k[2 * i] = w << 16 >= key.below;
      k[2 * i + 1] = (w & 0xffff0000u) >= key.below;
    }
  }
  // Eight values of which the first `moved` (1 to 7) are the last ones of the unit
  // before.
  __device__ __forceinline__ void draw_across(uint64_t unit, int moved, const Key& key) {
    draw(unit - 1, key);
    const uint32_t before = bits();
    draw(unit, key);
    const uint32_t both = before >> (8 - moved) | bits() << moved;
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = both >> i & 1;
  }
  __device__ __forceinline__ uint32_t bits() const {
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) b |= k[i] ? 1u << i : 0u;
    return b;
  }
  // one instruction for two
  static __device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
    return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
  }
};

// Eight values, a unit's.
template <typename T> struct Eight {
  static constexpr int VE = 16 / sizeof(T), NV = 8 / VE;
  Vec<T, VE> v[NV];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j].load(p + j * VE);
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j].store(p + j * VE);
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j].get(f + j * VE);
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j].set(f + j * VE);
  }
};

// out = (kept ? x * scale : 0) + residual, rounded once; res: none without RES.
template <bool RES, typename TX, typename TR, typename TO>
__device__ __forceinline__ void apply(const Eight<TX>& x, const Eight<TR>& res, TO* out, const Keep& keep, float scale) {
  float f[8], r[8];
  x.get(f);
  if constexpr (RES) res.get(r);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float base = RES ? r[i] : 0.f;
    f[i] = keep.k[i] ? fmaf(f[i], scale, base) : base;
  }
  Eight<TO> o;
  o.set(f);
  o.store(out);
}

// A decision for each value: units of eight values that lie one behind the other,
// four a thread.  The last one is moved back to end with the values, so its
// decisions come from two units.
template <bool RES, typename TX, typename TR, typename TO, int U>
__global__ __launch_bounds__(256) void dropout_flat_kernel(const TX* __restrict__ x, const TR* __restrict__ residual,
                                                           TO* __restrict__ out, int64_t n, Key key,
                                                           const uint64_t* __restrict__ seed_device, float scale) {
  if (seed_device) key.seed = *seed_device;
  const int64_t units = (n + 7) / 8;
  for (int64_t u0 = (int64_t)blockIdx.x * 256 * U + threadIdx.x; u0 < units; u0 += (int64_t)gridDim.x * 256 * U) {
    Eight<TX> xv[U];
    Eight<TR> rv[U];
    int64_t at[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int64_t u = u0 + j * 256;
      at[j] = u * 8 + 8 <= n ? u * 8 : n - 8;  // past the end: the last unit again, not stored
      xv[j].load(x + at[j]);
      if constexpr (RES) rv[j].load(residual + at[j]);
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int64_t u = u0 + j * 256;
      if (u >= units) break;
      const int moved = (int)(u * 8 - at[j]);
      Keep keep;
      if (moved)
        keep.draw_across(u, moved, key);
      else
        keep.draw(u, key);
      apply<RES>(xv[j], rv[j], out + at[j], keep, scale);
    }
  }
}

// One mask for all `shared` indices, at least eight values wide.  A thread has one
// unit of one outer index and walks `shared`; of a block's 256 threads `width` lie
// along the units, then `lanes` along the shared dimension, then `outers` along the
// outer one.  A block takes `steps` times `lanes` shared indices.
struct SharedShape {
  int64_t outer, shared, inner, units, tiles, chunks, columns;
  int width, lanes, outers, steps;
};

// a / b and a % b for a, b >= 0: in 32 bits where they fit, which takes a fifth of
// the instructions.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b, int64_t& rest) {
  if (((a | b) >> 32) == 0) {
    const uint32_t q = (uint32_t)a / (uint32_t)b;
    rest = (uint32_t)a - q * (uint32_t)b;
    return q;
  }
  const int64_t q = a / b;
  rest = a - q * b;
  return q;
}

template <bool RES, typename TX, typename TR, typename TO>
__global__ __launch_bounds__(256) void dropout_shared_kernel(const TX* __restrict__ x, const TR* __restrict__ residual,
                                                             TO* __restrict__ out, SharedShape g, Key key,
                                                             const uint64_t* __restrict__ seed_device, float scale) {
  constexpr int U = 4;  // rows in flight
  if (seed_device) key.seed = *seed_device;
  const int t = threadIdx.x, column = t % g.width, lane = t / g.width % g.lanes, place = t / (g.width * g.lanes);
  const int64_t items = g.tiles * g.chunks * g.columns;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    int64_t tile, chunk;
    const int64_t o = divide(divide(item, g.tiles, tile), g.chunks, chunk) * g.outers + place;
    const int64_t unit = tile * g.width + column, s0 = chunk * g.lanes * g.steps + lane;
    if (unit >= g.units || place >= g.outers || o >= g.outer || s0 >= g.shared) continue;
    // the last unit of an outer index is moved back to end with it
    const int64_t r = unit * 8 + 8 <= g.inner ? unit * 8 : g.inner - 8;
    const int moved = (int)(unit * 8 - r);
    const int64_t base = o * g.shared * g.inner + r;
    Keep keep;
    for (int k = 0; k < g.steps; k += U) {
      Eight<TX> xv[U];
      Eight<TR> rv[U];
      int64_t at[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int64_t s = s0 + (int64_t)(k + j) * g.lanes;
        at[j] = base + (s < g.shared ? s : g.shared - 1) * g.inner;
        xv[j].load(x + at[j]);
        if constexpr (RES) rv[j].load(residual + at[j]);
      }
      if (k == 0) {  // behind the first rows' loads
        if (moved)
          keep.draw_across(o * g.units + unit, moved, key);
        else
          keep.draw(o * g.units + unit, key);
      }
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (k + j < g.steps && s0 + (int64_t)(k + j) * g.lanes < g.shared)
          apply<RES>(xv[j], rv[j], out + at[j], keep, scale);
    }
  }
}

// Masks narrower than a unit: an outer index' is one unit.  A thread has eight
// values that lie one behind the other and draws again where the outer index
// changes.
template <bool RES, typename TX, typename TR, typename TO>
__global__ __launch_bounds__(256) void dropout_narrow_kernel(const TX* __restrict__ x, const TR* __restrict__ residual,
                                                             TO* __restrict__ out, int64_t shared, int inner,
                                                             int64_t n, Key key,
                                                             const uint64_t* __restrict__ seed_device, float scale) {
  if (seed_device) key.seed = *seed_device;
  const int64_t step = (int64_t)gridDim.x * 256 * 8;
  for (int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; at < n; at += step) {
    const int many = n - at < 8 ? (int)(n - at) : 8;
    int64_t rest, s;
    int64_t o = divide(divide(at, inner, rest), shared, s);
    int r = (int)rest;
    Keep keep;
    keep.draw(o, key);
    uint32_t mine = keep.bits(), bits = 0;
    for (int i = 0; i < many; ++i) {
      bits |= (mine >> r & 1) << i;
      if (++r < inner) continue;
      r = 0;
      if (++s < shared) continue;
      s = 0;
      if (i + 1 < many) {
        keep.draw(++o, key);
        mine = keep.bits();
      }
    }
    if (many == 8) {
      Eight<TX> xv;
      Eight<TR> rv;
      xv.load(x + at);
      if constexpr (RES) rv.load(residual + at);
#pragma unroll
      for (int i = 0; i < 8; ++i) keep.k[i] = bits >> i & 1;
      apply<RES>(xv, rv, out + at, keep, scale);
    } else {
      for (int i = 0; i < many; ++i) {
        const float base = RES ? to_f32(residual[at + i]) : 0.f;
        out[at + i] = cvt<TO>(bits >> i & 1 ? fmaf(to_f32(x[at + i]), scale, base) : base);
      }
    }
  }
}

constexpr int64_t kMostBlocks = 1 << 20;  // the kernels loop past that

template <bool RES, typename TX, typename TR, typename TO>
static int launch_dropout(const void* xp, const void* rp, void* op, int64_t outer, int64_t shared, int64_t inner,
                          const Key& key, const uint64_t* seed_device, float scale, hipStream_t st) {
  const TX* x = (const TX*)xp;
  const TR* residual = (const TR*)rp;
  TO* out = (TO*)op;
  const int64_t n = outer * shared * inner;
  StageTimer timer("dropout", st);
  if (shared == 1 && n >= 8 && (outer == 1 || inner % 8 == 0)) {
    constexpr int U = 4;
    const int64_t blocks = ((n + 7) / 8 + 256 * U - 1) / (256 * U);
    dropout_flat_kernel<RES, TX, TR, TO, U><<<(unsigned)std::min(blocks, kMostBlocks), 256, 0, st>>>(
        x, residual, out, n, key, seed_device, scale);
  } else if (inner >= 8) {
    SharedShape g{outer, shared, inner, (inner + 7) / 8, 0, 0, 0, 0, 0, 0, 0};
    g.width = (int)std::min<int64_t>(g.units, 256);
    g.tiles = (g.units + g.width - 1) / g.width;
    g.lanes = (int)std::min<int64_t>(shared, 256 / g.width);
    g.outers = 256 / (g.width * g.lanes);
    g.columns = (outer + g.outers - 1) / g.outers;
    const int64_t rows = (shared + g.lanes - 1) / g.lanes;
    g.steps = 8;
    while (g.steps > 1 && g.tiles * g.columns * ((rows + g.steps - 1) / g.steps) < 8 * (int64_t)device_cus()) g.steps /= 2;
    g.chunks = (rows + g.steps - 1) / g.steps;
    dropout_shared_kernel<RES, TX, TR, TO>
        <<<(unsigned)std::min(g.tiles * g.columns * g.chunks, kMostBlocks), 256, 0, st>>>(x, residual, out, g, key,
                                                                                         seed_device, scale);
  } else {
    dropout_narrow_kernel<RES, TX, TR, TO><<<(unsigned)std::min((n + 2047) / 2048, kMostBlocks), 256, 0, st>>>(
        x, residual, out, shared, (int)inner, n, key, seed_device, scale);
  }
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
  const Key key = Key::of(seed, offset, t);
  auto run = [&](auto res, auto tx, auto to) {
    typedef decltype(to) TO;
    return launch_dropout<decltype(res)::value, decltype(tx), TO, TO>(x, residual, out, outer, shared, inner, key,
                                                                      seed_device, scale, (hipStream_t)stream);
  };
  const std::true_type with;
  const std::false_type without;
  if (residual) {
    if (out_dtype == GTK_BF16) return run(with, bf16(), bf16());
    return dtype == GTK_BF16 ? run(with, bf16(), float()) : run(with, float(), float());
  }
  if (out_dtype == GTK_BF16) return dtype == GTK_BF16 ? run(without, bf16(), bf16()) : run(without, float(), bf16());
  return dtype == GTK_BF16 ? run(without, bf16(), float()) : run(without, float(), float());
}
