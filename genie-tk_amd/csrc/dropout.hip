// Dropout with a counter-based generator, for gfx950: the mask is a function of
// (seed, offset, place), computed where it is used, and in the backward pass again.
//
// One evaluation of the generator decides eight values (16 bits each, one unit);
// it is some 90 instructions, 20 of them wide products at a quarter of the rate.  A
// value of its own mask costs some 25 issue slots with its own arithmetic, and a bf16
// one moves 4 bytes: at 6 TB/s that is nearly what the memory takes, and the two
// overlap.  Under a mask that is shared along a dimension a draw serves several
// rows, and memory bounds it.  On MI355X, inputs in rotation: 512 x 512 x 128 bf16
// with residual 33 us (6.0 TB/s), its gradient 24 (5.6); 2 x 384 x 384 x 128 bf16
// added to fp32 58 us (6.5), its gradient 36 (6.3); 7.5 10^7 bf16 values with a mask
// of their own 52 us (5.8); 64 x 64 x 128 3.4 us, a launch's latency.
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

// N values that lie one behind the other, one access: 16 bytes, or 8 of bf16 beside
// fp32.
template <typename T, int N> struct Piece : Vec<T, N> {};
template <> struct Piece<bf16, 4> {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  typedef u32x2 u32x2_any __attribute__((aligned(2)));
  u32x2 raw;
  __device__ __forceinline__ void load(const bf16* p) { raw = __builtin_nontemporal_load((const u32x2_any*)p); }
  __device__ __forceinline__ void store(bf16* p) const { __builtin_nontemporal_store(raw, (u32x2_any*)p); }
  __device__ __forceinline__ void store_plain(bf16* p) const { *(u32x2_any*)p = raw; }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[2 * i] = __uint_as_float(raw[i] << 16);
      f[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int i = 0; i < 2; ++i) raw[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
  }
};

// The types of a call, and the values of a thread's access: where fp32 is among
// them a unit is two accesses, of neighbouring threads (two accesses of one thread,
// 32 bytes apart, read 36 MB of fp32 with residual in 40 us against 26).
template <bool RES_, typename TX_, typename TR_, typename TO_> struct Types {
  static constexpr bool RES = RES_;
  typedef TX_ TX;
  typedef TR_ TR;
  typedef TO_ TO;
  static constexpr int N = sizeof(TX) == 2 && sizeof(TR) == 2 && sizeof(TO) == 2 ? 8 : 4;
};

template <typename Y> struct Operands {
  Piece<typename Y::TX, Y::N> x;
  Piece<typename Y::TR, Y::N> r;
  __device__ __forceinline__ void load(const typename Y::TX* px, const typename Y::TR* pr, int64_t at) {
    x.load(px + at);
    if constexpr (Y::RES) r.load(pr + at);
  }
  // (kept ? x * scale : 0) + residual, rounded once.  NT: the result passes the caches
  template <bool NT> __device__ __forceinline__ void finish(typename Y::TO* out, const bool* keep, float scale) const {
    float f[Y::N], g[Y::N];
    x.get(f);
    if constexpr (Y::RES) r.get(g);
#pragma unroll
    for (int i = 0; i < Y::N; ++i) {
      const float base = Y::RES ? g[i] : 0.f;
      f[i] = keep[i] ? fmaf(f[i], scale, base) : base;
    }
    Piece<typename Y::TO, Y::N> o;
    o.set(f);
    if constexpr (NT)
      o.store(out);
    else
      o.store_plain(out);
  }
};

// The same for `many` values, one by one; bits: from the first one's on.
template <typename Y>
__device__ __forceinline__ void finish_single(const typename Y::TX* x, const typename Y::TR* residual,
                                              typename Y::TO* out, int many, uint32_t bits, float scale) {
  for (int i = 0; i < many; ++i) {
    const float base = Y::RES ? to_f32(residual[i]) : 0.f;
    out[i] = cvt<typename Y::TO>(bits >> i & 1 ? fmaf(to_f32(x[i]), scale, base) : base);
  }
}

// A decision for each value: a wave draws 64 units, a unit a lane, U times.  Pieces
// of four values lie in the order of the lanes, so their decisions come from the
// lanes that drew them.  What is left behind the last whole unit is one thread's.
template <typename Y, int U>
__global__ __launch_bounds__(256) void dropout_flat_kernel(const typename Y::TX* __restrict__ x,
                                                           const typename Y::TR* __restrict__ residual,
                                                           typename Y::TO* __restrict__ out, int64_t n, Key key,
                                                           const uint64_t* __restrict__ seed_device, float scale) {
  constexpr int N = Y::N, K = 8 / N;  // pieces a unit
  if (seed_device) key.seed = *seed_device;
  const int64_t units = n / 8, pieces = units * K;
  const int lane = threadIdx.x & 63;
  for (int64_t w = (int64_t)blockIdx.x * 256 * U + wave_id() * 64; w < units; w += (int64_t)gridDim.x * 256 * U) {
    Operands<Y> in[U][K];
    int64_t at[U][K];
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        at[j][k] = (w + j * 256) * K + k * 64 + lane;  // past the last one: that one again, not stored
        in[j][k].load(x, residual, (at[j][k] < pieces ? at[j][k] : pieces - 1) * N);
      }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      Keep keep;
      keep.draw(w + j * 256 + lane, key);
      const uint32_t mine = K > 1 ? keep.bits() : 0;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if constexpr (K > 1) {
          const uint32_t bits = (uint32_t)__shfl((int)mine, k * 32 + lane / 2, 64) >> (lane % 2 * 4);
#pragma unroll
          for (int i = 0; i < N; ++i) keep.k[i] = bits >> i & 1;
        }
        if (at[j][k] < pieces) in[j][k].template finish<true>(out + at[j][k] * N, keep.k, scale);
      }
    }
  }
  if (n % 8 && blockIdx.x == 0 && threadIdx.x == 0) {
    Keep keep;
    keep.draw(units, key);
    const int64_t at = units * 8;
    finish_single<Y>(x + at, residual + (Y::RES ? at : 0), out + at, (int)(n - at), keep.bits(), scale);
  }
}

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

// One mask for all `shared` indices, at least eight values wide.  A thread has one
// piece of one outer index and walks `shared`, ROWS indices; of a block's 256
// threads `width` lie along the pieces, then `lanes` along the shared dimension,
// then `outers` along the outer one.  Plain stores with a residual (bf16 onto fp32,
// 2 x 384 x 384 x 128: 58 us, non-temporal 61), non-temporal ones without (its
// backward pass in bf16, 512 x 512 x 128: 24 us, plain 25).
struct SharedShape {
  int64_t outer, shared, inner, units, pieces, tiles, chunks, columns;
  int width, lanes, outers;
};

template <typename Y, int ROWS>
__global__ __launch_bounds__(256) void dropout_shared_kernel(const typename Y::TX* __restrict__ x,
                                                             const typename Y::TR* __restrict__ residual,
                                                             typename Y::TO* __restrict__ out, SharedShape g, Key key,
                                                             const uint64_t* __restrict__ seed_device, float scale) {
  constexpr int N = Y::N;
  if (seed_device) key.seed = *seed_device;
  const int t = threadIdx.x, column = t % g.width, lane = t / g.width % g.lanes, place = t / (g.width * g.lanes);
  const int64_t items = g.tiles * g.chunks * g.columns;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    int64_t tile, chunk;
    const int64_t o = divide(divide(item, g.tiles, tile), g.chunks, chunk) * g.outers + place;
    const int64_t piece = tile * g.width + column, s0 = chunk * g.lanes * ROWS + lane;
    if (piece >= g.pieces || place >= g.outers || o >= g.outer || s0 >= g.shared) continue;
    // the last piece of an outer index is moved back to end with it
    const int64_t r = piece * N + N <= g.inner ? piece * N : g.inner - N;
    const int64_t base = o * g.shared * g.inner + r;
    Operands<Y> in[ROWS];
    int64_t at[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int64_t s = s0 + (int64_t)j * g.lanes;
      at[j] = base + (s < g.shared ? s : g.shared - 1) * g.inner;
      in[j].load(x, residual, at[j]);
    }
    Keep keep;
    keep.draw(o * g.units + r / 8, key);
    uint32_t bits = keep.bits();
    const int from = (int)(r % 8);
    if (from + N > 8) {  // a moved piece of two units
      keep.draw(o * g.units + r / 8 + 1, key);
      bits |= keep.bits() << 8;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) keep.k[i] = bits >> (from + i) & 1;
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
      if (s0 + (int64_t)j * g.lanes < g.shared) in[j].template finish<!Y::RES>(out + at[j], keep.k, scale);
  }
}

// Masks narrower than a unit: an outer index' is one unit.  A thread has eight
// values that lie one behind the other and draws again where the outer index
// changes.
template <typename Y>
__global__ __launch_bounds__(256) void dropout_narrow_kernel(const typename Y::TX* __restrict__ x,
                                                             const typename Y::TR* __restrict__ residual,
                                                             typename Y::TO* __restrict__ out, int64_t shared,
                                                             int inner, int64_t n, Key key,
                                                             const uint64_t* __restrict__ seed_device, float scale) {
  constexpr int N = Y::N, K = 8 / N;
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
    if (many < 8) {
      finish_single<Y>(x + at, residual + (Y::RES ? at : 0), out + at, many, bits, scale);
      continue;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) keep.k[i] = bits >> i & 1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      Operands<Y> in;
      in.load(x, residual, at + k * N);
      in.template finish<true>(out + at + k * N, keep.k + k * N, scale);
    }
  }
}

constexpr int64_t kMostBlocks = 1 << 20;  // the kernels loop past that

template <typename Y>
static int launch_dropout(const void* xp, const void* rp, void* op, int64_t outer, int64_t shared, int64_t inner,
                          const Key& key, const uint64_t* seed_device, float scale, hipStream_t st) {
  const auto* x = (const typename Y::TX*)xp;
  const auto* residual = (const typename Y::TR*)rp;
  auto* out = (typename Y::TO*)op;
  const int64_t n = outer * shared * inner;
  StageTimer timer("dropout", st);
  if (shared == 1 && n >= 8 && (outer == 1 || inner % 8 == 0)) {
    // two units a lane: 302 MB of bf16 moved in 50 us, with four 52
    constexpr int U = 2;
    const int64_t blocks = (n / 8 + 256 * U - 1) / (256 * U);
    dropout_flat_kernel<Y, U><<<(unsigned)std::min(blocks, kMostBlocks), 256, 0, st>>>(x, residual, out, n, key,
                                                                                       seed_device, scale);
  } else if (inner >= 8) {
    SharedShape g{outer, shared, inner, (inner + 7) / 8, (inner + Y::N - 1) / Y::N, 0, 0, 0, 0, 0, 0};
    g.width = (int)std::min<int64_t>(g.pieces, 256);
    g.tiles = (g.pieces + g.width - 1) / g.width;
    g.lanes = (int)std::min<int64_t>(shared, 256 / g.width);
    g.outers = 256 / (g.width * g.lanes);
    g.columns = (outer + g.outers - 1) / g.outers;
    const int64_t rows = (shared + g.lanes - 1) / g.lanes;
    auto run = [&](auto count) {
      constexpr int ROWS = decltype(count)::value;
      g.chunks = (rows + ROWS - 1) / ROWS;
      const int64_t blocks = g.tiles * g.columns * g.chunks;
      if (ROWS > 1 && (blocks < 2 * (int64_t)device_cus() || rows < ROWS)) return false;
      dropout_shared_kernel<Y, ROWS><<<(unsigned)std::min(blocks, kMostBlocks), 256, 0, st>>>(
          x, residual, out, g, key, seed_device, scale);
      return true;
    };
    // several rows a draw, unless that leaves the chip without blocks (twice as many
    // gain nothing: 604 MB of bf16 and fp32 moved in 96 us, with eight rows 98)
    run(std::integral_constant<int, 16 / Y::N>()) || run(std::integral_constant<int, 1>());
  } else {
    dropout_narrow_kernel<Y><<<(unsigned)std::min((n + 2047) / 2048, kMostBlocks), 256, 0, st>>>(
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
    return launch_dropout<Types<decltype(res)::value, decltype(tx), TO, TO>>(
        x, residual, out, outer, shared, inner, key, seed_device, scale, (hipStream_t)stream);
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
