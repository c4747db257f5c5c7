// Values as the normalisation and dropout kernels move them: 16-byte vectors at any
// address of the element's alignment (which gfx950 reads and writes as fast as
// aligned ones), parameter vectors of either type, and sums over lanes.
#pragma once
#include "common.hpp"

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

// VE values of T: 16 bytes, or one.  Loads and stores are non-temporal where each
// value is used once.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

template <typename T, int VE> struct Vec {
  u32x4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = __builtin_nontemporal_load((const u32x4_any*)p); }
  __device__ __forceinline__ void store(T* p) const { __builtin_nontemporal_store(raw, (u32x4_any*)p); }
  __device__ __forceinline__ void load_plain(const T* p) { raw = *(const u32x4_any*)p; }
  __device__ __forceinline__ void zero() { raw = u32x4{0, 0, 0, 0}; }
  // What was unpacked before is unpacked again, and need not be kept in registers.
  __device__ __forceinline__ void forget_unpacked() { asm volatile("" : "+v"(raw)); }
  __device__ __forceinline__ void store_plain(T* p) const { *(u32x4_any*)p = raw; }
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
  __device__ __forceinline__ void load_plain(const T* p) { v = *p; }
  __device__ __forceinline__ void zero() { v = cvt<T>(0.f); }
  __device__ __forceinline__ void forget_unpacked() {}
  __device__ __forceinline__ void store_plain(T* p) const { *p = v; }
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
}  // namespace gtk
