// Shared pieces of the view-token operators (dtk_*): element types, 16-byte vectors at any
// alignment, the counter-based generator.
#pragma once
#include "dsplat_common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace dtk {

using bf16 = __bf16;
using f16 = _Float16;

// One 16-byte vector of T. The loads and stores take any address (global memory accesses of
// this ISA need no alignment beyond the element's), so rows of odd widths and strides move
// as whole vectors too.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  Vec<T> r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& r) {
  __builtin_memcpy(p, &r, 16);
}

// The 32-bit value rounded to T. Without the empty statement a last f32 operation and f16's rounding become one
// instruction that rounds once, in some kernels and not in others; the plain and the fused norm give the same bits.
template <typename T>
__device__ __forceinline__ T rounded(float f) {
  if constexpr (__is_same(T, f16)) asm("" : "+v"(f));
  return (T)f;
}

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3",
// SC 2011): ten rounds of two 32 x 32 -> 64 bit products of the counter, keyed. Counter: the
// group's 64-bit number, the call's id, the step; key: the 64-bit seed. A round is two v_mad_u64_u32 (8 cycles a
// wave; separate upper and lower halves take half as long again) and two three-way exclusive ors.
struct RngKey {
  uint32_t k0, k1, call, step;
};
__device__ __forceinline__ RngKey rng_key(const int64_t* rng, uint32_t call) {
  const uint64_t seed = (uint64_t)rng[0], step = (uint64_t)rng[1];
  return {(uint32_t)seed, (uint32_t)(seed >> 32), call, (uint32_t)step};
}
__device__ __forceinline__ void philox(const RngKey& key, uint64_t group, uint32_t (&w)[4]) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = key.call, c3 = key.step;
  uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = __builtin_amdgcn_bitop3_b32((uint32_t)(b >> 32), c1, k0, 0x96);  // the three's exclusive or
    c1 = (uint32_t)b;
    c2 = __builtin_amdgcn_bitop3_b32((uint32_t)(a >> 32), c3, k1, 0x96);
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}
// keep[e] of the N elements from n0 on (both multiples of 4): element n takes word n % 4 of group n / 4, and
// is kept if that is above `least`.
template <int N>
__device__ __forceinline__ void keep_mask(const RngKey& key, uint64_t n0, uint32_t least, bool (&keep)[N]) {
#pragma unroll
  for (int g = 0; g < N / 4; ++g) {
    uint32_t w[4];
    philox(key, (n0 >> 2) + g, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) keep[4 * g + i] = w[i] > least;
  }
}

// The same from any element on: one group more where n0 lies inside one, and the bits shifted by its place.
template <int N>
__device__ __forceinline__ void keep_mask_anywhere(const RngKey& key, uint64_t n0, uint32_t least, bool (&keep)[N]) {
  const uint32_t sh = (uint32_t)n0 & 3u;
  uint32_t bits = 0;
#pragma unroll
  for (int g = 0; g < N / 4; ++g) {
    uint32_t w[4];
    philox(key, (n0 >> 2) + g, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) bits |= w[i] > least ? 1u << (4 * g + i) : 0u;
  }
  if (sh) {
    uint32_t w[4];
    philox(key, (n0 >> 2) + N / 4, w);
#pragma unroll
    for (int i = 0; i < 3; ++i) bits |= w[i] > least ? 1u << (N + i) : 0u;
  }
  bits >>= sh;
#pragma unroll
  for (int e = 0; e < N; ++e) keep[e] = (bits >> e) & 1u;
}

inline bool type_ok(int t) { return t >= DTK_F32 && t <= DTK_F16; }
inline size_t type_size(int t) { return t == DTK_F32 ? 4 : 2; }

}  // namespace dtk
