// 16-bit element types and short vectors of elements at any address, for the kernels that work on
// activations (linear_scan.hip).  Arithmetic is in 32 bits; a value is rounded once, when it is
// stored, to nearest with ties to even.
#pragma once
#include "common.h"

namespace tcd {

struct f16_t {
  uint16_t bits;
};
struct bf16_t {
  uint16_t bits;
};

__device__ inline uint32_t bf16_bits(float v) {
#if defined(__AMDGCN__)
  return bit_cast<uint16_t>((__bf16)v);  // one conversion instruction for two values
#else
  const uint32_t u = bit_cast<uint32_t>(v);  // the host pass and the emulator have no such instruction
  if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
  return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
#endif
}
__device__ inline uint32_t f16_bits(float v) { return bit_cast<uint16_t>((_Float16)v); }

// VEC consecutive elements in whole registers (a single 16-bit element in the lower half of one).
// Loads and stores take any address the element type allows (see tcd_v4u_anywhere).
template <class T, int VEC>
struct Pack {
  static constexpr int kBytes = (int)sizeof(T) * VEC;
  static constexpr int NW = (kBytes + 3) / 4;
  uint32_t w[NW];

  __device__ float value(int j) const {
    if constexpr (sizeof(T) == 4) return bit_cast<float>(w[j]);
    const uint32_t u = w[j / 2];
    if constexpr (std::is_same<T, bf16_t>::value) return bit_cast<float>(j & 1 ? u & 0xffff0000u : u << 16);
    else return (float)bit_cast<_Float16>((uint16_t)(j & 1 ? u >> 16 : u));
  }
  // Rounds to nearest, ties to even.
  __device__ static Pack of(const float (&v)[VEC]) {
    Pack r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < VEC; j++) r.w[j] = bit_cast<uint32_t>(v[j]);
    } else {
#pragma unroll
      for (int i = 0; i < NW; i++) {
        const float hi = 2 * i + 1 < VEC ? v[2 * i + 1 < VEC ? 2 * i + 1 : 0] : 0.f;
        if constexpr (std::is_same<T, bf16_t>::value) r.w[i] = bf16_bits(v[2 * i]) | bf16_bits(hi) << 16;
        else r.w[i] = f16_bits(v[2 * i]) | f16_bits(hi) << 16;
      }
    }
    return r;
  }
};
typedef unsigned int tcd_v2u __attribute__((ext_vector_type(2)));
typedef tcd_v2u tcd_v2u_anywhere __attribute__((aligned(1)));

template <class T, int VEC>
__device__ inline Pack<T, VEC> load_pack(const T* p) {
  Pack<T, VEC> r;
  if constexpr (Pack<T, VEC>::kBytes == 16) {
    const tcd_v4u u = __builtin_nontemporal_load(reinterpret_cast<const tcd_v4u_anywhere*>(p));
    __builtin_memcpy(&r, &u, 16);
  } else if constexpr (Pack<T, VEC>::kBytes == 8) {
    const tcd_v2u u = __builtin_nontemporal_load(reinterpret_cast<const tcd_v2u_anywhere*>(p));
    __builtin_memcpy(&r, &u, 8);
  } else {
    static_assert(VEC == 1, "one element, or 8 or 16 bytes of them");
    if constexpr (sizeof(T) == 2) r.w[0] = reinterpret_cast<const uint16_t*>(p)[0];
    else r.w[0] = bit_cast<uint32_t>(p[0]);
  }
  return r;
}
template <class T, int VEC>
__device__ inline void store_pack(T* p, const Pack<T, VEC>& r) {
  if constexpr (Pack<T, VEC>::kBytes == 16) {
    tcd_v4u u;
    __builtin_memcpy(&u, &r, 16);
    __builtin_nontemporal_store(u, reinterpret_cast<tcd_v4u_anywhere*>(p));
  } else if constexpr (Pack<T, VEC>::kBytes == 8) {
    tcd_v2u u;
    __builtin_memcpy(&u, &r, 8);
    __builtin_nontemporal_store(u, reinterpret_cast<tcd_v2u_anywhere*>(p));
  } else {
    static_assert(VEC == 1, "one element, or 8 or 16 bytes of them");
    if constexpr (sizeof(T) == 2) reinterpret_cast<uint16_t*>(p)[0] = (uint16_t)r.w[0];
    else p[0] = bit_cast<T>(r.w[0]);
  }
}
// The first n < VEC elements of a pack, one by one: the end of a row whose length is no multiple of VEC.
template <class T, int VEC>
__device__ inline Pack<T, VEC> load_part(const T* p, int n) {
  Pack<T, VEC> r{};
#pragma unroll
  for (int j = 0; j < VEC - 1; j++) {
    if (j < n) {
      if constexpr (sizeof(T) == 4) r.w[j] = bit_cast<uint32_t>(p[j]);
      else r.w[j / 2] |= (uint32_t)p[j].bits << 16 * (j & 1);
    }
  }
  return r;
}
template <class T, int VEC>
__device__ inline void store_part(T* p, const Pack<T, VEC>& r, int n) {
#pragma unroll
  for (int j = 0; j < VEC - 1; j++) {
    if (j < n) {
      if constexpr (sizeof(T) == 4) p[j] = bit_cast<T>(r.w[j]);
      else p[j].bits = (uint16_t)(r.w[j / 2] >> 16 * (j & 1));
    }
  }
}

// Makes the compiler forget what it derived from a pack: a second pass over packed 16-bit values then
// converts them again instead of keeping the 32-bit ones of the first in twice as many registers.
template <class T, int VEC>
__device__ inline void forget(Pack<T, VEC>& r) {
#pragma unroll
  for (int i = 0; i < r.NW; i++) asm volatile("" : "+v"(r.w[i]));
}

inline int activation_size(int dt) {
  return dt == THRUST_CDNA4_F32 ? 4 : dt == THRUST_CDNA4_F16 || dt == THRUST_CDNA4_BF16 ? 2 : 0;
}

}  // namespace tcd
