// Device helpers of the operators on paged caches (qd_paged.hip, qd_tree.hip,
// qd_sparse.hip): the storage types, moves between lanes, and the launch.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "qd_device.hpp"
#include "qd_device_math.hpp"

namespace qd {
namespace dev {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
// Lengths, tables and positions are written before the kernel starts: they may
// be read through the scalar cache.
typedef const __attribute__((address_space(4))) int32_t const_i32;

__device__ __forceinline__ int32_t load_uniform(const int32_t *p) { return *(const_i32 *)p; }

__device__ __forceinline__ void raise_error(uint32_t *errors, uint32_t bit) {
  if (errors) atomicOr(errors, bit);
}

// Waits until this thread's vector memory operations have completed.
__device__ __forceinline__ void wait_vm_stores() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// The storage types' conversions; two values share a 32-bit register, low half first.
struct Half {
  static __device__ __forceinline__ float lo(uint32_t v) { return half_lo(v); }
  static __device__ __forceinline__ float hi(uint32_t v) { return half_hi(v); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const f16x2 v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};  // to nearest even
    return __builtin_bit_cast(uint32_t, v);
  }
  static __device__ __forceinline__ f4v mfma(u4v a, u4v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
struct Brain {
  static __device__ __forceinline__ float lo(uint32_t v) { return __uint_as_float(v << 16); }
  static __device__ __forceinline__ float hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};  // to nearest even
    return __builtin_bit_cast(uint32_t, v);
  }
  static __device__ __forceinline__ f4v mfma(u4v a, u4v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

// Four consecutive elements as FP32, and back.
template <typename E>
__device__ __forceinline__ float4 load4(const void *base, int64_t i) {
  if constexpr (std::is_same_v<E, float>) {
    return *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + i);
  } else {
    const uint2 v = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(base) + i);
    return make_float4(E::lo(v.x), E::hi(v.x), E::lo(v.y), E::hi(v.y));
  }
}
template <typename E>
__device__ __forceinline__ void store4(void *base, int64_t i, float4 v) {
  if constexpr (std::is_same_v<E, float>)
    *reinterpret_cast<float4 *>(static_cast<float *>(base) + i) = v;
  else
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(base) + i) = make_uint2(E::pack(v.x, v.y), E::pack(v.z, v.w));
}

// Values of lanes l and l ^ 32 in a and b (any order).
__device__ __forceinline__ void half_swap(float v, float &a, float &b) {
  unsigned x = __builtin_bit_cast(unsigned, v), y = x;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  a = __builtin_bit_cast(float, x);
  b = __builtin_bit_cast(float, y);
}
// Over lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float quarters_max(float v) {
  float a, b;
  v = row_pair_max(v);
  half_swap(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float quarters_sum(float v) {
  float a, b;
  v = row_pair_sum(v);
  half_swap(v, a, b);
  return a + b;
}

// Lane `from`'s value.
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int from) {
  const uint32_t lo = __builtin_amdgcn_ds_bpermute(from << 2, static_cast<int>(v));
  const uint32_t hi = __builtin_amdgcn_ds_bpermute(from << 2, static_cast<int>(v >> 32));
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ double lane_of(double v, int from) {
  return __builtin_bit_cast(double, lane_of(__builtin_bit_cast(uint64_t, v), from));
}

// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ uint32_t lanes_upto(uint32_t v) {
  int x = static_cast<int>(v);
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row 0 to 1, 2 to 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row 1 to 2 and 3
  return static_cast<uint32_t>(x);
}

// Maximum over the wave of numbers below 2^31.
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  int x = static_cast<int>(v);
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kDppXor1, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kDppXor2, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kDppHalfMirror, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kDppMirror, 0xf, 0xf, false));
  return static_cast<uint32_t>(max(max(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)),
                                   max(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48))));
}

}  // namespace dev

inline uint32_t log2_of(uint32_t v) { return static_cast<uint32_t>(__builtin_ctz(v)); }

template <typename... A>
hipError_t launch(void (*kernel)(A...), dim3 grid, dim3 block, hipStream_t s, A... args) {
  void *packed[] = {&args...};
  return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, packed, 0, s);
}

inline size_t round256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace qd
