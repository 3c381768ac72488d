// Shared pieces of the voxel-block kernels: 16-byte fragments, the 32x32
// matrix instructions on them, and direct-to-LDS loads.
#pragma once

#include "common.hpp"

namespace tsc {

typedef int int4v __attribute__((ext_vector_type(4)));
typedef int int2v __attribute__((ext_vector_type(2)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <typename T> constexpr bool kIs16 = sizeof(T) == 2;
template <typename T> constexpr int kPer16 = 16 / sizeof(T);  // elements of 16 bytes

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == TSC_F32) return static_cast<const float*>(p)[i];
  if (dtype == TSC_F16) return to_f32(static_cast<const __half*>(p)[i]);
  return to_f32(static_cast<const __hip_bfloat16*>(p)[i]);
}

// c += a b for a 32x32 tile: lane l holds row (a) or column (b) l % 32, and of
// the products' sum the 16 bytes' elements of its half l / 32.  Which values
// of the sum those are is the caller's choice, the same for a and b.  c: lane
// l holds column l % 32, register r row 8 (r / 4) + 4 (l / 32) + r % 4.
template <typename T>
__device__ __forceinline__ f32x16 mma32(int4v a, int4v b, f32x16 c) {
  if constexpr (std::is_same_v<T, __half>) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else if constexpr (std::is_same_v<T, __hip_bfloat16>) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
    return c;
  }
}

// Two f32 values rounded to nearest even as 16-bit values of T.
template <typename T>
__device__ __forceinline__ int pack2(float a, float b) {
  const f32x2 v = {a, b};
  if constexpr (std::is_same_v<T, __half>)
    return __builtin_bit_cast(int, __builtin_convertvector(v, f16x2));
  else
    return __builtin_bit_cast(int, __builtin_convertvector(v, bf16x2));
}

// N (even) f32 values rounded to T.
template <typename T, int N>
__device__ __forceinline__ void round_to(const float* v, T* e) {
  if constexpr (kIs16<T>) {
    int w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    __builtin_memcpy(e, w, N * sizeof(T));
  } else {
    __builtin_memcpy(e, v, N * sizeof(T));
  }
}

// 16 bytes per lane from base (wave uniform) + offset into LDS at byte address
// m0 (wave uniform) + 16 * lane, without passing through registers; lanes
// that are not in leave their place as it is.  The compiler does not know of
// the load: the kernels wait for it themselves.  Nothing else in these
// kernels uses M0.  Nor does it know the load's hazards: one wait state after
// M0's write, and five after a vector instruction that wrote the base (a
// spilled base comes back through v_readlane): the move and four more.
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t m0, bool in = true) {
  if (in)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(m0) : "memory");
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p));
}

// 16 bytes from an address aligned to its elements only.
template <typename T>
__device__ __forceinline__ int4v load16_unaligned(const T* p) {
  int4v v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

// The first `count` of 16 bytes' elements, the others 0, from any address.
template <typename T>
__device__ __forceinline__ int4v load16_partial(const T* p, int count) {
  T e[kPer16<T>];
#pragma unroll
  for (int i = 0; i < kPer16<T>; ++i) e[i] = i < count ? p[i] : from_f32<T>(0.f);
  int4v v;
  __builtin_memcpy(&v, e, 16);
  return v;
}

}  // namespace tsc
