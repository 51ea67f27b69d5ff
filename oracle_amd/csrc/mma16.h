// The two 16-bit element types of the attention operators (attn_packed.hip, attn_paged.hip) and their matrix instructions.
#pragma once
#include <hip/hip_runtime.h>

#include "common.h"

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
typedef __attribute__((address_space(3))) void lds_void_t;

template <typename T> struct Mma;
template <> struct Mma<__bf16> {
  static constexpr bool BF16 = true;
  typedef bf16x8 v8;
  typedef __attribute__((ext_vector_type(2))) __bf16 v2;
  static __device__ __forceinline__ f32x16 m32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 m16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<_Float16> {
  static constexpr bool BF16 = false;
  typedef f16x8 v8;
  typedef __attribute__((ext_vector_type(2))) _Float16 v2;
  static __device__ __forceinline__ f32x16 m32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 m16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
// two floats rounded to nearest even, packed
template <typename T> __device__ __forceinline__ uint32_t cvt2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, typename Mma<T>::v2));
}
// 4 rows x 16 columns of 16-bit values, transposed by a group of 16 lanes: lane i passes the address of 8 bytes (row i / 4, columns
// 4 (i % 4) ...) and gets column i, rows 0..3
template <typename T> __device__ __forceinline__ u32x2 lds_tr16(const char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)p));
}
template <typename T> __device__ __forceinline__ typename Mma<T>::v8 join8(u32x2 a, u32x2 b) {
  return __builtin_bit_cast(typename Mma<T>::v8, (u32x4){a[0], a[1], b[0], b[1]});
}

// `bytes` bytes from base on; a lane that asks beyond them gets zeros
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, 0x00020000);
}
// 16 bytes a lane, from byte `at`: into registers, or by LDS-DMA to `to` + 16 lane
__device__ __forceinline__ u32x4 buffer_load16(__amdgpu_buffer_rsrc_t r, int at) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
}
__device__ __forceinline__ void buffer_load16_lds(__amdgpu_buffer_rsrc_t r, int at, char* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)to, 16, at, 0, 0, 0);
}
