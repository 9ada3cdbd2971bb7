// The two 16-bit types that the kernels for batches of streams take, behind one interface.
#pragma once
#include "ll_common.h"

namespace ll {

typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_hw __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_hw __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_hw __attribute__((ext_vector_type(2)));

struct Bf16 {
  static constexpr uint32_t kInfinity = 0x7F80;  // magnitudes from here on are not finite
  static constexpr float kWeightShift = 0.0f;    // log2 of what a softmax's probabilities are held times
  static __device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xFFFF0000u);
  }
  // round to nearest even
  static __device__ __forceinline__ uint32_t pack2(float a, float b) { return pack_bf16x2(a, b); }
  // c + the two values of w
  static __device__ __forceinline__ float add2(uint32_t w, float c) {
    const bf16x2_hw one = {(__bf16)1.0f, (__bf16)1.0f};
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_hw, w), one, c, false);
  }
  static __device__ __forceinline__ float16v mfma(short8v a, short8v b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_hw, a), __builtin_bit_cast(bf16x8_hw, b), c, 0, 0, 0);
  }
};

struct F16 {
  static constexpr uint32_t kInfinity = 0x7C00;
  // The range ends 2^24 below 1 and 2^16 above it: near its upper end, keys down to 2^-37 of the largest keep a weight.
  static constexpr float kWeightShift = 13.0f;
  static __device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
    const f16x2_hw h = __builtin_bit_cast(f16x2_hw, w);
    a = (float)h[0];
    b = (float)h[1];
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2_hw v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_hw));
  }
  static __device__ __forceinline__ float add2(uint32_t w, float c) {
    const f16x2_hw one = {(_Float16)1.0f, (_Float16)1.0f};
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_hw, w), one, c, false);
  }
  static __device__ __forceinline__ float16v mfma(short8v a, short8v b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_hw, a), __builtin_bit_cast(f16x8_hw, b), c, 0, 0, 0);
  }
};

}  // namespace ll
