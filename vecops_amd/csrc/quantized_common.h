// What the kernels of quantised elements share (fp8_block.hip, mx_block.hip, row_quantize.hip): loads at any address, scales of
// 8-bit floats, fragments, results of a product.
#ifndef VECOPS_HIP_QUANTIZED_COMMON_H
#define VECOPS_HIP_QUANTIZED_COMMON_H

#include "fp8_block.h"
#include "tile_gemm.h"

namespace vecops_hip {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
// the same at any address: the memory system takes them, and the compiler then makes one access of each
typedef __attribute__((ext_vector_type(2), aligned(1))) uint32_t u32x2_anywhere;
typedef __attribute__((ext_vector_type(4), aligned(1))) uint32_t u32x4_anywhere;

template <class Pointer>
__device__ __forceinline__ u32x4 load_16(Pointer at) { return *(const VECOPS_GLOBAL u32x4_anywhere*)at; }

__device__ __forceinline__ float real_bits_to_f32(uint32_t bits, int kind) {
  return kind == FP8_REAL_BF16 ? __uint_as_float(bits << 16) : f16_bits_to_f32(bits);
}

// Four quotients to four e4m3 bytes.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true));
}

__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
  const float s = __uint_as_float(amax_bits) / 448.0f;
  return s < 0x1p-126f ? 0x1p-126f : s;  // (NaN stays)
}

// x / s for a whole block.  With r = 1/s rounded, one step of Markstein's division (t = x r; t + (x - t s) r) gives the correctly
// rounded quotient in three operations where a division takes about ten, as long as nothing under- or overflows: scales outside
// [2^-80, 2^120] (uniform over the block) divide.
struct Quotient {
  float s, r;
  bool plain;
  __device__ __forceinline__ explicit Quotient(float scale) : s(scale), r(1.0f / scale), plain(!(scale >= 0x1p-80f && scale <= 0x1p120f)) {}
  __device__ __forceinline__ float operator()(float x) const {
    if (plain) return x / s;
    const float t = x * r;
    return copysignf(fmaf(fmaf(-t, s, x), r, t), x);   // (the sum of -0 and its remainder 0 is +0)
  }
};

__device__ __forceinline__ i32x8 fragment_of(const u32x4& lo, const u32x4& hi) {
  return i32x8{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(lo[2]), static_cast<int>(lo[3]),
               static_cast<int>(hi[0]), static_cast<int>(hi[1]), static_cast<int>(hi[2]), static_cast<int>(hi[3])};
}

// COUNT consecutive results of a row from column n on (`at`: the first one's place in elements); those past n_end stay unwritten.
template <int COUNT>
__device__ __forceinline__ void store_results(void* c, int64_t at, int64_t cs, int out_kind, int64_t n, int64_t n_end, const float (&v)[COUNT]) {
  if (out_kind == FP8_REAL_F32) {
    VECOPS_GLOBAL float* to = (VECOPS_GLOBAL float*)c + at;
    if (cs == 1 && n + COUNT <= n_end) {
#pragma unroll
      for (int e = 0; e < COUNT; e += 4)
        *(VECOPS_GLOBAL u32x4_anywhere*)(to + e) = u32x4{__float_as_uint(v[e]), __float_as_uint(v[e + 1]), __float_as_uint(v[e + 2]), __float_as_uint(v[e + 3])};
    } else {
#pragma unroll
      for (int e = 0; e < COUNT; ++e)
        if (n + e < n_end) to[e * cs] = v[e];
    }
    return;
  }
  uint32_t w[COUNT / 2];
#pragma unroll
  for (int e = 0; e < COUNT / 2; ++e)
    w[e] = out_kind == FP8_REAL_BF16 ? cvt_pk_bf16(v[2 * e], v[2 * e + 1]) : f16_bits_rne(v[2 * e]) | static_cast<uint32_t>(f16_bits_rne(v[2 * e + 1])) << 16;
  VECOPS_GLOBAL uint16_t* to = (VECOPS_GLOBAL uint16_t*)c + at;
  if (cs == 1 && n + COUNT <= n_end) {
    if constexpr (COUNT == 8) *(VECOPS_GLOBAL u32x4_anywhere*)to = u32x4{w[0], w[1], w[2], w[3]};
    else *(VECOPS_GLOBAL u32x2_anywhere*)to = u32x2{w[0], w[1]};
  } else {
#pragma unroll
    for (int e = 0; e < COUNT; ++e)
      if (n + e < n_end) to[e * cs] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
  }
}

typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) float lds_float;
typedef __attribute__((address_space(3))) uint32_t lds_word;
typedef __attribute__((address_space(3))) uint16_t lds_short;
typedef __attribute__((address_space(3))) char lds_char;

// (`offset`, a constant, goes into the instruction)
__device__ __forceinline__ u32x4 read_lds(uint32_t at, int offset) {
  return *reinterpret_cast<const lds_u32x4*>(reinterpret_cast<const lds_char*>(static_cast<uintptr_t>(at)) + offset);
}
__device__ __forceinline__ void write_lds(uint32_t at, const u32x4& v) {
  *reinterpret_cast<lds_u32x4*>(reinterpret_cast<lds_char*>(static_cast<uintptr_t>(at))) = v;
}
__device__ __forceinline__ uint32_t read_lds_word(uint32_t at, int offset) {
  return *reinterpret_cast<const lds_word*>(reinterpret_cast<const lds_char*>(static_cast<uintptr_t>(at)) + offset);
}
__device__ __forceinline__ uint32_t read_lds_short(uint32_t at, int offset) {
  return *reinterpret_cast<const lds_short*>(reinterpret_cast<const lds_char*>(static_cast<uintptr_t>(at)) + offset);
}
__device__ __forceinline__ float read_lds_float(uint32_t at, int offset) {
  return *reinterpret_cast<const lds_float*>(reinterpret_cast<const lds_char*>(static_cast<uintptr_t>(at)) + offset);
}

}  // namespace vecops_hip
#endif
