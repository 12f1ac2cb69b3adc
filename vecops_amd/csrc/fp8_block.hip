// 8-bit floats (e4m3: 4 exponent bits, 3 mantissa bits, largest number 448) with an fp32 scale for each block of 128: the
// quantiser, and the product of quantised operands.
#include "fp8_block.h"

#include <algorithm>
#include <utility>

#include "tile_gemm.h"

namespace vecops_hip {

namespace {

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

// ---------------------------------------------------------------------------------------------------------------------
// Quantiser.  s = max(amax / 448, 2^-126), q = e4m3(x / s), both divisions correctly rounded, then to the nearest e4m3, ties
// to even.  The maximum is taken on the bits of |x|, so that a NaN in a block makes its scale NaN and an infinity makes it
// infinite: what is not finite stays visible in every product with the block.
// ---------------------------------------------------------------------------------------------------------------------

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

// Eight consecutive elements of a row from k on as fp32; those past K are zeros.  `whole`: they are contiguous and all there.
template <int KIND>
__device__ __forceinline__ void load_eight(const Fp8QuantizeParams& p, int64_t at, int k, bool whole, float (&v)[8]) {
  if constexpr (KIND == FP8_REAL_F32) {
    const VECOPS_GLOBAL float* x = (const VECOPS_GLOBAL float*)p.x + at;
    if (whole) {
      const u32x4 lo = load_16(x), hi = load_16(x + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = __uint_as_float(lo[e]);
        v[4 + e] = __uint_as_float(hi[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = k + e < p.k ? x[e * p.x_cs] : 0.0f;
    }
  } else {
    const VECOPS_GLOBAL uint16_t* x = (const VECOPS_GLOBAL uint16_t*)p.x + at;
    if (whole) {
      const u32x4 w = load_16(x);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = real_bits_to_f32((w[e >> 1] >> (16 * (e & 1))) & 0xffffu, KIND);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = k + e < p.k ? real_bits_to_f32(x[e * p.x_cs], KIND) : 0.0f;
    }
  }
}

__device__ __forceinline__ uint32_t most_of(const float (&v)[8], uint32_t most) {
#pragma unroll
  for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
  return most;
}

__device__ __forceinline__ void store_eight(const Fp8QuantizeParams& p, int64_t at, int k, bool whole, const float (&v)[8], const Quotient& by) {
  const u32x2 q = {pack_e4m3(by(v[0]), by(v[1]), by(v[2]), by(v[3])), pack_e4m3(by(v[4]), by(v[5]), by(v[6]), by(v[7]))};
  if (whole) {
    *(VECOPS_GLOBAL u32x2_anywhere*)((VECOPS_GLOBAL uint8_t*)p.q + at) = q;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < p.k) ((VECOPS_GLOBAL uint8_t*)p.q)[at + e * p.q_cs] = static_cast<uint8_t>(q[e >> 2] >> (8 * (e & 3)));
  }
}

// A scale for each 128 of a row: sixteen lanes a block, eight elements a lane.  Bound by HBM.
template <int KIND>
__global__ __launch_bounds__(256) void fp8_quantize_rows_kernel(const Fp8QuantizeParams p, uint32_t blocks) {
  for (uint32_t block = blockIdx.x * 16u + (threadIdx.x >> 4); block < blocks; block += gridDim.x * 16u) {   // (the same for sixteen lanes)
    const uint32_t line = block / static_cast<uint32_t>(p.groups), g = block - line * p.groups;
    const uint32_t batch = line / static_cast<uint32_t>(p.rows), row = line - batch * p.rows;
    const int k = static_cast<int>(g) * kFp8Block + (threadIdx.x & 15) * 8;
    const bool there = k + 8 <= p.k;
    float v[8];
    load_eight<KIND>(p, batch * p.x_bs + row * p.x_rs + k * p.x_cs, k, there && p.x_cs == 1, v);
    uint32_t most = most_of(v, 0u);
#pragma unroll
    for (int d = 1; d < 16; d *= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d, 16)));
    const float s = block_scale(most);
    store_eight(p, batch * p.q_bs + row * p.q_rs + k * p.q_cs, k, there && p.q_cs == 1, v, Quotient(s));
    if ((threadIdx.x & 15) == 0) p.scales[batch * p.s_bs + row * p.s_rs + g * p.s_cs] = s;
  }
}

// A scale for each block of 128 x 128: a workgroup a block, which stays in its registers between the maximum and the
// quotients.  Bound by HBM.
template <int KIND>
__global__ __launch_bounds__(256) void fp8_quantize_tiles_kernel(const Fp8QuantizeParams p, uint32_t row_blocks) {
  __shared__ uint32_t meet[4];
  const uint32_t line = blockIdx.x / static_cast<uint32_t>(p.groups), g = blockIdx.x - line * p.groups;
  const uint32_t batch = line / row_blocks, i = line - batch * row_blocks;
  const int k = static_cast<int>(g) * kFp8Block + (threadIdx.x & 15) * 8;
  const bool there = k + 8 <= p.k;
  float v[8][8];
  uint32_t most = 0;
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const int64_t row = static_cast<int64_t>(i) * kFp8Block + t * 16 + (threadIdx.x >> 4);
    if (row < p.rows) {
      load_eight<KIND>(p, batch * p.x_bs + row * p.x_rs + k * p.x_cs, k, there && p.x_cs == 1, v[t]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[t][e] = 0.0f;
    }
  }
#pragma unroll
  for (int t = 0; t < 8; ++t) most = most_of(v[t], most);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d, 64)));
  if ((threadIdx.x & 63) == 0) meet[threadIdx.x >> 6] = most;
  __syncthreads();
  most = max(max(meet[0], meet[1]), max(meet[2], meet[3]));
  const float s = block_scale(most);
  const Quotient by(s);
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const int64_t row = static_cast<int64_t>(i) * kFp8Block + t * 16 + (threadIdx.x >> 4);
    if (row < p.rows) store_eight(p, batch * p.q_bs + row * p.q_rs + k * p.q_cs, k, there && p.q_cs == 1, v[t], by);
  }
  if (threadIdx.x == 0) p.scales[batch * p.s_bs + i * p.s_rs + g * p.s_cs] = s;
}

// Rows whose k are not contiguous, laid out so that they are: 64 x 64 elements through LDS, each side in its own order.
__global__ __launch_bounds__(256) void fp8_rows_kernel(const uint8_t* in, int64_t bs, int64_t rs, int64_t cs, uint8_t* out, int64_t ld,
                                                       int32_t rows, int32_t k, uint32_t tiles_k) {
  __shared__ uint8_t tile[64][68];
  const uint32_t row_tile = blockIdx.x / tiles_k;
  const int64_t r0 = static_cast<int64_t>(row_tile) * 64, k0 = static_cast<int64_t>(blockIdx.x - row_tile * tiles_k) * 64;
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  in += blockIdx.y * bs;
  out += static_cast<int64_t>(blockIdx.y) * rows * ld;
  for (int i = y; i < 64; i += 4)   // consecutive lanes: consecutive rows (the contiguous side of a [K, rows] matrix)
    if (r0 + x < rows && k0 + i < k) tile[x][i] = in[(r0 + x) * rs + (k0 + i) * cs];
  __syncthreads();
  for (int i = y; i < 64; i += 4)
    if (r0 + i < rows && k0 + x < k) out[(r0 + i) * ld + k0 + x] = tile[i][x];
}

// ---------------------------------------------------------------------------------------------------------------------
// Product.  c[m,n] = sum_g (sa[m,g] sb[n/128,g]) (sum_{k in g} a[m,k] b[n,k]): matrix instructions give the inner sums of 16 x 16
// results over one block of 128 from a zero accumulator; an fp32 fused multiply-add a result puts them, scaled, onto the outer
// sum.  Weights are the instruction's rows and activations its columns: lane l holds results n = 4 (l / 16) + 0..3 of
// activation row l % 16, so that its scale is one number a block.  Each lane's 32 bytes of an operand are two chunks of 16: any
// order of k does, if it is the same on both sides.
//
// Two ways to an inner sum.  v_mfma_f32_16x16x128_f8f6f4 takes the bytes as they are, at 2.8 times the rate of bf16 (random
// bytes, nothing but the instruction: 3200 TFLOP/s, bf16 1145).  It aligns each eight products that lie together along k to
// the largest of them and drops what is 2^-13 of its power of two or less (2^16 + 2^2 gave 2^16, 2^16 + 2^3 was exact; across
// eights nothing is lost): on normally distributed operands results are 1.4e-5 off, which a 16-bit result does not show (its
// own rounding: bf16 1.7e-3, f16 2.1e-4).  For fp32 results, and for few rows, where the rate does not count, the bytes are
// widened to bf16, exactly, and the bf16 instruction sums exact products in fp32.
// ---------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ f32x4 mfma_e4m3(const i32x8& w, const i32x8& x) {
  // (scale exponents that are the constant zero select the instruction without scales; formats 0 are e4m3)
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// Eight e4m3 bytes as eight bf16 (exact).
__device__ __forceinline__ u32x4 widen(int lo, int hi) {
#if defined(__HIP_DEVICE_COMPILE__)
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true))};
#else
  (void)lo; (void)hi;
  return u32x4{0u, 0u, 0u, 0u};
#endif
}

// A lane's 32 bytes of an operand, as the instruction of a kernel takes them.
template <bool WIDE>
struct Fragment;
template <>
struct Fragment<false> {
  i32x8 v;
  __device__ __forceinline__ explicit Fragment(const i32x8& bytes) : v(bytes) {}
  __device__ __forceinline__ f32x4 dot(const Fragment& x) const { return mfma_e4m3(v, x.v); }
};
template <>
struct Fragment<true> {
  u32x4 v[4];
  __device__ __forceinline__ explicit Fragment(const i32x8& bytes) {
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = widen(bytes[2 * c], bytes[2 * c + 1]);
  }
  __device__ __forceinline__ f32x4 dot(const Fragment& x) const {
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 4; ++c)
      sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v[c]), __builtin_bit_cast(bf16x8, x.v[c]), sum, 0, 0, 0);
    return sum;
  }
};

__device__ __forceinline__ i32x8 fragment_of(const u32x4& lo, const u32x4& hi) {
  return i32x8{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(lo[2]), static_cast<int>(lo[3]),
               static_cast<int>(hi[0]), static_cast<int>(hi[1]), static_cast<int>(hi[2]), static_cast<int>(hi[3])};
}

template <bool WIDE, int COUNT>
struct Fragments {
  Fragment<WIDE> v[COUNT];
};
template <bool WIDE, int COUNT, int... I>
__device__ __forceinline__ Fragments<WIDE, COUNT> fragments(const i32x8 (&bytes)[COUNT], std::integer_sequence<int, I...>) {
  return {{Fragment<WIDE>(bytes[I])...}};
}
template <bool WIDE, int COUNT>
__device__ __forceinline__ Fragments<WIDE, COUNT> fragments(const i32x8 (&bytes)[COUNT]) {
  return fragments<WIDE>(bytes, std::make_integer_sequence<int, COUNT>{});
}

// Sixteen bytes of a row from `k` on, zeros past K; reads nothing past the row's last byte.
__device__ __forceinline__ u32x4 load_chunk_until(const VECOPS_GLOBAL uint8_t* row, int k, int k_end) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if (k + 16 <= k_end) {
    v = load_16(row + k);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (k + e < k_end) v[e >> 2] |= static_cast<uint32_t>(row[k + e]) << (8 * (e & 3));
  }
  return v;
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

// One 4-byte load per lane that writes LDS itself (as load_16_bytes_into_lds).
__device__ __forceinline__ void load_4_bytes_into_lds(const u32x4& descriptor, uint32_t address, uint32_t lane_offset, uint32_t uniform_offset) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
               :
               : "s"(address), "v"(lane_offset), "s"(descriptor), "s"(uniform_offset)
               : "memory", "m0");
#else
  (void)descriptor; (void)address; (void)lane_offset; (void)uniform_offset;
#endif
}

typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) float lds_float;

__device__ __forceinline__ u32x4 read_lds(uint32_t at) { return *reinterpret_cast<const lds_u32x4*>(static_cast<uintptr_t>(at)); }
__device__ __forceinline__ float read_lds_float(uint32_t at) { return *reinterpret_cast<const lds_float*>(static_cast<uintptr_t>(at)); }

// Many rows: WN x WM wavefronts, each NT x MT blocks of 16 x 16.  A stage is one block of 128 k of both operands and the
// activations' scales; it arrives by loads that write LDS while the stage before it is multiplied.
// The rows of a wavefront's weights are dealt to its 16-row blocks so that a lane's results of two blocks are eight
// consecutive n (row r of block 2 p + h is n = 32 p + 8 (r / 4) + 4 h + r % 4): sixteen bytes of a 16-bit result a store.
template <int WN, int WM, int NT, int MT>
struct Fp8Tile {
  static constexpr int kBN = WN * NT * 16, kBM = WM * MT * 16, kThreads = 64 * WN * WM;
  static constexpr int kBytesW = kBN * 128, kBytesX = kBM * 128;
  // behind the operands: the scales of the kBM activation rows, and those of the tile's weight blocks in 64 places
  static constexpr int kScalesX = kBytesW + kBytesX, kScalesW = kScalesX + kBM * 4, kStage = kScalesW + 256;
  static constexpr int kLoadsW = kBytesW / (kThreads * 16), kLoadsX = kBytesX / (kThreads * 16);
  static_assert(kBM % 64 == 0 && kThreads >= kBM + 64, "a wavefront loads scales of 64 rows, another those of the weights");
  static_assert(NT % 2 == 0 && 128 % (NT * 16) == 0 && kBN % 8 == 0, "a wavefront's weights share their scale");
  static_assert(kBytesW % (kThreads * 16) == 0 && kBytesX % (kThreads * 16) == 0, "whole loads");
};

// slot of a chunk in its row of 128 bytes: rows that a fragment reads together lie in different slots
__device__ __forceinline__ int slot_key_w(int row) { return (row & 3) | ((row >> 1) & 4); }
__device__ __forceinline__ int slot_key_x(int row) { return row & 7; }

template <int WN, int WM, int NT, int MT, bool WIDE>
__global__ __launch_bounds__(64 * WN * WM, 2) void fp8_tile_kernel(const Fp8MatmulParams p, uint32_t tiles_n, uint32_t tiles_m) {
  using T = Fp8Tile<WN, WM, NT, MT>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lds0 = lds_address_of(lds);
  const int batch = blockIdx.y;

  // neighbouring tiles on one die: each die's workgroups (every eighth) take a contiguous run of tiles, walked in groups of
  // eight tile rows
  uint32_t pid = blockIdx.x;
  {
    const uint32_t total = tiles_n * tiles_m, xcd = pid & 7, share = total >> 3, extra = total & 7;
    pid = xcd * share + min(xcd, extra) + (pid >> 3);
  }
  const uint32_t per_group = 8 * tiles_n, group = pid / per_group, first = group * 8;
  const uint32_t height = min(tiles_m - first, 8u), in_group = pid - group * per_group;
  const uint32_t tile_m = first + in_group % height, tile_n = in_group / height;
  const int64_t m0 = static_cast<int64_t>(tile_m) * T::kBM, n0 = static_cast<int64_t>(tile_n) * T::kBN;
  const int last_m = static_cast<int>(min(p.m - m0, static_cast<int64_t>(T::kBM))) - 1, last_n = static_cast<int>(min(p.n - n0, static_cast<int64_t>(T::kBN))) - 1;

  const VECOPS_GLOBAL uint8_t* w_base = (const VECOPS_GLOBAL uint8_t*)p.b + batch * p.b_bs + n0 * p.ldb;
  const VECOPS_GLOBAL uint8_t* x_base = (const VECOPS_GLOBAL uint8_t*)p.a + batch * p.a_bs + m0 * p.lda;
  const VECOPS_GLOBAL float* sx_base = (const VECOPS_GLOBAL float*)p.a_scales + batch * p.as_bs + m0 * p.as_rs;
  const u32x4 desc_w = tile_buffer_words((const VECOPS_GLOBAL char*)w_base);
  const u32x4 desc_x = tile_buffer_words((const VECOPS_GLOBAL char*)x_base);

  // load i of a thread: sixteen bytes of row i * threads / 8 + tid / 8, the chunk whose slot is tid % 8
  uint32_t from_w[T::kLoadsW], from_x[T::kLoadsX];
#pragma unroll
  for (int i = 0; i < T::kLoadsW; ++i) {
    const int row = i * (T::kThreads / 8) + (tid >> 3);
    from_w[i] = static_cast<uint32_t>(min(row, last_n) * p.ldb) + (((tid & 7) ^ slot_key_w(row)) << 4);
  }
#pragma unroll
  for (int i = 0; i < T::kLoadsX; ++i) {
    const int row = i * (T::kThreads / 8) + (tid >> 3);
    from_x[i] = static_cast<uint32_t>(min(row, last_m) * p.lda) + (((tid & 7) ^ slot_key_x(row)) << 4);
  }
  // scales: the first wavefronts load those of the activations, 64 rows each, the next one those of the weights
  const bool loads_sw = wave == T::kBM / 64;
  const int64_t scale_row0 = n0 / kFp8Block, last_scale_row = (static_cast<int64_t>(p.n) - 1) / kFp8Block - scale_row0;
  const VECOPS_GLOBAL float* s_base = loads_sw ? (const VECOPS_GLOBAL float*)p.b_scales + batch * p.bs_bs + scale_row0 * p.bs_rs : sx_base;
  const int64_t s_step = loads_sw ? p.bs_gs : p.as_gs;
  const uint32_t from_s = loads_sw ? static_cast<uint32_t>(min(static_cast<int64_t>(min(lane, T::kBN / kFp8Block)), last_scale_row) * p.bs_rs * 4)
                                   : static_cast<uint32_t>(min(tid, last_m) * p.as_rs * 4);

  auto issue = [&](int g) {
    const uint32_t stage = lds0 + (g & 1) * T::kStage;
    const int k0 = g * kFp8Block;
    if (k0 + kFp8Block <= p.k) {
#pragma unroll
      for (int i = 0; i < T::kLoadsW; ++i)
        load_16_bytes_into_lds(desc_w, stage, __builtin_amdgcn_readfirstlane(i * (T::kThreads * 16) + wave * 1024), from_w[i],
                               __builtin_amdgcn_readfirstlane(k0));
#pragma unroll
      for (int i = 0; i < T::kLoadsX; ++i)
        load_16_bytes_into_lds(desc_x, stage, __builtin_amdgcn_readfirstlane(T::kBytesW + i * (T::kThreads * 16) + wave * 1024),
                               from_x[i], __builtin_amdgcn_readfirstlane(k0));
    } else {  // the last, partial block: through registers, byte by byte where K ends
#pragma unroll
      for (int i = 0; i < T::kLoadsW; ++i) {
        const int row = i * (T::kThreads / 8) + (tid >> 3), chunk = (tid & 7) ^ slot_key_w(row);
        const u32x4 v = load_chunk_until(w_base + min(row, last_n) * p.ldb, k0 + chunk * 16, p.k);
        *reinterpret_cast<lds_u32x4*>(static_cast<uintptr_t>(stage + i * (T::kThreads * 16) + tid * 16)) = v;
      }
#pragma unroll
      for (int i = 0; i < T::kLoadsX; ++i) {
        const int row = i * (T::kThreads / 8) + (tid >> 3), chunk = (tid & 7) ^ slot_key_x(row);
        const u32x4 v = load_chunk_until(x_base + min(row, last_m) * p.lda, k0 + chunk * 16, p.k);
        *reinterpret_cast<lds_u32x4*>(static_cast<uintptr_t>(stage + T::kBytesW + i * (T::kThreads * 16) + tid * 16)) = v;
      }
    }
    if (wave <= T::kBM / 64)
      load_4_bytes_into_lds(tile_buffer_words((const VECOPS_GLOBAL char*)(s_base + g * s_step)),
                            __builtin_amdgcn_readfirstlane(stage + T::kScalesX + wave * 256), from_s, 0);
  };

  const int wn = wave / WM, wm = wave % WM;
  const int col = lane & 15, quarter = lane >> 4;
  uint32_t at_w[2], at_x[2];   // a lane's two chunks of its row in block 0 (blocks apart by whole rows of equal keys)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int chunk = quarter + 4 * h;
    const int row_w = wn * (NT * 16) + 8 * (col >> 2) + (col & 3), row_x = wm * (MT * 16) + col;
    at_w[h] = lds0 + row_w * 128 + ((chunk ^ slot_key_w(row_w)) << 4);
    at_x[h] = lds0 + T::kBytesW + row_x * 128 + ((chunk ^ slot_key_x(row_x)) << 4);
  }
  const uint32_t at_sx = lds0 + T::kScalesX + (wm * (MT * 16) + col) * 4;
  const uint32_t at_sw = lds0 + T::kScalesW + static_cast<uint32_t>((n0 + wn * (NT * 16)) / kFp8Block - scale_row0) * 4;

  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (p.groups > 0) issue(0);
  for (int g = 0; g < p.groups; ++g) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // this stage has landed
    __builtin_amdgcn_s_barrier();                                 // and every wavefront has left the one before it
    asm volatile("" ::: "memory");
    if (g + 1 < p.groups) issue(g + 1);
    const uint32_t stage = (g & 1) * T::kStage;
    const float sw = read_lds_float(at_sw + stage);
    float scale[MT];
    i32x8 xb[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      xb[j] = fragment_of(read_lds(at_x[0] + stage + j * 2048), read_lds(at_x[1] + stage + j * 2048));
      scale[j] = read_lds_float(at_sx + stage + j * 64) * sw;
    }
    const auto x = fragments<WIDE>(xb);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      // block 2 p + h starts 32 p + 4 h rows down; 4 rows down the key stays
      const uint32_t down = stage + (i >> 1) * 4096 + (i & 1) * 512;
      const Fragment<WIDE> w(fragment_of(read_lds(at_w[0] + down), read_lds(at_w[1] + down)));
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const f32x4 part = w.dot(x.v[j]);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(part[r], scale[j], acc[i][j][r]);
      }
    }
  }

#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int64_t m = m0 + wm * (MT * 16) + j * 16 + col;
    if (m < p.m) {
#pragma unroll
      for (int i = 0; i < NT; i += 2) {
        const int64_t n = n0 + wn * (NT * 16) + i * 16 + quarter * 8;
        const float v[8] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3],
                            acc[i + 1][j][0], acc[i + 1][j][1], acc[i + 1][j][2], acc[i + 1][j][3]};
        store_results<8>(p.c, batch * p.c_bs + m * p.c_rs + n * p.c_cs, p.c_cs, p.out_kind, n, p.n, v);
      }
    }
  }
}

// Few rows (m <= 16 MT): bound by HBM.  A workgroup owns 16 NT weight rows and all m; its wavefronts take the blocks of k in
// turn, loads of DEPTH blocks under way in each, and their sums meet in LDS.  The scales sa sb of a run of blocks are
// multiplied beforehand into a table in LDS.
template <int NT, int MT, int WAVES, int DEPTH>
__global__ __launch_bounds__(64 * WAVES) void fp8_skinny_kernel(const Fp8MatmulParams p) {
  constexpr int RUN = 128, ROWS = MT * 16;
  constexpr int kTable = RUN * ROWS, kSums = WAVES * NT * MT * 256;
  __shared__ float shared[kTable > kSums ? kTable : kSums];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quarter = lane >> 4;
  const int batch = blockIdx.y;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * NT);
  const VECOPS_GLOBAL uint8_t *w[NT], *x[MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
    w[i] = (const VECOPS_GLOBAL uint8_t*)p.b + batch * p.b_bs + min(n0 + i * 16 + col, static_cast<int64_t>(p.n) - 1) * p.ldb;
#pragma unroll
  for (int j = 0; j < MT; ++j) x[j] = (const VECOPS_GLOBAL uint8_t*)p.a + batch * p.a_bs + static_cast<int64_t>(min(j * 16 + col, p.m - 1)) * p.lda;

  u32x4 wv[DEPTH][NT][2], xv[DEPTH][MT][2];
  auto load = [&](auto slot_tag, int g) {
    constexpr int slot = decltype(slot_tag)::value;
    if (g >= p.groups) return;
    const int k0 = g * kFp8Block + quarter * 16;
    if ((g + 1) * kFp8Block <= p.k) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < NT; ++i) wv[slot][i][h] = load_16(w[i] + k0 + 64 * h);
#pragma unroll
        for (int j = 0; j < MT; ++j) xv[slot][j][h] = load_16(x[j] + k0 + 64 * h);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < NT; ++i) wv[slot][i][h] = load_chunk_until(w[i], k0 + 64 * h, p.k);
#pragma unroll
        for (int j = 0; j < MT; ++j) xv[slot][j][h] = load_chunk_until(x[j], k0 + 64 * h, p.k);
      }
    }
  };
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const VECOPS_GLOBAL float* sx_base = (const VECOPS_GLOBAL float*)p.a_scales + batch * p.as_bs;
  const VECOPS_GLOBAL float* sw_base = (const VECOPS_GLOBAL float*)p.b_scales + batch * p.bs_bs + n0 / kFp8Block * p.bs_rs;  // (16 NT divides 128)
  for (int run = 0; run < p.groups; run += RUN) {
    const int end = min(run + RUN, p.groups);
    constexpr int ENTRIES = RUN * ROWS / (64 * WAVES);
    float sx[ENTRIES], sw[ENTRIES];
#pragma unroll
    for (int e = 0; e < ENTRIES; ++e) {   // (in front of the operands' loads, which the table then does not wait for)
      const int at = e * (64 * WAVES) + tid, g = run + at / ROWS, m = min(at % ROWS, p.m - 1);
      if (g < end) {
        sx[e] = sx_base[m * p.as_rs + g * p.as_gs];
        sw[e] = sw_base[g * p.bs_gs];
      }
    }
    static_for<DEPTH>([&](auto u) { load(u, run + wave + decltype(u)::value * WAVES); });
    if (run > 0) __syncthreads();   // the table's last readers are done
#pragma unroll
    for (int e = 0; e < ENTRIES; ++e) {
      const int at = e * (64 * WAVES) + tid;
      if (run + at / ROWS < end) shared[at] = sx[e] * sw[e];
    }
    __syncthreads();
    for (int g0 = run + wave; g0 < end; g0 += DEPTH * WAVES) {
      static_for<DEPTH>([&](auto u) {
        constexpr int slot = decltype(u)::value;
        const int g = g0 + slot * WAVES;
        if (g < end) {
          i32x8 wb[NT];
#pragma unroll
          for (int i = 0; i < NT; ++i) wb[i] = fragment_of(wv[slot][i][0], wv[slot][i][1]);
          const auto wf = fragments<true>(wb);
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            const float scale = shared[(g - run) * ROWS + j * 16 + col];
            const Fragment<true> xf(fragment_of(xv[slot][j][0], xv[slot][j][1]));
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              const f32x4 part = wf.v[i].dot(xf);
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(part[r], scale, acc[i][j][r]);
            }
          }
          if (g + DEPTH * WAVES < end) load(u, g + DEPTH * WAVES);
        }
      });
    }
  }

  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4*>(&shared[((wave * NT + i) * MT + j) * 256 + lane * 4]) = acc[i][j];
  __syncthreads();
  for (int at = wave; at < NT * MT; at += WAVES) {
    const int i = at / MT, j = at % MT;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < WAVES; ++u) {
      const f32x4 part = *reinterpret_cast<const f32x4*>(&shared[((u * NT + i) * MT + j) * 256 + lane * 4]);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += part[r];
    }
    const int m = j * 16 + col;
    const int64_t n = n0 + i * 16 + quarter * 4;
    if (m < p.m && n < p.n) store_results<4>(p.c, batch * p.c_bs + m * p.c_rs + n * p.c_cs, p.c_cs, p.out_kind, n, p.n, v);
  }
}

template <int NT, int MT, int WAVES, int DEPTH>
hipError_t launch_skinny(const Fp8MatmulParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>((p.n + 16 * NT - 1) / (16 * NT)), static_cast<uint32_t>(p.batch));
  hipLaunchKernelGGL((fp8_skinny_kernel<NT, MT, WAVES, DEPTH>), grid, dim3(64 * WAVES), 0, stream, p);
  return hipGetLastError();
}

template <int WN, int WM, int NT, int MT, bool WIDE>
hipError_t launch_tile(const Fp8MatmulParams& p, hipStream_t stream) {
  using T = Fp8Tile<WN, WM, NT, MT>;
  const void* kernel = reinterpret_cast<const void*>(&fp8_tile_kernel<WN, WM, NT, MT, WIDE>);
  if constexpr (2 * T::kStage > 65536) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 2 * T::kStage);
    if (e != hipSuccess) return e;
  }
  const uint32_t tiles_n = static_cast<uint32_t>((p.n + T::kBN - 1) / T::kBN), tiles_m = static_cast<uint32_t>((p.m + T::kBM - 1) / T::kBM);
  hipLaunchKernelGGL((fp8_tile_kernel<WN, WM, NT, MT, WIDE>), dim3(tiles_n * tiles_m, static_cast<uint32_t>(p.batch)), dim3(T::kThreads),
                     2 * T::kStage, stream, p, tiles_n, tiles_m);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_fp8_quantize(const Fp8QuantizeParams& p, int block_rows, hipStream_t stream) {
  if (block_rows == 1) {
    const uint32_t blocks = static_cast<uint32_t>(static_cast<int64_t>(p.batch) * p.rows * p.groups);
    const dim3 grid(std::min((blocks + 15) / 16, 1u << 22));
    if (p.kind == FP8_REAL_BF16) hipLaunchKernelGGL((fp8_quantize_rows_kernel<FP8_REAL_BF16>), grid, dim3(256), 0, stream, p, blocks);
    else if (p.kind == FP8_REAL_F16) hipLaunchKernelGGL((fp8_quantize_rows_kernel<FP8_REAL_F16>), grid, dim3(256), 0, stream, p, blocks);
    else hipLaunchKernelGGL((fp8_quantize_rows_kernel<FP8_REAL_F32>), grid, dim3(256), 0, stream, p, blocks);
  } else {
    const uint32_t row_blocks = static_cast<uint32_t>((p.rows + kFp8Block - 1) / kFp8Block);
    const dim3 grid(static_cast<uint32_t>(p.batch) * row_blocks * static_cast<uint32_t>(p.groups));
    if (p.kind == FP8_REAL_BF16) hipLaunchKernelGGL((fp8_quantize_tiles_kernel<FP8_REAL_BF16>), grid, dim3(256), 0, stream, p, row_blocks);
    else if (p.kind == FP8_REAL_F16) hipLaunchKernelGGL((fp8_quantize_tiles_kernel<FP8_REAL_F16>), grid, dim3(256), 0, stream, p, row_blocks);
    else hipLaunchKernelGGL((fp8_quantize_tiles_kernel<FP8_REAL_F32>), grid, dim3(256), 0, stream, p, row_blocks);
  }
  return hipGetLastError();
}

hipError_t launch_fp8_rows(const uint8_t* in, int64_t bs, int64_t rs, int64_t cs, uint8_t* out, int64_t ld, int32_t batch,
                           int32_t rows, int32_t k, hipStream_t stream) {
  const uint32_t tiles_k = static_cast<uint32_t>((static_cast<int64_t>(k) + 63) / 64), tiles_r = static_cast<uint32_t>((static_cast<int64_t>(rows) + 63) / 64);
  hipLaunchKernelGGL(fp8_rows_kernel, dim3(tiles_r * tiles_k, static_cast<uint32_t>(batch)), dim3(256), 0, stream, in, bs, rs, cs, out, ld,
                     rows, k, tiles_k);
  return hipGetLastError();
}

hipError_t launch_fp8_matmul(const Fp8MatmulParams& p, hipStream_t stream) {
  if (p.m <= 16) return launch_skinny<1, 1, 8, 4>(p, stream);
  if (p.m <= 32) return launch_skinny<1, 2, 8, 4>(p, stream);
  if (p.m <= 64) return launch_skinny<2, 4, 8, 2>(p, stream);
  if (p.out_kind == FP8_REAL_F32) return launch_tile<2, 2, 4, 4, true>(p, stream);
  const int64_t tiles_256 = ((static_cast<int64_t>(p.m) + 255) / 256) * ((static_cast<int64_t>(p.n) + 255) / 256) * p.batch;
  if (tiles_256 >= 256) return launch_tile<2, 4, 8, 4, false>(p, stream);
  return launch_tile<2, 2, 4, 4, false>(p, stream);
}

}  // namespace vecops_hip
