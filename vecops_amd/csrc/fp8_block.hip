// 8-bit floats (e4m3: 4 exponent bits, 3 mantissa bits, largest number 448) with an fp32 scale for each block of 128: the
// quantiser, and the product of quantised operands.
#include "fp8_block.h"

#include <algorithm>
#include <utility>

#include "lane_exchange.h"

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
// quotients.  Bound by HBM.  Workgroups go to the eight dies in turn, each with a cache of its own; with `runs`, of a grid of a
// multiple of eight every die takes a run of neighbouring blocks, so that the lines that two blocks share meet in one cache.
template <int KIND>
__global__ __launch_bounds__(256) void fp8_quantize_tiles_kernel(const Fp8QuantizeParams p, uint32_t row_blocks, bool runs) {
  __shared__ uint32_t meet[4];
  const uint32_t block = runs ? (blockIdx.x & 7u) * (gridDim.x >> 3) + (blockIdx.x >> 3) : blockIdx.x, line = block / static_cast<uint32_t>(p.groups), g = block - line * p.groups;
  const uint32_t batch = line / row_blocks, i = line - batch * row_blocks;
  if (batch >= static_cast<uint32_t>(p.batch)) return;
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

// Scales whose blocks of k do not follow one another, laid out so that they do.
__global__ __launch_bounds__(256) void fp8_scales_kernel(const float* in, int64_t bs, int64_t rs, int64_t gs, float* out, int64_t total, int32_t rows,
                                                         int32_t groups) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= total) return;
  const int64_t row = at % rows, line = at / rows;   // (consecutive lanes: consecutive rows)
  const int64_t g = line % groups, batch = line / groups;
  out[(batch * rows + row) * groups + g] = in[batch * bs + row * rs + g * gs];
}

// Rows whose k are not contiguous, or few, laid out so that they are, with zeros up to `ld`: 64 x 64 elements through LDS, each
// side in its own order.
__global__ __launch_bounds__(256) void fp8_rows_kernel(const uint8_t* in, int64_t bs, int64_t rs, int64_t cs, uint8_t* out, int64_t ld,
                                                       int32_t rows, int32_t k, uint32_t tiles_k) {
  __shared__ uint8_t tile[64][68];
  const uint32_t row_tile = blockIdx.x / tiles_k;
  const int64_t r0 = static_cast<int64_t>(row_tile) * 64, k0 = static_cast<int64_t>(blockIdx.x - row_tile * tiles_k) * 64;
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  in += blockIdx.y * bs;
  out += static_cast<int64_t>(blockIdx.y) * rows * ld;
  for (int i = y; i < 64; i += 4)   // consecutive lanes: consecutive rows (the contiguous side of a [K, rows] matrix)
    tile[x][i] = r0 + x < rows && k0 + i < k ? in[(r0 + x) * rs + (k0 + i) * cs] : 0;
  __syncthreads();
  for (int i = y; i < 64; i += 4)
    if (r0 + i < rows && k0 + x < ld) out[(r0 + i) * ld + k0 + x] = tile[i][x];
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
// the largest of them and drops what is below 2^-13 of its power of two (2^16 + 2^2 gave 2^16, 2^16 + 2^3 was exact; across
// eights nothing is lost): on normally distributed operands results are 1.4e-5 off, which a 16-bit result does not show (its
// own rounding: bf16 1.7e-3, f16 2.1e-4); a sum that cancels can be off by up to 7 * 2^-13 of its terms' sizes.  For fp32 results the bytes are widened to bf16, exactly, and the bf16
// instruction sums exact products in fp32.
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

typedef __attribute__((address_space(3))) char lds_char;

// (`offset`, a constant, goes into the instruction)
__device__ __forceinline__ u32x4 read_lds(uint32_t at, int offset) {
  return *reinterpret_cast<const lds_u32x4*>(reinterpret_cast<const lds_char*>(static_cast<uintptr_t>(at)) + offset);
}
__device__ __forceinline__ float read_lds_float(uint32_t at, int offset) {
  return *reinterpret_cast<const lds_float*>(reinterpret_cast<const lds_char*>(static_cast<uintptr_t>(at)) + offset);
}

// Many rows: WN x WM wavefronts, each NT x MT blocks of 16 x 16.  A stage is one block of 128 k of both operands and their
// scales; STAGES of them are under way or in use, by loads that write LDS.
// The rows of a wavefront's weights are dealt to its 16-row blocks so that a lane's results of two blocks are eight
// consecutive n (row r of block 2 p + h is n = 32 p + 8 (r / 4) + 4 h + r % 4): sixteen bytes of a 16-bit result a store.
template <int WN, int WM, int NT, int MT, int STAGES>
struct Fp8Tile {
  static constexpr int kBN = WN * NT * 16, kBM = WM * MT * 16, kWaves = WN * WM, kThreads = 64 * kWaves;
  static constexpr int kBytesW = kBN * 128, kBytesX = kBM * 128;
  static constexpr int kStage = kBytesW + kBytesX;
  // Scales arrive four blocks of k at a time (sixteen bytes of each row: a line holds many blocks' scales of one row): the first
  // wavefronts load those of 64 activation rows each, the others those of the weights' blocks.  In three of four stages the
  // load fetches nothing and writes where nobody reads, so that all wavefronts have the same number of loads under way.
  // Of four runs' places one is free again by the time that its next run is asked for, up to twelve stages ahead.
  static constexpr int kRuns = 4, kRunX = kBM * 16, kRunW = 1024;
  static constexpr int kScalesX = STAGES * kStage, kScalesW = kScalesX + kRuns * kRunX, kNobody = kScalesW + kRuns * kRunW, kLds = kNobody + 1024;
  static constexpr int kLoadsW = kBytesW / (kThreads * 16), kLoadsX = kBytesX / (kThreads * 16), kLoads = kLoadsW + kLoadsX + 1;
  static_assert(kBM % 64 == 0 && kWaves > kBM / 64 && STAGES <= 12, "wavefronts to load all scales, and room for them");
  static_assert(NT % 2 == 0 && 128 % (NT * 16) == 0, "a wavefront's weights share their scale");
  static_assert(kBytesW % (kThreads * 16) == 0 && kBytesX % (kThreads * 16) == 0, "whole loads");
  static_assert(kLds <= 160 * 1024 && STAGES >= 2 && (STAGES - 1) * kLoads < 64, "LDS of a compute unit; the counter of loads");
};

// slot of a chunk in its row of 128 bytes: rows that a fragment reads together lie in different slots
__device__ __forceinline__ int slot_key_w(int row) { return (row & 3) | ((row >> 1) & 4); }
__device__ __forceinline__ int slot_key_x(int row) { return row & 7; }

// What bounds the large tiles is the matrix pipe and the power it draws; a result's multiply-add every block of 128 takes half
// the vector unit's time beside it.  So the two run side by side: a block row's multiply-adds are issued while the next one's
// products are formed, and the stage is left, and the next one's first fragments are fetched, behind the last block row.
template <int WN, int WM, int NT, int MT, bool WIDE, int STAGES, bool HALVES>
__global__ __launch_bounds__(64 * WN * WM, 2) void fp8_tile_kernel(const Fp8MatmulParams p, uint32_t tiles_n, uint32_t tiles_m) {
  using T = Fp8Tile<WN, WM, NT, MT, STAGES>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lds0 = lds_address_of(lds);
  const int batch = blockIdx.y;
  // this workgroup's share of the blocks of k
  const int g_begin = static_cast<int>(static_cast<int64_t>(p.groups) * blockIdx.z / p.splits);
  const int g_end = static_cast<int>(static_cast<int64_t>(p.groups) * (blockIdx.z + 1) / p.splits);

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
  const int last_m = static_cast<int>(min(p.m - m0, static_cast<int64_t>(T::kBM))) - 1;
  const int last_n = static_cast<int>(min(p.n - n0, static_cast<int64_t>(T::kBN))) - 1;

  const VECOPS_GLOBAL uint8_t* w_base = (const VECOPS_GLOBAL uint8_t*)p.b + batch * p.b_bs + n0 * p.ldb;
  const VECOPS_GLOBAL uint8_t* x_base = (const VECOPS_GLOBAL uint8_t*)p.a + batch * p.a_bs + m0 * p.lda;
  u32x4 desc_w = tile_buffer_words((const VECOPS_GLOBAL char*)w_base);
  u32x4 desc_x = tile_buffer_words((const VECOPS_GLOBAL char*)x_base);
  // the last block of k, where K ends inside it: `tail` bytes of each row.  The chunk that K ends in is fetched as the sixteen
  // bytes in front of K (rows have at least sixteen): the same order of k on both sides, and the `again` bytes of it that the
  // chunk before it holds too are cleared on one side when they are read.
  const int tail = p.k % kFp8Block, again = tail % 16 ? 16 - tail % 16 : 0;

  // load i of a thread: sixteen bytes of row i * threads / 8 + tid / 8, the chunk whose slot is tid % 8 (rows apart by threads
  // / 8 have equal keys).  Rows past the operand's last one lie past the descriptor's end: zeros arrive.
  constexpr int kRows = T::kThreads / 8;
  static_assert(kRows % 16 == 0, "equal keys");
  constexpr uint32_t kNowhere = 0x80000000u;   // past every descriptor's end
  const int row = tid >> 3, chunk_w = ((tid & 7) ^ slot_key_w(row)) << 4, chunk_x = ((tid & 7) ^ slot_key_x(row)) << 4;
  const uint32_t from_w = static_cast<uint32_t>(row * p.ldb) + chunk_w, from_x = static_cast<uint32_t>(row * p.lda) + chunk_x;
  // (the tail's with their k: no part of an offset is negative.  Chosen without a branch: the loop below has to stay one block,
  // or the compiler gathers the multiply-adds behind it.)
  const uint32_t k_tail = static_cast<uint32_t>(p.groups - 1) * kFp8Block;
  const uint32_t tail_w = chunk_w + 16 <= tail ? from_w + k_tail : chunk_w < tail ? from_w + k_tail - (chunk_w + 16 - tail) : kNowhere;
  const uint32_t tail_x = chunk_x + 16 <= tail ? from_x + k_tail : chunk_x < tail ? from_x + k_tail - (chunk_x + 16 - tail) : kNowhere;
  const uint32_t end_w = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(last_n * p.ldb + p.k));
  const uint32_t end_x = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(last_m * p.lda + p.k));
  const uint32_t step_w = static_cast<uint32_t>(kRows * p.ldb), step_x = static_cast<uint32_t>(kRows * p.lda);
  const bool loads_sw = wave >= T::kBM / 64;
  const int64_t scale_row0 = n0 / kFp8Block, last_scale_row = (static_cast<int64_t>(p.n) - 1) / kFp8Block - scale_row0;
  u32x4 desc_s = tile_buffer_words((const VECOPS_GLOBAL char*)(loads_sw ? p.b_scales + batch * p.bs_bs + scale_row0 * p.bs_rs
                                                                        : p.a_scales + batch * p.as_bs + m0 * p.as_rs));
  const int64_t scale_rs = loads_sw ? p.bs_rs : p.as_rs, scale_rows = loads_sw ? min(static_cast<int64_t>(T::kBN / kFp8Block), last_scale_row) : last_m;
  const uint32_t from_s = static_cast<uint32_t>(min(static_cast<int64_t>(loads_sw ? lane : tid), scale_rows) * scale_rs * 4);
  const uint32_t end_s = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>((scale_rows * scale_rs + p.groups) * 4));
  const uint32_t to_s = __builtin_amdgcn_readfirstlane(loads_sw ? T::kScalesW : T::kScalesX + wave * 1024);
  const uint32_t run_shift = __builtin_amdgcn_readfirstlane(loads_sw ? 10 : T::kBM == 256 ? 12 : T::kBM == 128 ? 11 : 10);
  static_assert(T::kBM == 256 || T::kBM == 128 || T::kBM == 64, "the shift");

  // load PIECE of those that fill stage `slot` with block g (weights, activations, scales); past the last block nothing is
  // fetched (but as many loads are issued)
  auto issue_piece = [&](auto piece_tag, int g, int slot) {
    constexpr int PIECE = decltype(piece_tag)::value;
    const uint32_t stage = lds0 + slot * T::kStage;
    const bool there = g < g_end, at_tail = tail != 0 && g == p.groups - 1;
    const uint32_t k0 = at_tail ? 0u : static_cast<uint32_t>(g) * kFp8Block;
    if constexpr (PIECE < T::kLoadsW) {
      desc_w[2] = there ? end_w : 0u;
      load_16_bytes_into_lds(desc_w, stage, __builtin_amdgcn_readfirstlane(PIECE * (T::kThreads * 16) + wave * 1024), at_tail ? tail_w : from_w,
                             __builtin_amdgcn_readfirstlane(PIECE * step_w + k0));
    } else if constexpr (PIECE < T::kLoadsW + T::kLoadsX) {
      constexpr int AT = PIECE - T::kLoadsW;
      desc_x[2] = there ? end_x : 0u;
      load_16_bytes_into_lds(desc_x, stage, __builtin_amdgcn_readfirstlane(T::kBytesW + AT * (T::kThreads * 16) + wave * 1024),
                             at_tail ? tail_x : from_x, __builtin_amdgcn_readfirstlane(AT * step_x + k0));
    } else {
      const bool begins = (g & 3) == 0 || g == g_begin;   // with the first stage of a run its scales
      const uint32_t to = to_s + (static_cast<uint32_t>((g >> 2) & (T::kRuns - 1)) << run_shift);
      desc_s[2] = there && begins ? end_s : 0u;
      load_16_bytes_into_lds(desc_s, lds0, __builtin_amdgcn_readfirstlane(begins ? to : T::kNobody),
                             from_s, __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(g & ~3) * 4));
    }
  };
  auto issue = [&](int g, int slot) { static_for<T::kLoads>([&](auto piece) { issue_piece(piece, g, slot); }); };
  // HALVES: a stage's buffer is refilled in two parts.  The first, once every wavefront has passed the middle of the stage: the
  // activations (in registers since the stage began), the weights of the block rows done, the scales; the second, the rest,
  // behind the stage's end.  Each load stands among matrix instructions: all of them together would hold those up for as long
  // as the loads take to be accepted.
  constexpr int kSecond = HALVES ? T::kLoadsW / 2 : 0, kFirst = T::kLoads - kSecond;
  // loads that are issued behind the wait of a stage's end, among the matrix instructions of its last block row
  constexpr int kLate = HALVES ? (kFirst > (NT / 2 - 1) * MT ? kFirst - (NT / 2 - 1) * MT : 0) : T::kLoads - (NT - 1) * MT * T::kLoads / (NT * MT);
  static_assert(HALVES || STAGES >= 3, "a stage that is asked for while another one is multiplied");
  static_assert(!HALVES || (STAGES == 2 && kSecond <= MT && kFirst <= NT / 2 * MT), "loads among a stage's matrix instructions");
  auto issue_first = [&](auto nth, int g, int slot) {   // nth of kFirst: weights 0, 2, .., then the others
    constexpr int N = decltype(nth)::value;
    issue_piece(std::integral_constant<int, N < T::kLoadsW / 2 ? 2 * N : N + T::kLoadsW / 2>{}, g, slot);
  };
  auto issue_second = [&](auto nth, int g, int slot) { issue_piece(std::integral_constant<int, 2 * decltype(nth)::value + 1>{}, g, slot); };

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
  const uint32_t at_sx = lds0 + T::kScalesX + (wm * (MT * 16) + col) * 16;
  const uint32_t at_sw = lds0 + T::kScalesW + static_cast<uint32_t>((n0 + wn * (NT * 16)) / kFp8Block - scale_row0) * 16;
  auto read_w = [&](uint32_t stage, int i) {
    // block 2 p + h starts 32 p + 4 h rows down; 4 rows down the key stays
    const int down = (i >> 1) * 4096 + (i & 1) * 512;
    return fragment_of(read_lds(at_w[0] + stage, down), read_lds(at_w[1] + stage, down));
  };

  f32x4 acc[NT][MT], part[2][MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    part[0][j] = part[1][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  i32x8 xb[MT], wb[2];
  float scale[MT], next_scale[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) scale[j] = 0.f;

  auto read_x = [&](uint32_t stage, int j) { xb[j] = fragment_of(read_lds(at_x[0] + stage, j * 2048), read_lds(at_x[1] + stage, j * 2048)); };
  auto read_scales = [&](int g) {
    const uint32_t run = (g >> 2) & (T::kRuns - 1), in_run = (g & 3) * 4;
    const float sw = read_lds_float(at_sw + run * T::kRunW + in_run, 0);
#pragma unroll
    for (int j = 0; j < MT; ++j) next_scale[j] = read_lds_float(at_sx + run * T::kRunX + in_run, j * 256) * sw;
  };
  // clears what the chunk that K ends in repeats
  auto clear_again = [&] {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool mine = quarter + 4 * h == (tail >> 4);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int z = again - 4 * d;   // bytes of this word to clear
        const uint32_t mask = !mine || z <= 0 ? 0xffffffffu : z >= 4 ? 0u : 0xffffffffu << (8 * z);
#pragma unroll
        for (int j = 0; j < MT; ++j) xb[j][4 * h + d] = static_cast<int>(static_cast<uint32_t>(xb[j][4 * h + d]) & mask);
      }
    }
  };

  // one block of k: the block rows in turn, and behind the last one the next stage's first fragments
  auto multiply = [&](auto last_tag, int g, uint32_t stage, uint32_t next, int slot, int next_slot) {
    constexpr bool LAST = decltype(last_tag)::value;
    const auto x = fragments<WIDE>(xb);
    float mine[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) mine[j] = next_scale[j];
    static_for<NT>([&](auto row_tag) {
      constexpr int i = decltype(row_tag)::value;
      __builtin_amdgcn_sched_barrier(0);
      const Fragment<WIDE> w(wb[i & 1]);
      if constexpr (HALVES && !LAST && i == NT / 2) {   // every wavefront is past the first half of this stage
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      if constexpr (i + 1 < NT) {
        wb[(i + 1) & 1] = read_w(stage, i + 1);
      } else if constexpr (!LAST) {
        // every fragment of this stage is in registers: the next one has landed, and this one is free for all wavefronts
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(HALVES ? kFirst - kLate : (STAGES - 2) * T::kLoads - kLate) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      static_for<MT>([&](auto column_tag) {
        constexpr int j = decltype(column_tag)::value;
        part[i & 1][j] = w.dot(x.v[j]);
        if constexpr (!LAST && i + 1 == NT) {
          __builtin_amdgcn_sched_barrier(0);   // (its registers take the next fragment)
          read_x(next, j);
        }
        // the block row before this one (in front of the first one: the last of the stage before, by that stage's scale)
        constexpr int kBefore = i == 0 ? NT - 1 : i - 1;
        const f32x4 from = part[(i & 1) ^ 1][j];
        const float by = i == 0 ? scale[j] : mine[j];
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[kBefore][j][r] = fmaf(from[r], by, acc[kBefore][j][r]);
        if constexpr (HALVES && !LAST) {
          if constexpr (i == 0 && j < kSecond) issue_second(column_tag, g + 1, next_slot);
          constexpr int kStep = (i - NT / 2) * MT + j;
          if constexpr (kStep >= 0 && kStep < kFirst) issue_first(std::integral_constant<int, kStep < 0 ? 0 : kStep>{}, g + 2, slot);
          __builtin_amdgcn_sched_barrier(0);
        } else if constexpr (!LAST) {   // a stage's loads evenly among the matrix instructions
          constexpr int kFrom = (i * MT + j) * T::kLoads / (NT * MT), kTo = (i * MT + j + 1) * T::kLoads / (NT * MT);
          static_for<kTo - kFrom>([&](auto nth) {
            issue_piece(std::integral_constant<int, kFrom + decltype(nth)::value>{}, g + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
          });
          __builtin_amdgcn_sched_barrier(0);
        }
      });
      if constexpr (!LAST && i + 1 == NT) {
        wb[0] = read_w(next, 0);
        read_scales(g + 1);
      }
    });
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < MT; ++j) scale[j] = mine[j];
  };

  if (g_begin < g_end) {
    if constexpr (HALVES) {
      issue(g_begin, 0);
      static_for<kFirst>([&](auto nth) { issue_first(nth, g_begin + 1, 1); });
    } else {
#pragma unroll
      for (int g = 0; g < STAGES - 1; ++g) issue(g_begin + g, g);
    }
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(HALVES ? kFirst : (STAGES - 2) * T::kLoads) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < MT; ++j) read_x(0, j);
    wb[0] = read_w(0, 0);
    read_scales(g_begin);
    int slot = 0;
    for (int g = g_begin; g + 1 < g_end; ++g) {
      const int next_slot = slot + 1 == STAGES ? 0 : slot + 1;
      multiply(std::integral_constant<bool, false>{}, g, slot * T::kStage, next_slot * T::kStage, slot, next_slot);
      slot = next_slot;
    }
    if (again != 0 && g_end == p.groups) clear_again();
    multiply(std::integral_constant<bool, true>{}, g_end - 1, slot * T::kStage, 0, slot, 0);
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[NT - 1][j][r] = fmaf(part[(NT - 1) & 1][j][r], scale[j], acc[NT - 1][j][r]);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (no load may write LDS once the workgroup is gone)

#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int64_t m = m0 + wm * (MT * 16) + j * 16 + col;
    if (m < p.m) {
#pragma unroll
      for (int i = 0; i < NT; i += 2) {
        const int64_t n = n0 + wn * (NT * 16) + i * 16 + quarter * 8;
        const float v[8] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3],
                            acc[i + 1][j][0], acc[i + 1][j][1], acc[i + 1][j][2], acc[i + 1][j][3]};
        if (p.splits == 1) {
          store_results<8>(p.c, batch * p.c_bs + m * p.c_rs + n * p.c_cs, p.c_cs, p.out_kind, n, p.n, v);
        } else {
          const int64_t line = (static_cast<int64_t>(blockIdx.z) * p.batch + batch) * p.m + m;
          store_results<8>(p.partial, line * p.n + n, 1, FP8_REAL_F32, n, p.n, v);
        }
      }
    }
  }
}

// The shares of a split K added, in order: a thread four columns.
__global__ __launch_bounds__(256) void fp8_join_kernel(const Fp8MatmulParams p, uint32_t quads, int64_t total) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= total) return;
  const int64_t line = at / quads, n = (at - line * quads) * 4, batch = line / p.m, m = line - batch * p.m;
  const int64_t share = static_cast<int64_t>(p.batch) * p.m * p.n;
  const VECOPS_GLOBAL float* from = (const VECOPS_GLOBAL float*)p.partial + line * p.n + n;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (n + 4 <= p.n) {
    for (int s = 0; s < p.splits; ++s) {
      const u32x4 w = load_16(from + s * share);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += __uint_as_float(w[e]);
    }
  } else {
    for (int s = 0; s < p.splits; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.n) v[e] += from[s * share + e];
  }
  store_results<4>(p.c, batch * p.c_bs + m * p.c_rs + n * p.c_cs, p.c_cs, p.out_kind, n, p.n, v);
}

// Up to sixteen rows: bound by HBM, so that what counts is how many bytes of the weights are under way.  A workgroup owns sixteen
// weight rows; its wavefronts share the blocks of k, a run of neighbouring ones each, with the loads of four blocks of both
// operands under way, straight into the registers that the matrix instruction reads; scales come four blocks a load.  The
// wavefronts' sums meet in LDS.
template <int WAVES, int NT, bool WIDE>
__global__ __launch_bounds__(64 * WAVES, NT == 1 ? 4 : 2) void fp8_few_rows_kernel(const Fp8MatmulParams p) {
  constexpr int DEPTH = 4;
  __shared__ f32x4 sums[WAVES][NT][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quarter = lane >> 4;
  const int batch = blockIdx.y;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * NT);   // (16 NT divides 128: one row of scales)
  // Rows past the last one lie past the descriptors' ends: zeros arrive.
  const int last_n = static_cast<int>(min(p.n - n0, static_cast<int64_t>(16 * NT))) - 1;
  const auto operand = [](const VECOPS_GLOBAL char* base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)uniform_ptr(base), 0, __builtin_amdgcn_readfirstlane(static_cast<int>(bytes)), 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t desc_w = operand((const VECOPS_GLOBAL char*)p.b + batch * p.b_bs + n0 * p.ldb, last_n * p.ldb + p.k);
  const __amdgpu_buffer_rsrc_t desc_x = operand((const VECOPS_GLOBAL char*)p.a + batch * p.a_bs, (p.m - 1) * p.lda + p.k);
  const __amdgpu_buffer_rsrc_t desc_sx =
      operand((const VECOPS_GLOBAL char*)(p.a_scales + batch * p.as_bs), ((p.m - 1) * p.as_rs + p.groups) * 4);
  const __amdgpu_buffer_rsrc_t desc_sw =
      operand((const VECOPS_GLOBAL char*)(p.b_scales + batch * p.bs_bs + n0 / kFp8Block * p.bs_rs), static_cast<int64_t>(p.groups) * 4);
  // Two neighbouring lanes load thirty-two bytes of one row, once of either's, and exchange them: sixteen bytes of a row each
  // are a look-up in the cache for every lane.
  uint32_t from_w[NT][2], from_x[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = (col & 14) + h, k = quarter * 32 + (col & 1) * 16;
#pragma unroll
    for (int i = 0; i < NT; ++i) from_w[i][h] = static_cast<uint32_t>((i * 16 + row) * p.ldb) + k;
    from_x[h] = static_cast<uint32_t>(row * p.lda) + k;
  }
  const uint32_t from_sx = static_cast<uint32_t>(min(col, p.m - 1) * p.as_rs * 4);

  const int whole = p.k / kFp8Block;   // blocks of k without the partial one
  const int begin = static_cast<int>(static_cast<int64_t>(whole) * wave / WAVES), end = static_cast<int>(static_cast<int64_t>(whole) * (wave + 1) / WAVES);
  u32x4 wv[DEPTH][NT][2], xv[DEPTH][2];
  auto load = [&](auto slot_tag, int g) {
    constexpr int slot = decltype(slot_tag)::value;
    const uint32_t k0 = static_cast<uint32_t>(g) * kFp8Block;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < NT; ++i) wv[slot][i][h] = __builtin_amdgcn_raw_buffer_load_b128(desc_w, from_w[i][h], k0, 0);
      xv[slot][h] = __builtin_amdgcn_raw_buffer_load_b128(desc_x, from_x[h], k0, 0);
    }
  };
  f32x4 acc[NT], sx, sw;
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto load_scales = [&](int g) {   // of four blocks (past a row's end the next one's, or zeros: not used)
    sx = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(desc_sx, from_sx, static_cast<uint32_t>(g) * 4, 0));
    sw = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(desc_sw, 0, static_cast<uint32_t>(g) * 4, 0));
  };
  if (begin < end) {
    static_for<DEPTH>([&](auto u) {
      if (begin + decltype(u)::value < end) load(u, begin + decltype(u)::value);
    });
    load_scales(begin);
    for (int g0 = begin; g0 < end; g0 += DEPTH) {
      f32x4 scale;
#pragma unroll
      for (int e = 0; e < 4; ++e) scale[e] = sx[e] * sw[e];
      load_scales(g0 + DEPTH);
      static_for<DEPTH>([&](auto u) {
        constexpr int slot = decltype(u)::value;
        const int g = g0 + slot;
        if (g < end) {
          f32x4 part[NT];
          exchange_lanes<kNextLane>(xv[slot][0], xv[slot][1], lane & 1);
          const Fragment<WIDE> x(fragment_of(xv[slot][0], xv[slot][1]));
#pragma unroll
          for (int i = 0; i < NT; ++i) exchange_lanes<kNextLane>(wv[slot][i][0], wv[slot][i][1], lane & 1);
#pragma unroll
          for (int i = 0; i < NT; ++i) part[i] = Fragment<WIDE>(fragment_of(wv[slot][i][0], wv[slot][i][1])).dot(x);
          // (In front of the branch below: the compiler has been seen to leave too few wait states between a matrix instruction
          // and the use of its result where one path between them is longer than the other.)
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][r] = fmaf(part[i][r], scale[slot], acc[i][r]);
#pragma unroll
          for (int i = 0; i < NT; ++i) asm volatile("" : "+v"(acc[i]));   // (held here)
          if (g + DEPTH < end) load(u, g + DEPTH);
        }
      });
    }
  }
  if (whole < p.groups && wave == WAVES - 1) {
    // The partial block: a chunk that K ends in, or in front of, is the sixteen bytes in front of K (rows have at least
    // sixteen), the same on both sides; of the activations only those are kept that no other chunk has.
    u32x4 w[NT][2], x[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = whole * kFp8Block + quarter * 16 + 64 * h, at = min(k, p.k - 16);
#pragma unroll
      for (int i = 0; i < NT; ++i) w[i][h] = __builtin_amdgcn_raw_buffer_load_b128(desc_w, static_cast<uint32_t>((i * 16 + col) * p.ldb) + at, 0, 0);
      x[h] = __builtin_amdgcn_raw_buffer_load_b128(desc_x, static_cast<uint32_t>(col * p.lda) + at, 0, 0);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int z = k + 16 - p.k - 4 * d;   // bytes of this word to clear
        x[h][d] &= z <= 0 ? 0xffffffffu : z >= 4 ? 0u : 0xffffffffu << (8 * z);
      }
    }
    load_scales(whole);
    const Fragment<WIDE> xf(fragment_of(x[0], x[1]));
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const f32x4 part = Fragment<WIDE>(fragment_of(w[i][0], w[i][1])).dot(xf);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][r] = fmaf(part[r], sx[0] * sw[0], acc[i][r]);
    }
  }

#pragma unroll
  for (int i = 0; i < NT; ++i) sums[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave < NT) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < WAVES; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += sums[u][wave][lane][r];
    const int64_t n = n0 + wave * 16 + quarter * 4;
    if (col < p.m && n < p.n) store_results<4>(p.c, batch * p.c_bs + col * p.c_rs + n * p.c_cs, p.c_cs, p.out_kind, n, p.n, v);
  }
}

// 16-bit results by the 8-bit instruction, as many rows have them.  What exact products cost here, as those in fp32 have them (us):
// 1 x 14336 x 4096 13.1 -> 13.3, 1 x 4096 x 14336 12.8 -> 12.9, 8 x 14336 x 4096 13.7 -> 13.9, 16 x 14336 x 4096 13.8 -> 15.0.
template <int WAVES, int NT>
hipError_t launch_few_rows_as(const Fp8MatmulParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>((static_cast<int64_t>(p.n) + 16 * NT - 1) / (16 * NT)), static_cast<uint32_t>(p.batch));
  if (p.out_kind == FP8_REAL_F32) hipLaunchKernelGGL((fp8_few_rows_kernel<WAVES, NT, true>), grid, dim3(64 * WAVES), 0, stream, p);
  else hipLaunchKernelGGL((fp8_few_rows_kernel<WAVES, NT, false>), grid, dim3(64 * WAVES), 0, stream, p);
  return hipGetLastError();
}

// us, weights past the caches.  Blocks of 64 weight rows, which read the activations a fourth as often: 16 x 14336 x 4096 13.9,
// of 16 rows 16.0 (8 rows of activations 13.6 and 13.7, 4 rows 13.5 and 13.3).  Eight wavefronts a block, for a workgroup a
// compute unit or fewer: 1 x 4096 x 14336 12.9, four 14.4 (16 x 8192 x 8192 16.7 and 15.5, 1 x 4096 x 4096 7.3 and 6.3).
int few_rows_weights(int64_t m, int64_t n, int64_t batch) { return m > 8 && (n + 63) / 64 * batch >= 160 ? 64 : 16; }

hipError_t launch_few_rows(const Fp8MatmulParams& p, hipStream_t stream) {
  if (few_rows_weights(p.m, p.n, p.batch) == 64) return launch_few_rows_as<4, 4>(p, stream);
  if ((static_cast<int64_t>(p.n) + 15) / 16 * p.batch <= 256 && p.groups >= 64) return launch_few_rows_as<8, 1>(p, stream);
  return launch_few_rows_as<4, 1>(p, stream);
}

template <int WN, int WM, int NT, int MT, bool WIDE, int STAGES, bool HALVES = false>
hipError_t launch_tile(const Fp8MatmulParams& p, hipStream_t stream) {
  using T = Fp8Tile<WN, WM, NT, MT, STAGES>;
  const void* kernel = reinterpret_cast<const void*>(&fp8_tile_kernel<WN, WM, NT, MT, WIDE, STAGES, HALVES>);
  if constexpr (T::kLds > 65536) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds);
    if (e != hipSuccess) return e;
  }
  const uint32_t tiles_n = static_cast<uint32_t>((p.n + T::kBN - 1) / T::kBN), tiles_m = static_cast<uint32_t>((p.m + T::kBM - 1) / T::kBM);
  hipLaunchKernelGGL((fp8_tile_kernel<WN, WM, NT, MT, WIDE, STAGES, HALVES>), dim3(tiles_n * tiles_m, static_cast<uint32_t>(p.batch), static_cast<uint32_t>(p.splits)),
                     dim3(T::kThreads), T::kLds, stream, p, tiles_n, tiles_m);
  if (p.splits > 1) {
    const uint32_t quads = static_cast<uint32_t>((p.n + 3) / 4);
    const int64_t total = static_cast<int64_t>(p.batch) * p.m * quads;
    hipLaunchKernelGGL(fp8_join_kernel, dim3(static_cast<uint32_t>((total + 255) / 256)), dim3(256), 0, stream, p, quads, total);
  }
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
    const uint32_t total = static_cast<uint32_t>(p.batch) * row_blocks * static_cast<uint32_t>(p.groups);
    // Runs of blocks a die where rows are not whole lines: 11000 x 4001 in bf16 45.4 us without, 39.6 with; 8192 x 4096 28.1 and 29.8.
    const bool runs = (p.x_rs * (p.kind == FP8_REAL_F32 ? 4 : 2) % 128 != 0 || p.q_rs % 128 != 0) && total <= (1u << 24) - 16;
    const dim3 grid(runs ? (total + 7) / 8 * 8 : total);
    if (p.kind == FP8_REAL_BF16) hipLaunchKernelGGL((fp8_quantize_tiles_kernel<FP8_REAL_BF16>), grid, dim3(256), 0, stream, p, row_blocks, runs);
    else if (p.kind == FP8_REAL_F16) hipLaunchKernelGGL((fp8_quantize_tiles_kernel<FP8_REAL_F16>), grid, dim3(256), 0, stream, p, row_blocks, runs);
    else hipLaunchKernelGGL((fp8_quantize_tiles_kernel<FP8_REAL_F32>), grid, dim3(256), 0, stream, p, row_blocks, runs);
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

hipError_t launch_fp8_scales(const float* in, int64_t bs, int64_t rs, int64_t gs, float* out, int32_t batch, int32_t rows, int32_t groups,
                             hipStream_t stream) {
  const int64_t total = static_cast<int64_t>(batch) * rows * groups;
  hipLaunchKernelGGL(fp8_scales_kernel, dim3(static_cast<uint32_t>((total + 255) / 256)), dim3(256), 0, stream, in, bs, rs, gs, out, total, rows,
                     groups);
  return hipGetLastError();
}

// Which kernel a product takes, and in how many shares of K: the cheapest by an estimate whose numbers were fitted to times of 260
// shapes on one MI355X - 24 to 3000 rows, 512 to 14336 columns, K 1024 to 14336, every tile, K whole, in two and in four (by it
// the product takes 1.004 times the best of them on average, 1.2 times at the worst).
//   time = start + rounds * (tile start + blocks of k * time a block) + join,  at least the operands' bytes at 6.7 TB/s
// Tiles of which two share a compute unit take `alone` a block with at most one on each, `paired` else.
Fp8Plan fp8_plan(int64_t m, int64_t n, int64_t k, int64_t batch, int out_kind) {
  if (m <= 16) return {FP8_FEW_ROWS, 1, 16, few_rows_weights(m, n, batch)};
  if (k == 0) return {FP8_TILE_64, 1, 64, 64};
  struct Cost {
    int kind, n, m, slots;
    double start[2], alone[2], paired[2];   // us; [1]: fp32 results
  };
  static constexpr Cost kCosts[] = {
      {FP8_TILE_64, 64, 64, 512, {1.83, 2.08}, {0.313, 0.489}, {0.470, 0.711}},
      {FP8_TILE_128X64, 64, 128, 256, {2.28, 2.33}, {0.430, 0.704}, {0.430, 0.704}},
      {FP8_TILE_128_ALONE, 128, 128, 256, {2.55, 3.23}, {0.592, 1.000}, {0.592, 1.000}},
      {FP8_TILE_128_PAIRED, 128, 128, 512, {3.19, 3.93}, {0.718, 1.079}, {1.036, 1.683}},
      {FP8_TILE_256, 256, 256, 256, {6.11, 1e9}, {1.458, 0.0}, {1.458, 0.0}},
  };
  const int wide = out_kind == FP8_REAL_F32;
  const int64_t groups = (k + kFp8Block - 1) / kFp8Block;
  Fp8Plan best = {FP8_TILE_64, 1, 64, 64};
  double least = 1e30;
  for (const Cost& c : kCosts) {
    for (int splits = 1; splits <= 4; splits *= 2) {
      if (splits > 1 && groups < 4 * splits) break;
      const int64_t units = ((m + c.m - 1) / c.m) * ((n + c.n - 1) / c.n) * batch * splits, blocks = (groups + splits - 1) / splits;
      const int64_t rounds = units / c.slots, rest = units - rounds * c.slots;
      double us = rounds * (c.start[wide] + c.paired[wide] * blocks);
      if (rest > 0) us += c.start[wide] + (rest <= 256 ? c.alone[wide] : c.paired[wide]) * blocks;
      us = std::max(us, static_cast<double>(m + n) * k * batch / 6.7e6);
      if (splits > 1) us += 2.5 + 8.0 * splits * m * n * batch / 4.9e6;
      if (us < least) least = us, best = {c.kind, splits, c.m, c.n};
    }
  }
  return best;
}

hipError_t launch_fp8_matmul(const Fp8MatmulParams& p, int kind, hipStream_t stream) {
  const bool wide = p.out_kind == FP8_REAL_F32;
  switch (kind) {
    case FP8_FEW_ROWS: return launch_few_rows(p, stream);
    case FP8_TILE_64: return wide ? launch_tile<2, 2, 2, 2, true, 4>(p, stream) : launch_tile<2, 2, 2, 2, false, 4>(p, stream);
    case FP8_TILE_128X64: return wide ? launch_tile<2, 4, 2, 2, true, 4>(p, stream) : launch_tile<2, 4, 2, 2, false, 4>(p, stream);
    case FP8_TILE_128_ALONE: return wide ? launch_tile<2, 4, 4, 2, true, 3>(p, stream) : launch_tile<2, 4, 4, 2, false, 3>(p, stream);
    case FP8_TILE_128_PAIRED: return wide ? launch_tile<2, 2, 4, 4, true, 2, true>(p, stream) : launch_tile<2, 2, 4, 4, false, 2, true>(p, stream);
    case FP8_TILE_256: return wide ? hipErrorInvalidValue : launch_tile<2, 4, 8, 4, false, 2, true>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace vecops_hip
