// Microscaled copies of matrices, and the operators between a layer's products: the root-mean-square norm with the residual's
// addition and the gated activation, whose results leave quantised as the products take them.
#include "row_quantize.h"

#include <algorithm>

#include "quantized_common.h"

namespace vecops_hip {

namespace {

typedef __attribute__((aligned(1))) uint32_t u32_anywhere;

template <int KIND>
struct Real {
  using type = uint16_t;
};
template <>
struct Real<FP8_REAL_F32> {
  using type = float;
};

// Eight consecutive elements as fp32 (`at`: the first one's place, `cs` elements apart); those from `left` on are zeros.
// `whole`: they are contiguous and all there.
template <int KIND>
__device__ __forceinline__ void load_row_eight(const void* base, int64_t at, int64_t cs, int left, bool whole, float (&v)[8]) {
  const VECOPS_GLOBAL auto* x = (const VECOPS_GLOBAL typename Real<KIND>::type*)base + at;
  if constexpr (KIND == FP8_REAL_F32) {
    if (whole) {
      const u32x4 lo = load_16(x), hi = load_16(x + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = __uint_as_float(lo[e]);
        v[4 + e] = __uint_as_float(hi[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < left ? x[e * cs] : 0.0f;
    }
  } else {
    if (whole) {
      const u32x4 w = load_16(x);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = real_bits_to_f32((w[e >> 1] >> (16 * (e & 1))) & 0xffffu, KIND);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < left ? real_bits_to_f32(x[e * cs], KIND) : 0.0f;
    }
  }
}

// The same in two steps, so that many loads can be under way: what memory holds, then its numbers.
template <int KIND>
struct RawEight {
  u32x4 w[KIND == FP8_REAL_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    const VECOPS_GLOBAL auto* x = (const VECOPS_GLOBAL typename Real<KIND>::type*)base + at;
    w[0] = load_16(x);
    if constexpr (KIND == FP8_REAL_F32) w[1] = load_16(x + 4);
  }
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (KIND == FP8_REAL_F32) return __uint_as_float(w[e >> 2][e & 3]);
    else return real_bits_to_f32((w[0][e >> 1] >> (16 * (e & 1))) & 0xffffu, KIND);
  }
  // where less than eight are there: one by one, zeros behind them
  __device__ __forceinline__ void load_part(const void* base, int64_t at, int left) {
    const VECOPS_GLOBAL auto* x = (const VECOPS_GLOBAL typename Real<KIND>::type*)base + at;
#pragma unroll
    for (int d = 0; d < (KIND == FP8_REAL_F32 ? 2 : 1); ++d) w[d] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= left) continue;
      if constexpr (KIND == FP8_REAL_F32) w[e >> 2][e & 3] = __float_as_uint(x[e]);
      else w[0][e >> 1] |= static_cast<uint32_t>(x[e]) << (16 * (e & 1));
    }
  }
};

__device__ __forceinline__ uint32_t most_bits(const float (&v)[8]) {
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
  return most;
}

// Moves within sixteen lanes: to the next lane, the next but one, mirrored within eight, mirrored within sixteen.  In this order each
// brings in what the lanes before have not seen.
constexpr int kMoves[4] = {0xb1, 0x4e, 0x141, 0x140};
template <int MOVE>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
#if defined(__HIP_DEVICE_COMPILE__)
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0u, v, MOVE, 0xf, 0xf, true));
#else
  return v;
#endif
}
__device__ __forceinline__ uint32_t most_of_4(uint32_t v) {
  v = max(v, moved<kMoves[0]>(v));
  return max(v, moved<kMoves[1]>(v));
}
__device__ __forceinline__ uint32_t most_of_16(uint32_t v) {
  v = most_of_4(v);
  v = max(v, moved<kMoves[2]>(v));
  return max(v, moved<kMoves[3]>(v));
}
__device__ __forceinline__ uint32_t most_of_64(uint32_t v) {
  v = most_of_16(v);
  v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16, 64)));
  return max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 32, 64)));
}
__device__ __forceinline__ float sum_of_64(float v) {
  v += __uint_as_float(moved<kMoves[0]>(__float_as_uint(v)));
  v += __uint_as_float(moved<kMoves[1]>(__float_as_uint(v)));
  v += __uint_as_float(moved<kMoves[2]>(__float_as_uint(v)));
  v += __uint_as_float(moved<kMoves[3]>(__float_as_uint(v)));
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// ---------------------------------------------------------------------------------------------------------------------
// Microscaled blocks.  The scale is the power of two that brings the block's largest number into the element type's highest
// binade (e2m1: 4..6, e4m3: 256..448), by its exponent field: byte E = max(field - 2 or 8, 0) stands for 2^(E - 127).  Elements are
// x 2^(127 - E), exact but where it is far below the type's smallest number, to the nearest, ties to even, and what is past the largest number becomes that.  A block
// with an infinity or a NaN gets the scale's only other value, NaN, and elements of zero.
// ---------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t mx_scale(uint32_t most, int top) {   // `most`: the bits of the largest |x|
  const int field = static_cast<int>(most >> 23);
  return field == 255 ? 255u : static_cast<uint32_t>(max(field - top, 0));
}

// Eight elements of a block, e2m1: four bytes.
__device__ __forceinline__ uint32_t mx_e2m1(const float (&v)[8], uint32_t scale) {
#if defined(__HIP_DEVICE_COMPILE__)
  // (the instruction divides by the power of two whose exponent field this is, field 0 standing for 2^-127, and saturates)
  const float by = __uint_as_float((scale & 0xffu) << 23);
  uint32_t q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], by, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], by, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], by, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], by, 3);
  return scale == 255u ? 0u : q;
#else
  (void)v; (void)scale;
  return 0u;
#endif
}

// The same, e4m3: eight bytes.
__device__ __forceinline__ u32x2 mx_e4m3(const float (&v)[8], uint32_t scale) {
  const float by = __uint_as_float((254u - min(scale, 253u)) << 23);
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = fminf(fmaxf(v[e] * by, -448.0f), 448.0f);
  const u32x2 q = {pack_e4m3(y[0], y[1], y[2], y[3]), pack_e4m3(y[4], y[5], y[6], y[7])};
  return scale == 255u ? u32x2{0u, 0u} : q;
}

// BYTES bytes of quantised elements (`cs` bytes apart); those from `left` on stay unwritten.
template <int BYTES>
__device__ __forceinline__ void store_bytes(uint8_t* base, int64_t at, int64_t cs, int left, bool whole, const uint32_t (&w)[BYTES / 4]) {
  VECOPS_GLOBAL uint8_t* to = (VECOPS_GLOBAL uint8_t*)base + at;
  if (whole) {
    if constexpr (BYTES == 8) *(VECOPS_GLOBAL u32x2_anywhere*)to = u32x2{w[0], w[1]};
    else *(VECOPS_GLOBAL u32_anywhere*)to = w[0];
  } else {
#pragma unroll
    for (int e = 0; e < BYTES; ++e)
      if (e < left) to[e * cs] = static_cast<uint8_t>(w[e >> 2] >> (8 * (e & 3)));
  }
}

// Eight elements a lane, four lanes a block.  Bound by HBM: 11008 x 4096 bf16 to e2m1 29.3 us, and back 21.2 (3.9 and 5.4 TB/s read and written; of a matrix
// that the last cache holds 21.8 and 20.8).
template <int KIND, int FORMAT>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const MxCopyParams p, uint32_t total) {
  const uint32_t per_line = static_cast<uint32_t>(p.groups) * 4u;
  for (uint32_t at = blockIdx.x * 256u + threadIdx.x; at < total; at += gridDim.x * 256u) {   // (the same for four lanes)
    const uint32_t line = at / per_line, piece = at - line * per_line;
    const uint32_t batch = line / static_cast<uint32_t>(p.rows), row = line - batch * p.rows;
    const int k = static_cast<int>(piece) * 8, left = p.k - k;
    float v[8];
    load_row_eight<KIND>(p.x, batch * p.x_bs + row * p.x_rs + k * p.x_cs, p.x_cs, left, left >= 8 && p.x_cs == 1, v);
    const uint32_t scale = mx_scale(most_of_4(most_bits(v)), FORMAT == ROW_MX_E2M1 ? 2 : 8);
    if constexpr (FORMAT == ROW_MX_E2M1) {
      const uint32_t q[1] = {mx_e2m1(v, scale)};
      store_bytes<4>(p.q, batch * p.q_bs + row * p.q_rs + (k / 2) * p.q_cs, p.q_cs, left / 2, left >= 8 && p.q_cs == 1, q);
    } else {
      const u32x2 w = mx_e4m3(v, scale);
      const uint32_t q[2] = {w[0], w[1]};
      store_bytes<8>(p.q, batch * p.q_bs + row * p.q_rs + k * p.q_cs, p.q_cs, left, left >= 8 && p.q_cs == 1, q);
    }
    if ((piece & 3) == 0) p.scales[batch * p.s_bs + row * p.s_rs + (piece >> 2) * p.s_cs] = static_cast<uint8_t>(scale);
  }
}

// The way back.  An element times its power of two in fp32, rounded once to the result's type.
template <int KIND, int FORMAT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const MxCopyParams p, uint32_t total) {
  const uint32_t per_line = (static_cast<uint32_t>(p.k) + 7u) / 8u;
  for (uint32_t at = blockIdx.x * 256u + threadIdx.x; at < total; at += gridDim.x * 256u) {
    const uint32_t line = at / per_line, piece = at - line * per_line;
    const uint32_t batch = line / static_cast<uint32_t>(p.rows), row = line - batch * p.rows;
    const int k = static_cast<int>(piece) * 8, left = p.k - k;
    constexpr int BYTES = FORMAT == ROW_MX_E2M1 ? 4 : 8;
    const VECOPS_GLOBAL uint8_t* from = (const VECOPS_GLOBAL uint8_t*)p.q + batch * p.q_bs + row * p.q_rs + (k / (8 / BYTES)) * p.q_cs;
    uint32_t w[2] = {0u, 0u};
    if (left >= 8 && p.q_cs == 1) {
      w[0] = *(const VECOPS_GLOBAL u32_anywhere*)from;
      if constexpr (BYTES == 8) w[1] = *(const VECOPS_GLOBAL u32_anywhere*)(from + 4);
    } else {
#pragma unroll
      for (int e = 0; e < BYTES; ++e)
        if (e * (8 / BYTES) < left) w[e >> 2] |= static_cast<uint32_t>(from[e * p.q_cs]) << (8 * (e & 3));
    }
    const uint32_t scale = p.scales[batch * p.s_bs + row * p.s_rs + (piece >> 2) * p.s_cs];
    // (2^-127 has no normal fp32 number)
    const float by = __uint_as_float(scale == 255u ? 0x7fc00000u : scale == 0u ? 0x00400000u : scale << 23);
    float v[8] = {};
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((ext_vector_type(2))) float f32x2_local;
    f32x2_local pair[4];
    if constexpr (FORMAT == ROW_MX_E2M1) {
      pair[0] = __builtin_bit_cast(f32x2_local, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.0f, 0));
      pair[1] = __builtin_bit_cast(f32x2_local, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.0f, 1));
      pair[2] = __builtin_bit_cast(f32x2_local, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.0f, 2));
      pair[3] = __builtin_bit_cast(f32x2_local, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.0f, 3));
    } else {
      pair[0] = __builtin_bit_cast(f32x2_local, __builtin_amdgcn_cvt_pk_f32_fp8(w[0], false));
      pair[1] = __builtin_bit_cast(f32x2_local, __builtin_amdgcn_cvt_pk_f32_fp8(w[0], true));
      pair[2] = __builtin_bit_cast(f32x2_local, __builtin_amdgcn_cvt_pk_f32_fp8(w[1], false));
      pair[3] = __builtin_bit_cast(f32x2_local, __builtin_amdgcn_cvt_pk_f32_fp8(w[1], true));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = pair[e >> 1][e & 1] * by;
#endif
    store_results<8>(p.x, batch * p.x_bs + row * p.x_rs + k * p.x_cs, p.x_cs, KIND, k, p.k, v);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Rows.  T threads a row (64: four rows a workgroup, no barrier; else a workgroup a row), eight elements a thread a piece, HELD
// pieces of a thread in registers: a row of up to 8 HELD T elements is read once.  A longer one is read again behind each sum or
// maximum over it, by the threads that read (and wrote) the same places before.  Bound by HBM (4096 x 8192 bf16 with the residual to e4m3 by 32 50.8 us, 4.6 TB/s, and 42 where
// the last cache holds most of the operands; the gate of 1999 x 11000 f16 to e4m3 by 128 26-27 us, 4.1 TB/s, and 24), for a few rows by the launch and one
// row's way through memory and barriers: rows that a piece a thread holds have kernels of their own, a quarter as much code to fetch, and weights
// under way beside the row (4 x 4096 with the residual, bf16 to e4m3 by 128: 4.0 us a call rather than 5.0; a launch alone is 2.5).
// ---------------------------------------------------------------------------------------------------------------------

enum : int { SOURCE_NORM = 0, SOURCE_GATE = 1 };
constexpr int kHeld = 4;   // of rows that one piece a thread does not hold

// g / (1 + e^-g) * u.  The exponent's product with log2 e is off by 1.25 * 2^-24 of itself, which is as much of e^-g as |g| times that; v_exp_f32,
// the sum, v_rcp_f32 and the products add a unit of the last place each.  v_rcp_f32 gives no subnormal number, and e^-g ends at 2^128: FAR, for wavefronts with a
// gate of such a size (1999 x 11000 26.1 us; without it 25.8, for every element 27.2, lane by lane 28.5): from 2^120 on, where the 1 is no part of the sum, 2^-100 of e^-g is taken, and as much of the result (down to g = -156, from where on
// it is -0; NaN for -infinity).
constexpr float kFarGate = -83.0f;   // (e^83 = 2^119.7)
template <bool FAR>
__device__ __forceinline__ float silu_mul(float g, float u) {
  const float t = g * -1.44269504f;
  const bool far = FAR && t > 120.0f;
  const float e = __builtin_amdgcn_exp2f(far ? t - 100.0f : t);
  const float y = g * __builtin_amdgcn_rcpf(far ? e : 1.0f + e) * u;
  return far ? y * 0x1p-100f : y;
}

template <int KIND>
__device__ __forceinline__ float as_held(float v) {   // rounded to the type
  if constexpr (KIND == FP8_REAL_BF16) return __uint_as_float(cvt_pk_bf16(v, 0.0f) << 16);
  else if constexpr (KIND == FP8_REAL_F16) return f16_bits_to_f32(f16_bits_rne(v));
  else return v;
}

template <int SOURCE, int KIND, int FORMAT, int HELD>
__global__ __launch_bounds__(1024) void row_quantize_kernel(const RowQuantizeParams p, int threads, uint32_t lines) {
  __shared__ float sums[2][16];
  __shared__ uint32_t mosts[2][16];
  const int waves = threads >> 6, own = threads == 64 ? threadIdx.x & 63 : threadIdx.x, wave = threadIdx.x >> 6;
  const uint32_t rows_here = threads == 64 ? blockDim.x >> 6 : 1u;
  const int span = threads * (8 * HELD);
  const bool held = HELD == 1 || p.k <= span;   // (uniform)
  // the gate's blocks know nothing of one another: workgroups share a row
  constexpr bool kParts = SOURCE == SOURCE_GATE && FORMAT != ROW_INT8;
  const int spans_begin = kParts ? static_cast<int>(blockIdx.y) * span : 0, spans_step = kParts ? static_cast<int>(gridDim.y) * span : span;
  const int spans_end = HELD == 1 && !kParts ? 1 : p.k;
  int turn = 0;

  for (uint32_t line = blockIdx.x * rows_here + (threads == 64 ? static_cast<uint32_t>(wave) : 0u); line < lines; line += gridDim.x * rows_here) {
    const uint32_t batch = line / static_cast<uint32_t>(p.rows), row = line - batch * p.rows;
    const int64_t x_at = batch * p.x_bs + row * p.x_rs, summed_at = batch * p.summed_bs + row * p.summed_rs;
    const int64_t residual_at = batch * p.residual_bs + row * p.residual_rs;
    float v[HELD][8];
    constexpr bool kWeightsToo = SOURCE == SOURCE_NORM && HELD == 1;   // (of more pieces they would take the registers of other rows)
    RawEight<KIND> weight;
    RawEight<FP8_REAL_F32> wide_weight;
    const bool same_kind = p.weight_kind == KIND;

    // the pieces of a span from k0 on, all their loads under way at once; `again`: the residual has been added
    auto load = [&](int k0, bool again) {
      constexpr int kSources = 2;
      RawEight<KIND> raw[HELD][kSources];
      const bool adds = SOURCE == SOURCE_NORM && p.residual != nullptr && !again, two = SOURCE == SOURCE_GATE || adds;
      const bool sum = SOURCE == SOURCE_NORM && p.residual != nullptr && again;
      const void* const first = sum ? p.summed : p.x;
      const void* const second = SOURCE == SOURCE_GATE ? p.x : p.residual;
      const int64_t first_at = sum ? summed_at : x_at, second_at = SOURCE == SOURCE_GATE ? x_at + p.k : residual_at;
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        const int k = k0 + (i * threads + own) * 8;
        if (p.k - k < 8) continue;
        raw[i][0].load(first, first_at + k);
        if (two) raw[i][1].load(second, second_at + k);
        if constexpr (kWeightsToo) {
          if (same_kind) weight.load(p.weight, k);
          else wide_weight.load(p.weight, k);
        }
      }
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        const int k = k0 + (i * threads + own) * 8, left = p.k - k;
        if (left < 8) {
          raw[i][0].load_part(first, first_at + k, left);
          if (two) raw[i][1].load_part(second, second_at + k, left);
          if constexpr (kWeightsToo) {
            if (same_kind) weight.load_part(p.weight, k, left);
            else wide_weight.load_part(p.weight, k, left);
          }
        }
        if (HELD > 1 && k0 + i * threads * 8 >= p.k) {   // (uniform)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
          continue;
        }
        if constexpr (SOURCE == SOURCE_GATE) {
          float least = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[i][e] = silu_mul<false>(raw[i][0][e], raw[i][1][e]);   // (what is not there: 0)
            least = fminf(least, raw[i][0][e]);
          }
          if (__builtin_expect(__builtin_amdgcn_ballot_w64(least < kFarGate) != 0, 0)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = silu_mul<true>(raw[i][0][e], raw[i][1][e]);
          }
        } else {
          if (adds) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = as_held<KIND>(raw[i][0][e] + raw[i][1][e]);
            store_results<8>(p.summed, summed_at + k, 1, KIND, k, p.k, v[i]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = raw[i][0][e];
          }
        }
      }
    };
    float norm = 1.0f;
    // a span's results, from what load() left
    auto finish = [&](int k0) {
      if constexpr (SOURCE == SOURCE_NORM) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
          const int k = k0 + (i * threads + own) * 8, left = p.k - k;
          if (HELD > 1 && k0 + i * threads * 8 >= p.k) continue;
          float w[8];
          if constexpr (kWeightsToo) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = same_kind ? weight[e] : wide_weight[e];
          } else if (same_kind) load_row_eight<KIND>(p.weight, k, 1, left, left >= 8, w);
          else load_row_eight<FP8_REAL_F32>(p.weight, k, 1, left, left >= 8, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * norm * w[e];   // (what is not there: 0, but for a norm that is not finite)
          if (left < 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = e < left ? v[i][e] : 0.0f;
          }
        }
      }
    };

    if constexpr (SOURCE == SOURCE_NORM) {
      float sum = 0.0f;
      for (int k0 = 0; k0 < spans_end; k0 += span) {
        load(k0, false);
#pragma unroll
        for (int i = 0; i < HELD; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) sum = fmaf(v[i][e], v[i][e], sum);
      }
      sum = sum_of_64(sum);
      if (waves > 1) {
        if (own % 64 == 0) sums[turn][wave] = sum;
        __syncthreads();
        sum = 0.0f;
        for (int u = 0; u < waves; ++u) sum += sums[turn][u];
      }
      norm = 1.0f / sqrtf(sum / static_cast<float>(p.k) + p.eps);
    }
    float row_scale = 0.0f;
    if constexpr (FORMAT == ROW_INT8) {
      uint32_t most = 0;
      for (int k0 = 0; k0 < spans_end; k0 += span) {
        if (SOURCE == SOURCE_GATE || !held) load(k0, true);
        finish(k0);
#pragma unroll
        for (int i = 0; i < HELD; ++i) most = max(most, most_bits(v[i]));
      }
      most = most_of_64(most);
      if (waves > 1) {
        if (own % 64 == 0) mosts[turn][wave] = most;
        __syncthreads();
        for (int u = 0; u < waves; ++u) most = max(most, mosts[turn][u]);
      }
      row_scale = __uint_as_float(most) / 127.0f;
      row_scale = row_scale < 0x1p-126f ? 0x1p-126f : row_scale;   // (NaN stays)
      if (own == 0) static_cast<float*>(p.scales)[batch * p.s_bs + row * p.s_rs] = row_scale;
    }
    turn ^= 1;   // (a wavefront that is a row ahead writes beside what others still read; two ahead it cannot be)

    for (int k0 = spans_begin; k0 < spans_end; k0 += spans_step) {
      if (kParts || !held) load(k0, true);
      if (FORMAT != ROW_INT8 || !held) finish(k0);
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        const int k = k0 + (i * threads + own) * 8, left = p.k - k;
        if (HELD > 1 && k0 + i * threads * 8 >= p.k) continue;   // (uniform: the moves between lanes below have all of them)
        if constexpr (SOURCE == SOURCE_NORM)
          if (p.out != nullptr && left > 0) store_results<8>(p.out, batch * p.out_bs + row * p.out_rs + k, 1, KIND, k, p.k, v[i]);
        const int64_t q_at = batch * p.q_bs + row * p.q_rs, s_at = batch * p.s_bs + row * p.s_rs;
        if constexpr (FORMAT == ROW_INT8) {
          const Quotient by(row_scale);
          uint32_t q[2] = {0u, 0u};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = rintf(by(v[i][e]));
            q[e >> 2] |= (static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(y == y ? y : 0.0f, -127.0f), 127.0f))) & 0xffu) << (8 * (e & 3));
          }
          store_bytes<8>(p.q, q_at + k, 1, left, left >= 8, q);
        } else if constexpr (FORMAT == ROW_E4M3_128) {
          const float s = block_scale(most_of_16(most_bits(v[i])));
          const Quotient by(s);
          const uint32_t q[2] = {pack_e4m3(by(v[i][0]), by(v[i][1]), by(v[i][2]), by(v[i][3])), pack_e4m3(by(v[i][4]), by(v[i][5]), by(v[i][6]), by(v[i][7]))};
          store_bytes<8>(p.q, q_at + k, 1, left, left >= 8, q);
          if ((own & 15) == 0 && left > 0) static_cast<float*>(p.scales)[s_at + (k >> 7) * p.s_cs] = s;
        } else if constexpr (FORMAT == ROW_MX_E4M3 || FORMAT == ROW_MX_E2M1) {
          const uint32_t scale = mx_scale(most_of_4(most_bits(v[i])), FORMAT == ROW_MX_E2M1 ? 2 : 8);
          if constexpr (FORMAT == ROW_MX_E2M1) {
            const uint32_t q[1] = {mx_e2m1(v[i], scale)};
            store_bytes<4>(p.q, q_at + k / 2, 1, left / 2, left >= 8, q);
          } else {
            const u32x2 w = mx_e4m3(v[i], scale);
            const uint32_t q[2] = {w[0], w[1]};
            store_bytes<8>(p.q, q_at + k, 1, left, left >= 8, q);
          }
          if ((own & 3) == 0 && left > 0) static_cast<uint8_t*>(p.scales)[s_at + (k >> 5) * p.s_cs] = static_cast<uint8_t>(scale);
        }
      }
    }
  }
}

template <int SOURCE, int KIND, int HELD>
hipError_t launch_rows_held(const RowQuantizeParams& p, int threads, int parts, hipStream_t stream) {
  const int64_t lines = static_cast<int64_t>(p.batch) * p.rows;
  const int64_t rows_here = threads == 64 ? 4 : 1, groups = (lines + rows_here - 1) / rows_here;
  const dim3 grid(static_cast<uint32_t>(std::min<int64_t>(groups, 1 << 20)), static_cast<uint32_t>(parts)), block(threads == 64 ? 256 : threads);
  const uint32_t n = static_cast<uint32_t>(lines);
  switch (p.format) {
    case ROW_INT8: hipLaunchKernelGGL((row_quantize_kernel<SOURCE, KIND, ROW_INT8, HELD>), grid, block, 0, stream, p, threads, n); break;
    case ROW_E4M3_128: hipLaunchKernelGGL((row_quantize_kernel<SOURCE, KIND, ROW_E4M3_128, HELD>), grid, block, 0, stream, p, threads, n); break;
    case ROW_MX_E4M3: hipLaunchKernelGGL((row_quantize_kernel<SOURCE, KIND, ROW_MX_E4M3, HELD>), grid, block, 0, stream, p, threads, n); break;
    case ROW_MX_E2M1: hipLaunchKernelGGL((row_quantize_kernel<SOURCE, KIND, ROW_MX_E2M1, HELD>), grid, block, 0, stream, p, threads, n); break;
    default:
      if constexpr (SOURCE == SOURCE_NORM) {
        hipLaunchKernelGGL((row_quantize_kernel<SOURCE, KIND, ROW_NONE, HELD>), grid, block, 0, stream, p, threads, n);
        break;
      } else {
        return hipErrorInvalidValue;
      }
  }
  return hipGetLastError();
}

template <int SOURCE, int KIND>
hipError_t launch_rows_as(const RowQuantizeParams& p, hipStream_t stream) {
  const int64_t lines = static_cast<int64_t>(p.batch) * p.rows;
  // as few threads as hold a row, but enough wavefronts for the chip and a piece for each thread
  int threads = 64;
  while (threads < 1024 && (threads * 8 * kHeld < p.k || (threads * 8 < p.k && lines * threads < 256 * 1024))) threads *= 2;
  // (the gate's, up to 2^23 elements: bf16 to e4m3 by 32, 64 x 14336 in 2.9 us rather than 5.3, 2048 x 14336 and 4096 x 4096 in as long, 8192 x 14336 in 118
  // rather than 103, as more rows leave enough loads under way to a thread's four pieces)
  if (SOURCE == SOURCE_GATE && p.format != ROW_INT8 && p.k > 2048 && lines * p.k <= 1 << 23)
    return launch_rows_held<SOURCE, KIND, 1>(p, 256, (p.k + 2047) / 2048, stream);
  return threads * 8 >= p.k ? launch_rows_held<SOURCE, KIND, 1>(p, threads, 1, stream) : launch_rows_held<SOURCE, KIND, kHeld>(p, threads, 1, stream);
}

template <int SOURCE>
hipError_t launch_rows(const RowQuantizeParams& p, hipStream_t stream) {
  switch (p.kind) {
    case FP8_REAL_BF16: return launch_rows_as<SOURCE, FP8_REAL_BF16>(p, stream);
    case FP8_REAL_F16: return launch_rows_as<SOURCE, FP8_REAL_F16>(p, stream);
    default: return launch_rows_as<SOURCE, FP8_REAL_F32>(p, stream);
  }
}

template <int FORMAT>
void launch_quantize_as(const MxCopyParams& p, dim3 grid, uint32_t total, hipStream_t stream) {
  if (p.kind == FP8_REAL_BF16) hipLaunchKernelGGL((mx_quantize_kernel<FP8_REAL_BF16, FORMAT>), grid, dim3(256), 0, stream, p, total);
  else if (p.kind == FP8_REAL_F16) hipLaunchKernelGGL((mx_quantize_kernel<FP8_REAL_F16, FORMAT>), grid, dim3(256), 0, stream, p, total);
  else hipLaunchKernelGGL((mx_quantize_kernel<FP8_REAL_F32, FORMAT>), grid, dim3(256), 0, stream, p, total);
}

template <int FORMAT>
void launch_dequantize_as(const MxCopyParams& p, dim3 grid, uint32_t total, hipStream_t stream) {
  if (p.kind == FP8_REAL_BF16) hipLaunchKernelGGL((mx_dequantize_kernel<FP8_REAL_BF16, FORMAT>), grid, dim3(256), 0, stream, p, total);
  else if (p.kind == FP8_REAL_F16) hipLaunchKernelGGL((mx_dequantize_kernel<FP8_REAL_F16, FORMAT>), grid, dim3(256), 0, stream, p, total);
  else hipLaunchKernelGGL((mx_dequantize_kernel<FP8_REAL_F32, FORMAT>), grid, dim3(256), 0, stream, p, total);
}

}  // namespace

hipError_t launch_mx_quantize(const MxCopyParams& p, hipStream_t stream) {
  const uint32_t total = static_cast<uint32_t>(static_cast<int64_t>(p.batch) * p.rows * p.groups * 4);
  const dim3 grid(std::min((total + 255u) / 256u, 1u << 22));
  if (p.format == ROW_MX_E2M1) launch_quantize_as<ROW_MX_E2M1>(p, grid, total, stream);
  else launch_quantize_as<ROW_MX_E4M3>(p, grid, total, stream);
  return hipGetLastError();
}

hipError_t launch_mx_dequantize(const MxCopyParams& p, hipStream_t stream) {
  const uint32_t total = static_cast<uint32_t>(static_cast<int64_t>(p.batch) * p.rows * ((static_cast<int64_t>(p.k) + 7) / 8));
  const dim3 grid(std::min((total + 255u) / 256u, 1u << 22));
  if (p.format == ROW_MX_E2M1) launch_dequantize_as<ROW_MX_E2M1>(p, grid, total, stream);
  else launch_dequantize_as<ROW_MX_E4M3>(p, grid, total, stream);
  return hipGetLastError();
}

hipError_t launch_rms_norm(const RowQuantizeParams& p, hipStream_t stream) { return launch_rows<SOURCE_NORM>(p, stream); }
hipError_t launch_silu_mul(const RowQuantizeParams& p, hipStream_t stream) { return launch_rows<SOURCE_GATE>(p, stream); }

}  // namespace vecops_hip
