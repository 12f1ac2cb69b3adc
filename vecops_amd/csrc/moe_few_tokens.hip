// A mixture-of-experts layer for a few tokens:
//   l = x . router^T;  the experts of the largest scores;  out = sum_r w_r down[e_r] . (silu(gate[e_r] . x) * (up[e_r] . x))
// What bounds it: the weights of the experts that the tokens name are read once from HBM, against a handful of rows; the rest
// is latency.  Four launches: the logits, the choice, gate and up with the activation, down with the sum over a token's
// experts.  The tokens of an expert are the columns of a matrix instruction whose rows are sixteen rows of weights, which go
// from memory straight into its operand registers.
#include "moe_few_tokens.h"

#include <algorithm>

#include "tile_gemm.h"

namespace vecops_hip {

namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4), aligned(1))) uint32_t u32x4_anywhere;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

__device__ __forceinline__ u32x4 load_16(const VECOPS_GLOBAL char* at) { return *(const VECOPS_GLOBAL u32x4_anywhere*)at; }

// Sixteen bytes of a row of `count` elements of EB bytes from element k on, zeros past the row's end (which is not read past).
template <int EB>
__device__ __forceinline__ u32x4 load_16_until(const VECOPS_GLOBAL char* row, int k, int count) {
  constexpr int EPC = 16 / EB;
  if (k + EPC <= count) return load_16(row + static_cast<int64_t>(k) * EB);
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < EPC; ++e)
    if (k + e < count) {
      uint32_t bits;
      if constexpr (EB == 1) bits = ((const VECOPS_GLOBAL uint8_t*)row)[k + e];
      else if constexpr (EB == 2) bits = ((const VECOPS_GLOBAL uint16_t*)row)[k + e];
      else bits = ((const VECOPS_GLOBAL uint32_t*)row)[k + e];
      v[e * EB / 4] |= bits << (8 * (e * EB % 4));
    }
  return v;
}

template <bool F16>
__device__ __forceinline__ f32x4 mfma_16(const u32x4& w, const u32x4& x, const f32x4& acc) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, x), acc, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), acc, 0, 0, 0);
}

// Eight e4m3 bytes as eight bf16 or f16 (exact).
template <bool F16>
__device__ __forceinline__ u32x4 widen(uint32_t lo, uint32_t hi) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int a = static_cast<int>(lo), b = static_cast<int>(hi);
  if constexpr (F16)
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true))};
  else
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true))};
#else
  (void)lo; (void)hi;
  return u32x4{0u, 0u, 0u, 0u};
#endif
}

// ---------------------------------------------------------------------------------------------------------------------
// Router: logits in fp32.  A workgroup has sixteen experts, sixteen tokens and one of `parts` shares of the hidden axis, which
// its wavefronts split again; the shares are added where the experts are chosen.
// ---------------------------------------------------------------------------------------------------------------------

constexpr int kRouteWaves = 4, kRouteSteps = 4;  // steps of 32 that a wavefront has at most in its share

template <bool F16, bool R32>
__global__ __launch_bounds__(64 * kRouteWaves) void moe_logits_kernel(const MoeRouteParams p) {
  __shared__ float meet[kRouteWaves][256];
  const int lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e0 = blockIdx.x * 16, t0 = blockIdx.z * 16;
  const VECOPS_GLOBAL char* r = (const VECOPS_GLOBAL char*)p.router + static_cast<int64_t>(min(e0 + col, p.experts - 1)) * p.ld_router * (R32 ? 4 : 2);
  const VECOPS_GLOBAL char* x = (const VECOPS_GLOBAL char*)p.x + static_cast<int64_t>(min(t0 + col, p.tokens - 1)) * p.ldx * 2;
  const int steps = (p.hidden + 31) / 32, first = static_cast<int>(static_cast<int64_t>(steps) * blockIdx.y / p.parts),
            end = static_cast<int>(static_cast<int64_t>(steps) * (blockIdx.y + 1) / p.parts);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s = first + wave; s < end; s += kRouteWaves) {
    const int k = s * 32 + quarter * 8;
    const u32x4 xv = load_16_until<2>(x, k, p.hidden);
    if constexpr (R32) {
      const u32x4 lo = load_16_until<4>(r, k, p.hidden), hi = load_16_until<4>(r, k + 4, p.hidden);
#pragma unroll
      for (int i = 0; i < 8; ++i) {   // instruction i multiplies element i of every lane
        const uint32_t bits = (xv[i >> 1] >> (16 * (i & 1))) & 0xffffu;
        const float xf = F16 ? f16_bits_to_f32(bits) : __uint_as_float(bits << 16);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(i < 4 ? lo[i & 3] : hi[i & 3]), xf, acc, 0, 0, 0);
      }
    } else {
      acc = mfma_16<F16>(load_16_until<2>(r, k, p.hidden), xv, acc);
    }
  }
  *reinterpret_cast<f32x4*>(&meet[wave][lane * 4]) = acc;
  __syncthreads();
  const int at = threadIdx.x, e = e0 + (at >> 6) * 4 + (at & 3), t = t0 + ((at >> 2) & 15);   // (lane at / 4, its result at % 4)
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < kRouteWaves; ++w) sum += meet[w][at];
  if (e < p.experts && t < p.tokens) p.logits[(static_cast<int64_t>(blockIdx.y) * p.tokens + t) * p.experts + e] = sum;
}

// fp32 bits as an integer of the same order; every NaN above everything.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t bits = __float_as_uint(v == 0.0f ? 0.0f : v);   // (-0 ties with 0)
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = fmaxf(v, __shfl_xor(v, d, 64));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d, 64);
  return v;
}

// The choice: a wavefront a token, lane l has the experts l, l + 64, ...; `top` times the largest that is left, the lower
// index among equals.
__global__ __launch_bounds__(64) void moe_choose_kernel(const MoeRouteParams p) {
  constexpr int MOST = kMoeMostExperts / 64;
  const int t = blockIdx.x, lane = threadIdx.x;
  float score[MOST];
  uint32_t key[MOST];
  float most = -__builtin_huge_valf();
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    const int e = lane + 64 * j;
    score[j] = -__builtin_huge_valf();
    key[j] = 0;
    if (e < p.experts) {
      float l = 0.f;
      for (int s = 0; s < p.parts; ++s) l += p.logits[(static_cast<int64_t>(s) * p.tokens + t) * p.experts + e];
      score[j] = l;
      key[j] = order_of(l);   // (0 is below every number's)
      most = fmaxf(most, l);
    }
  }
  if (p.sigmoid) {
#pragma unroll
    for (int j = 0; j < MOST; ++j) score[j] = 1.0f / (1.0f + expf(-score[j]));
  } else {
    most = wave_max(most);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < MOST; ++j) {
      score[j] = lane + 64 * j < p.experts ? expf(score[j] - most) : 0.f;
      sum += score[j];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < MOST; ++j) score[j] /= sum;
  }
  if (p.bias != nullptr) {
#pragma unroll
    for (int j = 0; j < MOST; ++j)
      if (lane + 64 * j < p.experts) key[j] = order_of(score[j] + p.bias[lane + 64 * j]);
  }
  float chosen = 0.f, total = 0.f;   // lane r keeps the score of choice r
  int id = 0;
  for (int r = 0; r < p.top; ++r) {
    uint64_t best = 0;   // (the order, then the lower index first)
    float its = 0.f;
#pragma unroll
    for (int j = 0; j < MOST; ++j) {
      const uint64_t mine = static_cast<uint64_t>(key[j]) << 32 | static_cast<uint32_t>(~(lane + 64 * j));
      if (key[j] != 0 && mine > best) best = mine, its = score[j];
    }
    uint64_t top = best;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t hi = static_cast<uint32_t>(__shfl_xor(static_cast<int>(top >> 32), d, 64));
      const uint32_t lo = static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d, 64));
      const uint64_t other = static_cast<uint64_t>(hi) << 32 | lo;
      top = other > top ? other : top;
    }
    const int e = static_cast<int>(~static_cast<uint32_t>(top));
    its = __shfl(its, e & 63, 64);
#pragma unroll
    for (int j = 0; j < MOST; ++j)
      if (e == lane + 64 * j) key[j] = 0;   // taken
    if (lane == r) chosen = its, id = e;
    total += its;
  }
  if (lane < p.top) {
    p.ids[t * p.ids_rs + lane * p.ids_cs] = id;
    p.weights[t * p.weights_rs + lane * p.weights_cs] = (p.renormalize ? chosen / total : chosen) * p.scale;
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Experts.  A place (token, choice) whose expert an earlier choice of the same token names too adds its weight to that one.
// ---------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ int expert_at(const MoeExpertsParams& p, int token, int choice) { return p.ids[token * p.ids_rs + choice * p.ids_cs]; }

__device__ __forceinline__ bool named_before(const MoeExpertsParams& p, int token, int choice, int expert) {
  for (int r = 0; r < choice; ++r)
    if (expert_at(p, token, r) == expert) return true;
  return false;
}

// element index, in a block of 128 k, of chunk c (eight elements) of quarter q: a 16-byte load of weights is two chunks of
// e4m3, one of 16-bit elements
template <bool W8>
__device__ __forceinline__ int chunk_k(int c, int quarter) { return W8 ? (c >> 1) * 64 + quarter * 16 + (c & 1) * 8 : c * 32 + quarter * 8; }

constexpr int kUpWaves = 4;

// gate and up.  A workgroup: one expert, the tokens that name it (16 MT at a time), blocks of sixteen gate rows and their up
// rows.  Its wavefronts take the blocks of 128 of the hidden axis in turn.
template <bool F16, bool W8, int MT>
__global__ __launch_bounds__(64 * kUpWaves) void moe_up_kernel(const MoeExpertsParams p, int by_place) {
  constexpr int EB = W8 ? 1 : 2, LOADS = W8 ? 2 : 4;
  __shared__ float meet[kUpWaves][2][MT][256];
  __shared__ int places[kMoeMostTokens];
  __shared__ float weight[kMoeMostTokens];
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int total = p.tokens * p.top;

  // the expert: blockIdx.y itself, or the one that place blockIdx.y is the first to name
  int expert = blockIdx.y;
  if (by_place) {
    const int mine = blockIdx.y;
    expert = expert_at(p, mine / p.top, mine % p.top);
    if (expert < 0 || expert >= p.experts) return;
    int earlier = 0;
    for (int s = tid; s < mine; s += 64 * kUpWaves) earlier |= expert_at(p, s / p.top, s % p.top) == expert;
    if (__syncthreads_or(earlier)) return;
  }
  if (tid == 0) found = 0;
  __syncthreads();
  for (int s = tid; s < total; s += 64 * kUpWaves) {
    const int t = s / p.top, r = s - t * p.top;
    if (expert_at(p, t, r) == expert && !named_before(p, t, r, expert)) {
      float w = p.weights[t * p.weights_rs + r * p.weights_cs];
      for (int u = r + 1; u < p.top; ++u)
        if (expert_at(p, t, u) == expert) w += p.weights[t * p.weights_rs + u * p.weights_cs];
      const int at = atomicAdd(&found, 1);   // (in any order: a token's column does not touch its numbers)
      places[at] = s;
      weight[at] = w;
    }
  }
  __syncthreads();
  const int rows = found;
  if (rows == 0) return;

  const VECOPS_GLOBAL char* w_base = (const VECOPS_GLOBAL char*)p.gate_up + expert * p.gate_up_es * EB;
  const VECOPS_GLOBAL float* s_base = (const VECOPS_GLOBAL float*)p.gate_up_scales + expert * p.gs_es;
  const int blocks = (p.hidden + 127) / 128, tiles = p.inner_pad / 16;
  for (int base = 0; base < rows; base += 16 * MT) {
    const VECOPS_GLOBAL char* x[MT];
    bool there[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int at = base + j * 16 + col;
      there[j] = at < rows;
      x[j] = (const VECOPS_GLOBAL char*)p.x + (places[min(at, rows - 1)] / p.top) * p.ldx * 2;
    }
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      const int i0 = tile * 16, i = min(i0 + col, p.inner - 1);
      const VECOPS_GLOBAL char* w[2] = {w_base + i * p.gate_up_rs * EB, w_base + (static_cast<int64_t>(p.inner) + i) * p.gate_up_rs * EB};
      f32x4 acc[2][MT];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[h][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int b = wave; b < blocks; b += kUpWaves) {
        const int k0 = b * 128;
        u32x4 wv[2][LOADS], xv[MT][4];
        float scale[2][4];
        const bool whole = k0 + 128 <= p.hidden;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < LOADS; ++c) {
            const int k = k0 + chunk_k<W8>(W8 ? 2 * c : c, quarter);
            wv[h][c] = whole ? load_16(w[h] + k * EB) : load_16_until<EB>(w[h], k, p.hidden);
          }
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int k = k0 + chunk_k<W8>(c, quarter);
            xv[j][c] = u32x4{0u, 0u, 0u, 0u};
            if (there[j]) xv[j][c] = whole ? load_16(x[j] + k * 2) : load_16_until<2>(x[j], k, p.hidden);
          }
        if constexpr (W8) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) {   // (rows past the last one: a scale that exists)
              const int row = (h ? p.inner : 0) + min(i0 + quarter * 4 + r, p.inner - 1);
              scale[h][r] = s_base[(row >> 7) * p.gs_rs + b * p.gs_cs];
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            if constexpr (W8) {
              f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int c = 0; c < 4; ++c) part = mfma_16<F16>(widen<F16>(wv[h][c >> 1][(c & 1) * 2], wv[h][c >> 1][(c & 1) * 2 + 1]), xv[j][c], part);
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[h][j][r] = fmaf(part[r], scale[h][r], acc[h][j][r]);
            } else {
#pragma unroll
              for (int c = 0; c < 4; ++c) acc[h][j] = mfma_16<F16>(wv[h][c], xv[j][c], acc[h][j]);
            }
          }
      }
      __syncthreads();   // (the last tile's sums have been read)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4*>(&meet[wave][h][j][lane * 4]) = acc[h][j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int in_tile = (tid >> 6) * 4 + (tid & 3), row = base + j * 16 + ((tid >> 2) & 15);   // (lane tid / 4, its result tid % 4)
        if (row < rows) {
          float g = 0.f, u = 0.f;
#pragma unroll
          for (int s = 0; s < kUpWaves; ++s) g += meet[s][0][j][tid], u += meet[s][1][j][tid];
          const float v = i0 + in_tile < p.inner ? g / (1.0f + expf(-g)) * u * weight[row] : 0.0f;
          const uint32_t hi = bf16_bits_rne(v);
          const uint32_t lo = (hi & 0x7f80u) == 0x7f80u ? 0u : bf16_bits_rne(v - __uint_as_float(hi << 16));
          const int64_t at = static_cast<int64_t>(places[row]) * p.inner_pad + i0 + in_tile;
          p.middle[at] = static_cast<uint16_t>(hi);
          p.middle[static_cast<int64_t>(total) * p.inner_pad + at] = static_cast<uint16_t>(lo);
        }
      }
    }
  }
}

constexpr int kDownWaves = 8;

// A block of 16-bit weights as bf16: itself, or (f16) a bf16 and what that leaves, together exact.
__device__ __forceinline__ void split_f16(const u32x4& v, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float a = f16_bits_to_f32(v[c] & 0xffffu), b = f16_bits_to_f32(v[c] >> 16);
    hi[c] = cvt_pk_bf16(a, b);
    lo[c] = cvt_pk_bf16(a - __uint_as_float(hi[c] << 16), b - __uint_as_float(hi[c] & 0xffff0000u));
  }
}

// down, and the sum over a token's experts.  A workgroup owns sixteen columns of the result for all tokens: its wavefronts
// share the (expert, block of 128 inner) pairs out evenly, in order; a wavefront adds an expert's columns to its own sums of
// the tokens in LDS when it leaves the expert, and the wavefronts' sums are added at the end.  No sum depends on timing.
template <bool F16, bool W8, int MT>
__global__ __launch_bounds__(64 * kDownWaves) void moe_down_kernel(const MoeExpertsParams p) {
  constexpr int EB = W8 ? 1 : 2, LOADS = W8 ? 2 : 4;
  constexpr bool SPLIT = F16 && !W8;   // f16 weights against bf16 pairs
  extern __shared__ __attribute__((aligned(16))) float sums[];   // [wavefronts][tokens][16]
  __shared__ uint32_t named[kMoeMostExperts];                    // how often; then packed: first place of its run << 16 | length, of the active ones
  __shared__ uint16_t active[kMoeMostExperts];
  __shared__ uint16_t order[kMoeMostTokens * kMoeMostChoices];   // places by expert
  __shared__ uint32_t carry[kDownWaves];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int total = p.tokens * p.top;
  constexpr int THREADS = 64 * kDownWaves, PLACES = kMoeMostTokens * kMoeMostChoices / THREADS;
  static_assert(THREADS >= kMoeMostExperts, "a thread an expert");

  named[tid] = 0;
  for (int at = tid; at < kDownWaves * p.tokens * 16; at += THREADS) sums[at] = 0.f;
  __syncthreads();
  int expert_of[PLACES], nth[PLACES];
#pragma unroll
  for (int u = 0; u < PLACES; ++u) {
    const int s = u * THREADS + tid;
    expert_of[u] = -1;
    if (s < total) {
      const int t = s / p.top, r = s - t * p.top, e = expert_at(p, t, r);
      if (e >= 0 && e < p.experts && !named_before(p, t, r, e)) {
        expert_of[u] = e;
        nth[u] = static_cast<int>(atomicAdd(&named[e], 1u));   // (in any order, as above)
      }
    }
  }
  __syncthreads();
  // running sums over the experts of (places, active experts), packed
  const uint32_t mine = named[tid], pair = mine << 16 | (mine != 0 ? 1u : 0u);
  uint32_t run = pair;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t other = static_cast<uint32_t>(__shfl_up(static_cast<int>(run), d, 64));
    if (lane >= d) run += other;
  }
  if (lane == 63) carry[wave] = run;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w) before += carry[w];
  run += before;
  const uint32_t start = run - pair;   // what lies in front of this expert
  if (tid == THREADS - 1) count = static_cast<int>(run & 0xffffu);
  named[tid] = start >> 16;   // the first place of this expert's run
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PLACES; ++u)
    if (expert_of[u] >= 0) order[named[expert_of[u]] + nth[u]] = static_cast<uint16_t>(u * THREADS + tid);
  __syncthreads();
  if (mine != 0) active[start & 0xffffu] = static_cast<uint16_t>(tid);
  __syncthreads();
  named[tid] = (start >> 16) << 16 | mine;   // by expert: its run's first place and length
  __syncthreads();

  const int h0 = blockIdx.x * 16;
  const int blocks = (p.inner + 127) / 128, units = count * blocks;
  const int64_t row = min(h0 + col, p.hidden - 1);
  const int64_t lo_plane = static_cast<int64_t>(total) * p.inner_pad * 2;
  int unit = static_cast<int>(static_cast<int64_t>(units) * wave / kDownWaves);
  const int unit_end = static_cast<int>(static_cast<int64_t>(units) * (wave + 1) / kDownWaves);
  while (unit < unit_end) {
    const int nth_expert = unit / blocks, first = unit - nth_expert * blocks;
    const int last = min(blocks, first + unit_end - unit);
    const int expert = __builtin_amdgcn_readfirstlane(active[nth_expert]);
    const uint32_t its = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(named[expert])));
    const int from = static_cast<int>(its >> 16), rows = static_cast<int>(its & 0xffffu);
    const VECOPS_GLOBAL char* w = (const VECOPS_GLOBAL char*)p.down + (expert * p.down_es + row * p.down_rs) * EB;
    const VECOPS_GLOBAL float* s_base = (const VECOPS_GLOBAL float*)p.down_scales + expert * p.ds_es + (h0 >> 7) * p.ds_rs;
    for (int base = 0; base < rows; base += 16 * MT) {
      const VECOPS_GLOBAL char* x[MT];
      bool there[MT];
      int token[MT];
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int at = base + j * 16 + col, place = order[from + min(at, rows - 1)];
        there[j] = at < rows;
        token[j] = place / p.top;
        x[j] = (const VECOPS_GLOBAL char*)p.middle + static_cast<int64_t>(place) * p.inner_pad * 2;
      }
      f32x4 acc[MT];
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int b = first; b < last; ++b) {
        const int k0 = b * 128;
        const bool whole = k0 + 128 <= p.inner;
        u32x4 wv[LOADS], xh[MT][4], xl[MT][4];
        float scale = 1.0f;
#pragma unroll
        for (int c = 0; c < LOADS; ++c) {
          const int k = k0 + chunk_k<W8>(W8 ? 2 * c : c, quarter);
          wv[c] = whole ? load_16(w + k * EB) : load_16_until<EB>(w, k, p.inner);
        }
        if constexpr (W8) scale = s_base[b * p.ds_cs];
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int k = k0 + chunk_k<W8>(c, quarter);
            xh[j][c] = xl[j][c] = u32x4{0u, 0u, 0u, 0u};
            if (there[j] && k < p.inner) {   // (inner_pad, a multiple of sixteen, holds zeros past inner)
              xh[j][c] = load_16(x[j] + k * 2);
              xl[j][c] = load_16(x[j] + lo_plane + k * 2);
            }
          }
        f32x4 part[MT];
#pragma unroll
        for (int j = 0; j < MT; ++j) part[j] = W8 ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[j];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          u32x4 wh, wl;
          if constexpr (W8) wh = widen<false>(wv[c >> 1][(c & 1) * 2], wv[c >> 1][(c & 1) * 2 + 1]);
          else if constexpr (SPLIT) split_f16(wv[c], wh, wl);
          else wh = wv[c];
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            part[j] = mfma_16<false>(wh, xh[j][c], part[j]);
            part[j] = mfma_16<false>(wh, xl[j][c], part[j]);
            if constexpr (SPLIT) part[j] = mfma_16<false>(wl, xh[j][c], part[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          if constexpr (W8) {
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[j][r] = fmaf(part[j][r], scale, acc[j][r]);
          } else {
            acc[j] = part[j];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < MT; ++j)
        if (there[j]) {
          f32x4* at = reinterpret_cast<f32x4*>(&sums[(wave * p.tokens + token[j]) * 16 + quarter * 4]);
          f32x4 v = *at;
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] += acc[j][r];
          *at = v;
        }
    }
    unit += last - first;
  }
  __syncthreads();
  for (int at = tid; at < p.tokens * 16; at += THREADS) {
    const int t = at >> 4, h = h0 + (at & 15);
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kDownWaves; ++w) v += sums[(w * p.tokens + t) * 16 + (at & 15)];
    if (h < p.hidden) {
      const int64_t to = t * p.out_rs + h * p.out_cs;
      if (p.out_f32) static_cast<float*>(p.out)[to] = v;
      else static_cast<uint16_t*>(p.out)[to] = static_cast<uint16_t>(p.x_f16 ? f16_bits_rne(v) : bf16_bits_rne(v));
    }
  }
}

template <bool F16, bool W8, int MT>
hipError_t launch_experts(const MoeExpertsParams& p, hipStream_t stream) {
  const int places = p.tokens * p.top;
  if (places > 0 && p.inner > 0 && p.experts > 0) {
    // a workgroup an expert, or one a place where the places are fewer
    const int by_place = places < p.experts;
    const int tiles = p.inner_pad / 16;
    hipLaunchKernelGGL((moe_up_kernel<F16, W8, MT>), dim3(static_cast<uint32_t>(tiles), static_cast<uint32_t>(by_place ? places : p.experts)),
                       dim3(64 * kUpWaves), 0, stream, p, by_place);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const void* kernel = reinterpret_cast<const void*>(&moe_down_kernel<F16, W8, MT>);
  const int lds = kDownWaves * p.tokens * 16 * static_cast<int>(sizeof(float));
  if (lds > 32 * 1024) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kDownWaves * kMoeMostTokens * 16 * 4);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((moe_down_kernel<F16, W8, MT>), dim3(static_cast<uint32_t>((p.hidden + 15) / 16)), dim3(64 * kDownWaves), lds, stream, p);
  return hipGetLastError();
}

template <bool F16, bool W8>
hipError_t launch_experts_for(const MoeExpertsParams& p, hipStream_t stream) {
  if (p.tokens <= 16) return launch_experts<F16, W8, 1>(p, stream);
  if (p.tokens <= 32) return launch_experts<F16, W8, 2>(p, stream);
  return launch_experts<F16, W8, 4>(p, stream);
}

}  // namespace

int moe_route_parts(int hidden) {
  const int steps = (hidden + 31) / 32;
  return std::max(1, (steps + kRouteWaves * kRouteSteps - 1) / (kRouteWaves * kRouteSteps));
}

hipError_t launch_moe_route(const MoeRouteParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>((p.experts + 15) / 16), static_cast<uint32_t>(p.parts), static_cast<uint32_t>((p.tokens + 15) / 16));
  if (p.router_f32) {
    if (p.x_f16) hipLaunchKernelGGL((moe_logits_kernel<true, true>), grid, dim3(64 * kRouteWaves), 0, stream, p);
    else hipLaunchKernelGGL((moe_logits_kernel<false, true>), grid, dim3(64 * kRouteWaves), 0, stream, p);
  } else {
    if (p.x_f16) hipLaunchKernelGGL((moe_logits_kernel<true, false>), grid, dim3(64 * kRouteWaves), 0, stream, p);
    else hipLaunchKernelGGL((moe_logits_kernel<false, false>), grid, dim3(64 * kRouteWaves), 0, stream, p);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(moe_choose_kernel, dim3(static_cast<uint32_t>(p.tokens)), dim3(64), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_moe_experts(const MoeExpertsParams& p, hipStream_t stream) {
  if (p.x_f16) return p.w_e4m3 ? launch_experts_for<true, true>(p, stream) : launch_experts_for<true, false>(p, stream);
  return p.w_e4m3 ? launch_experts_for<false, true>(p, stream) : launch_experts_for<false, false>(p, stream);
}

}  // namespace vecops_hip
