// A mixture-of-experts layer for a few tokens:
//   l = x . router^T;  the experts of the largest scores;  out = sum_r w_r down[e_r] . (silu(gate[e_r] . x) * (up[e_r] . x))
// What bounds it: the weights of the experts that the tokens name are read once from HBM, against a handful of rows; the rest
// is latency.  Launches: the logits, the choice (for a few tokens in front of the next, in it), gate and up with the
// activation, down with the sum over a token's experts.  The tokens of an expert are the columns of a matrix instruction whose
// rows are sixteen rows of weights, which go from memory straight into registers.
#include "moe_few_tokens.h"

#include <algorithm>

#include "lane_exchange.h"

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

// The first elements of a 16-bit chunk cleared: those that lie below `clear` (0 or less: none).
__device__ __forceinline__ u32x4 cleared(const u32x4& v, int clear) {
  u32x4 out;
#pragma unroll
  for (int d = 0; d < 4; ++d) out[d] = v[d] & (clear <= 2 * d ? 0xffffffffu : clear == 2 * d + 1 ? 0xffff0000u : 0u);
  return out;
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
// its wavefronts split again; the shares are added where the experts are chosen.  A wavefront asks for all that it multiplies at
// once (64 tokens, 128 experts, hidden 2048: 8.4 us with a step's loads behind the step before, 4.7 so).
// ---------------------------------------------------------------------------------------------------------------------

constexpr int kRouteWaves = 4, kRouteSteps = 4;  // steps of 32 that a wavefront has at most in its share

template <bool F16, bool R32, bool TINY>
__global__ __launch_bounds__(64 * kRouteWaves) void moe_logits_kernel(const MoeRouteParams p) {
  __shared__ float meet[kRouteWaves][256];
  const int lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e0 = blockIdx.x * 16, t0 = blockIdx.z * 16;
  const VECOPS_GLOBAL char* r = (const VECOPS_GLOBAL char*)p.router + static_cast<int64_t>(min(e0 + col, p.experts - 1)) * p.ld_router * (R32 ? 4 : 2);
  const VECOPS_GLOBAL char* x = (const VECOPS_GLOBAL char*)p.x + static_cast<int64_t>(min(t0 + col, p.tokens - 1)) * p.ldx * 2;
  const int steps = (p.hidden + 31) / 32, first = static_cast<int>(static_cast<int64_t>(steps) * blockIdx.y / p.parts),
            end = static_cast<int>(static_cast<int64_t>(steps) * (blockIdx.y + 1) / p.parts);
  u32x4 xv[kRouteSteps], rv[kRouteSteps][R32 ? 2 : 1];
  int clear[kRouteSteps];   // of the eight elements, those that another step or lane has
#pragma unroll
  for (int u = 0; u < kRouteSteps; ++u) {
    const int s = first + wave + u * kRouteWaves, k = s * 32 + quarter * 8, from = TINY ? k : min(k, p.hidden - 8);
    clear[u] = s < end ? k - from : 8;
    if constexpr (TINY) {
      xv[u] = load_16_until<2>(x, k, p.hidden);
      rv[u][0] = load_16_until<R32 ? 4 : 2>(r, k, p.hidden);
      if constexpr (R32) rv[u][1] = load_16_until<4>(r, k + 4, p.hidden);
    } else {
      xv[u] = load_16(x + static_cast<int64_t>(from) * 2);
      rv[u][0] = load_16(r + static_cast<int64_t>(from) * (R32 ? 4 : 2));
      if constexpr (R32) rv[u][1] = load_16(r + static_cast<int64_t>(from) * 4 + 16);
    }
  }
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < kRouteSteps; ++u) {
    const u32x4 xs = cleared(xv[u], clear[u]);
    if constexpr (R32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {   // instruction i multiplies element i of every lane
        const uint32_t bits = (xs[i >> 1] >> (16 * (i & 1))) & 0xffffu;
        const float xf = F16 ? f16_bits_to_f32(bits) : __uint_as_float(bits << 16);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(i >= clear[u] ? __uint_as_float(rv[u][i >> 2][i & 3]) : 0.0f, xf, acc, 0, 0, 0);
      }
    } else {
      acc = mfma_16<F16>(cleared(rv[u][0], clear[u]), xs, acc);
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

// A reduction over the wavefront, by moves within rows of sixteen lanes and from row to row: the last lane has all of it.
template <typename Join>
__device__ __forceinline__ uint32_t over_wave(uint32_t v, uint32_t none, Join join) {
#if defined(__HIP_DEVICE_COMPILE__)
  v = join(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(none, v, 0x111, 0xf, 0xf, false)));   // from one, two, four, eight
  v = join(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(none, v, 0x112, 0xf, 0xf, false)));   // lanes below in the row
  v = join(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(none, v, 0x114, 0xf, 0xf, false)));
  v = join(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(none, v, 0x118, 0xf, 0xf, false)));
  v = join(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(none, v, 0x142, 0xa, 0xf, false)));   // rows 0, 2 into 1, 3
  v = join(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(none, v, 0x143, 0xc, 0xf, false)));   // row 1 into 2, 3
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
#else
  (void)none; (void)join;
  return v;
#endif
}
__device__ __forceinline__ float wave_max(float v) {
  return __uint_as_float(over_wave(__float_as_uint(v), 0xff800000u, [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
__device__ __forceinline__ float wave_sum(float v) {
  return __uint_as_float(over_wave(__float_as_uint(v), 0u, [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}

// The choice for a token, by a wavefront: lane l has the experts l, l + 64, ...; `top` times the largest that is left, the lower
// index among equals.  Lane r returns choice r and its weight.  What bounds it
// is the chain from choice to choice: each is a reduction of 32 bits by moves between lanes and a search for the first lane that
// has them, none of it through LDS (64 tokens, 8 of 128 experts: 5.5 us).
__device__ __forceinline__ void choose(const MoeRouteParams& p, int t, int lane, int& id, float& weight) {
  constexpr int MOST = kMoeMostExperts / 64;
  float score[MOST], bias[MOST];
  uint32_t key[MOST];
  float most = -__builtin_huge_valf();
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    const int e = lane + 64 * j;
    score[j] = -__builtin_huge_valf();
    key[j] = 0;
    bias[j] = 0.f;
    if (e < p.experts) {
      if (p.bias != nullptr) bias[j] = p.bias[e];
      float l = 0.f;
#pragma unroll 4
      for (int s = 0; s < p.parts; ++s) l += p.logits[(static_cast<int64_t>(s) * p.tokens + t) * p.experts + e];
      score[j] = l;
      key[j] = order_of(l);   // (0 is below every number's)
      most = fmaxf(most, l);
    }
  }
  if (p.sigmoid) {
#pragma unroll
    for (int j = 0; j < MOST; ++j)
      if (64 * j < p.experts) score[j] = 1.0f / (1.0f + expf(-score[j]));
  } else {
    most = wave_max(most);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < MOST; ++j)
      if (64 * j < p.experts) {
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
      if (lane + 64 * j < p.experts) key[j] = order_of(score[j] + bias[j]);
  }
  float chosen = 0.f, total = 0.f;   // lane r keeps the score of choice r
  id = 0;
  for (int r = 0; r < p.top; ++r) {
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < MOST; ++j) mine = max(mine, key[j]);
    const uint32_t best = over_wave(mine, 0u, [](uint32_t a, uint32_t b) { return max(a, b); });
    int e = -1;
    float its = 0.f;
#pragma unroll
    for (int j = 0; j < MOST; ++j) {
      if (e < 0 && 64 * j < p.experts) {   // (the same in all lanes)
        const uint64_t have = __ballot(key[j] == best);
        if (have != 0) {
          const int first = __builtin_ctzll(have);
          e = 64 * j + first;
          its = __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(score[j])), first)));
          if (lane == first) key[j] = 0;   // taken
        }
      }
    }
    if (lane == r) chosen = its, id = e;
    total += its;
  }
  weight = (p.renormalize ? chosen / total : chosen) * p.scale;
}

__global__ __launch_bounds__(64) void moe_choose_kernel(const MoeRouteParams p) {
  const int t = blockIdx.x, lane = threadIdx.x;
  int id;
  float weight;
  choose(p, t, lane, id, weight);
  if (lane < p.top) {
    p.ids[t * p.ids_rs + lane * p.ids_cs] = id;
    p.weights[t * p.weights_rs + lane * p.weights_cs] = weight;
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Experts.  A place (token, choice) whose expert an earlier choice of the same token names too adds its weight to that one.
// ---------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ int expert_at(const MoeExpertsParams& p, int place) {
  const int t = place / p.top;
  return p.ids[t * p.ids_rs + (place - t * p.top) * p.ids_cs];
}

// Whether an earlier choice of a place's token names the same expert (ids: all of them, by place).
__device__ __forceinline__ bool named_before(const int* ids, int place, int choice) {
  bool found = false;
  for (int r = 1; r <= choice; ++r) found |= ids[place - r] == ids[place];
  return found;
}

// Weights from memory into a matrix instruction's operand: a lane there holds sixteen bytes of row (lane % 16), the lanes of a
// quarter of the wavefront the same bytes of their rows.  Loaded like that every lane is a look-up in the cache of its own, and
// those bound the kernels (0.7 of them a cycle).  So neighbouring lanes load neighbouring sixteen bytes of one row, as many as
// there are loads (four, or two of e4m3, whose scales end a block of 128 k), a load each of as many rows, and exchange them, and
// activations likewise.  Gate and up, then down (us): 5 tokens, 4 of 60 of 1001 x 1411 in f16 35, 25.4 -> 24.4, 22.7; 64 tokens,
// 8 of 128 of 2048 x 768 in e4m3 90, 59 -> 86, 53; 16 tokens, 2 of 8 of 4096 x 14336 in bf16 315, 196 -> 309 (6.1 TB/s), 174 (5.4).
// Lane l holds then, of a block of 128 k, the thirty-two from 32 (l / 16) on, and so it has the activations.
//
// A row ends where it ends: sixteen bytes that the end lies in, or in front of, are replaced by those in front of the end, and so
// are the activations that go with them; what another lane or load has is cleared when they are used, in both, since either
// may hold an infinity (an e4m3 has none, and its NaN reaches the result from the other load as well).  (Rows of less than
// sixteen bytes, TINY, are read element by element.)
template <bool W8, bool TINY>
struct Chunks {
  static constexpr int EB = W8 ? 1 : 2, EPL = 16 / EB, LOADS = W8 ? 2 : 4;   // bytes, elements a load, loads of weights
  __device__ __forceinline__ static int from(int k, int count) { return min(k, count - EPL); }
  // which of sixteen rows load c of this lane is of
  __device__ __forceinline__ static int row(int c, int lane) { return (lane & 15 & ~(LOADS - 1)) + c; }
  __device__ __forceinline__ static u32x4 weight(const VECOPS_GLOBAL char* row, int k0, int lane, int count) {
    const int k = k0 + (lane >> 4) * 32 + (lane & (LOADS - 1)) * EPL;
    if constexpr (TINY) return load_16_until<EB>(row, k, count);
    else return load_16(row + static_cast<int64_t>(from(k, count)) * EB);
  }
  // load c of lane l becomes load l % COUNT of lane c of its group
  template <int COUNT>
  __device__ __forceinline__ static void exchange(u32x4 (&v)[COUNT], int lane) {
    exchange_lanes<kNextLane>(v[0], v[1], lane & 1);
    if constexpr (COUNT == 4) {
      exchange_lanes<kNextLane>(v[2], v[3], lane & 1);
      exchange_lanes<kNextButOne>(v[0], v[2], lane & 2);
      exchange_lanes<kNextButOne>(v[1], v[3], lane & 2);
    }
  }
  // four chunks of eight 16-bit elements, of a token each as a load of weights is of a row each
  __device__ __forceinline__ static int token(int c, int lane) { return (lane & 12) + c; }
  __device__ __forceinline__ static u32x4 activation(const VECOPS_GLOBAL char* row, int k0, int lane, int count, bool there) {
    const int chunk = lane & 3, in = W8 ? (chunk & 1) * 8 : 0, k = k0 + (lane >> 4) * 32 + chunk * 8 - in;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (there) {
      if constexpr (TINY) v = load_16_until<2>(row, k + in, count);
      else v = load_16(row + static_cast<int64_t>(from(k, count) + in) * 2);
    }
    return v;
  }
  // at the block that `count` lies in
  __device__ __forceinline__ static void clear(u32x4 (&v)[4], int k0, int quarter, int count) {
    if constexpr (!TINY) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int in = W8 ? (c & 1) * 8 : 0, k = k0 + quarter * 32 + c * 8 - in;
        v[c] = cleared(v[c], k - from(k, count) - in);
      }
    }
  }
  __device__ __forceinline__ static void clear_weights(u32x4 (&v)[LOADS], int k0, int quarter, int count) {
    if constexpr (!TINY && !W8) clear(v, k0, quarter, count);
  }
};

constexpr int kUpWaves = 4;

// gate and up.  A workgroup: one expert, the tokens that name it (16 MT at a time), every gridDim.x-th block of sixteen gate rows
// and their up rows.  Its wavefronts take the blocks of 128 of the hidden axis in turn, the loads of DEPTH of them under way,
// across the ends of row blocks; their sums meet in LDS.  (More workgroups a compute unit do better than more blocks
// under way in each: 128 tokens, 2 of 8 of 4096 x 4096 in bf16, two with one block 225 us, one with two 286; 64 tokens, 8 of 128
// of 2048 x 768 in e4m3, three with two blocks 138, two with four 144.)
// (Loads return in order: activations asked for when they are needed would wait for the weights asked for ahead of them.)
// CHOOSES: the experts are not chosen yet, and every workgroup chooses them, a wavefront a token; the first one writes the choice.
template <bool F16, bool W8, int MT, bool TINY, bool CHOOSES>
__global__ __launch_bounds__(64 * kUpWaves, MT == 4 ? 2 : 3) void moe_up_kernel(const MoeExpertsParams p, const MoeRouteParams route, int by_place) {
  using C = Chunks<W8, TINY>;
  constexpr int EB = C::EB, LOADS = C::LOADS, DEPTH = !TINY && MT == 1 ? 2 : 1, THREADS = 64 * kUpWaves;
  __shared__ f32x4 meet[2][kUpWaves][2][MT][64];
  __shared__ int ids[kMoeMostTokens * kMoeMostChoices];
  __shared__ int places[kMoeMostTokens];
  __shared__ float weight[kMoeMostTokens];
  __shared__ float chosen[CHOOSES ? kUpWaves * kMoeMostChoices : 1];   // the weights
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int total = p.tokens * p.top;

  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int at = tid; at < (p.hidden + 15) / 16; at += THREADS) p.arrived[at] = 0;   // for the kernel behind this one
  if constexpr (CHOOSES) {
    if (wave < p.tokens) {
      int id;
      float w;
      choose(route, wave, lane, id, w);
      if (lane < p.top) {
        ids[wave * p.top + lane] = id;
        chosen[wave * p.top + lane] = w;
        if (blockIdx.x == 0 && blockIdx.y == 0) {
          route.ids[wave * p.ids_rs + lane * p.ids_cs] = id;
          route.weights[wave * p.weights_rs + lane * p.weights_cs] = w;
        }
      }
    }
  } else {
    for (int s = tid; s < total; s += THREADS) ids[s] = expert_at(p, s);
  }
  if (tid == 0) found = 0;
  __syncthreads();
  // the expert: blockIdx.y itself, or the one that place blockIdx.y is the first to name
  int expert = blockIdx.y;
  if (by_place) {
    const int mine = blockIdx.y;
    expert = ids[mine];
    if (expert < 0 || expert >= p.experts) return;
    int earlier = 0;
    for (int s = tid; s < mine; s += THREADS) earlier |= ids[s] == expert;
    if (__syncthreads_or(earlier)) return;
  }
  for (int s = tid; s < total; s += THREADS) {
    const int t = s / p.top, r = s - t * p.top;
    if (ids[s] == expert && !named_before(ids, s, r)) {
      float w;
      if constexpr (CHOOSES) {   // (no expert twice)
        w = chosen[s];
      } else {
        w = p.weights[t * p.weights_rs + r * p.weights_cs];
        for (int u = r + 1; u < p.top; ++u)
          if (ids[t * p.top + u] == expert) w += p.weights[t * p.weights_rs + u * p.weights_cs];
      }
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
  const int mine = wave < blocks ? (blocks - wave + kUpWaves - 1) / kUpWaves : 0;   // this wavefront's blocks of a row block
  const int tile_count = (tiles - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const int steps = mine * tile_count;
  for (int base = 0; base < rows; base += 16 * MT) {
    const VECOPS_GLOBAL char* x[MT][4];
    bool there[MT][4];
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int at = base + j * 16 + C::token(c, lane);
        there[j][c] = at < rows;
        x[j][c] = (const VECOPS_GLOBAL char*)p.x + (places[min(at, rows - 1)] / p.top) * p.ldx * 2;
      }
    u32x4 wv[DEPTH][2][LOADS], xv[DEPTH][MT][4];
    float sv[DEPTH][2][2];
    // where the next loads go: row block, block of k
    int load_tile = blockIdx.x, load_block = wave;
    auto load = [&](auto slot_tag) __attribute__((always_inline)) {
      constexpr int slot = decltype(slot_tag)::value;
      const int i0 = load_tile * 16, k0 = load_block * 128;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < LOADS; ++c) {
          const int64_t row = (h ? p.inner : 0) + min(i0 + C::row(c, lane), p.inner - 1);
          wv[slot][h][c] = C::weight(w_base + row * p.gate_up_rs * EB, k0, lane, p.hidden);
        }
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) xv[slot][j][c] = C::activation(x[j][c], k0, lane, p.hidden, there[j][c]);
      if constexpr (W8) {   // the scales of a lane's first row and of its last one, which may lie in another block of rows
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            sv[slot][h][e] = s_base[(((h ? p.inner : 0) + min(i0 + quarter * 4 + 3 * e, p.inner - 1)) >> 7) * p.gs_rs + load_block * p.gs_cs];
      }
      load_block += kUpWaves;
      if (load_block >= blocks) load_block = wave, load_tile += gridDim.x;
    };
    f32x4 acc[2][MT];
    int tile = blockIdx.x, nth = 0, block = 0;   // the row block that is multiplied, its number here, and the block of k
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[h][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    // the end of a row block: sums, activation, the inner values' pairs
    auto finish = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < MT; ++j) meet[nth & 1][wave][h][j][lane] = acc[h][j];
      __syncthreads();   // (the other half of `meet` is written next: its readers have passed this)
      for (int at = tid; at < MT * 256; at += THREADS) {
        const int j = at >> 8, in = at & 255, in_tile = (in >> 6) * 4 + (in & 3), row = base + j * 16 + ((in >> 2) & 15);   // (lane in / 4, its result in % 4)
        if (row < rows) {
          float g = 0.f, u = 0.f;
#pragma unroll
          for (int s = 0; s < kUpWaves; ++s) {
            g += reinterpret_cast<const float*>(&meet[nth & 1][s][0][j][0])[in];
            u += reinterpret_cast<const float*>(&meet[nth & 1][s][1][j][0])[in];
          }
          const int i = tile * 16 + in_tile;
          const float v = i < p.inner ? g / (1.0f + expf(-g)) * u * weight[row] : 0.0f;
          const uint32_t hi = bf16_bits_rne(v);
          const uint32_t lo = (hi & 0x7f80u) == 0x7f80u ? 0u : bf16_bits_rne(v - __uint_as_float(hi << 16));
          const int64_t to = static_cast<int64_t>(places[row]) * p.inner_pad + i;
          p.middle[to] = static_cast<uint16_t>(hi);
          p.middle[static_cast<int64_t>(total) * p.inner_pad + to] = static_cast<uint16_t>(lo);
        }
      }
      tile += gridDim.x;
      ++nth;
      block = 0;
      clear();
    };
    clear();
    static_for<DEPTH>([&](auto u) {
      if (decltype(u)::value < steps) load(u);
    });
    if (mine == 0) {   // (fewer blocks than wavefronts)
      for (int t = 0; t < tile_count; ++t) finish();
    }
    for (int s0 = 0; s0 < steps; s0 += DEPTH) {
      static_for<DEPTH>([&](auto slot_tag) {
        constexpr int slot = decltype(slot_tag)::value;
        if (s0 + slot < steps) {
          const int i0 = tile * 16 + quarter * 4, k0 = (wave + block * kUpWaves) * 128;
#pragma unroll
          for (int h = 0; h < 2; ++h) C::exchange(wv[slot][h], lane);
#pragma unroll
          for (int j = 0; j < MT; ++j) C::exchange(xv[slot][j], lane);
          if (k0 + 128 > p.hidden) {
#pragma unroll
            for (int j = 0; j < MT; ++j) C::clear(xv[slot][j], k0, quarter, p.hidden);
#pragma unroll
            for (int h = 0; h < 2; ++h) C::clear_weights(wv[slot][h], k0, quarter, p.hidden);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              if constexpr (W8) {
                f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 4; ++c)
                  part = mfma_16<F16>(widen<F16>(wv[slot][h][c >> 1][(c & 1) * 2], wv[slot][h][c >> 1][(c & 1) * 2 + 1]), xv[slot][j][c], part);
                const int row = (h ? p.inner : 0) + i0;
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[h][j][r] = fmaf(part[r], ((row + r) ^ row) >> 7 ? sv[slot][h][1] : sv[slot][h][0], acc[h][j][r]);
              } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[h][j] = mfma_16<F16>(wv[slot][h][c], xv[slot][j][c], acc[h][j]);
              }
            }
          if (s0 + slot + DEPTH < steps) load(slot_tag);
          if (++block == mine) finish();
        }
      });
    }
    if (base + 16 * MT < rows) __syncthreads();   // (`meet` begins again)
  }
}

// f16 weights as a bf16 and what that leaves, together exact (an infinity leaves nothing).
__device__ __forceinline__ void split_f16(const u32x4& v, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float a = f16_bits_to_f32(v[c] & 0xffffu), b = f16_bits_to_f32(v[c] >> 16);
    hi[c] = cvt_pk_bf16(a, b);
    const float la = a - __uint_as_float(hi[c] << 16), lb = b - __uint_as_float(hi[c] & 0xffff0000u);
    lo[c] = cvt_pk_bf16(la == la ? la : 0.0f, lb == lb ? lb : 0.0f);
  }
}

// down, and the sum over a token's experts.  A workgroup owns sixteen columns of the result for all tokens, and one of gridDim.y
// shares of the work: the tokens of an expert, 8 MT at most, are a segment, and the wavefronts of all shares split the (segment,
// block of 128 inner) pairs evenly among them, in order, the loads of DEPTH pairs under way across the ends of segments.  Of a
// matrix instruction's sixteen columns eight take the upper halves of eight tokens' inner values and eight the lower ones,
// which meet when a wavefront leaves a segment and adds its columns to its own sums of the tokens in LDS.  The wavefronts' sums
// are added at the end, and the shares' by the workgroup that comes last, in order: no sum depends on which one that is.
constexpr int kDownWaves = 8;

template <bool F16, bool W8, int MT, bool TINY>
__global__ __launch_bounds__(64 * kDownWaves, 2) void moe_down_kernel(const MoeExpertsParams p) {
  using C = Chunks<W8, TINY>;
  constexpr int EB = C::EB, LOADS = C::LOADS, DEPTH = TINY ? 1 : MT == 1 ? (W8 ? 6 : 4) : MT == 2 ? 2 : 1;
  constexpr bool SPLIT = F16 && !W8;   // f16 weights against bf16 pairs
  constexpr int THREADS = 64 * kDownWaves, PLACES = kMoeMostTokens * kMoeMostChoices / THREADS, TOKENS = 8 * MT;
  constexpr int SEGMENTS = kMoeMostExperts + kMoeMostTokens * kMoeMostChoices / TOKENS;
  static_assert(THREADS >= kMoeMostExperts, "a thread an expert");
  extern __shared__ __attribute__((aligned(16))) float sums[];   // [wavefronts][tokens][16]
  __shared__ int ids[kMoeMostTokens * kMoeMostChoices];
  __shared__ uint32_t naming[kMoeMostExperts][kMoeMostTokens / 32];   // by expert: a bit for each token that names it
  __shared__ uint16_t first_of[kMoeMostExperts];                 // where an expert's run in `order` begins
  __shared__ uint32_t segment[SEGMENTS];                         // expert << 20 | tokens << 12 | first of them in `order`
  __shared__ uint16_t order[kMoeMostTokens * kMoeMostChoices];   // places by expert, then by token: the same in every workgroup
  __shared__ uint32_t carry[kDownWaves];
  __shared__ int count, last;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int total = p.tokens * p.top;

#pragma unroll
  for (int w = 0; w < kMoeMostTokens / 32; ++w) naming[tid][w] = 0;
  for (int s = tid; s < total; s += THREADS) ids[s] = expert_at(p, s);
  for (int at = tid; at < kDownWaves * p.tokens * 16; at += THREADS) sums[at] = 0.f;
  __syncthreads();
  int expert_of[PLACES];   // of this thread's places: -1 for those that name none, or none for the first time
#pragma unroll
  for (int u = 0; u < PLACES; ++u) {
    const int s = u * THREADS + tid;
    expert_of[u] = -1;
    if (s < total) {
      const int e = ids[s], t = s / p.top;
      if (e >= 0 && e < p.experts && !named_before(ids, s, s - t * p.top)) {
        expert_of[u] = e;
        atomicOr(&naming[e][t >> 5], 1u << (t & 31));
      }
    }
  }
  __syncthreads();
  // running sums over the experts of (places, segments), packed
  uint32_t mine = 0;
#pragma unroll
  for (int w = 0; w < kMoeMostTokens / 32; ++w) mine += __popc(naming[tid][w]);
  const uint32_t segments = (mine + TOKENS - 1) / TOKENS, pair = mine << 16 | segments;
  uint32_t run = pair;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t other = static_cast<uint32_t>(__shfl_up(static_cast<int>(run), d, 64));
    if (lane >= d) run += other;
  }
  if (lane == 63) carry[wave] = run;
  __syncthreads();
  for (int w = 0; w < wave; ++w) run += carry[w];
  const uint32_t start = run - pair;   // what lies in front of this expert
  if (tid == THREADS - 1) count = static_cast<int>(run & 0xffffu);
  first_of[tid] = static_cast<uint16_t>(start >> 16);
  for (uint32_t g = 0; g < segments; ++g)
    segment[(start & 0xffffu) + g] = static_cast<uint32_t>(tid) << 20 | min(mine - g * TOKENS, static_cast<uint32_t>(TOKENS)) << 12 | ((start >> 16) + g * TOKENS);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PLACES; ++u)
    if (expert_of[u] >= 0) {
      const int s = u * THREADS + tid, t = s / p.top;
      int at = first_of[expert_of[u]];
#pragma unroll
      for (int w = 0; w < kMoeMostTokens / 32; ++w) {
        const uint32_t bits = naming[expert_of[u]][w];
        at += __popc(t >= 32 * (w + 1) ? bits : t < 32 * w ? 0u : bits & ((1u << (t & 31)) - 1u));
      }
      order[at] = static_cast<uint16_t>(s);
    }
  __syncthreads();

  const int h0 = blockIdx.x * 16;
  const int blocks = (p.inner + 127) / 128;
  const int64_t units = static_cast<int64_t>(count) * blocks;
  const int shares = gridDim.y * kDownWaves, share = blockIdx.y * kDownWaves + wave;
  const int begin = static_cast<int>(units * share / shares), end = static_cast<int>(units * (share + 1) / shares);
  if (begin < end) {
    const VECOPS_GLOBAL char* w_row[LOADS];
#pragma unroll
    for (int c = 0; c < LOADS; ++c)
      w_row[c] = (const VECOPS_GLOBAL char*)p.down + static_cast<int64_t>(min(h0 + C::row(c, lane), p.hidden - 1)) * p.down_rs * EB;
    const VECOPS_GLOBAL float* s_row = (const VECOPS_GLOBAL float*)p.down_scales + (h0 >> 7) * p.ds_rs;
    // upper halves for the columns below eight, lower ones for the others
    const VECOPS_GLOBAL char* x_plane = (const VECOPS_GLOBAL char*)p.middle + (col >> 3) * (static_cast<int64_t>(total) * p.inner_pad * 2);
    u32x4 wv[DEPTH][LOADS], xv[DEPTH][MT][4];
    float sv[DEPTH];
    // where the next loads go
    int load_segment = begin / blocks, load_block = begin - load_segment * blocks;
    int64_t load_expert = 0;
    const VECOPS_GLOBAL char* x[MT][4];
    bool there[MT][4];
    auto aim = [&]() __attribute__((always_inline)) {
      const uint32_t its = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(segment[min(load_segment, count - 1)])));
      const int from = static_cast<int>(its & 0xfffu), rows = static_cast<int>(its >> 12 & 0xffu);
      load_expert = static_cast<int64_t>(its >> 20);
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int at = j * 8 + (C::token(c, lane) & 7);
          there[j][c] = at < rows;
          x[j][c] = x_plane + static_cast<int64_t>(order[from + min(at, rows - 1)]) * p.inner_pad * 2;
        }
    };
    auto load = [&](auto slot_tag) __attribute__((always_inline)) {
      constexpr int slot = decltype(slot_tag)::value;
      const int k0 = load_block * 128;
#pragma unroll
      for (int c = 0; c < LOADS; ++c) wv[slot][c] = C::weight(w_row[c] + load_expert * p.down_es * EB, k0, lane, p.inner);
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) xv[slot][j][c] = C::activation(x[j][c], k0, lane, p.inner, there[j][c]);
      if constexpr (W8) sv[slot] = s_row[load_expert * p.ds_es + load_block * p.ds_cs];
      if (++load_block == blocks) {
        load_block = 0;
        ++load_segment;
        aim();
      }
    };
    f32x4 acc[MT], less[SPLIT ? MT : 1];   // `less`: what a weight's second half gives
    int at_segment = load_segment, block = load_block;
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (SPLIT) less[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    };
    auto leave = [&]() __attribute__((always_inline)) {
      const uint32_t its = segment[at_segment];
      const int from = static_cast<int>(its & 0xfffu), rows = static_cast<int>(its >> 12 & 0xffu);
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // what the second halves give; next to an infinity it may be a NaN, or of the other sign
          float second = __shfl_xor(acc[j][r], 8, 64);
          if constexpr (SPLIT) second += less[j][r] + __shfl_xor(less[j][r], 8, 64);
          v[r] = acc[j][r] + (fabsf(acc[j][r]) < __builtin_huge_valf() ? second : 0.0f);
        }
        const int at = j * 8 + col;
        if (col < 8 && at < rows) {
          f32x4* to = reinterpret_cast<f32x4*>(&sums[(wave * p.tokens + order[from + at] / p.top) * 16 + quarter * 4]);
          const f32x4 old = *to;
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] += old[r];
          *to = v;
        }
      }
    };
    aim();
    static_for<DEPTH>([&](auto u) {
      if (begin + decltype(u)::value < end) load(u);
    });
    clear();
    for (int u0 = begin; u0 < end; u0 += DEPTH) {
      static_for<DEPTH>([&](auto slot_tag) {
        constexpr int slot = decltype(slot_tag)::value;
        if (u0 + slot < end) {
          C::exchange(wv[slot], lane);
#pragma unroll
          for (int j = 0; j < MT; ++j) C::exchange(xv[slot][j], lane);
          if ((block + 1) * 128 > p.inner) {
#pragma unroll
            for (int j = 0; j < MT; ++j) C::clear(xv[slot][j], block * 128, quarter, p.inner);
            C::clear_weights(wv[slot], block * 128, quarter, p.inner);
          }
          f32x4 part[MT];
#pragma unroll
          for (int j = 0; j < MT; ++j) part[j] = W8 ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[j];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            u32x4 wh, wl;
            if constexpr (W8) wh = widen<false>(wv[slot][c >> 1][(c & 1) * 2], wv[slot][c >> 1][(c & 1) * 2 + 1]);
            else if constexpr (SPLIT) split_f16(wv[slot][c], wh, wl);
            else wh = wv[slot][c];
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              part[j] = mfma_16<false>(wh, xv[slot][j][c], part[j]);
              if constexpr (SPLIT) less[j] = mfma_16<false>(wl, xv[slot][j][c], less[j]);
            }
          }
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            if constexpr (W8) {
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[j][r] = fmaf(part[j][r], sv[slot], acc[j][r]);
            } else {
              acc[j] = part[j];
            }
          }
          if (u0 + slot + DEPTH < end) load(slot_tag);
          if (++block == blocks || u0 + slot + 1 == end) {
            leave();
            clear();
            block = 0;
            ++at_segment;
          }
        }
      });
    }
  }
  __syncthreads();
  const bool alone = gridDim.y == 1;
  for (int at = tid; at < p.tokens * 16; at += THREADS) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kDownWaves; ++w) v += sums[w * p.tokens * 16 + at];
    if (alone) sums[at] = v;   // (this thread's own number of the first wavefront's)
    else __hip_atomic_store(&p.shares[(static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * p.tokens * 16 + at], v, __ATOMIC_RELAXED,
                            __HIP_MEMORY_SCOPE_AGENT);
  }
  if (!alone) {
    // Each wavefront's numbers have to be in memory before the counter says so: neither the barrier nor the release below, which
    // is one wavefront's, waits for another one's stores.  (A release by every wavefront would, but it writes the
    // die's cache back each time.)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) last = __hip_atomic_fetch_add(&p.arrived[blockIdx.x], 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == static_cast<int>(gridDim.y) - 1;
    __syncthreads();
    if (!last) return;
  }
  for (int at = tid; at < p.tokens * 16; at += THREADS) {
    const int t = at >> 4, h = h0 + (at & 15);
    float v = 0.f;
    if (alone) {
      v = sums[at];
    } else {
      for (uint32_t s = 0; s < gridDim.y; ++s)
        v += __hip_atomic_load(&p.shares[(static_cast<int64_t>(s) * gridDim.x + blockIdx.x) * p.tokens * 16 + at], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (h < p.hidden) {
      const int64_t to = t * p.out_rs + h * p.out_cs;
      if (p.out_f32) static_cast<float*>(p.out)[to] = v;
      else static_cast<uint16_t*>(p.out)[to] = static_cast<uint16_t>(p.x_f16 ? f16_bits_rne(v) : bf16_bits_rne(v));
    }
  }
}

bool has_work(const MoeExpertsParams& p) { return p.tokens * p.top > 0 && p.inner > 0 && p.experts > 0; }
// Rows of less than sixteen bytes of e4m3.
bool is_tiny(const MoeExpertsParams& p) { return std::min(p.hidden, p.inner) < 16; }

template <bool F16, bool W8, int MT, bool TINY, bool CHOOSES>
hipError_t launch_up(const MoeExpertsParams& p, const MoeRouteParams& route, hipStream_t stream) {
  // a workgroup an expert, or one a place where the places are fewer
  const int places = p.tokens * p.top, by_place = places < p.experts;
  const int tiles = p.inner_pad / 16, lines = by_place ? places : p.experts;
  // About six workgroups a compute unit, of equally many blocks of rows: fewer leave compute units without work where experts
  // are named unevenly (4 tokens x 6 of 64 experts, 2048 x 1408: 89 us with 512, 76 with 1536), more have each too little
  // behind its search for tokens (64 x 8 of 128, 2048 x 768 in e4m3: 147 us with 1536, 170 with 4096).
  constexpr int kUpWorkgroups = 1536;
  const int each = std::max(1, tiles * lines / kUpWorkgroups);
  const int across = (tiles + each - 1) / each;
  hipLaunchKernelGGL((moe_up_kernel<F16, W8, MT, TINY, CHOOSES>), dim3(static_cast<uint32_t>(across), static_cast<uint32_t>(lines)), dim3(64 * kUpWaves), 0,
                     stream, p, route, by_place);
  return hipGetLastError();
}

template <bool F16, bool W8, int MT, bool TINY = false>
hipError_t launch_experts(const MoeExpertsParams& p, const MoeRouteParams* route, hipStream_t stream) {
  const bool work = has_work(p);
  if (work) {
    hipError_t e;
    if constexpr (MT == 1 && !TINY) e = route != nullptr ? launch_up<F16, W8, MT, TINY, true>(p, *route, stream) : launch_up<F16, W8, MT, TINY, false>(p, MoeRouteParams{}, stream);
    else e = launch_up<F16, W8, MT, TINY, false>(p, MoeRouteParams{}, stream);
    if (e != hipSuccess) return e;
  }
  const void* kernel = reinterpret_cast<const void*>(&moe_down_kernel<F16, W8, MT, TINY>);
  const int lds = kDownWaves * p.tokens * 16 * static_cast<int>(sizeof(float));
  if (lds > 32 * 1024) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kDownWaves * kMoeMostTokens * 16 * 4);
    if (e != hipSuccess) return e;
  }
  const uint32_t columns = static_cast<uint32_t>((p.hidden + 15) / 16);
  hipLaunchKernelGGL((moe_down_kernel<F16, W8, MT, TINY>), dim3(columns, static_cast<uint32_t>(work ? moe_down_shares(p.hidden) : 1)), dim3(64 * kDownWaves), lds,
                     stream, p);
  return hipGetLastError();
}

// Columns of sixteen (in down eight) tokens that a pass over an expert's weights serves, by the tokens an expert has on average
// (known here; how many really name it, and how many ids name none, only the kernels know): more
// take registers from the loads ahead, fewer read the weights again.  Measured with one, two and four (us): 6 (64 tokens, 6 of 64
// of 2048 x 1408, bf16) 217, 220, 245; 8 (128 tokens, 8 of 128 of 2048 x 768) e4m3 169, 179, 248, bf16 251, 244, 270; 10 (40
// tokens, 2 of 8 of 4096 x 4096, bf16) 170, 161, 176; 25 (128 tokens, 2 of 10 of 2048 x 4096, e4m3) 140, 123, 133; 32 (128
// tokens, 2 of 8 of 4096 x 4096, bf16) 356, 241, 224.
template <bool F16, bool W8>
hipError_t launch_experts_for(const MoeExpertsParams& p, const MoeRouteParams* route, hipStream_t stream) {
  const int mean = p.experts > 0 ? p.tokens * p.top / p.experts : 0;
  if (is_tiny(p)) return launch_experts<F16, W8, 1, true>(p, route, stream);
  if (mean <= 8 || p.tokens <= 8) return launch_experts<F16, W8, 1>(p, route, stream);
  if (mean <= 28 || p.tokens <= 32) return launch_experts<F16, W8, 2>(p, route, stream);
  return launch_experts<F16, W8, 4>(p, route, stream);
}

}  // namespace

// A workgroup a compute unit: without shares the few columns of a small hidden axis leave units idle (1001 x 1411, f16, five tokens:
// 62 us with 63 workgroups, 24.6 with 252), and with more than one a unit the sums that meet in memory cost more than they
// bring (37 us with 504; 2048 x 768, 64 tokens: 98 us with 128 workgroups, 63 with 256, 75 with 512).
int moe_down_shares(int hidden) { return std::max(1, std::min(kMoeMostShares, 256 / std::max((hidden + 15) / 16, 1))); }

int moe_route_parts(int hidden) {
  const int steps = (hidden + 31) / 32;
  return std::max(1, (steps + kRouteWaves * kRouteSteps - 1) / (kRouteWaves * kRouteSteps));
}

namespace {

template <bool F16, bool R32>
hipError_t launch_logits(const MoeRouteParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>((p.experts + 15) / 16), static_cast<uint32_t>(p.parts), static_cast<uint32_t>((p.tokens + 15) / 16));
  if (p.hidden < 8) hipLaunchKernelGGL((moe_logits_kernel<F16, R32, true>), grid, dim3(64 * kRouteWaves), 0, stream, p);
  else hipLaunchKernelGGL((moe_logits_kernel<F16, R32, false>), grid, dim3(64 * kRouteWaves), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_for(const MoeExpertsParams& p, const MoeRouteParams* route, hipStream_t stream) {
  if (p.x_f16) return p.w_e4m3 ? launch_experts_for<true, true>(p, route, stream) : launch_experts_for<true, false>(p, route, stream);
  return p.w_e4m3 ? launch_experts_for<false, true>(p, route, stream) : launch_experts_for<false, false>(p, route, stream);
}

}  // namespace

hipError_t launch_moe_experts(const MoeExpertsParams& p, hipStream_t stream) { return launch_for(p, nullptr, stream); }

hipError_t launch_moe_layer(const MoeRouteParams& r, const MoeExpertsParams& p, hipStream_t stream) {
  if (r.top > 0) {
    hipError_t e;
    if (r.router_f32) e = r.x_f16 ? launch_logits<true, true>(r, stream) : launch_logits<false, true>(r, stream);
    else e = r.x_f16 ? launch_logits<true, false>(r, stream) : launch_logits<false, false>(r, stream);
    if (e != hipSuccess) return e;
    // For as many tokens as a workgroup of gate and up has wavefronts the choice is its first work: for one token of 6 of 64
    // experts of 2048 x 1408 a launch of its own makes the layer 41.9 us instead of 40.1.
    if (r.tokens <= kUpWaves && has_work(p) && !is_tiny(p)) return launch_for(p, &r, stream);
    hipLaunchKernelGGL(moe_choose_kernel, dim3(static_cast<uint32_t>(r.tokens)), dim3(64), 0, stream, r);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return launch_for(p, nullptr, stream);
}

}  // namespace vecops_hip
