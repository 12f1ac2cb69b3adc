// The product of microscaled operands: e2m1 or e4m3 activations, e2m1 weights, a power of two for each 32 elements of a row.
#include "mx_block.h"

#include <algorithm>
#include <utility>

#include "lane_exchange.h"
#include "quantized_common.h"

namespace vecops_hip {

namespace {

// ---------------------------------------------------------------------------------------------------------------------
// c[m,n] = sum over blocks of 32 k of 2^(sa[m] - 127) 2^(sb[n] - 127) sum a[m,k] b[n,k].  v_mfma_scale_f32_16x16x128_f8f6f4 does
// all of it: 16 x 16 results over 128 k, a power of two for each row's and column's 32 k, onto an fp32 accumulator.  Weights are
// its rows, activations its columns: lane l holds results n = 4 (l / 16) + 0..3 of activation row l % 16.
// A lane's e2m1 operand is 32 k of one row (16 bytes), lanes 16 q .. 16 q + 15 block q of four, and its scale is that block's.
// An e4m3 operand is 32 bytes: k 16 q .. 16 q + 15 and 64 + 16 q .., so that block b lies in the lanes of 2 b and 2 b + 1 (of
// eight halves), while its scale is still taken from the lanes of quarter b.
// Which block of a row goes into which of the four places is free, as long as both operands and scales agree: a step of 256 k is
// two instructions, and instruction h has block 2 q + h in place q.  A lane then holds the scales of neighbouring blocks.
// e2m1 times e2m1 is exact up to one rounding to fp32 an instruction (measured: 3e-8 of the terms' sizes).  With e4m3 the instruction aligns
// each eight products along k to the largest and drops what is below 2^-13 of it: 1.4e-5 of a result on normally distributed
// operands.  A scale that is NaN makes the result NaN, also over elements of zero.
// ---------------------------------------------------------------------------------------------------------------------

constexpr int kStepBlocks = 8;                  // blocks of 32 k in a step
constexpr uint32_t kNowhere = 0x80000000u;      // an offset past every descriptor's end: zeros arrive

// OPSEL: which byte of the scales' registers counts.
template <bool A8, int OPSEL>
__device__ __forceinline__ f32x4 mfma_mx(const i32x8& w, const i32x8& x, const f32x4& c, uint32_t sw, uint32_t sx) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, A8 ? 0 : 4, OPSEL, static_cast<int>(sw), OPSEL, static_cast<int>(sx));
}

__device__ __forceinline__ i32x8 narrow_fragment(const u32x4& v) {
  return i32x8{static_cast<int>(v[0]), static_cast<int>(v[1]), static_cast<int>(v[2]), static_cast<int>(v[3]), 0, 0, 0, 0};
}

// One buffer load of 4 bytes a lane that writes LDS itself, as load_16_bytes_into_lds: lane l's land at tile_address + tile_offset + 4 l.
__device__ __forceinline__ void load_4_bytes_into_lds(const u32x4& descriptor, uint32_t tile_address, uint32_t tile_offset, uint32_t lane_offset) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dword %2, %3, 0 offen lds"
               :
               : "s"(tile_address), "s"(tile_offset), "v"(lane_offset), "s"(descriptor)
               : "memory", "m0", "scc");
#else
  (void)descriptor; (void)tile_address; (void)tile_offset; (void)lane_offset;
#endif
}

// Matrix results are read by other instructions only behind this: the compiler has been seen to leave too few wait states where a
// branch stands between the two.
template <int N>
__device__ __forceinline__ void settle(f32x4 (&acc)[N]) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 15\n\ts_nop 3" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(acc[i]));
#else
  (void)acc;
#endif
}

// Scales arrive as words of four blocks; a row's last word is its last four bytes, so that no load passes a row's end (rows have at least
// four).  Word `word` of a row of `groups` is fetched from byte scale_word_at() on, and holds its own blocks from bit scale_shift() on (with blocks
// past the row's end as zeros, which stand for 2^-127).
__device__ __forceinline__ int scale_word_at(int word, int groups) { return min(4 * word, groups - 4); }
__device__ __forceinline__ uint32_t scale_shift(int word, int groups) { return static_cast<uint32_t>(min(max(4 * word + 4 - groups, 0) * 8, 31)); }

// Many rows: WN x WM wavefronts, each NT x MT blocks of 16 x 16.  A stage is a step of 256 k of both operands and their scales;
// STAGES of them are under way or in use, by loads that write LDS.
// The rows of a wavefront's weights are dealt to its 16-row blocks so that a lane's results of two blocks are eight
// consecutive n (row r of block 2 p + h is n = 32 p + 8 (r / 4) + 4 h + r % 4): sixteen bytes of a 16-bit result a store.
template <int WN, int WM, int NT, int MT, bool A8, int STAGES>
struct MxTile {
  static constexpr int kBN = WN * NT * 16, kBM = WM * MT * 16, kWaves = WN * WM, kThreads = 64 * kWaves;
  static constexpr int kRowX = A8 ? 256 : 128, kChunksX = kRowX / 16;
  static constexpr int kBytesW = kBN * 128, kBytesX = kBM * kRowX, kScalesW = kBytesW + kBytesX, kScalesX = kScalesW + kBN * 8;
  static constexpr int kLoadsS = (kBN + kBM + 32 * kWaves - 1) / (32 * kWaves);   // (32 rows of scales a load; what the last ones load past the tile's rows is not read)
  static constexpr int kStage = kScalesW + kLoadsS * kWaves * 256, kLds = STAGES * kStage;
  static constexpr int kLoadsW = kBytesW / (kThreads * 16), kLoadsX = kBytesX / (kThreads * 16);
  static constexpr int kLoads = kLoadsW + kLoadsX + kLoadsS;
  static_assert(NT % 2 == 0, "results of two blocks leave together");
  static_assert(kBytesW % (kThreads * 16) == 0 && kBytesX % (kThreads * 16) == 0, "whole loads");
  static_assert(kLds <= 160 * 1024 && STAGES >= 2 && (STAGES - 1) * kLoads < 64, "LDS of a compute unit; the counter of loads");
};

// slot of a chunk in its 128 bytes: rows that a fragment reads together lie in different slots
__device__ __forceinline__ int slot_key_w(int row) { return (row & 3) | ((row >> 1) & 4); }
__device__ __forceinline__ int slot_key_x(int row) { return row & 7; }

template <int WN, int WM, int NT, int MT, bool A8, int STAGES>
__global__ __launch_bounds__(64 * WN * WM, 2) void mx_tile_kernel(const MxMatmulParams p, uint32_t tiles_n, uint32_t tiles_m) {
  using T = MxTile<WN, WM, NT, MT, A8, STAGES>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lds0 = lds_address_of(lds);
  const int batch = blockIdx.y;
  // this workgroup's share of the steps
  const int steps = (p.groups + kStepBlocks - 1) / kStepBlocks;
  const int g_begin = static_cast<int>(static_cast<int64_t>(steps) * blockIdx.z / p.splits);
  const int g_end = static_cast<int>(static_cast<int64_t>(steps) * (blockIdx.z + 1) / p.splits);

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

  // Rows past the operand's last one lie past the descriptors' ends: zeros arrive.
  const uint32_t row_w = static_cast<uint32_t>(p.groups) * 16u, row_x = static_cast<uint32_t>(p.groups) * (A8 ? 32u : 16u);
  u32x4 desc_w = tile_buffer_words((const VECOPS_GLOBAL char*)p.b + batch * p.b_bs + n0 * p.ldb);
  u32x4 desc_x = tile_buffer_words((const VECOPS_GLOBAL char*)p.a + batch * p.a_bs + m0 * p.lda);
  u32x4 desc_sw = tile_buffer_words((const VECOPS_GLOBAL char*)p.b_scales + batch * p.bs_bs + n0 * p.bs_rs);
  u32x4 desc_sx = tile_buffer_words((const VECOPS_GLOBAL char*)p.a_scales + batch * p.as_bs + m0 * p.as_rs);
  const uint32_t end_w = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(last_n * p.ldb) + row_w);
  const uint32_t end_x = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(last_m * p.lda) + row_x);
  const uint32_t end_sw = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(last_n * p.bs_rs + p.row_scales));
  const uint32_t end_sx = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(last_m * p.as_rs + p.row_scales));

  // load i of a thread: sixteen bytes of row i * kRowsW + tid / 8, the chunk whose slot is tid % 8 (rows apart by kRowsW have
  // equal keys); e4m3 rows have sixteen slots
  constexpr int kRowsW = T::kThreads / 8, kRowsX = T::kThreads / T::kChunksX;
  static_assert(kRowsW % 16 == 0 && kRowsX % 8 == 0, "equal keys");
  const int at_row_w = tid / 8, at_row_x = tid / T::kChunksX;
  const uint32_t chunk_w = ((tid & 7) ^ slot_key_w(at_row_w)) << 4, chunk_x = ((tid & (T::kChunksX - 1)) ^ slot_key_x(at_row_x)) << 4;
  const uint32_t from_w = static_cast<uint32_t>(at_row_w * p.ldb) + chunk_w, from_x = static_cast<uint32_t>(at_row_x * p.lda) + chunk_x;
  const uint32_t add_w = static_cast<uint32_t>(kRowsW * p.ldb), add_x = static_cast<uint32_t>(kRowsX * p.lda);
  // the scales: 32 rows an instruction, a lane one of a row's two words; instruction u of the stage goes to wavefront u % waves
  uint32_t from_s[T::kLoadsS];
#pragma unroll
  for (int i = 0; i < T::kLoadsS; ++i) {
    const int u = i * T::kWaves + wave, row = 32 * u + (lane >> 1);
    from_s[i] = u < T::kBN / 32 ? static_cast<uint32_t>(row * p.bs_rs) : static_cast<uint32_t>((row - T::kBN) * p.as_rs);
  }

  // load PIECE of those that fill stage `slot` with step g; past the last step nothing is fetched (but as many loads are issued)
  auto issue_piece = [&](auto piece_tag, int g, int slot) {
    constexpr int PIECE = decltype(piece_tag)::value;
    const uint32_t stage = lds0 + slot * T::kStage;
    const bool there = g < g_end;
    if constexpr (PIECE < T::kLoadsW) {
      const uint32_t k0 = static_cast<uint32_t>(g) * 128u;
      desc_w[2] = there ? end_w : 0u;
      load_16_bytes_into_lds(desc_w, stage, __builtin_amdgcn_readfirstlane(PIECE * (T::kThreads * 16) + wave * 1024),
                             k0 + chunk_w < row_w ? from_w : kNowhere, __builtin_amdgcn_readfirstlane(PIECE * add_w + k0));
    } else if constexpr (PIECE < T::kLoadsW + T::kLoadsX) {
      constexpr int AT = PIECE - T::kLoadsW;
      const uint32_t k0 = static_cast<uint32_t>(g) * T::kRowX;
      desc_x[2] = there ? end_x : 0u;
      load_16_bytes_into_lds(desc_x, stage, __builtin_amdgcn_readfirstlane(T::kBytesW + AT * (T::kThreads * 16) + wave * 1024),
                             k0 + chunk_x < row_x ? from_x : kNowhere, __builtin_amdgcn_readfirstlane(AT * add_x + k0));
    } else {
      constexpr int AT = PIECE - T::kLoadsW - T::kLoadsX;
      const int u = AT * T::kWaves + wave;
      const bool weights = u < T::kBN / 32;
      u32x4 desc = weights ? desc_sw : desc_sx;
      desc[2] = there ? (weights ? end_sw : end_sx) : 0u;
      load_4_bytes_into_lds(desc, stage, __builtin_amdgcn_readfirstlane(T::kScalesW + u * 256), from_s[AT] + scale_word_at(2 * g + (lane & 1), p.row_scales));
    }
  };
  auto issue = [&](int g, int slot) { static_for<T::kLoads>([&](auto piece) { issue_piece(piece, g, slot); }); };

  const int wn = wave / WM, wm = wave % WM;
  const int col = lane & 15, quarter = lane >> 4;
  // a lane's chunks of its row in block 0 (blocks apart by whole rows of equal keys)
  uint32_t at_w[2], at_x[A8 ? 4 : 2];
  {
    const int row = wn * (NT * 16) + 8 * (col >> 2) + (col & 3), row_of_x = wm * (MT * 16) + col;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      at_w[h] = lds0 + row * 128 + (((2 * quarter + h) ^ slot_key_w(row)) << 4);
      if constexpr (A8) {
        const int chunk = 4 * (quarter >> 1) + (quarter & 1) + 2 * h;   // half quarter % 2 of block 2 (quarter / 2) + h; the other: of that plus four blocks
        at_x[2 * h] = lds0 + T::kBytesW + row_of_x * 256 + ((chunk ^ slot_key_x(row_of_x)) << 4);
        at_x[2 * h + 1] = lds0 + T::kBytesW + row_of_x * 256 + (((chunk + 8) ^ slot_key_x(row_of_x)) << 4);
      } else {
        at_x[h] = lds0 + T::kBytesW + row_of_x * 128 + (((2 * quarter + h) ^ slot_key_x(row_of_x)) << 4);
      }
    }
  }
  const uint32_t at_sw = lds0 + T::kScalesW + (wn * (NT * 16) + 8 * (col >> 2) + (col & 3)) * 8 + (quarter >> 1) * 4;
  const uint32_t at_sx = lds0 + T::kScalesX + (wm * (MT * 16) + col) * 8 + (quarter >> 1) * 4;

  f32x4 acc[NT * MT];
#pragma unroll
  for (int i = 0; i < NT * MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (g_begin < g_end) {
#pragma unroll
    for (int g = 0; g < STAGES - 1; ++g) issue(g_begin + g, g);
    int slot = 0;
    for (int g = g_begin; g < g_end; ++g) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * T::kLoads) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      issue(g + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
      const uint32_t stage = slot * T::kStage;
      const uint32_t shift = 16u * (quarter & 1) + scale_shift(2 * g + (quarter >> 1), p.row_scales);
      i32x8 x[MT][2];
      uint32_t sx[MT];
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        sx[j] = read_lds_word(at_sx + stage, j * 128) >> min(shift, 31u);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (A8) x[j][h] = fragment_of(read_lds(at_x[2 * h] + stage, j * 4096), read_lds(at_x[2 * h + 1] + stage, j * 4096));
          else x[j][h] = narrow_fragment(read_lds(at_x[h] + stage, j * 2048));
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        // block 2 p + h starts 32 p + 4 h rows down; 4 rows down the key stays
        const int down = (i >> 1) * 32 + (i & 1) * 4;
        const uint32_t sw = read_lds_word(at_sw + stage, down * 8) >> min(shift, 31u);
        const i32x8 w0 = narrow_fragment(read_lds(at_w[0] + stage, down * 128)), w1 = narrow_fragment(read_lds(at_w[1] + stage, down * 128));
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i * MT + j] = mfma_mx<A8, 0>(w0, x[j][0], acc[i * MT + j], sw, sx[j]);
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i * MT + j] = mfma_mx<A8, 1>(w1, x[j][1], acc[i * MT + j], sw, sx[j]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (this stage may be overwritten behind the next barrier)
      slot = slot + 1 == STAGES ? 0 : slot + 1;
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (no load may write LDS once the workgroup is gone)
  settle(acc);

#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int64_t m = m0 + wm * (MT * 16) + j * 16 + col;
    if (m < p.m) {
#pragma unroll
      for (int i = 0; i < NT; i += 2) {
        const int64_t n = n0 + wn * (NT * 16) + i * 16 + quarter * 8;
        const f32x4 lo = acc[i * MT + j], hi = acc[(i + 1) * MT + j];
        const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
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

// Up to sixteen rows: bound by HBM, so that what counts is how many bytes of the weights are under way.  A workgroup owns sixteen
// weight rows; its wavefronts share the steps of 256 k, a run of neighbouring ones each, with the loads of DEPTH steps of both
// operands and their scales under way, straight into the registers that the matrix instruction reads.  The wavefronts' sums meet in LDS.
template <int WAVES, bool A8>
__global__ __launch_bounds__(64 * WAVES, A8 ? 3 : 4) void mx_few_rows_kernel(const MxMatmulParams p) {
  constexpr int DEPTH = 4, X = A8 ? 4 : 2;
  __shared__ f32x4 sums[WAVES][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quarter = lane >> 4;
  const int batch = blockIdx.y;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int last_n = static_cast<int>(min(p.n - n0, static_cast<int64_t>(16))) - 1;
  const uint32_t row_w = static_cast<uint32_t>(p.groups) * 16u, row_x = static_cast<uint32_t>(p.groups) * (A8 ? 32u : 16u);
  // Rows past the last one lie past the descriptors' ends: zeros arrive.
  const auto operand = [](const uint8_t* base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)uniform_ptr((const VECOPS_GLOBAL char*)base), 0, __builtin_amdgcn_readfirstlane(static_cast<int>(bytes)), 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t desc_w = operand(p.b + batch * p.b_bs + n0 * p.ldb, last_n * p.ldb + row_w);
  const __amdgpu_buffer_rsrc_t desc_x = operand(p.a + batch * p.a_bs, (p.m - 1) * p.lda + row_x);
  const __amdgpu_buffer_rsrc_t desc_sw = operand(p.b_scales + batch * p.bs_bs + n0 * p.bs_rs, last_n * p.bs_rs + p.row_scales);
  const __amdgpu_buffer_rsrc_t desc_sx = operand(p.a_scales + batch * p.as_bs, (p.m - 1) * p.as_rs + p.row_scales);
  // Two neighbouring lanes load thirty-two bytes of one row of weights, once of either's, and exchange them: sixteen bytes of a row
  // each are a look-up in the cache for every lane.
  uint32_t from_w[2], chunk_x[X];
  const uint32_t chunk_w = quarter * 32 + (col & 1) * 16;
#pragma unroll
  for (int h = 0; h < 2; ++h) from_w[h] = static_cast<uint32_t>(((col & 14) + h) * p.ldb) + chunk_w;
#pragma unroll
  for (int c = 0; c < X; ++c) chunk_x[c] = (A8 ? 4 * (quarter >> 1) + (quarter & 1) + 2 * (c >> 1) + 8 * (c & 1) : 2 * quarter + c) * 16;
  const uint32_t from_x = static_cast<uint32_t>(col * p.lda);
  const uint32_t from_sw = static_cast<uint32_t>(col * p.bs_rs), from_sx = static_cast<uint32_t>(col * p.as_rs);

  const int steps = (p.groups + kStepBlocks - 1) / kStepBlocks;
  const int begin = static_cast<int>(static_cast<int64_t>(steps) * wave / WAVES), end = static_cast<int>(static_cast<int64_t>(steps) * (wave + 1) / WAVES);
  u32x4 wv[DEPTH][2], xv[DEPTH][X];
  uint32_t sw[DEPTH], sx[DEPTH];
  auto load = [&](auto slot_tag, int g) {
    constexpr int slot = decltype(slot_tag)::value;
    const uint32_t kw = static_cast<uint32_t>(g) * 128u, kx = static_cast<uint32_t>(g) * (A8 ? 256u : 128u);
#pragma unroll
    for (int h = 0; h < 2; ++h) wv[slot][h] = __builtin_amdgcn_raw_buffer_load_b128(desc_w, kw + chunk_w < row_w ? from_w[h] : kNowhere, kw, 0);
#pragma unroll
    for (int c = 0; c < X; ++c) xv[slot][c] = __builtin_amdgcn_raw_buffer_load_b128(desc_x, kx + chunk_x[c] < row_x ? from_x + chunk_x[c] : kNowhere, kx, 0);
    const int word = scale_word_at(2 * g + (quarter >> 1), p.row_scales);
    sw[slot] = __builtin_amdgcn_raw_buffer_load_b32(desc_sw, from_sw + word, 0, 0);
    sx[slot] = __builtin_amdgcn_raw_buffer_load_b32(desc_sx, from_sx + word, 0, 0);
  };
  f32x4 acc[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
  static_for<DEPTH>([&](auto u) {
    if (begin + decltype(u)::value < end) load(u, begin + decltype(u)::value);
  });
  for (int g0 = begin; g0 < end; g0 += DEPTH) {
    static_for<DEPTH>([&](auto u) {
      constexpr int slot = decltype(u)::value;
      const int g = g0 + slot;
      if (g < end) {
        const uint32_t shift = min(16u * (quarter & 1) + scale_shift(2 * g + (quarter >> 1), p.row_scales), 31u);
        const uint32_t by_w = sw[slot] >> shift, by_x = sx[slot] >> shift;
        exchange_lanes<kNextLane>(wv[slot][0], wv[slot][1], lane & 1);
        i32x8 x[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (A8) x[h] = fragment_of(xv[slot][2 * h], xv[slot][2 * h + 1]);
          else x[h] = narrow_fragment(xv[slot][h]);
        }
        acc[0] = mfma_mx<A8, 0>(narrow_fragment(wv[slot][0]), x[0], acc[0], by_w, by_x);
        acc[0] = mfma_mx<A8, 1>(narrow_fragment(wv[slot][1]), x[1], acc[0], by_w, by_x);
        if (g + DEPTH < end) load(u, g + DEPTH);
      }
    });
  }
  settle(acc);

  sums[wave][lane] = acc[0];
  __syncthreads();
  if (wave == 0) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < WAVES; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += sums[u][lane][r];
    const int64_t n = n0 + quarter * 4;
    if (col < p.m && n < p.n) store_results<4>(p.c, batch * p.c_bs + col * p.c_rs + n * p.c_cs, p.c_cs, p.out_kind, n, p.n, v);
  }
}

template <bool A8>
hipError_t launch_few_rows(const MxMatmulParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>((static_cast<int64_t>(p.n) + 15) / 16), static_cast<uint32_t>(p.batch));
  hipLaunchKernelGGL((mx_few_rows_kernel<4, A8>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <int WN, int WM, int NT, int MT, bool A8, int STAGES>
hipError_t launch_tile(const MxMatmulParams& p, hipStream_t stream) {
  using T = MxTile<WN, WM, NT, MT, A8, STAGES>;
  const void* kernel = reinterpret_cast<const void*>(&mx_tile_kernel<WN, WM, NT, MT, A8, STAGES>);
  if constexpr (T::kLds > 65536) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds);
    if (e != hipSuccess) return e;
  }
  const uint32_t tiles_n = static_cast<uint32_t>((p.n + T::kBN - 1) / T::kBN), tiles_m = static_cast<uint32_t>((p.m + T::kBM - 1) / T::kBM);
  hipLaunchKernelGGL((mx_tile_kernel<WN, WM, NT, MT, A8, STAGES>), dim3(tiles_n * tiles_m, static_cast<uint32_t>(p.batch), static_cast<uint32_t>(p.splits)),
                     dim3(T::kThreads), T::kLds, stream, p, tiles_n, tiles_m);
  if (p.splits > 1) {
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_join_shares({p.partial, p.c, p.c_rs, p.c_cs, p.c_bs, p.m, p.n, p.batch, p.splits, p.out_kind}, stream);
  }
  return hipGetLastError();
}

}  // namespace

MxPlan mx_plan(int64_t m, int64_t n, int64_t k, int64_t batch, bool a_wide) {
  (void)k;
  if (m <= 16) return {MX_FEW_ROWS, 1, 16, 16};
  const int64_t big = ((m + (a_wide ? 127 : 255)) / (a_wide ? 128 : 256)) * ((n + 255) / 256) * batch, middle = ((m + 127) / 128) * ((n + 127) / 128) * batch;
  if (big >= 192) return {MX_TILE_256, 1, a_wide ? 128 : 256, 256};
  if (middle >= 128) return {MX_TILE_128, 1, 128, 128};
  return {MX_TILE_64, 1, 64, 64};
}

hipError_t launch_mx_matmul(const MxMatmulParams& p, int kind, hipStream_t stream) {
  switch (kind) {
    case MX_FEW_ROWS: return p.a_wide ? launch_few_rows<true>(p, stream) : launch_few_rows<false>(p, stream);
    case MX_TILE_64: return p.a_wide ? launch_tile<2, 2, 2, 2, true, 4>(p, stream) : launch_tile<2, 2, 2, 2, false, 4>(p, stream);
    case MX_TILE_128: return p.a_wide ? launch_tile<2, 2, 4, 4, true, 3>(p, stream) : launch_tile<2, 2, 4, 4, false, 4>(p, stream);
    case MX_TILE_256: return p.a_wide ? launch_tile<2, 4, 8, 2, true, 2>(p, stream) : launch_tile<2, 4, 8, 4, false, 2>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace vecops_hip
