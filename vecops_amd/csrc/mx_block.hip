// The product of microscaled operands: e2m1 or e4m3 activations, e2m1 weights, a power of two for each 32 elements of a row.
#include "mx_block.h"

#include <algorithm>
#include <cmath>
#include <utility>

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
// Which block of a row goes into which of the four places is free, as long as both operands and scales agree: blocks are dealt so that a lane's scales of
// several instructions are neighbours, bytes of one word.
// e2m1 times e2m1 is exact up to one rounding to fp32 an instruction (measured: 3e-8 of the terms' sizes).  With e4m3 the instruction aligns
// each eight products along k to the largest and drops what is below 2^-13 of it: 1.4e-5 of a result on normally distributed
// operands, at worst 7 * 2^-13 of the terms' sizes.  Results of 16 bits, whose own rounding is 2^-8 or 2^-11, are left with it.  For results in f32 the activations are taken in two parts by size, an instruction each, whose products
// are exact as e2m1's are: 30 to 70 % more time where many rows share weights (4096 x 11008 x 4096 290 us rather than 177, 128 x 11008 x 4096 21.6 rather than 17.1),
// for a few rows 1 us of 7 (M up to 4) or less.  A scale that is NaN makes the result NaN, also over elements of zero.
// ---------------------------------------------------------------------------------------------------------------------

constexpr uint32_t kNowhere = 0x80000000u;      // an offset past every descriptor's end: zeros arrive

// OPSEL: which byte of the scales' registers counts.
template <bool A8, int OPSEL>
__device__ __forceinline__ f32x4 mfma_mx(const i32x8& w, const i32x8& x, const f32x4& c, uint32_t sw, uint32_t sx) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, A8 ? 0 : 4, OPSEL, static_cast<int>(sw), OPSEL, static_cast<int>(sx));
}

// The same of 32 x 32 results over 64 k.
template <bool A8, int OPSEL>
__device__ __forceinline__ f32x16 mfma_mx_32(const i32x8& w, const i32x8& x, const f32x16& c, uint32_t sw, uint32_t sx) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, c, 4, A8 ? 0 : 4, OPSEL, static_cast<int>(sw), OPSEL, static_cast<int>(sx));
}

__device__ __forceinline__ i32x8 narrow_fragment(const u32x4& v) {
  return i32x8{static_cast<int>(v[0]), static_cast<int>(v[1]), static_cast<int>(v[2]), static_cast<int>(v[3]), 0, 0, 0, 0};
}

// e4m3 elements of 2 and more (bit 6 of a byte; NaN has it too) with zeros for the others, and the others.  A product with e2m1 is a multiple of 2^-4 of its
// element's power of two, and a part has at most eight of these powers: none of eight products has a bit that is dropped beside the largest.
__device__ __forceinline__ void part_by_size(const i32x8& x, i32x8& high, i32x8& low) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t v = static_cast<uint32_t>(x[i]), there = (v >> 6) & 0x01010101u, mask = (there << 8) - there;
    high[i] = static_cast<int>(v & mask);
    low[i] = static_cast<int>(v & ~mask);
  }
}

// Matrix results are read by other instructions only behind this: the compiler has been seen to leave too few wait states where a
// branch stands between the two.
__device__ __forceinline__ void settle() {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
#endif
}

// Scales arrive sixteen of a row a load, a row's last sixteen by one that ends with the row.  Rows of fewer (K of up to 480): a lane reads those that there are,
// byte by byte, and writes them to LDS itself, with zeros behind, where a load has left zeros (1 x 640 x 256 4.9 us a call, 109 x 3200 x 256 6.5; with rows laid out in the workspace first 6.4 and 8.7.  It costs 64 x 64
// tiles of longer rows 0.15 us of 7.6).  MX_TILE_256, whose workgroups go on to other tiles, has them laid out.
__device__ __forceinline__ u32x4 few_scales(const uint8_t* base, int64_t at, int groups, bool there) {
  u32x4 v = {0u, 0u, 0u, 0u};
  const VECOPS_GLOBAL uint8_t* from = (const VECOPS_GLOBAL uint8_t*)base + at;
#pragma unroll
  for (int e = 0; e < 15; ++e)
    if (there && e < groups) v[e >> 2] |= static_cast<uint32_t>(from[e]) << (8 * (e & 3));
  return v;
}

// Many rows: WN x WM wavefronts, each NT x MT blocks of 32 x 32.  v_mfma_scale_f32_32x32x64_f8f6f4: a lane's e2m1 operand is the
// place l / 32 of two of row l % 32, an e4m3 one half l / 32 of either place; its scale is that of place l / 32.  Of a stage's eight blocks of
// 32 k instruction s of four has block 4 q + s in place q: a lane's four scales are one word, the instruction's byte of it a constant.  (One wavefront
// on a SIMD keeps the matrix pipe to 8.5 PFLOP/s with it, on operands of zeros, and with the 16 x 16 one to 4.9: an instruction with scales
// takes two issues.)
// A stage is 256 k of both operands: whole lines of e2m1 rows (of half lines each is fetched twice).  STAGES of them are under way or
// in use, by loads that write LDS.  Scales come two stages a run, sixteen bytes of a row a load: each is a request of its own to
// the cache, which a word a row for each 128 k had by the half of all requests.  A row's last run is its last sixteen scales; what of it
// has been summed before gets zeros for elements.
// 4096 x 11008 x 4096 on weights that no cache holds: e2m1 102 us (3.6 PFLOP/s; the matrix pipes busy 54 % of the cycles of a clock that they pull down to
// 1.65 GHz, 38 GB/s of loads a compute unit, and 8 us a tile in which all of them write), e4m3 167 us (2.2 PFLOP/s).
// 128 weight rows by 64, two wavefronts sharing k: a third less to load a result than 64 x 64; on such weights 128 x 11008 x 4096 with e4m3 16.4 us rather than 20.4,
// 512 x 4096 x 11008 35.4 rather than 44, 1024 x 2048 x 8192 25.7 rather than 31.6 (e2m1 22.4 and 23.5).
// The rows of a block of weights are dealt so that a lane's sixteen results are neighbouring n (the instruction's row
// 8 g + 4 h + e, which lane half h holds, is n = 16 h + 4 g + e).
constexpr int kRunBlocks = 16;
constexpr int min_of(int a, int b) { return a < b ? a : b; }
template <int WN, int WM, int WK, int NT, int MT, bool A8, int STAGES, bool GOES_ON>
struct MxTile {
  static constexpr int kBN = WN * NT * 32, kBM = WM * MT * 32, kWaves = WN * WM * WK, kThreads = 64 * kWaves;
  static constexpr int kRowX = A8 ? 256 : 128, kChunksX = kRowX / 16;
  static constexpr int kBytesW = kBN * 128, kBytesX = kBM * kRowX, kStage = kBytesW + kBytesX;
  static constexpr int kLoadsW = kBytesW / (kThreads * 16), kLoadsX = kBytesX / (kThreads * 16), kLoadsS = (kBN + kBM + 64 * kWaves - 1) / (64 * kWaves);
  static constexpr int kRuns = STAGES > 3 ? 4 : 2, kRun = kLoadsS * kWaves * 1024;   // (what the last loads of scales bring past the tile's rows is not read)
  // Results leave by way of 4 KiB a wavefront: of their own where the next tile's stages are under way meanwhile
  static constexpr int kScales = STAGES * kStage, kResults = GOES_ON ? kScales + kRuns * kRun : 0;
  static constexpr int kLds = kScales + kRuns * kRun + (GOES_ON ? kWaves * 4096 : 0);
  static constexpr int loads(int stage) { return kLoadsW + kLoadsX + (stage % 2 == 0 ? kLoadsS : 0); }   // a run's scales come with its first stage
  // loads of the stages from..to - 1 (of which only whether they are even matters)
  static constexpr int loads_between(int from, int to) { return from >= to ? 0 : loads(from) + loads_between(from + 1, to); }
  // kEarly: of a buffer that is multiplied, only the second pair of block rows is still to be read soon after the stage has begun.  The rest of it -
  // activations, the first pair's weights (a load is 32 rows, a block row), scales - is refilled from there on, kFirst loads of it beside the
  // first pair.
  static constexpr bool kEarly = STAGES == 2 && NT == 4 && kThreads == 256;
  static constexpr int kFirst = kEarly ? 11 : 0;
  // nth load of a stage
  static constexpr int piece(int nth, int stage) {
    return !kEarly ? nth : nth < kLoadsW / 2 ? nth / 2 * 4 + nth % 2 : nth < loads(stage) - kLoadsW / 2 ? nth + kLoadsW / 2 : late(nth - loads(stage) + kLoadsW / 2);
  }
  static constexpr int late(int nth) { return nth / 2 * 4 + 2 + nth % 2; }
  static_assert(NT % 2 == 0 && kBN % 64 == 0 && kBM % 64 == 0 && kBytesW % (kThreads * 16) == 0 && kBytesX % (kThreads * 16) == 0, "pairs of block rows; whole loads");
  static_assert(kThreads / 8 % 16 == 0 && kThreads / kChunksX % 8 == 0, "a thread's rows have equal keys, or two in turn");
  static_assert(kLds <= 160 * 1024 && STAGES >= 2 && STAGES <= 6 && loads_between(1, STAGES) < 63, "LDS of a compute unit; places for runs; the counter of loads");
};

// Slot of a chunk among a row's.  LDS serves sixteen-byte reads of lanes 0-3, 12-15, 20-27 together, then of 4-11, 16-19, 28-31, and so on: rows
// of either set (in both orders in which lanes have them) lie in different sixteen bytes of 256.
template <int BYTES>
__device__ __forceinline__ int slot_key(int row) { return BYTES == 128 ? (row >> 1) & 7 : row & 15; }

// Sixteen bytes of a row's results (`row`: the row's place in elements) from column n on; those from n_end on stay unwritten.
template <int KIND>
__device__ __forceinline__ void store_sixteen(char* c, int64_t row, int64_t cs, int64_t n, int64_t n_end, const u32x4& v) {
  constexpr int BYTES = KIND == FP8_REAL_F32 ? 4 : 2, COUNT = 16 / BYTES;
  VECOPS_GLOBAL char* const to = (VECOPS_GLOBAL char*)c + (row + n * cs) * BYTES;
  if (cs == 1 && n + COUNT <= n_end) {
    *(VECOPS_GLOBAL u32x4_anywhere*)to = v;
  } else {
#pragma unroll
    for (int e = 0; e < COUNT; ++e) {
      if (n + e >= n_end) continue;
      if constexpr (BYTES == 4) *(VECOPS_GLOBAL uint32_t*)(to + e * cs * 4) = v[e];
      else *(VECOPS_GLOBAL uint16_t*)(to + e * cs * 2) = static_cast<uint16_t>(v[e >> 1] >> (16 * (e & 1)));
    }
  }
}

// One wavefront: two block rows at a time against every block column of the activations, whose fragments stay in registers for the
// stage.  While a pair's products are formed the next one's weights are fetched, and beside the last pair the next stage's
// activations, each into the registers that its last product has read.  So in front of the last pair all of the stage has been read: there the next stage
// has landed, the wavefronts meet, and behind that this stage's buffer is refilled, a load behind each matrix instruction.
// GOES_ON: a workgroup goes from tile to tile, and the next one's first stages are fetched while it writes results: with a workgroup a
// compute unit nothing else would.
// OUT: the type in which results leave (a template's argument: with a branch the compiler makes copies of all of the way out and reads every
// accumulator in front of them).
template <int WN, int WM, int WK, int NT, int MT, bool A8, int STAGES, int WAVES_A_SIMD, bool GOES_ON, int OUT, bool PARTS>
__global__ __launch_bounds__(64 * WN * WM * WK, WAVES_A_SIMD) void mx_tile_kernel(const MxMatmulParams p, uint32_t tiles_n, uint32_t tiles_m) {
  using T = MxTile<WN, WM, WK, NT, MT, A8, STAGES, GOES_ON>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lds0 = lds_address_of(lds);
  const int batch = blockIdx.y;
  // this workgroup's share of the runs
  const int runs = (p.groups + kRunBlocks - 1) / kRunBlocks;
  const int run_begin = static_cast<int>(static_cast<int64_t>(runs) * blockIdx.z / p.splits);
  const int run_end = static_cast<int>(static_cast<int64_t>(runs) * (blockIdx.z + 1) / p.splits);

  // Neighbouring tiles on one die: each die's units (every eighth) are a contiguous run of tiles, walked in groups of eight tile rows.
  const uint32_t units = tiles_n * tiles_m;
  struct Tile {
    int64_t m0, n0;
    int last_m, last_n;
  };
  auto tile_of = [&](uint32_t unit) {
    const uint32_t xcd = unit & 7, share = units >> 3, extra = units & 7;
    const uint32_t pid = xcd * share + min(xcd, extra) + (unit >> 3);
    const uint32_t per_group = 8 * tiles_n, group = pid / per_group, first = group * 8;
    const uint32_t height = min(tiles_m - first, 8u), in_group = pid - group * per_group;
    Tile t;
    t.m0 = static_cast<int64_t>(first + in_group % height) * T::kBM, t.n0 = static_cast<int64_t>(in_group / height) * T::kBN;
    t.last_m = static_cast<int>(min(p.m - t.m0, static_cast<int64_t>(T::kBM))) - 1;
    t.last_n = static_cast<int>(min(p.n - t.n0, static_cast<int64_t>(T::kBN))) - 1;
    return t;
  };

  // load i of a thread: sixteen bytes of row i * kRowsW + tid / chunks, the chunk whose slot is tid % chunks
  constexpr int kRowsW = T::kThreads / 8, kRowsX = T::kThreads / T::kChunksX;
  const int at_row_w = tid / 8, at_row_x = tid / T::kChunksX;
  const int chunk_w = (tid & 7) ^ slot_key<128>(at_row_w), chunk_x = (tid & (T::kChunksX - 1)) ^ slot_key<T::kRowX>(at_row_x);
  constexpr int kTurn = kRowsX % 16 == 0 ? 0 : 8;   // (rows sixteen apart have equal keys; eight apart, those of 256 bytes, keys that differ by eight)
  const uint32_t from_w = static_cast<uint32_t>(at_row_w * p.ldb) + chunk_w * 16, from_x = static_cast<uint32_t>(at_row_x * p.lda) + chunk_x * 16;
  const uint32_t from_x_odd = static_cast<uint32_t>(at_row_x * p.lda) + (chunk_x ^ kTurn) * 16;
  const uint32_t add_w = static_cast<uint32_t>(kRowsW * p.ldb), add_x = static_cast<uint32_t>(kRowsX * p.lda);
  const int block_x = A8 ? chunk_x >> 1 : chunk_x, block_x_odd = A8 ? (chunk_x ^ kTurn) >> 1 : chunk_x;   // of the stage's eight
  // the scales: 64 rows an instruction; instruction u goes to wavefront u % waves
  uint32_t from_s[T::kLoadsS];
#pragma unroll
  for (int i = 0; i < T::kLoadsS; ++i) {
    const int rows = 64 * (i * T::kWaves + wave);
    from_s[i] = static_cast<uint32_t>(rows < T::kBN ? (rows + lane) * p.bs_rs : (rows - T::kBN + lane) * p.as_rs);
  }

  // What is fetched: a unit's tile, a run of it, and which run that is of the workgroup's.  Rows past the operand's last one lie past the
  // descriptors' ends: zeros arrive.
  uint32_t fetch_unit = blockIdx.x, end_w = 0, end_x = 0, end_s[T::kLoadsS], fetch_turn = 0;
  int fetch_run = run_begin;
  u32x4 desc_w, desc_x, desc_s[T::kLoadsS];
  const bool few = !GOES_ON && p.row_scales < kRunBlocks;
  const int last_first = few ? 0 : p.row_scales - kRunBlocks;
  auto aim = [&] {
    const bool there = fetch_unit < units && run_begin < run_end;   // (past the last tile nothing is fetched, but as many loads are issued)
    const Tile t = tile_of(there ? fetch_unit : 0);
    desc_w = tile_buffer_words((const VECOPS_GLOBAL char*)p.b + batch * p.b_bs + t.n0 * p.ldb);
    desc_x = tile_buffer_words((const VECOPS_GLOBAL char*)p.a + batch * p.a_bs + t.m0 * p.lda);
    end_w = __builtin_amdgcn_readfirstlane(there ? static_cast<uint32_t>(t.last_n * p.ldb) + static_cast<uint32_t>(p.groups) * 16u : 0u);
    end_x = __builtin_amdgcn_readfirstlane(there ? static_cast<uint32_t>(t.last_m * p.lda) + static_cast<uint32_t>(p.groups) * (A8 ? 32u : 16u) : 0u);
    desc_w[2] = end_w;
    desc_x[2] = end_x;
#pragma unroll
    for (int i = 0; i < T::kLoadsS; ++i) {
      const bool weights = 64 * (i * T::kWaves + wave) < T::kBN;
      desc_s[i] = tile_buffer_words(weights ? (const VECOPS_GLOBAL char*)p.b_scales + batch * p.bs_bs + t.n0 * p.bs_rs
                                            : (const VECOPS_GLOBAL char*)p.a_scales + batch * p.as_bs + t.m0 * p.as_rs);
      end_s[i] = __builtin_amdgcn_readfirstlane(there && !few ? static_cast<uint32_t>((weights ? t.last_n * p.bs_rs : t.last_m * p.as_rs) + p.row_scales) : 0u);
      desc_s[i][2] = end_s[i];
    }
  };
  auto advance = [&] {   // to the next run
    ++fetch_turn;
    if (++fetch_run < run_end) return;
    fetch_run = run_begin;
    fetch_unit = GOES_ON ? fetch_unit + gridDim.x : units;
    aim();
  };

  // load PIECE of those that fill buffer `slot` with half PAR of the run that is fetched
  auto issue_piece = [&](auto piece_tag, auto par_tag, int slot) {
    constexpr int PIECE = decltype(piece_tag)::value, PAR = decltype(par_tag)::value;
    const int first_block = min(fetch_run * kRunBlocks, last_first);   // the run's sixteen blocks
    // those before `old` have been summed; those from `most` on are not there
    const int old = fetch_run * kRunBlocks - first_block - 8 * PAR, most = p.groups - first_block - 8 * PAR;
    if constexpr (PIECE < T::kLoadsW) {
      load_16_bytes_into_lds(desc_w, lds0 + slot * T::kStage, __builtin_amdgcn_readfirstlane(PIECE * (T::kThreads * 16) + wave * 1024),
                             chunk_w >= old && chunk_w < most ? from_w : kNowhere,
                             __builtin_amdgcn_readfirstlane(PIECE * add_w + static_cast<uint32_t>(first_block + 8 * PAR) * 16u));
    } else if constexpr (PIECE < T::kLoadsW + T::kLoadsX) {
      constexpr int AT = PIECE - T::kLoadsW;
      const int block = AT % 2 ? block_x_odd : block_x;
      load_16_bytes_into_lds(desc_x, lds0 + slot * T::kStage, __builtin_amdgcn_readfirstlane(T::kBytesW + AT * (T::kThreads * 16) + wave * 1024),
                             block >= old && block < most ? (AT % 2 ? from_x_odd : from_x) : kNowhere,
                             __builtin_amdgcn_readfirstlane(AT * add_x + static_cast<uint32_t>(first_block + 8 * PAR) * (A8 ? 32u : 16u)));
    } else {
      constexpr int AT = PIECE - T::kLoadsW - T::kLoadsX;
      load_16_bytes_into_lds(desc_s[AT], lds0 + T::kScales + (fetch_turn & (T::kRuns - 1)) * T::kRun, __builtin_amdgcn_readfirstlane((AT * T::kWaves + wave) * 1024),
                             from_s[AT], __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(first_block)));
    }
  };

  const int wn = wave / (WM * WK), wm = wave / WK % WM, wk = wave % WK;
  const int col = lane & 31, half = lane >> 5;
  // a lane's chunks of its row in block 0 (blocks apart by whole rows of equal keys)
  const int row_of_w = wn * (NT * 32) + 16 * ((col >> 2) & 1) + 4 * (col >> 3) + (col & 3), row_of_x = wm * (MT * 32) + col;
  constexpr int kSets = 4 / WK;   // of 64 k, of a stage's four, that a wavefront multiplies
  uint32_t at_w[kSets], at_x[kSets][A8 ? 2 : 1];
#pragma unroll
  for (int s = 0; s < kSets; ++s) {
    at_w[s] = lds0 + row_of_w * 128 + (((4 * half + wk * kSets + s) ^ slot_key<128>(row_of_w)) << 4);
#pragma unroll
    for (int h = 0; h < (A8 ? 2 : 1); ++h)
      at_x[s][h] = lds0 + T::kBytesW + row_of_x * T::kRowX + (((A8 ? 8 * h + 2 * (wk * kSets + s) + half : 4 * half + wk * kSets + s) ^ slot_key<T::kRowX>(row_of_x)) << 4);
  }
  const uint32_t at_sw = lds0 + T::kScales + row_of_w * 16 + half * 4 + wk * kSets, at_sx = lds0 + T::kScales + (T::kBN + row_of_x) * 16 + half * 4 + wk * kSets;

  f32x16 acc[NT * MT];
  i32x8 x[kSets][MT], w[2][2][kSets];
  uint32_t sx[2][MT], sw[2][2];   // byte s: of set s
  constexpr int kPairs = NT / 2, kMeet = 5;
  // a stage's scales of one row
  auto scales_at = [&](uint32_t at, int offset) { return WK == 2 ? read_lds_short(at, offset) : read_lds_word(at, offset); };
  auto read_w = [&](auto to_tag, auto i_tag, auto s_tag, uint32_t stage) {
    constexpr int to = decltype(to_tag)::value, i = decltype(i_tag)::value, s = decltype(s_tag)::value;
    w[to][i & 1][s] = narrow_fragment(read_lds(at_w[s] + stage, i * 4096));
  };
  auto read_x = [&](auto s_tag, auto j_tag, uint32_t stage) {
    constexpr int s = decltype(s_tag)::value, j = decltype(j_tag)::value;
    if constexpr (A8) x[s][j] = fragment_of(read_lds(at_x[s][0] + stage, j * 8192), read_lds(at_x[s][1] + stage, j * 8192));
    else x[s][j] = narrow_fragment(read_lds(at_x[s][0] + stage, j * 4096));
  };

  // half PAR of the workgroup's run `turn`, in buffer `slot`
  auto multiply = [&](auto par_tag, uint32_t turn, int slot) {
    constexpr int PAR = decltype(par_tag)::value;
    constexpr int AHEAD = PAR + STAGES;   // the stage, counted from the run's first, that takes this one's buffer
    const int next_slot = slot + 1 == STAGES ? 0 : slot + 1;
    const uint32_t stage = slot * T::kStage, next = next_slot * T::kStage;
    const uint32_t run_at = (turn & (T::kRuns - 1)) * T::kRun, next_run_at = PAR == 0 ? run_at : ((turn + 1) & (T::kRuns - 1)) * T::kRun;
    if constexpr (AHEAD % 2 == 0) advance();
    static_for<kPairs>([&](auto pair_tag) {
      constexpr int pair = decltype(pair_tag)::value, now = (PAR * kPairs + pair) & 1, then = now ^ 1;
      constexpr bool final_pair = pair + 1 == kPairs;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (final_pair) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(T::kEarly ? T::kFirst : T::loads_between(PAR + 2, PAR + STAGES)) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      // behind matrix instruction AT of the pair: the next pair's weights and scales, the next stage's activations, loads
      auto beside = [&](auto at_tag) {
        constexpr int AT = decltype(at_tag)::value, kAll = 2 * kSets * MT, kParts = 2 * kSets;
        // of the pair's fragments (beside the first of several pairs not before the wavefronts have met; all some time before they are waited for)
        constexpr int start = T::kEarly && !final_pair ? kMeet : 0, step = kAll >= 32 ? 2 : 1, many = (kParts * step + kAll - 1) / kAll;
        constexpr int from = AT < start ? 0 : min_of((AT - start + step - 1) / step * many, kParts), to = AT < start ? 0 : min_of((AT - start + step) / step * many, kParts);
        static_for<to - from>([&](auto nth) {
          constexpr int f = from + decltype(nth)::value;
          constexpr int i = final_pair ? f & 1 : 2 * pair + 2 + (f & 1);
          read_w(std::integral_constant<int, then>{}, std::integral_constant<int, i>{}, std::integral_constant<int, (f >> 1)>{}, final_pair ? next : stage);
          if constexpr (f < 2)
            sw[then][f] = scales_at(at_sw + (final_pair ? next_run_at : run_at), i * 512 + 8 * (final_pair ? 1 - PAR : PAR));
        });
        if constexpr (final_pair) {
          if constexpr (AT < MT) sx[1 - PAR][AT] = scales_at(at_sx + next_run_at, AT * 512 + 8 * (1 - PAR));
          if constexpr (AT % 2 == 1) read_x(std::integral_constant<int, AT / 2 / MT>{}, std::integral_constant<int, AT / 2 % MT>{}, next);
        }
        if constexpr (T::kEarly && !final_pair && AT == kMeet) {   // every wavefront has read what is refilled from here on
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        // loads evenly
        constexpr int all = T::loads(AHEAD), first = final_pair ? T::kFirst : 0, count = final_pair ? all - T::kFirst : T::kFirst, room = kAll - start;
        constexpr int a = AT < start ? 0 : (AT - start) * count / room, b = AT < start ? 0 : (AT - start + 1) * count / room;
        static_for<b - a>([&](auto nth) {
          issue_piece(std::integral_constant<int, T::piece(first + a + decltype(nth)::value, AHEAD)>{}, std::integral_constant<int, AHEAD % 2>{}, slot);
        });
      };
      static_for<kSets>([&](auto s_tag) {
        static_for<MT>([&](auto j_tag) {
          i32x8 high, low;
          if constexpr (PARTS) {
            constexpr int s = decltype(s_tag)::value, j = decltype(j_tag)::value, at = 2 * pair * MT + j;
            part_by_size(x[s][j], high, low);
            acc[at] = mfma_mx_32<A8, s>(w[now][0][s], low, acc[at], sw[now][0], sx[PAR][j]);
            acc[at + MT] = mfma_mx_32<A8, s>(w[now][1][s], low, acc[at + MT], sw[now][1], sx[PAR][j]);
          }
          static_for<2>([&](auto i_tag) {
            constexpr int s = decltype(s_tag)::value, j = decltype(j_tag)::value, i = decltype(i_tag)::value, at = (2 * pair + i) * MT + j;
            acc[at] = mfma_mx_32<A8, s>(w[now][i][s], PARTS ? high : x[s][j], acc[at], sw[now][i], sx[PAR][j]);
            __builtin_amdgcn_sched_barrier(0);
            beside(std::integral_constant<int, (s * MT + j) * 2 + i>{});
            __builtin_amdgcn_sched_barrier(0);
          });
        });
      });
    });
  };

  aim();
  static_for<STAGES>([&](auto g) {
    constexpr int G = decltype(g)::value;
    if constexpr (G > 0 && G % 2 == 0) advance();
    static_for<T::loads(G)>([&](auto piece) { issue_piece(piece, std::integral_constant<int, G % 2>{}, G); });
  });
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(T::loads_between(1, STAGES)) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (__builtin_expect(few, 0)) {
    const Tile t = tile_of(blockIdx.x);
    for (int row = tid; row < T::kBN + T::kBM; row += T::kThreads) {
      const bool weights = row < T::kBN;
      const int64_t n = t.n0 + row, m = t.m0 + row - T::kBN;
      write_lds(lds0 + T::kScales + row * 16, weights ? few_scales(p.b_scales, batch * p.bs_bs + n * p.bs_rs, p.groups, n < p.n)
                                                      : few_scales(p.a_scales, batch * p.as_bs + m * p.as_rs, p.groups, m < p.m));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
  static_for<2 * kSets>([&](auto f) {
    constexpr int F = decltype(f)::value;
    read_w(std::integral_constant<int, 0>{}, std::integral_constant<int, (F & 1)>{}, std::integral_constant<int, (F >> 1)>{}, 0);
    if constexpr (F < 2) sw[0][F] = scales_at(at_sw, F * 512);
  });
  static_for<MT>([&](auto j) {
    sx[0][decltype(j)::value] = scales_at(at_sx, decltype(j)::value * 512);
    static_for<kSets>([&](auto s) { read_x(s, j, 0); });
  });
  const bool shares = p.splits > 1;
  const int64_t c_rs = shares ? p.n : p.c_rs, c_cs = shares ? 1 : p.c_cs;
  char* const c = shares ? reinterpret_cast<char*>(p.partial + (static_cast<int64_t>(blockIdx.z) * p.batch + batch) * p.m * p.n)
                         : static_cast<char*>(p.c) + batch * p.c_bs * (OUT == FP8_REAL_F32 ? 4 : 2);
  const uint32_t mine = lds0 + T::kResults + wave / WK * 4096;
  int slot = 0;
  uint32_t turn = 0;
  const auto following = [](int at) { return at + 1 == STAGES ? 0 : at + 1; };
  // (behind the last tile's last stage: reads of a buffer that nothing has been fetched for, and loads that fetch nothing)
#pragma unroll 1
  for (uint32_t unit = blockIdx.x; unit < units; unit = GOES_ON ? unit + gridDim.x : units) {
#pragma unroll
    for (int i = 0; i < NT * MT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
#pragma unroll 1
    for (int run = run_begin; run < run_end; ++run) {
      multiply(std::integral_constant<int, 0>{}, turn, slot);
      slot = following(slot);
      multiply(std::integral_constant<int, 1>{}, turn, slot);
      slot = following(slot);
      ++turn;
    }
    settle();
    if constexpr (!GOES_ON) {   // (no load may write LDS once results pass through it; other wavefronts are done with what they replace)
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
    if constexpr (WK == 2) {   // the second wavefront's sums onto the first one's, which writes them
      static_assert(!GOES_ON && T::kWaves / 2 * NT * MT * 4096 <= T::kStage * STAGES, "room for them");
      const uint32_t meet = lds0 + wave / 2 * (NT * MT * 4096) + lane * 16;
      if (wk == 1) {
        static_for<NT * MT>([&](auto i) {
          constexpr int I = decltype(i)::value;
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            write_lds(meet + I * 4096 + e * 256, u32x4{__float_as_uint(acc[I][e]), __float_as_uint(acc[I][e + 1]), __float_as_uint(acc[I][e + 2]), __float_as_uint(acc[I][e + 3])});
        });
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (wk == 0) {
        static_for<NT * MT>([&](auto i) {
          constexpr int I = decltype(i)::value;
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const u32x4 v = read_lds(meet + I * 4096, e * 256);
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[I][e + d] += __uint_as_float(v[d]);
          }
        });
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (wk == 1) return;
    }
    // 32 rows of 128 bytes at a time pass through LDS, so that a store instruction fills lines: sixteen bytes of a row lie in slot
    // (place ^ row / 2 % 8) of eight.
    const Tile t = tile_of(unit);
    const auto write_row = [&](int place, const u32x4& v) { write_lds(mine + col * 128 + ((place ^ ((col >> 1) & 7)) << 4), v); };
    const auto read_row = [&](int row, int place) { return read_lds(mine + row * 128 + ((place ^ ((row >> 1) & 7)) << 4), 0); };
    static_for<MT>([&](auto j_tag) {
      static_for<NT / 2>([&](auto pair_tag) {
        constexpr int j = decltype(j_tag)::value, i = 2 * decltype(pair_tag)::value;
        const int64_t m = t.m0 + wm * (MT * 32) + j * 32 + (lane >> 3), n = t.n0 + wn * (NT * 32) + i * 32;
        if constexpr (OUT == FP8_REAL_F32) {
          static_for<2>([&](auto u_tag) {
            constexpr int u = decltype(u_tag)::value;
            const f32x16 a = acc[(i + u) * MT + j];
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              write_row(e / 4 + half * 4, u32x4{__float_as_uint(a[e]), __float_as_uint(a[e + 1]), __float_as_uint(a[e + 2]), __float_as_uint(a[e + 3])});
#pragma unroll
            for (int r = 0; r < 32; r += 8)
              store_sixteen<FP8_REAL_F32>(c, (m + r) * c_rs, c_cs, n + u * 32 + (lane & 7) * 4, m + r < p.m ? p.n : 0, read_row(r + (lane >> 3), lane & 7));
          });
        } else {
          static_for<2>([&](auto u_tag) {
            constexpr int u = decltype(u_tag)::value;
            const f32x16 a = acc[(i + u) * MT + j];
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
              u32x4 v;
#pragma unroll
              for (int d = 0; d < 4; ++d)
                v[d] = OUT == FP8_REAL_BF16 ? cvt_pk_bf16(a[e + 2 * d], a[e + 2 * d + 1])
                                            : f16_bits_rne(a[e + 2 * d]) | static_cast<uint32_t>(f16_bits_rne(a[e + 2 * d + 1])) << 16;
              write_row(u * 4 + half * 2 + e / 8, v);
            }
          });
#pragma unroll
          for (int r = 0; r < 32; r += 8)
            store_sixteen<FP8_REAL_BF16>(c, (m + r) * c_rs, c_cs, n + (lane & 7) * 8, m + r < p.m ? p.n : 0, read_row(r + (lane >> 3), lane & 7));
        }
        __builtin_amdgcn_sched_barrier(0);   // (two blocks at a time leave the accumulators)
      });
    });
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (no load may write LDS once the workgroup is gone)
}

// Few rows, or few results: R weight rows (16 or 32) and XR activation rows a workgroup, whose wavefronts share k without a barrier: each
// has its own runs of 512 k, every WAVES-th, and its own DEPTH places for them in LDS, filled by loads that write LDS (whole lines, so that a load is
// a look-up in the cache for every eight lanes or more).  Bound by HBM, or by what a compute unit can have under way: about 40 GB/s as soon as some of its
// lines come from beyond its die's cache.  On weights that no cache holds: 1 x 14336 x 4096 8.3 us and 1 x 28672 x 4096 13.8 (3.8 and 4.5 TB/s), 16 x 14336 x
// 4096 10.5, 64 x 4096 x 4096 7.1 (as 64 x 64 tiles 10.4), with e4m3 16 x 4096 x 14336 11.3 (fragments fetched into registers, four wavefronts: 16.3) and
// 32 x 4096 x 14336 17.9 (64 x 64 tiles 29.5).  Two wavefronts of four rows where workgroups are many (1 x 28672 x 4096 13.8 us, with four 14.2, with two
// places each 16), four with two places where they are few (1 x 4096 x 14336 8.2, 10.0 with one place, 14.1 with two wavefronts).
// R = 16: v_mfma_scale_f32_16x16x128_f8f6f4, place q of instruction t of a run has block 4 q + t of sixteen; R = 32: 32x32x64, place q of
// instruction t has block 8 q + t.  Either way a lane's scales are whole words whose byte is a constant of the instruction.
template <int R, int XR, bool A8, int WAVES, int DEPTH>
struct MxSlim {
  static constexpr int kRowX = A8 ? 512 : 256, kChunksX = kRowX / 16;
  static constexpr int kBytesW = R * 256, kBytesX = XR * kRowX, kScales = kBytesW + kBytesX, kPlace = kScales + 2048;
  static constexpr int kLoadsW = kBytesW / 1024, kLoadsX = kBytesX / 1024, kLoads = kLoadsW + kLoadsX + 2;
  static constexpr int kColumns = XR < R ? 1 : XR / R;                       // blocks of R activation rows
  static constexpr int kSum = kColumns * R * R * 4;                         // bytes of a wavefront's sums
  static constexpr int kLds = WAVES * DEPTH * kPlace > WAVES * kSum ? WAVES * DEPTH * kPlace : WAVES * kSum;
  static_assert((R == 16 || R == 32) && XR % 4 == 0 && XR <= 64 && kLds <= 160 * 1024 && (DEPTH - 1) * kLoads < 63, "rows of scales a load; LDS; the counter of loads");
};

template <int R, int XR, bool A8, int WAVES, int DEPTH>
__global__ __launch_bounds__(64 * WAVES, 2) void mx_slim_kernel(const MxMatmulParams p, uint32_t tiles_m, uint32_t units) {
  using T = MxSlim<R, XR, A8, WAVES, DEPTH>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lds0 = lds_address_of(lds), own = lds0 + wave * (DEPTH * T::kPlace);
  const int batch = blockIdx.y;
  const int runs = (p.groups + kRunBlocks - 1) / kRunBlocks;
  const int run_begin = static_cast<int>(static_cast<int64_t>(runs) * blockIdx.z / p.splits);
  const int run_end = static_cast<int>(static_cast<int64_t>(runs) * (blockIdx.z + 1) / p.splits);
  // each die a contiguous run of tiles: those of the same weights are neighbours
  const uint32_t xcd = blockIdx.x & 7, share = units >> 3, extra = units & 7;
  const uint32_t pid = xcd * share + min(xcd, extra) + (blockIdx.x >> 3);
  const int64_t n0 = static_cast<int64_t>(pid / tiles_m) * R, m0 = static_cast<int64_t>(pid % tiles_m) * XR;
  const int last_n = static_cast<int>(min(p.n - n0, static_cast<int64_t>(R))) - 1, last_m = static_cast<int>(min(p.m - m0, static_cast<int64_t>(XR))) - 1;

  // Rows past the last one lie past the descriptors' ends: zeros arrive.
  const u32x4 desc_w = tile_buffer_words((const VECOPS_GLOBAL char*)p.b + batch * p.b_bs + n0 * p.ldb);
  const u32x4 desc_x = tile_buffer_words((const VECOPS_GLOBAL char*)p.a + batch * p.a_bs + m0 * p.lda);
  const u32x4 desc_sw = tile_buffer_words((const VECOPS_GLOBAL char*)p.b_scales + batch * p.bs_bs + n0 * p.bs_rs);
  const u32x4 desc_sx = tile_buffer_words((const VECOPS_GLOBAL char*)p.a_scales + batch * p.as_bs + m0 * p.as_rs);
  const uint32_t end_w = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(last_n * p.ldb) + static_cast<uint32_t>(p.groups) * 16u);
  const uint32_t end_x = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(last_m * p.lda) + static_cast<uint32_t>(p.groups) * (A8 ? 32u : 16u));
  const bool few = p.row_scales < kRunBlocks;
  const int last_first = few ? 0 : p.row_scales - kRunBlocks;
  const uint32_t end_sw = __builtin_amdgcn_readfirstlane(few ? 0u : static_cast<uint32_t>(last_n * p.bs_rs + p.row_scales));
  const uint32_t end_sx = __builtin_amdgcn_readfirstlane(few ? 0u : static_cast<uint32_t>(last_m * p.as_rs + p.row_scales));

  // Slot of a chunk: (chunk ^ (row + 4) % 16), of which LDS serves the rows that it reads together without conflicts (R = 16: of two places,
  // rows 0-3 and 12-15 of one, 4-11 of the other).  Load i of the weights: rows 4 i + lane / 16, slot lane % 16.
  const uint32_t from_sw = lane < R ? static_cast<uint32_t>(lane * p.bs_rs) : kNowhere, from_sx = lane < XR ? static_cast<uint32_t>(lane * p.as_rs) : kNowhere;
  auto issue = [&](int its_run, int place) {
    const int run = __builtin_amdgcn_readfirstlane(its_run);   // (the same in all lanes, which the compiler does not see)
    const uint32_t to = __builtin_amdgcn_readfirstlane(own + place * T::kPlace);
    const bool there = run < run_end;
    const int first_block = __builtin_amdgcn_readfirstlane(min(run * kRunBlocks, last_first)), old = run * kRunBlocks - first_block, most = p.groups - first_block;
    const uint32_t at_w = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(first_block) * 16u), at_x = __builtin_amdgcn_readfirstlane(at_w * (A8 ? 2u : 1u));
    const auto ending = [&](const u32x4& desc, uint32_t end) {
      u32x4 words = {desc[0], desc[1], there ? end : 0u, desc[3]};
#pragma unroll
      for (int i = 0; i < 4; ++i) words[i] = __builtin_amdgcn_readfirstlane(words[i]);
      return words;
    };
    const u32x4 of_w = ending(desc_w, end_w), of_x = ending(desc_x, end_x), of_sw = ending(desc_sw, end_sw), of_sx = ending(desc_sx, end_sx);
    const uint32_t at_s = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(first_block));
    load_16_bytes_into_lds(of_sw, to, T::kScales, from_sw, at_s);
    load_16_bytes_into_lds(of_sx, to, T::kScales + 1024, from_sx, at_s);
    static_for<T::kLoadsW>([&](auto i_tag) {
      constexpr int i = decltype(i_tag)::value;
      const int row = 4 * i + (lane >> 4), chunk = (lane & 15) ^ ((row + 4) & 15);
      load_16_bytes_into_lds(of_w, to, i * 1024, chunk >= old && chunk < most ? static_cast<uint32_t>(row * p.ldb) + chunk * 16 : kNowhere, at_w);
    });
    static_for<T::kLoadsX>([&](auto i_tag) {
      constexpr int i = decltype(i_tag)::value;
      const int row = A8 ? 2 * i + (lane >> 5) : 4 * i + (lane >> 4), chunk = (lane & (T::kChunksX - 1)) ^ ((row + 4) & 15), block = A8 ? chunk >> 1 : chunk;
      load_16_bytes_into_lds(of_x, to, T::kBytesW + i * 1024, block >= old && block < most ? static_cast<uint32_t>(row * p.lda) + chunk * 16 : kNowhere, at_x);
    });
  };

  constexpr int kSteps = R == 16 ? 4 : 8, kWords = kSteps / 4;
  const int col = lane & (R - 1), part = lane / R;   // a lane's row, and its place in the instruction
  const int row_w = R == 16 ? col : 16 * ((col >> 2) & 1) + 4 * (col >> 3) + (col & 3);
  typedef typename std::conditional<R == 16, f32x4, f32x16>::type Sums;
  Sums acc[T::kColumns];
#pragma unroll
  for (int j = 0; j < T::kColumns; ++j)
#pragma unroll
    for (int e = 0; e < (R == 16 ? 4 : 16); ++e) acc[j][e] = 0.f;

  const int mine = run_begin + wave;
  static_for<DEPTH>([&](auto d) { issue(mine + decltype(d)::value * WAVES, decltype(d)::value); });
  int place = 0;
  // all of this wavefront's runs; PARTS: e4m3 activations in two parts
  auto all_runs = [&](auto parts_tag) {
    constexpr bool PARTS = decltype(parts_tag)::value;
#pragma unroll 1
    for (int run = mine; run < run_end; run += WAVES) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DEPTH - 1) * T::kLoads) : "memory");
      const uint32_t at = own + place * T::kPlace;
      if (__builtin_expect(few, 0)) {   // (the only run)
        if (lane < R) write_lds(at + T::kScales + lane * 16, few_scales(p.b_scales, batch * p.bs_bs + (n0 + lane) * p.bs_rs, p.groups, lane <= last_n));
        if (lane < XR) write_lds(at + T::kScales + 1024 + lane * 16, few_scales(p.a_scales, batch * p.as_bs + (m0 + lane) * p.as_rs, p.groups, lane <= last_m));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      i32x8 w[kSteps];
      uint32_t sw[kWords];
#pragma unroll
      for (int u = 0; u < kWords; ++u) sw[u] = read_lds_word(at + T::kScales + row_w * 16 + part * (4 * kWords), 4 * u);
      static_for<kSteps>([&](auto t_tag) {
        constexpr int t = decltype(t_tag)::value;
        w[t] = narrow_fragment(read_lds(at + row_w * 256 + (((part * kSteps + t) ^ ((row_w + 4) & 15)) << 4), 0));
      });
      static_for<T::kColumns>([&](auto j_tag) {
        constexpr int j = decltype(j_tag)::value;
        const int row = min(j * R + col, XR - 1);   // (columns past the last row are not written)
        uint32_t sx[kWords];
#pragma unroll
        for (int u = 0; u < kWords; ++u) sx[u] = read_lds_word(at + T::kScales + 1024 + row * 16 + part * (4 * kWords), 4 * u);
        static_for<kSteps>([&](auto t_tag) {
          constexpr int t = decltype(t_tag)::value;
          const uint32_t x_at = at + T::kBytesW + row * T::kRowX;
          const int key = (row + 4) & 15;
          const auto multiply = [&](const i32x8& x) {
            if constexpr (R == 16) acc[j] = mfma_mx<A8, (t & 3)>(w[t], x, acc[j], sw[0], sx[0]);
            else acc[j] = mfma_mx_32<A8, (t & 3)>(w[t], x, acc[j], sw[t >> 2], sx[t >> 2]);
          };
          if constexpr (A8) {   // R = 16: half part % 2 of places part / 2 and 2 + part / 2; R = 32: half `part` of both places
            const int chunk = R == 16 ? 8 * (part >> 1) + 2 * t + (part & 1) : 2 * t + part;
            const i32x8 x = fragment_of(read_lds(x_at + ((chunk ^ key) << 4), 0), read_lds(x_at + ((chunk ^ key) << 4), 256));
            if constexpr (PARTS) {
              i32x8 high, low;
              part_by_size(x, high, low);
              multiply(low);
              multiply(high);
            } else {
              multiply(x);
            }
          } else {
            multiply(narrow_fragment(read_lds(x_at + (((part * kSteps + t) ^ key) << 4), 0)));
          }
        });
      });
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (what has been read may be overwritten)
      issue(run + DEPTH * WAVES, place);
      place = place + 1 == DEPTH ? 0 : place + 1;
    }
  };
  if constexpr (A8) {   // (uniform; one loop with a branch in it cost 16-bit results of 32 rows 4 %)
    if (p.out_kind == FP8_REAL_F32) all_runs(std::true_type{});
    else all_runs(std::false_type{});
  } else {
    all_runs(std::false_type{});
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  settle();
  __syncthreads();

  // The wavefronts' sums meet, [m][n] each: four neighbouring n a thread.
  static_for<T::kColumns>([&](auto j_tag) {
    constexpr int j = decltype(j_tag)::value;
    const uint32_t to = lds0 + wave * T::kSum + (j * R + col) * (R * 4) + part * (R == 16 ? 16 : 64);
#pragma unroll
    for (int e = 0; e < (R == 16 ? 4 : 16); e += 4)
      write_lds(to + e * 4, u32x4{__float_as_uint(acc[j][e]), __float_as_uint(acc[j][e + 1]), __float_as_uint(acc[j][e + 2]), __float_as_uint(acc[j][e + 3])});
  });
  __syncthreads();
  constexpr int kQuads = T::kColumns * R * R / 4;
#pragma unroll
  for (int q0 = 0; q0 < kQuads; q0 += 64 * WAVES) {
    const int q = q0 + tid;
    if (q >= kQuads) break;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < WAVES; ++u) {
      const u32x4 one = read_lds(lds0 + u * T::kSum + q * 16, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += __uint_as_float(one[e]);
    }
    const int64_t m = m0 + q / (R / 4), n = n0 + q % (R / 4) * 4;
    if (q / (R / 4) > last_m || n >= p.n) continue;
    if (p.splits == 1) store_results<4>(p.c, batch * p.c_bs + m * p.c_rs + n * p.c_cs, p.c_cs, p.out_kind, n, p.n, v);
    else store_results<4>(p.partial, ((static_cast<int64_t>(blockIdx.z) * p.batch + batch) * p.m + m) * p.n + n, 1, FP8_REAL_F32, n, p.n, v);
  }
}

// Operands whose rows are laid out in another way, all of them by one launch (171 x 426 x 12582, whose K is no whole blocks, 15.3 us a call; with a launch
// each that moves single bytes 28.7).  A unit of work is 256 times sixteen bytes of rows that are contiguous, else 64 x 64 bytes through LDS, each side in
// its own order.
__global__ __launch_bounds__(256) void mx_copies_kernel(const MxCopies copies) {
  __shared__ uint8_t tile[64][68];
  for (int64_t unit = blockIdx.x; unit < copies.of[copies.count - 1].end; unit += gridDim.x) {
    int which = 0;
    while (unit >= copies.of[which].end) ++which;   // (uniform)
    const MxCopy c = copies.of[which];
    const int64_t begin = which == 0 ? 0 : copies.of[which - 1].end, per_batch = (c.end - begin) / c.batch, batch = (unit - begin) / per_batch;
    const int64_t at = unit - begin - batch * per_batch;
    const VECOPS_GLOBAL uint8_t* in = (const VECOPS_GLOBAL uint8_t*)c.in + batch * c.bs;
    VECOPS_GLOBAL uint8_t* out = (VECOPS_GLOBAL uint8_t*)c.out + batch * c.rows * c.ld;
    if (c.cs == 1) {
      const int64_t pieces = c.ld / 16, piece = at * 256 + threadIdx.x, row = piece / pieces, from = (piece - row * pieces) * 16;
      if (row >= c.rows) continue;
      u32x4 v = {0u, 0u, 0u, 0u};
      if (from + 16 <= c.cols) {
        v = load_16(in + row * c.rs + from);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (from + e < c.cols) v[e >> 2] |= static_cast<uint32_t>(in[row * c.rs + from + e]) << (8 * (e & 3));
      }
      *(VECOPS_GLOBAL u32x4*)(out + piece * 16) = v;
    } else {
      const int64_t tiles = (c.ld + 63) / 64, r0 = at / tiles * 64, k0 = (at - at / tiles * tiles) * 64;
      const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
      for (int i = y; i < 64; i += 4)   // consecutive lanes: consecutive rows (the contiguous side of a [K, rows] matrix)
        tile[x][i] = r0 + x < c.rows && k0 + i < c.cols ? in[(r0 + x) * c.rs + (k0 + i) * c.cs] : 0;
      __syncthreads();
      for (int i = y; i < 64; i += 4)
        if (r0 + i < c.rows && k0 + x < c.ld) out[(r0 + i) * c.ld + k0 + x] = tile[i][x];
      __syncthreads();
    }
  }
}

hipError_t join(const MxMatmulParams& p, hipStream_t stream) {
  const hipError_t e = hipGetLastError();
  if (p.splits == 1 || e != hipSuccess) return e;
  return launch_join_shares({p.partial, p.c, p.c_rs, p.c_cs, p.c_bs, p.m, p.n, p.batch, p.splits, p.out_kind}, stream);
}

template <int R, int XR, bool A8, int WAVES, int DEPTH>
hipError_t launch_slim(const MxMatmulParams& p, hipStream_t stream) {
  using T = MxSlim<R, XR, A8, WAVES, DEPTH>;
  constexpr auto kernel = &mx_slim_kernel<R, XR, A8, WAVES, DEPTH>;
  if constexpr (T::kLds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds);
    if (e != hipSuccess) return e;
  }
  const uint32_t tiles_m = static_cast<uint32_t>((p.m + XR - 1) / XR), units = static_cast<uint32_t>((static_cast<int64_t>(p.n) + R - 1) / R) * tiles_m;
  hipLaunchKernelGGL(kernel, dim3(units, static_cast<uint32_t>(p.batch), static_cast<uint32_t>(p.splits)), dim3(64 * WAVES), T::kLds, stream, p, tiles_m, units);
  return join(p, stream);
}

template <int WN, int WM, int WK, int NT, int MT, bool A8, int STAGES, int WAVES_A_SIMD, bool GOES_ON, int OUT, bool PARTS = false>
hipError_t launch_tile_as(const MxMatmulParams& p, hipStream_t stream) {
  using T = MxTile<WN, WM, WK, NT, MT, A8, STAGES, GOES_ON>;
  constexpr auto kernel = &mx_tile_kernel<WN, WM, WK, NT, MT, A8, STAGES, WAVES_A_SIMD, GOES_ON, OUT, PARTS>;
  if constexpr (T::kLds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds);
    if (e != hipSuccess) return e;
  }
  const uint32_t tiles_n = static_cast<uint32_t>((p.n + T::kBN - 1) / T::kBN), tiles_m = static_cast<uint32_t>((p.m + T::kBM - 1) / T::kBM);
  const uint32_t units = tiles_n * tiles_m;
  hipLaunchKernelGGL(kernel, dim3(GOES_ON ? std::min(units, 256u) : units, static_cast<uint32_t>(p.batch), static_cast<uint32_t>(p.splits)), dim3(T::kThreads), T::kLds, stream, p, tiles_n,
                     tiles_m);
  return hipGetLastError();
}

template <int WN, int WM, int WK, int NT, int MT, bool A8, int STAGES, int WAVES_A_SIMD, bool GOES_ON>
hipError_t launch_tile(const MxMatmulParams& p, hipStream_t stream) {
  if (p.splits == 1 && p.out_kind == FP8_REAL_BF16) return launch_tile_as<WN, WM, WK, NT, MT, A8, STAGES, WAVES_A_SIMD, GOES_ON, FP8_REAL_BF16>(p, stream);
  if (p.splits == 1 && p.out_kind == FP8_REAL_F16) return launch_tile_as<WN, WM, WK, NT, MT, A8, STAGES, WAVES_A_SIMD, GOES_ON, FP8_REAL_F16>(p, stream);
  // (shares of 16-bit results too are added in fp32, but of products as those have them)
  const hipError_t e = A8 && p.out_kind == FP8_REAL_F32 ? launch_tile_as<WN, WM, WK, NT, MT, A8, STAGES, WAVES_A_SIMD, GOES_ON, FP8_REAL_F32, A8>(p, stream)
                                                        : launch_tile_as<WN, WM, WK, NT, MT, A8, STAGES, WAVES_A_SIMD, GOES_ON, FP8_REAL_F32>(p, stream);
  return e != hipSuccess ? e : join(p, stream);
}

}  // namespace

// Which kernel, and how many shares of k: the least of fitted times.  A kernel's workgroups (those of all shares) go in rounds over 256 compute units
// with `slots` of them each, as their LDS allows; a round of c on a compute unit takes start + runs (alone + more (c - 1)) us, where `runs` are the runs of
// 512 k that a wavefront has to do, and the bytes at 5.5 TB/s and 2 us are joined to that as a fourth power (the longer of the two counts, the other
// decides between equals).  Shares cost the joining launch and its bytes.  The constants were fitted to 4200 timings of every kernel and of 1 and 2
// shares at 620 products of random sizes (M 1 .. 4096, N 256 .. 28000, K 512 .. 16384) on weights that no cache held.  What the rule takes is 0.6 %
// slower than the fastest of them on average and 1.19 times at worst.  The best choice without one of them would be slower by 2.2 % (MX_ROWS_4),
// 2.1 % (MX_TILE_256), 1.5 % (MX_TILE_128), 1.1 % (MX_ROWS_32), 0.9 % (MX_ROWS_4_DEEP), 0.6 % (MX_TILE_128X64, MX_TILE_128_DEEP), 0.5 % (MX_ROWS_16_DEEP) and
// 0.3 % (shares, 1.38 times at worst; four shares rather than two, or of few rows, 0.04 %); 32 x 64 results a workgroup and 4 x 16 by four wavefronts
// brought 0.2 % each and are left out.  K of up to 512 lie at the fit's edge or past it: of 92 such products (M 256 .. 8192, N 2048 .. 16384, K 128, 256, 480, 512)
// with e4m3 what it takes is 0.1 % slower than the fastest, 1.04 times at worst, with e2m1 5 % and 1.51 times (MX_TILE_128 where MX_TILE_256 has three rounds and
// more: 4096 x 16384 x 480 71 us rather than 47).  Up to four rows only kernels of four are weighed: on a tie of latencies the fit's errors would decide.
MxPlan mx_plan(int64_t m, int64_t n, int64_t k, int64_t batch, bool a_wide) {
  struct Cost {
    int rows_a, rows_b, wavefronts, slots;   // as powers of two; wavefronts that share k by whole runs
    float once, start, alone, more;          // us
  };
  constexpr Cost kCosts[2][MX_KINDS] = {
      {{2, 4, 1, 3, 1.99f, 0.64f, 0.51f, 0.22f},    // MX_ROWS_4
       {2, 4, 2, 1, 1.06f, 1.85f, 0.52f, 0.42f},    // MX_ROWS_4_DEEP
       {4, 4, 2, 2, 1.58f, 0.94f, 0.85f, 0.50f},    // MX_ROWS_16
       {4, 4, 2, 1, 1.24f, 1.72f, 0.56f, 0.72f},    // MX_ROWS_16_DEEP
       {5, 5, 2, 1, 1.83f, 0.85f, 1.50f, 1.23f},    // MX_ROWS_32
       {6, 6, 0, 1, 1.87f, 2.37f, 0.70f, 0.75f},    // MX_TILE_64
       {6, 7, 0, 1, 1.96f, 3.53f, 1.15f, 0.90f},    // MX_TILE_128X64
       {7, 7, 0, 1, 1.16f, 3.47f, 1.89f, 0.86f},    // MX_TILE_128
       {7, 7, 0, 0, 1.60f, 5.14f, 1.48f, 0.f},      // MX_TILE_128_DEEP
       {8, 8, 0, 0, 4.85f, 9.57f, 3.14f, 0.f}},     // MX_TILE_256
      {{2, 4, 1, 3, 2.46f, 0.f, 0.60f, 0.26f},
       {2, 4, 2, 1, 1.04f, 1.94f, 0.46f, 0.64f},
       {4, 4, 2, 1, 1.33f, 1.21f, 1.02f, 0.62f},
       {4, 4, 3, 0, 0.91f, 1.30f, 1.69f, 0.f},
       {5, 5, 2, 0, 1.04f, 1.66f, 1.98f, 0.f},
       {6, 6, 0, 1, 1.73f, 2.56f, 0.93f, 0.87f},
       {6, 7, 0, 0, 2.07f, 3.44f, 1.37f, 0.f},
       {7, 7, 0, -1, 0.f, 0.f, 0.f, 0.f},           // (two workgroups of such tiles a compute unit: of e2m1 only)
       {7, 7, 0, 0, 2.06f, 4.88f, 1.96f, 0.f},
       {7, 8, 0, 0, 5.70f, 3.25f, 2.98f, 0.f}}};
  const int64_t runs = (k + 511) / 512;
  const auto shared = [](int64_t x, int by) { return (x + (int64_t{1} << by) - 1) >> by; };
  const float bytes = (static_cast<float>(n) * k * (17 / 32.f) + static_cast<float>(m) * k * (a_wide ? 33 / 32.f : 17 / 32.f) + 2.f * m * n) * batch;
  const float moved = 2.f + bytes / 5.5e6f;
  MxPlan best{};
  float least = INFINITY;
  for (int kind = 0; kind < MX_KINDS; ++kind) {
    const Cost& cost = kCosts[a_wide][kind];
    if (cost.slots < 0 || (m <= 4 && kind >= MX_ROWS_16) || (kind < MX_TILE_64 && m > 1 << (2 * cost.rows_a))) continue;   // (few rows up to M = 16, 256 and 1024, as they were timed)
    const int64_t tiles = shared(m, cost.rows_a) * shared(n, cost.rows_b);
    // (a grid holds fewer than 2^32 threads, of which a workgroup has up to 512; those of MX_TILE_256 go from tile to tile)
    if (tiles > (kind == MX_ROWS_16_DEEP || kind == MX_TILE_128_DEEP ? 1 << 22 : 1 << 23) && kind != MX_TILE_256) continue;
    for (int split = 0; split == 0 || (split == 1 && kind >= MX_TILE_64 && runs >= 4); ++split) {
      const int64_t each = shared(shared(runs, split), cost.wavefronts), depth = shared((tiles * batch) << split, 8), rounds = depth >> cost.slots;
      const int slots = 1 << cost.slots, rest = static_cast<int>(depth - (rounds << cost.slots));
      float us = cost.once + rounds * (cost.start + (cost.alone + cost.more * (slots - 1)) * each);
      if (rest > 0) us += cost.start + (cost.alone + cost.more * (rest - 1)) * each;
      us = std::sqrt(std::sqrt(us * us * us * us + moved * moved * moved * moved));
      if (kind == MX_TILE_256 && k % kMxBlock == 0 && k / kMxBlock < kRunBlocks) us += 2.5f;   // (for the launch that lays out scales too few a row; a K of no whole blocks has one anyway)
      if (split > 0) us += 3.2f + 2.8e-6f * (static_cast<float>(m) * n * batch);
      if (us < least) least = us, best = {kind, 1 << split, 1 << cost.rows_a, 1 << cost.rows_b, kind == MX_TILE_256 ? kRunBlocks : 0};
    }
  }
  return best;
}

hipError_t launch_mx_copies(MxCopies& copies, hipStream_t stream) {
  int64_t end = 0;
  for (int i = 0; i < copies.count; ++i) {
    MxCopy& c = copies.of[i];
    end += c.batch * (c.cs == 1 ? (c.rows * (c.ld / 16) + 255) / 256 : (static_cast<int64_t>(c.rows) + 63) / 64 * ((c.ld + 63) / 64));
    c.end = end;
  }
  hipLaunchKernelGGL(mx_copies_kernel, dim3(static_cast<uint32_t>(std::min<int64_t>(end, 1 << 20))), dim3(256), 0, stream, copies);
  return hipGetLastError();
}

hipError_t launch_mx_matmul(const MxMatmulParams& p, int kind, hipStream_t stream) {
  switch (kind) {
    case MX_ROWS_4: return p.a_wide ? launch_slim<16, 4, true, 2, 1>(p, stream) : launch_slim<16, 4, false, 2, 1>(p, stream);
    case MX_ROWS_4_DEEP: return p.a_wide ? launch_slim<16, 4, true, 4, 2>(p, stream) : launch_slim<16, 4, false, 4, 2>(p, stream);
    case MX_ROWS_16: return p.a_wide ? launch_slim<16, 16, true, 4, 1>(p, stream) : launch_slim<16, 16, false, 4, 1>(p, stream);
    case MX_ROWS_16_DEEP: return p.a_wide ? launch_slim<16, 16, true, 8, 1>(p, stream) : launch_slim<16, 16, false, 4, 2>(p, stream);
    case MX_ROWS_32: return p.a_wide ? launch_slim<32, 32, true, 4, 1>(p, stream) : launch_slim<32, 32, false, 4, 1>(p, stream);
    case MX_TILE_64: return p.a_wide ? launch_tile<1, 2, 2, 2, 1, true, 3, 2, false>(p, stream) : launch_tile<1, 2, 2, 2, 1, false, 4, 2, false>(p, stream);
    case MX_TILE_128X64: return p.a_wide ? launch_tile<2, 1, 2, 2, 2, true, 3, 2, false>(p, stream) : launch_tile<2, 1, 2, 2, 2, false, 3, 2, false>(p, stream);
    case MX_TILE_128: return p.a_wide ? hipErrorInvalidValue : launch_tile<2, 2, 1, 2, 2, false, 2, 2, false>(p, stream);
    case MX_TILE_128_DEEP: return p.a_wide ? launch_tile<2, 2, 2, 2, 2, true, 3, 2, false>(p, stream) : launch_tile<2, 2, 2, 2, 2, false, 4, 2, false>(p, stream);
    case MX_TILE_256: return p.a_wide ? launch_tile<2, 2, 1, 4, 2, true, 2, 1, true>(p, stream) : launch_tile<2, 2, 1, 4, 4, false, 2, 1, true>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace vecops_hip
