// Parameters and launchers of the 8-bit float kernels (fp8_block.hip): quantisation to e4m3 with a scale for each block of
// 128, and the product of such operands.
#ifndef VECOPS_HIP_FP8_BLOCK_H
#define VECOPS_HIP_FP8_BLOCK_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vecops_hip {

constexpr int kFp8Block = 128;  // k (and, for weights, rows) that share a scale

enum Fp8Real : int { FP8_REAL_BF16 = 0, FP8_REAL_F16 = 1, FP8_REAL_F32 = 2 };

struct Fp8QuantizeParams {
  const void* x;   // [batch][rows][k] of `kind`
  uint8_t* q;      // e4m3
  float* scales;   // [batch][ceil(rows / block rows)][groups]
  int64_t x_bs, x_rs, x_cs;
  int64_t q_bs, q_rs, q_cs;
  int64_t s_bs, s_rs, s_cs;
  int32_t batch, rows, k, groups;
  int32_t kind;    // Fp8Real
};

struct Fp8MatmulParams {
  const uint8_t* a;  // activations [batch][m][k], k contiguous
  const uint8_t* b;  // weights [batch][n][k], k contiguous
  const float* a_scales;  // [batch][m][groups]
  const float* b_scales;  // [batch][ceil(n / 128)][groups]
  void* c;                // [batch][m][n]
  int64_t lda, ldb, a_bs, b_bs;
  int64_t as_rs, as_bs;   // (a row's scales follow one another)
  int64_t bs_rs, bs_bs;
  int64_t c_rs, c_cs, c_bs;
  int32_t m, n, k, batch;  // k: 0, or at least 16
  int32_t groups;    // ceil(k / 128)
  int32_t out_kind;  // Fp8Real
  int32_t splits;    // shares of K; more than one leave through `partial`, [splits][batch][m][n]
  float* partial;
};

// block_rows 1 or 128
hipError_t launch_fp8_quantize(const Fp8QuantizeParams& p, int block_rows, hipStream_t stream);

// out[batch][row][0..k) = in with element strides rs, cs, then zeros; rows of `ld` < k + 64 bytes
hipError_t launch_fp8_rows(const uint8_t* in, int64_t bs, int64_t rs, int64_t cs, uint8_t* out, int64_t ld, int32_t batch,
                           int32_t rows, int32_t k, hipStream_t stream);

// out[batch][row][group] = in with element strides bs, rs, gs
hipError_t launch_fp8_scales(const float* in, int64_t bs, int64_t rs, int64_t gs, float* out, int32_t batch, int32_t rows, int32_t groups,
                             hipStream_t stream);

// The kernels of the product: up to sixteen rows; tiles of 64 x 64, 128 rows x 64, 128 x 128 (one workgroup of eight
// wavefronts a compute unit, or two of four), 256 x 256 (16-bit results only).
enum Fp8Kind : int { FP8_FEW_ROWS = 0, FP8_TILE_64, FP8_TILE_128X64, FP8_TILE_128_ALONE, FP8_TILE_128_PAIRED, FP8_TILE_256 };
struct Fp8Plan {
  int kind;
  int splits;  // shares of K; more than one need `partial`
  // Rows of a and of b that a workgroup reaches from its first one, by offsets of 32 bits whose upper half means nothing there:
  // (rows - 1) * ld + k + 128 has to stay below 2^31.
  int rows_a, rows_b;
};
Fp8Plan fp8_plan(int64_t m, int64_t n, int64_t k, int64_t batch, int out_kind);
hipError_t launch_fp8_matmul(const Fp8MatmulParams& p, int kind, hipStream_t stream);

}  // namespace vecops_hip
#endif
