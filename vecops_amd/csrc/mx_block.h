// Parameters and launchers of the product of microscaled operands (mx_block.hip).
#ifndef VECOPS_HIP_MX_BLOCK_H
#define VECOPS_HIP_MX_BLOCK_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "row_quantize.h"

namespace vecops_hip {

struct MxMatmulParams {
  const uint8_t* a;  // activations [batch][m][k]: e2m1 two a byte, or e4m3; a row's bytes follow one another
  const uint8_t* b;  // weights [batch][n][k], e2m1
  const uint8_t* a_scales;  // [batch][m][groups], a row's follow one another
  const uint8_t* b_scales;  // [batch][n][groups]
  void* c;                  // [batch][m][n]
  int64_t lda, ldb, a_bs, b_bs;   // bytes
  int64_t as_rs, as_bs, bs_rs, bs_bs;
  int64_t c_rs, c_cs, c_bs;
  int32_t m, n, batch;
  int32_t groups;      // blocks of 32 along k, each whole
  int32_t row_scales;  // scales of a row that can be read: groups, or sixteen where rows of fewer have been padded (what MX_TILE_256 needs)
  int32_t a_wide;    // a is e4m3
  int32_t out_kind;  // Fp8Real
  int32_t splits;    // shares of k; more than one leave through `partial`, [splits][batch][m][n]
  float* partial;
};

// Rows brought together: out[batch][row][0..cols) = in with strides rs, cs, then zeros up to `ld`, a multiple of sixteen bytes.  Up to four at once.
struct MxCopy {
  const uint8_t* in;
  uint8_t* out;
  int64_t bs, rs, cs, ld;
  int32_t batch, rows, cols;
  int64_t end;   // units of work, those of the copies before included (the launcher's)
};
struct MxCopies {
  MxCopy of[4];
  int32_t count;
};
hipError_t launch_mx_copies(MxCopies& copies, hipStream_t stream);

// The kernels.  MX_ROWS_r: r activation rows by 16 (r = 4, 16) or 32 weight rows a workgroup, whose wavefronts share k; MX_TILE_t: tiles of t x t,
// MX_TILE_128X64 of 128 weight rows by 64, MX_TILE_256 of 256 by 256, with e4m3 activations by 128.  _DEEP: more of k under way a workgroup, for products of few workgroups.
enum MxKind : int { MX_ROWS_4 = 0, MX_ROWS_4_DEEP, MX_ROWS_16, MX_ROWS_16_DEEP, MX_ROWS_32, MX_TILE_64, MX_TILE_128X64, MX_TILE_128, MX_TILE_128_DEEP, MX_TILE_256, MX_KINDS };
struct MxPlan {
  int kind;
  int splits;  // shares of k; more than one need `partial`
  int rows_a, rows_b;  // of an operand, that a workgroup reaches by offsets below 2 GiB
  int scales;          // the fewest of a row
};
MxPlan mx_plan(int64_t m, int64_t n, int64_t k, int64_t batch, bool a_wide);
hipError_t launch_mx_matmul(const MxMatmulParams& p, int kind, hipStream_t stream);

}  // namespace vecops_hip
#endif
