// Parameters and launchers of row_quantize.hip: microscaled copies of matrices and what they stand for, and the operators between
// a layer's products whose results are quantised by rows - the root-mean-square norm and the gated activation.
#ifndef VECOPS_HIP_ROW_QUANTIZE_H
#define VECOPS_HIP_ROW_QUANTIZE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fp8_block.h"

namespace vecops_hip {

constexpr int kMxBlock = 32;  // elements along k that share a power of two

// How results are held.  ROW_INT8: int8, an fp32 scale a row.  ROW_E4M3_128: e4m3, an fp32 scale for each 128.
// ROW_MX_E4M3, ROW_MX_E2M1: e4m3, or e2m1 two a byte, a power of two for each 32.
enum RowFormat : int { ROW_NONE = 0, ROW_INT8, ROW_E4M3_128, ROW_MX_E4M3, ROW_MX_E2M1 };

struct MxCopyParams {   // between a matrix and its microscaled copy
  void* x;          // [batch][rows][k] of `kind`
  uint8_t* q;       // e4m3, or e2m1 (strides in bytes)
  uint8_t* scales;  // [batch][rows][groups]
  int64_t x_bs, x_rs, x_cs;
  int64_t q_bs, q_rs, q_cs;
  int64_t s_bs, s_rs, s_cs;
  int32_t batch, rows, k, groups;
  int32_t kind;    // Fp8Real
  int32_t format;  // ROW_MX_E4M3 or ROW_MX_E2M1
};
hipError_t launch_mx_quantize(const MxCopyParams& p, hipStream_t stream);
hipError_t launch_mx_dequantize(const MxCopyParams& p, hipStream_t stream);

// Rows are contiguous (q, x, residual, summed, out); scales have any strides.
struct RowQuantizeParams {
  const void* x;         // norm: [batch][rows][k]; gated activation: [batch][rows][2 k], the gates first
  const void* residual;  // norm, or null
  void* summed;          // norm with a residual: x + residual in x's type (may be the residual itself)
  const void* weight;    // norm: [k]
  void* out;             // norm, or null: the result in x's type
  uint8_t* q;            // (null with ROW_NONE)
  void* scales;
  int64_t x_bs, x_rs, residual_bs, residual_rs, summed_bs, summed_rs, out_bs, out_rs, q_bs, q_rs;
  int64_t s_bs, s_rs, s_cs;
  int32_t batch, rows, k, groups;
  int32_t kind, weight_kind;  // Fp8Real
  int32_t format;             // RowFormat
  float eps;
};
hipError_t launch_rms_norm(const RowQuantizeParams& p, hipStream_t stream);
hipError_t launch_silu_mul(const RowQuantizeParams& p, hipStream_t stream);

}  // namespace vecops_hip
#endif
