// Parameters and launchers of the mixture-of-experts layer for a few tokens (moe_few_tokens.hip).
#ifndef VECOPS_HIP_MOE_FEW_TOKENS_H
#define VECOPS_HIP_MOE_FEW_TOKENS_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vecops_hip {

constexpr int kMoeMostTokens = 128, kMoeMostExperts = 512, kMoeMostChoices = 16, kMoeMostShares = 8;

struct MoeRouteParams {
  const void* x;       // [tokens][hidden], bf16 or f16
  const void* router;  // [experts][hidden], x's type or fp32
  const float* bias;   // [experts] or null
  float* logits;       // [parts][tokens][experts]: sums over parts of the hidden axis
  int32_t* ids;        // [tokens][top]
  float* weights;      // [tokens][top]
  int64_t ldx, ld_router;
  int64_t ids_rs, ids_cs, weights_rs, weights_cs;
  int32_t tokens, experts, hidden, top;
  int32_t parts;
  int32_t x_f16, router_f32;
  int32_t sigmoid, renormalize;
  float scale;
};

struct MoeExpertsParams {
  const void* x;         // [tokens][hidden], bf16 or f16
  const int32_t* ids;    // [tokens][top]; numbers outside 0..experts-1 name no expert
  const float* weights;  // [tokens][top]
  const void* gate_up;   // [experts][2 inner][hidden]: x's type or e4m3
  const void* down;      // [experts][hidden][inner]
  const float* gate_up_scales;  // e4m3: [experts][ceil(2 inner / 128)][ceil(hidden / 128)]
  const float* down_scales;     // e4m3: [experts][ceil(hidden / 128)][ceil(inner / 128)]
  uint16_t* middle;      // [2][tokens * top][inner_pad]: the experts' inner values, weighted, as a bf16 and what that leaves
  float* shares;         // [moe_down_shares][ceil(hidden / 16)][tokens][16]: parts of the result
  int32_t* arrived;      // [ceil(hidden / 16)]: how many of them are there
  void* out;             // [tokens][hidden], x's type or fp32
  int64_t ldx, ids_rs, ids_cs, weights_rs, weights_cs;
  int64_t gate_up_es, gate_up_rs, down_es, down_rs;  // in elements
  int64_t gs_es, gs_rs, gs_cs, ds_es, ds_rs, ds_cs;
  int64_t out_rs, out_cs;
  int32_t tokens, experts, hidden, inner, inner_pad, top;
  int32_t x_f16, w_e4m3, out_f32;
};

int moe_route_parts(int hidden);
int moe_down_shares(int hidden);
hipError_t launch_moe_experts(const MoeExpertsParams& p, hipStream_t stream);
hipError_t launch_moe_layer(const MoeRouteParams& route, const MoeExpertsParams& p, hipStream_t stream);

}  // namespace vecops_hip
#endif
