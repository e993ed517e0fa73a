// group_norm.h — geometry and launch interface of group normalisation with an activation (group_norm.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <cstddef>

namespace rst {

struct GroupNormArgs {
    const void* x;            // [B][hw][C], f32 or bf16 bits
    const void* dy;           // backward: gradient of the output
    void* out;                // forward: y; backward: dx
    const float* scale;       // [C] or [B][C]
    const float* bias;
    long aff_stride;          // 0: one affine for all images, C: one per image
    float* mean;              // [B][G], written by the forward (or null), read by the backward
    float* rstd;
    float* dscale;            // backward, shaped as scale / bias
    float* dbias;
    void* workspace;
    long hw;
    int batch, C, G;
    float eps;
    int act;                  // RST_ACT_*
    int bf16;
};

size_t group_norm_workspace_bytes(int batch, long hw, int C, int G);
bool group_norm_supported(int batch, long hw, int C, int G);
size_t group_norm_bwd_workspace_bytes(int batch, long hw, int C, int G);
hipError_t group_norm_launch(const GroupNormArgs& a, hipStream_t st);
hipError_t group_norm_bwd_launch(const GroupNormArgs& a, hipStream_t st);

}  // namespace rst
