// adamw.h — kernel interface of the AdamW step over many tensors (adamw.hip), used by adamw_api.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <cstddef>

namespace rst {

constexpr int ADAMW_BLOCK = 128;       // elements of one 8-bit state block (and its scale)
constexpr int ADAMW_CHUNK = 4096;      // elements of one workgroup: a multiple of the block
constexpr int ADAMW_MAX_PARTIALS = 1024;
constexpr int ADAMW_TICKETS = 64;      // workgroups that share a counter
constexpr int ADAMW_TICKET_STRIDE = 32;   // a cache line
constexpr int ADAMW_PTRS = 256;        // gradient pointers that one launch carries to the device

// A workgroup's share of one variable
struct AdamwChunk {
    float* param;
    long long grad_at;                 // element of the gradient bucket
    long long tensor_at;               // element of the variable
    long long state_at;                // element of the states
    int count;
    int tensor;
    int decay;
    int pad;
};

struct AdamwArgs {
    const AdamwChunk* chunks;
    const void* bucket;                // all gradients in one buffer, or null:
    const void* const* grad_ptrs;      // (device) one pointer per variable
    int grad_bf16;
    int num_chunks;
    void* m;                           // f32, or e4m3 codes with m_scale / v_scale per block
    void* v;
    float* m_scale;
    float* v_scale;
    long long* iterations;
    float* global_norm;                // may be null without clipping
    unsigned* tickets;                 // a root and one per ADAMW_TICKETS workgroups, ADAMW_TICKET_STRIDE apart
    const double* partials;            // sums of squares of the gradient
    int num_partials;                  // 0: no clipping
    double lr, decay, b1, b2, eps, clip;
    double log_b1, log_b2;
    unsigned seed;
};

struct AdamwPtrs {
    const void* p[ADAMW_PTRS];
};

hipError_t adamw_set_pointers_launch(const AdamwPtrs& p, const void** dst, int n, hipStream_t st);
hipError_t adamw_norm_launch(const AdamwArgs& a, double* partials, hipStream_t st);
// past: loads and stores past the caches
hipError_t adamw_step_launch(const AdamwArgs& a, int state_bits, bool past, hipStream_t st);

}  // namespace rst
