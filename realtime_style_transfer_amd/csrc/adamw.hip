// adamw.hip — the AdamW step over many tensors in one launch, states in 32 or in 8 bits, global-norm clipping.
//
// Step t, gradient g, c = min(1, clip / |g|) over all variables:
//   m = b1 m + (1 - b1) c g,  v = b2 v + (1 - b2) (c g)^2
//   p -= lr (m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps) + decay p)
// One pass over the data: every element's g, p, m, v are read once and p, m, v written once (28 bytes in 32 bits, 16.1
// with 8-bit states), which is all that bounds it. A workgroup takes one chunk of at most 4096 elements of one variable
// from a table made once, so a step over hundreds of small variables is one launch. The step count is on the device
// (a captured step replays as the next one): every workgroup reads t, and the last one to finish writes t + 1.
//
// 8-bit states: blocks of 128 elements of one variable with a scale s = max / 448 each, codes in e4m3. m / s rounds to
// nearest. v / s is rounded up or down at random with the right mean: (1 - b2) of a change is far below half a code, so
// that rounding to nearest would leave v where it is for ever. The random bits are a hash of (element, step, seed), so
// a step is reproducible. A v above zero keeps a code above zero: its root divides. Moments, scales and codes are
// formed in 64 bits, which issue at the f32 rate here, so that a code does not depend on the order of operations.
#include <hip/hip_runtime.h>

#include "adamw.h"

namespace rst {
namespace {

constexpr int NT = 256;

// Vectors of data whose alignment is the element's only: variables lie anywhere in a flat buffer
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef u16x4 u16x4_u __attribute__((aligned(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float widen(unsigned short v) { return __uint_as_float((unsigned)v << 16); }

__device__ __forceinline__ f32x4 load_grad4(const void* g, long long i, int bf16) {
    if (bf16) {
        const u16x4 v = *(const u16x4_u*)((const unsigned short*)g + i);
        return f32x4{widen(v.x), widen(v.y), widen(v.z), widen(v.w)};
    }
    return *(const f32x4_u*)((const float*)g + i);
}
__device__ __forceinline__ float load_grad(const void* g, long long i, int bf16) {
    return bf16 ? widen(((const unsigned short*)g)[i]) : ((const float*)g)[i];
}

// The chunk's gradient: a base and an element index
__device__ __forceinline__ const void* grad_of(const AdamwArgs& a, const AdamwChunk& c, long long& at) {
    at = a.bucket != nullptr ? c.grad_at : c.tensor_at;
    return a.bucket != nullptr ? a.bucket : a.grad_ptrs[c.tensor];
}

__device__ __forceinline__ double block_sum(double v, double* red) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(ADAMW_PTRS) void set_pointers_kernel(AdamwPtrs p, const void** dst, int n) {
    if ((int)threadIdx.x < n) dst[threadIdx.x] = p.p[threadIdx.x];
}

// Sums of squares over the chunks blockIdx, blockIdx + grid, ...: one partial per workgroup, merged by the step
__global__ __launch_bounds__(NT) void norm_kernel(AdamwArgs a, double* __restrict__ partials) {
    __shared__ double red[4];
    double s = 0.0;
    for (int k = blockIdx.x; k < a.num_chunks; k += gridDim.x) {
        const AdamwChunk c = a.chunks[k];
        long long at;
        const void* g = grad_of(a, c, at);
        for (int i = threadIdx.x * 4; i < c.count; i += NT * 4) {
            if (i + 4 <= c.count) {
                const f32x4 v = load_grad4(g, at + i, a.grad_bf16);
                s = fma((double)v.x, (double)v.x, fma((double)v.y, (double)v.y,
                    fma((double)v.z, (double)v.z, fma((double)v.w, (double)v.w, s))));
            } else {
                for (int j = i; j < c.count; ++j) {
                    const double v = load_grad(g, at + j, a.grad_bf16);
                    s = fma(v, v, s);
                }
            }
        }
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// What the whole step shares: the clipping factor, the step number and its corrections; false: nothing to do, the
// gradient's norm is not finite
struct StepScalars {
    double coef, inv_bc1, inv_bc2;
    long long t;
};
__device__ __forceinline__ bool step_scalars(const AdamwArgs& a, StepScalars& s, double* red) {
    s.t = *a.iterations + 1;
    s.coef = 1.0;
    if (a.num_partials > 0) {
        double q = 0.0;
        for (int i = threadIdx.x; i < a.num_partials; i += NT) q += a.partials[i];
        const double norm = sqrt(block_sum(q, red));
        if (blockIdx.x == 0 && threadIdx.x == 0 && a.global_norm != nullptr) *a.global_norm = (float)norm;
        if (!(norm < __builtin_inf())) return false;
        if (norm > a.clip) s.coef = a.clip / norm;
    }
    s.inv_bc1 = -1.0 / expm1((double)s.t * a.log_b1);
    s.inv_bc2 = -1.0 / expm1((double)s.t * a.log_b2);
    return true;
}

// The last workgroup moves the step count on: every other one has read it
__device__ __forceinline__ void step_done(const AdamwArgs& a, long long t) {
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned n = __hip_atomic_fetch_add(a.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (n == (unsigned)a.num_chunks - 1) {
            *a.ticket = 0;
            *a.iterations = t;
        }
    }
}

struct Scalars32 {
    float b1, c1, b2, c2, inv_bc1, inv_bc2, eps, lr, decay;
};

__device__ __forceinline__ void adamw_element(float g, float& p, float& m, float& v, const Scalars32& s) {
    m = fmaf(s.b1, m, s.c1 * g);
    v = fmaf(s.b2, v, s.c2 * (g * g));
    const float q = (m * s.inv_bc1) / (sqrtf(v * s.inv_bc2) + s.eps);
    p = fmaf(-s.lr, fmaf(s.decay, p, q), p);
}

__global__ __launch_bounds__(NT) void adamw32_kernel(AdamwArgs a) {
    __shared__ double red[4];
    const AdamwChunk c = a.chunks[blockIdx.x];
    StepScalars st;
    const bool go = step_scalars(a, st, red);
    if (!go) return;
    const Scalars32 s{(float)a.b1, (float)(1.0 - a.b1), (float)a.b2, (float)(1.0 - a.b2), (float)st.inv_bc1,
                      (float)st.inv_bc2, (float)a.eps, (float)a.lr, c.decay ? (float)a.decay : 0.f};
    const float coef = (float)st.coef;
    long long at;
    const void* g = grad_of(a, c, at);
    float* __restrict__ p = c.param;
    float* __restrict__ m = (float*)a.m + c.state_at;
    float* __restrict__ v = (float*)a.v + c.state_at;
    for (int i = threadIdx.x * 4; i < c.count; i += NT * 4) {
        if (i + 4 <= c.count) {
            const f32x4 gv = load_grad4(g, at + i, a.grad_bf16);
            f32x4 pv = *(const f32x4_u*)(p + i), mv = *(const f32x4_u*)(m + i), vv = *(const f32x4_u*)(v + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float pk = pv[k], mk = mv[k], vk = vv[k];
                adamw_element(gv[k] * coef, pk, mk, vk, s);
                pv[k] = pk;
                mv[k] = mk;
                vv[k] = vk;
            }
            *(f32x4_u*)(p + i) = pv;
            *(f32x4_u*)(m + i) = mv;
            *(f32x4_u*)(v + i) = vv;
        } else {
            for (int j = i; j < c.count; ++j) adamw_element(load_grad(g, at + j, a.grad_bf16) * coef, p[j], m[j], v[j], s);
        }
    }
    step_done(a, st.t);
}

// ---- 8-bit states --------------------------------------------------------------------------------------------------

// Two rounds of xor-shift and multiply: a bijection of 32 bits whose outputs look random
__device__ __forceinline__ unsigned mix(unsigned x) {
    x = (x ^ (x >> 16)) * 0x7FEB352Du;
    x = (x ^ (x >> 15)) * 0x846CA68Bu;
    return x ^ (x >> 16);
}

// y in [0, 448] to an e4m3 code, up with the probability of its place between two codes (u: 16 random bits)
__device__ __forceinline__ unsigned round_random(float y, unsigned u) {
    const unsigned r = u << 4;       // an f32 has 20 bits below e4m3's three
    unsigned code;
    if (y < 0.015625f)               // below 2^-6 codes are 2^-9 apart
        code = ((unsigned)(y * 536870912.f) + r) >> 20;
    else
        code = ((__float_as_uint(y) + r) >> 20) - ((127 - 7) << 3);
    return code > 0x7Eu ? 0x7Eu : code;
}

__device__ __forceinline__ double max16(double v) {     // over the 16 lanes of a block
    for (int o = 8; o > 0; o >>= 1) {
        const double w = __shfl_xor(v, o);
        v = (w > v || w != w) ? w : v;                  // a NaN wins
    }
    return v;
}

// Eight elements per lane, 16 lanes per block
__global__ __launch_bounds__(NT) void adamw8_kernel(AdamwArgs a) {
    __shared__ double red[4];
    const AdamwChunk c = a.chunks[blockIdx.x];
    StepScalars st;
    const bool go = step_scalars(a, st, red);
    if (!go) return;
    const unsigned key = mix(a.seed + (unsigned)st.t * 0x9E3779B9u);
    const float inv_bc1 = (float)st.inv_bc1, inv_bc2 = (float)st.inv_bc2, eps = (float)a.eps, lr = (float)a.lr,
                decay = c.decay ? (float)a.decay : 0.f;
    const double b1 = a.b1, c1 = 1.0 - a.b1, b2 = a.b2, c2 = 1.0 - a.b2;
    long long at;
    const void* gp = grad_of(a, c, at);
    float* __restrict__ p = c.param;
    unsigned char* __restrict__ m8 = (unsigned char*)a.m + c.state_at;
    unsigned char* __restrict__ v8 = (unsigned char*)a.v + c.state_at;
    const int blocks = (c.count + ADAMW_BLOCK - 1) / ADAMW_BLOCK;
    const long long block0 = c.state_at / ADAMW_BLOCK;
    for (int i = threadIdx.x * 8; i < blocks * ADAMW_BLOCK; i += NT * 8) {
        const long long block = block0 + i / ADAMW_BLOCK;
        const u32x2 mc = *(const u32x2*)(m8 + i), vc = *(const u32x2*)(v8 + i);
        const double ms = b1 * (double)a.m_scale[block], vs = b2 * (double)a.v_scale[block];
        float g[8], pv[8];
        const int n = min(8, c.count - i);              // may be below zero at a block's filled end
        if (n == 8) {
#pragma unroll
            for (int k = 0; k < 8; k += 4) {
                const f32x4 x = load_grad4(gp, at + i + k, a.grad_bf16), y = *(const f32x4_u*)(p + i + k);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    g[k + q] = x[q];
                    pv[k + q] = y[q];
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                g[k] = k < n ? load_grad(gp, at + i + k, a.grad_bf16) : 0.f;
                pv[k] = k < n ? p[i + k] : 0.f;
            }
        }
        float mf[8], vf[8];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            mf[4 * k] = __builtin_amdgcn_cvt_f32_fp8(mc[k], 0);
            mf[4 * k + 1] = __builtin_amdgcn_cvt_f32_fp8(mc[k], 1);
            mf[4 * k + 2] = __builtin_amdgcn_cvt_f32_fp8(mc[k], 2);
            mf[4 * k + 3] = __builtin_amdgcn_cvt_f32_fp8(mc[k], 3);
            vf[4 * k] = __builtin_amdgcn_cvt_f32_fp8(vc[k], 0);
            vf[4 * k + 1] = __builtin_amdgcn_cvt_f32_fp8(vc[k], 1);
            vf[4 * k + 2] = __builtin_amdgcn_cvt_f32_fp8(vc[k], 2);
            vf[4 * k + 3] = __builtin_amdgcn_cvt_f32_fp8(vc[k], 3);
        }
        double m[8], v[8], mm = 0.0, vm = 0.0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const double gd = (double)g[k] * st.coef;
            m[k] = fma(ms, (double)mf[k], c1 * gd);
            v[k] = fma(vs, (double)vf[k], c2 * (gd * gd));
            const double am = fabs(m[k]);
            mm = (am > mm || am != am) ? am : mm;
            vm = (v[k] > vm || v[k] != v[k]) ? v[k] : vm;
            const float q = ((float)m[k] * inv_bc1) / (sqrtf((float)v[k] * inv_bc2) + eps);
            pv[k] = fmaf(-lr, fmaf(decay, pv[k], q), pv[k]);
        }
        if (n == 8) {
#pragma unroll
            for (int k = 0; k < 8; k += 4) *(f32x4_u*)(p + i + k) = f32x4{pv[k], pv[k + 1], pv[k + 2], pv[k + 3]};
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < n) p[i + k] = pv[k];
        }
        const float new_ms = (float)(max16(mm) / 448.0), new_vs = (float)(max16(vm) / 448.0);
        const double im = new_ms > 0.f || new_ms != new_ms ? 1.0 / (double)new_ms : 0.0,
                     iv = new_vs > 0.f || new_vs != new_vs ? 1.0 / (double)new_vs : 0.0;
        const unsigned pair = (unsigned)((unsigned long long)(c.state_at + i) >> 1);
        u32x2 mo, vo;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float y[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                y[q] = (float)(m[4 * k + q] * im);
                y[q] = y[q] > 448.f ? 448.f : (y[q] < -448.f ? -448.f : y[q]);      // keeps a NaN
            }
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
            mo[k] = (unsigned)w;
            unsigned b = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const unsigned h = mix((pair + 2 * k + q / 2) ^ key);
                const double x = v[4 * k + q];
                const float z = (float)(x * iv);
                unsigned code = round_random(z, (q & 1) ? h >> 16 : h & 0xFFFFu);
                code = code == 0 && x > 0.0 && new_vs > 0.f ? 1u : code;
                if (z != z) code = 0x7Fu;
                b |= code << (8 * q);
            }
            vo[k] = b;
        }
        *(u32x2*)(m8 + i) = mo;
        *(u32x2*)(v8 + i) = vo;
        if ((threadIdx.x & 15) == 0) {
            a.m_scale[block] = new_ms;
            a.v_scale[block] = new_vs;
        }
    }
    step_done(a, st.t);
}

}  // namespace

hipError_t adamw_set_pointers_launch(const AdamwPtrs& p, const void** dst, int n, hipStream_t st) {
    hipLaunchKernelGGL(set_pointers_kernel, dim3(1), dim3(ADAMW_PTRS), 0, st, p, dst, n);
    return hipGetLastError();
}

hipError_t adamw_norm_launch(const AdamwArgs& a, double* partials, hipStream_t st) {
    hipLaunchKernelGGL(norm_kernel, dim3((unsigned)a.num_partials), dim3(NT), 0, st, a, partials);
    return hipGetLastError();
}

hipError_t adamw_step_launch(const AdamwArgs& a, int state_bits, hipStream_t st) {
    if (state_bits == 8)
        hipLaunchKernelGGL(adamw8_kernel, dim3((unsigned)a.num_chunks), dim3(NT), 0, st, a);
    else
        hipLaunchKernelGGL(adamw32_kernel, dim3((unsigned)a.num_chunks), dim3(NT), 0, st, a);
    return hipGetLastError();
}

}  // namespace rst
