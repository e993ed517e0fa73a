// adamw.hip — the AdamW step over many tensors in one launch, states in 32 or in 8 bits, global-norm clipping.
//
// Step t, gradient g, c = min(1, clip / |g|) over all variables:
//   m = b1 m + (1 - b1) c g,  v = b2 v + (1 - b2) (c g)^2
//   p -= lr (m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps) + decay p)
// One pass over the data: every element's g, p, m, v are read once and p, m, v written once (28 bytes in 32 bits, 16.1
// with 8-bit states), which is all that bounds it. A workgroup takes one chunk of at most 4096 elements of one variable
// from a table made once, so a step over hundreds of small variables is one launch. The step count is on the device
// (a captured step replays as the next one): every workgroup reads t, and the last one to have read it writes t + 1.
//
// 8-bit states: blocks of 128 elements of one variable with a scale s = max / 448 each, codes in e4m3. m / s rounds to
// nearest. v / s is rounded up or down at random with the right mean: (1 - b2) of a change is far below half a code, so
// that rounding to nearest would leave v where it is for ever. The random bits are a hash of (element, step, seed), so
// a step is reproducible. A v above zero keeps a code above zero: its root divides. Moments, scales and codes are
// formed in 64 bits, which issue at the f32 rate here, so that a code does not depend on the order of operations. The
// variable's step itself is in 32 bits, about 10 units of 2^-24 of it: learning_rate times that is far below the rounding of
// the variable.
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

// (pointers out of a table are generic: say that they are global)
template <typename T>
using Global = T __attribute__((address_space(1)))*;

// PAST: past the caches, for a step whose data does not stay in them
template <bool PAST, typename T>
__device__ __forceinline__ T load(const void* p, long long i) {
    const Global<const T> g = (Global<const T>)((const char*)p + i);
    if constexpr (PAST) return __builtin_nontemporal_load(g);
    else return *g;
}
template <bool PAST, typename T>
__device__ __forceinline__ void store(void* p, long long i, T v) {
    const Global<T> g = (Global<T>)((char*)p + i);
    if constexpr (PAST) __builtin_nontemporal_store(v, g);
    else *g = v;
}

template <bool BF16, bool PAST>
__device__ __forceinline__ f32x4 load_grad4(const void* g, long long i) {
    if constexpr (BF16) {
        const u16x4 v = load<PAST, u16x4_u>(g, 2 * i);
        return f32x4{widen(v.x), widen(v.y), widen(v.z), widen(v.w)};
    }
    return load<PAST, f32x4_u>(g, 4 * i);
}
template <bool BF16>
__device__ __forceinline__ float load_grad(const void* g, long long i) {
    if constexpr (BF16) return widen(load<false, unsigned short>(g, 2 * i));
    return load<false, float>(g, 4 * i);
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

// Sums of squares over the chunks blockIdx, blockIdx + grid, ...: one partial per workgroup, merged by the step. 192 MB in
// 32 us (6.0 TB/s: reading bound), 11 MB in 4.6
template <bool BF16>
__global__ __launch_bounds__(NT) void norm_kernel(AdamwArgs a, double* partials) {
    __shared__ double red[4];
    constexpr int R = ADAMW_CHUNK / (4 * NT);
    double s = 0.0;
    for (int k = blockIdx.x; k < a.num_chunks; k += gridDim.x) {
        const AdamwChunk c = a.chunks[k];
        long long at;
        const void* g = grad_of(a, c, at);
        const int i0 = threadIdx.x * 4;
        const int vectors = c.count / 4, tail = vectors * 4 + threadIdx.x;
        if (vectors > 0) {
            f32x4 v[R];
#pragma unroll
            for (int r = 0; r < R; ++r) v[r] = load_grad4<BF16, false>(g, at + (i0 / 4 + r * NT < vectors ? i0 + r * 4 * NT : 0));
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (i0 / 4 + r * NT < vectors)
#pragma unroll
                    for (int q = 0; q < 4; ++q) s = fma((double)v[r][q], (double)v[r][q], s);
        }
        if (tail < c.count) {
            const double v = load_grad<BF16>(g, at + tail);
            s = fma(v, v, s);
        }
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// Whether this is the last of n to count; the counter is then zero again for the next step
__device__ __forceinline__ bool last_of(unsigned* ticket, unsigned n) {
    const bool last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
    if (last) *ticket = 0;
    return last;
}

// What the whole step shares: the clipping factor, the step number and its corrections; `last`: this workgroup is the
// last one to have read the step count and moves it on at its end. False: nothing to do, the gradient's norm is not
// finite. Called with the chunk's loads under way.
struct StepScalars {
    double coef;
    float inv_bc1, inv_bc2;
    long long t;
    bool last;
};
__device__ __forceinline__ bool step_scalars(const AdamwArgs& a, StepScalars& s, double* red) {
    s.t = *a.iterations + 1;
    // 1 - beta^t: f32 is enough for the relative size of a step (the argument in 64 bits: t may be large)
    s.inv_bc1 = -1.f / expm1f((float)((double)s.t * a.log_b1));
    s.inv_bc2 = -1.f / expm1f((float)((double)s.t * a.log_b2));
    s.coef = 1.0;
    if (a.num_partials > 0) {
        double q = 0.0;
#pragma unroll
        for (int i = 0; i < ADAMW_MAX_PARTIALS / NT; ++i) {
            const int k = i * NT + threadIdx.x;
            const double v = a.partials[min(k, a.num_partials - 1)];
            q += k < a.num_partials ? v : 0.0;
        }
        const double norm = sqrt(block_sum(q, red));
        if (blockIdx.x == 0 && threadIdx.x == 0 && a.global_norm != nullptr) *a.global_norm = (float)norm;
        if (!(norm < __builtin_inf())) return false;
        if (norm > a.clip) s.coef = a.clip / norm;
    }
    __syncthreads();             // every wave has read the count
    s.last = threadIdx.x == 0 && last_of(a.tickets + (1 + blockIdx.x / ADAMW_TICKETS) * ADAMW_TICKET_STRIDE,
                                         min((unsigned)ADAMW_TICKETS, (unsigned)a.num_chunks - blockIdx.x / ADAMW_TICKETS * ADAMW_TICKETS));
    return true;
}

// Workgroups count in groups of 64, and the last of each group at the root: with 872 workgroups at one address the step
// took 18.2 us (8-bit states 21.4), like this 13.9 (16.0)
__device__ __forceinline__ void step_done(const AdamwArgs& a, const StepScalars& s) {
    if (s.last && last_of(a.tickets, (a.num_chunks + ADAMW_TICKETS - 1) / ADAMW_TICKETS)) *a.iterations = s.t;
}

// m / bc1 / (sqrt(v / bc2) + eps) through the hardware's root and reciprocal, one unit in the last place each
__device__ __forceinline__ float quotient(float m, float v, float inv_bc1, float inv_bc2, float eps) {
    return m * inv_bc1 * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v * inv_bc2) + eps);
}

// These two take a subnormal for 0, and v / bc2 can pass f32 (v too, in 64 bits), as 1 / bc2 goes to 2^53. Up to this v there
// is no overflow; from this eps on a root below 2^-63, which was taken for 0, is less than a rounding of the sum
constexpr float PLAIN_V = 0x1p64f, PLAIN_EPS = 0x1p-39f;

// The same for every v: a large one goes by 2^-184 and the quotient's two terms by 2^-92 (what that flushes is below 2^-72 of the
// other one), a small one by 2^170 and its root by 2^-85: f32's normal numbers for 2^-296 <= v < 2^257, and below that a
// root that no eps sees. In place of the plain form for every element the step took 2.5 % more (2.7 M elements 17.6 us,
// so 18.1; 8-bit states 48 M 181 and 185.6)
template <typename D>
__device__ __forceinline__ float any_quotient(float m, D v, float inv_bc1, float inv_bc2, float eps) {
    const bool large = v > (D)PLAIN_V, small = v < (D)0x1p-100;
    const float x = (float)ldexp(v, large ? -184 : (small ? 170 : 0)) * inv_bc2;
    const float root = ldexp(__builtin_amdgcn_sqrtf(x), small ? -85 : 0);
    const int down = large ? -92 : 0;
    return ldexp(m * inv_bc1, down) * __builtin_amdgcn_rcpf(root + ldexp(eps, down));
}

struct Scalars32 {
    float b1, c1, b2, c2, inv_bc1, inv_bc2, eps, lr, decay, coef;
};

// N elements' step
template <int N>
__device__ __forceinline__ void adamw_elements(const float (&g)[N], float (&p)[N], float (&m)[N], float (&v)[N], const Scalars32& s) {
    float q[N], most = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float x = g[k] * s.coef;
        m[k] = fmaf(s.b1, m[k], s.c1 * x);
        v[k] = fmaf(s.b2, v[k], s.c2 * x * x);       // (x * x alone would pass f32 from 1.8e19 on)
        most = __builtin_fmaxf(most, v[k]);
        q[k] = quotient(m[k], v[k], s.inv_bc1, s.inv_bc2, s.eps);
    }
    if (__builtin_expect(most > PLAIN_V || s.eps < PLAIN_EPS, 0)) {
#pragma unroll
        for (int k = 0; k < N; ++k) q[k] = any_quotient(m[k], v[k], s.inv_bc1, s.inv_bc2, s.eps);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) p[k] = fmaf(-s.lr, fmaf(s.decay, p[k], q[k]), p[k]);
}

// Bound by memory: 48 M elements with bf16 gradients, 1.25 GB, in 216 us (5.8 TB/s; torch's copy of 1 GiB 5.1), 2.7 M
// elements in 13.7 (their 76 MB stay in the Infinity Cache). Every load of a thread comes before the first use, the step's
// scalars in between
template <bool BF16, bool PAST>
__global__ __launch_bounds__(NT) void adamw32_kernel(AdamwArgs a) {
    __shared__ double red[4];
    constexpr int R = ADAMW_CHUNK / (4 * NT);
    const AdamwChunk c = a.chunks[blockIdx.x];
    long long at;
    const void* g = grad_of(a, c, at);
    float* p = c.param;
    float* m = (float*)a.m + c.state_at;
    float* v = (float*)a.v + c.state_at;
    const int i0 = threadIdx.x * 4;
    const bool full = c.count == ADAMW_CHUNK;
    // whole vectors first, then one element for each of the first count % 4 threads. Loads are unconditional (a guarded
    // one would be waited for by itself): where there is no vector, the variable's first elements again
    const int vectors = c.count / 4, rest = c.count % 4, tail = vectors * 4 + threadIdx.x;
    f32x4 gv[R], pv[R], mv[R], vv[R];
    float gt = 0.f, pt = 0.f, mt = 0.f, vt = 0.f;
    if (vectors > 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r * NT >= vectors) break;
            const int i = full || i0 / 4 + r * NT < vectors ? i0 + r * 4 * NT : 0;
            gv[r] = load_grad4<BF16, PAST>(g, at + i);
            pv[r] = load<PAST, f32x4_u>(p, 4ll * i);
            mv[r] = load<PAST, f32x4_u>(m, 4ll * i);
            vv[r] = load<PAST, f32x4_u>(v, 4ll * i);
        }
    }
    if ((int)threadIdx.x < rest) {
        gt = load_grad<BF16>(g, at + tail);
        pt = load<false, float>(p, 4ll * tail);
        mt = load<false, float>(m, 4ll * tail);
        vt = load<false, float>(v, 4ll * tail);
    }
    __builtin_amdgcn_sched_barrier(0);
    StepScalars st;
    const bool go = step_scalars(a, st, red);
    if (!go) return;
    const Scalars32 s{(float)a.b1, (float)(1.0 - a.b1), (float)a.b2, (float)(1.0 - a.b2), st.inv_bc1, st.inv_bc2,
                      (float)a.eps, (float)a.lr, c.decay ? (float)a.decay : 0.f, (float)st.coef};
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (!(full || i0 / 4 + r * NT < vectors)) break;
        const int i = i0 + r * 4 * NT;
        float g4[4], p4[4], m4[4], v4[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            g4[k] = gv[r][k];
            p4[k] = pv[r][k];
            m4[k] = mv[r][k];
            v4[k] = vv[r][k];
        }
        adamw_elements<4>(g4, p4, m4, v4, s);
        store<PAST, f32x4_u>(p, 4ll * i, f32x4{p4[0], p4[1], p4[2], p4[3]});
        store<PAST, f32x4_u>(m, 4ll * i, f32x4{m4[0], m4[1], m4[2], m4[3]});
        store<PAST, f32x4_u>(v, 4ll * i, f32x4{v4[0], v4[1], v4[2], v4[3]});
    }
    if ((int)threadIdx.x < rest) {
        const float g1[1] = {gt};
        float p1[1] = {pt}, m1[1] = {mt}, v1[1] = {vt};
        adamw_elements<1>(g1, p1, m1, v1, s);
        store<false, float>(p, 4ll * tail, p1[0]);
        store<false, float>(m, 4ll * tail, m1[0]);
        store<false, float>(v, 4ll * tail, v1[0]);
    }
    step_done(a, st);
}

// ---- 8-bit states --------------------------------------------------------------------------------------------------

// Two rounds of xor-shift and multiply, a bijection of 32 bits whose outputs look random: the published integer hash lowbias32
__device__ __forceinline__ unsigned mix(unsigned x) {
    x = (x ^ (x >> 16)) * 0x7FEB352Du;
    x = (x ^ (x >> 15)) * 0x846CA68Bu;
    return x ^ (x >> 16);
}

// y in [0, 448] to an e4m3 code, up with the probability of its place between two codes (u: 16 random bits). An f32 has
// 20 bits below e4m3's three; below 2^-6 codes are 2^-9 apart. A NaN gives the NaN code.
__device__ __forceinline__ unsigned round_random(float y, unsigned u) {
    const unsigned bits = y < 0.015625f ? (unsigned)(y * 536870912.f) : __float_as_uint(y) - ((127u - 7u) << 23);
    return min((bits + (u << 4)) >> 20, 0x7Fu);
}

// Over the 16 lanes of a block, by permutations within the row of lanes
template <int CTRL>
__device__ __forceinline__ double max_dpp(double v) {
    const long long b = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)(b & 0xFFFFFFFFll), CTRL, 0xF, 0xF, true);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_fmax(v, __longlong_as_double(((long long)hi << 32) | (unsigned)lo));
}
__device__ __forceinline__ double max16(double v) {
    return max_dpp<0x140>(max_dpp<0x141>(max_dpp<0x4E>(max_dpp<0xB1>(v))));   // lanes xor 1, xor 2, the half mirrored, the row
}

// A block's scale from its largest value. One that would be subnormal is 0: the block counts as zeros
constexpr double LARGEST = 448.0 * 3.4028234663852886e38;
__device__ __forceinline__ float scale_of(double largest) {
    const float s = (float)(largest * (1.0 / 448.0));
    return s < 1.17549435e-38f ? 0.f : s;
}
// 1 / s in 64 bits (one Newton step on the hardware's reciprocal: about one unit in the last place), 0 of 0
__device__ __forceinline__ double inverse(float s) {
    const double d = (double)s;
    const double r = __builtin_amdgcn_rcp(d);
    return s == 0.f ? 0.0 : fma(fma(-d, r, 1.0), r, r);
}

// One lane's eight elements: gradient, variable, codes, the block's scales
struct Eight {
    float g[8], p[8];
    u32x2 m, v;
    float ms, vs;
};

// Loads eight elements from element i of the chunk on; n of them are the variable's (the others: zeros)
template <bool BF16, bool PAST, bool FULL>
__device__ __forceinline__ void load8(Eight& e, const AdamwArgs& a, const AdamwChunk& c, const void* g, long long at, int i, int n) {
    if constexpr (FULL) {
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
            const f32x4 x = load_grad4<BF16, PAST>(g, at + i + k), y = load<PAST, f32x4_u>(c.param, 4ll * (i + k));
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                e.g[k + q] = x[q];
                e.p[k + q] = y[q];
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {        // (unconditional loads, of the variable's last element beyond it)
            const int q = min(i + k, c.count - 1);
            e.g[k] = load_grad<BF16>(g, at + q);
            e.p[k] = load<false, float>(c.param, 4ll * q);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k >= n) e.g[k] = 0.f;
    }
    e.m = load<PAST, u32x2>(a.m, c.state_at + i);
    e.v = load<PAST, u32x2>(a.v, c.state_at + i);
    const long long block = (c.state_at + i) / ADAMW_BLOCK;
    e.ms = a.m_scale[block];
    e.vs = a.v_scale[block];
}

struct Scalars8 {
    double b1, c1, b2, c2;        // c1, c2 with the clipping factor and its square
    float inv_bc1, inv_bc2, eps, lr, decay;
    unsigned key;
};

// Their step: 16 lanes are a block
template <bool PAST>
__device__ __forceinline__ void step8(Eight& e, const AdamwArgs& a, const AdamwChunk& c, int i, int n, const Scalars8& s) {
    float mf[8], vf[8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        mf[4 * k] = __builtin_amdgcn_cvt_f32_fp8(e.m[k], 0);
        mf[4 * k + 1] = __builtin_amdgcn_cvt_f32_fp8(e.m[k], 1);
        mf[4 * k + 2] = __builtin_amdgcn_cvt_f32_fp8(e.m[k], 2);
        mf[4 * k + 3] = __builtin_amdgcn_cvt_f32_fp8(e.m[k], 3);
        vf[4 * k] = __builtin_amdgcn_cvt_f32_fp8(e.v[k], 0);
        vf[4 * k + 1] = __builtin_amdgcn_cvt_f32_fp8(e.v[k], 1);
        vf[4 * k + 2] = __builtin_amdgcn_cvt_f32_fp8(e.v[k], 2);
        vf[4 * k + 3] = __builtin_amdgcn_cvt_f32_fp8(e.v[k], 3);
    }
    const double ms = s.b1 * (double)e.ms, vs = s.b2 * (double)e.vs;
    double m[8], v[8], mm = 0.0, vm = 0.0;
    float q[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const double gd = (double)e.g[k];
        m[k] = fma(ms, (double)mf[k], s.c1 * gd);
        v[k] = fma(vs, (double)vf[k], s.c2 * (gd * gd));
        mm = __builtin_fmax(mm, fabs(m[k]));      // (leaves a NaN out: it stays with its element)
        vm = __builtin_fmax(vm, v[k]);
        q[k] = quotient((float)m[k], (float)v[k], s.inv_bc1, s.inv_bc2, s.eps);
    }
    if (__builtin_expect(vm > (double)PLAIN_V || s.eps < PLAIN_EPS, 0)) {
#pragma unroll
        for (int k = 0; k < 8; ++k) q[k] = any_quotient((float)m[k], v[k], s.inv_bc1, s.inv_bc2, s.eps);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) e.p[k] = fmaf(-s.lr, fmaf(s.decay, e.p[k], q[k]), e.p[k]);
    if (n >= 8) {
#pragma unroll
        for (int k = 0; k < 8; k += 4)
            store<PAST, f32x4_u>(c.param, 4ll * (i + k), f32x4{e.p[k], e.p[k + 1], e.p[k + 2], e.p[k + 3]});
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < n) store<false, float>(c.param, 4ll * (i + k), e.p[k]);
    }
    float new_ms = scale_of(max16(mm)), new_vs = scale_of(max16(vm));
    if (!(new_ms < __builtin_inff() && new_vs < __builtin_inff())) {
        // beyond f32's range: an infinity is left out of its block's scale and becomes a NaN code, a finite v saturates
        mm = vm = 0.0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (v[k] < __builtin_inf()) v[k] = __builtin_fmin(v[k], LARGEST);
            mm = __builtin_fmax(mm, fabs(m[k]) < __builtin_inf() ? fabs(m[k]) : 0.0);
            vm = __builtin_fmax(vm, v[k] < __builtin_inf() ? v[k] : 0.0);
        }
        new_ms = scale_of(max16(mm));
        new_vs = scale_of(max16(vm));
    }
    const double im = inverse(new_ms), iv = inverse(new_vs);
    const unsigned least = new_vs > 0.f ? 1u : 0u, pair = (unsigned)((unsigned long long)(c.state_at + i) >> 1);
    u32x2 mo, vo;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        // (a finite |m / s| is at most 448 and a rounding: no clamp)
        int w = __builtin_amdgcn_cvt_pk_fp8_f32((float)(m[4 * k] * im), (float)(m[4 * k + 1] * im), 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32((float)(m[4 * k + 2] * im), (float)(m[4 * k + 3] * im), w, true);
        mo[k] = (unsigned)w;
        unsigned b = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const unsigned h = mix((pair + 2 * k + q / 2) ^ s.key);
            const double x = v[4 * k + q];
            b |= max(round_random((float)(x * iv), (q & 1) ? h >> 16 : h & 0xFFFFu), x > 0.0 ? least : 0u) << (8 * q);
        }
        vo[k] = b;
    }
    store<PAST, u32x2>(a.m, c.state_at + i, mo);
    store<PAST, u32x2>(a.v, c.state_at + i, vo);
    if ((threadIdx.x & 15) == 0) {
        const long long block = (c.state_at + i) / ADAMW_BLOCK;
        a.m_scale[block] = new_ms;
        a.v_scale[block] = new_vs;
    }
}

// Eight elements per lane and round: a chunk is at most two rounds. Bound by memory with about 50 instructions an element
// beside it: 48 M elements, 774 MB, in 147 to 158 us (from card to card; 4.9 to 5.3 TB/s); 61 k elements in 4.8, latency; 2.7 M in 13.1,
// with clipping 14.5: each of its 1537 workgroups then merges the norm's partial sums by itself, 8 KB, before its first
// element. (Three waves per SIMD: at four the registers spill, 12 M elements 51 us for 48)
template <bool BF16, bool PAST>
__global__ __launch_bounds__(NT, 3) void adamw8_kernel(AdamwArgs a) {
    __shared__ double red[4];
    constexpr int R = ADAMW_CHUNK / (8 * NT);
    const AdamwChunk c = a.chunks[blockIdx.x];
    long long at;
    const void* g = grad_of(a, c, at);
    const int i0 = threadIdx.x * 8;
    const int filled = (c.count + ADAMW_BLOCK - 1) / ADAMW_BLOCK * ADAMW_BLOCK;      // with the last block's zeros
    Eight e[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = i0 + r * 8 * NT;
        if (i + 8 <= c.count) load8<BF16, PAST, true>(e[r], a, c, g, at, i, 8);
        else if (i < filled) load8<BF16, PAST, false>(e[r], a, c, g, at, i, c.count - i);
    }
    __builtin_amdgcn_sched_barrier(0);
    StepScalars st;
    const bool go = step_scalars(a, st, red);
    if (!go) return;
    const Scalars8 s{a.b1, (1.0 - a.b1) * st.coef, a.b2, (1.0 - a.b2) * st.coef * st.coef, st.inv_bc1, st.inv_bc2,
                     (float)a.eps, (float)a.lr, c.decay ? (float)a.decay : 0.f, mix(a.seed + (unsigned)st.t * 0x9E3779B9u)};
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = i0 + r * 8 * NT;
        if (i < filled) step8<PAST>(e[r], a, c, i, c.count - i, s);
        __builtin_amdgcn_sched_barrier(0);      // one after the other: together they take 154 registers
    }
    step_done(a, st);
}

}  // namespace

hipError_t adamw_set_pointers_launch(const AdamwPtrs& p, const void** dst, int n, hipStream_t st) {
    hipLaunchKernelGGL(set_pointers_kernel, dim3(1), dim3(ADAMW_PTRS), 0, st, p, dst, n);
    return hipGetLastError();
}

hipError_t adamw_norm_launch(const AdamwArgs& a, double* partials, hipStream_t st) {
    if (a.grad_bf16)
        hipLaunchKernelGGL(norm_kernel<true>, dim3((unsigned)a.num_partials), dim3(NT), 0, st, a, partials);
    else
        hipLaunchKernelGGL(norm_kernel<false>, dim3((unsigned)a.num_partials), dim3(NT), 0, st, a, partials);
    return hipGetLastError();
}

hipError_t adamw_step_launch(const AdamwArgs& a, int state_bits, bool past, hipStream_t st) {
    const dim3 grid((unsigned)a.num_chunks), block(NT);
#define ADAMW(K)                                                                                 \
    if (a.grad_bf16 && past) hipLaunchKernelGGL((K<true, true>), grid, block, 0, st, a);         \
    else if (a.grad_bf16) hipLaunchKernelGGL((K<true, false>), grid, block, 0, st, a);           \
    else if (past) hipLaunchKernelGGL((K<false, true>), grid, block, 0, st, a);                  \
    else hipLaunchKernelGGL((K<false, false>), grid, block, 0, st, a);
    if (state_bits == 8) {
        ADAMW(adamw8_kernel)
    } else {
        ADAMW(adamw32_kernel)
    }
#undef ADAMW
    return hipGetLastError();
}

}  // namespace rst
