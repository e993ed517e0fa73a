// group_norm.hip — group normalisation with an activation over channels-last tensors, forward and backward.
//
// x (B, hw, C), G groups of Cg = C / G channels; per image b and group g
//   mean, var = moments over hw * Cg values (biased), rstd = 1 / sqrt(var + eps)
//   y = act(z), z = scale_c (x - mean) rstd + bias_c = a_c x + c_c,  a = scale rstd, c = bias - mean a
// and with dz = dy act'(z), h = (x - mean) rstd, n = hw * Cg
//   dbias_c = sum dz, dscale_c = sum dz h
//   dx = rstd (scale dz - S1 / n - h S2 / n),  S1 = sum_g scale dz, S2 = sum_g scale dz h
//
// Channels last puts a group's values Cg at a time into every pixel, so a workgroup takes a range of pixels with all
// their channels (up to 256 vectors of them: a channel block) and reduces every group it meets: loads are whole lines.
// A launch per pass over the data, and the partial sums of the workgroups are merged in a fixed order (no atomics: the
// same inputs give the same bits).
//
// Arithmetic: the moments are sums of x and x^2 in 64 bits: f64 adds and FMAs issue at the rate of the scalar f32 ones
// on this chip, and E[x^2] - mean^2 then loses log2(mean^2 / var) of 53 bits, not of 24. z = a x + c is one f64 FMA for
// the same reason (c ~ mean / std large), which also settles on which side of act's kinks z lies.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/rst.h"
#include "group_norm.h"

namespace rst {
namespace {

constexpr int NT = 256;

typedef unsigned short bf16_t;
template <typename T, int V>
using Pack = T __attribute__((ext_vector_type(V)));

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(bf16_t v) { return __uint_as_float((unsigned)v << 16); }
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16_t narrow<bf16_t>(float v) { return __builtin_bit_cast(bf16_t, (__bf16)v); }

// One launch's split of the tensor. A vector is V channels; a channel block nvb <= 256 vectors, its workgroup `rows`
// pixels high; a tile tile_px pixels. slots: the channel blocks that one group can meet.
struct Geom {
    long hw, tile_px;
    int B, C, G, Cg;
    int nv, nvb, CB, rows, tiles, slots;
    double inv_n;
};

// About 1024 workgroups (four of 256 threads per CU), four pixels at least and 64 at most per thread: the backward
// sums a thread's pixels in f32.
constexpr int TARGET_WGS = 1024;

Geom geometry(int B, long hw, int C, int G, int V) {
    Geom g{};
    g.hw = hw;
    g.B = B;
    g.C = C;
    g.G = G;
    g.Cg = C / G;
    g.nv = C / V;
    g.CB = (g.nv + NT - 1) / NT;
    g.nvb = (g.nv + g.CB - 1) / g.CB;
    g.CB = (g.nv + g.nvb - 1) / g.nvb;
    g.rows = NT / g.nvb;
    const long per = std::max(1L, (long)TARGET_WGS / ((long)B * g.CB));
    long px = (hw + per - 1) / per;
    px = std::min(std::max(px, 4L * g.rows), 64L * g.rows);
    g.tile_px = px;
    g.tiles = (int)((hw + px - 1) / px);
    g.slots = std::min(g.CB, (g.Cg - 1) / (g.nvb * V) + 2);
    g.inv_n = 1.0 / ((double)hw * g.Cg);
    return g;
}

struct Place {
    int b, cb, tile, lane, row, vec;
    bool active;
    long p0, p1;
};

__device__ __forceinline__ Place place(const Geom& g) {
    Place w;
    const int per = g.CB * g.tiles;
    w.b = blockIdx.x / per;
    const int r = blockIdx.x - w.b * per;
    w.cb = r / g.tiles;
    w.tile = r - w.cb * g.tiles;
    w.row = threadIdx.x / g.nvb;
    w.lane = threadIdx.x - w.row * g.nvb;
    w.vec = w.cb * g.nvb + w.lane;
    w.active = w.row < g.rows && w.vec < g.nv;
    w.p0 = (long)w.tile * g.tile_px;
    w.p1 = min(g.hw, w.p0 + g.tile_px);
    return w;
}

// body(U packs, count) over the thread's pixels, U loads in flight
template <int U, typename P, typename F>
__device__ __forceinline__ void each_pixel(const P* __restrict__ x, const Geom& g, const Place& w, F&& body) {
    const P* base = x + ((size_t)w.b * g.hw) * g.nv + w.vec;
    long p = w.p0 + w.row;
    for (; p + (long)(U - 1) * g.rows < w.p1; p += (long)U * g.rows) {
        P v[U];
#pragma unroll
        for (int k = 0; k < U; ++k) v[k] = base[(size_t)(p + (long)k * g.rows) * g.nv];
#pragma unroll
        for (int k = 0; k < U; ++k) body(v[k], p + (long)k * g.rows);
    }
    for (; p < w.p1; p += g.rows) body(base[(size_t)p * g.nv], p);
}

// The groups [g0, g1] that a channel block meets, and threads per group for their sums
struct Groups {
    int c0, c1, g0, ng, tpg;
};
template <int V>
__device__ __forceinline__ Groups groups_of(const Geom& g, int cb) {
    Groups r;
    r.c0 = cb * g.nvb * V;
    r.c1 = min(g.C, r.c0 + g.nvb * V);
    r.g0 = r.c0 / g.Cg;
    r.ng = (r.c1 - 1) / g.Cg - r.g0 + 1;
    r.tpg = r.ng >= NT ? 1 : min(64, 1 << (31 - __clz(NT / r.ng)));
    return r;
}

// Where group gi's partials of the channel blocks start: [b][g][slot][tile]
__device__ __forceinline__ size_t part_index(const Geom& g, int b, int group) {
    return ((size_t)b * g.G + group) * g.slots * g.tiles;
}

// Pass 1: sums of x and x^2 of every (image, group) over a tile. UNI: a vector lies in one group (Cg % V == 0).
template <typename T, int V, bool UNI>
__global__ __launch_bounds__(NT) void gn_stats_kernel(const void* __restrict__ x, double2* __restrict__ part, Geom g) {
    constexpr int E = UNI ? 1 : V;
    __shared__ double2 red[NT * E];
    const Place w = place(g);
    if (w.active) {
        double s[E], q[E];
#pragma unroll
        for (int k = 0; k < E; ++k) s[k] = q[k] = 0.0;
        each_pixel<4>((const Pack<T, V>*)x, g, w, [&](const Pack<T, V>& v, long) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const double d = (double)widen((T)v[k]);
                s[UNI ? 0 : k] += d;
                q[UNI ? 0 : k] = fma(d, d, q[UNI ? 0 : k]);
            }
        });
#pragma unroll
        for (int k = 0; k < E; ++k) red[threadIdx.x * E + k] = make_double2(s[k], q[k]);
    }
    __syncthreads();
    const Groups r = groups_of<V>(g, w.cb);
    const int j = threadIdx.x % r.tpg;
    for (int gi = threadIdx.x / r.tpg; gi < r.ng; gi += NT / r.tpg) {
        const int group = r.g0 + gi;
        const int lo = (max(r.c0, group * g.Cg) - r.c0) / (V / E), hi = (min(r.c1, (group + 1) * g.Cg) - r.c0) / (V / E);
        const int width = hi - lo;
        double s = 0.0, q = 0.0;
        for (int e = j; e < width * g.rows; e += r.tpg) {
            const int row = e / width;
            const double2 v = red[row * g.nvb * E + lo + (e - row * width)];
            s += v.x;
            q += v.y;
        }
        for (int o = r.tpg / 2; o > 0; o >>= 1) {
            s += __shfl_xor(s, o);
            q += __shfl_xor(q, o);
        }
        if (j == 0) {
            const int slot = w.cb - (group * g.Cg) / (g.nvb * V);
            part[part_index(g, w.b, group) + (size_t)slot * g.tiles + w.tile] = make_double2(s, q);
        }
    }
}

// One wave per (image, group): merge its partials into mean and rstd
__global__ __launch_bounds__(NT) void gn_finalize_kernel(const double2* __restrict__ part, double2* __restrict__ stat,
                                                         float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                         Geom g, int block_channels, float eps) {
    const long bg = (long)blockIdx.x * (NT / 64) + threadIdx.x / 64;
    if (bg >= (long)g.B * g.G) return;
    const int lane = threadIdx.x & 63, group = (int)(bg % g.G);
    const int used = ((group + 1) * g.Cg - 1) / block_channels - (group * g.Cg) / block_channels + 1;
    const double2* p = part + (size_t)bg * g.slots * g.tiles;
    double s = 0.0, q = 0.0;
#pragma unroll 4
    for (int i = lane; i < used * g.tiles; i += 64) {
        const double2 v = p[i];
        s += v.x;
        q += v.y;
    }
    for (int o = 32; o > 0; o >>= 1) {
        s += __shfl_xor(s, o);
        q += __shfl_xor(q, o);
    }
    if (lane == 0) {
        const double mean = s * g.inv_n;
        double var = q * g.inv_n - mean * mean;
        var = var < 0.0 ? 0.0 : var;          // keeps a NaN
        const double rstd = 1.0 / sqrt(var + (double)eps);
        stat[bg] = make_double2(mean, rstd);
        if (mean_out != nullptr) mean_out[bg] = (float)mean;
        if (rstd_out != nullptr) rstd_out[bg] = (float)rstd;
    }
}

// exp through the hardware's 2^x and 1/x: about 2 units in the last place
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == RST_ACT_RELU) return z < 0.f ? 0.f : z;             // keeps a NaN
    if constexpr (ACT == RST_ACT_SWISH) return z * sigmoid(z);
    if constexpr (ACT == RST_ACT_HARD_SWISH) return z <= -3.f ? 0.f : (z >= 3.f ? z : z * (z + 3.f) * (1.f / 6.f));
    return z;
}

template <int ACT>
__device__ __forceinline__ float act_slope(double z) {
    if constexpr (ACT == RST_ACT_RELU) return z > 0.0 ? 1.f : 0.f;
    if constexpr (ACT == RST_ACT_SWISH) {
        const float f = (float)z, s = sigmoid(f);
        return s * (1.f + f * (1.f - s));
    }
    if constexpr (ACT == RST_ACT_HARD_SWISH)
        return z >= 3.0 ? 1.f : (z > -3.0 ? ((float)z + 1.5f) * (1.f / 3.f) : 0.f);
    return 1.f;
}

// Pass 2: y = act(a x + c)
template <typename T, int V, int ACT>
__global__ __launch_bounds__(NT) void gn_apply_kernel(GroupNormArgs a, const double2* __restrict__ stat, Geom g) {
    const Place w = place(g);
    if (!w.active) return;
    double ka[V], kc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int c = w.vec * V + k;
        const double2 st = stat[(size_t)w.b * g.G + c / g.Cg];
        ka[k] = (double)a.scale[w.b * a.aff_stride + c] * st.y;
        kc[k] = fma(-st.x, ka[k], (double)a.bias[w.b * a.aff_stride + c]);
    }
    Pack<T, V>* __restrict__ y = (Pack<T, V>*)a.out + ((size_t)w.b * g.hw) * g.nv + w.vec;
    each_pixel<4>((const Pack<T, V>*)a.x, g, w, [&](const Pack<T, V>& v, long p) __attribute__((always_inline)) {
        Pack<T, V> o;
#pragma unroll
        for (int k = 0; k < V; ++k)
            o[k] = narrow<T>(act_value<ACT>((float)fma(ka[k], (double)widen((T)v[k]), kc[k])));
        y[(size_t)p * g.nv] = o;
    });
}

// ---- backward ------------------------------------------------------------------------------------------------------

// Per channel: what dz and h need
template <int V>
struct ChannelConsts {
    double a[V], c[V];        // z = a x + c
    float mean[V], rstd[V], scale[V];
};

template <int V>
__device__ __forceinline__ void load_consts(const GroupNormArgs& a, const Geom& g, const Place& w, ChannelConsts<V>& k) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = w.vec * V + i;
        const size_t bg = (size_t)w.b * g.G + c / g.Cg;
        k.mean[i] = a.mean[bg];
        k.rstd[i] = a.rstd[bg];
        k.scale[i] = a.scale[w.b * a.aff_stride + c];
        k.a[i] = (double)k.scale[i] * (double)k.rstd[i];
        k.c[i] = fma(-(double)k.mean[i], k.a[i], (double)a.bias[w.b * a.aff_stride + c]);
    }
}

template <int U, typename P, typename F>
__device__ __forceinline__ void each_pixel2(const P* __restrict__ x, const P* __restrict__ y, const Geom& g,
                                            const Place& w, F&& body) {
    const size_t o = ((size_t)w.b * g.hw) * g.nv + w.vec;
    const P* xb = x + o;
    const P* yb = y + o;
    long p = w.p0 + w.row;
    for (; p + (long)(U - 1) * g.rows < w.p1; p += (long)U * g.rows) {
        P v[U], u[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            v[k] = xb[(size_t)(p + (long)k * g.rows) * g.nv];
            u[k] = yb[(size_t)(p + (long)k * g.rows) * g.nv];
        }
#pragma unroll
        for (int k = 0; k < U; ++k) body(v[k], u[k], p + (long)k * g.rows);
    }
    for (; p < w.p1; p += g.rows) body(xb[(size_t)p * g.nv], yb[(size_t)p * g.nv], p);
}

// Pass 1: per (image, channel) and tile the sums of dz and dz h; part [b][tile][C]. At most 64 pixels per thread are
// summed in f32, everything beyond in f64.
template <typename T, int V, int ACT>
__global__ __launch_bounds__(NT) void gn_bwd_stats_kernel(GroupNormArgs a, float2* __restrict__ part, Geom g) {
    __shared__ float2 red[NT * V];
    const Place w = place(g);
    if (w.active) {
        ChannelConsts<V> k;
        load_consts<V>(a, g, w, k);
        float s1[V], s2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
        each_pixel2<2>((const Pack<T, V>*)a.x, (const Pack<T, V>*)a.dy, g, w,
                       [&](const Pack<T, V>& v, const Pack<T, V>& u, long) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float x = widen((T)v[i]);
                const float dz = widen((T)u[i]) * act_slope<ACT>(fma(k.a[i], (double)x, k.c[i]));
                s1[i] += dz;
                s2[i] = fmaf(dz, (x - k.mean[i]) * k.rstd[i], s2[i]);
            }
        });
#pragma unroll
        for (int i = 0; i < V; ++i) red[threadIdx.x * V + i] = make_float2(s1[i], s2[i]);
    }
    __syncthreads();
    const int c0 = w.cb * g.nvb * V, width = min(g.C, c0 + g.nvb * V) - c0;
    for (int c = threadIdx.x; c < width; c += NT) {
        double s1 = 0.0, s2 = 0.0;
        for (int r = 0; r < g.rows; ++r) {
            const float2 v = red[r * g.nvb * V + c];
            s1 += v.x;
            s2 += v.y;
        }
        part[((size_t)w.b * g.tiles + w.tile) * g.C + c0 + c] = make_float2((float)s1, (float)s2);
    }
}

// Sums over the tiles: 32 channels by 8 slices per workgroup; sums [b][c] {S1, S2}
constexpr int FC = 32, FS = NT / FC;
__global__ __launch_bounds__(NT) void gn_bwd_finalize_kernel(const float2* __restrict__ part,
                                                             double2* __restrict__ sums, float* __restrict__ dscale,
                                                             float* __restrict__ dbias, Geom g, int per_image) {
    __shared__ double2 red[NT];
    const int cbs = (g.C + FC - 1) / FC;
    const int b = blockIdx.x / cbs, c = (blockIdx.x - b * cbs) * FC + (threadIdx.x % FC), sl = threadIdx.x / FC;
    double s1 = 0.0, s2 = 0.0;
    if (c < g.C) {
#pragma unroll 4
        for (int t = sl; t < g.tiles; t += FS) {
            const float2 v = part[((size_t)b * g.tiles + t) * g.C + c];
            s1 += v.x;
            s2 += v.y;
        }
    }
    red[threadIdx.x] = make_double2(s1, s2);
    __syncthreads();
    if (sl == 0 && c < g.C) {
        for (int k = 1; k < FS; ++k) {
            s1 += red[threadIdx.x + k * FC].x;
            s2 += red[threadIdx.x + k * FC].y;
        }
        sums[(size_t)b * g.C + c] = make_double2(s1, s2);
        if (per_image) {
            dbias[(size_t)b * g.C + c] = (float)s1;
            dscale[(size_t)b * g.C + c] = (float)s2;
        }
    }
}

// dscale, dbias of an affine shared by the batch: the sum over the images
__global__ __launch_bounds__(NT) void gn_bwd_shared_kernel(const double2* __restrict__ sums, float* __restrict__ dscale,
                                                           float* __restrict__ dbias, int B, int C) {
    __shared__ double2 red[NT];
    const int c = blockIdx.x * FC + (threadIdx.x % FC), sl = threadIdx.x / FC;
    double s1 = 0.0, s2 = 0.0;
    if (c < C)
        for (int b = sl; b < B; b += FS) {
            s1 += sums[(size_t)b * C + c].x;
            s2 += sums[(size_t)b * C + c].y;
        }
    red[threadIdx.x] = make_double2(s1, s2);
    __syncthreads();
    if (sl == 0 && c < C) {
        for (int k = 1; k < FS; ++k) {
            s1 += red[threadIdx.x + k * FC].x;
            s2 += red[threadIdx.x + k * FC].y;
        }
        dbias[c] = (float)s1;
        dscale[c] = (float)s2;
    }
}

// Pass 2: dx = rstd (scale dz - S1 / n - h S2 / n); the workgroup first forms its groups' sums
template <typename T, int V, int ACT>
__global__ __launch_bounds__(NT) void gn_bwd_apply_kernel(GroupNormArgs a, const double2* __restrict__ sums, Geom g) {
    __shared__ float2 cg[NT * V];     // {S1 / n, S2 / n} of the block's groups (at most one per channel)
    const Place w = place(g);
    const Groups r = groups_of<V>(g, w.cb);
    const int j = threadIdx.x % r.tpg;
    for (int gi = threadIdx.x / r.tpg; gi < r.ng; gi += NT / r.tpg) {
        const int first = (r.g0 + gi) * g.Cg;
        double s1 = 0.0, s2 = 0.0;
        for (int c = j; c < g.Cg; c += r.tpg) {
            const double2 v = sums[(size_t)w.b * g.C + first + c];
            const double sc = a.scale[w.b * a.aff_stride + first + c];
            s1 = fma(sc, v.x, s1);
            s2 = fma(sc, v.y, s2);
        }
        for (int o = r.tpg / 2; o > 0; o >>= 1) {
            s1 += __shfl_xor(s1, o);
            s2 += __shfl_xor(s2, o);
        }
        if (j == 0) cg[gi] = make_float2((float)(s1 * g.inv_n), (float)(s2 * g.inv_n));
    }
    __syncthreads();
    if (!w.active) return;
    ChannelConsts<V> k;
    load_consts<V>(a, g, w, k);
    float c1[V], c2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 v = cg[(w.vec * V + i) / g.Cg - r.g0];
        c1[i] = v.x;
        c2[i] = v.y;
    }
    Pack<T, V>* __restrict__ dx = (Pack<T, V>*)a.out + ((size_t)w.b * g.hw) * g.nv + w.vec;
    each_pixel2<2>((const Pack<T, V>*)a.x, (const Pack<T, V>*)a.dy, g, w,
                   [&](const Pack<T, V>& v, const Pack<T, V>& u, long p) __attribute__((always_inline)) {
        Pack<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float x = widen((T)v[i]);
            const float dz = widen((T)u[i]) * act_slope<ACT>(fma(k.a[i], (double)x, k.c[i]));
            const float h = (x - k.mean[i]) * k.rstd[i];
            o[i] = narrow<T>(k.rstd[i] * (fmaf(k.scale[i], dz, -c1[i]) - h * c2[i]));
        }
        dx[(size_t)p * g.nv] = o;
    });
}

// ---- host ----------------------------------------------------------------------------------------------------------

// The widest vector that divides the channels and that every tensor is aligned to
template <typename T>
int vector_width(const GroupNormArgs& a) {
    int v = 16 / (int)sizeof(T);
    const size_t at = (size_t)a.x | (size_t)a.out | (size_t)a.dy;
    while (v > 1 && (a.C % v != 0 || at % (v * sizeof(T)) != 0)) v /= 2;
    return v;
}

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

size_t part_bytes_fwd(const Geom& g) { return (size_t)g.B * g.G * g.slots * g.tiles * sizeof(double2); }
size_t part_bytes_bwd(const Geom& g) { return align16((size_t)g.B * g.tiles * g.C * sizeof(float2)); }

template <typename T, int V>
hipError_t forward_t(const GroupNormArgs& a, hipStream_t st) {
    const Geom g = geometry(a.batch, a.hw, a.C, a.G, V);
    const dim3 grid((unsigned)((long)g.B * g.CB * g.tiles));
    double2* stat = (double2*)a.workspace;
    double2* part = stat + (size_t)g.B * g.G;
    if (g.Cg % V == 0)
        hipLaunchKernelGGL((gn_stats_kernel<T, V, true>), grid, dim3(NT), 0, st, a.x, part, g);
    else
        hipLaunchKernelGGL((gn_stats_kernel<T, V, false>), grid, dim3(NT), 0, st, a.x, part, g);
    const long bg = (long)g.B * g.G;
    hipLaunchKernelGGL(gn_finalize_kernel, dim3((unsigned)((bg + 3) / 4)), dim3(NT), 0, st, part, stat, a.mean, a.rstd, g,
                       g.nvb * V, a.eps);
    switch (a.act) {
        case RST_ACT_RELU: hipLaunchKernelGGL((gn_apply_kernel<T, V, RST_ACT_RELU>), grid, dim3(NT), 0, st, a, stat, g); break;
        case RST_ACT_SWISH: hipLaunchKernelGGL((gn_apply_kernel<T, V, RST_ACT_SWISH>), grid, dim3(NT), 0, st, a, stat, g); break;
        case RST_ACT_HARD_SWISH: hipLaunchKernelGGL((gn_apply_kernel<T, V, RST_ACT_HARD_SWISH>), grid, dim3(NT), 0, st, a, stat, g); break;
        default: hipLaunchKernelGGL((gn_apply_kernel<T, V, RST_ACT_LINEAR>), grid, dim3(NT), 0, st, a, stat, g); break;
    }
    return hipGetLastError();
}

template <typename T, int V, int ACT>
void backward_act(const GroupNormArgs& a, float2* part, double2* sums, const Geom& g, dim3 grid, hipStream_t st) {
    const int cbs = (g.C + FC - 1) / FC;
    hipLaunchKernelGGL((gn_bwd_stats_kernel<T, V, ACT>), grid, dim3(NT), 0, st, a, part, g);
    hipLaunchKernelGGL(gn_bwd_finalize_kernel, dim3((unsigned)(g.B * (long)cbs)), dim3(NT), 0, st, part, sums, a.dscale,
                       a.dbias, g, a.aff_stride != 0);
    if (a.aff_stride == 0)
        hipLaunchKernelGGL(gn_bwd_shared_kernel, dim3((unsigned)cbs), dim3(NT), 0, st, sums, a.dscale, a.dbias, g.B, g.C);
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT>), grid, dim3(NT), 0, st, a, sums, g);
}

template <typename T, int V>
hipError_t backward_t(const GroupNormArgs& a, hipStream_t st) {
    const Geom g = geometry(a.batch, a.hw, a.C, a.G, V);
    const dim3 grid((unsigned)((long)g.B * g.CB * g.tiles));
    double2* sums = (double2*)a.workspace;
    float2* part = (float2*)(sums + (size_t)g.B * g.C);
    switch (a.act) {
        case RST_ACT_RELU: backward_act<T, V, RST_ACT_RELU>(a, part, sums, g, grid, st); break;
        case RST_ACT_SWISH: backward_act<T, V, RST_ACT_SWISH>(a, part, sums, g, grid, st); break;
        case RST_ACT_HARD_SWISH: backward_act<T, V, RST_ACT_HARD_SWISH>(a, part, sums, g, grid, st); break;
        default: backward_act<T, V, RST_ACT_LINEAR>(a, part, sums, g, grid, st); break;
    }
    return hipGetLastError();
}

__global__ __launch_bounds__(NT) void gn_zero_kernel(float* a, float* b, long n) {
    const long i = blockIdx.x * (long)NT + threadIdx.x;
    if (i < n) a[i] = b[i] = 0.f;
}

}  // namespace

// The grids are flat: every (image, channel block, tile) has to be countable in 31 bits at every vector width
bool group_norm_supported(int batch, long hw, int C, int G) {
    if (batch == 0 || hw == 0) return true;
    for (int V = 1; V <= 8; V *= 2) {
        if (C % V != 0) break;
        const Geom g = geometry(batch, hw, C, G, V);
        if ((double)g.B * g.CB * g.tiles >= 2147483647.0 || (double)g.B * std::max(g.G, (g.C + FC - 1) / FC) >= 2147483647.0)
            return false;
    }
    return true;
}

size_t group_norm_workspace_bytes(int batch, long hw, int C, int G) {
    size_t n = 16;
    if (batch <= 0 || hw <= 0 || C <= 0 || G <= 0 || C % G != 0) return n;
    for (int V = 1; V <= 8; V *= 2) {
        if (C % V != 0) break;
        const Geom g = geometry(batch, hw, C, G, V);
        n = std::max(n, (size_t)batch * G * sizeof(double2) + part_bytes_fwd(g));
        n = std::max(n, (size_t)batch * C * sizeof(double2) + part_bytes_bwd(g));
    }
    return n;
}

hipError_t group_norm_launch(const GroupNormArgs& a, hipStream_t st) {
    if (a.batch == 0 || a.hw == 0) return hipSuccess;
    if (a.bf16) switch (vector_width<bf16_t>(a)) {
        case 8: return forward_t<bf16_t, 8>(a, st);
        case 4: return forward_t<bf16_t, 4>(a, st);
        case 2: return forward_t<bf16_t, 2>(a, st);
        default: return forward_t<bf16_t, 1>(a, st);
    }
    switch (vector_width<float>(a)) {
        case 4: return forward_t<float, 4>(a, st);
        case 2: return forward_t<float, 2>(a, st);
        default: return forward_t<float, 1>(a, st);
    }
}

hipError_t group_norm_bwd_launch(const GroupNormArgs& a, hipStream_t st) {
    if (a.batch == 0 || a.hw == 0) {      // no pixel: the gradients of the affine are empty sums
        const long n = (long)a.C * (a.aff_stride != 0 ? a.batch : 1);
        if (n > 0)
            hipLaunchKernelGGL(gn_zero_kernel, dim3((unsigned)((n + NT - 1) / NT)), dim3(NT), 0, st, a.dscale, a.dbias, n);
        return hipGetLastError();
    }
    if (a.bf16) switch (vector_width<bf16_t>(a)) {
        case 8: return backward_t<bf16_t, 8>(a, st);
        case 4: return backward_t<bf16_t, 4>(a, st);
        case 2: return backward_t<bf16_t, 2>(a, st);
        default: return backward_t<bf16_t, 1>(a, st);
    }
    switch (vector_width<float>(a)) {
        case 4: return backward_t<float, 4>(a, st);
        case 2: return backward_t<float, 2>(a, st);
        default: return backward_t<float, 1>(a, st);
    }
}

}  // namespace rst
