// group_norm.hip — group normalisation with an activation over channels-last tensors, forward (group_norm_bwd.hip: the
// backward).
//
// x (B, hw, C), G groups of Cg = C / G channels; per image b and group g
//   mean, var = moments over hw * Cg values (biased), rstd = 1 / sqrt(var + eps)
//   y = act(z), z = scale_c (x - mean) rstd + bias_c = a_c x + c_c,  a = scale rstd, c = bias - mean a
//
// Channels last puts a group's values Cg at a time into every pixel, so a workgroup takes a range of pixels with all
// their channels (up to 1024 vectors of them: a channel block) and reduces every group it meets: loads are whole lines.
// Two launches, each one pass over x: sums per (tile, group), then the affine and the activation, whose workgroups first
// merge the sums of their image (a third launch merges where that would be more than a workgroup should read). The
// second pass finds x in the caches while it has less than their 256 MB. An image whose groups fit a workgroup's
// registers takes one launch and one pass.
// Sums are merged in a fixed order, without atomics: the same inputs give the same bits.
//
// Arithmetic: the moments are sums of x and x^2 in 64 bits: f64 adds and FMAs issue at the rate of the scalar f32 ones
// on this chip, and E[x^2] - mean^2 then loses log2(mean^2 / var) of 53 bits, not of 24. z = a x + c is one f64 FMA for
// the same reason (c ~ mean / std large).
#include <hip/hip_runtime.h>

#include "group_norm_device.h"

namespace rst {
namespace {

using namespace gn;

constexpr int U = 4;          // vectors of a batch per thread

// The first pass's split, as the second pass has to know it: sums part [b][g][slot][tile], slots: channel blocks that
// one group can meet; merge: the second pass merges them (else stat [b][g] has been formed)
struct Parts {
    const double2* part;
    double2* stat;
    int block_channels, slots, tiles, merge;
};

struct Groups {
    int c0, c1, g0, ng;       // a channel block's channels and the groups it meets
};
template <int V>
__device__ __forceinline__ Groups groups_of(const Geom& g, int cb) {
    Groups r;
    r.c0 = cb * g.nvb * V;
    r.c1 = min(g.C, r.c0 + g.nvb * V);
    r.g0 = r.c0 / g.Cg;
    r.ng = (r.c1 - 1) / g.Cg - r.g0 + 1;
    return r;
}

// {mean, rstd} of the sums {x, x^2}
__device__ __forceinline__ double2 moments(double2 s, double inv_n, float eps) {
    const double mean = s.x * inv_n;
    double var = s.y * inv_n - mean * mean;
    var = var < 0.0 ? 0.0 : var;          // keeps a NaN
    // one Newton step on the hardware's 1 / sqrt: about one unit in the last place, where 0 and infinity keep theirs
    const double d = var + (double)eps, r = __builtin_amdgcn_rsq(d), s1 = fma(0.5 * r, fma(-d * r, r, 1.0), r);
    return make_double2(mean, s1 == s1 ? s1 : r);
}

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == RELU) return z < 0.f ? 0.f : z;             // keeps a NaN
    if constexpr (ACT == SWISH) return z * sigmoid(z);
    if constexpr (ACT == HARD_SWISH) return z <= -3.f ? 0.f : (z >= 3.f ? z : z * (z + 3.f) * (1.f / 6.f));
    return z;
}

// x and x^2 of a vector into its sums. UNI: the vector lies in one group
template <typename T, int V, bool UNI>
__device__ __forceinline__ void add_moments(const Pack<T, V>& v, double* s, double* q) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const double d = (double)widen((T)v[k]);
        s[UNI ? 0 : k] += d;
        q[UNI ? 0 : k] = fma(d, d, q[UNI ? 0 : k]);
    }
}

// Pass 1: sums of x and x^2 of every (image, group) over a tile. Bound by reading x: 59 MB bf16 in 11.9 us (5.0 TB/s),
// 236 MB f32 in 40.6 (5.8 TB/s; a kernel that only reads: 6.4)
template <typename T, int V, bool UNI>
__global__ __launch_bounds__(NT) void gn_stats_kernel(const void* x, Parts parts, Geom g, int block0) {
    constexpr int E = UNI ? 1 : V;
    __shared__ double2 red[NT * E];
    const Place w = place(g, blockIdx.x + block0);
    double s[E], q[E];
#pragma unroll
    for (int k = 0; k < E; ++k) s[k] = q[k] = 0.0;
    if (w.active) {
        Walk<Pack<T, V>, 1, U, false> walk;
        const void* in[1] = {x};
        walk.start(in, g, w);
        walk.run([&](const Pack<T, V>(&v)[1], size_t, unsigned) __attribute__((always_inline)) { add_moments<T, V, UNI>(v[0], s, q); });
    }
#pragma unroll
    for (int k = 0; k < E; ++k) red[threadIdx.x * E + k] = make_double2(s[k], q[k]);
    __syncthreads();
    const Groups r = groups_of<V>(g, w.cb);
    const int t = team(NT, r.ng), j = threadIdx.x % t;
    for (int gi = threadIdx.x / t; gi < r.ng; gi += NT / t) {
        const int group = r.g0 + gi;
        const int lo = (max(r.c0, group * g.Cg) - r.c0) / (V / E), hi = (min(r.c1, (group + 1) * g.Cg) - r.c0) / (V / E);
        const double2 sum = team_block_sum(red, g.rows, g.nvb * E, lo, hi - lo, j, t);
        if (j == 0) {
            const int slot = w.cb - (group * g.Cg) / parts.block_channels;
            const_cast<double2*>(parts.part)[(((size_t)w.b * g.G + group) * parts.slots + slot) * parts.tiles + w.tile] = sum;
        }
    }
}

// A team's sum over the parts of (image, group), its first AHEAD loads apart from their use
struct Merge {
    static constexpr int AHEAD = 8;
    const double2* at;
    int n, j, t;
    double2 v[AHEAD];
    __device__ __forceinline__ void load(const Parts& p, const Geom& g, size_t bg, int group, int j_, int t_) {
        j = j_;
        t = t_;
        n = (((group + 1) * g.Cg - 1) / p.block_channels - (group * g.Cg) / p.block_channels + 1) * p.tiles;
        at = p.part + bg * p.slots * p.tiles;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) v[i] = at[min(j + i * t, n - 1)];
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ double2 sum() {
        double2 s = make_double2(0.0, 0.0);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (j + i * t < n) {
                s.x += v[i].x;
                s.y += v[i].y;
            }
#pragma unroll 4
        for (int i = j + AHEAD * t; i < n; i += t) {
            s.x += at[i].x;
            s.y += at[i].y;
        }
        return team_sum(s, t);
    }
};

// The merge as a launch of its own, one wave per (image, group)
__global__ __launch_bounds__(256) void gn_finalize_kernel(Parts p, float* mean, float* rstd, Geom g, float eps, int block0) {
    const long bg = ((long)blockIdx.x + block0) * 4 + threadIdx.x / 64;
    if (bg >= (long)g.B * g.G) return;
    Merge merge;
    merge.load(p, g, (size_t)bg, (int)(bg % g.G), threadIdx.x & 63, 64);
    const double2 s = merge.sum();
    if ((threadIdx.x & 63) == 0) {
        const double2 m = moments(s, g.inv_n, eps);
        p.stat[bg] = m;
        if (mean != nullptr) mean[bg] = (float)m.x;
        if (rstd != nullptr) rstd[bg] = (float)m.y;
    }
}

// Pass 2: y = act(a x + c). MERGE: the image's sums are merged here, while the first loads are under way. Bound by memory:
// 59 + 59 MB bf16 in 21 us (5.6 TB/s), 236 + 236 MB f32 stored past the caches in 68 (7.0 TB/s: more than HBM gives, so some
// of x comes from the Infinity Cache; all of it comes from behind L2). 32-bit arithmetic instead of the f64 FMA was no
// faster. One image has less of both than of the merge's: 28800 pixels x 128 channels f32 are 14.7 MB, and each of the 225
// workgroups merges 115 KB of sums, 26 MB in all, which L2 holds (8.2 us)
constexpr int MERGE_GROUPS = 1024;
template <typename T, int V, int ACT, bool MERGE, bool PAST>
__global__ __launch_bounds__(NT) void gn_apply_kernel(GroupNormArgs a, Parts p, Geom g, int block0) {
    __shared__ double2 stat[MERGE ? MERGE_GROUPS : 1];
    const Place w = place(g, blockIdx.x + block0);
    const Groups r = groups_of<V>(g, w.cb);
    const int t = team(NT, r.ng);
    int gi = threadIdx.x / t;
    Merge merge;       // loads return in order: the sums first, then the pixels
    if (MERGE && gi < r.ng) merge.load(p, g, (size_t)w.b * g.G + r.g0 + gi, r.g0 + gi, threadIdx.x % t, t);
    Walk<Pack<T, V>, 1, U, PAST> walk;
    const void* in[1] = {a.x};
    double ka[V], kc[V];
    if (w.active) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            ka[k] = (double)a.scale[w.b * a.aff_stride + w.vec * V + k];
            kc[k] = (double)a.bias[w.b * a.aff_stride + w.vec * V + k];
        }
        walk.start(in, g, w);
    }
    if constexpr (MERGE) {
        while (gi < r.ng) {
            const size_t bg = (size_t)w.b * g.G + r.g0 + gi;
            const double2 s = merge.sum();
            if (merge.j == 0) {
                const double2 m = moments(s, g.inv_n, a.eps);
                stat[gi] = m;
                if (w.tile == 0) {        // (a group of two channel blocks: both write the same)
                    if (a.mean != nullptr) a.mean[bg] = (float)m.x;
                    if (a.rstd != nullptr) a.rstd[bg] = (float)m.y;
                }
            }
            gi += NT / t;
            if (gi < r.ng) merge.load(p, g, bg + NT / t, r.g0 + gi, merge.j, t);
        }
        __syncthreads();
    }
    if (!w.active) return;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int c = w.vec * V + k;
        const double2 m = MERGE ? stat[c / g.Cg - r.g0] : p.stat[(size_t)w.b * g.G + c / g.Cg];
        ka[k] *= m.y;
        kc[k] = fma(-m.x, ka[k], kc[k]);
    }
    walk.run([&](const Pack<T, V>(&v)[1], size_t at, unsigned off) __attribute__((always_inline)) {
        Pack<T, V> o;
#pragma unroll
        for (int k = 0; k < V; ++k)
            o[k] = narrow<T>(act_value<ACT>((float)fma(ka[k], (double)widen((T)v[0][k]), kc[k])));
        put<PAST>((char*)a.out, at, off, o);
    });
}

// One launch: the bundle's values stay in registers between the moments and the output. Bound by latency: 450 pixels x 96
// channels 6.1 us, an almost empty image 3.6 in a graph. (The widest form, bf16 with 16 vectors of eight, spills 8 registers)
template <typename T, int V, bool UNI, int R>
__global__ __launch_bounds__(NT) void gn_fused_kernel(GroupNormArgs a, Bundle u, int block0) {
    constexpr int E = UNI ? 1 : V;
    __shared__ double2 red[(UNI ? NT : NT / 2) * E];
    __shared__ double2 stat[BUNDLE_GROUPS];
    const int block = blockIdx.x + block0, b = block / u.bundles, first = (block - b * u.bundles) * u.groups;   // first group
    const int row = threadIdx.x / u.bv, lane = threadIdx.x - row * u.bv;
    const int vec = first * u.Cg / V + lane;
    const size_t at = ((size_t)b * u.hw + row) * u.nv + vec, step = (size_t)u.rows * u.nv;
    const bool active = row < u.rows && row < u.hw;
    Pack<T, V> v[R];
    double s[E], q[E];
#pragma unroll
    for (int k = 0; k < E; ++k) s[k] = q[k] = 0.0;
    double ka[V], kc[V];
    if (active) {
        const Pack<T, V>* x = (const Pack<T, V>*)a.x + at;
#pragma unroll
        for (int k = 0; k < R; ++k) v[k] = x[row + k * u.rows < u.hw ? k * step : 0];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            ka[k] = (double)a.scale[b * a.aff_stride + vec * V + k];
            kc[k] = (double)a.bias[b * a.aff_stride + vec * V + k];
        }
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (row + k * u.rows < u.hw) add_moments<T, V, UNI>(v[k], s, q);
    }
#pragma unroll
    for (int k = 0; k < E; ++k) red[threadIdx.x * E + k] = make_double2(s[k], q[k]);
    __syncthreads();
    const int t = team(u.threads, u.groups), j = threadIdx.x % t;
    for (int gi = threadIdx.x / t; gi < u.groups; gi += u.threads / t) {
        const int width = u.Cg / (V / E);
        const double2 sum = team_block_sum(red, u.rows, u.bv * E, gi * width, width, j, t);
        if (j == 0) {
            const double2 m = moments(sum, u.inv_n, a.eps);
            stat[gi] = m;
            const size_t bg = (size_t)b * u.G + first + gi;
            if (a.mean != nullptr) a.mean[bg] = (float)m.x;
            if (a.rstd != nullptr) a.rstd[bg] = (float)m.y;
        }
    }
    __syncthreads();
    if (!active) return;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const double2 m = stat[(vec * V + k) / u.Cg - first];
        ka[k] *= m.y;
        kc[k] = fma(-m.x, ka[k], kc[k]);
    }
    Pack<T, V>* y = (Pack<T, V>*)a.out + at;
#pragma unroll
    for (int k = 0; k < R; ++k)
        if (row + k * u.rows < u.hw) {
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float z = (float)fma(ka[i], (double)widen((T)v[k][i]), kc[i]);
                float f;
                switch (a.act) {          // one branch per vector of a small tensor: not worth four kernels
                    case RELU: f = act_value<RELU>(z); break;
                    case SWISH: f = act_value<SWISH>(z); break;
                    case HARD_SWISH: f = act_value<HARD_SWISH>(z); break;
                    default: f = z;
                }
                o[i] = narrow<T>(f);
            }
            y[k * step] = o;
        }
}

// ---- host ----------------------------------------------------------------------------------------------------------

// The second pass merges where its workgroups read at most this, else a launch of its own does: one image of 28800 pixels
// x 128 channels, 115 KB 13.6 us (with the launch 13.9, and 3 us more on the host), 230 KB 14.8 (13.8)
constexpr size_t MERGE_BYTES = 160 << 10;

Geom geometry_of(const GroupNormArgs& a, int V) {
    return geometry(a.batch, a.hw, a.C, a.G, V, U, a.bf16 ? 4 : 8, 1 << 30);
}

Parts parts_of(const Geom& g, int V) {
    Parts p{};
    p.block_channels = g.nvb * V;
    p.slots = std::min(g.CB, (g.Cg - 1) / p.block_channels + 2);
    p.tiles = g.tiles;
    return p;
}

// The widths that the two passes (or the one) can use
template <int V, typename T, bool UNI>
hipError_t fused_launch(const GroupNormArgs& a, const Bundle& u, hipStream_t st) {
    in_launches((long)u.B * u.bundles, u.threads, [&](int first, dim3 grid) {
        const dim3 block(u.threads);
        switch (u.R) {
            case 1: hipLaunchKernelGGL((gn_fused_kernel<T, V, UNI, 1>), grid, block, 0, st, a, u, first); break;
            case 2: hipLaunchKernelGGL((gn_fused_kernel<T, V, UNI, 2>), grid, block, 0, st, a, u, first); break;
            case 4: hipLaunchKernelGGL((gn_fused_kernel<T, V, UNI, 4>), grid, block, 0, st, a, u, first); break;
            case 8: hipLaunchKernelGGL((gn_fused_kernel<T, V, UNI, 8>), grid, block, 0, st, a, u, first); break;
            default: hipLaunchKernelGGL((gn_fused_kernel<T, V, UNI, 16>), grid, block, 0, st, a, u, first); break;
        }
    });
    return hipGetLastError();
}

template <typename T, int V>
hipError_t apply_launch(const GroupNormArgs& a, const Parts& p, hipStream_t st) {
    const Geom g = geometry_of(a, V);
#define GN_APPLY(ACT)                                                                                                         \
    if (p.merge && g.streaming) hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT, true, true>), grid, dim3(NT), 0, st, a, p, g, first); \
    else if (p.merge) hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT, true, false>), grid, dim3(NT), 0, st, a, p, g, first);   \
    else if (g.streaming) hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT, false, true>), grid, dim3(NT), 0, st, a, p, g, first); \
    else hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT, false, false>), grid, dim3(NT), 0, st, a, p, g, first);
    in_launches((long)g.B * g.CB * g.tiles, NT, [&](int first, dim3 grid) {
        switch (a.act) {
            case RELU: GN_APPLY(RELU) break;
            case SWISH: GN_APPLY(SWISH) break;
            case HARD_SWISH: GN_APPLY(HARD_SWISH) break;
            default: GN_APPLY(LINEAR) break;
        }
    });
#undef GN_APPLY
    return hipGetLastError();
}

template <typename T, int V, bool UNI>
hipError_t stats_launch(const GroupNormArgs& a, hipStream_t st) {
    Bundle u;
    if (forward_in_one(a.hw, (size_t)a.batch * a.hw * a.C * sizeof(T)) &&
        bundle(a.batch, a.hw, a.C, a.G, V, MAX_R, UNI ? NT : NT / 2, u))
        return fused_launch<V, T, UNI>(a, u, st);
    const Geom g = geometry_of(a, V);
    Parts p = parts_of(g, V);
    p.stat = (double2*)a.workspace;
    p.part = p.stat + (size_t)g.B * g.G;
    const int av = vector_width<T>((size_t)a.x | (size_t)a.out, a.C);
    const Geom ga = geometry_of(a, av);
    const int block_groups = std::min(a.G, (ga.nvb * av - 1) / ga.Cg + 2);
    p.merge = block_groups <= MERGE_GROUPS && (size_t)block_groups * p.slots * g.tiles * sizeof(double2) <= MERGE_BYTES;
    in_launches((long)g.B * g.CB * g.tiles, NT, [&](int first, dim3 grid) {
        hipLaunchKernelGGL((gn_stats_kernel<T, V, UNI>), grid, dim3(NT), 0, st, a.x, p, g, first);
    });
    if (!p.merge)
        in_launches(((long)g.B * g.G + 3) / 4, 256, [&](int first, dim3 grid) {
            hipLaunchKernelGGL(gn_finalize_kernel, grid, dim3(256), 0, st, p, a.mean, a.rstd, g, a.eps, first);
        });
    switch (av) {
        case 8:
            if constexpr (sizeof(T) == 2) return apply_launch<T, 8>(a, p, st);
        case 4: return apply_launch<T, 4>(a, p, st);
        case 2: return apply_launch<T, 2>(a, p, st);
        default: return apply_launch<T, 1>(a, p, st);
    }
}

// The moments go by the widest vector that lies in one group (one pair of sums per thread), or by four channels with a
// pair of sums each where the groups are narrower
struct Width {
    int V;
    bool uni;
};
Width moments_width(int wide, int uni) {
    if (uni >= 4) return {uni, true};
    if (wide >= 4) return {4, false};
    if (uni == 2) return {2, true};
    if (wide == 2) return {2, false};
    return {1, true};
}

template <typename T>
hipError_t forward(const GroupNormArgs& a, hipStream_t st) {
    const size_t at = (size_t)a.x | (size_t)a.out;
    const Width w = moments_width(vector_width<T>(at, a.C), vector_width<T>(at, a.C / a.G));
    switch (w.V) {
        case 8:
            if constexpr (sizeof(T) == 2) return stats_launch<T, 8, true>(a, st);
        case 4: return w.uni ? stats_launch<T, 4, true>(a, st) : stats_launch<T, 4, false>(a, st);
        case 2: return w.uni ? stats_launch<T, 2, true>(a, st) : stats_launch<T, 2, false>(a, st);
        default: return stats_launch<T, 1, true>(a, st);
    }
}

}  // namespace

// Workgroups are counted over all launches: every (image, channel block, tile) has to be countable in 31 bits at every vector width. A batch of
// four pixels of f32 is addressed in 32 bits: fewer than 2^28 channels
bool group_norm_supported(int batch, long hw, int C, int G) {
    if (batch == 0 || hw == 0) return true;
    if (C > 1 << 27) return false;
    const Geom g = geometry(batch, hw, C, G, 1, 1, 4, 1);
    return (double)g.B * g.CB * g.tiles < 2147483000.0 && (double)g.B * std::max(g.G, g.C) < 2147483000.0;
}

// What a call may need, whatever its tensors' alignment (in elements: 1, 2, 4 or 8)
size_t group_norm_workspace_bytes(int batch, long hw, int C, int G) {
    if (batch <= 0 || hw <= 0 || C <= 0 || G <= 0 || C % G != 0) return 0;
    size_t n = 0;
    for (size_t a = 1; a <= 8; a *= 2) {
        const Width w = moments_width(vector_width<bf16_t>(2 * a, C), vector_width<bf16_t>(2 * a, C / G));
        Bundle u;
        if (forward_in_one(hw, (size_t)batch * hw * C * 4) && bundle(batch, hw, C, G, w.V, MAX_R, w.uni ? NT : NT / 2, u))
            continue;
        const Geom g = geometry(batch, hw, C, G, w.V, U, 4, 1 << 30);
        n = std::max(n, (size_t)batch * G * sizeof(double2) * ((size_t)parts_of(g, w.V).slots * g.tiles + 1));
    }
    return n;
}

hipError_t group_norm_launch(const GroupNormArgs& a, hipStream_t st) {
    if (a.batch == 0 || a.hw == 0) return hipSuccess;
    return a.bf16 ? forward<bf16_t>(a, st) : forward<float>(a, st);
}

}  // namespace rst
