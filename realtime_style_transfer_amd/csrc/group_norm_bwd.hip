// group_norm_bwd.hip — the gradients of group normalisation with an activation (group_norm.hip).
//
// With dz = dy act'(z), h = (x - mean) rstd, z = scale h + bias and n = hw * Cg
//   dbias_c = sum dz, dscale_c = sum dz h
//   dx = rstd (scale dz - S1 / n - h S2 / n),  S1 = sum_g scale dz, S2 = sum_g scale dz h
// Two launches, each one pass over x and dy: sums per (tile, channel), then dx, whose workgroups first merge the sums of
// their image (a third launch where that is too much for each of them); workgroups behind those write the affine's
// gradients where it is shared by the batch. An image whose groups fit a workgroup's registers takes one launch for dx, and
// a few of them no other for a shared affine's gradients.
//
// On which side of a kink z lies is one f32 comparison per value: z > k is x > x0 (for scale > 0) with x0 = mean + (k - bias) /
// (scale rstd) formed in 64 bits and rounded down to f32 once per channel, z >= k is x beyond the f32 number below x0. The
// slopes on the kinks: relu 0 at 0; hard_swish 0 at -3 and 1 at 3, where its forward's branches are.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "group_norm_device.h"

namespace rst {
namespace {

using namespace gn;

// vectors of a batch per thread: 32 bytes of each tensor (hard_swish has too many constants for that beside them)
template <typename T, int ACT>
constexpr int U = ACT == HARD_SWISH ? 2 : 8 / (int)sizeof(T);
constexpr int THREAD_PX = 64;                  // values that a thread sums
// A thread's sums are in 64 bits in the first of two passes. In 32 where that would cost more than it gives: swish over bf16
// tensors (64 values of 8 bits lose less by it than by their own rounding: the affine's gradients are off by 1.5e-7, in 64
// bits by 0.8e-7; the registers would spill, 4 x 480 x 960 x 32 101 us, so 116), and the one launch, whose threads add up eight
// values at most (in 64 bits its widest forms spill: 2048 pixels x 128 channels in groups of 16, relu 11.8 us, so 13.7,
// hard_swish 17.2, so 21.0). Elsewhere it costs 0 to 1 % (four activations, 1 to 118 MB)
template <typename T, int ACT>
using Sum = typename std::conditional<sizeof(T) == 2 && ACT == SWISH, float, double>::type;
constexpr int MERGE_CHANNELS = 2048;
// As the forward's, per workgroup of the second pass: one image of 28800 pixels, 128 channels (256 KB) 22.8 us (with the
// launch 22.1, and 3 us more on the host), 256 channels x 14400 pixels (512 KB) 26.4 (22.1)
constexpr size_t MERGE_BYTES = 256 << 10;
constexpr int SHARED_C = 32;                   // channels of a workgroup that sums over the batch

struct BwdParts {
    float2* part;             // [b][tile][C] {sum dz, sum dz h}
    double2* sums;            // [b][C], where a launch has merged them
    int merge;
    int main_blocks;          // the second pass's workgroups before the shared affine's
};

// The largest f32 number up to x (UP_TO) or below it
template <bool UP_TO>
__device__ __forceinline__ float round_down(double x) {
    const float f = (float)x;
    if ((UP_TO ? (double)f <= x : (double)f < x) || !(f > -__builtin_inff())) return f;      // (-inf and NaN stay)
    const unsigned b = __float_as_uint(f);
    return __uint_as_float(b == 0u || b == 0x80000000u ? 0x80000001u : ((int)b < 0 ? b + 1 : b - 1));
}

// Per channel: d = x - mean, z = slope d + bias with slope = scale rstd; kinks: flip x > at
template <int ACT, int V>
struct Channels {
    float mean[V], rstd[V], slope[V], bias[V], flip[V], at0[V], at1[V];

    // z > k, or z >= k (INCLUSIVE)
    template <bool INCLUSIVE>
    __device__ __forceinline__ float threshold(double a, int i, double k) {
        const double b = (double)bias[i];
        if (!(a != 0.0)) return (INCLUSIVE ? b >= k : b > k) ? -__builtin_inff() : __builtin_inff();
        const double x0 = (double)mean[i] + (k - b) / a;
        return round_down<!INCLUSIVE>(a > 0.0 ? x0 : -x0);
    }
    __device__ __forceinline__ void load(const GroupNormArgs& g, int b, int G, int Cg, int vec) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = vec * V + i;
            const size_t bg = (size_t)b * G + c / Cg;
            mean[i] = g.mean[bg];
            rstd[i] = g.rstd[bg];
            bias[i] = g.bias[b * g.aff_stride + c];
            const double a = (double)g.scale[b * g.aff_stride + c] * (double)rstd[i];
            slope[i] = (float)a;
            if constexpr (ACT == RELU || ACT == HARD_SWISH) {
                flip[i] = a < 0.0 ? -1.f : 1.f;
                at0[i] = threshold<false>(a, i, ACT == RELU ? 0.0 : -3.0);
                if constexpr (ACT == HARD_SWISH) at1[i] = threshold<true>(a, i, 3.0);
            }
        }
    }
    // dz of one value; d = x - mean
    __device__ __forceinline__ float dz(float x, float d, float dy, int i) const {
        if constexpr (ACT == RELU) return flip[i] * x > at0[i] ? dy : 0.f;
        if constexpr (ACT == SWISH) {
            const float z = fmaf(slope[i], d, bias[i]), s = sigmoid(z);
            return dy * (s * fmaf(z, 1.f - s, 1.f));
        }
        if constexpr (ACT == HARD_SWISH) {
            const float t = flip[i] * x, z = fmaf(slope[i], d, bias[i]);
            return t > at1[i] ? dy : (t > at0[i] ? dy * ((z + 1.5f) * (1.f / 3.f)) : 0.f);
        }
        return dy;
    }
    // a value's share of the sums of dz and dz h (dz d, to be multiplied by rstd later, can pass f32)
    template <typename S>
    __device__ __forceinline__ void add(float x, float dy, int i, S& s1, S& s2) const {
        const float d = x - mean[i], g = dz(x, d, dy, i);
        s1 += (S)g;
        s2 = fma((S)g, (S)(d * rstd[i]), s2);
    }
};

// dx = slope dz - k1 - h k2 with k1 = rstd S1 / n, k2 = rstd S2 / n
template <typename T, int V, int ACT>
__device__ __forceinline__ Pack<T, V> dx_of(const Channels<ACT, V>& k, const Pack<T, V>& xs, const Pack<T, V>& dys,
                                            const float (&k1)[V], const float (&k2)[V]) {
    Pack<T, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float x = widen((T)xs[i]), d = x - k.mean[i];
        o[i] = narrow<T>(fmaf(k.slope[i], k.dz(x, d, widen((T)dys[i]), i), -fmaf(d * k.rstd[i], k2[i], k1[i])));
    }
    return o;
}

// Sums over the rows of red [rows][width] by teams; put(column, sum)
template <typename F>
__device__ __forceinline__ void column_sums(const float2* red, int rows, int width, int stride, int threads, F&& put) {
    const int t = team(threads, width), j = threadIdx.x % t;
    for (int c = threadIdx.x / t; c < width; c += threads / t) {
        double2 s = make_double2(0.0, 0.0);
        for (int r = j; r < rows; r += t) {
            const float2 v = red[r * stride + c];
            s.x += v.x;
            s.y += v.y;
        }
        s = team_sum(s, t);
        if (j == 0) put(c, s);
    }
}

// Pass 1. 118 + 118 MB bf16 with swish in 45 us (5.2 TB/s), 59 + 59 MB f32 with relu in 23 (5.1 TB/s): bound by reading;
// swish's 17 instructions a value would take 26 of the 45 by themselves. Partials are rounded to f32, which halves what the
// merges read: a large tensor has 200 of them or more, each off by half a step at most
template <typename T, int V, int ACT>
__global__ __launch_bounds__(NT) void gn_bwd_stats_kernel(GroupNormArgs a, BwdParts p, Geom g, int block0) {
    __shared__ float2 red[NT * V];
    const Place w = place(g, blockIdx.x + block0);
    Sum<T, ACT> s1[V], s2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0;
    if (w.active) {
        Walk<Pack<T, V>, 2, U<T, ACT>, false> walk;
        const void* in[2] = {a.x, a.dy};
        walk.start(in, g, w);
        Channels<ACT, V> k;
        k.load(a, w.b, g.G, g.Cg, w.vec);
        walk.run([&](const Pack<T, V>(&v)[2], size_t, unsigned) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < V; ++i) k.add(widen((T)v[0][i]), widen((T)v[1][i]), i, s1[i], s2[i]);
        });
    }
#pragma unroll
    for (int i = 0; i < V; ++i) red[threadIdx.x * V + i] = make_float2((float)s1[i], (float)s2[i]);
    __syncthreads();
    const int c0 = w.cb * g.nvb * V, width = min(g.C, c0 + g.nvb * V) - c0;
    float2* out = p.part + ((size_t)w.b * g.tiles + w.tile) * g.C + c0;
    column_sums(red, g.rows, width, g.nvb * V, NT,
                [&](int c, double2 s) __attribute__((always_inline)) { out[c] = make_float2((float)s.x, (float)s.y); });
}

// The merge as a launch of its own: sums over the tiles, 32 channels by 8 slices per workgroup
constexpr int FC = 32, FS = 8;
__global__ __launch_bounds__(FC * FS) void gn_bwd_finalize_kernel(BwdParts p, Geom g, int block0) {
    __shared__ double2 red[FC * FS];
    const int cbs = (g.C + FC - 1) / FC;
    const int block = blockIdx.x + block0, b = block / cbs, c = (block - b * cbs) * FC + (threadIdx.x % FC), sl = threadIdx.x / FC;
    double2 s = make_double2(0.0, 0.0);
    if (c < g.C) {
#pragma unroll 4
        for (int t = sl; t < g.tiles; t += FS) {
            const float2 v = p.part[((size_t)b * g.tiles + t) * g.C + c];
            s.x += v.x;
            s.y += v.y;
        }
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (sl == 0 && c < g.C) {
        for (int k = 1; k < FS; ++k) {
            s.x += red[threadIdx.x + k * FC].x;
            s.y += red[threadIdx.x + k * FC].y;
        }
        p.sums[(size_t)b * g.C + c] = s;
    }
}

// The affine's gradients over the whole batch: 32 channels per workgroup, n rows of partial sums
template <typename D>
__device__ __forceinline__ void shared_affine(const D* from, long n, int C, int block, int threads, float* dscale,
                                              float* dbias, double2* red) {
    const int c = block * SHARED_C + threadIdx.x % SHARED_C, slices = threads / SHARED_C;
    double2 s = make_double2(0.0, 0.0);
    if (c < C) {
#pragma unroll 4
        for (long r = threadIdx.x / SHARED_C; r < n; r += slices) {
            const D v = from[(size_t)r * C + c];
            s.x += v.x;
            s.y += v.y;
        }
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if ((int)threadIdx.x < SHARED_C && c < C) {
        for (int k = 1; k < slices; ++k) {
            s.x += red[threadIdx.x + k * SHARED_C].x;
            s.y += red[threadIdx.x + k * SHARED_C].y;
        }
        dbias[c] = (float)s.x;
        dscale[c] = (float)s.y;
    }
}

__global__ __launch_bounds__(256) void gn_bwd_shared_kernel(const double2* sums, int B, int C, float* dscale,
                                                            float* dbias) {
    __shared__ double2 red[256];
    shared_affine(sums, B, C, blockIdx.x, 256, dscale, dbias, red);
}

// {S1 / n, S2 / n} of groups from their channels' sums; sum(c): channel c's
template <typename S, typename F>
__device__ __forceinline__ void group_sums(const GroupNormArgs& a, int b, int g0, int ng, int Cg, double inv_n, int threads,
                                           S&& sum, F&& put) {
    const int t = team(threads, ng), j = threadIdx.x % t;
    for (int gi = threadIdx.x / t; gi < ng; gi += threads / t) {
        const int first = (g0 + gi) * Cg;
        double2 s = make_double2(0.0, 0.0);
        for (int c = first + j; c < first + Cg; c += t) {
            const double2 v = sum(c);
            const double sc = a.scale[b * a.aff_stride + c];
            s.x = fma(sc, v.x, s.x);
            s.y = fma(sc, v.y, s.y);
        }
        s = team_sum(s, t);
        if (j == 0) put(gi, make_float2((float)(s.x * inv_n), (float)(s.y * inv_n)));
    }
}

// Pass 2. MERGE: the image's sums are merged here, while the first loads are under way (one channel block only). Bound by
// memory: 236 MB read, 118 MB written in 55.7 us (6.4 TB/s), 118 and 59 MB in 28.9 (6.1 TB/s)
template <typename T, int V, int ACT, bool MERGE, bool PAST>
__global__ __launch_bounds__(NT) void gn_bwd_apply_kernel(GroupNormArgs a, BwdParts p, Geom g, int block0) {
    __shared__ double2 chan[MERGE ? MERGE_CHANNELS : 1];
    __shared__ double2 red[NT];
    __shared__ float2 cg[MERGE ? MERGE_CHANNELS : NT * V];     // the block's groups, at most one per channel
    const int block = blockIdx.x + block0;
    if (block >= p.main_blocks) {
        if constexpr (MERGE)
            shared_affine(p.part, (long)g.B * g.tiles, g.C, block - p.main_blocks, NT, a.dscale, a.dbias, red);
        else
            shared_affine(p.sums, g.B, g.C, block - p.main_blocks, NT, a.dscale, a.dbias, red);
        return;
    }
    const Place w = place(g, block);
    Walk<Pack<T, V>, 2, U<T, ACT>, PAST> walk;
    const void* in[2] = {a.x, a.dy};
    if (w.active) walk.start(in, g, w);
    const int c0 = w.cb * g.nvb * V, c1 = min(g.C, c0 + g.nvb * V), g0 = c0 / g.Cg, ng = (c1 - 1) / g.Cg - g0 + 1;
    if constexpr (MERGE) {
        const int across = min(g.C, NT), slices = NT / across;
        const float2* part = p.part + (size_t)w.b * g.tiles * g.C;
        for (int base = 0; base < g.C; base += across) {
            const int sl = threadIdx.x / across, c = base + threadIdx.x - sl * across;
            double2 s = make_double2(0.0, 0.0);
            if (sl < slices && c < g.C) {
#pragma unroll 4
                for (int t = sl; t < g.tiles; t += slices) {
                    const float2 v = part[(size_t)t * g.C + c];
                    s.x += v.x;
                    s.y += v.y;
                }
            }
            red[threadIdx.x] = s;
            __syncthreads();
            if (sl == 0 && c < g.C) {
                for (int k = 1; k < slices; ++k) {
                    s.x += red[threadIdx.x + k * across].x;
                    s.y += red[threadIdx.x + k * across].y;
                }
                chan[c] = s;
            }
            __syncthreads();
        }
        group_sums(a, w.b, g0, ng, g.Cg, g.inv_n, NT, [&](int c) __attribute__((always_inline)) { return chan[c]; },
                   [&](int gi, float2 v) __attribute__((always_inline)) { cg[gi] = v; });
    } else {
        group_sums(a, w.b, g0, ng, g.Cg, g.inv_n, NT,
                   [&](int c) __attribute__((always_inline)) { return p.sums[(size_t)w.b * g.C + c]; },
                   [&](int gi, float2 v) __attribute__((always_inline)) { cg[gi] = v; });
    }
    if (w.tile == 0 && a.aff_stride != 0)
        for (int c = c0 + threadIdx.x; c < c1; c += NT) {
            const double2 s = MERGE ? chan[MERGE ? c : 0] : p.sums[(size_t)w.b * g.C + c];
            a.dbias[w.b * a.aff_stride + c] = (float)s.x;
            a.dscale[w.b * a.aff_stride + c] = (float)s.y;
        }
    __syncthreads();
    if (!w.active) return;
    Channels<ACT, V> k;
    k.load(a, w.b, g.G, g.Cg, w.vec);
    float k1[V], k2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 v = cg[(w.vec * V + i) / g.Cg - g0];
        k1[i] = k.rstd[i] * v.x;
        k2[i] = k.rstd[i] * v.y;
    }
    walk.run([&](const Pack<T, V>(&v)[2], size_t at, unsigned off) __attribute__((always_inline)) {
        put<PAST>((char*)a.out, at, off, dx_of<T, V, ACT>(k, v[0], v[1], k1, k2));
    });
}

// One launch: the bundle's x and dy stay in registers between the sums and dx. A shared affine's gradients over several
// images: workgroups behind those sum the bundle over all images once more (u.shared), or the launch of
// gn_bwd_shared_kernel does
template <typename T, int V, int ACT, int R>
__global__ __launch_bounds__(NT) void gn_bwd_fused_kernel(GroupNormArgs a, double2* sums, Bundle u, int block0) {
    __shared__ float2 red[NT * V];
    __shared__ double2 chan[NT];
    __shared__ float2 cg[BUNDLE_GROUPS];
    const int block = blockIdx.x + block0, image = block / u.bundles, first = (block - image * u.bundles) * u.groups;
    const bool all = image == u.B;
    const int row = threadIdx.x / u.bv, lane = threadIdx.x - row * u.bv;
    const int vec = first * u.Cg / V + lane, c0 = first * u.Cg;
    const size_t step = (size_t)u.rows * u.nv;
    const bool active = row < u.rows && row < u.hw;
    int b = all ? 0 : image;
    size_t at = ((size_t)b * u.hw + row) * u.nv + vec;
    Pack<T, V> x[R], dy[R];
    float s1[V], s2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
    Channels<ACT, V> k;
    if (active)
        for (;;) {
            const Pack<T, V>* xs = (const Pack<T, V>*)a.x + at;
            const Pack<T, V>* ys = (const Pack<T, V>*)a.dy + at;
#pragma unroll
            for (int n = 0; n < R; ++n) {
                const size_t o = row + n * u.rows < u.hw ? n * step : 0;
                x[n] = xs[o];
                dy[n] = ys[o];
            }
            k.load(a, b, u.G, u.Cg, vec);
#pragma unroll
            for (int n = 0; n < R; ++n)
                if (row + n * u.rows < u.hw) {
#pragma unroll
                    for (int i = 0; i < V; ++i) k.add(widen((T)x[n][i]), widen((T)dy[n][i]), i, s1[i], s2[i]);
                }
            if (!all || b == u.B - 1) break;
            ++b;
            at += (size_t)u.hw * u.nv;
        }
#pragma unroll
    for (int i = 0; i < V; ++i) red[threadIdx.x * V + i] = make_float2((float)s1[i], (float)s2[i]);
    __syncthreads();
    const bool own = all || a.aff_stride != 0 || u.B == 1;
    column_sums(red, u.rows, u.bv * V, u.bv * V, u.threads, [&](int c, double2 s) __attribute__((always_inline)) {
        chan[c] = s;
        if (own) {
            a.dbias[b * a.aff_stride + c0 + c] = (float)s.x;
            a.dscale[b * a.aff_stride + c0 + c] = (float)s.y;
        } else if (!u.shared) {
            sums[(size_t)b * u.C + c0 + c] = s;
        }
    });
    if (all) return;
    __syncthreads();
    group_sums(a, b, first, u.groups, u.Cg, u.inv_n, u.threads,
               [&](int c) __attribute__((always_inline)) { return chan[c - c0]; },
               [&](int gi, float2 v) __attribute__((always_inline)) { cg[gi] = v; });
    __syncthreads();
    if (!active) return;
    float k1[V], k2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 v = cg[(vec * V + i) / u.Cg - first];
        k1[i] = k.rstd[i] * v.x;
        k2[i] = k.rstd[i] * v.y;
    }
    Pack<T, V>* dx = (Pack<T, V>*)a.out + at;
#pragma unroll
    for (int n = 0; n < R; ++n)
        if (row + n * u.rows < u.hw) dx[n * step] = dx_of<T, V, ACT>(k, x[n], dy[n], k1, k2);
}

__global__ __launch_bounds__(256) void gn_zero_kernel(float* a, float* b, long n, int block0) {
    const long i = ((long)blockIdx.x + block0) * 256 + threadIdx.x;
    if (i < n) a[i] = b[i] = 0.f;
}

// ---- host ----------------------------------------------------------------------------------------------------------

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

bool fused(int B, long hw, int C, int G, int V, int elem, Bundle& u) {
    return backward_in_one(hw, (size_t)B * hw * C * elem) && bundle(B, hw, C, G, V, MAX_R / 2, NT, u) && u.bv * V <= NT;
}

// Whether workgroups of the same launch sum a shared affine's gradients over the images, one image after the other, each in
// R loads: us in a graph so / with the other launch (4 us more on the host): 1024 pixels x 128 channels f32, R = 4,
// 2 images 7.3 / 8.6, 3 images 11.3 / 10.0; 256 x 256, R = 2, 4 images 6.0 / 6.6, 8 images 10.6 / 7.1; 64 x 512, R = 1,
// 8 images 6.6 / 6.5
bool shared_in_one(const Bundle& u) { return u.B > 1 && u.B * u.R <= 8; }

template <typename T, int V, int ACT>
void fused_launch(const GroupNormArgs& a, double2* sums, const Bundle& u, int block0, int blocks, hipStream_t st) {
    in_launches(blocks, u.threads, [&](int first, dim3 grid) {
        const dim3 block(u.threads);
        first += block0;
        switch (u.R) {
            case 1: hipLaunchKernelGGL((gn_bwd_fused_kernel<T, V, ACT, 1>), grid, block, 0, st, a, sums, u, first); break;
            case 2: hipLaunchKernelGGL((gn_bwd_fused_kernel<T, V, ACT, 2>), grid, block, 0, st, a, sums, u, first); break;
            case 4: hipLaunchKernelGGL((gn_bwd_fused_kernel<T, V, ACT, 4>), grid, block, 0, st, a, sums, u, first); break;
            default: hipLaunchKernelGGL((gn_bwd_fused_kernel<T, V, ACT, 8>), grid, block, 0, st, a, sums, u, first); break;
        }
    });
}

template <typename T, int V, int ACT>
hipError_t backward_act(const GroupNormArgs& a, hipStream_t st) {
    BwdParts p{};
    p.sums = (double2*)a.workspace;
    p.part = (float2*)(p.sums + (size_t)a.batch * a.C);
    const int shared_blocks = (a.C + SHARED_C - 1) / SHARED_C;
    Bundle u;
    if (fused(a.batch, a.hw, a.C, a.G, V, sizeof(T), u)) {
        u.shared = a.aff_stride == 0 && shared_in_one(u);
        const int images = u.B * u.bundles;
        if (!u.shared) {
            fused_launch<T, V, ACT>(a, p.sums, u, 0, images, st);
        } else if (a.out == a.dy || a.out == a.x) {      // before dx takes the place of what they read
            fused_launch<T, V, ACT>(a, p.sums, u, images, u.bundles, st);
            fused_launch<T, V, ACT>(a, p.sums, u, 0, images, st);
        } else {
            fused_launch<T, V, ACT>(a, p.sums, u, 0, images + u.bundles, st);
        }
        if (a.aff_stride == 0 && a.batch > 1 && !u.shared)
            hipLaunchKernelGGL(gn_bwd_shared_kernel, dim3((unsigned)shared_blocks), dim3(256), 0, st, p.sums, a.batch, a.C,
                               a.dscale, a.dbias);
        return hipGetLastError();
    }
    const Geom g = geometry(a.batch, a.hw, a.C, a.G, V, U<T, ACT>, 3 * sizeof(T), THREAD_PX / U<T, ACT>);
    p.merge = g.CB == 1 && a.C <= MERGE_CHANNELS && (size_t)g.tiles * a.C * sizeof(float2) <= MERGE_BYTES;
    p.main_blocks = (int)((long)g.B * g.CB * g.tiles);
    in_launches(p.main_blocks, NT, [&](int first, dim3 grid) {
        hipLaunchKernelGGL((gn_bwd_stats_kernel<T, V, ACT>), grid, dim3(NT), 0, st, a, p, g, first);
    });
    if (!p.merge)
        in_launches((long)g.B * ((a.C + FC - 1) / FC), FC * FS, [&](int first, dim3 grid) {
            hipLaunchKernelGGL(gn_bwd_finalize_kernel, grid, dim3(FC * FS), 0, st, p, g, first);
        });
    in_launches((long)p.main_blocks + (a.aff_stride == 0 ? shared_blocks : 0), NT, [&](int first, dim3 grid) {
        if (p.merge && g.streaming)
            hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT, true, true>), grid, dim3(NT), 0, st, a, p, g, first);
        else if (p.merge)
            hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT, true, false>), grid, dim3(NT), 0, st, a, p, g, first);
        else if (g.streaming)
            hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT, false, true>), grid, dim3(NT), 0, st, a, p, g, first);
        else
            hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT, false, false>), grid, dim3(NT), 0, st, a, p, g, first);
    });
    return hipGetLastError();
}

template <typename T, int V>
hipError_t backward_t(const GroupNormArgs& a, hipStream_t st) {
    switch (a.act) {
        case RELU: return backward_act<T, V, RELU>(a, st);
        case SWISH: return backward_act<T, V, SWISH>(a, st);
        case HARD_SWISH: return backward_act<T, V, HARD_SWISH>(a, st);
        default: return backward_act<T, V, LINEAR>(a, st);
    }
}

template <typename T>
hipError_t backward(const GroupNormArgs& a, hipStream_t st) {
    // four channels at most: with eight, their constants (mean, rstd, scale, thresholds, ...) spill at 1024 threads. (With four,
    // hard_swish in the one-launch form of eight f32 vectors a thread does, 12 registers)
    switch (vector_width<T>((size_t)a.x | (size_t)a.dy | (size_t)a.out, a.C, 4)) {
        case 4: return backward_t<T, 4>(a, st);
        case 2: return backward_t<T, 2>(a, st);
        default: return backward_t<T, 1>(a, st);
    }
}

}  // namespace

size_t group_norm_bwd_workspace_bytes(int batch, long hw, int C, int G) {
    if (batch <= 0 || hw <= 0 || C <= 0 || G <= 0 || C % G != 0) return 0;
    size_t n = 0;
    for (size_t a = 1; a <= 4; a *= 2) {
        const int V = vector_width<bf16_t>(2 * a, C, 4);
        Bundle u;
        if (batch > 1 && fused(batch, hw, C, G, V, 2, u) && !shared_in_one(u)) n = std::max(n, (size_t)batch * C * sizeof(double2));   // a shared affine's
        if (fused(batch, hw, C, G, V, 4, u)) continue;
        for (int w : {2, 4})
            n = std::max(n, (size_t)batch * C * sizeof(double2) +
                                align16((size_t)batch * geometry(batch, hw, C, G, V, w, 4, THREAD_PX / w).tiles * C * sizeof(float2)));
    }
    return n;
}

hipError_t group_norm_bwd_launch(const GroupNormArgs& a, hipStream_t st) {
    if (a.batch == 0 || a.hw == 0) {      // no pixel: the gradients of the affine are empty sums
        const long n = (long)a.C * (a.aff_stride != 0 ? a.batch : 1);
        in_launches((n + 255) / 256, 256, [&](int first, dim3 grid) {
            hipLaunchKernelGGL(gn_zero_kernel, grid, dim3(256), 0, st, a.dscale, a.dbias, n, first);
        });
        return hipGetLastError();
    }
    return a.bf16 ? backward<bf16_t>(a, st) : backward<float>(a, st);
}

}  // namespace rst
