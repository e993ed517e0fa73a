// group_norm_device.h — what the forward (group_norm.hip) and the backward (group_norm_bwd.hip) of group normalisation
// share: the split of a channels-last tensor over workgroups, its pipelined walk, sums over columns, activations.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/rst.h"
#include "group_norm.h"

namespace rst {
namespace gn {

constexpr int NT = 1024;            // threads of a workgroup
constexpr int LINEAR = RST_ACT_LINEAR, RELU = RST_ACT_RELU, SWISH = RST_ACT_SWISH, HARD_SWISH = RST_ACT_HARD_SWISH;

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

// How a launch splits the tensor. A vector is V channels; a channel block nvb <= NT vectors; `rows` pixels of it are one
// vector per thread, U times as many a batch; workgroup t of an image's `tiles` takes its batches t, t + tiles, ...: the
// workgroups sweep the image together (each in a range of its own, reads were 5 to 10 % slower).
struct Geom {
    long hw;
    int B, C, G, Cg;
    int nv, nvb, CB, rows, tiles, batches;
    int streaming;            // outputs and last reads past the caches
    double inv_n;
};

// One workgroup of 1024 threads per CU over the whole batch: sixteen waves with four 16-byte loads each keep about twice
// the bytes in flight that HBM's latency needs, and the fewer workgroups, the less those of the second pass have to merge.
// More than 128 images get one workgroup each until there are 256: 129 of 3600 x 64 f32 take 3 % more a byte than 128 (backward
// 9 %). Channels that no 16-byte vector divides go by narrower ones, with as many fewer bytes in flight, and more than 512
// vectors a pixel leave the lanes beyond them idle: C = 515 for 512, 59 MB f32 33.0 us for 29.8, backward 77 for 53; 29 MB
// bf16 24.7 for 19.5, backward 56 for 37; C = 63 for 64 31.7 for 29.8, 55 for 49, 20.8 for 19.4, 32 for 33.
constexpr int WORKGROUPS = 256;

// A call that touches more than half of the 256 MB Infinity Cache stores past it, and does not keep what it reads for the
// second time: dirty lines written back under the next reads cost more than that cache then saves. Forward, us past the
// caches / through them: 118 MB 35.7 / 33.3, 177 MB 43.1 / 48.9, 236 MB 61 / 74, 472 MB 109 / 138; backward: 133 MB 45.9
// through them, 177 MB 52 / 59, 354 MB 100 / 119.
constexpr size_t STREAMING_BYTES = 128u << 20;

// bytes: of all tensors, per element
inline Geom geometry(int B, long hw, int C, int G, int V, int U, int bytes, int thread_batches) {
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
    g.batches = (int)((hw + (long)U * g.rows - 1) / ((long)U * g.rows));
    g.tiles = std::min(std::max(1, WORKGROUPS / B), g.batches);
    g.tiles = std::max(g.tiles, (g.batches + thread_batches - 1) / thread_batches);
    g.streaming = (size_t)B * hw * C * bytes > STREAMING_BYTES;
    g.inv_n = 1.0 / ((double)hw * g.Cg);
    return g;
}

struct Place {
    int b, cb, tile, lane, row, vec;
    bool active;
};

// HIP launches fewer than 2^32 threads: more workgroups (many tiny images) go in several launches, launch(first workgroup, grid)
template <typename F>
void in_launches(long blocks, int threads, F&& launch) {
    const long most = 0xFFFFFFFFL / threads;
    for (long first = 0; first < blocks; first += most) launch((int)first, dim3((unsigned)std::min(most, blocks - first)));
}

__device__ __forceinline__ Place place(const Geom& g, int block) {
    Place w;
    const int per = g.CB * g.tiles;
    w.b = block / per;
    const int r = block - w.b * per;
    w.cb = r / g.tiles;
    w.tile = r - w.cb * g.tiles;
    w.row = threadIdx.x / g.nvb;
    w.lane = threadIdx.x - w.row * g.nvb;
    w.vec = w.cb * g.nvb + w.lane;
    w.active = w.row < g.rows && w.vec < g.nv;
    return w;
}

// The thread's pixels in batches of U vectors from each of N tensors, one batch ahead: two buffers by turns in
// straight-line code (copying one to the other would wait for the loads under way). Addresses are a batch's first byte,
// the same for the workgroup, and 32 bits of offset that stay. The last batch's loads beyond the image read its first
// pixel instead (a guarded load would be waited for by itself). start() may be called long before the first use.
// PAST: what is loaded is not to be kept in the caches.
template <typename P, int N, int U, bool PAST>
struct Walk {
    const char* base[N];
    P v[N][U], u[N][U];
    unsigned off[U], idle;    // bytes from a batch's first; to its first pixel
    size_t stride, at;        // bytes from one of the workgroup's batches to the next; to the current one
    int row, rows, left, last;     // batches left; pixels of the last one

    template <bool FULL>
    __device__ __forceinline__ void fetch(P (&to)[N][U], int ahead) {
        const size_t s = at + ahead * stride;
        unsigned o[U];
#pragma unroll
        for (int k = 0; k < U; ++k) o[k] = FULL || k * rows + row < last ? off[k] : idle;
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const P* x = (const P*)(base[n] + s + o[k]);
                to[n][k] = PAST ? __builtin_nontemporal_load(x) : *x;
            }
        __builtin_amdgcn_sched_barrier(0);      // else the scheduler moves them behind the arithmetic that follows
    }
    __device__ __forceinline__ void start(const void* const (&x)[N], const Geom& g, const Place& w) {
        row = w.row;
        rows = g.rows;
        left = (g.batches - w.tile + g.tiles - 1) / g.tiles;
        const int end = w.tile + (left - 1) * g.tiles;             // the workgroup's last batch
        last = (int)min((long)U * rows, g.hw - (long)end * U * rows);
        const size_t pixel = (size_t)g.nv * sizeof(P);
#pragma unroll
        for (int k = 0; k < U; ++k) off[k] = (unsigned)(((k * rows + row) * g.nv + w.vec) * (unsigned)sizeof(P));
        idle = (unsigned)w.vec * (unsigned)sizeof(P);
        stride = (size_t)g.tiles * U * rows * pixel;
        at = ((size_t)w.b * g.hw + (size_t)w.tile * U * rows) * pixel;
#pragma unroll
        for (int n = 0; n < N; ++n) base[n] = (const char*)x[n];
        if (left > 1) fetch<true>(v, 0);
        else fetch<false>(v, 0);
    }
    template <bool FULL, typename F>
    __device__ __forceinline__ void use(P (&from)[N][U], int ahead, F& body) {
        const size_t s = at + ahead * stride;
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (FULL || k * rows + row < last) {
                P one[N];
#pragma unroll
                for (int n = 0; n < N; ++n) one[n] = from[n][k];
                body(one, s, off[k]);
            }
        __builtin_amdgcn_sched_barrier(0);
    }
    // body(vectors of one pixel, its batch's offset and its own in bytes)
    template <typename F>
    __device__ __forceinline__ void run(F&& body) {
        for (; left > 3; left -= 2, at += 2 * stride) {     // all but the last batch are full
            fetch<true>(u, 1);
            use<true>(v, 0, body);
            fetch<true>(v, 2);
            use<true>(u, 1, body);
        }
        if (left == 3) {
            fetch<true>(u, 1);
            use<true>(v, 0, body);
            fetch<false>(v, 2);
            use<true>(u, 1, body);
            use<false>(v, 2, body);
        } else if (left == 2) {
            fetch<false>(u, 1);
            use<true>(v, 0, body);
            use<false>(u, 1, body);
        } else {
            use<false>(v, 0, body);
        }
    }
};

template <bool PAST, typename P>
__device__ __forceinline__ void put(char* base, size_t at, unsigned off, const P& v) {
    if constexpr (PAST) __builtin_nontemporal_store(v, (P*)(base + at + off));
    else *(P*)(base + at + off) = v;
}

// Threads (a power of two, within a wave) that share each of n sums of a workgroup
__device__ __forceinline__ int team(int threads, int n) {
    return n >= threads ? 1 : min(64, 1 << (31 - __clz(threads / n)));
}

// Lane permutations within a row on the halves of a double: the chain of cross-lane reads through LDS that __shfl_xor is
// would take most of a small sum's time
template <int CTRL>
__device__ __forceinline__ double row_permuted(double v) {
    const long long b = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)(b & 0xFFFFFFFFll), CTRL, 0xF, 0xF, true);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xF, 0xF, true);
    return __longlong_as_double(((long long)hi << 32) | (unsigned)lo);
}
// Every member of a team gets its sum
__device__ __forceinline__ double team_sum(double v, int t) {
    if (t >= 2) v += row_permuted<0xB1>(v);      // lanes xor 1
    if (t >= 4) v += row_permuted<0x4E>(v);      // lanes xor 2
    if (t >= 8) v += row_permuted<0x141>(v);     // the half row mirrored
    if (t >= 16) v += row_permuted<0x140>(v);    // the row mirrored
    if (t >= 32) v += __shfl_xor(v, 16);
    if (t >= 64) v += __shfl_xor(v, 32);
    return v;
}
__device__ __forceinline__ double2 team_sum(double2 v, int t) { return make_double2(team_sum(v.x, t), team_sum(v.y, t)); }

// Sums by a team (member j of t) over the rows of red [rows][stride], columns lo .. lo + width
__device__ __forceinline__ double2 team_block_sum(const double2* red, int rows, int stride, int lo, int width, int j, int t) {
    double2 s = make_double2(0.0, 0.0);
    const float inv = 1.f / (float)width;
    for (int e = j; e < width * rows; e += t) {
        const int row = (int)(((float)e + 0.5f) * inv);      // e / width: e < 2^13, half a step from every border
        const double2 v = red[row * stride + lo + (e - row * width)];
        s.x += v.x;
        s.y += v.y;
    }
    return team_sum(s, t);
}

// exp through the hardware's 2^x and 1/x: their argument's rounding counts |z| times, (5 + 2 |z|) 2^-24 relative in all
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

// The widest vector of at most `v` channels (16 bytes) that divides n channels and that every tensor is aligned to
template <typename T>
int vector_width(size_t addresses, int n, int v = 16 / (int)sizeof(T)) {
    while (v > 1 && (n % v != 0 || addresses % (v * sizeof(T)) != 0)) v /= 2;
    return v;
}

// One-launch form: a workgroup takes a bundle of whole groups of one image, bv vectors per pixel, and holds its values
// in registers: `rows` pixels at a time, R pixels per thread.
struct Bundle {
    int B, C, G, Cg, hw;
    int nv, bv, groups, bundles, rows, R, threads;
    int shared;               // backward: workgroups behind the images' form a shared affine's gradients
    double inv_n;
};
constexpr int MAX_R = 16;
constexpr int BUNDLE_GROUPS = 64;   // 8 to make whole vectors, or as many as make 64 bytes: at most 32

// false: the bundle does not fit one workgroup (whether one launch is also faster: forward_in_one, backward_in_one)
inline bool bundle(int B, long hw, int C, int G, int V, int max_r, int max_threads, Bundle& u) {
    const int Cg = C / G;
    int groups = 1;
    while (groups * Cg % V != 0) ++groups;              // divides G: C is a multiple of V
    const auto fits = [&](int n) {
        const long bv = (long)n * Cg / V;
        return bv <= max_threads && (hw + max_threads / bv - 1) / (max_threads / bv) <= max_r;
    };
    if (!fits(groups)) return false;
    // whole 64-byte sectors where that leaves a workgroup for every second CU
    while (groups * 2 <= G && G % (groups * 2) == 0 && groups * Cg / V * 16 < 64 && fits(groups * 2) &&
           (long)B * (G / groups) >= WORKGROUPS)
        groups *= 2;
    u = Bundle{};
    u.B = B;
    u.C = C;
    u.G = G;
    u.Cg = Cg;
    u.hw = (int)hw;
    u.nv = C / V;
    u.bv = groups * Cg / V;
    u.groups = groups;
    u.bundles = G / groups;
    u.threads = 256;      // four vectors a thread where fewer threads do: a small launch's cost is its waves
    while (u.threads < max_threads && (4L * u.threads < hw * u.bv || u.threads < u.bv)) u.threads *= 2;
    u.rows = u.threads / u.bv;
    u.R = 1;
    while (u.R * u.rows < hw) u.R *= 2;
    u.inv_n = 1.0 / ((double)hw * Cg);
    return u.R <= max_r && (double)(B + 1) * u.bundles < 2147483647.0;
}

// When the one-launch form is taken, f32 and bf16 with 32 to 512 channels in groups of 1 to 16 measured: its workgroups
// are few and fetch lines of which they use a bundle's share. Forward, us in one launch / in two: 1024 pixels x 128
// channels f32 x 1 image 5.2 / 11.5, x 32 images (17 MB) 11.5 / 14.9; 4096 pixels x 8 images 19.4 / 14.3. Backward: 1024
// pixels x 128 channels f32 x 8 images (4 MB) 12.3 / 13.3, x 32 images 21.3 / 19.4; 256 pixels x 32 images 7.8 / 12.8;
// 4096 pixels x 1 image 18.3 / 13.3.
inline bool forward_in_one(long hw, size_t bytes) { return hw <= 2048 && bytes <= (16u << 20); }
inline bool backward_in_one(long hw, size_t bytes) { return hw <= 2048 && (size_t)hw * bytes <= ((size_t)1 << 32); }

}  // namespace gn
}  // namespace rst
