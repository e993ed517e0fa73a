// adamw_api.hip — C ABI of the AdamW step over many tensors (include/rst.h rst_adamw_*).
//
// rst_adamw_create cuts the variables into chunks once and keeps the table on the device; a step is then one launch
// (three with global-norm clipping and separate gradient tensors: pointers, norm, step). Nothing is allocated or
// synchronised by a step.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "../../include/rst.h"
#include "adamw.h"
#include "common.h"

using namespace rst;

struct rst_adamw {
    int device = 0, bits = 32, num_tensors = 0, num_chunks = 0;
    size_t num_blocks = 0;
    std::vector<bool> filled;          // per variable: it has elements
    bool past = false;                 // the step's data does not stay in the caches
    rst_adamw_state state{};
    AdamwChunk* d_chunks = nullptr;    // one allocation: the table, the step counters (zero), partials, gradient pointers
    unsigned* d_tickets = nullptr;
    double* d_partials = nullptr;
    const void** d_ptrs = nullptr;
    ~rst_adamw() { (void)hipFree(d_chunks); }
};

namespace {

// A step that touches more than half of the 256 MB Infinity Cache loads and stores past it (with the larger chunks and 32-bit
// states, 12 M elements 70 us, through it 80; 6 M 38.9 and 44.4)
constexpr size_t STREAMING_BYTES = 128u << 20;
constexpr size_t MAX_CHUNKS = 0xFFFFFFFFu / 256;     // HIP launches fewer than 2^32 threads, 256 of them a chunk's
// The kernels take the reciprocal of sqrt(v) + epsilon in f32: below 2^-126 it is infinite, and an element with m = v = 0 a NaN
constexpr float SMALLEST_EPSILON = 1.17549435e-38f;
constexpr size_t MAX_ELEMENTS = (size_t)1 << 36;     // 256 GB of variables

int step_args(rst_adamw* h, const char* who, int dtype, const rst_adamw_config* c, AdamwArgs& a) {
    const char* what = nullptr;      // (no string is made where nothing is wrong)
    int dev = 0, code = RST_ERR_INVALID;
    RST_HIP_TRY(hipGetDevice(&dev));
    if (dtype != RST_DTYPE_FLOAT32 && dtype != RST_DTYPE_BFLOAT16) {
        what = "gradients are float32 or bfloat16";
        code = RST_ERR_UNSUPPORTED;
    } else if (!(c->beta_1 >= 0.0 && c->beta_1 < 1.0 && c->beta_2 >= 0.0 && c->beta_2 < 1.0)) {
        what = "beta_1 and beta_2 must lie in [0, 1)";
    } else if (!std::isfinite((float)c->learning_rate) || !std::isfinite((float)c->weight_decay) ||
               !((float)c->epsilon >= SMALLEST_EPSILON) || !std::isfinite((float)c->epsilon) ||
               !(c->global_clipnorm >= 0.0) || !std::isfinite(c->global_clipnorm)) {
        what = "hyperparameters must be finite in 32 bits, epsilon at least 2^-126 and global_clipnorm not negative";
    } else if (dev != h->device) {
        what = "called on another device than the handle was made on";
    }
    if (what != nullptr) return set_error(code, std::string(who) + ": " + what);
    a.chunks = h->d_chunks;
    a.grad_ptrs = h->d_ptrs;
    a.grad_bf16 = dtype == RST_DTYPE_BFLOAT16;
    a.num_chunks = h->num_chunks;
    a.m = h->state.m;
    a.v = h->state.v;
    a.m_scale = h->state.m_scale;
    a.v_scale = h->state.v_scale;
    a.iterations = h->state.iterations;
    a.global_norm = h->state.global_norm;
    a.tickets = h->d_tickets;
    a.partials = h->d_partials;
    a.num_partials = c->global_clipnorm > 0.0 ? std::min(h->num_chunks, ADAMW_MAX_PARTIALS) : 0;
    a.lr = c->learning_rate;
    a.decay = c->weight_decay;
    a.b1 = c->beta_1;
    a.b2 = c->beta_2;
    a.eps = c->epsilon;
    a.clip = c->global_clipnorm;
    a.log_b1 = std::log(c->beta_1);
    a.log_b2 = std::log(c->beta_2);
    a.seed = c->seed;
    return RST_OK;
}

int launch(rst_adamw* h, const AdamwArgs& a, hipStream_t st) {
    if (a.num_partials > 0) RST_HIP_TRY(adamw_norm_launch(a, h->d_partials, st));
    RST_HIP_TRY(adamw_step_launch(a, h->bits, h->past, st));
    return RST_OK;
}

// Elements per workgroup. 32-bit states: one vector per thread where the step streams through HBM (the workgroups' reads
// then sweep closely: 48 M elements 217 us, with 4096 252; 12 M 60 and 68), four where latency counts (2.7 M with
// clipping 17.6 us, with 1024 20.7). 8-bit states: two rounds of eight per thread pay for large steps (48 M 181 us, with
// one 193), one for small (12 M 39.5 us, with two 43.4; 2.7 M 18.7 and 19.0).
size_t chunk_size(size_t elements, int bits, bool past) {
    if (bits == 32) return past ? ADAMW_CHUNK / 4 : ADAMW_CHUNK;
    return elements < ((size_t)16 << 20) ? ADAMW_CHUNK / 2 : ADAMW_CHUNK;
}

int create(const rst_adamw_tensor* tensors, int n, int bits, const rst_adamw_state* state, rst_adamw* h) {
    std::vector<AdamwChunk> chunks;
    size_t blocks = 0, elements = 0, total = 0;
    for (int k = 0; k < n; ++k) {
        if (tensors[k].count > MAX_ELEMENTS || (total += tensors[k].count) > MAX_ELEMENTS)
            return set_error(RST_ERR_INVALID, "rst_adamw_create: more elements than a device holds");
    }
    h->past = total * (bits == 8 ? 14 : 26) > STREAMING_BYTES;
    const auto count = [&](size_t chunk) {
        size_t num = 0;
        for (int k = 0; k < n; ++k) num += (tensors[k].count + chunk - 1) / chunk;
        return num;
    };
    size_t chunk = chunk_size(total, bits, h->past);
    if (count(chunk) > MAX_CHUNKS) chunk = ADAMW_CHUNK;
    if (count(chunk) > MAX_CHUNKS)
        return set_error(RST_ERR_UNSUPPORTED, "rst_adamw_create: more workgroups than one launch takes");
    chunks.reserve(count(chunk));
    for (int k = 0; k < n; ++k) {
        const rst_adamw_tensor& t = tensors[k];
        if (t.count != 0 && t.param == nullptr) return set_error(RST_ERR_INVALID, "rst_adamw_create: null variable");
        for (size_t i = 0; i < t.count; i += chunk) {
            AdamwChunk c{};
            c.param = t.param + i;
            c.grad_at = (long long)(t.grad_offset + i);
            c.tensor_at = (long long)i;
            c.state_at = (long long)(bits == 8 ? blocks * ADAMW_BLOCK + i : elements + i);
            c.count = (int)std::min(chunk, t.count - i);
            c.tensor = k;
            c.decay = t.decay != 0;
            chunks.push_back(c);
        }
        h->filled.push_back(t.count != 0);
        blocks += (t.count + ADAMW_BLOCK - 1) / ADAMW_BLOCK;
        elements += t.count;
    }
    if (elements == 0) return set_error(RST_ERR_INVALID, "rst_adamw_create: no variable has an element");
    if (state->m == nullptr || state->v == nullptr ||
        (bits == 8 && (state->m_scale == nullptr || state->v_scale == nullptr)))
        return set_error(RST_ERR_INVALID, "rst_adamw_create: null state");
    if (bits == 8 && (((size_t)state->m | (size_t)state->v) & 7) != 0)
        return set_error(RST_ERR_INVALID, "rst_adamw_create: 8-bit states must be aligned to 8 bytes");
    RST_HIP_TRY(hipGetDevice(&h->device));
    h->bits = bits;
    h->num_tensors = n;
    h->num_chunks = (int)chunks.size();
    h->num_blocks = blocks;
    h->state = *state;
    const size_t line = ADAMW_TICKET_STRIDE * sizeof(unsigned);
    const auto lines = [&](size_t bytes) { return (bytes + line - 1) / line * line; };
    const size_t table = lines(chunks.size() * sizeof(AdamwChunk));
    const size_t tickets = (1 + (chunks.size() + ADAMW_TICKETS - 1) / ADAMW_TICKETS) * line;
    const size_t partials = ADAMW_MAX_PARTIALS * sizeof(double);
    chunks.resize((table + tickets + sizeof(AdamwChunk) - 1) / sizeof(AdamwChunk), AdamwChunk{});   // zeros behind the table
    char* base = nullptr;
    if (hipMalloc(&base, chunks.size() * sizeof(AdamwChunk) + line + partials + n * sizeof(void*)) != hipSuccess)
        return set_error(RST_ERR_ALLOC, "rst_adamw_create: device allocation failed");
    h->d_chunks = (AdamwChunk*)base;
    h->d_tickets = (unsigned*)(base + table);
    h->d_partials = (double*)(base + lines(chunks.size() * sizeof(AdamwChunk)));
    h->d_ptrs = (const void**)(h->d_partials + ADAMW_MAX_PARTIALS);
    RST_HIP_TRY(hipMemcpy(base, chunks.data(), chunks.size() * sizeof(AdamwChunk), hipMemcpyHostToDevice));
    return RST_OK;
}

}  // namespace

extern "C" {

int rst_adamw_create(const rst_adamw_tensor* tensors, int num_tensors, int state_bits, const rst_adamw_state* state,
                     rst_adamw** out) {
    if (tensors == nullptr || state == nullptr || out == nullptr || num_tensors <= 0 || state->iterations == nullptr)
        return set_error(RST_ERR_INVALID, "rst_adamw_create: bad argument");
    if (state_bits != 8 && state_bits != 32)
        return set_error(RST_ERR_UNSUPPORTED, "rst_adamw_create: state_bits must be 8 or 32");
    *out = nullptr;
    rst_adamw* h = nullptr;
    int rc;
    try {
        h = new rst_adamw;
        rc = create(tensors, num_tensors, state_bits, state, h);
    } catch (const std::exception&) {
        rc = set_error(RST_ERR_ALLOC, "rst_adamw_create: out of host memory");
    }
    if (rc != RST_OK) {
        delete h;
        return rc;
    }
    *out = h;
    return RST_OK;
}

void rst_adamw_destroy(rst_adamw* h) { delete h; }

size_t rst_adamw_num_blocks(const rst_adamw* h) { return h ? h->num_blocks : 0; }

int rst_adamw_step(rst_adamw* h, const void* gradients, int dtype, const rst_adamw_config* config, void* stream) {
    if (h == nullptr || config == nullptr || gradients == nullptr)
        return set_error(RST_ERR_INVALID, "rst_adamw_step: null argument");
    AdamwArgs a{};
    const int rc = step_args(h, "rst_adamw_step", dtype, config, a);
    if (rc != RST_OK) return rc;
    a.bucket = gradients;
    return launch(h, a, static_cast<hipStream_t>(stream));
}

int rst_adamw_step_tensors(rst_adamw* h, const void* const* gradients, int num_tensors, int dtype,
                           const rst_adamw_config* config, void* stream) {
    if (h == nullptr || config == nullptr || gradients == nullptr || num_tensors != h->num_tensors)
        return set_error(RST_ERR_INVALID, "rst_adamw_step_tensors: null argument, or not one gradient per variable");
    for (int k = 0; k < num_tensors; ++k)
        if (gradients[k] == nullptr && h->filled[k])
            return set_error(RST_ERR_INVALID, "rst_adamw_step_tensors: null gradient");
    AdamwArgs a{};
    const int rc = step_args(h, "rst_adamw_step_tensors", dtype, config, a);
    if (rc != RST_OK) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    for (int k = 0; k < num_tensors; k += ADAMW_PTRS) {
        AdamwPtrs p{};
        const int n = std::min(ADAMW_PTRS, num_tensors - k);
        std::copy(gradients + k, gradients + k + n, p.p);
        RST_HIP_TRY(adamw_set_pointers_launch(p, h->d_ptrs + k, n, st));
    }
    return launch(h, a, st);
}

}  // extern "C"
