// Penalties, biases and grammar masks on logits (logits_process, include/nn.h).
//
// One pass: every logit is read and written once, and that is the bound. A
// workgroup takes CHUNK ids of one row. It counts the row's history in LDS
// (one word an id: bit 31 for the prompt, the rest counts the output; whole
// numbers, so the order of the atomics changes nothing), notes for each biased
// id the last entry of its list, then streams its logits.
#include <limits.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/nn.h"
#include "launch.hpp"
#include "common.hpp"

namespace bmb {
namespace {

constexpr int THREADS = 256;
constexpr int CHUNK = 4096;
constexpr uint32_t IN_PROMPT = 0x80000000u;

struct LogitsArgs {
    LogitsRules r;
    char *out;
    const char *logits;
    long long stride;
    int rows, V, chunks;
};

// One id's logit under the rules; each operation rounds once (no contraction),
// as written.
struct RowRules {
    float repetition, frequency, presence;
    bool penalties;
};
__device__ __forceinline__ float penalise(float x, uint32_t seen, const RowRules &r) {
#pragma clang fp contract(off)
    if (seen) {
        x = x > 0.0f ? x / r.repetition : x * r.repetition;
        const uint32_t n = seen & ~IN_PROMPT;
        if (n) {
            x = x - r.frequency * (float)n;
            x = x - r.presence;
        }
    }
    return x;
}

template <typename T>
__global__ __launch_bounds__(THREADS) void logits_kernel(LogitsArgs a) {
    constexpr int N = 16 / sizeof(T);  // elements of a 16-byte piece
    extern __shared__ uint32_t lds[];
    const LogitsRules &r = a.r;
    const int row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, tid = threadIdx.x;
    T *out = (T *)a.out + row * a.stride;
    const T *in = (const T *)a.logits + row * a.stride;
    // Pieces start where the output row is a multiple of 16 bytes: `skew` ids
    // come before the first one, and belong to the first chunk.
    const int skew = (int)((16 - ((uintptr_t)out & 15)) & 15) / (int)sizeof(T);
    const int lo = chunk == 0 ? 0 : min(a.V, skew + chunk * CHUNK);
    const int hi = min(a.V, skew + (chunk + 1) * CHUNK);
    if (lo >= hi) return;
    uint32_t *seen = lds, *bias = lds + (r.tokens ? CHUNK + N : 0);

    RowRules rules = {r.repetition ? r.repetition[row] : 1.0f,
                      r.frequency ? r.frequency[row] : 0.0f, r.presence ? r.presence[row] : 0.0f,
                      r.tokens != nullptr};
    int b0 = 0, b1 = 0;
    if (r.bias_offsets) {
        b0 = min(max(r.bias_offsets[row], 0), r.biases);
        b1 = min(max(r.bias_offsets[row + 1], 0), r.biases);
    }
    const uint32_t *mask = nullptr;
    if (r.mask) {
        const int m = r.mask_index ? r.mask_index[row] : row;
        if ((unsigned)m < (unsigned)r.masks) mask = r.mask + m * r.mask_stride;
    }
    if (r.tokens) {
        for (int i = tid; i < hi - lo; i += THREADS) seen[i] = 0;
    }
    if (r.bias_offsets) {
        for (int i = tid; i < hi - lo; i += THREADS) bias[i] = 0;
    }
    __syncthreads();
    if (r.tokens) {
        const int *tokens = r.tokens + row * r.token_stride;
        const int len = (int)min((long long)max(r.lens[row], 0), r.token_stride);
        const int prompt = r.prompt_lens ? r.prompt_lens[row] : 0;
        for (int i = tid; i < len; i += THREADS) {
            const int id = tokens[i];
            if (id >= lo && id < hi) {
                if (i < prompt)
                    atomicOr(&seen[id - lo], IN_PROMPT);
                else
                    atomicAdd(&seen[id - lo], 1u);
            }
        }
    }
    for (int i = b0 + tid; i < b1; i += THREADS) {
        const int id = r.bias_ids[i];
        if (id >= lo && id < hi) atomicMax(&bias[id - lo], (uint32_t)(i - b0) + 1);
    }
    __syncthreads();

    const auto one = [&](int id, T v) -> T {
        if (mask && !(mask[id >> 5] >> (id & 31) & 1)) return (T)-INFINITY;
        float x = (float)v;
        if (rules.penalties) x = penalise(x, seen[id - lo], rules);
        if (r.bias_offsets) {
            const uint32_t e = bias[id - lo];
            if (e) x += r.bias_values[b0 + (int)e - 1];
        }
        return (T)x;
    };
    typedef T Piece __attribute__((ext_vector_type(N)));
    const int first = chunk == 0 ? min(skew, a.V) : lo;  // of the whole pieces
    const int last = first + (hi - first) / N * N;
    if (lo + tid < first) out[lo + tid] = one(lo + tid, in[lo + tid]);
    if (last + tid < hi) out[last + tid] = one(last + tid, in[last + tid]);
    const bool same = (((uintptr_t)out ^ (uintptr_t)in) & 15) == 0;
    for (int id = first + tid * N; id < last; id += THREADS * N) {
        Piece x;
        if (same) {
            x = *(const Piece *)(in + id);
        } else {
            for (int e = 0; e < N; ++e) x[e] = in[id + e];
        }
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = one(id + e, x[e]);
        *(Piece *)(out + id) = x;
    }
}

int refuse(const char *why) {
    fprintf(stderr, "bmb: logits_process: %s\n", why);
    return -1;
}

}  // namespace
}  // namespace bmb

extern "C" int logits_process(void *out, const void *logits, int type, int rows, int V,
                              long long stride, const LogitsRules *r, hipStream_t stream) {
    using namespace bmb;
    if (type != BMB_F32 && type != BMB_F16 && type != BMB_BF16)
        return refuse("unknown element type");
    if (rows < 0 || V < 1 || stride < V) return refuse("rows, V or stride is below its least");
    if (rows == 0) return 0;
    if (out == nullptr || logits == nullptr || r == nullptr) return refuse("a null pointer");
    const size_t size = type == BMB_F32 ? 4 : 2;
    if (((uintptr_t)out | (uintptr_t)logits) % size != 0)
        return refuse("a buffer is no multiple of its element's size");
    if (out != logits) {
        const char *o = (const char *)out, *i = (const char *)logits;
        const size_t n = ((size_t)(rows - 1) * stride + V) * size;
        if (o < i + n && i < o + n) return refuse("out overlaps logits in part");
    }
    if (r->tokens && (r->lens == nullptr || r->token_stride < 0))
        return refuse("tokens without lens, or a negative token_stride");
    if (!r->tokens && (r->repetition || r->frequency || r->presence))
        return refuse("penalties without tokens");
    if (r->bias_offsets && (r->biases < 0 || !r->bias_ids || !r->bias_values))
        return refuse("bias_offsets without ids and values");
    if (r->mask && (r->mask_stride < (V + 31ll) / 32 || r->masks < 1))
        return refuse("mask rows that do not hold V bits");
    if (r->mask && !r->mask_index && r->masks < rows) return refuse("fewer masks than rows");
    // (one piece more than V: up to a piece of ids may come before the first whole one)
    const long long chunks = ((long long)V + CHUNK - 1) / CHUNK;
    if (chunks * rows > INT_MAX || V > INT_MAX - 2 * CHUNK) return refuse("too many logits for one call");
    LogitsArgs a = {*r, (char *)out, (const char *)logits, stride, rows, V, (int)chunks};
    const int n = CHUNK + 16 / (int)size;
    const size_t lds = ((r->tokens ? n : 0) + (r->bias_offsets ? n : 0)) * sizeof(uint32_t);
    const dim3 grid((unsigned)(chunks * rows)), block(THREADS);
    if (type == BMB_F32)
        launch(logits_kernel<float>, grid, block, lds, stream, a);
    else if (type == BMB_F16)
        launch(logits_kernel<_Float16>, grid, block, lds, stream, a);
    else
        launch(logits_kernel<__bf16>, grid, block, lds, stream, a);
    return 0;
}
