// Penalties, biases and grammar masks on logits (logits_process, include/nn.h).
//
// One pass: every logit is read and written once, and that is the bound (512
// rows of 50257 in fp32: 41.6 us, 5.0 TB/s, the rate of a copy). A workgroup
// takes a chunk of the ids of one row. It counts the row's history in LDS
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
constexpr uint32_t IN_PROMPT = 0x80000000u;

struct LogitsArgs {
    LogitsRules r;
    char *out;
    const char *logits;
    long long stride;
    int rows, V, chunks;
    int first;  // the launch's first workgroup of the call's
};

// Each operation rounds once, as written (no contraction).
__device__ __forceinline__ float penalise(float x, uint32_t seen, float repetition,
                                          float frequency, float presence) {
#pragma clang fp contract(off)
    if (seen) {
        x = x > 0.0f ? x / repetition : x * repetition;
        const uint32_t n = seen & ~IN_PROMPT;
        if (n) {
            x = x - frequency * (float)n;
            x = x - presence;
        }
    }
    return x;
}

// Elements of a 16-byte piece, and ids of a workgroup whose threads take
// `pieces` of them each.
template <typename T>
constexpr int piece_of() { return 16 / sizeof(T); }
template <typename T>
constexpr int chunk_of(int pieces) { return THREADS * pieces * piece_of<T>(); }

template <typename T, int PIECES, bool STREAM>
__global__ __launch_bounds__(THREADS) void logits_kernel(LogitsArgs a) {
    constexpr int N = piece_of<T>(), CHUNK = chunk_of<T>(PIECES), WORDS = CHUNK + 2 * N;
    typedef T Piece __attribute__((ext_vector_type(N)));
    extern __shared__ uint4 lds[];
    const LogitsRules &r = a.r;
    const uint32_t block = a.first + blockIdx.x;
    const int row = block / a.chunks, chunk = block % a.chunks, tid = threadIdx.x;
    T *out = (T *)a.out + row * a.stride;
    const T *in = (const T *)a.logits + row * a.stride;
    // Pieces start where the output row is a multiple of 16 bytes: `skew` ids
    // come before the first one, and belong to the first chunk.
    const int skew = (int)((16 - ((uintptr_t)out & 15)) & 15) / (int)sizeof(T);
    const int lo = chunk == 0 ? 0 : min(a.V, skew + chunk * CHUNK);
    const int hi = min(a.V, skew + (chunk + 1) * CHUNK);
    if (lo >= hi) return;
    const int first = chunk == 0 ? min(skew, a.V) : lo;  // of the whole pieces
    const int last = first + (hi - first) / N * N;

    // The logits and the mask's words are on their way while the history is
    // counted.
    const uint32_t *mask = nullptr;
    if (r.mask) {
        const int m = r.mask_index ? r.mask_index[row] : row;
        if ((unsigned)m < (unsigned)r.masks) mask = r.mask + m * r.mask_stride;
    }
    Piece x[PIECES];
    uint32_t bits[PIECES];
    const bool same = (((uintptr_t)out ^ (uintptr_t)in) & 15) == 0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int id = first + (i * THREADS + tid) * N;
        bits[i] = ~0u;
        if (id < last) {
            if (same) {
                x[i] = *(const Piece *)(in + id);
            } else {
                for (int e = 0; e < N; ++e) x[i][e] = in[id + e];
            }
            if (mask)  // (a piece may reach into the next word)
                bits[i] =
                    __builtin_amdgcn_alignbit(mask[(id + N - 1) >> 5], mask[id >> 5], id & 31);
        }
    }

    // LDS: id's word at id + word.
    const bool counts = r.tokens != nullptr;
    const int word = N - first;
    uint32_t *seen = (uint32_t *)lds, *bias = seen + (counts ? WORDS : 0);
    int b0 = 0, b1 = 0;
    if (r.bias_offsets) {
        b0 = min(max(r.bias_offsets[row], 0), r.biases);
        b1 = min(max(r.bias_offsets[row + 1], 0), r.biases);
    }
    const bool biased = b0 < b1;
    const int words = ((counts ? WORDS : 0) + (biased ? WORDS : 0)) / 4;
    for (int i = tid; i < words; i += THREADS) lds[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (counts) {
        const int *tokens = r.tokens + row * r.token_stride;
        // (32 unsigned bits: steps behind the end of up to 2^31 - 1 tokens)
        const uint32_t len = (uint32_t)min((long long)max(r.lens[row], 0), r.token_stride);
        const uint32_t prompt = r.prompt_lens ? max(r.prompt_lens[row], 0) : 0;
        constexpr int AHEAD = 4;  // loads in flight
        for (uint32_t base = tid; base < len; base += AHEAD * THREADS) {
            int id[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                id[j] = base + j * THREADS < len ? tokens[base + j * THREADS] : -1;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                if (id[j] < lo || id[j] >= hi) continue;
                if (base + j * THREADS < prompt)
                    atomicOr(&seen[id[j] + word], IN_PROMPT);
                else
                    atomicAdd(&seen[id[j] + word], 1u);
            }
        }
    }
    for (uint32_t i = b0 + tid; i < (uint32_t)b1; i += THREADS) {
        const int id = r.bias_ids[i];
        if (id >= lo && id < hi) atomicMax(&bias[id + word], i - b0 + 1);
    }
    __syncthreads();

    const float repetition = r.repetition ? r.repetition[row] : 1.0f;
    const float frequency = r.frequency ? r.frequency[row] : 0.0f;
    const float presence = r.presence ? r.presence[row] : 0.0f;
    const auto one = [&](T v, uint32_t n, uint32_t entry) -> T {
        float y = penalise((float)v, n, repetition, frequency, presence);
        if (entry) y += r.bias_values[b0 + (int)entry - 1];
        return (T)y;
    };
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int id = first + (i * THREADS + tid) * N;
        if (id >= last) break;
        // Most pieces have no word of the history and no bias.
        uint32_t n[N] = {}, entry[N] = {}, any = 0;
        if (counts) {
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const uint4 w = *(const uint4 *)(seen + (id + word + e));
                n[e] = w.x, n[e + 1] = w.y, n[e + 2] = w.z, n[e + 3] = w.w;
                any |= w.x | w.y | w.z | w.w;
            }
        }
        if (biased) {
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const uint4 w = *(const uint4 *)(bias + (id + word + e));
                entry[e] = w.x, entry[e + 1] = w.y, entry[e + 2] = w.z, entry[e + 3] = w.w;
                any |= w.x | w.y | w.z | w.w;
            }
        }
        if (any) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (n[e] | entry[e]) x[i][e] = one(x[i][e], n[e], entry[e]);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) x[i][e] = bits[i] >> e & 1 ? x[i][e] : (T)-INFINITY;
        if constexpr (STREAM)
            __builtin_nontemporal_store(x[i], (Piece *)(out + id));
        else
            *(Piece *)(out + id) = x[i];
    }
    // What is left before the first whole piece and behind the last.
    const int edge = tid < first - lo ? lo + tid : last + tid - (first - lo);
    if (edge < hi) {
        const bool on = !mask || (mask[edge >> 5] >> (edge & 31) & 1);
        const uint32_t n = counts ? seen[edge + word] : 0, entry = biased ? bias[edge + word] : 0;
        out[edge] = on ? one(in[edge], n, entry) : (T)-INFINITY;
    }
}

// What the L2 caches of the eight XCDs hold together.
constexpr long long L2_BYTES = 32 << 20;

template <typename T>
void launch_logits(LogitsArgs &a, hipStream_t stream) {
    // Ids of a workgroup: 2048, since more take LDS from the workgroups beside
    // it (512 rows of 50257, fp32, penalties, biases and masks: 4096 ids 48.7
    // us, 2048 41.6; bf16: 34.9 and 28.1), and fewer count the same history
    // more often. Few fp32 rows: 1024, so that more workgroups share a row's
    // latency. Results that do not fit the L2 caches are stored past them (48.2
    // -> 41.6 us).
    constexpr int MOST = sizeof(T) == 4 ? 2 : 1;
    const long long all = (long long)a.rows * a.V;
    const bool few = all < 512ll * chunk_of<T>(MOST);
    const bool past = all * (int)sizeof(T) > L2_BYTES;
    const int chunk = chunk_of<T>(few ? 1 : MOST);
    a.chunks = (a.V + chunk - 1) / chunk;
    const size_t words = chunk + 2 * piece_of<T>();
    const int tables = (a.r.tokens != nullptr) + (a.r.bias_offsets != nullptr);
    const size_t lds = tables * words * sizeof(uint32_t);
    const auto kernel = few    ? logits_kernel<T, 1, false>
                        : past ? logits_kernel<T, MOST, true>
                               : logits_kernel<T, MOST, false>;
    in_launches((long long)a.chunks * a.rows, THREADS, [&](long long first, unsigned n) {
        a.first = (int)first;
        launch(kernel, dim3(n), dim3(THREADS), lds, stream, a);
    });
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
    if ((V + 1023ll) / 1024 * rows > INT_MAX || V > INT_MAX - 16384)
        return refuse("too many logits for one call");
    LogitsArgs a = {*r, (char *)out, (const char *)logits, stride, rows, V, 0, 0};
    if (type == BMB_F32)
        launch_logits<float>(a, stream);
    else if (type == BMB_F16)
        launch_logits<_Float16>(a, stream);
    else
        launch_logits<__bf16>(a, stream);
    return 0;
}
