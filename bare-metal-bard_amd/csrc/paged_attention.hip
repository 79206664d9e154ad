// Attention of one new token a request over a paged key-value cache
// (paged_attention, include/flash.h).
//
// out = sum_j p_j v_j / sum_j p_j with p_j = 2^(x_j - max x), x_j = scale
// log2(e) q.k_j: one pass over the keys and values with a running maximum and
// sum. Every key and value is read once for all the query heads that share it,
// so the bound is the cache's bytes.
//
// A workgroup of four waves takes one part of a request's tokens for one kv
// head and up to 16 query heads. A wave takes STEP keys at a time and keeps
// everything in registers: the matrix cores' own layouts chain the two
// products. With lane = 16 g + c, a 16x16 product leaves lane (g, c) rows
// 4g..4g+3 of column c:
//   S^T = K Q^T   rows: keys, columns: heads. Lane (g, c) loads key c (16
//                 bytes at a time) and holds the scores of keys 4g..4g+3 for
//                 head c;
//   O^T = V^T P^T rows: head elements, contracted over keys, where the order
//                 of the keys is free: lane (g, c) contributes keys 4g..4g+3,
//                 whose probabilities it holds already, and the elements
//                 c*DPL..c*DPL+DPL-1 of their values, which are contiguous in
//                 memory; product j takes element j of each lane's.
// So neither the probabilities nor the values pass through LDS, and loads are
// whole rows.
#include "launch.hpp"
#include "paged.hpp"
#include "workspace.hpp"

namespace bmb {
namespace {

constexpr int WAVES = 4, THREADS = WAVES * WAVE, COLS = 16;
constexpr int UNIT = 128;  // a part is a whole number of these keys
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
template <typename T, int N>
using vec __attribute__((ext_vector_type(N))) = T;

struct AttendArgs {
    const char *q, *k, *v;
    char *out;
    float *lse;
    const int *table, *lens, *rows;
    float *part_o;     // (slots, heads, HS)
    float2 *part_ml;   // (slots, heads): running maximum (log2 units) and sum
    int2 *parts;       // (requests): first slot, number of parts
    long long page_stride, token_stride, head_stride, q_stride, out_stride;
    int requests, heads, kv_heads, group, tiles, pages, table_stride, max_len, n_rows;
    int slots;     // parts that the launch has room for
    int workers;   // parts aimed at; 0: one part a request
    float scale;   // times log2(e)
    FastDiv page;
};

// The part of a request that a slot stands for; n: how many the request has (0: none here).
struct Part {
    int r, i, n, begin, end, row;
};

__device__ __forceinline__ int row_of(const AttendArgs &a, int r) {
    const int row = a.rows ? a.rows[r] : r;
    return (unsigned)row < (unsigned)a.n_rows ? row : -1;
}

__device__ __forceinline__ int len_of(const AttendArgs &a, int r) {
    return min(max(a.lens[r], 0), a.max_len);
}

// All parts are of one length, ceil(total / workers) units, so that their work
// is alike whatever the lengths; the last part of each request is shorter.
// (Sum of ceil(len / part) <= requests + workers: the slots.) Every wave finds
// its slot's request by itself, 64 requests at a time.
__device__ __forceinline__ Part find_part(const AttendArgs &a, int slot) {
    const int lane = threadIdx.x & 63;
    Part p = {slot, 0, 0, 0, 0, -1};
    if (a.workers == 0) {
        p.row = row_of(a, slot);
        p.n = p.row >= 0;
        p.end = len_of(a, slot);
        return p;
    }
    uint32_t total = 0;
    for (int base = 0; base < a.requests; base += WAVE) {
        const int r = base + lane;
        uint32_t units = 0;
        if (r < a.requests && row_of(a, r) >= 0) units = (len_of(a, r) + UNIT - 1) / UNIT;
        total += __builtin_amdgcn_readlane(wave_scan(units), 63);
    }
    const uint32_t size = max((total + a.workers - 1) / a.workers, 1u);
    uint32_t before = 0;
    for (int base = 0; base < a.requests; base += WAVE) {
        const int r = base + lane;
        int len = 0, row = -1;
        uint32_t n = 0;
        if (r < a.requests) {
            row = row_of(a, r);
            len = len_of(a, r);
            if (row >= 0) n = max(((len + UNIT - 1) / UNIT + size - 1) / size, 1u);
        }
        const uint32_t upto = before + wave_scan(n);
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > (uint32_t)slot);
        if (past) {
            const int l = __builtin_ctzll(past);
            p.r = base + l;
            p.n = __builtin_amdgcn_readlane(n, l);
            p.i = slot - (int)(__builtin_amdgcn_readlane(upto, l) - p.n);
            p.row = __builtin_amdgcn_readlane(row, l);
            p.end = __builtin_amdgcn_readlane(len, l);
            const long long keys = (long long)size * UNIT;
            p.begin = (int)(p.i * keys);
            p.end = (int)min((long long)p.end, p.begin + keys);
            return p;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return p;
}

// Maximum (sum) over the four lanes g of a column: row pairs, then halves.
__device__ __forceinline__ float col_max(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float col_sum(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

__device__ __forceinline__ f32x4 mfma(vec<_Float16, 8> a, vec<_Float16, 8> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(vec<__bf16, 8> a, vec<__bf16, 8> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// What a wave holds of the queries and of one step's keys and values, and the
// two products on it. TILES groups of 16 keys a step.
//
// 16-bit cache and queries: 16-bit products (exact in fp32), 32 keys a step.
// The probabilities go in as a 16-bit rounding and the 16-bit rounding of what
// it left (2^-16 of a probability in bf16, 2^-22 in fp16): a single bf16 (2^-9)
// would add as much error as the result's own rounding, and the second product
// costs nothing beside the loads.
template <typename T, int HS>
struct Half {
    using Q = T;
    static constexpr int TILES = 2, KV = 4 * TILES, DPL = HS / 16;
    using V8 = vec<T, 8>;
    using Row = vec<uint32_t, DPL / 2>;
    struct Query {
        V8 q[HS / 32];
    };
    struct Regs {
        V8 k[TILES][HS / 32];
        Row v[KV];
    };
    static __device__ __forceinline__ void load_q(Query &q, const T *row, int g) {
        typedef V8 U __attribute__((aligned(4)));
        for (int s = 0; s < HS / 32; ++s) q.q[s] = *(const U *)(row + s * 32 + g * 8);
    }
    static __device__ __forceinline__ void zero_q(Query &q) {
        for (int s = 0; s < HS / 32; ++s) q.q[s] = (V8)(T)0.0f;
    }
    static __device__ __forceinline__ void load_k(Regs &x, int t, const char *row, int g) {
        for (int s = 0; s < HS / 32; ++s)
            x.k[t][s] = *(const V8 *)(row + (s * 32 + g * 8) * sizeof(T));
    }
    static __device__ __forceinline__ void load_v(Regs &x, int i, const char *row, int c) {
        x.v[i] = *(const Row *)(row + c * DPL * sizeof(T));
    }
    static __device__ __forceinline__ void zero_v(Regs &x, int i) { x.v[i] = (Row)0u; }
    static __device__ __forceinline__ f32x4 scores(const Regs &x, int t, const Query &q) {
        f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < HS / 32; ++i) s = mfma(x.k[t][i], q.q[i], s);
        return s;
    }
    static __device__ __forceinline__ void values(f32x4 (&o)[DPL], const Regs &x,
                                                  const float (&p)[KV]) {
        V8 hi, lo;
#pragma unroll
        for (int i = 0; i < KV; ++i) {
            hi[i] = (T)p[i];
            lo[i] = (T)(p[i] - (float)hi[i]);
        }
#pragma unroll
        for (int j = 0; j < DPL; ++j) {
            // element j of the lane's eight values, two to a register
            vec<uint32_t, 4> f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                f[i] = __builtin_amdgcn_perm(x.v[2 * i + 1][j / 2], x.v[2 * i][j / 2],
                                             j & 1 ? 0x07060302u : 0x05040100u);
            const V8 v = __builtin_bit_cast(V8, f);
            o[j] = mfma(v, hi, o[j]);
            o[j] = mfma(v, lo, o[j]);
        }
    }
};

// fp32 queries: fp32 products on 16x16x4 matrix instructions, the cache's
// 16-bit values widened in registers (exactly). 16 keys a step.
template <typename T, int HS>
struct Full {
    using Q = float;
    static constexpr int TILES = 1, KV = 4, DPL = HS / 16;
    static constexpr int EPL = 16 / sizeof(T);  // elements of a 16-byte load
    using VE = vec<T, EPL>;
    struct Query {
        float q[HS / 4];
    };
    struct Regs {
        VE k[TILES][HS / (4 * EPL)];
        vec<T, DPL> v[KV];
    };
    // Product (s, t) contracts elements s*4*EPL + g*EPL + t, g = 0..3.
    static __device__ __forceinline__ void load_q(Query &q, const float *row, int g) {
        typedef vec<float, EPL> U __attribute__((aligned(4)));
        for (int s = 0; s < HS / (4 * EPL); ++s) {
            const vec<float, EPL> x = *(const U *)(row + (s * 4 + g) * EPL);
            for (int t = 0; t < EPL; ++t) q.q[s * EPL + t] = x[t];
        }
    }
    static __device__ __forceinline__ void zero_q(Query &q) {
        for (int s = 0; s < HS / 4; ++s) q.q[s] = 0.0f;
    }
    static __device__ __forceinline__ void load_k(Regs &x, int t, const char *row, int g) {
        for (int s = 0; s < HS / (4 * EPL); ++s)
            x.k[t][s] = *(const VE *)(row + (s * 4 + g) * 16);
    }
    static __device__ __forceinline__ void load_v(Regs &x, int i, const char *row, int c) {
        x.v[i] = *(const vec<T, DPL> *)(row + c * DPL * sizeof(T));
    }
    static __device__ __forceinline__ void zero_v(Regs &x, int i) {
        x.v[i] = (vec<T, DPL>)(T)0.0f;
    }
    static __device__ __forceinline__ f32x4 scores(const Regs &x, int t, const Query &q) {
        f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < HS / (4 * EPL); ++i)
#pragma unroll
            for (int e = 0; e < EPL; ++e) s = mfma((float)x.k[t][i][e], q.q[i * EPL + e], s);
        return s;
    }
    static __device__ __forceinline__ void values(f32x4 (&o)[DPL], const Regs &x,
                                                  const float (&p)[KV]) {
#pragma unroll
        for (int i = 0; i < KV; ++i)
#pragma unroll
            for (int j = 0; j < DPL; ++j) o[j] = mfma((float)x.v[i][j], p[i], o[j]);
    }
};

// Loads the step of keys from kb on. Returns which of the lane's KV keys (4g +
// r of each 16) count. ALIGNED: 16 keys from a multiple of 16 on lie in one
// page, so a page id is read once, by the scalar unit, and keys behind `end`
// are read (inside their page) and left out; otherwise each lane looks its
// own keys' pages up.
template <typename P, bool ALIGNED>
__device__ __forceinline__ unsigned load_step(typename P::Regs &x, const AttendArgs &a,
                                              const int *table, const char *k, const char *v,
                                              int esize, int kb, int end, int g, int c) {
    unsigned live = 0;
#pragma unroll
    for (int t = 0; t < P::TILES; ++t) {
        const int base = kb + 16 * t;
        if constexpr (ALIGNED) {
            const int b = base < end ? base : 0;
            const int j = a.page.quot(b);
            int page = base < end ? table[j] : -1;
            const int n = (unsigned)page < (unsigned)a.pages ? min(end - base, 16) : 0;
            page = n > 0 ? page : 0;
            const long long at = page * a.page_stride + (b - j * (int)a.page.d) * a.token_stride;
            P::load_k(x, t, k + (at + c * a.token_stride) * esize, g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                P::load_v(x, 4 * t + r, v + (at + (4 * g + r) * a.token_stride) * esize, c);
                live |= (4 * g + r < n ? 1u : 0u) << (4 * t + r);
            }
        } else {
            const auto find = [&](int key, bool &ok) {
                const int n = key < end ? key : 0;
                const int j = a.page.quot(n);
                int page = key < end ? table[j] : -1;
                ok = (unsigned)page < (unsigned)a.pages;
                page = ok ? page : 0;
                return page * a.page_stride + (n - j * (int)a.page.d) * a.token_stride;
            };
            bool ok;
            P::load_k(x, t, k + find(base + c, ok) * esize, g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                P::load_v(x, 4 * t + r, v + find(base + 4 * g + r, ok) * esize, c);
                live |= (ok ? 1u : 0u) << (4 * t + r);
            }
        }
    }
    return live;
}

template <template <typename, int> class POLICY, typename TC, int HS, bool ALIGNED>
__global__ __launch_bounds__(THREADS) void attend_kernel(AttendArgs a) {
    using P = POLICY<TC, HS>;
    using TQ = typename P::Q;
    constexpr int STEP = 16 * P::TILES, DPL = P::DPL, KV = P::KV;
    __shared__ float part_ml[WAVES][2][COLS];
    __shared__ float part_o[WAVES][COLS][HS];

    // Workgroups go to the XCDs in turn: all heads of a slot on one of them,
    // since rows of neighbouring heads can share cache lines.
    const int per = 8 * a.kv_heads * a.tiles;
    const int in = blockIdx.x % per, slot = blockIdx.x / per * 8 + in % 8;
    if (slot >= a.slots) return;
    const int kv_head = in / 8 / a.tiles, tile = in / 8 % a.tiles;
    const Part part = find_part(a, slot);
    if (part.n == 0) return;

    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cols = min(a.group - tile * COLS, COLS);
    const int head0 = kv_head * a.group + tile * COLS;  // the first query head here
    const int *table = a.table + (size_t)part.r * a.table_stride;
    const char *k = a.k + kv_head * a.head_stride * (long long)sizeof(TC);
    const char *v = a.v + kv_head * a.head_stride * (long long)sizeof(TC);

    typename P::Query q;
    if (c < cols)
        P::load_q(q, (const TQ *)a.q + part.row * a.q_stride + (head0 + c) * HS, g);
    else
        P::zero_q(q);

    f32x4 o[DPL];
#pragma unroll
    for (int j = 0; j < DPL; ++j) o[j] = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;  // of column c; l of this lane's keys only
    for (int kb = part.begin + wave * STEP; kb < part.end; kb += WAVES * STEP) {
        typename P::Regs x;
        const unsigned live =
            load_step<P, ALIGNED>(x, a, table, k, v, sizeof(TC), kb, part.end, g, c);
        const bool whole = __builtin_amdgcn_ballot_w64(live != (1u << KV) - 1) == 0;
        float p[KV];
#pragma unroll
        for (int t = 0; t < P::TILES; ++t) {
            const f32x4 s = P::scores(x, t, q);
#pragma unroll
            for (int r = 0; r < 4; ++r) p[4 * t + r] = s[r] * a.scale;
        }
        if (!whole) {
            // What lies in an absent place may be NaN or infinite: the score
            // and the value are replaced, not multiplied by 0.
#pragma unroll
            for (int i = 0; i < KV; ++i) {
                const bool on = live >> i & 1;
                p[i] = on ? p[i] : -INFINITY;
                if (!on) P::zero_v(x, i);
            }
        }
        float top = p[0];
#pragma unroll
        for (int i = 1; i < KV; ++i) top = fmaxf(top, p[i]);
        const float m1 = fmaxf(m, col_max(top));
        const float ref = m1 == -INFINITY ? 0.0f : m1;  // no live score yet: all 2^-inf
        const float keep = __builtin_amdgcn_exp2f(m - ref);
        m = m1;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < KV; ++i) {
            p[i] = __builtin_amdgcn_exp2f(p[i] - ref);
            sum += p[i];
        }
        l = l * keep + sum;
#pragma unroll
        for (int j = 0; j < DPL; ++j) o[j] *= keep;
        P::values(o, x, p);
    }
    l = col_sum(l);

    // The four waves' results through LDS; the first to read a column's
    // maxima weighs each wave's share.
    if (g == 0) {
        part_ml[wave][0][c] = m;
        part_ml[wave][1][c] = l;
    }
    if (c < cols) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < DPL; ++j) part_o[wave][c][(4 * g + r) * DPL + j] = o[j][r];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < cols * HS; i += THREADS) {
        const int col = i / HS, d = i % HS;
        float top = part_ml[0][0][col];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) top = fmaxf(top, part_ml[w][0][col]);
        const float ref = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(part_ml[w][0][col] - ref);
            sum += f * part_ml[w][1][col];
            acc += f * part_o[w][col][d];
        }
        const int head = head0 + col;
        if (part.n == 1) {
            const float y = sum == 0.0f ? 0.0f : acc / sum;
            ((TQ *)a.out)[part.row * a.out_stride + head * HS + d] = (TQ)y;
            if (a.lse && d == 0)
                a.lse[(long long)part.row * a.heads + head] =
                    sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * LN2;
        } else {
            const long long at = (long long)slot * a.heads + head;
            a.part_o[at * HS + d] = acc;
            if (d == 0) a.part_ml[at] = make_float2(top, sum);
        }
    }
    if (a.workers && threadIdx.x == 0 && part.i == 0 && kv_head == 0 && tile == 0)
        a.parts[part.r] = make_int2(slot, part.n);
}

// Joins the parts of split requests: one workgroup a request and head.
template <typename TQ, int HS>
__global__ __launch_bounds__(THREADS) void join_kernel(AttendArgs a) {
    constexpr int LANES = HS / 4, SHARES = THREADS / LANES;
    __shared__ float4 acc_s[SHARES][LANES];
    __shared__ float sum_s[SHARES];
    const int r = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
    const int row = row_of(a, r);
    if (row < 0) return;
    const int2 parts = a.parts[r];
    if (parts.y < 2) return;
    const int d = threadIdx.x % LANES, share = threadIdx.x / LANES;
    const long long at = (long long)parts.x * a.heads + head;
    float top = -INFINITY;
    for (int i = 0; i < parts.y; ++i) top = fmaxf(top, a.part_ml[at + (long long)i * a.heads].x);
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    float4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = share; i < parts.y; i += SHARES) {
        const long long s = at + (long long)i * a.heads;
        const float2 ml = a.part_ml[s];
        const float f = __builtin_amdgcn_exp2f(ml.x - ref);
        const float4 x = ld4(a.part_o + s * HS + 4 * d);
        sum += f * ml.y;
        acc.x += f * x.x;
        acc.y += f * x.y;
        acc.z += f * x.z;
        acc.w += f * x.w;
    }
    acc_s[share][d] = acc;
    if (d == 0) sum_s[share] = sum;
    __syncthreads();
    if (share != 0) return;
    for (int i = 1; i < SHARES; ++i) {
        sum += sum_s[i];
        acc.x += acc_s[i][d].x;
        acc.y += acc_s[i][d].y;
        acc.z += acc_s[i][d].z;
        acc.w += acc_s[i][d].w;
    }
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    typedef vec<TQ, 4> U __attribute__((aligned(4)));
    const vec<TQ, 4> y = {(TQ)(acc.x * f), (TQ)(acc.y * f), (TQ)(acc.z * f), (TQ)(acc.w * f)};
    *(U *)((TQ *)a.out + row * a.out_stride + head * HS + 4 * d) = y;
    if (a.lse && d == 0)
        a.lse[(long long)row * a.heads + head] =
            sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * LN2;
}

// How a call is split, from what the host knows of it.
struct Split {
    int slots, workers;
    size_t ml_at, parts_at, bytes;  // offsets of the workspace's pieces; its size
};

constexpr int CUS = 256, WORKGROUPS_PER_CU = 4;
constexpr int WHOLE = 256;  // sequences up to this stay whole

Split split_of(const PagedCache &c, const PagedBatch &b) {
    Split s = {b.requests, 0, 0, 0, 0};
    const long long group = b.heads / c.kv_heads, tiles = (group + COLS - 1) / COLS;
    const long long rows = c.kv_heads * tiles;  // workgroups of one slot
    if (b.max_len > WHOLE) {
        long long workers = CUS * WORKGROUPS_PER_CU / rows;
        workers = workers < 1 ? 1 : workers;
        const long long units = (b.max_len + UNIT - 1) / UNIT;
        const long long most = b.requests * units;
        workers = workers < most ? workers : most;
        s.workers = (int)workers;
        const long long slots = b.requests + workers < most ? b.requests + workers : most;
        s.slots = (int)slots;
        const size_t o = (size_t)s.slots * b.heads * c.head_size * sizeof(float);
        const size_t ml = (size_t)s.slots * b.heads * sizeof(float2);
        s.ml_at = o;
        s.parts_at = o + ml;
        s.bytes = o + ml + (size_t)b.requests * sizeof(int2);
    }
    return s;
}

const char *batch_fault(const PagedCache *c, const PagedBatch *b) {
    if (const char *why = cache_fault(c)) return why;
    if (b == nullptr) return "no batch";
    if (b->requests < 1 || b->max_len < 0 || b->heads < 1 || b->n_rows < 1)
        return "a size is below its least";
    if (b->heads % c->kv_heads != 0) return "heads is no multiple of kv_heads";
    if (b->type != BMB_F32 && b->type != BMB_F16 && b->type != BMB_BF16)
        return "unknown element type";
    if (b->type != BMB_F32 && b->type != c->type)
        return "16-bit queries need a cache of their own type";
    if (((long long)b->max_len + c->page_size - 1) / c->page_size > b->table_stride)
        return "table_stride is less than max_len needs";
    if ((long long)b->requests * (b->max_len / UNIT + 1) > INT_MAX / 4 ||
        (long long)(b->requests + CUS * WORKGROUPS_PER_CU + 8) * b->heads > INT_MAX)
        return "too many requests for one call";
    const long long size = element_size(b->type);
    if (b->q_stride * size % 4 != 0 || b->out_stride * size % 4 != 0)
        return "rows are no multiples of 4 bytes";
    return nullptr;
}

template <template <typename, int> class POLICY, typename TC, int HS>
void launch_attend(const AttendArgs &a, hipStream_t stream) {
    using TQ = typename POLICY<TC, HS>::Q;
    const dim3 grid((unsigned)((a.slots + 7) / 8 * 8 * a.kv_heads * a.tiles)), block(THREADS);
    if (a.page.d % 16 == 0)
        launch(attend_kernel<POLICY, TC, HS, true>, grid, block, 0, stream, a);
    else
        launch(attend_kernel<POLICY, TC, HS, false>, grid, block, 0, stream, a);
    if (a.workers)
        launch(join_kernel<TQ, HS>, dim3((unsigned)(a.requests * a.heads)), block, 0, stream, a);
}

template <template <typename, int> class POLICY, typename TC>
void launch_attend(int hs, const AttendArgs &a, hipStream_t stream) {
    if (hs == 32)
        launch_attend<POLICY, TC, 32>(a, stream);
    else if (hs == 64)
        launch_attend<POLICY, TC, 64>(a, stream);
    else
        launch_attend<POLICY, TC, 128>(a, stream);
}

}  // namespace
}  // namespace bmb

extern "C" {

size_t paged_attention_workspace(const PagedCache *cache, const PagedBatch *batch) {
    if (bmb::batch_fault(cache, batch)) return 0;
    return bmb::split_of(*cache, *batch).bytes;
}

int paged_attention(const PagedCache *c, const PagedBatch *b, void *out, float *lse, const void *q,
                    hipStream_t stream) {
    using namespace bmb;
    const char *me = "paged_attention";
    if (const char *why = batch_fault(c, b)) return refuse(me, why);
    if (!out || !q || !b->block_table || !b->lens) return refuse(me, "a null pointer");
    if (((uintptr_t)q | (uintptr_t)out) % 4 != 0)
        return refuse(me, "rows are no multiples of 4 bytes");
    const Split s = split_of(*c, *b);
    char *work = (char *)b->work;
    if (work != nullptr && b->work_bytes < s.bytes) return refuse(me, "the workspace is too small");
    if ((uintptr_t)work % 16 != 0) return refuse(me, "the workspace is no multiple of 16 bytes");
    const bool lease = s.bytes > 0 && work == nullptr;
    if (lease && stream_capturing(stream))
        return refuse(me, "a call under graph capture needs a workspace of its caller's");
    ScratchLease ws(SCRATCH_PAGED, lease ? s.bytes : 0, stream);
    if (lease) {
        if (!ws) return refuse(me, "cannot allocate the workspace");
        work = (char *)ws.get();
    }
    const int group = b->heads / c->kv_heads;
    AttendArgs a = {(const char *)q, (const char *)c->k, (const char *)c->v, (char *)out, lse,
                    b->block_table, b->lens, b->rows, (float *)work, (float2 *)(work + s.ml_at),
                    (int2 *)(work + s.parts_at), c->page_stride, c->token_stride, c->head_stride,
                    b->q_stride, b->out_stride, b->requests, b->heads, c->kv_heads, group,
                    (group + COLS - 1) / COLS, c->pages, b->table_stride, b->max_len, b->n_rows,
                    s.slots, s.workers, b->scale * LOG2E, FastDiv::of(c->page_size)};
    const int hs = c->head_size;
    if (b->type == BMB_F16)
        launch_attend<Half, _Float16>(hs, a, stream);
    else if (b->type == BMB_BF16)
        launch_attend<Half, __bf16>(hs, a, stream);
    else if (c->type == BMB_F16)
        launch_attend<Full, _Float16>(hs, a, stream);
    else if (c->type == BMB_BF16)
        launch_attend<Full, __bf16>(hs, a, stream);
    else
        launch_attend<Full, float>(hs, a, stream);
    return 0;
}

}  // extern "C"
