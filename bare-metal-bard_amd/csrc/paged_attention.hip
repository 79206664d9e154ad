// Attention of one new token a request over a paged key-value cache
// (paged_attention, include/flash.h).
//
// out = sum_j p_j v_j / sum_j p_j with p_j = 2^(x_j - max x), x_j = scale
// log2(e) q.k_j: one pass over the keys and values with a running maximum and
// sum. Every key and value is read once for all the query heads that share it,
// so the bound is the cache's bytes.
//
// Measured: two contexts of 131072 tokens, 8 kv heads of 128 in bf16 (1.07 GB)
// 175 us back to back in a graph, 6.1 TB/s; an fp32 cache (460 MB) 6.1 TB/s; a
// plain copy moves 5.1 TB/s here. A single sequence of 1000 tokens takes 7.6 us
// in two launches: latency.
//
// A workgroup of four waves takes one part of a request's tokens for one kv
// head and up to 16 (or 32) query heads. A wave takes STEP keys at a time and
// keeps everything in registers: the matrix cores' own layouts chain the two
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
#include <optional>

#include "launch.hpp"
#include "paged.hpp"
#include "workspace.hpp"

namespace bmb {
namespace {

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
    int4 *parts;       // (requests): whole parts' first slot and number, the rest's slot or -1
    long long page_stride, token_stride, head_stride, q_stride, out_stride;
    int requests, heads, kv_heads, group, tiles, pages, table_stride, max_len, n_rows;
    int slots;          // parts that the launch has room for
    int workers;        // most parts; 0: one part a request
    int few;            // parts that give each CU a workgroup
    int least, enough;  // units of a part: at least; more than `enough` only past `few` parts
    int cached;         // units that stay in the caches; without workers: whether they do
    int first;          // the launch's first workgroup of the call's
    float scale;        // times log2(e)
    FastDiv page;
    uint32_t page16, token16;  // strides in units of 16 bytes
};

// The part of a request that a slot stands for; n: how many the request has (0: none here).
struct Part {
    int r, i, n, whole, begin, end, row;  // (whole: those of full length, which come first)
    bool nt;  // the step's batch passes the caches
};

__device__ __forceinline__ int row_of(const AttendArgs &a, int r) {
    const int row = a.rows ? a.rows[r] : r;
    return (unsigned)row < (unsigned)a.n_rows ? row : -1;
}

__device__ __forceinline__ int len_of(const AttendArgs &a, int r) {
    return min(max(a.lens[r], 0), a.max_len);
}

// A request's tokens, in units, and how they come apart: whole parts of `size` units
// and a rest (an empty sequence is one empty rest).
struct Asks {
    int row, len;
    uint32_t units, whole, rest;
};
__device__ __forceinline__ Asks asks_of(const AttendArgs &a, int r, uint32_t size) {
    Asks x = {-1, 0, 0, 0, 0};
    if (r < a.requests) {
        x.row = row_of(a, r);
        x.len = len_of(a, r);
    }
    if (x.row < 0) return x;
    x.units = (x.len + UNIT - 1) / UNIT;
    x.whole = x.units / size;
    x.rest = x.whole * size < x.units || x.units == 0;
    return x;
}

// All parts are of one length, `size` units, whatever the sequences' lengths, but
// for what is left of each sequence; those rests (and the sequences shorter than a
// part) come behind the whole parts, so that the device ends on the short ones.
// (Sum of ceil(len / part) <= requests + workers: the slots.) Every wave finds its
// slot's request by itself: each lane counts a share of the requests, which takes
// three scans however many they are, then the wave looks into the share that holds
// the slot. (Rests among the whole parts: 16 sequences of 3000-4000 tokens 79.5 us,
// behind them 76.1; 256 requests, 64 to a scan: 81.3 us, in shares 78.2.)
__device__ __forceinline__ Part find_part(const AttendArgs &a, int slot) {
    const int lane = threadIdx.x & 63;
    Part p = {slot, 0, 0, 0, 0, 0, -1, a.cached == 0 && a.tiles == 1};
    if (a.workers == 0) {
        p.row = row_of(a, slot);
        p.n = p.row >= 0;
        p.end = len_of(a, slot);
        return p;
    }
    const int share = (a.requests + WAVE - 1) / WAVE;
    uint32_t units = 0;
    for (int i = 0; i < share; ++i) units += asks_of(a, lane * share + i, 1).units;
    const uint32_t total = __builtin_amdgcn_readlane(wave_scan(units), 63);
    p.nt = total >= (uint32_t)a.cached && a.tiles == 1;  // (several tiles read the same rows)
    uint32_t size = (total + a.workers - 1) / a.workers;
    size = max(size, min((total + a.few - 1) / a.few, (uint32_t)a.enough));
    size = max(size, (uint32_t)a.least);

    uint32_t whole = 0, rest = 0;
    Asks x;
    for (int i = 0; i < share; ++i) {
        x = asks_of(a, lane * share + i, size);
        whole += x.whole;
        rest += x.rest;
    }
    const uint32_t whole_upto = wave_scan(whole), rest_upto = wave_scan(rest);
    const uint32_t all_whole = __builtin_amdgcn_readlane(whole_upto, 63);
    const bool rests = (uint32_t)slot >= all_whole;
    uint32_t left = rests ? slot - all_whole : slot;  // slots before this one, from here on
    const uint32_t upto = rests ? rest_upto : whole_upto;
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > left);
    if (past == 0) return p;
    int l = __builtin_ctzll(past);
    left -= __builtin_amdgcn_readlane(upto - (rests ? rest : whole), l);
    p.r = l * share;
    if (share > 1) {
        for (int base = 0;; base += WAVE) {  // (ends: the share holds the slot)
            x = asks_of(a, base + lane < share ? p.r + base + lane : a.requests, size);
            const uint32_t n = rests ? x.rest : x.whole, sum = wave_scan(n);
            const uint64_t here = __builtin_amdgcn_ballot_w64(sum > left);
            l = here ? __builtin_ctzll(here) : 63;
            left -= __builtin_amdgcn_readlane(here ? sum - n : sum, l);
            if (here || base + WAVE >= share) {
                p.r += base + l;
                break;
            }
        }
    }
    p.whole = __builtin_amdgcn_readlane(x.whole, l);
    p.n = p.whole + __builtin_amdgcn_readlane(x.rest, l);
    p.i = rests ? p.whole : left;
    p.row = __builtin_amdgcn_readlane(x.row, l);
    p.end = __builtin_amdgcn_readlane(x.len, l);
    const long long keys = (long long)size * UNIT;
    p.begin = (int)(p.i * keys);
    p.end = (int)min((long long)p.end, p.begin + keys);
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

// A load of the cache. NT: not kept in the caches behind it (non-temporal), for
// batches that do not fit them anyway.
// A wave-uniform base and 32 bits of each lane's own: no address arithmetic
// in the vector unit.
template <bool NT, typename R>
__device__ __forceinline__ R load(const char *p, uint32_t lane) {
    if constexpr (NT)
        return __builtin_nontemporal_load((const R *)(p + lane));
    else
        return *(const R *)(p + lane);
}

// What a wave holds of the queries and of one step's keys and values, and the
// two products on it. TILES groups of 16 keys a step.
//
// 16-bit cache and queries: 16-bit products (exact in fp32), 32 keys a step.
// The probabilities go in as a 16-bit rounding and the 16-bit rounding of what
// it left: a single bf16 would add as much error as the result's own rounding,
// and the second product costs nothing beside the loads. What the two lose is
// at most 2^-17 of a probability in bf16 and 2^-23 in fp16, or there, if that is
// more, 2^-40 of the largest: fp16 holds nothing below 2^-24, so probabilities
// (at most 1) go in times 2^15, which the sums carry until the wave's end.
template <typename T, int HS>
struct Half {
    using Q = T;
    static constexpr int SIZE = sizeof(T);
    static constexpr int TILES = 2, KV = 4 * TILES, DPL = HS / 16;
    static constexpr float P_SCALE = __is_same(T, _Float16) ? 0x1p15f : 1.0f;
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
    template <bool NT>
    static __device__ __forceinline__ void load_k(Regs &x, int t, const char *p, uint32_t lane) {
        for (int s = 0; s < HS / 32; ++s)
            x.k[t][s] = load<NT, V8>(p + s * 64, lane);
    }
    template <bool NT>
    static __device__ __forceinline__ void load_v(Regs &x, int i, const char *p, uint32_t lane) {
        x.v[i] = load<NT, Row>(p, lane);
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
            const float x = p[i] * P_SCALE;
            hi[i] = (T)x;
            lo[i] = (T)(x - (float)hi[i]);
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
    static constexpr int SIZE = sizeof(T);
    // (32 keys of 16-bit heads of 128 take too many registers: 64 -> 82 us.)
    static constexpr int TILES = sizeof(T) == 2 && HS <= 64 ? 2 : 1, KV = 4 * TILES, DPL = HS / 16;
    static constexpr float P_SCALE = 1.0f;
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
    template <bool NT>
    static __device__ __forceinline__ void load_k(Regs &x, int t, const char *p, uint32_t lane) {
        for (int s = 0; s < HS / (4 * EPL); ++s)
            x.k[t][s] = load<NT, VE>(p + s * 64, lane);
    }
    template <bool NT>
    static __device__ __forceinline__ void load_v(Regs &x, int i, const char *p, uint32_t lane) {
        x.v[i] = load<NT, vec<T, DPL>>(p, lane);
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

// The pages of one step's keys, read one step ahead of their rows. ALIGNED: 16
// keys from a multiple of 16 on lie in one page, so a page id is read once a
// tile, by the scalar unit. Otherwise each lane looks up one of the step's keys
// and the lanes exchange the rows' places (in units of 16 bytes, as every
// stride is a multiple of that): with every lane looking up the pages of its
// own rows, pages of 24 keys took 137 us where pages of 16 took 99 (16
// sequences of 16000 keys, 4 heads of 128, bf16).
constexpr uint32_t NO_ROW = 0xffffffffu;
template <bool ALIGNED, int TILES>
struct Pages {
    int id[ALIGNED ? TILES : 1];
    // (Steps behind `end`, which is at least 1, look up the last tile or key
    // again: a branch here would have the scalar loads waited for at once.)
    static __device__ __forceinline__ int tile_at(int t, int kb, int end) {
        return min(kb + 16 * t, (end - 1) & ~15);
    }
    static __device__ __forceinline__ int key_at(int kb) {
        return kb + (int)(threadIdx.x & (16 * TILES - 1));
    }
    __device__ __forceinline__ void fetch(const AttendArgs &a, const int *table, int kb, int end) {
        if constexpr (ALIGNED) {
#pragma unroll
            for (int t = 0; t < TILES; ++t) id[t] = table[a.page.quot(tile_at(t, kb, end))];
        } else {
            id[0] = table[a.page.quot(min(key_at(kb), end - 1))];
        }
    }
    // Not ALIGNED: the place of this lane's key.
    __device__ __forceinline__ uint32_t place(const AttendArgs &a, int kb, int end) const {
        const int key = key_at(kb);
        const uint32_t in = key - a.page.quot(key) * (int)a.page.d;
        const bool ok = key < end && (unsigned)id[0] < (unsigned)a.pages;
        return ok ? id[0] * a.page16 + in * a.token16 : NO_ROW;
    }
    // ALIGNED: bytes to a tile's first key, and how many of its keys count (with
    // none, the rows that are read all the same are some of the cache's).
    __device__ __forceinline__ long long tile(const AttendArgs &a, int t, int kb, int end,
                                              int esize, int &n) const {
        const int base = tile_at(t, kb, end), in = base - a.page.quot(base) * (int)a.page.d;
        const bool ok = (unsigned)id[t] < (unsigned)a.pages;
        n = ok ? min(end - (kb + 16 * t), 16) : 0;
        return ((ok ? id[t] : 0) * a.page_stride + in * a.token_stride) * esize;
    }
};

// Which keys of a step count.
template <bool ALIGNED, int TILES>
struct Live {
    bool whole;  // all of them, for every lane
    int n[TILES];   // ALIGNED: the first n of each tile
    uint32_t bits;  // otherwise: by this lane's keys
    // Of this lane's 4 * TILES keys, of which the r-th of a tile is its key
    // `first` + r * `step`.
    __device__ __forceinline__ uint32_t mask(int first, int step) const {
        if constexpr (!ALIGNED) return bits;
        uint32_t m = 0;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) m |= (first + r * step < n[t] ? 1u : 0u) << (4 * t + r);
        return m;
    }
};

// Loads the step of keys from kb on. k and v: a row's start in the cache's first
// page, for the wave.
template <typename P, bool ALIGNED, bool NT>
__device__ __forceinline__ Live<ALIGNED, P::TILES> load_step(typename P::Regs &x,
                                                             const AttendArgs &a,
                                                             const Pages<ALIGNED, P::TILES> &pages,
                                                             const char *k, const char *v, int kb,
                                                             int end, int g, int c) {
    Live<ALIGNED, P::TILES> live = {true, {}, 0};
    const uint32_t row = (uint32_t)a.token_stride * P::SIZE;
    const uint32_t k_at = g * 16, v_at = c * P::DPL * P::SIZE;  // in a row
    if constexpr (ALIGNED) {
#pragma unroll
        for (int t = 0; t < P::TILES; ++t) {
            const long long at = pages.tile(a, t, kb, end, P::SIZE, live.n[t]);
            live.whole &= live.n[t] == 16;
            P::template load_k<NT>(x, t, k + at, c * row + k_at);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                P::template load_v<NT>(x, 4 * t + r, v + at + r * (size_t)row, 4 * g * row + v_at);
        }
    } else {
        const uint32_t place = pages.place(a, kb, end);
#pragma unroll
        for (int t = 0; t < P::TILES; ++t) {
            const uint32_t at = __shfl(place, 16 * t + c);
            P::template load_k<NT>(x, t, k + (at == NO_ROW ? 0ull : at * 16ull), k_at);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t to = __shfl(place, 16 * t + 4 * g + r);
                P::template load_v<NT>(x, 4 * t + r, v + (to == NO_ROW ? 0ull : to * 16ull), v_at);
                live.bits |= (to != NO_ROW ? 1u : 0u) << (4 * t + r);
            }
        }
        live.whole = __builtin_amdgcn_ballot_w64(place == NO_ROW) == 0;
    }
    return live;
}

// LDS of a workgroup: each wave's running maxima and sums, and its share of
// the result for the columns in use, `used` of `cols`.
constexpr size_t merge_bytes(int waves, int cols, int used, int hs) {
    return (size_t)waves * (2 * cols + used * hs) * sizeof(float);
}

// The waves' results, each weighed by its maximum: to the result, or as a part
// of a split request.
template <typename TQ, int HS, int WAVES, int COLS>
__device__ __forceinline__ void merge_waves(const AttendArgs &a, const Part &part, int slot,
                                            int head0, int cols) {
    extern __shared__ float merge[];
    const float(*part_ml)[2][COLS] = (const float(*)[2][COLS])merge;
    const float *part_o = merge + WAVES * 2 * COLS;
    __syncthreads();
    for (int i = threadIdx.x; i < cols * HS; i += WAVES * WAVE) {
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
            acc += f * part_o[w * cols * HS + i];
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
    if (a.workers && threadIdx.x == 0 && head0 == 0) {
        int4 &parts = a.parts[part.r];
        if (part.i == part.whole) parts.z = slot;
        if (part.i == 0) {
            parts.x = slot;
            parts.y = part.whole;
            if (part.n == part.whole) parts.z = -1;
        }
    }
}

// A wave's share of a part: steps of keys from `first` on, `step` apart, for QT
// groups of 16 query heads.
template <typename P, bool ALIGNED, bool NT, int QT>
__device__ __forceinline__ void attend_steps(f32x4 (&o)[QT][P::DPL], float (&m)[QT], float (&l)[QT],
                                             const AttendArgs &a, const Part &part,
                                             const typename P::Query (&q)[QT], const int *table,
                                             const char *k, const char *v, int first, int step,
                                             int g, int c) {
    constexpr int DPL = P::DPL, KV = P::KV;
    Pages<ALIGNED, P::TILES> pages, next;
    if (part.begin + first >= part.end) return;
    pages.fetch(a, table, part.begin + first, part.end);
    for (int kb = part.begin + first; kb < part.end; kb += step, pages = next) {
        typename P::Regs x;
        next.fetch(a, table, kb + step, part.end);
        const auto live = load_step<P, ALIGNED, NT>(x, a, pages, k, v, kb, part.end, g, c);
        const bool whole = live.whole;
        const uint32_t on = whole ? 0u : live.mask(4 * g, 1);
        if (!whole) {
            // What lies in an absent place may be NaN or infinite: the value
            // (and the score, below) is replaced, not multiplied by 0.
#pragma unroll
            for (int i = 0; i < KV; ++i)
                if (!(on >> i & 1)) P::zero_v(x, i);
        }
#pragma unroll
        for (int u = 0; u < QT; ++u) {
            float p[KV];
#pragma unroll
            for (int t = 0; t < P::TILES; ++t) {
                const f32x4 s = P::scores(x, t, q[u]);
#pragma unroll
                for (int r = 0; r < 4; ++r) p[4 * t + r] = s[r] * a.scale;
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < KV; ++i) p[i] = on >> i & 1 ? p[i] : -INFINITY;
            }
            float top = p[0];
#pragma unroll
            for (int i = 1; i < KV; ++i) top = fmaxf(top, p[i]);
            const float m1 = fmaxf(m[u], col_max(top));
            const float ref = m1 == -INFINITY ? 0.0f : m1;  // no live score yet: all 2^-inf
            const float keep = __builtin_amdgcn_exp2f(m[u] - ref);
            m[u] = m1;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < KV; ++i) {
                p[i] = __builtin_amdgcn_exp2f(p[i] - ref);
                sum += p[i];
            }
            l[u] = l[u] * keep + sum;
#pragma unroll
            for (int j = 0; j < DPL; ++j) o[u][j] *= keep;
            P::values(o[u], x, p);
        }
    }
}

// (QT = 2, for more than 16 query heads a kv head: 32 heads on 16 x 16000 keys
// of 128 in bf16 191 us in two workgroups of 16, 156 in one.)
template <template <typename, int> class POLICY, typename TC, int HS, bool ALIGNED, int QT>
__global__ __launch_bounds__(256) void attend_kernel(AttendArgs a) {
    using P = POLICY<TC, HS>;
    using TQ = typename P::Q;
    constexpr int WAVES = 4, STEP = 16 * P::TILES, DPL = P::DPL, COLS = 16 * QT;
    extern __shared__ float merge[];
    float *part_ml = merge;                     // (wave, maximum and sum, column)
    float *part_o = merge + WAVES * 2 * COLS;  // (wave, column, element)

    // Workgroups go to the XCDs in turn: all heads of a slot on one of them,
    // since rows of neighbouring heads can share cache lines.
    const uint32_t per = 8 * a.kv_heads * a.tiles, block = a.first + blockIdx.x;
    const int in = block % per, slot = block / per * 8 + in % 8;
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

    typename P::Query q[QT];
    f32x4 o[QT][DPL];
    float m[QT], l[QT];  // of column c; l of this lane's keys only
#pragma unroll
    for (int u = 0; u < QT; ++u) {
        const int col = 16 * u + c;
        if (col < cols)
            P::load_q(q[u], (const TQ *)a.q + part.row * a.q_stride + (head0 + col) * HS, g);
        else
            P::zero_q(q[u]);
#pragma unroll
        for (int j = 0; j < DPL; ++j) o[u][j] = {0.0f, 0.0f, 0.0f, 0.0f};
        m[u] = -INFINITY;
        l[u] = 0.0f;
    }
    if (part.nt)
        attend_steps<P, ALIGNED, true, QT>(o, m, l, a, part, q, table, k, v, wave * STEP,
                                           WAVES * STEP, g, c);
    else
        attend_steps<P, ALIGNED, false, QT>(o, m, l, a, part, q, table, k, v, wave * STEP,
                                            WAVES * STEP, g, c);
#pragma unroll
    for (int u = 0; u < QT; ++u) {
        const int col = 16 * u + c;
        const float sum = col_sum(l[u]);
        if (g == 0) {
            part_ml[(wave * 2 + 0) * COLS + col] = m[u];
            part_ml[(wave * 2 + 1) * COLS + col] = sum;
        }
        if (col < cols) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < DPL; ++j)
                    part_o[(wave * cols + col) * HS + (4 * g + r) * DPL + j] =
                        o[u][j][r] * (1.0f / P::P_SCALE);
        }
    }
    merge_waves<TQ, HS, WAVES, COLS>(a, part, slot, head0, cols);
}

// ---- few query heads to a kv head, fp32 queries: 16 matrix columns would
// mostly be empty, and fp32 matrix instructions have no rate to spare (one CU
// a head, 1000 fp32 keys of 64: 16.9 us with them, 10.2 so; 16 x 8000 keys of
// 128 in fp32, groups of 4: 128 and 93 us). Sixteen lanes take a key, each
// HS/16 of its elements, so a wave's load is four whole rows; KEYS loads make a
// step, lane (g, c) with keys 4 i + g. A key's partial sums are added over its
// lanes while they are spread over them (half of the keys kept, half sent, at
// each step), which leaves lane c with the score of key i = c mod KEYS; the
// probabilities come back for the values' sums as broadcasts of a lane over
// its row of 16. Each row of 16 lanes keeps its own running maximum.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
constexpr int XOR1 = 0xB1, XOR2 = 0x4E, XOR7 = 0x141, ROR4 = 0x124, ROR8 = 0x128;

// s[0..N-1] of each lane to the sums over lanes: lanes whose `up` bit is set
// keep the upper half.
template <int CTRL, int N>
__device__ __forceinline__ void halve(float *s, bool up) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float keep = up ? s[i + N / 2] : s[i], send = up ? s[i] : s[i + N / 2];
        s[i] = keep + dpp<CTRL>(send);
    }
}
// (The partners 8, 7, 2 and 1 apart, as exclusive or, reach all sixteen lanes,
// and each pair still holds the same keys when it meets.)
template <int KEYS>
__device__ __forceinline__ float spread_sum(float (&s)[KEYS], int c) {
    if constexpr (KEYS == 16) halve<ROR8, 16>(s, c & 8);
    if constexpr (KEYS >= 8) halve<XOR7, 8>(s, c & 4);
    halve<XOR2, 4>(s, c & 2);
    halve<XOR1, 2>(s, c & 1);
    float x = s[0];
    if constexpr (KEYS == 4) x += dpp<ROR4>(x);
    if constexpr (KEYS <= 8) x += dpp<ROR8>(x);
    return x;
}
template <int KEYS>
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, dpp<XOR1>(x));
    x = fmaxf(x, dpp<XOR2>(x));
    if constexpr (KEYS >= 8) x = fmaxf(x, dpp<XOR7>(x));
    if constexpr (KEYS == 16) x = fmaxf(x, dpp<ROR8>(x));
    return x;
}

template <int I, int KEYS, int DPL, typename Row>
__device__ __forceinline__ void add_values(float *acc, float p, const Row (&v)[KEYS]) {
    if constexpr (I < KEYS) {
        const float w = dpp<0x150 + I>(p);
#pragma unroll
        for (int j = 0; j < DPL; ++j) acc[j] = fma_rn(w, (float)v[I][j], acc[j]);
        add_values<I + 1, KEYS, DPL>(acc, p, v);
    }
}

// Lane c's HS/16 elements of a row: contiguous, or two pieces of 16 bytes half a
// row apart, so that each load covers whole lines.
template <typename T, int HS>
__device__ __forceinline__ constexpr int row_at(int c, int j) {
    constexpr int DPL = HS / 16, E = 16 / sizeof(T);
    return DPL <= E ? c * DPL + j : (j / E) * (HS / 2) + c * E + j % E;
}
template <typename T, int HS, bool NT>
__device__ __forceinline__ vec<T, HS / 16> load_row(const char *p, uint32_t lane) {
    constexpr int DPL = HS / 16, E = 16 / sizeof(T);
    if constexpr (DPL <= E) {
        return load<NT, vec<T, DPL>>(p, lane);
    } else {
        const vec<T, E> x = load<NT, vec<T, E>>(p, lane);
        const vec<T, E> y = load<NT, vec<T, E>>(p + HS / 2 * sizeof(T), lane);
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// A step's rows of K and V, and which of the lane's keys (kb + 4 i + g) count; as
// load_step.
template <typename T, int HS, int KEYS, bool ALIGNED, bool NT>
__device__ __forceinline__ Live<ALIGNED, KEYS / 4> load_rows(
    vec<T, HS / 16> (&kr)[KEYS], vec<T, HS / 16> (&vr)[KEYS], const AttendArgs &a,
    const Pages<ALIGNED, KEYS / 4> &pages, const char *k, const char *v, int kb, int end, int g,
    int c) {
    Live<ALIGNED, KEYS / 4> live = {true, {}, 0};
    const uint32_t row = (uint32_t)a.token_stride * (uint32_t)sizeof(T);
    const uint32_t in_row = row_at<T, HS>(c, 0) * sizeof(T);
    if constexpr (ALIGNED) {
#pragma unroll
        for (int t = 0; t < KEYS / 4; ++t) {
            const long long at = pages.tile(a, t, kb, end, sizeof(T), live.n[t]);
            live.whole &= live.n[t] == 16;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const size_t to = at + 4 * r * (size_t)row;
                kr[4 * t + r] = load_row<T, HS, NT>(k + to, g * row + in_row);
                vr[4 * t + r] = load_row<T, HS, NT>(v + to, g * row + in_row);
            }
        }
    } else {
        const uint32_t place = pages.place(a, kb, end);
#pragma unroll
        for (int i = 0; i < KEYS; ++i) {
            const uint32_t at = __shfl(place, 4 * i + g);
            const size_t to = at == NO_ROW ? 0 : at * (size_t)16;
            kr[i] = load_row<T, HS, NT>(k + to, in_row);
            vr[i] = load_row<T, HS, NT>(v + to, in_row);
            live.bits |= (at != NO_ROW ? 1u : 0u) << i;
        }
        live.whole = __builtin_amdgcn_ballot_w64(place == NO_ROW) == 0;
    }
    return live;
}

template <typename T, int HS, int G, int KEYS, bool ALIGNED, bool NT>
__device__ __forceinline__ void rows_steps(float (&acc)[G][HS / 16], float (&m)[G], float (&l)[G],
                                           const AttendArgs &a, const Part &part,
                                           const float (&q)[G][HS / 16], const int *table,
                                           const char *k, const char *v, int first, int step,
                                           int g, int c) {
    constexpr int DPL = HS / 16;
    using Row = vec<T, DPL>;
    Pages<ALIGNED, KEYS / 4> pages, next;
    if (part.begin + first >= part.end) return;
    pages.fetch(a, table, part.begin + first, part.end);
    for (int kb = part.begin + first; kb < part.end; kb += step, pages = next) {
        Row kr[KEYS], vr[KEYS];
        next.fetch(a, table, kb + step, part.end);
        const auto live =
            load_rows<T, HS, KEYS, ALIGNED, NT>(kr, vr, a, pages, k, v, kb, part.end, g, c);
        const bool whole = live.whole;
        const uint32_t on = whole ? 0u : live.mask(g, 4);
        if (!whole) {
            // (the value itself is replaced: 0 times an infinity is no 0)
#pragma unroll
            for (int i = 0; i < KEYS; ++i)
                if (!(on >> i & 1)) vr[i] = (Row)(T)0.0f;
        }
#pragma unroll
        for (int h = 0; h < G; ++h) {
            float s[KEYS];
#pragma unroll
            for (int i = 0; i < KEYS; ++i) {
                s[i] = q[h][0] * (float)kr[i][0];
#pragma unroll
                for (int j = 1; j < DPL; ++j) s[i] = fma_rn(q[h][j], (float)kr[i][j], s[i]);
            }
            float x = spread_sum<KEYS>(s, c);
            if (!whole) x = on >> (c & (KEYS - 1)) & 1 ? x : -INFINITY;
            const float m1 = fmaxf(m[h], row_max<KEYS>(x));
            const float ref = m1 == -INFINITY ? 0.0f : m1;
            const float keep = __builtin_amdgcn_exp2f(m[h] - ref);
            const float p = __builtin_amdgcn_exp2f(x - ref);
            m[h] = m1;
            l[h] = l[h] * keep + p;
#pragma unroll
            for (int j = 0; j < DPL; ++j) acc[h][j] *= keep;
            add_values<0, KEYS, DPL>(acc[h], p, vr);
        }
    }
}

template <typename T, int HS, int G, bool ALIGNED, int WAVES>
__global__ __launch_bounds__(WAVES *WAVE) void attend_rows_kernel(AttendArgs a) {
    constexpr int DPL = HS / 16, BYTES = DPL * sizeof(T);
    // Loads of a step, by a row's bytes a lane. Smaller steps start sooner and
    // leave registers for more waves, until the loads in flight are too few
    // (64 ragged sequences of bf16 heads of 64: 16 loads 13.7 us, 8 12.5; one
    // short one 3.8 and 3.1; heads of 32: 16 20.9, 8 21.8, 4 27.6).
    constexpr int KEYS = BYTES == 4 ? 16 : BYTES == 8 || (BYTES == 16 && sizeof(T) == 4) ? 8 : 4;
    constexpr int STEP = 4 * KEYS;
    extern __shared__ float merge[];
    float(*part_ml)[2][G] = (float(*)[2][G])merge;
    float *part_o = merge + WAVES * 2 * G;  // (wave, head, element)

    const uint32_t per = 8 * a.kv_heads * a.tiles, block = a.first + blockIdx.x;
    const int in = block % per, slot = block / per * 8 + in % 8;
    if (slot >= a.slots) return;
    const int kv_head = in / 8 / a.tiles, tile = in / 8 % a.tiles;
    const Part part = find_part(a, slot);
    if (part.n == 0) return;

    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cols = min(a.group - tile * G, G);
    const int head0 = kv_head * a.group + tile * G;
    const int *table = a.table + (size_t)part.r * a.table_stride;
    const char *k = a.k + kv_head * a.head_stride * (int)sizeof(T);
    const char *v = a.v + kv_head * a.head_stride * (int)sizeof(T);

    float q[G][DPL], acc[G][DPL], m[G], l[G];
#pragma unroll
    for (int h = 0; h < G; ++h) {
        const float *row = (const float *)a.q + part.row * a.q_stride +
                           (head0 + min(h, cols - 1)) * HS;
#pragma unroll
        for (int j = 0; j < DPL; ++j) {
            q[h][j] = row[row_at<T, HS>(c, j)] * a.scale;
            acc[h][j] = 0.0f;
        }
        m[h] = -INFINITY;
        l[h] = 0.0f;
    }
    if (part.nt)
        rows_steps<T, HS, G, KEYS, ALIGNED, true>(acc, m, l, a, part, q, table, k, v, wave * STEP,
                                                  WAVES * STEP, g, c);
    else
        rows_steps<T, HS, G, KEYS, ALIGNED, false>(acc, m, l, a, part, q, table, k, v, wave * STEP,
                                                   WAVES * STEP, g, c);
    // The four rows of the wave into one.
#pragma unroll
    for (int h = 0; h < G; ++h) {
        const float top = col_max(m[h]);
        const float f = __builtin_amdgcn_exp2f(m[h] - (top == -INFINITY ? 0.0f : top));
        float sum = l[h] * f;  // of this lane's key: 16 / KEYS lanes have the same
        sum += dpp<XOR1>(sum);
        sum += dpp<XOR2>(sum);
        sum += dpp<ROR4>(sum);
        sum += dpp<ROR8>(sum);
        sum = col_sum(sum) * (KEYS / 16.0f);
#pragma unroll
        for (int j = 0; j < DPL; ++j) acc[h][j] = col_sum(acc[h][j] * f);
        if (h < cols && g == 0) {
            if (c == 0) {
                part_ml[wave][0][h] = top;
                part_ml[wave][1][h] = sum;
            }
#pragma unroll
            for (int j = 0; j < DPL; ++j)
                part_o[(wave * cols + h) * HS + row_at<T, HS>(c, j)] = acc[h][j];
        }
    }
    merge_waves<float, HS, WAVES, G>(a, part, slot, head0, cols);
}

// Joins the parts of split requests: one workgroup a request and head. The
// request's number of parts is not known before its lens are, so the launch
// covers all; a request of one part is done already. Each share of the threads
// takes every SHARES-th part and keeps its own running maximum, so the parts'
// maxima and results are loaded together (the 128 parts of two long contexts: 25
// us with the maximum found first, by one thread after another, 7 so).
constexpr int JOIN_THREADS = 256;
template <typename TQ, int HS>
__global__ __launch_bounds__(JOIN_THREADS) void join_kernel(AttendArgs a) {
    constexpr int LANES = HS / 4, SHARES = JOIN_THREADS / LANES;
    __shared__ float4 acc_s[SHARES][LANES];
    __shared__ float sum_s[SHARES], top_s[SHARES];
    const uint32_t block = a.first + blockIdx.x;
    const int r = block / a.heads, head = block % a.heads, tid = threadIdx.x;
    const int row = row_of(a, r), len = len_of(a, r);
    const int4 parts = a.parts[r];
    const int n = parts.y + (parts.z >= 0);
    if ((row < 0) | (len <= UNIT) | (n < 2)) return;  // (one wait for the three loads)
    const int d = tid % LANES, share = tid / LANES;
    float top = -INFINITY, sum = 0.0f;
    float4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    const auto add = [&](float m, float l, float4 y) {
        const float top1 = fmaxf(top, m), ref = top1 == -INFINITY ? 0.0f : top1;
        const float f = __builtin_amdgcn_exp2f(top - ref), e = __builtin_amdgcn_exp2f(m - ref);
        top = top1;
        sum = sum * f + l * e;
        acc.x = acc.x * f + y.x * e;
        acc.y = acc.y * f + y.y * e;
        acc.z = acc.z * f + y.z * e;
        acc.w = acc.w * f + y.w * e;
    };
#pragma unroll 4
    for (int i = share; i < n; i += SHARES) {
        const int slot = i < parts.y ? parts.x + i : parts.z;
        const long long at = (long long)slot * a.heads + head;
        const float2 x = a.part_ml[at];
        add(x.x, x.y, ld4(a.part_o + at * HS + 4 * d));
    }
    acc_s[share][d] = acc;
    if (d == 0) {
        sum_s[share] = sum;
        top_s[share] = top;
    }
    __syncthreads();
    if (share != 0) return;
#pragma unroll
    for (int i = 1; i < SHARES; ++i) add(top_s[i], sum_s[i], acc_s[i][d]);
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    typedef vec<TQ, 4> U __attribute__((aligned(4)));
    const vec<TQ, 4> y = {(TQ)(acc.x * f), (TQ)(acc.y * f), (TQ)(acc.z * f), (TQ)(acc.w * f)};
    *(U *)((TQ *)a.out + row * a.out_stride + head * HS + 4 * d) = y;
    if (a.lse && d == 0)
        a.lse[(long long)row * a.heads + head] =
            sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * LN2;
}

// How a call is split, from what the host knows of it (the lengths are the
// device's).
struct Split {
    int slots, workers, few, least, enough, cached;  // as in AttendArgs
    size_t ml_at, parts_at, bytes;  // offsets of the workspace's pieces; its size
};

constexpr int CUS = 256;

// A split costs the join and the search for a part, about 4 us; a whole
// sequence is bound by what one CU reads, about 70 GB/s. Measured, whole against
// split, by the bytes of a sequence's keys and values of one head: 12
// workgroups, 256 KB 7.8 and 7.9 us, 512 KB 12.5 and 8.1; 128 workgroups, 512
// KB 15 and 20, 1 MB 33 and 29; 768 workgroups, 512 KB 75 and 84. The device
// reads 70 times as fast as a CU, so with very many workgroups one longer
// sequence still ends with the others.
constexpr long long WHOLE_FEW = 256 << 10, WHOLE_MANY = 512 << 10;
constexpr int MANY = 96;
constexpr long long WHOLE_SHARE = 256;  // bytes a workgroup

// Parts: up to 8 workgroups a CU in all, for balance (128 requests of 1 to 8192
// tokens: 4 a CU 135 us, 8 123, 16 124; two of 131072: 172, 175, 183); parts
// of at least 64 KB; parts of up to 256 KB while that leaves a workgroup a CU
// (16 x 2000 tokens: parts of 64 KB 36 us, of 256 KB 31).
constexpr int WORKGROUPS_PER_CU = 8;
constexpr long long PART_LEAST = 64 << 10, PART_ENOUGH = 256 << 10;

// Keys and values that pass the device's caches (256 MB, half of it what the
// other tensors of a step leave) are read non-temporally: two contexts of
// 131072 tokens 198 -> 177 us, 64 x 2000 tokens 105 -> 94; what fits is kept
// (16 x 1000 tokens, 66 MB, read again and again: 14.9 us, non-temporally 20.6).
constexpr double CACHES = 1.2e8;

// Query heads of a kv head up to which fp32 queries go by attend_rows_kernel, whose
// registers grow with them (4, on 16 x 8000 keys of 64 in bf16: 33 us, 42 by the
// matrix kernel).
constexpr int ROWS = 4;

// Workgroups that share a kv head's query heads.
int tiles_of(const PagedCache &c, const PagedBatch &b) {
    const int group = b.heads / c.kv_heads;
    const int cols = b.type != BMB_F32 && group > 16 ? 32 : 16;
    return (group + cols - 1) / cols;
}

Split split_of(const PagedCache &c, const PagedBatch &b) {
    Split s = {b.requests, 0, 0, 0, 0, 0, 0, 0, 0};
    const long long heads = (long long)c.kv_heads * tiles_of(c, b);  // workgroups of one slot
    const long long key_bytes = 2ll * c.head_size * element_size(c.type);
    const long long all = b.requests * heads;
    // Whole sequences do not look at each other's lengths: the batch is taken
    // for half of the most it can be.
    s.cached = 0.5 * b.requests * b.max_len * key_bytes * c.kv_heads < CACHES;
    long long whole = all >= MANY ? WHOLE_MANY : WHOLE_FEW;
    if (whole < all * WHOLE_SHARE) whole = all * WHOLE_SHARE;
    if (b.max_len * key_bytes <= whole) return s;

    const auto at_least_1 = [](long long x) { return x < 1 ? 1ll : x; };
    const long long units = (b.max_len + UNIT - 1) / UNIT, most = b.requests * units;
    long long workers = at_least_1(CUS * WORKGROUPS_PER_CU / heads);
    workers = workers < most ? workers : most;
    s.workers = (int)workers;
    s.slots = (int)(b.requests + workers < most ? b.requests + workers : most);
    s.few = (int)at_least_1(CUS / heads);
    s.least = (int)at_least_1(PART_LEAST / (key_bytes * UNIT));
    s.enough = (int)at_least_1(PART_ENOUGH / (key_bytes * UNIT));
    const double cached = CACHES / ((double)key_bytes * c.kv_heads * UNIT);
    s.cached = cached < 1.0 ? 1 : (int)cached;
    const size_t rows = (size_t)s.slots * b.heads;
    s.ml_at = rows * c.head_size * sizeof(float);
    s.parts_at = (s.ml_at + rows * sizeof(float2) + 15) / 16 * 16;
    s.bytes = s.parts_at + (size_t)b.requests * sizeof(int4);
    return s;
}

// (`buffers`: as for cache_fault.)
const char *batch_fault(const PagedCache *c, const PagedBatch *b, bool buffers) {
    if (const char *why = cache_fault(c, buffers)) return why;
    if (b == nullptr) return "no batch";
    if (b->requests < 1 || b->max_len < 0 || b->heads < 1 || b->n_rows < 1)
        return "a size is below its least";
    if (b->max_len > INT_MAX - 4096) return "max_len is more than 2^31 - 4097";
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
    if (b->n_rows > 1 && b->out_stride < (long long)b->heads * c->head_size)
        return "rows of out overlap";
    return nullptr;
}

// `blocks` workgroups of `kernel`.
void launch_blocks(void (*kernel)(AttendArgs), long long blocks, int threads, size_t lds,
                   AttendArgs a, hipStream_t stream) {
    in_launches(blocks, threads, [&](long long first, unsigned n) {
        a.first = (int)first;
        launch(kernel, dim3(n), dim3(threads), lds, stream, a);
    });
}

// The parts by `kernel`, whose workgroups of `waves` waves take `cols` heads each.
void launch_parts(void (*kernel)(AttendArgs), int waves, int cols, int hs, const AttendArgs &a,
                  hipStream_t stream) {
    const size_t lds = merge_bytes(waves, cols, a.group < cols ? a.group : cols, hs);
    allow_smem(kernel, lds);
    launch_blocks(kernel, (a.slots + 7ll) / 8 * 8 * a.kv_heads * a.tiles, waves * WAVE, lds, a,
                  stream);
}

template <template <typename, int> class POLICY, typename TC, int HS, int QT>
void launch_matrix(const AttendArgs &a, hipStream_t stream) {
    launch_parts(a.page.d % 16 == 0 ? attend_kernel<POLICY, TC, HS, true, QT>
                                    : attend_kernel<POLICY, TC, HS, false, QT>,
                 4, 16 * QT, HS, a, stream);
}

// Few whole sequences: 8 waves share one (192 workgroups, 1000 keys: 12.6 us with
// 4, 11.2 with 8); many: 4, which start sooner (768 workgroups of one key: 4.3
// and 6.8 us).
template <typename TC, int HS, int G>
void launch_rows(const AttendArgs &a, hipStream_t stream) {
    const bool aligned = a.page.d % 16 == 0;
    if (a.workers == 0 && a.requests * a.kv_heads * a.tiles < 512)
        launch_parts(aligned ? attend_rows_kernel<TC, HS, G, true, 8>
                             : attend_rows_kernel<TC, HS, G, false, 8>,
                     8, G, HS, a, stream);
    else
        launch_parts(aligned ? attend_rows_kernel<TC, HS, G, true, 4>
                             : attend_rows_kernel<TC, HS, G, false, 4>,
                     4, G, HS, a, stream);
}

template <typename TQ, typename TC, int HS>
void launch_attend(const AttendArgs &a, hipStream_t stream) {
    if constexpr (sizeof(TQ) == 2) {
        if (a.group <= 16)
            launch_matrix<Half, TC, HS, 1>(a, stream);
        else
            launch_matrix<Half, TC, HS, 2>(a, stream);
    } else {
        if (a.group == 1)
            launch_rows<TC, HS, 1>(a, stream);
        else if (a.group == 2)
            launch_rows<TC, HS, 2>(a, stream);
        else if (a.group <= ROWS)
            launch_rows<TC, HS, 4>(a, stream);
        else
            launch_matrix<Full, TC, HS, 1>(a, stream);
    }
    if (a.workers)
        launch_blocks(join_kernel<TQ, HS>, (long long)a.requests * a.heads, JOIN_THREADS, 0, a,
                      stream);
}

template <typename TQ, typename TC>
void launch_attend(int hs, const AttendArgs &a, hipStream_t stream) {
    if (hs == 32)
        launch_attend<TQ, TC, 32>(a, stream);
    else if (hs == 64)
        launch_attend<TQ, TC, 64>(a, stream);
    else
        launch_attend<TQ, TC, 128>(a, stream);
}

}  // namespace
}  // namespace bmb

extern "C" {

size_t paged_attention_workspace(const PagedCache *cache, const PagedBatch *batch) {
    if (bmb::batch_fault(cache, batch, false)) return 0;
    return bmb::split_of(*cache, *batch).bytes;
}

int paged_attention(const PagedCache *c, const PagedBatch *b, void *out, float *lse, const void *q,
                    hipStream_t stream) {
    using namespace bmb;
    const char *me = "paged_attention";
    if (const char *why = batch_fault(c, b, true)) return refuse(me, why);
    if (!out || !q || !b->block_table || !b->lens) return refuse(me, "a null pointer");
    if (((uintptr_t)q | (uintptr_t)out) % 4 != 0)
        return refuse(me, "rows are no multiples of 4 bytes");
    const int size = element_size(c->type);
    if (c->page_size % 16 != 0 &&
        ((c->pages - 1) * c->page_stride + (c->page_size - 1) * c->token_stride) * size / 16 >=
            NO_ROW)
        return refuse(me, "tokens 64 GiB apart need pages of a multiple of 16 tokens");
    const Split s = split_of(*c, *b);
    char *work = (char *)b->work;
    if (work != nullptr && b->work_bytes < s.bytes) return refuse(me, "the workspace is too small");
    if ((uintptr_t)work % 16 != 0) return refuse(me, "the workspace is no multiple of 16 bytes");
    const bool lease = s.bytes > 0 && work == nullptr;
    if (lease && stream_capturing(stream))
        return refuse(me, "a call under graph capture needs a workspace of its caller's");
    std::optional<ScratchLease> ws;
    if (lease) {
        ws.emplace(SCRATCH_PAGED, s.bytes, stream);
        if (!*ws) return refuse(me, "cannot allocate the workspace");
        work = (char *)ws->get();
    }
    const int group = b->heads / c->kv_heads;
    AttendArgs a = {(const char *)q, (const char *)c->k, (const char *)c->v, (char *)out, lse,
                    b->block_table, b->lens, b->rows, (float *)work, (float2 *)(work + s.ml_at),
                    (int4 *)(work + s.parts_at), c->page_stride, c->token_stride, c->head_stride,
                    b->q_stride, b->out_stride, b->requests, b->heads, c->kv_heads, group,
                    tiles_of(*c, *b), c->pages, b->table_stride, b->max_len, b->n_rows,
                    s.slots, s.workers, s.few, s.least, s.enough, s.cached, 0, b->scale * LOG2E,
                    FastDiv::of(c->page_size),
                    (uint32_t)(c->page_stride * size / 16),
                    (uint32_t)(c->token_stride * size / 16)};
    const int hs = c->head_size;
    if (b->type == BMB_F16)
        launch_attend<_Float16, _Float16>(hs, a, stream);
    else if (b->type == BMB_BF16)
        launch_attend<__bf16, __bf16>(hs, a, stream);
    else if (c->type == BMB_F16)
        launch_attend<float, _Float16>(hs, a, stream);
    else if (c->type == BMB_BF16)
        launch_attend<float, __bf16>(hs, a, stream);
    else
        launch_attend<float, float>(hs, a, stream);
    return 0;
}

}  // extern "C"
