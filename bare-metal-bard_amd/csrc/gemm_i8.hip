// 8-bit linear layers (gemm_i8, include/gemm.h).
//
// C = A B^T on v_mfma_i32_32x32x32_i8: both operands have k contiguous, so lane
// l supplies 16 consecutive bytes of row l % 32 at k = 16 (l / 32), and since
// both supply the same k in the same place, their order inside the instruction
// does not matter. Sums are whole numbers in 32 bits: exact, in any order.
//
// A stage is 128 k. Its tile of A and of B goes from global memory straight into
// LDS (16 bytes a lane, no registers). LDS holds three stages of A and two or
// three of B (all 160 KB for 256 x 256 tiles): what bounds a tile is how long
// before its use a load is issued. In steps of 32 k a wave multiplies what it has
// read, and between the products reads the next step's operands and issues loads;
// one barrier a stage. 8192^3 (256 x 256 tiles): two stages of both, all loads at
// the stage's start 525 us; spread 510; scales by LDS instead of from memory
// between the stores, which waited for the stores, 477; A three stages deep 446;
// results by LDS in whole rows 429; no wait in the loop but for the next stage 423
// (2600 TOP/s; up to 448 on other boxes, and 440-515 for the first passes after other
// work. The matrix cores are busy 77% of the cycles at about 1.55 of 2.4 GHz: power
// bounds the clock; on zeros it takes 281).
// 256 x 256 tiles take a whole CU, so their stores overlap no products: 1000 x 50257 x
// 768 in fp32 takes 83-91 us, the stores alone 42. 256 x 128 tiles with stages of 64 k,
// two workgroups a CU, took 71 instead of 79 where rows are whole lines, but 59 instead
// of 54 for 1024 x 49152 in 16 bits and 581 instead of 435 for 8192^3.
//
// Edges. Rows past the last are loaded from the last one and reach only
// results that are not stored. In a last stage that is not whole, chunks past
// the row's last one are loaded from that, and A's bytes from K on are masked
// to zero before they are multiplied (so B's need no mask).
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "args.hpp"
#include "common.hpp"
#include "launch.hpp"
#include "paged.hpp"
#include "workspace.hpp"
#include "../../include/gemm.h"

namespace bmb {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int MAX_K = 131071;  // 128 * 128 * MAX_K < 2^31
constexpr int BK = 128, STEPS = BK / 32;  // k of a stage, and steps of 32 k
constexpr int CHUNK = 16, CHUNKS = BK / CHUNK;

struct I8Args {
    const signed char *A, *B;
    const float *a_scales, *b_scales, *bias;
    char *C;
    long long lda, ldb, ldc;
    int M, N, K, tiles_m, tiles_n;
    int span;   // K of a workgroup (a multiple of 128), or all of it
    int *part;  // span < K: (ranges of K, M, N) sums
    long long part_stride;
    int first;  // few rows: the launch's first workgroup of the call's
};

// DA, DB: stages of A and of B in LDS.
template <int BM_, int BN_, int WAVES_M_, int WAVES_N_, int DA_, int DB_>
struct I8Tile {
    static constexpr int DA = DA_, DB = DB_;
    static constexpr int BM = BM_, BN = BN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_;
    static constexpr int NT = 64 * WAVES_M * WAVES_N;
    static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, FM = WM / 32, FN = WN / 32;
};

typedef __attribute__((address_space(3))) void lds_void;

// A stage's rows in LDS: 128 bytes, their 16-byte chunks permuted by the row so
// that the groups of 16 lanes in which a 128-bit read of 32 rows is served, {0-3,
// 12-15, 20-27}, {4-11, 16-19, 28-31}, touch 16 different places modulo 256
// bytes (no bank conflict is counted).
__device__ __forceinline__ int permuted(int row, int chunk) { return chunk ^ ((row >> 1) & 7); }

// ROWS rows of one operand's stage into LDS: lane i of a wave fills the i-th
// chunk of 1 KB, eight rows; the workgroup's load i rows i * STEP on, where
// chunks are permuted alike (STEP is a multiple of 16).
template <int ROWS, int NT>
struct Staging {
    static constexpr int LOADS = ROWS * CHUNKS / NT, STEP = NT / CHUNKS;
    static_assert(STEP % 16 == 0, "permutations depend on the row modulo 16");
    int row, chunk;      // byte offsets of this lane's first row, and in it
    int step, last_row;  // of the next load's row, and of the operand's last row
    __device__ __forceinline__ void setup(int rows, int ld) {
        const int r = threadIdx.x / CHUNKS;
        row = r * ld;
        chunk = permuted(r, threadIdx.x % CHUNKS) * CHUNK;
        step = STEP * ld;
        last_row = (min(rows, ROWS) - 1) * ld;
    }
    // Load i of a stage. k0: the stage's first k; last: the first k of the
    // operand's last chunk.
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t p, char *lds, int k0, int last,
                                         int i) const {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        [[maybe_unused]] char *to = lds + (i * NT + wave * 64) * CHUNK;
        [[maybe_unused]] const int at = min(row + i * step, last_row) + min(chunk + k0, last);
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass does not know loads of 16 bytes)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(p, (lds_void *)to, 16, at, 0, 0, 0);
#endif
    }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t operand(const signed char *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<signed char *>(p), 0, 0xffffffff,
                                             0x00027000);
}

// Where this lane finds its operand of a stage's first step in row r of the
// tile; those of step kk are at place ^ 32 kk, and of rows 32 i on 32 i rows on.
__device__ __forceinline__ int place_of(int r, int half) {
    return r * BK + permuted(r, half) * CHUNK;
}
__device__ __forceinline__ i32x4 operand_at(const char *lds, int place, int kk, int i) {
    return *(const i32x4 *)(lds + ((place ^ (32 * kk)) + i * 32 * BK));
}

// The first n bytes of a chunk (n any number).
__device__ __forceinline__ i32x4 first_bytes(i32x4 x, int n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int m = n - 4 * e;
        x[e] = m >= 4 ? x[e] : m <= 0 ? 0 : x[e] & (int)((1u << (8 * m)) - 1);
    }
    return x;
}

// f(0), ..., f(N - 1) as constants.
template <int N, typename F>
__device__ __forceinline__ void for_each(F &&f) {
    if constexpr (N > 0) {
        for_each<N - 1>(f);
        f(std::integral_constant<int, N - 1>());
    }
}

// s_waitcnt's operand: at most n loads from memory on their way, whatever else.
constexpr int vmcnt(int n) { return 0x0f70 | (n & 15) | (n >> 4) << 14; }

// Waits until at most n loads from memory are on their way and every access to
// LDS is done.
template <int N>
__device__ __forceinline__ void wait() {
    asm volatile("" ::: "memory");  // (the compiler moves no access over it)
    __builtin_amdgcn_s_waitcnt(vmcnt(N) & 0xf0ff);
}
// A barrier that waits for nothing but the other waves (__syncthreads() also
// waits for every load into LDS, and every store, that is on its way). The
// caller has waited for what the others will read.
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// xcd_remap() for any number of workgroups: XCD x, which is given ids x, x + 8,
// ..., takes consecutive tiles.
__device__ __forceinline__ int xcd_order(int id, int blocks) {
    const int x = id % 8, each = blocks / 8, more = blocks % 8;
    return x * each + min(x, more) + id / 8;
}

// A sum's result. (Told nothing, the compiler rounds fp16 results once, of
// the exact product and sum, where it finds both in one place: the bits would
// depend on how a product is cut.)
template <typename T>
__device__ __forceinline__ T result(int sum, float a_scale, float b_scale, float bias) {
    float y = __builtin_fmaf((float)sum * a_scale, b_scale, bias);
    asm("" : "+v"(y));
    return (T)y;
}

// A wave's operands of one step of 32 k.
template <int FM, int FN>
struct Operands {
    i32x4 a[FM], b[FN];
};

// T: of C, or int for sums of a range of K. PAST: stores go past the L2 caches.
template <typename Tile, typename T, bool PAST>
__global__ __launch_bounds__(Tile::NT) void i8_kernel(I8Args a) {
    constexpr int BM = Tile::BM, BN = Tile::BN, FM = Tile::FM, FN = Tile::FN;
    // Objects of their own, so that reads of one stage do not wait for the
    // loads into the other.
    constexpr int DA = Tile::DA, DB = Tile::DB;
    static_assert(DA == 3 && (DB == 2 || DB == 3), "stages in LDS");
    __shared__ __attribute__((aligned(256))) char a0[BM * BK], a1[BM * BK], a2[BM * BK];
    __shared__ __attribute__((aligned(256))) char b0[BN * BK], b1[BN * BK];
    char *b2 = nullptr;
    if constexpr (DB == 3) {
        __shared__ __attribute__((aligned(256))) char more[BN * BK];
        b2 = more;
    }
    char *const as[3] = {a0, a1, a2}, *const bs[3] = {b0, b1, b2};
    int tm, tn;
    const int tiles = a.tiles_m * a.tiles_n, range = blockIdx.x / tiles;
    group_tile(xcd_order((int)blockIdx.x - range * tiles, tiles), a.tiles_m, a.tiles_n, 8, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int from = range * a.span, K = min(a.span, a.K - from);
    const __amdgpu_buffer_rsrc_t A = operand(a.A + m0 * a.lda + from);
    const __amdgpu_buffer_rsrc_t B = operand(a.B + n0 * a.ldb + from);
    Staging<BM, Tile::NT> sa;
    Staging<BN, Tile::NT> sb;
    sa.setup(a.M - m0, (int)a.lda);
    sb.setup(a.N - n0, (int)a.ldb);
    static_assert(BM <= Tile::NT && BN <= Tile::NT, "a scale a thread");
    const int tid = threadIdx.x;
    const float scale_of_m = a.a_scales[min(m0 + min(tid, BM - 1), a.M - 1)];
    const float scale_of_n = a.b_scales[min(n0 + min(tid, BN - 1), a.N - 1)];
    const float bias_of_n = a.bias ? a.bias[min(n0 + min(tid, BN - 1), a.N - 1)] : 0.0f;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / Tile::WAVES_N * Tile::WM, wn = wave % Tile::WAVES_N * Tile::WN;
    const int r = lane & 31, half = lane >> 5;

    int place_a = place_of(wm + r, half), place_b = place_of(wn + r, half);

    i32x16 acc[FM][FN] = {};
    // Operands of one step of 32 k, and of the next while it is multiplied.
    typedef Operands<FM, FN> Step;
    Step even, odd;
    const int last = (K - 1) / CHUNK * CHUNK;
    constexpr int LA = decltype(sa)::LOADS, LB = decltype(sb)::LOADS;
    // Load i of a pair of stages: of B's stage kb into lb, then of A's stage ka into la.
    const auto load = [&](char *la, int ka, char *lb, int kb, int i) {
        if (i < LB) {
            if (kb < K) sb.load(B, lb, kb, last, i);
        } else {
            if (ka < K) sa.load(A, la, ka, last, i - LB);
        }
    };
    // Read i of a step's operands, in the order in which the products want them.
    const auto read = [&](Step &f, const char *la, const char *lb, int kk, int i) {
        if (i == 0 || i > FN)
            f.a[i ? i - FN : 0] = operand_at(la, place_a, kk, i ? i - FN : 0);
        else
            f.b[i - 1] = operand_at(lb, place_b, kk, i - 1);
    };
    const auto product = [&](const Step &f, int t) {
        const int i = t / FN, j = t % FN;
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.a[i], f.b[j], acc[i][j], 0, 0, 0);
    };
    // One step: its products, and between them the reads of the next step's
    // operands (step kk of stage la, lb) and loads [first, first + n) of a pair of
    // stages into ga, gb. Fenced, since the compiler gathers them.
    const auto step = [&](const Step &now, Step &next, const char *la, const char *lb, int kk,
                          char *ga, int ka, char *gb, int kb, int first, int n) {
        // (not all steps' places at once: they do not fit the registers)
        asm volatile("" : "+v"(place_a), "+v"(place_b));
#pragma unroll
        for (int t = 0; t < FM * FN; ++t) {
#pragma unroll
            for (int i = t * (FM + FN) / (FM * FN); i < (t + 1) * (FM + FN) / (FM * FN); ++i)
                read(next, la, lb, kk, i);
#pragma unroll
            for (int i = t * n / (FM * FN); i < (t + 1) * n / (FM * FN); ++i)
                load(ga, ka, gb, kb, first + i);
            product(now, t);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Stage k0, the i-th, in its places (the operands of its first step are read), up
    // to the first step of the next. Behind the barrier its places are free for A's
    // stage DA and B's stage DB after it; these loads (the first L0 in the last step,
    // the others in the next stage) are spread over the steps: a wave that issues
    // them all at once waits until the memory pipeline has taken them.
    constexpr int LOADS = LA + LB, L0 = (3 * LOADS + 7) / 8, L1 = L0, L2 = LOADS - L0 - L1;
    // Loads that may be on their way when the next stage has to be there.
    constexpr int LATER = (DA - 2) * LA + (DB - 2) * LB;
    const auto stage = [&](int i, int k0) {
        char *la = as[i % DA], *lb = bs[i % DB], *pa = as[(i + DA - 1) % DA];
        char *pb = bs[(i + DB - 1) % DB], *na = as[(i + 1) % DA], *nb = bs[(i + 1) % DB];
        step(even, odd, la, lb, 1, pa, k0 + (DA - 1) * BK, pb, k0 + (DB - 1) * BK, L0, L1);
        step(odd, even, la, lb, 2, pa, k0 + (DA - 1) * BK, pb, k0 + (DB - 1) * BK, L0 + L1, L2);
        step(even, odd, la, lb, 3, pa, 0, pb, 0, 0, 0);
        // This wave has read the stage, and its loads of the next are in LDS; behind
        // the barrier everybody's are. (The last stages have fewer loads behind them.)
        wait<LATER>();
        if (k0 + (DA - 1) * BK >= K) wait<0>();
        barrier();
        step(odd, even, na, nb, 0, la, k0 + DA * BK, lb, k0 + DB * BK, 0, L0);
    };
    // The last stage, of `rest` k.
    int rest = 0;
    const auto finish = [&](const char *la, const char *lb) {
#pragma unroll
        for (int kk = 0; kk < STEPS; ++kk) {
            if (kk > 0) {
#pragma unroll
                for (int i = 0; i < FM + FN; ++i) read(even, la, lb, kk, i);
            }
            if (rest < BK) {
#pragma unroll
                for (int i = 0; i < FM; ++i)
                    even.a[i] = first_bytes(even.a[i], rest - (2 * kk + half) * CHUNK);
            }
#pragma unroll
            for (int t = 0; t < FM * FN; ++t) product(even, t);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (K > 0) {
#pragma unroll
        for (int x = 0; x < DA - 1; ++x) {
#pragma unroll
            for (int i = x < DB - 1 ? 0 : LB; i < LOADS; ++i) load(as[x], x * BK, bs[x], x * BK, i);
        }
#pragma unroll
        for (int i = 0; i < L0; ++i)
            load(as[DA - 1], (DA - 1) * BK, bs[DB - 1], (DB - 1) * BK, i);
        static_assert(L0 <= LB, "these are B's");
        wait<LATER + L0>();
        if (K <= (DA - 1) * BK) wait<0>();
        barrier();
#pragma unroll
        for (int i = 0; i < FM + FN; ++i) read(even, a0, b0, 0, i);
        // As many stages as bring every one back to its places.
        constexpr int TURN = DA == DB ? DA : DA * DB;
        int k0 = 0;
        for (; k0 + (TURN + DA - 1) * BK < K; k0 += TURN * BK)
            for_each<TURN>([&](auto i) { stage(i(), k0 + i() * BK); });
        rest = K - k0;
        const char *la = a0, *lb = b0;
        const auto left = [&](auto self, auto number) {
            constexpr int i = decltype(number)::value;
            if constexpr (i + 1 < TURN + DA) {
                if (rest <= BK) return;
                stage(i, k0 + i * BK);
                rest -= BK;
                la = as[(i + 1) % DA];
                lb = bs[(i + 1) % DB];
                self(self, std::integral_constant<int, i + 1>());
            }
        };
        left(left, std::integral_constant<int, 0>());
        finish(la, lb);
    }

    // Results leave by LDS, eight rows of each wave row at a time, in two places in
    // turn: lane l has column l % 32, rows 8 g + 4 (l / 32) + 0..3 of a 32 x 32 block
    // in registers 4 g + 0..3; a lane then stores four columns of a row, so that
    // a store takes 256 columns in a piece, wherever rows begin. The scales come
    // by LDS too: loads from memory would wait for the stores before them.
    constexpr bool PART = std::is_same_v<T, int>;
    typedef std::conditional_t<PART, int, float> V;
    constexpr int ROWS = Tile::WAVES_M * 8, LINE = BN / 4;  // lanes of a row
    static_assert(ROWS * BN * 4 <= BN * BK && (BM + 2 * BN) * 4 <= BM * BK, "they fit the stages");
    float *scale_m = (float *)a0, *scale_n = scale_m + BM, *bias_n = scale_n + BN;
    __syncthreads();  // the stages have been read
    if (tid < BM) scale_m[tid] = scale_of_m;
    if (tid < BN) scale_n[tid] = scale_of_n;
    if (tid < BN) bias_n[tid] = bias_of_n;
    __syncthreads();
    const long long ldc = PART ? (long long)a.N : a.ldc;
    T *C = (T *)(PART ? (char *)(a.part + range * a.part_stride) : a.C) + n0;
    float sn[FN], bias[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        sn[j] = scale_n[wn + j * 32 + r];
        bias[j] = bias_n[wn + j * 32 + r];
    }
    // (rows 4..7 of eight move by 32 columns: both halves of a wave write at once)
    const auto at = [](int row, int c) { return row * BN + (c ^ ((row & 4) << 3)); };
    const int columns = min(BN, a.N - n0);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            V *place = (V *)((i * 4 + g) % 2 ? b1 : b0);
            const float4 sm = *(const float4 *)(scale_m + wm + i * 32 + 8 * g + 4 * half);
            const float each[4] = {sm.x, sm.y, sm.z, sm.w};
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int sum = acc[i][j][4 * g + e];
                    place[at(wm / Tile::WM * 8 + 4 * half + e, wn + j * 32 + r)] =
                        PART ? (V)sum : (V)result<float>(sum, each[e], sn[j], bias[j]);
                }
            wait<63>();
            barrier();
#pragma unroll
            for (int x = 0; x < ROWS * LINE / Tile::NT; ++x) {
                const int t = x * Tile::NT + tid, row = t / LINE, c = t % LINE * 4;
                const int m = m0 + row / 8 * Tile::WM + i * 32 + 8 * g + row % 8;
                typedef V V4 __attribute__((ext_vector_type(4)));
                const V4 v = *(const V4 *)(place + at(row, c));
                typedef T T4 __attribute__((ext_vector_type(4)));
                typedef T4 Unaligned __attribute__((aligned(sizeof(T))));
                const T4 y = __builtin_convertvector(v, T4);
                T *to = C + m * ldc + c;
                if (m < a.M && c + 4 <= columns) {
                    if (PAST)
                        __builtin_nontemporal_store(y, (Unaligned *)to);
                    else
                        *(Unaligned *)to = y;
                } else if (m < a.M) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < columns) to[e] = y[e];
                }
            }
        }
}

// Few rows: bound by the weights' bytes and by latency. A workgroup takes 16
// columns, each of its waves a range of K, and no stage passes through LDS: a
// wave's loads are the operands of v_mfma_i32_16x16x64_i8 (lane l: 16 bytes of
// row l % 16 at k = 16 (l / 16)), several on their way at once. The waves' sums
// meet in LDS. 1 x 16384 x 16384 49.5 us, 5.4 TB/s, the rate of a copy.
template <int FM, typename T>
__global__ __launch_bounds__(1024) void i8_few_kernel(I8Args a) {
    extern __shared__ i32x4 sums[];  // (waves, FM, 64 lanes)
    constexpr int UNIT = 64, AHEAD = 4;
    const int lane = threadIdx.x & 63, r = lane & 15, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int n0 = (a.first + (int)blockIdx.x) * 16;
    const int units = (a.K + UNIT - 1) / UNIT, last = (a.K - 1) / CHUNK * CHUNK;
    const int first = (int)((long long)units * wave / waves);
    const int end = (int)((long long)units * (wave + 1) / waves);
    const signed char *A[FM], *B = a.B + min(n0 + r, a.N - 1) * a.ldb;
#pragma unroll
    for (int i = 0; i < FM; ++i) A[i] = a.A + min(16 * i + r, a.M - 1) * a.lda;

    i32x4 acc[FM] = {};
    for (int u = first; u < end; u += AHEAD) {
        i32x4 fa[AHEAD][FM], fb[AHEAD];
#pragma unroll
        for (int x = 0; x < AHEAD; ++x) {
            if (u + x >= end) break;
            const int k = min((u + x) * UNIT + quarter * CHUNK, last);
            fb[x] = *(const i32x4 *)(B + k);
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[x][i] = *(const i32x4 *)(A[i] + k);
        }
#pragma unroll
        for (int x = 0; x < AHEAD; ++x) {
            if (u + x >= end) break;
            if ((u + x + 1) * UNIT > a.K) {
#pragma unroll
                for (int i = 0; i < FM; ++i)
                    fa[x][i] = first_bytes(fa[x][i], a.K - (u + x) * UNIT - quarter * CHUNK);
            }
#pragma unroll
            for (int i = 0; i < FM; ++i)
                acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[x][i], fb[x], acc[i], 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) sums[(wave * FM + i) * 64 + lane] = acc[i];
    __syncthreads();
    // Register e of lane l is row 4 (l / 16) + e, column l % 16 of its block.
    const int *part = (const int *)sums;
    for (int at = threadIdx.x; at < FM * 256; at += blockDim.x) {
        const int m = at / 16, c = at % 16, n = n0 + c;
        if (m >= a.M || n >= a.N) continue;
        const int from = (m / 16 * 64 + (m % 16 / 4) * 16 + c) * 4 + m % 4;
        int sum = 0;
        for (int w = 0; w < waves; ++w) sum += part[w * FM * 256 + from];
        ((T *)a.C)[m * a.ldc + n] =
            result<T>(sum, a.a_scales[m], a.b_scales[n], a.bias ? a.bias[n] : 0.0f);
    }
}

template <int FM, typename T>
void launch_few(I8Args &a, hipStream_t stream) {
    // Three units of K a wave, up to 16 waves. One to eight units are the same within
    // 4% wherever the rule sends few rows (1 x 2304 x 768 2.63-2.74 us, three 2.69; 1 x 768 x
    // 6400 5.60-5.74) but for 32 x 2304 x 768: one 3.48, three 3.68, eight 4.12.
    const int waves = std::min(16, std::max(1, ceil_div(ceil_div(a.K, 64), 3)));
    in_launches(ceil_div(a.N, 16), 64 * waves, [&](long long first, unsigned n) {
        a.first = (int)first;
        launch(i8_few_kernel<FM, T>, dim3(n), dim3(64 * waves), waves * FM * 64 * sizeof(i32x4),
               stream, a);
    });
}

// C from the sums of the ranges of K: four results a thread.
template <typename T>
__global__ __launch_bounds__(256) void i8_join_kernel(I8Args a, int ranges, FastDiv columns) {
    const long long all = (long long)a.M * a.N;
    const long long first = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (first >= all) return;
    i32x4 sum = *(const i32x4 *)(a.part + first);
    for (int x = 1; x < ranges; ++x) sum += *(const i32x4 *)(a.part + x * a.part_stride + first);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (first + e >= all) return;
        const int m = columns.quot((int)(first + e)), n = (int)(first + e) - m * a.N;
        ((T *)a.C)[m * a.ldc + n] =
            result<T>(sum[e], a.a_scales[m], a.b_scales[n], a.bias ? a.bias[n] : 0.0f);
    }
}

// What the L2 caches of the eight XCDs hold together.
constexpr long long L2_BYTES = 32 << 20;

// How a product is cut. tile: an index below; ranges: of K.
struct I8Plan {
    int tile, ranges, span;
    bool deep;  // of tiles of 64 x 64 and 128 x 128: three stages of B
};

// Tiles at most that are deep (plan_of says why).
constexpr int DEEP_64 = 768, DEEP_128 = 256;

template <typename Tile>
dim3 grid_of(I8Args &a, int ranges) {
    a.tiles_m = ceil_div(a.M, Tile::BM);
    a.tiles_n = ceil_div(a.N, Tile::BN);
    return dim3(a.tiles_m * a.tiles_n * ranges);
}

// Results that do not fit the L2 caches are stored past them (1000 x 50257 x 768
// in fp32: 94 -> 86 us). FIT: they always fit.
template <typename Tile, typename T, bool FIT>
void launch_tile(I8Args &a, hipStream_t stream) {
    const dim3 grid = grid_of<Tile>(a, 1);
    if constexpr (!FIT) {
        if ((long long)a.M * a.N * (int)sizeof(T) > L2_BYTES) {
            launch(i8_kernel<Tile, T, true>, grid, dim3(Tile::NT), 0, stream, a);
            return;
        }
    }
    launch(i8_kernel<Tile, T, false>, grid, dim3(Tile::NT), 0, stream, a);
}

// The sums of each range of K, and what joins them.
template <typename Tile, typename T>
void launch_ranges(I8Args &a, int ranges, hipStream_t stream) {
    launch(i8_kernel<Tile, int, false>, grid_of<Tile>(a, ranges), dim3(Tile::NT), 0, stream, a);
    launch(i8_join_kernel<T>, dim3((unsigned)(((long long)a.M * a.N + 1023) / 1024)), dim3(256), 0,
           stream, a, ranges, FastDiv::of(a.N));
}

enum { FEW, TILE_64, TILE_128, TILE_256 };

// The rule, and its limits with both sides measured: us of a call among others in a
// graph, 16-bit results, three sets of operands in turn; * is what the rule takes
// (64 x 64 and so on: tiles; "in 4": ranges of K, and what joins them).
//   Few rows, up to 32 where N <= 4096 and K <= 8192, up to 4 where N > 4096 and K >
//   8192. Rows 1, 4, 16 and 32:
//                   few rows              64 x 64               64 x 64, split
//     2304 x 768    2.7* 2.8* 3.0* 3.7*   3.9  4.0  4.0  4.1
//     4096 x 4096   5.9* 6.1* 6.8* 8.4*   9.9  10.0 10.0 10.1   9.0  9.2  9.4  10.0 in 4
//     4096 x 8192   8.5* 8.8* 10.3* 14.1*     16.2 16.3 16.4 16.6   11.1 11.4 11.7 12.2 in 4
//     4096 x 8208   8.1  8.4  9.8  13.5   16.8 17.0 17.1 17.7   11.5* 11.8* 12.2* 12.7* in 4
//     4096 x 16384  14.0 14.4 17.5 24.1   28.6 29.0 29.2 29.5   15.4* 15.6* 16.0* 16.4* in 4
//     768 x 16384   12.0 13.0 16.9 24.0   28.0 27.9 27.9 29.0   10.5* 11.1* 11.8* 12.1* in 12
//     4112 x 768    2.9  3.0  3.4  4.4    4.0* 4.0* 4.1* 4.2*
//     8192 x 768    3.3  3.4  3.8  4.9    4.1* 4.1* 4.2* 4.2*
//     8192 x 4096   8.5  8.9  10.2 14.8   10.2* 10.3* 10.4* 10.6*   10.7 10.8 11.0 11.4 in 2
//     11008 x 4096  11.6 12.2 13.6 20.7   10.5* 10.6* 10.6* 10.9*
//     16384 x 1600  7.0  6.9  7.9  10.6   7.4* 7.5* 7.7* 7.9*
//     50257 x 768   8.6  9.3  12.1 17.2   9.1* 9.1* 9.4* 9.8*
//     8192 x 8192   12.8 13.4 17.2 25.3   16.8 16.9 17.0 17.4   15.0* 15.1* 15.5* 16.2* in 2
//     8192 x 8208   12.9* 13.3* 15.9 24.2     17.7 17.7 18.0 18.6   15.6 15.7 16.2* 16.8* in 2
//     16384 x 16384 48.8* 51.9* 73.6 105.6    60.1 60.4 61.0* 61.7*
//   (N = 4096 and K = 8192 are where 32 rows change sides. One to four rows are faster
//   as few rows on both sides of either, but for 768 x 16384, 11008 x 4096 and four of
//   50257 x 768: the limits cost them up to 3.4 us.)
//   64 x 64 split, from 36 stages on and ten a range:
//     64 x 2048 x 4480 (35 stages)   10.7*, in 2 10.2, in 4 9.1
//     64 x 2048 x 4608 (36)          10.7, in 2 10.3, in 3 9.5*, in 4 9.2
//     64 x 4096 x 4096 (32)          10.4*, in 2 10.4, in 4 10.1
//     64 x 6400 x 1600 (13)          6.7*, in 2 9.2
//     128 x 1600 x 4800 (38)         12.3, in 2 11.4, in 3 10.2*, in 4 9.9
//     256 x 768 x 6400 (50)          14.1, in 2 12.1, in 4 10.2, in 5 10.3*
//   64 x 64, then 128 x 128 from 192 of these on:
//     512 x 1600 x 6400 (52 tiles)   14.6*, 22.3
//     512 x 4096 x 4096 (128)        14.9*, 16.5
//     768 x 4096 x 4096 (192)        21.5, 17.5*
//     1024 x 4096 x 4096 (256)       27.3, 19.9*
//   128 x 128, then 256 x 256 where they fill 70% of their rounds of 256 CUs:
//     2048 x 4096 x 4096 (50%)       36.6*, 40.7
//     8192 x 2304 x 768 (56%)        24.6*, 29.1
//     1000 x 50257 x 768 (77%)       72, 66*
//     8192 x 1600 x 6400 (88%)       93, 80*
//     65 x 50257 x 768 (77%)         12.1, 16.8* (rows that a tile wastes are not counted)
// A tile has to leave few CUs idle; a larger one reads less.
I8Plan plan_of(int M, int N, int K) {
    I8Plan p = {TILE_64, 1, K, false};
    const auto tiles = [&](long long bm, long long bn) {
        return (M + bm - 1) / bm * ((N + bn - 1) / bn);
    };
    // The share of 256 CUs that whole rounds of 256 x 256 tiles keep busy.
    const long long t256 = tiles(256, 256);
    const bool full = t256 * 10 >= (t256 + 255) / 256 * 256 * 7;
    const int stages = std::max(1, ceil_div(K, 128));
    if (N <= 4096 ? M <= 32 && K <= 8192 : M <= 4 && K > 8192) {
        p.tile = FEW;
    } else if (M > 64 && full) {
        p.tile = TILE_256;
    } else if (M > 64 && tiles(128, 128) >= 192) {
        p.tile = TILE_128;
    } else {
        // Few tiles of many k, which make up for a second launch: at most a workgroup
        // a CU, ranges of at least ten stages.
        const long long t64 = std::max(1ll, tiles(64, 64));
        const int ranges = (int)std::min(256 / t64, stages / 10ll);
        if (ranges > 1 && stages >= 36) {
            p.span = ceil_div(stages, ranges) * 128;
            p.ranges = ceil_div(K, p.span);
        }
    }
    // A third stage of B hides more of a load's way, where the LDS that it takes
    // keeps no workgroup from a CU (256 x 4096 x 4096 14.4 -> 10.6 us, 64 x 6400 x 1600
    // 7.9 -> 6.6, 1024 x 4096 x 4096 21.7 -> 19.7; 16 x 50257 x 768, 786 tiles, it would
    // be 9.1 -> 10.6, 2048 x 4096 x 4096 36 -> 38).
    if (p.tile == TILE_64) p.deep = tiles(64, 64) * p.ranges <= DEEP_64;
    if (p.tile == TILE_128) p.deep = tiles(128, 128) <= DEEP_128;
    return p;
}

template <typename T>
void launch_i8(I8Args &a, const I8Plan &p, hipStream_t stream) {
    a.span = p.span;
    a.part_stride = ((long long)a.M * a.N + 3) / 4 * 4;
    typedef I8Tile<64, 64, 2, 2, 3, 3> Deep64;
    typedef I8Tile<128, 128, 2, 2, 3, 3> Deep128;
    static_assert(DEEP_64 * Deep64::BM * Deep64::BN * 4ll <= L2_BYTES &&
                      DEEP_128 * Deep128::BM * Deep128::BN * 4ll <= L2_BYTES,
                  "results of deep tiles fit the L2 caches");
    if (p.tile == FEW)
        a.M <= 16 ? launch_few<1, T>(a, stream) : launch_few<2, T>(a, stream);
    else if (p.ranges > 1)  // (at most 256 workgroups of 64 x 64 tiles)
        launch_ranges<Deep64, T>(a, p.ranges, stream);
    else if (p.tile == TILE_64)
        p.deep ? launch_tile<Deep64, T, true>(a, stream)
               : launch_tile<I8Tile<64, 64, 2, 2, 3, 2>, T, false>(a, stream);
    else if (p.tile == TILE_128)
        p.deep ? launch_tile<Deep128, T, true>(a, stream)
               : launch_tile<I8Tile<128, 128, 2, 2, 3, 2>, T, false>(a, stream);
    else
        launch_tile<I8Tile<256, 256, 2, 4, 3, 2>, T, false>(a, stream);
}

size_t bytes_of(const I8Plan &p, int M, int N) {
    return p.ranges == 1 ? 0 : ((size_t)M * N + 3) / 4 * 4 * sizeof(int) * p.ranges;
}

const char *size_fault(const GemmI8 *g) {
    if (g == nullptr) return "no arguments";
    if (element_size(g->type) == 0) return "unknown element type";
    if (g->M < 0 || g->N < 0 || g->K < 0) return "a negative size";
    if (g->K > MAX_K) return "K is above 131071";
    if (((long long)g->M + 63) / 64 * (((long long)g->N + 63) / 64) > (1 << 22))
        return "too many results for one call";
    return nullptr;
}

}  // namespace
}  // namespace bmb

extern "C" {

size_t gemm_i8_workspace(const GemmI8 *g) {
    using namespace bmb;
    if (size_fault(g) || g->M == 0 || g->N == 0) return 0;
    return bytes_of(plan_of(g->M, g->N, g->K), g->M, g->N);
}

int gemm_i8(const GemmI8 *g, hipStream_t stream) {
    using namespace bmb;
    const char *me = "gemm_i8";
    if (const char *why = size_fault(g)) return refuse(me, why);
    if (g->M == 0 || g->N == 0) return 0;
    if ((g->K > 0 && (!g->A || !g->B)) || !g->a_scales || !g->b_scales || !g->C)
        return refuse(me, "a null pointer");
    const int size = element_size(g->type);
    if (g->K > 0) {
        if (g->lda < g->K || g->ldb < g->K || g->lda >= (1 << 23) || g->ldb >= (1 << 23))
            return refuse(me, "lda or ldb is below K or not below 2^23");
        if (((uintptr_t)g->A | (uintptr_t)g->B | (unsigned long long)g->lda |
             (unsigned long long)g->ldb) % 16 != 0)
            return refuse(me, "A, B or their strides are no multiples of 16 bytes");
    }
    if (g->ldc < g->N || g->ldc >= (1 << 30)) return refuse(me, "ldc is below N or not below 2^30");
    if ((uintptr_t)g->C % size != 0 ||
        ((uintptr_t)g->a_scales | (uintptr_t)g->b_scales | (uintptr_t)g->bias) % 4 != 0)
        return refuse(me, "a buffer is no multiple of its element's size");
    const long long M = g->M, N = g->N;
    const auto clash = [&](const void *p, long long rows, long long stride, long long width) {
        const char *c = (const char *)g->C, *in = (const char *)p;
        return in != nullptr && width > 0 && c < in + ((rows - 1) * stride + width) &&
               in < c + ((M - 1) * g->ldc + N) * size;
    };
    if (clash(g->A, M, g->lda, g->K) || clash(g->B, N, g->ldb, g->K) ||
        clash(g->a_scales, M, 4, 4) || clash(g->b_scales, N, 4, 4) || clash(g->bias, N, 4, 4))
        return refuse(me, "C overlaps an input");
    I8Plan plan = plan_of(g->M, g->N, g->K);
    const size_t need = bytes_of(plan, g->M, g->N);
    if (g->work != nullptr && need > 0) {
        if (g->work_bytes < need) return refuse(me, "the workspace is too small");
        if ((uintptr_t)g->work % 16 != 0)
            return refuse(me, "the workspace is no multiple of 16 bytes");
        const char *w = (const char *)g->work;
        const auto within = [&](const void *p, long long rows, long long stride, long long width) {
            const char *in = (const char *)p;
            return in != nullptr && width > 0 && w < in + ((rows - 1) * stride + width) &&
                   in < w + need;
        };
        if (clash(w, 1, 0, need) || within(g->A, M, g->lda, g->K) ||
            within(g->B, N, g->ldb, g->K) || within(g->a_scales, M, 4, 4) ||
            within(g->b_scales, N, 4, 4) || within(g->bias, N, 4, 4))
            return refuse(me, "the workspace overlaps another buffer");
    }
    const auto go = [&](void *work) {
        I8Args a = {g->A, g->B, g->a_scales, g->b_scales, g->bias, (char *)g->C, g->lda, g->ldb,
                    g->ldc, g->M, g->N, g->K, 0, 0, 0, (int *)work, 0, 0};
        if (g->type == BMB_F32)
            launch_i8<float>(a, plan, stream);
        else if (g->type == BMB_F16)
            launch_i8<_Float16>(a, plan, stream);
        else
            launch_i8<__bf16>(a, plan, stream);
    };
    if (need == 0 || g->work != nullptr) {
        go(g->work);
        return 0;
    }
    if (!stream_capturing(stream)) {
        ScratchLease ws(SCRATCH_GEMM, need, stream);
        if (ws) {
            go(ws.get());
            return 0;
        }
    }
    plan.ranges = 1;
    plan.span = g->K;
    go(nullptr);
    return 0;
}

}  // extern "C"
