// 8-bit linear layers (gemm_i8, include/gemm.h).
//
// C = A B^T on v_mfma_i32_32x32x32_i8: both operands have k contiguous, so lane
// l supplies 16 consecutive bytes of row l % 32 at k = 16 (l / 32), and since
// both supply the same k in the same place, their order inside the instruction
// does not matter. Sums are whole numbers in 32 bits: exact, in any order.
// B goes in as the instruction's first operand, so a lane holds four
// consecutive columns of C in four registers.
//
// A stage is 128 k. Its tile of A and of B goes from global memory straight
// into LDS (16 bytes a lane, no registers), rows of 128 bytes whose eight
// 16-byte chunks are permuted by their row (chunk ^ (row / 2) % 8): the groups of 16
// lanes that a 128-bit read is served in then touch 16 different places
// modulo 256 bytes. Two stages in turn; the loads of the next are on their way
// while one is multiplied.
//
// Edges. Rows past the last are loaded from the last one and reach only
// results that are not stored. In a last stage that is not whole, chunks past
// the row's last one are loaded from that, and A's bytes from K on are masked
// to zero before they are multiplied (so B's need no mask).
#include <limits.h>

#include "args.hpp"
#include "common.hpp"
#include "launch.hpp"
#include "workspace.hpp"
#include "../../include/gemm.h"

namespace bmb {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int MAX_K = 131071;      // 128 * 128 * MAX_K < 2^31
constexpr int BK = 128, CHUNK = 16, CHUNKS = BK / CHUNK;

struct I8Args {
    const signed char *A, *B;
    const float *a_scales, *b_scales, *bias;
    char *C;
    long long lda, ldb, ldc;
    int M, N, K, tiles_m, tiles_n;
    long long first;
};

template <int BM_, int BN_, int WAVES_M_, int WAVES_N_>
struct I8Tile {
    static constexpr int BM = BM_, BN = BN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_;
    static constexpr int NT = 64 * WAVES_M * WAVES_N;
    static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, FM = WM / 32, FN = WN / 32;
};

typedef __attribute__((address_space(3))) void lds_void;

// ROWS rows of one operand's stage into LDS: lane i of a wave fills the i-th
// chunk of 1 KB, eight rows.
template <int ROWS, int NT>
struct Staging {
    static constexpr int LOADS = ROWS * CHUNKS / NT;
    int row[LOADS];  // byte offset of this lane's row
    int chunk[LOADS];
    __device__ __forceinline__ void setup(int rows, int ld) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int at = i * NT + threadIdx.x, r = at / CHUNKS;
            row[i] = min(r, rows - 1) * ld;
            chunk[i] = ((at % CHUNKS) ^ ((r >> 1) & 7)) * CHUNK;
        }
    }
    // k0: the stage's first k; last: the first k of the operand's last chunk.
    template <bool WHOLE>
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t p, char *lds, int k0,
                                         int last) const {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            char *to = lds + (i * NT + wave * 64) * CHUNK;
            const int off = WHOLE ? row[i] + chunk[i] : row[i] + min(chunk[i], last - k0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(p, (lds_void *)to, 16, off, k0, 0, 0);
        }
    }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t operand(const signed char *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<signed char *>(p), 0, 0xffffffff,
                                             0x00027000);
}

// Chunk c of row r of a staged tile.
__device__ __forceinline__ i32x4 chunk_at(const char *lds, int r, int c) {
    return *(const i32x4 *)(lds + r * BK + ((c ^ ((r >> 1) & 7)) * CHUNK));
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

template <typename Tile, typename T>
__global__ __launch_bounds__(Tile::NT) void i8_kernel(I8Args a) {
    constexpr int BM = Tile::BM, BN = Tile::BN, FM = Tile::FM, FN = Tile::FN;
    // Objects of their own, so that reads of one stage do not wait for the
    // loads into the other.
    __shared__ __attribute__((aligned(256))) char a0[BM * BK], a1[BM * BK];
    __shared__ __attribute__((aligned(256))) char b0[BN * BK], b1[BN * BK];
    int tm, tn;
    group_tile(xcd_remap((int)blockIdx.x, (int)gridDim.x), a.tiles_m, a.tiles_n, 8, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const __amdgpu_buffer_rsrc_t A = operand(a.A + (long long)m0 * a.lda);
    const __amdgpu_buffer_rsrc_t B = operand(a.B + (long long)n0 * a.ldb);
    Staging<BM, Tile::NT> sa;
    Staging<BN, Tile::NT> sb;
    sa.setup(a.M - m0, (int)a.lda);
    sb.setup(a.N - n0, (int)a.ldb);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / Tile::WAVES_N * Tile::WM, wn = wave % Tile::WAVES_N * Tile::WN;
    const int r = lane & 31, half = lane >> 5;

    i32x16 acc[FM][FN] = {};
    const auto load = [&](char *la, char *lb, int k0) {
        if (k0 + BK <= a.K) {
            sa.template load<true>(A, la, k0, 0);
            sb.template load<true>(B, lb, k0, 0);
        } else if (k0 < a.K) {
            const int last = (a.K - 1) / CHUNK * CHUNK;
            sa.template load<false>(A, la, k0, last);
            sb.template load<false>(B, lb, k0, last);
        }
    };
    const auto multiply = [&](const char *la, const char *lb, int k0) {
        const bool whole = k0 + BK <= a.K;
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) {
            i32x4 fa[FM], fb[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[i] = chunk_at(la, wm + i * 32 + r, 2 * kk + half);
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[j] = chunk_at(lb, wn + j * 32 + r, 2 * kk + half);
            if (!whole) {
#pragma unroll
                for (int i = 0; i < FM; ++i)
                    fa[i] = first_bytes(fa[i], a.K - k0 - (2 * kk + half) * CHUNK);
            }
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[j], fa[i], acc[i][j], 0, 0, 0);
        }
    };
    // vmcnt(0): this wave's loads are in LDS; the barrier: everybody's are.
    const auto ready = [] {
        __builtin_amdgcn_s_waitcnt(0x0f70);
        __syncthreads();
    };
    load(a0, b0, 0);
    for (int k0 = 0; k0 < a.K; k0 += 2 * BK) {
        ready();
        load(a1, b1, k0 + BK);
        multiply(a0, b0, k0);
        ready();
        if (k0 + BK < a.K) {
            load(a0, b0, k0 + 2 * BK);
            multiply(a1, b1, k0 + BK);
        }
    }

    // Lane: row l % 32 of C, columns 8 g + 4 (l / 32) + 0..3 in registers 4 g + 0..3.
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int m = m0 + wm + i * 32 + r;
        if (m >= a.M) continue;
        const float sm = a.a_scales[m];
        T *row = (T *)a.C + m * a.ldc;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int n = n0 + wn + j * 32 + 8 * (e / 4) + 4 * half + e % 4;
                if (n >= a.N) continue;
                const float y = (float)acc[i][j][e] * sm;
                row[n] = (T)__builtin_fmaf(y, a.b_scales[n], a.bias ? a.bias[n] : 0.0f);
            }
    }
}

template <typename Tile, typename T>
void launch_tile(I8Args &a, hipStream_t stream) {
    a.tiles_m = ceil_div(a.M, Tile::BM);
    a.tiles_n = ceil_div(a.N, Tile::BN);
    launch(i8_kernel<Tile, T>, dim3((long long)a.tiles_m * a.tiles_n), dim3(Tile::NT), 0, stream, a);
}

template <typename T>
void launch_i8(I8Args &a, hipStream_t stream) {
    const auto tiles = [&](long long bm, long long bn) {
        return (a.M + bm - 1) / bm * ((a.N + bn - 1) / bn);
    };
    if (tiles(256, 256) >= 256)
        launch_tile<I8Tile<256, 256, 2, 4>, T>(a, stream);
    else if (tiles(128, 128) >= 256)
        launch_tile<I8Tile<128, 128, 2, 2>, T>(a, stream);
    else
        launch_tile<I8Tile<64, 64, 2, 2>, T>(a, stream);
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

size_t gemm_i8_workspace(const GemmI8 *g) { return 0; }

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
    if (g->ldc < g->N || g->ldc > (1ll << 40)) return refuse(me, "ldc is below N or above 2^40");
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
    I8Args a = {g->A, g->B, g->a_scales, g->b_scales, g->bias, (char *)g->C, g->lda, g->ldb,
                g->ldc, g->M, g->N, g->K, 0, 0, 0};
    if (g->type == BMB_F32)
        launch_i8<float>(a, stream);
    else if (g->type == BMB_F16)
        launch_i8<_Float16>(a, stream);
    else
        launch_i8<__bf16>(a, stream);
    return 0;
}

}  // extern "C"
