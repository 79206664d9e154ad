// Root-mean-square norm with the residual's addition, out in the input's type
// or in 8 bits, its backward pass, and rows to 8 bits (include/nn.h states all
// three).
//
// All of them are bound by HBM: a row is read once, kept in registers across
// its reduction, and written once. G threads share a row (one, four, eight or
// sixteen waves), each with P pieces of 16 bytes, at most 16 elements, so that
// enough rows are on their way. Rows of more than 16384 take kernels that read
// them twice. At 5.15 TB/s, the rate of a copy: 8192 x 768 in fp32 with residual and
// sum 21.3 us (floor 19.6), its backward 22.6 (19.6; the next row is loaded while
// one is reduced, without that 28), 16381 x 4096 in bf16 113 (104), 50257 x 768 in
// fp32 to 8 bits 39 (37.5).
//
// The mean of the squares is held in 64 bits, and so are the products of the
// result: squares of fp32 numbers pass fp32's range, and so can rstd (1 ULP of
// the result is all that is lost). It costs nothing: HBM bounds.
//
// 8 bits. The values are v = s * w (exact in 64 bits: 24 x 24 bits), a = max
// |v|, and rstd cancels in q = 127 v / a. In fp32, y = s * w * (127 / a) is off
// by three roundings, at most 127 * 3 * 2^-24 < 2.3e-5, so unless y is that
// near to half-way between two whole numbers, rounding it gives q. Where it
// is near, the exact side of the half-way point decides: 254 v against (2
// floor(y) + 1) a, in 64 bits. So q is what exact arithmetic gives, whatever
// the order of anything.
#include <float.h>
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "args.hpp"
#include "common.hpp"
#include "launch.hpp"
#include "workspace.hpp"

namespace bmb {
namespace {

constexpr int MAX_C = 1 << 24;

template <typename T>
constexpr int piece_of() { return 16 / sizeof(T); }
// Rows start where their element's alignment lets them: 16-byte accesses at
// any multiple of it.
template <typename T, int N>
using Piece __attribute__((ext_vector_type(N))) = T;
template <typename T, int N>
struct Unaligned {
    typedef Piece<T, N> type __attribute__((aligned(sizeof(T))));
};

// Elements c .. c + N - 1 of a row of C as floats, zeros behind the last.
template <typename T, int N>
__device__ __forceinline__ void load_piece(const T *row, int c, int C, float (&v)[N]) {
    if (c + N <= C) {
        const Piece<T, N> x = *(const typename Unaligned<T, N>::type *)(row + c);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = (float)x[e];
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = c + e < C ? (float)row[c + e] : 0.0f;
    }
}
// The same as they are.
template <typename T, int N>
__device__ __forceinline__ Piece<T, N> load_raw(const T *row, int c, int C) {
    Piece<T, N> x = {};
    if (c + N <= C) {
        x = *(const typename Unaligned<T, N>::type *)(row + c);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (c + e < C) x[e] = row[c + e];
    }
    return x;
}
template <typename T, int N, typename V>
__device__ __forceinline__ void store_piece(T *row, int c, int C, const V (&v)[N]) {
    if (c + N <= C) {
        Piece<T, N> x;
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = (T)v[e];
        *(typename Unaligned<T, N>::type *)(row + c) = x;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (c + e < C) row[c + e] = (T)v[e];
    }
}

// The value of another lane of the DPP row or row group, 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ float from_lane(float x) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double from_lane(double x) {
    const int2 v = __builtin_bit_cast(int2, x);
    return __builtin_bit_cast(
        double, make_int2(__builtin_amdgcn_update_dpp(0, v.x, CTRL, ROWS, 0xf, false),
                          __builtin_amdgcn_update_dpp(0, v.y, CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ float last_lane(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ double last_lane(double x) {
    const int2 v = __builtin_bit_cast(int2, x);
    return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_readlane(v.x, 63),
                                                __builtin_amdgcn_readlane(v.y, 63)));
}
// f, for which 0 changes nothing, over the 64 lanes: inside rows of 16 lanes,
// then from row to row into lane 63, and to all.
template <typename V, typename F>
__device__ __forceinline__ V wave_all(V x, F &&f) {
    x = f(x, from_lane<0x111, 0xf>(x));
    x = f(x, from_lane<0x112, 0xf>(x));
    x = f(x, from_lane<0x114, 0xf>(x));
    x = f(x, from_lane<0x118, 0xf>(x));
    x = f(x, from_lane<0x142, 0xa>(x));
    x = f(x, from_lane<0x143, 0xc>(x));
    return last_lane(x);
}
// f over the G threads of a row (G = 64, or the whole workgroup), in a fixed
// order.
template <int G, typename V, typename F>
__device__ __forceinline__ V row_all(V x, V *part, F &&f) {
    x = wave_all(x, f);
    if constexpr (G > WAVE) {
        __syncthreads();  // part may still be read by the reduction before
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
        __syncthreads();
        x = part[0];
#pragma unroll
        for (int w = 1; w < G / WAVE; ++w) x = f(x, part[w]);
    }
    return x;
}
struct Add {
    template <typename V>
    __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Max {
    __device__ __forceinline__ double operator()(double a, double b) const { return fmax(a, b); }
};

// How a row's values become 8-bit numbers, from their largest magnitude.
struct Steps {
    double a;
    float inv;
    bool plain;  // fp32 may decide (no product of it is subnormal or infinite)
    bool none;   // q = 0: a row of zeros, or one with an infinity or a NaN
    __device__ __forceinline__ explicit Steps(double top) : a(top) {
        plain = a > 1e-30 && a < 1e30;
        none = !(a > 0.0 && a <= DBL_MAX);
        inv = plain ? (float)(127.0 / a) : 0.0f;
    }
    __device__ __forceinline__ int of(float s, float w) const {
        if (none) return 0;
        float y = s * w * inv, k = __builtin_rintf(y);
        if (!plain || fabsf(y - k) > 0.4999f) {
            const double v = (double)s * w;
            // (a is subnormal at the least: the quotient is finite)
            const double f =
                plain ? floor((double)y) : fmin(fmax(floor(v / a * 127.0), -127.0), 126.0);
            // (254 v takes up to 55 bits: it and what its rounding lost)
            const double most = 254.0 * v, rest = __builtin_fma(254.0, v, -most);
            const double side = __builtin_fma(-(2.0 * f + 1.0), a, most) + rest;
            const bool odd = ((int)f & 1) != 0;
            k = (float)(side > 0.0 || (side == 0.0 && odd) ? f + 1.0 : f);
        }
        return (int)k;
    }
    __device__ __forceinline__ float scale(double rstd) const {
        return a <= DBL_MAX ? (float)(a * rstd / 127.0) : NAN;
    }
};

struct NormArgs {
    const char *x, *residual;
    char *sum, *out;
    const float *weight;
    float *scales, *rstd;
    long long x_stride, residual_stride, sum_stride, out_stride;  // elements
    long long first;                                              // the launch's first row
    int rows, C;
    float eps;
};

// NORM: the norm, else (quantize_rows) the rows themselves. I8: out in 8 bits.
template <typename T, bool NORM, bool I8, int G, int P>
__global__ __launch_bounds__(G < 256 ? 256 : G) void rows_kernel(NormArgs a) {
    constexpr int N = piece_of<T>(), ROWS = G < 256 ? 256 / G : 1;
    __shared__ double part[2][G / WAVE];
    const int t = G < 256 ? threadIdx.x % G : threadIdx.x;
    const long long row = a.first + (long long)blockIdx.x * ROWS + (G < 256 ? threadIdx.x / G : 0);
    if (row >= a.rows) return;
    const T *x = (const T *)a.x + row * a.x_stride;
    const T *res = (const T *)a.residual + row * a.residual_stride;
    float s[P][N], w[P][N];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int c = (i * G + t) * N;
        load_piece<T, N>(x, c, a.C, s[i]);
        if constexpr (NORM) load_piece<float, N>(a.weight, c, a.C, w[i]);
    }
    if constexpr (NORM) {
        if (a.residual) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                float r[N];
                load_piece<T, N>(res, (i * G + t) * N, a.C, r);
#pragma unroll
                for (int e = 0; e < N; ++e) s[i][e] = (float)(T)(s[i][e] + r[e]);
            }
            if (a.sum) {
                T *sum = (T *)a.sum + row * a.sum_stride;
#pragma unroll
                for (int i = 0; i < P; ++i) store_piece<T, N>(sum, (i * G + t) * N, a.C, s[i]);
            }
        }
    }
    double square = 0.0, top = 0.0;
    bool bad = false;  // an infinity or a NaN
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if constexpr (NORM) square = __builtin_fma((double)s[i][e], (double)s[i][e], square);
            if constexpr (I8) {
                const double v = NORM ? (double)s[i][e] * w[i][e] : (double)s[i][e];
                top = fmax(top, fabs(v));
                bad |= !(fabsf(s[i][e]) <= FLT_MAX);
                if constexpr (NORM) bad |= !(fabsf(w[i][e]) <= FLT_MAX);
            }
        }
    double rstd = 1.0;
    if constexpr (NORM) {
        square = row_all<G>(square, part[0], Add());
        rstd = 1.0 / sqrt(square / a.C + (double)a.eps);
        if (a.rstd && t == 0) a.rstd[row] = (float)rstd;
    }
    if constexpr (I8) {
        top = row_all<G>(bad ? INFINITY : top, part[1], Max());
        const Steps steps(top);
        if (t == 0) a.scales[row] = steps.scale(rstd);
        signed char *out = (signed char *)a.out + row * a.out_stride;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            int q[N];
#pragma unroll
            for (int e = 0; e < N; ++e) q[e] = steps.of(s[i][e], NORM ? w[i][e] : 1.0f);
            store_piece<signed char, N>(out, (i * G + t) * N, a.C, q);
        }
    } else {
        T *out = (T *)a.out + row * a.out_stride;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float y[N];
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = (float)(s[i][e] * rstd * w[i][e]);
            store_piece<T, N>(out, (i * G + t) * N, a.C, y);
        }
    }
}

// Rows wider than the registers hold: a workgroup reads its row once for the
// reduction and once more for the result. Each thread reads again what it
// read before, so a result may be written over its input.
template <typename T, bool NORM, bool I8>
__global__ __launch_bounds__(1024) void wide_rows_kernel(NormArgs a) {
    constexpr int N = piece_of<T>(), G = 1024;
    __shared__ double part[2][G / WAVE];
    const long long row = a.first + blockIdx.x;
    const int t = threadIdx.x;
    const T *x = (const T *)a.x + row * a.x_stride;
    const T *res = (const T *)a.residual + row * a.residual_stride;
    T *sum = (T *)a.sum + row * a.sum_stride;
    const bool added = NORM && a.residual, kept = added && a.sum;
    const auto load = [&](int c, bool again, float(&s)[N]) {
        load_piece<T, N>(again && kept ? sum : x, c, a.C, s);
        if (added && !(again && kept)) {
            float r[N];
            load_piece<T, N>(res, c, a.C, r);
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] = (float)(T)(s[e] + r[e]);
        }
    };
    double square = 0.0, top = 0.0;
    bool bad = false;
    for (int c = t * N; c < a.C; c += G * N) {
        float s[N], w[N];
        load(c, false, s);
        if (kept) store_piece<T, N>(sum, c, a.C, s);
        if constexpr (NORM) load_piece<float, N>(a.weight, c, a.C, w);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if constexpr (NORM) square = __builtin_fma((double)s[e], (double)s[e], square);
            if constexpr (I8) {
                const double v = NORM ? (double)s[e] * w[e] : (double)s[e];
                top = fmax(top, fabs(v));
                bad |= !(fabsf(s[e]) <= FLT_MAX);
                if constexpr (NORM) bad |= !(fabsf(w[e]) <= FLT_MAX);
            }
        }
    }
    double rstd = 1.0;
    if constexpr (NORM) {
        square = row_all<G>(square, part[0], Add());
        rstd = 1.0 / sqrt(square / a.C + (double)a.eps);
        if (a.rstd && t == 0) a.rstd[row] = (float)rstd;
    }
    if constexpr (I8) top = row_all<G>(bad ? INFINITY : top, part[1], Max());
    const Steps steps(top);
    if (I8 && t == 0) a.scales[row] = steps.scale(rstd);
    for (int c = t * N; c < a.C; c += G * N) {
        float s[N], w[N];
        load(c, true, s);
        if constexpr (NORM) load_piece<float, N>(a.weight, c, a.C, w);
        if constexpr (I8) {
            int q[N];
#pragma unroll
            for (int e = 0; e < N; ++e) q[e] = steps.of(s[e], NORM ? w[e] : 1.0f);
            store_piece<signed char, N>((signed char *)a.out + row * a.out_stride, c, a.C, q);
        } else {
            float y[N];
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = (float)(s[e] * rstd * w[e]);
            store_piece<T, N>((T *)a.out + row * a.out_stride, c, a.C, y);
        }
    }
}

// ------------------------------------------------------------------ backward
struct GradArgs {
    const char *dout, *inp, *dres;
    char *dinp;
    const float *weight, *rstd;
    float *part;  // (blocks, C) sums of dout * xhat over a workgroup's rows, or null
    long long dout_stride, inp_stride, dres_stride, dinp_stride;
    long long first;    // the launch's first workgroup of the call's
    int rows, C, span;  // rows a workgroup
};

// A workgroup takes `span` consecutive rows, ROWS at a time, and keeps their
// sums for dweight in registers; a wave a row, the waves' sums meet in LDS.
template <typename T, int G, int P>
__global__ __launch_bounds__(G < 256 ? 256 : G) void grad_kernel(GradArgs a) {
    constexpr int N = piece_of<T>(), ROWS = G < 256 ? 256 / G : 1;
    extern __shared__ float sums[];  // ROWS > 1: (ROWS, C)
    __shared__ float part[G / WAVE];
    const int t = G < 256 ? threadIdx.x % G : threadIdx.x;
    const int lane_row = G < 256 ? threadIdx.x / G : 0;
    const long long block = a.first + blockIdx.x;
    const long long first = block * a.span, last = min((long long)a.rows, first + a.span);
    float w[P][N], dw[P][N];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        load_piece<float, N>(a.weight, (i * G + t) * N, a.C, w[i]);
#pragma unroll
        for (int e = 0; e < N; ++e) dw[i][e] = 0.0f;
    }
    // The next row's pieces are on their way while a row is reduced (1024 threads
    // have no registers for that).
    constexpr bool AHEAD = G < 1024;
    Piece<T, N> dr[P], xr[P], gr[P] = {};
    float rstd_next = 0.0f;
    const auto fetch = [&](long long row) {
        if (row >= last) return;
        const T *dout = (const T *)a.dout + row * a.dout_stride;
        const T *inp = (const T *)a.inp + row * a.inp_stride;
        const T *dres = (const T *)a.dres + row * a.dres_stride;
        rstd_next = a.rstd[row];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (i * G + t) * N;
            dr[i] = load_raw<T, N>(dout, c, a.C);
            xr[i] = load_raw<T, N>(inp, c, a.C);
            if (a.dres) gr[i] = load_raw<T, N>(dres, c, a.C);
        }
    };
    if (AHEAD) fetch(first + lane_row);
    for (long long row = first + lane_row; row < last; row += ROWS) {
        if (!AHEAD) fetch(row);
        const float rstd = rstd_next;
        float d[P][N], xhat[P][N], g[P][N], dot = 0.0f;
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                d[i][e] = (float)dr[i][e];
                xhat[i][e] = (float)xr[i][e] * rstd;
                g[i][e] = (float)gr[i][e];
                dw[i][e] = __builtin_fmaf(d[i][e], xhat[i][e], dw[i][e]);
                d[i][e] *= w[i][e];
                dot = __builtin_fmaf(d[i][e], xhat[i][e], dot);
            }
        if (AHEAD) fetch(row + ROWS);
        dot = row_all<G>(dot, part, Add()) / a.C;
        T *dinp = (T *)a.dinp + row * a.dinp_stride;
#pragma unroll
        for (int i = 0; i < P; ++i) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                g[i][e] += rstd * __builtin_fmaf(-xhat[i][e], dot, d[i][e]);
            store_piece<T, N>(dinp, (i * G + t) * N, a.C, g[i]);
        }
    }
    if (!a.part) return;
    float *out = a.part + block * a.C;
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int i = 0; i < P; ++i) store_piece<float, N>(out, (i * G + t) * N, a.C, dw[i]);
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i)
            store_piece<float, N>(sums + lane_row * a.C, (i * G + t) * N, a.C, dw[i]);
        __syncthreads();
        for (int c = threadIdx.x; c < a.C; c += 256) {
            float x = sums[c];
#pragma unroll
            for (int r = 1; r < ROWS; ++r) x += sums[r * a.C + c];
            out[c] = x;
        }
    }
}

// Wide rows: dinp with a second reading of the row. A thread adds up to 2^14 terms:
// in 64 bits (in fp32 their roundings reach 3400 u, u = 2^-24, in rows of 2^24) ...
template <typename T>
__global__ __launch_bounds__(1024) void wide_grad_kernel(GradArgs a) {
    constexpr int N = piece_of<T>(), G = 1024;
    __shared__ double part[G / WAVE];
    const long long row = a.first + blockIdx.x;
    const T *dout = (const T *)a.dout + row * a.dout_stride;
    const T *inp = (const T *)a.inp + row * a.inp_stride;
    const float rstd = a.rstd[row];
    float w[N], d[N], x[N];
    double sum = 0.0;
    for (int c = threadIdx.x * N; c < a.C; c += G * N) {
        load_piece<T, N>(dout, c, a.C, d);
        load_piece<T, N>(inp, c, a.C, x);
        load_piece<float, N>(a.weight, c, a.C, w);
#pragma unroll
        for (int e = 0; e < N; ++e)
            sum = __builtin_fma((double)(d[e] * w[e]), (double)(x[e] * rstd), sum);
    }
    const float dot = (float)(row_all<G>(sum, part, Add()) / a.C);
    for (int c = threadIdx.x * N; c < a.C; c += G * N) {
        float g[N];
        load_piece<T, N>(dout, c, a.C, d);
        load_piece<T, N>(inp, c, a.C, x);
        load_piece<float, N>(a.weight, c, a.C, w);
        if (a.dres) {
            load_piece<T, N>((const T *)a.dres + row * a.dres_stride, c, a.C, g);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) g[e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < N; ++e)
            g[e] += rstd * __builtin_fmaf(-(x[e] * rstd), dot, d[e] * w[e]);
        store_piece<T, N>((T *)a.dinp + row * a.dinp_stride, c, a.C, g);
    }
}
// ... and, before it (dinp may be dout or inp), the sums for dweight.
template <typename T>
__global__ __launch_bounds__(256) void wide_sums_kernel(GradArgs a) {
    constexpr int N = piece_of<T>();
    const int chunks = (a.C + 256 * N - 1) / (256 * N);
    const long long block = (a.first + blockIdx.x) / chunks;
    const int c = ((int)((a.first + blockIdx.x) % chunks) * 256 + threadIdx.x) * N;
    if (c >= a.C) return;
    const long long first = block * a.span, last = min((long long)a.rows, first + a.span);
    float dw[N] = {};
    for (long long row = first; row < last; ++row) {
        float d[N], x[N];
        load_piece<T, N>((const T *)a.dout + row * a.dout_stride, c, a.C, d);
        load_piece<T, N>((const T *)a.inp + row * a.inp_stride, c, a.C, x);
        const float rstd = a.rstd[row];
#pragma unroll
        for (int e = 0; e < N; ++e) dw[e] = __builtin_fmaf(d[e], x[e] * rstd, dw[e]);
    }
    store_piece<float, N>(a.part + block * a.C, c, a.C, dw);
}

// dweight += the workgroups' sums, in a fixed order, in 64 bits: 16 columns a
// workgroup, 256 rows of sums at once.
__global__ __launch_bounds__(1024) void join_sums_kernel(float *dweight, const float *part,
                                                         int blocks, int C) {
    __shared__ double lds[16][16];
    const int x = threadIdx.x % 4 * 4, y = threadIdx.x / 4, c = blockIdx.x * 16 + x;
    const int column = blockIdx.x * 16 + threadIdx.x;
    const float before = threadIdx.x < 16 && column < C ? dweight[column] : 0.0f;
    double s[4] = {};
    for (int b = y; b < blocks; b += 256) {
        float v[4];
        load_piece<float, 4>(part + (long long)b * C, c, C, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int d = 32; d > 2; d >>= 1) s[e] += __shfl_xor(s[e], d);
        if ((threadIdx.x & 63) < 4) lds[threadIdx.x >> 6][x + e] = s[e];
    }
    __syncthreads();
    if (threadIdx.x < 16 && column < C) {
        double sum = before;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += lds[i][threadIdx.x];
        dweight[column] = (float)sum;
    }
}

// Threads of a row and pieces of each, at most `elements` a thread; G = 0: the
// wide kernels.
struct Shape {
    int G, P;
};
Shape shape_of(int C, int size, int elements) {
    const int pieces = ceil_div(C, 16 / size), most = elements * size / 16;
    for (int G : {64, 256, 512, 1024})
        if (pieces <= most * G) return {G, ceil_div(pieces, G)};
    return {0, 0};
}

// f(G, P) as constants, for the P from LEAST to MOST that shape_of gives.
template <int LEAST, int MOST, int G, typename F>
void with_pieces(int P, F &&f) {
    if constexpr (MOST >= LEAST) {
        if (P == MOST)
            f(std::integral_constant<int, G>(), std::integral_constant<int, MOST>());
        else
            with_pieces<LEAST, MOST - 1, G>(P, f);
    }
}
// (G threads have more pieces than MOST times the next smaller G holds)
template <int MOST, typename F>
void with_shape(Shape s, F &&f) {
    if (s.G == 64) with_pieces<1, MOST, 64>(s.P, f);
    else if (s.G == 256) with_pieces<MOST * 64 / 256 + 1, MOST, 256>(s.P, f);
    else if (s.G == 512) with_pieces<MOST * 256 / 512 + 1, MOST, 512>(s.P, f);
    else with_pieces<MOST * 512 / 1024 + 1, MOST, 1024>(s.P, f);
}

template <typename T, bool NORM, bool I8>
void launch_rows(NormArgs &a, hipStream_t stream) {
    constexpr int MOST = 16 / piece_of<T>();  // 16 elements a thread
    const Shape s = shape_of(a.C, sizeof(T), 16);
    const auto go = [&](auto kernel, int threads, int rows_each) {
        in_launches(((long long)a.rows + rows_each - 1) / rows_each, threads,
                    [&](long long first, unsigned n) {
                        a.first = first * rows_each;
                        launch(kernel, dim3(n), dim3(threads), 0, stream, a);
                    });
    };
    if (s.G == 0)
        go(wide_rows_kernel<T, NORM, I8>, 1024, 1);
    else
        with_shape<MOST>(s, [&](auto G, auto P) {
            go(rows_kernel<T, NORM, I8, G(), P()>, std::max(256, (int)G),
               G() < 256 ? 256 / G() : 1);
        });
}

// Workgroups of the backward and rows of each.
struct Spans {
    int blocks, span;
};
Spans spans_of(int rows) {
    Spans s;
    // Two workgroups a CU (16381 x 4096 in bf16, where each is four times as wide:
    // one 104 us, two 108, four 116; 8192 x 768 in fp32: 20.8, 18.5 and 19.8), and
    // at most 64 rows.
    s.span = (int)std::min(64ll, std::max(4ll, (rows + 511ll) / 512));
    s.blocks = (int)(((long long)rows + s.span - 1) / s.span);
    return s;
}

template <typename T>
void launch_grad(GradArgs &a, hipStream_t stream) {
    constexpr int MOST = 16 / piece_of<T>();  // 16 elements a thread
    const Shape s = shape_of(a.C, sizeof(T), 16);
    const Spans n = spans_of(a.rows);
    a.span = n.span;
    const auto go = [&](auto kernel, long long blocks, int threads, size_t lds) {
        in_launches(blocks, threads, [&](long long first, unsigned count) {
            a.first = first;
            launch(kernel, dim3(count), dim3(threads), lds, stream, a);
        });
    };
    if (s.G == 0) {
        const long long chunks = ceil_div(a.C, 256 * piece_of<T>());
        if (a.part) go(wide_sums_kernel<T>, chunks * n.blocks, 256, 0);
        go(wide_grad_kernel<T>, a.rows, 1024, 0);
    } else {
        with_shape<MOST>(s, [&](auto G, auto P) {
            const size_t lds = G() < 256 ? (size_t)a.C * (256 / G()) * sizeof(float) : 0;
            go(grad_kernel<T, G(), P()>, n.blocks, std::max(256, (int)G), lds);
        });
    }
}

const char *grad_fault(const RmsNormGrad *g) {
    if (g == nullptr) return "no arguments";
    if (element_size(g->type) == 0) return "unknown element type";
    if (g->rows < 0 || g->C < 1 || g->C > MAX_C) return "rows is negative, or C not 1 to 2^24";
    return nullptr;
}

bool bad_stride(long long stride, long long width, bool result) {
    return (stride < width && (result || stride != 0)) || stride > (1ll << 40);
}

}  // namespace
}  // namespace bmb

extern "C" {

int rms_norm_forward(const RmsNorm *n, hipStream_t stream) {
    using namespace bmb;
    const char *me = "rms_norm_forward";
    if (n == nullptr) return refuse(me, "no arguments");
    const int size = element_size(n->type);
    if (size == 0) return refuse(me, "unknown element type");
    const bool i8 = n->out_type == BMB_I8;
    if (!i8 && n->out_type != n->type)
        return refuse(me, "out_type is neither the input's type nor BMB_I8");
    if (n->rows < 0 || n->C < 1 || n->C > MAX_C)
        return refuse(me, "rows is negative, or C not 1 to 2^24");
    if (!(n->eps > 0.0f) || !(n->eps <= FLT_MAX)) return refuse(me, "eps is not above 0");
    if (n->rows == 0) return 0;
    if (!n->x || !n->weight || !n->out || (i8 && !n->scales)) return refuse(me, "a null pointer");
    if (n->sum && !n->residual) return refuse(me, "sum without residual");
    const int out_size = i8 ? 1 : size;
    if (((uintptr_t)n->x | (uintptr_t)n->residual | (uintptr_t)n->sum) % size != 0 ||
        (uintptr_t)n->out % out_size != 0 ||
        ((uintptr_t)n->weight | (uintptr_t)n->scales | (uintptr_t)n->rstd) % 4 != 0)
        return refuse(me, "a buffer is no multiple of its element's size");
    if (bad_stride(n->x_stride, n->C, false) ||
        (n->residual && bad_stride(n->residual_stride, n->C, false)) ||
        (n->sum && bad_stride(n->sum_stride, n->C, true)) ||
        bad_stride(n->out_stride, n->C, true))
        return refuse(me, "a stride is below the row's width or above 2^40");
    const long long wide = (long long)n->C * size, R = n->rows;
    const Rows x = {n->x, n->x_stride * size, wide};
    const Rows res = {n->residual, n->residual_stride * size, wide};
    const Rows sum = {n->sum, n->sum_stride * size, wide};
    const Rows out = {n->out, n->out_stride * out_size, (long long)n->C * out_size};
    const Rows scales = {i8 ? n->scales : nullptr, 4, 4}, rstd = {n->rstd, 4, 4};
    const Rows weight = {n->weight, 0, 4ll * n->C};
    const auto clash = [&](const Rows &result, const Rows &input, bool in_place) {
        return overlap(result, input, R) && !(in_place && same(result, input, R));
    };
    if (clash(sum, x, true) || clash(sum, res, true) || clash(out, x, !i8) ||
        clash(out, res, !i8) || overlap(sum, out, R))
        return refuse(me, "results overlap inputs or each other in part");
    for (const Rows &r : {scales, rstd})
        for (const Rows &o : {x, res, sum, out, weight})
            if (overlap(r, o, R)) return refuse(me, "scales or rstd overlaps another buffer");
    if (overlap(scales, rstd, R) || overlap(sum, weight, R) || overlap(out, weight, R))
        return refuse(me, "results overlap weight or each other");
    NormArgs a = {(const char *)n->x, (const char *)n->residual, (char *)n->sum, (char *)n->out,
                  n->weight, n->scales, n->rstd, n->x_stride, n->residual_stride, n->sum_stride,
                  n->out_stride, 0, n->rows, n->C, n->eps};
    if (n->type == BMB_F32)
        i8 ? launch_rows<float, true, true>(a, stream) : launch_rows<float, true, false>(a, stream);
    else if (n->type == BMB_F16)
        i8 ? launch_rows<_Float16, true, true>(a, stream)
           : launch_rows<_Float16, true, false>(a, stream);
    else
        i8 ? launch_rows<__bf16, true, true>(a, stream)
           : launch_rows<__bf16, true, false>(a, stream);
    return 0;
}

int quantize_rows(signed char *out, long long out_stride, float *scales, const void *x,
                  long long x_stride, int type, int rows, int C, hipStream_t stream) {
    using namespace bmb;
    const char *me = "quantize_rows";
    const int size = element_size(type);
    if (size == 0) return refuse(me, "unknown element type");
    if (rows < 0 || C < 1 || C > MAX_C) return refuse(me, "rows is negative, or C not 1 to 2^24");
    if (rows == 0) return 0;
    if (!out || !scales || !x) return refuse(me, "a null pointer");
    if ((uintptr_t)x % size != 0 || (uintptr_t)scales % 4 != 0)
        return refuse(me, "a buffer is no multiple of its element's size");
    if (bad_stride(x_stride, C, false) || bad_stride(out_stride, C, true))
        return refuse(me, "a stride is below the row's width or above 2^40");
    const Rows from = {x, x_stride * size, (long long)C * size}, to = {out, out_stride, C};
    const Rows s = {scales, 4, 4};
    if (overlap(to, from, rows) || overlap(s, from, rows) || overlap(s, to, rows))
        return refuse(me, "results overlap the input or each other");
    NormArgs a = {(const char *)x, nullptr, nullptr, (char *)out, nullptr, scales, nullptr,
                  x_stride, 0, 0, out_stride, 0, rows, C, 0.0f};
    if (type == BMB_F32)
        launch_rows<float, false, true>(a, stream);
    else if (type == BMB_F16)
        launch_rows<_Float16, false, true>(a, stream);
    else
        launch_rows<__bf16, false, true>(a, stream);
    return 0;
}

size_t rms_norm_backward_workspace(const RmsNormGrad *g) {
    using namespace bmb;
    if (grad_fault(g) || g->rows == 0 || !g->dweight) return 0;
    return (size_t)spans_of(g->rows).blocks * g->C * sizeof(float);
}

int rms_norm_backward(const RmsNormGrad *g, hipStream_t stream) {
    using namespace bmb;
    const char *me = "rms_norm_backward";
    if (const char *why = grad_fault(g)) return refuse(me, why);
    if (g->rows == 0) return 0;
    const int size = element_size(g->type);
    if (!g->dout || !g->inp || !g->weight || !g->rstd || !g->dinp)
        return refuse(me, "a null pointer");
    if (((uintptr_t)g->dout | (uintptr_t)g->inp | (uintptr_t)g->dres | (uintptr_t)g->dinp) % size !=
            0 ||
        ((uintptr_t)g->weight | (uintptr_t)g->rstd | (uintptr_t)g->dweight | (uintptr_t)g->work) %
                4 !=
            0)
        return refuse(me, "a buffer is no multiple of its element's size");
    if (bad_stride(g->dout_stride, g->C, false) || bad_stride(g->inp_stride, g->C, false) ||
        (g->dres && bad_stride(g->dres_stride, g->C, false)) ||
        bad_stride(g->dinp_stride, g->C, true))
        return refuse(me, "a stride is below the row's width or above 2^40");
    const long long wide = (long long)g->C * size, R = g->rows;
    const Rows dinp = {g->dinp, g->dinp_stride * size, wide};
    const Rows dw = {g->dweight, 0, 4ll * g->C}, weight = {g->weight, 0, 4ll * g->C};
    const Rows rstd = {g->rstd, 4, 4};
    for (const Rows &in : {Rows{g->dout, g->dout_stride * size, wide},
                           Rows{g->inp, g->inp_stride * size, wide},
                           Rows{g->dres, g->dres_stride * size, wide}}) {
        if (overlap(dinp, in, R) && !same(dinp, in, R))
            return refuse(me, "dinp overlaps an input in part");
        if (overlap(dw, in, R)) return refuse(me, "dweight overlaps another buffer");
    }
    if (overlap(dw, dinp, R) || overlap(dw, weight, R) || overlap(dw, rstd, R) ||
        overlap(dinp, weight, R) || overlap(dinp, rstd, R))
        return refuse(me, "results overlap weight, rstd or each other");
    const size_t need = rms_norm_backward_workspace(g);
    if (need > 0 && g->work == nullptr && stream_capturing(stream))
        return refuse(me, "a captured call needs a workspace of the caller's");
    if (g->work != nullptr && g->work_bytes < need) return refuse(me, "the workspace is too small");
    const Rows work = {need > 0 ? g->work : nullptr, 0, (long long)need};
    for (const Rows &o : {dinp, dw, weight, rstd, Rows{g->dout, g->dout_stride * size, wide},
                          Rows{g->inp, g->inp_stride * size, wide},
                          Rows{g->dres, g->dres_stride * size, wide}})
        if (overlap(work, o, R)) return refuse(me, "the workspace overlaps another buffer");
    const auto go = [&](float *part) {
        GradArgs a = {(const char *)g->dout, (const char *)g->inp, (const char *)g->dres,
                      (char *)g->dinp, g->weight, g->rstd, part, g->dout_stride, g->inp_stride,
                      g->dres_stride, g->dinp_stride, 0, g->rows, g->C, 0};
        if (g->type == BMB_F32)
            launch_grad<float>(a, stream);
        else if (g->type == BMB_F16)
            launch_grad<_Float16>(a, stream);
        else
            launch_grad<__bf16>(a, stream);
        if (part)
            launch(join_sums_kernel, dim3(ceil_div(g->C, 16)), dim3(1024), 0, stream, g->dweight,
                   part, spans_of(g->rows).blocks, g->C);
    };
    if (need == 0) {
        go(nullptr);
    } else if (g->work != nullptr) {
        go((float *)g->work);
    } else {
        ScratchLease ws(SCRATCH_NN, need, stream);
        if (!ws) return refuse(me, "no memory for the workspace");
        go((float *)ws.get());
    }
    return 0;
}

}  // extern "C"
