// Rotary positions (include/nn.h states them).
//
// A pair (x, y) at position p becomes amplitude * (x cos - y sin, y cos + x
// sin) of the angle p * freq. The angle passes 2^17 radians in long contexts, so
// it is formed in 64 bits, in turns (p * freq / 2 pi), and its whole turns are
// dropped there; what is left is below half a turn and fp32 keeps it to 2^-25
// of a turn.
//
// Bound by HBM, or by a launch for a decoding step: each workgroup takes one
// or more tokens, its threads first put the sine and cosine of each pair into
// LDS (one sincospi each, for all heads of the token), then turn pieces of
// the heads. 8192 tokens of 24 heads in fp32, in place, 32 dims of each: 10.6-11.2
// us, 4.5-4.7 TB/s (the copy's rate gives 9.8); 64 tokens of 40 heads of 128: 3.5 us, a
// launch.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "args.hpp"
#include "common.hpp"
#include "launch.hpp"
#include "paged.hpp"

namespace bmb {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_HEAD = 256, MAX_PAIRS = MAX_HEAD / 2;

struct RotaryArgs {
    const char *in;
    char *out;
    const int *positions;
    long long in_stride, out_stride;  // elements
    long long first;                  // the launch's first workgroup of the call's
    int tokens, heads, head_size, pairs;
    int each;                // tokens a workgroup
    int turns, items;        // pieces to turn, and all pieces, of a token
    FastDiv per_head, rest;  // pieces of a head that turn, and that pass
    float amplitude, sign;
    double freq[MAX_PAIRS];  // turns a position
};

template <typename T, int N>
struct Elements {
    typedef T vec __attribute__((ext_vector_type(N)));
    typedef vec type __attribute__((aligned(sizeof(T))));
};
template <typename T>
struct Elements<T, 1> {
    typedef T vec, type;
};
template <typename T, int N>
__device__ __forceinline__ void load_n(const T *p, float (&v)[N]) {
    const typename Elements<T, N>::vec x = *(const typename Elements<T, N>::type *)p;
    if constexpr (N == 1) {
        v[0] = (float)x;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = (float)x[e];
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T *p, const float (&v)[N]) {
    typename Elements<T, N>::vec x;
    if constexpr (N == 1) {
        x = (T)v[0];
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = (T)v[e];
    }
    *(typename Elements<T, N>::type *)p = x;
}

// A piece is N pairs: N elements of either half, or 2 N neighbours. Elements
// that pass are copied N at a time.
template <typename T, bool HALF, int N>
__global__ __launch_bounds__(THREADS) void rotary_kernel(RotaryArgs a) {
    extern __shared__ float2 turn[];  // (each, pairs): cos, sin
    const long long token0 = (a.first + blockIdx.x) * a.each;
    const int count = (int)min((long long)a.each, a.tokens - token0);
    for (int i = threadIdx.x; i < count * a.pairs; i += THREADS) {
        const int t = i / a.pairs, p = i - t * a.pairs;
        const double turns = a.positions[token0 + t] * a.freq[p];
        float sin, cos;
        sincospif(2.0f * (float)(turns - rint(turns)), &sin, &cos);
        turn[i] = make_float2(a.amplitude * cos, a.amplitude * a.sign * sin);
    }
    __syncthreads();
    for (int t = 0; t < count; ++t) {
        const T *in = (const T *)a.in + (token0 + t) * a.in_stride;
        T *out = (T *)a.out + (token0 + t) * a.out_stride;
        for (int i = threadIdx.x; i < a.items; i += THREADS) {
            if (i < a.turns) {
                const int head = a.per_head.quot(i), p = (i - head * (int)a.per_head.d) * N;
                const int at = head * a.head_size;
                float x[N], y[N], u[N], v[N];
                if constexpr (HALF) {
                    load_n<T, N>(in + at + p, x);
                    load_n<T, N>(in + at + p + a.pairs, y);
                } else {
                    float xy[2 * N];
                    load_n<T, 2 * N>(in + at + 2 * p, xy);
#pragma unroll
                    for (int e = 0; e < N; ++e) x[e] = xy[2 * e], y[e] = xy[2 * e + 1];
                }
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float2 cs = turn[t * a.pairs + p + e];
                    u[e] = x[e] * cs.x - y[e] * cs.y;
                    v[e] = y[e] * cs.x + x[e] * cs.y;
                }
                if constexpr (HALF) {
                    store_n<T, N>(out + at + p, u);
                    store_n<T, N>(out + at + p + a.pairs, v);
                } else {
                    float xy[2 * N];
#pragma unroll
                    for (int e = 0; e < N; ++e) xy[2 * e] = u[e], xy[2 * e + 1] = v[e];
                    store_n<T, 2 * N>(out + at + 2 * p, xy);
                }
            } else {
                const int j = i - a.turns, head = a.rest.quot(j);
                const int at = head * a.head_size + 2 * a.pairs + (j - head * (int)a.rest.d) * N;
                float x[N];
                load_n<T, N>(in + at, x);
                store_n<T, N>(out + at, x);
            }
        }
    }
}

// Most pairs of a piece: 16 bytes of either half, or of neighbours.
template <typename T, bool HALF>
constexpr int most_pairs() { return 16 / sizeof(T) / (HALF ? 1 : 2); }

// f(N) as a constant, for N from MOST down in halves.
template <int MOST, typename F>
void with_pairs(int N, F &&f) {
    if (N == MOST)
        f(std::integral_constant<int, MOST>());
    else if constexpr (MOST > 1)
        with_pairs<MOST / 2>(N, f);
}

// rest: elements of a head that are copied.
template <typename T, bool HALF>
void launch_rotary(RotaryArgs &a, int rest, hipStream_t stream) {
    int N = most_pairs<T, HALF>();
    while (a.pairs % N != 0 || rest % N != 0) N /= 2;
    a.turns = a.heads * (a.pairs / N);
    a.items = a.turns + (rest ? a.heads * (rest / N) : 0);
    a.per_head = FastDiv::of(a.pairs / N);
    a.rest = FastDiv::of(std::max(1, rest / N));
    a.each = std::max(1, THREADS / a.items);
    with_pairs<most_pairs<T, HALF>()>(N, [&](auto pairs) {
        in_launches(((long long)a.tokens + a.each - 1) / a.each, THREADS,
                    [&](long long first, unsigned n) {
                        a.first = first;
                        const size_t lds = a.each * a.pairs * sizeof(float2);
                        launch(rotary_kernel<T, HALF, pairs()>, dim3(n), dim3(THREADS), lds, stream,
                               a);
                    });
    });
}

const char *plan_fault(const Rotary *r) {
    if (r == nullptr) return "no plan";
    if (r->head_size < 2 || r->head_size > MAX_HEAD) return "head size is not 2 to 256";
    if (r->dims < 2 || r->dims % 2 != 0 || r->dims > r->head_size)
        return "dims is odd, or not 2 to the head size";
    return nullptr;
}

int run(const char *me, const Rotary *r, void *out, long long out_stride, const void *in,
        long long in_stride, int type, int tokens, int heads, const int *positions, float sign,
        hipStream_t stream) {
    if (const char *why = plan_fault(r)) return refuse(me, why);
    if (r->layout != BMB_ROTARY_HALF && r->layout != BMB_ROTARY_PAIRS)
        return refuse(me, "unknown layout");
    const int size = element_size(type);
    if (size == 0) return refuse(me, "unknown element type");
    if (tokens < 0 || heads < 1 || heads > 65536)
        return refuse(me, "tokens is negative, or heads not 1 to 65536");
    if (tokens == 0) return 0;
    if (!out || !in || !positions) return refuse(me, "a null pointer");
    if (((uintptr_t)out | (uintptr_t)in) % size != 0 || (uintptr_t)positions % 4 != 0)
        return refuse(me, "a buffer is no multiple of its element's size");
    const long long width = (long long)heads * r->head_size;
    if (out_stride < width || (in_stride < width && in_stride != 0) || out_stride > (1ll << 40) ||
        in_stride > (1ll << 40))
        return refuse(me, "a stride is below the heads' width or above 2^40");
    const Rows from = {in, in_stride * size, width * size};
    const Rows to = {out, out_stride * size, width * size};
    const Rows pos = {positions, 4, 4};
    const bool in_place = same(to, from, tokens);
    if (overlap(to, from, tokens) && !in_place)
        return refuse(me, "the result overlaps the input in part");
    if (overlap(to, pos, tokens)) return refuse(me, "the result overlaps positions");
    RotaryArgs a = {};
    a.in = (const char *)in;
    a.out = (char *)out;
    a.positions = positions;
    a.in_stride = in_stride;
    a.out_stride = out_stride;
    a.tokens = tokens;
    a.heads = heads;
    a.head_size = r->head_size;
    a.pairs = r->dims / 2;
    a.amplitude = r->amplitude;
    a.sign = sign;
    for (int i = 0; i < a.pairs; ++i) a.freq[i] = r->freq[i] / (2.0 * M_PI);
    // What passes is copied, but for in place.
    const int rest = in_place ? 0 : r->head_size - r->dims;
    const bool half = r->layout == BMB_ROTARY_HALF;
    if (type == BMB_F32)
        half ? launch_rotary<float, true>(a, rest, stream)
             : launch_rotary<float, false>(a, rest, stream);
    else if (type == BMB_F16)
        half ? launch_rotary<_Float16, true>(a, rest, stream)
             : launch_rotary<_Float16, false>(a, rest, stream);
    else
        half ? launch_rotary<__bf16, true>(a, rest, stream)
             : launch_rotary<__bf16, false>(a, rest, stream);
    return 0;
}

}  // namespace
}  // namespace bmb

extern "C" {

int rotary_frequencies(Rotary *r, double base, int scaling, double factor, int trained_len,
                       double slow, double fast) {
    using namespace bmb;
    const char *me = "rotary_frequencies";
    if (const char *why = plan_fault(r)) return refuse(me, why);
    if (!(base > 0.0) || !std::isfinite(base)) return refuse(me, "base is not above 0");
    if (scaling < BMB_ROTARY_UNSCALED || scaling > BMB_ROTARY_PARTS)
        return refuse(me, "unknown scaling");
    if (scaling != BMB_ROTARY_UNSCALED && (!(factor >= 1.0) || !std::isfinite(factor)))
        return refuse(me, "factor is below 1");
    if (scaling == BMB_ROTARY_PARTS &&
        (trained_len < 1 || !(slow >= 0.0) || !(fast > slow) || !std::isfinite(fast)))
        return refuse(me, "trained_len is below 1, or not 0 <= slow < fast");
    const double n = r->dims;
    if (scaling == BMB_ROTARY_BASE && r->dims > 2) base *= pow(factor, n / (n - 2.0));
    // (the last frequency is the farthest from 1)
    if (!std::isfinite(base) || !std::isfinite(pow(base, 2.0 / n - 1.0)))
        return refuse(me, "the scaled base or a frequency is not finite");
    for (int i = 0; i < r->dims / 2; ++i) {
        double f = pow(base, -2.0 * i / n);
        if (scaling == BMB_ROTARY_LINEAR) f /= factor;
        if (scaling == BMB_ROTARY_PARTS) {
            const double turns = trained_len * f / (2.0 * M_PI);
            const double keep = std::min(1.0, std::max(0.0, (turns - slow) / (fast - slow)));
            f = f * keep + f / factor * (1.0 - keep);
        }
        r->freq[i] = f;
    }
    return 0;
}

int rotary_forward(const Rotary *plan, void *out, long long out_stride, const void *inp,
                   long long inp_stride, int type, int tokens, int heads, const int *positions,
                   hipStream_t stream) {
    return bmb::run("rotary_forward", plan, out, out_stride, inp, inp_stride, type, tokens, heads,
                    positions, 1.0f, stream);
}

int rotary_backward(const Rotary *plan, void *dinp, long long dinp_stride, const void *dout,
                    long long dout_stride, int type, int tokens, int heads, const int *positions,
                    hipStream_t stream) {
    return bmb::run("rotary_backward", plan, dinp, dinp_stride, dout, dout_stride, type, tokens,
                    heads, positions, -1.0f, stream);
}

}  // extern "C"
