// Pages, slots and positions of a generation step (paged_plan) and the copy of
// its keys and values into the paged cache (paged_append); include/flash.h
// states both.
#include "launch.hpp"
#include "paged.hpp"

namespace bmb {
namespace {

constexpr int PLAN_MAX_REQUESTS = 8192;  // 16 bytes of LDS each
constexpr int PLAN_MAX_BLOCKS = 512;

struct PlanArgs {
    PagedPlan p;
    FastDiv page;
    bool fill, finish;  // which halves this launch does
};

// One request's part in the step, before the pool's limits.
struct Ask {
    int held, have;  // tokens, pages
    uint32_t want, need;
    bool ended;
};

__device__ __forceinline__ Ask ask_of(const PlanArgs &a, int r) {
    const PagedPlan &p = a.p;
    const int cap = p.max_pages * p.page_size;
    Ask x;
    const int n = p.new_tokens[r];
    x.held = min(max(p.lens[r], 0), cap);
    x.have = a.page.quot(x.held + p.page_size - 1);
    x.ended = n < 0;
    x.want = n > 0 && n <= cap - x.held ? n : 0;
    x.need = x.want ? a.page.quot(x.held + (int)x.want + p.page_size - 1) - x.have : 0;
    return x;
}

// Inclusive scans of two counts over the workgroup; totals are their last
// values. A wave sums its rows of 64 in registers, then every wave adds the
// sums of the waves before it.
template <int THREADS>
__device__ __forceinline__ void block_scan(uint32_t &x, uint32_t &y, uint32_t &tx, uint32_t &ty,
                                           uint32_t (*part)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    x = wave_scan(x);
    y = wave_scan(y);
    __syncthreads();  // part may still be read by the scan before
    if (lane == 63) {
        part[wave][0] = x;
        part[wave][1] = y;
    }
    __syncthreads();
    uint32_t bx = 0, by = 0;
    tx = ty = 0;
#pragma unroll
    for (int w = 0; w < THREADS / WAVE; ++w) {
        if (w == wave) {
            bx = tx;
            by = ty;
        }
        tx = add_sat(tx, part[w][0]);
        ty = add_sat(ty, part[w][1]);
    }
    x = add_sat(bx, x);
    y = add_sat(by, y);
}

// Latency, not bytes: a decoding step of 64 requests takes 4.2 us, 512 requests
// with 260 000 prompt tokens 6.4, and a launch that does nothing about 2.
//
// Every workgroup scans all requests (pages asked for, tokens granted, pages
// given back) into LDS and fills its share of the tokens from there: a search
// of the offsets finds a token's request. A new page's first token is new by
// definition, so the thread of that token writes the table. Nothing read here
// is written in the same launch: the pages taken lie in the ring before its
// count and the ones given back behind it, and the tables' old columns stay.
// Only lens and state may be the caller's outputs too (in place): then those
// are written by a launch of their own, or, with one workgroup, behind a
// barrier.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void plan_kernel(PlanArgs a) {
    extern __shared__ uint32_t plan_lds[];
    __shared__ uint32_t part[THREADS / WAVE][2];
    __shared__ uint32_t n_gone, taken, limit;
    const PagedPlan &p = a.p;
    const int R = p.requests, tid = threadIdx.x;
    uint32_t *off = plan_lds;          // R + 1: tokens before a request
    uint32_t *first = off + R + 1;     // R: pages taken (given back) before it
    uint32_t *held = first + R;        // R: tokens held
    uint32_t *gone = held + R;         // ended requests this workgroup handles
    const uint32_t pages = p.pages;
    const uint32_t head = (uint32_t)p.state[0] % pages;
    const uint32_t count = min((uint32_t)max(p.state[1], 0), pages);

    if (tid == 0) {
        n_gone = taken = 0;
        limit = 0xffffffffu;
        off[0] = 0;
    }
    uint32_t asked = 0, back = 0, tokens_asked = 0;
    for (int base = 0; base < R; base += THREADS) {
        const int r = base + tid;
        Ask x = {0, 0, 0u, 0u, false};
        if (r < R) x = ask_of(a, r);
        uint32_t pages_upto = x.need, back_upto = x.ended ? x.have : 0, t0, t1;
        block_scan<THREADS>(pages_upto, back_upto, t0, t1, part);
        pages_upto = add_sat(asked, pages_upto);
        back_upto = add_sat(back, back_upto);
        asked = add_sat(asked, t0);
        back = add_sat(back, t1);
        const bool has_pages = x.want > 0 && (x.need == 0 || pages_upto <= count);
        uint32_t tok = has_pages ? x.want : 0, none = 0;
        block_scan<THREADS>(tok, none, t0, t1, part);
        tok = add_sat(tokens_asked, tok);
        tokens_asked = add_sat(tokens_asked, t0);
        // The granted requests are those before the first that would pass
        // max_tokens (sums only grow), so their pages are a first part of the
        // pages asked for, and every later offset is the first one's start.
        const bool ok = has_pages && tok <= (uint32_t)p.max_tokens;
        if (has_pages && !ok) atomicMin(&limit, tok - x.want);
        if (ok && x.need > 0) atomicMax(&taken, pages_upto);
        if (r < R) {
            off[r + 1] = tok;
            held[r] = x.held;
            first[r] = x.ended ? back_upto - x.have : pages_upto - x.need;
            if (x.ended && x.have > 0 && r % gridDim.x == blockIdx.x)
                gone[atomicAdd(&n_gone, 1u)] = r;
        }
    }
    __syncthreads();
    for (int r = tid; r < R; r += THREADS) off[r + 1] = min(off[r + 1], limit);
    __syncthreads();

    if (a.fill) {
        const uint32_t T = p.max_tokens, tokens = off[R];
        for (uint32_t t = blockIdx.x * THREADS + tid; t < T; t += gridDim.x * THREADS) {
            int slot = -1, pos = 0;
            if (t < tokens) {
                int r = 0, hi = R - 1;  // t's request: the first that ends behind it
                while (r < hi) {
                    const int mid = (r + hi) >> 1;
                    if (off[mid + 1] <= t)
                        r = mid + 1;
                    else
                        hi = mid;
                }
                const int have = a.page.quot(held[r] + p.page_size - 1);
                pos = (int)(held[r] + (t - off[r]));
                const int j = a.page.quot(pos), in = pos - j * p.page_size;
                int *row = p.block_table + (size_t)r * p.max_pages;
                int page;
                if (j >= have) {
                    page = p.free_pages[(head + first[r] + (uint32_t)(j - have)) % pages];
                    if (in == 0) row[j] = page;
                } else {
                    page = row[j];
                }
                if ((uint32_t)page < pages) slot = page * p.page_size + in;
            }
            p.slots[t] = slot;
            p.positions[t] = pos;
        }
        for (uint32_t i = tid >> 6; i < n_gone; i += THREADS / WAVE) {
            const int r = gone[i], have = a.page.quot(held[r] + p.page_size - 1);
            const int *row = p.block_table + (size_t)r * p.max_pages;
            const uint32_t to = head + count + first[r];
            for (int j = tid & 63; j < have; j += WAVE)
                p.free_pages[(to + (uint32_t)j) % pages] = row[j];
        }
    }
    if (a.finish && blockIdx.x == 0) {
        __syncthreads();  // lens and state may be the results too
        for (int r = tid; r < R; r += THREADS) {
            const uint32_t grant = off[r + 1] - off[r];
            const bool ended = p.new_tokens[r] < 0;
            p.lens_out[r] = ended ? 0 : (int)(held[r] + grant);
            p.rows[r] = grant ? (int)off[r + 1] - 1 : -1;
            p.offsets[r + 1] = off[r + 1];
        }
        if (tid == 0) {
            p.offsets[0] = 0;
            p.state_out[0] = (head + taken) % pages;
            p.state_out[1] = min(count - taken + back, pages);
        }
    }
}

// ---------------------------------------------------------------- append
struct AppendArgs {
    const char *k, *v;
    char *kc, *vc;
    const int *slots;
    long long row_stride, page_stride, token_stride, head_stride;  // elements
    long long items;   // 8-element pieces of one half
    long long first;   // the launch's first workgroup of the call's
    int capacity;      // slots of the cache
    FastDiv page, heads;
    int page_size, kv_heads;
};

template <typename T>
using Vec8 __attribute__((ext_vector_type(8))) = T;

// One thread moves eight elements of a key and of the value beside it. The
// rows come at any multiple of 4 bytes, the cache in multiples of 16. Bound by
// HBM: 65536 tokens of 8 heads of 128 in bf16 (537 MB read and written) take 104
// us, 5.2 TB/s, the rate of a copy; 32 tokens 2.0 us, a launch. (Non-temporal
// stores gain 2% there and lose a third where fp32 goes to fp32.)
template <typename TS, typename TC, int HS>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    constexpr int PIECES = HS / 8;
    const long long i = (a.first + blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.items) return;
    const int piece = (int)(i % PIECES), row = (int)(i / PIECES);  // row: (token, head)
    const int token = a.heads.quot(row), head = row - token * a.kv_heads;
    const int slot = a.slots[token];
    if ((unsigned)slot >= (unsigned)a.capacity) return;
    const int page = a.page.quot(slot), in = slot - page * a.page_size;
    const long long from = token * a.row_stride + head * HS + piece * 8;
    const long long to = page * a.page_stride + in * a.token_stride + head * a.head_stride +
                         piece * 8;
    typedef Vec8<TS> VS __attribute__((aligned(4)));
    const Vec8<TS> k = *(const VS *)(a.k + from * (long long)sizeof(TS));
    const Vec8<TS> v = *(const VS *)(a.v + from * (long long)sizeof(TS));
    *(Vec8<TC> *)(a.kc + to * (long long)sizeof(TC)) = __builtin_convertvector(k, Vec8<TC>);
    *(Vec8<TC> *)(a.vc + to * (long long)sizeof(TC)) = __builtin_convertvector(v, Vec8<TC>);
}

template <typename TS, typename TC>
void launch_append(int hs, AppendArgs &a, hipStream_t stream) {
    const auto kernel = hs == 32   ? append_kernel<TS, TC, 32>
                        : hs == 64 ? append_kernel<TS, TC, 64>
                                   : append_kernel<TS, TC, 128>;
    in_launches((a.items + 255) / 256, 256, [&](long long first, unsigned n) {
        a.first = first;
        launch(kernel, dim3(n), dim3(256), 0, stream, a);
    });
}

}  // namespace
}  // namespace bmb

extern "C" {

int paged_plan(const PagedPlan *p, hipStream_t stream) {
    using namespace bmb;
    const char *me = "paged_plan";
    if (p == nullptr) return refuse(me, "no plan");
    if (p->requests < 1 || p->requests > PLAN_MAX_REQUESTS)
        return refuse(me, "requests is not 1 to 8192");
    if (p->max_pages < 1 || p->pages < 1 || p->page_size < 1 || p->max_tokens < 0)
        return refuse(me, "a size is below its least");
    if ((long long)p->pages * p->page_size > INT_MAX ||
        ((long long)p->max_pages + 1) * p->page_size > INT_MAX)
        return refuse(me, "2^31 or more tokens in the cache or in a request");
    if (!p->new_tokens || !p->lens || !p->lens_out || !p->state || !p->state_out ||
        !p->free_pages || !p->block_table || !p->rows || !p->offsets ||
        (p->max_tokens > 0 && (!p->slots || !p->positions)))
        return refuse(me, "a null pointer");
    const size_t R = p->requests;
    const auto apart = [](const int *a, const int *b, size_t n) {
        return a + n <= b || b + n <= a;
    };
    if ((p->lens != p->lens_out && !apart(p->lens, p->lens_out, R)) ||
        (p->state != p->state_out && !apart(p->state, p->state_out, 2)))
        return refuse(me, "lens or state overlaps its result in part");
    const bool in_place = p->lens == p->lens_out || p->state == p->state_out;
    PlanArgs a = {*p, FastDiv::of(p->page_size), true, true};
    // As many waves as one round of the scan needs: 64 decoding requests take
    // 4.8 us with 64 threads (their tables and ended requests then go one by
    // one), 4.1 with 256, 4.7 with 1024; 8 requests 3.2, 3.5 and 4.2; 1024
    // requests 18.6, 9.0 and 6.6.
    const int threads = R <= 32 ? 64 : R <= 256 ? 256 : 1024;
    const auto kernel = threads == 64    ? plan_kernel<64>
                        : threads == 256 ? plan_kernel<256>
                                         : plan_kernel<1024>;
    const size_t lds = (4 * R + 1) * sizeof(uint32_t);
    allow_smem(kernel, lds + 256);
    int blocks = (int)(((long long)p->max_tokens + threads - 1) / threads);
    blocks = blocks < 1 ? 1 : blocks > PLAN_MAX_BLOCKS ? PLAN_MAX_BLOCKS : blocks;
    a.finish = blocks == 1 || !in_place;
    launch(kernel, dim3(blocks), dim3(threads), lds, stream, a);
    if (!a.finish) {
        a.fill = false;
        a.finish = true;
        launch(kernel, dim3(1), dim3(threads), lds, stream, a);
    }
    return 0;
}

int paged_append(const PagedCache *c, const void *k, const void *v, int type, long long row_stride,
                 const int *slots, int tokens, hipStream_t stream) {
    using namespace bmb;
    const char *me = "paged_append";
    if (const char *why = cache_fault(c, true)) return refuse(me, why);
    const int size = element_size(type);
    if (size == 0) return refuse(me, "unknown element type");
    if (type != BMB_F32 && type != c->type)
        return refuse(me, "16-bit rows go into a cache of their own type only");
    if (tokens < 0) return refuse(me, "negative number of tokens");
    if (tokens == 0) return 0;
    if (k == nullptr || v == nullptr || slots == nullptr) return refuse(me, "a null pointer");
    if ((long long)tokens * c->kv_heads > INT_MAX)
        return refuse(me, "too many tokens for one call");
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)(row_stride * size)) % 4 != 0)
        return refuse(me, "rows are no multiples of 4 bytes");
    AppendArgs a = {(const char *)k, (const char *)v, (char *)c->k, (char *)c->v, slots, row_stride,
                    c->page_stride, c->token_stride, c->head_stride,
                    (long long)tokens * c->kv_heads * (c->head_size / 8), 0,
                    c->pages * c->page_size, FastDiv::of(c->page_size), FastDiv::of(c->kv_heads),
                    c->page_size, c->kv_heads};
    const int hs = c->head_size;
    if (type == BMB_F32 && c->type == BMB_F32)
        launch_append<float, float>(hs, a, stream);
    else if (type == BMB_F32 && c->type == BMB_F16)
        launch_append<float, _Float16>(hs, a, stream);
    else if (type == BMB_F32)
        launch_append<float, __bf16>(hs, a, stream);
    else
        launch_append<uint16_t, uint16_t>(hs, a, stream);
    return 0;
}

}  // extern "C"
