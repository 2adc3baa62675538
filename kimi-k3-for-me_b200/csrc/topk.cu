// topk.cu -- the K largest logits of each row of a verify sweep's logits, the targets a
// draft head is distilled from (k3gpu_lm_head_distill).
//
// Order: values descending, equal values by ascending id; NaN is never taken (argmax's
// rule), -inf is taken after every finite value. Each value becomes a 32-bit key that
// orders as the floats do (the sign folded in, -0 as +0, NaN as 0, below -inf's key); key and
// complemented id make a 64-bit rank, and no two ranks are equal.
//
// The row is read once, a block per segment of it, 8192 values a round, 32 a thread in
// registers. The first round's bar: each warp's ceil(K / 8)-th largest of its lanes' maxima,
// the least of the warps' (so at least K values reach it; of random values about 1% pass).
// One comparison for four values; a quad with one above the bar is put aside whole in
// shared memory, and after the round the block takes its values apart into the candidate
// list, which is trimmed to about the K best by bisection on the ranks, raising the bar. Past
// the first round the bar is strict: ids ascend, so an equal value comes behind K better ones.
// A round with more such quads than fit (long runs of ascending values) is taken again in
// small steps with a trim after each; the result is exact whatever the order.
// A second kernel joins the segments' lists the same way and writes the K in order.
// Bound by the read, about two instructions a value.
#include <math.h>

#include "common.cuh"
#include "pdl.cuh"

namespace k3 {
namespace topk {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int QUADS = 8;                     // float4s a thread holds of a round
constexpr int ROUND = THREADS * QUADS * 4;
constexpr int MAXK = 128;
constexpr int MORE = 64;                     // candidates past K before a trim is due
constexpr int SLACK = 16;                    // a trim leaves at most K + SLACK
constexpr int STEP = 1024;                   // values a step of a round taken again
constexpr int ASIDE = 512;                   // quads a round puts aside
constexpr int LIST = 2304;
constexpr int HOLD = LIST / THREADS;         // candidates a thread holds in a trim
constexpr int MAX_SEG = 32;
constexpr int MERGE = MAX_SEG * MAXK / THREADS;   // candidates a thread holds in the merge
static_assert(MAXK + MORE + 4 * ASIDE <= LIST && MAXK + MORE + STEP <= LIST, "what joins fits behind what is kept");
static_assert(MAXK + MORE <= THREADS, "one candidate a thread in the last sort");

__device__ __forceinline__ uint32_t key_of(float v)
{
    if (v != v) return 0u;
    const uint32_t u = __float_as_uint(__fadd_rn(v, 0.0f));   // -0 + 0 = +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k)
{
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

__device__ __forceinline__ uint64_t rank_of(uint32_t key, int id) { return (uint64_t)key << 32 | (uint32_t)~id; }

struct Shared {
    uint64_t rank[LIST];
    float4 quad[ASIDE];
    int quad_id[ASIDE];
    int n, n_quads;                 // candidates; quads above the bar (those past ASIDE were dropped)
    uint32_t bar;                   // a value joins when its key is above this
    int part[2][WARPS];
    uint32_t low[WARPS];
};

// block-wide sum of a count, one barrier (the partial array alternates)
__device__ __forceinline__ int block_count(int c, int *part)
{
    c = __reduce_add_sync(0xffffffffu, c);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = c;
    __syncthreads();
    int t = 0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) t += part[w];
    return t;
}

// A first bar from the threads' largest keys: at least K values have a key above it.
__device__ __forceinline__ void first_bar(Shared &s, uint32_t most, int K)
{
    const int need = (K + WARPS - 1) / WARPS;
    uint32_t t = 0;
#pragma unroll
    for (int b = 31; b >= 0; b--) {
        const uint32_t mid = t | (1u << b);
        if (__popc(__ballot_sync(0xffffffffu, most >= mid)) >= need) t = mid;
    }
    if ((threadIdx.x & 31) == 0) s.low[threadIdx.x >> 5] = t;
    __syncthreads();
    uint32_t low = s.low[0];
#pragma unroll
    for (int w = 1; w < WARPS; w++) low = min(low, s.low[w]);
    // just below it; -0 has no key of its own, and as a float it is not below 0
    if (threadIdx.x == 0) s.bar = low == 0x80000000u ? low - 2 : low ? low - 1 : 0u;
    __syncthreads();
}

__device__ __forceinline__ void join(Shared &s, uint32_t key, int id, uint32_t bar)
{
    if (key > bar) s.rank[atomicAdd(&s.n, 1)] = rank_of(key, id);
}

// Trim the list to between K and K + SLACK of its best and raise the bar to them. Called by
// the whole block with n = s.n read by all; leaves the list, n and the bar visible; returns n.
__device__ __forceinline__ int trim(Shared &s, int n, int K)
{
    uint64_t r[HOLD];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < HOLD; i++) {
        const int x = threadIdx.x + i * THREADS;
        r[i] = x < n ? s.rank[x] : 0ull;
        top = max(top, (uint32_t)(r[i] >> 32));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) s.low[threadIdx.x >> 5] = top;
    uint64_t lo = (uint64_t)(s.bar + 1u) << 32;        // n ranks at or above it
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; w++) top = max(top, s.low[w]);
    uint64_t hi = (uint64_t)(top + 1u) << 32;          // none
    int flip = 0;
    while (hi - lo > 1) {
        const uint64_t mid = lo + (hi - lo) / 2;
        int c = 0;
#pragma unroll
        for (int i = 0; i < HOLD; i++) c += r[i] >= mid;
        c = block_count(c, s.part[flip ^= 1]);
        if (c >= K) {
            lo = mid;
            if (c <= K + SLACK) break;
        } else {
            hi = mid;
        }
    }
    __syncthreads();                // every thread holds its candidates: the list is rewritten
    if (threadIdx.x == 0) {
        s.n = 0;
        s.bar = (uint32_t)(lo >> 32);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < HOLD; i++)
        if (r[i] >= lo) s.rank[atomicAdd(&s.n, 1)] = r[i];
    __syncthreads();
    n = s.n;
    __syncthreads();
    return n;
}

// The list's K best in order, by counting each one's place; places past the list are 0.
__device__ __forceinline__ void sort(Shared &s, int n, int K)
{
    if (n > K + MORE) n = trim(s, n, K);
    if (n + threadIdx.x < (unsigned)((n + 3) & ~3)) s.rank[n + threadIdx.x] = 0;
    __syncthreads();
    const uint64_t r = (int)threadIdx.x < n ? s.rank[threadIdx.x] : 0;
    int place = (int)threadIdx.x < n ? 0 : THREADS;
#pragma unroll 2
    for (int j = 0; j < n; j += 4) {
        const ulonglong2 a = *reinterpret_cast<const ulonglong2 *>(&s.rank[j]);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2 *>(&s.rank[j + 2]);
        place += (a.x > r) + (a.y > r) + (b.x > r) + (b.y > r);
    }
    __syncthreads();
    if ((int)threadIdx.x >= n && (int)threadIdx.x < K) s.rank[threadIdx.x] = 0;
    if (place < K) s.rank[place] = r;
    __syncthreads();
}

__device__ __forceinline__ void write_out(const Shared &s, int *idx, float *val, int K)
{
    for (int k = threadIdx.x; k < K; k += THREADS) {
        const uint64_t r = s.rank[k];
        idx[k] = r ? (int)~(uint32_t)r : -1;
        val[k] = r ? value_of((uint32_t)(r >> 32)) : -INFINITY;
    }
}

// grid (segments, rows): the segment's K best, in order, to cand [rows][segments][K] (0 past its
// candidates), or, of a row that is one segment, to idx and val
__global__ void __launch_bounds__(THREADS, 4) segment_kernel(uint64_t *cand, int *idx, float *val, const float *logits,
                                                             int vocab, int seg_len, int K)
{
    __shared__ __align__(16) Shared s;
    const float *row = logits + (size_t)blockIdx.y * vocab;
    const int begin = blockIdx.x * seg_len, end = min(vocab, begin + seg_len);
    if (threadIdx.x == 0) { s.n = s.n_quads = 0; s.bar = 0; }
    __syncthreads();
    pdl_wait();
    pdl_release();
    // quads lie on 16-byte boundaries; the first may start before the segment
    const int skew = (int)((reinterpret_cast<uintptr_t>(row + begin) & 15u) / 4);
    int n = 0;
    float4 v[QUADS];
    auto fetch = [&](int base) {
#pragma unroll
        for (int i = 0; i < QUADS; i++) {
            const int x = base + (i * THREADS + (int)threadIdx.x) * 4;
            if (x >= begin && x + 4 <= end) {
                v[i] = __ldcs(reinterpret_cast<const float4 *>(row + x));
            } else {
                v[i].x = x >= begin && x < end ? row[x] : NAN;
                v[i].y = x + 1 >= begin && x + 1 < end ? row[x + 1] : NAN;
                v[i].z = x + 2 >= begin && x + 2 < end ? row[x + 2] : NAN;
                v[i].w = x + 3 >= begin && x + 3 < end ? row[x + 3] : NAN;
            }
        }
    };
    fetch(begin - skew);
    for (int base = begin - skew; base < end; base += ROUND) {
        // fmaxf passes over NaN
        auto most = [](const float4 &q) { return fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w)); };
        if (base + skew == begin) {
            float m = NAN;
#pragma unroll
            for (int i = 0; i < QUADS; i++) m = fmaxf(m, most(v[i]));
            first_bar(s, key_of(m), K);
        }
        const uint32_t bar = s.bar;
        const float bar_f = value_of(bar);            // NaN for an open bar: every quad passes
#pragma unroll
        for (int i = 0; i < QUADS; i++)
            if (!(most(v[i]) <= bar_f)) {
                const int p = atomicAdd(&s.n_quads, 1);
                if (p < ASIDE) {
                    s.quad[p] = v[i];
                    s.quad_id[p] = base + (i * THREADS + (int)threadIdx.x) * 4;
                }
            }
        if (base + ROUND < end) fetch(base + ROUND);   // on its way while the block sorts this one out
        __syncthreads();
        const int aside = s.n_quads;
        if (aside == 0) {                              // (read by all before anyone adds to it:
            __syncthreads();                           //  the loads of the next round come between)
            continue;
        }
        if (aside <= ASIDE) {
            for (int p = threadIdx.x; p < aside; p += THREADS) {
                const float4 q = s.quad[p];
                const int x = s.quad_id[p];
                join(s, key_of(q.x), x, bar);
                join(s, key_of(q.y), x + 1, bar);
                join(s, key_of(q.z), x + 2, bar);
                join(s, key_of(q.w), x + 3, bar);
            }
            __syncthreads();
            n = s.n;
            if (threadIdx.x == 0) s.n_quads = 0;
            __syncthreads();
            if (n > K + MORE) n = trim(s, n, K);
        } else {                                       // again, in steps that fit
            const int stop = min(base + ROUND, end);
            for (int x0 = max(base, begin); x0 < stop; x0 += STEP) {
                const uint32_t now = s.bar;
                for (int x = x0 + (int)threadIdx.x; x < min(x0 + STEP, stop); x += THREADS)
                    join(s, key_of(row[x]), x, now);
                __syncthreads();
                n = s.n;
                if (threadIdx.x == 0) s.n_quads = 0;
                __syncthreads();
                if (n > K + MORE) n = trim(s, n, K);
            }
        }
    }
    sort(s, n, K);
    if (gridDim.x == 1) {
        write_out(s, idx + (size_t)blockIdx.y * K, val + (size_t)blockIdx.y * K, K);
        return;
    }
    cand += ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * K;
    for (int k = threadIdx.x; k < K; k += THREADS) cand[k] = s.rank[k];
}

// grid (rows): the K best of the segments' lists, in order
__global__ void __launch_bounds__(THREADS) merge_kernel(int *idx, float *val, const uint64_t *cand, int nseg, int K)
{
    __shared__ __align__(16) Shared s;
    const int total = nseg * K;
    cand += (size_t)blockIdx.x * total;
    if (threadIdx.x == 0) s.n = 0;
    pdl_wait();
    pdl_release();
    uint64_t r[MERGE];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < MERGE; i++) {
        const int x = threadIdx.x + i * THREADS;
        r[i] = x < total ? cand[x] : 0ull;
        most = max(most, (uint32_t)(r[i] >> 32));
    }
    first_bar(s, most, K);
    // a step of four candidates a thread at a time (MERGE steps fit the list only trimmed)
    int n = 0;
    for (int i0 = 0; i0 < MERGE && i0 * THREADS < total; i0 += 4) {
        const uint32_t bar = s.bar;
#pragma unroll
        for (int i = 0; i < MERGE; i++)
            if (i / 4 == i0 / 4 && (uint32_t)(r[i] >> 32) > bar) s.rank[atomicAdd(&s.n, 1)] = r[i];
        __syncthreads();
        n = s.n;
        __syncthreads();
        if (n > K + MORE) n = trim(s, n, K);
    }
    sort(s, n, K);
    write_out(s, idx + (size_t)blockIdx.x * K, val + (size_t)blockIdx.x * K, K);
}

static int segments(int rows, int vocab)
{
    // at most four blocks an SM, one wave, no more segments than the row has rounds: 576 rows in
    // one segment each take 63 us (in two, before the loads ran ahead, 76 against 69)
    const int want = 4 * PLAN_SMS / rows, most = ceil_div(vocab, ROUND);
    return std::max(1, std::min(std::min(want, most), MAX_SEG));
}

static size_t a256(size_t b) { return (b + 255) & ~(size_t)255; }

}  // namespace topk
}  // namespace k3

extern "C" size_t k3gpu_topk_logits_workspace(int rows, int vocab, int K)
{
    using namespace k3::topk;
    if (rows <= 0 || vocab <= 0 || K <= 0 || K > MAXK) return 0;
    return a256((size_t)rows * segments(rows, vocab) * K * 8);
}

extern "C" int k3gpu_topk_logits(int *idx, float *val, const float *logits, int rows, int vocab, int K,
                                 void *workspace, size_t ws_bytes, void *stream)
{
    using namespace k3::topk;
    if (!idx || !val || !logits || !workspace || rows <= 0 || vocab <= 0 || K <= 0 || K > MAXK) return K3GPU_EINVAL;
    if (rows > 65535 || vocab > 1 << 30 || !k3::aligned(logits, 4) || !k3::aligned(idx, 4) || !k3::aligned(val, 4) ||
        !k3::aligned(workspace, 16))
        return K3GPU_EINVAL;
    if (ws_bytes < k3gpu_topk_logits_workspace(rows, vocab, K)) return K3GPU_ECAPACITY;
    const int nseg = segments(rows, vocab);
    const int seg_len = k3::ceil_div(k3::ceil_div(vocab, nseg), 4) * 4;
    uint64_t *cand = static_cast<uint64_t *>(workspace);
    cudaStream_t s = k3::as_stream(stream);
    const int st = k3::launch_pdl(segment_kernel, dim3(nseg, rows), THREADS, 0, s, 1, cand, idx, val, logits, vocab,
                                  seg_len, K);
    if (st || nseg == 1) return st;
    return k3::launch_pdl(merge_kernel, dim3(rows), THREADS, 0, s, 1, idx, val, cand, nseg, K);
}
