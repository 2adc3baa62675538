// topk.cu -- the K largest logits of each row of a verify sweep's logits, the targets a
// draft head is distilled from (k3gpu_lm_head_distill).
//
// Order: values descending, equal values by ascending id; NaN is never taken (argmax's
// rule), -inf is taken after every finite value. Each value becomes a 32-bit key that
// orders as the floats do (the sign folded in, -0 as +0, NaN as 0, below -inf's key).
//
// The row is read once. A block walks its segment of the row in tiles; a value joins the
// block's candidate list when its key is above the K-th largest kept so far (strictly:
// tiles ascend in id, so an equal value comes after K better ones), and a tile that makes
// the list outgrow KEEP is followed by a selection that cuts it to K and raises the bar.
// Random rows take a handful of selections a segment (the expected number of values above
// a running K-th largest grows with the log of the length); an ascending row takes one per
// tile and is still exact. A second kernel selects among the segments' lists and writes
// the K in order, each value's place counted directly (K <= 128).
// Bound by the read: K << vocab, about four instructions a value.
#include <math.h>

#include "common.cuh"

namespace k3 {
namespace topk {

constexpr int THREADS = 512;
constexpr int PER = 8;                       // values a thread holds of a tile
constexpr int TILE = THREADS * PER;
constexpr int MAXK = 128;
constexpr int KEEP = 1024;                   // candidates kept before a selection is due
constexpr int CAP = KEEP + TILE;             // a tile can join whole
constexpr int MAX_SEG = 32;                  // segments a row: their lists fit one selection
constexpr int HOLD = (CAP + THREADS - 1) / THREADS;   // candidates a thread holds in a selection
static_assert(MAX_SEG * MAXK <= CAP, "the merge holds every segment's list");

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

struct Shared {
    uint32_t key[CAP];
    int id[CAP];
    int n;                          // candidates in the list
    uint32_t bar;                   // a value joins when its key is above this
    int part[2][THREADS / 32];
};

// block-wide sum of a count, one barrier (the partial array alternates)
__device__ __forceinline__ int block_count(int c, int *part)
{
    c = __reduce_add_sync(0xffffffffu, c);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = c;
    __syncthreads();
    int t = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) t += part[w];
    return t;
}

// Cut the list to its K best, in any order. Called by the whole block with the list and n
// visible; leaves them, and the bar, visible. The K-th largest key is the largest t with at
// least K keys >= t, found bit by bit; where its equals overflow the K places, the largest
// id that still fits is found the same way.
__device__ void select(Shared &s, int K)
{
    const int n = s.n;
    if (n <= K) {
        __syncthreads();
        return;
    }
    uint32_t key[HOLD];
    int id[HOLD];
#pragma unroll
    for (int i = 0; i < HOLD; i++) {
        const int x = threadIdx.x + i * THREADS;
        key[i] = x < n ? s.key[x] : 0u;
        id[i] = x < n ? s.id[x] : 0x7fffffff;
    }
    uint32_t t = 0;
    int flip = 0, at_least = n;
    for (int b = 31; b >= 0; b--) {
        const uint32_t mid = t | (1u << b);
        int c = 0;
#pragma unroll
        for (int i = 0; i < HOLD; i++) c += key[i] >= mid;
        c = block_count(c, s.part[flip ^= 1]);
        if (c >= K) {
            t = mid;
            at_least = c;
            if (c == K) break;
        }
    }
    int last = 0x7fffffff;          // keys equal to t stay up to this id
    if (at_least > K) {
        int above = 0;
#pragma unroll
        for (int i = 0; i < HOLD; i++) above += key[i] > t;
        above = block_count(above, s.part[flip ^= 1]);
        // the smallest id with (K - above) equals at or below it
        int lo = 0;
        for (int b = 30; b >= 0; b--) {
            const int mid = lo | (1 << b);
            int c = 0;
#pragma unroll
            for (int i = 0; i < HOLD; i++) c += key[i] == t && id[i] < mid;
            c = block_count(c, s.part[flip ^= 1]);
            if (c < K - above) lo = mid;
        }
        last = lo;
    }
    __syncthreads();                // every thread holds its candidates: the list is rewritten
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < HOLD; i++) {
        const int x = threadIdx.x + i * THREADS;
        if (x < n && (key[i] > t || (key[i] == t && id[i] <= last))) {
            const int p = atomicAdd(&s.n, 1);
            s.key[p] = key[i];
            s.id[p] = id[i];
        }
    }
    if (threadIdx.x == 0) s.bar = t;
    __syncthreads();
}

// grid (segments, rows): the segment's K best to cand_key/cand_id [rows][segments][K], the
// places past its candidates with key 0
__global__ void __launch_bounds__(THREADS) segment_kernel(uint32_t *__restrict__ cand_key, int *__restrict__ cand_id,
                                                          const float *__restrict__ logits, int vocab, int seg_len,
                                                          int K)
{
    extern __shared__ __align__(16) unsigned char topk_dyn[];
    Shared &s = *reinterpret_cast<Shared *>(topk_dyn);
    const float *row = logits + (size_t)blockIdx.y * vocab;
    const int begin = blockIdx.x * seg_len, end = min(vocab, begin + seg_len);
    if (threadIdx.x == 0) { s.n = 0; s.bar = 0; }
    float v[PER];
    auto fetch = [&](int base) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int x = base + i * THREADS + (int)threadIdx.x;
            v[i] = x < end ? __ldg(row + x) : NAN;
        }
    };
    fetch(begin);
    __syncthreads();
    for (int base = begin; base < end; base += TILE) {
        uint32_t key[PER];
#pragma unroll
        for (int i = 0; i < PER; i++) key[i] = key_of(v[i]);
        if (base + TILE < end) fetch(base + TILE);
        const uint32_t bar = s.bar;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (key[i] > bar) {
                const int p = atomicAdd(&s.n, 1);
                s.key[p] = key[i];
                s.id[p] = base + i * THREADS + (int)threadIdx.x;
            }
        __syncthreads();
        if (s.n > KEEP || (base == begin && s.n > K)) select(s, K);
        __syncthreads();
    }
    select(s, K);
    const size_t out = ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * K;
    for (int k = threadIdx.x; k < K; k += THREADS) {
        cand_key[out + k] = k < s.n ? s.key[k] : 0u;
        cand_id[out + k] = k < s.n ? s.id[k] : 0x7fffffff;
    }
}

// grid (rows): the K best of the segments' lists, in order
__global__ void __launch_bounds__(THREADS) merge_kernel(int *__restrict__ idx, float *__restrict__ val,
                                                        const uint32_t *__restrict__ cand_key,
                                                        const int *__restrict__ cand_id, int nseg, int K)
{
    extern __shared__ __align__(16) unsigned char topk_dyn[];
    Shared &s = *reinterpret_cast<Shared *>(topk_dyn);
    const size_t in = (size_t)blockIdx.x * nseg * K, out = (size_t)blockIdx.x * K;
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    for (int x = threadIdx.x; x < nseg * K; x += THREADS) {
        const uint32_t k = cand_key[in + x];
        if (k) {
            const int p = atomicAdd(&s.n, 1);
            s.key[p] = k;
            s.id[p] = cand_id[in + x];
        }
    }
    __syncthreads();
    select(s, K);
    const int n = s.n;
    for (int k = threadIdx.x; k < K; k += THREADS) {
        if (k < n) {
            int place = 0;
            for (int j = 0; j < n; j++)
                place += s.key[j] > s.key[k] || (s.key[j] == s.key[k] && s.id[j] < s.id[k]);
            idx[out + place] = s.id[k];
            val[out + place] = value_of(s.key[k]);
        } else {
            idx[out + k] = -1;
            val[out + k] = -INFINITY;
        }
    }
}

static int segments(int rows, int vocab)
{
    // about four blocks an SM of 148, no segment shorter than two tiles
    const int want = ceil_div(4 * 148, rows), most = ceil_div(vocab, 2 * TILE);
    return std::max(1, std::min(std::min(want, most), MAX_SEG));
}

static size_t a256(size_t b) { return (b + 255) & ~(size_t)255; }

}  // namespace topk
}  // namespace k3

extern "C" size_t k3gpu_topk_logits_workspace(int rows, int vocab, int K)
{
    using namespace k3::topk;
    if (rows <= 0 || vocab <= 0 || K <= 0 || K > MAXK) return 0;
    return 2 * a256((size_t)rows * segments(rows, vocab) * K * 4);
}

extern "C" int k3gpu_topk_logits(int *idx, float *val, const float *logits, int rows, int vocab, int K,
                                 void *workspace, size_t ws_bytes, void *stream)
{
    using namespace k3::topk;
    if (!idx || !val || !logits || !workspace || rows <= 0 || vocab <= 0 || K <= 0 || K > MAXK) return K3GPU_EINVAL;
    if (rows > 65535 || !k3::aligned(workspace, 16)) return K3GPU_EINVAL;
    if (ws_bytes < k3gpu_topk_logits_workspace(rows, vocab, K)) return K3GPU_ECAPACITY;
    const int nseg = segments(rows, vocab);
    const int seg_len = k3::ceil_div(k3::ceil_div(vocab, nseg), 4) * 4;
    uint32_t *ck = static_cast<uint32_t *>(workspace);
    int *ci = reinterpret_cast<int *>(static_cast<char *>(workspace) + a256((size_t)rows * nseg * K * 4));
    cudaStream_t s = k3::as_stream(stream);
    segment_kernel<<<dim3(nseg, rows), THREADS, sizeof(Shared), s>>>(ck, ci, logits, vocab, seg_len, K);
    int st = k3::launch_status();
    if (st) return st;
    merge_kernel<<<rows, THREADS, sizeof(Shared), s>>>(idx, val, ck, ci, nseg, K);
    return k3::launch_status();
}
