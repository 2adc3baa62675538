// head.cu -- the losses a draft head is fitted with, over the lm_head product without its
// logits: softmax cross entropy and distillation from a teacher's top logits, forward and
// backward (k3gpu_lm_head_xent*, k3gpu_lm_head_distill*).
//
//   z[t][v] = sum_i X[t][i] W[v][i]     X [T][in], W [vocab][in] bf16, sums fp32
//   p[t][v] = e^(z/temp - lse[t]),      lse[t] = ln sum_v e^(z/temp)
//   loss[t] = sum_k q_k (ln q_k - z[t][id_k]/temp + lse[t])       (cross entropy: one target
//                                        of mass 1, temp 1: lse - z[label])
//   dz[t][v] = g[t]/temp (p[t][v] - sum_{k: id_k = v} q_k)
//   dX = dz W,  dW = dz^T X
//
// Rows without a target (a negative label; no teacher entry) are left out before the first
// product: a scan numbers the rows that count, and where some do not, their hidden states
// are gathered into a packed copy -- so such a row costs nothing and nothing of it (a NaN
// of its padding, say) reaches a sum. When every row counts, X is read in place.
//
// Forward: one pass over the vocabulary in 128 x 256 tiles; the epilogue keeps each row's
// running maximum and sum of 2^(z c - max) over its tile half (c = log2(e)/temp) and picks
// out the targets' z; a second kernel joins the halves' statistics per row in double.
// Backward: the vocabulary in pieces. Per piece the tile products run again, the epilogue
// turns z into dz from the saved lse and writes it as bf16 to the workspace [T][piece];
// then one launch forms dX += dz W_piece (fp32 between pieces, bf16 at the end) and
// dW_piece = dz^T X. dz is rounded to bf16 once, relative error 2^-9 an element, the size
// of the outputs' own rounding and independent between elements; all sums are fp32.
//
// One persistent CTA per SM walks tiles (10 warps):
//   warp 0     TMA, a ring of 64-K stages: A 128 rows (16 KB), B 256 rows (32 KB)
//   warp 1     one thread issues the MMAs (128 x 256 x 16) into one of two TMEM
//              accumulators of 256 columns
//   warps 2-9  epilogue of the finished accumulator while the next tile runs: warp w reads
//              the TMEM lane quarter w % 4, columns 128 ((w - 2) / 4) ..
// Every wait is bounded (a wait that gives up has waited seconds, longer than any copy in
// flight takes); TMEM is freed on every exit path. No TMA multicast.
#include <cuda_bf16.h>
#include <math.h>

#include <mutex>

#include "common.cuh"
#include "tc.cuh"

namespace k3 {
namespace head {

using namespace tc;

constexpr int THREADS = 10 * 32;
constexpr int BM = 128, BN = 256, KB = 64;
constexpr int NS = 4;
constexpr int A_BYTES = BM * KB * 2, B_BYTES = BN * KB * 2, STAGE = A_BYTES + B_BYTES;
constexpr int SMEM = NS * STAGE + 256;
constexpr int MAXK = 128;
constexpr int ROW_PAD = 256;               // packed rows are padded to this
constexpr float LOG2E = 1.4426950408889634f;

enum Mode { LOSS, DZ, GRADS };

struct Args {
    int T, in, vocab;
    const int *n_live;          // rows that count
    const int *row_of;          // [T] packed row -> row
    int Tpad;
    // targets, by row: entry e of row t is ids[t * K + e] (ascending), mass[t * K + e]
    const int *ids;
    const float *mass;          // nullptr: cross entropy (K = 1, mass 1)
    const int *count;           // entries of a row; nullptr: 1
    int K;
    float c;                    // log2(e) / temp
    // LOSS
    float2 *part;               // [2 * vocabulary tiles][Tpad] (max, sum), base 2
    float *zt;                  // [T][K] z of the targets
    // DZ and GRADS: this piece of the vocabulary
    int v0, vc;                 // first id, ids
    const float *lse, *g;       // by row; g may be nullptr (1)
    float inv_temp;
    __nv_bfloat16 *dz;          // [Tpad][ldz]
    int ldz;
    // GRADS
    int want_dx, want_dw, first, last;
    float *acc;                 // [Tpad][in] dX between pieces
    __nv_bfloat16 *dX, *dW;
    int lddx, vec_dx;
    int x_direct_ok;            // X itself can be read by TMA when every row counts
    int group;                  // row tiles walked together
};

struct Maps {
    CUtensorMap x_k, xp_k;      // X and packed X, K-major boxes (64 x BM)
    CUtensorMap w_k;            // W, K-major boxes (64 x BN)
    CUtensorMap x_mn, xp_mn, w_mn;   // 64 x 64 boxes of rows as K
    CUtensorMap dz_k, dz_mn;    // the piece's dz, 64 x BM and 64 x 64 boxes
};

// A tile of the launch: which product, its first row and column, its K steps.
struct Tile {
    int kind;                   // 0: z (LOSS, DZ); 1: dX; 2: dW
    int m0, n0, steps;
};

__device__ __forceinline__ void place(int i, int mt, int nt, int group, int &m, int &n)
{
    // groups of row tiles; inside a group the rows run fastest, so a wave shares both the
    // group's rows and a few column tiles through L2
    const int per = group * nt, gr = i / per, r = i - gr * per;
    const int size = min(group, mt - gr * group);
    n = r / size;
    m = gr * group + (r - n * size);
}

template <int MODE>
struct Walk {
    int n, mt, nt, mt2, nt2, first2, total, steps_k, steps_v, steps_n;
    __device__ __forceinline__ Walk(const Args &a, int n_live)
    {
        n = n_live;
        mt = (n + BM - 1) / BM;
        if (MODE != GRADS) {
            nt = (a.vc + BN - 1) / BN;
            steps_k = (a.in + KB - 1) / KB;
            first2 = total = mt * nt;
            mt2 = nt2 = steps_v = steps_n = 0;
        } else {
            nt = nt2 = (a.in + BN - 1) / BN;
            mt2 = (a.vc + BM - 1) / BM;
            steps_k = 0;
            steps_v = (a.vc + KB - 1) / KB;
            steps_n = (n + KB - 1) / KB;
            first2 = a.want_dx ? mt * nt : 0;
            total = first2 + (a.want_dw ? mt2 * nt2 : 0);
        }
    }
    __device__ __forceinline__ Tile at(int i, const Args &a) const
    {
        Tile t;
        int m, c;
        if (MODE != GRADS) {
            t.kind = 0;
            place(i, mt, nt, a.group, m, c);
            t.steps = steps_k;
        } else if (i < first2) {
            t.kind = 1;
            place(i, mt, nt, a.group, m, c);
            t.steps = steps_v;
        } else {
            t.kind = 2;
            place(i - first2, mt2, nt2, a.group, m, c);
            t.steps = steps_n;
        }
        t.m0 = m * BM;
        t.n0 = c * BN;
        return t;
    }
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
}
__device__ __forceinline__ float pick(const uint32_t (&v)[32], int j)
{
    float z = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; i++)
        if (i == j) z = __uint_as_float(v[i]);
    return z;
}
// the first of row t's entries at or past id v
__device__ __forceinline__ int first_entry(const Args &a, int t, int cnt, int v)
{
    const int *ids = a.ids + (size_t)t * a.K;
    int lo = 0, hi = cnt;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(ids + mid) < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <int MODE>
__global__ void __launch_bounds__(THREADS, 1) head_kernel(const __grid_constant__ Maps maps, const Args a)
{
    extern __shared__ __align__(1024) unsigned char smem[];
    if ((s_addr(smem) & 1023u) != 0u) {   // never expected: refuse rather than mis-swizzle
        if (threadIdx.x == 0) flag(DEV_BAD_INDEX);
        return;
    }
    uint64_t *b_full = reinterpret_cast<uint64_t *>(smem + NS * STAGE), *b_empty = b_full + NS;
    uint64_t *b_done = b_empty + NS, *b_free = b_done + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(b_free + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; s++) {
            bar_init(s_addr(&b_full[s]), 1);
            bar_init(s_addr(&b_empty[s]), 1);
        }
        for (int d = 0; d < 2; d++) {
            bar_init(s_addr(&b_done[d]), 1);
            bar_init(s_addr(&b_free[d]), 8);       // the epilogue warps
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(s_addr(tmem_slot))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    const int n_live = *a.n_live;
    const Walk<MODE> walk(a, n_live);
    const bool direct = a.x_direct_ok && n_live == a.T;
    bool failed = false;

    if (warp == 0) {
        if (lane == 0) {
            const CUtensorMap *xk = direct ? &maps.x_k : &maps.xp_k, *xmn = direct ? &maps.x_mn : &maps.xp_mn;
            int item = 0;
            for (int i = blockIdx.x; i < walk.total && !failed; i += gridDim.x) {
                const Tile t = walk.at(i, a);
                for (int ks = 0; ks < t.steps; ks++, item++) {
                    const int st = item % NS;
                    if (!bar_wait(s_addr(&b_empty[st]), (uint32_t)((item / NS) & 1) ^ 1u)) { failed = true; break; }
                    const uint32_t sa = s_addr(smem + st * STAGE), sb = sa + A_BYTES, full = s_addr(&b_full[st]);
                    bar_expect(full, STAGE);
                    const int k = ks * KB;
                    if (MODE != GRADS) {
                        tma2d(sa, xk, k, t.m0, full);
                        tma2d(sb, &maps.w_k, k, a.v0 + t.n0, full);
                    } else if (t.kind == 1) {
                        tma2d(sa, &maps.dz_k, k, t.m0, full);
#pragma unroll
                        for (int b = 0; b < BN / 64; b++)
                            tma2d(sb + b * 8192, &maps.w_mn, t.n0 + b * 64, a.v0 + k, full);
                    } else {
#pragma unroll
                        for (int b = 0; b < BM / 64; b++)
                            tma2d(sa + b * 8192, &maps.dz_mn, t.m0 + b * 64, k, full);
#pragma unroll
                        for (int b = 0; b < BN / 64; b++) tma2d(sb + b * 8192, xmn, t.n0 + b * 64, k, full);
                    }
                }
            }
            if (failed) flag(DEV_TIMEOUT);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int item = 0, use = 0;
            for (int i = blockIdx.x; i < walk.total && !failed; i += gridDim.x, use++) {
                const Tile t = walk.at(i, a);
                const int d = use & 1;
                if (!bar_wait(s_addr(&b_free[d]), (uint32_t)((use >> 1) & 1) ^ 1u)) { failed = true; break; }
                fence_after();
                const uint32_t dt = tmem + (uint32_t)(d * BN);
                // A and B: K-major for z; dX takes W as rows of K, dW both operands so
                const uint32_t idesc = bf16_idesc(BN, t.kind >= 1) | (t.kind == 2 ? (1u << 15) : 0u);
                const uint32_t da = t.kind == 2 ? 2048u >> 4 : 32u >> 4, db = t.kind >= 1 ? 2048u >> 4 : 32u >> 4;
                for (int ks = 0; ks < t.steps; ks++, item++) {
                    const int st = item % NS;
                    if (!bar_wait(s_addr(&b_full[st]), (uint32_t)((item / NS) & 1))) { failed = true; break; }
                    fence_after();
                    const uint32_t sa = s_addr(smem + st * STAGE), sb = sa + A_BYTES;
                    const uint64_t ad = t.kind == 2 ? sw128_mn_desc(sa, 8192) : sw128_desc(sa);
                    const uint64_t bd = t.kind >= 1 ? sw128_mn_desc(sb, 8192) : sw128_desc(sb);
#pragma unroll
                    for (int u = 0; u < KB / 16; u++)
                        mma_ss(dt, ad + u * da, bd + u * db, idesc, (uint32_t)(ks > 0 || u > 0));
                    mma_commit(s_addr(&b_empty[st]));
                }
                if (failed) break;
                if (t.steps > 0) mma_commit(s_addr(&b_done[d]));
                else bar_arrive(s_addr(&b_done[d]));
            }
            if (failed) flag(DEV_TIMEOUT);
        }
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2;
        const int r = q * 32 + lane;
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        int use = 0;
        for (int i = blockIdx.x; i < walk.total && !failed; i += gridDim.x, use++) {
            const Tile t = walk.at(i, a);
            const int d = use & 1;
            const int row = t.m0 + r;              // packed row (z, dX) or id of the piece (dW)
            const int col0 = t.n0 + half * (BN / 2);
            const uint32_t src = tmem + lanes + (uint32_t)(d * BN + half * (BN / 2));
            if constexpr (MODE != GRADS) {
                // what the row needs is fetched while the tile's products still run
                const bool live = row < n_live;
                const int tr = live ? a.row_of[row] : 0;
                const int cnt = live ? (a.count ? a.count[tr] : 1) : 0;
                const int *ids = a.ids + (size_t)tr * a.K;
                int e = cnt > 0 ? first_entry(a, tr, cnt, a.v0 + col0) : 0;
                int next = e < cnt ? ids[e] - a.v0 : 0x7fffffff;
                float l2 = 0.0f, gt = 0.0f;
                if (MODE == DZ && live) {
                    l2 = a.lse[tr] * LOG2E;
                    gt = (a.g ? a.g[tr] : 1.0f) * a.inv_temp;
                }
                if (!bar_wait(s_addr(&b_done[d]), (uint32_t)((use >> 1) & 1))) { failed = true; break; }
                fence_after();
                float mx = -INFINITY, sum = 0.0f;
                for (int c0 = 0; c0 < BN / 2; c0 += 32) {
                    uint32_t v[32];
                    __syncwarp();                  // the targets' branches below part the lanes
                    tmem_ld32(src + (uint32_t)c0, v);
                    tmem_wait_ld();
                    const int col = col0 + c0;
                    if constexpr (MODE == LOSS) {
                        while (next < col + 32) {
                            a.zt[(size_t)tr * a.K + e] = pick(v, next - col);
                            e++;
                            next = e < cnt ? ids[e] - a.v0 : 0x7fffffff;
                        }
                        const int left = a.vc - col;
                        float cm = -INFINITY;
#pragma unroll
                        for (int j = 0; j < 32; j++) {
                            const float z = j < left ? __uint_as_float(v[j]) * a.c : -INFINITY;
                            v[j] = __float_as_uint(z);
                            cm = fmaxf(cm, z);
                        }
                        const float mn = fmaxf(mx, cm), ref = mn == -INFINITY ? 0.0f : mn;
                        float cs = 0.0f;
#pragma unroll
                        for (int j = 0; j < 32; j++) cs += ex2(__uint_as_float(v[j]) - ref);
                        sum = sum * ex2(mx - ref) + cs;
                        mx = mn;
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            v[j] = __float_as_uint(live ? ex2(__uint_as_float(v[j]) * a.c - l2) : 0.0f);
                        while (next < col + 32) {
                            const float q_e = a.mass ? a.mass[(size_t)tr * a.K + e] : 1.0f;
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (j == next - col) v[j] = __float_as_uint(__uint_as_float(v[j]) - q_e);
                            e++;
                            next = e < cnt ? ids[e] - a.v0 : 0x7fffffff;
                        }
                        uint32_t o[16];
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            o[j] = live ? pack_bf16(__uint_as_float(v[2 * j]) * gt, __uint_as_float(v[2 * j + 1]) * gt)
                                        : 0u;
                        if (col < a.ldz) {          // ldz is a multiple of 64
                            uint4 *dst = reinterpret_cast<uint4 *>(a.dz + (size_t)row * a.ldz + col);
#pragma unroll
                            for (int j = 0; j < 4; j++) dst[j] = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                        }
                    }
                }
                if (MODE == LOSS && live) a.part[(size_t)(col0 / (BN / 2)) * a.Tpad + row] = make_float2(mx, sum);
            } else {
                if (!bar_wait(s_addr(&b_done[d]), (uint32_t)((use >> 1) & 1))) { failed = true; break; }
                fence_after();
                const bool dx = t.kind == 1;
                const bool live = dx ? row < n_live : row < a.vc;
                float *acc = a.acc + (size_t)row * a.in;
                __nv_bfloat16 *out = nullptr;
                if (live) out = dx ? a.dX + (size_t)a.row_of[row] * a.lddx : a.dW + (size_t)(a.v0 + row) * a.in;
                const bool vec = dx ? a.vec_dx : 1;
                for (int c0 = 0; c0 < BN / 2; c0 += 32) {
                    const int col = col0 + c0;
                    uint32_t v[32];
                    __syncwarp();
                    if (t.steps > 0) {
                        tmem_ld32(src + (uint32_t)c0, v);
                        tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j++) v[j] = 0u;
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {      // `in` is a multiple of 8
                        if (!live || col + j >= a.in) continue;
                        float f[8];
#pragma unroll
                        for (int u = 0; u < 8; u++) f[u] = __uint_as_float(v[j + u]);
                        if (dx && !a.first) {
                            const float4 p0 = *reinterpret_cast<const float4 *>(acc + col + j);
                            const float4 p1 = *reinterpret_cast<const float4 *>(acc + col + j + 4);
                            f[0] += p0.x; f[1] += p0.y; f[2] += p0.z; f[3] += p0.w;
                            f[4] += p1.x; f[5] += p1.y; f[6] += p1.z; f[7] += p1.w;
                        }
                        if (dx && !a.last) {
                            *reinterpret_cast<float4 *>(acc + col + j) = make_float4(f[0], f[1], f[2], f[3]);
                            *reinterpret_cast<float4 *>(acc + col + j + 4) = make_float4(f[4], f[5], f[6], f[7]);
                        } else if (vec) {
                            *reinterpret_cast<uint4 *>(out + col + j) =
                                make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]),
                                           pack_bf16(f[6], f[7]));
                        } else {
#pragma unroll
                            for (int u = 0; u < 8; u++) out[col + j + u] = __float2bfloat16_rn(f[u]);
                        }
                    }
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(s_addr(&b_free[d]));
        }
        if (failed && lane == 0) flag(DEV_TIMEOUT);
    }
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// One block per row: the row's teacher entries as masses over ids in ascending order.
// An entry counts when its id lies in the vocabulary and its logit is not -inf;
// mass = softmax(top / temp) over those. entropy = sum mass ln mass. The maximum carries a
// NaN (fmaxf would drop it): such a row's masses, loss and gradient are NaN.
__global__ void __launch_bounds__(MAXK) teacher_kernel(int *__restrict__ s_ids, float *__restrict__ s_mass,
                                                       int *__restrict__ count, float *__restrict__ entropy,
                                                       const int *__restrict__ ids, const float *__restrict__ top,
                                                       int K, int vocab, float inv_temp)
{
    __shared__ int sid[MAXK];
    __shared__ float st[MAXK];
    __shared__ double se[MAXK];
    const size_t base = (size_t)blockIdx.x * K;
    const int k = threadIdx.x;
    int id = -1;
    float t = -INFINITY;
    if (k < K) {
        id = ids[base + k];
        t = top[base + k];
        if (id >= vocab) flag(DEV_BAD_INDEX);
    }
    const bool ok = id >= 0 && id < vocab && t != -INFINITY;
    sid[k] = ok ? id : -1;
    st[k] = ok ? t : -INFINITY;
    __syncthreads();
    float mx = -INFINITY;
    int nan = 0;
    for (int j = 0; j < K; j++) {
        nan |= st[j] != st[j];
        mx = fmaxf(mx, st[j]);
    }
    if (nan) mx = NAN;
    const double l = ok ? ((double)st[k] - (double)mx) * (double)inv_temp : 0.0;
    const double e = ok ? exp(l) : 0.0;
    se[k] = e;
    __syncthreads();
    double sum = 0.0;
    int place = 0, n = 0;
    for (int j = 0; j < K; j++) {
        sum += se[j];
        n += sid[j] >= 0;
        place += sid[j] >= 0 && (sid[j] < id || (sid[j] == id && j < k));
    }
    const double m = e / sum;
    if (ok) {
        s_ids[base + place] = id;
        s_mass[base + place] = (float)m;
    }
    __syncthreads();
    se[k] = ok ? (e == 0.0 ? 0.0 : m * (l - log(sum))) : 0.0;
    __syncthreads();
    if (k == 0) {
        double h = 0.0;
        for (int j = 0; j < K; j++) h += se[j];
        count[blockIdx.x] = n;
        entropy[blockIdx.x] = (float)h;
    }
}

// One block numbers the rows that count, in order: place[t] (-1: none), row_of[place] = t.
__global__ void __launch_bounds__(1024) plan_kernel(int *__restrict__ place, int *__restrict__ row_of,
                                                    int *__restrict__ n_live, const int *__restrict__ label,
                                                    const int *__restrict__ count, int T, int vocab)
{
    __shared__ int warp_n[32];
    __shared__ int base;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) base = 0;
    __syncthreads();
    for (int t0 = 0; t0 < T; t0 += 1024) {
        const int t = t0 + threadIdx.x;
        bool live = false;
        if (t < T) {
            if (label) {
                const int l = label[t];
                if (l >= vocab) flag(DEV_BAD_INDEX);
                live = l >= 0 && l < vocab;
            } else {
                live = count[t] > 0;
            }
        }
        const unsigned m = __ballot_sync(0xffffffffu, live);
        if (lane == 0) warp_n[warp] = __popc(m);
        __syncthreads();
        int before = base;
        for (int w = 0; w < warp; w++) before += warp_n[w];
        const int p = before + __popc(m & ((1u << lane) - 1));
        if (t < T) place[t] = live ? p : -1;
        if (live) row_of[p] = t;
        __syncthreads();
        if (threadIdx.x == 1023) base = before + __popc(m);
        __syncthreads();
    }
    if (threadIdx.x == 0) *n_live = base;
}

// Block t < T: row t's hidden state to its packed place, or, for a row that does not count,
// zeros to its outputs. Blocks T ..: the zero rows behind the last packed one. Nothing is
// copied when every row counts and X can be read in place.
__global__ void __launch_bounds__(256) gather_kernel(__nv_bfloat16 *__restrict__ Xp, float *__restrict__ loss,
                                                     float *__restrict__ lse, __nv_bfloat16 *__restrict__ dX, int lddx,
                                                     const uint16_t *__restrict__ X, int ldx,
                                                     const int *__restrict__ place, const int *__restrict__ n_live,
                                                     int T, int in, int Tpad, int direct_ok)
{
    const int n = *n_live;
    const bool copy = !(direct_ok && n == T);
    uint16_t *xp = reinterpret_cast<uint16_t *>(Xp);
    if ((int)blockIdx.x >= T) {
        const int p = n + (int)blockIdx.x - T;
        if (copy && p < Tpad)
            for (int i = threadIdx.x; i < in; i += 256) xp[(size_t)p * in + i] = 0;
        return;
    }
    const int t = blockIdx.x, p = place[t];
    if (p >= 0) {
        if (!copy) return;
        const uint16_t *x = X + (size_t)t * ldx;
        if (direct_ok) {                           // rows 16-byte aligned
            for (int i = threadIdx.x; i < in / 8; i += 256)
                reinterpret_cast<uint4 *>(xp + (size_t)p * in)[i] = reinterpret_cast<const uint4 *>(x)[i];
        } else {
            for (int i = threadIdx.x; i < in; i += 256) xp[(size_t)p * in + i] = x[i];
        }
        return;
    }
    if (loss && threadIdx.x == 0) {
        loss[t] = 0.0f;
        lse[t] = 0.0f;
    }
    if (dX)
        for (int i = threadIdx.x; i < in; i += 256) dX[(size_t)t * lddx + i] = __float2bfloat16_rn(0.0f);
}

// 32 packed rows a block, 32 threads a row: the tile halves' statistics joined in double.
__global__ void __launch_bounds__(1024) join_kernel(float *__restrict__ loss, float *__restrict__ lse,
                                                    const float2 *__restrict__ part, int halves, int Tpad,
                                                    const int *__restrict__ row_of, const int *__restrict__ n_live,
                                                    const float *__restrict__ zt, const float *__restrict__ mass,
                                                    const int *__restrict__ count,
                                                    const float *__restrict__ entropy, int K, float inv_temp)
{
    __shared__ float sm[32][33];
    __shared__ float ss[32][33];
    const int r = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int row = blockIdx.x * 32 + r, n = *n_live;
    if ((int)blockIdx.x * 32 >= n) return;
    float m = -INFINITY, s = 0.0f;
    if (row < n)
        for (int h = w; h < halves; h += 32) {
            const float2 p = part[(size_t)h * Tpad + row];
            const float mn = fmaxf(m, p.x), ref = mn == -INFINITY ? 0.0f : mn;
            s = s * exp2f(m - ref) + p.y * exp2f(p.x - ref);
            m = mn;
        }
    sm[w][r] = m;
    ss[w][r] = s;
    __syncthreads();
    // warp w finishes row w
    const int mine = blockIdx.x * 32 + w;
    if (mine >= n) return;
    const float lm = sm[r][w], ls = ss[r][w];
    float M = lm;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float ref = M == -INFINITY ? 0.0f : M;
    double S = (double)ls * exp2((double)lm - (double)ref);
    const int t = row_of[mine];
    const int cnt = count ? count[t] : 1;
    double zq = 0.0;
    for (int e = r; e < cnt; e += 32) {
        const double q = mass ? (double)mass[(size_t)t * K + e] : 1.0;
        if (q != 0.0) zq += q * (double)zt[(size_t)t * K + e];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        S += __shfl_xor_sync(0xffffffffu, S, o);
        zq += __shfl_xor_sync(0xffffffffu, zq, o);
    }
    if (r == 0) {
        const double l = ((double)ref + log2(S)) * 0.69314718055994530942;
        lse[t] = (float)l;
        loss[t] = (float)(l - zq * (double)inv_temp + (entropy ? (double)entropy[t] : 0.0));
    }
}

// ---- host ----------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn()
{
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *q = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &r) == cudaSuccess &&
            r == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(q);
    });
    return fn;
}

// bf16 [rows][ld] of which cols columns exist; reads outside give zeros
static int map2d(CUtensorMap *m, const void *base, long long cols, long long ld, long long rows, int box_rows)
{
    EncodeTiledFn fn = encode_fn();
    if (!fn) return K3GPU_ECUDA;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(ld * 2)};
    cuuint32_t box[2] = {(cuuint32_t)KB, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1u, 1u};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        g_last_cuda_error = (int)r;
        return K3GPU_ECUDA;
    }
    return K3GPU_OK;
}

constexpr long long MAX_T = 1 << 20, MAX_VOCAB = 1 << 24, MAX_IN = 1 << 16;

static size_t a256(size_t b) { return (b + 255) & ~(size_t)255; }

struct Plan {
    int Tpad, tiles, piece, ldz;       // vocabulary tiles; ids per piece of the backward
};

static Plan plan(int T, int vocab)
{
    Plan p;
    p.Tpad = ceil_div(T, ROW_PAD) * ROW_PAD;
    p.tiles = ceil_div(vocab, BN);
    // a piece's dz takes about 64 MB, at least eight tiles
    const long long tiles = std::max<long long>(8, (64LL << 20) / ((long long)p.Tpad * 2 * BN));
    p.piece = (int)std::min<long long>(tiles, p.tiles) * BN;
    p.ldz = p.piece;
    return p;
}

struct Ws {
    int *n_live, *place, *row_of, *ids, *count;
    float *mass, *entropy, *zt, *acc;
    float2 *part;
    __nv_bfloat16 *xp, *dz;
};

// K = 0: cross entropy
static size_t layout(Ws *w, char *base, const Plan &p, int T, int in, int K, bool grad)
{
    size_t o = 0;
    auto take = [&](size_t bytes) {
        char *r = base ? base + o : nullptr;
        o += a256(bytes);
        return r;
    };
    Ws x{};
    x.n_live = (int *)take(4);
    x.place = (int *)take((size_t)T * 4);
    x.row_of = (int *)take((size_t)T * 4);
    x.xp = (__nv_bfloat16 *)take((size_t)p.Tpad * in * 2);
    if (K) {
        x.ids = (int *)take((size_t)T * K * 4);
        x.mass = (float *)take((size_t)T * K * 4);
        x.count = (int *)take((size_t)T * 4);
        x.entropy = (float *)take((size_t)T * 4);
    }
    if (!grad) {
        x.part = (float2 *)take((size_t)p.tiles * 2 * p.Tpad * 8);
        x.zt = (float *)take((size_t)T * (K ? K : 1) * 4);
    } else {
        x.dz = (__nv_bfloat16 *)take((size_t)p.Tpad * p.ldz * 2);
        if (p.piece < p.tiles * BN) x.acc = (float *)take((size_t)p.Tpad * in * 4);
    }
    if (w) *w = x;
    return o;
}

static bool sizes_ok(int T, int in, int vocab)
{
    return T > 0 && T <= MAX_T && vocab > 0 && vocab <= MAX_VOCAB && in > 0 && in <= MAX_IN && in % 8 == 0;
}

static int prepare_device(int *sms)
{
    int dev = 0;
    int st = cuda_status(cudaGetDevice(&dev));
    if (st) return st;
    if ((st = cuda_status(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev)))) return st;
    static std::atomic<uint64_t> ready{0};          // devices whose kernels have their shared memory
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (ready.load() & bit)) return K3GPU_OK;
    for (const void *f : {(const void *)head_kernel<LOSS>, (const void *)head_kernel<DZ>,
                          (const void *)head_kernel<GRADS>})
        if ((st = cuda_status(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM)))) return st;
    if (dev < 64) ready.fetch_or(bit);
    return K3GPU_OK;
}

struct Call {
    const uint16_t *X, *W;
    int ldx, in, vocab, T;
    const int *label;                  // cross entropy
    const int *ids;                    // distillation
    const float *top;
    int K;
    float temp;
    cudaStream_t s;
};

// The targets, the rows that count and their hidden states; fills the common arguments.
static int set_up(Args *a, Maps *maps, const Call &c, const Plan &p, const Ws &w, float *loss, float *lse,
                  uint16_t *dX, int lddx)
{
    int st;
    if (c.K) {
        teacher_kernel<<<c.T, MAXK, 0, c.s>>>(w.ids, w.mass, w.count, w.entropy, c.ids, c.top, c.K, c.vocab,
                                              1.0f / c.temp);
        if ((st = launch_status())) return st;
    }
    plan_kernel<<<1, 1024, 0, c.s>>>(w.place, w.row_of, w.n_live, c.K ? nullptr : c.label, w.count, c.T, c.vocab);
    if ((st = launch_status())) return st;
    const int direct_ok = c.ldx % 8 == 0 && aligned(c.X, 16);
    gather_kernel<<<c.T + ROW_PAD, 256, 0, c.s>>>(w.xp, loss, lse, reinterpret_cast<__nv_bfloat16 *>(dX), lddx, c.X,
                                                  c.ldx, w.place, w.n_live, c.T, c.in, p.Tpad, direct_ok);
    if ((st = launch_status())) return st;
    *a = Args{};
    a->T = c.T; a->in = c.in; a->vocab = c.vocab;
    a->n_live = w.n_live; a->row_of = w.row_of; a->Tpad = p.Tpad;
    a->ids = c.K ? w.ids : c.label;
    a->mass = w.mass; a->count = w.count;
    a->K = c.K ? c.K : 1;
    a->inv_temp = c.K ? 1.0f / c.temp : 1.0f;
    a->c = c.K ? (float)(1.4426950408889634 / (double)c.temp) : LOG2E;
    a->x_direct_ok = direct_ok;
    // the group's hidden states take at most about 32 MB
    a->group = std::max(1, std::min(64, (int)((32LL << 20) / ((long long)BM * c.in * 2))));
    const void *x = direct_ok ? (const void *)c.X : (const void *)w.xp;
    const long long ldx = direct_ok ? c.ldx : c.in, xr = direct_ok ? c.T : p.Tpad;
    if ((st = map2d(&maps->x_k, x, c.in, ldx, xr, BM))) return st;
    if ((st = map2d(&maps->x_mn, x, c.in, ldx, xr, 64))) return st;
    if ((st = map2d(&maps->xp_k, w.xp, c.in, c.in, p.Tpad, BM))) return st;
    if ((st = map2d(&maps->xp_mn, w.xp, c.in, c.in, p.Tpad, 64))) return st;
    if ((st = map2d(&maps->w_k, c.W, c.in, c.in, c.vocab, BN))) return st;
    return map2d(&maps->w_mn, c.W, c.in, c.in, c.vocab, 64);
}

static int forward(float *loss, float *lse, const Call &c, void *ws)
{
    int sms = 0, st = prepare_device(&sms);
    if (st) return st;
    const Plan p = plan(c.T, c.vocab);
    Ws w;
    layout(&w, static_cast<char *>(ws), p, c.T, c.in, c.K, false);
    Args a;
    Maps maps{};
    if ((st = set_up(&a, &maps, c, p, w, loss, lse, nullptr, 0))) return st;
    a.part = w.part; a.zt = w.zt;
    a.v0 = 0; a.vc = c.vocab;
    head_kernel<LOSS><<<sms, THREADS, SMEM, c.s>>>(maps, a);
    if ((st = launch_status())) return st;
    join_kernel<<<p.Tpad / 32, 1024, 0, c.s>>>(loss, lse, w.part, 2 * p.tiles, p.Tpad, w.row_of, w.n_live, w.zt, w.mass,
                                               w.count, w.entropy, a.K, a.inv_temp);
    return launch_status();
}

static int backward(uint16_t *dX, int lddx, uint16_t *dW, const float *g, const float *lse, const Call &c, void *ws)
{
    int sms = 0, st = prepare_device(&sms);
    if (st) return st;
    const Plan p = plan(c.T, c.vocab);
    Ws w;
    layout(&w, static_cast<char *>(ws), p, c.T, c.in, c.K, true);
    Args a;
    Maps maps{};
    if ((st = set_up(&a, &maps, c, p, w, nullptr, nullptr, dX, lddx))) return st;
    a.lse = lse; a.g = g;
    a.dz = w.dz; a.ldz = p.ldz; a.acc = w.acc;
    a.dX = reinterpret_cast<__nv_bfloat16 *>(dX);
    a.dW = reinterpret_cast<__nv_bfloat16 *>(dW);
    a.want_dx = dX != nullptr; a.want_dw = dW != nullptr;
    a.lddx = lddx; a.vec_dx = lddx % 8 == 0 && aligned(dX, 16);
    for (int v0 = 0; v0 < c.vocab; v0 += p.piece) {
        a.v0 = v0;
        a.vc = std::min(p.piece, c.vocab - v0);
        a.first = v0 == 0; a.last = v0 + p.piece >= c.vocab;
        if ((st = map2d(&maps.dz_k, w.dz, a.vc, p.ldz, p.Tpad, BM))) return st;
        if ((st = map2d(&maps.dz_mn, w.dz, a.vc, p.ldz, p.Tpad, 64))) return st;
        head_kernel<DZ><<<sms, THREADS, SMEM, c.s>>>(maps, a);
        if ((st = launch_status())) return st;
        head_kernel<GRADS><<<sms, THREADS, SMEM, c.s>>>(maps, a);
        if ((st = launch_status())) return st;
    }
    return K3GPU_OK;
}

static size_t workspace_bytes(int T, int in, int vocab, int K)
{
    const Plan p = plan(T, vocab);
    return std::max(layout(nullptr, nullptr, p, T, in, K, false), layout(nullptr, nullptr, p, T, in, K, true));
}

static bool head_ok(const uint16_t *X, int ldx, const uint16_t *W, int in, int vocab, int T, const void *ws)
{
    return X && W && ws && sizes_ok(T, in, vocab) && ldx >= in && aligned(W, 16) && aligned(X, 2) && aligned(ws, 256);
}

static bool grads_ok(const uint16_t *dX, int lddx, const uint16_t *dW, int in)
{
    return (dX || dW) && (!dX || (lddx >= in && aligned(dX, 2))) && (!dW || aligned(dW, 16));
}

static bool teacher_ok(const int *ids, const float *top, int K, float temp)
{
    return ids && top && K > 0 && K <= MAXK && temp > 0.0f && isfinite(temp) && isfinite(1.0f / temp);
}

}  // namespace head
}  // namespace k3

extern "C" size_t k3gpu_lm_head_xent_workspace(int T, int in, int vocab)
{
    return k3::head::sizes_ok(T, in, vocab) ? k3::head::workspace_bytes(T, in, vocab, 0) : 0;
}

extern "C" int k3gpu_lm_head_xent(float *loss, float *lse, const uint16_t *X, int ldx, const uint16_t *W,
                                  const int *label, int in, int vocab, int T, void *workspace, size_t ws_bytes,
                                  void *stream)
{
    using namespace k3::head;
    if (!loss || !lse || !label || !head_ok(X, ldx, W, in, vocab, T, workspace)) return K3GPU_EINVAL;
    if (ws_bytes < workspace_bytes(T, in, vocab, 0)) return K3GPU_ECAPACITY;
    const Call c{X, W, ldx, in, vocab, T, label, nullptr, nullptr, 0, 1.0f, k3::as_stream(stream)};
    return forward(loss, lse, c, workspace);
}

extern "C" int k3gpu_lm_head_xent_grad(uint16_t *dX, int lddx, uint16_t *dW, const float *g, const float *lse,
                                       const uint16_t *X, int ldx, const uint16_t *W, const int *label, int in,
                                       int vocab, int T, void *workspace, size_t ws_bytes, void *stream)
{
    using namespace k3::head;
    if (!lse || !label || !head_ok(X, ldx, W, in, vocab, T, workspace) || !grads_ok(dX, lddx, dW, in))
        return K3GPU_EINVAL;
    if (ws_bytes < workspace_bytes(T, in, vocab, 0)) return K3GPU_ECAPACITY;
    const Call c{X, W, ldx, in, vocab, T, label, nullptr, nullptr, 0, 1.0f, k3::as_stream(stream)};
    return backward(dX, lddx, dW, g, lse, c, workspace);
}

extern "C" size_t k3gpu_lm_head_distill_workspace(int T, int in, int vocab, int K)
{
    using namespace k3::head;
    return sizes_ok(T, in, vocab) && K > 0 && K <= MAXK ? workspace_bytes(T, in, vocab, K) : 0;
}

extern "C" int k3gpu_lm_head_distill(float *loss, float *lse, const uint16_t *X, int ldx, const uint16_t *W,
                                     const int *ids, const float *top, int K, float temp, int in, int vocab, int T,
                                     void *workspace, size_t ws_bytes, void *stream)
{
    using namespace k3::head;
    if (!loss || !lse || !teacher_ok(ids, top, K, temp) || !head_ok(X, ldx, W, in, vocab, T, workspace))
        return K3GPU_EINVAL;
    if (ws_bytes < workspace_bytes(T, in, vocab, K)) return K3GPU_ECAPACITY;
    const Call c{X, W, ldx, in, vocab, T, nullptr, ids, top, K, temp, k3::as_stream(stream)};
    return forward(loss, lse, c, workspace);
}

extern "C" int k3gpu_lm_head_distill_grad(uint16_t *dX, int lddx, uint16_t *dW, const float *g, const float *lse,
                                          const uint16_t *X, int ldx, const uint16_t *W, const int *ids,
                                          const float *top, int K, float temp, int in, int vocab, int T,
                                          void *workspace, size_t ws_bytes, void *stream)
{
    using namespace k3::head;
    if (!lse || !teacher_ok(ids, top, K, temp) || !head_ok(X, ldx, W, in, vocab, T, workspace) ||
        !grads_ok(dX, lddx, dW, in))
        return K3GPU_EINVAL;
    if (ws_bytes < workspace_bytes(T, in, vocab, K)) return K3GPU_ECAPACITY;
    const Call c{X, W, ldx, in, vocab, T, nullptr, ids, top, K, temp, k3::as_stream(stream)};
    return backward(dX, lddx, dW, g, lse, c, workspace);
}
