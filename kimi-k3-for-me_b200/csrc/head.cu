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
// maximum and sum of 2^(z c - max) over its tile half (c = log2(e)/temp) and picks out the
// targets' z; a second kernel joins the halves' statistics per row.
// Backward: the vocabulary in pieces. Per piece the tile products run again, the epilogue
// turns z into dz from the saved lse and writes it as bf16 to the workspace [T][piece]; the
// next launch forms dX += dz W_piece (fp32 between pieces, bf16 at the end) and
// dW_piece = dz^T X, beside the dz of the piece after it (two buffers), so each launch has
// several kinds of units to fill the SMs with. dz leaves out the factors common to all of
// it (1/temp, the largest weight's mantissa; the outputs get them in fp32) and is rounded to bf16
// once: at most 2^-8 of an element, as much as the outputs' own rounding, independent
// between elements. All sums are fp32.
// Few elements that matter do not average that rounding out (4 rows of 2 entries: dX off by
// 0.0025, by 0.0016 with an exact dz). Up to 32 rows a tile has room for as many again: there the
// rest of each rounding, as bf16, is a second set of rows, against W for dX (whose last sum joins
// the two) and against a copy of X for dW; rows and rests together are one K step of it, the
// products no more tiles than without. Loss and gradient of 4 rows of 1024 over 32,000 ids take 84
// us against 80, of 32 rows of 7168 over 163,840 1.81 ms against 1.77. (Up to 64 rows it would
// be two K steps: 94 against 77 us at 64 rows of 1024, which are off by 0.0019 to 0.0024 without.)
//
// One persistent CTA per SM takes every n-th unit of work (10 warps):
//   warp 0     TMA, a ring of 64-K stages: A 128 rows (16 KB), B 256 rows (32 KB)
//   warp 1     one thread issues the MMAs (128 x 256 x 16) into one of two TMEM
//              accumulators of 256 columns
//   warps 2-9  epilogue of the finished accumulator while the next one fills: warp w reads
//              the TMEM lane quarter w % 4, columns 128 ((w - 2) / 4) ..
// In the backward of larger batches two CTAs of a cluster share a 256 x 256 unit
// (cta_group::2): each loads its 128 rows of A and half of B.
// The tensor core's fp32 sums are cut, not rounded, as they grow, an error with one sign; z
// therefore leaves TMEM every 1024 of K (256 for a weight stream) and is summed in the
// epilogue's registers: over 7168 wide hidden states the loss is 5.6e-7 from its 64-bit value,
// without that 4.4e-6, and it costs 0.3% (the MMAs do not wait, two accumulators alternate;
// every 512: 2.6e-7 and 1.5%). dX and dW end in bf16 and stay in TMEM.
//
// What bounds it: the tensor cores, and the power limit that holds their clock down. One call after
// a pause, 2048 rows of 7168 over 163,840 ids: the loss 3.2 ms (1.48 PFLOP/s, 0.87 of the measured
// burst rate), the gradient 9.8 ms for the three products it runs (1.47), the tensor pipe 87-90%
// busy while the clock falls to 1.34-1.45 GHz; back to back 14.8-15.2 ms together, 1.28 PFLOP/s of
// the four products, where a library product sustains 1.41. A handful of rows is a weight stream:
// 9 rows 372 us of kernel (6.3 TB/s of W), 417-428 us a pass.
// Units dealt out by a counter instead of in turn cost 2-3% (neighbouring SMs then no longer
// read the same W tile together), pairs in the forward 3%.
// Every wait is bounded (a wait that gives up has waited seconds, longer than any copy in
// flight takes); TMEM is freed on every exit path. No TMA multicast.
#include <cuda_bf16.h>
#include <math.h>

#include <mutex>

#include "common.cuh"
#include "pdl.cuh"
#include "tc.cuh"

namespace k3 {
namespace head {

using namespace tc;

constexpr int THREADS = 10 * 32;
constexpr int BM = 128, BN = 256, KB = 64; // rows a CTA, columns a unit
constexpr int NU = 4;                      // units published ahead
constexpr int A_BYTES = BM * KB * 2;
constexpr int RING = 192 * 1024;           // the stages: 4 of 48 KB, or 6 of 32 KB in a pair
constexpr int OUT_BYTES = 32 * 64 * 2;     // a warp's 32 rows x 64 columns on their way out
constexpr int SMEM = RING + 8 * OUT_BYTES + 512;
template <int CG> struct Stage {
    static constexpr int B_COLS = BN / CG, BYTES = A_BYTES + B_COLS * KB * 2, N = RING / BYTES;
};
constexpr int HALF = BN / 2;               // columns an epilogue thread holds
constexpr int GROUP_D = 16 * BM;           // rows of dX and dW walked together: 16 x 9 tiles in flight
constexpr int MAXK = 128;
constexpr int ROW_PAD = 2 * BM;            // packed rows end on a pair's tile
constexpr int PACK_BLOCKS = 512, PACK_ROWS = 2048, PACK_COLS = 1024;
constexpr float LOG2E = 1.4426950408889634f;

enum Mode { LOSS, GRAD, GRAD_RESTS };      // GRAD_RESTS: dz in two parts (Args::rest)
enum Kind { Z, DX, DW };                   // what a unit of work forms

// A vocabulary piece of the backward: ids v0 .. v0 + vc - 1, their dz [dz_rows][piece].
struct Piece {
    int v0, vc;
    __nv_bfloat16 *dz;
};

struct Args {
    int T, in;
    const int *n_live;          // rows that count
    const int4 *rows;           // [T] of a packed row: its row t, its label or count of entries, lse log2(e), weight
    int Tpad;
    int x_in_place;             // X itself can be read by TMA when every row counts
    // targets, by row: entry e of row t is ids[t * K + e] (ascending), mass[t * K + e]
    const int *ids;             // nullptr: cross entropy (K = 1, mass 1, the label in `rows`)
    const float *mass;
    int K;
    float c;                    // log2(e) / temp
    int chunk;                  // 64-K steps of z summed in TMEM before they join the registers
    Piece z;                    // vc = 0: no z units in this launch
    // LOSS
    float2 *part;               // [2 * vocabulary tiles][Tpad] (max, sum), base 2
    float *zt;                  // [T][K] z of the targets
    // GRAD
    const float *g_scale;       // what the weights in `rows` were divided by; nullptr: nothing
    float inv_temp;
    Piece d;                    // vc = 0: no dX and dW units in this launch
    int want_dx, want_dw, first, last;
    int dz_rows;                // rows that dz has a place for: T rounded up to a K step of dW
    int rest;                   // GRAD_RESTS: from this row on dz holds what rounding the rows before left
    int splits, split_steps;    // dX: K splits, 64-K steps of each
    int acc_groups;             // 32-row groups of acc, to the end of T
    float4 *acc;                // dX before its last sum: by split, 32 rows x 128 columns, 4 columns, lane
    __nv_bfloat16 *dX;
    int lddx, vec_dx;
    int z_before_dw;            // the longer units come first
    int group_z;                // rows of z walked together
};

struct Maps {
    CUtensorMap x_k, xp_k;      // X and packed X, K-major boxes (64 x BM)
    CUtensorMap w_k;            // W, K-major boxes (64 x a CTA's columns)
    CUtensorMap x_mn, xp_mn, w_mn;   // 64 x 64 boxes of rows as K
    CUtensorMap dz_k, dz_mn;    // piece d's dz, 64 x BM and 64 x 64 boxes
    CUtensorMap z_out, w_out;   // piece z's dz and dW to write, 64 x 32 boxes
};

// A unit: a 128 CG x 256 tile of one product (or of one K split of it), worked on by a CTA
// (CG = 1) or a pair of them. The producer publishes it to its CTA's warps as four words.
struct Unit {
    int kind, m0, n0, split, step0, steps;
    __device__ __forceinline__ int4 words() const { return make_int4(kind | (split << 4), m0, n0, steps); }
    static __device__ __forceinline__ Unit of(const int4 &w)
    {
        return Unit{w.x < 0 ? -1 : (w.x & 15), w.y, w.z, w.x >> 4, 0, w.w};
    }
};

template <int MODE, int CG>
struct Units {
    static constexpr int TM = BM * CG;
    int n_dx, n_dw, n_z, total;
    int mt, nt_in, nt_z, mt_w, steps_in, steps_v, steps_n;
    __device__ __forceinline__ Units(const Args &a, int n)
    {
        mt = (n + TM - 1) / TM;
        nt_in = (a.in + BN - 1) / BN;
        nt_z = (a.z.vc + BN - 1) / BN;
        mt_w = (a.d.vc + TM - 1) / TM;
        steps_in = (a.in + KB - 1) / KB;
        steps_v = (a.d.vc + KB - 1) / KB;
        steps_n = (n + KB - 1) / KB;
        n_z = mt * nt_z;
        n_dx = MODE != LOSS && a.want_dx && a.d.vc ? mt * nt_in * a.splits : 0;
        n_dw = MODE != LOSS && a.want_dw ? mt_w * nt_in : 0;
        total = n_dx + n_dw + n_z;
    }
    // groups of row tiles; inside a group the rows run fastest, so the units in flight share
    // both the group's rows and a few column tiles through L2
    static __device__ __forceinline__ void place(int i, int m_tiles, int n_tiles, int group, int &m, int &n)
    {
        const int per = group * n_tiles, gr = i / per, r = i - gr * per;
        const int size = min(group, m_tiles - gr * group);
        n = r / size;
        m = gr * group + (r - n * size);
    }
    __device__ __forceinline__ Unit at(int i, const Args &a) const
    {
        Unit u;
        int m = 0, c = 0;
        u.split = 0;
        u.step0 = 0;
        if (MODE != LOSS && i < n_dx) {
            u.kind = DX;
            u.split = i / (mt * nt_in);
            place(i - u.split * (mt * nt_in), mt, nt_in, GROUP_D / TM, m, c);
            u.step0 = u.split * a.split_steps;
            u.steps = max(0, min(a.split_steps, steps_v - u.step0));
        } else {
            i -= n_dx;
            const bool z = MODE == LOSS || (a.z_before_dw ? i < n_z : i >= n_dw);
            if (z) {
                u.kind = Z;
                place(MODE == LOSS || a.z_before_dw ? i : i - n_dw, mt, nt_z, a.group_z / TM, m, c);
                u.steps = steps_in;
            } else {
                u.kind = DW;
                place(a.z_before_dw ? i - n_z : i, mt_w, nt_in, GROUP_D / TM, m, c);
                u.steps = steps_n;
            }
        }
        u.m0 = m * TM;
        u.n0 = c * BN;
        return u;
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
// The pair's forms (CG = 2, a cluster of two CTAs, rank 0 leads): loads signal the leader's
// barrier, the leader's MMAs read both CTAs' shared memory and write both's TMEM, a commit
// arrives at the barrier of the same place in both.
__device__ __forceinline__ uint32_t at_rank0(uint32_t saddr)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(saddr));
    return r;
}
template <int CG>
__device__ __forceinline__ void load2d(uint32_t dst, const CUtensorMap *m, int x, int y, uint32_t bar)
{
    if (CG == 1) {
        tma2d(dst, m, x, y, bar);
    } else {
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
            "{%2, %3}], [%4];" ::"r"(dst),
            "l"(m), "r"(x), "r"(y), "r"(bar)
            : "memory");
    }
}
template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t more)
{
    if (CG == 1) {
        mma_ss(d, ad, bd, idesc, more);
    } else {
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
            "l"(ad), "l"(bd), "r"(idesc), "r"(more)
            : "memory");
    }
}
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar)
{
    if (CG == 1) {
        mma_commit(bar);
    } else {
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                bar),
            "h"((uint16_t)3)
            : "memory");
    }
}
// every thread of the cluster; orders what came before it for what comes after
template <int CG>
__device__ __forceinline__ void sync_all()
{
    if (CG == 1) {
        __syncthreads();
    } else {
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 64 columns of a warp's 32 rows, lane = row, from registers to an output: through shared
// memory in the 128-byte swizzle and one TMA store. Lanes storing 16 bytes each to 32 rows
// took 13,000 clocks a 128 x 256 unit; this takes a tenth. `off`: nothing is written.
__device__ __forceinline__ void out_wait()
{
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
template <typename F>
__device__ __forceinline__ void store64(uint32_t buf, const CUtensorMap *m, int x, int y, bool off, int lane, F &&word8)
{
    if (lane == 0) out_wait();             // the buffer's last store has read it
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint4 o = word8(j);
        const uint32_t at = buf + (uint32_t)(lane * 128 + ((j ^ (lane & 7)) * 16));
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(o.x), "r"(o.y), "r"(o.z), "r"(o.w)
                     : "memory");
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0 && !off) {
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(m), "r"(x),
                     "r"(y), "r"(buf)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
}
// the first of a row's entries at or past id v
__device__ __forceinline__ int first_entry(const int *ids, int cnt, int v)
{
    int lo = 0, hi = cnt;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ids[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// The targets of the thread's row from the unit's column col0 on.
struct RowTargets {
    int e, cnt, next;           // the next entry, entries, the next entry's column in the piece
    __device__ __forceinline__ void start(const Args &a, const int4 &r, bool live, int col0)
    {
        if (!a.ids) {
            e = 0;
            cnt = 1;
            next = live && r.y - a.z.v0 >= col0 ? r.y - a.z.v0 : 0x7fffffff;
            return;
        }
        const int *ids = a.ids + (size_t)r.x * a.K;
        cnt = live ? r.y : 0;
        e = first_entry(ids, cnt, a.z.v0 + col0);
        next = e < cnt ? ids[e] - a.z.v0 : 0x7fffffff;
    }
    __device__ __forceinline__ void step(const Args &a, int t)
    {
        e++;
        next = e < cnt ? a.ids[(size_t)t * a.K + e] - a.z.v0 : 0x7fffffff;
    }
};

__device__ __forceinline__ void loss_epilogue(const Args &a, float (&z)[HALF], RowTargets &tg, int t, int row,
                                              bool live, int col0)
{
#pragma unroll
    for (int c0 = 0; c0 < HALF; c0 += 32)
        while (tg.next < col0 + c0 + 32) {
            const uint32_t at = 1u << (tg.next - col0 - c0);   // a bit, so that z stays in registers
            float v = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; j++)
                if (at & (1u << j)) v = z[c0 + j];
            a.zt[(size_t)t * a.K + tg.e] = v;
            tg.step(a, t);
        }
    const int left = a.z.vc - col0;
    if (left < HALF) {                     // the vocabulary ends here
#pragma unroll
        for (int j = 0; j < HALF; j++) z[j] = j < left ? z[j] : -INFINITY;
    }
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < HALF; j += 2) mx[(j >> 1) & 3] = fmaxf(mx[(j >> 1) & 3], fmaxf(z[j], z[j + 1]));
    const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.c, ref = m == -INFINITY ? 0.0f : m;
    float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < HALF; j++) s[j & 7] += ex2(fmaf(z[j], a.c, -ref));
    if (live)
        a.part[(size_t)(col0 / HALF) * a.Tpad + row] =
            make_float2(m, ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7])));
}

template <bool RESTS>
__device__ __forceinline__ void dz_epilogue(const Args &a, const CUtensorMap *out, uint32_t buf, float (&z)[HALF],
                                            RowTargets &tg, int t, int row0, int lane, bool live, int col0, float l2,
                                            float gt)
{
#pragma unroll
    for (int j = 0; j < HALF; j++) z[j] = ex2(fmaf(z[j], a.c, -l2));
#pragma unroll
    for (int c0 = 0; c0 < HALF; c0 += 32)
        while (tg.next < col0 + c0 + 32) {
            const uint32_t at = 1u << (tg.next - col0 - c0);   // a bit, so that z stays in registers
            const float q = a.mass ? a.mass[(size_t)t * a.K + tg.e] : 1.0f;
#pragma unroll
            for (int j = 0; j < 32; j++)
                if (at & (1u << j)) z[c0 + j] -= q;
            tg.step(a, t);
        }
    // rows of the tile past the live ones are zeros: dW sums over them
    if (!live) {
#pragma unroll
        for (int j = 0; j < HALF; j++) z[j] = 0.0f;
        gt = 0.0f;
    }
    if (row0 >= (RESTS ? a.rest : a.dz_rows)) return;      // (multiples of 32: a warp's rows lie on one side)
#pragma unroll 1
    for (int part = 0;; part++) {
#pragma unroll
        for (int c0 = 0; c0 < HALF; c0 += 64)
            store64(buf, out, col0 + c0, RESTS ? row0 + part * a.rest : row0, false, lane, [&](int j) {
                const float *f = z + c0 + 8 * j;
                return make_uint4(pack_bf16(f[0] * gt, f[1] * gt), pack_bf16(f[2] * gt, f[3] * gt),
                                  pack_bf16(f[4] * gt, f[5] * gt), pack_bf16(f[6] * gt, f[7] * gt));
            });
        if (!RESTS || part == 1) break;
        if constexpr (RESTS) {
#pragma unroll
            for (int j = 0; j < HALF; j++) {
                const float v = z[j] * gt, r = __bfloat162float(__float2bfloat16_rn(v));
                z[j] = fabsf(r) < INFINITY ? v - r : 0.0f; // exact; nothing beside an infinity or a NaN
            }
            gt = 1.0f;
        }
    }
}

// dz was formed without these: exactly common factors add no rounding of their own to it
__device__ __forceinline__ float out_scale(const Args &a) { return (a.g_scale ? *a.g_scale : 1.0f) * a.inv_temp; }
// where a warp's 32 rows x 128 columns of a dX tile lie in acc (float4s; its lanes follow)
__device__ __forceinline__ size_t acc_at(const Args &a, int split, int row0, int col0)
{
    const size_t groups = (size_t)split * a.acc_groups + row0 / 32;
    return (groups * ((a.in + BN - 1) / BN * 2) + col0 / HALF) * (HALF / 4) * 32;
}
__device__ __forceinline__ void put8(__nv_bfloat16 *out, const float4 &f0, const float4 &f1, float k, bool vec)
{
    const uint4 o = make_uint4(pack_bf16(f0.x * k, f0.y * k), pack_bf16(f0.z * k, f0.w * k),
                               pack_bf16(f1.x * k, f1.y * k), pack_bf16(f1.z * k, f1.w * k));
    if (vec) {
        *reinterpret_cast<uint4 *>(out) = o;
    } else {
        uint16_t *u = reinterpret_cast<uint16_t *>(out);
        u[0] = (uint16_t)o.x; u[1] = (uint16_t)(o.x >> 16); u[2] = (uint16_t)o.y; u[3] = (uint16_t)(o.y >> 16);
        u[4] = (uint16_t)o.z; u[5] = (uint16_t)(o.z >> 16); u[6] = (uint16_t)o.w; u[7] = (uint16_t)(o.w >> 16);
    }
}

template <int MODE, int CG>
__global__ void __launch_bounds__(THREADS, 1) head_kernel(const __grid_constant__ Maps maps, const Args a)
{
    using St = Stage<CG>;
    constexpr int NS = St::N;
    extern __shared__ __align__(1024) unsigned char smem[];
    uint64_t *b_full = reinterpret_cast<uint64_t *>(smem + RING + 8 * OUT_BYTES), *b_empty = b_full + NS;
    uint64_t *b_done = b_empty + NS, *b_free = b_done + 2, *b_unit = b_free + 2, *b_took = b_unit + NU;
    int4 *unit_slot = reinterpret_cast<int4 *>(b_took + NU);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(unit_slot + NU);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CG == 1 ? 0 : blockIdx.x & 1;   // in the cluster of two
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; s++) {
            bar_init(s_addr(&b_full[s]), 1);
            bar_init(s_addr(&b_empty[s]), 1);
        }
        for (int d = 0; d < 2; d++) {
            bar_init(s_addr(&b_done[d]), 1);
            bar_init(s_addr(&b_free[d]), 8 * CG);  // the epilogue warps
        }
        for (int u = 0; u < NU; u++) {
            bar_init(s_addr(&b_unit[u]), 1);
            bar_init(s_addr(&b_took[u]), rank == 0 ? 9 : 8);   // the MMA thread and the epilogue warps
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(s_addr(tmem_slot))
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(s_addr(tmem_slot))
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    fence_before();
    sync_all<CG>();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_release();
    const int n_live = *a.n_live, n_rows = MODE == GRAD_RESTS && n_live ? a.rest + n_live : n_live;
    bool failed = false;

    if (warp == 0) {
        if (lane == 0) {
            const bool in_place = a.x_in_place && n_live == a.T;
            const CUtensorMap *xk = in_place ? &maps.x_k : &maps.xp_k, *xmn = in_place ? &maps.x_mn : &maps.xp_mn;
            if (MODE == GRAD_RESTS) xmn = &maps.xp_mn;             // (its rows twice)
            const Units<MODE, CG> units(a, n_rows);
            int item = 0, n_units = 0;
            for (int i = blockIdx.x / CG; !failed; i += gridDim.x / CG) {
                const int slot = n_units % NU;
                if (!bar_wait(s_addr(&b_took[slot]), (uint32_t)((n_units / NU) & 1) ^ 1u)) { failed = true; break; }
                const bool end = i >= units.total;
                Unit t{};
                if (!end) t = units.at(i, a);
                unit_slot[slot] = end ? make_int4(-1, 0, 0, 0) : t.words();
                bar_arrive(s_addr(&b_unit[slot]));
                n_units++;
                if (end) break;
                const int m0 = t.m0 + rank * BM, n0 = t.n0 + rank * St::B_COLS;
                for (int ks = 0; ks < t.steps; ks++, item++) {
                    const int st = item % NS;
                    if (!bar_wait(s_addr(&b_empty[st]), (uint32_t)((item / NS) & 1) ^ 1u)) { failed = true; break; }
                    const uint32_t sa = s_addr(smem + st * St::BYTES), sb = sa + A_BYTES;
                    uint32_t full = s_addr(&b_full[st]);
                    if (rank == 0) bar_expect(full, CG * St::BYTES);
                    if (CG > 1) full = at_rank0(full);
                    const int k = (t.step0 + ks) * KB;
                    if (MODE == LOSS || t.kind == Z) {
                        load2d<CG>(sa, xk, k, m0, full);
                        load2d<CG>(sb, &maps.w_k, k, a.z.v0 + n0, full);
                    } else if (t.kind == DX) {
                        load2d<CG>(sa, &maps.dz_k, k, m0, full);
#pragma unroll
                        for (int b = 0; b < St::B_COLS / 64; b++)
                            load2d<CG>(sb + b * 8192, &maps.w_mn, n0 + b * 64, a.d.v0 + k, full);
                    } else {
#pragma unroll
                        for (int b = 0; b < BM / 64; b++)
                            load2d<CG>(sa + b * 8192, &maps.dz_mn, m0 + b * 64, k, full);
#pragma unroll
                        for (int b = 0; b < St::B_COLS / 64; b++)
                            load2d<CG>(sb + b * 8192, xmn, n0 + b * 64, k, full);
                    }
                }
            }
            if (failed) flag(DEV_TIMEOUT);
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int item = 0, use = 0;
            for (int n_units = 0; !failed; n_units++) {
                const int slot = n_units % NU;
                if (!bar_wait(s_addr(&b_unit[slot]), (uint32_t)((n_units / NU) & 1))) { failed = true; break; }
                const Unit t = Unit::of(unit_slot[slot]);
                bar_arrive(s_addr(&b_took[slot]));
                if (t.kind < 0) break;
                // A and B are K-major for z; dX takes W as rows of K, dW both operands so
                const bool b_mn = MODE != LOSS && t.kind != Z, a_mn = MODE != LOSS && t.kind == DW;
                const uint32_t idesc = (bf16_idesc(BN, b_mn) + ((uint32_t)(CG - 1) << 27)) | (a_mn ? (1u << 15) : 0u);
                const uint32_t da = a_mn ? 2048u >> 4 : 32u >> 4, db = b_mn ? 2048u >> 4 : 32u >> 4;
                const int chunk = b_mn ? t.steps : a.chunk;
                for (int ks = 0; ks < t.steps && !failed; use++) {
                    const int d = use & 1, end = min(t.steps, ks + chunk);
                    if (!bar_wait(s_addr(&b_free[d]), (uint32_t)((use >> 1) & 1) ^ 1u)) { failed = true; break; }
                    fence_after();
                    const uint32_t dt = tmem + (uint32_t)(d * BN);
                    for (uint32_t more = 0; ks < end; ks++, item++) {
                        const int st = item % NS;
                        if (!bar_wait(s_addr(&b_full[st]), (uint32_t)((item / NS) & 1))) { failed = true; break; }
                        fence_after();
                        const uint32_t sa = s_addr(smem + st * St::BYTES), sb = sa + A_BYTES;
                        const uint64_t ad = a_mn ? sw128_mn_desc(sa, 8192) : sw128_desc(sa);
                        const uint64_t bd = b_mn ? sw128_mn_desc(sb, 8192) : sw128_desc(sb);
#pragma unroll
                        for (int u = 0; u < KB / 16; u++) {
                            mma<CG>(dt, ad + u * da, bd + u * db, idesc, more);
                            more = 1;
                        }
                        commit<CG>(s_addr(&b_empty[st]));
                    }
                    if (!failed) commit<CG>(s_addr(&b_done[d]));
                }
            }
            if (failed) flag(DEV_TIMEOUT);
        }
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        const uint32_t buf = s_addr(smem + RING + (warp - 2) * OUT_BYTES);
        int use = 0;
        // the next finished accumulator
        auto finished = [&]() {
            if (!bar_wait(s_addr(&b_done[use & 1]), (uint32_t)((use >> 1) & 1))) return false;
            fence_after();
            return true;
        };
        // the leader's MMAs may write this accumulator again
        auto release = [&]() {
            fence_before();
            __syncwarp();
            if (lane == 0) {
                const uint32_t b = s_addr(&b_free[use & 1]);
                if (CG == 1 || rank == 0) bar_arrive(b);
                else
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(at_rank0(b))
                                 : "memory");
            }
            use++;
        };
        // the next unit, and of its packed row what `rows` says (on its way while this one ends)
        int n_units = 0;
        auto take = [&](int4 &words, int4 &r) {
            const int slot = n_units % NU;
            words.x = -1;
            if (!bar_wait(s_addr(&b_unit[slot]), (uint32_t)((n_units / NU) & 1))) { failed = true; return; }
            n_units++;
            words = unit_slot[slot];
            __syncwarp();
            if (lane == 0) bar_arrive(s_addr(&b_took[slot]));
            const int row = words.y + rank * BM + q * 32 + lane;
            if (words.x >= 0 && row < n_live) r = a.rows[row];   // (of a dW unit it means nothing)
        };
        int4 words, words_next, r = make_int4(0, 0, 0, 0), r_next = r;
        for (take(words, r); words.x >= 0 && !failed; words = words_next, r = r_next) {
            const Unit t = Unit::of(words);
            const int row0 = t.m0 + rank * BM + q * 32, row = row0 + lane;   // packed row (z, dX), id of the piece (dW)
            const int col0 = t.n0 + half * HALF;
            const uint32_t src = tmem + lanes + (uint32_t)(half * HALF);
            if (MODE == LOSS || t.kind == Z) {
                const bool live = row < n_live;
                RowTargets tg;
                tg.start(a, r, live, col0);
                float z[HALF];
                __syncwarp();
                if (!finished()) { failed = true; break; }
#pragma unroll
                for (int c0 = 0; c0 < HALF; c0 += 32)
                    tmem_ld32(src + (uint32_t)((use & 1) * BN + c0), *reinterpret_cast<uint32_t(*)[32]>(z + c0));
                tmem_wait_ld();
                release();
#pragma unroll 1
                for (int ks = a.chunk; ks < t.steps; ks += a.chunk) {
                    if (!finished()) { failed = true; break; }
#pragma unroll
                    for (int c0 = 0; c0 < HALF; c0 += 16) {
                        uint32_t v[16];
                        tmem_ld16(src + (uint32_t)((use & 1) * BN + c0), v);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; j++) z[c0 + j] += __uint_as_float(v[j]);
                    }
                    release();
                }
                if (failed) break;
                if (MODE == LOSS) take(words_next, r_next);
                if (MODE == LOSS) loss_epilogue(a, z, tg, r.x, row, live, col0);
                else
                    dz_epilogue<MODE == GRAD_RESTS>(a, &maps.z_out, buf, z, tg, r.x, row0, lane, live, col0,
                                                    __int_as_float(r.z), __int_as_float(r.w));
                __syncwarp();
                if (MODE != LOSS) take(words_next, r_next);
            } else if (t.kind == DW) {
                const float scale = out_scale(a);
                take(words_next, r_next);
                if (t.steps > 0 && !finished()) { failed = true; break; }
                for (int c0 = 0; c0 < HALF; c0 += 64) {
                    uint32_t v[2][32];
                    if (t.steps > 0) {
                        tmem_ld32(src + (uint32_t)((use & 1) * BN + c0), v[0]);
                        tmem_ld32(src + (uint32_t)((use & 1) * BN + c0 + 32), v[1]);
                        tmem_wait_ld();
                        if (c0 + 64 == HALF) release();
                    } else {               // no row counts
#pragma unroll
                        for (int j = 0; j < 32; j++) v[0][j] = v[1][j] = 0u;
                    }
                    const int col = col0 + c0;
                    store64(buf, &maps.w_out, col, a.d.v0 + row0, col >= a.in || row0 >= a.d.vc, lane, [&](int j) {
                        const uint32_t *f = v[j >> 2] + 8 * (j & 3);
                        auto pk = [&](int k) {
                            return pack_bf16(__uint_as_float(f[k]) * scale, __uint_as_float(f[k + 1]) * scale);
                        };
                        return make_uint4(pk(0), pk(2), pk(4), pk(6));
                    });
                }
            } else {
                const bool live = row < n_live || (MODE == GRAD_RESTS && row >= a.rest && row < n_rows);
                const float scale = out_scale(a);
                const bool sum = MODE == GRAD_RESTS || a.splits > 1 || !a.last, add = !a.first;
                float4 *acc = a.acc + acc_at(a, t.split, row0, col0) + lane;
                __nv_bfloat16 *out = row < n_live ? a.dX + (size_t)r.x * a.lddx : nullptr;
                take(words_next, r_next);
                if (t.steps > 0 && !finished()) { failed = true; break; }
                for (int c0 = 0; c0 < HALF; c0 += 32) {
                    uint32_t v[32];
                    __syncwarp();
                    if (t.steps > 0) {
                        tmem_ld32(src + (uint32_t)((use & 1) * BN + c0), v);
                        tmem_wait_ld();
                    } else {               // a split past a short last piece
#pragma unroll
                        for (int j = 0; j < 32; j++) v[j] = 0u;
                    }
                    if (!live) continue;
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {      // `in` is a multiple of 8
                        float4 f0, f1;
                        f0 = make_float4(__uint_as_float(v[j]), __uint_as_float(v[j + 1]), __uint_as_float(v[j + 2]),
                                         __uint_as_float(v[j + 3]));
                        f1 = make_float4(__uint_as_float(v[j + 4]), __uint_as_float(v[j + 5]),
                                         __uint_as_float(v[j + 6]), __uint_as_float(v[j + 7]));
                        const int at = (c0 + j) / 4 * 32;
                        if (add) {
                            const float4 p0 = acc[at], p1 = acc[at + 32];
                            f0.x += p0.x; f0.y += p0.y; f0.z += p0.z; f0.w += p0.w;
                            f1.x += p1.x; f1.y += p1.y; f1.z += p1.z; f1.w += p1.w;
                        }
                        if (sum) {
                            acc[at] = f0;
                            acc[at + 32] = f1;
                        } else if (col0 + c0 + j < a.in) {
                            put8(out + col0 + c0 + j, f0, f1, scale, a.vec_dx);
                        }
                    }
                }
                __syncwarp();
                if (t.steps > 0) release();
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        if (failed && lane == 0) flag(DEV_TIMEOUT);
    }
    fence_before();
    __syncwarp();
    sync_all<CG>();
    if (warp == 1) {
        fence_after();
        if (CG == 1)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// dX = the splits' sums in order, each with its row's rest, as bf16. Block (tile, p): columns 8 p ..
// and 128 + 8 p .. of a 128 x 256 tile, a warp for 32 rows of each half.
__global__ void __launch_bounds__(256) sum_splits_kernel(const Args a)
{
    const int cols = (a.in + BN - 1) / BN, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = (int)(blockIdx.x / cols) * BM, n0 = (int)(blockIdx.x % cols) * BN;
    const int group = row0 + (w & 3) * 32, row = group + lane, half = n0 + (w >> 2) * HALF;
    const int col = half + (int)blockIdx.y * 8;
    pdl_wait();
    pdl_release();
    if (row >= *a.n_live || col >= a.in) return;
    float4 f0 = make_float4(0, 0, 0, 0), f1 = f0;
    const float4 *p = a.acc + acc_at(a, 0, group, half) + (int)blockIdx.y * 64 + lane;
    const size_t step = acc_at(a, 1, 0, 0), rest = acc_at(a, 0, a.rest, 0);
    auto add = [&](const float4 *q) {
        const float4 p0 = q[0], p1 = q[32];
        f0.x += p0.x; f0.y += p0.y; f0.z += p0.z; f0.w += p0.w;
        f1.x += p1.x; f1.y += p1.y; f1.z += p1.z; f1.w += p1.w;
    };
    if (rest) {
#pragma unroll 4
        for (int s = 0; s < a.splits; s++, p += step) {
            add(p);
            add(p + rest);
        }
    } else {
#pragma unroll 4
        for (int s = 0; s < a.splits; s++, p += step) add(p);
    }
    put8(a.dX + (size_t)a.rows[row].x * a.lddx + col, f0, f1, out_scale(a), a.vec_dx);
}

// One warp per row: the row's teacher entries as masses over ids in ascending order.
// An entry counts when its id lies in the vocabulary and its logit is not -inf;
// mass = softmax(top / temp) over those. entropy = sum mass ln mass. The maximum carries a
// NaN (fmaxf would drop it): such a row's masses, loss and gradient are NaN.
constexpr int TEACHER_ROWS = 4, PER_LANE = MAXK / 32;
__global__ void __launch_bounds__(32 * TEACHER_ROWS) teacher_kernel(int *s_ids, float *s_mass, int *count, float *entropy,
                                                                    const int *ids, const float *top, int T, int K,
                                                                    int vocab, float inv_temp)
{
    __shared__ __align__(16) int sid_all[TEACHER_ROWS][MAXK];
    pdl_wait();
    pdl_release();
    const int lane = threadIdx.x & 31, row = blockIdx.x * TEACHER_ROWS + (threadIdx.x >> 5);
    if (row >= T) return;
    int *sid = sid_all[threadIdx.x >> 5];
    const size_t base = (size_t)row * K;
    int id[PER_LANE], place[PER_LANE];
    float t[PER_LANE], e[PER_LANE];
    float mx = -INFINITY;
    bool nan = false;
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER_LANE; i++) {
        const int k = lane + 32 * i;
        id[i] = k < K ? ids[base + k] : -1;
        t[i] = k < K ? top[base + k] : -INFINITY;
        if (id[i] >= vocab) {
            flag(DEV_BAD_INDEX);
            id[i] = -1;
        }
        if (id[i] < 0 || t[i] == -INFINITY) id[i] = 0x7fffffff;    // empty: behind every id
        else {
            n++;
            nan |= t[i] != t[i];
            mx = fmaxf(mx, t[i]);
        }
        sid[k] = id[i];
        place[i] = 0;
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (__any_sync(0xffffffffu, nan)) mx = NAN;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, mx, o);
        mx = mx != mx ? mx : fmaxf(mx, other);
    }
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < PER_LANE; i++) {
        t[i] = (t[i] - mx) * inv_temp;
        e[i] = id[i] != 0x7fffffff ? expf(t[i]) : 0.0f;
        sum += (double)e[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncwarp();
    // each entry's place among the ids; equal ids by position
    const int used = (K + 31) & ~31;
    for (int j = 0; j < used; j += 4) {
        const int4 o = *reinterpret_cast<const int4 *>(sid + j);
#pragma unroll
        for (int i = 0; i < PER_LANE; i++) {
            const int k = lane + 32 * i;
            place[i] += (o.x < id[i] || (o.x == id[i] && j < k)) + (o.y < id[i] || (o.y == id[i] && j + 1 < k)) +
                        (o.z < id[i] || (o.z == id[i] && j + 2 < k)) + (o.w < id[i] || (o.w == id[i] && j + 3 < k));
        }
    }
    const double log_sum = log(sum);
    double h = 0.0;
#pragma unroll
    for (int i = 0; i < PER_LANE; i++)
        if (id[i] != 0x7fffffff) {
            const double m = (double)e[i] / sum;
            s_ids[base + place[i]] = id[i];
            s_mass[base + place[i]] = (float)m;
            if (e[i] != 0.0f) h += m * ((double)t[i] - log_sum);   // (a NaN is not equal to 0)
        }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) h += __shfl_xor_sync(0xffffffffu, h, o);
    if (lane == 0) {
        count[row] = n;
        entropy[row] = (float)h;
    }
}

// Numbers the rows that count, in order (rows[place], *n_live), copies their hidden states to
// their places and writes zeros for the others' outputs. Each block takes `per` rows and
// counts the live ones before them itself (T * 4 bytes from L2, at most PACK_BLOCKS blocks),
// so one launch does it. When every row counts and X can be read in place nothing is copied;
// else the rows from the last packed one to the end of its K step become zeros: dW sums over
// them. (What z's tiles read past those is of rows that do not count.) With `rest` all of it stands
// there a second time: what dW takes with the rests of dz.
// The weights are divided by the mantissa of the largest of them (*g_scale): a mean's common
// 1 / n is then a power of two, which rounds nothing when dz becomes bf16, and weights of
// any ratio keep their range. (Where the largest is 0 or not finite, by 1.)
struct Pack {
    int4 *rows;
    int *n_live;
    float *g_scale;
    uint16_t *xp;
    float *loss, *lse_out;             // forward
    __nv_bfloat16 *dX;                 // backward
    const float *lse, *g;
    const uint16_t *X;
    const int *label, *count;          // one of them
    int lddx, ldx, vec, in_place;      // vec: X's rows lie on 16 bytes
    int rest;                          // the packed rows stand at this row again (0: once)
    int T, in, vocab, per;
};

__global__ void __launch_bounds__(256) pack_kernel(const Pack k)
{
    __shared__ int red[2][8];
    __shared__ float red_g[8];
    __shared__ int place[PACK_ROWS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_release();
    const int T = k.T, in = k.in, t0 = blockIdx.x * k.per, t1 = min(T, t0 + k.per);
    auto counts = [&](int t) {
        if (!k.label) return k.count[t] > 0;
        const int l = k.label[t];
        return l >= 0 && l < k.vocab;
    };
    int before = 0, total = 0;
    float g_max = 0.0f;
    for (int t = tid; t < T; t += 256) {
        const int c = counts(t);
        total += c;
        before += t < t0 ? c : 0;
        if (c && k.g) g_max = fmaxf(g_max, fabsf(k.g[t]));
    }
    before = __reduce_add_sync(0xffffffffu, before);
    total = __reduce_add_sync(0xffffffffu, total);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) g_max = fmaxf(g_max, __shfl_xor_sync(0xffffffffu, g_max, o));
    if (lane == 0) { red[0][warp] = before; red[1][warp] = total; red_g[warp] = g_max; }
    __syncthreads();
    before = total = 0;
#pragma unroll
    for (int w = 0; w < 8; w++) {
        before += red[0][w];
        total += red[1][w];
        g_max = fmaxf(g_max, red_g[w]);
    }
    // the mantissa in [1, 2); of an extreme weight all of it
    float g_scale = 1.0f;
    if (k.g && g_max > 0.0f && g_max < INFINITY) {
        const unsigned bits = __float_as_uint(g_max), e = bits >> 23;
        g_scale = e >= 27 && e <= 227 ? __uint_as_float((bits & 0x7FFFFFu) | 0x3F800000u) : g_max;
    }
    if (warp == 0) {
        for (int b = t0; b < t1; b += 32) {
            const int t = b + lane;
            const bool live = t < t1 && counts(t);
            if (t < t1 && k.label && k.label[t] >= k.vocab) flag(DEV_BAD_INDEX);
            const unsigned m = __ballot_sync(0xffffffffu, live);
            const int p = before + __popc(m & ((1u << lane) - 1));
            if (t < t1) place[t - t0] = live ? p : -1;
            if (live) {
                const float l2 = k.lse ? k.lse[t] * LOG2E : 0.0f, g = k.g ? k.g[t] / g_scale : 1.0f;
                k.rows[p] = make_int4(t, k.label ? k.label[t] : k.count[t], __float_as_int(l2), __float_as_int(g));
            }
            before += __popc(m);
        }
    }
    if (blockIdx.x == 0 && tid == 0) {
        *k.n_live = total;
        *k.g_scale = g_scale;
    }
    __syncthreads();
    const bool copy = k.rest || !(k.in_place && total == T);
    // a warp takes a row's next PACK_COLS columns
    const int parts = (in + PACK_COLS - 1) / PACK_COLS;
    for (int w = warp; w < (t1 - t0) * parts; w += 8) {
        const int t = t0 + w / parts, p = place[t - t0], c0 = w % parts * PACK_COLS, c1 = min(in, c0 + PACK_COLS);
        if (p >= 0 && copy) {
            const uint16_t *x = k.X + (size_t)t * k.ldx;
            uint16_t *o = k.xp + (size_t)p * in;
            const size_t again = (size_t)k.rest * in;
            if (k.vec) {
#pragma unroll
                for (int i = 0; i < PACK_COLS / 256; i++) {
                    const int c = c0 + (i * 32 + lane) * 8;
                    if (c < c1) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(x + c);
                        *reinterpret_cast<uint4 *>(o + c) = v;
                        if (again) *reinterpret_cast<uint4 *>(o + again + c) = v;
                    }
                }
            } else {
#pragma unroll 8
                for (int c = c0 + lane; c < c1; c += 32) {
                    const uint16_t v = x[c];
                    o[c] = v;
                    if (again) o[again + c] = v;
                }
            }
        }
        if (p < 0) {
            if (k.loss && c0 == 0 && lane == 0) {
                k.loss[t] = 0.0f;
                k.lse_out[t] = 0.0f;
            }
            if (k.dX)
                for (int c = c0 + lane; c < c1; c += 32) k.dX[(size_t)t * k.lddx + c] = __float2bfloat16_rn(0.0f);
        }
    }
    if (copy) {
        const int end = k.rest ? k.rest : (total + KB - 1) / KB * KB;
        for (int p = total + (int)blockIdx.x * 8 + warp; p < end; p += (int)gridDim.x * 8)
            for (int i = lane; i < in / 8; i += 32) {
                reinterpret_cast<uint4 *>(k.xp + (size_t)p * in)[i] = make_uint4(0u, 0u, 0u, 0u);
                if (k.rest) reinterpret_cast<uint4 *>(k.xp + (size_t)(k.rest + p) * in)[i] = make_uint4(0u, 0u, 0u, 0u);
            }
    }
}

// 32 packed rows a block, 32 threads a row: the tile halves' statistics joined in double.
__global__ void __launch_bounds__(1024) join_kernel(float *loss, float *lse, const float2 *part, int halves, int Tpad,
                                                    const int4 *rows, const int *n_live, const float *zt,
                                                    const float *mass, const float *entropy, int K, float c)
{
    __shared__ float sm[32][33];
    __shared__ float ss[32][33];
    const int r = threadIdx.x & 31, w = threadIdx.x >> 5;
    pdl_wait();
    pdl_release();
    const int row = blockIdx.x * 32 + r, n = *n_live;
    if ((int)blockIdx.x * 32 >= n) return;
    float m = -INFINITY, s = 0.0f;
    if (row < n)
        for (int h = w; h < halves; h += 32 * 8) {
            float2 p[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
                p[i] = h + 32 * i < halves ? part[(size_t)(h + 32 * i) * Tpad + row] : make_float2(-INFINITY, 0.0f);
            float mn = m;
#pragma unroll
            for (int i = 0; i < 8; i++) mn = fmaxf(mn, p[i].x);
            const float ref = mn == -INFINITY ? 0.0f : mn;
            s *= exp2f(m - ref);
#pragma unroll
            for (int i = 0; i < 8; i++) s += p[i].y * exp2f(p[i].x - ref);
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
    const int4 info = rows[mine];
    const int t = info.x, cnt = mass ? info.y : 1;
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
        // in base 2 until the difference is taken: a sure row's loss is small against both, and
        // the targets' z meet the sum's with the factor that it has
        const double l = (double)ref + log2(S), ln2 = 0.69314718055994530942;
        lse[t] = (float)(l * ln2);
        loss[t] = (float)((l - zq * (double)c) * ln2 + (entropy ? (double)entropy[t] : 0.0));
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

constexpr size_t MAX_SUMS = 256 << 20;
// workspaces come in whole 256 KB: batches of about one size share one, and the smallest have one size
// for both directions
constexpr size_t GRAIN = 256 << 10;

static size_t a256(size_t b) { return (b + 255) & ~(size_t)255; }

struct Plan {
    int cg;                            // CTAs that share a unit of the backward
    int Tpad, tiles, piece, pieces;    // vocabulary tiles; ids per piece of the backward; pieces
    int rest, dz_rows, acc_groups;     // where dz's rests begin (0: none), its rows, 32-row groups of dX's sums
    int splits, split_steps;           // of dX's K (a piece)
    size_t dz_bytes, acc_bytes;        // of one piece; of dX's sums in fp32
};

// The steps of the busiest worker when units of three kinds are dealt out in turn: each kind
// gives every worker n / workers units and one more to the n % workers after its start, so
// the busiest is a worker at which some kind starts.
static double busiest(const long long (&n)[3], const double (&cost)[3], int workers)
{
    const int start[3] = {0, (int)(n[0] % workers), (int)((n[0] + n[1]) % workers)};
    double most = 0.0;
    for (int w : start) {
        double t = 0.0;
        for (int k = 0; k < 3; k++)
            t += cost[k] * (double)(n[k] / workers + ((w - start[k] + workers) % workers < n[k] % workers ? 1 : 0));
        most = std::max(most, t);
    }
    return most;
}

static Plan plan(int T, int in, int vocab)
{
    Plan p;
    // Pairs take 7% less time a row where both halves of their 256-row tiles are full (2048 x
    // 7168 over 163,840 ids: 15.4 against 16.4 ms for loss and gradient); 576 rows, 2.25
    // of their tiles, take 18% more.
    p.cg = 100LL * ceil_div(T, 2 * BM) * 2 < 107LL * ceil_div(T, BM) ? 2 : 1;
    p.Tpad = ceil_div(T, ROW_PAD) * ROW_PAD;
    p.tiles = ceil_div(vocab, BN);
    // A piece's dz takes about 128 MB, at least eight tiles: with 64 MB the gradients take 1-4%
    // longer (each launch ends unevenly), with 256 MB -1 to +2%.
    const long long tiles = std::max<long long>(8, (128LL << 20) / ((long long)p.Tpad * 2 * BN));
    p.piece = (int)std::min<long long>(tiles, p.tiles) * BN;
    p.pieces = ceil_div(vocab, p.piece);
    p.rest = T <= 32 ? 32 : 0;
    p.dz_rows = p.rest ? 2 * p.rest : ceil_div(T, KB) * KB;
    p.dz_bytes = (size_t)p.dz_rows * p.piece * 2;
    // dX has few tiles with long sums over the ids: split them where that shortens the busiest
    // worker of the launches, each unit's fp32 sums costing about 16 steps to write
    // and read back; the sums of all splits take 256 MB at most (a limit that only hidden states
    // wider than 16,384 reach)
    const int rows = ceil_div(T, BM * p.cg), cols = ceil_div(in, BN), steps = p.piece / KB;
    const int workers = PLAN_SMS / p.cg;
    const long long n_w = (long long)ceil_div(p.piece, BM * p.cg) * cols, n_z = (long long)rows * (p.piece / BN);
    p.acc_groups = p.rest ? 2 * p.rest / 32 : ceil_div(T, 32);
    const size_t sums = (size_t)p.acc_groups * 32 * cols * BN * 4;
    double best = 0.0;
    p.splits = 1;
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
        if (s > 1 && (steps / s < 4 || s * sums > MAX_SUMS)) break;
        const int len = ceil_div(steps, s);
        const double cost[3] = {len + (s > 1 || p.pieces > 1 ? 16.0 : 4.0), ceil_div(T, KB) + 4.0,
                                ceil_div(in, KB) + 4.0};
        const double t = busiest({(long long)rows * cols * s, n_w, 0}, cost, workers) +
                         (p.pieces - 1) * busiest({(long long)rows * cols * s, n_w, n_z}, cost, workers);
        if (s == 1 || t < 0.98 * best) {
            best = t;
            p.splits = s;
        }
    }
    p.split_steps = ceil_div(steps, p.splits);
    p.splits = ceil_div(steps, p.split_steps);
    p.acc_bytes = p.pieces > 1 || p.splits > 1 || p.rest ? p.splits * sums : 0;
    return p;
}

struct Ws {
    int *n_live, *ids, *count;
    int4 *rows;
    float *g_scale, *mass, *entropy, *zt;
    float4 *acc;
    float2 *part;
    __nv_bfloat16 *xp, *dz[2];
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
    x.g_scale = (float *)take(4);
    x.rows = (int4 *)take((size_t)T * 16);
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
        x.dz[0] = (__nv_bfloat16 *)take(p.dz_bytes);
        x.dz[1] = p.pieces > 1 ? (__nv_bfloat16 *)take(p.dz_bytes) : x.dz[0];
        if (p.acc_bytes) x.acc = (float4 *)take(p.acc_bytes);
    }
    if (w) *w = x;
    return (o + GRAIN - 1) / GRAIN * GRAIN;
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
    for (const void *f : {(const void *)head_kernel<LOSS, 1>, (const void *)head_kernel<GRAD, 1>,
                          (const void *)head_kernel<GRAD, 2>, (const void *)head_kernel<GRAD_RESTS, 1>})
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

// The targets, the rows that count and their hidden states; fills the common arguments. `k`
// holds what one direction adds.
static int set_up(Args *a, Maps *maps, const Call &c, const Plan &p, const Ws &w, Pack k, int cg, bool grad)
{
    int st;
    const float inv_temp = c.K ? 1.0f / c.temp : 1.0f;
    if (c.K) {
        st = launch_pdl(teacher_kernel, dim3(ceil_div(c.T, TEACHER_ROWS)), 32 * TEACHER_ROWS, 0, c.s, 1, w.ids, w.mass,
                        w.count, w.entropy, c.ids, c.top, c.T, c.K, c.vocab, inv_temp);
        if (st) return st;
    }
    // Read in place where TMA can, and where the rows span 128 KB: with a smaller tensor map the
    // weight stream beside it is a fifth slower (9 rows of 7168 over 163,840 ids 490 us, 10 rows
    // 400, the 9 copied to a map of 256 rows 411; the same step at 12 to 16 rows of 4096).
    const int vec = c.ldx % 8 == 0 && aligned(c.X, 16), in_place = vec && (long long)c.T * c.ldx >= (64 << 10);
    k.rows = w.rows; k.n_live = w.n_live; k.g_scale = w.g_scale;
    k.xp = reinterpret_cast<uint16_t *>(w.xp);
    k.X = c.X; k.label = c.label; k.count = w.count;
    k.ldx = c.ldx; k.vec = vec; k.in_place = in_place;
    k.T = c.T; k.in = c.in; k.vocab = c.vocab;
    k.per = ceil_div(c.T, PACK_BLOCKS);
    if ((st = launch_pdl(pack_kernel, dim3(ceil_div(c.T, k.per)), 256, 0, c.s, 1, k))) return st;
    *a = Args{};
    a->T = c.T; a->in = c.in;
    a->n_live = w.n_live; a->rows = w.rows; a->Tpad = p.Tpad;
    a->x_in_place = in_place;
    // the hidden states of a group stay in L2 while the vocabulary streams by: 48 MB of them
    a->group_z = (int)std::max<long long>(ROW_PAD, std::min<long long>(MAX_T, (48LL << 20) / (c.in * 2LL)));
    a->ids = w.ids; a->mass = w.mass;
    a->K = c.K ? c.K : 1;
    // the same in both directions: where p is near 1, p - 1 lives on z and lse agreeing
    a->chunk = c.T <= BM ? 4 : 16;         // (a weight stream leaves the time for it)
    a->inv_temp = inv_temp;
    a->c = c.K ? (float)(1.4426950408889634 / (double)c.temp) : LOG2E;
    const void *x = in_place ? (const void *)c.X : (const void *)w.xp;
    const long long ldx = in_place ? c.ldx : c.in, xr = in_place ? c.T : p.Tpad;
    if ((st = map2d(&maps->x_k, x, c.in, ldx, xr, BM))) return st;
    if ((st = map2d(&maps->xp_k, w.xp, c.in, c.in, p.Tpad, BM))) return st;
    if ((st = map2d(&maps->w_k, c.W, c.in, c.in, c.vocab, BN / cg))) return st;
    if (!grad) return K3GPU_OK;
    if ((st = map2d(&maps->x_mn, x, c.in, ldx, xr, 64))) return st;
    if ((st = map2d(&maps->xp_mn, w.xp, c.in, c.in, p.Tpad, 64))) return st;
    return map2d(&maps->w_mn, c.W, c.in, c.in, c.vocab, 64);
}

template <int MODE, int CG>
static int launch_head(const Maps &maps, const Args &a, int sms, cudaStream_t s)
{
    return launch_pdl(head_kernel<MODE, CG>, dim3(sms / CG * CG), THREADS, SMEM, s, CG, maps, a);
}

static int forward(float *loss, float *lse, const Call &c, void *ws)
{
    int sms = 0, st = prepare_device(&sms);
    if (st) return st;
    const Plan p = plan(c.T, c.in, c.vocab);
    Ws w;
    layout(&w, static_cast<char *>(ws), p, c.T, c.in, c.K, false);
    Args a;
    Maps maps{};
    Pack k{};
    k.loss = loss; k.lse_out = lse;
    if ((st = set_up(&a, &maps, c, p, w, k, 1, false))) return st;
    a.part = w.part; a.zt = w.zt;
    a.z = Piece{0, c.vocab, nullptr};
    if ((st = launch_head<LOSS, 1>(maps, a, sms, c.s))) return st;
    return launch_pdl(join_kernel, dim3(p.Tpad / 32), 1024, 0, c.s, 1, loss, lse, w.part, 2 * p.tiles, p.Tpad, w.rows,
                      w.n_live, w.zt, w.mass, w.entropy, a.K, a.c);
}

// Launch i forms piece i's dz beside the dX and dW of piece i - 1 (two dz buffers), so each
// launch has both kinds of units to fill the SMs with.
static int backward(uint16_t *dX, int lddx, uint16_t *dW, const float *g, const float *lse, const Call &c, void *ws)
{
    int sms = 0, st = prepare_device(&sms);
    if (st) return st;
    const Plan p = plan(c.T, c.in, c.vocab);
    Ws w;
    layout(&w, static_cast<char *>(ws), p, c.T, c.in, c.K, true);
    Args a;
    Maps maps{};
    Pack k{};
    k.dX = reinterpret_cast<__nv_bfloat16 *>(dX); k.lddx = lddx; k.lse = lse; k.g = g;
    k.rest = p.rest;
    if ((st = set_up(&a, &maps, c, p, w, k, p.cg, true))) return st;
    a.g_scale = g ? w.g_scale : nullptr;
    a.acc = w.acc;
    a.dz_rows = p.dz_rows; a.rest = p.rest; a.acc_groups = p.acc_groups;
    a.splits = p.splits; a.split_steps = p.split_steps;
    a.dX = reinterpret_cast<__nv_bfloat16 *>(dX);
    a.want_dx = dX != nullptr; a.want_dw = dW != nullptr;
    a.lddx = lddx; a.vec_dx = lddx % 8 == 0 && aligned(dX, 16);
    a.z_before_dw = c.in > c.T;
    if (dW && (st = map2d(&maps.w_out, dW, c.in, c.in, c.vocab, 32))) return st;
    for (int i = 0; i <= p.pieces; i++) {
        a.d = a.z;
        a.first = i == 1; a.last = i == p.pieces;
        const int v0 = i * p.piece;
        a.z = i < p.pieces ? Piece{v0, std::min(p.piece, c.vocab - v0), w.dz[i & 1]} : Piece{};
        if (i < p.pieces && (st = map2d(&maps.z_out, a.z.dz, p.piece, p.piece, p.dz_rows, 32))) return st;
        if (i > 0) {
            if ((st = map2d(&maps.dz_k, a.d.dz, a.d.vc, p.piece, p.dz_rows, BM))) return st;
            if ((st = map2d(&maps.dz_mn, a.d.dz, a.d.vc, p.piece, p.dz_rows, 64))) return st;
        }
        st = p.rest      ? launch_head<GRAD_RESTS, 1>(maps, a, sms, c.s)
             : p.cg == 1 ? launch_head<GRAD, 1>(maps, a, sms, c.s)
                         : launch_head<GRAD, 2>(maps, a, sms, c.s);
        if (st) return st;
    }
    if (dX && (p.splits > 1 || p.rest)) {
        return launch_pdl(sum_splits_kernel, dim3(ceil_div(c.T, BM) * ceil_div(c.in, BN), HALF / 8), 256, 0, c.s, 1, a);
    }
    return K3GPU_OK;
}

// what one direction needs (K = 0: cross entropy)
static size_t workspace_bytes(int T, int in, int vocab, int K, bool grad)
{
    return layout(nullptr, nullptr, plan(T, in, vocab), T, in, K, grad);
}
static size_t workspace_both(int T, int in, int vocab, int K)
{
    return std::max(workspace_bytes(T, in, vocab, K, false), workspace_bytes(T, in, vocab, K, true));
}

static bool head_ok(const uint16_t *X, int ldx, const uint16_t *W, int in, int vocab, int T, const void *ws)
{
    return X && W && ws && sizes_ok(T, in, vocab) && ldx >= in && aligned(W, 16) && aligned(X, 2) && aligned(ws, 256);
}

// 32-bit values on their boundaries (a NULL passes: what may not be absent is checked beside)
template <typename... P>
static bool words_ok(const P *...p)
{
    return (aligned(p, 4) && ...);
}

static bool grads_ok(const uint16_t *dX, int lddx, const uint16_t *dW, int in)
{
    return (dX || dW) && (!dX || (lddx >= in && aligned(dX, 2))) && (!dW || aligned(dW, 16));
}

static bool teacher_ok(const int *ids, const float *top, int K, float temp)
{
    // (log2(e) / temp is what multiplies the logits)
    return ids && top && words_ok(ids, top) && K > 0 && K <= MAXK && temp > 0.0f && isfinite(temp) &&
           isfinite((float)(1.4426950408889634 / (double)temp));
}

}  // namespace head
}  // namespace k3

extern "C" size_t k3gpu_lm_head_xent_workspace(int T, int in, int vocab)
{
    return k3::head::sizes_ok(T, in, vocab) ? k3::head::workspace_both(T, in, vocab, 0) : 0;
}

extern "C" size_t k3gpu_lm_head_xent_loss_workspace(int T, int in, int vocab)
{
    return k3::head::sizes_ok(T, in, vocab) ? k3::head::workspace_bytes(T, in, vocab, 0, false) : 0;
}

extern "C" int k3gpu_lm_head_xent(float *loss, float *lse, const uint16_t *X, int ldx, const uint16_t *W,
                                  const int *label, int in, int vocab, int T, void *workspace, size_t ws_bytes,
                                  void *stream)
{
    using namespace k3::head;
    if (!loss || !lse || !label || !words_ok(loss, lse, label) || !head_ok(X, ldx, W, in, vocab, T, workspace))
        return K3GPU_EINVAL;
    if (ws_bytes < workspace_bytes(T, in, vocab, 0, false)) return K3GPU_ECAPACITY;
    const Call c{X, W, ldx, in, vocab, T, label, nullptr, nullptr, 0, 1.0f, k3::as_stream(stream)};
    return forward(loss, lse, c, workspace);
}

extern "C" int k3gpu_lm_head_xent_grad(uint16_t *dX, int lddx, uint16_t *dW, const float *g, const float *lse,
                                       const uint16_t *X, int ldx, const uint16_t *W, const int *label, int in,
                                       int vocab, int T, void *workspace, size_t ws_bytes, void *stream)
{
    using namespace k3::head;
    if (!lse || !label || !words_ok(lse, label, g) || !head_ok(X, ldx, W, in, vocab, T, workspace) ||
        !grads_ok(dX, lddx, dW, in))
        return K3GPU_EINVAL;
    if (ws_bytes < workspace_bytes(T, in, vocab, 0, true)) return K3GPU_ECAPACITY;
    const Call c{X, W, ldx, in, vocab, T, label, nullptr, nullptr, 0, 1.0f, k3::as_stream(stream)};
    return backward(dX, lddx, dW, g, lse, c, workspace);
}

extern "C" size_t k3gpu_lm_head_distill_workspace(int T, int in, int vocab, int K)
{
    using namespace k3::head;
    return sizes_ok(T, in, vocab) && K > 0 && K <= MAXK ? workspace_both(T, in, vocab, K) : 0;
}

extern "C" size_t k3gpu_lm_head_distill_loss_workspace(int T, int in, int vocab, int K)
{
    using namespace k3::head;
    return sizes_ok(T, in, vocab) && K > 0 && K <= MAXK ? workspace_bytes(T, in, vocab, K, false) : 0;
}

extern "C" int k3gpu_lm_head_distill(float *loss, float *lse, const uint16_t *X, int ldx, const uint16_t *W,
                                     const int *ids, const float *top, int K, float temp, int in, int vocab, int T,
                                     void *workspace, size_t ws_bytes, void *stream)
{
    using namespace k3::head;
    if (!loss || !lse || !words_ok(loss, lse) || !teacher_ok(ids, top, K, temp) ||
        !head_ok(X, ldx, W, in, vocab, T, workspace))
        return K3GPU_EINVAL;
    if (ws_bytes < workspace_bytes(T, in, vocab, K, false)) return K3GPU_ECAPACITY;
    const Call c{X, W, ldx, in, vocab, T, nullptr, ids, top, K, temp, k3::as_stream(stream)};
    return forward(loss, lse, c, workspace);
}

extern "C" int k3gpu_lm_head_distill_grad(uint16_t *dX, int lddx, uint16_t *dW, const float *g, const float *lse,
                                          const uint16_t *X, int ldx, const uint16_t *W, const int *ids,
                                          const float *top, int K, float temp, int in, int vocab, int T,
                                          void *workspace, size_t ws_bytes, void *stream)
{
    using namespace k3::head;
    if (!lse || !words_ok(lse, g) || !teacher_ok(ids, top, K, temp) || !head_ok(X, ldx, W, in, vocab, T, workspace) ||
        !grads_ok(dX, lddx, dW, in))
        return K3GPU_EINVAL;
    if (ws_bytes < workspace_bytes(T, in, vocab, K, true)) return K3GPU_ECAPACITY;
    const Call c{X, W, ldx, in, vocab, T, nullptr, ids, top, K, temp, k3::as_stream(stream)};
    return backward(dX, lddx, dW, g, lse, c, workspace);
}
