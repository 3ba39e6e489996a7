// Prompt attention over the paged KV cache on the tensor cores (include/vx27_paged.h): causal,
// or the last `window` slots and the first `sinks` ones.
//
// A 2-CTA cluster serves two tiles of 128 query rows against the same keys: the rows of two
// query heads of one KV head, or (odd group sizes) two neighbouring row tiles of one head.
// Its tcgen05 MMAs span both SMs (M = 256): each SM holds its rows' Q, S, P and O and half of
// every K and V tile. Per 128-slot key tile
//     S = Q K^T (fp32, tensor memory), p = 2^(s - m) as bf16 in tensor memory, O += P V,
// with O rescaled only when a row's maximum has grown by more than 2^8.
//
// The clusters are persistent: the next pair's keys and rows are fetched and its first scores
// made while a pair is finished. Pairs are dealt out in turn, as many rounds as all clusters
// share, so that clusters that run at the same time read the same keys (with a stretch of
// neighbouring pairs per cluster they read them all over the sequence, and the L2 does not hold
// that: 13.1 ms instead of 9.6 for 32768 causal rows). The key tiles of the pairs that are left
// are cut into a run per cluster, equal ones where that pays (make_plan): the last round ends
// everywhere at once, and a few rows over a long cache use every SM. A pair that a cut goes
// through leaves a record (O, m, l) per part, which prompt_join_k merges.
//
// Only key tiles with a slot that some row of the pair sees are gone through: the sinks'
// tiles, then those from the first row's window on; masks are applied on tiles that some row
// sees in part. Within a tile the copies fetch page by page; a box without a seen slot reads
// past the pool instead, which fills it with zeros, so freed pages are not touched. The last
// 64-slot block, whose end nothing has written, comes from a zero-padded copy (prompt_tail_k).
//
// What bounds it: the tensor cores and the softmax warps that feed them (4 T_keys 128 256 FLOP
// per row tile); K and V come from L2, which the heads of a KV head share. 2048 rows after 14001
// slots take 570 us at 1965 MHz (1330 TFLOP/s, 0.81 of the cuBLAS rate; 1.8 us a key tile of a
// pair) and 650-670 under the power cap; 300 rows after 130, one round, 20 us, of which the last
// pair's rows are 5: two SFU operations per gate and 32 rows an access. A tile holds rows of one
// head, so few rows leave most of it empty: one row after 8000 slots takes 46 us, 8 rows 48,
// against 5 for the bytes.
//
// p is rounded to bf16, half a step of 2^-8 relative, and l sums it unrounded: results are off by
// 2.1e-3 to 2.4e-3 of their size, of which their own rounding to bf16 makes 1.7e-3. A second
// term of p would take as many O MMAs again (half as many tensor operations more in all), and
// tensor memory is full.
//
// Warps of a CTA: 0 copies K (and Q), 11 copies V, 1 S MMAs, 10 O MMAs, 2-9 softmax (two
// threads a row, one per half of the keys and of the output columns). Rank 0 issues the
// pair's MMAs. Waits are bounded (2 s).
#include <math.h>
#include <algorithm>
#include "common.cuh"
#include "gqa_paged.cuh"
#include "tc.cuh"

namespace vx27 {
namespace {

constexpr int HD = PG_HD;
constexpr int QT = 128;           // query rows of a CTA
constexpr int KT = 128;           // slots of a key tile
constexpr int NK = 10, NV = 9;    // ring slots of K and V
constexpr int CHUNK = 8192;       // K: 64 slots x 64 dims; V: 32 slots x 128 dims
constexpr int TAIL = 64;          // slots of the padded last block
constexpr int O_WARP = 10, V_WARP = 11;
constexpr int THREADS = 384;
constexpr float RESCALE_LOG2 = 8.0f;
constexpr int MAX_RUNS = 96;
constexpr int CUT_COST = 6;       // what a cut costs, in key tiles (a record's write and merge: ~10 us)
// tensor memory: S at [0, 128), O at [128, 384), P as bf16 pairs at [384, 512), two buffers
constexpr uint32_t TM_O = 128, TM_P = 384;

struct Smem {
    uint8_t q[4][QT * 128];
    uint8_t ring[NK + NV][CHUNK];  // K slots, then V slots
    float xmax[2][2][QT], xsum[2][2][QT];
    uint64_t qfull, q_empty, o_empty, full[NK + NV], empty[NK + NV], s_full, s_empty, p_full[2], pv_done[2],
        o_final, mma_done, qk_done;
    int pages[2][2][KT / 16];  // K and V: of the tile being copied and of the next one
    uint32_t tmem_base;
    int abort;
};
static_assert(sizeof(Smem) + 1024 <= 232448, "smem");

// First `rounds` rounds of a pair per cluster, every second one in reverse; then, dealt out in
// the same way, run c begins with key tile tile[c] of pair item[c], u[c] tiles into what is left.
struct PromptPlan {
    int clusters, rounds, runs, cuts;  // cuts: runs that begin inside a pair
    int item[MAX_RUNS + 1], tile[MAX_RUNS + 1], u[MAX_RUNS + 1];
};

struct PromptArgs {
    const uint16_t *gate;
    const int *table;
    uint16_t *out;
    float *rec_o;    // [runs][2: begun earlier, begun here][2 CTAs][128][256], O not divided by l
    float2 *rec_ml;  // [runs][2][2][128] (m in log2 units, l)
    PagePool pool;
    int max_pages, s0, T, nq, window, sinks, by_heads;
    PromptPlan plan;
};

__device__ __forceinline__ bool try_wait(uint32_t addr, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; "
        "selp.u32 %0, 1, 0, p; }"
        : "=r"(ok) : "r"(addr), "r"(parity) : "memory");
    return ok;
}
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Bounded wait that goes on after an abort: what must be done before a CTA may leave.
__device__ __forceinline__ void drain(uint64_t *bar, uint32_t parity) {
    const uint32_t addr = smem_u32(bar);
    for (int it = 0; it < (1 << 20); it++)
        if (try_wait(addr, parity)) return;
}
// The pair's waits: one that runs out aborts both CTAs.
struct Sync {
    int *abort;
    uint32_t *status;
    uint32_t peer_abort;  // shared::cluster address of the other CTA's abort word
    __device__ void fail(uint32_t code) const {
        *(volatile int *)abort = 1;
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_abort), "r"(1) : "memory");
        dev_flag(status, code);
    }
    __device__ bool aborted() const { return *(volatile int *)abort != 0; }
    // only the first try is inlined: the roles' loops share the instruction cache
    __device__ __noinline__ bool wait_long(uint32_t addr, uint32_t parity, uint32_t code) const {
        const uint64_t t0 = now_ns();
        for (;;) {
            if (try_wait(addr, parity)) return true;
            if (aborted()) return false;
            if (now_ns() - t0 > 2000000000ull) break;
        }
        fail(code);
        return false;
    }
    __device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, uint32_t code) const {
        const uint32_t addr = smem_u32(bar);
        return try_wait(addr, parity) || wait_long(addr, parity, code);
    }
    // a softmax warp's arrival on rank 0's barrier (16 of the pair's)
    __device__ void arrive(uint64_t *bar) const {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive_cluster(mapa_shared(bar, 0));
    }
};

// The key tiles of a pair whose rows sit in slots [a, e): the sinks' tiles, then [win0, end).
struct KeyTiles {
    int lo, sink_end, sink_tiles, win0, n;
    __host__ __device__ KeyTiles(int a, int e, int window, int sinks) {
        const SeenSlots first(a + 1, window, sinks);
        lo = first.win_begin;
        sink_end = first.sink_end;
        win0 = lo / KT;
        const int st = (sink_end + KT - 1) / KT;
        sink_tiles = st < win0 ? st : win0;
        n = sink_tiles + (e + KT - 1) / KT - win0;
    }
    __device__ int slot0(int m) const { return (m < sink_tiles ? m : win0 + m - sink_tiles) * KT; }
    // does some row see a slot of [s, s + len)? (up to the pair's end, which the caller knows)
    __device__ bool seen(int s, int len) const { return s + len > lo || s < sink_end; }
};

// Rows [ta, tb) of pair p, those with most keys first; its tiles of 128 rows start at ta.
__host__ __device__ inline void pair_rows(int p, int T, int nq, int by_heads, int *ta, int *tb) {
    const int step = by_heads ? QT : 2 * QT, per = by_heads ? nq / 2 : nq;
    *ta = ((T + step - 1) / step - 1 - p / per) * step;
    *tb = *ta + step < T ? *ta + step : T;
}

// A CTA's way through its pairs, each with its key tiles [v0, v0 + cnt).
struct Walk {
    const PromptArgs &a;
    int c, rank, round, run, left, p, v0, cnt, h, t0;  // left: tiles to go in the run
    bool over;
    KeyTiles kt;
    __device__ __forceinline__ Walk(const PromptArgs &a_, int c_, int rank_)
        : a(a_), c(c_), rank(rank_), round(-1), run(0), left(0), p(0), v0(0), cnt(0), h(0), t0(0),
          over(false), kt(0, 1, 0, 0) {
        next();
    }
    __device__ __forceinline__ bool done() const { return over; }
    __device__ __forceinline__ bool whole() const { return cnt == kt.n; }
    __device__ __forceinline__ void next() {
        const PromptPlan &pl = a.plan;
        v0 = 0;
        const int turn = ++round & 1 ? pl.clusters - 1 - c : c;
        if (round < pl.rounds) {
            p = round * pl.clusters + turn;
        } else if (round == pl.rounds) {
            run = turn;
            p = pl.item[run];
            v0 = pl.tile[run];
            left = pl.u[run + 1] - pl.u[run];
            over = left <= 0;
        } else {
            p++;
            left -= cnt;
            over = left <= 0;
        }
        if (over) return;
        int ta, tb;
        pair_rows(p, a.T, a.nq, a.by_heads, &ta, &tb);
        kt = KeyTiles(a.s0 + ta, a.s0 + tb, a.window, a.sinks);
        h = a.by_heads ? 2 * (p % (a.nq / 2)) + rank : p % a.nq;
        t0 = a.by_heads ? ta : ta + QT * rank;
        cnt = round < pl.rounds ? kt.n : min(kt.n - v0, left);
    }
};

// The result of a pair's 128 rows: O / l * sigmoid(gate), or a record of the part. By 32
// columns, in a loop that is not unrolled (its code is shared by all of the row's columns),
// the gate requested one round ahead; its sigmoid uses the SFU's 2^x and reciprocal.
__device__ __forceinline__ bool write_rows(Smem &sm, const Sync &sy, const PromptArgs &a, uint32_t to,
                                           int k, bool whole, int h, int t_row, size_t rec_row, int hf,
                                           float m, float l) {
    const size_t base = ((size_t)t_row * a.nq + h) * HD + hf * (HD / 2);
    const bool gated = whole && a.gate && t_row < a.T;
    uint4 gate[4], next[4];
    auto request = [&](int i) {
        const uint4 *gp = reinterpret_cast<const uint4 *>(a.gate + base) + 4 * i;
#pragma unroll
        for (int e = 0; e < 4; e++) next[e] = gp[e];
    };
    if (gated) request(0);
    bool ok = sy.wait(&sm.o_final, k & 1, VX_DEV_TIMEOUT_MMA);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) return false;
    tc_fence_after();
    const float inv = whole ? 1.0f / l : 1.0f;
    if (!whole && hf == 0) a.rec_ml[rec_row] = make_float2(m, l);
#pragma unroll 1
    for (int i = 0; i < HD / 64; i++) {
        float o[32];
        __syncwarp();  // rows past T store nothing; the loads want the whole warp
        tmem_ld16(to + 32 * i, o);
        tmem_ld16(to + 32 * i + 16, o + 16);
        if (!whole) {
            float4 *d = reinterpret_cast<float4 *>(a.rec_o + rec_row * HD + hf * (HD / 2) + 32 * i);
#pragma unroll
            for (int e = 0; e < 8; e++) d[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            continue;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) gate[e] = next[e];
        if (gated && i < HD / 64 - 1) request(i + 1);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = o[8 * q + e] * inv;
            if (gated) {
                const uint32_t gw[4] = {gate[q].x, gate[q].y, gate[q].z, gate[q].w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[2 * e] *= __fdividef(1.0f, 1.0f + __expf(-bf16_to_f32(gw[e] & 0xffffu)));
                    x[2 * e + 1] *= __fdividef(1.0f, 1.0f + __expf(-bf16_to_f32(gw[e] >> 16)));
                }
            }
            if (t_row < a.T) st8_bf16(a.out + base + 32 * i + 8 * q, x);
        }
    }
    tc_fence_before();
    return true;
}

// Softmax, rescale and results of this CTA's 128 rows, two threads a row.
__device__ __forceinline__ void softmax_role(Smem &sm, const Sync &sy, const PromptArgs &a,
                                             Walk w, uint32_t tmem, int warp, int lane) {
    const uint32_t tO = tmem + TM_O;
    const int q4 = warp & 3, hf = (warp - 2) >> 2, r = q4 * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
    const float sc2 = 1.4426950408889634f * 0.0625f;  // log2(e) / sqrt(256)
    float m_run = -INFINITY, l_run = 0.0f;
    bool ok = true;
    int g = 0, k = 0;                       // key tiles and pairs so far
    int e_h = 0, e_t0 = 0;                  // the pair that has ended
    bool e_whole = false;
    size_t e_rec = 0;
    // every softmax warp goes through all tiles and the named barrier of each, also after a
    // failed wait (then skipping the tensor-memory work), so none is left waiting
    for (int i = 0;;) {  // tile i of the pair; after the last tile once more, to finish it
        const bool last = w.done(), ended = i == 0 && g > 0;
        const int b = g & 1;
        constexpr int HK = KT / 2;
        float s[HK];
        float mloc = -INFINITY;
        if (!last) {
            if (ok) ok = sy.wait(&sm.s_full, b, VX_DEV_TIMEOUT_MMA);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
                tc_fence_after();
                tmem_ld64(tmem + lane_off + hf * HK, s);
                tc_fence_before();
                sy.arrive(&sm.s_empty);
                const int s0 = w.kt.slot0(w.v0 + i), k0 = s0 + hf * HK, q0 = a.s0 + w.t0;
                // masks on tiles that some row does not see whole
                if (s0 > q0 - (KT - 1) || (a.window && s0 < q0 + QT - a.window)) {
                    const int qpos = q0 + r;
                    const int row_lo = a.window ? qpos - a.window : -1;  // the window is above it
#pragma unroll
                    for (int e = 0; e < HK; e++)
                        if (k0 + e > qpos || (k0 + e <= row_lo && k0 + e >= a.sinks)) s[e] = -INFINITY;
                }
                float mx[16];
#pragma unroll
                for (int e = 0; e < 16; e++)
                    mx[e] = fmaxf(fmaxf(s[4 * e], s[4 * e + 1]), fmaxf(s[4 * e + 2], s[4 * e + 3]));
#pragma unroll
                for (int x = 8; x >= 1; x >>= 1)
#pragma unroll
                    for (int e = 0; e < x; e++) mx[e] = fmaxf(mx[e], mx[e + x]);
                mloc = mx[0];
            }
        }
        // the two threads of a row meet: this tile's maxima, the ended pair's sums
        sm.xmax[b][hf][r] = mloc;
        if (ended) sm.xsum[k & 1][hf][r] = l_run;
        named_bar_sync(1, 256);
        const float mpart = sm.xmax[b][hf ^ 1][r];
        float l_old = 0.f;
        const float m_old = m_run;
        if (ended) {
            l_old = l_run + sm.xsum[k & 1][hf ^ 1][r];
            m_run = -INFINITY;
            l_run = 0.f;
        }
        if (!last && ok) {
            const float mt = fmaxf(mloc, mpart) * sc2;
            float alpha = 1.0f;
            const bool grow = mt > m_run + RESCALE_LOG2;
            if (grow) {
                alpha = ex2_approx(m_run - mt);
                m_run = mt;
            }
            // not on a pair's first tile, where O holds nothing yet; alpha may be 0 (a row that
            // has seen nothing, or whose weights underflow), which clears O
            if (__any_sync(0xffffffffu, grow && i > 0)) {
                ok = sy.wait(&sm.pv_done[b ^ 1], ((g - 1) >> 1) & 1, VX_DEV_TIMEOUT_MMA);
                ok = __all_sync(0xffffffffu, ok);
                if (ok) {
                    tc_fence_after();
#pragma unroll 1
                    for (int e = 0; e < HD / 32; e++) {
                        float o[16];
                        const uint32_t ta = tO + lane_off + hf * (HD / 2) + 16 * e;
                        tmem_ld16(ta, o);
#pragma unroll
                        for (int x = 0; x < 16; x++) o[x] *= alpha;
                        tmem_st16(ta, o);
                    }
                }
            }
            // P buffer b is free once O += P(g-2) V(g-2) is done
            if (ok && g >= 2) {
                ok = sy.wait(&sm.pv_done[b], ((g >> 1) - 1) & 1, VX_DEV_TIMEOUT_MMA);
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after();
            }
            if (ok) {
                float ls[4] = {0.f, 0.f, 0.f, 0.f};
                const float nm = m_run == -INFINITY ? 0.0f : -m_run;  // nothing seen: p = 2^-inf = 0
                uint32_t pw[32];
#pragma unroll
                for (int u = 0; u < 8; u++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float pa = ex2_approx(fmaf(s[u * 8 + 2 * e], sc2, nm));
                        const float pb = ex2_approx(fmaf(s[u * 8 + 2 * e + 1], sc2, nm));
                        ls[e] += pa + pb;
                        pw[4 * u + e] = pack_bf16x2(pa, pb);
                    }
                }
                tmem_st32(tmem + TM_P + 64u * b + lane_off + 32 * hf, pw);
                tmem_st_wait();
                tc_fence_before();
                l_run = fmaf(l_run, alpha, (ls[0] + ls[1]) + (ls[2] + ls[3]));
                sy.arrive(&sm.p_full[b]);
            }
        }
        // the ended pair's rows, behind the next one's first P: O += P V then waits for them,
        // S does not
        if (ended) {
            if (ok) ok = write_rows(sm, sy, a, tO + lane_off + hf * (HD / 2), k, e_whole, e_h, e_t0 + r,
                                    e_rec + r, hf, m_old, l_old);
            if (ok) sy.arrive(&sm.o_empty);
            k++;
        }
        if (last) break;
        g++;
        if (++i == w.cnt) {
            i = 0;
            e_h = w.h;
            e_t0 = w.t0;
            e_whole = w.whole();
            e_rec = (size_t)((2 * w.run + (w.v0 > 0 ? 0 : 1)) * 2 + w.rank) * QT;
            w.next();
        }
    }
    if (!ok) *(volatile int *)sy.abort = 1;
}

__global__ void __launch_bounds__(THREADS, 1)
paged_prompt_k(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
               const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmtk,
               const __grid_constant__ CUtensorMap tmtv, const __grid_constant__ PromptArgs a,
               uint32_t *status) {
    extern __shared__ uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_rank();
    const int nkv = a.pool.nkv, group = a.nq / nkv, c = (int)(blockIdx.x >> 1);

    if (tid == 32) {  // not of warp 0, which allocates as a whole
        mbar_init(&sm.qfull, 1);
        mbar_init(&sm.q_empty, 1);
        mbar_init(&sm.o_empty, 16);
        for (int i = 0; i < NK + NV; i++) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], 1);
        }
        mbar_init(&sm.s_full, 1);
        mbar_init(&sm.s_empty, 16);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sm.p_full[i], 16);
            mbar_init(&sm.pv_done[i], 1);
        }
        mbar_init(&sm.o_final, 1);
        mbar_init(&sm.mma_done, 1);
        mbar_init(&sm.qk_done, 1);
        sm.abort = 0;
        fence_barrier_init();
    }
    if (warp == 0) {
        tmem_alloc_pair(&sm.tmem_base, 512);
        tmem_relinquish_pair();
        if (lane == 0) {
            tma_prefetch_desc(&tmq);
            tma_prefetch_desc(&tmk);
            tma_prefetch_desc(&tmv);
        }
    }
    tc_fence_before();
    __syncwarp();
    cluster_sync();  // both CTAs' barriers initialised and tensor memory allocated
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;
    const uint32_t tO = tmem + TM_O;
    const Sync sy{&sm.abort, status, mapa_shared(&sm.abort, rank ^ 1u)};
    grid_dep_wait();
    Walk w(a, c, (int)rank);

    if (warp == 0 || warp == V_WARP) {
        // ---- copies: this CTA's halves of the K chunks (warp 0) and of the V chunks ----------
        // Lane i < 8 has the box that begins at the i-th 16-slot group: of this CTA's 64 slots
        // of a K tile, of the 128 of a V tile (bigger boxes: every second or fourth lane).
        const bool is_k = warp == 0;
        const int ps = 1 << a.pool.ps_log, end = a.s0 + a.T;
        const int tail0 = end / TAIL * TAIL;  // first slot of the padded block
        const int none = (int)((size_t)a.pool.n_pages * nkv << a.pool.ps_log);  // past the pool
        const int box = min(ps, is_k ? 64 : 32);
        const bool leads = lane < (is_k ? 4 : 8) && 16 * lane % box == 0;
        const int rel = (is_k ? 64 * (int)rank : 0) + 16 * lane;  // first slot, from the tile's
        // The page goes to shared memory by an asynchronous copy, a tile ahead (a load into a
        // register is waited for at once where it leaves its branch).
        auto fetch = [&](const Walk &f, int m, int g) {
            if (!leads || f.done()) return;
            const int s = f.kt.slot0(m) + rel;
            if (s >= tail0 || !f.kt.seen(s, box)) return;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;"
                         ::"r"(smem_u32(&sm.pages[!is_k][g & 1][lane])),
                         "l"(a.table + (s >> a.pool.ps_log)) : "memory");
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        const int slots = is_k ? NK : NV, ring0 = is_k ? 0 : NK;
        const uint32_t full0 = mapa_shared(&sm.full[ring0], 0);
        bool ok = true;
        // Q of the k-th pair, once the S MMAs of the pair before are done: asked for after two
        // tiles of its K, which the ring holds meanwhile
        auto load_q = [&](const Walk &w, int k) {
            if (k > 0) ok = __all_sync(0xffffffffu, sy.wait(&sm.q_empty, (k - 1) & 1, VX_DEV_TIMEOUT_MMA));
            if (!ok || lane != 0) return;
            if (rank == 0) mbar_arrive_expect_tx(&sm.qfull, 2 * 4 * QT * 128);
            const uint32_t lq = mapa_shared(&sm.qfull, 0);
            for (int e = 0; e < 4; e++) tma_load_3d_pair(sm.q[e], &tmq, e * 64, w.h, w.t0, lq);
        };
        Walk f = w;               // one tile ahead of w
        int fm = f.v0;
        int n = 0, sl = 0, g = 0, k = 0;  // chunks; the next one's ring slot; tiles; pairs
        uint32_t phase = 1;       // of its empty barrier (the first round waits for nothing)
        fetch(f, fm, 0);
        if (is_k && !w.done()) load_q(w, 0);
        for (; !w.done() && ok; w.next(), k++) {
            const int kvh = w.h / group;
            for (int i = 0; i < w.cnt && ok; i++, g++) {
                if (is_k && k > 0 && i == 2) load_q(w, k);
                asm volatile("cp.async.wait_all;" ::: "memory");
                const int s = w.kt.slot0(w.v0 + i) + rel;
                const bool tail = s >= tail0;
                bool issue = leads;
                int y = none;
                if (leads && tail) {  // the padded block (64 slots of K, 32 of V at a time), or zeros
                    issue = is_k ? lane == 0 : (lane & 1) == 0;
                    y = kvh * TAIL + s - tail0;
                    if (s >= tail0 + TAIL) y = nkv * TAIL;
                } else if (leads && w.kt.seen(s, box)) {
                    const int page = sm.pages[!is_k][g & 1][lane];
                    if (a.pool.has(page)) y = (int)a.pool.row(page, kvh, s);
                    else dev_flag(status, VX_DEV_BAD_ARG);
                }
                if (++fm == f.v0 + f.cnt) {
                    f.next();
                    fm = f.v0;
                }
                fetch(f, fm, g + 1);
                const CUtensorMap *map = is_k ? (tail ? &tmtk : &tmk) : (tail ? &tmtv : &tmv);
                const bool halves = !is_k && !tail && ps == 16;  // V boxes of 16 slots, one block each
                const int off = is_k ? lane * 2048 : halves ? (lane & 1) * 2048 : 0;
                for (int e = 0; e < 4 && ok; e++) {
                    if (n >= slots)
                        ok = __all_sync(0xffffffffu,
                                        sy.wait(&sm.empty[ring0 + sl], phase, VX_DEV_TIMEOUT_TMA));
                    if (!ok) break;
                    if (lane == 0 && rank == 0) mbar_arrive_expect_tx(&sm.full[ring0 + sl], 2 * CHUNK);
                    uint8_t *dst = sm.ring[ring0 + sl] + off;
                    const uint32_t bar = full0 + 8 * sl;
                    if (is_k) {  // dims [64 e, 64 e + 64)
                        if (issue) tma_load_2d_pair(dst, map, e * 64, y, bar);
                    } else if (issue && (lane >> 1) == e) {  // slots [32 e, ..), two blocks of 64 dims
                        tma_load_3d_pair(dst, map, 0, y, 2 * (int)rank, bar);
                        if (halves) tma_load_3d_pair(dst + 4096, map, 0, y, 2 * (int)rank + 1, bar);
                    }
                    n++;
                    if (++sl == slots) {
                        sl = 0;
                        phase ^= 1;
                    }
                }
            }
            if (is_k && k > 0 && w.cnt <= 2 && ok) load_q(w, k);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (rank == 0) {  // every copy of both CTAs lands before this CTA can leave
            for (int i = max(0, n - slots); i < n; i++)
                drain(&sm.full[ring0 + i % slots], (i / slots) & 1);
            if (is_k && k > 0) drain(&sm.qfull, (k - 1) & 1);
        }
        if (sy.aborted()) {
            // the two CTAs may have issued different numbers of copies, which no barrier then
            // tracks: 200 us for those in flight
            const uint64_t tw = now_ns();
            while (now_ns() - tw < 200000ull) {
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {  // ---- S = Q K(m)^T once the softmax has read S(m-1)
            const uint32_t id1 = idesc_bf16(256, KT, false, false);
            const uint64_t dq0 = sdesc_sw128(smem_u32(sm.q[0]), 16, 1024);
            const uint64_t dr0 = sdesc_sw128(smem_u32(sm.ring[0]), 16, 1024);
            bool ok = true;
            int g = 0, sl = 0;
            uint32_t phase = 0;
            for (int k = 0; !w.done() && ok; w.next(), k++) {
                ok = sy.wait(&sm.qfull, k & 1, VX_DEV_TIMEOUT_TMA);
                for (int i = 0; i < w.cnt && ok; i++, g++) {
                    if (g >= 1) ok = sy.wait(&sm.s_empty, (g - 1) & 1, VX_DEV_TIMEOUT_MMA);
                    for (int e = 0; e < 4 && ok; e++) {
                        ok = sy.wait(&sm.full[sl], phase, VX_DEV_TIMEOUT_TMA);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t dq = sdesc_add(dq0, e * (QT * 128));
                        const uint64_t dk = sdesc_add(dr0, sl * CHUNK);
#pragma unroll
                        for (int kk = 0; kk < 4; kk++)
                            mma_bf16_pair(tmem, sdesc_add(dq, kk * 32), sdesc_add(dk, kk * 32), id1,
                                          (e | kk) != 0);
                        mma_commit_pair_both(&sm.empty[sl]);
                        if (++sl == NK) {
                            sl = 0;
                            phase ^= 1;
                        }
                    }
                    if (ok) mma_commit_pair_both(&sm.s_full);
                }
                if (ok) mma_commit_pair_both(&sm.q_empty);
            }
            mma_commit_pair(mapa_shared(&sm.qk_done, 0));
            drain(&sm.qk_done, 0);
        }
    } else if (warp == O_WARP) {
        if (lane == 0 && rank == 0) {  // ---- O += P(t) V(t)
            const uint32_t id2 = idesc_bf16(256, HD, false, true);
            const uint64_t dv0 = sdesc_sw128(smem_u32(sm.ring[0]), 32 * 128, 1024);
            bool ok = true;
            int g = 0, sl = 0;
            uint32_t phase = 0;
            for (int k = 0; !w.done() && ok; w.next(), k++) {
                for (int i = 0; i < w.cnt && ok; i++, g++) {
                    const int pb = g & 1;
                    ok = sy.wait(&sm.p_full[pb], (g >> 1) & 1, VX_DEV_TIMEOUT_MMA);
                    // the rows of the pair before have been read
                    if (ok && i == 0 && k > 0) ok = sy.wait(&sm.o_empty, (k - 1) & 1, VX_DEV_TIMEOUT_MMA);
                    for (int e = 0; e < 4 && ok; e++) {
                        ok = sy.wait(&sm.full[NK + sl], phase, VX_DEV_TIMEOUT_TMA);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t dv = sdesc_add(dv0, (NK + sl) * CHUNK);
#pragma unroll
                        for (int k2 = 0; k2 < 2; k2++) {
                            const int kk = 2 * e + k2;
                            mma_bf16_pair_ts(tO, tmem + TM_P + 64u * pb + 8u * kk,
                                             sdesc_add(dv, k2 * 2048), id2, (i > 0 || kk > 0) ? 1u : 0u);
                        }
                        mma_commit_pair_both(&sm.empty[NK + sl]);
                        if (++sl == NV) {
                            sl = 0;
                            phase ^= 1;
                        }
                    }
                    if (ok) mma_commit_pair_both(&sm.pv_done[pb]);
                }
                if (ok) mma_commit_pair_both(&sm.o_final);
            }
            mma_commit_pair(mapa_shared(&sm.mma_done, 0));
            drain(&sm.mma_done, 0);
        }
    } else {
        softmax_role(sm, sy, a, w, tmem, warp, lane);
    }
    __syncwarp();
    __syncthreads();
    // neither CTA leaves (or frees tensor memory) while the other may still arrive on its
    // barriers or rank 0's MMAs may touch its memory
    tc_fence_before();
    __syncwarp();
    cluster_sync();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

// The last 64-slot block, zero behind slot `end` and where no row sees it: [2][nkv][64][256],
// one warp per row.
__global__ void __launch_bounds__(256)
prompt_tail_k(const uint16_t *kp, const uint16_t *vp, uint16_t *tail, PagePool pool,
              const int *table, int s0, int end, int window, int sinks, uint32_t *status) {
    grid_dep_wait();
    grid_dep_launch();
    const int row = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
    if (row >= 2 * pool.nkv * TAIL) return;
    const int i = row % TAIL, h = row / TAIL % pool.nkv;
    const int slot = end / TAIL * TAIL + i;
    const SeenSlots first(s0 + 1, window, sinks);  // what the first row does not see in front of
    uint4 x = make_uint4(0, 0, 0, 0);              // its window, none sees
    if (slot < end && (slot >= first.win_begin || slot < first.sink_end)) {
        const int page = table[slot >> pool.ps_log];
        if (pool.has(page))
            x = reinterpret_cast<const uint4 *>((row < pool.nkv * TAIL ? kp : vp) +
                                                pool.row(page, h, slot) * HD)[lane];
        else
            dev_flag(status, VX_DEV_BAD_ARG);
    }
    reinterpret_cast<uint4 *>(tail + (size_t)row * HD)[lane] = x;
}

// Rows of a pair that runs c1 .. c2 share: o = sum_i O_i 2^(m_i - m) / sum_i l_i 2^(m_i - m) *
// sigmoid(gate). Block (16 rows, CTA, boundary c) works if run c is the second one; a warp per
// two rows, 8 dims a lane.
__global__ void __launch_bounds__(256)
prompt_join_k(const __grid_constant__ PromptArgs a) {
    grid_dep_wait();
    const int c = blockIdx.z + 1, rank = blockIdx.y, lane = threadIdx.x & 31;
    const PromptPlan &pl = a.plan;
    if (pl.tile[c] == 0 || (pl.item[c - 1] == pl.item[c] && pl.tile[c - 1] > 0)) return;
    int c2 = c;
    while (c2 + 1 < pl.runs && pl.item[c2 + 1] == pl.item[c] && pl.tile[c2 + 1] > 0) c2++;
    int ta, tb;
    pair_rows(pl.item[c], a.T, a.nq, a.by_heads, &ta, &tb);
    const int h = a.by_heads ? 2 * (pl.item[c] % (a.nq / 2)) + rank : pl.item[c] % a.nq;
    const int t0 = a.by_heads ? ta : ta + QT * rank;
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int r = blockIdx.x * 16 + 2 * (threadIdx.x >> 5) + u;
        if (t0 + r >= a.T) return;
        // parts: the item begins in run c - 1 (its last), runs c .. c2 go on with it (their first)
        auto row = [&](int i) { return (size_t)((2 * i + (i < c ? 1 : 0)) * 2 + rank) * QT + r; };
        // the first two parts' rows and the gate in one round trip
        const size_t at = ((size_t)(t0 + r) * a.nq + h) * HD + 8 * lane, r0 = row(c - 1), r1 = row(c);
        float o[8], x[8], gate[8];
        ld8_f32(o, a.rec_o + r0 * HD + 8 * lane);
        ld8_f32(x, a.rec_o + r1 * HD + 8 * lane);
        if (a.gate) ld8_bf16(gate, a.gate + at);
        const float2 ml0 = a.rec_ml[r0], ml1 = a.rec_ml[r1];
        float m = fmaxf(ml0.x, ml1.x);
        for (int i = c + 1; i <= c2; i++) m = fmaxf(m, a.rec_ml[row(i)].x);
        // a part without a seen slot has m = -inf (and l = 0)
        const float f0 = ml0.x == -INFINITY ? 0.f : exp2f(ml0.x - m);
        const float f1 = ml1.x == -INFINITY ? 0.f : exp2f(ml1.x - m);
        float l = fmaf(ml1.y, f1, ml0.y * f0);
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = fmaf(x[e], f1, o[e] * f0);
        for (int i = c + 1; i <= c2; i++) {
            const float2 ml = a.rec_ml[row(i)];
            const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m);
            ld8_f32(x, a.rec_o + row(i) * HD + 8 * lane);
            l = fmaf(ml.y, f, l);
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = fmaf(x[e], f, o[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            o[e] /= l;
            if (a.gate) o[e] *= __fdividef(1.0f, 1.0f + __expf(-gate[e]));
        }
        st8_bf16(a.out + at, o);
    }
}

// The rounds, and the runs of what is left: equal ones, or a pair each where cutting pairs
// saves no more than it costs.
int make_plan(PromptPlan &pl, int clusters, int s0, int T, int nq, int by_heads, int window,
              int sinks) {
    const int step = by_heads ? QT : 2 * QT, per = by_heads ? nq / 2 : nq;
    const int groups = (T + step - 1) / step;  // of `per` pairs with the same rows
    const long long pairs = (long long)groups * per;
    if (pairs > 0x7fffffffLL / 2) return -1;
    auto tiles = [&](int i) {
        int ta, tb;
        pair_rows(i * per, T, nq, by_heads, &ta, &tb);
        return KeyTiles(s0 + ta, s0 + tb, window, sinks).n;
    };
    pl.clusters = (int)std::min<long long>(clusters, pairs);
    pl.rounds = (int)(pairs / clusters);
    const int p0 = pl.rounds * clusters;  // first pair that is left
    long long total = 0;
    for (int i = p0 / per; i < groups; i++) total += (long long)tiles(i) * (per - std::max(p0 - i * per, 0));
    if (total > 0x7fffffffLL) return -1;
    // equal runs of at least CUT_COST tiles, or one run a pair
    const int equal = (int)std::min<long long>(clusters, std::max<long long>(1, total / CUT_COST));
    const bool cut = p0 < pairs && tiles(p0 / per) > total / equal + 2 * CUT_COST;
    pl.runs = cut ? equal : (int)(pairs - p0);
    pl.cuts = 0;
    int c = 0;
    long long u = 0;  // tiles before group i
    for (int i = p0 / per; i < groups; i++) {
        const int n = tiles(i), first = std::max(i * per, p0), held = (i + 1) * per - first;
        for (; c < pl.runs; c++) {
            const long long to = cut ? total * c / pl.runs : u + (long long)n * (p0 + c - first);
            if (to >= u + (long long)n * held) break;
            pl.item[c] = first + (int)(to - u) / n;
            pl.tile[c] = (int)(to - u) % n;
            pl.u[c] = (int)to;
            pl.cuts += pl.tile[c] > 0;
        }
        u += (long long)n * held;
    }
    for (; c <= MAX_RUNS; c++) {
        pl.item[c] = (int)pairs;
        pl.tile[c] = 0;
        pl.u[c] = (int)total;
    }
    if (pl.rounds == 0) pl.clusters = pl.runs;
    return 0;
}

}  // namespace

size_t paged_prompt_workspace(int nkv) {
    return (size_t)2 * nkv * TAIL * HD * sizeof(uint16_t) +
           (size_t)MAX_RUNS * 4 * QT * (HD * sizeof(float) + sizeof(float2));
}

int launch_paged_prompt(const void *q, const void *gate, const void *k_pages, const void *v_pages,
                        const PagePool &pool, const int *table, int max_pages, int s0, int window,
                        int sinks, void *out, void *workspace, int T, int nq, cudaStream_t st,
                        char *err, size_t errlen) {
    const int ps = 1 << pool.ps_log, nkv = pool.nkv;
    PromptArgs a{};
    a.gate = (const uint16_t *)gate;
    a.table = table;
    a.out = (uint16_t *)out;
    a.rec_o = (float *)workspace;
    a.rec_ml = (float2 *)(a.rec_o + (size_t)MAX_RUNS * 4 * QT * HD);
    uint16_t *tail = (uint16_t *)(a.rec_ml + (size_t)MAX_RUNS * 4 * QT);
    uint16_t *tail_v = tail + (size_t)nkv * TAIL * HD;
    const uint64_t rows = (uint64_t)pool.n_pages * nkv * ps;
    CUtensorMap mq, mk, mv, mtk, mtv;
    // V as [64-dim block][slot][64 dims]: a copy brings a chunk's two blocks one after the
    // other (one block for pages of 16 slots, half a chunk's rows)
    if (make_tmap_bf16_3d(&mq, q, HD, nq, T, HD * 2, (uint64_t)nq * HD * 2, 64, 1, QT, err, errlen) ||
        make_tmap_bf16_2d(&mk, k_pages, rows, HD, HD * 2, 64, std::min(ps, 64), err, errlen) ||
        make_tmap_bf16_3d(&mv, v_pages, 64, rows, HD / 64, HD * 2, 128, 64, std::min(ps, 32),
                          ps >= 32 ? 2 : 1, err, errlen) ||
        make_tmap_bf16_2d(&mtk, tail, (uint64_t)nkv * TAIL, HD, HD * 2, 64, TAIL, err, errlen) ||
        make_tmap_bf16_3d(&mtv, tail_v, 64, (uint64_t)nkv * TAIL, HD / 64, HD * 2, 128, 64, 32, 2,
                          err, errlen))
        return -1;
    a.pool = pool;
    a.max_pages = max_pages;
    a.s0 = s0;
    a.T = T;
    a.nq = nq;
    a.window = window;
    a.sinks = sinks;
    a.by_heads = nq / nkv % 2 == 0;
    if (make_plan(a.plan, std::min(num_sms() / 2, MAX_RUNS), s0, T, nq, a.by_heads, window, sinks))
        return fail(err, errlen, "vx27_gqa_paged_prefill: T=%d over %d slots: over 2^31 tiles", T, s0);
    const size_t smem = sizeof(Smem) + 1024;
    if (ensure_smem_attr((const void *)paged_prompt_k, smem, err, errlen)) return -1;
    VX_CK(launch_pdl(prompt_tail_k, dim3((2 * nkv * TAIL + 7) / 8), dim3(256), 0, st,
                     (const uint16_t *)k_pages, (const uint16_t *)v_pages, tail, pool, table, s0,
                     s0 + T, window, sinks, dev_status()));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * a.plan.clusters));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    VX_CK(cudaLaunchKernelEx(&cfg, paged_prompt_k, mq, mk, mv, mtk, mtv, a, dev_status()));
    if (a.plan.cuts)
        VX_CK(launch_pdl(prompt_join_k, dim3(QT / 16, 2, a.plan.runs - 1), dim3(256), 0, st, a));
    return 0;
}

}  // namespace vx27
