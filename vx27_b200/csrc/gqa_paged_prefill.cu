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
// Only key tiles with a slot that some row of the pair sees are gone through: the sinks'
// tiles, then those from the first row's window on; masks are applied on tiles that some row
// sees in part. Within a tile the copies fetch page by page; a box without a seen slot reads
// past the pool instead, which fills it with zeros, so freed pages are not touched. The last
// 64-slot block, whose end nothing has written, comes from a zero-padded copy (prompt_tail_k).
//
// What bounds it: the tensor cores and the softmax warps that feed them (4 T_keys 128 256 FLOP
// per row tile); K and V come from L2, which the heads of a KV head share.
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
// tensor memory: S at [0, 128), O at [128, 384), P as bf16 pairs at [384, 512), two buffers
constexpr uint32_t TM_O = 128, TM_P = 384;

struct Smem {
    uint8_t q[4][QT * 128];
    uint8_t ring[NK + NV][CHUNK];  // K slots, then V slots
    float xmax[2][2][QT], xsum[2][QT];
    uint64_t qfull, full[NK + NV], empty[NK + NV], s_full, s_empty, p_full[2], pv_done[2],
        o_final, mma_done, qk_done;
    int pages[2][2][KT / 16];  // K and V: of the tile being copied and of the next one
    uint32_t tmem_base;
    int abort;
};
static_assert(sizeof(Smem) + 1024 <= 232448, "smem");

struct PromptArgs {
    const uint16_t *gate;
    const int *table;
    uint16_t *out;
    PagePool pool;
    int max_pages, s0, T, nq, window, sinks, by_heads;
};

__device__ __forceinline__ bool try_wait(uint32_t addr, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; "
        "selp.u32 %0, 1, 0, p; }"
        : "=r"(ok) : "r"(addr), "r"(parity) : "memory");
    return ok;
}
__device__ __forceinline__ bool test_wait(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; "
        "selp.u32 %0, 1, 0, p; }"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
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
    __device__ KeyTiles(int a, int e, int window, int sinks) {
        const SeenSlots first(a + 1, window, sinks);
        lo = first.win_begin;
        sink_end = first.sink_end;
        win0 = lo / KT;
        sink_tiles = min((sink_end + KT - 1) / KT, win0);
        n = sink_tiles + (e + KT - 1) / KT - win0;
    }
    __device__ int slot0(int m) const { return (m < sink_tiles ? m : win0 + m - sink_tiles) * KT; }
    // does some row see a slot of [s, s + len)? (up to the pair's end, which the caller knows)
    __device__ bool seen(int s, int len) const { return s + len > lo || s < sink_end; }
};

// Softmax, rescale and result of this CTA's 128 rows.
__device__ __forceinline__ void softmax_role(Smem &sm, const Sync &sy, const PromptArgs &a,
                                             const KeyTiles &kt, uint32_t tmem, int warp, int lane,
                                             int h, int t0) {
    const uint32_t tO = tmem + TM_O;
    const int q4 = warp & 3, hf = (warp - 2) >> 2, r = q4 * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
    const int qpos = a.s0 + t0 + r;
    const float sc2 = 1.4426950408889634f * 0.0625f;  // log2(e) / sqrt(256)
    // tiles from full0 on to full1 are seen whole by every row of the tile
    const int full1 = a.s0 + t0 - (KT - 1);
    const int full0 = a.window ? a.s0 + t0 + QT - a.window : 0;
    const int row_lo = a.window ? qpos - a.window : -1;  // slots above it are in the window
    float m_run = -INFINITY, l_run = 0.0f;
    bool ok = true;
    for (int j = 0; j < kt.n; j++) {
        const int b = j & 1;
        if (ok) ok = sy.wait(&sm.s_full, j & 1, VX_DEV_TIMEOUT_MMA);
        ok = __all_sync(0xffffffffu, ok);
        constexpr int HK = KT / 2;
        float s[HK];
        float mloc = -INFINITY;
        if (ok) {
            tc_fence_after();
            tmem_ld64(tmem + lane_off + hf * HK, s);
            tc_fence_before();
            sy.arrive(&sm.s_empty);
            const int s0 = kt.slot0(j), k0 = s0 + hf * HK;
            if (s0 > full1 || s0 < full0) {
#pragma unroll
                for (int c = 0; c < HK; c++)
                    if (k0 + c > qpos || (k0 + c <= row_lo && k0 + c >= a.sinks)) s[c] = -INFINITY;
            }
            float mx[16];
#pragma unroll
            for (int i = 0; i < 16; i++)
                mx[i] = fmaxf(fmaxf(s[4 * i], s[4 * i + 1]), fmaxf(s[4 * i + 2], s[4 * i + 3]));
#pragma unroll
            for (int w = 8; w >= 1; w >>= 1)
#pragma unroll
                for (int i = 0; i < w; i++) mx[i] = fmaxf(mx[i], mx[i + w]);
            mloc = mx[0];
        }
        sm.xmax[b][hf][r] = mloc;  // the two threads of a row meet here
        named_bar_sync(1, 256);
        const float mpart = sm.xmax[b][hf ^ 1][r];
        if (!ok) continue;
        const float mt = fmaxf(mloc, mpart) * sc2;
        float alpha = 1.0f;
        const bool grow = mt > m_run + RESCALE_LOG2;
        if (grow) {
            alpha = (m_run == -INFINITY) ? 0.0f : exp2f(m_run - mt);
            m_run = mt;
        }
        // a row that has seen nothing yet has O = 0, and nothing to rescale
        if (__any_sync(0xffffffffu, grow && alpha > 0.0f)) {
            ok = sy.wait(&sm.pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1, VX_DEV_TIMEOUT_MMA);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) continue;
            tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < HD / 32; i++) {
                float o[16];
                const uint32_t ta = tO + lane_off + hf * (HD / 2) + 16 * i;
                tmem_ld16(ta, o);
#pragma unroll
                for (int e = 0; e < 16; e++) o[e] *= alpha;
                tmem_st16(ta, o);
            }
        }
        // P buffer b is free once O += P(j-2) V(j-2) is done
        if (j >= 2) {
            ok = sy.wait(&sm.pv_done[b], ((j >> 1) - 1) & 1, VX_DEV_TIMEOUT_MMA);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) continue;
            tc_fence_after();
        }
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
    sm.xsum[hf][r] = l_run;
    named_bar_sync(1, 256);
    const float l_row = l_run + sm.xsum[hf ^ 1][r];
    // the result by 32 columns, in a loop that is not unrolled (its code is shared by all of
    // the row's columns), the gate requested one round ahead; its sigmoid uses the SFU's 2^x
    // and reciprocal
    const int t_row = t0 + r;
    const size_t base = ((size_t)t_row * a.nq + h) * HD + hf * (HD / 2);
    const bool gated = a.gate && t_row < a.T;
    uint4 gate[4], next[4];
    auto request = [&](int i) {
        const uint4 *gp = reinterpret_cast<const uint4 *>(a.gate + base) + 4 * i;
#pragma unroll
        for (int k = 0; k < 4; k++) next[k] = gp[k];
    };
    if (gated) request(0);
    if (ok) ok = sy.wait(&sm.o_final, 0, VX_DEV_TIMEOUT_MMA);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) {
        *(volatile int *)sy.abort = 1;
        return;
    }
    tc_fence_after();
    const float inv = 1.0f / l_row;
#pragma unroll 1
    for (int i = 0; i < HD / 64; i++) {
        float o[32];
        tmem_ld16(tO + lane_off + hf * (HD / 2) + 32 * i, o);
        tmem_ld16(tO + lane_off + hf * (HD / 2) + 32 * i + 16, o + 16);
        if (t_row >= a.T) continue;
#pragma unroll
        for (int k = 0; k < 4; k++) gate[k] = next[k];
        if (gated && i < HD / 64 - 1) request(i + 1);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = o[8 * k + e] * inv;
            if (gated) {
                const uint32_t gw[4] = {gate[k].x, gate[k].y, gate[k].z, gate[k].w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[2 * e] *= __fdividef(1.0f, 1.0f + __expf(-bf16_to_f32(gw[e] & 0xffffu)));
                    x[2 * e + 1] *= __fdividef(1.0f, 1.0f + __expf(-bf16_to_f32(gw[e] >> 16)));
                }
            }
            st8_bf16(a.out + base + 32 * i + 8 * k, x);
        }
    }
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
    const int nkv = a.pool.nkv, pr = (int)(blockIdx.x >> 1);
    int h, t0, ta, tb;  // this CTA's head and first row; the pair's rows [ta, tb)
    if (a.by_heads) {
        const int per = a.nq >> 1, n_t = (a.T + QT - 1) / QT;
        h = 2 * (pr % per) + (int)rank;
        ta = t0 = (n_t - 1 - pr / per) * QT;  // the tiles with most keys first
        tb = min(a.T, ta + QT);
    } else {
        const int n_t = (a.T + 2 * QT - 1) / (2 * QT);
        h = pr % a.nq;
        ta = (n_t - 1 - pr / a.nq) * 2 * QT;
        t0 = ta + QT * (int)rank;
        tb = min(a.T, ta + 2 * QT);
    }
    const int kvh = h / (a.nq / nkv);
    const KeyTiles kt(a.s0 + ta, a.s0 + tb, a.window, a.sinks);

    if (tid == 0) {
        mbar_init(&sm.qfull, 1);
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
        auto fetch = [&](int m) {
            if (!leads || m >= kt.n) return;
            const int s = kt.slot0(m) + rel;
            if (s >= tail0 || !kt.seen(s, box)) return;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;"
                         ::"r"(smem_u32(&sm.pages[!is_k][m & 1][lane])),
                         "l"(a.table + (s >> a.pool.ps_log)) : "memory");
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        const int slots = is_k ? NK : NV, ring0 = is_k ? 0 : NK;
        const uint32_t full0 = mapa_shared(&sm.full[ring0], 0);
        fetch(0);
        if (is_k && lane == 0) {
            if (rank == 0) mbar_arrive_expect_tx(&sm.qfull, 2 * 4 * QT * 128);
            const uint32_t lq = mapa_shared(&sm.qfull, 0);
            for (int c = 0; c < 4; c++) tma_load_3d_pair(sm.q[c], &tmq, c * 64, h, t0, lq);
        }
        bool ok = true;
        int n = 0, sl = 0;        // chunks issued; the next one's ring slot
        uint32_t phase = 1;       // of its empty barrier (the first round waits for nothing)
        for (int m = 0; m < kt.n && ok; m++) {
            asm volatile("cp.async.wait_all;" ::: "memory");
            const int s = kt.slot0(m) + rel;
            const bool tail = s >= tail0;
            bool issue = leads;
            int y = none;
            if (leads && tail) {  // the padded block (64 slots of K, 32 of V at a time), or zeros
                issue = is_k ? lane == 0 : (lane & 1) == 0;
                y = kvh * TAIL + s - tail0;
                if (s >= tail0 + TAIL) y = nkv * TAIL;
            } else if (leads && kt.seen(s, box)) {
                const int page = sm.pages[!is_k][m & 1][lane];
                if (a.pool.has(page)) y = (int)a.pool.row(page, kvh, s);
                else dev_flag(status, VX_DEV_BAD_ARG);
            }
            fetch(m + 1);
            const CUtensorMap *map = is_k ? (tail ? &tmtk : &tmk) : (tail ? &tmtv : &tmv);
            const bool halves = !is_k && !tail && ps == 16;  // V boxes of 16 slots, one block each
            const int off = is_k ? lane * 2048 : halves ? (lane & 1) * 2048 : 0;
            for (int c = 0; c < 4; c++) {
                uint64_t *empty = &sm.empty[ring0 + sl];
                if (n >= slots && !test_wait(empty, phase)) ok = sy.wait(empty, phase, VX_DEV_TIMEOUT_TMA);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0 && rank == 0) mbar_arrive_expect_tx(&sm.full[ring0 + sl], 2 * CHUNK);
                uint8_t *dst = sm.ring[ring0 + sl] + off;
                const uint32_t bar = full0 + 8 * sl;
                if (is_k) {  // dims [64 c, 64 c + 64)
                    if (issue) tma_load_2d_pair(dst, map, c * 64, y, bar);
                } else if (issue && (lane >> 1) == c) {  // slots [32 c, ..), two blocks of 64 dims
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
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (rank == 0) {  // every copy of both CTAs lands before this CTA can leave
            for (int i = max(0, n - slots); i < n; i++)
                drain(&sm.full[ring0 + i % slots], (i / slots) & 1);
            if (is_k) drain(&sm.qfull, 0);
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
            bool ok = sy.wait(&sm.qfull, 0, VX_DEV_TIMEOUT_TMA);
            for (int m = 0; m < kt.n && ok; m++) {
                if (m >= 1) ok = sy.wait(&sm.s_empty, (m - 1) & 1, VX_DEV_TIMEOUT_MMA);
                for (int c = 0; c < 4 && ok; c++) {
                    const uint32_t i = 4u * m + c, sl = i % NK;
                    ok = sy.wait(&sm.full[sl], (i / NK) & 1, VX_DEV_TIMEOUT_TMA);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t dq = sdesc_add(dq0, c * (QT * 128));
                    const uint64_t dk = sdesc_add(dr0, sl * CHUNK);
#pragma unroll
                    for (int kk = 0; kk < 4; kk++)
                        mma_bf16_pair(tmem, sdesc_add(dq, kk * 32), sdesc_add(dk, kk * 32), id1,
                                      (c | kk) != 0);
                    mma_commit_pair_both(&sm.empty[sl]);
                }
                if (!ok) break;
                mma_commit_pair_both(&sm.s_full);
            }
            mma_commit_pair(mapa_shared(&sm.qk_done, 0));
            drain(&sm.qk_done, 0);
        }
    } else if (warp == O_WARP) {
        if (lane == 0 && rank == 0) {  // ---- O += P(t) V(t)
            const uint32_t id2 = idesc_bf16(256, HD, false, true);
            const uint64_t dv0 = sdesc_sw128(smem_u32(sm.ring[0]), 32 * 128, 1024);
            bool ok = true;
            for (int t = 0; t < kt.n && ok; t++) {
                const int pb = t & 1;
                ok = sy.wait(&sm.p_full[pb], (t >> 1) & 1, VX_DEV_TIMEOUT_MMA);
                for (int c = 0; c < 4 && ok; c++) {
                    const uint32_t i = 4u * t + c, sl = NK + i % NV;
                    ok = sy.wait(&sm.full[sl], (i / NV) & 1, VX_DEV_TIMEOUT_TMA);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t dv = sdesc_add(dv0, sl * CHUNK);
#pragma unroll
                    for (int k2 = 0; k2 < 2; k2++) {
                        const int kk = 2 * c + k2;
                        mma_bf16_pair_ts(tO, tmem + TM_P + 64u * pb + 8u * kk,
                                         sdesc_add(dv, k2 * 2048), id2, (t > 0 || kk > 0) ? 1u : 0u);
                    }
                    mma_commit_pair_both(&sm.empty[sl]);
                }
                if (!ok) break;
                mma_commit_pair_both(&sm.pv_done[pb]);
                if (t == kt.n - 1) mma_commit_pair_both(&sm.o_final);
            }
            mma_commit_pair(mapa_shared(&sm.mma_done, 0));
            drain(&sm.mma_done, 0);
        }
    } else {
        softmax_role(sm, sy, a, kt, tmem, warp, lane, h, t0);
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

}  // namespace

size_t paged_prompt_workspace(int nkv) { return (size_t)2 * nkv * TAIL * HD * sizeof(uint16_t); }

int launch_paged_prompt(const void *q, const void *gate, const void *k_pages, const void *v_pages,
                        const PagePool &pool, const int *table, int max_pages, int s0, int window,
                        int sinks, void *out, void *workspace, int T, int nq, cudaStream_t st,
                        char *err, size_t errlen) {
    const int ps = 1 << pool.ps_log, nkv = pool.nkv;
    uint16_t *tail = (uint16_t *)workspace, *tail_v = tail + (size_t)nkv * TAIL * HD;
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
    PromptArgs a{};
    a.gate = (const uint16_t *)gate;
    a.table = table;
    a.out = (uint16_t *)out;
    a.pool = pool;
    a.max_pages = max_pages;
    a.s0 = s0;
    a.T = T;
    a.nq = nq;
    a.window = window;
    a.sinks = sinks;
    a.by_heads = nq / nkv % 2 == 0;
    const long long pairs = a.by_heads ? (long long)(nq / 2) * ((T + QT - 1) / QT)
                                       : (long long)nq * ((T + 2 * QT - 1) / (2 * QT));
    if (pairs > 0x3fffffffLL)
        return fail(err, errlen, "vx27_gqa_paged_prefill: bad shape T=%d nq=%d", T, nq);
    const size_t smem = sizeof(Smem) + 1024;
    if (ensure_smem_attr((const void *)paged_prompt_k, smem, err, errlen)) return -1;
    VX_CK(launch_pdl(prompt_tail_k, dim3((2 * nkv * TAIL + 7) / 8), dim3(256), 0, st,
                     (const uint16_t *)k_pages, (const uint16_t *)v_pages, tail, pool, table,
                     s0, s0 + T, window, sinks, dev_status()));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * pairs));
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
    return 0;
}

}  // namespace vx27
