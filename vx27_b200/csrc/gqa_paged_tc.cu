// Decode attention over the paged KV cache on the tensor cores (include/vx27_paged.h).
//
// The seen slots of the whole batch are counted in tiles of 128 aligned slots, sequence by
// sequence and KV head by KV head, and cut into P equal runs, one per CTA (P = the SM
// count): a run holds whole (sequence, KV head) items and at most two cut ones. Lengths are
// on the device, so every CTA finds its run by a scan over them. A whole item is finished
// by its CTA (gate and rounding included); a cut one leaves a record (o / l, m, l) per part,
// which the join kernel merges. The run, not the number of sequences or their lengths,
// decides a CTA's work: with one CTA per item or a fixed split per sequence a ragged batch
// waits for its longest.
//
// Per tile:  S^T[128 x N] = K[128 x 256] Q^T       (tcgen05, tensor memory, fp32)
//            p = 2^(s - m), one thread per slot, running maximum m per head
//            O^T[256 x N] = V^T[256 x 128] P^T     folded into fp32 registers
// The N columns hold each head of the group TERMS times: q (and p) split into bf16 terms,
// x = hi + mid (+ lo), whose products with the bf16 cache are exact in fp32. Two terms carry
// 16 bits (bf16 output), three 24 (fp32 output, weight sums).
//
// What bounds it: the cache bytes, 128 KB per tile through two rings of 6 chunks of 16 KB (128
// slots x 64 dims) per SM, one for K and one for V, each with a copying and a multiplying warp
// of its own. 128 sequences of 2112 slots (1.1 GB) take 177-180 us, 0.94-0.95 of the copy
// rate (0.84 with one ring, one copying and one multiplying warp, where a wait for K holds up
// V); 128 ragged ones 174. About 15 us of a call are its ends, whatever the size: the scan of
// the lengths 2 us, the first data 4, the last tile's products and rows 4, the join 3, and
// with the memory busy the last CTA ends 4-8% after the middle one. (Handing the last 3-8% of the
// tiles out late, to CTAs that start where others end, cost more than that: 107 us instead of 99
// for 64 sequences.) Short sequences are bound by the chain of each item through the warps:
// 256 of 100 slots take 38 us (48 with q and the results in one warp).
// A page is a box of its own: boxes of min(page_size, 128) rows where all of them are seen,
// else boxes of the 16-row groups with a seen slot. The O MMAs take 16 slots each and leave
// the other groups out; unseen rows of a copied group are zeroed.
//
// Warps: 0 copies K and 7 copies V (lane i: rows 16 i .. of the tile; page ids come a tile
// ahead), 1 issues the S MMAs and 8 the O MMAs, 2-5 softmax and accumulation, 6 q, 9-11 gate
// and results. Waits are bounded (2 s).
#include <math.h>
#include <algorithm>
#include "common.cuh"
#include "paged.cuh"
#include "tc.cuh"
#include "gqa_paged.cuh"

namespace vx27 {
namespace {

constexpr int HD = PG_HD;
constexpr int TILE = 128;
constexpr int NK = 6, NV = 6;      // ring slots; NV even: a V operand is two neighbouring chunks
constexpr int CHUNK = 16384;       // 128 slots x 64 dims, 128-byte swizzle
constexpr int THREADS = 384;
constexpr int SM_WARP0 = 2, Q_WARP = 6, V_WARP = 7, O_WARP = 8;  // 0: K copies, 1: S MMAs
constexpr int OUT_WARP0 = 9, OUT_WARPS = 3;
constexpr int JOIN_MAX = 1024;     // runs at most (records of one item)
constexpr int RUN_LENS = 128;      // lengths kept in shared memory

__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ bool bar_test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; "
        "selp.u32 %0, 1, 0, p; }"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool bar_try(uint32_t addr, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; "
        "selp.u32 %0, 1, 0, p; }"
        : "=r"(ok) : "r"(addr), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded wait: false when the CTA has aborted or 2 s have passed (then it aborts). Only the
// first try is inlined: the roles' loops share the instruction cache, and with the whole wait
// in each of them (and 64-bit divisions in their walks) a third of the warps' time went by
// waiting for instructions.
__device__ __noinline__ bool bar_wait_long(uint32_t addr, uint32_t parity, int *abort,
                                           uint32_t *status, uint32_t code) {
    const uint64_t t0 = now_ns();
    for (;;) {
        if (bar_try(addr, parity)) return true;
        if (*(volatile int *)abort) return false;
        if (now_ns() - t0 > 2000000000ull) break;
    }
    *(volatile int *)abort = 1;
    dev_flag(status, code);
    return false;
}
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, int *abort,
                                         uint32_t *status, uint32_t code) {
    const uint32_t addr = smem_u32(bar);
    return bar_try(addr, parity) || bar_wait_long(addr, parity, abort, status, code);
}
// (a b + add) / c, a quotient that fits 32 bits.
__device__ __noinline__ int mul_div(int a, int b, int c, int add = 0) {
    const unsigned long long x = (unsigned long long)a * b + add;
    return (int)(x >> 32 ? x / c : (unsigned)x / (unsigned)c);
}
// Bounded wait that goes on after an abort: what must be done before the CTA may leave.
__device__ __forceinline__ void bar_drain(uint64_t *bar, uint32_t parity) {
    for (int it = 0; it < (1 << 20); it++)
        if (bar_test(bar, parity)) return;
}
// N consecutive fp32 columns of this thread's tensor-memory lane, one wait.
template <int N>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, float (&v)[N]) {
    if constexpr (N == 32) {
        uint32_t r[32];
#pragma unroll
        for (int k = 0; k < 2; k++)
            asm volatile(
                "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,"
                "%12,%13,%14,%15}, [%16];"
                : "=r"(r[16 * k]), "=r"(r[16 * k + 1]), "=r"(r[16 * k + 2]), "=r"(r[16 * k + 3]),
                  "=r"(r[16 * k + 4]), "=r"(r[16 * k + 5]), "=r"(r[16 * k + 6]),
                  "=r"(r[16 * k + 7]), "=r"(r[16 * k + 8]), "=r"(r[16 * k + 9]),
                  "=r"(r[16 * k + 10]), "=r"(r[16 * k + 11]), "=r"(r[16 * k + 12]),
                  "=r"(r[16 * k + 13]), "=r"(r[16 * k + 14]), "=r"(r[16 * k + 15])
                : "r"(taddr + 16 * k));
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
    } else {
        tmem_ld16(taddr, v);
    }
}
// The largest value of the warp (the sm_100a reduction over fp32; NaN loses).
__device__ __forceinline__ float warp_max_redux(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// Byte offset of element (row, col) of a K-major operand in 128-byte swizzled rows.
__device__ __forceinline__ uint32_t sw128(int row, int col) {
    return (uint32_t)(row * 128 + ((((col >> 3) ^ (row & 7)) & 7) << 4) + (col & 7) * 2);
}

template <int G, int TERMS>
struct Smem {
    static constexpr int ROWS = (G * TERMS + 7) / 8 * 8;    // operand rows held
    static constexpr int N = (G * TERMS + 15) / 16 * 16;    // MMA columns (rows past ROWS are
                                                            // whatever follows, and not used)
    static constexpr int QB = TERMS == 2 ? 2 : 1;           // q buffers
    uint8_t ring[NK + NV][CHUNK];    // K slots, then V slots
    uint8_t q[QB][4][ROWS * 128];    // 4 chunks of 64 dims
    uint8_t p[2][2][ROWS * 128];     // 2 chunks of 64 slots
    float ob[G][HD];                 // an item's normalised rows, for the staging warp
    uint64_t full[NK + NV], empty[NK + NV];
    uint64_t s_full[2], s_empty[2], p_full[2], o_full[2], o_empty[2], v_ok[2], q_full[QB], q_empty[QB];
    uint64_t grp[2], grp_end[2], ob_full, ob_empty, mma_done[2];
    float red_max[2][4][G], red_sum[2][4][G];
    float ml[G][2];
    int pages[2][2][8];              // K and V: of the tile being copied and of the next one
    int scan[THREADS / 32];          // start: the warps' tiles
    int run_b, run_off;              // start: the run's first sequence, its tiles before the run
    int lens[RUN_LENS];              // of the run's first sequences
    float m_fin[2][G];
    uint32_t tmem_base;
    int abort;
};
static_assert(sizeof(Smem<8, 2>) + 1024 <= 232448 && sizeof(Smem<8, 3>) + 1024 <= 232448, "smem");

// Tiles that sequence b's slots are seen in, per KV head; the sink tiles first.
struct SeqTiles {
    SeenSlots see;
    int sink_tiles, win_tile0, tiles;
    __device__ SeqTiles(int n, int window, int sinks) : see(n, window, sinks) {
        win_tile0 = see.win_begin / TILE;
        sink_tiles = min((see.sink_end + TILE - 1) / TILE, win_tile0);
        tiles = sink_tiles + (n + TILE - 1) / TILE - win_tile0;
    }
    __device__ int first_slot(int v) const {                // of the v-th tile
        return (v < sink_tiles ? v : win_tile0 + v - sink_tiles) * TILE;
    }
    // 16-slot groups of the tile at s0 that hold a slot of [from, to)
    __device__ static uint32_t groups(int s0, int from, int to) {
        from = max(from - s0, 0);
        to = min(to - s0, TILE);
        return from < to ? (2u << ((to - 1) >> 4)) - (1u << (from >> 4)) : 0u;
    }
    __device__ uint32_t seen_groups(int s0) const {
        return groups(s0, see.win_begin, see.n) | groups(s0, 0, see.sink_end);
    }
};

// Length of sequence b, clipped to its table.
__device__ __forceinline__ int seq_len(const DecodeArgs &a, int b) {
    return min(max(a.lens[b], 0), a.max_pages << a.pool.ps_log);
}

// A CTA's run: items (b, h), each with its tiles [v0, v0 + cnt). Sequences without slots are
// not met. The lengths of the first ones are in shared memory (with the memory busy a load
// takes as long as one or two tiles).
struct Walk {
    const DecodeArgs &a;
    const int *lens;
    int run_b, left;  // first sequence; tiles to go, the item's included
    int b, h, v0, cnt;
    SeqTiles t;
    __device__ __forceinline__ SeqTiles seq() const {
        const int i = b - run_b;
        return SeqTiles(i < RUN_LENS ? lens[i] : seq_len(a, b), a.window, a.sinks);
    }
    __device__ __forceinline__ Walk(const DecodeArgs &a_, const int *lens_, int run_b_, int off,
                                    int left_)
        : a(a_), lens(lens_), run_b(run_b_), left(left_), b(run_b_), h(0), v0(off), cnt(0),
          t(left_ > 0 ? seq() : SeqTiles(0, 0, 0)) {
        if (left > 0) {
            h = off / t.tiles;
            v0 = off % t.tiles;
            cnt = min(t.tiles - v0, left);
        }
    }
    __device__ __forceinline__ bool done() const { return left <= 0; }
    __device__ __forceinline__ bool whole() const { return cnt == t.tiles; }
    __device__ __forceinline__ void next() {
        left -= cnt;
        v0 = 0;
        if (left <= 0) return;
        if (++h == a.pool.nkv) {
            h = 0;
            do {
                b++;
                t = seq();
            } while (t.tiles == 0);
        }
        cnt = min(t.tiles, left);
    }
};

template <int G, int TERMS>
__global__ void __launch_bounds__(THREADS, 1)
paged_decode_tc(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                const __grid_constant__ CUtensorMap tmk16,
                const __grid_constant__ CUtensorMap tmv16, const __grid_constant__ DecodeArgs a,
                uint32_t *status) {
    extern __shared__ uint8_t smem_raw[];
    using Sm = Smem<G, TERMS>;
    Sm &sm = *reinterpret_cast<Sm *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    constexpr int N = Sm::N, QB = Sm::QB;
    constexpr uint32_t TM_COLS = N == 16 ? 128 : 256, TM_O = 2 * N;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nkv = a.pool.nkv;

    if (tid == 0) {
        for (int i = 0; i < NK + NV; i++) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.s_empty[i], 128);
            mbar_init(&sm.p_full[i], 128);
            mbar_init(&sm.v_ok[i], 1);
            mbar_init(&sm.o_full[i], 1);
            mbar_init(&sm.o_empty[i], 128);
            mbar_init(&sm.grp[i], 128);
            mbar_init(&sm.grp_end[i], 128);
        }
        for (int i = 0; i < QB; i++) {
            mbar_init(&sm.q_full[i], 32);
            mbar_init(&sm.q_empty[i], 1);
        }
        mbar_init(&sm.ob_full, 128);
        mbar_init(&sm.ob_empty, OUT_WARPS);
        mbar_init(&sm.mma_done[0], 1);
        mbar_init(&sm.mma_done[1], 1);
        sm.abort = 0;
        fence_barrier_init();
    }
    if (warp == 0) {
        tmem_alloc(&sm.tmem_base, TM_COLS);
        tmem_relinquish();
        if (lane == 0) {
            tma_prefetch_desc(&tmk);
            tma_prefetch_desc(&tmv);
        }
    }
    if (warp >= SM_WARP0 && warp < Q_WARP) {  // operand rows that no term fills stay zero
        uint4 *z = reinterpret_cast<uint4 *>(&sm.q[0][0][0]);
        for (int e = tid - 64; e < (int)(sizeof(sm.q) + sizeof(sm.p)) / 16; e += 128)
            z[e] = make_uint4(0, 0, 0, 0);
        fence_proxy_async();
    }
    grid_dep_wait();  // lengths, q, cache rows come from the kernels before
    if (tid == 0) grid_dep_launch();

    // ---- the run of this CTA: tiles [c T / P, (c + 1) T / P) of the T in all ------------
    const int cb = (a.B + THREADS - 1) / THREADS;  // consecutive sequences per thread
    const int b_lo = min(tid * cb, a.B), b_hi = min(b_lo + cb, a.B);
    int mine = 0, n0 = 0;  // tiles of the thread's sequences; the first one's length
    for (int b = b_lo; b < b_hi; b++) {
        const int n = a.lens[b], nc = min(max(n, 0), a.max_pages << a.pool.ps_log);
        if (n != nc) dev_flag(status, VX_DEV_BAD_ARG);
        if (b == b_lo) n0 = nc;
        mine += SeqTiles(nc, a.window, a.sinks).tiles * nkv;
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) sm.scan[warp] = incl;
    __syncthreads();
    int before = incl - mine, total = 0;
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < warp) before += sm.scan[w];
        total += sm.scan[w];
    }
    const int P = min((int)gridDim.x, total), c = blockIdx.x;
    const int begin = c < P ? mul_div(c, total, P) : 0, end = c < P ? mul_div(c + 1, total, P) : 0;
    if (begin < end && begin >= before && begin < before + mine) {
        int b = b_lo, at = before;
        for (; cb > 1; b++) {
            const int k = SeqTiles(seq_len(a, b), a.window, a.sinks).tiles * nkv;
            if (begin < at + k) break;
            at += k;
        }
        sm.run_b = b;
        sm.run_off = begin - at;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;
    const int run_b = begin < end ? sm.run_b : 0;
    if (cb == 1) {  // thread b has the length of sequence b
        if (tid >= run_b && tid < run_b + RUN_LENS) sm.lens[tid - run_b] = n0;
    } else if (tid < RUN_LENS && run_b + tid < a.B) {
        sm.lens[tid] = seq_len(a, run_b + tid);
    }
    __syncthreads();
    const Walk start(a, sm.lens, run_b, begin < end ? sm.run_off : 0, end - begin);
    // the run that holds tile u
    auto owner = [&](int u) { return mul_div(u + 1, P, total, -1); };

    if (warp == 0 || warp == V_WARP) {
        // ---- copies of K (warp 0) and of V: lane i < 8 has rows [16 i, 16 i + 16) of a tile ----
        const bool is_k = warp == 0;
        const int ring0 = is_k ? 0 : NK, slots = is_k ? NK : NV;
        const int seg = min(1 << a.pool.ps_log, TILE) / 16;  // lanes of a page's share
        const uint32_t seg_mask = (1u << seg) - 1;
        const int lead = lane & ~(seg - 1);
        // The page of this lane's rows of tile v of the walk's item goes to shared memory by an
        // asynchronous copy, a tile ahead (a load into a register is waited for at once where
        // it leaves its branch).
        auto fetch = [&](const Walk &w, int v, int g) {
            if (w.done() || lane >= 8) return;
            const int s0 = w.t.first_slot(v);
            if ((w.t.seen_groups(s0) >> lane) & 1)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;"
                             ::"r"(smem_u32(&sm.pages[!is_k][g & 1][lane])),
                             "l"(a.table + (size_t)w.b * a.max_pages +
                                 ((s0 + 16 * lane) >> a.pool.ps_log)) : "memory");
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        // V rows of copied groups that are not seen may hold anything, and 0 * NaN is NaN: once
        // the tile has landed they are zeroed. Until then the tile is due (its slots, 1 due).
        bool due = false, ok = true;
        int due_g = 0, due_s0 = 0;
        SeenSlots due_see(0, 0, 0);
        auto landed = [&]() {
            const int j = 4 * due_g + (lane & 3);
            return (bool)__all_sync(0xffffffffu, bar_test(&sm.full[NK + j % NV], (j / NV) & 1));
        };
        // V(g) may be multiplied once it has landed. It is copied over V(g - 1)'s first half, so
        // v_ok(g - 2), on the same barrier, is over.
        auto v_done = [&](int g) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.v_ok[g & 1]);
        };
        auto zero_edges = [&]() {
#pragma unroll 1
            for (int e = 0; e < 3; e++) {  // the groups that n, the window or the sinks end in
                const int at = e == 0 ? due_see.n : e == 1 ? due_see.win_begin : due_see.sink_end;
                if ((at & 15) == 0 || at < due_s0 || at >= due_s0 + TILE) continue;
                for (int i = lane >> 3; i < 16; i += 4) {
                    const int slot = (at & ~15) + i;
                    if (due_see.sees(slot)) continue;
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        *reinterpret_cast<uint4 *>(sm.ring[NK + (4 * due_g + k) % NV] +
                                                   (slot - due_s0) * 128 + (lane & 7) * 16) =
                            make_uint4(0, 0, 0, 0);
                }
            }
            due = false;
            v_done(due_g);
        };
        // Waits for a ring slot (bar), or for the due tile (NULL); a due tile may land meanwhile.
        auto wait_for = [&](uint64_t *bar, uint32_t parity) {
            if (!due)
                return !bar || (bool)__all_sync(0xffffffffu, bar_wait(bar, parity, &sm.abort, status,
                                                                      VX_DEV_TIMEOUT_TMA));
            const uint64_t t0 = now_ns();
            for (;;) {
                if (due && landed()) zero_edges();
                if (bar ? (bool)__all_sync(0xffffffffu, bar_test(bar, parity)) : !due) return true;
                bool stop = *(volatile int *)&sm.abort;
                if (now_ns() - t0 > 2000000000ull) {
                    *(volatile int *)&sm.abort = 1;
                    dev_flag(status, VX_DEV_TIMEOUT_TMA);
                    stop = true;
                }
                if (__any_sync(0xffffffffu, stop)) return false;
            }
        };
        Walk w = start;
        int v = w.done() ? 0 : w.v0, g = 0, j = 0;  // tiles and chunks of this ring so far
        fetch(w, v, 0);
        for (; !w.done() && ok; g++) {
            const int s0 = w.t.first_slot(v), h = w.h;
            const SeenSlots see = w.t.see;
            const uint32_t seen = w.t.seen_groups(s0);
            asm volatile("cp.async.wait_all;" ::: "memory");
            const int page = lane < 8 ? sm.pages[!is_k][g & 1][lane] : 0;
            const bool want = (seen >> lane) & 1, need = want && a.pool.has(page);
            if (want && !need) dev_flag(status, VX_DEV_BAD_ARG);
            const uint32_t mask = __ballot_sync(0xffffffffu, need);
            const bool big = ((mask >> lead) & seg_mask) == seg_mask;
            const bool issue = need && (!big || lane == lead);
            const int y = need ? (int)a.pool.row(page, h, s0 + 16 * lane) : 0;
            const uint32_t bytes = __popc(mask) * 2048;
            if (++v == w.v0 + w.cnt) {
                w.next();
                v = w.done() ? 0 : w.v0;
            }
            fetch(w, v, g + 1);
            const CUtensorMap *map = is_k ? (big ? &tmk : &tmk16) : (big ? &tmv : &tmv16);
            for (int r = 0; r < 4; r++, j++) {
                const int slot = ring0 + j % slots, round = j / slots;
                if (round > 0) ok = wait_for(&sm.empty[slot], (round - 1) & 1);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(&sm.full[slot], bytes);
                __syncwarp();
                if (issue) tma_load_2d(sm.ring[slot] + lane * 2048, map, r * 64, y, &sm.full[slot]);
            }
            if (is_k || !ok) continue;
            ok = wait_for(nullptr, 0);
            auto cuts = [&](int at) { return (at & 15) && at > s0 && at < s0 + TILE; };
            if (!cuts(see.n) && !cuts(see.win_begin) && !cuts(see.sink_end)) {
                v_done(g);
            } else {
                due = true;
                due_g = g;
                due_s0 = s0;
                due_see = see;
            }
        }
        if (ok) wait_for(nullptr, 0);
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (*(volatile int *)&sm.abort) {  // copies in flight land before the CTA leaves
            for (int k = max(0, j - slots); k < j; k++)
                bar_drain(&sm.full[ring0 + k % slots], (k / slots) & 1);
        }
    } else if (warp == 1) {
        // ---- S(g) = K(g) Q^T, as the softmax frees its buffer and K lands --------------------
        if (lane == 0) {
            const uint32_t id = idesc_bf16(128, N, false, false);
            const uint64_t dk0 = sdesc_sw128(smem_u32(sm.ring[0]), 16, 1024);
            const uint64_t dq0 = sdesc_sw128(smem_u32(sm.q[0][0]), 16, 1024);
            bool ok = true;
            int g = 0, kq = 0, sl = 0;
            uint32_t phase = 0;
            Walk w = start;
            for (; !w.done() && ok; w.next(), kq++) {
                const uint64_t dq = sdesc_add(dq0, (kq % QB) * (uint32_t)sizeof(sm.q[0]));
                ok = bar_wait(&sm.q_full[kq % QB], (kq / QB) & 1, &sm.abort, status, VX_DEV_TIMEOUT_MMA);
                for (int i = 0; i < w.cnt && ok; i++, g++) {
                    const int bb = g & 1;
                    if (g >= 2)
                        ok = bar_wait(&sm.s_empty[bb], ((g >> 1) - 1) & 1, &sm.abort, status,
                                      VX_DEV_TIMEOUT_MMA);
                    for (int c = 0; c < 4 && ok; c++) {
                        ok = bar_wait(&sm.full[sl], phase, &sm.abort, status, VX_DEV_TIMEOUT_TMA);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t dk = sdesc_add(dk0, sl * CHUNK);
                        const uint64_t dqc = sdesc_add(dq, c * (Sm::ROWS * 128));
#pragma unroll
                        for (int kk = 0; kk < 4; kk++)
                            mma_bf16(tmem + bb * N, sdesc_add(dk, kk * 32), sdesc_add(dqc, kk * 32), id,
                                     (c | kk) != 0);
                        mma_commit(&sm.empty[sl]);
                        if (++sl == NK) {
                            sl = 0;
                            phase ^= 1;
                        }
                    }
                    if (ok) mma_commit(&sm.s_full[bb]);
                }
                if (ok) mma_commit(&sm.q_empty[kq % QB]);
            }
            mma_commit(&sm.mma_done[0]);
            bar_drain(&sm.mma_done[0], 0);  // also after an abort
        }
    } else if (warp == O_WARP) {
        // ---- O(g) = V(g)^T P(g)^T, half by half as P is written and V lands -------------------
        if (lane == 0) {
            const uint32_t id = idesc_bf16(128, N, true, false);
            const uint64_t dv0 = sdesc_sw128(smem_u32(sm.ring[NK]), CHUNK, 1024);
            const uint64_t dp0 = sdesc_sw128(smem_u32(sm.p[0][0]), 16, 1024);
            bool ok = true;
            int g = 0, sl = 0;
            uint32_t phase = 0;
            Walk w = start;
            for (; !w.done() && ok; w.next()) {
                for (int i = 0; i < w.cnt && ok; i++, g++) {
                    const int bb = g & 1;
                    const uint32_t seen = w.t.seen_groups(w.t.first_slot(w.v0 + i));
                    const uint64_t dp = sdesc_add(dp0, bb * (uint32_t)sizeof(sm.p[0]));
                    if (g >= 2)
                        ok = bar_wait(&sm.o_empty[bb], ((g >> 1) - 1) & 1, &sm.abort, status,
                                      VX_DEV_TIMEOUT_MMA);
                    ok = ok && bar_wait(&sm.p_full[bb], (g >> 1) & 1, &sm.abort, status, VX_DEV_TIMEOUT_MMA);
                    ok = ok && bar_wait(&sm.v_ok[bb], (g >> 1) & 1, &sm.abort, status, VX_DEV_TIMEOUT_TMA);
                    for (int ho = 0; ho < 2 && ok; ho++) {
                        ok = bar_wait(&sm.full[NK + sl], phase, &sm.abort, status, VX_DEV_TIMEOUT_TMA) &&
                             bar_wait(&sm.full[NK + sl + 1], phase, &sm.abort, status, VX_DEV_TIMEOUT_TMA);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t dv = sdesc_add(dv0, sl * CHUNK);
                        const uint32_t d = tmem + TM_O + (bb * 2 + ho) * N;
                        uint32_t acc = 0;
#pragma unroll 2
                        for (int kk = 0; kk < 8; kk++) {  // the 16-slot groups with a seen slot
                            if (!((seen >> kk) & 1)) continue;
                            mma_bf16(d, sdesc_add(dv, kk * 2048),
                                     sdesc_add(dp, (kk >> 2) * (Sm::ROWS * 128) + (kk & 3) * 32), id, acc);
                            acc = 1;
                        }
                        mma_commit(&sm.empty[NK + sl]);
                        mma_commit(&sm.empty[NK + sl + 1]);
                        if ((sl += 2) == NV) {
                            sl = 0;
                            phase ^= 1;
                        }
                    }
                    if (ok) mma_commit(&sm.o_full[bb]);
                }
            }
            mma_commit(&sm.mma_done[1]);
            bar_drain(&sm.mma_done[1], 0);
        }
    } else if (warp < Q_WARP) {
        // ---- softmax: thread = slot r of the tile; then output dims r and r + 128 ----------
        const int q4 = warp & 3, r = q4 * 32 + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)(q4 * 32) << 16);
        const float sc2 = 1.4426950408889634f * 0.0625f;  // log2(e) / sqrt(256)
        bool ok = true;
        int g = 0, kq = 0;  // tiles and items so far
        float m2[G], l[G], acc_a[G], acc_b[G], al[G], al_prev[G];
        auto reset = [&]() {
#pragma unroll
            for (int h = 0; h < G; h++) {
                m2[h] = -INFINITY;
                l[h] = 0.f;
            }
        };
#pragma unroll
        for (int h = 0; h < G; h++) acc_a[h] = acc_b[h] = al[h] = al_prev[h] = 0.f;
        reset();
        auto fold = [&](int t) {  // O(t), with the rescale of its tile
            const int bb = t & 1;
            ok = ok && bar_wait(&sm.o_full[bb], (t >> 1) & 1, &sm.abort, status, VX_DEV_TIMEOUT_MMA);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) return;
            tc_fence_after();
            auto half = [&](int ho, float (&acc)[G]) {
                float o[N];
                tmem_ld_cols(lane_addr + TM_O + (bb * 2 + ho) * N, o);
#pragma unroll
                for (int h = 0; h < G; h++) {
                    float x = o[h + (TERMS - 1) * G];
#pragma unroll
                    for (int k = TERMS - 2; k >= 0; k--) x += o[h + k * G];  // small terms first
                    acc[h] = fmaf(acc[h], al_prev[h], x);
                }
            };
            half(0, acc_a);
            half(1, acc_b);
            tc_fence_before();
            mbar_arrive(&sm.o_empty[bb]);
        };
        // An item ends in two steps: its sums and maxima go to shared memory (close) before the
        // next item's first tile uses the registers, its rows to the output buffer (finish)
        // after that tile's P is written: the wait for the last O does not hold the next S up.
        auto close = [&](int k) {
            const int eb = k & 1;
#pragma unroll
            for (int h = 0; h < G; h++) {
                const float t = warp_sum(l[h]);
                if (lane == 0) sm.red_sum[eb][q4][h] = t;
                if (r == 0) sm.m_fin[eb][h] = m2[h];
            }
            mbar_arrive(&sm.grp_end[eb]);
            reset();
        };
        auto finish = [&](int k) {
            const int eb = k & 1;
            ok = bar_wait(&sm.grp_end[eb], (k >> 1) & 1, &sm.abort, status, VX_DEV_TIMEOUT_MMA) && ok;
            if (k > 0)
                ok = bar_wait(&sm.ob_empty, (k - 1) & 1, &sm.abort, status, VX_DEV_TIMEOUT_MMA) && ok;
            ok = __all_sync(0xffffffffu, ok);
#pragma unroll
            for (int h = 0; h < G; h++) {
                const float L = sm.red_sum[eb][0][h] + sm.red_sum[eb][1][h] +
                                sm.red_sum[eb][2][h] + sm.red_sum[eb][3][h];
                const float inv = 1.0f / L;
                sm.ob[h][r] = acc_a[h] * inv;
                sm.ob[h][r + 128] = acc_b[h] * inv;
                acc_a[h] = acc_b[h] = 0.f;
                if (r == 0) {
                    sm.ml[h][0] = sm.m_fin[eb][h];
                    sm.ml[h][1] = L;
                }
            }
            mbar_arrive(&sm.ob_full);
        };
        Walk w = start;
        for (int i = 0;;) {  // tile i of the item; after the last tile once more, to finish it
            const bool last = w.done(), ended = i == 0 && g > 0;
            const int bb = g & 1;
            if (ended) close(kq - 1);
            if (!last) {
                ok = bar_wait(&sm.s_full[bb], (g >> 1) & 1, &sm.abort, status, VX_DEV_TIMEOUT_MMA);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                float s[N], x[G];
                tmem_ld_cols(lane_addr + bb * N, s);
                tc_fence_before();
                mbar_arrive(&sm.s_empty[bb]);
                const bool valid = w.t.see.sees(w.t.first_slot(w.v0 + i) + r);
#pragma unroll
                for (int h = 0; h < G; h++) {
                    float t = s[h + (TERMS - 1) * G];
#pragma unroll
                    for (int k = TERMS - 2; k >= 0; k--) t += s[h + k * G];
                    x[h] = valid ? t * sc2 : -INFINITY;
                    t = warp_max_redux(x[h]);
                    if (lane == 0) sm.red_max[bb][q4][h] = t;
                }
                mbar_arrive(&sm.grp[bb]);  // all four warps' maxima
                if constexpr (TERMS == 3)
                    if (a.scores && valid) {  // [G][slots] of the item, for the weight sums
                        float *sc = a.scores + (size_t)(w.b * nkv + w.h) * G * a.score_stride +
                                    (w.v0 + i) * TILE + r;
#pragma unroll
                        for (int h = 0; h < G; h++) sc[(size_t)h * a.score_stride] = x[h];
                    }
                ok = bar_wait(&sm.grp[bb], (g >> 1) & 1, &sm.abort, status, VX_DEV_TIMEOUT_MMA);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                uint8_t *pbuf = sm.p[bb][r >> 6];
#pragma unroll
                for (int h = 0; h < G; h++) {
                    const float t = fmaxf(fmaxf(sm.red_max[bb][0][h], sm.red_max[bb][1][h]),
                                          fmaxf(sm.red_max[bb][2][h], sm.red_max[bb][3][h]));
                    const float mn = fmaxf(m2[h], t);
                    al[h] = ex2_approx(m2[h] - mn);
                    m2[h] = mn;
                    x[h] = ex2_approx(x[h] - mn);
                    l[h] = fmaf(l[h], al[h], x[h]);
                }
#pragma unroll
                for (int k = 0; k < TERMS; k++)
#pragma unroll
                    for (int h = 0; h < G; h += 2) {  // two heads per conversion
                        const int h1 = h + 1 < G ? h + 1 : h;
                        const uint32_t t = pack_bf16x2(x[h], x[h1]);
                        *reinterpret_cast<uint16_t *>(pbuf + sw128(h + k * G, r & 63)) = (uint16_t)t;
                        x[h] -= bf16_to_f32(t & 0xffffu);
                        if (h1 > h) {
                            *reinterpret_cast<uint16_t *>(pbuf + sw128(h1 + k * G, r & 63)) =
                                (uint16_t)(t >> 16);
                            x[h1] -= __uint_as_float(t & 0xffff0000u);
                        }
                    }
                fence_proxy_async();
                mbar_arrive(&sm.p_full[bb]);
            }
            if (g > 0) fold(g - 1);
            if (ended) finish(kq - 1);
            if (last || !ok) break;
#pragma unroll
            for (int h = 0; h < G; h++) al_prev[h] = al[h];
            g++;
            if (++i == w.cnt) {
                i = 0;
                kq++;
                w.next();
            }
        }
    } else if (warp == Q_WARP) {
        // ---- q, split into terms --------------------------------------------------------------
        if (lane == 0) {
            // an item that began in an earlier run is joined by the block of its second run
            int4 j = make_int4(-1, 0, 0, 0);
            if (!start.done() && start.v0 > 0) {
                const int c1 = owner(begin - start.v0), c2 = owner(begin - start.v0 + start.t.tiles - 1);
                if (c == c1 + 1) j = make_int4(start.b * nkv + start.h, c1, c2, 0);
            }
            a.join[c] = j;
        }
        const int d0 = 8 * lane;
        bool ok = true;
        int kq = 0;
        for (Walk w = start; !w.done(); w.next(), kq++) {
            float x[G][8];
#pragma unroll
            for (int h = 0; h < G; h++)
                ld8_f32(x[h], a.q + ((size_t)w.b * a.nq + w.h * G + h) * HD + d0);
            if (kq >= QB)  // the S MMAs of the item that used the buffer before are complete
                ok = bar_wait(&sm.q_empty[kq % QB], ((kq - QB) / QB) & 1, &sm.abort, status,
                              VX_DEV_TIMEOUT_MMA);
            if (!__all_sync(0xffffffffu, ok)) break;
            uint8_t *dst = sm.q[kq % QB][d0 >> 6];
#pragma unroll
            for (int h = 0; h < G; h++)
#pragma unroll
                for (int k = 0; k < TERMS; k++) {
                    uint32_t wd[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        wd[e] = pack_bf16x2(x[h][2 * e], x[h][2 * e + 1]);
                        x[h][2 * e] -= bf16_to_f32(wd[e] & 0xffffu);
                        x[h][2 * e + 1] -= bf16_to_f32(wd[e] >> 16);
                    }
                    *reinterpret_cast<uint4 *>(dst + sw128(h + k * G, d0 & 63)) =
                        make_uint4(wd[0], wd[1], wd[2], wd[3]);
                }
            fence_proxy_async();
            mbar_arrive(&sm.q_full[kq % QB]);
        }
    } else {
        // ---- results: warp OUT_WARP0 + i has heads i, i + OUT_WARPS, .. of the group -----------
        constexpr int HW = (G + OUT_WARPS - 1) / OUT_WARPS;
        const int h0 = warp - OUT_WARP0, d0 = 8 * lane;
        bool ok = true;
        int kq = 0;
        for (Walk w = start; !w.done(); w.next(), kq++) {
            const size_t base = ((size_t)w.b * a.nq + w.h * G) * HD + d0;
            const bool whole = w.whole();
            float gv[HW][8], o[HW][8];
            if (whole && a.gate) {
#pragma unroll
                for (int u = 0; u < HW; u++) {
                    const int h = h0 + u * OUT_WARPS;
                    if (h >= G) break;
                    if (a.gate_bf16) ld8_bf16(gv[u], static_cast<const uint16_t *>(a.gate) + base + h * HD);
                    else ld8_f32(gv[u], static_cast<const float *>(a.gate) + base + h * HD);
                }
            }
            ok = bar_wait(&sm.ob_full, kq & 1, &sm.abort, status, VX_DEV_TIMEOUT_MMA);
            if (!__all_sync(0xffffffffu, ok)) break;
            // the buffer is free once it is in registers (an arrival after the global stores
            // waits for them)
#pragma unroll
            for (int u = 0; u < HW; u++)
                if (h0 + u * OUT_WARPS < G) ld8_f32(o[u], &sm.ob[h0 + u * OUT_WARPS][d0]);
            const float2 ml = lane < G ? make_float2(sm.ml[lane][0], sm.ml[lane][1]) : make_float2(0, 0);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.ob_empty);
            const size_t rec = (size_t)(2 * c + (w.v0 > 0 ? 0 : 1)) * G;
            const int item = w.b * nkv + w.h;
#pragma unroll
            for (int u = 0; u < HW; u++) {
                const int h = h0 + u * OUT_WARPS;
                if (h >= G) break;
                if (!whole) {
                    st8_f32(a.rec_o + (rec + h) * HD + d0, o[u]);
                } else {
                    if (a.gate)
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            o[u][e] *= __fdividef(1.0f, 1.0f + __expf(-gv[u][e]));
                    if (a.out_bf16) st8_bf16(static_cast<uint16_t *>(a.out) + base + h * HD, o[u]);
                    else st8_f32(static_cast<float *>(a.out) + base + h * HD, o[u]);
                }
            }
            if (h0 == 0 && lane < G) {
                if (!whole) a.rec_ml[rec + lane] = ml;
                else if (a.scores) a.item_ml[(size_t)item * G + lane] = ml;
            }
            // which runs hold the item, for the weight sums
            if (h0 == 0 && lane == 0 && a.scores && w.v0 == 0)
                a.span[item] = make_int2(c, owner(end - w.left + w.t.tiles - 1));
        }
    }
    __syncwarp();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, TM_COLS);
    }
}

// ---- join and weight sums ---------------------------------------------------------------
// Blocks [0, B): zeros for a sequence without slots. Then (P - 1) G blocks: (c, h) merges head
// h of the item that run c continues, if c is the second run of it: o = sum_r w_r o_r / sum_r
// w_r, w_r = l_r 2^(m_r - m). The other blocks add the weights of 1024 slots of an item: sum_h
// 2^(s_h - m_h) / l_h.
// Nothing but round trips and instructions bound it. The first two records of an item are those
// of runs c - 1 and c, so they are requested along with the plan. Items of more records take 38
// more of them in the first round trip (FEW: at most an eighth as many items as runs), or 4, in
// fewer registers; what is left after that comes four at a time. Replayed from a graph, one
// sequence of 8192 slots (37 runs an item) takes 17.3 us in all with FEW and 19.2 without, 4 of
// them 34.3 and 34.0, 8 of 2112 21.4 and 20.3, 16 of them 37.1 and 35.3. The lengths are on the
// device, so the rule counts lanes: one such sequence among 64 lanes takes 20.7, with FEW 18.0.
// WEIGHTS is an instance of its own, whose registers the others need not have; sums are read and
// written four at a time, requested with the scores (32 ragged sequences 62.5 us in all, 65.7
// with scalar sums added at the end, 56 without sums). Their blocks, and the scores, are as many
// as the tables' slots need: the same call with tables of 65536 slots takes 69 us, of 262144 94.
template <bool FEW, bool WEIGHTS>
__global__ void __launch_bounds__(256, FEW ? 3 : WEIGHTS ? 4 : 5)
paged_join_k(const __grid_constant__ DecodeArgs a, int P, int G, int slot_blocks) {
    grid_dep_wait();
    __shared__ float w_s[JOIN_MAX];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n_join = (P - 1) * G, blk = (int)blockIdx.x - a.B;
    if (blk < 0) {
        if (a.lens[blockIdx.x] > 0) return;
        for (int i = tid; i < a.nq * HD; i += 256) {
            const size_t at = (size_t)blockIdx.x * a.nq * HD + i;
            if (a.out_bf16) act_st<true>(a.out, at, 0.f);
            else act_st<false>(a.out, at, 0.f);
        }
        return;
    }
    // records of runs c1 .. c2: the first is that run's last item, the others first items
    auto rec_of = [](int c1, int r) { return (size_t)(r == 0 ? 2 * c1 + 1 : 2 * (c1 + r)); };
    if (blk < n_join) {
        const int c = blk / G + 1, h = blk % G;
        const float *ro = a.rec_o + (size_t)(2 * c - 1) * G * HD + h * HD + tid;
        const float2 *rm = a.rec_ml + (size_t)(2 * c - 1) * G + h;
        const float v0 = ro[0], v1 = ro[G * HD];
        const float2 ml0 = rm[0], ml1 = rm[G];
        const int4 j = a.join[c];
        if (j.x < 0) return;
        const int n = j.z - j.y + 1;
        const size_t i = ((size_t)(j.x / a.pool.nkv) * a.nq + (j.x % a.pool.nkv) * G + h) * HD + tid;
        const float g = !a.gate ? 0.f : a.gate_bf16 ? act_ld<true>(a.gate, i) : act_ld<false>(a.gate, i);
        float L, O;
        if (n == 2) {
            const float m = fmaxf(ml0.x, ml1.x);
            const float w0 = ml0.y * exp2f(ml0.x - m), w1 = ml1.y * exp2f(ml1.x - m);
            L = w0 + w1;
            O = fmaf(w1, v1, w0 * v0);
        } else {
            constexpr int RU = FEW ? 38 : 4;
            ro += (size_t)G * HD;  // record r >= 1 of the item is at 2 (r - 1) records from here
            rm += G;
            float v[RU];
#pragma unroll
            for (int u = 0; u < RU; u++) v[u] = u + 2 < n ? ro[(u + 1) * 2 * G * HD] : 0.f;
            float m = fmaxf(ml0.x, ml1.x);  // every warp makes it
            for (int r = 2 + lane; r < n; r += 32) m = fmaxf(m, rm[(size_t)(r - 1) * 2 * G].x);
            m = warp_max(m);
            for (int r = 2 + tid; r < n; r += 256) {
                const float2 ml = rm[(size_t)(r - 1) * 2 * G];
                w_s[r] = ml.y * exp2f(ml.x - m);
            }
            const float w0 = ml0.y * exp2f(ml0.x - m), w1 = ml1.y * exp2f(ml1.x - m);
            L = w0 + w1;
            O = fmaf(w1, v1, w0 * v0);
            __syncthreads();
#pragma unroll
            for (int u = 0; u < RU; u++) {
                const float wr = u + 2 < n ? w_s[u + 2] : 0.f;
                L += wr;
                O = fmaf(wr, v[u], O);
            }
#pragma unroll 4
            for (int r = RU + 2; r < n; r++) {
                L += w_s[r];
                O = fmaf(w_s[r], ro[(size_t)(r - 1) * 2 * G * HD], O);
            }
        }
        float o = O / L;
        if (a.gate) o *= 1.0f / (1.0f + expf(-g));
        if (a.out_bf16) act_st<true>(a.out, i, o);
        else act_st<false>(a.out, i, o);
        return;
    }
    if constexpr (!WEIGHTS) return;
    // 4 slots a thread; their scores and sums are requested before the statistics, which warp h
    // makes for head h
    const int bi = blk - n_join, item = bi / slot_blocks, k0 = (bi % slot_blocks) * 1024 + 4 * tid;
    const SeqTiles t(seq_len(a, item / a.pool.nkv), a.window, a.sinks);
    if ((bi % slot_blocks) * 1024 >= t.tiles * TILE) return;
    const int slot = t.first_slot(k0 / TILE) + k0 % TILE;
    const bool seen[4] = {t.see.sees(slot), t.see.sees(slot + 1), t.see.sees(slot + 2), t.see.sees(slot + 3)};
    const bool any = k0 < t.tiles * TILE && (seen[0] || seen[1] || seen[2] || seen[3]);
    const float *sc = a.scores + (size_t)item * G * a.score_stride + k0;
    float4 *ws = reinterpret_cast<float4 *>(a.wsum + (size_t)item * ((size_t)a.max_pages << a.pool.ps_log) +
                                            slot);
    const float4 old = any ? *ws : make_float4(0, 0, 0, 0);
    float4 x[8];
#pragma unroll
    for (int h = 0; h < 8; h++)
        x[h] = h < G && any ? *reinterpret_cast<const float4 *>(sc + (size_t)h * a.score_stride)
                            : make_float4(0, 0, 0, 0);
    __shared__ float2 ml_s[8];
    if (warp < G) {
        const int2 span = a.span[item];
        const int n = span.y - span.x + 1;
        float2 ml = make_float2(-INFINITY, 0.f);
        if (n == 1) {
            ml = a.item_ml[(size_t)item * G + warp];
        } else {
            for (int r = lane; r < n; r += 32)
                ml.x = fmaxf(ml.x, a.rec_ml[rec_of(span.x, r) * G + warp].x);
            ml.x = warp_max(ml.x);
            for (int r = lane; r < n; r += 32) {
                const float2 e = a.rec_ml[rec_of(span.x, r) * G + warp];
                ml.y = fmaf(e.y, exp2f(e.x - ml.x), ml.y);
            }
            ml.y = warp_sum(ml.y);
        }
        if (lane == 0) ml_s[warp] = make_float2(ml.x, 1.0f / ml.y);
    }
    __syncthreads();
    float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int h = 0; h < 8; h++) {
        if (h >= G) break;
        const float2 ml = ml_s[h];
        sum.x = fmaf(exp2f(x[h].x - ml.x), ml.y, sum.x);
        sum.y = fmaf(exp2f(x[h].y - ml.x), ml.y, sum.y);
        sum.z = fmaf(exp2f(x[h].z - ml.x), ml.y, sum.z);
        sum.w = fmaf(exp2f(x[h].w - ml.x), ml.y, sum.w);
    }
    if (any)
        *ws = make_float4(seen[0] ? old.x + sum.x : old.x, seen[1] ? old.y + sum.y : old.y,
                          seen[2] ? old.z + sum.z : old.z, seen[3] ? old.w + sum.w : old.w);
}

}  // namespace

int paged_decode_parts(int n_parts) {
    if (n_parts <= 0) n_parts = num_sms();
    return std::min(n_parts, JOIN_MAX);
}

// Slots that an item's scores may take: the table's, or the sinks' and the window's tiles.
static size_t score_slots(int max_slots, int window, int sinks) {
    const long long all = ((long long)max_slots + TILE - 1) / TILE;
    if (!window) return (size_t)all * TILE;
    const long long w = ((long long)window + TILE - 1) / TILE + 1 + ((long long)sinks + TILE - 1) / TILE;
    return (size_t)std::min(all, w) * TILE;
}

size_t paged_decode_layout(DecodeArgs &a, void *workspace, int B, int nq, int nkv, int max_slots,
                           int window, int sinks, bool weights, int P) {
    const size_t G = nq / nkv;
    char *p = (char *)workspace;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        char *at = p ? p + off : nullptr;
        off += (bytes + 15) & ~(size_t)15;
        return at;
    };
    a.join = (int4 *)take((size_t)P * sizeof(int4));
    a.rec_o = (float *)take((size_t)2 * P * G * HD * sizeof(float));
    a.rec_ml = (float2 *)take((size_t)2 * P * G * sizeof(float2));
    a.scores = nullptr;
    a.score_stride = 0;
    if (weights) {
        a.span = (int2 *)take((size_t)B * nkv * sizeof(int2));
        a.item_ml = (float2 *)take((size_t)B * nq * sizeof(float2));
        a.score_stride = score_slots(max_slots, window, sinks);
        a.scores = (float *)take((size_t)B * nq * a.score_stride * sizeof(float));
    }
    return off;
}

int launch_paged_decode(const DecodeArgs &a, const void *k_pages, const void *v_pages, int P,
                        cudaStream_t st, char *err, size_t errlen) {
    const uint64_t rows = (uint64_t)a.pool.n_pages * a.pool.nkv << a.pool.ps_log;
    const uint32_t box = std::min(1 << a.pool.ps_log, TILE);
    CUtensorMap mk, mv, mk16, mv16;
    if (make_tmap_bf16_2d(&mk, k_pages, rows, HD, HD * 2, 64, box, err, errlen) ||
        make_tmap_bf16_2d(&mv, v_pages, rows, HD, HD * 2, 64, box, err, errlen) ||
        make_tmap_bf16_2d(&mk16, k_pages, rows, HD, HD * 2, 64, 16, err, errlen) ||
        make_tmap_bf16_2d(&mv16, v_pages, rows, HD, HD * 2, 64, 16, err, errlen))
        return -1;
    const int G = a.nq / a.pool.nkv;
    const int slot_blocks = a.scores ? (int)((a.score_stride + 1023) / 1024) : 0;
    const long long blocks = a.B + (long long)(P - 1) * G + (long long)slot_blocks * a.B * a.pool.nkv;
    if (blocks > 0x7fffffffLL)
        return fail(err, errlen, "vx27_gqa_paged_decode: weight sums over %d sequences of %zu slots",
                    a.B, a.score_stride);
    const bool three = !a.out_bf16 || a.scores;
#define VX_D(G_, T_)                                                                          \
    {                                                                                         \
        const size_t smem = sizeof(Smem<G_, T_>) + 1024;                                      \
        if (ensure_smem_attr((const void *)paged_decode_tc<G_, T_>, smem, err, errlen))       \
            return -1;                                                                        \
        VX_CK(launch_pdl(paged_decode_tc<G_, T_>, dim3(P), dim3(THREADS), smem, st, mk, mv, mk16, \
                         mv16, a, dev_status()));                                             \
    }
#define VX_G(G_) \
    case G_: if (three) VX_D(G_, 3) else VX_D(G_, 2) break;
    switch (G) {
        VX_G(1) VX_G(2) VX_G(3) VX_G(4) VX_G(5)
        VX_G(6) VX_G(7) VX_G(8)
    }
#undef VX_G
#undef VX_D
    const bool few = 8LL * a.B * a.pool.nkv < P;
    auto join = a.scores ? (few ? paged_join_k<true, true> : paged_join_k<false, true>)
                         : (few ? paged_join_k<true, false> : paged_join_k<false, false>);
    VX_CK(launch_pdl(join, dim3((unsigned)blocks), dim3(256), 0, st, a, P, G, slot_blocks));
    return 0;
}

}  // namespace vx27
