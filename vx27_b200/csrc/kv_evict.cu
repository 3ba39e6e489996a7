// Eviction from the paged KV cache (include/vx27_paged.h): per (sequence, KV head) the first
// sinks slots, the last recent ones and the middle slots with the largest weight sums stay.
//   evict_select_k   the kept slots in order (kept, weight_sum_out, lens_out): one CTA per
//                    (KV head, sequence) finds the smallest kept sum by a radix select over
//                    the order-preserving bits, 11 at a time, then compacts the slots above it
//   evict_copy_k     the kept K and V rows to their new pages, one warp per row pair
#include <math.h>
#include <algorithm>
#include "common.cuh"
#include "paged.cuh"
#include "../../include/vx27_paged.h"

namespace vx27 {
namespace {

constexpr int SEL_THREADS = 1024;

struct EvictArgs {
    uint16_t *kp, *vp;
    const int *table, *table_out, *lens;
    const float *wsum;
    float *wsum_out;
    int *lens_out, *kept;
    PagePool pool;
    int max_pages, max_pages_out, keep, sinks, recent, B;
};

// Unsigned integers in the order of the floats, -0 as +0 and NaN as -infinity.
__device__ __forceinline__ uint32_t sum_key(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Length of sequence b, clipped to what its table can hold.
__device__ __forceinline__ int seq_len(const EvictArgs &a, int b, uint32_t *status) {
    const int n = a.lens[b], cap = a.max_pages << a.pool.ps_log;
    if (n < 0 || n > cap) {
        dev_flag(status, VX_DEV_BAD_ARG);
        return n < 0 ? 0 : cap;
    }
    return n;
}

// Inclusive scan over the warp.
__device__ __forceinline__ int warp_scan(int x, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// Four slots a thread and round; 11 bits of the threshold a pass, counted in shared memory.
// Bytes do not bound it: three passes over a row that the L1 holds, the barriers between them
// and the compaction's round per 4096 slots do. With the copy, one sequence cut from 5001 slots
// to 2048 takes 15 us (8 bits a pass, four passes: 18), 64 sequences of up to 4163 cut to 1024
// take 96 us (113); sums that are all alike, and so one bin, take as long. Long sequences are
// bound by one load in flight a thread, four passes of n / 4096 rounds: 65536 slots cut to 4096
// take 69 us, 262144 take 232 (the copy's bytes are 5 of them).
__global__ void __launch_bounds__(SEL_THREADS)
evict_select_k(const __grid_constant__ EvictArgs a, uint32_t *status) {
    grid_dep_wait();
    grid_dep_launch();
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = seq_len(a, b, status), m = min(n, a.keep);
    const size_t bh = (size_t)b * a.pool.nkv + h;
    const float *ws = a.wsum + bh * ((size_t)a.max_pages << a.pool.ps_log);
    const int cap_out = a.max_pages_out << a.pool.ps_log;
    float *wo = a.wsum_out + bh * cap_out;
    int *kept = a.kept + bh * a.keep;
    if (h == 0 && tid == 0) a.lens_out[b] = m;
    for (int j = m + tid; j < cap_out; j += SEL_THREADS) wo[j] = 0.0f;
    for (int j = m + tid; j < a.keep; j += SEL_THREADS) kept[j] = -1;
    if (n <= a.keep) {
        for (int j = tid; j < m; j += SEL_THREADS) {
            kept[j] = j;
            wo[j] = ws[j];
        }
        return;
    }
    const int lo = a.sinks, hi = n - a.recent;
    int want = a.keep - a.sinks - a.recent;  // of the hi - lo middle slots; fewer than all
    const bool any = want > 0;
    constexpr int BINS = 2048, PER = BINS / SEL_THREADS;
    __shared__ int hist[BINS], sums[32], s_want;
    __shared__ uint32_t s_prefix;
    uint32_t prefix = 0;
    for (int pass = 0; any && pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;  // digits of 11, 11 and 10 bits
        const int bins = pass == 2 ? 1024 : 2048;
        const uint32_t above = pass == 0 ? 0 : 0xffffffffu << (pass == 1 ? 21 : 10);
        for (int i = tid; i < BINS; i += SEL_THREADS) hist[i] = 0;
        __syncthreads();
        for (int j0 = 0; j0 < n; j0 += 4 * SEL_THREADS) {
            const int j = j0 + 4 * tid;
            if (j >= n) continue;
            const float4 f = *reinterpret_cast<const float4 *>(ws + j);
            const float w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t k = sum_key(w[e]);
                if (j + e >= lo && j + e < hi && ((k ^ prefix) & above) == 0)
                    atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
            }
        }
        __syncthreads();
        // counts from the largest digit down: thread i has digits BINS - 1 - PER i - (0 .. PER - 1)
        int count[PER], mine = 0;
#pragma unroll
        for (int u = 0; u < PER; u++) mine += count[u] = hist[BINS - 1 - PER * tid - u];
        int incl = warp_scan(mine, lane);
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        const int part = warp_scan(sums[lane], lane);
        incl += warp ? __shfl_sync(0xffffffffu, part, warp - 1) : 0;
        int upto = incl - mine;
#pragma unroll
        for (int u = 0; u < PER; u++) {
            if (upto < want && upto + count[u] >= want) {  // one digit in all: the threshold's
                s_want = want - upto;
                s_prefix = prefix | ((uint32_t)(BINS - 1 - PER * tid - u) << shift);
            }
            upto += count[u];
        }
        __syncthreads();
        want = s_want;
        prefix = s_prefix;
    }
    // the slots above the threshold `prefix` stay, and the first `want` equal to it
    int base = 0, base_eq = 0;
    for (int j0 = 0; j0 < n; j0 += 4 * SEL_THREADS) {
        const int j = j0 + 4 * tid;
        const float4 f = j < n ? *reinterpret_cast<const float4 *>(ws + j) : make_float4(0, 0, 0, 0);
        const float w[4] = {f.x, f.y, f.z, f.w};
        uint32_t gt = 0, eq = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t k = sum_key(w[e]);
            const bool in = j + e < n, fixed = in && (j + e < lo || j + e >= hi);
            gt |= (uint32_t)(fixed || (in && any && k > prefix)) << e;
            eq |= (uint32_t)(in && !fixed && any && k == prefix) << e;
        }
        // up to 4096 of each a round: two counts in one word
        const int mine = __popc(gt) | (__popc(eq) << 16);
        const int incl = warp_scan(mine, lane);
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        const int part = warp_scan(sums[lane], lane);  // every warp, over the warps' sums
        const int upto = __shfl_sync(0xffffffffu, part, 31);
        const int warps = warp ? __shfl_sync(0xffffffffu, part, warp - 1) : 0;
        const int excl = warps + incl - mine;
        int rg = base + (excl & 0xffff), re = base_eq + (excl >> 16);  // before this slot
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool g = (gt >> e) & 1, q = (eq >> e) & 1;
            if (g || (q && re < want)) {
                const int at = rg + min(re, want);
                kept[at] = j + e;
                wo[at] = w[e];
            }
            rg += g;
            re += q;
        }
        base += upto & 0xffff;
        base_eq += upto >> 16;
        __syncthreads();
    }
}

__global__ void __launch_bounds__(256)
evict_copy_k(const __grid_constant__ EvictArgs a, uint32_t *status) {
    grid_dep_wait();
    const int lane = threadIdx.x & 31;
    const long long rows = (long long)a.B * a.pool.nkv * a.keep;
    for (long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; i < rows;
         i += ((long long)gridDim.x * blockDim.x) >> 5) {
        const int slot = a.kept[i];
        if (slot < 0) continue;
        const int j = (int)(i % a.keep);
        const long long bh = i / a.keep;
        const int h = (int)(bh % a.pool.nkv), b = (int)(bh / a.pool.nkv);
        const int src = a.table[(size_t)b * a.max_pages + (slot >> a.pool.ps_log)];
        const int dst = a.table_out[(size_t)b * a.max_pages_out + (j >> a.pool.ps_log)];
        if (!a.pool.has(src) || !a.pool.has(dst)) {
            dev_flag(status, VX_DEV_BAD_ARG);
            continue;
        }
        const size_t from = a.pool.row(src, h, slot) * PG_HD + lane * 8;
        const size_t to = a.pool.row(dst, h, j) * PG_HD + lane * 8;
        const uint4 k = *reinterpret_cast<const uint4 *>(a.kp + from);
        const uint4 v = *reinterpret_cast<const uint4 *>(a.vp + from);
        *reinterpret_cast<uint4 *>(a.kp + to) = k;
        *reinterpret_cast<uint4 *>(a.vp + to) = v;
    }
}

}  // namespace
}  // namespace vx27

using namespace vx27;

extern "C" int vx27_kv_evict(void *k_pages, void *v_pages, int n_pages, int page_size,
                             const int *page_table, int max_pages, const int *lens,
                             const float *weight_sum, const int *page_table_out,
                             int max_pages_out, int *lens_out, float *weight_sum_out, int *kept,
                             int keep, int sinks, int recent, int B, int nkv, int hd,
                             void *stream, char *err, size_t errlen) {
    const char *fn = "vx27_kv_evict";
    if (check_pool(fn, k_pages, v_pages, n_pages, page_size, page_table, max_pages, nkv, hd, err,
                   errlen))
        return -1;
    if (B <= 0 || B > 65535) return fail(err, errlen, "%s: B=%d", fn, B);
    if (keep <= 0 || sinks < 0 || recent < 0 || (long long)sinks + recent > keep)
        return fail(err, errlen, "%s: keep=%d with sinks=%d and recent=%d", fn, keep, sinks, recent);
    if (max_pages_out <= 0 || (long long)max_pages_out * page_size < keep ||
        (long long)max_pages_out * page_size > 0x7fffffffLL - 256)
        return fail(err, errlen, "%s: %d pages of %d slots for keep=%d", fn, max_pages_out,
                    page_size, keep);
    if (!lens || !weight_sum || !page_table_out || !lens_out || !weight_sum_out || !kept)
        return fail(err, errlen, "%s: null pointer argument", fn);
    if ((uintptr_t)weight_sum & 15)
        return fail(err, errlen, "%s: weight_sum must be 16-byte aligned", fn);
    if (page_table_out == page_table || lens_out == lens || weight_sum_out == weight_sum ||
        k_pages == v_pages)
        return fail(err, errlen, "%s: an output is an input (eviction is not in place)", fn);
    EvictArgs a{};
    a.kp = (uint16_t *)k_pages;
    a.vp = (uint16_t *)v_pages;
    a.table = page_table;
    a.table_out = page_table_out;
    a.lens = lens;
    a.wsum = weight_sum;
    a.wsum_out = weight_sum_out;
    a.lens_out = lens_out;
    a.kept = kept;
    a.pool = PagePool{n_pages, nkv, page_size_log(page_size)};
    a.max_pages = max_pages;
    a.max_pages_out = max_pages_out;
    a.keep = keep;
    a.sinks = sinks;
    a.recent = recent;
    a.B = B;
    cudaStream_t st = (cudaStream_t)stream;
    VX_CK(launch_pdl(evict_select_k, dim3(nkv, B), dim3(SEL_THREADS), 0, st, a, dev_status()));
    const long long rows = (long long)B * nkv * keep;
    const int grid = (int)std::min<long long>((rows + 7) / 8, (long long)num_sms() * 8);
    VX_CK(launch_pdl(evict_copy_k, dim3(grid), dim3(256), 0, st, a, dev_status()));
    return 0;
}
