// GQA over the paged KV cache (include/vx27_paged.h): the append kernel, and the entry points
// of the decode (gqa_paged_tc.cu) and prompt attention (gqa_paged_prefill.cu).
#include <algorithm>
#include "common.cuh"
#include "gqa_paged.cuh"
#include "../../include/vx27_paged.h"

namespace vx27 {
namespace {

constexpr int HD = PG_HD;

// ---- append ---------------------------------------------------------------------------
// y = x * rsqrt(mean x^2 + eps) * w, then the rotation (x0, x1) -> (x0 c - x1 s, x0 s + x1 c)
// of dims (i, i + rope_dim / 2). A warp takes `rows` rows (q, k or v) of one token, so that its
// position, slot, page and rope row are looked up once; the loads of four rows are in flight
// while the four before them are worked on. Lane l < rope_dim / 8 holds dims 4 l .. and their
// partners rope_dim / 2 + 4 l .., the others 8 l .., so a rotation needs no other lane; lanes
// without one rotate by (1, 0). The square sum is a tree of fp32 sums.
// Bound by the activations' bytes when there are many tokens: 4096 tokens of 24 + 4 heads take
// 31 us, 4.3 TB/s (one head per warp at a time, everything looked up per head: 53 us; a plain
// copy of the bytes: 24 us). Their 2048 blocks run in 2.3 rounds of 6 per SM, each with the chain
// of lookups in front. One token takes 3.1 us, the chain slot -> page -> store.
constexpr int APPEND_THREADS = 128;
struct AppendArgs {
    const void *q_in, *k_in, *v_in;
    const float *qw, *kw, *rope;
    const int *pos, *slots, *seq, *table;
    uint16_t *kp, *vp;
    void *q_out;
    PagePool pool;
    int rope_len, rope_dim, n_seqs, max_pages, n, nq, rows;
    float eps;
    int one_p, q_bf16;
};

// A lane's 8 values of a row: 4 from d0 and 4 from d1.
template <bool BF16>
struct Row8 {
    uint2 a[2];
    __device__ __forceinline__ void load(const void *p, size_t i, int d0, int d1) {
        const uint16_t *r = static_cast<const uint16_t *>(p) + i;
        a[0] = *reinterpret_cast<const uint2 *>(r + d0);
        a[1] = *reinterpret_cast<const uint2 *>(r + d1);
    }
    __device__ __forceinline__ float get(int e) const {
        const uint32_t w = (e & 2) ? a[e >> 2].y : a[e >> 2].x;
        return (e & 1) ? __uint_as_float(w & 0xffff0000u) : __uint_as_float(w << 16);
    }
};
template <>
struct Row8<false> {
    float4 a[2];
    __device__ __forceinline__ void load(const void *p, size_t i, int d0, int d1) {
        const float *r = static_cast<const float *>(p) + i;
        a[0] = *reinterpret_cast<const float4 *>(r + d0);
        a[1] = *reinterpret_cast<const float4 *>(r + d1);
    }
    __device__ __forceinline__ float get(int e) const {
        const float4 &f = a[e >> 2];
        return (e & 3) == 0 ? f.x : (e & 3) == 1 ? f.y : (e & 3) == 2 ? f.z : f.w;
    }
};
__device__ __forceinline__ void st_row_bf16(uint16_t *p, int d0, int d1, const float (&y)[8]) {
    *reinterpret_cast<uint2 *>(p + d0) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    *reinterpret_cast<uint2 *>(p + d1) = make_uint2(pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
}

template <bool ACT_BF16>
__global__ void __launch_bounds__(APPEND_THREADS, ACT_BF16 ? 6 : 4)
paged_append_k(const __grid_constant__ AppendArgs a, uint32_t *status) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    const int nkv = a.pool.nkv, nh = a.nq + 2 * nkv, parts = (nh + a.rows - 1) / a.rows;
    const long long item = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (item >= (long long)a.n * parts) return;
    const int t = (int)(item / parts), h0 = (int)(item % parts) * a.rows, h1 = min(h0 + a.rows, nh);
    const bool rot = lane < a.rope_dim / 8;
    const int d0 = rot ? 4 * lane : 8 * lane, d1 = rot ? a.rope_dim / 2 + 4 * lane : 8 * lane + 4;
    // the token: position, slot and page are looked up while the first rows come
    const int p = a.pos[t], slot = a.slots[t], b = a.seq ? a.seq[t] : t;
    float wq[8], wk[8], c[4], s[4];
    auto weights = [&](float (&w)[8], const float *from) {
        const float4 f = *reinterpret_cast<const float4 *>(from + d0);
        const float4 g = *reinterpret_cast<const float4 *>(from + d1);
        const float one = a.one_p ? 1.0f : 0.0f;
        w[0] = f.x + one; w[1] = f.y + one; w[2] = f.z + one; w[3] = f.w + one;
        w[4] = g.x + one; w[5] = g.y + one; w[6] = g.z + one; w[7] = g.w + one;
    };
    weights(wq, a.qw);
    weights(wk, a.kw);
    const bool p_ok = p >= 0 && p < a.rope_len;
    if (a.rope_dim && !p_ok && lane == 0) dev_flag(status, VX_DEV_BAD_ARG);
    float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
    if (rot && p_ok) {
        const float *rr = a.rope + (size_t)p * a.rope_dim + d0;
        cs = *reinterpret_cast<const float4 *>(rr);
        sn = *reinterpret_cast<const float4 *>(rr + a.rope_dim / 2);
    }
    c[0] = cs.x; c[1] = cs.y; c[2] = cs.z; c[3] = cs.w;
    s[0] = sn.x; s[1] = sn.y; s[2] = sn.z; s[3] = sn.w;
    int page = -1;
    if (slot >= 0 && h1 > a.nq) {
        const bool ok = b >= 0 && b < a.n_seqs && (slot >> a.pool.ps_log) < a.max_pages;
        if (ok) page = a.table[(size_t)b * a.max_pages + (slot >> a.pool.ps_log)];
        if (!a.pool.has(page)) {
            page = -1;
            if (lane == 0) dev_flag(status, VX_DEV_BAD_ARG);
        }
    }
    auto request = [&](Row8<ACT_BF16> (&x)[4], int h) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int i = h + u;
            if (i >= h1) continue;
            const int j = i < a.nq ? i : i < a.nq + nkv ? i - a.nq : i - a.nq - nkv;
            x[u].load(i < a.nq ? a.q_in : i < a.nq + nkv ? a.k_in : a.v_in,
                      ((size_t)t * (i < a.nq ? a.nq : nkv) + j) * HD, d0, d1);
        }
    };
    Row8<ACT_BF16> x[4], next[4];
    request(next, h0);
    for (int h = h0; h < h1; h += 4) {
#pragma unroll
        for (int u = 0; u < 4; u++) x[u] = next[u];
        request(next, h + 4);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int i = h + u;
            if (i >= h1) continue;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = x[u].get(e);
            if (i >= a.nq + nkv) {
                if (page >= 0) st_row_bf16(a.vp + a.pool.row(page, i - a.nq - nkv, slot) * HD, d0, d1, y);
                continue;
            }
            const bool is_q = i < a.nq;
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) ss = fmaf(y[e], y[e], ss);
            const float r = rsqrtf(warp_sum(ss) * (1.0f / HD) + a.eps);
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = y[e] * r * (is_q ? wq[e] : wk[e]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float x0 = y[e], x1 = y[e + 4];
                y[e] = fmaf(x0, c[e], -x1 * s[e]);
                y[e + 4] = fmaf(x1, c[e], x0 * s[e]);
            }
            if (!is_q) {
                if (page >= 0) st_row_bf16(a.kp + a.pool.row(page, i - a.nq, slot) * HD, d0, d1, y);
            } else if (a.q_bf16) {
                st_row_bf16(static_cast<uint16_t *>(a.q_out) + ((size_t)t * a.nq + i) * HD, d0, d1, y);
            } else {
                float *o = static_cast<float *>(a.q_out) + ((size_t)t * a.nq + i) * HD;
                *reinterpret_cast<float4 *>(o + d0) = make_float4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<float4 *>(o + d1) = make_float4(y[4], y[5], y[6], y[7]);
            }
        }
    }
}

}  // namespace
}  // namespace vx27

using namespace vx27;

extern "C" {

int vx27_gqa_paged_append(const void *q_in, const void *k_in, const void *v_in,
                          const float *q_norm_w, const float *k_norm_w, const float *rope_table,
                          int rope_table_len, const int *pos, const int *slots, const int *seq,
                          const int *page_table, int n_seqs, int max_pages, void *k_pages,
                          void *v_pages, int n_pages, int page_size, void *q_out, int n, int nq,
                          int nkv, int hd, int rope_dim, float eps, int flags, void *stream,
                          char *err, size_t errlen) {
    const char *fn = "vx27_gqa_paged_append";
    if (check_pool(fn, k_pages, v_pages, n_pages, page_size, page_table, max_pages, nkv, hd, err,
                   errlen) ||
        check_heads(fn, nq, nkv, err, errlen))
        return -1;
    if (n <= 0 || n_seqs <= 0) return fail(err, errlen, "%s: n=%d n_seqs=%d", fn, n, n_seqs);
    if (!seq && n > n_seqs)
        return fail(err, errlen, "%s: %d tokens for %d sequences without seq", fn, n, n_seqs);
    if (rope_dim < 0 || rope_dim > hd || (rope_dim & 15))
        return fail(err, errlen, "%s: rope_dim=%d (a multiple of 16 up to 256)", fn, rope_dim);
    if (!q_in || !k_in || !v_in || !q_norm_w || !k_norm_w || !pos || !slots || !q_out ||
        (rope_dim && (!rope_table || rope_table_len <= 0)))
        return fail(err, errlen, "%s: null pointer argument", fn);
    if (((uintptr_t)q_in | (uintptr_t)k_in | (uintptr_t)v_in | (uintptr_t)q_out |
         (uintptr_t)q_norm_w | (uintptr_t)k_norm_w | (uintptr_t)rope_table) & 15)
        return fail(err, errlen,
                    "%s: activations, norm weights, rope_table and q_out must be 16-byte aligned", fn);
    AppendArgs a{};
    a.q_in = q_in;
    a.k_in = k_in;
    a.v_in = v_in;
    a.qw = q_norm_w;
    a.kw = k_norm_w;
    a.rope = rope_table;
    a.pos = pos;
    a.slots = slots;
    a.seq = seq;
    a.table = page_table;
    a.kp = (uint16_t *)k_pages;
    a.vp = (uint16_t *)v_pages;
    a.q_out = q_out;
    a.pool = PagePool{n_pages, nkv, page_size_log(page_size)};
    a.rope_len = rope_dim ? rope_table_len : 0x7fffffff;
    a.rope_dim = rope_dim;
    a.n_seqs = n_seqs;
    a.max_pages = max_pages;
    a.n = n;
    a.nq = nq;
    a.eps = eps;
    a.one_p = (flags & VX27_F_NORM_1P) != 0;
    a.q_bf16 = (flags & VX27_F_OUT_BF16) != 0;
    // heads per warp: four (one round of loads) until the warps fill the SMs, then more, for
    // fewer lookups; in equal parts
    const int nh = nq + 2 * nkv;
    const long long rounds = (long long)n * ((nh + 3) / 4), fill = (long long)num_sms() * 32;
    const int rows = (int)std::min<long long>(nh, 4 * std::max<long long>(1, rounds / fill));
    const int parts = (nh + rows - 1) / rows;
    a.rows = ((nh + parts - 1) / parts + 3) / 4 * 4;
    const long long warps = (long long)n * ((nh + a.rows - 1) / a.rows);
    if (warps > (1LL << 33)) return fail(err, errlen, "%s: n=%d", fn, n);
    const unsigned grid = (unsigned)((warps + APPEND_THREADS / 32 - 1) / (APPEND_THREADS / 32));
    cudaStream_t st = (cudaStream_t)stream;
    if (flags & VX27_F_ACT_BF16)
        VX_CK(launch_pdl(paged_append_k<true>, dim3(grid), dim3(APPEND_THREADS), 0, st, a, dev_status()));
    else
        VX_CK(launch_pdl(paged_append_k<false>, dim3(grid), dim3(APPEND_THREADS), 0, st, a, dev_status()));
    return 0;
}

size_t vx27_gqa_paged_workspace_size(int B, int nq, int nkv, int hd, int max_slots, int window,
                                     int sinks, int weights, int n_parts) {
    if (B <= 0 || nq <= 0 || nkv <= 0 || nq % nkv || hd != HD || max_slots <= 0 || window < 0 ||
        sinks < 0)
        return 0;
    DecodeArgs a{};
    return paged_decode_layout(a, nullptr, B, nq, nkv, max_slots, window, sinks, weights != 0,
                               paged_decode_parts(n_parts));
}

int vx27_gqa_paged_decode(const float *q, const void *gate, const void *k_pages,
                          const void *v_pages, int n_pages, int page_size, const int *page_table,
                          int max_pages, const int *lens, int window, int sinks,
                          float *weight_sum, void *out, void *workspace, size_t workspace_bytes,
                          int B, int nq, int nkv, int hd, int n_parts, int flags, void *stream,
                          char *err, size_t errlen) {
    const char *fn = "vx27_gqa_paged_decode";
    if (check_pool(fn, k_pages, v_pages, n_pages, page_size, page_table, max_pages, nkv, hd, err,
                   errlen) ||
        check_heads(fn, nq, nkv, err, errlen) || check_window(fn, window, sinks, err, errlen))
        return -1;
    if (B <= 0 || B > 65535) return fail(err, errlen, "%s: B=%d", fn, B);
    if (!q || !lens || !out || !workspace) return fail(err, errlen, "%s: null pointer argument", fn);
    if (((uintptr_t)q | (uintptr_t)gate | (uintptr_t)out | (uintptr_t)workspace | (uintptr_t)weight_sum) & 15)
        return fail(err, errlen, "%s: q, gate, out, weight_sum and the workspace must be 16-byte aligned",
                    fn);
    DecodeArgs a{};
    int P = paged_decode_parts(n_parts);
    const size_t need = paged_decode_layout(a, workspace, B, nq, nkv, max_pages * page_size, window,
                                            sinks, weight_sum != nullptr, P);
    if (workspace_bytes < need)
        return fail(err, errlen, "%s: workspace of %zu bytes, need %zu", fn, workspace_bytes, need);
    a.q = q;
    a.gate = gate;
    a.table = page_table;
    a.lens = lens;
    a.wsum = weight_sum;
    a.out = out;
    a.pool = PagePool{n_pages, nkv, page_size_log(page_size)};
    a.max_pages = max_pages;
    a.B = B;
    a.window = window;
    a.sinks = sinks;
    a.nq = nq;
    a.gate_bf16 = (flags & VX27_F_ACT_BF16) != 0;
    a.out_bf16 = (flags & VX27_F_OUT_BF16) != 0;
    // no more runs than the tables have tiles of 128 slots
    const long long tiles = ((long long)max_pages * page_size + 127) / 128;
    if (tiles * B * nkv > 0x7fffffffLL)
        return fail(err, errlen, "%s: %d sequences of %d pages: over 2^31 tiles of 128 slots", fn, B,
                    max_pages);
    P = (int)std::min<long long>(P, tiles * B * nkv);
    return launch_paged_decode(a, k_pages, v_pages, P, (cudaStream_t)stream, err, errlen);
}

size_t vx27_gqa_paged_prefill_workspace_size(int nkv, int hd) {
    return nkv <= 0 || hd != HD ? 0 : paged_prompt_workspace(nkv);
}

int vx27_gqa_paged_prefill(const void *q, const void *gate, const void *k_pages,
                           const void *v_pages, int n_pages, int page_size,
                           const int *page_table, int max_pages, int s0, int window, int sinks,
                           void *out, void *workspace, size_t workspace_bytes, int T, int nq,
                           int nkv, int hd, int flags, void *stream, char *err, size_t errlen) {
    const char *fn = "vx27_gqa_paged_prefill";
    if (check_pool(fn, k_pages, v_pages, n_pages, page_size, page_table, max_pages, nkv, hd, err,
                   errlen) ||
        check_heads(fn, nq, nkv, err, errlen) || check_window(fn, window, sinks, err, errlen))
        return -1;
    if (!(flags & VX27_F_ACT_BF16) || !(flags & VX27_F_OUT_BF16))
        return fail(err, errlen, "%s: q, gate and out must be bf16", fn);
    if (T <= 0 || s0 < 0 || (long long)s0 + T > (long long)max_pages * page_size)
        return fail(err, errlen, "%s: slots [%d, %d + %d) outside %d pages of %d", fn, s0, s0, T,
                    max_pages, page_size);
    if (!q || !out || !workspace) return fail(err, errlen, "%s: null pointer argument", fn);
    if (((uintptr_t)q | (uintptr_t)gate | (uintptr_t)out | (uintptr_t)workspace) & 15)
        return fail(err, errlen, "%s: q, gate, out and the workspace must be 16-byte aligned", fn);
    if (workspace_bytes < vx27_gqa_paged_prefill_workspace_size(nkv, hd))
        return fail(err, errlen, "%s: workspace of %zu bytes, need %zu", fn, workspace_bytes,
                    vx27_gqa_paged_prefill_workspace_size(nkv, hd));
    return launch_paged_prompt(q, gate, k_pages, v_pages,
                               PagePool{n_pages, nkv, page_size_log(page_size)}, page_table,
                               max_pages, s0, window, sinks, out, workspace, T, nq,
                               (cudaStream_t)stream, err, errlen);
}

}  // extern "C"
