// GQA over the paged KV cache (include/vx27_paged.h): the append kernel, and the entry points
// of the decode (gqa_paged_tc.cu) and prompt attention (gqa_paged_prefill.cu).
#include <algorithm>
#include "common.cuh"
#include "gqa_paged.cuh"
#include "../../include/vx27_paged.h"

namespace vx27 {
namespace {

constexpr int HD = PG_HD;

// 8 consecutive activations.
template <bool BF16>
__device__ __forceinline__ void ld8(float (&x)[8], const void *p, size_t i) {
    if constexpr (BF16) ld8_bf16(x, static_cast<const uint16_t *>(p) + i);
    else ld8_f32(x, static_cast<const float *>(p) + i);
}

// ---- append ---------------------------------------------------------------------------
// One warp per (token, head) row, 8 consecutive dims per lane; y = x * rsqrt(mean x^2 + eps)
// * w, then the rotation (x0, x1) -> (x0 c - x1 s, x0 s + x1 c) of dims (i, i + rope_dim/2),
// whose partner is rope_dim/16 lanes away. The square sum is a tree of fp32 sums.
struct AppendArgs {
    const void *q_in, *k_in, *v_in;
    const float *qw, *kw, *rope;
    const int *pos, *slots, *seq, *table;
    uint16_t *kp, *vp;
    void *q_out;
    PagePool pool;
    int rope_len, rope_dim, n_seqs, max_pages, n, nq;
    float eps;
    int one_p, q_bf16;
};

template <bool ACT_BF16>
__global__ void __launch_bounds__(256)
paged_append_k(const __grid_constant__ AppendArgs a, uint32_t *status) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, d0 = lane * 8;
    const int nkv = a.pool.nkv, nh = a.nq + nkv;
    const long long n_rows = (long long)a.n * nh;
    const int half = a.rope_dim / 2;
    const bool rot = d0 < a.rope_dim, lo = d0 < half;
    const int i0 = lo ? d0 : d0 - half;
    const int partner = (lo ? lane + half / 8 : lane - half / 8) & 31;
    for (long long item = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; item < n_rows;
         item += ((long long)gridDim.x * blockDim.x) >> 5) {
        const int t = (int)(item / nh), head = (int)(item % nh);
        const bool is_q = head < a.nq;
        const int h = is_q ? head : head - a.nq;
        const size_t row = (is_q ? (size_t)t * a.nq + h : (size_t)t * nkv + h) * HD + d0;
        float x[8], v[8];
        ld8<ACT_BF16>(x, is_q ? a.q_in : a.k_in, row);
        const int p = a.pos[t];
        const bool p_ok = p >= 0 && p < a.rope_len;
        size_t dst = 0;
        bool store = false;
        if (!is_q) {
            const int slot = a.slots[t], b = a.seq ? a.seq[t] : t;
            if (slot >= 0) {
                bool ok = b >= 0 && b < a.n_seqs && (slot >> a.pool.ps_log) < a.max_pages;
                const int page =
                    ok ? a.table[(size_t)b * a.max_pages + (slot >> a.pool.ps_log)] : -1;
                ok = ok && a.pool.has(page);
                if (!ok) dev_flag(status, VX_DEV_BAD_ARG);
                store = ok;
                if (ok) dst = a.pool.row(page, h, slot) * HD + d0;
            }
            ld8<ACT_BF16>(v, a.v_in, row);
        }
        float c[8], s[8];
        if (rot && p_ok) {
            const float *rr = a.rope + (size_t)p * a.rope_dim + i0;
            ld8<false>(c, rr, 0);
            ld8<false>(s, rr, half);
        }
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) ss = fmaf(x[e], x[e], ss);
        ss = warp_sum(ss);
        const float r = __fdiv_rn(1.0f, __fsqrt_rn(ss * (1.0f / HD) + a.eps));
        const float *wp = (is_q ? a.qw : a.kw) + d0;
        float y[8], yp[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float w = __ldg(wp + e);
            y[e] = x[e] * r * (a.one_p ? w + 1.0f : w);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) yp[e] = __shfl_sync(0xffffffffu, y[e], partner);
        if (rot) {
            if (!p_ok) {
                dev_flag(status, VX_DEV_BAD_ARG);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    y[e] = lo ? fmaf(y[e], c[e], -yp[e] * s[e]) : fmaf(yp[e], s[e], y[e] * c[e]);
            }
        }
        if (is_q) {
            if (a.q_bf16) st8_bf16(static_cast<uint16_t *>(a.q_out) + row, y);
            else st8_f32(static_cast<float *>(a.q_out) + row, y);
        } else if (store) {
            st8_bf16(a.kp + dst, y);
            st8_bf16(a.vp + dst, v);
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
         (uintptr_t)rope_table) & 15)
        return fail(err, errlen, "%s: activations, rope_table and q_out must be 16-byte aligned", fn);
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
    const long long rows = (long long)n * (nq + nkv);
    const int grid = (int)std::min<long long>((rows + 7) / 8, (long long)num_sms() * 8);
    cudaStream_t st = (cudaStream_t)stream;
    if (flags & VX27_F_ACT_BF16)
        VX_CK(launch_pdl(paged_append_k<true>, dim3(grid), dim3(256), 0, st, a, dev_status()));
    else
        VX_CK(launch_pdl(paged_append_k<false>, dim3(grid), dim3(256), 0, st, a, dev_status()));
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
    if (((uintptr_t)q | (uintptr_t)gate | (uintptr_t)out | (uintptr_t)workspace) & 15)
        return fail(err, errlen, "%s: q, gate, out and the workspace must be 16-byte aligned", fn);
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
