// What the entry points of the paged cache's attention (gqa_paged.cu) and its kernels
// (gqa_paged_tc.cu, gqa_paged_prefill.cu) share; 8-element loads and stores.
#pragma once
#include "common.cuh"
#include "paged.cuh"

namespace vx27 {

struct DecodeArgs {
    const float *q;
    const void *gate;
    const int *table, *lens;
    float *wsum;  // NULL: no weight sums
    void *out;
    // workspace
    int4 *join;      // [P] item, first and last run of the item that this run continues
    float *rec_o;    // [2 P][G][256] parts of cut items: first item of a run, last item
    float2 *rec_ml;  // [2 P][G] (m in log2 units, l)
    int2 *span;      // [B nkv] first and last run of an item
    float2 *item_ml; // [B nkv][G] of whole items
    float *scores;   // [B nkv][G][score_stride], log2 units, by tile
    size_t score_stride;
    PagePool pool;
    int max_pages, B, window, sinks, nq, gate_bf16, out_bf16;
};

// Runs that a call cuts the batch into.
int paged_decode_parts(int n_parts);
// Sets the workspace pointers of a (NULL workspace: sizes only); bytes used.
size_t paged_decode_layout(DecodeArgs &a, void *workspace, int B, int nq, int nkv, int max_slots,
                           int window, int sinks, bool weights, int P);
int launch_paged_decode(const DecodeArgs &a, const void *k_pages, const void *v_pages, int P,
                        cudaStream_t st, char *err, size_t errlen);

// Prompt attention: T rows in slots s0 .. of the sequence with this table row.
size_t paged_prompt_workspace(int nkv);
int launch_paged_prompt(const void *q, const void *gate, const void *k_pages, const void *v_pages,
                        const PagePool &pool, const int *table, int max_pages, int s0, int window,
                        int sinks, void *out, void *workspace, int T, int nq, cudaStream_t st,
                        char *err, size_t errlen);

__device__ __forceinline__ void ld8_bf16(float (&x)[8], const uint16_t *p) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
        x[2 * k] = bf16_to_f32(w[k] & 0xffffu);
        x[2 * k + 1] = bf16_to_f32(w[k] >> 16);
    }
}
__device__ __forceinline__ void ld8_f32(float (&x)[8], const float *p) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0];
    const float4 b = reinterpret_cast<const float4 *>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void st8_bf16(uint16_t *p, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(p) =
        make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                   pack_bf16x2(x[6], x[7]));
}
__device__ __forceinline__ void st8_f32(float *p, const float (&x)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

}  // namespace vx27
