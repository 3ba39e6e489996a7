/*
 * GQA over a paged BF16 KV cache on B200 (libvx27cuda): append, decode attention, prompt
 * attention, eviction. No counterpart in the reference, which keeps one contiguous fp32
 * cache per layer (src/vx27_qfwd.c:183-185).
 *
 * The cache of a layer is a pool of pages, two planes k_pages and v_pages, each bf16
 * [n_pages][nkv][page_size][hd], and a table page_table int32 [n_seqs][max_pages] on the
 * device: slot s of sequence b is row s % page_size of every KV head of page
 * page_table[b][s / page_size]. A sequence's slots are numbered in the order in which its
 * tokens came. page_size is 16, 32, 64, 128 or 256, hd is 256, nq / nkv is 1 to 8; caches,
 * activations, norm weights, weight sums, outputs and workspaces are 16-byte aligned and
 * contiguous. A table holds at most 2^31 - 256 slots per sequence.
 *
 * A window keeps the last `window` slots in sight and the first `sinks` ones: with n slots
 * up to and with its own, a token attends to slot j when j >= n - window or j < sinks. window
 * = 0: all n slots (sinks is then 0). Table entries whose slots no token of the call attends
 * to are not read, so the pages between the sinks and the window may be freed (entry -1).
 *
 * The values of the tables are on the device, so the host cannot check them. A page outside
 * [0, n_pages), a sequence index or a position outside its table, and a length above max_pages *
 * page_size put 3 into the status word (vx27cuda_device_status); nothing outside the pool
 * is then read or written, and the results of that sequence are unspecified.
 *
 * All calls enqueue on the stream and return; they allocate nothing and may be captured
 * into a graph, which keeps the addresses: tables, lengths, caches and workspace live as long
 * as it does. Calls that overlap on the GPU need workspaces of their own.
 */
#ifndef VX27_PAGED_H
#define VX27_PAGED_H
#include <stddef.h>
#include "vx27cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * n tokens enter the cache: RMSNorm of q and k per head (eps, weights [hd]; VX27_F_NORM_1P:
 * zero-centred), NeoX rotation of the first rope_dim dims at position pos[i] (row pos[i] of a
 * table from vx27_rope_table_build), bf16 store of k and v into slot slots[i] of sequence
 * seq[i] (seq NULL: sequence i). A slot below 0 stores nothing (an idle lane of a padded
 * batch); its q_out row is written all the same. Two tokens of one call must not name the
 * same slot of the same sequence.
 *   q_in [n][nq][hd], k_in, v_in [n][nkv][hd]  (act dtype)
 *   q_out [n][nq][hd]: fp32 for vx27_gqa_paged_decode, or bf16 (VX27_F_OUT_BF16) for
 *         vx27_gqa_paged_prefill
 * rope_dim is a multiple of 16 up to hd.
 */
int vx27_gqa_paged_append(const void *q_in, const void *k_in, const void *v_in,
                          const float *q_norm_w, const float *k_norm_w, const float *rope_table,
                          int rope_table_len, const int *pos, const int *slots, const int *seq,
                          const int *page_table, int n_seqs, int max_pages, void *k_pages,
                          void *v_pages, int n_pages, int page_size, void *q_out, int n, int nq,
                          int nkv, int hd, int rope_dim, float eps, int flags, void *stream,
                          char *err, size_t errlen);

/*
 * Attention of one token per sequence over the lens[b] slots that the sequence holds (the
 * token's own is the last), or those of them in the window: out = softmax(q k^T / sqrt(hd)) v
 * * sigmoid(gate) per query head (head h reads KV head h * nkv / nq). lens[b] = 0: a row of
 * zeros. What lies in masked slots, NaN and infinities among it, has no effect; seen K and V rows
 * and q are finite (an infinity among them gives NaN, since q is split into terms).
 *   q [B][nq][hd] fp32; gate [B][nq][hd] (act dtype) or NULL; out [B][nq][hd] (fp32, or bf16
 *   with VX27_F_OUT_BF16)
 *   weight_sum fp32 [B][nkv][max_pages * page_size] or NULL: to the entry of each slot attended
 *   to, the softmax weights that the heads of its group gave it are added (vx27_kv_evict)
 *   workspace: vx27_gqa_paged_workspace_size(...) bytes, 16-byte aligned; with weight sums it
 *   holds B * nq * max_slots floats (with a window only as many slots as that and the sinks span)
 * The slots that the batch attends to are counted in tiles of 128 and cut into n_parts equal
 * runs (0: one per SM; at most 1024), which are joined where a cut goes through a sequence. So the
 * lengths of the other sequences move the cuts, and with them the last bits of a result; the
 * same call always gives the same bits. With fp32 out or weight_sum, q and the softmax's
 * weights enter the tensor cores as three bf16 terms (24 bits), else as two (16 bits).
 * Batches of over 2^31 tiles are refused.
 */
size_t vx27_gqa_paged_workspace_size(int B, int nq, int nkv, int hd, int max_slots, int window,
                                     int sinks, int weights, int n_parts);
int vx27_gqa_paged_decode(const float *q, const void *gate, const void *k_pages,
                          const void *v_pages, int n_pages, int page_size, const int *page_table,
                          int max_pages, const int *lens, int window, int sinks,
                          float *weight_sum, void *out, void *workspace, size_t workspace_bytes,
                          int B, int nq, int nkv, int hd, int n_parts, int flags, void *stream,
                          char *err, size_t errlen);

/*
 * Causal attention of T prompt tokens of one sequence, in slots s0 .. s0 + T - 1 (already
 * appended): token t attends to slots [0, s0 + t], or those of them in its window.
 *   q, gate, out [T][nq][hd] bf16 (gate may be NULL; the flags are VX27_F_ACT_BF16 |
 *   VX27_F_OUT_BF16, other types are refused: the softmax's weights enter the tensor cores
 *   as bf16); page_table [max_pages], the sequence's row
 *   workspace: vx27_gqa_paged_prefill_workspace_size(nkv, hd) bytes (51 MB, whatever T)
 * K and V of the slots up to s0 + T - 1 in the pages that are attended to have to be
 * finite: a NaN or infinite V value reaches every token of its block of 128, masked or not.
 */
size_t vx27_gqa_paged_prefill_workspace_size(int nkv, int hd);
int vx27_gqa_paged_prefill(const void *q, const void *gate, const void *k_pages,
                           const void *v_pages, int n_pages, int page_size,
                           const int *page_table, int max_pages, int s0, int window, int sinks,
                           void *out, void *workspace, size_t workspace_bytes, int T, int nq,
                           int nkv, int hd, int flags, void *stream, char *err, size_t errlen);

/*
 * Cuts every sequence back to at most keep slots, per KV head: the first sinks slots, the
 * last recent ones, and of the others those with the largest weight_sum (ties: the lowest
 * slot; NaN ranks as -infinity). The kept rows and sums are copied, in slot order, to the
 * pages of page_table_out [B][max_pages_out] of the same pool; a sequence with at most keep slots
 * is copied whole. The old pages keep their contents, so sequences may share them.
 *   lens, lens_out [B]; weight_sum [B][nkv][max_pages * page_size], weight_sum_out
 *   [B][nkv][max_pages_out * page_size] (zero behind the kept slots)
 *   kept int32 [B][nkv][keep]: the old slot of each new one, -1 behind the last
 * Per head the kept slots differ, so afterwards a new slot's row is another token's in every
 * head; rows of the new pages behind lens_out are left as they were.
 * sinks + recent <= keep <= max_pages_out * page_size. No page of page_table_out may be a page
 * of page_table or occur twice, and no output may be an input: a call whose output
 * pointers equal its input pointers is refused.
 * Rotations are part of the stored K rows, so a kept row keeps its token's position; the
 * next token's slot is lens_out[b], its position goes on from the old count.
 */
int vx27_kv_evict(void *k_pages, void *v_pages, int n_pages, int page_size,
                  const int *page_table, int max_pages, const int *lens,
                  const float *weight_sum, const int *page_table_out, int max_pages_out,
                  int *lens_out, float *weight_sum_out, int *kept, int keep, int sinks,
                  int recent, int B, int nkv, int hd, void *stream, char *err, size_t errlen);

#ifdef __cplusplus
}
#endif
#endif
