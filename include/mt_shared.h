/* Attention of a batch whose requests share a long prefix, and the append that
 * reads a slot map: C-ABI of minitorch_amd/cuda_kernels/shared_prefix_kernel.so
 * (gfx950). Status, dtype, slab and stream conventions as in mt_paged.h.
 *
 * The prefix is prefix_tokens tokens (0: none) whose pages prefix_table (device,
 * ceil(prefix_tokens / page_size) entries; may be null without a prefix) names
 * once for the whole batch. A request's own tokens follow it: token s of request
 * r is at position prefix_tokens + s, in page table[r, s / page_size] of the
 * block table [b, columns] (a page of its own, also where the prefix ends inside
 * a page). Every query attends the whole prefix, then its request's own tokens
 * up to itself. The prefix is read once for many requests' queries (tiles of up
 * to 256), not once per request. A missing page (mt_paged.h) makes every query
 * that attends it NaN; one of the prefix all of them. Inf and NaN of K and V reach
 * the queries that attend them and no others (rows beside or behind such values
 * in V are computed once more one by one, which is slow).
 *
 * Workspace: partial results, of the size that mt_paged_shared_workspace_bytes
 * reports for the same sizes (0: none is needed, and it may be null), 16-byte
 * aligned, with no content to keep between calls; calls that share one must not
 * overlap, nor must replays of graphs captured with it. Fewer rows can need more
 * (their keys are cut more often): one for several sizes takes the largest of theirs.
 * `out` overlaps no input.
 * Sizes: h <= 65535 / b; rows * h * d, prefix and own tokens of a table together
 * below 2^31; for rows of whole 16-byte chunks also rows * h < 2^26, and at most 2^22
 * pieces of work of one kind (tiles of up to 256 rows x the cuts of the longest
 * keys). What is past them is refused with hipErrorInvalidValue.
 */
#ifndef MT_SHARED_H
#define MT_SHARED_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* K/V rows [rows, kv_stride] (head j at columns [j*d, (j+1)*d); kv_stride 0 =
 * h*d) to their pages through a slot map (device): row t goes to row slots[t] %
 * page_size of page slots[t] / page_size. Rows whose slot is negative, past the
 * pool or in an absent slab are skipped. Of rows with the same slot any one
 * may be the one that stays, 16 bytes by 16 bytes. rows * kv_stride < 2^31; h*d
 * <= kv_stride. No reference counterpart (reference mt_paged_append,
 * src/paged_attention_kernel.cu:96-106, takes one offset for the batch). */
int mt_paged_append_slots(const void* k, const void* v, const uint64_t* slabs, const int64_t* slots, int rows,
                          int h, int d, int page_size, int pages_per_slab, int num_slabs, int layer, int layers,
                          int dtype, int kv_stride);

/* Bytes of workspace the two attentions below need on the current device: for
 * mt_paged_shared_decode rows = b and max_tokens = 1. */
int mt_paged_shared_workspace_bytes(int rows, int b, int h, int d, int page_size, int prefix_tokens, int columns,
                                    int max_tokens, int dtype, size_t* bytes);

/* One token per request: q/k/v/out [b, h, 1, d] (rows of q, k and v qkv_stride
 * elements apart, 0 = h*d; out contiguous). Writes k/v as own token offsets[r]
 * (device) of request r, then attends the prefix and its own offsets[r] + 1
 * tokens. A request of negative offset is padding: its output row is zero and
 * nothing is written. One past the table's columns has a NaN row and writes
 * nothing. Without a prefix this is mt_paged_decode_batch up to the order of
 * its sums. Two launches at most; nothing is allocated, so that the call can be
 * captured. Requests must not share a page that this call writes. No reference
 * counterpart (the reference reads a shared prefix once per request,
 * src/paged_attention_kernel.cu:121-137). */
int mt_paged_shared_decode(void* out, const void* q, const void* k, const void* v, const uint64_t* slabs,
                           const int* prefix_table, const int* table, const int* offsets, int b, int h, int d,
                           int page_size, int pages_per_slab, int num_slabs, int prefix_tokens, int columns,
                           int layer, int layers, int dtype, int qkv_stride, void* workspace,
                           size_t workspace_bytes);

/* Several new tokens per request, whose K/V are in the pages already
 * (mt_paged_append_slots): request r has query rows [cu_tokens[r], cu_tokens[r +
 * 1]) (device [b + 1], ascending from 0; what mt_sched_batch_tables writes) of q [rows,
 * q_stride] and out [rows, out_stride] (head j at columns [j*d, (j+1)*d);
 * strides 0 = h*d). Its query i attends the prefix and its own tokens [0,
 * lengths[r] + i] (lengths: device, own tokens before the new ones; negative:
 * padding, whose rows are zero). max_tokens bounds the new tokens of any one
 * request: rows past it, like those behind the last request's, are not
 * written. 1 <= b <= 65535, max_tokens <= rows. No launch depends on device
 * values, and nothing is allocated, so that the call can be captured. No
 * reference counterpart. */
int mt_paged_shared_attention(void* out, const void* q, const uint64_t* slabs, const int* prefix_table,
                              const int* table, const int* lengths, const int* cu_tokens, int b, int rows,
                              int max_tokens, int h, int d, int page_size, int pages_per_slab, int num_slabs,
                              int prefix_tokens, int columns, int layer, int layers, int dtype, int q_stride,
                              int out_stride, void* workspace, size_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif /* MT_SHARED_H */
