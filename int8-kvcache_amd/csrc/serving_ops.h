/*
 * serving_ops.h -- operators of a serving step over many requests, exported by libint8kv.so for the
 * package's Python entry points (int8kv.build_batch_tables, lora_plan, lora_add, sample_tokens),
 * next to the cache operators of int8kv.h and the layer steps of int8kv_decode_loop.h.  Not part
 * of the public C ABI (include/).
 *   1. block tables, slot mapping, positions and lengths of a ragged batch, from request lengths;
 *   2. low-rank adapters of many requests beside a shared projection;
 *   3. sampling with temperature, top-k, top-p and min-p from given random numbers.
 *
 * They have no counterpart among the reference's own operators: in its end-to-end runs
 * (bench/run_qwen_case_final.py of cjsmt/Int8-kvcache) vLLM's scheduler, model and sampler around
 * the attention do this work.
 *
 * Conventions are those of int8kv.h: device pointers, element strides, a hipStream_t as void*,
 * 0 / negative INT8KV_E_* / positive hipError_t returns, no allocation, no synchronisation.
 */
#ifndef INT8KV_SERVING_OPS_H
#define INT8KV_SERVING_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "../../include/int8kv.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Block tables and per-token indices of one step of a batch, built from request lengths.
 * Request r holds c_r = computed_lens[r] tokens in the paged cache and brings n_r = new_lens[r]
 * more (both read as clamp(length, 0, 2^31 - 1)).  Its tokens follow those of request r - 1 in
 * the token outputs; tokens past num_tokens are dropped, as if their request brought fewer (n_r
 * below is what is left).
 *
 *   Blocks: request r has ceil(c_r / block_size) and needs ceil((c_r + n_r) / block_size), both at
 *   most table_width; the blocks it lacks come from the free list, in request order:
 *     block_tables[r, j] = free_blocks[free_start + (blocks taken by requests before r) + j - have]
 *   for have <= j < need, -1 where that index lies outside [0, num_free).  Other entries are left
 *   as they are.  free_end = free_start + all blocks taken (above num_free: the list ran out).
 *
 *   query_starts[r] = first token of request r, query_starts[requests] = tokens held (int32)
 *   seq_lens[r] = min(c_r + n_r, 2^31 - 1)                                          (int32)
 *   for the i-th new token of request r, at p = c_r + i:
 *     positions = p, token_requests = r,
 *     slot_mapping = block_tables[r, p / block_size] * block_size + p % block_size, or -1 where
 *     p / block_size >= table_width or the block is negative
 *   rows behind the last token: position 0, slot -1, request -1.
 *
 *   computed_lens, new_lens: [requests] of lens_dtype (I32 or I64), contiguous.  block_tables:
 *   int32 [requests, table_width], unit inner stride.  free_blocks: int32 [num_free].
 *   free_start: one int64 on the device, or NULL for 0; free_end may be the same location.  No
 *   other output may overlap an input.
 *   workspace: int8kv_batch_tables_workspace_bytes(requests) bytes, 16-byte aligned, no
 *   initialisation needed; calls that share one must not overlap.  block_size in [1, 65536].
 */
size_t int8kv_batch_tables_workspace_bytes(int64_t requests);
int int8kv_batch_tables(const void* computed_lens, const void* new_lens, int lens_dtype,
                        int64_t requests, int32_t* block_tables, int64_t table_width,
                        int64_t table_row_stride, int32_t block_size, const int32_t* free_blocks,
                        int64_t num_free, const int64_t* free_start, int64_t num_tokens,
                        int32_t* query_starts, int32_t* seq_lens, int64_t* positions,
                        int64_t* slot_mapping, int32_t* token_requests, int64_t* free_end,
                        void* workspace, size_t workspace_bytes, void* stream);

/*
 * Low-rank adapters: out[t, :] = bf16(base[t, :] + scales[a] * (x[t, :] A[a]^T) B[a]^T) with
 * a = adapter_ids[t]; rows whose id lies outside [0, num_adapters) get out[t, :] = base[t, :].
 * Products and sums in fp32; the rank-wide intermediate is kept in fp32 and enters the second
 * product as two bf16 parts (17 bits).
 *
 * int8kv_lora_plan groups a step's tokens by adapter, once for all projections of the step: it
 * fills `plan` (int8kv_lora_plan_bytes(tokens, num_adapters) bytes, 16-byte aligned, no
 * initialisation needed).  adapter_ids: [tokens] of ids_dtype (I32 or I64), contiguous.
 * tokens <= 2^24, num_adapters <= 4096 (else the size is 0 and the call INT8KV_E_SHAPE).
 */
size_t int8kv_lora_plan_bytes(int64_t tokens, int32_t num_adapters);
int int8kv_lora_plan(const void* adapter_ids, int ids_dtype, int64_t tokens, int32_t num_adapters,
                     void* plan, size_t plan_bytes, void* stream);

/*
 * The product, with the plan of the same tokens and num_adapters.  All matrices bf16 with unit
 * inner strides and 16-byte aligned rows: x [tokens, k], base and out [tokens, n] (out may be
 * base itself, and must not otherwise overlap the inputs: rows that overlap base's or x's give
 * INT8KV_E_STRIDE), lora_a [num_adapters, rank, k] and
 * lora_b [num_adapters, n, rank] (strides of the adapters and of the rows).  scales: fp32
 * [num_adapters], or NULL for 1.  k, n and rank multiples of 8, rank at most 128, k and n at most
 * 2^20.  workspace: int8kv_lora_workspace_bytes(...) bytes, 16-byte aligned, no initialisation
 * needed; calls that share one must not overlap.
 */
size_t int8kv_lora_workspace_bytes(int64_t tokens, int32_t num_adapters, int64_t k, int32_t rank);
int int8kv_lora_add(const void* base, int64_t base_row_stride, const void* x, int64_t tokens,
                    int64_t k, int64_t x_row_stride, const void* lora_a,
                    const int64_t lora_a_strides[2], const void* lora_b,
                    const int64_t lora_b_strides[2], int32_t num_adapters, int32_t rank, int64_t n,
                    const float* scales, const void* plan, size_t plan_bytes, void* out,
                    int64_t out_row_stride, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Sampling: one token per row r of logits [rows, vocab] (F32, F16 or BF16, row stride >= vocab).
 * With v the row's logits (a NaN counts as -inf), M their maximum and T = temperature[r]:
 *   w_i = exp((v_i - M) / T)   (1 where v_i = M, 0 where v_i = -inf)
 *   order the tokens by v, largest first, equal ones by index; S(j) = sum of the first j weights;
 *   n_k = top_k[r] if 0 < top_k[r] < vocab, else vocab
 *   n_p = #{j < n_k : S(j) < top_p[r] * S(n_k)}, at least 1, if top_p[r] < 1, else n_k
 *   n_m = #{j : w_j >= min_p[r]}, at least 1, if min_p[r] > 0, else vocab
 * keeps the first min(n_k, n_p, n_m) tokens of that order.  out[r] is the first kept token, in
 * index order, at which the sum of the kept weights up to it exceeds uniforms[r] times the sum of
 * all kept weights (uniforms below 0 or NaN count as 0, from 1 on as the largest number below 1).
 * Rows with T <= 0 (or NaN), or whose logits are all -inf or NaN, give the first maximum of v.
 *
 * Weights are rounded to multiples of 2^-41 or finer (2^-44 at vocab 152064), computed in 64 bits,
 * and summed as integers, so that a row's token depends on nothing but its inputs.
 *
 *   uniforms: fp32 [rows]; temperature, top_p, min_p: fp32 [rows] or NULL (1, 1, 0); top_k: int32
 *   [rows] or NULL (0); all contiguous.
 *   vocab in [1, 2^21], rows at most 2^16.  out: int64 [rows].
 *   workspace: int8kv_sample_workspace_bytes(rows, vocab) bytes, 16-byte aligned, no
 *   initialisation needed; calls that share one must not overlap.
 */
size_t int8kv_sample_workspace_bytes(int64_t rows, int64_t vocab);
int int8kv_sample_rows(const void* logits, int logits_dtype, int64_t rows, int64_t vocab,
                       int64_t row_stride, const float* uniforms, const float* temperature,
                       const int32_t* top_k, const float* top_p, const float* min_p, int64_t* out,
                       void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* INT8KV_SERVING_OPS_H */
