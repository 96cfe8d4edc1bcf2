// Internal launch interface between the C ABI (capi.cu) and the kernels.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "fa_b200.h"

namespace fa {

// ---- prefill (prefill_sm100.cu) -------------------------------------------
const void *prefill_kernel_ptr(int dtype = FA_DTYPE_F16);
int prefill_threads();
const void *prefill_solo_kernel_ptr(int dtype = FA_DTYPE_F16);
int prefill_solo_smem_bytes();
int prefill_solo_threads();
const void *prefill_split_kernel_ptr(int dtype = FA_DTYPE_F16);
int prefill_split_smem_bytes();
const void *prefill_d128_solo_kernel_ptr(int dtype = FA_DTYPE_F16);
int prefill_d128_solo_smem_bytes();
const void *prefill_d128_wide_kernel_ptr(int dtype = FA_DTYPE_F16);
int prefill_d128_wide_smem_bytes();
int prefill_smem_bytes();
cudaError_t launch_prefill_kernel(const CUtensorMap &tm_q,
                                  const CUtensorMap &tm_k,
                                  const CUtensorMap &tm_v, __half *out, int B,
                                  int H, int N, bool causal, float scale,
                                  int H_kv, int sms, int dtype,
                                  cudaStream_t stream, long long plan_bh = 0);
// CTA form of the head_dim-64 prefill for BH (batch x head) pairs of N
// tokens (FA_PREFILL_FORM_*); *ctas (if given) receives the grid size.
// plan_bh > 0: the form of a chunk of a larger problem of plan_bh pairs.
int prefill_form_of(long long BH, int N, bool causal, int sms,
                    long long plan_bh, int *ctas);
// fa_prefill_ex for one chunk of a larger problem of plan_bh (batch x head)
// pairs: the CTA form is chosen for the whole problem, so a head's output
// does not depend on how the problem was cut into launches (capi.cu).
int prefill_chunk_ex(const void *q, const void *k, const void *v, void *o,
                     int B, int H, int H_kv, int N, int head_dim, int dtype,
                     int causal, float scale, void *stream, long long plan_bh);

// ---- prefill, head_dim 128 (prefill_d128_sm100.cu) -------------------------
const void *prefill_d128_kernel_ptr(int dtype = FA_DTYPE_F16);
int prefill_d128_smem_bytes();
cudaError_t launch_prefill_d128_kernel(const CUtensorMap &tm_q,
                                       const CUtensorMap &tm_k,
                                       const CUtensorMap &tm_v, __half *out,
                                       int B, int H, int N, bool causal,
                                       float scale, int H_kv, int sms,
                                       int dtype, cudaStream_t stream);

// ---- decode (decode_sm100.cu) ---------------------------------------------
struct DecodeArgs {
  const __half *q;
  const __half *k;
  const __half *v;
  const int32_t *seq_lens;
  __half *out;           // final fp16 output, or
  float *partial_out;    // (B, H, 68) log-sum-exp partials when non-null
  float *ws_partials;    // (B*H + grid) x 68 fp32
  uint32_t *ws_counters; // B*H arrival counters, zero between calls
  // fused append (null when not appending): the new token's K/V rows
  // (B, H_kv, 64), stored at row seq_lens[b] of the caches (written through
  // k_cache_w / v_cache_w, the same caches as k / v) and attended
  const __half *k_new;
  const __half *v_new;
  __half *k_cache_w;
  __half *v_cache_w;
  // cross-GPU exchange (null when not sharded): x_peers[r] is rank r's
  // exchange buffer, two epoch-parity banks of (x_world, B*H, 4 + D) fp32
  // partials then B*H uint32
  // arrival counters; each finished segment is sent to every rank and the
  // merged output written once all x_world partials of it are present
  // (counters reach x_epoch * x_world)
  float *const *x_peers;
  int x_rank, x_world;
  uint32_t x_epoch;
  int B, H, S_max;
  int H_kv;  // K/V heads; H / H_kv query heads share each
  float scale_log2;
  long long rows_per_cta;  // 0: balance the valid rows over the grid
  int grid;
  int dtype;  // FA_DTYPE_F16 or FA_DTYPE_BF16 (q, caches, new rows, out)
};

constexpr int kPartialFloats = 68;  // m, l, pad, pad, acc[64]

const void *decode_kernel_ptr(int dtype = FA_DTYPE_F16);
int decode_threads();
int decode_smem_bytes();
int decode_ctas_per_sm();
int decode_min_rows_per_cta();
cudaError_t launch_decode_kernel(const DecodeArgs &args, cudaStream_t stream);

// Grouped-query decode: K/V read once per group of query heads. The grid is
// one CTA per SM at most; segments are (b, K/V head, chunk of up to
// decode_gqa_max_heads() query heads).
// (decode_gqa_sm100.cu) head_dim 64 or 128; K/V TMA boxes of
// decode_gqa_box_rows(head_dim) rows; partials of 4 + head_dim floats.
const void *decode_gqa_kernel_ptr(int head_dim, int dtype = FA_DTYPE_F16);
int decode_gqa_smem_bytes(int head_dim);
int decode_gqa_max_heads();
// Partial records of one segment one round of the final merge gathers.
int decode_gqa_merge_batch(int head_dim, int heads_per_seg);
int decode_gqa_box_rows(int head_dim);
cudaError_t launch_decode_gqa_kernel(const DecodeArgs &args,
                                     const CUtensorMap &tm_k,
                                     const CUtensorMap &tm_v, int head_dim,
                                     cudaStream_t stream);

// head_dim 128 per-head decode (decode_d128_sm100.cu); partials are
// decode_d128_partial_floats() = 132 floats, grid as decode_kernel's.
const void *decode_d128_kernel_ptr(int dtype = FA_DTYPE_F16);
int decode_d128_smem_bytes();
int decode_d128_partial_floats();
cudaError_t launch_decode_d128_kernel(const DecodeArgs &args,
                                      cudaStream_t stream);

const void *merge_kernel_ptr();
int merge_threads();
cudaError_t launch_merge_kernel(const float *partials, int G, __half *out,
                                int B, int H, cudaStream_t stream);

// ---- rotary positions and the paged append (rope_sm100.cu) ------------------
struct RopeArgs {
  const __half *q;  // null with H == 0: none
  const __half *k;
  const __half *v;  // append only
  __half *q_out;
  __half *k_out;  // append: the K pages
  __half *v_out;  // append: the V pages
  // element strides per batch entry, head and token
  int64_t q_sb, q_sh, q_sn, qo_sb, qo_sh, qo_sn;
  int64_t k_sb, k_sh, k_sn, ko_sb, ko_sh, ko_sn;
  int64_t v_sh, v_sn;
  int H, H_kv, N, D, rot;
  int tokens;  // B * N, or the step's
  const int32_t *positions;  // append: null for the cache row
  int64_t position_stride;
  const double *freqs;
  float amplitude, sign;
  // set by the launch: how a warp's lanes lie on units and rows, the chunks
  // that a token's rows (q's, from k_before on k's, from v_before on v's) are
  // cut into, and from a warp's token to its next
  int unit_lanes, row_lanes, rows_per_chunk, chunks, k_before, v_before;
  int token_step;
  // append
  const int32_t *starts;
  const int32_t *seq_lens;
  const int32_t *page_table;
  int64_t table_stride;
  int64_t kp_sp, kp_sh, kp_sr, vp_sp, vp_sh, vp_sr;  // page, head, row
  int batch, table_width, page_rows, num_pages;
};
// vector: every row is 16-byte aligned and rotates in whole 16-byte units.
cudaError_t launch_rope_kernel(const RopeArgs &a, bool interleaved,
                               bool append, bool vector, int dtype, int sms,
                               cudaStream_t stream);

// ---- attention over a paged cache (paged_attend_sm100.cu) -------------------
struct PagedArgs {
  const __half *q;
  int64_t q_st, q_sh;  // element strides per token and head
  __half *out;         // (tokens, H, D)
  float *lse;          // (tokens, H) or null
  const __half *k_pages;
  const __half *v_pages;
  int64_t kp_sp, kp_sh, kp_sr, vp_sp, vp_sh, vp_sr;
  const int32_t *page_table;
  int64_t table_stride;
  const int32_t *starts;
  const int32_t *seq_lens;
  int batch, tokens, H, H_kv, D, table_width, page_rows, num_pages;
  float scale_log2;
  int causal;
  // set by the launch: rows of a TMA box, new tokens of an item, and the
  // division of the work (paged_sm100.cuh)
  int box_rows, item_tokens, item_cost, min_piece, min_part, whole_tiles;
  float *partials;
  uint32_t *counters;
};
// Form of the call: few query rows per sequence and K/V head
// (paged_few_sm100.cu) or many (paged_many_sm100.cu).
enum { kPagedFew = 0, kPagedMany = 1, kPagedForms = 2 };
const void *attend_paged_kernel_ptr(int form, int head_dim, int dtype);
int attend_paged_smem_bytes(int form, int head_dim);
size_t attend_paged_workspace_bytes(int head_dim, int sms);
// Sets the fields above and launches; tm_q is used by kPagedMany.
int attend_paged_form(const PagedArgs &a);
void attend_paged_plan(PagedArgs &a, int form);
cudaError_t launch_attend_paged_kernel(const PagedArgs &a, int form,
                                       const CUtensorMap &tm_q,
                                       const CUtensorMap &tm_k,
                                       const CUtensorMap &tm_v, int dtype,
                                       int sms, cudaStream_t stream);

// ---- single-head fp32 attention (legacy_sm100.cu) -------------------------
cudaError_t launch_legacy_kernel(const float *q, const float *k, const float *v,
                                 float *o, int N, cudaStream_t stream);

}  // namespace fa
