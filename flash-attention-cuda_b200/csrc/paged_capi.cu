// C ABI of the paged-cache operators (include/fa_b200.h): argument checks and
// launches. No allocation happens here; callers own every buffer.

#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "fa_b200.h"
#include "fa_kernels.h"
#include "fa_sm100.cuh"

namespace fa {
namespace {

bool dtype_ok(int dtype) {
  return dtype == FA_DTYPE_F16 || dtype == FA_DTYPE_BF16;
}

bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// Strides that keep every row 16-byte aligned (a dimension of one element
// has none).
bool strides_vector(const int64_t *strides, const int *sizes, int n) {
  for (int i = 0; i < n; ++i)
    if (sizes[i] > 1 && strides[i] % 8 != 0) return false;
  return true;
}

int check_rotary(int head_dim, int rotary_dim, float amplitude,
                 const double *freqs) {
  if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim ||
      !isfinite(amplitude))
    return FA_EINVAL;
  return (reinterpret_cast<uintptr_t>(freqs) & 7u) ? FA_EALIGN : FA_OK;
}

int check_cache(const fa_paged_cache *c) {
  if (!c || !c->k_pages || !c->v_pages || !c->page_table) return FA_EINVAL;
  if (c->head_dim != FA_HEAD_DIM && c->head_dim != 128) return FA_EINVAL;
  if (c->num_pages <= 0 || c->kv_heads <= 0 || c->page_rows <= 0 ||
      c->table_width <= 0 || c->table_stride < 0)
    return FA_EINVAL;
  if (c->page_rows % 8 != 0) return FA_EINVAL;
  const int sizes[3] = {c->num_pages, c->kv_heads, c->page_rows};
  const int64_t ks[3] = {c->k_page_stride, c->k_head_stride, c->k_row_stride};
  const int64_t vs[3] = {c->v_page_stride, c->v_head_stride, c->v_row_stride};
  for (int i = 0; i < 3; ++i)
    if (sizes[i] > 1 && (ks[i] <= 0 || vs[i] <= 0)) return FA_EINVAL;
  if (!aligned16(c->k_pages) || !aligned16(c->v_pages) ||
      !strides_vector(ks, sizes, 3) || !strides_vector(vs, sizes, 3) ||
      !aligned4(c->page_table))
    return FA_EALIGN;
  return FA_OK;
}

// 4-D view of 16-bit elements (64 of the innermost a box), 128-byte swizzle;
// what lies outside reads as zero. A dimension of one element takes any
// stride. Rows that follow one another are fetched into L2 by 256 bytes,
// rows with others between them by 128, so that nobody else's are.
int make_map(CUtensorMap *map, const void *base, int dtype, const int (&sizes)[4],
             const int64_t (&strides)[3], int box1, int box3) {
  cuuint64_t dims[4], bytes[3];
  for (int i = 0; i < 4; ++i) dims[i] = static_cast<cuuint64_t>(sizes[i]);
  for (int i = 0; i < 3; ++i)
    bytes[i] = 2 * static_cast<cuuint64_t>(sizes[i + 1] > 1 ? strides[i] : sizes[0]);
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box1), 1,
                             static_cast<cuuint32_t>(box3)};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  return g_encode(map,
                  dtype == FA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                         : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                  4, const_cast<void *>(base), dims, bytes, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  strides[0] == sizes[0] || sizes[0] == 128
                      ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B
                      : CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? FA_OK
             : FA_EINVAL;
}

int check_step(const fa_new_tokens *s) {
  if (!s || !s->starts || !s->seq_lens || s->batch <= 0 || s->tokens <= 0)
    return FA_EINVAL;
  return aligned4(s->starts) && aligned4(s->seq_lens) ? FA_OK : FA_EALIGN;
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" {

int fa_rope(const void *q, const int64_t q_strides[3], void *q_out,
            const void *k, const int64_t k_strides[3], void *k_out, int B,
            int H, int H_kv, int N, int head_dim, const int32_t *positions,
            int64_t position_stride, const double *freqs, int rotary_dim,
            float amplitude, int flags, int dtype, void *stream) {
  if (!dtype_ok(dtype) || (flags & ~(FA_ROPE_INTERLEAVED | FA_ROPE_INVERSE)))
    return FA_EINVAL;
  if (!q || !q_out || !q_strides || !positions || !freqs) return FA_EINVAL;
  if ((k != nullptr) != (k_out != nullptr) || (k && !k_strides)) return FA_EINVAL;
  if (B <= 0 || H <= 0 || N <= 0 || (k && H_kv <= 0) || head_dim <= 0 ||
      head_dim > 1024 || static_cast<long long>(B) * N > INT_MAX ||
      static_cast<long long>(H) + (k ? H_kv : 0) > 65535)
    return FA_EINVAL;
  int rc = check_rotary(head_dim, rotary_dim, amplitude, freqs);
  if (rc != FA_OK) return rc;
  if (!aligned4(positions) || (reinterpret_cast<uintptr_t>(q) & 1u) ||
      (reinterpret_cast<uintptr_t>(q_out) & 1u) ||
      (reinterpret_cast<uintptr_t>(k) & 1u) ||
      (reinterpret_cast<uintptr_t>(k_out) & 1u))
    return FA_EALIGN;
  int dev = 0;
  rc = ensure_device(&dev);
  if (rc != FA_OK) return rc;

  RopeArgs a{};
  a.q = static_cast<const __half *>(q);
  a.q_out = static_cast<__half *>(q_out);
  a.q_sb = q_strides[0];
  a.q_sh = q_strides[1];
  a.q_sn = q_strides[2];
  a.qo_sn = head_dim;
  a.qo_sh = static_cast<int64_t>(N) * head_dim;
  a.qo_sb = a.qo_sh * H;
  a.H = H;
  if (k) {
    a.k = static_cast<const __half *>(k);
    a.k_out = static_cast<__half *>(k_out);
    a.k_sb = k_strides[0];
    a.k_sh = k_strides[1];
    a.k_sn = k_strides[2];
    a.ko_sn = head_dim;
    a.ko_sh = a.qo_sh;
    a.ko_sb = a.ko_sh * H_kv;
    a.H_kv = H_kv;
  }
  a.tokens = B * N;
  a.N = N;
  a.D = head_dim;
  a.rot = rotary_dim;
  a.positions = positions;
  a.position_stride = position_stride;
  a.freqs = freqs;
  a.amplitude = amplitude;
  a.sign = flags & FA_ROPE_INVERSE ? -1.f : 1.f;
  const bool interleaved = (flags & FA_ROPE_INTERLEAVED) != 0;
  const int q_sizes[3] = {B, H, N}, k_sizes[3] = {B, H_kv, N};
  const bool vector = head_dim % 8 == 0 &&
                      rotary_dim % (interleaved ? 8 : 16) == 0 &&
                      aligned16(q) && aligned16(q_out) &&
                      strides_vector(q_strides, q_sizes, 3) &&
                      (!k || (aligned16(k) && aligned16(k_out) &&
                              strides_vector(k_strides, k_sizes, 3)));
  return launch_rope_kernel(a, interleaved, false, vector, dtype,
                            g_devices[dev].sms,
                            static_cast<cudaStream_t>(stream)) == cudaSuccess
             ? FA_OK
             : FA_ECUDA;
}

int fa_append_paged(const void *q, const int64_t q_strides[2], void *q_out,
                    const void *k_new, const int64_t k_strides[2],
                    const void *v_new, const int64_t v_strides[2], int H,
                    const fa_paged_cache *cache, const fa_new_tokens *step,
                    const int32_t *positions, const double *freqs,
                    int rotary_dim, float amplitude, int flags, int dtype,
                    void *stream) {
  if (!dtype_ok(dtype) || (flags & ~FA_ROPE_INTERLEAVED)) return FA_EINVAL;
  int rc = check_cache(cache);
  if (rc != FA_OK) return rc;
  rc = check_step(step);
  if (rc != FA_OK) return rc;
  if (!k_new || !v_new || !k_strides || !v_strides) return FA_EINVAL;
  if ((q != nullptr) != (q_out != nullptr) ||
      (q && (!q_strides || H <= 0 || !freqs)))
    return FA_EINVAL;
  if (static_cast<long long>(q ? H : 0) + 2ll * cache->kv_heads > 65535)
    return FA_EINVAL;
  if (freqs) {
    rc = check_rotary(cache->head_dim, rotary_dim, amplitude, freqs);
    if (rc != FA_OK) return rc;
  }
  if (!aligned4(positions) || (reinterpret_cast<uintptr_t>(q) & 1u) ||
      (reinterpret_cast<uintptr_t>(q_out) & 1u) ||
      (reinterpret_cast<uintptr_t>(k_new) & 1u) ||
      (reinterpret_cast<uintptr_t>(v_new) & 1u))
    return FA_EALIGN;
  int dev = 0;
  rc = ensure_device(&dev);
  if (rc != FA_OK) return rc;

  const fa_paged_cache &c = *cache;
  RopeArgs a{};
  if (q) {
    a.q = static_cast<const __half *>(q);
    a.q_out = static_cast<__half *>(q_out);
    a.q_sn = q_strides[0];
    a.q_sh = q_strides[1];
    a.qo_sn = static_cast<int64_t>(H) * c.head_dim;
    a.qo_sh = c.head_dim;
    a.H = H;
  }
  a.k = static_cast<const __half *>(k_new);
  a.v = static_cast<const __half *>(v_new);
  a.k_sn = k_strides[0];
  a.k_sh = k_strides[1];
  a.v_sn = v_strides[0];
  a.v_sh = v_strides[1];
  a.k_out = static_cast<__half *>(c.k_pages);
  a.v_out = static_cast<__half *>(c.v_pages);
  a.kp_sp = c.k_page_stride;
  a.kp_sh = c.k_head_stride;
  a.kp_sr = c.k_row_stride;
  a.vp_sp = c.v_page_stride;
  a.vp_sh = c.v_head_stride;
  a.vp_sr = c.v_row_stride;
  a.H_kv = c.kv_heads;
  a.tokens = step->tokens;
  a.N = step->tokens;
  a.D = c.head_dim;
  a.rot = freqs ? rotary_dim : 0;
  a.positions = positions;
  a.freqs = freqs;
  a.amplitude = amplitude;
  a.sign = 1.f;
  a.starts = step->starts;
  a.seq_lens = step->seq_lens;
  a.batch = step->batch;
  a.page_table = c.page_table;
  a.table_stride = c.table_stride;
  a.table_width = c.table_width;
  a.page_rows = c.page_rows;
  a.num_pages = c.num_pages;
  const bool interleaved = (flags & FA_ROPE_INTERLEAVED) != 0;
  const int q_sizes[2] = {step->tokens, H}, k_sizes[2] = {step->tokens, c.kv_heads};
  const bool vector = a.rot % (interleaved ? 8 : 16) == 0 &&
                      aligned16(k_new) && aligned16(v_new) &&
                      strides_vector(k_strides, k_sizes, 2) &&
                      strides_vector(v_strides, k_sizes, 2) &&
                      (!q || (aligned16(q) && aligned16(q_out) &&
                              strides_vector(q_strides, q_sizes, 2)));
  return launch_rope_kernel(a, interleaved, true, vector, dtype,
                            g_devices[dev].sms,
                            static_cast<cudaStream_t>(stream)) == cudaSuccess
             ? FA_OK
             : FA_ECUDA;
}

size_t fa_attend_paged_workspace_bytes(int head_dim, int device) {
  if (head_dim != FA_HEAD_DIM && head_dim != 128) return 0;
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) !=
      cudaSuccess)
    return 0;
  return attend_paged_workspace_bytes(head_dim, sms);
}

int fa_attend_paged(const void *q, const int64_t q_strides[2], void *o,
                    float *lse, int H, const fa_paged_cache *cache,
                    const fa_new_tokens *step, float scale, int causal,
                    int dtype, void *workspace, size_t workspace_bytes,
                    uint32_t *counters, size_t counter_count, void *stream) {
  if (!dtype_ok(dtype) || !isfinite(scale)) return FA_EINVAL;
  int rc = check_cache(cache);
  if (rc != FA_OK) return rc;
  rc = check_step(step);
  if (rc != FA_OK) return rc;
  const fa_paged_cache &c = *cache;
  if (!q || !q_strides || !o || !workspace || !counters) return FA_EINVAL;
  if (H <= 0 || H % c.kv_heads != 0 || H / c.kv_heads > 128) return FA_EINVAL;
  if (static_cast<long long>(step->tokens) * H > INT_MAX) return FA_EINVAL;
  const int sizes[2] = {step->tokens, H};
  if ((sizes[0] > 1 && q_strides[0] <= 0) || (sizes[1] > 1 && q_strides[1] <= 0))
    return FA_EINVAL;
  if (!aligned16(q) || !aligned16(o) || !strides_vector(q_strides, sizes, 2) ||
      !aligned16(workspace) || !aligned4(lse) || !aligned4(counters))
    return FA_EALIGN;
  int dev = 0;
  rc = ensure_device(&dev);
  if (rc != FA_OK) return rc;
  const int sms = g_devices[dev].sms;
  if (workspace_bytes < attend_paged_workspace_bytes(c.head_dim, sms) ||
      counter_count < 2 * static_cast<size_t>(sms))
    return FA_ENOSPACE;

  PagedArgs a{};
  a.q = static_cast<const __half *>(q);
  a.q_st = q_strides[0];
  a.q_sh = q_strides[1];
  a.out = static_cast<__half *>(o);
  a.lse = lse;
  a.k_pages = static_cast<const __half *>(c.k_pages);
  a.v_pages = static_cast<const __half *>(c.v_pages);
  a.kp_sp = c.k_page_stride;
  a.kp_sh = c.k_head_stride;
  a.kp_sr = c.k_row_stride;
  a.vp_sp = c.v_page_stride;
  a.vp_sh = c.v_head_stride;
  a.vp_sr = c.v_row_stride;
  a.page_table = c.page_table;
  a.table_stride = c.table_stride;
  a.table_width = c.table_width;
  a.num_pages = c.num_pages;
  a.page_rows = c.page_rows;
  a.starts = step->starts;
  a.seq_lens = step->seq_lens;
  a.batch = step->batch;
  a.tokens = step->tokens;
  a.H = H;
  a.H_kv = c.kv_heads;
  a.D = c.head_dim;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.causal = causal != 0;
  a.partials = static_cast<float *>(workspace);
  a.counters = counters;
  const int form = attend_paged_form(a);
  attend_paged_plan(a, form);
  const int group = H / c.kv_heads;
  const int kv_sizes[4] = {c.head_dim, c.page_rows, c.kv_heads, c.num_pages};
  const int64_t k_str[3] = {c.k_row_stride, c.k_head_stride, c.k_page_stride};
  const int64_t v_str[3] = {c.v_row_stride, c.v_head_stride, c.v_page_stride};
  CUtensorMap tq{}, tk, tv;
  if (make_map(&tk, c.k_pages, dtype, kv_sizes, k_str, a.box_rows, 1) != FA_OK ||
      make_map(&tv, c.v_pages, dtype, kv_sizes, v_str, a.box_rows, 1) != FA_OK)
    return FA_EINVAL;
  if (form == kPagedMany) {
    // (dims, heads of a group, groups, tokens): a box is a tile's rows in
    // the order (token, head)
    const int q_sizes[4] = {c.head_dim, group, c.kv_heads, step->tokens};
    const int64_t q_str[3] = {q_strides[1], q_strides[1] * group, q_strides[0]};
    if (make_map(&tq, q, dtype, q_sizes, q_str, group, a.item_tokens / 2) != FA_OK)
      return FA_EINVAL;
  }
  return launch_attend_paged_kernel(a, form, tq, tk, tv, dtype, sms,
                                    static_cast<cudaStream_t>(stream)) ==
                 cudaSuccess
             ? FA_OK
             : FA_ECUDA;
}

}  // extern "C"
