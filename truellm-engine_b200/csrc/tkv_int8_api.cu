// tkv_int8_api.cu -- the extern "C" boundary of the paged int8 cache and of the
// rotary step (declared in include/truellm_kivi.h): argument validation and
// launches.  Nothing here allocates device memory or synchronises the host.
#include <limits.h>
#include <math.h>
#include <string.h>

#include "tkv_int8.cuh"

using namespace tkv;

namespace {

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool half_type(int t) { return t == TKV_F16 || t == TKV_BF16; }
// strides of 16-byte vectors of 16-bit elements
bool vec_strides(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || s[i] % 8 != 0) return false;
  return true;
}
bool cache_ok(const tkv_int8_cache_t* c) {
  return c && c->pool && al16(c->pool) && c->num_pages > 0 && c->n_kv_heads > 0 &&
         (c->head_dim == 64 || c->head_dim == 128);
}

}  // namespace

extern "C" {

int tkv_rope_plan_init(tkv_rope_plan_t* plan, int rotary_dim, double theta,
                       const int32_t* sections, int n_axes, int order, int pairing) {
  if (!plan || !sections) return TKV_INVALID_ARGUMENT;
  if (rotary_dim <= 0 || rotary_dim % 16 != 0 || rotary_dim > 2 * TKV_ROPE_MAX_PAIRS)
    return TKV_NOT_IMPLEMENTED;
  if (n_axes < 1 || n_axes > TKV_ROPE_MAX_AXES || !(theta > 0.) || !isfinite(theta))
    return TKV_INVALID_ARGUMENT;
  if ((order != TKV_ROPE_BLOCKS && order != TKV_ROPE_ROUND_ROBIN) ||
      (pairing != TKV_ROPE_HALVES && pairing != TKV_ROPE_ADJACENT))
    return TKV_INVALID_ARGUMENT;
  const int pairs = rotary_dim / 2;
  int left[TKV_ROPE_MAX_AXES];
  long long sum = 0;
  for (int a = 0; a < n_axes; ++a) {
    if (sections[a] < 0) return TKV_INVALID_ARGUMENT;
    left[a] = sections[a];
    sum += sections[a];
  }
  if (sum != pairs) return TKV_INVALID_ARGUMENT;
  memset(plan, 0, sizeof(*plan));
  plan->rotary_dim = rotary_dim;
  plan->n_axes = n_axes;
  plan->pairing = pairing;
  for (int i = 0, a = 0; i < pairs; ++i) {
    while (left[a] == 0) a = (a + 1) % n_axes;
    --left[a];
    plan->axis[i] = static_cast<uint8_t>(a);
    if (order == TKV_ROPE_ROUND_ROBIN) a = (a + 1) % n_axes;
    plan->turns[i] = pow(theta, -2.0 * i / rotary_dim) / 6.283185307179586476925286766559;
  }
  return TKV_OK;
}

int tkv_rope_axes(const tkv_rope_plan_t* plan, const void* q, const void* k, void* q_out,
                  void* k_out, int dtype, int num_q_heads, int num_k_heads, int head_dim,
                  int n_tokens, const int64_t* strides, const int32_t* positions,
                  int64_t axis_stride, int inverse, void* stream) {
  if (!plan || !strides) return TKV_INVALID_ARGUMENT;
  if (!half_type(dtype)) return TKV_NOT_IMPLEMENTED;
  const int r = plan->rotary_dim;
  if (r <= 0 || r % 16 != 0 || r > 2 * TKV_ROPE_MAX_PAIRS || plan->n_axes < 1 ||
      plan->n_axes > TKV_ROPE_MAX_AXES ||
      (plan->pairing != TKV_ROPE_HALVES && plan->pairing != TKV_ROPE_ADJACENT))
    return TKV_INVALID_ARGUMENT;
  for (int i = 0; i < r / 2; ++i)
    if (plan->axis[i] >= plan->n_axes || !isfinite(plan->turns[i])) return TKV_INVALID_ARGUMENT;
  if (head_dim < r || head_dim % 8 != 0) return TKV_INVALID_ARGUMENT;
  if (head_dim > 512) return TKV_NOT_IMPLEMENTED;
  if (num_q_heads < 0 || num_k_heads < 0 || n_tokens < 0) return TKV_INVALID_ARGUMENT;
  if (n_tokens == 0 || num_q_heads + static_cast<long long>(num_k_heads) == 0) return TKV_OK;
  if (num_q_heads + static_cast<long long>(num_k_heads) > INT_MAX) return TKV_INVALID_ARGUMENT;
  if (!positions || axis_stride < 0 || !vec_strides(strides, 8)) return TKV_INVALID_ARGUMENT;
  if (num_q_heads && (!q || !q_out || !al16(q) || !al16(q_out))) return TKV_INVALID_ARGUMENT;
  if (num_k_heads && (!k || !k_out || !al16(k) || !al16(k_out))) return TKV_INVALID_ARGUMENT;
  RopeArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_out = static_cast<uint16_t*>(k_out);
  a.q_t = strides[0], a.q_h = strides[1], a.k_t = strides[2], a.k_h = strides[3];
  a.qo_t = strides[4], a.qo_h = strides[5], a.ko_t = strides[6], a.ko_h = strides[7];
  a.hq = num_q_heads;
  a.hk = num_k_heads;
  a.head_dim = head_dim;
  a.n_tokens = n_tokens;
  a.inverse = inverse ? 1 : 0;
  a.positions = positions;
  a.axis_stride = axis_stride;
  return launch_rope(*plan, a, dtype == TKV_BF16, static_cast<cudaStream_t>(stream));
}

int64_t tkv_int8_page_bytes(int head_dim) {
  return head_dim == 128 ? Int8Fmt<128>::BYTES : head_dim == 64 ? Int8Fmt<64>::BYTES : 0;
}

int tkv_int8_append(const tkv_int8_cache_t* cache, const void* k_new, const void* v_new,
                    int in_dtype, const int64_t* strides, const int32_t* cu_new,
                    const int32_t* seq_lens_old, const int32_t* block_tables,
                    int max_blocks_per_seq, int num_seqs, int total_new_tokens,
                    int max_new_tokens, int* err_flag, void* stream) {
  if (!cache_ok(cache)) return TKV_INVALID_ARGUMENT;
  if (!half_type(in_dtype)) return TKV_NOT_IMPLEMENTED;
  if (num_seqs < 0 || total_new_tokens < 0 || max_new_tokens < 0 || max_blocks_per_seq <= 0)
    return TKV_INVALID_ARGUMENT;
  if (num_seqs == 0 || total_new_tokens == 0 || max_new_tokens == 0) return TKV_OK;
  if (!k_new || !v_new || !strides || !cu_new || !seq_lens_old || !block_tables)
    return TKV_INVALID_ARGUMENT;
  if (!al16(k_new) || !al16(v_new) || !vec_strides(strides, 4)) return TKV_INVALID_ARGUMENT;
  Int8AppendArgs a;
  a.pool = static_cast<uint8_t*>(cache->pool);
  a.num_pages = cache->num_pages;
  a.n_kv_heads = cache->n_kv_heads;
  a.k = static_cast<const uint16_t*>(k_new);
  a.v = static_cast<const uint16_t*>(v_new);
  a.k_t = strides[0], a.k_h = strides[1], a.v_t = strides[2], a.v_h = strides[3];
  a.cu = cu_new;
  a.lens_old = seq_lens_old;
  a.block_tables = block_tables;
  a.max_blocks = max_blocks_per_seq;
  a.num_seqs = num_seqs;
  a.total = total_new_tokens;
  a.max_new = max_new_tokens;
  a.err = err_flag;
  return launch_int8_append(a, cache->head_dim, in_dtype == TKV_BF16,
                            static_cast<cudaStream_t>(stream));
}

int tkv_int8_read(const tkv_int8_cache_t* cache, void* k_out, void* v_out, int out_dtype,
                  const int32_t* block_tables, int max_blocks_per_seq, const int32_t* starts,
                  const int32_t* cu, int num_seqs, int total_tokens, int max_tokens,
                  int* err_flag, void* stream) {
  if (!cache_ok(cache)) return TKV_INVALID_ARGUMENT;
  if (!half_type(out_dtype) && out_dtype != TKV_F32) return TKV_NOT_IMPLEMENTED;
  if (num_seqs < 0 || total_tokens < 0 || max_tokens < 0 || max_blocks_per_seq <= 0)
    return TKV_INVALID_ARGUMENT;
  if (num_seqs == 0 || total_tokens == 0 || max_tokens == 0) return TKV_OK;
  if ((!k_out && !v_out) || !block_tables || !starts || !cu) return TKV_INVALID_ARGUMENT;
  if (!al16(k_out) || !al16(v_out)) return TKV_INVALID_ARGUMENT;
  Int8ReadArgs a;
  a.pool = static_cast<const uint8_t*>(cache->pool);
  a.num_pages = cache->num_pages;
  a.n_kv_heads = cache->n_kv_heads;
  a.k_out = k_out;
  a.v_out = v_out;
  a.block_tables = block_tables;
  a.max_blocks = max_blocks_per_seq;
  a.starts = starts;
  a.cu = cu;
  a.num_seqs = num_seqs;
  a.total = total_tokens;
  a.max_tokens = max_tokens;
  a.err = err_flag;
  return launch_int8_read(a, cache->head_dim, out_dtype, static_cast<cudaStream_t>(stream));
}

static bool attend_sizes_ok(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                            int max_q_tokens, int max_context_len) {
  return num_seqs >= 0 && num_seqs <= 65535 && num_q_heads > 0 && num_kv_heads > 0 &&
         num_q_heads % num_kv_heads == 0 && (head_dim == 64 || head_dim == 128) &&
         max_q_tokens >= 0 && max_context_len >= 0 && max_context_len <= INT_MAX - 1024 &&
         static_cast<long long>(max_q_tokens) * (num_q_heads / num_kv_heads) < 1ll << 30;
}

size_t tkv_int8_attend_workspace_bytes(int num_seqs, int num_q_heads, int num_kv_heads,
                                       int head_dim, int max_q_tokens, int max_context_len) {
  if (!attend_sizes_ok(num_seqs, num_q_heads, num_kv_heads, head_dim, max_q_tokens,
                       max_context_len))
    return 0;
  return int8_attend_workspace(num_seqs, num_q_heads, num_kv_heads, head_dim, max_q_tokens,
                               max_context_len);
}

int tkv_int8_attend(const tkv_int8_cache_t* cache, const void* q, int q_dtype,
                    const int64_t* q_stride, void* out, int out_dtype, const int32_t* cu_q,
                    const int32_t* block_tables, int max_blocks_per_seq, const int32_t* seq_lens,
                    int num_seqs, int num_q_heads, int total_q_tokens, int max_q_tokens,
                    int max_context_len, int window, float scale, void* workspace,
                    size_t workspace_bytes, int* err_flag, void* stream) {
  if (!cache_ok(cache)) return TKV_INVALID_ARGUMENT;
  if (!half_type(q_dtype) || !half_type(out_dtype)) return TKV_NOT_IMPLEMENTED;
  if (!attend_sizes_ok(num_seqs, num_q_heads, cache->n_kv_heads, cache->head_dim, max_q_tokens,
                       max_context_len) ||
      total_q_tokens < 0 || max_blocks_per_seq <= 0 || window < 0 || !(scale > 0.f) ||
      !isfinite(scale * 1.4426950408889634f))
    return TKV_INVALID_ARGUMENT;
  if (num_seqs == 0 || total_q_tokens == 0 || max_q_tokens == 0) return TKV_OK;
  if (!q || !q_stride || !out || !cu_q || !block_tables || !seq_lens || !workspace)
    return TKV_INVALID_ARGUMENT;
  if (!al16(q) || !al16(out) || !al16(workspace) || !vec_strides(q_stride, 2))
    return TKV_INVALID_ARGUMENT;
  if (workspace_bytes < int8_attend_workspace(num_seqs, num_q_heads, cache->n_kv_heads,
                                              cache->head_dim, max_q_tokens, max_context_len))
    return TKV_INVALID_ARGUMENT;
  Int8AttendArgs a;
  a.pool = static_cast<const uint8_t*>(cache->pool);
  a.num_pages = cache->num_pages;
  a.n_kv_heads = cache->n_kv_heads;
  a.q = static_cast<const uint16_t*>(q);
  a.q_t = q_stride[0];
  a.q_h = q_stride[1];
  a.q_bf16 = q_dtype == TKV_BF16;
  a.out = static_cast<uint16_t*>(out);
  a.out_bf16 = out_dtype == TKV_BF16;
  a.cu_q = cu_q;
  a.block_tables = block_tables;
  a.max_blocks = max_blocks_per_seq;
  a.seq_lens = seq_lens;
  a.num_seqs = num_seqs;
  a.num_q_heads = num_q_heads;
  a.grp = num_q_heads / cache->n_kv_heads;
  a.total_q = total_q_tokens;
  a.max_q = max_q_tokens;
  a.max_len = max_context_len;
  a.window = window;
  a.alpha = scale * 1.4426950408889634f;
  a.err = err_flag;
  return launch_int8_attend(a, cache->head_dim, workspace, workspace_bytes,
                            static_cast<cudaStream_t>(stream));
}

}  // extern "C"
