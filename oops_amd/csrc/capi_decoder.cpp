// C entry points of softmax attention in a decoder (norm and rotation of
// queries and keys, causal attention, the 4-bit key/value cache): host checks,
// then the launchers.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "decoder_kernels.h"
#include "layer_kernels.h"

namespace {

using oops::report;
using oops::report_launch;

bool known_dtype(int dtype) { return dtype == OOPS_F32 || dtype == OOPS_BF16 || dtype == OOPS_F16; }
size_t align256(size_t b) { return (b + 255) / 256 * 256; }
int element(int dtype) { return dtype == OOPS_F32 ? 4 : 2; }
constexpr int64_t kMax31 = (int64_t(1) << 31) - 1;
// a * b * c <= limit, all >= 0
bool fits(int64_t a, int64_t b, int64_t c, int64_t limit) {
  if (a == 0 || b == 0 || c == 0) return true;
  return a <= limit / b && a * b <= limit / c;
}

// ---- norm and rotation
int check_rotary(const oops_rotary_geometry* g) {
  if (!g) return report(OOPS_EINVAL, "rms_norm_rotary geometry is NULL");
  if (!known_dtype(g->dtype)) return report(OOPS_EINVAL, "unknown dtype %lld", g->dtype);
  if (g->size <= 0 || g->size > 256) return report(OOPS_EINVAL, "size must be in 1..256, got %lld", g->size);
  if (g->rotary < 0 || g->rotary > g->size || g->rotary % 2)
    return report(OOPS_EINVAL, "rotary must be even and in 0..size, got %lld", g->rotary);
  if (g->heads[0] <= 0 || g->heads[1] <= 0)
    return report(OOPS_EINVAL, "heads must be positive, got %lld and %lld", g->heads[0], g->heads[1]);
  if (g->batch < 0 || g->length < 0 || g->table_rows < 0 ||
      !fits(g->batch, g->length, std::max(g->heads[0], g->heads[1]), kMax31))
    return report(OOPS_EINVAL, "batch (%lld) x length (%lld) x heads must be in 0..2^31-1", g->batch, g->length);
  if (g->batch * g->length > 0 && g->table_rows < 1) return report(OOPS_EINVAL, "the table has no rows");
  for (const auto& operand : g->stride)
    for (const auto& side : operand)
      for (int64_t s : side)
        if (s < 0) return report(OOPS_EINVAL, "an operand has a negative stride");
  return OOPS_OK;
}
size_t rotary_parts_bytes(const oops_rotary_geometry& g) {
  return align256((size_t)oops::rotary_parts(g) * (size_t)g.size * sizeof(float));
}

// ---- causal attention
// strides of dimensions of one element are nobody's
oops_causal_geometry with_strides(oops_causal_geometry g) {
  for (int i = 0; i < OOPS_CA_OPERANDS; ++i) {
    const bool kv = i == OOPS_CA_K || i == OOPS_CA_V || i == OOPS_CA_DK || i == OOPS_CA_DV;
    if (g.batch <= 1) g.stride[i][0] = 0;
    if ((kv ? g.kv_heads : g.heads) <= 1) g.stride[i][1] = 0;
    if (g.length <= 1) g.stride[i][2] = 0;
  }
  return g;
}
int check_causal(const oops_causal_geometry* g, bool offsets) {
  if (!g) return report(OOPS_EINVAL, "causal attention geometry is NULL");
  if (!known_dtype(g->dtype)) return report(OOPS_EINVAL, "unknown dtype %lld", g->dtype);
  if (g->kv_heads <= 0 || g->heads <= 0 || g->heads % g->kv_heads)
    return report(OOPS_EINVAL, "heads (%lld) must be a positive multiple of kv_heads (%lld)", g->heads, g->kv_heads);
  const int el = element(g->dtype);
  if (g->key_size <= 0 || g->key_size > 128 || g->value_size <= 0 || g->value_size > 128 || g->key_size * el % 16 ||
      g->value_size * el % 16)
    return report(OOPS_EINVAL, "key_size and value_size must be in 1..128 and of whole 16-byte pieces, got %lld and %lld",
                  g->key_size, g->value_size);
  if (g->batch < 0 || g->length < 0 || g->length > kMax31 - 256 || !fits(g->batch, g->heads, (g->length + 127) / 128, 1 << 24))
    return report(OOPS_EINVAL, "batch (%lld) x heads x blocks of 128 tokens (%lld tokens) must be at most 2^24", g->batch,
                  g->length);
  if (offsets && (g->sequences < 0 || g->sequences > kMax31 - 1))
    return report(OOPS_EINVAL, "sequences must not be negative, got %lld", g->sequences);
  const oops_causal_geometry own = with_strides(*g);
  for (const auto& s : own.stride) {
    if (s[0] < 0 || s[1] < 0 || s[2] < 0) return report(OOPS_EINVAL, "an operand has a negative stride");
    if (s[2] * el >= (1 << 24)) return report(OOPS_EINVAL, "tokens must be less than 2^24 bytes apart, got %lld elements", s[2]);
    if (s[0] * el % 16 || s[1] * el % 16 || s[2] * el % 16) return report(OOPS_EINVAL, "strides must be of whole 16-byte pieces");
  }
  return OOPS_OK;
}
bool aligned(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}
void set3(int64_t (&to)[3], const int64_t (&from)[3]) { std::copy(from, from + 3, to); }
oops::CausalArgs causal_args(const oops_causal_geometry& given, const void* q, const void* k, const void* v, const void* offsets) {
  const oops_causal_geometry g = with_strides(given);
  oops::CausalArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.offsets = offsets;
  set3(a.q_stride, g.stride[OOPS_CA_Q]);
  set3(a.k_stride, g.stride[OOPS_CA_K]);
  set3(a.v_stride, g.stride[OOPS_CA_V]);
  set3(a.o_stride, g.stride[OOPS_CA_O]);
  set3(a.do_stride, g.stride[OOPS_CA_DO]);
  set3(a.dq_stride, g.stride[OOPS_CA_DQ]);
  set3(a.dk_stride, g.stride[OOPS_CA_DK]);
  set3(a.dv_stride, g.stride[OOPS_CA_DV]);
  a.batch = g.batch;
  a.length = g.length;
  a.heads = g.heads;
  a.kv_heads = g.kv_heads;
  a.group = g.heads / g.kv_heads;
  a.key_size = g.key_size;
  a.value_size = g.value_size;
  a.sequences = g.sequences;
  a.offsets_i64 = g.offsets_i64;
  a.flip = std::signbit(g.scale);
  a.scale = std::fabs(g.scale);
  a.parts = a.key_splits = a.query_splits = 1;
  a.blocks = (int32_t)((g.length + 127) / 128);
  return a;
}
size_t stat_bytes(const oops_causal_geometry& g) { return align256((size_t)(g.batch * g.heads * g.length) * sizeof(float)); }
size_t order_bytes(const oops_causal_geometry& g) {
  return g.sequences > 0 && oops::causal_ordered(g) ? align256((size_t)((g.length + 127) / 128) * 2 * sizeof(int32_t)) : 0;
}
size_t part_bytes(const oops_causal_geometry& g, int heads, int parts, int size) {
  return parts > 1 ? align256((size_t)(g.batch * heads * g.length) * size * parts * sizeof(float)) : 0;
}
// parts of the queries' keys, and of the keys' queries
int key_splits(const oops_causal_geometry& g) { return oops::causal_splits(g, (g.length + 127) / 128 * g.batch * g.heads); }
int query_splits(const oops_causal_geometry& g) {
  return oops::causal_splits(g, (g.length + 127) / 128 * g.batch * g.kv_heads * oops::causal_grad_parts(g));
}

// ---- cache
int check_cache_shape(int dtype, int heads, int size, int page, int64_t pages) {
  if (!known_dtype(dtype)) return report(OOPS_EINVAL, "unknown dtype %lld", dtype);
  if (heads <= 0) return report(OOPS_EINVAL, "heads must be positive, got %lld", heads);
  if (size <= 0 || size > 128 || size % 32) return report(OOPS_EINVAL, "size must be 32, 64, 96 or 128, got %lld", size);
  if (page <= 0 || page % 16 || page > (1 << 20)) return report(OOPS_EINVAL, "page must be a multiple of 16 up to 2^20, got %lld", page);
  if (pages < 0 || !fits(pages, page, 1, kMax31)) return report(OOPS_EINVAL, "pages (%lld) x page (%lld) must be in 0..2^31-1", pages, page);
  return OOPS_OK;
}
int check_cache(const oops_cache_geometry* g) {
  if (!g) return report(OOPS_EINVAL, "cache geometry is NULL");
  if (int rc = check_cache_shape(g->dtype, g->heads, g->size, g->page, g->pages)) return rc;
  if (g->heads > (1 << 16)) return report(OOPS_EINVAL, "heads must be at most 2^16, got %lld", g->heads);
  if (g->batch < 0 || g->length < 0 || !fits(g->batch, g->length, (int64_t)g->heads * (g->size / 4), int64_t(1) << 31))
    return report(OOPS_EINVAL, "batch (%lld) x length (%lld) tokens are too many for one call", g->batch, g->length);
  for (const auto& operand : g->stride)
    for (int64_t s : operand)
      if (s < 0) return report(OOPS_EINVAL, "an operand has a negative stride");
  return OOPS_OK;
}
int check_cache_attn(const oops_cache_attn_geometry* g) {
  if (!g) return report(OOPS_EINVAL, "cache attention geometry is NULL");
  if (g->kv_heads <= 0 || g->heads <= 0 || g->heads % g->kv_heads)
    return report(OOPS_EINVAL, "heads (%lld) must be a positive multiple of kv_heads (%lld)", g->heads, g->kv_heads);
  if (int rc = check_cache_shape(g->dtype, g->kv_heads, g->size, g->page, g->pages)) return rc;
  if (g->batch < 0 || g->max_pages < 0 || !fits(g->max_pages, g->page, 1, kMax31 - 256) || !fits(g->batch, g->heads, 256, 1 << 30))
    return report(OOPS_EINVAL, "batch (%lld) x heads must be at most 2^22 and max_pages (%lld) x page below 2^31", g->batch,
                  g->max_pages);
  if (g->stride[0] < 0 || g->stride[1] < 0) return report(OOPS_EINVAL, "the query has a negative stride");
  return OOPS_OK;
}

}  // namespace

extern "C" {

int oops_rms_norm_rotary_forward(const oops_rotary_geometry* geo, const void* query, const void* key,
                                 const void* query_weight, const void* key_weight, const float* table,
                                 const void* positions, void* query_out, void* key_out, void* stream) {
  oops::clear_report();
  if (int rc = check_rotary(geo)) return rc;
  if (geo->batch * geo->length == 0) return OOPS_OK;
  if (!query || !key || !query_out || !key_out || (geo->rotary > 0 && !table))
    return report(OOPS_EINVAL, "query, key, their outputs and the table must be non-NULL");
  return report_launch(oops::launch_rotary_forward(*geo, {query, key}, {query_weight, key_weight}, table, positions,
                                                   {query_out, key_out}, static_cast<hipStream_t>(stream)),
                       "rms_norm_rotary forward");
}

size_t oops_rms_norm_rotary_backward_workspace_bytes(const oops_rotary_geometry* geo) {
  oops::clear_report();
  if (check_rotary(geo)) return 0;
  return 2 * rotary_parts_bytes(*geo);
}

int oops_rms_norm_rotary_backward(const oops_rotary_geometry* geo, const void* query, const void* key,
                                  const void* query_weight, const void* key_weight, const float* table,
                                  const void* positions, const void* grad_query_out, const void* grad_key_out,
                                  void* grad_query, void* grad_key, void* grad_query_weight, void* grad_key_weight,
                                  void* workspace, size_t ws_bytes, void* stream) {
  oops::clear_report();
  if (int rc = check_rotary(geo)) return rc;
  if (geo->batch * geo->length == 0) return report(OOPS_EINVAL, "the backward needs tokens");
  if (!query || !key || (geo->rotary > 0 && !table)) return report(OOPS_EINVAL, "query, key and the table must be non-NULL");
  if ((!grad_query_out && (grad_query || grad_query_weight)) || (!grad_key_out && (grad_key || grad_key_weight)))
    return report(OOPS_EINVAL, "a gradient of the inputs needs that of the output");
  const bool weights = grad_query_weight || grad_key_weight;
  if (weights)
    if (int rc = oops::report_workspace(workspace, ws_bytes, oops_rms_norm_rotary_backward_workspace_bytes(geo))) return rc;
  float* first = static_cast<float*>(workspace);
  float* second = weights ? first + rotary_parts_bytes(*geo) / sizeof(float) : nullptr;
  return report_launch(
      oops::launch_rotary_backward(*geo, {query, key}, {query_weight, key_weight}, table, positions,
                                   {grad_query_out, grad_key_out}, {grad_query, grad_key},
                                   {grad_query_weight ? first : nullptr, grad_key_weight ? second : nullptr},
                                   {grad_query_weight, grad_key_weight}, static_cast<hipStream_t>(stream)),
      "rms_norm_rotary backward");
}

size_t oops_causal_attn_forward_workspace_bytes(const oops_causal_geometry* geo) {
  oops::clear_report();
  if (check_causal(geo, true)) return 0;
  const int splits = key_splits(*geo);
  return order_bytes(*geo) + part_bytes(*geo, geo->heads, splits, geo->value_size) + part_bytes(*geo, geo->heads, splits, 2);
}

int oops_causal_attn_forward(const oops_causal_geometry* geo, const void* q, const void* k, const void* v,
                             const void* offsets, void* out, void* out_low, float* lse, void* workspace, size_t ws_bytes,
                             void* stream) {
  oops::clear_report();
  if (int rc = check_causal(geo, offsets)) return rc;
  if (geo->batch * geo->length == 0) return OOPS_OK;
  if (!q || !k || !v || !out) return report(OOPS_EINVAL, "q, k, v and out must be non-NULL");
  if (!aligned({q, k, v, out, out_low})) return report(OOPS_EINVAL, "operands must lie at multiples of 16 bytes");
  const size_t order = offsets ? order_bytes(*geo) : 0;
  if (int rc = oops::report_workspace(workspace, ws_bytes, oops_causal_attn_forward_workspace_bytes(geo))) return rc;
  oops::CausalArgs a = causal_args(*geo, q, k, v, offsets);
  a.out = out;
  a.low = geo->dtype == OOPS_F32 ? nullptr : out_low;
  a.lse = lse;
  a.key_splits = key_splits(*geo);
  char* ws = static_cast<char*>(workspace) + order_bytes(*geo);
  a.o_parts = reinterpret_cast<float*>(ws);
  a.stat_parts = reinterpret_cast<float*>(ws + part_bytes(*geo, geo->heads, a.key_splits, geo->value_size));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e = hipSuccess;
  if (order) {
    e = oops::launch_causal_order(a, static_cast<int32_t*>(workspace), st);
    a.order = static_cast<int32_t*>(workspace);
  }
  if (e == hipSuccess) e = oops::launch_causal_forward(geo->dtype, a, st);
  return report_launch(e, "causal attention forward");
}

size_t oops_causal_attn_backward_workspace_bytes(const oops_causal_geometry* geo) {
  oops::clear_report();
  if (check_causal(geo, true)) return 0;
  const int parts = oops::causal_grad_parts(*geo) * query_splits(*geo);
  return order_bytes(*geo) + 2 * stat_bytes(*geo) + part_bytes(*geo, geo->heads, key_splits(*geo), geo->key_size) +
         part_bytes(*geo, geo->kv_heads, parts, geo->key_size) + part_bytes(*geo, geo->kv_heads, parts, geo->value_size);
}

int oops_causal_attn_backward(const oops_causal_geometry* geo, const void* q, const void* k, const void* v,
                              const void* offsets, const void* out, const void* out_low, const float* lse,
                              const void* grad_out, void* grad_q, void* grad_k, void* grad_v, void* workspace,
                              size_t ws_bytes, void* stream) {
  oops::clear_report();
  if (int rc = check_causal(geo, offsets)) return rc;
  if (geo->batch * geo->length == 0) return OOPS_OK;
  if (!q || !k || !v || !out || !lse || !grad_out) return report(OOPS_EINVAL, "q, k, v, out, lse and grad_out must be non-NULL");
  if (!aligned({q, k, v, out, out_low, grad_out, grad_q, grad_k, grad_v}))
    return report(OOPS_EINVAL, "operands must lie at multiples of 16 bytes");
  if (int rc = oops::report_workspace(workspace, ws_bytes, oops_causal_attn_backward_workspace_bytes(geo))) return rc;
  oops::CausalArgs a = causal_args(*geo, q, k, v, offsets);
  a.out = const_cast<void*>(out);
  a.low = geo->dtype == OOPS_F32 ? nullptr : const_cast<void*>(out_low);
  a.lse = const_cast<float*>(lse);
  a.dout = grad_out;
  a.dq = grad_q;
  a.dk = grad_k;
  a.dv = grad_v;
  a.parts = oops::causal_grad_parts(*geo);
  a.query_splits = query_splits(*geo);
  a.key_splits = grad_q ? key_splits(*geo) : 1;
  char* ws = static_cast<char*>(workspace);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e = hipSuccess;
  if (offsets && order_bytes(*geo)) {
    e = oops::launch_causal_order(a, reinterpret_cast<int32_t*>(ws), st);
    a.order = reinterpret_cast<int32_t*>(ws);
  }
  ws += order_bytes(*geo);
  a.neg_lse = reinterpret_cast<float*>(ws);
  a.neg_delta = reinterpret_cast<float*>(ws += stat_bytes(*geo));
  a.dq_parts = reinterpret_cast<float*>(ws += stat_bytes(*geo));
  a.dk_parts = reinterpret_cast<float*>(ws += part_bytes(*geo, geo->heads, key_splits(*geo), geo->key_size));
  a.dv_parts = reinterpret_cast<float*>(ws + part_bytes(*geo, geo->kv_heads, a.parts * a.query_splits, geo->key_size));
  if (e == hipSuccess) e = oops::launch_causal_backward(geo->dtype, a, st);
  return report_launch(e, "causal attention backward");
}

size_t oops_cache_write_workspace_bytes(const oops_cache_geometry* geo) {
  oops::clear_report();
  if (check_cache(geo)) return 0;
  return oops::cache_write_workspace_bytes(*geo);
}

int oops_cache_write(const oops_cache_geometry* geo, void* codes, void* scales, const void* key, const void* value,
                     const void* slots, void* workspace, size_t ws_bytes, void* stream) {
  oops::clear_report();
  if (int rc = check_cache(geo)) return rc;
  if (geo->batch * geo->length == 0 || geo->pages == 0) return OOPS_OK;
  if (!codes || !scales || !key || !value || !slots)
    return report(OOPS_EINVAL, "codes, scales, key, value and slots must be non-NULL");
  if (!aligned({codes})) return report(OOPS_EINVAL, "codes must lie at a multiple of 16 bytes");
  if (int rc = oops::report_workspace(workspace, ws_bytes, oops::cache_write_workspace_bytes(*geo))) return rc;
  return report_launch(oops::launch_cache_write(*geo, codes, scales, key, value, slots, workspace, static_cast<hipStream_t>(stream)),
                       "cache_write");
}

int oops_cache_read(const oops_cache_geometry* geo, const void* codes, const void* scales, const void* slots, void* key,
                    void* value, void* stream) {
  oops::clear_report();
  if (int rc = check_cache(geo)) return rc;
  if (geo->batch * geo->length == 0) return OOPS_OK;
  if ((geo->pages > 0 && (!codes || !scales)) || !key || !value || !slots)
    return report(OOPS_EINVAL, "codes, scales, key, value and slots must be non-NULL");
  if (!aligned({codes, key, value})) return report(OOPS_EINVAL, "codes, key and value must lie at multiples of 16 bytes");
  for (const auto& operand : geo->stride)
    for (int64_t s : operand)
      if (s % 8) return report(OOPS_EINVAL, "the results' strides must be of whole blocks of eight elements");
  return report_launch(oops::launch_cache_read(*geo, codes, scales, slots, key, value, static_cast<hipStream_t>(stream)), "cache_read");
}

size_t oops_cache_attn_workspace_bytes(const oops_cache_attn_geometry* geo) {
  oops::clear_report();
  if (check_cache_attn(geo)) return 0;
  return oops::cache_attn_workspace_bytes(*geo);
}

int oops_cache_attn(const oops_cache_attn_geometry* geo, const void* query, const void* codes, const void* scales,
                    const int32_t* table, const void* lengths, void* out, void* workspace, size_t ws_bytes,
                    void* stream) {
  oops::clear_report();
  if (int rc = check_cache_attn(geo)) return rc;
  if (geo->batch == 0) return OOPS_OK;
  if (!query || !lengths || !out || (geo->pages > 0 && (!codes || !scales)) || (geo->max_pages > 0 && !table))
    return report(OOPS_EINVAL, "query, codes, scales, table, lengths and out must be non-NULL");
  if (!aligned({codes})) return report(OOPS_EINVAL, "codes must lie at a multiple of 16 bytes");
  if (int rc = oops::report_workspace(workspace, ws_bytes, oops::cache_attn_workspace_bytes(*geo))) return rc;
  return report_launch(oops::launch_cache_attn(*geo, query, codes, scales, table, lengths, out, workspace,
                                               static_cast<hipStream_t>(stream)),
                       "cache_attention");
}

}  // extern "C"
