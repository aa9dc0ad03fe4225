// Operators of softmax attention in a decoder: launchers behind the
// oops_rms_norm_rotary_*, oops_causal_attn_* and oops_cache_* C entry points.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/oops_amd.h"

namespace oops {

// ---- rotary.hip
hipError_t launch_rotary_forward(const oops_rotary_geometry& g, const void* const (&x)[2], const void* const (&weight)[2],
                                 const float* table, const void* positions, void* const (&y)[2], hipStream_t stream);
int rotary_parts(const oops_rotary_geometry& g);  // rows of each side's weight-gradient partials
hipError_t launch_rotary_backward(const oops_rotary_geometry& g, const void* const (&x)[2], const void* const (&weight)[2],
                                  const float* table, const void* positions, const void* const (&dy)[2],
                                  void* const (&dx)[2], float* const (&parts)[2], void* const (&dweight)[2],
                                  hipStream_t stream);

// ---- causal_attn.hip, causal_attn_bwd.hip
struct CausalArgs {
  const void *q, *k, *v, *offsets, *dout;
  void *out, *low, *dq, *dk, *dv;
  float* lse;          // (batch, heads, length), log2 units
  float *neg_lse, *neg_delta;  // the same shape: -lse over the scores' factor, -delta
  const int32_t* order;        // blocks of queries, then of keys, the heaviest first (NULL: by their place)
  float *o_parts, *dq_parts, *dk_parts, *dv_parts;
  float* stat_parts;           // of o_parts: maximum and sum (-1: a row without keys)
  int64_t q_stride[3], k_stride[3], v_stride[3], o_stride[3], do_stride[3], dq_stride[3], dk_stride[3], dv_stride[3];
  int64_t batch, length;
  int32_t heads, kv_heads, group, key_size, value_size, sequences, offsets_i64;
  int32_t flip;        // the scale is negative: `scale` is its magnitude, and the scores' sign is changed
  float scale;
  int32_t parts;       // of the query heads of a group in the key/value gradient
  int32_t key_splits;   // of a block of queries' keys, in the forward or the queries' gradient
  int32_t query_splits; // of a block of keys' queries
  int32_t blocks;       // of 128 tokens
};
bool causal_ordered(const oops_causal_geometry& g);
hipError_t launch_causal_order(const CausalArgs& a, int32_t* order, hipStream_t stream);
hipError_t launch_causal_forward(int dtype, const CausalArgs& a, hipStream_t stream);
int causal_grad_parts(const oops_causal_geometry& g);
int causal_splits(const oops_causal_geometry& g, int64_t workgroups);
hipError_t launch_causal_backward(int dtype, const CausalArgs& a, hipStream_t stream);

// ---- cache.hip
hipError_t launch_cache_write(const oops_cache_geometry& g, void* codes, void* scales, const void* key, const void* value,
                              const void* slots, void* workspace, hipStream_t stream);
size_t cache_write_workspace_bytes(const oops_cache_geometry& g);
hipError_t launch_cache_read(const oops_cache_geometry& g, const void* codes, const void* scales, const void* slots,
                             void* key, void* value, hipStream_t stream);
size_t cache_attn_workspace_bytes(const oops_cache_attn_geometry& g);
hipError_t launch_cache_attn(const oops_cache_attn_geometry& g, const void* query, const void* codes, const void* scales,
                             const int32_t* pages, const void* lengths, void* out, void* workspace, hipStream_t stream);

}  // namespace oops
