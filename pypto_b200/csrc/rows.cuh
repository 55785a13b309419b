// Parameter blocks of the row kernels (rows.cu): norm and rotation of heads, rows into a quantised cache and back.
#pragma once
#include "common.cuh"

namespace pto {

// one of the two tensors [t, heads, d] of a norm_rope call; strides in elements
struct NormRopeSide {
  const void* in;
  void* out;
  const void* weight;  // [d] or null: no norm
  int64_t in_token, in_head, out_token, out_head;
  int64_t warps;      // of the launch that work on it
  int heads, d;
  int lanes;          // a head
  int split;          // warps that share the heads of a token
  int rotation_only;  // in place and without a norm
};
struct NormRopeParams {
  NormRopeSide side[2];
  const void* positions;   // int32 or int64 [t]
  const uint64_t* turns;   // [rotary/2]: turns a position, a binary fraction of 64 bits
  float amplitude, eps;
  int positions64, rotary, rope_last;
};
void norm_rope_plan(NormRopeSide* s, int64_t t, int num_sms);
cudaError_t launch_norm_rope(const NormRopeParams& p, int dtype, int layout, cudaStream_t stream);

struct KvWriteParams {
  const void *nope, *rope;  // [t, groups*128], bf16 [t, 64] or null
  int64_t nope_ld, rope_ld;
  const int64_t* index;  // [t]
  int8_t* cache;         // [rows, groups*128] or null
  void* rope_cache;      // bf16 [rows, 64]
  void* scales;          // [rows, groups]
  int8_t* packed;        // [rows, 656] or null
  int64_t rows;
  int t, groups, chunks, scale_f16;
  int32_t* status;
};
cudaError_t launch_kv_write(const KvWriteParams& p, int dtype, cudaStream_t stream);

struct KvReadParams {
  const int8_t* cache;
  const void *rope, *scales;
  const int8_t* packed;
  const int32_t *table, *cu, *first;  // [b, max_blocks], [b+1], [b] or null
  void *out, *rope_out;               // [n, groups*128], bf16 [n, 64] or null
  int64_t out_ld, rope_out_ld, rows, n;
  int b, max_blocks, block_size, groups, chunks, scale_f16, per_warp;
  int32_t* status;
};
cudaError_t launch_kv_read(KvReadParams p, int dtype, int num_sms, cudaStream_t stream);

}  // namespace pto
