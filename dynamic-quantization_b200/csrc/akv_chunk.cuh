// The tensor-core (tcgen05) form of chunk attention: what akv_chunk_attention
// hands to it.
#pragma once

#include "akv_common.cuh"

namespace akv {

struct ChunkArgs {
  const uint8_t *arena;
  int64_t arena_bytes;
  const int64_t *table;
  int64_t table_stride;
  const int32_t *seq_blocks;
  int32_t columns;  // of the table
  const int32_t *tokens;
  int32_t uniform_tokens;
  const __half *q;
  int64_t q_bs, q_hs, q_ts;
  __half *out;
  int64_t o_bs, o_hs, o_ts;
  int32_t batch, rows, q_heads, kv_heads, head_dim, log2_group;
  int32_t kv_first, page_heads;  // a call's slice has KV heads kv_first .. of the page_heads that pages hold
  int32_t window, sinks, lead;
  float scale;
  int32_t *status;
  cudaStream_t stream;
};

// Bytes of workspace the call needs (-1: unsupported, or no device).
int64_t chunk_tiles_bytes(const ChunkArgs &a);
int chunk_tiles_launch(const ChunkArgs &a, void *workspace, int64_t workspace_bytes);

}  // namespace akv
