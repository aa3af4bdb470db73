// What the attention entry points (attention.cu) hand to the tensor-core kernel
// (attention_tc.cu).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mtrtq {

struct TcAttention {
  const int32_t* cu_rows;
  const int32_t* kv_len;  // paged only, like table
  const int32_t* table;
  int64_t table_ld;
  int64_t rows;
  int batch, kv_heads, group, head_dim, page_size;
  int slot_tokens;   // 128 / group: tokens in a tile slot's 128 rows
  int64_t max_keys;  // paged: tokens the table's columns hold
  int64_t min_steps; // fewest steps worth a CTA
  float scale;
  __nv_bfloat16* out;
  int64_t out_row, out_head;
  const __nv_bfloat16* v;  // as the tensor map has it, for values taken out of a block
  int64_t v_row, v_head;   // paged: v_row is the page stride
  unsigned* counters;      // [grid] tickets, zero
  float* partials;         // [grid][2][head_dim rounded to 64 or 128 / 4][part_rows] float4
  float2* part_ml;         // [grid][2][part_rows]
  int part_rows;           // rows a tile can have, at most 256
  unsigned* status;
};

cudaError_t launch_attention_tc(const TcAttention& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                                int grid, bool pdl, cudaStream_t st);

}  // namespace mtrtq
