// What the attention entry points (attention.cu) hand to the tensor-core kernel
// (attention_tc.cu).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mtrtq {

// What a call's list of steps (attention_sched.cuh) is made from.
struct AttentionList {
  const int32_t* cu_rows;
  const int32_t* kv_len;  // paged only, like table
  const int32_t* table;
  int64_t table_ld;
  int64_t rows;
  int batch, kv_heads, group, head_dim, page_size;
  int slot_tokens;    // tensor cores: 128 / group, the tokens in a slot's 128 rows
  int q_buffers;      // and whether the next tile's Q has a place of its own (2)
  int tile_tokens;
  int least, most;    // tokens of the requests that this launch takes
  int64_t max_keys;   // paged: tokens the table's columns hold
  int64_t min_steps;  // fewest steps worth a CTA
  int tile_cost, pair_cost;  // steps that a tile takes besides its own, in one slot's rows or more
};

struct TcAttention : AttentionList {
  float scale;
  bool planes;  // q lies in two planes of `rows` rows
  __nv_bfloat16* out;
  int64_t out_row, out_head;
  bool out32;  // rows of out start on 32 bytes
  const __nv_bfloat16* v;  // as the tensor map has it, for values taken out of a block
  int64_t v_row, v_head;   // paged: v_row is the page stride
  unsigned* counters;      // [grid] tickets, zero
  float* partials;         // [grid][2][head_dim rounded to 64 or 128 / 4][part_rows] float4
  float2* part_ml;         // [grid][2][part_rows]
  int part_rows;           // rows a tile can have, at most 256
  unsigned* status;
};

// fp32 throughout, on the CUDA cores (attention_f32.cu): tiles of 1, 2, 4, 8, 16, 64 or
// 128 rows; those of 1 and 2 also with pages and out (pages16) and q (q16) in bf16.
struct F32Attention : AttentionList {
  float scale;
  bool pages16, q16;
  const float *q, *k, *v;  // paged: k and v are the pages, k_row and v_row the page stride
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  float* out;
  int64_t out_row, out_head;
  unsigned* counters;  // [grid] tickets, zero
  int64_t num_pages;
  float* partials;     // [grid][2][tile_rows][head_dim rounded to 64 or 128]
  float2* part_ml;     // [grid][2][tile_rows]
  int tile_rows;
};

// The same on the tensor cores (attention_f32_tc.cu): whole prompts, up to 64 dimensions, in
// tiles of 128 rows. q, k and v lie as three bf16 planes.
struct F32TcAttention : F32Attention {
  const int* flags;  // of split_rows: whether a block of rows has infinities or NaN in v
  unsigned* status;
};
constexpr int kSplitRows = 8;  // rows of a block of split_rows
cudaError_t launch_split_rows(const F32Attention& p, int heads, __nv_bfloat16* planes, int* flags, cudaStream_t st);
cudaError_t launch_attention_f32_tc(const F32TcAttention& p, const CUtensorMap& q, const CUtensorMap& k,
                                    const CUtensorMap& v, int grid, cudaStream_t st);

cudaError_t launch_attention_f32(const F32Attention& p, int grid, bool pdl, cudaStream_t st);

cudaError_t launch_attention_tc(const TcAttention& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                                int grid, bool pdl, cudaStream_t st);

}  // namespace mtrtq
