// Beam search: the selection over beams and vocabulary, and the reordering of the
// beams' cached states (include/mtrtq.h, mtrtq_beam_select and mtrtq_beam_reorder).
#include <math.h>

#include "../../include/mtrtq.h"
#include "q8_common.cuh"

namespace mtrtq {

int report_error(int code, const char* fmt, ...);
int report_cuda_error(cudaError_t e, const char* what);
unsigned* device_status_address(int* rc);

namespace {

// A candidate as one 64-bit number that is larger for a larger score and, between
// equal scores, for a lower index: the score's bits made monotonic, then ~index.
// -0 counts as +0.
__device__ __forceinline__ unsigned long long candidate_key(float score, uint32_t index) {
  const uint32_t u = __float_as_uint(score + 0.0f);
  const uint32_t hi = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)hi << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_score(unsigned long long key) {
  const uint32_t hi = (uint32_t)(key >> 32);
  return __uint_as_float((hi & 0x80000000u) ? (hi & 0x7fffffffu) : ~hi);
}
__device__ __forceinline__ uint32_t key_index(unsigned long long key) { return ~(uint32_t)key; }

__device__ __forceinline__ float logit(float x) { return x == x ? x : -INFINITY; }

constexpr int kThreads = 256;

__device__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < kThreads / 32; ++w) v = fmaxf(v, red[w]);
  return v;
}
__device__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < kThreads / 32; ++w) v += red[w];
  return v;
}

// One block per row: log sum_t exp(logit_t) = max + log sum exp(logit - max).
__global__ void __launch_bounds__(kThreads) row_lse_kernel(const float* logits, int64_t ldl, int vocab, float* lse) {
  __shared__ float red[kThreads / 32];
  const float* x = logits + blockIdx.x * ldl;
  float m = -INFINITY;
  for (int t = threadIdx.x; t < vocab; t += kThreads) m = fmaxf(m, logit(x[t]));
  m = block_max(m, red);
  float s = 0.0f;
  for (int t = threadIdx.x; t < vocab; t += kThreads) s += expf(logit(x[t]) - m);
  s = block_sum(s, red);
  if (threadIdx.x == 0) lse[blockIdx.x] = m + logf(s);
}

// One block per request: `beams` times the best candidate below the last one.
__global__ void __launch_bounds__(kThreads)
    pick_kernel(const float* logits, int64_t ldl, const float* lse, const float* scores, const uint8_t* done,
                int32_t eos, int beams, int vocab, float* out_scores, int32_t* parent, int32_t* token,
                uint8_t* out_done) {
  __shared__ unsigned long long best[kThreads];
  const int64_t r0 = (int64_t)blockIdx.x * beams;
  unsigned long long below = ~0ull;
  for (int i = 0; i < beams; ++i) {
    unsigned long long k = 0;
    for (int w = 0; w < beams; ++w) {
      const float* x = logits + (r0 + w) * ldl;
      const float base = scores[r0 + w], z = lse[r0 + w];
      const bool ended = done[r0 + w] != 0;
      for (int t = threadIdx.x; t < vocab; t += kThreads) {
        float s = ended ? (t == eos ? base : -INFINITY) : base + (logit(x[t]) - z);
        if (s != s) s = -INFINITY;
        const unsigned long long c = candidate_key(s, (uint32_t)w * vocab + t);
        if (c < below && c > k) k = c;
      }
    }
    best[threadIdx.x] = k;
    __syncthreads();
    for (int n = kThreads / 2; n > 0; n >>= 1) {
      if (threadIdx.x < n && best[threadIdx.x + n] > best[threadIdx.x]) best[threadIdx.x] = best[threadIdx.x + n];
      __syncthreads();
    }
    below = best[0];
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint32_t at = key_index(below);
      const int w = at / vocab, t = at % vocab;
      out_scores[r0 + i] = key_score(below);
      parent[r0 + i] = w;
      token[r0 + i] = t;
      out_done[r0 + i] = done[r0 + w] != 0 || t == eos;
    }
  }
}

// The partly filled pages' tokens move along with their beams, in place: a thread
// reads its 16 bytes of every beam's parent before it writes any beam's, and no other
// thread touches those. Grid (chunks of a page, layers, requests); the request's
// first block moves the table's rows the same way.
template <int W>
__global__ void __launch_bounds__(kThreads)
    reorder_kernel(const int32_t* parent, int beams, int32_t* table, int64_t table_ld, const int32_t* owned,
                   int64_t owned_ld, int64_t width, const int32_t* kv_len, uint4* k_pages, uint4* v_pages,
                   int64_t layer_vecs, int64_t page_vecs, int64_t num_pages, int kv_heads, int page_size,
                   int token_vecs) {
  const int64_t r0 = (int64_t)blockIdx.z * beams;
  const int64_t n = kv_len[blockIdx.z] < 0 ? 0 : kv_len[blockIdx.z];
  const int64_t full = n / page_size < width ? n / page_size : width;
  const int rest = n / page_size < width ? (int)(n % page_size) : 0;
  int from[W];
  bool moves = false;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const int p = i < beams ? parent[r0 + i] : i;
    from[i] = p >= 0 && p < beams ? p : i;
    moves |= from[i] != i;
  }
  if (rest > 0 && moves) {
    const int chunk = rest * token_vecs, total = kv_heads * chunk;
    for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kThreads) {
      const int64_t in_page = blockIdx.y * layer_vecs + e / chunk * (int64_t)page_size * token_vecs + e % chunk;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        uint4* pages = kv ? v_pages : k_pages;
        uint4 x[W];
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const int64_t page = i < beams ? owned[(r0 + from[i]) * owned_ld + full] : -1;
          if (from[i] != i && page >= 0 && page < num_pages) x[i] = pages[page * page_vecs + in_page];
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
          if (i >= beams || from[i] == i) continue;
          const int64_t page = owned[(r0 + i) * owned_ld + full], source = owned[(r0 + from[i]) * owned_ld + full];
          if (page >= 0 && page < num_pages && source >= 0 && source < num_pages)
            pages[page * page_vecs + in_page] = x[i];
        }
      }
    }
  }
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    for (int64_t c = threadIdx.x; c < width; c += kThreads) {
      int32_t x[W];
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i < beams) x[i] = c < full ? table[(r0 + from[i]) * table_ld + c] : owned[(r0 + i) * owned_ld + c];
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i < beams) table[(r0 + i) * table_ld + c] = x[i];
    }
  }
}

int check_beams(int64_t requests, int64_t beams) {
  if (requests < 1 || requests > 65535 || beams < 1 || beams > MTRTQ_MAX_BEAMS)
    return report_error(MTRTQ_ERR_INVALID_ARG, "requests (%lld) is 1 to 65535, beams (%lld) 1 to %d",
                        (long long)requests, (long long)beams, MTRTQ_MAX_BEAMS);
  return MTRTQ_OK;
}

int check_select(int64_t requests, int64_t beams, int64_t vocab) {
  if (int rc = check_beams(requests, beams)) return rc;
  if (vocab < 1 || vocab * beams > 2147483647 || vocab > 2147483647)
    return report_error(MTRTQ_ERR_INVALID_ARG, "vocab (%lld) times beams is 1 to 2^31 - 1", (long long)vocab);
  return MTRTQ_OK;
}

}  // namespace
}  // namespace mtrtq

using namespace mtrtq;

extern "C" {

int64_t mtrtq_beam_workspace_bytes(int64_t requests, int64_t beams, int64_t vocab) {
  if (check_select(requests, beams, vocab)) return -1;
  return requests * beams * (int64_t)sizeof(float);
}

int mtrtq_beam_select(const float* logits, int64_t ldl, const float* scores, const uint8_t* done, int32_t eos,
                      int64_t requests, int64_t beams, int64_t vocab, float* out_scores, int32_t* parent,
                      int32_t* token, uint8_t* out_done, void* workspace, size_t workspace_bytes, void* stream) {
  if (!logits || !scores || !done || !out_scores || !parent || !token || !out_done)
    return report_error(MTRTQ_ERR_INVALID_ARG, "null pointer");
  if (int rc = check_select(requests, beams, vocab)) return rc;
  if (ldl < vocab || eos < -1 || eos >= vocab)
    return report_error(MTRTQ_ERR_INVALID_ARG, "ldl (%lld) is at least vocab, eos (%d) -1 or a token", (long long)ldl,
                        eos);
  int rc;
  device_status_address(&rc);
  if (rc) return rc;
  if (!workspace || (int64_t)workspace_bytes < mtrtq_beam_workspace_bytes(requests, beams, vocab))
    return report_error(MTRTQ_ERR_WORKSPACE, "workspace %zu bytes < %lld", workspace_bytes,
                        (long long)mtrtq_beam_workspace_bytes(requests, beams, vocab));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* lse = static_cast<float*>(workspace);
  row_lse_kernel<<<(unsigned)(requests * beams), kThreads, 0, st>>>(logits, ldl, (int)vocab, lse);
  pick_kernel<<<(unsigned)requests, kThreads, 0, st>>>(logits, ldl, lse, scores, done, eos, (int)beams, (int)vocab,
                                                       out_scores, parent, token, out_done);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MTRTQ_OK : report_cuda_error(e, "beam selection launch");
}

int mtrtq_beam_reorder(const int32_t* parent, int64_t requests, int64_t beams, int32_t* table, int64_t table_ld,
                       const int32_t* owned, int64_t owned_ld, int64_t width, const int32_t* kv_len,
                       void* k_pages, void* v_pages, int64_t layers, int64_t layer_stride, int64_t page_stride,
                       int64_t num_pages, int kv_heads, int page_size, int head_dim, int dtype, void* stream) {
  if (!parent || !table || !owned || !kv_len || !k_pages || !v_pages)
    return report_error(MTRTQ_ERR_INVALID_ARG, "null pointer");
  if (int rc = check_beams(requests, beams)) return rc;
  if (dtype != MTRTQ_DTYPE_F32 && dtype != MTRTQ_DTYPE_BF16)
    return report_error(MTRTQ_ERR_INVALID_ARG, "dtype must be MTRTQ_DTYPE_F32 or MTRTQ_DTYPE_BF16");
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
    return report_error(MTRTQ_ERR_INVALID_ARG, "page_size (%d) is 16, 32, 64 or 128", page_size);
  if (head_dim < 8 || head_dim > 128 || head_dim % 8 || kv_heads < 1 || kv_heads > 65535)
    return report_error(MTRTQ_ERR_INVALID_ARG, "head_dim (%d) is a multiple of 8 up to 128, kv_heads (%d) positive",
                        head_dim, kv_heads);
  const int64_t page = (int64_t)kv_heads * page_size * head_dim;
  if (layers < 1 || layers > 65535 || width < 1 || width * page_size > 2147483647 || table_ld < width ||
      owned_ld < width || num_pages < 1 || num_pages > 2147483647 || page_stride < page ||
      page_stride >= (int64_t(1) << 36) || layer_stride < 0 || (layers > 1 && layer_stride < page))
    return report_error(MTRTQ_ERR_INVALID_ARG, "layers, width, num_pages or a stride is out of range");
  const int size = dtype == MTRTQ_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(k_pages) % 16 || reinterpret_cast<uintptr_t>(v_pages) % 16 ||
      page_stride * size % 16 || layer_stride * size % 16)
    return report_error(MTRTQ_ERR_ALIGNMENT, "pages must be 16-byte aligned with strides of whole 16 bytes");
  int rc;
  device_status_address(&rc);
  if (rc) return rc;
  const int vec = 16 / size;
  const int64_t most = (page / vec + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)(most < 8 ? most : 8), (unsigned)layers, (unsigned)requests);
  auto run = [&](auto kernel) {
    kernel<<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        parent, (int)beams, table, table_ld, owned, owned_ld, width, kv_len, static_cast<uint4*>(k_pages),
        static_cast<uint4*>(v_pages), layer_stride / vec, page_stride / vec, num_pages, kv_heads, page_size,
        head_dim / vec);
  };
  if (beams <= 4) run(reorder_kernel<4>);
  else if (beams <= 8) run(reorder_kernel<8>);
  else if (beams <= 16) run(reorder_kernel<16>);
  else run(reorder_kernel<32>);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MTRTQ_OK : report_cuda_error(e, "beam reorder launch");
}

}  // extern "C"
