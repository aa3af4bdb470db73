// Attention of packed rows: over whole prompts, and of new tokens over a paged
// key/value cache (include/mtrtq.h, mtrtq_prompt_attention and mtrtq_paged_attention).
#include <math.h>

#include "../../include/mtrtq.h"
#include "q8_common.cuh"

namespace mtrtq {

int report_error(int code, const char* fmt, ...);
int report_cuda_error(cudaError_t e, const char* what);
unsigned* device_status_address(int* rc);
bool overlap_launch_enabled();

namespace {

typedef mtrtq_attention_args Args;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Rows of request b, with malformed bounds clamped so that no access leaves the rows.
__device__ __forceinline__ void request_rows(const Args& a, int64_t b, int64_t& r0, int64_t& r1) {
  const int64_t lo = a.cu_rows[b], hi = a.cu_rows[b + 1];
  r0 = lo < 0 ? 0 : lo > a.rows ? a.rows : lo;
  r1 = hi < r0 ? r0 : hi > a.rows ? a.rows : hi;
}

// The request that owns row r, or -1: the last b with cu_rows[b] <= r.
__device__ int64_t request_of(const Args& a, int64_t r) {
  int64_t lo = 0, hi = a.batch;
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (mid < a.batch && a.cu_rows[mid] <= r) lo = mid; else hi = mid - 1;
  }
  int64_t r0, r1;
  request_rows(a, lo, r0, r1);
  return r >= r0 && r < r1 ? lo : -1;
}

// Where token i of request b lies in the pages of head g (elements), or -1.
__device__ __forceinline__ int64_t page_offset(const Args& a, int64_t b, int64_t i, int64_t g) {
  const int64_t c = i / a.page_size;
  if (i < 0 || c >= a.table_width) return -1;
  const int64_t n = a.table[b * a.table_ld + c];
  if (n < 0 || n >= a.num_pages) return -1;
  return n * a.page_stride + (g * a.page_size + i % a.page_size) * a.head_dim;
}

// One block per new row: its k and v go to its position's page, rounded to the
// cache's type.
template <typename TX, typename TC>
__global__ void append_kernel(const __grid_constant__ Args a) {
  const int64_t r = blockIdx.x;
  const int64_t b = request_of(a, r);
  if (b < 0) return;
  int64_t r0, r1;
  request_rows(a, b, r0, r1);
  const int64_t i = (int64_t)a.kv_len[b] - (r1 - r0) + (r - r0);
  for (int e = threadIdx.x; e < a.kv_heads * a.head_dim; e += blockDim.x) {
    const int g = e / a.head_dim, d = e - g * a.head_dim;
    const int64_t at = page_offset(a, b, i, g);
    if (at < 0) continue;
    static_cast<TC*>(a.k_pages)[at + d] =
        from_f32<TC>(to_f32(static_cast<const TX*>(a.k)[r * a.k_row + g * a.k_head + d]));
    static_cast<TC*>(a.v_pages)[at + d] =
        from_f32<TC>(to_f32(static_cast<const TX*>(a.v)[r * a.v_row + g * a.v_head + d]));
  }
}

// One warp per (row, head), lanes over the dimensions: the running maximum m, sum l
// and output o of a softmax over the keys in order.
template <typename TX, typename TC, bool PAGED>
__global__ void __launch_bounds__(32) rows_kernel(const __grid_constant__ Args a) {
  const int64_t r = blockIdx.x;
  const int h = blockIdx.y, lane = threadIdx.x;
  const int64_t b = request_of(a, r);
  if (b < 0) return;
  int64_t r0, r1;
  request_rows(a, b, r0, r1);
  const int g = h / (a.heads / a.kv_heads);
  int64_t last = PAGED ? (int64_t)a.kv_len[b] - (r1 - r0) + (r - r0) : r - r0;
  if (PAGED && last >= a.table_width * a.page_size) last = a.table_width * a.page_size - 1;
  float q[4], o[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int d = c * 32 + lane;
    q[c] = d < a.head_dim ? to_f32(static_cast<const TX*>(a.q)[r * a.q_row + h * a.q_head + d]) * a.scale : 0.0f;
    o[c] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int64_t j = 0; j <= last; ++j) {
    const int64_t at = PAGED ? page_offset(a, b, j, g) : 0;
    if (at < 0) continue;
    float s = 0.0f, v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int d = c * 32 + lane;
      float k = 0.0f;
      v[c] = 0.0f;
      if (d < a.head_dim) {
        if (PAGED) {
          k = to_f32(static_cast<const TC*>(a.k_pages)[at + d]);
          v[c] = to_f32(static_cast<const TC*>(a.v_pages)[at + d]);
        } else {
          k = to_f32(from_f32<TC>(to_f32(static_cast<const TX*>(a.k)[(r0 + j) * a.k_row + g * a.k_head + d])));
          v[c] = to_f32(from_f32<TC>(to_f32(static_cast<const TX*>(a.v)[(r0 + j) * a.v_row + g * a.v_head + d])));
        }
      }
      s += q[c] * k;
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float top = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.0f : expf(m - top), p = top == -INFINITY ? 0.0f : expf(s - top);
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = o[c] * keep + p * v[c];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int d = c * 32 + lane;
    if (d < a.head_dim)
      static_cast<TC*>(a.out)[r * a.out_row + h * a.out_head + d] = from_f32<TC>(l == 0.0f ? 0.0f : o[c] * inv);
  }
}

bool on16(const void* p, int64_t s0, int64_t s1, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s0 * size % 16 == 0 && s1 * size % 16 == 0;
}

int check_args(const Args* a, bool paged) {
  if (!a || !a->cu_rows || (a->rows != 0 && (!a->q || !a->out)))
    return report_error(MTRTQ_ERR_INVALID_ARG, "null pointer");
  if (a->x_dtype != MTRTQ_DTYPE_F32 && a->x_dtype != MTRTQ_DTYPE_BF16)
    return report_error(MTRTQ_ERR_INVALID_ARG, "x_dtype must be MTRTQ_DTYPE_F32 or MTRTQ_DTYPE_BF16");
  if (a->dtype != MTRTQ_DTYPE_BF16 && (a->dtype != MTRTQ_DTYPE_F32 || a->x_dtype != MTRTQ_DTYPE_F32))
    return report_error(MTRTQ_ERR_INVALID_ARG, "dtype is MTRTQ_DTYPE_BF16, or MTRTQ_DTYPE_F32 with f32 rows");
  if (a->rows < 0 || a->rows > (int64_t(1) << 30) || a->batch < 1 || a->batch > MTRTQ_MAX_BATCH)
    return report_error(MTRTQ_ERR_INVALID_ARG, "rows (%lld) is 0 to 2^30, batch (%lld) 1 to %d", (long long)a->rows,
                        (long long)a->batch, MTRTQ_MAX_BATCH);
  if (a->kv_heads < 1 || a->heads < a->kv_heads || a->heads > 65535 || a->heads % a->kv_heads ||
      a->heads / a->kv_heads > 128)
    return report_error(MTRTQ_ERR_INVALID_ARG, "heads (%d) must be 1 to 128 times kv_heads (%d)", a->heads,
                        a->kv_heads);
  if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8)
    return report_error(MTRTQ_ERR_INVALID_ARG, "head_dim (%d) is a multiple of 8 up to 128", a->head_dim);
  if (!(a->scale > 0.0f) || !(a->scale < INFINITY))
    return report_error(MTRTQ_ERR_INVALID_ARG, "scale must be positive and finite");
  if (a->rows != 0 && (!a->k || !a->v) && !(paged && !a->k && !a->v))
    return report_error(MTRTQ_ERR_INVALID_ARG, "k and v are both needed%s", paged ? " or both NULL" : "");
  const int xs = a->x_dtype == MTRTQ_DTYPE_F32 ? 4 : 2, cs = a->dtype == MTRTQ_DTYPE_F32 ? 4 : 2;
  const int64_t strides[8] = {a->q_row, a->q_head, a->k_row, a->k_head, a->v_row, a->v_head, a->out_row, a->out_head};
  for (int64_t s : strides)
    if (s < 0 || s >= (int64_t(1) << 36)) return report_error(MTRTQ_ERR_INVALID_ARG, "a stride is out of range");
  if (a->out_row == 0 && a->rows > 1)
    return report_error(MTRTQ_ERR_INVALID_ARG, "the rows of out must not overlap");
  if (!on16(a->q, a->q_row, a->q_head, xs) || (a->k && !on16(a->k, a->k_row, a->k_head, xs)) ||
      (a->v && !on16(a->v, a->v_row, a->v_head, xs)) || !on16(a->out, a->out_row, a->out_head, cs))
    return report_error(MTRTQ_ERR_ALIGNMENT, "q, k, v and out must be 16-byte aligned with strides of whole 16 bytes");
  if (!paged) return MTRTQ_OK;
  if (!a->k_pages || !a->v_pages || !a->table || !a->kv_len) return report_error(MTRTQ_ERR_INVALID_ARG, "null pointer");
  if (a->page_size != 16 && a->page_size != 32 && a->page_size != 64 && a->page_size != 128)
    return report_error(MTRTQ_ERR_INVALID_ARG, "page_size (%d) is 16, 32, 64 or 128", a->page_size);
  if (a->num_pages < 1 || a->num_pages > 2147483647 || a->table_width < 1 ||
      a->table_width * a->page_size > 2147483647 || a->table_ld < a->table_width)
    return report_error(MTRTQ_ERR_INVALID_ARG, "num_pages (%lld), table_width (%lld) or table_ld (%lld) is out of range",
                        (long long)a->num_pages, (long long)a->table_width, (long long)a->table_ld);
  if (a->page_stride < (int64_t)a->kv_heads * a->page_size * a->head_dim || a->page_stride >= (int64_t(1) << 36))
    return report_error(MTRTQ_ERR_INVALID_ARG, "page_stride (%lld) is less than a page", (long long)a->page_stride);
  if (!on16(a->k_pages, a->page_stride, 0, cs) || !on16(a->v_pages, a->page_stride, 0, cs))
    return report_error(MTRTQ_ERR_ALIGNMENT, "pages must be 16-byte aligned, page_stride whole 16 bytes");
  return MTRTQ_OK;
}

template <typename TX, typename TC>
int launch(const Args& a, bool paged, cudaStream_t st) {
  if (paged) {
    if (a.k) append_kernel<TX, TC><<<(unsigned)a.rows, 128, 0, st>>>(a);
    rows_kernel<TX, TC, true><<<dim3((unsigned)a.rows, a.heads), 32, 0, st>>>(a);
  } else {
    rows_kernel<TX, TC, false><<<dim3((unsigned)a.rows, a.heads), 32, 0, st>>>(a);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MTRTQ_OK : report_cuda_error(e, "attention launch");
}

int attention(const Args* a, bool paged, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_args(a, paged)) return rc;
  int rc;
  device_status_address(&rc);
  if (rc) return rc;
  if (a->rows == 0) return MTRTQ_OK;
  const int64_t need = mtrtq_attention_workspace_bytes(a);
  if (!workspace || (int64_t)workspace_bytes < need)
    return report_error(MTRTQ_ERR_WORKSPACE, "workspace %zu bytes < %lld", workspace_bytes, (long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return report_error(MTRTQ_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->dtype == MTRTQ_DTYPE_F32) return launch<float, float>(*a, paged, st);
  if (a->x_dtype == MTRTQ_DTYPE_F32) return launch<float, __nv_bfloat16>(*a, paged, st);
  return launch<__nv_bfloat16, __nv_bfloat16>(*a, paged, st);
}

}  // namespace
}  // namespace mtrtq

using namespace mtrtq;

extern "C" {

int64_t mtrtq_attention_workspace_bytes(const mtrtq_attention_args* a) {
  if (check_args(a, a && a->k_pages)) return -1;
  return 4096;
}

int mtrtq_prompt_attention(const mtrtq_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  return attention(a, false, workspace, workspace_bytes, stream);
}

int mtrtq_paged_attention(const mtrtq_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  return attention(a, true, workspace, workspace_bytes, stream);
}

}  // extern "C"
