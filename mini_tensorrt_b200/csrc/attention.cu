// Attention of packed rows: over whole prompts, and of new tokens over a paged
// key/value cache (include/mtrtq.h, mtrtq_prompt_attention and mtrtq_paged_attention).
#include <limits.h>
#include <math.h>

#include "../../include/mtrtq.h"
#include "attention.h"
#include "q8_common.cuh"

namespace mtrtq {

int report_error(int code, const char* fmt, ...);
int report_cuda_error(cudaError_t e, const char* what);
unsigned* device_status_address(int* rc);

namespace {

typedef mtrtq_attention_args Args;

// Rows of request b, with malformed bounds clamped so that no access leaves the rows.
__device__ __forceinline__ void request_rows(const Args& a, int64_t b, int64_t& r0, int64_t& r1) {
  const int64_t lo = a.cu_rows[b], hi = a.cu_rows[b + 1];
  r0 = lo < 0 ? 0 : lo > a.rows ? a.rows : lo;
  r1 = hi < r0 ? r0 : hi > a.rows ? a.rows : hi;
}

// The request that owns row r, or -1: every thread of the block looks at a few requests
// (one round of loads; a row in two requests goes to the later one).
__device__ int request_of(const Args& a, int64_t r) {
  __shared__ int found;
  if (threadIdx.x == 0) found = -1;
  __syncthreads();
  for (int b = threadIdx.x; b < a.batch; b += blockDim.x) {
    int64_t r0, r1;
    request_rows(a, b, r0, r1);
    if (r >= r0 && r < r1) atomicMax(&found, b);
  }
  __syncthreads();
  return found;
}

// Where token i of request b lies in the pages of head g (elements); -1 if its page
// number is out of range.
__device__ __forceinline__ int64_t page_offset(const Args& a, int64_t b, int64_t i, int64_t g) {
  const int64_t c = i / a.page_size;
  if (i < 0 || c >= a.table_width) return -1;
  const int64_t n = a.table[b * a.table_ld + c];
  if (n < 0 || n >= a.num_pages) return -1;
  return n * a.page_stride + (g * a.page_size + i % a.page_size) * a.head_dim;
}

// Four elements from src, as TC, to dst (16-byte aligned f32, 8-byte aligned bf16).
__device__ __forceinline__ float4 load4(const float* src) { return *reinterpret_cast<const float4*>(src); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* src) {
  const uint2 u = *reinterpret_cast<const uint2*>(src);
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ void store4(float* dst, float4 x) { *reinterpret_cast<float4*>(dst) = x; }
__device__ __forceinline__ void store4(__nv_bfloat16* dst, float4 x) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x, x.y), hi = __floats2bfloat162_rn(x.z, x.w);
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(reinterpret_cast<const uint32_t&>(lo), reinterpret_cast<const uint32_t&>(hi));
}

// Four elements of q in the tensor cores' types: rounded to dst's type, or (f32 rows) as two
// bf16 planes, `plane` elements apart, of 16 bits together. The first is cut toward zero and the
// second is never zero where q is not, so that both have q's sign: their products with an
// infinite k are then both the infinity that q's is, and a zero q times it NaN in both.
template <typename TX>
__device__ __forceinline__ void store_q(__nv_bfloat16* dst, int64_t plane, float4 x) {
  if (sizeof(TX) == 2) {
    store4(dst, x);
    return;
  }
  const float v[4] = {x.x, x.y, x.z, x.w};
  float a[4], b[4];
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    a[y] = v[y] == v[y] ? __uint_as_float(__float_as_uint(v[y]) & 0xffff0000u) : v[y];
    b[y] = __bfloat162float(__float2bfloat16_rn(v[y] - a[y]));
    if (!(fabsf(b[y]) >= 1.1754944e-38f) && v[y] != 0.0f) b[y] = copysignf(1.1754944e-38f, v[y]);  // (2^-126; of infinities too)
  }
  store4(dst, make_float4(a[0], a[1], a[2], a[3]));
  store4(dst + plane, make_float4(b[0], b[1], b[2], b[3]));
}

// One block per new row: its k and v go to its position's page, rounded to the
// cache's type; q_rows (if not null) gets q, [rows, heads, head_dim], see store_q.
// 16 rows of 12 x 64 take 5.3 us on a B200 and 964 of 32 / 8 x 128 6.3: the latency of a load and
// a store, during which the attention kernel is launched and makes its list.
constexpr int kRowThreads = 256;
template <typename TX, typename TC>
__global__ void __launch_bounds__(kRowThreads) append_kernel(const __grid_constant__ Args a, __nv_bfloat16* q_rows) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t r = blockIdx.x;
  const int quads = a.head_dim / 4;
  if (q_rows) {
    for (int e = threadIdx.x; e < a.heads * quads; e += kRowThreads) {
      const int h = e / quads, d = (e - h * quads) * 4;
      store_q<TX>(q_rows + (r * a.heads + h) * a.head_dim + d, a.rows * a.heads * a.head_dim,
                  load4(static_cast<const TX*>(a.q) + r * a.q_row + h * a.q_head + d));
    }
  }
  if (!a.k) return;
  const int b = request_of(a, r);
  if (b < 0) return;
  int64_t r0, r1;
  request_rows(a, b, r0, r1);
  const int64_t i = (int64_t)a.kv_len[b] - (r1 - r0) + (r - r0);
  for (int e = threadIdx.x; e < a.kv_heads * quads; e += kRowThreads) {
    const int g = e / quads, d = (e - g * quads) * 4;
    const float4 k = load4(static_cast<const TX*>(a.k) + r * a.k_row + g * a.k_head + d);
    const float4 v = load4(static_cast<const TX*>(a.v) + r * a.v_row + g * a.v_head + d);
    const int64_t at = page_offset(a, b, i, g);
    if (at < 0) continue;
    store4(static_cast<TC*>(a.k_pages) + at + d, k);
    store4(static_cast<TC*>(a.v_pages) + at + d, v);
  }
}

// q (see store_q), [rows, heads, head_dim], and k and v in bf16, [rows, 2 kv_heads, head_dim]: 60
// rows of 12 x 64 4.2 us.
template <typename TX>
__global__ void __launch_bounds__(kRowThreads)
    cast_kernel(const __grid_constant__ Args a, __nv_bfloat16* q_rows, __nv_bfloat16* kv_rows) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t r = blockIdx.x;
  const int hq = a.heads, hk = a.kv_heads, quads = a.head_dim / 4;
  for (int e = threadIdx.x; e < (hq + 2 * hk) * quads; e += kRowThreads) {
    const int h = e / quads, d = (e - h * quads) * 4;
    if (h < hq) {
      store_q<TX>(q_rows + (r * hq + h) * a.head_dim + d, a.rows * hq * a.head_dim,
                  load4(static_cast<const TX*>(a.q) + r * a.q_row + h * a.q_head + d));
      continue;
    }
    const TX* src = h < hq + hk ? static_cast<const TX*>(a.k) + r * a.k_row + (h - hq) * a.k_head
                                : static_cast<const TX*>(a.v) + r * a.v_row + (h - hq - hk) * a.v_head;
    store4(kv_rows + (r * 2 * hk + h - hq) * a.head_dim + d, load4(src + d));
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
  if (!on16(a->q, a->q_row, a->q_head, xs) || (a->k && !on16(a->k, a->k_row, a->k_head, xs)) ||
      (a->v && !on16(a->v, a->v_row, a->v_head, xs)) || !on16(a->out, a->out_row, a->out_head, cs))
    return report_error(MTRTQ_ERR_ALIGNMENT, "q, k, v and out must be 16-byte aligned with strides of whole 16 bytes");
  if ((a->rows > 1 && a->out_row < a->head_dim) || (a->rows > 0 && a->heads > 1 && a->out_head < a->head_dim))
    return report_error(MTRTQ_ERR_INVALID_ARG, "the rows and heads of out must not overlap");
  if (!paged) {
    // (the layouts and the workspace query tell the calls apart by k_pages)
    if (a->k_pages || a->v_pages || a->table || a->kv_len)
      return report_error(MTRTQ_ERR_INVALID_ARG, "k_pages, v_pages, table and kv_len are for paged calls: NULL here");
    return MTRTQ_OK;
  }
  if (!a->k_pages || !a->v_pages || !a->table || !a->kv_len) return report_error(MTRTQ_ERR_INVALID_ARG, "null pointer");
  if (a->page_size != 16 && a->page_size != 32 && a->page_size != 64 && a->page_size != 128)
    return report_error(MTRTQ_ERR_INVALID_ARG, "page_size (%d) is 16, 32, 64 or 128", a->page_size);
  if (a->num_pages < 1 || a->num_pages > 2147483647 || a->table_width < 1 ||
      a->table_width * a->page_size > (int64_t(1) << 30) || a->table_ld < a->table_width)
    return report_error(MTRTQ_ERR_INVALID_ARG, "num_pages (%lld), table_width (%lld) or table_ld (%lld) is out of range",
                        (long long)a->num_pages, (long long)a->table_width, (long long)a->table_ld);
  if (a->page_stride < (int64_t)a->kv_heads * a->page_size * a->head_dim || a->page_stride >= (int64_t(1) << 36))
    return report_error(MTRTQ_ERR_INVALID_ARG, "page_stride (%lld) is less than a page", (long long)a->page_stride);
  if (!on16(a->k_pages, a->page_stride, 0, cs) || !on16(a->v_pages, a->page_stride, 0, cs))
    return report_error(MTRTQ_ERR_ALIGNMENT, "pages must be 16-byte aligned, page_stride whole 16 bytes");
  return MTRTQ_OK;
}

int cuda_status(cudaError_t e, const char* what) {
  return e == cudaSuccess ? MTRTQ_OK : report_cuda_error(e, what);
}

size_t round256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

// Workspace of the tensor-core path: 4 KiB of tickets, as in every call's | q's planes | whole
// prompts' k and v, where they are cast | partials of cut tiles.
struct TcLayout {
  int grid, slot_tokens, part_rows, planes;
  bool cast;
  size_t off_q, off_kv, off_ml, off_part, total;
};

// TMA reads rows of the kernel's own type whose strides are not zero.
bool needs_cast(const Args& a) {
  return a.x_dtype == MTRTQ_DTYPE_F32 || a.q_row == 0 || a.q_head == 0 ||
         (!a.k_pages && (a.k_row == 0 || a.k_head == 0 || a.v_row == 0 || a.v_head == 0));
}

TcLayout tc_layout(const Args& a, int sm_count) {
  TcLayout l;
  l.grid = sm_count < 1024 ? sm_count : 1024;  // a ticket each
  const int group = a.heads / a.kv_heads;
  l.slot_tokens = 128 / group;
  l.part_rows = a.rows > l.slot_tokens ? 256 : (int)((a.rows * group + 31) / 32 * 32);
  l.cast = needs_cast(a);
  l.planes = a.x_dtype == MTRTQ_DTYPE_F32 ? 2 : 1;
  const int dp = a.head_dim <= 64 ? 64 : 128;
  const size_t row = (size_t)a.rows * a.head_dim * 2;  // of one head
  l.off_q = 4096;
  l.off_kv = l.off_q + (l.cast ? round256(row * a.heads * l.planes) : 0);
  l.off_ml = l.off_kv + (l.cast && !a.k_pages ? round256(row * 2 * a.kv_heads) : 0);
  l.off_part = l.off_ml + round256((size_t)l.grid * 2 * l.part_rows * sizeof(float2));
  l.total = l.off_part + (size_t)l.grid * 2 * l.part_rows * dp * sizeof(float);
  return l;
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// bf16, 128-byte-swizzled boxes of 64 dimensions; strides in elements, of dimension 1 on.
int make_map(CUtensorMap* map, const void* base, int rank, const int64_t* dims, const int64_t* strides, const int* box) {
  static const EncodeFn encode = reinterpret_cast<EncodeFn>(tensor_map_encoder());
  if (!encode) return report_error(MTRTQ_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  cuuint64_t d[5], s[4];
  cuuint32_t b[5], one[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = (cuuint64_t)dims[i];
    b[i] = (cuuint32_t)box[i];
    one[i] = 1;
    if (i) s[i - 1] = (cuuint64_t)strides[i - 1] * 2;
  }
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), d, s, b, one,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MTRTQ_OK : report_error(MTRTQ_ERR_CUDA, "tensor map: driver error %d", (int)r);
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    return 148;
  }
  return n;
}

void fill_list(const Args& a, bool paged, AttentionList& p) {
  p.cu_rows = a.cu_rows;
  p.kv_len = paged ? a.kv_len : nullptr;
  p.table = paged ? a.table : nullptr;
  p.table_ld = a.table_ld;
  p.rows = a.rows;
  p.batch = (int)a.batch;
  p.kv_heads = a.kv_heads;
  p.group = a.heads / a.kv_heads;
  p.head_dim = a.head_dim;
  p.page_size = a.page_size;
  p.least = 1;
  p.most = INT_MAX;
  p.max_keys = a.table_width * a.page_size;
}

// Stores the new tokens' k and v in the pages, and writes q (whole prompts: q, k and v) for the
// tensor cores to q_rows (and kv_rows) if not null.
int launch_new_rows(const Args& a, bool paged, __nv_bfloat16* q_rows, __nv_bfloat16* kv_rows, cudaStream_t st) {
  const unsigned grid = (unsigned)a.rows;
  const bool x16 = a.x_dtype != MTRTQ_DTYPE_F32;
  if (!paged) {
    if (x16) cast_kernel<__nv_bfloat16><<<grid, kRowThreads, 0, st>>>(a, q_rows, kv_rows);
    else cast_kernel<float><<<grid, kRowThreads, 0, st>>>(a, q_rows, kv_rows);
  } else if (a.dtype == MTRTQ_DTYPE_F32) {
    append_kernel<float, float><<<grid, kRowThreads, 0, st>>>(a, nullptr);
  } else if (x16) {
    append_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, kRowThreads, 0, st>>>(a, q_rows);
  } else {
    append_kernel<float, __nv_bfloat16><<<grid, kRowThreads, 0, st>>>(a, q_rows);
  }
  return cuda_status(cudaGetLastError(), "attention rows launch");
}

// For requests of `least` tokens and more; after: it follows another kernel of the call.
int launch_tc(const Args& a, bool paged, const TcLayout& l, int least, bool after, void* workspace, unsigned* status,
              cudaStream_t st) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Args x = a;
  if (l.cast) {
    __nv_bfloat16* kv = reinterpret_cast<__nv_bfloat16*>(ws + l.off_kv);
    x.q = ws + l.off_q;
    x.q_row = (int64_t)a.heads * a.head_dim;
    x.k = kv;
    x.v = kv + (int64_t)a.kv_heads * a.head_dim;
    x.k_row = x.v_row = (int64_t)2 * a.kv_heads * a.head_dim;
    x.q_head = x.k_head = x.v_head = a.head_dim;
  }
  const int group = a.heads / a.kv_heads;
  CUtensorMap qm, km, vm;
  {
    const int64_t dims[4] = {a.head_dim, group, a.kv_heads, l.planes * a.rows};
    const int64_t strides[3] = {x.q_head, x.q_head * group, x.q_row};
    const int box[4] = {64, group, 1, l.slot_tokens};
    if (int rc = make_map(&qm, x.q, 4, dims, strides, box)) return rc;
  }
  for (int i = 0; i < 2; ++i) {
    int rc;
    if (paged) {
      const int64_t dims[3] = {a.head_dim, (int64_t)a.kv_heads * a.page_size, a.num_pages};
      const int64_t strides[2] = {a.head_dim, a.page_stride};
      const int box[3] = {64, a.page_size, 1};
      rc = make_map(i ? &vm : &km, i ? a.v_pages : a.k_pages, 3, dims, strides, box);
    } else {
      const int64_t dims[3] = {a.head_dim, a.kv_heads, a.rows};
      const int64_t strides[2] = {i ? x.v_head : x.k_head, i ? x.v_row : x.k_row};
      const int box[3] = {64, 1, 128};
      rc = make_map(i ? &vm : &km, i ? x.v : x.k, 3, dims, strides, box);
    }
    if (rc) return rc;
  }
  TcAttention p = {};
  fill_list(a, paged, p);
  p.least = least;
  p.slot_tokens = l.slot_tokens;
  p.planes = l.planes == 2;
  p.q_buffers = p.planes && a.head_dim > 64 ? 1 : 2;
  p.tile_tokens = p.q_buffers * l.slot_tokens;
  p.min_steps = 4;
  p.tile_cost = 3;
  p.pair_cost = 3;
  p.scale = a.scale;
  p.out32 = reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.out_row % 16 == 0 && a.out_head % 16 == 0;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.out_row = a.out_row;
  p.out_head = a.out_head;
  p.v = static_cast<const __nv_bfloat16*>(paged ? a.v_pages : x.v);
  p.v_row = paged ? a.page_stride : x.v_row;
  p.v_head = x.v_head;
  p.counters = reinterpret_cast<unsigned*>(ws);
  p.partials = reinterpret_cast<float*>(ws + l.off_part);
  p.part_ml = reinterpret_cast<float2*>(ws + l.off_ml);
  p.part_rows = l.part_rows;
  p.status = status;
  return cuda_status(launch_attention_tc(p, qm, km, vm, l.grid, after, st), "attention launch");
}

// The f32 path: tickets | partials of cut tiles. Tiles of up to 8 rows where requests have
// few rows each (a kernel of its own, bound by memory), else of 16, 64 or 128. A tile holds
// whole groups of heads.
struct F32Layout {
  int grid, tile_rows;
  bool tc;  // on the tensor cores
  size_t off_ml, off_part, off_flags, off_planes, total;
};

F32Layout f32_layout(const Args& a, int sm_count, bool many = false) {
  F32Layout l;
  const int group = a.heads / a.kv_heads, dp = a.head_dim <= 64 ? 64 : 128;
  const int64_t each = a.rows * group / a.batch;  // rows of a request's tiles, on average
  // Prompts from some 100 rows a request on, where the split pays (B200, 12 heads of 64: 4
  // requests of 64 tokens 23 us against 21 on the CUDA cores, of 130 27 against 38, 8 of 300
  // 52 against 97).
  l.tc = !many && !a.k_pages && a.head_dim <= 64 && each >= 96;
  if (many)
    l.tile_rows = 64;
  else if (l.tc)
    l.tile_rows = 128;
  else if (each <= 8 && group <= 8)
    l.tile_rows = each <= 1 && group == 1 ? 1 : each <= 2 && group <= 2 ? 2 : each <= 4 && group <= 4 ? 4 : 8;
  else
    l.tile_rows = each <= 16 && group <= 16 ? 16 : each <= 256 && group <= 64 ? 64 : 128;
  const int ctas = l.tc ? 1 : l.tile_rows <= 2 || l.tile_rows == 16 || (dp == 64 && l.tile_rows > 8) ? 2 : 1;
  l.grid = sm_count * ctas < 1024 ? sm_count * ctas : 1024;
  l.off_ml = 4096;
  l.off_part = l.off_ml + round256((size_t)l.grid * 2 * l.tile_rows * sizeof(float2));
  l.total = l.off_part + (size_t)l.grid * 2 * l.tile_rows * dp * sizeof(float);
  l.off_flags = round256(l.total);
  l.off_planes = l.off_flags + round256((size_t)((a.rows + kSplitRows - 1) / kSplitRows) * sizeof(int));
  if (l.tc) l.total = l.off_planes + (size_t)3 * a.rows * (a.heads + 2 * a.kv_heads) * a.head_dim * 2;
  return l;
}

// Which kernels a call takes, and its workspace. The kernel of few rows (tiles of up to 8) is
// chosen by the rows that requests have on average, which is all that the host knows.
//
// With a bf16 cache it takes tiles of a row or two, for which the tensor cores' 128 are mostly
// empty. On a B200, there and here: 16 requests of 20 to 1024 tokens, 12 heads of 64, 32.0 us and
// 15.7; 64 of 2000 141 and 91; 16 of 700, 16 heads of 128, 61 and 28, 16 over 8 25.5 and 22.5,
// 64 of 2000 149 and 136. Groups of four and more gain or lose with the lengths, which the host
// does not know (4 requests of 300, 32 heads over 8, 29 and 20; 64 of 100 to 8192 157 and 262),
// and stay.
//
// Single requests may have many rows all the same (a chunk of a prompt beside tokens that are
// decoded, or beside requests that wait), and their keys are read again for every tile. So
// where one can have more tokens than kFewTokens, such requests go to a second kernel, the
// tensor cores' or that of 64 rows; it takes up to 1 us (f32: 0.5) to find that there are none. On a
// B200, 12 heads of 64, with and without it, bf16 cache (f32): 511 requests that wait and a chunk of
// 512 over 8192 67 us and 2136 (430 and 2316), 31 and 32 over 8000 45 and 146, 63 and 64 over
// 1000 27 and 50, 63 that decode and 64 over 1000 78 and 90, 63 and 512 (231 and 297). A few
// tokens cost less where the others are: 31 that decode and 32 over 1000 54.7 and 52.8 (79 and
// 61), 63 that wait and 33 (43 and 34).
constexpr int kFewTokens16 = 16, kFewTokens32 = 64;
struct Plan {
  bool few, both;
  F32Layout f32, many;
  TcLayout tc;
  size_t off_few;  // of the few rows' parts, beside the tensor cores'
  size_t total;
};

Plan plan_call(const Args& a) {
  Plan p = {};
  const int sms = sm_count();
  const bool f32 = a.dtype == MTRTQ_DTYPE_F32;
  if (f32 || a.k_pages) p.f32 = f32_layout(a, sms);
  p.few = f32 ? p.f32.tile_rows <= 8 : a.k_pages && p.f32.tile_rows <= 2;
  p.both = p.few && a.batch > 1 && a.rows > (f32 ? kFewTokens32 : kFewTokens16);
  if (f32) {
    if (p.both) p.many = f32_layout(a, sms, true);
    p.total = p.f32.total > p.many.total ? p.f32.total : p.many.total;
    return p;
  }
  if (!p.few || p.both) p.tc = tc_layout(a, sms);
  p.off_few = round256(p.tc.total);
  p.total = p.few ? p.off_few + p.f32.total : p.tc.total;
  return p;
}

// For requests of least .. most tokens; after: it follows another kernel of the call. parts:
// where l's offsets count from.
int launch_f32(const Args& a, bool paged, const F32Layout& l, int least, int most, bool after, void* workspace,
               uint8_t* parts, unsigned* status, cudaStream_t st) {
  const bool pages16 = a.dtype != MTRTQ_DTYPE_F32, q16 = a.x_dtype != MTRTQ_DTYPE_F32;
  F32Attention p = {};
  fill_list(a, paged, p);
  p.least = least;
  p.most = most;
  p.slot_tokens = 0;
  p.q_buffers = 1;
  p.tile_tokens = l.tile_rows / p.group;
  p.min_steps = 2;
  p.pair_cost = l.tile_rows == 128;  // (every f32 tile is of that kind)
  p.pages16 = pages16;
  p.q16 = q16;
  p.scale = a.scale;
  p.q = static_cast<const float*>(a.q);
  p.k = static_cast<const float*>(paged ? a.k_pages : a.k);
  p.v = static_cast<const float*>(paged ? a.v_pages : a.v);
  p.q_row = a.q_row;
  p.q_head = a.q_head;
  p.k_row = paged ? a.page_stride : a.k_row;
  p.k_head = a.k_head;
  p.v_row = paged ? a.page_stride : a.v_row;
  p.v_head = a.v_head;
  p.num_pages = a.num_pages;
  p.out = static_cast<float*>(a.out);
  p.out_row = a.out_row;
  p.out_head = a.out_head;
  p.counters = static_cast<unsigned*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(parts + l.off_ml);
  p.partials = reinterpret_cast<float*>(parts + l.off_part);
  p.tile_rows = l.tile_rows;
  if (l.tc) {
    const int all = a.heads + 2 * a.kv_heads;
    __nv_bfloat16* planes = reinterpret_cast<__nv_bfloat16*>(parts + l.off_planes);
    int* flags = reinterpret_cast<int*>(parts + l.off_flags);
    F32TcAttention x = {};
    static_cast<F32Attention&>(x) = p;
    x.pair_cost = 2;
    x.flags = flags;
    x.status = status;
    CUtensorMap qm, km, vm;
    const int64_t row = (int64_t)all * a.head_dim;
    const int64_t q_dims[4] = {a.head_dim, p.group, a.kv_heads, 3 * a.rows};
    const int64_t q_strides[3] = {a.head_dim, (int64_t)a.head_dim * p.group, row};
    const int q_box[4] = {64, p.group, 1, x.tile_tokens};
    if (int rc = make_map(&qm, planes, 4, q_dims, q_strides, q_box)) return rc;
    const int64_t dims[3] = {a.head_dim, a.kv_heads, 3 * a.rows}, strides[2] = {a.head_dim, row};
    const int box[3] = {64, 1, 128};
    if (int rc = make_map(&km, planes + (int64_t)a.heads * a.head_dim, 3, dims, strides, box)) return rc;
    if (int rc = make_map(&vm, planes + (int64_t)(a.heads + a.kv_heads) * a.head_dim, 3, dims, strides, box)) return rc;
    if (int rc = cuda_status(launch_split_rows(p, a.heads, planes, flags, st), "attention rows launch")) return rc;
    return cuda_status(launch_attention_f32_tc(x, qm, km, vm, l.grid, st), "attention launch");
  }
  return cuda_status(launch_attention_f32(p, l.grid, after, st), "attention launch");
}

int attention(const Args* a, bool paged, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_args(a, paged)) return rc;
  int rc;
  unsigned* status = device_status_address(&rc);
  if (rc) return rc;
  if (a->rows == 0) return MTRTQ_OK;
  const int64_t need = mtrtq_attention_workspace_bytes(a);
  if (!workspace || (int64_t)workspace_bytes < need)
    return report_error(MTRTQ_ERR_WORKSPACE, "workspace %zu bytes < %lld", workspace_bytes, (long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return report_error(MTRTQ_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Plan p = plan_call(*a);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  __nv_bfloat16* q_rows = p.tc.cast ? reinterpret_cast<__nv_bfloat16*>(ws + p.tc.off_q) : nullptr;
  const bool before = q_rows || (paged && a->k);
  if (before) {
    rc = launch_new_rows(*a, paged, q_rows, reinterpret_cast<__nv_bfloat16*>(ws + p.tc.off_kv), st);
    if (rc) return rc;
  }
  if (a->dtype == MTRTQ_DTYPE_F32) {
    rc = launch_f32(*a, paged, p.f32, 1, p.both ? kFewTokens32 : INT_MAX, before, ws, ws, status, st);
    if (rc == MTRTQ_OK && p.both)
      rc = launch_f32(*a, paged, p.many, kFewTokens32 + 1, INT_MAX, true, ws, ws, status, st);
    return rc;
  }
  if (p.few) {
    rc = launch_f32(*a, paged, p.f32, 1, p.both ? kFewTokens16 : INT_MAX, before, ws, ws + p.off_few, status, st);
    if (rc != MTRTQ_OK || !p.both) return rc;
  }
  return launch_tc(*a, paged, p.tc, p.both ? kFewTokens16 + 1 : 1, before || p.both, ws, status, st);
}

}  // namespace
}  // namespace mtrtq

using namespace mtrtq;

extern "C" {

int64_t mtrtq_attention_workspace_bytes(const mtrtq_attention_args* a) {
  if (check_args(a, a && a->k_pages)) return -1;
  return (int64_t)plan_call(*a).total;
}

int mtrtq_prompt_attention(const mtrtq_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  return attention(a, false, workspace, workspace_bytes, stream);
}

int mtrtq_paged_attention(const mtrtq_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  return attention(a, true, workspace, workspace_bytes, stream);
}

}  // extern "C"
