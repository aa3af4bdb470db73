// What the attention kernels share: PTX wrappers, operand descriptors, the order of loads and
// bounded waits of those on the tensor cores (attention_tc.cu, attention_f32_tc.cu), and how
// f32 parts are joined.
#pragma once

#include <math.h>

#include "attention_sched.cuh"
#include "q8_common.cuh"

namespace mtrtq {

constexpr int kBlock = 128;  // keys per block, rows per tile slot

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
      "%5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}

// Operand descriptors, 128-byte swizzle: the low word has the address and the leading
// byte offset, the high word is the same for all (groups of 8 rows 1024 bytes apart). A step
// of the products moves the address alone, so one thread keeps the tensor cores fed: per
// product an addition or two, where whole descriptors took longer than the product.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
// Q and K: contiguous along the dimensions, which are summed over.
__device__ __forceinline__ uint32_t desc_qk(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | (1u << 16); }
// V as the B operand of O += P V: keys are summed over, dimensions contiguous; the next 64
// dimensions lie 128 rows further (leading byte offset).
__device__ __forceinline__ uint32_t desc_v(uint32_t addr) {
  return ((addr & 0x3FFFFu) >> 4) | ((uint32_t)(kBlock * 128 >> 4) << 16);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a_low), "r"(b_low), "r"(idesc), "r"((uint32_t)add), "r"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_low), "r"(idesc), "r"((uint32_t)add), "r"(kDescHigh)
      : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&u)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Largest of three.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// K and V blocks of a segment in the order the products need them, 2 n loads for n
// blocks; the at-th: whether it is V, and which block c.
__device__ __forceinline__ bool nth_load(bool pair, int at, int n, int& c) {
  if (pair) {
    c = at >> 1;
    return at & 1;
  }
  if (at < 2 && at < n) {
    c = at;
    return false;
  }
  if (at == 2 * n - 1) {
    c = n - 1;
    return true;
  }
  c = at & 1 ? (at + 1) >> 1 : (at - 2) >> 1;
  return !(at & 1);
}

// Tests the phase with the given parity, suspended for as long as the hardware sees fit.
__device__ __forceinline__ bool try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded waits that fail at once when another role has given up. (Many warps wait at any
// time: the clock and the flag are looked at every 64 tests only.)
__device__ __forceinline__ bool wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort_flag, unsigned* status) {
  const long long t0 = clock64();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (clock64() - t0 > kSpinLimitCycles) {
      *abort_flag = 1;
      atomicExch(status, 6u /* MTRTQ_ERR_TIMEOUT */);
      return false;
    }
  }
}
__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity, volatile int* abort_flag, unsigned* status) {
  if (__builtin_expect(try_wait(bar, parity), 1)) return true;
  return wait_slow(bar, parity, abort_flag, status);
}
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, volatile int* abort_flag, unsigned* status) {
  return __all_sync(0xffffffffu, wait_one(bar, parity, abort_flag, status));
}

// After an abort: the copies or products still in flight are waited for, with a limit.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity) && clock64() - t0 < kSpinLimitCycles) {}
}

// Four elements of a row of out, as its type.
__device__ __forceinline__ void put4(float* dst, float4 x) { *reinterpret_cast<float4*>(dst) = x; }
__device__ __forceinline__ void put4(__nv_bfloat16* dst, float4 x) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x, x.y), hi = __floats2bfloat162_rn(x.z, x.w);
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(reinterpret_cast<const uint32_t&>(lo), reinterpret_cast<const uint32_t&>(hi));
}

// The CTA that finishes a cut tile last joins its parts, in order: THREADS threads,
// from the first on.
template <int HD, int BM, int THREADS, typename T = float>
__device__ __forceinline__ void join_parts_f32(const F32Attention& p, const Segment& s) {
  const int c_first = s.c_first, c_last = s.c_last, rows = s.tokens * p.group, vecs = p.head_dim / 4;
#pragma unroll 1
  for (int e = threadIdx.x; e < rows * vecs; e += THREADS) {
    const int row = e / vecs, d = e % vecs * 4, token = row / p.group, head = row - token * p.group;
    float top = -INFINITY;
    for (int64_t c = c_first; c <= c_last; ++c)
      top = fmaxf(top, __ldcg(p.part_ml + (c * 2 + (c == c_first ? 1 : 0)) * BM + row).x);
    float sum = 0.0f;
    float4 x = make_float4(0, 0, 0, 0);
    for (int64_t c = c_first; c <= c_last; ++c) {
      const int64_t at = (c * 2 + (c == c_first ? 1 : 0)) * BM + row;
      const float2 ml = __ldcg(p.part_ml + at);
      if (ml.x == -INFINITY) continue;
      const float w = top == INFINITY ? 1.0f : ex2(ml.x - top);
      const float4 y = __ldcg(reinterpret_cast<const float4*>(p.partials + at * HD + d));
      sum += ml.y * w;
      x.x += y.x * w;
      x.y += y.y * w;
      x.z += y.z * w;
      x.w += y.w * w;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    put4(reinterpret_cast<T*>(p.out) + (s.row0 + (int64_t)token) * p.out_row +
             (int64_t)(s.h * p.group + head) * p.out_head + d,
         make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
  }
  if (threadIdx.x == 0) p.counters[c_first] = 0u;
}

}  // namespace mtrtq
