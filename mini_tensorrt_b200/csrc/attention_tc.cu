// Attention on the 5th-generation tensor cores: packed prompts, and new tokens over a
// paged cache (bf16 products, fp32 accumulators, maximum and sum).
//
// A softmax row needs its running maximum m and sum l alone, so keys are taken in
// blocks of 128 and nothing of a score leaves the SM:
//   S = Q K^T (tensor memory);  m' = max(m, max S);  P = 2^(S c - m');
//   l = l 2^(m - m') + sum P;   O = O 2^(m - m') + P V (tensor memory),  c = scale log2 e.
// m' replaces m only when it is larger by more than 8 (a factor of 2^8 in P, which fp32
// sums and bf16 weights carry without loss), so O is rescaled a few times per row.
//
// Rows: the G query heads of a key/value head read the same keys, so a tile's 128 rows
// are 128 / G tokens times G heads (one 4-D TMA box). Two tile slots run out of phase,
// so that one's exponentials overlap the other's products. With more rows than one
// slot's, the slots hold neighbouring tiles and share each K and V block ("pair");
// otherwise both hold the same rows and take alternate key blocks ("halves"), joined at
// the end -- which is what a single token over a long cache needs.
//
// Work: a step is one block for each slot. The steps of all tiles of all requests form
// one list, cut into equal runs over one CTA per SM; every CTA finds its own run from
// the lengths in device memory. A tile cut between CTAs leaves partial (m, l, O) in the
// workspace, and the CTA that finishes last joins them in order.
//
// One CTA = 12 warps: 0..3 and 4..7 the slots' softmax (a thread per row, also the
// epilogue), 8 TMA loads, 9 MMA issue, 10..11 look over the V blocks that not every row
// sees whole: rows past the request's keys are zeroed (a page's unused rows, the next
// request's rows: 0 * NaN would reach O), and infinities and NaN in rows that only later
// tokens see are taken out and listed; the epilogue adds them to the rows that see them.
#include <math.h>

#include <type_traits>

#include "../../include/mtrtq.h"
#include "attention_sched.cuh"
#include "q8_common.cuh"

namespace mtrtq {

namespace {

constexpr int kBlock = 128;  // keys per block, rows per slot
constexpr int kThreads = 384;
constexpr int kBadMax = 192;  // listed V rows per checking warp: three blocks of 64

template <int DP>
struct Cfg {
  static constexpr int TILE = kBlock * DP * 2;  // Q, K or V block in shared memory
  static constexpr int STAGES = DP == 128 ? 4 : 8;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int OFF_LIST = OFF_KV + STAGES * TILE;
  static constexpr int OFF_WALK = OFF_LIST + StepList::bytes(MTRTQ_MAX_BATCH);
  static constexpr int OFF_SEG = OFF_WALK + kThreads / 32 * ((sizeof(Walk) + 15) / 16 * 16);
  static constexpr int OFF_ML = OFF_SEG + kThreads / 32 * ((sizeof(Segment) + 15) / 16 * 16);  // slot 1's (m, l)
  static constexpr int OFF_BAD = OFF_ML + kBlock * 8;                                         // [2][2][kBadMax] keys
  static constexpr int OFF_BAR = OFF_BAD + 4 * kBadMax * 4;
  static constexpr int NBAR = 3 * STAGES + 17;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = OFF_MISC + 64 + 1024;
  static constexpr int COL_O = 256;
  // One pair of exponentials in this many is a polynomial on the FMA units: the special
  // function units alone would take as long as both products (128 dimensions) or twice
  // as long (64).
  static constexpr int POLY = DP == 128 ? 4 : 2;
  static_assert(BYTES <= 227 * 1024, "shared memory per CTA");
};

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

// V block as the B operand of O += P V: keys are its K side, dimensions (contiguous in
// memory) its N side: 128-byte-swizzled rows of 64 dimensions, 8 keys per 1024 bytes
// (stride byte offset), the next 64 dimensions 128 rows further (leading byte offset).
__device__ __forceinline__ uint64_t desc_v(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)((kBlock * 128) >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
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
// Largest of three, NaN if any is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// 2^x for finite x <= 8, below 2^-126 rounded up to about that: x = n + f with n whole and
// |f| <= 1/2, 2^f by the cubic with the least relative error (7.5e-5, an eighth of a bf16
// rounding), n added to the exponent.
__device__ __forceinline__ float2 exp2_cubic(float2 x) {
  x.x = fmaxf(x.x, -126.0f);
  x.y = fmaxf(x.y, -126.0f);
  const float2 big = make_float2(12582912.0f, 12582912.0f), nbig = make_float2(-12582912.0f, -12582912.0f);
  const float2 t = __fadd2_rn(x, big);  // n in the low bits
  const float2 n = __fadd2_rn(t, nbig);
  const float2 f = __fadd2_rn(x, make_float2(-n.x, -n.y));
  float2 y = fma2(f, make_float2(0.0551716685f, 0.0551716685f), make_float2(0.2426111251f, 0.2426111251f));
  y = fma2(y, f, make_float2(0.6932609677f, 0.6932609677f));
  y = fma2(y, f, make_float2(0.9999280572f, 0.9999280572f));
  return make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + __float_as_uint(y.x)),
                     __uint_as_float((__float_as_uint(t.y) << 23) + __float_as_uint(y.y)));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// K and V blocks of a segment in the order the products need them: `at` 0 .. 2 n - 1
// for n blocks.
__device__ __forceinline__ int order_k(bool pair, int c) { return pair ? 2 * c : c < 2 ? c : 2 * c - 1; }
__device__ __forceinline__ int order_v(bool pair, int c, int n) { return pair ? 2 * c + 1 : min(2 * c + 2, 2 * n - 1); }

// The at-th of them: whether it is V, and which block c.
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

// Bounded waits that fail at once when another role has given up.
__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity, volatile int* abort_flag, unsigned* status) {
  if (mbar_test_wait(bar, parity)) return true;
  if (*abort_flag) return false;
  return mbar_wait_bounded(bar, parity, abort_flag, status);
}
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, volatile int* abort_flag, unsigned* status) {
  return __all_sync(0xffffffffu, wait_one(bar, parity, abort_flag, status));
}

// After an abort: the copies or products still in flight are waited for, with a limit.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity) && clock64() - t0 < kSpinLimitCycles) {}
}

// One row of a cut tile from the parts of CTAs c_first .. c_last, in order.
template <int DP>
__device__ __noinline__ void join_parts(const TcAttention& p, int c_first, int c_last, int prow, __nv_bfloat16* out) {
  const int64_t rows = p.part_rows;
  float top = -INFINITY;
  for (int c = c_first; c <= c_last; ++c)
    top = fmaxf(top, __ldcg(p.part_ml + (c * 2 + (c == c_first)) * rows + prow).x);
  float sum = 0.0f;
  for (int c = c_first; c <= c_last; ++c) {
    const float2 ml = __ldcg(p.part_ml + (c * 2 + (c == c_first)) * rows + prow);
    if (ml.x != -INFINITY) sum += ml.y * (top == INFINITY ? 1.0f : ex2(ml.x - top));
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  for (int i = 0; i < p.head_dim; i += 8) {
    float o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int c = c_first; c <= c_last; ++c) {
      const int64_t part = c * 2 + (c == c_first);
      const float pm = __ldcg(p.part_ml + part * rows + prow).x;
      if (pm == -INFINITY) continue;
      const float w = top == INFINITY ? 1.0f : ex2(pm - top);
      const float4* po = reinterpret_cast<const float4*>(p.partials) + part * rows * (DP / 4) + prow;
      const float4 a = __ldcg(po + (i / 4) * rows), b = __ldcg(po + (i / 4 + 1) * rows);
      o[0] += w * a.x;
      o[1] += w * a.y;
      o[2] += w * a.z;
      o[3] += w * a.w;
      o[4] += w * b.x;
      o[5] += w * b.y;
      o[6] += w * b.z;
      o[7] += w * b.w;
    }
    *reinterpret_cast<uint4*>(out + i) = make_uint4(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv),
                                                    pack_bf16(o[4] * inv, o[5] * inv), pack_bf16(o[6] * inv, o[7] * inv));
  }
}

// After a bounded wait gives up, every role goes on through its loops without waiting,
// copying or multiplying (each wait returns at once), so that all reach the barriers
// between them and the end.
template <int DP, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1)
    attention_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap, const __grid_constant__ TcAttention p) {
  using C = Cfg<DP>;
  constexpr int NH = DP / 64;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const StepList list(smem + C::OFF_LIST, MTRTQ_MAX_BATCH);
  float2* ml1 = reinterpret_cast<float2*>(smem + C::OFF_ML);
  int* bad = reinterpret_cast<int*>(smem + C::OFF_BAD);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* empty = full + C::STAGES;
  uint64_t* checked = empty + C::STAGES;
  uint64_t* q_full = checked + C::STAGES;  // [2], a barrier for each slot or buffer
  uint64_t* q_free = q_full + 2;
  uint64_t* s_full = q_free + 2;
  uint64_t* p_half = s_full + 2;           // the weights of the block's first 64 keys
  uint64_t* p_full = p_half + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* o_free = o_full + 2;
  uint64_t* list_free = o_free + 2;
  uint64_t* drained = list_free + 2;
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* s_abort = reinterpret_cast<volatile int*>(misc + 1);
  volatile unsigned* s_ticket = misc + 2;
  volatile int* bad_count = reinterpret_cast<volatile int*>(misc + 4);  // [2][2]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Walk* walks = reinterpret_cast<Walk*>(smem + C::OFF_WALK);
  Walk& walk = walks[warp];
  Segment& s = reinterpret_cast<Segment*>(smem + C::OFF_SEG)[warp];

  if (tid == 0) {
    for (int x = 0; x < C::STAGES; ++x) {
      mbar_init(&full[x], 1);
      mbar_init(&empty[x], 3);  // the products, two checking warps
      mbar_init(&checked[x], 2);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_free[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_half[t], 4);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_free[t], 4);
      mbar_init(&list_free[t], 8);
    }
    mbar_init(drained, 1);
    *s_abort = 0;
    for (int x = 0; x < 4; ++x) bad_count[x] = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(misc, 512);
    tmem_relinquish();
  }
  if (warp == 8 && lane == 0) {
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  tc_fence_before();
  make_list<kBlock, kThreads>(p, list, walks);
  tc_fence_after();
  const uint32_t tmem = misc[0];
  // The kernel that stored the new keys and cast the rows is complete from here on.
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int ksteps = (p.head_dim + 15) / 16;

  // 256 threads of 200 registers and 128 of 104: the 384 x 168 of the launch.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---------------- softmax and epilogue ----------------
    const int t = warp >> 2;                           // slot
    const int row = tid & 127;                         // of the slot's tile
    const uint32_t quad = (uint32_t)(warp & 3) << 21;  // lanes 32 (warp & 3) .. of TMEM
    const uint32_t s_addr = tmem + quad + t * kBlock, o_addr = tmem + quad + C::COL_O + t * DP;
    const int token = row / p.group, head = row - token * p.group;
    const float c2 = p.scale * 1.4426950408889634f;  // scale log2 e
    const float2 cc = make_float2(c2, c2);
    uint32_t n_s = 0, n_o = 0;
    for (int seg = 0; next_segment<kBlock>(p, list, walk, s); ++seg) {
      const int tok = (s.pair ? t * p.slot_tokens : 0) + token;  // of the tile's
      const bool live = token < p.slot_tokens && tok < s.tokens;
      const int keys = live ? max(0, min(s.see0 + tok, s.keys)) : 0;  // that this row sees
      const bool warp_live = __any_sync(0xffffffffu, live);
      const int cnt = s.cnt[t], stride = s.pair ? kBlock : 2 * kBlock;
      int left = keys - (s.k0 + (s.pair ? 0 : t)) * kBlock;  // columns of the block that it sees
      float m = -INFINITY, l = 0.0f;
      for (int x = 0; x < cnt; ++x, left -= stride) {
        const bool ok = wait_all(&s_full[t], n_s & 1, s_abort, p.status);
        ++n_s;
        if (!ok || !warp_live) {
          if (lane == 0) {
            mbar_arrive(&p_half[t]);
            mbar_arrive(&p_full[t]);
          }
          continue;
        }
        tc_fence_after();
        float v[kBlock];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32(s_addr + 32 * i, v + 32 * i);
        tmem_wait_ld();
        if (__any_sync(0xffffffffu, left < kBlock)) {
#pragma unroll
          for (int i = 0; i < kBlock; ++i) v[i] = i < left ? v[i] : -INFINITY;
        }
        float top = max3(v[0], v[1], v[2]), top1 = max3(v[3], v[4], v[5]);
#pragma unroll
        for (int i = 6; i + 3 < kBlock; i += 4) {
          top = max3(top, v[i], v[i + 1]);
          top1 = max3(top1, v[i + 2], v[i + 3]);
        }
        top = max3(top, top1, max3(v[kBlock - 2], v[kBlock - 1], top1)) * c2;
        // Masked, infinite or NaN scores: every exponential by the instruction, which
        // keeps them exact.
        const bool exact = __any_sync(0xffffffffu, left < kBlock || !(fabsf(top) < INFINITY));
        const bool grow = top > m + 8.0f || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, grow)) {
          const float m1 = grow ? top : m;
          const float keep = m1 == -INFINITY ? 1.0f : ex2(m - m1);
          l *= keep;
          m = m1;
          if (x > 0) {
            // this slot's earlier products are complete: their scores came after them
#pragma unroll 1
            for (int i = 0; i < DP; i += 16) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(o_addr + i, o);
              tmem_wait_ld();
#pragma unroll
              for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * keep);
              tmem_st16(o_addr + i, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float2 sum = make_float2(0.0f, 0.0f);
        const float2 mm = make_float2(-base, -base);
        auto weights = [&](auto some_cubic) {
#pragma unroll
          for (int i = 0; i < kBlock; i += 32) {
            uint32_t w[16];
#pragma unroll
            for (int y = 0; y < 16; ++y) {
              float2 e = fma2(make_float2(v[i + 2 * y], v[i + 2 * y + 1]), cc, mm);
              if (decltype(some_cubic)::value && y % C::POLY == C::POLY - 1) {
                e = exp2_cubic(e);
              } else {
                e.x = ex2(e.x);
                e.y = ex2(e.y);
              }
              sum = __fadd2_rn(sum, e);
              w[y] = pack_bf16(e.x, e.y);
            }
            tmem_st16(s_addr + (i >> 1), w);
            if (i == kBlock / 2 - 32) {
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&p_half[t]);
            }
          }
        };
        if (exact) weights(std::false_type());
        else weights(std::true_type());
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
        l += sum.x + sum.y;
      }

      if (m == -INFINITY && l != l) m = 0.0f;  // every score it saw was NaN
      bool ok = true;
      if (cnt > 0) {
        ok = wait_all(&o_full[t], n_o & 1, s_abort, p.status);
        ++n_o;
        tc_fence_after();
      }
      // halves: slot 0's threads join the two slots' rows
      const bool mine = s.pair || t == 0, two = !s.pair && s.n > 1;
      float w0 = 1.0f, w1 = 0.0f;
      if (!s.pair) {
        if (t == 1) ml1[row] = make_float2(m, l);
        tc_fence_before();
        named_bar_sync(1, 256);
        tc_fence_after();
        if (two && t == 0) {
          const float2 ml = ml1[row];
          const float top = fmaxf(m, ml.x);
          w0 = m == -INFINITY ? 0.0f : top == INFINITY ? 1.0f : ex2(m - top);
          w1 = ml.x == -INFINITY ? 0.0f : top == INFINITY ? 1.0f : ex2(ml.x - top);
          l = l * w0 + ml.y * w1;
          m = top;
        }
      }
      if (m == -INFINITY) w0 = 0.0f;  // no key seen (and perhaps no product formed)
      const int prow = (s.pair ? t * kBlock : 0) + row;
      const int64_t at_out =
          (int64_t)(s.row0 + tok) * p.out_row + (int64_t)(s.h * p.group + head) * p.out_head;
      const int64_t part = (int64_t)blockIdx.x * 2 + s.part;
      float* to_part = p.partials + (part * p.part_rows * (DP / 4) + prow) * 4;
      if (mine && ok) {
        if (s.whole) {
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          w0 *= inv;
          w1 *= inv;
        }
#pragma unroll 1
        for (int i = 0; i < p.head_dim; i += 32) {
          float o[32];
          if (cnt > 0) {
            tmem_ld32(o_addr + i, o);
            tmem_wait_ld();
          }
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = w0 == 0.0f ? 0.0f : o[y] * w0;
          if (two) {
            float o1[32];
            tmem_ld32(o_addr + DP + i, o1);
            tmem_wait_ld();
            if (w1 != 0.0f) {
#pragma unroll
              for (int y = 0; y < 32; ++y) o[y] = fmaf(o1[y], w1, o[y]);
            }
          }
          if (live) {
            if (s.whole) {
#pragma unroll
              for (int y = 0; y < 32; y += 8) {
                if (i + y < p.head_dim)
                  *reinterpret_cast<uint4*>(p.out + at_out + i + y) =
                      make_uint4(pack_bf16(o[y], o[y + 1]), pack_bf16(o[y + 2], o[y + 3]),
                                 pack_bf16(o[y + 4], o[y + 5]), pack_bf16(o[y + 6], o[y + 7]));
              }
            } else {
#pragma unroll
              for (int y = 0; y < 32; y += 4)
                __stcg(reinterpret_cast<float4*>(to_part + (int64_t)(i + y) * p.part_rows),
                       make_float4(o[y], o[y + 1], o[y + 2], o[y + 3]));
            }
          }
        }
        if (live && !s.whole) __stcg(p.part_ml + part * p.part_rows + prow, make_float2(m, l));
        // The infinities and NaN that were taken out of the last blocks' V, for the rows
        // that see them. A slot without blocks here has not waited for the check, and
        // sees none of it.
        const int par = seg & 1;
        if (cnt > 0 && (s.k0 + s.n) * kBlock > s.all_see()) {
          for (int w = 0; w < 2; ++w) {
            const int have = min(kBadMax, bad_count[par * 2 + w]);
            for (int x = 0; x < have; ++x) {
              const int key = bad[(par * 2 + w) * kBadMax + x];
              if ((unsigned)key >= (unsigned)keys) continue;
              const __nv_bfloat16* src;
              if (PAGED) {
                const int64_t page = p.table[s.b * p.table_ld + key / p.page_size];
                src = p.v + page * p.v_row + ((int64_t)s.h * p.page_size + key % p.page_size) * p.head_dim;
              } else {
                src = p.v + (int64_t)(list.req[s.b].r0 + key) * p.v_row + s.h * p.v_head;
              }
              for (int d = 0; d < p.head_dim; ++d) {
                const float z = __bfloat162float(src[d]);
                if (fabsf(z) < INFINITY) continue;
                if (s.whole) {
                  p.out[at_out + d] = __float2bfloat16_rn(__bfloat162float(p.out[at_out + d]) + z);
                } else {
                  float* to = to_part + (int64_t)(d & ~3) * p.part_rows + (d & 3);
                  __stcg(to, __ldcg(to) + z);
                }
              }
            }
          }
        }
      }
      // O and the list have been read.
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (mine && cnt > 0) mbar_arrive(&o_free[t]);
        if (two && t == 0) mbar_arrive(&o_free[1]);
        mbar_arrive(&list_free[seg & 1]);
      }
      if (!s.pair) named_bar_sync(2, 256);  // ml1 has been read
      if (!s.whole && mine) {
        const int id = s.pair ? 3 : 4, count = s.pair ? 256 : 128;
        named_bar_sync(id, count);
        if (tid == 0) *s_ticket = ticket_acq_rel(p.counters + s.c_first);
        named_bar_sync(id, count);
        const bool last = *s_ticket == (unsigned)(s.c_last - s.c_first);
        if (last && live) join_parts<DP>(p, s.c_first, s.c_last, prow, p.out + at_out);
        if (last && tid == 0) p.counters[s.c_first] = 0u;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 8) {
      // ---------------- loads ----------------
      uint32_t seq = 0, sent = 0;
      int q_sent[2] = {0, 0};
      const int pages = PAGED ? kBlock / p.page_size : 1;
      const uint32_t box = (PAGED ? p.page_size : kBlock) * 128;
      const uint32_t rows_bytes = (uint32_t)p.slot_tokens * p.group * 128 * NH;
      while (next_segment<kBlock>(p, list, walk, s)) {
        const int k0 = s.k0, n = s.n;
        const bool pair = s.pair;
        for (int t = 0; t < (pair ? 2 : 1); ++t) {
          const int buf = pair ? t : s.buf;
          if (!wait_all(&q_free[buf], (s.q_use[buf] & 1) ^ 1, s_abort, p.status)) continue;
          ++q_sent[buf];
          if (lane == 0) mbar_arrive_expect_tx(&q_full[buf], rows_bytes);
          __syncwarp();
          if (lane < NH)
            tma_load_4d(smem + C::OFF_Q + buf * C::TILE + lane * kBlock * 128, &qmap, lane * 64, 0, s.h,
                        s.row0 + t * p.slot_tokens, &q_full[buf]);
        }
        const int r0 = PAGED ? 0 : list.req[s.b].r0;
        for (int at = 0; at < 2 * n; ++at, ++seq) {
          int c;
          const bool is_v = nth_load(pair, at, n, c);
          const int st = seq % C::STAGES;
          const int key0 = (k0 + c) * kBlock;
          const int pg = lane % pages, half = lane / pages;
          bool load = lane < pages * NH;
          int page = 0;
          if (PAGED) {
            load = load && key0 + pg * p.page_size < s.keys;
            if (load) page = p.table[s.b * p.table_ld + (k0 + c) * pages + pg];
          }
          if (!wait_all(&empty[st], ((seq / C::STAGES) & 1) ^ 1, s_abort, p.status)) continue;
          sent = seq + 1;
          const unsigned who = __ballot_sync(0xffffffffu, load);
          if (lane == 0) mbar_arrive_expect_tx(&full[st], box * __popc(who));
          __syncwarp();
          if (load) {
            uint8_t* dst = smem + C::OFF_KV + st * C::TILE + half * kBlock * 128 + (PAGED ? pg * box : 0);
            if (PAGED)
              tma_load_3d(dst, is_v ? &vmap : &kmap, half * 64, s.h * p.page_size, page, &full[st]);
            else
              tma_load_3d(dst, is_v ? &vmap : &kmap, half * 64, s.h, r0 + key0, &full[st]);
          }
        }
      }
      // No copy may be in flight when the CTA exits: without an abort the products have
      // waited for every one.
      if (*s_abort && lane == 0) {
        for (int t = 0; t < 2; ++t)
          if (q_sent[t]) drain(&q_full[t], (q_sent[t] - 1) & 1);
        for (uint32_t x = sent > C::STAGES ? sent - C::STAGES : 0; x < sent; ++x)
          drain(&full[x % C::STAGES], (x / C::STAGES) & 1);
      }
      __syncwarp();
    } else if (warp == 9) {
      // ---------------- products ----------------
      const uint32_t idesc_s = umma_idesc_bf16(kBlock, kBlock);
      const uint32_t idesc_o = umma_idesc_bf16(kBlock, ksteps * 16) | (1u << 16);  // B is contiguous along N
      const uint32_t q_addr = smem_u32(smem + C::OFF_Q), kv_addr = smem_u32(smem + C::OFF_KV);
      uint32_t base = 0, fixed = 0;  // loads so far; phase of each stage's check
      uint32_t n_p[2] = {0, 0}, n_seg[2] = {0, 0};
      while (next_segment<kBlock>(p, list, walk, s)) {
        if (lane == 0) {
          const bool pair = s.pair;
          const int n = s.n, k0 = s.k0, all_see = s.all_see();
          const int cnt[2] = {s.cnt[0], s.cnt[1]};
          auto block_of = [&](int t, int x) { return pair ? x : 2 * x + t; };
          auto wait_load = [&](uint32_t at) {
            return wait_one(&full[at % C::STAGES], (at / C::STAGES) & 1, s_abort, p.status);
          };
          auto scores = [&](int t, int x) {
            const int c = block_of(t, x), buf = pair ? t : s.buf;
            const uint32_t at = base + order_k(pair, c);
            if (!wait_load(at)) return;
            tc_fence_after();
            const uint32_t k = kv_addr + (at % C::STAGES) * C::TILE, q = q_addr + buf * C::TILE;
            for (int i = 0; i < ksteps; ++i) {
              const uint32_t off = (i >> 2) * kBlock * 128 + (i & 3) * 32;
              umma_ss(tmem + t * kBlock, umma_desc_sw128(q + off), umma_desc_sw128(k + off), idesc_s, i > 0);
            }
            umma_commit(&s_full[t]);
            if (!pair || t == 1) umma_commit(&empty[at % C::STAGES]);
            if (pair ? x == cnt[t] - 1 : c == n - 1) umma_commit(&q_free[buf]);
          };
          bool ok = true;
          for (int t = 0; t < (pair ? 2 : 1); ++t) {
            const int buf = pair ? t : s.buf;
            ok = wait_one(&q_full[buf], s.q_use[buf] & 1, s_abort, p.status) && ok;
          }
          for (int t = 0; t < 2; ++t)
            if (ok && cnt[t] > 0) scores(t, 0);
          if (pair && cnt[0] == 0) umma_commit(&q_free[0]);
          uint32_t was_checked = 0;  // pair: slot 0 has waited for this stage's check
          for (int x = 0; x < max(cnt[0], cnt[1]); ++x) {
            for (int t = 0; t < 2; ++t) {
              if (x >= cnt[t]) continue;
              const int c = block_of(t, x);
              const uint32_t at = base + order_v(pair, c, n), st = at % C::STAGES;
              if (x == 0) wait_one(&o_free[t], (n_seg[t] & 1) ^ 1, s_abort, p.status);
              wait_load(at);
              if ((k0 + c + 1) * kBlock > all_see && !(pair && t == 1 && (was_checked >> st & 1))) {
                wait_one(&checked[st], fixed >> st & 1, s_abort, p.status);
                fixed ^= 1u << st;
                was_checked |= 1u << st;
              }
              const uint32_t v = kv_addr + st * C::TILE;
              for (int half = 0; half < 2; ++half) {
                wait_one(half ? &p_full[t] : &p_half[t], n_p[t] & 1, s_abort, p.status);
                if (*s_abort) break;
                tc_fence_after();
#pragma unroll
                for (int i = half * 4; i < half * 4 + 4; ++i)
                  umma_ts(tmem + C::COL_O + t * DP, tmem + t * kBlock + i * 8, desc_v(v + i * 2048), idesc_o,
                          x > 0 || i > 0);
              }
              ++n_p[t];
              if (*s_abort) continue;
              if (!pair || t == 1) {
                umma_commit(&empty[st]);
                was_checked &= ~(1u << st);
              }
              if (x + 1 < cnt[t]) scores(t, x + 1);
              else umma_commit(&o_full[t]);
            }
          }
          for (int t = 0; t < 2; ++t)
            if (cnt[t] > 0) ++n_seg[t];
          base += 2 * n;
        }
        __syncwarp();
      }
      if (lane == 0 && *s_abort) {  // the products in flight end before TMEM is freed
        umma_commit(drained);
        drain(drained, 0);
      }
      __syncwarp();
    } else {
      // ---------------- V blocks that not every row sees whole ----------------
      const int w = warp - 10;
      uint32_t base = 0;
      for (int seg = 0; next_segment<kBlock>(p, list, walk, s); ++seg) {
        const bool pair = s.pair;
        const int n = s.n, k0 = s.k0, keys = s.keys, all_see = s.all_see(), par = seg & 1;
        bool first = true;
        for (int x = 0; x < 2 * n; ++x) {
          int c;
          const bool is_v = nth_load(pair, x, n, c);
          const int key0 = (k0 + c) * kBlock;
          const uint32_t at = base + x, st = at % C::STAGES;
          // every load is followed, so that no phase of its barrier is taken for another
          const bool landed = wait_all(&full[st], (at / C::STAGES) & 1, s_abort, p.status);
          if (!is_v || key0 + kBlock <= all_see) {
            if (lane == 0) mbar_arrive(&empty[st]);
            continue;
          }
          if (first) {
            wait_all(&list_free[par], ((seg >> 1) & 1) ^ 1, s_abort, p.status);
            if (lane == 0) bad_count[par * 2 + w] = 0;
            __syncwarp();
            first = false;
          }
          if (landed) {
            uint8_t* v = smem + C::OFF_KV + st * C::TILE;
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
              const int r = w * 64 + rr * 32 + lane;
              const bool kept = key0 + r < keys;
              bool broken = false;
              for (int y = 0; y < NH * 8; ++y) {
                uint4* at16 =
                    reinterpret_cast<uint4*>(v + (y >> 3) * kBlock * 128 + r * 128 + (((y & 7) ^ (r & 7)) << 4));
                if (!kept) {
                  *at16 = make_uint4(0, 0, 0, 0);
                  continue;
                }
                uint4 u = *at16;
                uint32_t* e = reinterpret_cast<uint32_t*>(&u);
                bool hit = false;
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                  if ((e[z] & 0x7f80u) == 0x7f80u) { e[z] &= 0xffff0000u; hit = true; }
                  if ((e[z] & 0x7f800000u) == 0x7f800000u) { e[z] &= 0xffffu; hit = true; }
                }
                if (hit) *at16 = u;
                broken |= hit;
              }
              const unsigned who = __ballot_sync(0xffffffffu, broken);
              if (who) {
                const int had = bad_count[par * 2 + w];
                __syncwarp();
                const int to = had + __popc(who & ((1u << lane) - 1));
                if (broken && to < kBadMax) bad[(par * 2 + w) * kBadMax + to] = key0 + r;
                __threadfence_block();  // slot 0 may read while slot 1's last blocks are looked over
                __syncwarp();
                if (lane == 0) bad_count[par * 2 + w] = min(kBadMax, had + __popc(who));
                __syncwarp();
              }
            }
            fence_proxy_async_smem();
          }
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&checked[st]);
            mbar_arrive(&empty[st]);
          }
        }
        base += 2 * n;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int DP, bool PAGED>
cudaError_t launch_one(const TcAttention& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, int grid,
                       bool pdl, cudaStream_t st) {
  auto kernel = attention_tc_kernel<DP, PAGED>;
  if (cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kernel), Cfg<DP>::BYTES)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<DP>::BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, q, k, v, p);
}

}  // namespace

cudaError_t launch_attention_tc(const TcAttention& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                                int grid, bool pdl, cudaStream_t st) {
  if (p.head_dim <= 64)
    return p.table ? launch_one<64, true>(p, q, k, v, grid, pdl, st) : launch_one<64, false>(p, q, k, v, grid, pdl, st);
  return p.table ? launch_one<128, true>(p, q, k, v, grid, pdl, st) : launch_one<128, false>(p, q, k, v, grid, pdl, st);
}

}  // namespace mtrtq
