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
  static constexpr int OFF_PREFIX = OFF_KV + STAGES * TILE;
  static constexpr int OFF_ML = OFF_PREFIX + (MTRTQ_MAX_BATCH + 1) * 8;  // slot 1's (m, l), then its rows
  static constexpr int OFF_BAD = OFF_ML + kBlock * 8;                    // [2][2][kBadMax] keys
  static constexpr int OFF_BAR = OFF_BAD + 4 * kBadMax * 4;
  static constexpr int NBAR = 3 * STAGES + 13;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = OFF_MISC + 64 + 1024;
  static constexpr int COL_O = 256;
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
  int64_t* prefix = reinterpret_cast<int64_t*>(smem + C::OFF_PREFIX);
  float2* ml1 = reinterpret_cast<float2*>(smem + C::OFF_ML);
  int* bad = reinterpret_cast<int*>(smem + C::OFF_BAD);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* empty = full + C::STAGES;
  uint64_t* checked = empty + C::STAGES;
  uint64_t* q_full = checked + C::STAGES;
  uint64_t* q_free = q_full + 1;
  uint64_t* s_full = q_free + 1;   // [2]
  uint64_t* p_full = s_full + 2;   // [2]
  uint64_t* o_full = p_full + 2;   // [2]
  uint64_t* o_free = o_full + 2;   // [2]
  uint64_t* list_free = o_free + 2;  // [2]
  uint64_t* drained = list_free + 2;
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* s_abort = reinterpret_cast<volatile int*>(misc + 1);
  volatile unsigned* s_ticket = misc + 2;
  volatile int* bad_count = reinterpret_cast<volatile int*>(misc + 4);  // [2][2]
  volatile int* s_start = reinterpret_cast<volatile int*>(misc + 8);    // b, h, i, j

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 3);  // the products, two checking warps
      mbar_init(&checked[s], 2);
    }
    mbar_init(q_full, 1);
    mbar_init(q_free, 1);
    mbar_init(drained, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_free[t], 4);
      mbar_init(&list_free[t], 8);
    }
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
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = misc[0];
  int64_t per;
  const Walk<kBlock> walk0 = find_run<kBlock, kThreads>(p, prefix, s_start, per);
  // The kernel that stored the new keys and cast the rows is complete from here on.
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int ksteps = (p.head_dim + 15) / 16;
  Segment s;
  Walk<kBlock> walk = walk0;

  // 256 threads of 200 registers and 128 of 104: the 384 x 168 of the launch.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---------------- softmax and epilogue ----------------
    const int t = warp >> 2;          // slot
    const int row = tid & 127;        // of the slot's tile
    const uint32_t quad = (uint32_t)(warp & 3) << 21;  // lanes 32 (warp & 3) .. of TMEM
    const uint32_t s_addr = tmem + quad + t * kBlock, o_addr = tmem + quad + C::COL_O + t * DP;
    const int token = row / p.group, head = row - token * p.group;
    const float c2 = p.scale * 1.4426950408889634f;  // scale log2 e
    uint32_t n_s = 0, n_o = 0;
    int seg = 0;
    for (; walk.next(p, s); ++seg) {
      const bool pair = s.tile.pair;
      const int k0 = pair ? s.j0 : 2 * s.j0;
      const int n = (pair ? s.j1 : min(2 * s.j1, s.tile.blocks)) - k0;
      const int tok = s.tile.t0 + (pair ? t * p.slot_tokens : 0) + token;
      const bool live = token < p.slot_tokens && tok < s.tile.t0 + s.tile.tokens;
      const int64_t seen = s.q.ctx + tok + 1;
      const int keys = !live ? 0 : (int)max((int64_t)0, min(seen, (int64_t)s.q.keys));  // this row sees
      int cnt;
      if (pair && t == 0) {
        const int64_t seen0 = s.q.ctx + s.tile.t0 + p.slot_tokens;
        const int keys0 = (int)(seen0 < s.q.keys ? seen0 : s.q.keys);
        cnt = max(0, min(s.j1, keys0 <= 0 ? 0 : (keys0 + kBlock - 1) / kBlock) - s.j0);
      } else {
        cnt = pair ? n : t == 0 ? (n + 1) >> 1 : n >> 1;
      }
      const bool warp_live = __any_sync(0xffffffffu, live);
      float m = -INFINITY, l = 0.0f;
      for (int x = 0; x < cnt; ++x) {
        const int key0 = (k0 + (pair ? x : 2 * x + t)) * kBlock;
        const bool ok = wait_all(&s_full[t], n_s & 1, s_abort, p.status);
        ++n_s;
        if (ok && warp_live) {
          tc_fence_after();
          float v[kBlock];
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_ld32(s_addr + 32 * i, v + 32 * i);
          tmem_wait_ld();
          const int left = keys - key0;  // columns this row sees
          if (__any_sync(0xffffffffu, left < kBlock)) {
#pragma unroll
            for (int i = 0; i < kBlock; ++i) v[i] = i < left ? v[i] : -INFINITY;
          }
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < kBlock; i += 2) top = fmaxf(top, fmaxf(v[i], v[i + 1]));
          top *= c2;
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
          const float2 cc = make_float2(c2, c2), mm = make_float2(-base, -base);
#pragma unroll
          for (int i = 0; i < kBlock; i += 32) {
            uint32_t w[16];
#pragma unroll
            for (int y = 0; y < 16; ++y) {
              float2 e = fma2(make_float2(v[i + 2 * y], v[i + 2 * y + 1]), cc, mm);
              e.x = ex2(e.x);
              e.y = ex2(e.y);
              sum = __fadd2_rn(sum, e);
              w[y] = pack_bf16(e.x, e.y);
            }
            tmem_st16(s_addr + (i >> 1), w);
          }
          l += sum.x + sum.y;
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (m == -INFINITY && l != l) m = 0.0f;  // every score it saw was NaN
      bool ok = true;
      if (cnt > 0) {
        ok = wait_all(&o_full[t], n_o & 1, s_abort, p.status);
        ++n_o;
        tc_fence_after();
      }
      // The V rows taken out of the last blocks (the epilogue of a whole tile or of the
      // CTA that joins one adds them; they are the same in every part that has them).
      const int par = seg & 1;
      const int64_t t0_sees = s.q.ctx + s.tile.t0 + 1;
      // A slot without blocks here has not waited for the check, and sees none of it.
      const bool any_checked = cnt > 0 && (int64_t)(k0 + n) * kBlock > min(t0_sees, (int64_t)s.q.keys);
      float other_m = -INFINITY, other_l = 0.0f;
      bool mine = pair || t == 0;  // this thread finishes its row
      if (!pair) {
        if (t == 1) ml1[row] = cnt > 0 ? make_float2(m, l) : make_float2(-INFINITY, 0.0f);
        tc_fence_before();
        named_bar_sync(1, 256);
        tc_fence_after();
        if (t == 0) {
          other_m = ml1[row].x;
          other_l = ml1[row].y;
        }
      }
      const bool two = !pair && n > 1;  // slot 1 has products too
      const float top = fmaxf(m, other_m);
      float w0 = m == -INFINITY ? 0.0f : ex2(m - top), w1 = other_m == -INFINITY ? 0.0f : ex2(other_m - top);
      if (top == INFINITY) w0 = w1 = 1.0f;  // sums and products are NaN by then
      const float lsum = l * w0 + other_l * w1;
      const bool whole = s.whole();
      const int64_t out_at = (s.q.r0 + tok) * p.out_row + (int64_t)(s.h * p.group + head) * p.out_head;
      const int rows_cap = p.part_rows;
      // Columns [i, i + 32) of this row's products, joined over the slots, with the
      // infinities and NaN that were taken out.
      auto columns = [&](int i, float* o) {
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
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] += w1 == 0.0f ? 0.0f : o1[y] * w1;
        }
        if (any_checked) {
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
                src = p.v + (s.q.r0 + key) * p.v_row + s.h * p.v_head;
              }
              for (int y = 0; y < 32 && i + y < p.head_dim; ++y) {
                const float z = __bfloat162float(src[i + y]);
                if (!(fabsf(z) < INFINITY)) {
#pragma unroll
                  for (int q = 0; q < 32; ++q)
                    if (q == y) o[q] += z;
                }
              }
            }
          }
        }
      };
      if (mine && ok && whole) {
        const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
#pragma unroll
        for (int i = 0; i < DP; i += 32) {
          float o[32];
          columns(i, o);
          if (live) {
#pragma unroll
            for (int y = 0; y < 32; y += 8) {
              if (i + y < p.head_dim)
                *reinterpret_cast<uint4*>(p.out + out_at + i + y) =
                    make_uint4(pack_bf16(o[y] * inv, o[y + 1] * inv), pack_bf16(o[y + 2] * inv, o[y + 3] * inv),
                               pack_bf16(o[y + 4] * inv, o[y + 5] * inv), pack_bf16(o[y + 6] * inv, o[y + 7] * inv));
            }
          }
        }
      } else if (mine && ok) {
        const int prow = (pair ? t * kBlock : 0) + row;
        const int64_t part = (int64_t)blockIdx.x * 2 + (s.j0 > 0 ? 0 : 1);
        float4* po = reinterpret_cast<float4*>(p.partials) + part * rows_cap * (DP / 4);
#pragma unroll
        for (int i = 0; i < DP; i += 32) {
          float o[32];
          columns(i, o);
          if (live) {
#pragma unroll
            for (int y = 0; y < 32; y += 4)
              __stcg(po + (int64_t)((i + y) / 4) * rows_cap + prow, make_float4(o[y], o[y + 1], o[y + 2], o[y + 3]));
          }
        }
        if (live) __stcg(p.part_ml + part * rows_cap + prow, make_float2(top, lsum));
      }
      // O and the list have been read.
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (mine && cnt > 0) mbar_arrive(&o_free[t]);
        if (two && t == 0) mbar_arrive(&o_free[1]);
        mbar_arrive(&list_free[par]);
      }
      if (!pair) named_bar_sync(2, 256);  // ml1 has been read
      if (!whole && mine) {
        const int id = pair ? 3 : 4, count = pair ? 256 : 128;
        const int64_t c_first = s.first / per, c_last = (s.first + s.tile.steps - 1) / per;
        named_bar_sync(id, count);
        if (tid == 0) *s_ticket = ticket_acq_rel(p.counters + c_first);
        named_bar_sync(id, count);
        const bool last = *s_ticket == (unsigned)(c_last - c_first);
        if (last && live) {
          const int prow = (pair ? t * kBlock : 0) + row;
          float mx = -INFINITY;
          for (int64_t c = c_first; c <= c_last; ++c)
            mx = fmaxf(mx, __ldcg(p.part_ml + (c * 2 + (c == c_first ? 1 : 0)) * rows_cap + prow).x);
          float sum = 0.0f;
          for (int64_t c = c_first; c <= c_last; ++c) {
            const float2 ml = __ldcg(p.part_ml + (c * 2 + (c == c_first ? 1 : 0)) * rows_cap + prow);
            if (ml.x != -INFINITY) sum += ml.y * (mx == INFINITY ? 1.0f : ex2(ml.x - mx));
          }
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          for (int i = 0; i < p.head_dim; i += 8) {
            float o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            for (int64_t c = c_first; c <= c_last; ++c) {
              const int64_t part = c * 2 + (c == c_first ? 1 : 0);
              const float pm = __ldcg(p.part_ml + part * rows_cap + prow).x;
              if (pm == -INFINITY) continue;
              const float w = mx == INFINITY ? 1.0f : ex2(pm - mx);
              const float4* po = reinterpret_cast<const float4*>(p.partials) + part * rows_cap * (DP / 4);
              const float4 a = __ldcg(po + (int64_t)(i / 4) * rows_cap + prow);
              const float4 b = __ldcg(po + (int64_t)(i / 4 + 1) * rows_cap + prow);
              o[0] += w * a.x;
              o[1] += w * a.y;
              o[2] += w * a.z;
              o[3] += w * a.w;
              o[4] += w * b.x;
              o[5] += w * b.y;
              o[6] += w * b.z;
              o[7] += w * b.w;
            }
            *reinterpret_cast<uint4*>(p.out + out_at + i) =
                make_uint4(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv),
                           pack_bf16(o[4] * inv, o[5] * inv), pack_bf16(o[6] * inv, o[7] * inv));
          }
        }
        if (last && tid == 0) p.counters[c_first] = 0u;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 8) {
      // ---------------- loads ----------------
      uint32_t seq = 0, sent = 0, q_sent = 0;
      int seg = 0;
      const int pages = PAGED ? kBlock / p.page_size : 1;
      const uint32_t box = (PAGED ? p.page_size : kBlock) * 128;
      for (; walk.next(p, s); ++seg) {
        if (wait_all(q_free, (seg & 1) ^ 1, s_abort, p.status)) {
          const int slots = s.tile.pair ? 2 : 1;
          const uint32_t rows_bytes = (uint32_t)p.slot_tokens * p.group * 128;
          ++q_sent;
          if (lane == 0) mbar_arrive_expect_tx(q_full, rows_bytes * NH * slots);
          __syncwarp();
          if (lane < slots * NH) {
            const int t = lane / NH, half = lane % NH;
            tma_load_4d(smem + C::OFF_Q + t * C::TILE + half * kBlock * 128, &qmap, half * 64, 0, s.h,
                        (int)s.q.r0 + s.tile.t0 + t * p.slot_tokens, q_full);
          }
        }
        const int k0 = s.tile.pair ? s.j0 : 2 * s.j0;
        const int n = (s.tile.pair ? s.j1 : min(2 * s.j1, s.tile.blocks)) - k0;
        for (int at = 0; at < 2 * n; ++at, ++seq) {
          int c;
          const bool is_v = nth_load(s.tile.pair, at, n, c);
          const int st = seq % C::STAGES;
          const int key0 = (k0 + c) * kBlock;
          const int pg = lane % pages, half = lane / pages;
          bool mine = lane < pages * NH;
          int page = 0;
          if (PAGED) {
            const int col = (k0 + c) * pages + pg;
            mine = mine && key0 + pg * p.page_size < s.q.keys;
            if (mine) page = p.table[s.b * p.table_ld + col];
          }
          if (!wait_all(&empty[st], ((seq / C::STAGES) & 1) ^ 1, s_abort, p.status)) continue;
          sent = seq + 1;
          const unsigned who = __ballot_sync(0xffffffffu, mine);
          if (lane == 0) mbar_arrive_expect_tx(&full[st], box * __popc(who));
          __syncwarp();
          if (mine) {
            uint8_t* dst = smem + C::OFF_KV + st * C::TILE + half * kBlock * 128 + (PAGED ? pg * box : 0);
            if (PAGED)
              tma_load_3d(dst, is_v ? &vmap : &kmap, half * 64, s.h * p.page_size, page, &full[st]);
            else
              tma_load_3d(dst, is_v ? &vmap : &kmap, half * 64, s.h, (int)s.q.r0 + key0, &full[st]);
          }
        }
      }
      // No copy may be in flight when the CTA exits: without an abort the products have
      // waited for every one.
      if (*s_abort && lane == 0) {
        if (q_sent) drain(q_full, (q_sent - 1) & 1);
        for (uint32_t x = sent > C::STAGES ? sent - C::STAGES : 0; x < sent; ++x)
          drain(&full[x % C::STAGES], (x / C::STAGES) & 1);
      }
      __syncwarp();
    } else if (warp == 9) {
      // ---------------- products ----------------
      if (lane == 0) {
        const uint32_t idesc_s = umma_idesc_bf16(kBlock, kBlock);
        const uint32_t idesc_o = umma_idesc_bf16(kBlock, ksteps * 16) | (1u << 16);  // B is contiguous along N
        uint32_t base = 0, fixed = 0;  // loads so far; phase of each stage's check
        uint32_t n_p[2] = {0, 0}, n_seg[2] = {0, 0};
        int seg = 0;
        const uint32_t q_addr = smem_u32(smem + C::OFF_Q), kv_addr = smem_u32(smem + C::OFF_KV);
        auto wait_load = [&](uint32_t at) {
          return wait_one(&full[at % C::STAGES], (at / C::STAGES) & 1, s_abort, p.status);
        };
        for (; walk.next(p, s); ++seg) {
          const bool pair = s.tile.pair;
          const int k0 = pair ? s.j0 : 2 * s.j0;
          const int n = (pair ? s.j1 : min(2 * s.j1, s.tile.blocks)) - k0;
          int cnt[2];  // blocks of each slot
          if (pair) {
            const int64_t seen = s.q.ctx + s.tile.t0 + p.slot_tokens;
            const int keys0 = (int)(seen < s.q.keys ? seen : s.q.keys);
            const int blocks0 = keys0 <= 0 ? 0 : (keys0 + kBlock - 1) / kBlock;
            cnt[0] = max(0, min(s.j1, blocks0) - s.j0);
            cnt[1] = n;
          } else {
            cnt[0] = (n + 1) >> 1;
            cnt[1] = n >> 1;
          }
          const int64_t t0_sees = s.q.ctx + s.tile.t0 + 1;
          const int64_t all_see = t0_sees < s.q.keys ? t0_sees : s.q.keys;  // keys that every row sees
          auto block_of = [&](int t, int x) { return pair ? x : 2 * x + t; };
          auto scores = [&](int t, int x) {
            const int c = block_of(t, x);
            const uint32_t at = base + order_k(pair, c);
            if (!wait_load(at)) return;
            tc_fence_after();
            const uint32_t k = kv_addr + (at % C::STAGES) * C::TILE, q = q_addr + (pair ? t : 0) * C::TILE;
            for (int i = 0; i < ksteps; ++i) {
              const uint32_t off = (i >> 2) * kBlock * 128 + (i & 3) * 32;
              umma_ss(tmem + t * kBlock, umma_desc_sw128(q + off), umma_desc_sw128(k + off), idesc_s, i > 0);
            }
            umma_commit(&s_full[t]);
            if (!pair || t == 1) umma_commit(&empty[at % C::STAGES]);
          };
          bool ok = wait_one(q_full, seg & 1, s_abort, p.status);
          for (int t = 0; t < 2; ++t)
            if (ok && cnt[t] > 0) scores(t, 0);
          uint32_t was_checked = 0;  // pair: slot 0 has waited for this stage's check
          for (int x = 0; x < max(cnt[0], cnt[1]); ++x) {
            for (int t = 0; t < 2; ++t) {
              if (x >= cnt[t]) continue;
              const int c = block_of(t, x);
              const uint32_t at = base + order_v(pair, c, n), st = at % C::STAGES;
              if (x == 0) wait_one(&o_free[t], (n_seg[t] & 1) ^ 1, s_abort, p.status);
              wait_load(at);
              if ((int64_t)(k0 + c + 1) * kBlock > all_see && !(pair && t == 1 && (was_checked >> st & 1))) {
                wait_one(&checked[st], fixed >> st & 1, s_abort, p.status);
                fixed ^= 1u << st;
                was_checked |= 1u << st;
              }
              wait_one(&p_full[t], n_p[t] & 1, s_abort, p.status);
              ++n_p[t];
              if (*s_abort) continue;
              tc_fence_after();
              const uint32_t v = kv_addr + st * C::TILE;
              for (int i = 0; i < kBlock / 16; ++i)
                umma_ts(tmem + C::COL_O + t * DP, tmem + t * kBlock + i * 8, desc_v(v + i * 2048), idesc_o, x > 0 || i > 0);
              if (!pair || t == 1) {
                umma_commit(&empty[st]);
                was_checked &= ~(1u << st);
              }
              if (x + 1 < cnt[t]) scores(t, x + 1);
              else umma_commit(&o_full[t]);
            }
          }
          // Q is free once the last scores are done; later commits only come after them.
          umma_commit(q_free);
          for (int t = 0; t < 2; ++t)
            if (cnt[t] > 0) ++n_seg[t];
          base += 2 * n;
        }
        if (*s_abort) {  // the products in flight end before TMEM is freed
          umma_commit(drained);
          drain(drained, 0);
        }
      }
      __syncwarp();
    } else if (warp >= 10) {
      // ---------------- V blocks that not every row sees whole ----------------
      const int w = warp - 10;
      uint32_t base = 0;
      int seg = 0;
      for (; walk.next(p, s); ++seg) {
        const bool pair = s.tile.pair;
        const int k0 = pair ? s.j0 : 2 * s.j0;
        const int n = (pair ? s.j1 : min(2 * s.j1, s.tile.blocks)) - k0;
        const int64_t t0_sees = s.q.ctx + s.tile.t0 + 1;
        const int64_t all_see = t0_sees < s.q.keys ? t0_sees : s.q.keys;
        const int par = seg & 1;
        bool first = true;
        for (int x = 0; x < 2 * n; ++x) {
          int c;
          const bool is_v = nth_load(pair, x, n, c);
          const int key0 = (k0 + c) * kBlock;
          const uint32_t at = base + x, st = at % C::STAGES;
          // every load is followed, so that no phase of its barrier is taken for another
          const bool landed = wait_all(&full[st], (at / C::STAGES) & 1, s_abort, p.status);
          if (!is_v || (int64_t)key0 + kBlock <= all_see) {
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
              const bool live = key0 + r < s.q.keys;
              bool broken = false;
              for (int x = 0; x < NH * 8; ++x) {
                uint4* at16 = reinterpret_cast<uint4*>(v + (x >> 3) * kBlock * 128 + r * 128 + (((x & 7) ^ (r & 7)) << 4));
                if (!live) {
                  *at16 = make_uint4(0, 0, 0, 0);
                  continue;
                }
                uint4 u = *at16;
                uint32_t* e = reinterpret_cast<uint32_t*>(&u);
                bool hit = false;
  #pragma unroll
                for (int y = 0; y < 4; ++y) {
                  if ((e[y] & 0x7f80u) == 0x7f80u) { e[y] &= 0xffff0000u; hit = true; }
                  if ((e[y] & 0x7f800000u) == 0x7f800000u) { e[y] &= 0xffffu; hit = true; }
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
