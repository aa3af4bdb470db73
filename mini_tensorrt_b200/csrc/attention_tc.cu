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
// Roundings: the weights to bf16 (their sum is that of the unrounded ones). f32 rows of q are two
// bf16 planes of 16 bits together (attention.cu, store_q) and S the sum of both products, the
// smaller first: half as many products again, which cost prompts of 1024 + 700 + 333 + 1019 tokens, 12
// heads of 64, 49 us in place of 46, and, as two planes of 128 dimensions leave room for one
// tile's Q only, 8192 tokens of 32 heads over 8 of 128 928 in place of 698. One plane left errors
// 1.7 times those of fp32 arithmetic (2.8e-3 against 1.6e-3 of the result) at scores of a few, and
// as many times more at larger ones. (A row or two of a request go to attention_f32.cu, which
// rounds neither.)
//
// Work: a step is one block for each slot. The steps of all tiles of all requests form
// one list, cut into equal runs over one CTA per SM; every CTA finds its own run from
// the lengths in device memory. A tile cut between CTAs leaves partial (m, l, O) in the
// workspace, and the CTA that finishes last joins them in order.
//
// Bound by a row's softmax chain (maximum, its exchange, exponentials), not by the products or the
// memory: on a B200 a prompt of 8192 tokens, 32 heads over 8 of 128 dimensions, takes 580 to 670 us
// with the clock, some 5,000 clocks a step of two blocks, of which the products are 2,048
// (tensor pipe 41 % of cycles); 64 requests of 100 to 8192 tokens decoding with the same heads
// 160 us, 3.8 TB/s of keys and values.
//
// One CTA = 20 warps: 0..7 and 8..15 the slots' softmax (two threads per row, of 64 keys
// each, also the epilogue), 16 TMA loads, 17 and 18 issue the slots' products, 19 looks over
// the V blocks that not every row sees whole: rows past the request's keys are zeroed (a
// page's unused rows, the next request's rows: 0 * NaN would reach O), and infinities and NaN
// in rows that only later tokens see are taken out and listed; the epilogue adds them to the
// rows that see them.
#include <math.h>

#include <type_traits>

#include "../../include/mtrtq.h"
#include "attention_mma.cuh"

namespace mtrtq {

namespace {

constexpr int kThreads = 640;
constexpr int kLoadWarp = 16;  // after the softmax warps
constexpr int kBadMax = 384;  // listed V rows of a tile: three blocks

constexpr int kRing = 4;  // segments that the roles may lie apart

// PLANES: of Q. Two of 128 dimensions leave shared memory for one tile's, so that the slots
// always have the same rows and the next tile's Q is not loaded ahead.
template <int DP, int PLANES>
struct Cfg {
  static constexpr int TILE = kBlock * DP * 2;  // Q, K or V block in shared memory
  static constexpr int STAGES = DP == 128 ? 4 : 8;
  static constexpr int Q_BUFFERS = DP == 128 && PLANES == 2 ? 1 : 2;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_KV = Q_BUFFERS * PLANES * TILE;
  static constexpr int OFF_LIST = OFF_KV + STAGES * TILE;
  static constexpr int OFF_SEG = OFF_LIST + MTRTQ_MAX_BATCH * sizeof(Request);
  static constexpr int OFF_ML = OFF_SEG + kRing * ((sizeof(Segment) + 15) / 16 * 16);  // slot 1's (m, l)
  static constexpr int OFF_TOP = OFF_ML + kBlock * 8;  // [2 phases][2 slots][2 halves][rows]
  static constexpr int OFF_BAD = OFF_TOP + 8 * kBlock * 4;                                  // [kRing][kBadMax] keys
  static constexpr int OFF_BAR = OFF_BAD + kRing * kBadMax * 4;
  static constexpr int NBAR = 3 * STAGES + 2 * kRing + 22;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = OFF_MISC + 128 + 1024;
  static constexpr int COL_O = 256;
  static_assert(BYTES <= 227 * 1024, "shared memory per CTA");
};

// 16 bf16 of a row, or 8 if only 8 are left: 32 bytes at a time where the rows allow it, as
// every row is a line of its own.
__device__ __forceinline__ void store_row(__nv_bfloat16* out, const uint32_t* u, int left, bool by32) {
  if (by32 && left >= 16) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), "r"(u[0]), "r"(u[1]), "r"(u[2]),
                 "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                 : "memory");
    return;
  }
  *reinterpret_cast<uint4*>(out) = make_uint4(u[0], u[1], u[2], u[3]);
  if (left > 8) *reinterpret_cast<uint4*>(out + 8) = make_uint4(u[4], u[5], u[6], u[7]);
}
// O's rows of this warp times keep.
template <int DP>
__device__ __forceinline__ void rescale(uint32_t o_addr, float keep) {
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

// Dimensions d0 .. d1 - 1 of one row of a cut tile from the parts of CTAs c_first .. c_last, in order.
template <int DP>
__device__ __forceinline__ void join_parts(const TcAttention& p, int c_first, int c_last, int prow, int d0, int d1,
                                           __nv_bfloat16* out) {
  const int64_t rows = p.part_rows;
  float top = -INFINITY;
#pragma unroll 1
  for (int c = c_first; c <= c_last; ++c)
    top = fmaxf(top, __ldcg(p.part_ml + (c * 2 + (c == c_first)) * rows + prow).x);
  float sum = 0.0f;
#pragma unroll 1
  for (int c = c_first; c <= c_last; ++c) {
    const float2 ml = __ldcg(p.part_ml + (c * 2 + (c == c_first)) * rows + prow);
    if (ml.x != -INFINITY) sum += ml.y * (top == INFINITY ? 1.0f : ex2(ml.x - top));
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll 1
  for (int i = d0; i < d1; i += 8) {
    float o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
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

// After a bounded wait gives up, every role's next wait fails at once and it leaves its
// loop for the barrier at the end; there is no other barrier without a limit.
template <int DP, bool PAGED, int PLANES>
__global__ void __launch_bounds__(kThreads, 1)
    attention_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap, const __grid_constant__ TcAttention p) {
  using C = Cfg<DP, PLANES>;
  constexpr int NH = DP / 64;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  // the prefix lies where K and V will
  const StepList list = {reinterpret_cast<Request*>(smem + C::OFF_LIST), reinterpret_cast<int64_t*>(smem + C::OFF_KV)};
  float* tops = reinterpret_cast<float*>(smem + C::OFF_TOP);
  float2* ml1 = reinterpret_cast<float2*>(smem + C::OFF_ML);
  int* bad = reinterpret_cast<int*>(smem + C::OFF_BAD);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* empty = full + C::STAGES;
  uint64_t* checked = empty + C::STAGES;
  uint64_t* q_full = checked + C::STAGES;  // [2], a barrier for each slot or buffer
  uint64_t* q_free = q_full + 2;
  uint64_t* s_full = q_free + 2;
  uint64_t* p_half = s_full + 2;           // the weights of the block's first 64 keys, and O rescaled
  uint64_t* p_full = p_half + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* o_free = o_full + 2;
  uint64_t* turn = o_free + 2;
  uint64_t* ml_full = turn + 2;
  uint64_t* ml_free = ml_full + 1;
  uint64_t* cut_in = ml_free + 1;   // a cut tile's part is stored
  uint64_t* cut_out = cut_in + 1;   // its ticket is here
  uint64_t* drained = cut_out + 1;
  uint64_t* seg_full = drained + 2;  // [kRing]
  uint64_t* seg_free = seg_full + kRing;
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* s_abort = reinterpret_cast<volatile int*>(misc + 1);
  volatile unsigned* s_ticket = misc + 2;
  volatile int* bad_count = reinterpret_cast<volatile int*>(misc + 4);  // [kRing]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Segment* segments = reinterpret_cast<Segment*>(smem + C::OFF_SEG);

  if (nothing_here<kThreads>(p)) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (the stream goes on when this kernel ends)
    return;
  }

  if (tid == 0) {
    for (int x = 0; x < C::STAGES; ++x) {
      mbar_init(&full[x], 1);
      mbar_init(&empty[x], 3);  // each slot's products, the check
      mbar_init(&checked[x], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_free[t], 2);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_half[t], 8);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_free[t], 8);
      mbar_init(&turn[t], 1);
    }
    mbar_init(&drained[0], 1);
    mbar_init(&drained[1], 1);
    mbar_init(ml_full, 4);
    mbar_init(ml_free, 8);
    mbar_init(cut_in, 16);
    for (int x = 0; x < 8; ++x) misc[8 + x] = 0;
    mbar_init(cut_out, 1);
    for (int r = 0; r < kRing; ++r) {
      mbar_init(&seg_full[r], 1);
      mbar_init(&seg_free[r], kLoadWarp + 3);  // all but the load warp
      bad_count[r] = 0;
    }
    *s_abort = 0;
    fence_barrier_init();
  }
  if (warp == kLoadWarp + 1) {
    tmem_alloc(misc, 512);
    tmem_relinquish();
  }
  if (warp == kLoadWarp && lane == 0) {
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  tc_fence_before();
  Walk walk;  // the load warp makes the segments
  make_list<kBlock, kThreads>(p, list, walk, reinterpret_cast<Walk*>(smem + C::OFF_SEG));
  tc_fence_after();
  const uint32_t tmem = misc[0];
  // The kernel that stored the new keys and cast the rows is complete from here on.
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int ksteps = (p.head_dim + 15) / 16;

  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_one(bar, parity, s_abort, p.status); };
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return wait_all(bar, parity, s_abort, p.status); };
  // The ring's next segment; false at the end of the run (a segment without blocks).
  auto next = [&](int seg) {
    return warp_wait(&seg_full[seg % kRing], (seg / kRing) & 1) && segments[seg % kRing].n > 0;
  };
  auto leave = [&](int seg) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&seg_free[seg % kRing]);
  };

  // 512 threads of 104 registers and 128 of 64: the 640 x 96 of the launch.
  if (warp < kLoadWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ---------------- softmax and epilogue ----------------
    const int t = warp >> 3, half = (warp >> 2) & 1;   // slot; which 64 keys, and half of the dimensions
    const int row = (warp & 3) * 32 + lane;            // of the slot's tile
    const uint32_t quad = (uint32_t)(warp & 3) << 21;  // lanes 32 (warp & 3) .. of TMEM
    const uint32_t s_addr = tmem + quad + t * kBlock + half * 64;  // scores
    const uint32_t p_addr = tmem + quad + t * kBlock + half * 32;  // weights, two keys a column
    const uint32_t o_addr = tmem + quad + C::COL_O + t * DP;
    const int d0 = half * (DP / 2), d1 = min(p.head_dim, d0 + DP / 2);
    volatile int* const pair_failed = reinterpret_cast<volatile int*>(misc + 8) + t * 4 + (warp & 3);
    float* const mine_top = tops + (t * 2 + half) * kBlock + row;
    const float* const other_top = tops + (t * 2 + (half ^ 1)) * kBlock + row;
    const int token = row / p.group, head = row - token * p.group;
    const float c2 = p.scale * 1.4426950408889634f;  // scale log2 e
    const float2 cc = make_float2(c2, c2);
    uint32_t n_s = 0, n_o = 0, n_x = 0;
    // Gives this half's value of the row to the other half's thread, and gets its; false
    // if either warp's last wait gave up (so both leave together: this barrier has no limit,
    // but neither warp can fail to reach it).
    auto swap = [&](bool fine, float x, float& y) {
      const uint32_t at = (n_x++ & 1) * 4 * kBlock;
      mine_top[at] = x;
      if (!fine) *pair_failed = 1;
      named_bar_sync(1 + t * 4 + (warp & 3), 64);
      y = other_top[at];
      return *pair_failed == 0;
    };
    uint32_t n_ml = 0, n_cut = 0;
    bool ok = true;
#pragma unroll 1
    for (int seg = 0; ok && next(seg); leave(seg), ++seg) {
      const Segment& s = segments[seg % kRing];
      const bool pair = s.pair;
      const int tok = (pair ? t * p.slot_tokens : 0) + token;  // of the tile's
      const bool live = token < p.slot_tokens && tok < s.tokens;
      const int keys = live ? max(0, min(s.see0 + tok, s.keys)) : 0;  // that this row sees
      const bool warp_live = __any_sync(0xffffffffu, live);
      const int cnt = s.cnt[t], stride = pair ? kBlock : 2 * kBlock;
      // Of these 64 columns it sees so many; rows that are no tokens' are left unmasked, so
      // that they do not put their warp on the masked path block after block.
      int left = (live ? keys : 0x40000000) - (s.k0 + (pair ? 0 : t)) * kBlock - half * 64;
      float m = -INFINITY, l = 0.0f;
#pragma unroll 1
      for (int x = 0; x < cnt; ++x, left -= stride, ++n_s) {
        ok = warp_wait(&s_full[t], n_s & 1);
        if (!warp_live) {
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive(&p_half[t]);
            if (half) mbar_arrive(&p_full[t]);
          }
          continue;
        }
        tc_fence_after();
        float v[64];
        tmem_ld32(s_addr, v);
        tmem_ld32(s_addr + 32, v + 32);
        tmem_wait_ld();
        if (__any_sync(0xffffffffu, left < 64)) {
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] = i < left ? v[i] : -INFINITY;
        }
        // The largest score (NaN ones aside: they make the sum NaN).
        float a[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int i = 4; i + 7 < 64; i += 8) {
#pragma unroll
          for (int y = 0; y < 4; ++y) a[y] = max3(a[y], v[i + 2 * y], v[i + 2 * y + 1]);
        }
        a[0] = max3(a[0], v[60], v[61]);
        a[1] = max3(a[1], v[62], v[63]);
        // The row's other half. Past the swap both have read their scores, which the
        // weights overwrite.
        float top = max3(a[0], a[1], fmaxf(a[2], a[3])), other;
        ok = swap(ok, top, other);
        if (!ok) break;
        top = fmaxf(top, other) * c2;
        const bool grow = live && (top > m + 8.0f || (m == -INFINITY && top > m));
        if (__any_sync(0xffffffffu, grow)) {
          const float m1 = grow ? top : m;
          const float keep = m1 == -INFINITY ? 1.0f : ex2(m - m1);
          l *= keep;
          m = m1;
          if (x > 0) rescale<DP / 2>(o_addr + d0, keep);  // the earlier products are complete: these scores came after
        }
        if (half) {
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_half[t]);
        }
        const float base = m == -INFINITY ? 0.0f : -m;
        const float2 mm = make_float2(base, base);
        float2 sum = make_float2(0.0f, 0.0f), sum1 = sum;
#pragma unroll
        for (int i = 0; i < 64; i += 32) {
          uint32_t w[16];
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            float2 e = fma2(make_float2(v[i + 2 * y], v[i + 2 * y + 1]), cc, mm);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            if (y & 1) sum1 = __fadd2_rn(sum1, e);
            else sum = __fadd2_rn(sum, e);
            w[y] = pack_bf16(e.x, e.y);
          }
          tmem_st16(p_addr + (i >> 1), w);
        }
        sum = __fadd2_rn(sum, sum1);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(half ? &p_full[t] : &p_half[t]);
        l += sum.x + sum.y;
      }
      if (!ok) break;
      if (warp_live) {  // the row's sum: its first half's and its second's
        float other;
        swap(true, l, other);
        l = half ? other + l : l + other;
      }

      if (m == -INFINITY && l != l) m = 0.0f;  // every score it saw was NaN
      if (cnt > 0) {
        ok = warp_wait(&o_full[t], n_o & 1);
        ++n_o;
        if (!ok) break;
      }
      // halves: slot 0's threads join the two slots' rows
      const bool mine = pair || t == 0, two = !pair && s.n > 1, whole = s.whole;
      float w0 = 1.0f, w1 = 0.0f;
      if (two) {
        if (t == 1 && half == 0) {
          ok = warp_wait(ml_free, (n_ml & 1) ^ 1);
          ml1[row] = make_float2(m, l);
          __syncwarp();
          if (lane == 0) mbar_arrive(ml_full);
        } else if (t == 0) {
          ok = warp_wait(ml_full, n_ml & 1);  // slot 1's warps have waited for their products
          const float2 ml = ml1[row];
          __syncwarp();
          if (lane == 0) mbar_arrive(ml_free);
          const float top = fmaxf(m, ml.x);
          w0 = m == -INFINITY ? 0.0f : top == INFINITY ? 1.0f : ex2(m - top);
          w1 = ml.x == -INFINITY ? 0.0f : top == INFINITY ? 1.0f : ex2(ml.x - top);
          l = l * w0 + ml.y * w1;
          m = top;
        }
        ++n_ml;
        if (!ok) break;
      }
      tc_fence_after();
      if (m == -INFINITY) w0 = 0.0f;  // no key seen (and perhaps no product formed)
      const int prow = (pair ? t * kBlock : 0) + row;
      __nv_bfloat16* out = p.out + (int64_t)(s.row0 + tok) * p.out_row + (int64_t)(s.h * p.group + head) * p.out_head;
      const int64_t part = (int64_t)blockIdx.x * 2 + s.part;
      float* to_part = p.partials + (part * p.part_rows * (DP / 4) + prow) * 4;
      if (mine) {
        if (whole) {
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          w0 *= inv;
          w1 *= inv;
        }
#pragma unroll 1
        for (int i = d0; i < d1; i += 16) {
          uint32_t u[16];
          float o[16];
          if (cnt > 0) {
            tmem_ld_32x32b_x16(o_addr + i, u);
            tmem_wait_ld();
          }
#pragma unroll
          for (int y = 0; y < 16; ++y) o[y] = w0 == 0.0f ? 0.0f : __uint_as_float(u[y]) * w0;
          if (two) {
            tmem_ld_32x32b_x16(o_addr + DP + i, u);
            tmem_wait_ld();
#pragma unroll
            for (int y = 0; y < 16; ++y) o[y] += w1 == 0.0f ? 0.0f : __uint_as_float(u[y]) * w1;
          }
          if (!live) continue;
          if (whole) {
#pragma unroll
            for (int y = 0; y < 8; ++y) u[y] = pack_bf16(o[2 * y], o[2 * y + 1]);
            store_row(out + i, u, d1 - i, p.out32);
          } else {
#pragma unroll
            for (int y = 0; y < 16; y += 4)
              __stcg(reinterpret_cast<float4*>(to_part + (int64_t)(i + y) * p.part_rows),
                     make_float4(o[y], o[y + 1], o[y + 2], o[y + 3]));
          }
        }
        if (live && half == 0 && !whole) __stcg(p.part_ml + part * p.part_rows + prow, make_float2(m, l));
        // The infinities and NaN that were taken out of the last blocks' V, for the rows
        // that see them. A slot without such blocks has not waited for the check (and sees
        // none of it): with a token a slot that is slot 0's case even where it has others.
        if (cnt > 0 && (s.k0 + (pair ? cnt : s.n)) * kBlock > s.all_see()) {
          const int have = min(kBadMax, bad_count[seg % kRing]);
#pragma unroll 1
          for (int x = 0; x < have; ++x) {
            const int key = bad[seg % kRing * kBadMax + x];
            if ((unsigned)key >= (unsigned)keys) continue;
            const __nv_bfloat16* src;
            if (PAGED) {
              const int64_t page = p.table[s.b * p.table_ld + key / p.page_size];
              src = p.v + page * p.v_row + ((int64_t)s.h * p.page_size + key % p.page_size) * p.head_dim;
            } else {
              src = p.v + (int64_t)(s.r0 + key) * p.v_row + s.h * p.v_head;
            }
#pragma unroll 1
            for (int d = d0; d < d1; ++d) {
              const float z = __bfloat162float(src[d]);
              if (fabsf(z) < INFINITY) continue;
              if (whole) {
                out[d] = __float2bfloat16_rn(__bfloat162float(out[d]) + z);
              } else {
                float* to = to_part + (int64_t)(d & ~3) * p.part_rows + (d & 3);
                __stcg(to, __ldcg(to) + z);
              }
            }
          }
        }
        // O has been read.
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (cnt > 0) mbar_arrive(&o_free[t]);
          if (two) mbar_arrive(&o_free[1]);
        }
      }
      if (!whole) {
        __syncwarp();
        if (lane == 0) mbar_arrive(cut_in);
        if (tid == 0) {
          wait(cut_in, n_cut & 1);
          *s_ticket = ticket_acq_rel(p.counters + s.c_first);
          mbar_arrive(cut_out);
        }
        __syncwarp();
        if (mine) {
          ok = warp_wait(cut_out, n_cut & 1);
          const bool last = *s_ticket == (unsigned)(s.c_last - s.c_first);
          if (ok && last && live) join_parts<DP>(p, s.c_first, s.c_last, prow, d0, d1, out);
          if (last && tid == 0) p.counters[s.c_first] = 0u;
        }
        ++n_cut;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == kLoadWarp) {
      // ---------------- loads ----------------
      uint32_t seq = 0;
      int q_sent[2] = {0, 0};
      const int pages = PAGED ? kBlock / p.page_size : 1;
      const uint32_t box = (PAGED ? p.page_size : kBlock) * 128;
      const uint32_t rows_bytes = (uint32_t)p.slot_tokens * p.group * 128 * NH * PLANES;
      bool ok = true;
#pragma unroll 1
      for (int seg = 0; ok; ++seg) {
        Segment& s = segments[seg % kRing];
        ok = warp_wait(&seg_free[seg % kRing], ((seg / kRing) & 1) ^ 1);
        if (!ok) break;
        if (lane == 0 && !next_segment<kBlock>(p, list, walk, s)) s.n = 0;
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_full[seg % kRing]);
        const int k0 = s.k0, n = s.n;
        if (n == 0) break;
        const bool pair = s.pair;
        // Page numbers of 64 columns, two in each lane, read well before they are used: a
        // read of the table on each copy's way cost more than the copy.
        const int columns = PAGED ? (s.keys + p.page_size - 1) / p.page_size : 0;
        auto column = [&](int col) { return col < columns ? p.table[s.b * p.table_ld + col] : 0; };
        int window = PAGED ? k0 * pages : 0, ahead[2];
        if (PAGED) {
          ahead[0] = column(window + lane);
          ahead[1] = column(window + 32 + lane);
        }
#pragma unroll 1
        for (int t = 0; ok && t < (pair ? 2 : 1); ++t) {
          const int buf = pair ? t : s.buf;
          ok = warp_wait(&q_free[buf], (s.q_use[buf] & 1) ^ 1);
          if (!ok) break;
          ++q_sent[buf];
          if (lane == 0) mbar_arrive_expect_tx(&q_full[buf], rows_bytes);
          __syncwarp();
          if (lane < NH * PLANES)
            tma_load_4d(smem + C::OFF_Q + (buf * PLANES * NH + lane) * kBlock * 128, &qmap, lane % NH * 64, 0, s.h,
                        lane / NH * (int)p.rows + s.row0 + t * p.slot_tokens, &q_full[buf]);
        }
#pragma unroll 1
        for (int at = 0; ok && at < 2 * n; ++at) {
          int c;
          const bool is_v = nth_load(pair, at, n, c);
          const int st = seq % C::STAGES;
          const int key0 = (k0 + c) * kBlock;
          const int pg = lane % pages, half = lane / pages;
          bool load = lane < pages * NH;
          int page = 0;
          if (PAGED) {
            load = load && key0 + pg * p.page_size < s.keys;
            const int col = (k0 + c) * pages;
            if (is_v && col >= window + 32) {  // every earlier column is done with
              window += 32;
              ahead[0] = ahead[1];
              ahead[1] = column(window + 32 + lane);
            }
            const int want = (col + pg - window) & 63;
            const int lo = __shfl_sync(0xffffffffu, ahead[0], want & 31), hi = __shfl_sync(0xffffffffu, ahead[1], want & 31);
            page = want < 32 ? lo : hi;
          }
          ok = warp_wait(&empty[st], ((seq / C::STAGES) & 1) ^ 1);
          if (!ok) break;
          ++seq;
          const unsigned who = __ballot_sync(0xffffffffu, load);
          if (lane == 0) mbar_arrive_expect_tx(&full[st], box * __popc(who));
          __syncwarp();
          if (load) {
            uint8_t* dst = smem + C::OFF_KV + st * C::TILE + half * kBlock * 128 + (PAGED ? pg * box : 0);
            if (PAGED)
              tma_load_3d(dst, is_v ? &vmap : &kmap, half * 64, s.h * p.page_size, page, &full[st]);
            else
              tma_load_3d(dst, is_v ? &vmap : &kmap, half * 64, s.h, s.r0 + key0, &full[st]);
          }
        }
      }
      // No copy may be in flight when the CTA exits: without an abort the products have
      // waited for every one.
      if (*s_abort && lane == 0) {
        for (int t = 0; t < 2; ++t)
          if (q_sent[t]) drain(&q_full[t], (q_sent[t] - 1) & 1);
        for (uint32_t x = seq > C::STAGES ? seq - C::STAGES : 0; x < seq; ++x)
          drain(&full[x % C::STAGES], (x / C::STAGES) & 1);
      }
      __syncwarp();
    } else if (warp < kLoadWarp + 3) {
      // ---------------- products: a warp for each slot ----------------
      // It follows every load in order (so that no phase of a barrier is taken for another)
      // and lets go at once of those that its slot does not use. A turn is one block's PV and
      // the next one's scores, with nothing but the products between them: whatever else
      // they need is waited for before. Slot 0 has the first turn; a slot with fewer blocks
      // passes its turns on. (Without turns the slots fall into step, and the tensor cores
      // wait for both.)
      const int t = warp - kLoadWarp - 1;
      const uint32_t idesc_s = umma_idesc_bf16(kBlock, kBlock);
      const uint32_t idesc_o = umma_idesc_bf16(kBlock, ksteps * 16) | (1u << 16);  // B is contiguous along N
      const uint32_t q_desc = desc_qk(smem_u32(smem + C::OFF_Q)), k_desc = desc_qk(smem_u32(smem + C::OFF_KV)),
                     v_desc = desc_v(smem_u32(smem + C::OFF_KV));
      const uint32_t s_col = tmem + t * kBlock, o_col = tmem + C::COL_O + t * DP;
      uint32_t seq = 0, fixed = 0;  // loads so far; phase of each stage's check
      uint32_t n_p = 0, n_o = 0, n_turn = 0;
      auto take_turn = [&]() { return wait(&turn[t], (n_turn++ & 1) ^ (t ^ 1)); };
      auto end_turn = [&]() { mbar_arrive(&turn[t ^ 1]); };
      auto landed = [&]() { return wait(&full[seq % C::STAGES], (seq / C::STAGES) & 1); };
      // The scores of a block, q's smaller plane first; the other slot may go on shortly
      // before the end.
      auto scores = [&](uint32_t q, uint32_t k) {
#pragma unroll
        for (int plane = PLANES - 1; plane >= 0; --plane) {
#pragma unroll
          for (int i = 0; i < DP / 16; ++i) {
            if (plane == 0 && i == DP / 32) end_turn();
            if (i < ksteps)
              mma_ss(s_col, q + plane * (C::TILE >> 4) + (i >> 2) * (kBlock * 128 >> 4) + (i & 3) * 2,
                     k + (i >> 2) * (kBlock * 128 >> 4) + (i & 3) * 2, idesc_s, plane < PLANES - 1 || i > 0);
          }
        }
        umma_commit(&s_full[t]);
      };
#pragma unroll 1
      for (int seg = 0; next(seg); leave(seg), ++seg) {
        if (lane == 0) {
          const Segment& s = segments[seg % kRing];
          const bool pair = s.pair;
          const uint32_t turns = n_turn + max(s.cnt[0], s.cnt[1]) + 1, end = seq + 2 * s.n;
          const int n = s.n, cnt = s.cnt[t], buf = pair ? t : s.buf;
          const int checked_from = max(0, s.all_see() / kBlock - s.k0);  // blocks from there on
          bool ok = true;
          if (pair) {
            ok = wait(&q_full[t ^ 1], s.q_use[t ^ 1] & 1);
            mbar_arrive(&q_free[t ^ 1]);
          }
          ok = ok && wait(&q_full[buf], s.q_use[buf] & 1);
          if (cnt == 0) mbar_arrive(&q_free[buf]);
          const uint32_t q = q_desc + buf * (PLANES * C::TILE >> 4), first = seq;
          // Passes over the loads of the other slot's blocks before `to`.
          auto skip = [&](uint32_t to) {
#pragma unroll 1
            for (; ok && seq < to; ++seq) {
              int c;
              const bool is_v = nth_load(pair, seq - first, n, c);
              ok = landed();
              if (is_v && c >= checked_from) fixed ^= 1u << (seq % C::STAGES);
              if (ok) mbar_arrive(&empty[seq % C::STAGES]);
            }
          };
          if (cnt > 0) {
            skip(first + (pair ? 0 : t));
            ok = ok && landed() && take_turn();
            if (ok) {
              tc_fence_after();
              scores(q, k_desc + seq % C::STAGES * (C::TILE >> 4));
              umma_commit(&empty[seq % C::STAGES]);
              if (cnt == 1) umma_commit(&q_free[buf]);
              ++seq;
            }
#pragma unroll 1
            for (int x = 0; ok && x < cnt; ++x) {
              const int c = pair ? x : 2 * x + t;
              skip(first + (pair ? 2 * c + 1 : min(2 * c + 2, 2 * n - 1)));
              ok = ok && landed();
              if (!ok) break;
              const uint32_t st_v = seq % C::STAGES, v = v_desc + st_v * (C::TILE >> 4);
              if (c >= checked_from) {
                ok = wait(&checked[st_v], fixed >> st_v & 1);
                fixed ^= 1u << st_v;
              }
              ++seq;
              const bool more = x + 1 < cnt;  // the next load is this slot's next K
              const uint32_t st_k = seq % C::STAGES, k = k_desc + st_k * (C::TILE >> 4);
              if (more) ok = ok && landed();
              if (x == 0) ok = ok && wait(&o_free[t], (n_o & 1) ^ 1);
              ok = ok && take_turn() && wait(&p_half[t], n_p & 1);
              if (!ok) break;
              tc_fence_after();
#pragma unroll
              for (int i = 0; i < 4; ++i) mma_ts(o_col, s_col + i * 8, v + i * (2048 >> 4), idesc_o, x > 0 || i > 0);
              ok = wait(&p_full[t], n_p & 1);
              if (!ok) break;
              tc_fence_after();
#pragma unroll
              for (int i = 4; i < 8; ++i) mma_ts(o_col, s_col + i * 8, v + i * (2048 >> 4), idesc_o, true);
              ++n_p;
              if (more) {
                scores(q, k);
                umma_commit(&empty[st_k]);
                if (x + 2 == cnt) umma_commit(&q_free[buf]);
                ++seq;
              } else {
                end_turn();
                umma_commit(&o_full[t]);
                ++n_o;
              }
              umma_commit(&empty[st_v]);
            }
          }
          skip(end);
#pragma unroll 1
          while (ok && n_turn < turns) {
            ok = take_turn();
            end_turn();
          }
        }
        __syncwarp();
      }
      if (lane == 0 && *s_abort) {  // the products in flight end before TMEM is freed
        umma_commit(&drained[t]);
        drain(&drained[t], 0);
      }
      __syncwarp();
    } else {
      // ---------------- V blocks that not every row sees whole ----------------
      uint32_t seq = 0;
      bool ok = true;
#pragma unroll 1
      for (int seg = 0; ok && next(seg); leave(seg), ++seg) {
        const Segment& s = segments[seg % kRing];
        const bool pair = s.pair;
        const int n = s.n, k0 = s.k0, keys = s.keys, slot = seg % kRing;
        const int checked_from = max(0, s.all_see() / kBlock - k0);
        if (lane == 0) bad_count[slot] = 0;
        __syncwarp();
#pragma unroll 1
        for (int at = 0; ok && at < 2 * n; ++at, ++seq) {
          int c;
          const bool is_v = nth_load(pair, at, n, c);
          const uint32_t st = seq % C::STAGES;
          ok = warp_wait(&full[st], (seq / C::STAGES) & 1);
          if (!ok) break;
          if (is_v && c >= checked_from) {
            uint8_t* v = smem + C::OFF_KV + st * C::TILE;
            const int key0 = (k0 + c) * kBlock;
#pragma unroll 1
            for (int r = lane; r < kBlock; r += 32) {
              const bool kept = key0 + r < keys;
              bool broken = false;
#pragma unroll
              for (int y = 0; y < NH * 8; ++y) {
                uint4* at16 =
                    reinterpret_cast<uint4*>(v + (y >> 3) * kBlock * 128 + r * 128 + (((y & 7) ^ (r & 7)) << 4));
                if (!kept) {
                  *at16 = make_uint4(0, 0, 0, 0);
                  continue;
                }
                const uint4 u = *at16;
                const uint32_t e[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int z = 0; z < 4; ++z)
                  broken |= (e[z] & 0x7f80u) == 0x7f80u || (e[z] & 0x7f800000u) == 0x7f800000u;
              }
              if (broken) {
#pragma unroll 1
                for (int y = 0; y < NH * 32; ++y) {
                  uint32_t* at4 = reinterpret_cast<uint32_t*>(v + (y >> 5) * kBlock * 128 + r * 128 +
                                                              ((((y >> 2) & 7) ^ (r & 7)) << 4) + (y & 3) * 4);
                  uint32_t e = *at4;
                  if ((e & 0x7f80u) == 0x7f80u) e &= 0xffff0000u;
                  if ((e & 0x7f800000u) == 0x7f800000u) e &= 0xffffu;
                  *at4 = e;
                }
              }
              const unsigned who = __ballot_sync(0xffffffffu, broken);
              if (who) {
                const int had = bad_count[slot];
                __syncwarp();
                const int to = had + __popc(who & ((1u << lane) - 1));
                if (broken && to < kBadMax) bad[slot * kBadMax + to] = key0 + r;
                __threadfence_block();  // slot 0 may read while slot 1's last blocks are looked over
                __syncwarp();
                if (lane == 0) bad_count[slot] = min(kBadMax, had + __popc(who));
                __syncwarp();
              }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&checked[st]);
          }
          if (lane == 0) mbar_arrive(&empty[st]);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kLoadWarp + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int DP, bool PAGED, int PLANES>
cudaError_t launch_one(const TcAttention& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, int grid,
                       bool pdl, cudaStream_t st) {
  auto kernel = attention_tc_kernel<DP, PAGED, PLANES>;
  if (cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kernel), Cfg<DP, PLANES>::BYTES)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<DP, PLANES>::BYTES;
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
  auto run = [&](auto planes) {
    constexpr int P = decltype(planes)::value;
    if (p.head_dim <= 64)
      return p.table ? launch_one<64, true, P>(p, q, k, v, grid, pdl, st) : launch_one<64, false, P>(p, q, k, v, grid, pdl, st);
    return p.table ? launch_one<128, true, P>(p, q, k, v, grid, pdl, st) : launch_one<128, false, P>(p, q, k, v, grid, pdl, st);
  };
  return p.planes ? run(std::integral_constant<int, 2>()) : run(std::integral_constant<int, 1>());
}

}  // namespace mtrtq
