// f32 attention of whole prompts on the tensor cores, up to 64 dimensions.
//
// An f32 number is the sum of three bf16 ones (8 bits each), x = x0 + x1 + x2, so a product
// of two is x0 y0 + (x0 y1 + x1 y0) + (x0 y2 + x1 y1 + x2 y0) and terms below 2^-24 of it: six
// bf16 products with fp32 accumulators, where the CUDA cores have one product per lane and
// clock (25 heads of 64, prompts of 3076 tokens on a B200: CUDA cores 302 us, 145 us here with the split).
// A first kernel splits q, k and v into planes; the weights are split where they are made.
//
// The tensor cores cut what their fp32 accumulator cannot hold (measured: toward zero, two
// bits below its last), so the smallest terms are added first, and no sum runs over more
// than one block of 128 keys: every block's P V is a new accumulator that the softmax threads
// add to the output in registers, rounded to nearest. Rescaling by the running maximum
// happens there too.
//
// Infinities and NaN do not survive the split (inf - inf). In q and k they become NaN, so that
// the rows that see them are NaN. In v they are left out (0 * NaN would reach rows that do
// not see them) and their rows flagged; a tile whose request has flags looks at v itself and
// adds them to the rows that do.
//
// Tiles, the list of steps and the joining of cut tiles are as in attention_tc.cu, with one
// tile of 128 rows (tokens times the group's heads) and its blocks at a time. One CTA = 12
// warps: 0..7 softmax (two threads per row, of 64 keys and 32 dimensions each), 8 loads, 9
// products. The scores have two buffers, so that the next block's are formed while this
// block's weights are: bound by the products, 24 + 48 of 128 x 128 (or 64) x 16 a block.
#include <math.h>

#include "../../include/mtrtq.h"
#include "attention_mma.cuh"

namespace mtrtq {

namespace {

constexpr int kThreads = 384;
constexpr int kRing = 4;
constexpr int kPlane = kBlock * 128;     // bytes of a tile's plane: 128 rows of 64 bf16
constexpr int kTile = 3 * kPlane;
constexpr int kStages = 3;
constexpr int kColP = 256, kColO = 448;  // TMEM: two score buffers, three planes of weights, P V

constexpr int kOffKV = kTile;
constexpr int kOffList = kOffKV + kStages * kTile;
constexpr int kOffSeg = kOffList + MTRTQ_MAX_BATCH * (int)sizeof(Request);
constexpr int kOffTop = kOffSeg + kRing * (((int)sizeof(Segment) + 15) / 16 * 16);  // [2][2][rows]
constexpr int kOffBar = kOffTop + 4 * kBlock * 4;
constexpr int kOffMisc = kOffBar + (2 * kStages + 2 * kRing + 12) * 8;
constexpr int kBytes = kOffMisc + 64 + 1024;
static_assert(kBytes <= 227 * 1024, "shared memory per CTA");

// The pairs of planes of a product, smallest terms first.
__host__ __device__ constexpr int plane_a(int i) { return i == 0 ? 2 : i == 1 ? 1 : i == 2 ? 0 : i == 3 ? 1 : 0; }
__host__ __device__ constexpr int plane_b(int i) { return i == 0 ? 0 : i == 1 ? 1 : i == 2 ? 2 : i == 3 ? 0 : i == 4 ? 1 : 0; }

// One block per kSplitRows rows: planes [3][rows][heads + 2 kv_heads][head_dim] of q, k and v.
// Bound by memory: 3076 rows of 25 heads of 64 take 26 us on a B200, 5.6 TB/s.
__global__ void __launch_bounds__(256) split_rows_kernel(const __grid_constant__ F32Attention p, int heads,
                                                         __nv_bfloat16* planes, int* flags) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int all = heads + 2 * p.kv_heads, quads = p.head_dim / 4, each = all * quads;
  const int64_t plane = p.rows * all * p.head_dim, r0 = (int64_t)blockIdx.x * kSplitRows;
  int odd = 0;  // of v
  for (int e = threadIdx.x; e < each; e += 256) {
    const int h = e / quads, d = (e - h * quads) * 4;
    const bool is_v = h >= heads + p.kv_heads;
    const float* src = (h < heads ? p.q + h * p.q_head : is_v ? p.v + (h - heads - p.kv_heads) * p.v_head
                                                              : p.k + (h - heads) * p.k_head) + d;
    const int64_t stride = h < heads ? p.q_row : is_v ? p.v_row : p.k_row;
    float4 u[kSplitRows];
#pragma unroll
    for (int r = 0; r < kSplitRows; ++r)
      if (r0 + r < p.rows) u[r] = *reinterpret_cast<const float4*>(src + (r0 + r) * stride);
#pragma unroll
    for (int r = 0; r < kSplitRows; ++r) {
      if (r0 + r >= p.rows) break;
      float x[4] = {u[r].x, u[r].y, u[r].z, u[r].w};
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        if (fabsf(x[y]) < INFINITY) continue;
        odd |= is_v;
        x[y] = is_v ? 0.0f : NAN;
      }
      __nv_bfloat16* dst = planes + ((r0 + r) * all + h) * p.head_dim + d;
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        float z[4];
#pragma unroll
        for (int y = 0; y < 4; ++y)  // (nothing rounds up to infinity)
          z[y] = i == 0 && fabsf(x[y]) > 3.3895314e38f ? copysignf(3.3895314e38f, x[y]) : x[y];
        const uint32_t lo = pack_bf16(z[0], z[1]), hi = pack_bf16(z[2], z[3]);
        *reinterpret_cast<uint2*>(dst + i * plane) = make_uint2(lo, hi);
        const float b[4] = {__uint_as_float(lo << 16), __uint_as_float(lo & 0xffff0000u), __uint_as_float(hi << 16),
                            __uint_as_float(hi & 0xffff0000u)};
#pragma unroll
        for (int y = 0; y < 4; ++y) x[y] = b[y] == b[y] ? x[y] - b[y] : 0.0f;
      }
    }
  }
  const int any = __syncthreads_or(odd);
  if (threadIdx.x == 0) flags[blockIdx.x] = any;
}

__global__ void __launch_bounds__(kThreads, 1)
    attention_f32_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                            const __grid_constant__ CUtensorMap vmap, const __grid_constant__ F32TcAttention p) {
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  // the prefix lies where K and V will
  const StepList list = {reinterpret_cast<Request*>(smem + kOffList), reinterpret_cast<int64_t*>(smem + kOffKV)};
  Segment* segments = reinterpret_cast<Segment*>(smem + kOffSeg);
  float* tops = reinterpret_cast<float*>(smem + kOffTop);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* empty = full + kStages;
  uint64_t* q_full = empty + kStages;
  uint64_t* q_free = q_full + 1;
  uint64_t* s_full = q_free + 1;  // [2]
  uint64_t* p_full = s_full + 2;  // a block's weights are written, the last P V has been read
  uint64_t* o_full = p_full + 1;  // a block's P V
  uint64_t* o_free = o_full + 1;  // the tile's last P V has been read
  uint64_t* cut_in = o_free + 1;
  uint64_t* cut_out = cut_in + 1;
  uint64_t* drained = cut_out + 1;
  uint64_t* seg_full = drained + 1;  // [kRing]
  uint64_t* seg_free = seg_full + kRing;
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + kOffMisc);
  volatile int* s_abort = reinterpret_cast<volatile int*>(misc + 1);
  volatile unsigned* s_ticket = misc + 2;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int x = 0; x < kStages; ++x) {
      mbar_init(&full[x], 1);
      mbar_init(&empty[x], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_free, 1);
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(p_full, 8);
    mbar_init(o_full, 1);
    mbar_init(o_free, 8);
    mbar_init(cut_in, 8);
    mbar_init(cut_out, 1);
    mbar_init(drained, 1);
    for (int r = 0; r < kRing; ++r) {
      mbar_init(&seg_full[r], 1);
      mbar_init(&seg_free[r], 9);  // softmax, products
    }
    *s_abort = 0;
    for (int x = 0; x < 4; ++x) misc[4 + x] = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(misc, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  Walk walk;  // the load warp makes the segments
  make_list<kBlock, kThreads>(p, list, walk, reinterpret_cast<Walk*>(smem + kOffSeg));
  tc_fence_after();
  const uint32_t tmem = misc[0];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the rows are split

  const int ksteps = (p.head_dim + 15) / 16;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_one(bar, parity, s_abort, p.status); };
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return wait_all(bar, parity, s_abort, p.status); };
  auto next = [&](int seg) {
    return warp_wait(&seg_full[seg % kRing], (seg / kRing) & 1) && segments[seg % kRing].n > 0;
  };
  auto leave = [&](int seg) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&seg_free[seg % kRing]);
  };

  if (warp < 8) {
    // ---------------- softmax, output ----------------
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t quad = tmem + ((uint32_t)(warp & 3) << 21);
    const int d0 = half * 32, d1 = min(p.head_dim, d0 + 32);
    volatile int* const pair_failed = reinterpret_cast<volatile int*>(misc + 4) + (warp & 3);
    float* const mine_top = tops + half * kBlock + row;
    const float* const other_top = tops + (half ^ 1) * kBlock + row;
    const int token = row / p.group, head = row - token * p.group;
    const float c2 = p.scale * 1.4426950408889634f;  // scale log2 e
    uint32_t n_s = 0, n_o = 0, n_x = 0, n_cut = 0;
    // As in attention_tc.cu: the row's other half, and whether both warps' waits were fine.
    auto swap = [&](bool fine, float x, float& y) {
      const uint32_t at = (n_x++ & 1) * 2 * kBlock;
      mine_top[at] = x;
      if (!fine) *pair_failed = 1;
      named_bar_sync(1 + (warp & 3), 64);
      y = other_top[at];
      return *pair_failed == 0;
    };
    bool ok = true;
#pragma unroll 1
    for (int seg = 0; ok && next(seg); leave(seg), ++seg) {
      const Segment& s = segments[seg % kRing];
      const bool live = token < p.tile_tokens && token < s.tokens;
      const int keys = live ? max(0, min(s.see0 + token, s.keys)) : 0x40000000;  // that this row sees
      const int n = s.n;
      int left = keys - s.k0 * kBlock - half * 64;  // of these 64 columns
      int flagged = 0;  // whether a row of the request up to this tile's has values left out of v
#pragma unroll 1
      for (int x = s.r0 / kSplitRows + lane; x <= (s.row0 + s.tokens - 1) / kSplitRows; x += 32) flagged |= p.flags[x];
      float m = -INFINITY, l = 0.0f, o[32];
#pragma unroll
      for (int y = 0; y < 32; ++y) o[y] = 0.0f;
      // Adds the last block's P V to the output.
      auto add_block = [&]() {
        if (!warp_wait(o_full, n_o++ & 1)) return false;
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < 32; i += 16) {
          uint32_t pv[16];
          tmem_ld_32x32b_x16(quad + kColO + d0 + i, pv);
          tmem_wait_ld();
#pragma unroll
          for (int y = 0; y < 16; ++y) o[i + y] += __uint_as_float(pv[y]);
        }
        return true;
      };
#pragma unroll 1
      for (int x = 0; x < n; ++x, left -= kBlock, ++n_s) {
        const uint32_t buf = n_s & 1;
        ok = warp_wait(&s_full[buf], (n_s >> 1) & 1);
        tc_fence_after();
        float v[64];
        tmem_ld32(quad + buf * kBlock + half * 64, v);
        tmem_ld32(quad + buf * kBlock + half * 64 + 32, v + 32);
        tmem_wait_ld();
        if (__any_sync(0xffffffffu, left < 64)) {
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] = i < left ? v[i] : -INFINITY;
        }
        float a[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int i = 4; i + 7 < 64; i += 8) {
#pragma unroll
          for (int y = 0; y < 4; ++y) a[y] = max3(a[y], v[i + 2 * y], v[i + 2 * y + 1]);
        }
        a[0] = max3(a[0], v[60], v[61]);
        a[1] = max3(a[1], v[62], v[63]);
        float top = max3(a[0], a[1], fmaxf(a[2], a[3])), other;
        ok = swap(ok, top, other);
        if (!ok) break;
        const float m1 = fmaxf(m, fmaxf(top, other) * c2);
        const float keep = m == -INFINITY ? 1.0f : ex2(m - m1);  // (no key seen so far: all zero)
        const float base = m1 == -INFINITY ? 0.0f : -m1;
        const float2 cc = make_float2(c2, c2), mm = make_float2(base, base);
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          float2 e = fma2(make_float2(v[i], v[i + 1]), cc, mm);
          e.x = ex2(e.x);
          e.y = ex2(e.y);
          sum = __fadd2_rn(sum, e);
          v[i] = e.x;
          v[i + 1] = e.y;
        }
        l = l * keep + (sum.x + sum.y);
        m = m1;
        // The weights' planes, while the last block's product is still being formed.
        uint32_t w[3][32];
#pragma unroll
        for (int plane = 0; plane < 3; ++plane)
#pragma unroll
          for (int y = 0; y < 32; ++y) {
            w[plane][y] = pack_bf16(v[2 * y], v[2 * y + 1]);
            if (plane < 2) {
              v[2 * y] -= __uint_as_float(w[plane][y] << 16);
              v[2 * y + 1] -= __uint_as_float(w[plane][y] & 0xffff0000u);
            }
          }
        // That product has to be in before its place and its weights' are used again.
        if (x > 0) ok = add_block();
        // (Leaving alone is safe: the other warp's next wait fails, and so does its swap.)
        if (!ok) *pair_failed = 1;
#pragma unroll
        for (int plane = 0; plane < 3; ++plane) {
          tmem_st16(quad + kColP + plane * 64 + half * 32, reinterpret_cast<const uint32_t(&)[16]>(w[plane][0]));
          tmem_st16(quad + kColP + plane * 64 + half * 32 + 16, reinterpret_cast<const uint32_t(&)[16]>(w[plane][16]));
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
#pragma unroll
        for (int y = 0; y < 32; ++y) o[y] *= keep;
      }
      if (ok) ok = add_block();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      // The row's sum, its first half's and its second's.
      float other;
      ok = swap(ok, l, other);
      if (!ok) break;
      l = half ? other + l : l + other;
      if (m == -INFINITY && l != l) m = 0.0f;  // every score it saw was NaN: the join must not pass it over
      if (__any_sync(0xffffffffu, flagged) && live) {
#pragma unroll 1
        for (int key = s.k0 * kBlock; key < min(keys, (s.k0 + n) * kBlock); ++key) {
          const float* v = p.v + (int64_t)(s.r0 + key) * p.v_row + s.h * p.v_head + d0;
#pragma unroll
          for (int y = 0; y < 32; ++y) {
            const float z = d0 + y < d1 ? v[y] : 0.0f;
            if (!(fabsf(z) < INFINITY)) o[y] += z;
          }
        }
      }
      const bool whole = s.whole;
      const int64_t part = (int64_t)blockIdx.x * 2 + s.part;
      if (live) {
        const float inv = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
        float* out = whole ? p.out + (s.row0 + (int64_t)token) * p.out_row + (int64_t)(s.h * p.group + head) * p.out_head + d0
                           : p.partials + (part * kBlock + row) * 64 + d0;
#pragma unroll
        for (int y = 0; y < 32; y += 4)
          if (d0 + y < d1) {
            const float4 u = make_float4(o[y] * inv, o[y + 1] * inv, o[y + 2] * inv, o[y + 3] * inv);
            if (whole) *reinterpret_cast<float4*>(out + y) = u;
            else __stcg(reinterpret_cast<float4*>(out + y), u);
          }
        if (!whole && half == 0) __stcg(p.part_ml + part * kBlock + row, make_float2(m, l));
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
        ok = warp_wait(cut_out, n_cut & 1);
        ++n_cut;
        if (ok && *s_ticket == (unsigned)(s.c_last - s.c_first)) join_parts_f32<64, kBlock, 256>(p, s);
      }
    }
  } else if (warp == 8) {
    // ---------------- loads ----------------
    uint32_t seq = 0;
    int q_sent = 0;
    bool ok = true;
#pragma unroll 1
    for (int seg = 0; ok; ++seg) {
      Segment& s = segments[seg % kRing];
      ok = warp_wait(&seg_free[seg % kRing], ((seg / kRing) & 1) ^ 1);
      if (!ok) break;
      if (lane == 0 && !next_segment<kBlock>(p, list, walk, s)) s.n = 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_full[seg % kRing]);
      const int n = s.n, k0 = s.k0;
      if (n == 0) break;
      ok = warp_wait(q_free, (seg & 1) ^ 1);
      if (!ok) break;
      ++q_sent;
      const int rows = (int)p.rows;
      if (lane == 0) mbar_arrive_expect_tx(q_full, (uint32_t)p.tile_tokens * p.group * 128 * 3);
      __syncwarp();
      if (lane < 3) tma_load_4d(smem + lane * kPlane, &qmap, 0, 0, s.h, lane * rows + s.row0, q_full);
#pragma unroll 1
      for (int at = 0; ok && at < 2 * n; ++at) {
        int c;
        const bool is_v = nth_load(false, at, n, c);
        const int st = seq % kStages;
        ok = warp_wait(&empty[st], ((seq / kStages) & 1) ^ 1);
        if (!ok) break;
        ++seq;
        if (lane == 0) mbar_arrive_expect_tx(&full[st], kTile);
        __syncwarp();
        if (lane < 3)
          tma_load_3d(smem + kOffKV + st * kTile + lane * kPlane, is_v ? &vmap : &kmap, 0, s.h,
                      lane * rows + s.r0 + (k0 + c) * kBlock, &full[st]);
      }
    }
    // No copy may be in flight when the CTA exits: without an abort the products have
    // waited for every one.
    if (*s_abort && lane == 0) {
      if (q_sent) drain(q_full, (q_sent - 1) & 1);
      for (uint32_t x = seq > kStages ? seq - kStages : 0; x < seq; ++x) drain(&full[x % kStages], (x / kStages) & 1);
    }
    __syncwarp();
  } else if (warp == 9) {
    // ---------------- products, in the order of the loads ----------------
    const uint32_t idesc_s = umma_idesc_bf16(kBlock, kBlock);
    const uint32_t idesc_o = umma_idesc_bf16(kBlock, ksteps * 16) | (1u << 16);  // B is contiguous along N
    const uint32_t q = desc_qk(smem_u32(smem)), k_desc = desc_qk(smem_u32(smem + kOffKV)),
                   v_desc = desc_v(smem_u32(smem + kOffKV));
    uint32_t seq = 0, n_s = 0, n_p = 0;
#pragma unroll 1
    for (int seg = 0; next(seg); leave(seg), ++seg) {
      if (lane == 0) {
        const int n = segments[seg % kRing].n;
        bool ok = wait(q_full, seg & 1);
        int scores = 0, sums = 0;
#pragma unroll 1
        for (int at = 0; ok && at < 2 * n; ++at, ++seq) {
          int c;
          const bool is_v = nth_load(false, at, n, c);
          const uint32_t st = seq % kStages;
          ok = wait(&full[st], (seq / kStages) & 1);
          if (!ok) break;
          if (!is_v) {
            // (the buffer's last scores were read before the weights that are waited for below)
            tc_fence_after();
            const uint32_t k = k_desc + st * (kTile >> 4), s_col = tmem + (n_s & 1) * kBlock;
#pragma unroll
            for (int i = 0; i < 6; ++i)
#pragma unroll
              for (int y = 0; y < 4; ++y)
                if (y < ksteps)
                  mma_ss(s_col, q + plane_a(i) * (kPlane >> 4) + y * 2, k + plane_b(i) * (kPlane >> 4) + y * 2, idesc_s,
                         i > 0 || y > 0);
            umma_commit(&s_full[n_s & 1]);
            umma_commit(&empty[st]);
            ++n_s;
            if (++scores == n) umma_commit(q_free);
          } else {
            if (sums == 0) ok = wait(o_free, (seg & 1) ^ 1);
            ok = ok && wait(p_full, n_p++ & 1);
            if (!ok) break;
            tc_fence_after();
            const uint32_t v = v_desc + st * (kTile >> 4);
#pragma unroll 1
            for (int i = 0; i < 6; ++i) {
              const uint32_t a = tmem + kColP + plane_a(i) * 64, b = v + plane_b(i) * (kPlane >> 4);
#pragma unroll
              for (int y = 0; y < 8; ++y) mma_ts(tmem + kColO, a + y * 8, b + y * (2048 >> 4), idesc_o, i > 0 || y > 0);
            }
            umma_commit(o_full);
            umma_commit(&empty[st]);
            ++sums;
          }
        }
      }
      __syncwarp();
    }
    if (lane == 0 && *s_abort) {  // the products in flight end before TMEM is freed
      umma_commit(drained);
      drain(drained, 0);
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

cudaError_t launch_split_rows(const F32Attention& p, int heads, __nv_bfloat16* planes, int* flags, cudaStream_t st) {
  split_rows_kernel<<<(unsigned)((p.rows + kSplitRows - 1) / kSplitRows), 256, 0, st>>>(p, heads, planes, flags);
  return cudaGetLastError();
}

cudaError_t launch_attention_f32_tc(const F32TcAttention& p, const CUtensorMap& q, const CUtensorMap& k,
                                    const CUtensorMap& v, int grid, cudaStream_t st) {
  if (cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(attention_f32_tc_kernel), kBytes)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attention_f32_tc_kernel, q, k, v, p);
}

}  // namespace mtrtq
