// The list of steps of an attention call (attention_tc.cu, attention_f32.cu): which rows
// and keys a CTA takes, worked out on the device from the lengths there.
//
// A tile is the rows of `tile_tokens` tokens of one request for one key/value head (with
// its group of query heads); its steps are its blocks of BLOCK keys, or half as many
// where two slots take alternate blocks of the same rows. The steps of all tiles, in the
// order request, head, tile, block, are cut into equal runs, one for each CTA.
#pragma once

#include "../../include/mtrtq.h"
#include "attention.h"
#include "q8_common.cuh"

namespace mtrtq {

// A request's rows r0 .. r0 + m - 1, the position of the first (negative: rows before
// the first position see nothing), and the keys it has.
struct Request {
  int r0, m, ctx, keys;
};

// A CTA's next run of one tile's steps: what its roles need to know of it.
struct Segment {
  int b, h;
  int r0, row0;    // the request's first row, the tile's
  int tokens;      // its tokens
  int see0;        // keys that the first row sees, if the request has them
  int keys;        // keys the request has
  int pair;        // the rows fill more than one slot (f32: always)
  int k0, n;       // blocks of keys k0 .. k0 + n - 1
  int cnt[2];      // of them, blocks of each slot
  int whole;       // all of the tile's steps
  int part;        // else: which of the CTA's two partials
  int c_first, c_last;  // else: the CTAs that have parts of the tile
  int buf;         // halves: which of the two Q buffers
  int q_use[2];    // earlier uses of the Q buffers
  __device__ int all_see() const { return min(see0, keys); }
};

struct Walk {
  int64_t u, end, per;
  int b, h, i, j;
  int buf, q_use[2];
};

struct StepList {
  Request* req;     // [batch]
  int64_t* prefix;  // [batch + 1] steps before each request, while the list is made
};

__device__ __forceinline__ Request load_request(const AttentionList& p, int b) {
  const int lo = p.cu_rows[b], hi = p.cu_rows[b + 1], rows = (int)p.rows;
  const int n = p.table ? p.kv_len[b] : 0;
  Request q;
  q.r0 = min(max(lo, 0), rows);
  q.m = min(max(hi, q.r0), rows) - q.r0;
  q.ctx = p.table ? max(n, -(1 << 30)) - q.m : 0;
  q.keys = p.table ? min(max(n, 0), (int)p.max_keys) : q.m;
  if (q.m < p.least || q.m > p.most) q.m = 0;  // another launch's
  return q;
}

__device__ __forceinline__ int tile_count(const AttentionList& p, const Request& q) {
  return (q.m + p.tile_tokens - 1) / p.tile_tokens;
}

// Blocks of keys that tokens t0 .. t0 + tokens - 1 see together; at least one, so that
// rows that see none are written too.
template <int BLOCK>
__device__ __forceinline__ int block_count(const Request& q, int t0, int tokens) {
  return max(1, (min(q.keys, q.ctx + t0 + tokens) + BLOCK - 1) / BLOCK);
}

template <int BLOCK>
__device__ __forceinline__ int tile_steps(const AttentionList& p, const Request& q, int i) {
  const int t0 = i * p.tile_tokens, tokens = min(p.tile_tokens, q.m - t0);
  const int blocks = block_count<BLOCK>(q, t0, tokens);
  return tokens > p.slot_tokens ? p.pair_cost + blocks : p.tile_cost + ((blocks + 1) >> 1);
}

// One thread's; false at the end of the CTA's run. A tile counts tile_cost or
// pair_cost steps more than it has: what starting and ending it takes.
template <int BLOCK>
__device__ bool next_segment(const AttentionList& p, const StepList list, Walk& w, Segment& s) {
#pragma unroll 1
  while (w.u < w.end) {
    const Request q = list.req[w.b];
    const int t0 = w.i * p.tile_tokens, tokens = min(p.tile_tokens, q.m - t0);
    const int blocks = block_count<BLOCK>(q, t0, tokens);
    const bool pair = tokens > p.slot_tokens;
    const int steps = pair ? blocks : (blocks + 1) >> 1;
    const int64_t first = w.u - w.j;  // of the tile's
    const int extra = pair ? p.pair_cost : p.tile_cost, cost = steps + extra;
    const int take = (int)min((int64_t)(cost - w.j), w.end - w.u);
    const int j0 = max(0, w.j - extra), j1 = max(0, w.j + take - extra);
    s.b = w.b;
    s.h = w.h;
    s.r0 = q.r0;
    s.row0 = q.r0 + t0;
    s.tokens = tokens;
    s.see0 = q.ctx + t0 + 1;
    s.keys = q.keys;
    s.pair = pair;
    s.k0 = pair ? j0 : 2 * j0;
    s.n = (pair ? j1 : min(2 * j1, blocks)) - s.k0;
    if (pair) {
      const int sees = min(q.keys, q.ctx + t0 + p.slot_tokens);  // slot 0's last row
      s.cnt[0] = max(0, min(j1, sees <= 0 ? 0 : (sees + BLOCK - 1) / BLOCK) - j0);
      s.cnt[1] = s.n;
    } else {
      s.cnt[0] = (s.n + 1) >> 1;
      s.cnt[1] = s.n >> 1;
    }
    s.whole = j1 - j0 == steps;
    if (!s.whole) {
      s.part = j0 > 0 ? 0 : 1;
      s.c_first = (int)((first + extra) / w.per);
      s.c_last = (int)((first + cost - 1) / w.per);
    }
    w.u += take;
    w.j += take;
    if (w.j == cost) {
      w.j = 0;
      if (++w.i == tile_count(p, q)) {
        w.i = 0;
        if (++w.h == p.kv_heads) {
          w.h = 0;
          if (w.u < w.end) {
            do ++w.b; while (list.req[w.b].m == 0);
          }
        }
      }
    }
    if (j1 == j0) continue;  // the end of the run lies in what starting the tile takes
    s.buf = w.buf;
    s.q_use[0] = w.q_use[0];
    s.q_use[1] = w.q_use[1];
    if (pair) {
      ++w.q_use[0];
      ++w.q_use[1];
      w.buf = 0;
    } else {
      ++w.q_use[w.buf];
      w.buf = p.q_buffers - 1 - w.buf;
    }
    return true;
  }
  return false;
}

// Whether the second kernel of a call (attention.cu) finds no request of its own, as is usual:
// it then leaves before it sets anything up. All threads.
template <int THREADS>
__device__ __forceinline__ bool nothing_here(const AttentionList& p) {
  if (p.least <= 1) return false;
  bool any = false;
  for (int b = threadIdx.x; b < p.batch; b += THREADS) any |= load_request(p, b).m > 0;
  return !__syncthreads_or(any);
}

// Fills the list and this CTA's walk, which every thread gets, through `shared`. All threads.
template <int BLOCK, int THREADS>
__device__ void make_list(const AttentionList& p, const StepList list, Walk& walk, Walk* shared) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // Requests, and the steps of those with few tiles: a thread each.
  bool many = false;
#pragma unroll 1
  for (int b = tid; b < p.batch; b += THREADS) {
    const Request q = load_request(p, b);
    list.req[b] = q;
    const int n = tile_count(p, q);
    int64_t sum = 0;
    if (n <= 8) {
#pragma unroll 1
      for (int i = 0; i < n; ++i) sum += tile_steps<BLOCK>(p, q, i);
    } else {
      sum = -1;
      many = true;
    }
    list.prefix[b + 1] = sum;
  }
  if (tid == 0) list.prefix[0] = 0;
  if (__syncthreads_or(many)) {
#pragma unroll 1
    for (int b = warp; b < p.batch; b += THREADS / 32) {
      if (list.prefix[b + 1] >= 0) continue;
      const Request q = list.req[b];
      const int n = tile_count(p, q);
      int64_t sum = 0;
#pragma unroll 1
      for (int i = lane; i < n; i += 32) sum += tile_steps<BLOCK>(p, q, i);
#pragma unroll 1
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      __syncwarp();
      if (lane == 0) list.prefix[b + 1] = sum;
    }
    __syncthreads();
  }
  if (warp == 0) {
    int64_t run = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      int64_t v = b0 + lane < p.batch ? list.prefix[b0 + lane + 1] * p.kv_heads : 0;
#pragma unroll 1
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
      }
      if (b0 + lane < p.batch) list.prefix[b0 + lane + 1] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
    __syncwarp();
    const int64_t total = run, per = max((total + gridDim.x - 1) / gridDim.x, p.min_steps);
    Walk w;
    w.per = per;
    w.u = min(total, per * blockIdx.x);
    w.end = min(total, w.u + per);
    w.b = w.h = w.i = w.j = w.buf = w.q_use[0] = w.q_use[1] = 0;
    if (w.u < w.end) {
      int lo = 0, hi = p.batch - 1;  // the last request whose first step is not after u
#pragma unroll 1
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (list.prefix[mid] <= w.u) lo = mid; else hi = mid - 1;
      }
      const Request q = list.req[lo];
      const int64_t each = (list.prefix[lo + 1] - list.prefix[lo]) / p.kv_heads;
      int64_t left = w.u - list.prefix[lo];
      w.b = lo;
      w.h = (int)(left / each);
      left -= w.h * each;
      const int n = tile_count(p, q);
#pragma unroll 1
      for (int i0 = 0; i0 < n; i0 += 32) {
        int64_t v = i0 + lane < n ? tile_steps<BLOCK>(p, q, i0 + lane) : 0;
        const int64_t mine = v;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t x = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, v > left);
        if (past) {
          const int at = __ffs(past) - 1;
          w.i = i0 + at;
          w.j = (int)__shfl_sync(0xffffffffu, left - (v - mine), at);
          break;
        }
        left -= __shfl_sync(0xffffffffu, v, 31);
      }
    }
    if (lane == 0) *shared = w;
  }
  fence_proxy_async_smem();  // bulk copies may land where the prefix was
  __syncthreads();
  walk = *shared;
  __syncthreads();
}

}  // namespace mtrtq
