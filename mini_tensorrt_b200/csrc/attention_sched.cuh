// The list of steps of an attention call (attention_tc.cu, attention_f32.cu): which rows
// and keys a CTA takes, worked out on the device from the lengths there.
//
// A tile is the rows of `tile_tokens` tokens of one request for one key/value head (with
// its group of query heads); its steps are its blocks of BLOCK keys, or half as many
// where two slots take alternate blocks of the same rows. The steps of all tiles, in the
// order request, head, tile, block, are cut into equal runs, one for each CTA.
#pragma once

#include "attention.h"

namespace mtrtq {

struct Request {
  int64_t r0;
  int m;        // rows
  int64_t ctx;  // position of row 0 (negative: rows before the first position see nothing)
  int keys;     // keys it has
};

struct Tile {
  int t0, tokens;  // its tokens, of the request's rows
  bool pair;       // its rows fill more than one slot (f32: always; slot_tokens is 0)
  int blocks, steps;
};

struct Segment {
  Request q;
  Tile tile;
  int b, h;
  int j0, j1;     // its steps of the tile's
  int64_t first;  // the tile's first step in the list
  __device__ bool whole() const { return j0 == 0 && j1 == tile.steps; }
};

__device__ __forceinline__ Request load_request(const AttentionList& p, int b) {
  Request q;
  const int64_t lo = p.cu_rows[b], hi = p.cu_rows[b + 1];
  q.r0 = lo < 0 ? 0 : lo > p.rows ? p.rows : lo;
  q.m = (int)((hi < q.r0 ? q.r0 : hi > p.rows ? p.rows : hi) - q.r0);
  if (p.table) {
    const int64_t n = p.kv_len[b];
    q.ctx = n - q.m;
    q.keys = (int)(n < 0 ? 0 : n < p.max_keys ? n : p.max_keys);
  } else {
    q.ctx = 0;
    q.keys = q.m;
  }
  return q;
}

template <int BLOCK>
__device__ __forceinline__ Tile make_tile(const AttentionList& p, const Request& q, int i) {
  Tile t;
  t.t0 = i * p.tile_tokens;
  t.tokens = min(p.tile_tokens, q.m - t.t0);
  t.pair = t.tokens > p.slot_tokens;
  const int64_t seen = q.ctx + t.t0 + t.tokens;
  const int keys = (int)(seen < q.keys ? seen : q.keys);
  t.blocks = keys <= 0 ? 1 : (keys + BLOCK - 1) / BLOCK;
  t.steps = t.pair ? t.blocks : (t.blocks + 1) >> 1;
  return t;
}

__device__ __forceinline__ int tile_count(const AttentionList& p, const Request& q) {
  return (q.m + p.tile_tokens - 1) / p.tile_tokens;
}

template <int BLOCK>
struct Walk {
  int64_t u, end;
  int b, h, i, j;
  Request q;

  __device__ bool next(const AttentionList& p, Segment& s) {
    if (u >= end) return false;
    s.q = q;
    s.tile = make_tile<BLOCK>(p, q, i);
    s.b = b;
    s.h = h;
    s.j0 = j;
    s.first = u - j;
    const int64_t take = min((int64_t)(s.tile.steps - j), end - u);
    s.j1 = j + (int)take;
    u += take;
    j = s.j1;
    if (j == s.tile.steps) {
      j = 0;
      if (++i == tile_count(p, q)) {
        i = 0;
        if (++h == p.kv_heads) {
          h = 0;
          if (u < end) {
            do q = load_request(p, ++b); while (q.m == 0);
          }
        }
      }
    }
    return true;
  }
};

// This CTA's run, and the steps of a run in `per`. All threads; prefix has batch + 1
// entries and start 4 in shared memory.
template <int BLOCK, int THREADS>
__device__ Walk<BLOCK> find_run(const AttentionList& p, int64_t* prefix, volatile int* start, int64_t& per) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Steps of each request, then their running total.
  for (int b = warp; b < p.batch; b += THREADS / 32) {
    const Request q = load_request(p, b);
    const int n = tile_count(p, q);
    int64_t sum = 0;
    for (int i = lane; i < n; i += 32) sum += make_tile<BLOCK>(p, q, i).steps;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) prefix[b + 1] = sum;
  }
  if (threadIdx.x == 0) prefix[0] = 0;
  __syncthreads();
  if (warp == 0) {
    int64_t run = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      int64_t v = b0 + lane < p.batch ? prefix[b0 + lane + 1] * p.kv_heads : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
      }
      if (b0 + lane < p.batch) prefix[b0 + lane + 1] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  const int64_t total = prefix[p.batch];
  per = (total + gridDim.x - 1) / gridDim.x;
  if (per < p.min_steps) per = p.min_steps;
  Walk<BLOCK> walk;
  walk.u = min(total, per * blockIdx.x);
  walk.end = min(total, walk.u + per);
  if (warp == 0 && walk.u < walk.end) {
    int lo = 0, hi = p.batch - 1;  // the last request whose first step is not after u
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= walk.u) lo = mid; else hi = mid - 1;
    }
    const Request q = load_request(p, lo);
    const int64_t each = (prefix[lo + 1] - prefix[lo]) / p.kv_heads;
    int64_t left = walk.u - prefix[lo];
    const int h = (int)(left / each);
    left -= h * each;
    const int n = tile_count(p, q);
    for (int i0 = 0; i0 < n; i0 += 32) {
      int64_t v = i0 + lane < n ? make_tile<BLOCK>(p, q, i0 + lane).steps : 0;
      const int64_t mine = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
      }
      const unsigned past = __ballot_sync(0xffffffffu, v > left);
      if (past) {
        if (lane == __ffs(past) - 1) {
          start[0] = lo;
          start[1] = h;
          start[2] = i0 + lane;
          start[3] = (int)(left - (v - mine));
        }
        break;
      }
      left -= __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  walk.b = walk.h = walk.i = walk.j = 0;
  if (walk.u < walk.end) {
    walk.b = start[0];
    walk.h = start[1];
    walk.i = start[2];
    walk.j = start[3];
    walk.q = load_request(p, walk.b);
  }
  return walk;
}

}  // namespace mtrtq
