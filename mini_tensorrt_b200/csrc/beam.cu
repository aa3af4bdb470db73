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

// A logit or score as it counts: NaN as -infinity.
__device__ __forceinline__ float number(float x) { return x == x ? x : -INFINITY; }

constexpr int kThreads = 256;
// Logits of one row that a block looks at: 16 per thread, 32 where that still leaves every
// SM several blocks (a block's fixed cost is that of some 20 logits per thread; for a few
// rows more blocks finish sooner). 64 x 8 x 50257 on a B200: 41.8 us with 32, 48.9 with 16.
constexpr int kChunk = 4096;
constexpr int kGroups = 64;    // of 4 threads: their maxima bound the best keys from below
constexpr int kList = 256;     // candidates above that bound which are ranked side by side

// Workspace: a ticket per request, 4 KiB of them | per row and chunk (max, sum of exponentials) | per row
// and chunk beams + 1 keys (logit, index in the row), best first, 0 where there are fewer.
struct BeamLayout {
  int chunk, chunks;
  size_t off_stats, off_keys, total;
};
inline BeamLayout beam_layout(int64_t requests, int64_t beams, int64_t vocab) {
  BeamLayout l;
  // rows start up to 3 floats past 16 bytes
  l.chunk = requests * beams * ((vocab + 3) / kChunk) >= 3000 ? 2 * kChunk : kChunk;
  l.chunks = (int)((vocab + 3 + l.chunk - 1) / l.chunk);
  const size_t parts = (size_t)requests * beams * l.chunks;
  l.off_stats = 4096;
  l.off_keys = (l.off_stats + parts * sizeof(float2) + 255) & ~(size_t)255;
  l.total = l.off_keys + parts * (beams + 1) * sizeof(unsigned long long);
  return l;
}

struct BeamArgs {
  const float* logits;
  int64_t ldl;
  const float* scores;
  const uint8_t* done;
  int eos, beams, vocab, chunk, chunks;
  float* out_scores;
  int32_t *parent, *token;
  uint8_t* out_done;
  unsigned* tickets;
  float2* stats;
  unsigned long long* keys;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// exp(x - m): the difference first, so that a large m costs no bits of the exponent.
__device__ __forceinline__ float exp_below(float x, float m) { return ex2((x - m) * 1.4426950408889634f); }

__device__ unsigned long long block_best(unsigned long long k, unsigned long long* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long x = __shfl_xor_sync(0xffffffffu, k, o);
    k = x > k ? x : k;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = k;
  __syncthreads();
  k = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) k = red[w] > k ? red[w] : k;
  return k;
}

struct Shared {
  unsigned long long list[kList];
  unsigned long long red[kThreads / 32];
  unsigned long long group[kGroups];
  unsigned long long best[MTRTQ_MAX_BEAMS + 1];
  unsigned long long tied[MTRTQ_MAX_BEAMS];
  float lse[MTRTQ_MAX_BEAMS];
  unsigned look[kThreads / 32];
  int ties[kThreads / 32];
  int count;
  // of a chunk
  float group_max[kGroups], warp_max[kThreads / 32], warp_sum[kThreads / 32], bound;
};

// The `want` largest of the block's keys (distinct, 0 = none), best first, in sh.best; 0
// where there are fewer. each(f) calls f with every key of the calling thread, in any
// order, any number of times over. The want-th largest of 64 groups' maxima is at most
// the want-th largest key, so only keys from it on are ranked (some 1.2 times `want`;
// when more than kList reach it, as with many equal logits, `want` rounds of a block-wide
// maximum do it instead).
template <typename Each>
__device__ void block_top(int want, Shared& sh, Each each) {
  const int tid = threadIdx.x, lane = tid & 31;
  unsigned long long k = 0;
  each([&](unsigned long long c) { k = c > k ? c : k; });
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const unsigned long long x = __shfl_xor_sync(0xffffffffu, k, o);
    k = x > k ? x : k;
  }
  __syncthreads();
  if ((lane & 3) == 0) sh.group[tid >> 2] = k;
  if (tid == 0) sh.count = 0;
  if (tid <= MTRTQ_MAX_BEAMS) sh.best[tid] = 0;
  __syncthreads();
  if (tid < kGroups) {
    const unsigned long long mine = sh.group[tid];
    int above = 0;
#pragma unroll 8
    for (int g = 0; g < kGroups; ++g) above += sh.group[g] > mine || (sh.group[g] == mine && g < tid);
    if (above == want - 1) sh.red[0] = mine;
  }
  __syncthreads();
  const unsigned long long bound = sh.red[0] ? sh.red[0] : 1ull;
  each([&](unsigned long long c) {
    if (c >= bound) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kList) sh.list[at] = c;
    }
  });
  __syncthreads();
  const int have = sh.count;
  if (have <= kList) {
    if (tid < have) {
      const unsigned long long mine = sh.list[tid];
      int above = 0;
      for (int x = 0; x < have; ++x) above += sh.list[x] > mine;
      if (above < want) sh.best[above] = mine;
    }
  } else {
    unsigned long long below = ~0ull;
    for (int i = 0; i < want && below; ++i) {
      k = 0;
      each([&](unsigned long long c) { k = c < below && c > k ? c : k; });
      below = block_best(k, sh.red);
      if (tid == 0) sh.best[i] = below;
    }
  }
  __syncthreads();
}

// Candidate (w, t)'s score, with what its row's logits are worth in all.
__device__ __forceinline__ float row_score(float base, float x, float lse) {
  return number(base + (x - lse));
}

// One block per (chunk, row). It reads its logits once: their maximum and the sum of
// exponentials below it, and the beams + 1 largest. The last block of a request then
// joins the rows' sums into log-sums and ranks the rows' candidates by their scores.
// The floor is memory's, 4 bytes of each logit once (rows of beams that are done or not in
// use are not read): 15.7 us for 64 x 8 x 50257, where a B200 takes 41, bound by latency and
// by the instructions of each logit (1.6 a clock, registers for 5 blocks an SM).
//
// Rounding can give two unequal logits of a row the same score, and the tie then goes to
// the lower index, perhaps to a logit that its chunk did not pass on. That needs a score
// of the first one left out, at most that of the last one passed on, no worse than the
// last beam chosen: where a chunk's (beams + 1)-th does reach it, its logits are looked at
// again.
template <int E>
__global__ void __launch_bounds__(kThreads, 5) beam_kernel(const __grid_constant__ BeamArgs p) {
  __shared__ Shared sh;
  __shared__ unsigned ticket;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int chunk = blockIdx.x, w0 = blockIdx.y, want = p.beams + 1;
  const int64_t request = blockIdx.z, first_row = request * p.beams, row = first_row + w0;
  const float* x = p.logits + row * p.ldl;
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) >> 2);
  const int64_t part = row * p.chunks + chunk;
  const bool used = p.done[row] == 0 && p.scores[row] > -INFINITY;
  if (used) {
    // 16-byte loads from the boundary before the row's first logit on
    const int t0 = chunk * E * kThreads + tid * 4 - shift;
    const bool inside = chunk > 0 && (chunk + 1) * E * kThreads - shift <= p.vocab;
    float v[E];
#pragma unroll
    for (int j = 0; j < E / 4; ++j) {
      const int t = t0 + j * kThreads * 4;
      float4 u = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (inside || (t < p.vocab && t + 3 >= 0)) u = __ldcs(reinterpret_cast<const float4*>(x + t));
      v[4 * j] = u.x;
      v[4 * j + 1] = u.y;
      v[4 * j + 2] = u.z;
      v[4 * j + 3] = u.w;
    }
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = fmaxf(v[j], -INFINITY);  // NaN counts as -infinity
    if (!inside) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int t = t0 + (j >> 2) * kThreads * 4 + (j & 3);
        if (t < 0 || t >= p.vocab) v[j] = -INFINITY;
      }
    }
    // Maxima of groups of threads (32 of eight while they bound `want` keys well, else 64 of
    // four) and of the warp; the warp's sum below its own maximum.
    const int group = want <= 16 ? 8 : 4, groups = kThreads / group;
    float m = v[0];
#pragma unroll
    for (int j = 1; j < E; ++j) m = fmaxf(m, v[j]);
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    if (group == 4 && (lane & 3) == 0) sh.group_max[tid >> 2] = m;
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
    if (group == 8 && (lane & 7) == 0) sh.group_max[tid >> 3] = m;
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < E; ++j) s[j & 3] += exp_below(v[j], m);
    float sum = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      sh.warp_max[warp] = m;
      sh.warp_sum[warp] = m == -INFINITY ? 0.0f : sum;
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
    if (tid < groups) {
      // the want-th largest of the groups' maxima
      const float mine = sh.group_max[tid];
      int above = 0;
#pragma unroll 8
      for (int g = 0; g < groups; ++g) {
        const float o = sh.group_max[g];
        above += o > mine || (o == mine && g < tid);
      }
      if (above == want - 1) sh.bound = mine;
    } else if (tid == kThreads - 1) {
      float top = sh.warp_max[0], all = 0.0f;
#pragma unroll
      for (int w = 1; w < kThreads / 32; ++w) top = fmaxf(top, sh.warp_max[w]);
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w)
        all += sh.warp_max[w] == top ? sh.warp_sum[w] : sh.warp_sum[w] * exp_below(sh.warp_max[w], top);
      __stcg(p.stats + part, make_float2(top, all));
    }
    __syncthreads();
    const float bound = sh.bound;
    auto key = [&](int j) {
      return candidate_key(v[j], (uint32_t)(t0 + (j >> 2) * kThreads * 4 + (j & 3)));
    };
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (v[j] >= bound && v[j] > -INFINITY) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kList) sh.list[at] = key(j);
      }
    }
    __syncthreads();
    const int have = sh.count;
    unsigned long long* out = p.keys + part * want;
    if (have <= kList) {
      if (tid < have) {
        const unsigned long long mine = sh.list[tid];
        int above = 0;
        for (int e = 0; e < have; ++e) above += sh.list[e] > mine;
        if (above < want) __stcg(out + above, mine);
      } else if (tid < want) {
        __stcg(out + tid, 0ull);
      }
    } else {
      // many logits reach the bound (equal ones, as a rule): a block-wide maximum each
      unsigned long long below = ~0ull;
      for (int i = 0; i < want; ++i) {
        unsigned long long k = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const unsigned long long c = v[j] > -INFINITY ? key(j) : 0ull;
          k = c < below && c > k ? c : k;
        }
        below = block_best(k, sh.red);
        if (tid == 0) __stcg(out + i, below);
      }
    }
  }
  __syncthreads();
  if (tid == 0) ticket = ticket_acq_rel(p.tickets + request);
  __syncthreads();
  if (ticket != (unsigned)(p.beams * p.chunks - 1)) return;

  // ---- the request's last block ----
  for (int w = warp; w < p.beams; w += kThreads / 32) {
    const int64_t r = first_row + w;
    float lse = -INFINITY;  // of a row that passes nothing on
    if (p.done[r] == 0 && p.scores[r] > -INFINITY) {
      float m = -INFINITY, s = 0.0f;
      for (int c = lane; c < p.chunks; c += 32) m = fmaxf(m, __ldcg(p.stats + r * p.chunks + c).x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      for (int c = lane; c < p.chunks; c += 32) {
        const float2 st = __ldcg(p.stats + r * p.chunks + c);
        s += st.x == m ? st.y : st.y * exp_below(st.x, m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      lse = m + logf(s);
    }
    if (lane == 0) sh.lse[w] = lse;
  }
  __syncthreads();
  const int per_row = p.chunks * want, all = p.beams * per_row;
  // Keys of what the chunks passed on (those of -infinity fill what is left at the end).
  auto passed = [&](auto f) {
    for (int e = tid; e < all; e += kThreads) {
      const int w = e / per_row;
      const int64_t r = first_row + w;
      if (p.done[r] != 0 || !(p.scores[r] > -INFINITY)) continue;
      const unsigned long long k = __ldcg(p.keys + r * per_row + (e - w * per_row));
      if (!k) continue;
      const float s = row_score(p.scores[r], key_score(k), sh.lse[w]);
      if (s > -INFINITY) f(candidate_key(s, (uint32_t)w * p.vocab + key_index(k)));
    }
    if (tid < p.beams && p.done[first_row + tid] != 0 && p.eos >= 0 && p.scores[first_row + tid] > -INFINITY)
      f(candidate_key(p.scores[first_row + tid], (uint32_t)tid * p.vocab + p.eos));
  };
  block_top(p.beams, sh, passed);
  const unsigned long long kth = sh.best[p.beams - 1];
  const float least = key_score(kth);
  // Which chunks may hold more: the last one each passed on reaches the last beam.
  auto reaches = [&](int w, int c) {
    const int64_t r = first_row + w;
    if (!kth || p.done[r] != 0 || !(p.scores[r] > -INFINITY)) return false;
    const unsigned long long k = __ldcg(p.keys + r * per_row + c * want + want - 1);
    return k && row_score(p.scores[r], key_score(k), sh.lse[w]) >= least;
  };
  bool again = false;
  for (int e = tid; e < p.beams * p.chunks; e += kThreads) again |= reaches(e / p.chunks, e % p.chunks);
  if (__syncthreads_or(again)) {
    // Whatever has a higher score than the last beam is here (as below), so the `open` places
    // from there on go to the lowest indices with its very score. Those chunks are looked
    // through in order, until they have given so many: with the type's lowest value as a
    // mask, which ties every masked token, and one beam of 8 x 50257 in use, 18 us, where a
    // pass for each place took 522.
    int better = 0;
    for (int i = 0; i < p.beams; ++i) better += key_score(sh.best[i]) > least;
    const int open = p.beams - better;
    int found = 0;
    for (int e0 = 0; e0 < p.beams * p.chunks && found < open; e0 += kThreads) {
      const int e1 = e0 + tid;
      const bool look = e1 < p.beams * p.chunks && reaches(e1 / p.chunks, e1 % p.chunks);
      unsigned bits = __ballot_sync(0xffffffffu, look);
      __syncthreads();
      if (lane == 0) sh.look[warp] = bits;
      __syncthreads();
      for (int x = 0; x < kThreads / 32; ++x) {
        for (bits = sh.look[x]; bits && found < open; bits &= bits - 1) {
          const int e = e0 + x * 32 + __ffs(bits) - 1, w = e / p.chunks, c = e % p.chunks;
          const int64_t r = first_row + w;
          const float* y = p.logits + r * p.ldl;
          const int skip = (int)((reinterpret_cast<uintptr_t>(y) & 15) >> 2);
          const int t1 = min(p.vocab, (c + 1) * p.chunk - skip);
          for (int t = max(0, c * p.chunk - skip); t < t1 && found < open; t += kThreads) {
            const int at = t + tid;
            const bool tie = at < t1 && row_score(p.scores[r], number(y[at]), sh.lse[w]) == least;
            const unsigned ties = __ballot_sync(0xffffffffu, tie);
            if (lane == 0) sh.ties[warp] = __popc(ties);
            __syncthreads();
            int to = found + __popc(ties & ((1u << lane) - 1));
            for (int v = 0; v < kThreads / 32; ++v) {
              to += v < warp ? sh.ties[v] : 0;
              found += sh.ties[v];
            }
            if (tie && to < open) sh.tied[to] = candidate_key(least, (uint32_t)w * p.vocab + at);
            __syncthreads();
          }
        }
      }
    }
    // Joined with those here already (some are in both), best first.
    if (warp == 0) {
      const unsigned long long a = lane < open ? sh.best[better + lane] : 0, b = lane < min(found, open) ? sh.tied[lane] : 0;
      bool twice = a == 0;
      for (int i = 0; i < 32; ++i) twice |= a == __shfl_sync(0xffffffffu, b, i);
      const unsigned own = __ballot_sync(0xffffffffu, !twice);
      int at_a = __popc(own & ((1u << lane) - 1)), at_b = lane;
      for (int i = 0; i < 32; ++i) {
        at_a += __shfl_sync(0xffffffffu, b, i) > a;
        at_b += __shfl_sync(0xffffffffu, a, i) > b && (own >> i & 1);
      }
      if (!twice && at_a < open) sh.best[better + at_a] = a;
      if (b && at_b < open) sh.best[better + at_b] = b;
    }
    __syncthreads();
  } else if (!kth) {
    // Fewer candidates have a score than there are beams, and all of those are here (a chunk
    // that left one out would have passed on beams + 1 others no worse). Every other's is
    // -infinity, so the lowest indices not taken follow, all of them below `beams`: with two
    // tokens of one beam of 8 x 50257 left 9.7 us, where looking the logits through again took
    // 1443.
    if (warp == 0) {
      int have = 0;
      bool open = lane < p.beams;
      for (int i = 0; i < p.beams; ++i) {
        const unsigned long long k = sh.best[i];
        have += k != 0;
        open &= k == 0 || key_index(k) != (uint32_t)lane;
      }
      const int at = have + __popc(__ballot_sync(0xffffffffu, open) & ((1u << lane) - 1));
      if (open && at < p.beams) sh.best[at] = candidate_key(-INFINITY, lane);
    }
    __syncthreads();
  }
  if (tid < p.beams) {
    const uint32_t at = key_index(sh.best[tid]);
    const int w = at / p.vocab, t = at % p.vocab;
    p.out_scores[first_row + tid] = key_score(sh.best[tid]);
    p.parent[first_row + tid] = w;
    p.token[first_row + tid] = t;
    p.out_done[first_row + tid] = p.done[first_row + w] != 0 || t == p.eos;
  }
  if (tid == 0) p.tickets[request] = 0u;
}

// The partly filled pages' tokens move along with their beams, in place: a thread
// reads its 16 bytes of every beam's parent before it writes any beam's, and no other
// thread touches those. Grid (chunks of a page, layers, requests); the request's
// first block moves the table's rows the same way. Bound by memory: 16 requests of 8 beams,
// 12 layers of 12 x 64 in bf16, take 42.5 us on a B200, 96 % of a plain copy's rate.
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
  if (requests < 1 || requests > MTRTQ_MAX_BATCH || beams < 1 || beams > MTRTQ_MAX_BEAMS)
    return report_error(MTRTQ_ERR_INVALID_ARG, "requests (%lld) is 1 to %d, beams (%lld) 1 to %d",
                        (long long)requests, MTRTQ_MAX_BATCH, (long long)beams, MTRTQ_MAX_BEAMS);
  return MTRTQ_OK;
}

int check_select(int64_t requests, int64_t beams, int64_t vocab) {
  if (int rc = check_beams(requests, beams)) return rc;
  // (32-bit places of a row, up to a block and a few past its end)
  constexpr int64_t most = (int64_t(1) << 31) - 2 * (2 * kChunk);
  if (vocab < 1 || vocab > most || vocab * beams > most)
    return report_error(MTRTQ_ERR_INVALID_ARG, "vocab (%lld) times beams is 1 to %lld", (long long)vocab,
                        (long long)most);
  return MTRTQ_OK;
}

}  // namespace
}  // namespace mtrtq

using namespace mtrtq;

extern "C" {

int64_t mtrtq_beam_workspace_bytes(int64_t requests, int64_t beams, int64_t vocab) {
  if (check_select(requests, beams, vocab)) return -1;
  return (int64_t)beam_layout(requests, beams, vocab).total;
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
  if (reinterpret_cast<uintptr_t>(workspace) % 256 || reinterpret_cast<uintptr_t>(logits) % 4)
    return report_error(MTRTQ_ERR_ALIGNMENT, "workspace must be 256-byte aligned, logits 4-byte");
  const BeamLayout l = beam_layout(requests, beams, vocab);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const BeamArgs p = {logits, ldl, scores, done, eos, (int)beams, (int)vocab, l.chunk, l.chunks, out_scores, parent, token,
                      out_done, reinterpret_cast<unsigned*>(ws), reinterpret_cast<float2*>(ws + l.off_stats),
                      reinterpret_cast<unsigned long long*>(ws + l.off_keys)};
  const dim3 grid(l.chunks, (unsigned)beams, (unsigned)requests);
  if (l.chunk == kChunk) beam_kernel<16><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  else beam_kernel<32><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
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
