// Attention with every product and sum in fp32, on the CUDA cores: packed prompts and new
// tokens over a paged cache whose rows and pages are f32 (for a row or two, bf16 too).
//
// The same online softmax as on the tensor cores (attention_tc.cu), over blocks of 64 keys:
// a CTA of 256 threads holds a tile of 16 RM rows (tokens times the group's heads), thread
// (ty, tx) the rows ty RM .. and the keys 4 tx .. of the scores, then the same rows and
// dimensions 4 tx .. of the output. Q and K lie transposed in shared memory, so that one
// dimension's step is RM + 4 values read for 4 RM products (packed two at a time), and P
// transposed for the same reason. Bound by these reads of shared
// memory (65 to 70 % of its rate with tiles of 128 rows; four chunks of 1 to 128 tokens, 25
// heads of 64, over up to 1000: 67 us, 44 %); 32 x 8 threads instead of 16 x 16 were slower.
//
// V rows past the request's keys are read as zeros; where a block not seen whole by every
// row holds an infinity or a NaN, its products are formed only for the rows that see them.
#include <limits.h>
#include <math.h>

#include "../../include/mtrtq.h"
#include "attention_mma.cuh"

namespace mtrtq {

namespace {

constexpr int kKeys = 64;
constexpr int kThreads = 256;

template <int HD, int RM>
struct Cfg {
  static constexpr int BM = 16 * RM;
  static constexpr int QS = BM + 4;    // row strides, in floats
  static constexpr int KS = kKeys + 4;
  static constexpr int OFF_Q = 0;                       // [HD][QS]
  static constexpr int OFF_K = OFF_Q + HD * QS;         // [HD][KS]
  static constexpr int OFF_V = OFF_K + HD * KS;         // [kKeys][HD]
  static constexpr int OFF_P = OFF_V + kKeys * HD;      // [kKeys][QS]
  static constexpr int FLOATS = OFF_P + kKeys * QS;
  static constexpr int BYTES = FLOATS * 4;  // and the list of steps
  static constexpr int CTAS = HD == 64 || RM == 1 ? 2 : 1;
  static_assert(CTAS * (BYTES + 5 * 1024) <= 228 * 1024 && FLOATS % 4 == 0, "shared memory per CTA");
};

__device__ __forceinline__ bool broken(float x) { return !(fabsf(x) < INFINITY); }

template <int HD, int RM, bool PAGED>
__global__ void __launch_bounds__(kThreads, Cfg<HD, RM>::CTAS)
    attention_f32_kernel(const __grid_constant__ F32Attention p) {
  using C = Cfg<HD, RM>;
  constexpr int RP = RM == 1 ? 1 : RM / 2;  // row pairs of a thread
  constexpr int NC = HD / 64;               // groups of four output columns of a thread
  constexpr int NL = HD / 16;               // 16-byte loads of K, and of V, of a thread
  constexpr bool AHEAD = RM < 8;
  extern __shared__ float4 raw4[];
  float* sm = reinterpret_cast<float*>(raw4);
  float *qs = sm + C::OFF_Q, *ks = sm + C::OFF_K, *vs = sm + C::OFF_V, *ps = sm + C::OFF_P;
  const StepList list = {reinterpret_cast<Request*>(sm + C::FLOATS), reinterpret_cast<int64_t*>(sm)};  // the prefix lies where Q will
  __shared__ Walk shared_walk;
  __shared__ Segment s;
  __shared__ int more;
  __shared__ unsigned ticket;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, lane = tid & 31, warp = tid >> 5;

  if (nothing_here<kThreads>(p)) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (the stream goes on when this kernel ends)
    return;
  }
  Walk walk;
  make_list<kKeys, kThreads>(p, list, walk, &shared_walk);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float c2 = p.scale * 1.4426950408889634f;  // scale log2 e

  while (true) {
    __syncthreads();
    if (tid == 0) more = next_segment<kKeys>(p, list, walk, s);
    __syncthreads();
    if (!more) break;
    const int64_t r0 = s.r0;  // where the request's rows start
    const int tokens = s.tokens, keys = s.keys;
    // K and V of a block, on their way together (and while the last block is worked on, where
    // registers allow it): a lane per key of K, which is transposed, V as it is. Tokens past
    // the keys, and pages out of range, read as zeros.
    float4 kr[NL], vr[NL];
    auto fetch = [&](int key0) {
      const int key = key0 + (warp & 1) * 32 + lane;
      const float* src = nullptr;
      if (key < keys) {
        if (PAGED) {
          const int64_t page = p.table[s.b * p.table_ld + key / p.page_size];
          if (page >= 0 && page < p.num_pages)
            src = p.k + page * p.k_row + ((int64_t)s.h * p.page_size + key % p.page_size) * p.head_dim;
        } else {
          src = p.k + (r0 + key) * p.k_row + s.h * p.k_head;
        }
      }
#pragma unroll
      for (int c = 0; c < NL; ++c) {
        const int d = (warp >> 1) * (HD / 4) + c * 4;
        kr[c] = src && d < p.head_dim ? *reinterpret_cast<const float4*>(src + d) : make_float4(0, 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < NL; ++c) {
        const int e = c * kThreads + tid, at = key0 + e / (HD / 4), d = e % (HD / 4) * 4;
        vr[c] = make_float4(0, 0, 0, 0);
        if (at < keys && d < p.head_dim) {
          if (PAGED) {
            const int64_t page = p.table[s.b * p.table_ld + at / p.page_size];
            if (page >= 0 && page < p.num_pages)
              vr[c] = *reinterpret_cast<const float4*>(
                  p.v + page * p.v_row + ((int64_t)s.h * p.page_size + at % p.page_size) * p.head_dim + d);
          } else {
            vr[c] = *reinterpret_cast<const float4*>(p.v + (r0 + at) * p.v_row + s.h * p.v_head + d);
          }
        }
      }
    };
    if (AHEAD) fetch(s.k0 * kKeys);
    // Q, transposed; rows past the tile's tokens and dimensions past the head's are zero.
    for (int e = tid; e < C::BM * (HD / 4); e += kThreads) {
      const int row = e % C::BM, d = e / C::BM * 4;
      const int token = row / p.group, head = row - token * p.group;
      float4 x = make_float4(0, 0, 0, 0);
      if (token < tokens && d < p.head_dim)
        x = *reinterpret_cast<const float4*>(p.q + (s.row0 + (int64_t)token) * p.q_row +
                                             (int64_t)(s.h * p.group + head) * p.q_head + d);
      qs[d * C::QS + row] = x.x;
      qs[(d + 1) * C::QS + row] = x.y;
      qs[(d + 2) * C::QS + row] = x.z;
      qs[(d + 3) * C::QS + row] = x.w;
    }
    float m[RM], l[RM], o[RM][4 * NC];
    int sees[RM];  // keys the row sees
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.0f;
#pragma unroll
      for (int c = 0; c < 4 * NC; ++c) o[r][c] = 0.0f;
      const int token = (ty * RM + r) / p.group;
      sees[r] = token < tokens ? max(0, min(s.see0 + token, keys)) : 0;
    }
    const int all_see = s.all_see(), k1 = s.k0 + s.n;

    for (int j = s.k0; j < k1; ++j) {
      const int key0 = j * kKeys;
      __syncthreads();
      bool odd = false;
      if (!AHEAD) fetch(key0);
#pragma unroll
      for (int c = 0; c < NL; ++c) {
        float* dst = ks + ((warp >> 1) * (HD / 4) + c * 4) * C::KS + (warp & 1) * 32 + lane;
        dst[0] = kr[c].x;
        dst[C::KS] = kr[c].y;
        dst[2 * C::KS] = kr[c].z;
        dst[3 * C::KS] = kr[c].w;
        *reinterpret_cast<float4*>(vs + (c * kThreads + tid) * 4) = vr[c];
        odd |= broken(vr[c].x) | broken(vr[c].y) | broken(vr[c].z) | broken(vr[c].w);
      }
      const bool partly = key0 + kKeys > all_see;
      const bool careful = __syncthreads_or(odd) && partly;
      if (AHEAD && j + 1 < k1) fetch(key0 + kKeys);

      // S: rows in pairs, four keys
      float2 a[RP][4];
#pragma unroll
      for (int r = 0; r < RP; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) a[r][c] = make_float2(0, 0);
#pragma unroll 8
      for (int d = 0; d < HD; ++d) {
        const float4 k4 = *reinterpret_cast<const float4*>(ks + d * C::KS + 4 * tx);
        const float kk[4] = {k4.x, k4.y, k4.z, k4.w};
        if (RM == 1) {
          const float q = qs[d * C::QS + ty];
#pragma unroll
          for (int c = 0; c < 4; c += 2) {
            const float2 t = fma2(make_float2(q, q), make_float2(kk[c], kk[c + 1]), make_float2(a[0][c].x, a[0][c + 1].x));
            a[0][c].x = t.x;
            a[0][c + 1].x = t.y;
          }
        } else {
          float q[RM];
#pragma unroll
          for (int r = 0; r < RM; r += 4)
            *reinterpret_cast<float4*>(q + r) = *reinterpret_cast<const float4*>(qs + d * C::QS + ty * RM + r);
#pragma unroll
          for (int r = 0; r < RP; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              a[r][c] = fma2(make_float2(q[2 * r], q[2 * r + 1]), make_float2(kk[c], kk[c]), a[r][c]);
        }
      }
      // softmax: a row's 64 scores lie in the 16 lanes of one ty
      float pr[RM][4];
#pragma unroll
      for (int r = 0; r < RM; ++r) {
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          pr[r][c] = (r & 1) ? a[r >> 1][c].y : a[r >> 1][c].x;
          if (partly && key0 + 4 * tx + c >= sees[r]) pr[r][c] = -INFINITY;
          top = fmaxf(top, pr[r][c]);
        }
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        top *= c2;
        const float now = fmaxf(m[r], top);
        const float base = now == -INFINITY ? 0.0f : now;
        const float keep = m[r] == -INFINITY ? 1.0f : ex2(m[r] - base);
        m[r] = now;
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          pr[r][c] = ex2(fmaf(pr[r][c], c2, -base));
          sum += pr[r][c];
        }
        l[r] = l[r] * keep + sum;  // this lane's share
#pragma unroll
        for (int c = 0; c < 4 * NC; ++c) o[r][c] *= keep;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float* dst = ps + (4 * tx + c) * C::QS + ty * RM;
        if (RM == 1) {
          dst[0] = pr[0][c];
        } else {
#pragma unroll
          for (int r = 0; r + 3 < RM; r += 4)
            *reinterpret_cast<float4*>(dst + r) = make_float4(pr[r][c], pr[r + 1][c], pr[r + 2][c], pr[r + 3][c]);
        }
      }
      __syncwarp();  // a row's weights are written and read by the same half warp
      if (!careful) {
#pragma unroll 4
        for (int y = 0; y < kKeys; ++y) {
          float w[RM];
          if (RM == 1) {
            w[0] = ps[y * C::QS + ty];
          } else {
#pragma unroll
            for (int r = 0; r + 3 < RM; r += 4)
              *reinterpret_cast<float4*>(w + r) = *reinterpret_cast<const float4*>(ps + y * C::QS + ty * RM + r);
          }
#pragma unroll
          for (int g = 0; g < NC; ++g) {
            const float4 v = *reinterpret_cast<const float4*>(vs + y * HD + g * 64 + 4 * tx);
#pragma unroll
            for (int r = 0; r < RM; ++r) {
              float2 t0 = fma2(make_float2(w[r], w[r]), make_float2(v.x, v.y), make_float2(o[r][4 * g], o[r][4 * g + 1]));
              float2 t1 =
                  fma2(make_float2(w[r], w[r]), make_float2(v.z, v.w), make_float2(o[r][4 * g + 2], o[r][4 * g + 3]));
              o[r][4 * g] = t0.x;
              o[r][4 * g + 1] = t0.y;
              o[r][4 * g + 2] = t1.x;
              o[r][4 * g + 3] = t1.y;
            }
          }
        }
      } else {
        for (int y = 0; y < kKeys; ++y) {
#pragma unroll
          for (int r = 0; r < RM; ++r) {
            if (key0 + y >= sees[r]) continue;
            const float w = ps[y * C::QS + ty * RM + r];
#pragma unroll
            for (int c = 0; c < 4 * NC; ++c) o[r][c] = fmaf(w, vs[y * HD + (c >> 2) * 64 + 4 * tx + (c & 3)], o[r][c]);
          }
        }
      }
    }

#pragma unroll
    for (int r = 0; r < RM; ++r) {
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
      if (m[r] == -INFINITY && l[r] != l[r]) m[r] = 0.0f;  // every score it saw was NaN
    }
    const bool whole = s.whole;
    const int64_t part = (int64_t)blockIdx.x * 2 + s.part;
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      const int row = ty * RM + r, token = row / p.group, head = row - token * p.group;
      if (token >= tokens) continue;
      if (whole) {
        const float inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
        float* dst = p.out + (s.row0 + (int64_t)token) * p.out_row + (int64_t)(s.h * p.group + head) * p.out_head;
#pragma unroll
        for (int g = 0; g < NC; ++g) {
          const int d = g * 64 + 4 * tx;
          if (d < p.head_dim)
            *reinterpret_cast<float4*>(dst + d) = make_float4(o[r][4 * g] * inv, o[r][4 * g + 1] * inv,
                                                              o[r][4 * g + 2] * inv, o[r][4 * g + 3] * inv);
        }
      } else {
        float* dst = p.partials + (part * C::BM + row) * HD;
#pragma unroll
        for (int g = 0; g < NC; ++g)
          __stcg(reinterpret_cast<float4*>(dst + g * 64 + 4 * tx),
                 make_float4(o[r][4 * g], o[r][4 * g + 1], o[r][4 * g + 2], o[r][4 * g + 3]));
        if (tx == 0) __stcg(p.part_ml + part * C::BM + row, make_float2(m[r], l[r]));
      }
    }
    if (!whole) {
      __syncthreads();
      if (tid == 0) ticket = ticket_acq_rel(p.counters + s.c_first);
      __syncthreads();
      if (ticket == (unsigned)(s.c_last - s.c_first)) join_parts_f32<HD, C::BM, kThreads>(p, s);
    }
  }
}

// ---- few rows: one token, or a few, over a cache ------------------------------------
//
// A tile of up to R rows (one token's group of heads, as a rule) needs 2 R products for each
// element of K and V, so the time is that of reading them. Eight lanes (16 for 128
// dimensions) share a key, eight dimensions each, with the rows of q in registers: four
// keys' K and V (eight of bf16) are loaded together and used straight from the registers,
// without shared memory or barriers. Every such group of lanes keeps its own maximum, sum and output; they
// are joined when the CTA's run of the tile ends. 32 requests of 1500 tokens, 12 heads of 64,
// take 56 us on a B200: 5.2 TB/s. With a bf16 cache, where q and the weights stay in fp32, the
// instructions for each element weigh twice as much: 64 requests of 2000 tokens take 91 us,
// 4.3 TB/s; with four keys of bf16 together 8 % more.
template <typename T>
struct Eight {  // dimensions of a row, as they are read
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (uint4& x : u) x = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void load(const T* src) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4*>(src)[i];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[4 * i] = __uint_as_float(u[i].x), x[4 * i + 1] = __uint_as_float(u[i].y);
        x[4 * i + 2] = __uint_as_float(u[i].z), x[4 * i + 3] = __uint_as_float(u[i].w);
      }
    } else {
      const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

template <int HD, int R, typename T>
struct Few {
  static constexpr int LANES = HD / 8;             // of a key
  static constexpr int KEYS = sizeof(T) == 4 ? 4 : 8;  // of a lane, loaded together (as many bytes)
  static constexpr int BLOCK = kThreads / LANES * KEYS;
  static constexpr int CTAS = R <= 2 ? 2 : 1;
};

// T: of k, v and out; TQ: of q.
template <int HD, int R, bool PAGED, typename T, typename TQ>
__global__ void __launch_bounds__(kThreads, Few<HD, R, T>::CTAS)
    attention_few_kernel(const __grid_constant__ F32Attention p) {
  using F = Few<HD, R, T>;
  constexpr int LANES = F::LANES, KEYS = F::KEYS;
  extern __shared__ float4 raw4[];
  float* joined = reinterpret_cast<float*>(raw4);  // [8 warps][R][HD], then their (m, l)
  float2* joined_ml = reinterpret_cast<float2*>(joined + 8 * R * HD);
  // the list's prefix lies where the rows are joined
  const StepList list = {reinterpret_cast<Request*>(joined + (8 * R * (HD + 2) > (MTRTQ_MAX_BATCH + 2) / 2 * 4 ? 8 * R * (HD + 2) : (MTRTQ_MAX_BATCH + 2) / 2 * 4)),
                         reinterpret_cast<int64_t*>(joined)};
  __shared__ Walk shared_walk;
  __shared__ Segment s;
  __shared__ int more;
  __shared__ unsigned ticket;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int d0 = lane % LANES * 8;             // this lane's dimensions
  const int mine = tid / LANES;                // and its first key of a block
  const bool in0 = d0 < p.head_dim;            // (head_dim is a multiple of 8)

  if (p.most != INT_MAX) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the call's second kernel
  Walk walk;
  make_list<F::BLOCK, kThreads>(p, list, walk, &shared_walk);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float c2 = p.scale * 1.4426950408889634f;  // scale log2 e

  while (true) {
    __syncthreads();
    if (tid == 0) more = next_segment<F::BLOCK>(p, list, walk, s);
    __syncthreads();
    if (!more) break;
    const int64_t r0 = s.r0;
    const int tokens = s.tokens, keys = s.keys, rows = tokens * p.group;
    float q[R][8], o[R][8], m[R], l[R];
    int sees[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int token = r / p.group, head = r - token * p.group;
      Eight<TQ> x;
      x.zero();
      if (r < rows && in0)
        x.load(reinterpret_cast<const TQ*>(p.q) + (s.row0 + (int64_t)token) * p.q_row + (int64_t)(s.h * p.group + head) * p.q_head + d0);
      x.get(q[r]);
      sees[r] = r < rows ? max(0, min(s.see0 + token, keys)) : 0;
      m[r] = -INFINITY;
      l[r] = 0.0f;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[r][d] = 0.0f;
    }
    const int k1 = s.k0 + s.n;
    for (int j = s.k0; j < k1; ++j) {
      Eight<T> k[KEYS], v[KEYS];
#pragma unroll
      for (int c = 0; c < KEYS; ++c) {
        const int key = j * F::BLOCK + c * (kThreads / LANES) + mine;
        k[c].zero();
        v[c].zero();
        if (key < keys && in0) {
          const T *ks = reinterpret_cast<const T*>(p.k), *vs = reinterpret_cast<const T*>(p.v);
          bool there = true;
          if (PAGED) {
            const int64_t page = p.table[s.b * p.table_ld + key / p.page_size];
            there = page >= 0 && page < p.num_pages;  // else the token reads as zeros
            const int64_t at = ((int64_t)s.h * p.page_size + key % p.page_size) * p.head_dim + d0;
            ks += page * p.k_row + at;
            vs += page * p.v_row + at;
          } else {
            ks += (r0 + key) * p.k_row + s.h * p.k_head + d0;
            vs += (r0 + key) * p.v_row + s.h * p.v_head + d0;
          }
          if (there) {
            k[c].load(ks);
            v[c].load(vs);
          }
        }
      }
      float e[R][KEYS];
#pragma unroll
      for (int c = 0; c < KEYS; ++c) {
        float y[8];
        k[c].get(y);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float x = q[r][0] * y[0];
#pragma unroll
          for (int d = 1; d < 8; ++d) x = fmaf(q[r][d], y[d], x);
#pragma unroll
          for (int w = LANES / 2; w > 0; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
          e[r][c] = x;
        }
      }
      float base[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float top = m[r];
#pragma unroll
        for (int c = 0; c < KEYS; ++c)
          if (j * F::BLOCK + c * (kThreads / LANES) + mine < sees[r]) top = fmaxf(top, e[r][c] * c2);
        base[r] = top == -INFINITY ? 0.0f : top;
        const float keep = m[r] == -INFINITY ? 1.0f : ex2(m[r] - base[r]);
        m[r] = top;
        l[r] *= keep;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[r][d] *= keep;
      }
#pragma unroll
      for (int c = 0; c < KEYS; ++c) {
        float y[8];
        v[c].get(y);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          // a key that the row does not see adds nothing, whatever its v
          if (j * F::BLOCK + c * (kThreads / LANES) + mine >= sees[r]) continue;
          const float w = ex2(fmaf(e[r][c], c2, -base[r]));
          l[r] += w;
#pragma unroll
          for (int d = 0; d < 8; ++d) o[r][d] = fmaf(w, y[d], o[r][d]);
        }
      }
    }
    // The groups of a warp, then the warps.
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (m[r] == -INFINITY && l[r] != l[r]) m[r] = 0.0f;  // every score it saw was NaN
#pragma unroll
      for (int w = LANES; w < 32; w <<= 1) {
        const float m1 = __shfl_xor_sync(0xffffffffu, m[r], w), l1 = __shfl_xor_sync(0xffffffffu, l[r], w);
        const float top = fmaxf(m[r], m1);
        // both lanes of a pair form the same sum
        const float a = m[r] == -INFINITY ? 0.0f : top == INFINITY ? 1.0f : ex2(m[r] - top);
        const float b = m1 == -INFINITY ? 0.0f : top == INFINITY ? 1.0f : ex2(m1 - top);
        const bool low = (lane & w) == 0;
        l[r] = low ? l[r] * a + l1 * b : l1 * b + l[r] * a;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const float x = o[r][d] * a, y = __shfl_xor_sync(0xffffffffu, o[r][d], w) * b;
          o[r][d] = low ? x + y : y + x;
        }
        m[r] = top;
      }
      if (lane < LANES) {
        float* dst = joined + (warp * R + r) * HD + d0;
        *reinterpret_cast<float4*>(dst) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(o[r][4], o[r][5], o[r][6], o[r][7]);
        if (lane == 0) joined_ml[warp * R + r] = make_float2(m[r], l[r]);
      }
    }
    __syncthreads();
    const bool whole = s.whole;
    const int64_t part = (int64_t)blockIdx.x * 2 + s.part;
    for (int e = tid; e < rows * (HD / 4); e += kThreads) {
      const int row = e / (HD / 4), d = e % (HD / 4) * 4, token = row / p.group, head = row - token * p.group;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) top = fmaxf(top, joined_ml[w * R + row].x);
      float4 x = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const float2 ml = joined_ml[w * R + row];
        const float a = ml.x == -INFINITY ? 0.0f : top == INFINITY ? 1.0f : ex2(ml.x - top);
        const float4 y = *reinterpret_cast<const float4*>(joined + (w * R + row) * HD + d);
        sum = fmaf(ml.y, a, sum);
        x.x = fmaf(y.x, a, x.x);
        x.y = fmaf(y.y, a, x.y);
        x.z = fmaf(y.z, a, x.z);
        x.w = fmaf(y.w, a, x.w);
      }
      if (whole) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (d < p.head_dim)
          put4(reinterpret_cast<T*>(p.out) + (s.row0 + (int64_t)token) * p.out_row +
                   (int64_t)(s.h * p.group + head) * p.out_head + d,
               make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
      } else {
        __stcg(reinterpret_cast<float4*>(p.partials + (part * R + row) * HD + d), x);
        if (d == 0) __stcg(p.part_ml + part * R + row, make_float2(top, sum));
      }
    }
    if (!whole) {
      __syncthreads();
      if (tid == 0) ticket = ticket_acq_rel(p.counters + s.c_first);
      __syncthreads();
      if (ticket == (unsigned)(s.c_last - s.c_first)) join_parts_f32<HD, R, kThreads, T>(p, s);
    }
  }
}

cudaError_t launch(void (*kernel)(F32Attention), const F32Attention& p, int bytes, int grid, bool pdl, cudaStream_t st) {
  if (cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kernel),
                                        bytes + MTRTQ_MAX_BATCH * (int)sizeof(Request)))
    return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes + p.batch * sizeof(Request);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int HD, int RM, bool PAGED>
cudaError_t launch_tile(const F32Attention& p, int grid, bool pdl, cudaStream_t st) {
  using C = Cfg<HD, RM>;
  static_assert(C::BYTES + MTRTQ_MAX_BATCH * (int)sizeof(Request) + 3 * 1024 <= 227 * 1024 &&
                    C::BYTES >= (MTRTQ_MAX_BATCH + 1) * 8, "shared memory per CTA");
  return launch(attention_f32_kernel<HD, RM, PAGED>, p, C::BYTES, grid, pdl, st);
}

template <int HD, int R, bool PAGED>
cudaError_t launch_few(const F32Attention& p, int grid, bool pdl, cudaStream_t st) {
  const int bytes = 8 * R * (HD * 4 + 8), prefix = (MTRTQ_MAX_BATCH + 2) / 2 * 16;
  const int all = bytes > prefix ? bytes : prefix;
  if constexpr (PAGED && R <= 2) {
    using bf16 = __nv_bfloat16;
    if (p.pages16 && p.q16) return launch(attention_few_kernel<HD, R, true, bf16, bf16>, p, all, grid, pdl, st);
    if (p.pages16) return launch(attention_few_kernel<HD, R, true, bf16, float>, p, all, grid, pdl, st);
  }
  return launch(attention_few_kernel<HD, R, PAGED, float, float>, p, all, grid, pdl, st);
}

template <int HD, bool PAGED>
cudaError_t launch_rows(const F32Attention& p, int grid, bool pdl, cudaStream_t st) {
  switch (p.tile_rows) {
    case 1: return launch_few<HD, 1, PAGED>(p, grid, pdl, st);
    case 2: return launch_few<HD, 2, PAGED>(p, grid, pdl, st);
    case 4: return launch_few<HD, 4, PAGED>(p, grid, pdl, st);
    case 8: return launch_few<HD, 8, PAGED>(p, grid, pdl, st);
    case 16: return launch_tile<HD, 1, PAGED>(p, grid, pdl, st);
    case 64: return launch_tile<HD, 4, PAGED>(p, grid, pdl, st);
    default: return launch_tile<HD, 8, PAGED>(p, grid, pdl, st);
  }
}

}  // namespace

cudaError_t launch_attention_f32(const F32Attention& p, int grid, bool pdl, cudaStream_t st) {
  if (p.head_dim <= 64)
    return p.table ? launch_rows<64, true>(p, grid, pdl, st) : launch_rows<64, false>(p, grid, pdl, st);
  return p.table ? launch_rows<128, true>(p, grid, pdl, st) : launch_rows<128, false>(p, grid, pdl, st);
}

}  // namespace mtrtq
