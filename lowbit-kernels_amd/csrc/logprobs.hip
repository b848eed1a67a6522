// Log probabilities of given tokens with the entropy and the most likely alternatives of each row of logits (token_logprobs), and
// the best continuations of several beams, which are chosen from the same (beam_select).
//
// A row is read once from memory. Every lane keeps, against its largest logit so far r, z = sum exp(x - r) and e = sum exp(x -
// r) (x - r); when all is read, the sums are moved to the row's maximum m: log p(t) = (x_t - m) - log z, H = log z - e / z.
// Every term of e, and what a move to a larger reference adds, is 0 or below, so nothing cancels (a reference that lags 16
// behind the maximum saves instructions and cost entropies up to 4e-5). Differences from a logit, not products with log2(e),
// are what is rounded, so rows far from zero (or at the type's lowest value throughout) lose nothing.
// The alternatives: the `top`-th largest of the lanes' maxima is a bound that `top` logits at least reach, and almost no other
// does; the maxima of the groups of vectors that each lane has read (kept in LDS) say which groups hold such logits, and only
// those are read again (from L2). What reaches the bound is ranked by counting.
// Where there are few rows, each is cut into slices of one workgroup, whose sums and alternatives a second launch joins.
#include <algorithm>
#include <cfloat>
#include <climits>

#include "kernels.hpp"

namespace lowbit {

namespace {

typedef __bf16 bf16;

constexpr int kThreads = 512;
constexpr int kUnroll = 4;               // 16-byte vectors of a lane in flight
constexpr int kGroups = 16;              // groups of vectors a lane keeps the maxima of
constexpr int kList = 1024;              // logits that may reach the bound on the fast path
constexpr int kMaxSlices = 64;

// (value, index) as one number, larger = earlier among the alternatives: the larger value (-0 equal to +0, a NaN above
// every number, as torch orders them), then the smaller index. Zero is below every key.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
  return x != x ? 0xFFFFFFFFu : (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __builtin_bit_cast(float, (k >> 31) ? (k & 0x7FFFFFFFu) : ~k);
}
__device__ __forceinline__ uint64_t rank_key(float x, int idx) {
  return ((uint64_t)order_key(x) << 32) | (uint32_t)(0x7FFFFFFF - idx);
}
__device__ __forceinline__ int rank_index(uint64_t key) { return 0x7FFFFFFF - (int)(uint32_t)key; }

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* red, Op op) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = op(v, __shfl_xor(v, off, 64));
  const int wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[wave] = v;
  __syncthreads();
  V t = red[0];
  for (int i = 1; i < nw; ++i) t = op(t, red[i]);
  return t;
}

// this wave's LDS writes so far come before its later reads (one wave: no barrier is needed)
__device__ __forceinline__ void lds_wave_order() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <typename T>
__device__ __forceinline__ float value(const u32x4& v, int i) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t w = v[i];                                  // (a bit cast of the element itself reads the first one)
    return __builtin_bit_cast(float, w);
  } else {
    const uint32_t w = v[i >> 1];
    if constexpr (__is_same(T, f16)) return (float)as_f16x2(w)[i & 1];
    return __builtin_bit_cast(float, i & 1 ? w & 0xFFFF0000u : w << 16);
  }
}
// bits of order_key that tell two values of T apart, from the top
template <typename T>
constexpr int key_bits() { return sizeof(T) == 4 ? 32 : __is_same(T, f16) ? 19 : 16; }

// a part's sums: maximum, z and e against it
struct Sums {
  float m, z, e;
};
// (z, e) moved from reference r to m >= r; r = -inf: nothing above it was seen, both are 0 (the difference is held above
// -inf, so that sums that vanish beside m vanish)
__device__ __forceinline__ void move_sums(float r, float m, float& z, float& e) {
  const float d = r == -INFINITY ? 0.f : fmaxf(r - m, -1e4f), f = __expf(d);
  e = f * fmaf(d, z, e);
  z *= f;
}

}  // namespace

// the row's two results from its whole sums, by one thread; false where the row has no distribution
template <typename T>
__device__ __forceinline__ void store_sums(const T* x, int V, int64_t t, const Sums& s, float* logprob, float* entropy) {
  const bool none = !(s.m > -INFINITY && s.m < INFINITY) || s.z != s.z;
  const float lz = logf(s.z);
  *logprob = t < 0 ? 0.f : none || t >= V ? NAN : ((float)x[t] - s.m) - lz;
  *entropy = none ? NAN : lz - s.e / s.z;
}

// Workgroup (row, slice): see the top of the file. part (S > 1, or beams): [row][slice] Sums, then keys [row][slice][top].
// kBeam: the rows of beams, scores theirs, by which one that holds nothing or is finished is not read; no entropy is summed, and
// the maxima kept are each vector's, so that of a group only the vectors that may reach the bound are read again (64 x 8 beams of
// 151936 in fp16, 16 alternatives: 42.6 us without, 35.8 so, 4.3 TB/s).
// Bound: memory, 2047 rows of 151665 in fp16 (621 MB) 126 us, 4.9 TB/s; of few rows the chain of load, sums, bound, reread and
// join: 48 rows of 151936 in fp32 18 us, one in fp16 13.
template <typename T, bool kBeam>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(const T* __restrict__ logits, int64_t stride,
                                                            const int64_t* __restrict__ targets,
                                                            float* __restrict__ logprob, float* __restrict__ entropy,
                                                            float* __restrict__ top_value, int64_t* __restrict__ top_id,
                                                            int V, int top, int S, Sums* __restrict__ part,
                                                            uint64_t* __restrict__ part_keys,
                                                            const float* __restrict__ scores,
                                                            const uint8_t* __restrict__ finished) {
  constexpr int kN = 16 / sizeof(T);
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  float* s_max = reinterpret_cast<float*>(smem);              // [group][thread]
  uint2* s_max4 = reinterpret_cast<uint2*>(smem);             // kBeam: the same of four vectors, the upper halves of their keys
  __shared__ uint64_t s_list[kList];
  __shared__ Sums s_sums[kThreads / 64];
  __shared__ uint64_t s_redk[kThreads / 64];
  __shared__ int s_wave[kThreads / 64];
  __shared__ float s_lane[kThreads];
  __shared__ int s_count;
  __shared__ uint32_t s_bound;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x / S;
  const int slice = blockIdx.x % S;
  const bool parts = kBeam || S > 1;
  if (kBeam && (!(fabsf(scores[row]) <= FLT_MAX) || (finished && finished[row]))) return;
  const T* x = logits + row * stride;
  // the row's 16-byte vectors, after a head and before a tail of single logits, which slice 0 and the last slice take
  const int head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
  const int nvec = (V - head) / kN, tail0 = head + nvec * kN;
  const int per = (nvec + S - 1) / S, v0 = min(nvec, slice * per), v1 = min(nvec, v0 + per);
  const T* body = x + head;
  const int steps = (v1 - v0 + kThreads * kUnroll - 1) / (kThreads * kUnroll), every = (steps + kGroups - 1) / kGroups;
  const int single = slice == 0 && tid < head ? tid : slice == S - 1 && tail0 + (int)tid - 16 < V && tid >= 16 ? tail0 + tid - 16 : -1;

  float r = -INFINITY, z = 0.f, e = 0.f;
  auto raise = [&](float v) {                                 // the lane's reference, to v where that is larger
    if (v > r) {
      move_sums(r, v, z, e);
      r = v;
    }
  };
  auto add = [&](float v, float ref) {                        // (p d with d held above -inf: 0 log 0 = 0)
    const float d = v - ref, p = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
    z += p;
    if constexpr (!kBeam) e = fmaf(p, fmaxf(d, -1e4f), e);
  };
  const int64_t end = (int64_t)(v1 - v0);
  float gm = -INFINITY;
  [[maybe_unused]] float gv[kUnroll] = {};
  for (int step = 0; step < steps; ++step) {
    u32x4 v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = (int64_t)(step * kUnroll + u) * kThreads + tid;
      v[u] = i < end ? load_stream(body + (v0 + i) * kN) : u32x4{0u, 0u, 0u, 0u};
    }
    float vm[kUnroll], sm = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      vm[u] = value<T>(v[u], 0);
#pragma unroll
      for (int i = 1; i < kN; ++i) vm[u] = fmaxf(vm[u], value<T>(v[u], i));
      if ((int64_t)(step * kUnroll + u) * kThreads + tid >= end) vm[u] = -INFINITY;
      sm = fmaxf(sm, vm[u]);
    }
    raise(sm);
    const float ref = r == -INFINITY ? 0.f : r;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if ((int64_t)(step * kUnroll + u) * kThreads + tid < end) {
#pragma unroll
        for (int i = 0; i < kN; ++i) add(value<T>(v[u], i), ref);
      }
    if constexpr (kBeam) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) gv[u] = step % every == 0 ? vm[u] : fmaxf(gv[u], vm[u]);
      static_assert(kUnroll == 4, "the maxima of a group");
      s_max4[step / every * kThreads + tid] = make_uint2(order_key(gv[0]) >> 16 | (order_key(gv[1]) & 0xFFFF0000u),
                                                         order_key(gv[2]) >> 16 | (order_key(gv[3]) & 0xFFFF0000u));
    } else {
      gm = step % every == 0 ? sm : fmaxf(gm, sm);
      s_max[step / every * kThreads + tid] = gm;
    }
  }
  if (single >= 0) {
    const float v = (float)x[single];
    raise(v);
    add(v, r == -INFINITY ? 0.f : r);
  }
  // the wave's sums against its maximum, then the workgroup's, added by every thread in order of the waves
  Sums s;
  s.m = wave_max(r);
  move_sums(r, s.m, z, e);
  s.z = wave_sum(z);
  s.e = wave_sum(e);
  if (lane == 0) s_sums[tid >> 6] = s;
  s_lane[tid] = r;
  if (tid == 0) s_count = 0;
  __syncthreads();
  s = s_sums[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) s.m = fmaxf(s.m, s_sums[w].m);
  s.z = s.e = 0.f;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    Sums o = s_sums[w];
    move_sums(o.m, s.m, o.z, o.e);
    s.z += o.z;
    s.e += o.e;
  }
  if (tid == 0) {
    if (!parts)
      store_sums(x, V, targets[row], s, logprob + row, entropy + row);
    else
      part[blockIdx.x] = s;
  }
  if (top == 0) return;

  // ---- the alternatives ----
  const bool none = !(s.m > -INFINITY && s.m < INFINITY) || s.z != s.z;
  const float lz = logf(s.z);
  auto give = [&](int rank, uint64_t key) {                   // by the thread that holds it
    if (parts) {
      part_keys[(int64_t)blockIdx.x * top + rank] = key;
    } else {
      const int idx = rank_index(key);
      top_id[row * top + rank] = idx;
      top_value[row * top + rank] = none ? NAN : ((float)x[idx] - s.m) - lz;
    }
  };
  const int held = (v1 - v0) * kN + (slice == 0 ? head : 0) + (slice == S - 1 ? V - tail0 : 0);   // logits of the slice
  // the bound: the top-th largest of 64 maxima, each of the threads of one lane number, found bit by bit by the first wave
  // (of 512 maxima it would be a little higher and leave 20 .. 35 logits, not 24 .. 45, but take 8 compares a bit)
  if (tid < 64) {
    float m = s_lane[lane];
#pragma unroll
    for (int i = 1; i < kThreads / 64; ++i) m = fmaxf(m, s_lane[64 * i + lane]);
    const uint32_t k = order_key(m);
    uint32_t bound = 0;
#pragma unroll
    for (int bit = 31; bit >= 32 - key_bits<T>(); --bit) {
      const uint32_t trial = bound | (1u << bit);
      if (__popcll(__ballot(k >= trial)) >= top) bound = trial;
    }
    if (key_bits<T>() < 32 && !(bound >> 31)) bound |= (1u << (32 - key_bits<T>())) - 1u;   // (negative: the bits are ones)
    if (lane == 0) s_bound = bound;
  }
  __syncthreads();
  const float bound = order_value(s_bound);
  auto push = [&](float v, int idx) {
    const int at = atomicAdd(&s_count, 1);
    if (at < kList) s_list[at] = rank_key(v, idx);
  };
  auto collect = [&](bool above) {                            // what reaches the bound, or passes it
    for (int g = 0; g * every < steps; ++g) {
      uint32_t may = (1u << kUnroll) - 1u;                    // vectors of a step that may hold such logits
      if constexpr (kBeam) {
        const uint2 k = s_max4[g * kThreads + tid];
        const uint32_t b = s_bound >> 16;
        may = ((k.x & 0xFFFFu) >= b ? 1u : 0u) | (k.x >> 16 >= b ? 2u : 0u) | ((k.y & 0xFFFFu) >= b ? 4u : 0u) | (k.y >> 16 >= b ? 8u : 0u);
        if (!may) continue;
      } else if (!(s_max[g * kThreads + tid] >= bound)) {
        continue;
      }
      for (int step = g * every; step < min(steps, (g + 1) * every); ++step) {
        u32x4 v[kUnroll];                                     // (asked for at once)
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int64_t i = (int64_t)(step * kUnroll + u) * kThreads + tid;
          if (i < end && (may >> u & 1u)) v[u] = load16(body + (v0 + i) * kN);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int64_t i = (int64_t)(step * kUnroll + u) * kThreads + tid;
          if (i >= end || !(may >> u & 1u)) continue;
#pragma unroll
          for (int k = 0; k < kN; ++k) {
            const float f = value<T>(v[u], k);
            if (above ? f > bound : f >= bound) push(f, head + (int)(v0 + i) * kN + k);
          }
        }
      }
    }
    if (single >= 0) {
      const float f = (float)x[single];
      if (above ? f > bound : f >= bound) push(f, single);
    }
  };
  bool by_rounds = s.z != s.z || s.m == INFINITY;             // NaN and +inf among the logits: ordered by rounds below
  if (!by_rounds) {
    collect(false);
    __syncthreads();
    int n = s_count;
    __syncthreads();
    if (n > kList) {
      // many equal to the bound (ties, banned tokens at -inf), or many above it in few lanes (sorted rows)
      if (tid == 0) s_count = 0;
      __syncthreads();
      collect(true);
      __syncthreads();
      n = s_count;
      __syncthreads();
      by_rounds = n > kList;
      if (!by_rounds && n < top) {
        // those above, and of the equal ones the first in order of index until there are `top`
        auto in_order = [&](int mine, auto idx_of) {          // the thread's `mine` (a bit mask) come before the next thread's
          const int c = __popc(mine);
          int upto = c;
#pragma unroll
          for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(upto, off, 64);
            if (lane >= off) upto += o;
          }
          if (lane == 63) s_wave[tid >> 6] = upto;
          __syncthreads();
          int at = n + upto - c, all = n;
          for (int w = 0; w < kThreads / 64; ++w) {
            if (w < (tid >> 6)) at += s_wave[w];
            all += s_wave[w];
          }
          for (int bits = mine; bits && at < top; bits &= bits - 1, ++at) s_list[at] = rank_key(bound, idx_of(__ffs(bits) - 1));
          __syncthreads();
          n = all;
        };
        if (slice == 0 && head > 0) in_order(tid < head && (float)x[tid] == bound ? 1 : 0, [&](int) { return tid; });
        for (int64_t i0 = 0; i0 < end && n < top; i0 += kThreads) {
          int mask = 0;
          if (i0 + tid < end) {
            const u32x4 v = load16(body + (v0 + i0 + tid) * kN);
#pragma unroll
            for (int k = 0; k < kN; ++k) mask |= value<T>(v, k) == bound ? 1 << k : 0;
          }
          in_order(mask, [&](int k) { return head + (int)(v0 + i0 + tid) * kN + k; });
        }
        if (slice == S - 1 && n < top && tail0 < V)
          in_order(tail0 + tid < V && (float)x[tail0 + tid] == bound ? 1 : 0, [&](int) { return tail0 + tid; });
        n = min(n, top);
      }
    }
    if (!by_rounds) {
      for (int i = tid; i < n; i += kThreads) {
        const uint64_t key = s_list[i];
        int rank = 0;
#pragma unroll 8
        for (int k = 0; k < n; ++k) rank += s_list[k] > key;
        if (rank < top) give(rank, key);
      }
      if (parts)                                              // a slice of fewer logits than `top`
        for (int i = min(n, held) + tid; i < top; i += kThreads) give(i, 0);
      return;
    }
  }
  // each the largest key below the one before
  uint64_t below = ~(uint64_t)0;
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    auto offer = [&](float v, int idx) {
      const uint64_t key = rank_key(v, idx);
      if (key < below && key > best) best = key;
    };
    for (int64_t i = tid; i < end; i += kThreads) {
      const u32x4 v = load16(body + (v0 + i) * kN);
#pragma unroll
      for (int j = 0; j < kN; ++j) offer(value<T>(v, j), head + (int)(v0 + i) * kN + j);
    }
    if (single >= 0) offer((float)x[single], single);
    below = block_reduce(best, s_redk, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
    if (tid == 0) give(k, below);                             // (of parts: 0 where the slice has no more)
  }
}

// One workgroup per row, whose first wave joins the slices' sums and alternatives.
template <typename T>
__global__ __launch_bounds__(256) void logprobs_join_kernel(const T* __restrict__ logits, int64_t stride,
                                                           const int64_t* __restrict__ targets,
                                                           float* __restrict__ logprob, float* __restrict__ entropy,
                                                           float* __restrict__ top_value, int64_t* __restrict__ top_id,
                                                           int V, int top, int S, const Sums* __restrict__ part,
                                                           const uint64_t* __restrict__ part_keys) {
  __shared__ uint64_t s_keys[kMaxSlices * kMaxTop], s_list[kMaxSlices * kMaxTop];
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * stride;
  const uint64_t* keys = part_keys + row * S * top;
  for (int i = threadIdx.x; i < S * top; i += 256) s_keys[i] = keys[i];
  __syncthreads();
  if (threadIdx.x >= 64) return;
  Sums s = lane < S ? part[row * S + lane] : Sums{-INFINITY, 0.f, 0.f};
  const float m = wave_max(s.m);
  move_sums(s.m, m, s.z, s.e);
  s.m = m;
  s.z = wave_sum(s.z);
  s.e = wave_sum(s.e);
  if (lane == 0) store_sums(x, V, targets[row], s, logprob + row, entropy + row);
  const bool none = !(s.m > -INFINITY && s.m < INFINITY) || s.z != s.z;
  const float lz = logf(s.z);
  if (top == 0) return;
  // the top-th largest of the slices' first alternatives bounds the row's: those of each slice's list down to it are ranked by
  // counting
  const uint64_t first = lane < S ? s_keys[lane * top] : 0;
  int above = 0;
  for (int l = 0; l < S; ++l) above += s_keys[l * top] > first;
  const uint64_t at_bound = __ballot(lane < S && above == top - 1);   // (keys are distinct; none where S < top)
  const uint64_t bound = at_bound ? s_keys[__builtin_ctzll(at_bound) * top] : 0;
  int mine = 0;
  if (lane < S)
    while (mine < top && s_keys[lane * top + mine] >= max(bound, (uint64_t)1)) ++mine;
  int upto = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(upto, off, 64);
    if (lane >= off) upto += o;
  }
  for (int i = 0; i < mine; ++i) s_list[upto - mine + i] = s_keys[lane * top + i];
  const int n = __shfl(upto, 63, 64);
  lds_wave_order();
  for (int i = lane; i < n; i += 64) {
    const uint64_t key = s_list[i];
    int rank = 0;
    for (int k = 0; k < n; ++k) rank += s_list[k] > key;
    if (rank >= top) continue;
    const int idx = rank_index(key);
    top_id[row * top + rank] = idx;
    top_value[row * top + rank] = none ? NAN : ((float)x[idx] - s.m) - lz;
  }
}

// ---- beam_select ----
// A workgroup per request. The slices' sums are joined, 16 lanes a beam; a candidate's score is then score + (x - max) - log z, in 64
// bits (which of two beams' tokens comes first goes by that difference). The n-th largest of 64 maxima, each of some of the slices'
// first scores, bounds what can be among the n best: of all slices' lists what reaches it is ranked by counting, a few lanes a
// candidate. Where that is too little (few beams hold anything) or too much (ties), each beam's own n best are made first, a
// wave a beam, and those ranked.
// Bound: its chain of round trips and barriers, 4.8 (1 x 4 beams) .. 5.8 us (64 x 8).
// A beam that holds nothing (a score that is no finite number) or whose row has no distribution has -inf for every token, a
// finished one its score for `pad` and -inf for the others; equal candidates rank by beam, then by token.
constexpr int kBeamSlices = 16, kBeamThreads = 512;
constexpr int kBeamList = 1024;
constexpr int kBeamWhole = 128 * 1024;   // LDS of the lists of whole beams
struct BeamJoin {
  const float* scores;
  const uint8_t* finished;
  float* out_scores;
  int64_t *out_beams, *out_tokens;
  int W, V, n, pad, S, depth;                                 // depth: of each slice's list, scores that the bound is taken of
  const Sums* part;
  const uint64_t* keys;
};

// each beam's n best, then the n best of those
__device__ __forceinline__ void beam_join_whole(const BeamJoin& a, uint8_t* smem, int req) {
  const int W = a.W, V = a.V, n = a.n, S = a.S, pad = a.pad;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int have = min(n, V);                                 // candidates of a beam
  double* s_value = reinterpret_cast<double*>(smem);          // [W][have]
  int* s_token = reinterpret_cast<int*>(s_value + W * n);     // (rounded up to a multiple of two)
  uint64_t* s_all = reinterpret_cast<uint64_t*>(s_token + ((W * n + 1) & ~1));
  const int waves = max(1, min(kBeamThreads / 64, (kBeamWhole - W * n * 12 - 8) / (16 * S * n)));   // as many as LDS holds the lists of
  uint64_t *s_keys = s_all + wave * 2 * S * n, *s_list = s_keys + S * n;
  for (int w = wave; w < W && wave < waves; w += waves) {
    const int64_t row = (int64_t)req * W + w;
    const uint64_t* keys = a.keys + row * S * n;
    const float score = a.scores[row];
    const uint8_t flag = a.finished ? a.finished[row] : 0;
    Sums s = lane < S ? a.part[row * S + lane] : Sums{-INFINITY, 0.f, 0.f};   // (of a row that was not read: not used)
    for (int i = lane; i < S * n; i += 64) s_keys[i] = keys[i];
    const bool held = fabsf(score) <= FLT_MAX, done = held && flag;
    bool none = !held;
    if (held && !done) {
      const float m = wave_max(s.m);
      move_sums(s.m, m, s.z, s.e);
      const float z = wave_sum(s.z);
      none = !(m > -INFINITY && m < INFINITY) || z != z;
      lds_wave_order();
      if (!none) {
        uint64_t bound;
        if (S >= n) {
          const uint64_t first = lane < S ? s_keys[lane * n] : 0;
          int above = 0;
#pragma unroll 8
          for (int l = 0; l < S; ++l) above += s_keys[l * n] > first;
          bound = s_keys[__builtin_ctzll(__ballot(lane < S && above == n - 1)) * n];   // (first keys are distinct)
        } else {
          const int at = (n + S - 1) / S - 1;
          bound = lane < S ? s_keys[lane * n + at] : ~(uint64_t)0;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) bound = min(bound, (uint64_t)__shfl_xor((unsigned long long)bound, off, 64));   // (S < n <= 32)
          bound = __shfl((unsigned long long)bound, 0, 64);
        }
        if (bound == 0) bound = 1;                            // (slices with fewer logits end in zeros)
        int all = 0;
        for (int i0 = 0; i0 < S * n; i0 += 64) {
          const uint64_t key = i0 + lane < S * n ? s_keys[i0 + lane] : 0;
          const uint64_t in = __ballot(key >= bound);
          if (key >= bound) s_list[all + __popcll(in & (((uint64_t)1 << lane) - 1))] = key;
          all += __popcll(in);
        }
        lds_wave_order();
        const double at = (double)score - log((double)z);
        for (int i = lane; i < all; i += 64) {
          const uint64_t key = s_list[i];
          int rank = 0;
#pragma unroll 8
          for (int k = 0; k < all; ++k) rank += s_list[k] > key;
          if (rank >= have) continue;
          s_value[w * have + rank] = at + ((double)order_value((uint32_t)(key >> 32)) - (double)m);
          s_token[w * have + rank] = rank_index(key);
        }
      }
    }
    if (none || done) {
      for (int i = lane; i < have; i += 64) {
        s_value[w * have + i] = done && i == 0 ? (double)score : -INFINITY;
        s_token[w * have + i] = !done ? i : i == 0 ? pad : i - 1 < pad ? i - 1 : i;
      }
    }
  }
  __syncthreads();
  // a candidate's rank, counted by `per` lanes side by side
  const int all = W * have;
  int per = 1;
  while (per < 16 && 2 * per * all <= kBeamThreads) per *= 2;
  for (int c0 = 0; c0 < all; c0 += kBeamThreads / per) {
    const int c = c0 + (int)threadIdx.x / per;
    const double v = c < all ? s_value[c] : 0.0;
    int rank = 0;
#pragma unroll 4
    for (int k = (int)threadIdx.x % per; k < all; k += per) {
      const double o = s_value[k];
      rank += o > v || (o == v && k < c);
    }
    for (int off = 1; off < per; off <<= 1) rank += __shfl_xor(rank, off, 64);
    if (c >= all || rank >= n || (int)threadIdx.x % per) continue;
    const int64_t to = (int64_t)req * n + rank;
    a.out_scores[to] = (float)v;
    a.out_beams[to] = c / have;
    a.out_tokens[to] = s_token[c];
  }
}

// the sum, or the largest, over the 16 lanes of a row; every lane of the row gets it
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, dpp<kQuadSwap1>(v));
  v = fmaxf(v, dpp<kQuadSwap2>(v));
  v = fmaxf(v, dpp<kRowHalfMirror>(v));
  return fmaxf(v, dpp<kRowMirror>(v));
}

__global__ __launch_bounds__(kBeamThreads) void beam_join_kernel(BeamJoin a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ double s_at[kMaxBeams];                          // score - log z
  __shared__ float s_max[kMaxBeams];                          // the row's largest logit; NaN: no candidate but, perhaps, `pad`
  __shared__ double s_value[kBeamList];
  __shared__ uint64_t s_key[kBeamList];
  __shared__ int s_beam[kBeamList], s_count;
  const int W = a.W, n = a.n, S = a.S, req = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const uint64_t* keys = a.keys + (int64_t)req * W * S * n;
  const int lists = W * S, all = lists * n;
  // the first keys of the lists and the first four of the thread's, asked for before anything is known (of rows that were not
  // read: not used)
  constexpr int kFirst = kMaxBeams * 8 / 64, kAhead = 4;
  uint64_t first[kFirst], mine[kAhead];
  const int firsts = lists * a.depth;
#pragma unroll
  for (int i = 0; i < kFirst; ++i) {
    const int e = lane + 64 * i, l = (int)((uint32_t)e / (uint32_t)a.depth);
    first[i] = e < firsts ? keys[l * n + (e - l * a.depth)] : 0;
  }
#pragma unroll
  for (int i = 0; i < kAhead; ++i) mine[i] = tid + kBeamThreads * i < all ? keys[tid + kBeamThreads * i] : 0;
  if (tid == 0) s_count = 0;
  for (int w0 = 0; w0 < W; w0 += kBeamThreads / 16) {
    const int w = w0 + tid / 16, l = tid & 15;
    const int64_t row = (int64_t)req * W + min(w, W - 1);
    const float score = a.scores[row];
    const bool held = fabsf(score) <= FLT_MAX, done = held && a.finished && a.finished[row];
    Sums s = l < S ? a.part[row * S + l] : Sums{-INFINITY, 0.f, 0.f};
    const float m = row_max(s.m);
    move_sums(s.m, m, s.z, s.e);
    const float z = row_sum(s.z);
    const bool none = !held || done || !(m > -INFINITY && m < INFINITY) || z != z;
    const double at = (double)score - log((double)z);
    if (l == 0 && w < W) {
      s_at[w] = at;
      s_max[w] = none ? NAN : m;
    }
  }
  __syncthreads();
  // a finished beam's one candidate (key 0: none of a list has it)
  auto push = [&](bool in, double v, uint64_t key, int w) {
    const uint64_t vote = __ballot(in);
    if (!vote) return;
    int at = 0;
    if (lane == __builtin_ctzll(vote)) at = atomicAdd(&s_count, __popcll(vote));
    at = __builtin_amdgcn_readlane(at, __builtin_ctzll(vote)) + __popcll(vote & (((uint64_t)1 << lane) - 1));
    if (in && at < kBeamList) {
      s_value[at] = v;
      s_key[at] = key;
      s_beam[at] = w;
    }
  };
  auto value = [&](uint64_t key, int w) { return s_at[w] + ((double)order_value((uint32_t)(key >> 32)) - (double)s_max[w]); };
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kFirst; ++i) {
    const int e = lane + 64 * i;
    if (e >= firsts) break;
    const int w = (int)((uint32_t)e / (uint32_t)(S * a.depth));
    if (s_max[w] == s_max[w] && first[i]) top = fmaxf(top, (float)value(first[i], w));
  }
  const uint32_t k = order_key(top);
  uint32_t nth = 0;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t trial = nth | (1u << bit);
    if (__popcll(__ballot(k >= trial)) >= n) nth = trial;
  }
  // (as a float it may be a step above the score itself; -inf where too few lanes hold anything)
  const float f = order_value(nth);
  const double bound = f == -INFINITY ? -DBL_MAX : (double)f - fabs((double)f) * 0x1p-22 - 0x1p-140;
  for (int i0 = 0; i0 < all; i0 += kAhead * kBeamThreads) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = i0 + tid + kBeamThreads * i;
      if (i0 + kBeamThreads * i >= all) break;
      const uint64_t key = i0 == 0 ? mine[i] : at < all ? keys[at] : 0;
      const int w = min((int)((uint32_t)at / (uint32_t)(S * n)), W - 1);
      const bool live = key != 0 && s_max[w] == s_max[w];
      const double v = live ? value(key, w) : -INFINITY;
      push(live && v >= bound, v, key, w);
    }
  }
  if (tid < 64 && a.finished)
    for (int w0 = 0; w0 < W; w0 += 64) {
      const int w = min(w0 + lane, W - 1);
      const int64_t row = (int64_t)req * W + w;
      const float score = a.scores[row];
      push(w0 + lane < W && fabsf(score) <= FLT_MAX && a.finished[row], (double)score, 0, w);
    }
  __syncthreads();
  const int found = s_count;
  if (found < n || found > kBeamList) {                       // (uniform)
    beam_join_whole(a, smem, req);
    return;
  }
  int per = 1;                                                // lanes side by side that count a candidate's rank
  while (per < 16 && 2 * per * found <= kBeamThreads) per *= 2;
  for (int c0 = 0; c0 < found; c0 += kBeamThreads / per) {
    const int c = c0 + tid / per;
    const double v = c < found ? s_value[c] : 0.0;
    const uint64_t key = c < found ? s_key[c] : 0;
    const int w = c < found ? s_beam[c] : 0;
    int rank = 0;
#pragma unroll 4
    for (int i = tid % per; i < found; i += per) {
      const double o = s_value[i];
      rank += o > v || (o == v && (s_beam[i] < w || (s_beam[i] == w && s_key[i] > key)));
    }
    for (int off = 1; off < per; off <<= 1) rank += __shfl_xor(rank, off, 64);
    if (c >= found || rank >= n || tid % per) continue;
    const int64_t to = (int64_t)req * n + rank;
    a.out_scores[to] = (float)v;
    a.out_beams[to] = w;
    a.out_tokens[to] = key ? rank_index(key) : a.pad;
  }
}

// slices of at least 2048 logits: up to `most` a row and `all` workgroups
static int row_slices(int M, int V, int top, int most, int all, size_t ws_bytes) {
  const int S = std::min({all / M, V / 2048, most});
  const size_t per = (size_t)M * (sizeof(Sums) + 4 + (size_t)top * 8);
  return (int)std::max<size_t>(1, std::min<size_t>((size_t)std::max(S, 1), ws_bytes / per));
}
// LDS of a slice's group maxima
static size_t slice_lds(int V, int dtype, int S, size_t each_max) {
  const int each = dtype == 0 ? 4 : 8;                        // logits of a vector
  const int64_t vectors = (V / each + S - 1) / S, steps = (vectors + kThreads * kUnroll - 1) / (kThreads * kUnroll);
  return (size_t)std::max<int64_t>(1, std::min<int64_t>(steps, kGroups)) * kThreads * each_max;
}

hipError_t token_logprobs_launch(const LogprobArgs& a, hipStream_t st) {
  // (four workgroups a CU; rows whole from 512 on)
  const int S = a.ws && a.M < 512 ? row_slices(a.M, a.V, a.top, kMaxSlices, 1024, a.ws_bytes) : 1;
  const size_t lds = slice_lds(a.V, a.dtype, S, sizeof(float));
  uint64_t* keys = static_cast<uint64_t*>(a.ws);              // [M][S][top] keys, then [M][S] sums
  Sums* part = reinterpret_cast<Sums*>(keys + (size_t)a.M * S * a.top);
  auto go = [&](auto first, auto second, auto* p) {
    hipError_t e = launch(first, dim3((unsigned)((int64_t)a.M * S)), dim3(kThreads), lds, st, p, a.stride, a.targets, a.logprob,
                          a.entropy, a.top_value, a.top_id, a.V, a.top, S, part, keys, static_cast<const float*>(nullptr),
                          static_cast<const uint8_t*>(nullptr));
    if (e != hipSuccess || S == 1) return e;
    return launch(second, dim3((unsigned)a.M), dim3(256), 0, st, p, a.stride, a.targets, a.logprob, a.entropy, a.top_value,
                  a.top_id, a.V, a.top, S, part, keys);
  };
  if (a.dtype == 0) return go(logprobs_kernel<float, false>, logprobs_join_kernel<float>, static_cast<const float*>(a.logits));
  if (a.dtype == 1) return go(logprobs_kernel<f16, false>, logprobs_join_kernel<f16>, static_cast<const f16*>(a.logits));
  return go(logprobs_kernel<bf16, false>, logprobs_join_kernel<bf16>, static_cast<const bf16*>(a.logits));
}

// few slices, whose lists the join has to read: at most 16 a row and 512 workgroups in all (vocabulary 151936, fp16, graph-timed us, so
// / otherwise: 1 x 4 beams 11.3, with 64 slices 12.9; 16 x 8 in 4 slices 20.3, in 8 22.1; 32 x 8 in 2 25.9, in 4 27.6; 64 x 8 in 1 38.8, in
// 2 39.6)
hipError_t beam_select_launch(const BeamArgs& a, hipStream_t st) {
  const int M = a.requests * a.beams, S = row_slices(M, a.V, a.n, kBeamSlices, 512, a.ws_bytes);
  const size_t lds = slice_lds(a.V, a.dtype, S, sizeof(uint2));
  uint64_t* keys = static_cast<uint64_t*>(a.ws);              // [M][S][n] keys, then [M][S] sums
  Sums* part = reinterpret_cast<Sums*>(keys + (size_t)M * S * a.n);
  auto go = [&](auto first, auto* p) {
    if (lds > 49152) {                                        // (beside 12 KB of the kernel's own)
      static std::atomic<uint64_t> done{0};
      if (hipError_t err = allow_lds_once(done, first, kGroups * kThreads * sizeof(uint2))) return err;
    }
    return launch(first, dim3((unsigned)((int64_t)M * S)), dim3(kThreads), lds, st, p, a.stride,
                  static_cast<const int64_t*>(nullptr), static_cast<float*>(nullptr), static_cast<float*>(nullptr),
                  static_cast<float*>(nullptr), static_cast<int64_t*>(nullptr), a.V, a.n, S, part, keys, a.scores, a.finished);
  };
  hipError_t e = a.dtype == 0   ? go(logprobs_kernel<float, true>, static_cast<const float*>(a.logits))
                 : a.dtype == 1 ? go(logprobs_kernel<f16, true>, static_cast<const f16*>(a.logits))
                                : go(logprobs_kernel<bf16, true>, static_cast<const bf16*>(a.logits));
  if (e != hipSuccess) return e;
  const int depth = std::min(a.n, std::max(1, 64 / (a.beams * S)));
  const BeamJoin j{a.scores, a.finished, a.out_scores, a.out_beams, a.out_tokens, a.beams, a.V, a.n, a.pad, S, depth, part, keys};
  const size_t fixed = (size_t)a.beams * a.n * 12 + 8, each = (size_t)2 * S * a.n * 8;
  const size_t join_lds = std::min<size_t>(kBeamWhole, fixed + kBeamThreads / 64 * each);
  if (join_lds > 32768) {
    static std::atomic<uint64_t> done{0};
    if ((e = allow_lds_once(done, beam_join_kernel, kBeamWhole))) return e;
  }
  return launch(beam_join_kernel, dim3((unsigned)a.requests), dim3(kBeamThreads), join_lds, st, j);
}

}  // namespace lowbit
