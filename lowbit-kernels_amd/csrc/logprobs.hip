// Log probabilities of given tokens with the entropy and the most likely alternatives of each row of logits.
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

// Workgroup (row, slice): see the top of the file. part (S > 1): [row][slice] Sums, then keys [row][slice][top].
// Bound: memory, 2047 rows of 151665 in fp16 (621 MB) 126 us, 4.9 TB/s; of few rows the chain of load, sums, bound, reread and
// join: 48 rows of 151936 in fp32 18 us, one in fp16 13.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(const T* __restrict__ logits, int64_t stride,
                                                            const int64_t* __restrict__ targets,
                                                            float* __restrict__ logprob, float* __restrict__ entropy,
                                                            float* __restrict__ top_value, int64_t* __restrict__ top_id,
                                                            int V, int top, int S, Sums* __restrict__ part,
                                                            uint64_t* __restrict__ part_keys) {
  constexpr int kN = 16 / sizeof(T);
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  float* s_max = reinterpret_cast<float*>(smem);              // [group][thread]
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
    e = fmaf(p, fmaxf(d, -1e4f), e);
  };
  const int64_t end = (int64_t)(v1 - v0);
  float gm = -INFINITY;
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
    gm = step % every == 0 ? sm : fmaxf(gm, sm);
    s_max[step / every * kThreads + tid] = gm;
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
    if (S == 1)
      store_sums(x, V, targets[row], s, logprob + row, entropy + row);
    else
      part[blockIdx.x] = s;
  }
  if (top == 0) return;

  // ---- the alternatives ----
  const bool none = !(s.m > -INFINITY && s.m < INFINITY) || s.z != s.z;
  const float lz = logf(s.z);
  auto give = [&](int rank, uint64_t key) {                   // by the thread that holds it
    if (S > 1) {
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
      if (!(s_max[g * kThreads + tid] >= bound)) continue;
      for (int step = g * every; step < min(steps, (g + 1) * every); ++step)
        for (int u = 0; u < kUnroll; ++u) {
          const int64_t i = (int64_t)(step * kUnroll + u) * kThreads + tid;
          if (i >= end) continue;
          const u32x4 v = load16(body + (v0 + i) * kN);
#pragma unroll
          for (int k = 0; k < kN; ++k) {
            const float f = value<T>(v, k);
            if (above ? f > bound : f >= bound) push(f, head + (int)(v0 + i) * kN + k);
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
        for (int k = 0; k < n; ++k) rank += s_list[k] > key;
        if (rank < top) give(rank, key);
      }
      if (S > 1)                                              // a slice of fewer logits than `top`
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
    if (tid == 0) give(k, below);                             // (S > 1: 0 where the slice has no more)
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

hipError_t token_logprobs_launch(const LogprobArgs& a, hipStream_t st) {
  // slices: up to 1024 workgroups, four a CU, of at least 2048 logits
  int S = 1;
  if (a.ws && a.M < 512) {
    S = (int)std::min<int64_t>({1024 / a.M, a.V / 2048, (int64_t)kMaxSlices});
    const size_t per = (size_t)a.M * (sizeof(Sums) + 4 + (size_t)a.top * 8);
    S = (int)std::max<size_t>(1, std::min<size_t>((size_t)std::max(S, 1), a.ws_bytes / per));
  }
  const int each = a.dtype == 0 ? 4 : 8;                      // logits of a vector
  const int64_t vectors = (a.V / each + S - 1) / S, steps = (vectors + kThreads * kUnroll - 1) / (kThreads * kUnroll);
  const size_t lds = (size_t)std::max<int64_t>(1, std::min<int64_t>(steps, kGroups)) * kThreads * sizeof(float);
  uint64_t* keys = static_cast<uint64_t*>(a.ws);              // [M][S][top] keys, then [M][S] sums
  Sums* part = reinterpret_cast<Sums*>(keys + (size_t)a.M * S * a.top);
  auto go = [&](auto first, auto second, auto* p) {
    hipError_t e = launch(first, dim3((unsigned)((int64_t)a.M * S)), dim3(kThreads), lds, st, p, a.stride, a.targets, a.logprob,
                          a.entropy, a.top_value, a.top_id, a.V, a.top, S, part, keys);
    if (e != hipSuccess || S == 1) return e;
    return launch(second, dim3((unsigned)a.M), dim3(256), 0, st, p, a.stride, a.targets, a.logprob, a.entropy, a.top_value,
                  a.top_id, a.V, a.top, S, part, keys);
  };
  if (a.dtype == 0) return go(logprobs_kernel<float>, logprobs_join_kernel<float>, static_cast<const float*>(a.logits));
  if (a.dtype == 1) return go(logprobs_kernel<f16>, logprobs_join_kernel<f16>, static_cast<const f16*>(a.logits));
  return go(logprobs_kernel<bf16>, logprobs_join_kernel<bf16>, static_cast<const bf16*>(a.logits));
}

}  // namespace lowbit
