// Log probabilities of given tokens with the entropy and the most likely alternatives of each row of logits.
#include <climits>

#include "kernels.hpp"

namespace lowbit {

namespace {

typedef __bf16 bf16;

// (value, index) as one number, larger = earlier among the alternatives: the larger value (-0 equal to +0, a NaN above
// every number, as torch orders them), then the smaller index. Zero is below every key.
__device__ __forceinline__ uint64_t rank_key(float x, int idx) {
  uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
  u = x != x ? 0xFFFFFFFFu : (u >> 31) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)(0x7FFFFFFF - idx);
}

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

}  // namespace

// One workgroup per row: the maximum, then the sums, then the alternatives one by one, each the largest key below the one
// before.
template <typename T>
__global__ __launch_bounds__(512) void logprobs_kernel(const T* __restrict__ logits, int64_t stride,
                                                       const int64_t* __restrict__ targets, float* __restrict__ logprob,
                                                       float* __restrict__ entropy, float* __restrict__ top_value,
                                                       int64_t* __restrict__ top_id, int V, int top) {
  __shared__ float red[8];
  __shared__ uint64_t redk[8];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * stride;
  float mx = -INFINITY;
  bool nan = false;
  for (int i = threadIdx.x; i < V; i += blockDim.x) {
    const float v = (float)x[i];
    mx = fmaxf(mx, v);
    nan |= v != v;
  }
  mx = block_reduce(nan ? INFINITY : mx, red, [](float a, float b) { return fmaxf(a, b); });
  // a NaN, a +inf or nothing above -inf leaves no distribution: every result is NaN, as log_softmax gives
  const bool none = !(mx < INFINITY) || mx == -INFINITY;
  float z = 0.f, e = 0.f;
  for (int i = threadIdx.x; i < V; i += blockDim.x) {
    const float d = (float)x[i] - mx, p = expf(d);
    z += p;
    e += p > 0.f ? p * d : 0.f;                             // 0 log 0 = 0
  }
  z = block_reduce(z, red, [](float a, float b) { return a + b; });
  e = block_reduce(e, red, [](float a, float b) { return a + b; });
  const float lz = logf(z);
  if (threadIdx.x == 0) {
    const int64_t t = targets[row];
    logprob[row] = t < 0 ? 0.f : none || t >= V ? NAN : ((float)x[t] - mx) - lz;
    entropy[row] = none ? NAN : lz - e / z;
  }
  uint64_t below = ~(uint64_t)0;
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < V; i += blockDim.x) {
      const uint64_t key = rank_key((float)x[i], i);
      if (key < below && key > best) best = key;
    }
    below = block_reduce(best, redk, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
    const int idx = 0x7FFFFFFF - (int)(uint32_t)below;
    if (threadIdx.x == 0) {
      top_id[row * top + k] = idx;
      top_value[row * top + k] = none ? NAN : ((float)x[idx] - mx) - lz;
    }
  }
}

hipError_t token_logprobs_launch(const LogprobArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.M), block(512);
  auto go = [&](auto kernel, auto* p) {
    return launch(kernel, grid, block, 0, st, p, a.stride, a.targets, a.logprob, a.entropy, a.top_value, a.top_id, a.V, a.top);
  };
  if (a.dtype == 0) return go(logprobs_kernel<float>, static_cast<const float*>(a.logits));
  if (a.dtype == 1) return go(logprobs_kernel<f16>, static_cast<const f16*>(a.logits));
  return go(logprobs_kernel<bf16>, static_cast<const bf16*>(a.logits));
}

}  // namespace lowbit
