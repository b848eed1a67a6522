// A batch of sequences over a paged KV cache: the q and k norms of every head with the position rotation and the write of
// k and v into the pages (norm_rope_paged), and causal GQA attention of each sequence's new tokens over its pages
// (attention_paged). Caches are [pages][Hkv][page size][D]; row r of page p is slot p * page size + r.
#include <algorithm>
#include <climits>

#include "kernels.hpp"

namespace lowbit {

namespace {

typedef __bf16 bf16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// cos and sin of p * inv_f: the product and its reduction to one turn in 64 bits (a position of 10^5 times a frequency of
// 1 keeps 2^-7 of a radian in 32), the functions of the remaining part of a turn in 32
__device__ __forceinline__ void turn_cos_sin(int64_t p, float inv_f, float& c, float& s) {
  const double turns = (double)p * (double)inv_f * 0.15915494309189533577;
  const float part = (float)(turns - rint(turns));
  sincospif(2.f * part, &s, &c);
}

}  // namespace

// One wave per (token, head), lane l < D / 2 the pair (l, l + D / 2): y = x / sqrt(mean(x^2) + eps) * w and the rotation in
// 32 bits, rounded once.
template <typename T, int D>
__global__ __launch_bounds__(256) void norm_rope_kernel(const T* __restrict__ qkv, int64_t stride,
                                                        const T* __restrict__ qw, const T* __restrict__ kw, float eps,
                                                        const int64_t* __restrict__ pos,
                                                        const float* __restrict__ inv_freq,
                                                        const int64_t* __restrict__ slots, T* __restrict__ q_out,
                                                        T* __restrict__ k_cache, T* __restrict__ v_cache, int M, int Hq,
                                                        int Hkv, int64_t pages, int page_size, bool permuted) {
  const int heads = Hq + 2 * Hkv;
  const int unit = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int m = unit / heads, h = unit - m * heads;
  if (m >= M) return;
  const T* src = qkv + m * stride + (int64_t)h * D;
  const bool live = lane < D / 2;
  const int i = live ? lane : 0, s1 = permuted ? rope_row(i) : i, s2 = permuted ? rope_row(i) + 8 : i + D / 2;
  const T r1 = src[s1], r2 = src[s2];
  T* dst;
  if (h < Hq) {
    dst = q_out + ((int64_t)m * Hq + h) * D;
  } else {
    const int64_t slot = slots[m];
    if (slot < 0 || slot >= pages * page_size) return;
    const int64_t page = slot / page_size, row = slot - page * page_size;
    const int hk = (h - Hq) % Hkv;
    dst = (h < Hq + Hkv ? k_cache : v_cache) + ((page * Hkv + hk) * page_size + row) * D;
  }
  T o1 = r1, o2 = r2;
  if (h < Hq + Hkv) {
    float x1 = (float)r1, x2 = (float)r2;
    const T* w = h < Hq ? qw : kw;
    if (w) {
      const float ss = wave_sum(live ? x1 * x1 + x2 * x2 : 0.f);
      const float r = rsqrtf(ss / (float)D + eps);
      x1 *= r * (float)w[i];
      x2 *= r * (float)w[i + D / 2];
    }
    float c, s;
    turn_cos_sin(pos[m], inv_freq[i], c, s);
    o1 = (T)(x1 * c - x2 * s);
    o2 = (T)(x2 * c + x1 * s);
  }
  if (live) {
    dst[i] = o1;
    dst[i + D / 2] = o2;
  }
}

// One wave per (token, query head), its lanes the head's dims.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_attention_kernel(const T* __restrict__ q, const T* __restrict__ k_cache,
                                                              const T* __restrict__ v_cache, PagedBatch b,
                                                              T* __restrict__ out, int Hq, int Hkv, float scale) {
  const int unit = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int t = unit / Hq, h = unit - t * Hq, hk = h / (Hq / Hkv);
  if (t >= b.T) return;
  int seq = -1, first = 0, end = 0;
  for (int i = 0; i < b.B && seq < 0; ++i) {
    first = min(max(b.q_starts[i], 0), b.T);
    end = min(max(b.q_starts[i + 1], first), b.T);
    if (t >= first && t < end) seq = i;
  }
  if (seq < 0) return;                                       // a row of no sequence is left as it is
  const int len = b.kv_lens[seq], last = min(len - (end - first) + (t - first), (int)min((int64_t)b.table_width * b.page_size, (int64_t)INT_MAX) - 1);
  constexpr int E = D / 64;
  float qv[E], o[E] = {}, mx = -INFINITY, sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) qv[e] = (float)q[((int64_t)t * Hq + h) * D + E * lane + e] * scale;
  for (int base = 0; base <= last; base += 16) {             // 16 keys' sums before they meet the running ones
    float sc[16], vv[16][E], bm = -INFINITY;
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int key = min(base + u, last);
      const int page = b.table[(int64_t)seq * b.table_width + key / b.page_size];
      const bool real = page >= 0 && page < b.pages;         // a page outside the cache reads as zeros
      const int64_t at = (((int64_t)(real ? page : 0) * Hkv + hk) * b.page_size + key % b.page_size) * D + E * lane;
      float a = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        a = fmaf(qv[e], real ? (float)k_cache[at + e] : 0.f, a);
        vv[u][e] = real ? (float)v_cache[at + e] : 0.f;
      }
      a = wave_sum(a);
      sc[u] = base + u <= last ? a : -INFINITY;
      bm = fmaxf(bm, sc[u]);
    }
    const float nm = fmaxf(mx, bm), corr = expf(mx - nm);
    float bs = 0.f, bo[E] = {};
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const float p = expf(sc[u] - nm);
      bs += p;
#pragma unroll
      for (int e = 0; e < E; ++e) bo[e] = fmaf(p, vv[u][e], bo[e]);
    }
    sum = sum * corr + bs;
    mx = nm;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * corr + bo[e];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) out[((int64_t)t * Hq + h) * D + E * lane + e] = last >= 0 ? (T)(o[e] / sum) : (T)0.f;
}

namespace {

template <typename T, int D>
hipError_t launch_norm_rope(const NormRopeArgs& a, hipStream_t st) {
  const int64_t units = (int64_t)a.M * (a.Hq + 2 * a.Hkv);
  return launch(norm_rope_kernel<T, D>, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, static_cast<const T*>(a.qkv),
                a.stride, static_cast<const T*>(a.q_weight), static_cast<const T*>(a.k_weight), a.eps, a.positions,
                a.inv_freq, a.slots, static_cast<T*>(a.q_out), static_cast<T*>(a.k_cache), static_cast<T*>(a.v_cache), a.M,
                a.Hq, a.Hkv, a.pages, a.page_size, a.permuted);
}

template <typename T, int D>
hipError_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t st) {
  const int64_t units = (int64_t)a.batch.T * a.Hq;
  return launch(paged_attention_kernel<T, D>, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st,
                static_cast<const T*>(a.q), static_cast<const T*>(a.k_cache), static_cast<const T*>(a.v_cache), a.batch,
                static_cast<T*>(a.out), a.Hq, a.Hkv, a.scale);
}

}  // namespace

hipError_t norm_rope_paged_launch(const NormRopeArgs& a, hipStream_t st) {
  if (a.bf16) return a.D == 64 ? launch_norm_rope<bf16, 64>(a, st) : launch_norm_rope<bf16, 128>(a, st);
  return a.D == 64 ? launch_norm_rope<f16, 64>(a, st) : launch_norm_rope<f16, 128>(a, st);
}

hipError_t attention_paged_launch(const PagedAttentionArgs& a, hipStream_t st) {
  if (a.bf16) return a.D == 64 ? launch_paged_attention<bf16, 64>(a, st) : launch_paged_attention<bf16, 128>(a, st);
  return a.D == 64 ? launch_paged_attention<f16, 64>(a, st) : launch_paged_attention<f16, 128>(a, st);
}

}  // namespace lowbit
