// A batch of sequences over a paged KV cache: the q and k norms of every head with the position rotation and the write of
// k and v into the pages (norm_rope_paged), and causal GQA attention of each sequence's new tokens over its pages
// (attention_paged). Caches are [pages][Hkv][page size][D]; row r of page p is slot p * page size + r.
#include "paged_attention.hpp"

namespace lowbit {

namespace {

// cos and sin of p * inv_f: the product and its reduction to one turn in 64 bits (a position of 10^5 times a frequency of
// 1 keeps 2^-7 of a radian in 32), the functions of the remaining part of a turn in 32
__device__ __forceinline__ void turn_cos_sin(int64_t p, float inv_f, float& c, float& s) {
  const double turns = (double)p * (double)inv_f * 0.15915494309189533577;
  const float part = (float)(turns - rint(turns));
  sincospif(2.f * part, &s, &c);
}

}  // namespace

// A workgroup takes kTokens tokens: their cos and sin, one pair a thread, go to LDS while the first heads are loaded; then D /
// 16 lanes a head, lane t the dims 8 t .. 8 t + 7 and their partners D / 2 + 8 t .. in two 16-byte pieces, so that the rotation
// stays in a lane and the norm's sum takes three (D = 128) or two lane exchanges. y = x / sqrt(mean(x^2) + eps) * w and the
// rotation in 32 bits, rounded once. Bound: memory (8192 tokens of 28 / 4 heads of 128 in fp16, 151 MB, 28 us, 5.3 TB/s), of few
// tokens the launch. Four tokens a workgroup, whose pairs keep all its threads busy, from kManyTokens on, else one (28 / 4
// heads, us, one / four: 67 tokens 3.4 / 5.7, 512 4.3 / 6.2, 1024 6.6 / 7.0, 2048 10.4 / 10.1, 8192 31 / 28; 16 / 2 heads 1024
// 5.4 / 4.9; 14 / 2 heads of 64 8192 20 / 12).
constexpr int kHeadsAhead = 3;           // heads of a lane group in flight
constexpr int kManyTokens = 1024;

template <typename T, int D, int kTokens>
__global__ __launch_bounds__(256) void norm_rope_kernel(const T* __restrict__ qkv, int64_t stride, const T* __restrict__ qw,
                                                        const T* __restrict__ kw, float eps,
                                                        const int64_t* __restrict__ pos,
                                                        const float* __restrict__ inv_freq,
                                                        const int64_t* __restrict__ slots, T* __restrict__ q_out,
                                                        T* __restrict__ k_cache, T* __restrict__ v_cache, int M, int Hq,
                                                        int Hkv, FastDiv by_heads, int64_t rows, int shift, bool permuted) {
  constexpr int kLanes = D / 16, kSlots = 256 / kLanes, kPairs = D / 2;
  typedef T x8 __attribute__((ext_vector_type(8)));
  __shared__ __attribute__((aligned(16))) float s_cos[kTokens][kPairs], s_sin[kTokens][kPairs];
  args_in_sgprs(qkv, stride, qw, kw, pos, inv_freq, slots, q_out, k_cache, v_cache, M, Hq, Hkv, rows, shift);
  const int heads = Hq + 2 * Hkv, m0 = blockIdx.x * kTokens, items = min(kTokens, M - m0) * heads;
  const int t = threadIdx.x % kLanes, from_lo = permuted ? 16 * t : 8 * t, from_hi = permuted ? 16 * t + 8 : D / 2 + 8 * t;
  u32x4 lo[kHeadsAhead], hi[kHeadsAhead];
  auto fetch = [&](int it, u32x4& a, u32x4& b) {
    if (it >= items) return;
    const int m = div(it, by_heads), h = it - m * heads;
    const T* src = qkv + (m0 + m) * stride + h * D;
    a = load16(src + from_lo);
    b = load16(src + from_hi);
  };
  int it = threadIdx.x / kLanes;
#pragma unroll
  for (int u = 0; u < kHeadsAhead; ++u) fetch(it + u * kSlots, lo[u], hi[u]);
  for (int i = threadIdx.x; i < kTokens * kPairs; i += 256) {
    const int m = i / kPairs, p = i % kPairs;
    if (m0 + m < M) turn_cos_sin(pos[m0 + m], inv_freq[p], s_cos[m][p], s_sin[m][p]);
  }
  u32x4 wq[2] = {}, wk[2] = {};
  if (qw) {
    wq[0] = load16(qw + 8 * t);
    wq[1] = load16(qw + D / 2 + 8 * t);
    wk[0] = load16(kw + 8 * t);
    wk[1] = load16(kw + D / 2 + 8 * t);
  }
  __syncthreads();
  auto put = [&](int at, const u32x4& a, const u32x4& b) {
    if (at >= items) return;
    const int m = div(at, by_heads), h = at - m * heads;
    T* dst;
    if (h < Hq) {
      dst = q_out + ((int64_t)(m0 + m) * Hq + h) * D;
    } else {
      const int64_t slot = slots[m0 + m];
      if (slot < 0 || slot >= rows) return;                   // (a whole lane group)
      const int hk = h < Hq + Hkv ? h - Hq : h - Hq - Hkv;
      dst = (h < Hq + Hkv ? k_cache : v_cache) + (((((slot >> shift) * Hkv + hk) << shift) + (slot & ((1 << shift) - 1))) * D);
    }
    u32x4 oa = a, ob = b;
    if (h < Hq + Hkv) {
      const x8 xa = __builtin_bit_cast(x8, a), xb = __builtin_bit_cast(x8, b);
      float ya[8], yb[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ya[i] = (float)xa[i];
        yb[i] = (float)xb[i];
      }
      if (qw) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(ya[i], ya[i], fmaf(yb[i], yb[i], ss));
        ss = quad_sum(ss);
        if constexpr (kLanes == 8) ss += dpp<kRowHalfMirror>(ss);
        const float r = rsqrtf(ss * (1.f / (float)D) + eps);
        const x8 wa = __builtin_bit_cast(x8, h < Hq ? wq[0] : wk[0]), wb = __builtin_bit_cast(x8, h < Hq ? wq[1] : wk[1]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ya[i] = ya[i] * r * (float)wa[i];
          yb[i] = yb[i] * r * (float)wb[i];
        }
      }
      x8 za, zb;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float c = s_cos[m][8 * t + i], s = s_sin[m][8 * t + i];
        za[i] = (T)(ya[i] * c - yb[i] * s);
        zb[i] = (T)(yb[i] * c + ya[i] * s);
      }
      oa = __builtin_bit_cast(u32x4, za);
      ob = __builtin_bit_cast(u32x4, zb);
    }
    *reinterpret_cast<u32x4*>(dst + 8 * t) = oa;
    *reinterpret_cast<u32x4*>(dst + D / 2 + 8 * t) = ob;
  };
  for (; it < items; it += kHeadsAhead * kSlots) {
#pragma unroll
    for (int u = 0; u < kHeadsAhead; ++u) {
      const u32x4 a = lo[u], b = hi[u];
      fetch(it + (kHeadsAhead + u) * kSlots, lo[u], hi[u]);
      put(it + u * kSlots, a, b);
    }
  }
}

namespace {

template <typename T, int D, int kTokens>
hipError_t launch_norm_rope(const NormRopeArgs& a, hipStream_t st) {
  return launch(norm_rope_kernel<T, D, kTokens>, dim3((unsigned)((a.M + kTokens - 1) / kTokens)), dim3(256), 0, st,
                static_cast<const T*>(a.qkv), a.stride, static_cast<const T*>(a.q_weight), static_cast<const T*>(a.k_weight),
                a.eps, a.positions, a.inv_freq, a.slots, static_cast<T*>(a.q_out), static_cast<T*>(a.k_cache),
                static_cast<T*>(a.v_cache), a.M, a.Hq, a.Hkv, fast_div(a.Hq + 2 * a.Hkv), a.pages * a.page_size,
                log2_of(a.page_size), a.permuted);
}
template <typename T, int D>
hipError_t pick_norm_rope(const NormRopeArgs& a, hipStream_t st) {
  return a.M >= kManyTokens ? launch_norm_rope<T, D, 4>(a, st) : launch_norm_rope<T, D, 1>(a, st);
}

}  // namespace

hipError_t norm_rope_paged_launch(const NormRopeArgs& a, hipStream_t st) {
  if (a.bf16) return a.D == 64 ? pick_norm_rope<bf16, 64>(a, st) : pick_norm_rope<bf16, 128>(a, st);
  return a.D == 64 ? pick_norm_rope<f16, 64>(a, st) : pick_norm_rope<f16, 128>(a, st);
}

size_t attention_paged_workspace(const PagedAttentionArgs& a) {
  const PagedLaunch l = paged_launch(a);
  return l.records * paged_record_bytes(l.rg, a.D);
}

hipError_t attention_paged_launch(const PagedAttentionArgs& a, hipStream_t st) {
  if (a.bf16) return a.D == 64 ? pick_paged_attention<bf16, 64>(a, st) : pick_paged_attention<bf16, 128>(a, st);
  return a.D == 64 ? pick_paged_attention<f16, 64>(a, st) : pick_paged_attention<f16, 128>(a, st);
}

}  // namespace lowbit
