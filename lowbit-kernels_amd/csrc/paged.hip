// A batch of sequences over a paged KV cache: the q and k norms of every head with the position rotation and the write of
// k and v into the pages (norm_rope_paged), and causal GQA attention of each sequence's new tokens over its pages
// (attention_paged). Caches are [pages][Hkv][page size][D]; row r of page p is slot p * page size + r.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "kernels.hpp"

namespace lowbit {

namespace {

typedef __bf16 bf16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct FastDiv {                                              // n / d = high word of n m >> s for 0 <= n < 2^31 (m 0: d is 1)
  uint32_t m;
  int s;
};
__device__ __forceinline__ int div(int n, const FastDiv& d) { return d.m ? (int)(__umulhi((uint32_t)n, d.m) >> d.s) : n; }

FastDiv fast_div(int d) {
  if (d == 1) return {0, 0};
  int l = 1;
  while ((int64_t)1 << l < d) ++l;
  return {(uint32_t)((((uint64_t)1 << (31 + l)) + (uint64_t)d - 1) / (uint64_t)d), l - 1};
}

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

// ---- attention_paged ----
// A workgroup takes 32 RG query rows of one sequence and KV head (row = new token * G + head in the group) and walks a
// range of the sequence's keys; see paged_attention. The work of a call is numbered along blockIdx.x, and every workgroup
// finds its own part from the sequences' lengths, so that a captured launch serves any lengths:
//   a sequence has tiles of rows, and its keys are cut into `parts` alike for all its tiles, `parts` being its blocks of keys
//   over a share that the whole call's blocks give each of the GPU's workgroup slots. A tile of one part writes its output,
//   the parts of another write records of the workspace that paged_attention_merge joins in order.
struct PagedPlan {
  int slots;         // workgroups that the GPU holds at once
  int least;         // blocks of a part at least
  int cap;           // parts of a tile at most (1: no split)
  int most;          // parts of split tiles in all at most (what the workspace holds, twice its share)
  int Hq, Hkv, G;
  FastDiv by_hkv, by_g;
};
struct PagedUnit {
  int seq, first, nq, len, tiles, parts, tile, hk, pid, rec;   // first: the sequence's first row of q; rec: the part's record (parts > 1)
};

// sum of the lanes up to and including this one
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8: within 16 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast 15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // row_bcast 31 into rows 2 and 3
  return v;
}

// What lane l knows of sequence b0 + l (all zero past the last one): its rows of q, keys, tiles of kRows and blocks of kBlock.
struct PagedSeq {
  int first, nq, len, tiles, blocks;
};
template <int kRows, int kBlock>
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, int G, int seq) {
  PagedSeq s{};
  if (seq >= b.B) return s;
  const int q0 = b.q_starts[seq], q1 = b.q_starts[seq + 1], n = b.kv_lens[seq];
  s.first = min(max(q0, 0), b.T);
  s.nq = min(max(q1, s.first), b.T) - s.first;
  s.len = max(n, 0);
  s.tiles = (s.nq * G + kRows - 1) / kRows;
  s.blocks = s.nq ? (min(s.len, b.table_width * b.page_size) + kBlock - 1) / kBlock : 0;
  return s;
}

// The parts' share in blocks. While tiles of one part leave a quarter of the GPU's slots free, the total over the free ones,
// so that the parts, each sequence's rounded up, run at once; else the total over one and a half rounds of slots, so that only
// keys far above the mean are cut (us with half a round, one, one and a half and two: 64 decode tokens of 32 / 8 heads on 300 ..
// 8000 keys 147, 133, 129 and 128; a prompt of 2000 tokens, 28 / 4 heads, 64, 71, 71 and 79; a mixed step 33.8, 34.2, 34.7 and
// 34.8). s0: the first 64 sequences.
template <int kRows, int kBlock>
__device__ __forceinline__ int paged_share(const PagedBatch& b, const PagedPlan& p, const PagedSeq& s0, int lane) {
  if (p.cap == 1) return 0x3FFFFFFF;
  float total = wave_sum((float)s0.tiles * (float)s0.blocks), units = wave_sum((float)s0.tiles);
  for (int b0 = 64; b0 < b.B; b0 += 64) {
    const PagedSeq s = paged_seq<kRows, kBlock>(b, p.G, b0 + lane);
    total += wave_sum((float)s.tiles * (float)s.blocks);
    units += wave_sum((float)s.tiles);
  }
  total *= (float)p.Hkv;
  units *= (float)p.Hkv;
  const float slots = (float)p.slots;
  const float free = fminf(units < 0.75f * slots ? slots - units : 1.5f * slots, (float)(p.most / 2));
  return max(p.least, (int)fminf(ceilf(total / free), 1e9f));
}

// The part of work `idx`; false past the last one. kMerge > 0: the chunk `idx` of kMerge rows (a divisor of kRows) of the split
// tiles, pid counting the chunk in its tile and rec the tile's first part.
template <int kRows, int kBlock, int kMerge>
__device__ __forceinline__ bool paged_unit(const PagedBatch& b, const PagedPlan& p, const PagedSeq& s0, int share, int idx,
                                           int lane, PagedUnit& u) {
  int before = 0, recs = 0;                                  // work and record groups of the sequences before
  for (int b0 = 0; b0 < b.B; b0 += 64) {
    const PagedSeq s = b0 == 0 ? s0 : paged_seq<kRows, kBlock>(b, p.G, b0 + lane);
    const int parts = p.cap == 1 ? 1 : max(1, min(p.cap, (s.blocks + share - 1) / share));
    const int tiles = s.tiles * p.Hkv, split = parts > 1 ? tiles * parts : 0;
    const int mine = kMerge == 0 ? tiles * parts : parts > 1 ? (s.nq * p.G + max(kMerge, 1) - 1) / max(kMerge, 1) * p.Hkv : 0;
    const int upto = wave_scan(mine), recs_upto = p.cap == 1 ? 0 : wave_scan(split);
    const uint64_t hit = __ballot(idx - before < upto);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto pick = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      u.seq = b0 + l;
      u.first = pick(s.first);
      u.nq = pick(s.nq);
      u.len = pick(s.len);
      u.tiles = pick(s.tiles);
      u.parts = p.cap == 1 ? 1 : pick(parts);
      const int at = idx - before - pick(upto - mine), rest = div(at, p.by_hkv);
      u.hk = at - rest * p.Hkv;                              // KV heads fastest: a head's keys stay in the L2 of its XCDs
      if constexpr (kMerge == 0) {
        const int t = u.parts == 1 ? rest : (int)((uint32_t)rest / (uint32_t)u.parts);
        u.pid = rest - t * u.parts;
        u.tile = u.tiles - 1 - t;                            // the last rows, which have the most keys, first
      } else {
        u.tile = rest / (kRows / kMerge);
        u.pid = rest % (kRows / kMerge);
      }
      u.rec = p.cap == 1 ? 0 : recs + pick(recs_upto - split) + (u.tile * p.Hkv + u.hk) * u.parts + (kMerge == 0 ? u.pid : 0);
      // (starts that fall, which the caller rules out, could number more work than 32 bits hold: never past the buffers. A
      // tile of one part has no record, whatever its number)
      return at >= 0 && (uint32_t)u.tile < (uint32_t)u.tiles &&
             (u.parts == 1 || (u.rec >= 0 && u.rec <= p.most - (kMerge == 0 ? 1 : u.parts)));
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    if (p.cap > 1) recs += __builtin_amdgcn_readlane(recs_upto, 63);
  }
  return false;
}

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct Mfma;
template <>
struct Mfma<f16> {
  typedef f16x8 x8;
  static __device__ __forceinline__ f32x16 go(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    typedef f16 x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, x2));
  }
  static __device__ __forceinline__ float sum2(uint32_t p, float c) {   // c + the two values
    return dot2(as_f16x2(p), f16x2{(f16)1.f, (f16)1.f}, c);
  }
  static constexpr uint32_t kExponent = 0x7C00u;              // all ones: an infinity or a NaN
  static __device__ __forceinline__ float half_of(uint32_t w, int i) { return (float)as_f16x2(w)[i]; }
};
template <>
struct Mfma<bf16> {
  typedef bf16x8 x8;
  static __device__ __forceinline__ f32x16 go(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    typedef bf16 x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, x2));
  }
  static __device__ __forceinline__ float sum2(uint32_t p, float c) {
    return c + (__builtin_bit_cast(float, p << 16) + __builtin_bit_cast(float, p & 0xFFFF0000u));
  }
  static constexpr uint32_t kExponent = 0x7F80u;
  static __device__ __forceinline__ float half_of(uint32_t w, int i) {
    return __builtin_bit_cast(float, i ? w & 0xFFFF0000u : w << 16);
  }
};

// the sign bits of a pair's values that are infinities or NaN (the exponent's ones carry into them, none past them)
template <typename T>
__device__ __forceinline__ uint32_t odd2(uint32_t w) {
  constexpr uint32_t one = Mfma<T>::kExponent & -Mfma<T>::kExponent;   // the exponent's last bit
  return ((w & 0x7FFF7FFFu) + (one | one << 16)) & 0x80008000u;
}
// a pair's finite values, zeros for the others
template <typename T>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  const uint32_t m = odd2<T>(w);
  return w & ~(m | (m - (m >> 15)));
}

// four values of a row's output; a row without a key gets zeros
template <typename T>
__device__ __forceinline__ void store_row(T* dst, const f32x4& num, float den, bool some) {
  const float inv = 1.f / den;
  *reinterpret_cast<uint2*>(dst) = some ? make_uint2(Mfma<T>::pack(num[0] * inv, num[1] * inv), Mfma<T>::pack(num[2] * inv, num[3] * inv))
                                        : make_uint2(0u, 0u);
}

// blocks ahead that K and V are requested, and the slots of LDS that takes
template <int RG, int KG>
constexpr int paged_ahead() { return KG == 4 || RG * KG == 1 ? 1 : 3; }
template <int D, int RG, int KG>
constexpr size_t paged_lds() {
  const size_t ring = (size_t)(paged_ahead<RG, KG>() + 1) * 2 * 32 * KG * D * 2;
  const size_t merge = KG > 1 ? (size_t)4 * 32 * (D + 4) * 4 : 0;
  return ring > merge ? ring : merge;
}
constexpr int paged_per_cu(int rg, int kg) { return kg > 1 ? 1 : rg == 1 ? 5 : 2; }   // workgroups, by their LDS at D = 128
template <int D>
constexpr int paged_rec() { return D + 4; }                  // floats of a row's record: reference, weight sum, -, -, output

// RG row groups of 32 rows times KG key groups, a wave each (4 x 1, 2 x 2, 1 x 4 or 1 x 1); a block is 32 KG keys, wave (rg, kg)
// taking the block's 32 keys of key group kg for its rows. Per 32 keys (32x32x16 MFMA, lane l: j = l % 32, h = l / 32):
//   S^T = K Q^T: A = 32 keys x 16 dims from LDS, B = 32 rows (registers); lane (j, h) holds row j's scores of keys 8 (v / 4) +
//   4 h + v % 4, v < 16.
//   Softmax in base 2 (c2 = |scale| log2 e) against a reference that follows the row's running maximum only when a score passes
//   it by more than kLag / c2, so that the output's registers are rescaled in the first blocks only. The products start at
//   minus the reference, so that a difference is scaled and rounded, never the score itself: above 2^24 / c2, scaled scores have
//   steps of 1 and more, and weights 2^(step / 2) too large leave fp16. Weights are 2^((score - reference) c2 + 15 - kLag), the
//   largest between 2^(15 - kLag) and 2^15, rounded to T for the second product: half a step of T for each weight, the same
//   relative step as the output's own rounding; in fp16 those below 2^-14 are off by 2^-25, i.e. 2^-32 of the largest. Their
//   sum, in 32 bits, is of the rounded weights, as the output's is. (As two halves, which leave the output's rounding alone: an
//   error of 2.0e-4 for 2.4e-4 .. 2.9e-4 of the output in fp16, 1.7e-3 for 2.2e-3 in bf16; but prompts 527 -> 690 us, a mixed
//   step 35.5 -> 40, one token 13.1 -> 13.8, 64 decode tokens 129.9 -> 130.6, and an infinity in V, times a second half of 0,
//   would become a NaN.)
//   O^T += V^T P^T: B = the weights as the lane holds them, A = V^T from LDS by transposing reads.
// K and V go from the pages straight to LDS, rows as they are: a wave-load takes 1 KB, 512 / D keys, in groups of up to 16 keys
// of one page, so that address and bound are scalar and looked up once a group; rows past the sequence's keys and pages
// outside the cache read as zeros through the bound, so nothing unwritten meets the products. The 16-byte pieces of a row are
// permuted by the key: K's so that the 32 rows of a fragment read meet different banks, V's so that the four rows of a
// transposing read do (no conflict is counted). K is requested paged_ahead + 1 blocks before its scores' weights, V
// paged_ahead, and a block's scores are multiplied while the vector unit evaluates the block before. With one row group a
// wave loads the keys it takes itself and no barrier is needed.
// Bounds (MI355X): few rows, the read of K and V: 64 decode tokens of 32 / 8 heads on 300 .. 8000 keys (626 MB) 130 us, 4.8
// TB/s; 3 tokens of 28 / 4 heads on 40000 .. 70000 70 us, 5.1 TB/s. Prompts, power: 8000 tokens of 28 / 4 heads 520 us in fp16
// and 503 in bf16, 0.88 and 0.91 PFLOP/s, on zeros 422, where the vector unit and the matrix cores are busy 43% and 42%. There,
// measured and not kept, against 500 us of that time's kernel: 64 rows a wave with one wave per SIMD (half the LDS reads) 703 us;
// eight waves in two turns, one four on the matrix cores while the other is on the vector unit, 509 us and 454 on zeros; three
// waves per SIMD (168 registers, spilled) 546; two blocks ahead instead of three 519 .. 536.
constexpr float kLag = 8.f;

// of scores to powers of 2 (a NaN stays one); a negative scale's sign goes into q
__device__ __forceinline__ float score_scale(float scale) {
  const float c2 = fabsf(scale) * 1.44269504088896340736f;
  return c2 < FLT_MIN ? FLT_MIN : c2;
}

template <typename T, int D, int RG, int KG>
__global__ __launch_bounds__(64 * RG * KG, KG > 1 ? 1 : 2) void paged_attention(
    const T* __restrict__ q, const T* __restrict__ k_cache, const T* __restrict__ v_cache, PagedBatch bt, PagedPlan plan,
    T* __restrict__ out, float* __restrict__ part, int shift, float scale) {
  constexpr int NW = RG * KG;
  constexpr int RB = D * 2;                                  // bytes of a row
  constexpr int PR = RB / 16;                                // its pieces
  constexpr int KL = 64 / PR;                                // keys of a wave-load
  constexpr int BK = 32 * KG;
  constexpr int BB = BK * RB;                                // bytes of a block of K, and of V
  constexpr int KW = BK / NW;                                // keys of a block that a wave loads
  constexpr int NG = (KW + 15) / 16, LG = KW / NG / KL;      // groups of them, wave-loads of a group
  constexpr int NP = NG * LG;                                // wave-loads of a wave and block, for K and for V
  constexpr int AH = paged_ahead<RG, KG>(), N = AH + 1;          // slots: [N] K blocks, [N] V blocks
  constexpr bool kOwn = RG == 1;                             // a wave loads its own keys
  constexpr int DT = D / 32, KS = D / 16;
  constexpr int kRows = 32 * RG;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  args_in_sgprs(q, k_cache, v_cache, bt.table, bt.q_starts, bt.kv_lens, bt.B, bt.T, bt.table_width, bt.page_size, plan.slots,
                plan.cap, plan.G, plan.by_hkv.m, plan.by_g.m, out, part, shift);
  const int Hq = plan.Hq, Hkv = plan.Hkv, G = plan.G;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 31, h = lane >> 5;
  PagedUnit un;
  const PagedSeq s0 = paged_seq<kRows, BK>(bt, G, lane);
  if (!paged_unit<kRows, BK, 0>(bt, plan, s0, paged_share<kRows, BK>(bt, plan, s0, lane), blockIdx.x, lane, un)) return;
  const int rgrp = wave % RG, kgrp = wave / RG;
  const int cap = bt.table_width * bt.page_size;
  const int len = min(un.len, cap);                  // keys that can be read
  const int rows = un.nq * G;
  const int tok_last = div(min(rows, (un.tile + 1) * kRows) - 1, plan.by_g);
  const int keys = min(un.len - un.nq + tok_last + 1, cap);  // of the tile's last row (none: 0 or less)
  const int nblk = (max(keys, 0) + BK - 1) / BK;
  const int per = un.parts == 1 ? nblk : (int)((uint32_t)(nblk + un.parts - 1) / (uint32_t)un.parts);
  const int b0 = min(nblk, un.pid * per), b1 = min(nblk, b0 + per);
  const int kend = min(keys, b1 * BK);
  // this lane's row: its last key (the least of the wave's rows: wmin) and q
  const float c2 = score_scale(scale), lag = fminf(kLag / c2, FLT_MAX);
  const uint32_t flip = scale < 0.f ? 0x80008000u : 0u;      // a negative scale is moved into q (exact)
  const int row = un.tile * kRows + 32 * rgrp + j, row_c = min(row, rows - 1), tok = div(row_c, plan.by_g);
  const bool live = row < rows;
  const int pr = live ? min(un.len - un.nq + tok, cap - 1) : -1;
  int wmin = live ? pr : INT_MAX;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) wmin = min(wmin, __shfl_xor(wmin, off, 64));
  wmin = __builtin_amdgcn_readfirstlane(wmin);
  const int64_t qrow = ((int64_t)(un.first + tok) * Hq + un.hk * G + (row_c - tok * G)) * D;
  u32x4 qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    qf[s] = load16(q + qrow + 16 * s + 8 * h);
#pragma unroll
    for (int e = 0; e < 4; ++e) qf[s][e] ^= flip;
  }
  const bool busy = wmin != INT_MAX;                         // a wave whose rows are all past the end only loads

  // ---- loads ----
  // where the 128 pages from `win` on begin in a cache, lane l holding pages win + l and win + 64 + l: byte offsets of this KV
  // head's rows, bit 63 set for a page outside the cache. They are waited for where they are fetched (the empty asm uses
  // them), so that no later use waits for the loads into LDS that were requested in between
  const int* table = bt.table + (int64_t)un.seq * bt.table_width;
  int win = (b0 * BK) >> shift;
  uint32_t wlo[2], whi[2];
  auto fetch = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = win + 64 * i + lane;
      const int id = at < bt.table_width ? table[at] : -1;
      const uint64_t off = ((uint64_t)(uint32_t)id * (uint32_t)Hkv + (uint32_t)un.hk) * (uint32_t)bt.page_size * RB;
      wlo[i] = (uint32_t)off;
      whi[i] = id >= 0 && id < bt.pages ? (uint32_t)(off >> 32) : 0x80000000u;
    }
    asm volatile("" : "+v"(wlo[0]), "+v"(wlo[1]), "+v"(whi[0]), "+v"(whi[1]));
  };
  fetch();
  const uint32_t lds0 = lds_addr(smem);
  // A wave loads keys KW wave .. + KW - 1 of every block (with KG == 4 the keys it takes), in groups of at most 16, which lie
  // in one page; a wave-load takes KL keys, lane l the 16-byte slot l % PR of key l / PR
  const int lk = lane / PR, ls = lane % PR;
  auto kswz = [](int key) { return D == 128 ? key & 15 : (key >> 1) & 7; };
  auto vswz = [](int key) { return D == 128 ? 4 * (key & 3) + 2 * ((key >> 2) & 1) : 4 * ((key >> 1) & 1); };
  int koff[LG], voff[LG];
#pragma unroll
  for (int u = 0; u < LG; ++u) {
    const int k = KW * wave + KL * u + lk;                    // (groups of 16 repeat)
    koff[u] = (KL * u + lk) * RB + 16 * (ls ^ kswz(k));
    voff[u] = (KL * u + lk) * RB + 16 * (ls ^ vswz(k));
  }
  struct Rows {
    uint32_t lo[NG], hi[NG], bytes[NG];                       // a group's rows: offset in a cache, bytes that exist
  };
  auto rows_of = [&](int blk) {
    if ((((blk + 1) * BK - 1) >> shift) - win >= 128) {       // (uniform)
      win = (blk * BK) >> shift;
      fetch();
    }
    Rows p;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int key = blk * BK + KW * wave + 16 * g, at = (key >> shift) - win;
      const uint32_t lo0 = __builtin_amdgcn_readlane(wlo[0], at & 63), lo1 = __builtin_amdgcn_readlane(wlo[1], at & 63);
      const uint32_t hi0 = __builtin_amdgcn_readlane(whi[0], at & 63), hi1 = __builtin_amdgcn_readlane(whi[1], at & 63);
      const uint32_t lo = at & 64 ? lo1 : lo0, hi = at & 64 ? hi1 : hi0;
      const uint64_t off = (((uint64_t)hi << 32) | lo) + (uint32_t)((key & (bt.page_size - 1)) * RB);
      p.lo[g] = (uint32_t)off;
      p.hi[g] = (uint32_t)(off >> 32);
      p.bytes[g] = blk < b1 && (int)hi >= 0 ? (uint32_t)(min(max(len - key, 0), KL * LG) * RB) : 0u;
    }
    return p;
  };
  const uint64_t kbase = reinterpret_cast<uint64_t>(k_cache), vbase = reinterpret_cast<uint64_t>(v_cache);
  auto load = [&](uint64_t cache, const Rows& p, const int (&off)[LG], uint32_t at) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint64_t base = cache + (((uint64_t)p.hi[g] << 32) | p.lo[g]);
      const uint64_t ub = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(base >> 32)) << 32) |
                          (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)base);   // (uniform; the compiler keeps it scalar then)
      const __amdgpu_buffer_rsrc_t rs = make_rsrc(reinterpret_cast<const void*>(ub), (uint32_t)__builtin_amdgcn_readfirstlane((int)p.bytes[g]));
#pragma unroll
      for (int u = 0; u < LG; ++u) dma16(rs, off[u], lds0 + at + (uint32_t)((KW * wave + 16 * g + KL * u) * RB));
    }
  };
  auto slot = [](int i) { return (uint32_t)(i * BB); };
  constexpr uint32_t kV = N * BB;                            // V's slots follow K's

  const uint32_t kr = (32 * kgrp + j) * RB + 16 * (h ^ kswz(j));
  const int vk = 4 * h + ((lane & 15) >> 2), vp = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t vr = kV + (32 * kgrp + vk) * RB + 16 * (vp ^ vswz(vk)) + 8 * (lane & 1);
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  auto v_frag = [&](uint32_t at) {                            // keys at .. and at + 8 rows, this lane's dim
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(smem + at));
    const s16x4 c = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(smem + at + 8 * RB));
    return __builtin_bit_cast(u32x4, __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  float lsum[2] = {0.f, 0.f};                                 // the lane's share of the weights' sum
  const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  f32x16 o[DT], st = zero, neg = zero;                        // output, scores of the wave's 32 keys of a block less the row's
  float pass = -INFINITY;                                     // reference, minus that; what a score passes to move it (-inf: none yet)
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = zero;
  auto k_frag = [&](uint32_t at, int s) { return *reinterpret_cast<const u32x4*>(smem + at + (kr ^ (32 * s))); };
  // some row leaves out a key of the 32 from kb on that is there (keys past the tile's last row may be, up to the sequence's
  // last)
  auto guarded = [&](int kb) { return wmin < min(kb + 31, len - 1); };
  bool some_odd = false;
  // One block: the weights of its scores, the weights times V and the next block's scores. Every fragment is read well before
  // its product (K's and V's first half at the start, V's other half while K's are multiplied)
  auto block = [&](uint32_t kat, uint32_t vat, int kb) {      // kb: the wave's first key
    u32x4 kf[KS], va[2][DT];
#pragma unroll
    for (int s = 0; s < KS; ++s) kf[s] = k_frag(kat, s);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) va[0][dt] = v_frag(vat + (vr ^ (64 * dt)));
    __builtin_amdgcn_sched_barrier(0);
    if (kb + 31 > min(wmin, kend - 1)) {                      // some row attends part of these keys only (uniform)
      const int last = min(pr, kend - 1) - kb - 4 * h;        // a key at or below it counts
#pragma unroll
      for (int v = 0; v < 16; ++v)
        if (8 * (v >> 2) + (v & 3) > last) st[v] = -INFINITY;
    }
    float bm = st[0];
#pragma unroll
    for (int v = 1; v < 16; ++v) bm = fmaxf(bm, st[v]);
    if (__any(bm > pass)) {                                   // (uniform; either lane of a row)
      const bool fresh = pass == -INFINITY;                   // (the row has seen no key: its reference counts as 0)
      const float top = fmaxf(bm, __shfl_xor(bm, 32, 64)), up = fresh ? (top == -INFINITY ? 0.f : top) : fmaxf(top, 0.f);
      const float ref = up - neg[0], d = ref + neg[0];        // (d: what the rounded reference moves by)
      const float corr = fresh ? 1.f : __builtin_amdgcn_exp2f(-d * c2);
      pass = top == -INFINITY ? pass : lag;
      lsum[0] *= corr;
      lsum[1] *= corr;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        st[v] -= d;
        neg[v] = -ref;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= corr;
    }
    // Where a row leaves out a key that the block holds, its weight 0 may meet an infinity or a NaN of that key's V: those are
    // taken out of the product, and the rows that do attend the key get them after the walk (uniform; rare)
    bool odd = false;
    if (guarded(kb)) {
      uint32_t any = 0;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u32x4 second = v_frag(vat + (vr ^ (64 * dt)) + 16 * RB);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t first = va[0][dt][e];
          asm("" : "+v"(first));                              // (else every block takes the steps shared with finite2 below)
          any |= odd2<T>(first) | odd2<T>(second[e]);
        }
      }
      odd = __any(any != 0);
      some_odd |= odd;
    }
    const f32x16 sc = st;
    st = neg;
#pragma unroll
    for (int s = 0; s < 2; ++s) {                             // 16 keys
      u32x4 ph;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ph[i] = Mfma<T>::pack(__builtin_amdgcn_exp2f(fmaf(sc[8 * s + 2 * i], c2, 15.f - kLag)),
                              __builtin_amdgcn_exp2f(fmaf(sc[8 * s + 2 * i + 1], c2, 15.f - kLag)));
        lsum[i & 1] = Mfma<T>::sum2(ph[i], lsum[i & 1]);
      }
#pragma unroll
      for (int i = KS / 2 * s; i < KS / 2 * s + KS / 2; ++i)  // the next block's (past the last one: of zeros, not used)
        st = Mfma<T>::go(kf[i], qf[i], st);
      if (s == 0) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) va[1][dt] = v_frag(vat + (vr ^ (64 * dt)) + 16 * RB);
      }
      if (odd) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int e = 0; e < 4; ++e) va[s][dt][e] = finite2<T>(va[s][dt][e]);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = Mfma<T>::go(va[s][dt], ph, o[dt]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (b0 < b1) {
    auto sync = [](auto n) {
      if constexpr (kOwn)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(n)::value) : "memory");
      else
        lds_wait_barrier<decltype(n)::value>();
    };
    Rows at = rows_of(b0);
    load(kbase, at, koff, slot(0));
#pragma unroll
    for (int t = 0; t < AH; ++t) {
      load(vbase, at, voff, kV + slot(t));
      at = rows_of(b0 + t + 1);
      load(kbase, at, koff, slot((t + 1) % N));
    }
    sync(std::integral_constant<int, 2 * NP * AH>{});
    if (busy) {
#pragma unroll
      for (int i = 0; i < KS; ++i) st = Mfma<T>::go(k_frag(slot(0), i), qf[i], st);
    }
    sync(std::integral_constant<int, 2 * NP * (AH - 1)>{});
    // unrolled over the slots, so that every LDS address is a register and a constant, and over two blocks, so that the
    // next block's scores need no copy
    constexpr int U = N % 2 ? 2 * N : N;
    for (int i = b0; i < b1; i += U) {
#pragma unroll
      for (int t = 0; t < U; ++t) {
        if (i + t >= b1) break;
        load(vbase, at, voff, kV + slot((t + AH) % N));
        at = rows_of(i + t + 1 + AH);
        load(kbase, at, koff, slot(t % N));
        if (busy) block(slot((t + 1) % N), slot(t % N), (i + t) * BK + 32 * kgrp);
        sync(std::integral_constant<int, 2 * NP * (AH - 1)>{});
      }
    }
    lds_wait_barrier<0>();                                    // nothing is left in flight, and the slots may be reused
    if (some_odd) {                                           // the values that the guarded blocks left out, from the pages again
#pragma unroll 1
      for (int i = b0; i < b1; ++i) {
        const int kb = i * BK + 32 * kgrp;
        if (!guarded(kb)) continue;
#pragma unroll 1
        for (int key = kb; key < min(kb + 32, kend); ++key) {
          const int id = table[key >> shift];
          if (id < 0 || id >= bt.pages) continue;             // (zeros)
          const T* from = v_cache + (((int64_t)id * Hkv + un.hk) * bt.page_size + (key & (bt.page_size - 1))) * D + 4 * h;
#pragma unroll
          for (int v = 0; v < D / 8; ++v) {
            const uint2 p = *reinterpret_cast<const uint2*>(from + 8 * v);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t w = e < 2 ? p.x : p.y;
              if (key <= pr && (odd2<T>(w) >> (16 * (e & 1)) & 0x8000u)) o[v >> 2][4 * (v & 3) + e] += Mfma<T>::half_of(w, e & 1);
            }
          }
        }
      }
    }
  }
  const float ref = pass == -INFINITY ? -INFINITY : -neg[0];
  float den = lsum[0] + lsum[1];
  den += __shfl_xor(den, 32, 64);
  if constexpr (KG > 1) {
    // the key groups' sums meet in LDS as rows, reference and weight sum behind each, and leave 16 bytes of a row a lane
    constexpr int kPitch = D + 4, kLanes = D / 4;
    float* sums = reinterpret_cast<float*>(smem);
    float* mine = sums + (size_t)(wave * 32 + j) * kPitch;
    if (live) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; v += 4)
          *reinterpret_cast<f32x4*>(mine + 32 * dt + 2 * v + 4 * h) = f32x4{o[dt][v], o[dt][v + 1], o[dt][v + 2], o[dt][v + 3]};
      if (h == 0) {
        mine[D] = ref;
        mine[D + 1] = den;
      }
    }
    lds_barrier();
    const int d = 4 * (tid % kLanes);
    for (int r = tid / kLanes; r < min(kRows, rows - un.tile * kRows); r += 256 / kLanes) {
      const float* at = sums + (size_t)((r >> 5) * 32 + (r & 31)) * kPitch;   // row group r / 32: waves r / 32 + RG k
      float top = -INFINITY, all = 0.f;
#pragma unroll
      for (int k = 0; k < KG; ++k) top = fmaxf(top, at[k * RG * 32 * kPitch + D]);
      f32x4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        const float* theirs = at + k * RG * 32 * kPitch;
        const float m = theirs[D], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - top) * c2);
        const f32x4 v = *reinterpret_cast<const f32x4*>(theirs + d);
        all = fmaf(f, theirs[D + 1], all);
#pragma unroll
        for (int e = 0; e < 4; ++e) num[e] = fmaf(f, v[e], num[e]);
      }
      const int at_row = un.tile * kRows + r, t = div(at_row, plan.by_g), g = at_row - t * G;
      if (un.parts == 1) {
        store_row<T>(out + ((int64_t)(un.first + t) * Hq + un.hk * G + g) * D + d, num, all, un.len - un.nq + t >= 0);
      } else {
        float* rec = part + ((size_t)un.rec * kRows + r) * paged_rec<D>();
        if (d == 0) {
          rec[0] = top;
          rec[1] = all;
        }
        *reinterpret_cast<f32x4*>(rec + 4 + d) = num;
      }
    }
    return;
  }
  if (!live) return;
  // lane (j, h) holds O^T[32 dt + 8 (v / 4) + 4 h + v % 4][row j]
  if (un.parts == 1) {
    T* dst = out + qrow + 4 * h;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int v = 0; v < 16; v += 4)
        store_row<T>(dst + 32 * dt + 2 * v, f32x4{o[dt][v], o[dt][v + 1], o[dt][v + 2], o[dt][v + 3]}, den, pr >= 0);
  } else {
    float* rec = part + ((size_t)un.rec * kRows + 32 * rgrp + j) * paged_rec<D>();
    if (h == 0) {
      rec[0] = ref;
      rec[1] = den;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int v = 0; v < 16; v += 4)
        *reinterpret_cast<f32x4*>(rec + 4 + 32 * dt + 2 * v + 4 * h) = f32x4{o[dt][v], o[dt][v + 1], o[dt][v + 2], o[dt][v + 3]};
  }
}

// The outputs of the split tiles: a workgroup takes chunks of paged_merge_rows rows, PG lane groups a row, each joining every
// PG-th part in order, their weights 2^((reference - largest reference) c2); then the groups' sums. Tiles of 32 rows, which few
// rows on many parts take, have four groups a row, the others one.
template <int kRows>
constexpr int paged_merge_groups() { return kRows == 32 ? 4 : 1; }
template <int D, int kRows>
constexpr int paged_merge_rows() { return 1024 / D / paged_merge_groups<kRows>(); }
template <typename T, int D, int kRows, int kBlock>
__global__ __launch_bounds__(256) void paged_attention_merge(const float* __restrict__ part, PagedBatch bt, PagedPlan plan,
                                                             T* __restrict__ out, float scale) {
  constexpr int kLanes = D / 4, PG = paged_merge_groups<kRows>(), kHere = paged_merge_rows<D, kRows>(), kRec = paged_rec<D>();
  __shared__ f32x4 s_num[256];
  __shared__ float s_top[256 / kLanes], s_den[256 / kLanes];
  args_in_sgprs(part, bt.table, bt.q_starts, bt.kv_lens, bt.B, bt.T, bt.table_width, bt.page_size, plan.slots, plan.cap, plan.G,
                plan.by_hkv.m, plan.by_g.m, out);
  const int lane = threadIdx.x & 63, grp = threadIdx.x / kLanes, c = threadIdx.x % kLanes;
  const float c2 = score_scale(scale);
  const PagedSeq s0 = paged_seq<kRows, kBlock>(bt, plan.G, lane);
  const int share = paged_share<kRows, kBlock>(bt, plan, s0, lane);
  PagedUnit un;
  for (int idx = blockIdx.x; paged_unit<kRows, kBlock, kHere>(bt, plan, s0, share, idx, lane, un); idx += gridDim.x) {
    const int r = un.pid * kHere + grp / PG, row = un.tile * kRows + r;
    const float* rec = part + ((size_t)un.rec * kRows + r) * kRec;
    const size_t step = (size_t)kRows * kRec;
    f32x4 num = {0.f, 0.f, 0.f, 0.f};
    float den = 0.f, top = -INFINITY;
    if (row < un.nq * plan.G) {
      for (int p0 = grp % PG; p0 < un.parts; p0 += 8 * PG) {       // eight records' loads in flight
        f32x4 v[8];
        float m[8], l[8], nm = top;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float* at = rec + (size_t)min(p0 + PG * i, un.parts - 1) * step;
          m[i] = at[0];
          l[i] = at[1];
          v[i] = *reinterpret_cast<const f32x4*>(at + 4 + 4 * c);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (p0 + PG * i >= un.parts) m[i] = -INFINITY;
          nm = fmaxf(nm, m[i]);
        }
        const float f0 = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((top - nm) * c2);
        den *= f0;
        num *= f0;
        top = nm;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (p0 + PG * i >= un.parts) continue;
          // (no score of a part's keys above -inf: its sums are zeros, or NaN where a score was, which factor 0 keeps)
          const float f = m[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[i] - top) * c2);
          den = fmaf(f, l[i], den);
#pragma unroll
          for (int e = 0; e < 4; ++e) num[e] = fmaf(f, v[i][e], num[e]);
        }
      }
    }
    if constexpr (PG > 1) {
      s_num[threadIdx.x] = num;
      if (c == 0) {
        s_top[grp] = top;
        s_den[grp] = den;
      }
      __syncthreads();
    }
    if (grp % PG == 0 && row < un.nq * plan.G) {
      if constexpr (PG > 1) {
#pragma unroll
        for (int i = 1; i < PG; ++i) top = fmaxf(top, s_top[grp + i]);
        num = f32x4{0.f, 0.f, 0.f, 0.f};
        den = 0.f;
#pragma unroll
        for (int i = 0; i < PG; ++i) {
          const float m = s_top[grp + i], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - top) * c2);
          den = fmaf(f, s_den[grp + i], den);
#pragma unroll
          for (int e = 0; e < 4; ++e) num[e] = fmaf(f, s_num[threadIdx.x + i * kLanes][e], num[e]);
        }
      }
      const int tok = div(row, plan.by_g), g = row - tok * plan.G;
      store_row<T>(out + ((int64_t)(un.first + tok) * plan.Hq + un.hk * plan.G + g) * D + 4 * c, num, den,
                   un.len - un.nq + tok >= 0);
    }
    if constexpr (PG > 1) __syncthreads();
  }
}

namespace {

int log2_of(int n) {
  int s = 0;
  while ((1 << s) < n) ++s;
  return s;
}

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

constexpr int kPagedParts = 256;                             // of a tile at most
constexpr int kPagedLeast = 256;                             // keys of a part at least
constexpr int kPagedWhole = 768;                             // keys up to which decode tiles are not split

// How a call is launched, from its sizes and bounds alone.
struct PagedLaunch {
  int rg, kg;                                                // the tile, as rows and keys of 32
  int slots;                                                 // workgroups that the GPU holds at once
  int64_t units;                                             // tiles times KV heads at most
  int least, cap;                                            // blocks of a part at least, parts of a tile at most (1: no split)
  int records;                                               // of split tiles that the workspace has use for
};

// Which tile serves a call; any serves every call. Sequences of at most 32 rows (decode, few drafted tokens) take four waves
// on four key groups (RG 1, KG 4), one workgroup a CU; where there are more tiles than those and the keys are few, or very many
// tiles, one wave, five a CU (28 / 4 heads, us, four waves / one: 100 tokens on 100 keys 13.5 / 9.6, 300 on 100 39 / 22, on 1000
// 153 / 152, 30 tokens of 32 / 32 heads on up to 2000 48 / 41; but 40 on 500 12.7 / 19.8, 100 on 2000 90 / 95, 64 of 32 / 8 heads
// on 300 .. 8000 130 / 141; 100 on 500 lie on the line, 26 / 21). More rows take four waves of 128 rows (RG 4), two workgroups
// a CU, or of 64 rows and two key groups while those tiles fit the CUs once and the keys are few, so that the serial walk counts
// (us, 128 rows / 64: 28 / 4 heads, one prompt of 500 24.5 / 17.8, of 1200 42 / 50, 500 on 2000 cached 41 / 62, 300 on 500 with
// 40 decode tokens 25.9 / 29.0; one of 8000 527 / 1042).
PagedLaunch paged_launch(const PagedAttentionArgs& a) {
  const int64_t G = a.Hq / a.Hkv, seqs = std::min(a.batch.B, a.batch.T);   // with new tokens
  auto tiles = [&](int rows) { return ((int64_t)a.batch.T * G / rows + seqs) * a.Hkv; };   // at most
  PagedLaunch p{};
  if (a.max_new * G <= 32) {
    p.rg = 1;
    p.kg = tiles(32) > 256 && (a.max_keys <= 512 || tiles(32) > 768) ? 1 : 4;
  } else if (tiles(64) <= 256 && a.max_keys <= 1024) {
    p.rg = p.kg = 2;
  } else {
    p.rg = 4;
    p.kg = 1;
  }
  const int rows = 32 * p.rg, block = 32 * p.kg;
  p.slots = 256 * paged_per_cu(p.rg, p.kg);
  p.units = (((int64_t)a.batch.T * G + rows - 1) / rows + seqs) * a.Hkv;
  p.least = std::max(1, kPagedLeast / block);
  // no split, and no launch of the merge, where it does not pay: decode tiles of few keys, other tiles of not many that fill
  // half the slots (28 / 4 heads, us, split or its idle merge / whole: one token on 700 keys 11.8 / 13.0, where the host saves a
  // launch, on 1000 12.0 / 15.5, on 3000 12.4 / 34; 8 on 500 12.1 / 11.0, on 1000 12.4 / 15.8; 40, whose tiles take 160 of the 256
  // slots, on 760 18.3 / 15.7, on 1500 26.7 / 24.1 and on 3000 43.4 / 41.1: the keys alone do not tell those; a prompt of 500 30.0
  // / 17.7, of 900 34.0 / 29.3; six prompts of 171 .. 794, 14 / 2 heads of 64, 23.7 / 20.2)
  const bool whole = p.rg == 1 ? a.max_keys <= kPagedWhole : a.max_keys <= 1024 && 2 * p.units >= p.slots;
  p.cap = whole ? 1 : std::min(kPagedParts, (int)((((int64_t)a.max_keys + block - 1) / block + p.least - 1) / p.least));
  // twice the free slots that paged_share gives parts at most, and twice what the tiles can be cut into
  p.records = p.cap == 1 ? 0 : (int)std::min<int64_t>(p.rg == 4 ? 2048 : 1024, 2 * p.units * p.cap);
  return p;
}

size_t paged_record_bytes(int rg, int D) { return (size_t)32 * rg * (D == 64 ? paged_rec<64>() : paged_rec<128>()) * sizeof(float); }

template <typename T, int D, int RG, int KG>
hipError_t launch_paged_attention(const PagedAttentionArgs& a, const PagedLaunch& l, hipStream_t st) {
  constexpr size_t lds = paged_lds<D, RG, KG>();
  constexpr int kRows = 32 * RG, kBlock = 32 * KG;
  const int G = a.Hq / a.Hkv;
  PagedPlan p{l.slots, l.least, 1, 0, a.Hq, a.Hkv, G, fast_div(a.Hkv), fast_div(G)};
  p.most = a.ws ? (int)std::min<size_t>((size_t)l.records, a.ws_bytes / paged_record_bytes(RG, D)) : 0;
  if (p.most >= 2) p.cap = l.cap;
  const int64_t grid = p.cap == 1 ? l.units : std::min<int64_t>(l.units * p.cap, l.units + p.most / 2 + 1);
  if (lds > 65536) {
    static std::atomic<uint64_t> done{0};
    if (hipError_t e = allow_lds_once(done, paged_attention<T, D, RG, KG>, lds)) return e;
  }
  const int shift = log2_of(a.batch.page_size);
  hipError_t e = launch(paged_attention<T, D, RG, KG>, dim3((unsigned)grid), dim3(64 * RG * KG), lds, st,
                        static_cast<const T*>(a.q), static_cast<const T*>(a.k_cache), static_cast<const T*>(a.v_cache),
                        a.batch, p, static_cast<T*>(a.out), static_cast<float*>(a.ws), shift, a.scale);
  if (e != hipSuccess || p.cap == 1) return e;
  constexpr int kHere = paged_merge_rows<D, kRows>();
  const int64_t seqs = std::min(a.batch.B, a.batch.T), chunks = (((int64_t)a.batch.T * G + kHere - 1) / kHere + seqs) * a.Hkv;
  return launch(paged_attention_merge<T, D, kRows, kBlock>, dim3((unsigned)std::min<int64_t>(chunks, 2048)), dim3(256), 0, st,
                static_cast<const float*>(a.ws), a.batch, p, static_cast<T*>(a.out), a.scale);
}

template <typename T, int D>
hipError_t pick_paged_attention(const PagedAttentionArgs& a, hipStream_t st) {
  const PagedLaunch l = paged_launch(a);
  if (l.rg == 4) return launch_paged_attention<T, D, 4, 1>(a, l, st);
  if (l.rg == 2) return launch_paged_attention<T, D, 2, 2>(a, l, st);
  return l.kg == 4 ? launch_paged_attention<T, D, 1, 4>(a, l, st) : launch_paged_attention<T, D, 1, 1>(a, l, st);
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
