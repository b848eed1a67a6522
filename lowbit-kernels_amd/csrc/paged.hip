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

// ---- attention_paged ----
// A workgroup takes 32 NR RG query rows of one sequence and KV head (row = new token * G + head in the group) and walks a
// range of the sequence's keys; see paged_attention. The work of a call is numbered along blockIdx.x, and every workgroup
// finds its own part from the sequences' lengths, so that a captured launch serves any lengths:
//   a sequence has tiles of rows, and its keys are cut into `parts` alike for all its tiles, `parts` being its blocks of keys
//   over a share that the whole call's blocks give each of the GPU's workgroup slots. A tile of one part writes its output,
//   the parts of another write records of the workspace that paged_attention_merge joins in order.
struct PagedPlan {
  int rows;          // query rows of a tile
  int block;         // keys of a block
  int slots;         // workgroups that the GPU holds at once
  int least;         // blocks of a part at least
  int cap;           // parts of a tile at most (1: no split)
  int most;          // parts of split tiles in all at most (what the workspace holds, twice its share)
};
struct PagedUnit {
  int seq, first, nq, len, tiles, parts, tile, hk, pid, rec;   // first: the sequence's first row of q; rec: the part's records
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

// What lane l knows of sequence b0 + l (all zero past the last one): its rows of q, keys, tiles and blocks of keys.
struct PagedSeq {
  int first, nq, len, tiles, blocks;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, const PagedPlan& p, int G, int seq) {
  PagedSeq s{};
  if (seq >= b.B) return s;
  s.first = min(max(b.q_starts[seq], 0), b.T);
  s.nq = min(max(b.q_starts[seq + 1], s.first), b.T) - s.first;
  s.len = max(b.kv_lens[seq], 0);
  s.tiles = (s.nq * G + p.rows - 1) / p.rows;
  s.blocks = s.nq ? (min(s.len, b.table_width * b.page_size) + p.block - 1) / p.block : 0;
  return s;
}

// The parts' share in blocks: total blocks over the slots that tiles of one part leave free in the call's rounds of
// workgroups (half a round at least), so that the parts, each sequence's rounded up, fill whole rounds.
__device__ __forceinline__ int paged_share(const PagedBatch& b, const PagedPlan& p, int G, int Hkv, int lane) {
  if (p.cap == 1) return 0x3FFFFFFF;
  float total = 0.f, units = 0.f;
  for (int b0 = 0; b0 < b.B; b0 += 64) {
    const PagedSeq s = paged_seq(b, p, G, b0 + lane);
    total += wave_sum((float)s.tiles * (float)s.blocks);
    units += wave_sum((float)s.tiles);
  }
  total *= (float)Hkv;
  units *= (float)Hkv;
  const float slots = (float)p.slots, rounds = ceilf((units + 0.5f * slots) / slots);
  const float free = fminf(rounds * slots - units, (float)(p.most / 2));
  return max(p.least, (int)fminf(ceilf(total / free), 1e9f));
}

// The unit of work `idx` (split: counted among the split tiles alone, without their parts). False past the last one.
template <bool kSplitTiles>
__device__ __forceinline__ bool paged_unit(const PagedBatch& b, const PagedPlan& p, int G, int Hkv, int idx, int lane,
                                           PagedUnit& u) {
  const int share = paged_share(b, p, G, Hkv, lane);
  int before = 0, recs = 0;                                  // units and record groups of the sequences before
  for (int b0 = 0; b0 < b.B; b0 += 64) {
    const PagedSeq s = paged_seq(b, p, G, b0 + lane);
    const int parts = max(1, min(p.cap, (s.blocks + share - 1) / share));
    const int tiles = s.tiles * Hkv, split = parts > 1 ? tiles * parts : 0;
    const int mine = kSplitTiles ? (parts > 1 ? tiles : 0) : tiles * parts;
    const int upto = wave_scan(mine), recs_upto = wave_scan(split);
    const uint64_t hit = __ballot(idx - before < upto);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto pick = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      u.seq = b0 + l;
      u.first = pick(s.first);
      u.nq = pick(s.nq);
      u.len = pick(s.len);
      u.tiles = pick(s.tiles);
      u.parts = pick(parts);
      int at = idx - before - pick(upto - mine);
      const int rec = recs + pick(recs_upto - split);
      u.hk = at % Hkv;                                       // KV heads fastest: a head's keys stay in the L2 of its XCDs
      at /= Hkv;
      u.pid = kSplitTiles ? 0 : at % u.parts;
      at = kSplitTiles ? at : at / u.parts;
      u.tile = u.tiles - 1 - at;                             // the last rows, which have the most keys, first
      u.rec = rec + ((u.tile * Hkv + u.hk) * u.parts + u.pid);
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    recs += __builtin_amdgcn_readlane(recs_upto, 63);
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
};

// blocks ahead that K and V are requested, and the slots of LDS that takes
template <int KG>
constexpr int paged_ahead() { return KG == 4 ? 1 : 2; }
template <int D, int RG, int KG>
constexpr size_t paged_lds() {
  const size_t ring = (size_t)(paged_ahead<KG>() + 1) * 2 * 32 * KG * D * 2;
  const size_t merge = (size_t)(KG - 1) * RG * (D / 2 + 2) * 256;
  return ring > merge ? ring : merge;
}
template <int D>
constexpr int paged_rec() { return D + 4; }                  // floats of a row's record: reference, weight sum, -, -, output

// Four waves: RG row groups of 32 NR rows times KG key groups; a block is 32 KG keys, wave (rg, kg) taking the block's 32 keys
// of key group kg for its rows. Per 32 keys (32x32x16 MFMA, lane l: j = l % 32, h = l / 32):
//   S^T = K Q^T: A = 32 keys x 16 dims from LDS, B = 32 rows (registers); lane (j, h) holds row j's scores of keys 8 (v / 4) +
//   4 h + v % 4, v < 16.
//   Softmax in base 2 against a reference that follows the running maximum only when a score passes it by more than kLag, so
//   that the output's registers are rescaled in the first blocks only. Weights are 2^(score - reference + 15 - kLag), the
//   largest between 2^(15 - kLag) and 2^15, rounded to T for the second product: half a step of T for each weight, the same
//   relative step as the output's own rounding (fp16: down to 2^-14, i.e. 2^-25 of the largest weight, and half of 2^-24
//   below); their sum is of the unrounded weights in 32 bits.
//   O^T += V^T P^T: B = the weights as the lane holds them, A = V^T from LDS by transposing reads.
// K and V go from the pages straight to LDS, rows as they are: a wave-load takes 1 KB, 512 / D keys, which lie in one page, so
// that its page number, address and bound are scalar; rows past the sequence's keys and pages outside the cache read as zeros
// through the bound, so nothing unwritten meets the products. The 16-byte pieces of a row are permuted by the key: K's so
// that the 32 rows of a fragment read meet different banks, V's so that the four rows of a transposing read do. K's are
// requested paged_ahead + 1 blocks before their scores' softmax, V's paged_ahead, and a block's scores are multiplied while
// the vector unit evaluates the block before. With KG == 4 a wave loads the keys it takes itself and no barrier is needed.
constexpr float kLag = 4.f;

template <typename T, int D, int RG, int KG, int NR>
__global__ __launch_bounds__(256, KG == 4 || NR > 1 ? 1 : 2) void paged_attention(
    const T* __restrict__ q, const T* __restrict__ k_cache, const T* __restrict__ v_cache, PagedBatch bt, PagedPlan plan,
    T* __restrict__ out, float* __restrict__ part, int Hq, int Hkv, int shift, float scale) {
  static_assert(RG * KG == 4, "four waves");
  constexpr int RB = D * 2;                                  // bytes of a row
  constexpr int PR = RB / 16;                                // its pieces
  constexpr int KL = 64 / PR;                                // keys of a wave-load
  constexpr int BK = 32 * KG;
  constexpr int BB = BK * RB;                                // bytes of a block of K, and of V
  constexpr int NP = BK / (4 * KL);                          // wave-loads of a wave and block, for K and for V
  constexpr int AH = paged_ahead<KG>(), N = AH + 1;          // slots: [N] K blocks, [N] V blocks
  constexpr bool kOwn = RG == 1;                             // a wave loads its own keys
  constexpr int DT = D / 32, KS = D / 16;
  constexpr int kRows = 32 * NR * RG;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int G = Hq / Hkv;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 31, h = lane >> 5;
  PagedUnit un;
  if (!paged_unit<false>(bt, plan, G, Hkv, blockIdx.x, lane, un)) return;
  const int rgrp = wave % RG, kgrp = wave / RG;
  const int cap = bt.table_width * bt.page_size;
  const int len = min(un.len, cap);                  // keys that can be read
  const int rows = un.nq * G;
  const int tok_last = (min(rows, (un.tile + 1) * kRows) - 1) / G;
  const int keys = min(un.len - un.nq + tok_last + 1, cap);  // of the tile's last row (none: 0 or less)
  const int nblk = (max(keys, 0) + BK - 1) / BK;
  const int per = (nblk + un.parts - 1) / un.parts;
  const int b0 = min(nblk, un.pid * per), b1 = min(nblk, b0 + per);
  const int kend = min(keys, b1 * BK);
  // the rows' last keys, least and most of a row group, and q
  int pr[NR], wmin[NR];
  bool live[NR];
  int64_t qrow[NR];
  u32x4 qf[NR][KS];
  const uint32_t flip = scale < 0.f ? 0x80008000u : 0u;      // a negative scale is moved into q (exact)
  const float c2 = fabsf(scale) * 1.44269504088896340736f < FLT_MIN ? FLT_MIN : fabsf(scale) * 1.44269504088896340736f;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int row = un.tile * kRows + 32 * (NR * rgrp + r) + j;
    live[r] = row < rows;
    const int c = min(row, rows - 1), tok = c / G, g = c - tok * G;
    pr[r] = live[r] ? min(un.len - un.nq + tok, cap - 1) : -1;
    wmin[r] = live[r] ? pr[r] : INT_MAX;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) wmin[r] = min(wmin[r], __shfl_xor(wmin[r], o, 64));
    wmin[r] = __builtin_amdgcn_readfirstlane(wmin[r]);
    qrow[r] = ((int64_t)(un.first + tok) * Hq + un.hk * G + g) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[r][s] = load16(q + qrow[r] + 16 * s + 8 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[r][s][e] ^= flip;
    }
  }
  const bool busy = wmin[0] != INT_MAX;                      // a wave whose rows are all past the end only loads

  // ---- loads ----
  // page numbers of window [win, win + 64) pages, a lane each; the next window requested when one is begun
  const int* table = bt.table + (int64_t)un.seq * bt.table_width;
  int win = (b0 * BK) >> shift;
  auto fetch = [&](int first) { return first + lane < bt.table_width ? table[first + lane] : -1; };
  int cur = fetch(win), nxt = fetch(win + 64);
  const uint64_t head_bytes = (uint64_t)bt.page_size * RB;   // a head's rows of a page
  const uint32_t lds0 = lds_addr(smem);
  // lane's row of a wave-load and its slot there
  const int lk = lane / PR, ls = lane % PR;
  auto kswz = [](int key) { return D == 128 ? key & 15 : (key >> 1) & 7; };
  auto vswz = [](int key) { return D == 128 ? 4 * (key & 3) + 2 * ((key >> 2) & 1) : 4 * ((key >> 1) & 1); };
  auto load_key = [&](int u) { return kOwn ? 32 * kgrp + KL * u : KL * (4 * u + wave); };   // first key of wave-load u
  struct Pages {
    int id[NP];
  };
  auto pages_of = [&](int blk) {
    Pages p;
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      const int key = blk * BK + load_key(u), pg = key >> shift;
      if (pg - win >= 64) {
        win += 64;
        cur = nxt;
        nxt = fetch(win + 64);
      }
      const int id = __builtin_amdgcn_readlane(cur, (pg - win) & 63);
      p.id[u] = blk < b1 && key < len && id >= 0 && id < bt.pages ? id : -1;
    }
    return p;
  };
  auto load = [&](const T* cache, const Pages& p, int blk, uint32_t at, bool is_k) {
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      const int lkey = load_key(u), key = blk * BK + lkey, row = key & (bt.page_size - 1);
      const int n = p.id[u] < 0 ? 0 : min(len - key, KL);    // rows that exist
      const uint64_t off = ((uint64_t)(uint32_t)max(p.id[u], 0) * (uint32_t)Hkv + (uint32_t)un.hk) * head_bytes + (uint64_t)(uint32_t)row * RB;
      const uint64_t base = reinterpret_cast<uint64_t>(cache) + off;
      const uint64_t ub = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(base >> 32)) << 32) |
                          (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)base);
      const __amdgpu_buffer_rsrc_t rs = make_rsrc(reinterpret_cast<const void*>(ub), (uint32_t)__builtin_amdgcn_readfirstlane(n * RB));
      const int k = lkey + lk, piece = ls ^ (is_k ? kswz(k) : vswz(k));
      dma16(rs, lk * RB + 16 * piece, lds0 + at + lkey * RB);
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

  float ref[NR], lsum[NR];
  f32x16 o[NR][DT], st[NR];
  const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    ref[r] = -INFINITY;
    lsum[r] = 0.f;
    st[r] = zero;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[r][dt] = zero;
  }
  auto scores = [&](uint32_t at, int s0, int s1) {
#pragma unroll
    for (int s = s0; s < s1; ++s) {
      const u32x4 kf = *reinterpret_cast<const u32x4*>(smem + at + (kr ^ (32 * s)));
#pragma unroll
      for (int r = 0; r < NR; ++r) st[r] = Mfma<T>::go(kf, qf[r][s], st[r]);
    }
  };
  auto block = [&](uint32_t kat, uint32_t vat, int kb) {      // kb: the wave's first key
    f32x16 sc[NR];
    float sub[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if (kb + 31 > min(wmin[r], kend - 1)) {                 // some row attends part of these keys only (uniform)
        const int last = min(pr[r], kend - 1) - kb - 4 * h;   // a key at or below it counts
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (8 * (v >> 2) + (v & 3) > last) st[r][v] = -INFINITY;
      }
      float bm = st[r][0];
#pragma unroll
      for (int v = 1; v < 16; ++v) bm = fmaxf(bm, st[r][v]);
      if (__any(bm * c2 > ref[r] + kLag)) {                   // (uniform; either lane of a row)
        const float nm = fmaxf(ref[r], fmaxf(bm, __shfl_xor(bm, 32, 64)) * c2);   // -inf while the row has seen no key
        const float corr = nm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref[r] - nm);
        ref[r] = nm;
        lsum[r] *= corr;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[r][dt] *= corr;
      }
      sub[r] = ref[r] == -INFINITY ? 0.f : ref[r] - (15.f - kLag);
      sc[r] = st[r];
      st[r] = zero;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {                             // 16 keys
      u32x4 ph[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        float ps[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[r][8 * s + 2 * i], c2, -sub[r]));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[r][8 * s + 2 * i + 1], c2, -sub[r]));
          ps[0] += p0;
          ps[1] += p1;
          ph[r][i] = Mfma<T>::pack(p0, p1);
        }
        lsum[r] += ps[0] + ps[1];
      }
      scores(kat, KS / 2 * s, KS / 2 * s + KS / 2);           // of the next block (past the last one: zeros, not used)
      u32x4 va[DT];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) va[dt] = v_frag(vat + (vr ^ (64 * dt)) + 16 * RB * s);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < NR; ++r) o[r][dt] = Mfma<T>::go(va[dt], ph[r], o[r][dt]);
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
    Pages pg = pages_of(b0);
    load(k_cache, pg, b0, slot(0), true);
#pragma unroll
    for (int t = 0; t < AH; ++t) {
      load(v_cache, pg, b0 + t, kV + slot(t), false);
      pg = pages_of(b0 + t + 1);
      load(k_cache, pg, b0 + t + 1, slot((t + 1) % N), true);
    }
    sync(std::integral_constant<int, 2 * NP * AH>{});
    if (busy) scores(slot(0), 0, KS);
    sync(std::integral_constant<int, 2 * NP * (AH - 1)>{});
    int a = 0;                                                // i % N
    for (int i = b0; i < b1; ++i) {
      const int a1 = a + 1 == N ? 0 : a + 1, am = a == 0 ? N - 1 : a - 1;
      load(v_cache, pg, i + AH, kV + slot(am), false);
      pg = pages_of(i + 1 + AH);
      load(k_cache, pg, i + 1 + AH, slot(a), true);
      if (busy) block(slot(a1), slot(a), i * BK + 32 * kgrp);
      sync(std::integral_constant<int, 2 * NP * (AH - 1)>{});
      a = a1;
    }
    lds_wait_barrier<0>();                                    // nothing is left in flight, and the slots may be reused
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) lsum[r] += __shfl_xor(lsum[r], 32, 64);
  if constexpr (KG > 1) {                                     // the key groups' sums, through LDS, into key group 0
    static_assert(NR == 1, "one row group a wave");
    constexpr int kRec = (D / 2 + 2) * 64 * 4;
    float* mine = reinterpret_cast<float*>(smem + (size_t)((kgrp - 1) * RG + rgrp) * kRec) + lane;
    if (kgrp > 0) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; ++v) mine[64 * (16 * dt + v)] = o[0][dt][v];
      mine[64 * (D / 2)] = ref[0];
      mine[64 * (D / 2 + 1)] = lsum[0];
    }
    lds_barrier();
    if (kgrp > 0) return;
    for (int g2 = 1; g2 < KG; ++g2) {
      const float* theirs = reinterpret_cast<const float*>(smem + (size_t)((g2 - 1) * RG + rgrp) * kRec) + lane;
      const float r2 = theirs[64 * (D / 2)], nm = fmaxf(ref[0], r2);
      const float f0 = ref[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref[0] - nm);
      const float f1 = r2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r2 - nm);
      ref[0] = nm;
      lsum[0] = lsum[0] * f0 + theirs[64 * (D / 2 + 1)] * f1;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[0][dt][v] = o[0][dt][v] * f0 + theirs[64 * (16 * dt + v)] * f1;
    }
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (!live[r]) continue;
    // lane (j, h) holds O^T[32 dt + 8 (v / 4) + 4 h + v % 4][row j]
    if (un.parts == 1) {
      const bool some = pr[r] >= 0;                           // a row without a key: zeros
      const float inv = some ? 1.f / lsum[r] : 0.f;
      T* dst = out + qrow[r] + 4 * h;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
          const uint32_t lo = some ? Mfma<T>::pack(o[r][dt][v] * inv, o[r][dt][v + 1] * inv) : 0u;
          const uint32_t hi = some ? Mfma<T>::pack(o[r][dt][v + 2] * inv, o[r][dt][v + 3] * inv) : 0u;
          *reinterpret_cast<uint2*>(dst + 32 * dt + 2 * v) = make_uint2(lo, hi);
        }
    } else {
      float* rec = part + ((size_t)un.rec * kRows + 32 * (NR * rgrp + r) + j) * paged_rec<D>();
      if (h == 0) {
        rec[0] = ref[r];
        rec[1] = lsum[r];
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; v += 4)
          *reinterpret_cast<f32x4*>(rec + 4 + 32 * dt + 2 * v + 4 * h) = f32x4{o[r][dt][v], o[r][dt][v + 1], o[r][dt][v + 2], o[r][dt][v + 3]};
    }
  }
}

// The outputs of the split tiles: a workgroup takes tile blockIdx.x of them and 1024 / D of its rows, D / 4 lanes a row; the
// parts are joined in order, their weights 2^(reference - largest reference) against the sum's.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_attention_merge(const float* __restrict__ part, PagedBatch bt, PagedPlan plan,
                                                             T* __restrict__ out, int Hq, int Hkv) {
  constexpr int kLanes = D / 4, kRowsHere = 256 / kLanes, kRec = paged_rec<D>();
  const int G = Hq / Hkv;
  PagedUnit un;
  if (!paged_unit<true>(bt, plan, G, Hkv, blockIdx.x, threadIdx.x & 63, un)) return;
  const int r = blockIdx.y * kRowsHere + threadIdx.x / kLanes, d = 4 * (threadIdx.x % kLanes);
  const int row = un.tile * plan.rows + r, tok = row / G, g = row - tok * G;
  if (row >= un.nq * G) return;
  const float* rec = part + ((size_t)un.rec * plan.rows + r) * kRec;
  const size_t step = (size_t)plan.rows * kRec;
  float top = -INFINITY;
  for (int p = 0; p < un.parts; ++p) top = fmaxf(top, rec[p * step]);
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
  float den = 0.f;
  for (int p0 = 0; p0 < un.parts; p0 += 8) {                  // eight records' loads in flight
    f32x4 v[8];
    float m[8], l[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float* at = rec + (size_t)min(p0 + i, un.parts - 1) * step;
      m[i] = at[0];
      l[i] = at[1];
      v[i] = *reinterpret_cast<const f32x4*>(at + 4 + d);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (p0 + i >= un.parts || m[i] == -INFINITY) continue;  // (a part that saw no key)
      const float f = __builtin_amdgcn_exp2f(m[i] - top);
      den = fmaf(f, l[i], den);
#pragma unroll
      for (int e = 0; e < 4; ++e) num[e] = fmaf(f, v[i][e], num[e]);
    }
  }
  const bool some = un.len - un.nq + tok >= 0;                // a row without a key: zeros
  const float inv = some ? 1.f / den : 0.f;
  T* dst = out + ((int64_t)(un.first + tok) * Hq + un.hk * G + g) * D + d;
  *reinterpret_cast<uint2*>(dst) = some ? make_uint2(Mfma<T>::pack(num[0] * inv, num[1] * inv), Mfma<T>::pack(num[2] * inv, num[3] * inv)) : make_uint2(0u, 0u);
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

constexpr int kPagedParts = 256;                             // of a tile at most
constexpr int kPagedLeast = 256;                             // keys of a part at least

template <typename T, int D, int RG, int KG, int NR>
hipError_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t st) {
  constexpr size_t lds = paged_lds<D, RG, KG>();
  const int G = a.Hq / a.Hkv;
  PagedPlan p{32 * NR * RG, 32 * KG, 256 * (KG == 4 || NR > 1 ? 1 : 2), 0, 1, 0};
  p.least = std::max(1, kPagedLeast / p.block);
  const int64_t units = (((int64_t)a.batch.T * G + p.rows - 1) / p.rows + std::min(a.batch.B, a.batch.T)) * a.Hkv;
  const size_t group = (size_t)p.rows * paged_rec<D>() * sizeof(float);
  p.most = (int)std::min<size_t>(3 * (size_t)p.slots, a.ws_bytes / group);
  if (a.ws && p.most >= 2)
    p.cap = std::min(kPagedParts, (int)((((int64_t)a.max_keys + p.block - 1) / p.block + p.least - 1) / p.least));
  const int64_t grid = p.cap == 1 ? units : std::min<int64_t>(units * p.cap, units + p.most / 2 + 1);
  if (lds > 65536) {
    static std::atomic<uint64_t> done{0};
    if (hipError_t e = allow_lds_once(done, paged_attention<T, D, RG, KG, NR>, lds)) return e;
  }
  int shift = 0;
  while ((1 << shift) < a.batch.page_size) ++shift;
  hipError_t e = launch(paged_attention<T, D, RG, KG, NR>, dim3((unsigned)grid), dim3(256), lds, st,
                        static_cast<const T*>(a.q), static_cast<const T*>(a.k_cache), static_cast<const T*>(a.v_cache),
                        a.batch, p, static_cast<T*>(a.out), static_cast<float*>(a.ws), a.Hq, a.Hkv, shift, a.scale);
  if (e != hipSuccess || p.cap == 1) return e;
  const int64_t split = std::min<int64_t>(units, p.most / 2 + 1);
  return launch(paged_attention_merge<T, D>, dim3((unsigned)split, (unsigned)(p.rows * D / 1024)), dim3(256), 0, st,
                static_cast<const float*>(a.ws), a.batch, p, static_cast<T*>(a.out), a.Hq, a.Hkv);
}

template <typename T, int D>
hipError_t pick_paged_attention(const PagedAttentionArgs& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.max_new * (a.Hq / a.Hkv);
  if (rows <= 32) return launch_paged_attention<T, D, 1, 4, 1>(a, st);
  return launch_paged_attention<T, D, 4, 1, 1>(a, st);
}

}  // namespace

hipError_t norm_rope_paged_launch(const NormRopeArgs& a, hipStream_t st) {
  if (a.bf16) return a.D == 64 ? launch_norm_rope<bf16, 64>(a, st) : launch_norm_rope<bf16, 128>(a, st);
  return a.D == 64 ? launch_norm_rope<f16, 64>(a, st) : launch_norm_rope<f16, 128>(a, st);
}

hipError_t attention_paged_launch(const PagedAttentionArgs& a, hipStream_t st) {
  if (a.bf16) return a.D == 64 ? pick_paged_attention<bf16, 64>(a, st) : pick_paged_attention<bf16, 128>(a, st);
  return a.D == 64 ? pick_paged_attention<f16, 64>(a, st) : pick_paged_attention<f16, 128>(a, st);
}

}  // namespace lowbit
