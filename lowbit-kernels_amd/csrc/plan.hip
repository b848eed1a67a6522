// The tables of a batch's step over a paged KV cache, built on the GPU from its sequences' lengths (plan_paged), and what becomes
// of a tree of drafted tokens once the model has picked its own (accept_drafts). Both are whole numbers and copies of rows of the
// cache; a step of a captured graph runs them without the host.
//
// plan_paged. Sequence b goes on from row r = rows[b] of the table: its past[r] keys lie in the row's first ceil(past / page
// size) pages, which it keeps. A page is in use while a sequence keeps it, free otherwise: no counts are carried from step to
// step, so nothing leaks when a sequence ends, a draft is rejected or a beam gives way. The free pages, in order, go to the
// sequences, in order. A page that a sequence is about to write (its last one, partly filled) and that another one reads is
// replaced by a copy first; of several sequences that could write it, the one with the most keys, then the first, keeps it.
#include "paged_attention.hpp"

namespace lowbit {

namespace {

constexpr int kThreads = 1024;
constexpr int kMasksPer = 4;             // words of 32 pages that a thread looks through in a later step of the search for free pages
// what one workgroup plans alone, its state in LDS
constexpr int kSmallSeqs = 1024, kSmallTokens = 4096, kSmallList = kSmallTokens / 16 + 2 * kSmallSeqs;
constexpr int kSmallPages = 1 << 18, kSmallEntries = 1 << 15;
constexpr int kHashSeqs = 1024;          // sequences whose hash lies in LDS
constexpr int kStartSeqs = 4096;         // sequences whose starts every workgroup copies to LDS
constexpr int kFinishTokens = 8192;      // tokens that the workgroup which hands out the pages numbers too
constexpr int kMostNodes = 64 * kMaxMaskWords;   // of a tree: later ones are attended by none

// The state of a call, in LDS or in the workspace: [B] each but off and start ([B + 1])
struct PlanState {
  int *row, *past, *fresh, *tail, *off, *start;   // tail: the last page kept; off: its first place in the list, ~off if that is a copy
  uint32_t* used;                                 // LDS: a bit a page, workspace: a byte: kept (while pages are marked: kept and full)
  int* hash_page;                                 // the pages that are partly filled, and whose they are (owner_key)
  uint64_t* hash_owner;
  int hash_mask;
  int* list;                                      // the free pages handed out, -1 where they ran out
  int list_cap;
};

__device__ __forceinline__ int pages_of(int keys, int shift) { return (keys + (1 << shift) - 1) >> shift; }

template <bool kLds>
__device__ __forceinline__ void use_page(const PlanState& s, int page) {
  if constexpr (kLds)
    atomicOr(s.used + (page >> 5), 1u << (page & 31));
  else
    reinterpret_cast<uint8_t*>(s.used)[page] = 1;             // (all writers write the same: no atomics)
}
template <bool kLds>
__device__ __forceinline__ bool page_used(const PlanState& s, int page) {
  if constexpr (kLds) return s.used[page >> 5] >> (page & 31) & 1u;
  return reinterpret_cast<const uint8_t*>(s.used)[page];
}
// pages 32 w .. + 31 that are free, a bit each
template <bool kLds>
__device__ __forceinline__ uint32_t free_pages(const PlanState& s, int w) {
  if constexpr (kLds) return ~s.used[w];
  const u32x4 a = load16(s.used + 8 * (int64_t)w), b = load16(s.used + 8 * (int64_t)w + 4);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t t = ~(i < 4 ? a[i & 3] : b[i & 3]) & 0x01010101u;
    m |= ((t | t >> 7 | t >> 14 | t >> 21) & 0xFu) << (4 * i);
  }
  return m;
}

// of the sequences that hold a partly filled page: the most keys, then one that writes, then the first
__device__ __forceinline__ uint64_t owner_key(int past, int fresh, int b) {
  return ((uint64_t)(uint32_t)past << 32) | (fresh > 0 ? 0x80000000u : 0u) | (uint32_t)(0x7FFFFFFF - b);
}
__device__ __forceinline__ int hash_slot(int page, int mask) { return (int)(((uint32_t)page * 2654435761u) >> 7) & mask; }

// sequence b's partly filled last page, if it has one
__device__ __forceinline__ int part_page(const PlanArgs& a, int shift, int past, int tail) {
  return (past & ((1 << shift) - 1)) && tail >= 0 && tail < a.pages ? tail : -1;
}

// the last b with of(b) <= v, of not falling and of(0) <= v
template <typename F>
__device__ __forceinline__ int last_at(int n, int v, F of) {
  int lo = 0;
  for (int hi = n; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if (of(mid) <= v)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Sums over the threads of a workgroup, held at `most` (values 0 .. most): of those before a thread and of all. s_wave has two rows,
// taken in turn, so that one barrier a sum is enough.
struct Scan {
  int before, all;
};
struct ScanWaves {
  int at[2][16];                                              // (zeros before: a smaller workgroup has fewer waves)
};
__device__ __forceinline__ Scan block_scan(int v, int most, ScanWaves& s, int& turn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int* at = s.at[turn];
  turn ^= 1;
  // (as wave_scan adds them, held at `most` in every step)
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false), most);
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false), most);
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false), most);
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false), most);
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false), most);
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false), most);
  if (lane == 63) at[wave] = v;
  const int ahead = __builtin_amdgcn_update_dpp(0, v, 0x138, 0xF, 0xF, false);   // wave_shr 1
  lds_barrier();
  int w[16], before = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < 16; i += 4) *reinterpret_cast<u32x4*>(w + i) = *reinterpret_cast<const u32x4*>(at + i);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    before = i == wave ? sum : before;
    sum = min(sum + w[i], most);
  }
  return {min(before + ahead, most), sum};
}

// q_starts, kv_lens and the sequences' lengths, by one workgroup
__device__ __forceinline__ void plan_lens(const PlanArgs& a, const PlanState& s, int shift, ScanWaves& s_wave, int& turn) {
  int done = 0;
  for (int b0 = 0; b0 < a.B; b0 += (int)blockDim.x) {
    const int b = b0 + threadIdx.x;
    int row = -1, past = 0, fresh = 0;
    if (b < a.B) {
      row = a.rows ? a.rows[b] : b;
      fresh = min(max(a.fresh[b], 0), a.T);
      if (row >= 0 && row < a.R) past = min(max(a.past[row], 0), a.width << shift);
    }
    const Scan sum = block_scan(fresh, a.T, s_wave, turn);
    if (b < a.B) {
      const int first = min(done + sum.before, a.T), upto = min(first + fresh, a.T);   // (held at T: tokens past it are left out)
      s.start[b + 1] = upto;
      a.q_starts[b + 1] = upto;
      s.row[b] = row;
      s.past[b] = past;
      s.tail[b] = -1;
      s.fresh[b] = upto - first;
      a.kv_lens[b] = past + upto - first;
      if (b == 0) {
        s.start[0] = 0;
        a.q_starts[0] = 0;
      }
    }
    done = min(done + sum.all, a.T);
  }
}

// Which sequences get how many of the free pages, and which pages those are, by one workgroup. The hash is empty before. s_free: a word
// of each step's pages (zeros before); s_before: how many free ones come before a thread's.
// The workspace's bytes of the first 32768 pages are asked for at once, before those of the last pages are marked: s_free has
// a bit for each of these.
template <bool kLds>
__device__ __forceinline__ void plan_assign(const PlanArgs& a, const PlanState& s, int shift, ScanWaves& s_wave, int& turn,
                                            int* s_over, uint32_t* s_free, int* s_before) {
  const int tid = threadIdx.x, threads = blockDim.x, words = (int)((a.pages + 31) >> 5);
  const bool far = !kLds && a.B > kHashSeqs;                  // the hash lies in the workspace
  auto mask = [&](int w) {
    const int64_t left = a.pages - 32 * (int64_t)w;
    return w < words ? free_pages<kLds>(s, w) & (left >= 32 ? ~0u : (1u << left) - 1u) : 0u;
  };
  uint32_t first_mask = 0;
  if constexpr (!kLds) first_mask = mask(tid);
  if (tid == 0) *s_over = 0;
  // a thread's first sequence in registers
  int past0 = 0, fresh0 = 0, tail0 = -1;
  if (tid < a.B) {
    past0 = s.past[tid];
    fresh0 = s.fresh[tid];
    tail0 = s.tail[tid];
  }
  auto sequence = [&](int b, int& past, int& fresh, int& page) {
    const bool first = b == tid;
    past = first ? past0 : s.past[b];
    fresh = first ? fresh0 : s.fresh[b];
    page = part_page(a, shift, past, first ? tail0 : s.tail[b]);
  };
  for (int b = tid; b < a.B; b += threads) {
    int past, fresh, page;
    sequence(b, past, fresh, page);
    if (page < 0) continue;
    for (int at = hash_slot(page, s.hash_mask);; at = (at + 1) & s.hash_mask) {   // (twice as many places as sequences)
      const int was = atomicCAS(s.hash_page + at, -1, page);
      if (was != -1 && was != page) continue;
      atomicMax(reinterpret_cast<unsigned long long*>(s.hash_owner) + at, (unsigned long long)owner_key(past, fresh, b));
      break;
    }
  }
  if (far) vm_drain();                                        // (the owners, which other waves read behind the barrier)
  lds_barrier();
  // (in the workspace: past the L1, which the atomics above pass by)
  auto hash_page = [&](int at) {
    return far ? __hip_atomic_load(s.hash_page + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : s.hash_page[at];
  };
  auto hash_owner = [&](int at) {
    return far ? __hip_atomic_load(s.hash_owner + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : s.hash_owner[at];
  };
  int total = 0;
  for (int b0 = 0; b0 < a.B; b0 += threads) {
    const int b = b0 + tid;
    int want = 0;
    bool copy = false;
    if (b < a.B) {
      int past, fresh, page;
      sequence(b, past, fresh, page);
      const int have = pages_of(past, shift), need = pages_of(past + fresh, shift);
      if (fresh > 0 && page >= 0) {
        copy = page_used<kLds>(s, page);                      // (within another's keys)
        int at = hash_slot(page, s.hash_mask);
        while (hash_page(at) != page) at = (at + 1) & s.hash_mask;
        copy |= hash_owner(at) != owner_key(past, fresh, b);
      }
      want = min(need, a.width) - have + (copy ? 1 : 0);
      if (need > a.width) atomicAdd(s_over, need - a.width);  // pages that the table has no place for
    }
    const Scan sum = block_scan(want, INT_MAX / 2, s_wave, turn);
    if (b < a.B) s.off[b] = copy ? ~(total + sum.before) : total + sum.before;
    total += sum.all;
  }
  total = min(total, s.list_cap);
  // (every sequence has looked for its page among the full ones: the barrier of the last sum)
  for (int b = tid; b < a.B; b += threads) {
    int past, fresh, page;
    sequence(b, past, fresh, page);
    if (page < 0) continue;
    if (kLds || page >= 32 * threads)
      use_page<kLds>(s, page);
    else
      atomicOr(s_free + (page >> 5), 1u << (page & 31));
  }
  __syncthreads();
  int found = 0, per = 1;
  for (int w0 = 0; w0 < words && found < total; w0 += threads * per, per = kMasksPer) {
    if (w0 > 0) lds_barrier();                                // (the step before has been read)
    int n = 0;
    for (int i = 0; i < per; ++i) {
      const uint32_t m = kLds || w0 > 0 ? mask(w0 + tid * per + i) : first_mask & ~s_free[tid];
      s_free[tid * per + i] = m;
      n += __popc(m);
    }
    const Scan sum = block_scan(n, INT_MAX / 2, s_wave, turn);
    s_before[tid] = sum.before;
    lds_barrier();
    // a thread a page: whose words hold it, then which bit it is
    for (int j = tid; j < min(sum.all, total - found); j += threads) {
      const int t = last_at(threads, j, [&](int i) { return s_before[i]; });
      int rest = j - s_before[t], w = t * per;
      for (int c = __popc(s_free[w]); rest >= c; c = __popc(s_free[w])) {
        rest -= c;
        ++w;
      }
      uint32_t m = s_free[w];
      int bit = 0;
#pragma unroll
      for (int half = 16; half > 0; half >>= 1) {
        const int c = __popc(m & ((1u << half) - 1u));
        if (rest >= c) {
          rest -= c;
          m >>= half;
          bit += half;
        }
      }
      s.list[found + j] = 32 * (w0 + w) + bit;
    }
    found = min(found + sum.all, total);
  }
  for (int i = found + tid; i < total; i += threads) s.list[i] = -1;
  if (tid == 0) {
    *a.missing = *s_over + total - found;
    s.off[a.B] = total;
  }
}

__device__ __forceinline__ int off_of(int v) { return v < 0 ? ~v : v; }

// place j of the list: into the table
__device__ __forceinline__ void give_page(const PlanArgs& a, const PlanState& s, int shift, int j) {
  const int b = last_at(a.B, j, [&](int i) { return off_of(s.off[i]); });
  const int off = s.off[b], first = off_of(off), have = pages_of(s.past[b], shift);
  a.table_out[(int64_t)b * a.width + have + (j - first) - (off < 0 ? 1 : 0)] = s.list[j];
}
__device__ __forceinline__ void give_copy(const PlanArgs& a, const PlanState& s, int shift, int b) {
  const bool copy = s.off[b] < 0;
  const int have = pages_of(s.past[b], shift);
  if (!copy && have > 0 && a.table_out != a.table) a.table_out[(int64_t)b * a.width + have - 1] = s.tail[b];
  a.copies[2 * b] = copy ? s.tail[b] : -1;
  a.copies[2 * b + 1] = copy ? s.list[~s.off[b]] : -1;
}

// token t's position, slot and mask; parent: of node i of its sequence
template <typename P>
__device__ __forceinline__ void give_token(const PlanArgs& a, const PlanState& s, int shift, int t, P parent) {
  if (t >= s.start[a.B]) {                                    // (a padded token)
    a.positions[t] = 0;
    a.slots[t] = -1;
    for (int w = 0; w < a.words; ++w) a.masks[(int64_t)t * a.words + w] = 0;
    return;
  }
  const int b = last_at(a.B, t, [&](int i) { return s.start[i]; });
  const int first = s.start[b], i = t - first, past = s.past[b], key = past + i;
  const int have = pages_of(past, shift), off = s.off[b], c = key >> shift;
  int page = -1;
  if (c < have && off >= 0)
    page = s.tail[b];                                         // (key >= past: of the pages kept, the last)
  else if (c < a.width)
    page = s.list[off_of(off) + c - have + (off < 0 ? 1 : 0)];
  a.slots[t] = page >= 0 && page < a.pages ? ((int64_t)page << shift) + (key & ((1 << shift) - 1)) : -1;
  if (!a.parents) {
    a.positions[t] = key;
    return;
  }
  // up to the root, each word's nodes in turn (a node hangs below an earlier one); past the words' most nodes there is no tree
  int depth = 0, n = i < kMostNodes ? i : -1;
  for (int w = a.words - 1; w >= 0; --w) {
    uint64_t bits = 0;
    while (n >= 64 * w) {
      if (n >> 6 == w) bits |= (uint64_t)1 << (n & 63);
      const int p = parent(first, n);
      if (p < 0 || p >= n) {
        n = -1;
        break;
      }
      n = p;
      ++depth;
    }
    a.masks[(int64_t)t * a.words + w] = bits;
  }
  a.positions[t] = past + depth;
}

}  // namespace

// The whole plan by one workgroup: what it takes is its chain of round trips to memory and of barriers (a tree of 26 tokens 6.8 us, 128
// beams' rows of 141 pages 12.4). Up to kSmallEntries table entries, which one CU reads as fast as the launches beyond take.
__global__ __launch_bounds__(kThreads) void plan_small_kernel(PlanArgs a, int lanes_log, int shift, int hash_mask) {
  extern __shared__ __attribute__((aligned(16))) uint32_t s_plan[];
  __shared__ __attribute__((aligned(16))) ScanWaves s_wave;
  __shared__ int s_over, s_before[kThreads];
  __shared__ uint32_t s_free[kThreads * kMasksPer];
  int turn = 0;
  const int tid = threadIdx.x, threads = blockDim.x, words = ((int)((a.pages + 31) >> 5) + 3) & ~3;
  PlanState s;
  s.hash_mask = hash_mask;
  s.list_cap = kSmallList;
  s.hash_owner = reinterpret_cast<uint64_t*>(s_plan);
  s.used = reinterpret_cast<uint32_t*>(s.hash_owner + hash_mask + 1);
  s.hash_page = reinterpret_cast<int*>(s.used + words);
  s.row = s.hash_page + hash_mask + 1;
  s.past = s.row + a.B;
  s.fresh = s.past + a.B;
  s.tail = s.fresh + a.B;
  s.off = s.tail + a.B;
  s.start = s.off + a.B + 1;
  s.list = s.start + a.B + 1;
  int* s_parent = s.list + kSmallList;
  if (a.parents)
    for (int i = tid; i < a.T; i += threads) s_parent[i] = a.parents[i];
  if (tid < 32) s_wave.at[0][tid] = 0;
  for (int i = tid; i < 2 * (hash_mask + 1) + words; i += threads) s_plan[i] = 0;
  for (int i = tid; i <= hash_mask; i += threads) s.hash_page[i] = -1;
  lds_barrier();
  plan_lens(a, s, shift, s_wave, turn);
  lds_barrier();
  const bool other = a.table_out != a.table;
  // 2^lanes_log threads a row, four rows and four pieces of each in flight
  const int lanes = 1 << lanes_log, step = threads >> lanes_log, c1 = tid & (lanes - 1);
  constexpr int kAhead = 4;
  for (int b0 = tid >> lanes_log; b0 < a.B; b0 += kAhead * step) {
    int past[kAhead];
    int64_t row[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int b = b0 + u * step;
      past[u] = b < a.B ? s.past[b] : 0;
      row[u] = b < a.B ? (int64_t)s.row[b] * a.width : 0;
    }
    for (int c0 = c1; c0 < a.width; c0 += kAhead * lanes) {
      int page[kAhead][kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int c = c0 + i * lanes;
          page[u][i] = -1;
          if (c < pages_of(past[u], shift)) page[u][i] = a.table[row[u] + c];
        }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int b = b0 + u * step;
        if (b >= a.B) break;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int c = c0 + i * lanes, got = page[u][i];
          if (c >= a.width) break;
          const bool last = c == pages_of(past[u], shift) - 1;
          if (last) s.tail[b] = got;
          if (c < past[u] >> shift && got >= 0 && got < a.pages) use_page<true>(s, got);
          if (other && !last) a.table_out[b * a.width + c] = got;   // (the last page kept, or its copy: below)
        }
      }
    }
  }
  lds_barrier();
  plan_assign<true>(a, s, shift, s_wave, turn, &s_over, s_free, s_before);
  lds_barrier();
  for (int j = tid; j < s.off[a.B]; j += threads) give_page(a, s, shift, j);
  for (int b = tid; b < a.B; b += threads) give_copy(a, s, shift, b);
  for (int t = tid; t < a.T; t += threads) give_token(a, s, shift, t, [&](int first, int n) { return s_parent[first + n]; });
}

// The same in three launches, the state in the workspace: the lengths, beside the clearing of what the pages are marked in; the pages
// kept, 1024 entries of a row a workgroup; the pages handed out, tables and tokens. 256 sequences on 300 .. 30000 keys in pages of 16,
// 4500 tokens: 2.3, 4.3 and 11.1 us, the chain of round trips of one workgroup (its bytes would take 0.5). Beyond kFinishTokens or
// kHashSeqs the tables and tokens take a launch of their own (6.2 and 4.1 us here, and one launch more of the host's). The pages handed
// out by the last workgroup that marks, whose marks then go past the L2: 17.9 us for both, not kept.
__global__ __launch_bounds__(kThreads) void plan_lens_kernel(PlanArgs a, PlanState s, int shift, int64_t clear) {
  __shared__ __attribute__((aligned(16))) ScanWaves s_wave;
  int turn = 0;
  if (blockIdx.x == 0) {
    if (threadIdx.x < 32) s_wave.at[0][threadIdx.x] = 0;
    lds_barrier();
    plan_lens(a, s, shift, s_wave, turn);
    return;
  }
  const int64_t step = (int64_t)(gridDim.x - 1) * kThreads, at = (int64_t)(blockIdx.x - 1) * kThreads + threadIdx.x;
  u32x4* zero = reinterpret_cast<u32x4*>(s.used);             // (the owners of a hash in the workspace follow)
  for (int64_t i = at; i < clear; i += step) zero[i] = u32x4{0u, 0u, 0u, 0u};
  if (s.hash_page)
    for (int64_t i = at; i <= s.hash_mask; i += step) s.hash_page[i] = -1;
}

__global__ __launch_bounds__(256) void plan_mark_kernel(PlanArgs a, PlanState s, int chunks, int shift) {
  const int b = blockIdx.x / chunks, c0 = (blockIdx.x - b * chunks) * 1024 + threadIdx.x;
  const int row = s.row[b], past = s.past[b], have = pages_of(past, shift);
  const bool other = a.table_out != a.table;
  int page[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) page[u] = c0 + 256 * u < have ? a.table[(int64_t)row * a.width + c0 + 256 * u] : -1;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int c = c0 + 256 * u;
    if (c == have - 1) s.tail[b] = page[u];
    if (c < past >> shift && page[u] >= 0 && page[u] < a.pages) use_page<false>(s, page[u]);
    if (other && c < a.width && c != have - 1) a.table_out[(int64_t)b * a.width + c] = page[u];
  }
}

__global__ __launch_bounds__(kThreads) void plan_assign_kernel(PlanArgs a, PlanState s, int shift, bool finish) {
  extern __shared__ __attribute__((aligned(16))) uint32_t s_plan[];
  __shared__ __attribute__((aligned(16))) ScanWaves s_wave;
  __shared__ int s_over, s_before[kThreads];
  __shared__ uint32_t s_free[kThreads * kMasksPer];
  int turn = 0;
  s_free[threadIdx.x] = 0;
  if (threadIdx.x < 32) s_wave.at[0][threadIdx.x] = 0;
  if (!s.hash_page) {
    s.hash_owner = reinterpret_cast<uint64_t*>(s_plan);
    s.hash_page = reinterpret_cast<int*>(s.hash_owner + s.hash_mask + 1);
    for (int i = threadIdx.x; i <= s.hash_mask; i += kThreads) {
      s.hash_owner[i] = 0;
      s.hash_page[i] = -1;
    }
    if (finish) {                                             // what the searches read, in LDS
      int* copy = s.hash_page + s.hash_mask + 1;
      for (int i = threadIdx.x; i <= a.B; i += kThreads) copy[i] = s.start[i];
      s.start = copy;
      s.off = copy + a.B + 1;
    }
  }
  __syncthreads();
  plan_assign<false>(a, s, shift, s_wave, turn, &s_over, s_free, s_before);
  if (!finish) return;
  __syncthreads();
  for (int j = threadIdx.x; j < s.off[a.B]; j += kThreads) give_page(a, s, shift, j);
  for (int b = threadIdx.x; b < a.B; b += kThreads) give_copy(a, s, shift, b);
  for (int t = threadIdx.x; t < a.T; t += kThreads)
    give_token(a, s, shift, t, [&](int first, int n) { return a.parents[first + n]; });
}

__global__ __launch_bounds__(256) void plan_fill_kernel(PlanArgs a, PlanState s, int shift) {
  extern __shared__ __attribute__((aligned(16))) uint32_t s_plan[];
  if (a.B <= kStartSeqs) {                                    // the searches' arrays
    int* copy = reinterpret_cast<int*>(s_plan);
    for (int i = threadIdx.x; i <= a.B; i += 256) {
      copy[i] = s.start[i];
      copy[a.B + 1 + i] = s.off[i];
    }
    s.start = copy;
    s.off = copy + a.B + 1;
    __syncthreads();
  }
  const int step = gridDim.x * 256, at = blockIdx.x * 256 + threadIdx.x;
  const int total = s.off[a.B];
  for (int j = at; j < total; j += step) give_page(a, s, shift, j);
  for (int b = at; b < a.B; b += step) give_copy(a, s, shift, b);
  for (int t = at; t < a.T; t += step)
    give_token(a, s, shift, t, [&](int first, int n) { return a.parents[first + n]; });
}

// Workgroup (sequence, layer): the filled rows of the page that is replaced, every head of k and v. Bound: memory and the
// launch (some 45 of 128 beams, 28 layers, 2 heads of 128, 19 MB read and written: 4.4 .. 6 us, 4.1 at a large copy's rate).
__global__ __launch_bounds__(256) void plan_copy_kernel(const int* __restrict__ copies, const int* __restrict__ q_starts,
                                                        const int* __restrict__ kv_lens, uint8_t* __restrict__ k,
                                                        uint8_t* __restrict__ v, int64_t pages, int Hkv, int row_bytes, int shift) {
  const int b = blockIdx.x, src = copies[2 * b], dst = copies[2 * b + 1];
  const int rows = (kv_lens[b] - (q_starts[b + 1] - q_starts[b])) & ((1 << shift) - 1);
  if (src < 0 || dst < 0) return;
  const int64_t head = (int64_t)row_bytes << shift, page = head * Hkv, layer = (int64_t)blockIdx.y * pages;
  const int vec = rows * (row_bytes / 16), n = vec * Hkv;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int h = i / vec, at = i - h * vec;
    const int64_t from = (layer + src) * page + h * head + 16 * (int64_t)at, to = (layer + dst) * page + h * head + 16 * (int64_t)at;
    const u32x4 x = load16(k + from), y = load16(v + from);
    *reinterpret_cast<u32x4*>(k + to) = x;
    *reinterpret_cast<u32x4*>(v + to) = y;
  }
}

// accept_drafts. Workgroup (sequence, layer): its first wave follows the picks from node 0 down the tree (the first 64 nodes in its
// lanes, a ballot a step), then the workgroup moves the confirmed nodes' rows of its layer, every head of k and v, to the places
// behind the sequence's keys: one launch, the walk repeated in every layer. Node d of the path comes to lie at place d <= the node's
// own, so rows are read and written in order of the path, a chunk's all read before one is written.
// Bound: without moves the chain of round trips (one tree of 26 4.4 us, 64 trees 3.8); with them the chain walk, table, rows, stores,
// which every workgroup of the one round goes through: 64 trees, 28 layers, 26 MB read and written, 14.6 us, 1.8 TB/s (several layers
// a workgroup 16.6). Waves wait 63% of their cycles; 2100 of 410000 address translations miss, so scattered rows are not it.
constexpr int kMostPath = 1024;
__device__ __forceinline__ int64_t readlane64(int64_t v, int lane) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
                   (uint32_t)__builtin_amdgcn_readlane((int)v, lane));
}
__global__ __launch_bounds__(256) void accept_kernel(AcceptArgs a, int shift) {
  __shared__ int s_path[kMostPath], s_table[64];
  __shared__ int s_count;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int first = min(max(a.q_starts[b], 0), a.T), nodes = min(max(a.q_starts[b + 1], first), a.T) - first;
  const int past = a.kv_lens[b] - nodes, tree = min(nodes, kMostNodes);
  const int* table = a.table + (int64_t)b * a.width;
  const int c0 = max(past, 0) >> shift;                       // s_table: the entries from there on
  if (tid < 64) {
    const int64_t* tokens = a.tokens + first;
    const int64_t* picks = a.picks + first;
    const int* parents = a.parents ? a.parents + first : nullptr;
    int64_t token = 0, pick = 0;
    int parent = -1;
    if (lane < tree) {
      token = tokens[lane];
      pick = picks[lane];
      parent = parents ? parents[lane] : lane - 1;
    }
    // (a token below 0 cannot be confirmed: no node's child, and nothing if it is node 0's)
    parent = token < 0 ? -1 : parent;
    int count = 0, cur = __builtin_amdgcn_readlane((int)(token >> 32), 0) < 0 ? tree : 0;
    while (count < a.longest && cur < tree) {
      if (lane == 0) s_path[count] = cur;
      ++count;
      const int64_t want = cur < 64 ? readlane64(pick, cur) : picks[cur];
      const uint64_t hit = __ballot(lane > cur && lane < tree && parent == cur && token == want);
      int next = hit ? __builtin_ctzll(hit) : tree;
      if (!hit && (parents || cur >= 63)) {
        for (int n0 = max(64, cur + 1); n0 < tree && next == tree; n0 += 64) {
          const int n = n0 + lane;
          const uint64_t any = __ballot(n < tree && want >= 0 && (parents ? parents[n] : n - 1) == cur && tokens[n] == want);
          if (any) next = n0 + __builtin_ctzll(any);
          if (!parents) break;                                // (a chain: the next token or none)
        }
      }
      cur = next;
    }
    if (lane == 0) s_count = count;
    if (blockIdx.y == 0) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      for (int d = lane; d < a.longest; d += 64) {
        const int n = d < count ? s_path[d] : -1;
        a.path[(int64_t)b * a.longest + d] = n;
        a.accepted[(int64_t)b * a.longest + d] = n < 0 ? -1 : picks[n];   // (a confirmed node's token is its parent's pick)
      }
      if (lane == 0) {
        a.counts[b] = count;
        a.lens[b] = past + count;
      }
    }
  } else if (tid < 128 && a.k) {
    s_table[lane] = c0 + lane < a.width ? table[c0 + lane] : -1;
  }
  __syncthreads();
  const int count = s_count;
  if (!a.k || count == 0 || s_path[count - 1] == count - 1) return;   // (a path that is in its place, as every chain's is)
  int from = 0;                                               // the first node that is not in its place; none behind it is
  for (int n = count - 1; from < n;) {
    const int mid = (from + n) >> 1;
    if (s_path[mid] == mid)
      from = mid + 1;
    else
      n = mid;
  }
  const int pieces = a.row_bytes / 16, heads = 2 * a.Hkv, groups = 256 / pieces;
  const int64_t head = (int64_t)a.row_bytes << shift, page = head * a.Hkv, layer = (int64_t)blockIdx.y * a.pages;
  // where key `key` lies in this layer, below 0: nowhere
  auto place = [&](int key) -> int64_t {
    const int c = key >> shift;
    if (key < 0 || c >= a.width) return -1;
    const int id = c - c0 < 64 ? s_table[c - c0] : table[c];
    return id < 0 || id >= a.pages ? -1 : (layer + id) * page + (int64_t)(key & ((1 << shift) - 1)) * a.row_bytes;
  };
  // a lane group a row of one head; kHeld rows of a group in a chunk
  constexpr int kHeld = 8;
  const int grp = tid / pieces, piece = tid - grp * pieces;
  const int rows = min(count - from, kHeld * groups), together = max(1, kHeld * groups / rows);
  for (int h0 = 0; h0 < heads; h0 += together)
    for (int d0 = from; d0 < count; d0 += rows) {
      const int n = min(rows, count - d0), items = n * min(together, heads - h0);
      u32x4 held[kHeld];
      int64_t to[kHeld];
#pragma unroll
      for (int u = 0; u < kHeld; ++u) {
        const int i = grp + groups * u;
        to[u] = -1;
        if (grp >= groups || i >= items) continue;
        const int q = (int)((uint32_t)i / (uint32_t)n), hv = h0 + q, d = d0 + i - q * n;
        const int64_t src = place(past + s_path[d]), dst = place(past + d);
        if (src < 0 || dst < 0) continue;
        const int64_t at = (int64_t)(hv >> 1) * head + 16 * piece;
        held[u] = load16((hv & 1 ? a.v : a.k) + src + at);
        to[u] = 2 * (dst + at) + (hv & 1);
      }
      vm_drain();
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kHeld; ++u)
        if (to[u] >= 0) *reinterpret_cast<u32x4*>((to[u] & 1 ? a.v : a.k) + (to[u] >> 1)) = held[u];
      __syncthreads();
    }
}

namespace {

bool plan_is_small(const PlanArgs& a) {
  return a.B <= kSmallSeqs && a.T <= kSmallTokens && a.pages <= kSmallPages && (int64_t)a.B * a.width <= kSmallEntries;
}
int hash_places(int B) {
  int n = 64;
  while (n < 2 * B) n *= 2;
  return n;
}
int64_t map_words(int64_t pages) { return ((pages + 31) / 32 + 3) & ~(int64_t)3; }
int64_t list_places(const PlanArgs& a, int shift) { return (a.T >> shift) + 2 * (int64_t)a.B + 1; }

}  // namespace

// [used][hash_owner, beyond kHashSeqs][hash_page, likewise][row .. start][list]
static int64_t plan_clear(const PlanArgs& a) {   // 16-byte pieces that have to be zero before
  return (a.pages + 31) / 32 * 2 + (a.B > kHashSeqs ? hash_places(a.B) / 2 : 0);
}
size_t plan_paged_workspace(const PlanArgs& a) {
  if (plan_is_small(a)) return 0;
  const int64_t hash = a.B > kHashSeqs ? hash_places(a.B) : 0;
  const int64_t ints = 4 * plan_clear(a) + hash + 6 * (int64_t)a.B + 2 + list_places(a, log2_of(a.page_size));
  return (size_t)(4 * ints + 15) / 16 * 16;
}

hipError_t plan_paged_launch(const PlanArgs& a, hipStream_t st) {
  const int shift = log2_of(a.page_size), places = hash_places(a.B);
  hipError_t e;
  if (plan_is_small(a)) {
    const size_t words = (size_t)map_words(a.pages);
    const size_t lds = 4 * (3 * (size_t)places + words + 6 * (size_t)a.B + 2 + kSmallList + kSmallTokens);
    constexpr size_t most = 4 * (3 * 2 * kSmallSeqs + kSmallPages / 32 + 6 * kSmallSeqs + 2 + kSmallList + kSmallTokens);
    static_assert(most <= 138 * 1024, "LDS");
    static std::atomic<uint64_t> done{0};
    if ((e = allow_lds_once(done, plan_small_kernel, most))) return e;
    // a few sequences and tokens are waves that wait for one another at the barriers: 256 threads then (graph-timed us, 256 / 1024: one
    // sequence of 26 tokens 6.1 / 6.8, 16 of 16 on 2000 keys 7.5 / 8.0, 16 with 256 tokens 7.2 / 7.9; with 1024 tokens 8.7 / 7.9, 32 with
    // 32 8.7 / 8.5, 48 10.4 / 9.1, 128 beams of 141 pages 23.1 / 13.2)
    const bool few = a.B <= 16 && a.T <= 256 && (int64_t)a.B * a.width <= 2048 && a.pages <= 32768;
    e = launch(plan_small_kernel, dim3(1), dim3(few ? 256 : kThreads), lds, st, a, std::min(6, log2_of(a.width)), shift, places - 1);
  } else {
    const bool far = a.B > kHashSeqs;                         // the hash in the workspace
    PlanState s;
    s.hash_mask = places - 1;
    s.used = static_cast<uint32_t*>(a.ws);
    int* at = reinterpret_cast<int*>(s.used + 4 * plan_clear(a));
    s.hash_owner = far ? reinterpret_cast<uint64_t*>(s.used + (a.pages + 31) / 32 * 8) : nullptr;
    s.hash_page = far ? at : nullptr;
    s.row = at + (far ? places : 0);
    s.past = s.row + a.B;
    s.fresh = s.past + a.B;
    s.tail = s.fresh + a.B;
    s.off = s.tail + a.B;
    s.start = s.off + a.B + 1;
    s.list = s.start + a.B + 1;
    s.list_cap = (int)list_places(a, shift);
    const int64_t clear = plan_clear(a);
    e = launch(plan_lens_kernel, dim3((unsigned)(1 + std::min<int64_t>((clear + kThreads - 1) / kThreads, 512))), dim3(kThreads), 0, st,
               a, s, shift, clear);
    const int chunks = (a.width + 1023) / 1024;
    if (e == hipSuccess) e = launch(plan_mark_kernel, dim3((unsigned)(a.B * chunks)), dim3(256), 0, st, a, s, chunks, shift);
    const bool finish = !far && a.T <= kFinishTokens;
    static_assert(12 * 2 * kHashSeqs + 8 * (kHashSeqs + 1) + 24 * 1024 <= 64 * 1024, "LDS");
    if (e == hipSuccess)
      e = launch(plan_assign_kernel, dim3(1), dim3(kThreads), far ? 0 : 12 * (size_t)places + (finish ? 8 * (size_t)(a.B + 1) : 0),
                 st, a, s, shift, finish);
    const int64_t items = std::max<int64_t>(a.T, a.B);
    if (e == hipSuccess && !finish)
      e = launch(plan_fill_kernel, dim3((unsigned)std::min<int64_t>((items + 255) / 256, 4096)), dim3(256),
                 a.B <= kStartSeqs ? 8 * (size_t)(a.B + 1) : 0, st, a, s, shift);
  }
  if (e != hipSuccess || !a.k) return e;
  return launch(plan_copy_kernel, dim3((unsigned)a.B, (unsigned)a.layers), dim3(256), 0, st, static_cast<const int*>(a.copies),
                static_cast<const int*>(a.q_starts), static_cast<const int*>(a.kv_lens), a.k, a.v, a.pages, a.Hkv, a.row_bytes, shift);
}

hipError_t accept_drafts_launch(const AcceptArgs& a, hipStream_t st) {
  return launch(accept_kernel, dim3((unsigned)a.B, (unsigned)(a.k ? a.layers : 1)), dim3(256), 0, st, a, log2_of(a.page_size));
}

}  // namespace lowbit
