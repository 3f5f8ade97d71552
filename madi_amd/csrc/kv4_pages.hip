// kv4_pages.hip -- page tables built, shared and taken back on the GPU
// (madi_kv4_grow, madi_kv4_trim, madi_kv4_fork), and the pages' copies (madi_kv4_copy).
#include "kv4.h"

using namespace madi;

namespace {

constexpr uint32_t kNone = 0xffffffffu;

struct Pages {
  uint32_t *refs, *mark, *state, *table, *lens;
  uint32_t n_pages, shift, b, max_pages;
};

__device__ inline uint32_t pages_of(uint32_t len, uint32_t shift) {
  return (len >> shift) + ((len & ((1u << shift) - 1)) != 0);
}
__device__ inline uint32_t length(const Pages &p, uint32_t i) {
  const uint32_t reach = p.max_pages << p.shift, len = p.lens[i];
  return len < reach ? len : reach;
}
// One holder more or less; how the number of free pages changes by it.  (Sums of these
// over any order of the atomics are the same: a page's steps to and from 0 cancel out.)
__device__ inline int take(const Pages &p, uint32_t page) {
  if (page >= p.n_pages) return 0;
  return __hip_atomic_fetch_add(p.refs + page, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0 ? -1 : 0;
}
__device__ inline int give(const Pages &p, uint32_t page) {
  if (page >= p.n_pages) return 0;
  return __hip_atomic_fetch_sub(p.refs + page, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 1 ? 1 : 0;
}
// The workgroup's sum added to the number of free pages: one atomic a workgroup (one a wave, all to the same
// word, took 5 of 10 us for 256 sequences).
__device__ inline void add_free(const Pages &p, int n) {
  __shared__ int sum;
  if (threadIdx.x == 0) sum = 0;
  __syncthreads();
#pragma unroll
  for (int s = 32; s; s >>= 1) n += __shfl_xor(n, s);
  if ((threadIdx.x & 63) == 0 && n) atomicAdd(&sum, n);
  __syncthreads();
  if (threadIdx.x == 0 && sum) __hip_atomic_fetch_add(p.state, (uint32_t)sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---------------------------------------------------------------- fork
// A workgroup per group (it alone reads and writes the group's rows and lengths), a
// thread per column: the column's entries of all beams go through LDS, so that each is
// read before one is written (in registers a column of 32 spilled).  Bound by latency: parents, lengths, entries, counts
// one after the other; 64 groups of 8 beams with 1024 columns 5.4 us (12.3 with 256 threads a group, whose passes
// follow one another), 8 groups of 5 with 7 4.4, where no entry changes; where every beam's last pages do, 11.2 (18.2)
// and 8.1: the counts' atomics, and the sum's.
constexpr uint32_t kMaxBeams = 32, kForkLds = 32 << 10;
__global__ __launch_bounds__(1024) void kv4_fork_kernel(Pages p, const uint32_t *__restrict__ parent, uint32_t ldp,
                                                         uint32_t beams) {
  __shared__ uint32_t from[kMaxBeams], held[kMaxBeams];
  extern __shared__ uint32_t tile[];  // [beams][threads]
  const uint32_t g = blockIdx.x, t = threadIdx.x, wide = blockDim.x;
  uint32_t *table = p.table + (size_t)g * beams * p.max_pages;
  uint32_t len = 0;
  bool moves = false;
  if (t < beams) {
    const uint32_t f = parent[(size_t)g * ldp + t];
    from[t] = f;
    held[t] = pages_of(length(p, g * beams + t), p.shift);
    if (f < beams) len = length(p, g * beams + f);
    moves = f != t;
  }
  __syncthreads();  // every length is read
  if (moves) p.lens[g * beams + t] = len;
  uint32_t most = 0;
  for (uint32_t i = 0; i < beams; ++i) most = held[i] > most ? held[i] : most;
  int freed = 0;
  for (uint32_t c = t; c < most; c += wide) {
#pragma unroll 4
    for (uint32_t i = 0; i < beams; ++i)
      tile[i * wide + t] = c < held[i] ? table[(size_t)i * p.max_pages + c] : kNone;
    for (uint32_t i = 0; i < beams; ++i) {
      const uint32_t f = from[i];
      if (f == i) continue;
      const uint32_t had = held[i], has = f < beams ? held[f] : 0;
      if (c >= had && c >= has) continue;
      const uint32_t old = tile[i * wide + t], now = c < has ? tile[f * wide + t] : kNone;
      if (old != now) freed += take(p, now) + give(p, old);
      table[(size_t)i * p.max_pages + c] = now;
    }
  }
  add_free(p, freed);
}

// ---------------------------------------------------------------- trim
// A workgroup per sequence.  (256 sequences of 512 columns 5.5 us, 48 3.6: length, entries, counts and the sum's
// atomic one after the other.)
__global__ __launch_bounds__(256) void kv4_trim_kernel(Pages p, const uint32_t *__restrict__ to) {
  const uint32_t i = blockIdx.x, len = length(p, i), want = to[i];
  if (want >= len) return;
  uint32_t *row = p.table + (size_t)i * p.max_pages;
  const uint32_t had = pages_of(len, p.shift);
  int freed = 0;
  for (uint32_t c = pages_of(want, p.shift) + threadIdx.x; c < had; c += blockDim.x) {
    freed += give(p, row[c]);
    row[c] = kNone;
  }
  add_free(p, freed);
  __syncthreads();  // every thread has the length
  if (threadIdx.x == 0) p.lens[i] = want;
}

// ---------------------------------------------------------------- grow
struct Rows {
  uint32_t *row_off, *copies, *row_seq, *row_pos;
  int64_t *slot;
  uint32_t m, kept;
};

constexpr uint32_t kGrow = 1024;         // threads, and sequences of a tile
constexpr uint32_t kScan = 16;           // refs a thread looks at per step
// a + b, or the largest number where that is more: sums of these do not depend on the order
__device__ inline uint32_t sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
// The sums of the threads' v[] before the calling one; `all` are the whole sums.  (Row shifts and broadcasts:
// a shift through the LDS crossbar at each of the six steps took three times as long.)
template <int N>
__device__ inline void before(uint32_t (&v)[N], uint32_t (*lds)[kGrow / 64], uint32_t (&all)[N]) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t sum[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint32_t x = v[i];
    x = sat(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true));  // lanes 1, 2, 4, 8 lower in the row of 16
    x = sat(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true));
    x = sat(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true));
    x = sat(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true));
    x = sat(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, true));  // lane 15 to row 1, 47 to row 3
    sum[i] = sat(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, true));  // lane 31 to rows 2 and 3
  }
  __syncthreads();
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < N; ++i) lds[i][wave] = sum[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint32_t base = 0, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kGrow / 64; ++w) {
      const uint32_t x = w < blockDim.x / 64 ? lds[i][w] : 0;
      if (w < wave) base = sat(base, x);
      total = sat(total, x);
    }
    all[i] = total;
    v[i] = sat(base, __builtin_amdgcn_update_dpp(0, sum[i], 0x138, 0xf, 0xf, true));  // of the lane before
  }
}

// The maps of a row: its sequence by bisection of the offsets, len(sequence) the length after the call.
template <typename F>
__device__ inline void put_row(const Pages &p, const Rows &r, uint32_t row, uint32_t rows, const uint32_t *offs, F len) {
  uint32_t seq = kNone, pos = 0;
  int64_t slot = -1;
  if (row < rows) {
    uint32_t lo = 0, hi = p.b;  // offs[lo] <= row < offs[hi]
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (offs[mid] <= row) lo = mid;
      else hi = mid;
    }
    seq = lo;
    pos = len(seq) - (offs[seq + 1] - row);
    if (r.slot) {
      const uint32_t page = p.table[(size_t)seq * p.max_pages + (pos >> p.shift)];
      if (page < p.n_pages) slot = ((int64_t)page << p.shift) + (pos & ((1u << p.shift) - 1));
    }
  }
  if (r.row_seq) r.row_seq[row] = seq;
  if (r.row_pos) r.row_pos[row] = pos;
  if (r.slot) r.slot[row] = slot;
}

// A sequence of a grow: its length, and its tokens (0 where the table has no room for them).
struct Seq {
  uint32_t len, add;
  bool wants;
};
__device__ inline Seq seq_of(const Pages &p, const uint32_t *add, uint32_t i) {
  Seq s{0, 0, false};
  if (i < p.b) {
    s.len = length(p, i);
    const uint32_t a = add[i];
    s.wants = a != 0;
    s.add = a <= (p.max_pages << p.shift) - s.len ? a : 0;
  }
  return s;
}
// The page that its next token goes to, if it has one.
__device__ inline uint32_t last_page(const Pages &p, uint32_t i, const Seq &s) {
  return s.add && (s.len & ((1u << p.shift) - 1)) ? p.table[(size_t)i * p.max_pages + (s.len >> p.shift)] : kNone;
}
// Which of refs[at .. at + 15] are 0.  (Past the end the last sixteen are read, not one word after the other: 48
// sequences of a pool of 16383 pages 12.3 -> 11.2 us with a trim.)
__device__ inline uint32_t look(const Pages &p, uint32_t at) {
  typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(4)));
  uint32_t is_free = 0;
  if (p.n_pages >= kScan) {
    const uint32_t from = at <= p.n_pages - kScan ? at : p.n_pages - kScan;
    u32x4_any v[kScan / 4];
#pragma unroll
    for (uint32_t j = 0; j < kScan / 4; ++j) v[j] = *reinterpret_cast<const u32x4_any *>(p.refs + from + 4 * j);
#pragma unroll
    for (uint32_t j = 0; j < kScan; ++j) is_free |= (v[j / 4][j % 4] == 0) << j;
    return at < p.n_pages ? is_free >> (at - from) : 0;
  }
  for (uint32_t j = 0; j < kScan && at + j < p.n_pages; ++j) is_free |= (p.refs[at + j] == 0) << j;
  return is_free;
}

// Where a grow of several launches keeps what it needs from one to the next, behind mark's n_pages words.
constexpr uint32_t kSegment = 64 * kScan;  // pages that a wave looks through
__device__ __host__ inline uint32_t segments(uint32_t n_pages) { return n_pages / kSegment + (n_pages % kSegment != 0); }
struct Plan {
  uint32_t *first;   // [b + 1]: number of the sequence's first page among the free ones; of all
  uint32_t *counts;  // [segments]: free pages of 1024
  uint32_t *bits;    // [segments * 64]: which, of 16
};
__device__ inline Plan plan_of(const Pages &p) {
  uint32_t *first = p.mark + p.n_pages;
  return {first, first + p.b + 1, first + p.b + 1 + segments(p.n_pages)};
}

// A sequence whose last page has `held` holders, more than itself.
struct Sharer {
  uint32_t seq, page, len, held, copies;
};
// Whether another sequence has a sharer's page, at the same place of its row.  Up to kNear sequences a wave of
// the grow looks through them; of more kv4_others_kernel has noted it.  (One token each, every page held elsewhere too: 128
// sequences 15.6 us, 129 13.0 with 3.7 of that kernel before; 1000, of which 50 are such, 34 looked up by the grow's
// workgroup, 13.0 and 7.2 so.)
constexpr uint32_t kNear = 128;
__device__ inline bool has(const Pages &p, uint32_t j, const Sharer &s) {
  const uint32_t i = j < p.b ? j : s.seq, c = s.len >> p.shift;
  return p.table[(size_t)i * p.max_pages + c] == s.page && i != s.seq && pages_of(length(p, i), p.shift) > c;
}
__device__ inline uint32_t *others_have_of(const Pages &p) { return plan_of(p).first; }  // (until the plan is there)
__device__ inline bool others_have(const Pages &p, const Sharer &s) {
  if (p.b > kNear) return others_have_of(p)[s.seq];
  bool found = false;
#pragma unroll
  for (uint32_t u = 0; u < kNear; u += 64) found |= has(p, u + (threadIdx.x & 63), s);
  return __any(found);
}
// A wave per sequence, 256 others at a time from its neighbours on.  (What is read goes with the sharers times the
// sequences: 256 prompts 4.1 us, 4096 sequences with 205 sharers 17, 16384 that all are 675.)
__global__ __launch_bounds__(256) void kv4_others_kernel(Pages p, const uint32_t *__restrict__ add) {
  const uint32_t lane = threadIdx.x & 63, i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Seq s = seq_of(p, add, i);
  const uint32_t q = last_page(p, i, s);
  if (q >= p.n_pages || p.refs[q] <= 1) return;  // (not asked for)
  const Sharer own{i, q, s.len, 0, 0};
  const uint32_t chunks = (p.b + 63) / 64;
  bool found = false;
  for (uint32_t k = 0; k < chunks && !found; k += 4) {
    bool here = false;
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) here |= has(p, (i / 64 + k + u) % chunks * 64 + lane, own);
    found = __any(here);
  }
  if (lane == 0) others_have_of(p)[i] = found;
}

// Up to so many of them find one another in LDS, at a cost that goes with their square; more through mark's six phases.  (A
// step of as many beams: 40 8.6 / 10.8 us, 128 10.7 / 11.0, 192 12.1 / 11.4, 800 50 / 16; 48 sequences, two of them on kept
// prompts' pages, 10.0 / 12.0.)
constexpr uint32_t kFew = 128;

// One workgroup.  Sequences in tiles of 1024, thread t has sequence 1024 j + t of tile j.
//  1. holders of a shared last page that grow: where all holders do, the one with the most tokens in it keeps it, the
//     others get copies (one that finds no page for its copy goes on holding the page, and no row of a longer one's is
//     written where it has tokens); with `kept`, a page that no other sequence has is left to its sequence
//  2. a tile's sums of the pages and rows asked for decide who grows; lengths and row offsets
//  3. refs are looked through from page 0 for as many free pages as that takes, 16384 at a time
//     (the first ones are asked for at the start: a page that is free then is so until it is given out)
// Bound by latency, about ten dependent steps: 48 sequences of up to 5 tokens 8.0 us with the maps and no copies asked for,
// 8.6 with copies where no page has other holders, 9.6 where two are kept prompts'; as kPlan, 256 prompts of up to 4096
// tokens, 4.2, 5.7 and 6.5.  A step of 40 beams on shared pages 8.7, of 512 20 (of which the look from page 0 through
// 36000 used ones is a part).
// kMaps (one tile): the rows' maps too.  kPlan: 3 is left to kv4_give_kernel, and the grid's other workgroups
// note the free pages for it meanwhile (a page in use has a holder at every moment of 1 and 2).
enum Grow { kPlain, kMaps, kPlan };
template <Grow MODE>
__global__ __launch_bounds__(kGrow) void kv4_grow_kernel(Pages p, const uint32_t *__restrict__ add, Rows r) {
  constexpr bool MAPS = MODE == kMaps;
  __shared__ uint32_t list[MODE == kPlan ? kFew * sizeof(Sharer) / 4 : kGrow * kScan], lds[2][kGrow / 64], asking;
  __shared__ uint32_t offs[MAPS ? kGrow + 1 : 1], ends[MAPS ? kGrow : 1];
  const uint32_t tid = threadIdx.x, tiles = MAPS ? 1 : (p.b + kGrow - 1) / kGrow, mask = (1u << p.shift) - 1;
  if (MODE == kPlan && blockIdx.x) {
    const uint32_t at = (blockIdx.x - 1) * kGrow + tid, mine = look(p, at * kScan);
    uint32_t n = __builtin_popcount(mine);
#pragma unroll
    for (int s = 32; s; s >>= 1) n += __shfl_xor(n, s);
    const Plan plan = plan_of(p);
    if (at / 64 < segments(p.n_pages)) {
      plan.bits[at] = mine;
      if (tid % 64 == 0) plan.counts[at / 64] = n;
    }
    return;
  }
  const auto seq = [&](uint32_t i) { return seq_of(p, add, i); };
  const uint32_t free = p.state[0];
  uint32_t is_free = MODE == kPlan ? 0 : look(p, tid * kScan);

  const uint32_t lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  uint64_t copy = 0;
  if (r.copies) {
    uint64_t shared = 0;
    Sharer own{};  // of the last tile
    for (uint32_t t = 0; t < tiles; ++t) {
      const uint32_t i = t * kGrow + tid;
      const Seq s = seq(i);
      const uint32_t q = last_page(p, i, s), held = q < p.n_pages ? p.refs[q] : 0;
      own = {i, q, s.len, held, 0};
      if (held > 1) shared |= 1ull << t;
    }
    if (tid == 0) asking = 0;
    const uint32_t some = __syncthreads_count(shared != 0);
    if (some && some <= kFew && tiles == 1) {  // a wave counts a sharer's page among the others
      Sharer *sharers = reinterpret_cast<Sharer *>(list);
      uint32_t mine = 0;
      if (shared) {
        mine = atomicAdd(&asking, 1u);
        sharers[mine] = own;
      }
      __syncthreads();
      for (uint32_t e = wave; e < some; e += kGrow / 64) {
        const Sharer s = sharers[e];
        uint32_t grow = 0;
        bool most = true;
        for (uint32_t x = lane; x - lane < some; x += 64) {
          const Sharer o = sharers[x < some ? x : e];
          const bool same = x < some && o.page == s.page;
          grow += __builtin_popcountll(__ballot(same));
          most &= !same || (o.len & mask) < (s.len & mask) || ((o.len & mask) == (s.len & mask) && o.seq <= s.seq);
        }
        const bool copies = grow < s.held ? !r.kept || grow > 1 || others_have(p, s) : !__all(most);
        if (lane == 0) sharers[e].copies = copies;
      }
      __syncthreads();
      copy = shared && sharers[mine].copies;
    } else if (some) {
      // through mark, which is 0 before and after: how many of a page's holders grow, then the longest of them
      const auto each = [&](uint64_t who, auto f) {
        for (uint32_t t = 0; t < tiles; ++t)
          if (who >> t & 1) {
            const uint32_t i = t * kGrow + tid;
            f(t, i, last_page(p, i, seq(i)));
          }
        __syncthreads();
      };
      const auto load = [&](uint32_t q) { return __hip_atomic_load(p.mark + q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
      const auto clear = [&](uint32_t, uint32_t, uint32_t q) {
        __hip_atomic_store(p.mark + q, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      };
      each(shared, [&](uint32_t, uint32_t, uint32_t q) {
        __hip_atomic_fetch_add(p.mark + q, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      });
      uint64_t single = 0;  // of whose page one holder grows
      each(shared, [&](uint32_t t, uint32_t, uint32_t q) {
        const uint32_t n = load(q);
        if (n < p.refs[q]) copy |= 1ull << t;
        if (n == 1) single |= 1ull << t;
      });
      each(shared, clear);
      const uint64_t whole = shared & ~copy;  // of whose page all holders grow
      if (r.kept)
        for (uint32_t t = 0; t < tiles; ++t) {
          const uint32_t i = t * kGrow + tid;
          if (copy >> t & single >> t & 1 && !others_have_of(p)[i]) copy &= ~(1ull << t);
        }
      if (__syncthreads_or(whole != 0)) {
        const auto tokens = [&](uint32_t i) { return length(p, i) & mask; };  // (at least one)
        const auto most = [&](auto number) {  // keeps the page, so far; the others copy
          const uint64_t left = whole & ~copy;
          each(left, [&](uint32_t, uint32_t i, uint32_t q) {
            __hip_atomic_fetch_max(p.mark + q, number(i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          });
          each(left, [&](uint32_t t, uint32_t i, uint32_t q) {
            if (load(q) != number(i)) copy |= 1ull << t;
          });
          each(left, clear);
        };
        // of equals the last: one number (sequences are 2^16 - 1 at most), or two for pages of more than 2^16 tokens
        if (p.shift <= 16) {
          most([&](uint32_t i) { return tokens(i) << 16 | i; });
        } else {
          most(tokens);
          most([&](uint32_t i) { return i + 1; });
        }
      }
    }
  }

  const Plan plan = plan_of(p);
  uint32_t asked = 0, rows_asked = 0, rows = 0, total = 0, left_out = 0;
  // list: free pages number found .. found + n - 1; `at`: where to look on
  uint32_t found = 0, n = 0, at = 0;
  for (uint32_t t = 0; t < tiles; ++t) {
    const uint32_t i = t * kGrow + tid;
    const Seq s = seq(i);
    const bool cp = copy >> t & 1;
    const uint32_t src = cp ? last_page(p, i, s) : kNone, col = pages_of(s.len, p.shift);
    const uint32_t want = pages_of(s.len + s.add, p.shift) - col + cp;
    uint32_t ask[] = {want, s.add}, all[2], get[2], took_all[2];
    before(ask, lds, all);
    const uint32_t first = sat(asked, ask[0]), row = sat(rows_asked, ask[1]);
    const bool grows = s.add && (want == 0 || sat(first, want) <= free) && sat(row, s.add) <= r.m;
    // (those that grow and want pages are the first that want any: their pages have no gaps)
    const uint32_t need = grows ? want : 0, own = need - (grows && cp);
    get[0] = need, get[1] = grows ? s.add : 0;
    before(get, lds, took_all);
    const uint32_t given = total + get[0], off = rows + get[1], took = took_all[0], some = took_all[1];
    if (i < p.b) {
      r.row_off[i] = off;
      if (grows) p.lens[i] = s.len + s.add;
      if (grows && cp) __hip_atomic_fetch_sub(p.refs + src, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (MODE == kPlan) plan.first[i] = given;
      if (r.copies) {  // (its target once the page is there)
        uint32_t *c = r.copies + (size_t)i * 3;
        c[0] = grows && cp ? src : kNone;
        c[1] = kNone;
        c[2] = grows && cp ? s.len & mask : kNone;
      }
    }
    if (MAPS) {
      offs[tid] = off;
      ends[tid] = s.len + (grows ? s.add : 0);
      if (tid == kGrow - 1) offs[kGrow] = rows + some;
    }
    asked = sat(asked, all[0]);
    rows_asked = sat(rows_asked, all[1]);
    rows += some;
    total += took;
    left_out += __syncthreads_count(s.wants && !grows);

    while (MODE != kPlan && took) {
      // its pages first .. first + need - 1, of which found .. found + n - 1 are there: the
      // table's new columns, then the copy
      const uint32_t lo = first > found ? first : found;
      const uint32_t hi = first + own < found + n ? first + own : found + n;
      const bool some_here = need && lo < hi, longer = some_here && hi > lo + 4;
      const auto put = [&](uint32_t row, uint32_t c, uint32_t lo, uint32_t hi, uint32_t f, uint32_t from, uint32_t step) {
        for (uint32_t x = lo + from; x < hi; x += step) {
          const uint32_t page = list[x - found];
          p.table[(size_t)row * p.max_pages + c + (x - f)] = page;
          p.refs[page] = 1;
        }
      };
      if (some_here && !longer) put(i, col, lo, hi, first, 0, 1);
      for (uint64_t todo = __ballot(longer); todo; todo &= todo - 1) {
        const int l = __builtin_ctzll(todo);
        put(__shfl(i, l), __shfl(col, l), __shfl(lo, l), __shfl(hi, l), __shfl(first, l), tid & 63, 64);
      }
      if (grows && cp && first + own >= found && first + own < found + n) {
        const uint32_t page = list[first + own - found];
        r.copies[(size_t)i * 3 + 1] = page;
        p.table[(size_t)i * p.max_pages + (s.len >> p.shift)] = page;
        p.refs[page] = 1;
      }
      if (found + n >= total || at >= p.n_pages) break;
      __syncthreads();  // the list is read
      found += n;
      if (at) is_free = look(p, at + tid * kScan);
      uint32_t ranks[] = {(uint32_t)__builtin_popcount(is_free)}, count[1];
      before(ranks, lds, count);
      n = count[0];
      for (uint32_t k = ranks[0]; is_free; is_free &= is_free - 1, ++k) list[k] = at + tid * kScan + __builtin_ctz(is_free);
      at += kGrow * kScan;
      __syncthreads();
    }
  }
  if (tid == 0) {
    r.row_off[p.b] = rows;
    p.state[0] = free - total;
    p.state[1] = left_out;
    if (MODE == kPlan) plan.first[p.b] = total;
  }
  if constexpr (MAPS) {
    __syncthreads();  // offsets, lengths and table are there
    for (uint32_t row = tid; row < r.m; row += kGrow) put_row(p, r, row, rows, offs, [&](uint32_t i) { return ends[i]; });
  }
}

// After a plan: a workgroup per segment gives out its free pages, a thread one of them at a time.  (33000 pages of
// 131072 7 us; by the one workgroup of the plan 50, with a thread for 16384 pages' words each 16.)
__global__ __launch_bounds__(256) void kv4_give_kernel(Pages p, Rows r) {
  __shared__ uint32_t lds[2][kGrow / 64], list[kSegment];
  const Plan plan = plan_of(p);
  const uint32_t tid = threadIdx.x, seg = blockIdx.x, total = plan.first[p.b];
  uint32_t bits = plan.bits[seg * 64 + tid / 4] >> tid % 4 * 4 & 15;
  uint32_t sums[] = {(uint32_t)__builtin_popcount(bits), 0}, all[2];
  for (uint32_t s = tid; s < seg; s += 256) sums[1] += plan.counts[s];
  before(sums, lds, all);
  const uint32_t k0 = all[1];  // its first page's number among the free ones
  if (k0 >= total || !all[0]) return;
  const uint32_t n = all[0] < total - k0 ? all[0] : total - k0;
  for (; bits; bits &= bits - 1) list[sums[0]++] = seg * kSegment + tid * 4 + __builtin_ctz(bits);
  // the sequence of page number k: first[seq] <= k < first[seq + 1]
  const auto seq_at = [&](uint32_t k, uint32_t lo, uint32_t hi) {
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (plan.first[mid] <= k) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  const uint32_t from = seq_at(k0, 0, p.b), to = seq_at(k0 + n - 1, from, p.b) + 1;
  __syncthreads();
  for (uint32_t x = tid; x < n; x += 256) {
    const uint32_t i = seq_at(k0 + x, from, to), j = k0 + x - plan.first[i], page = list[x];
    const uint32_t len = p.lens[i], old = len - (r.row_off[i + 1] - r.row_off[i]);
    const uint32_t col = pages_of(old, p.shift), own = pages_of(len, p.shift) - col;
    if (j >= own) r.copies[(size_t)i * 3 + 1] = page;
    p.table[(size_t)i * p.max_pages + (j < own ? col + j : old >> p.shift)] = page;
    p.refs[page] = 1;
  }
}

// A thread per row.  (524288 of them 5.8 us.)
__global__ __launch_bounds__(256) void kv4_rows_kernel(Pages p, Rows r) {
  const uint32_t row = blockIdx.x * 256 + threadIdx.x;
  if (row < r.m) put_row(p, r, row, r.row_off[p.b], r.row_off, [&](uint32_t i) { return p.lens[i]; });
}

// ---------------------------------------------------------------- copy
// A workgroup per entry and head; each of K, V and the scales has the first tokens in front.  (512 entries of 8 heads
// of 64, half of them copies of 16 tokens, 3.1 us.)
__global__ __launch_bounds__(256) void kv4_copy_kernel(uint8_t *data, uint32_t n_pages, uint32_t shift, uint32_t nkv,
                                                       uint32_t d, const uint32_t *__restrict__ copies) {
  const uint32_t *c = copies + (size_t)blockIdx.x * 3;
  const uint32_t from = c[0], to = c[1], page = 1u << shift, head = blockIdx.y;
  uint32_t tokens = c[2];
  if (from >= n_pages || to >= n_pages) return;
  tokens = (tokens < page ? tokens + 3 : page) & ~3u;
  const size_t blk = kv4_block_bytes(shift, d), half = (size_t)page * (d / 2);
  const uint8_t *src = data + ((size_t)from * nkv + head) * blk;
  uint8_t *dst = data + ((size_t)to * nkv + head) * blk;
  const uint32_t kv = tokens * (d / 32), sc = tokens * d / 128;  // in 16 bytes
  for (uint32_t x = threadIdx.x; x < 2 * kv + sc; x += 256) {
    const size_t off = x < kv ? (size_t)x * 16 : x < 2 * kv ? half + (size_t)(x - kv) * 16 : 2 * half + (size_t)(x - 2 * kv) * 16;
    *reinterpret_cast<u32x4 *>(dst + off) = *reinterpret_cast<const u32x4 *>(src + off);
  }
}

// ---------------------------------------------------------------- checks
int pages_args(const char *what, const madi_kv4_pages *p, Pages *a) {
  if (!p) return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (p->page < 16 || p->page > (1u << 20) || (p->page & (p->page - 1)))
    return fail(MADI_ERR_SHAPE, "%s: page %u (a power of two from 16 to 2^20)", what, p->page);
  if (p->b > 65535) return fail(MADI_ERR_SHAPE, "%s: %u sequences (at most 65535)", what, p->b);
  if (p->n_pages == 0 || p->n_pages > 0x7fffffffu)
    return fail(MADI_ERR_SHAPE, "%s: %u pages (1 to 2^31 - 1)", what, p->n_pages);
  if (p->b && p->max_pages == 0) return fail(MADI_ERR_SHAPE, "%s: max_pages is 0", what);
  if ((uint64_t)p->max_pages * p->page > 0x7ffff000u)
    return fail(MADI_ERR_SHAPE, "%s: max_pages * page = %u * %u positions (at most 2^31 - 4096)", what, p->max_pages,
                p->page);
  if (!p->refs || !p->mark || !p->state || (p->b && (!p->table || !p->lens)))
    return fail(MADI_ERR_NULL, "%s: null pointer", what);
  for (const void *q : {p->refs, p->mark, p->state, p->table, p->lens})
    if (!aligned(q, 4)) return fail(MADI_ERR_ALIGN, "%s: arrays must be 4-byte aligned", what);
  *a = {p->refs, p->mark, p->state, p->table, p->lens, p->n_pages, (uint32_t)__builtin_ctz(p->page), p->b, p->max_pages};
  return MADI_OK;
}
#define PAGES_EXTENTS(p)                                                                                    \
  {(p)->refs, (size_t)(p)->n_pages * 4, true}, {(p)->mark, ((size_t)(p)->n_pages + (p)->n_pages / 8 + (p)->b + 1024) * 4, true}, {(p)->state, 8, true}, \
      {(p)->table, (size_t)(p)->b * (p)->max_pages * 4, true}, {(p)->lens, (size_t)(p)->b * 4, true}

int not_ready(const char *what) {
  return initialized() ? MADI_OK : fail(MADI_ERR_NOT_INIT, "%s: madi_init has not succeeded", what);
}

}  // namespace

extern "C" int madi_kv4_grow(const madi_kv4_pages *pages, const uint32_t *add, const madi_kv4_rows *rows) {
  const char *what = "madi_kv4_grow";
  Pages a;
  if (int rc = pages_args(what, pages, &a)) return rc;
  if (!rows || !rows->row_off || !add) return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (rows->m > 0x7fffffffu) return fail(MADI_ERR_SHAPE, "%s: %u rows (below 2^31)", what, rows->m);
  for (const void *q : {(const void *)rows->row_off, (const void *)rows->copies, (const void *)rows->row_seq,
                        (const void *)rows->row_pos, (const void *)add})
    if (!aligned(q, 4)) return fail(MADI_ERR_ALIGN, "%s: arrays must be 4-byte aligned", what);
  if (!aligned(rows->slot, 8)) return fail(MADI_ERR_ALIGN, "%s: slot must be 8-byte aligned", what);
  const size_t b = pages->b, m = rows->m;
  const Extent x[] = {PAGES_EXTENTS(pages), {add, b * 4, false}, {rows->row_off, (b + 1) * 4, true},
                      {rows->copies, rows->copies ? b * 12 : 0, true}, {rows->row_seq, rows->row_seq ? m * 4 : 0, true},
                      {rows->row_pos, rows->row_pos ? m * 4 : 0, true}, {rows->slot, rows->slot ? m * 8 : 0, true}};
  if (int rc = disjoint(what, x)) return rc;
  if (int rc = not_ready(what)) return rc;
  if (int rc = ready(x)) return rc;
  const Rows r{rows->row_off, rows->copies, rows->row_seq, rows->row_pos, rows->slot, rows->m, rows->kept};
  const bool maps = m && (r.row_seq || r.row_pos || r.slot);
  if (r.copies && r.kept && a.b > kNear) {
    kv4_others_kernel<<<(a.b + 3) / 4, 256, 0, stream()>>>(a, add);
    if (int rc = check_launch(what)) return rc;
  }
  // Few rows: one workgroup.  More: the plan's launches, 3 us more, with the pages and maps over all CUs.  (Measured with
  // a trim and without copies, whose cost is the same in both, one workgroup against the plan: 48 sequences of 20 rows 11.7 / 14.4 us, of 80 20.8 / 14.4; 256 of 16
  // 17.0 / 18.2, of 64 29 / 21, of 256 82 / 21; 1024 of 4 27 / 33.)
  if (m <= 2048 + 8 * (a.b < kGrow ? a.b : kGrow)) {
    if (maps && b <= kGrow) kv4_grow_kernel<kMaps><<<1, kGrow, 0, stream()>>>(a, add, r);
    else kv4_grow_kernel<kPlain><<<1, kGrow, 0, stream()>>>(a, add, r);
    if (int rc = check_launch(what)) return rc;
    if (b <= kGrow) return MADI_OK;
  } else {
    const uint32_t segs = segments(a.n_pages);
    kv4_grow_kernel<kPlan><<<1 + (segs + 15) / 16, kGrow, 0, stream()>>>(a, add, r);
    if (int rc = check_launch(what)) return rc;
    kv4_give_kernel<<<segs, 256, 0, stream()>>>(a, r);
    if (int rc = check_launch(what)) return rc;
  }
  if (maps) kv4_rows_kernel<<<(uint32_t)((m + 255) / 256), 256, 0, stream()>>>(a, r);
  return check_launch(what);
}

extern "C" int madi_kv4_trim(const madi_kv4_pages *pages, const uint32_t *to) {
  const char *what = "madi_kv4_trim";
  Pages a;
  if (int rc = pages_args(what, pages, &a)) return rc;
  if (!to) return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (!aligned(to, 4)) return fail(MADI_ERR_ALIGN, "%s: arrays must be 4-byte aligned", what);
  const Extent x[] = {PAGES_EXTENTS(pages), {to, (size_t)pages->b * 4, false}};
  if (int rc = disjoint(what, x)) return rc;
  if (int rc = not_ready(what)) return rc;
  if (a.b == 0) return MADI_OK;
  if (int rc = ready(x)) return rc;
  kv4_trim_kernel<<<a.b, 256, 0, stream()>>>(a, to);
  return check_launch(what);
}

extern "C" int madi_kv4_fork(const madi_kv4_pages *pages, const uint32_t *parent, uint32_t ldp, uint32_t beams) {
  const char *what = "madi_kv4_fork";
  Pages a;
  if (int rc = pages_args(what, pages, &a)) return rc;
  if (beams < 1 || beams > kMaxBeams || a.b % beams)
    return fail(MADI_ERR_SHAPE, "%s: %u beams (1 to 32) of %u sequences", what, beams, a.b);
  if (ldp < beams) return fail(MADI_ERR_SHAPE, "%s: rows of parent are %u apart but %u long", what, ldp, beams);
  if (!parent) return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (!aligned(parent, 4)) return fail(MADI_ERR_ALIGN, "%s: arrays must be 4-byte aligned", what);
  const uint32_t groups = a.b / beams;
  const Extent x[] = {PAGES_EXTENTS(pages), {parent, groups ? ((size_t)(groups - 1) * ldp + beams) * 4 : 0, false}};
  if (int rc = disjoint(what, x)) return rc;
  if (int rc = not_ready(what)) return rc;
  if (a.b == 0) return MADI_OK;
  if (int rc = ready(x)) return rc;
  // as many threads as the table has columns, while their tile fits the LDS
  uint32_t threads = 64;
  while (threads < 1024 && threads < a.max_pages && threads * 2 * beams * 4 <= kForkLds) threads *= 2;
  kv4_fork_kernel<<<groups, threads, beams * threads * 4, stream()>>>(a, parent, ldp, beams);
  return check_launch(what);
}

extern "C" int madi_kv4_copy(const madi_kv4 *cache, const uint32_t *copies, uint32_t n) {
  const char *what = "madi_kv4_copy";
  if (!cache) return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (madi_kv4_bytes(1, cache->page, cache->nkv, cache->d) == 0 || kv4_cache_bytes(cache) == 0)
    return fail(MADI_ERR_SHAPE, "%s: a cache of %u pages of %u tokens, %u heads of %u", what, cache->n_pages, cache->page,
                cache->nkv, cache->d);
  if (n > 65535) return fail(MADI_ERR_SHAPE, "%s: %u entries (at most 65535)", what, n);
  if (!cache->data || (n && !copies)) return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (!aligned(cache->data, 16) || !aligned(copies, 4))
    return fail(MADI_ERR_ALIGN, "%s: data must be 16-byte, copies 4-byte aligned", what);
  const Extent x[] = {{cache->data, kv4_cache_bytes(cache), true}, {copies, (size_t)n * 12, false}};
  if (int rc = disjoint(what, x)) return rc;
  if (int rc = not_ready(what)) return rc;
  if (n == 0) return MADI_OK;
  if (int rc = ready(x)) return rc;
  kv4_copy_kernel<<<dim3(n, cache->nkv), 256, 0, stream()>>>(static_cast<uint8_t *>(cache->data), cache->n_pages,
                                                              (uint32_t)__builtin_ctz(cache->page), cache->nkv, cache->d, copies);
  return check_launch(what);
}
