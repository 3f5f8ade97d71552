// beam.hip -- beam search: the n best continuations of each group of beams
// (madi_beam_select) and the beams' dense states in their new order (madi_beam_gather).
//
// Selection in two kernels.  The first takes a piece of one row per workgroup, once through memory: the
// running maximum and sum of exponentials, and the n best tokens of the piece by logit
// (within a beam the logits' order is the candidates' order).  The second joins a group: each row's
// log sum from its pieces' sums, in 64 bits, and the n best of the pieces' candidates.
#include <float.h>

#include "kv4.h"

using namespace madi;

namespace {

constexpr uint32_t kMaxBeams = 32, kMaxBest = 64;
constexpr uint32_t kTokenBits = 27, kTokenMask = (1u << kTokenBits) - 1;  // vocab is at most kTokenMask
constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;
constexpr uint32_t kPer = 16, kTile = kThreads * kPer;  // logits a thread holds, and a workgroup
constexpr uint32_t kRank = 512;                         // up to so many keys are ranked by counting
constexpr uint32_t kMaxPieces = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kMost = 0x1p126f;  // logits below -kMost are banned, so differences are finite

// Whole numbers in the order of the floats (-0 and 0 made one by the caller; no NaN).
__device__ inline uint32_t order(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ inline float unorder(uint32_t k) {
  return __builtin_bit_cast(float, k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ inline uint64_t order(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ inline double unorder(uint64_t k) {
  return __builtin_bit_cast(double, k ^ (k >> 63 ? 0x8000000000000000ull : ~0ull));
}
constexpr uint64_t kNoCandidate = 0x000fffffffffffffull;    // order(-(double)inf)

// f over the wave's values, the result in every lane: four steps within 16 lanes (DPP) and two exchanges of
// rows, where a shuffle through LDS takes 60 cycles a step.
template <int CTRL>
__device__ inline uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <typename T, typename F>
__device__ inline T over_wave(T v, F f) {
  constexpr int kWords = sizeof(T) / 4;
  struct Words {
    uint32_t w[kWords];
  };
  const auto moved = [&](auto move) {
    Words x = __builtin_bit_cast(Words, v);
#pragma unroll
    for (int i = 0; i < kWords; ++i) x.w[i] = move(x.w[i]);
    return __builtin_bit_cast(T, x);
  };
  v = f(v, moved([](uint32_t x) { return dpp<0xb1>(x); }));   // lane ^ 1
  v = f(v, moved([](uint32_t x) { return dpp<0x4e>(x); }));   // lane ^ 2
  v = f(v, moved([](uint32_t x) { return dpp<0x141>(x); }));  // 7 - lane of 8
  v = f(v, moved([](uint32_t x) { return dpp<0x140>(x); }));  // 15 - lane of 16
  const auto both = [&](auto swap) {
    Words x = __builtin_bit_cast(Words, v), y;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const auto r = swap(x.w[i]);
      x.w[i] = r[0];
      y.w[i] = r[1];
    }
    v = f(__builtin_bit_cast(T, x), __builtin_bit_cast(T, y));
  };
  both([](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
  both([](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
  return v;
}
__device__ inline float wave_max(float v) {
  return over_wave(v, [](float a, float b) { return __builtin_fmaxf(a, b); });
}
__device__ inline double wave_sum(double v) {
  return over_wave(v, [](double a, double b) { return a + b; });
}

// A number that at least k (1 to 64) of the wave's v reach: the k-th largest, but for the last BITS bits, or a
// lower one where some are equal.
template <int BITS>
__device__ inline uint32_t reached_by(uint32_t v, uint32_t k) {
  uint32_t t = 0;
  if (k <= 6) {  // the largest taken away k times, 60 cycles each; else a bit at a time, 30 each
    for (uint32_t r = 0; r < k; ++r) {
      t = over_wave(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
      v = v == t ? 0 : v;
    }
    return __builtin_amdgcn_readfirstlane(t);
  }
#pragma unroll
  for (int b = 31; b >= BITS; --b) {
    const uint32_t x = t | 1u << b;
    if ((uint32_t)__builtin_popcountll(__ballot(v >= x)) >= k) t = x;
  }
  return t;
}

// A list of unequal keys in LDS; A of one word, or of two where equal first words are told apart by the second.
struct Key1 {
  uint64_t a;
  __device__ bool over(const Key1 &o) const { return a > o.a; }
  __device__ Key1 from(int lane) const { return {__shfl_xor(a, lane)}; }
};
struct Key2 {
  uint64_t a, b;
  __device__ bool over(const Key2 &o) const { return a > o.a || (a == o.a && b > o.b); }
  __device__ Key2 from(int lane) const { return {__shfl_xor(a, lane), __shfl_xor(b, lane)}; }
};

// The largest of the threads' keys, for all of them.
template <uint32_t WAVES, typename K>
__device__ inline K largest(K best, K *waves) {
#pragma unroll
  for (int s = 32; s; s >>= 1) {
    const K o = best.from(s);
    if (o.over(best)) best = o;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = best;
  __syncthreads();
  best = waves[0];
#pragma unroll
  for (uint32_t w = 1; w < WAVES; ++w)
    if (waves[w].over(best)) best = waves[w];
  return best;
}

// The n largest of list[0 .. count - 1] to its front, in order.  Few keys are ranked by counting
// those over each; of many (a threshold that let equal logits through) the largest is taken n times.
template <uint32_t WAVES, typename K>
__device__ inline uint32_t keep_best(K *list, uint32_t count, uint32_t n, K none, K *waves, K *best) {
  constexpr uint32_t kT = WAVES * 64, kMine = (kRank + kT - 1) / kT;
  __syncthreads();
  if (count <= kRank) {
    K mine[kMine];
    uint32_t rank[kMine];
#pragma unroll
    for (uint32_t j = 0; j < kMine; ++j) {
      const uint32_t i = threadIdx.x + j * kT;
      mine[j] = i < count ? list[i] : none;
      rank[j] = i < count ? 0 : n;
    }
    if ((threadIdx.x & ~63u) < count) {  // (waves without a key do not count)
      for (uint32_t i = 0; i < count; ++i) {
        const K k = list[i];
#pragma unroll
        for (uint32_t j = 0; j < kMine; ++j) rank[j] += k.over(mine[j]);
      }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kMine; ++j)
      if (rank[j] < n) list[rank[j]] = mine[j];
  } else {
    K top = none;
    top.a = ~0ull;  // (over every key)
    for (uint32_t r = 0; r < n; ++r) {
      K mine = none;
      for (uint32_t i = threadIdx.x; i < count; i += kT) {
        const K k = list[i];
        if (top.over(k) && k.over(mine)) mine = k;
      }
      top = largest<WAVES>(mine, waves);
      if (threadIdx.x == 0) best[r] = top;
    }
    __syncthreads();
    if (threadIdx.x < n) list[threadIdx.x] = best[threadIdx.x];
  }
  __syncthreads();
  return count < n ? count : n;
}

// The sum over a piece of 2^(L (x - top)), L log2(e) in f32, top its largest logit: the log of a row's sum of
// exponentials is top + log2(sum) / L.
struct Stat {
  double sum;
  float top, pad;
};

// kPer logits of a thread as they lie in memory, in vectors of V.  A thread sums its powers about a point of
// the largest so far, power(x, point(top)) = 2^(L (x - top)) but for a factor that `rest` makes up for.
// f32: the difference is rounded, then the product.  f16: one fused multiply-add with the f16 as it is; the point L top is
// rounded, by 2^-8 at most, which all powers have in common.
template <typename T>
struct Logits;
template <>
struct Logits<float> {
  static constexpr uint32_t V = 4;
  typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
  vec v[kPer / V];
  __device__ void nothing(uint32_t e) { v[e / V][e % V] = -INFINITY; }
  __device__ void ban(uint32_t j, uint32_t bits) {
#pragma unroll
    for (uint32_t e = 0; e < V; ++e) v[j][e] = bits >> e & 1 ? -INFINITY : v[j][e];
  }
  __device__ void clean() {
#pragma unroll
    for (uint32_t e = 0; e < kPer; ++e) {
      const float x = v[e / V][e % V];
      v[e / V][e % V] = x > -INFINITY ? __builtin_fminf(x, kMost) : -INFINITY;
    }
  }
  static constexpr float kTop = kMost;
  static __device__ float point(float top) { return top; }
  __device__ float power(uint32_t e, float c) const { return __builtin_amdgcn_exp2f((at(e) - c) * kLog2e); }
  static __device__ float shift(float from, float to) { return __builtin_amdgcn_exp2f((from - to) * kLog2e); }
  static __device__ float rest(float, float) { return 1.0f; }
  __device__ float at(uint32_t e) const { return v[e / V][e % V]; }
  __device__ float most() const {
    float m = at(0);
#pragma unroll
    for (uint32_t e = 1; e < kPer; ++e) m = __builtin_fmaxf(m, at(e));
    return m;
  }
};
template <>
struct Logits<f16> {
  static constexpr uint32_t V = 8;
  typedef f16 vec __attribute__((ext_vector_type(8), aligned(2)));
  vec v[kPer / V];
  __device__ void nothing(uint32_t e) { v[e / V][e % V] = -(f16)INFINITY; }
  __device__ void ban(uint32_t j, uint32_t bits) {
    u32x4 w = __builtin_bit_cast(u32x4, (f16x8)v[j]);
#pragma unroll
    for (uint32_t e = 0; e < V; e += 2) {
      const uint32_t lo = (uint32_t)__builtin_amdgcn_sbfe((int)bits, e, 1), hi = (uint32_t)__builtin_amdgcn_sbfe((int)bits, e + 1, 1);
      const uint32_t m = (lo & 0xffffu) | (hi & 0xffff0000u);
      w[e / 2] = (w[e / 2] & ~m) | (0xfc00fc00u & m);
    }
    v[j] = __builtin_bit_cast(f16x8, w);
  }
  __device__ void clean() {
#pragma unroll
    for (uint32_t e = 0; e < kPer; ++e) {
      const float x = (float)v[e / V][e % V];
      v[e / V][e % V] = (f16)(x > -INFINITY ? __builtin_fminf(x, kTop) : -INFINITY);
    }
  }
  static constexpr float kTop = 65504;
  static __device__ float point(float top) { return top * kLog2e; }
  __device__ float power(uint32_t e, float c) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(at(e), kLog2e, -c)); }
  static __device__ float shift(float from, float to) { return __builtin_amdgcn_exp2f(from - to); }
  static __device__ float rest(float top, float c) { return __builtin_amdgcn_exp2f(__builtin_fmaf(-top, kLog2e, c)); }
  __device__ float at(uint32_t e) const { return (float)v[e / V][e % V]; }
  __device__ float most() const {
    f16x8 m = v[0];
#pragma unroll
    for (uint32_t j = 1; j < kPer / V; ++j) m = __builtin_elementwise_max(m, (f16x8)v[j]);
    const f16x4 a = __builtin_elementwise_max((f16x4){m[0], m[1], m[2], m[3]}, (f16x4){m[4], m[5], m[6], m[7]});
    const f16x2 b = __builtin_elementwise_max((f16x2){a[0], a[1]}, (f16x2){a[2], a[3]});
    return __builtin_fmaxf((float)b[0], (float)b[1]);
  }
};

// The n largest of a wave's list[0 .. count - 1] to its front, in order; returns how many there are.  (The
// wave alone reads and writes the list.)
__device__ inline uint32_t keep_in_wave(uint64_t *list, uint32_t count, uint32_t n) {
  const uint32_t lane = threadIdx.x & 63;
  constexpr uint32_t kMine = 4;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (count <= 64 * kMine) {
    uint64_t mine[kMine];
    uint32_t rank[kMine];
#pragma unroll
    for (uint32_t j = 0; j < kMine; ++j) {
      mine[j] = lane + j * 64 < count ? list[lane + j * 64] : 0;
      rank[j] = lane + j * 64 < count ? 0 : n;
    }
    if (count <= 64) {
#pragma unroll 8
      for (uint32_t i = 0; i < count; ++i) rank[0] += list[i] > mine[0];
    } else if (count <= 128) {
#pragma unroll 4
      for (uint32_t i = 0; i < count; ++i) {
        const uint64_t k = list[i];
        rank[0] += k > mine[0];
        rank[1] += k > mine[1];
      }
    } else {
#pragma unroll 4
      for (uint32_t i = 0; i < count; ++i) {
        const uint64_t k = list[i];
#pragma unroll
        for (uint32_t j = 0; j < kMine; ++j) rank[j] += k > mine[j];
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (uint32_t j = 0; j < kMine; ++j)
      if (rank[j] < n) list[rank[j]] = mine[j];
  } else {  // (a threshold that let many equal logits through)
    uint64_t top = ~0ull, found = 0;
    for (uint32_t r = 0; r < n; ++r) {
      Key1 best{0};
      for (uint32_t i = lane; i < count; i += 64)
        if (list[i] < top && list[i] > best.a) best.a = list[i];
#pragma unroll
      for (int s = 32; s; s >>= 1) {
        const Key1 o = best.from(s);
        if (o.over(best)) best = o;
      }
      top = best.a;
      if (lane == r) found = top;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (lane < n) list[lane] = found;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  return count < n ? count : n;
}

// Those of a wave's keys whose logit reaches `least` to the list's front, as they come; returns how many.
__device__ inline uint32_t sift_in_wave(uint64_t *list, uint32_t count, uint32_t least) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t kept = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (uint32_t i = 0; i < count; i += 64) {
    const uint64_t k = i + lane < count ? list[i + lane] : 0;
    const bool in = (uint32_t)(k >> 32) >= least;
    const uint64_t who = __ballot(in);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in) list[kept + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = k;
    kept += (uint32_t)__builtin_popcountll(who);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  return kept;
}

// Grid (pieces, rows).  keys [rows][pieces][n], stats [rows][pieces].
// A wave goes through its quarter of every tile by itself, with a list of its own of the logits that may be among the n
// best; the waves tell each other how many of theirs reach what (the n-th best of any is a bound for all), and meet at the end.
constexpr uint32_t kMore = 48, kList = 64 * kPer + kMaxBest + kMore;  // a list is cut down from n + kMore keys on
template <typename T, bool BAN>
__global__ __launch_bounds__(kThreads) void beam_part_kernel(const T *__restrict__ logits, uint32_t ld, uint32_t vocab,
                                                             uint32_t piece, uint32_t n, const uint32_t *__restrict__ ban,
                                                             uint32_t ban_ld, const float *__restrict__ score,
                                                             const uint8_t *__restrict__ done, uint64_t *keys, Stat *stats) {
  typedef Logits<T> L;
  constexpr uint32_t V = L::V;
  __shared__ uint64_t lists[kWaves][kList];
  __shared__ uint32_t reached, counts[kWaves];
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves];
  const uint32_t row = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T *x = logits + (size_t)row * ld;
  if (BAN) ban += (size_t)row * ban_ld;
  const uint32_t first = blockIdx.x * piece, last = vocab - first < piece ? vocab : first + piece;
  struct Tile {
    L l;
    uint32_t bits[kPer / V];
  };
  const auto fetch = [&](uint32_t at, Tile &t) {  // a whole tile
#pragma unroll
    for (uint32_t j = 0; j < kPer / V; ++j) {
      const uint32_t i = (j * kThreads + threadIdx.x) * V;
      t.l.v[j] = *reinterpret_cast<const typename L::vec *>(x + at + i);
      if (BAN) t.bits[j] = ban[at / 32 + i / 32] >> (i % 32);
    }
  };
  // the row's whole tiles, the next one always on its way, then what is left of a tile
  const uint32_t whole = first + (last - first) / kTile * kTile;
  const auto fetch_rest = [&](Tile &t) {
#pragma unroll
    for (uint32_t j = 0; j < kPer / V; ++j) {
      const uint32_t i = whole + (j * kThreads + threadIdx.x) * V;
#pragma unroll
      for (uint32_t e = 0; e < V; ++e) {
        t.l.nothing(j * V + e);
        if (i + e < last) t.l.v[j][e] = x[i + e];
      }
      if (BAN) t.bits[j] = i < last ? ban[i / 32] >> (i % 32) : 0;
    }
  };
  Tile now;
  if (whole > first) {
    fetch(first, now);
  } else {
    fetch_rest(now);
  }
  if (!(score[row] > -INFINITY) || (done && done[row])) return;  // (the second kernel does not ask)
  constexpr uint32_t kLeast = 0x017fffffu;  // order(-kMost)
  if (threadIdx.x == 0) reached = kLeast;

  uint64_t *list = lists[wave];
  uint32_t held = 0, mine = kLeast;
  float top = -INFINITY, c = 0, sum = 0;
  const auto take = [&](uint32_t at) {
    if (BAN) {
#pragma unroll
      for (uint32_t j = 0; j < kPer / V; ++j) now.l.ban(j, now.bits[j]);
    }
    // One pass over the thread's logits.  A NaN or an infinity among them (rare, and only asked
    // of the results: the maximum passes over a NaN) takes another over what they count as.
    float m, top1, c1, sum1;
    const auto pass = [&] {
      m = now.l.most();
      top1 = top;
      c1 = c;
      sum1 = sum;
      if (m > top && m >= -kMost) {
        top1 = m;
        c1 = L::point(m);
        sum1 = top > -INFINITY ? sum * L::shift(c, c1) : 0.0f;
      }
      if (top1 > -INFINITY) {
        float s[4];
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) s[e] = now.l.power(e, c1);
#pragma unroll
        for (uint32_t e = 4; e < kPer; ++e) s[e % 4] += now.l.power(e, c1);
        sum1 += (s[0] + s[1]) + (s[2] + s[3]);
      }
      return m <= L::kTop && sum1 == sum1;
    };
    if (!pass()) {
      now.l.clean();
      pass();
    }
    top = top1;
    c = c1;
    sum = sum1;
    // `mine`: what n logits reach.  At the first tile n / 4 lanes of each wave reach its bound, so n reach the least of
    // the four; later n keys of the wave's list reach the n-th of them, which holds for the other waves too.
    if (at == first) {
      const uint32_t b = reached_by<8>(order(m + 0.0f), (n + kWaves - 1) / kWaves);
      if (lane == 0) counts[wave] = b;
      __syncthreads();
      uint32_t least = counts[0];
#pragma unroll
      for (uint32_t w = 1; w < kWaves; ++w) least = counts[w] < least ? counts[w] : least;
      mine = __builtin_amdgcn_readfirstlane(least > mine ? least : mine);
    } else {
      const uint32_t all = __builtin_amdgcn_readfirstlane(*(volatile uint32_t *)&reached);
      mine = all > mine ? all : mine;
      if (held > n + kMore) {
        held = sift_in_wave(list, held, mine);
        if (held > n + kMore / 2) {
          held = keep_in_wave(list, held, n);
          mine = __builtin_amdgcn_readfirstlane((uint32_t)(list[n - 1] >> 32));
          if (lane == 0) atomicMax(&reached, mine);
        }
      }
    }
    const float threshold = unorder(mine);
    if (!__any(m >= threshold)) return;
#pragma unroll
    for (uint32_t e = 0; e < kPer; ++e) {
      const bool in = now.l.at(e) >= threshold;
      const uint64_t who = __ballot(in);
      if (who) {
        const uint32_t token = at + ((e / V) * kThreads + threadIdx.x) * V + e % V;
        if (in) list[held + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] =
            (uint64_t)order(now.l.at(e) + 0.0f) << 32 | (uint32_t)~token;
        held += (uint32_t)__builtin_popcountll(who);
      }
    }
  };
  for (uint32_t at = first; at < whole; at += kTile) {
    Tile next;
    fetch(at + kTile < whole ? at + kTile : at, next);
    take(at);
    now = next;
  }
  if (whole < last) {
    if (whole > first) fetch_rest(now);
    take(whole);
  }
  if (held > 64) {
    const uint32_t all_reach = __builtin_amdgcn_readfirstlane(*(volatile uint32_t *)&reached);
    held = sift_in_wave(list, held, all_reach > mine ? all_reach : mine);
  }
  held = keep_in_wave(list, held, n);
  // the sum over the threads, about the largest logit
  float all = wave_max(top);
  double total = wave_sum(top > -INFINITY ? (double)(sum * L::rest(top, c) * __builtin_amdgcn_exp2f((top - all) * kLog2e)) : 0.0);
  __syncthreads();  // (the bounds in counts are read)
  if (lane == 0) {
    counts[wave] = held;
    tops[wave] = all;
    sums[wave] = total;
  }
  __syncthreads();
  // a key's place: its place in its wave's list, and those over it in the others'
  const size_t out = (size_t)row * gridDim.x + blockIdx.x;
  uint32_t rank = lane, found = 0;
  const uint64_t key = lane < held ? list[lane] : 0;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) {
    const uint32_t k = counts[w];
    found += k;
    if (w != wave) {
#pragma unroll 4
      for (uint32_t i = 0; i < k; ++i) rank += lists[w][i] > key;
    }
  }
  if (lane < held && rank < n) keys[out * n + rank] = key;
  if (threadIdx.x >= found && threadIdx.x < n) keys[out * n + threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    all = tops[0];
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) all = __builtin_fmaxf(all, tops[w]);
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w)
      if (tops[w] > -INFINITY) total += sums[w] * (double)__builtin_amdgcn_exp2f((tops[w] - all) * kLog2e);
    stats[out] = {total, all, 0};
  }
}

// A workgroup per group, its waves dealt out to the beams; a wave works out its beam's log sum
// by itself.  The second word of a key tells equal candidates apart: the lower beam, then (as within a
// beam everywhere) the larger logit, then the lower token.
constexpr uint32_t kJoin = 1024, kJoinWaves = kJoin / 64;
constexpr uint32_t kHeld = 2048;
__global__ __launch_bounds__(kJoin) void beam_join_kernel(const uint64_t *__restrict__ keys, const Stat *__restrict__ stats,
                                                          const float *score, const uint8_t *__restrict__ done,
                                                          uint32_t beams, uint32_t pieces, uint32_t n, uint32_t eos,
                                                          float *out_score, uint32_t *out_parent, uint32_t *out_token) {
  __shared__ Key2 list[kHeld], waves[kJoinWaves], best[kMaxBest];
  __shared__ uint32_t count_, bound[kJoinWaves];
  __shared__ uint8_t over[kMaxBeams];
  const uint32_t g = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) count_ = 0;
  const uint32_t each = pieces * n;
  // beams at most 16: `parts` waves each; more: two or less a wave
  const uint32_t parts = beams <= kJoinWaves ? kJoinWaves / beams : 1;
  const uint32_t part = beams <= kJoinWaves ? wave / beams : 0, first_beam = beams <= kJoinWaves ? wave % beams : wave;
  const Key2 none{0, 0};
  // f(k) for every candidate of the wave's beams
  const auto every = [&](auto f) {
    if (part >= parts) return;
    for (uint32_t w = first_beam; w < beams; w += kJoinWaves) {
      const size_t row = (size_t)g * beams + w;
      const uint64_t *mine = keys + row * each;
      const Stat t = lane < pieces ? stats[row * pieces + lane] : Stat{0, -INFINITY, 0};
      const uint32_t at = part * 64 + lane;
      uint64_t k = at < each ? mine[at] : 0;
      const float s = __builtin_fminf(__builtin_fmaxf(score[row], -INFINITY), FLT_MAX);
      const bool is_done = done && done[row];
      const uint64_t tie = (uint64_t)(kMaxBeams - 1 - w) << 59;
      if (lane == 0 && part == 0) over[w] = is_done;
      if (!(s > -INFINITY)) continue;
      if (is_done) {
        if (at == 0) f(Key2{order((double)s + 0.0), tie});
        continue;
      }
      const float top = wave_max(t.top);
      if (!(top > -INFINITY)) continue;  // nothing is left of the row
      const double sum = wave_sum(t.top > -INFINITY ? t.sum * (double)__builtin_amdgcn_exp2f((t.top - top) * kLog2e) : 0.0);
      const double lse = (double)top + log2(sum) * (1.0 / (double)kLog2e);
      for (uint32_t i = at; i < each; i += parts * 64) {
        const uint64_t after = i + parts * 64 < each ? mine[i + parts * 64] : 0;
        if (k)
          f(Key2{order((double)s + ((double)unorder((uint32_t)(k >> 32)) - lse) + 0.0),
                 tie | (k >> 32) << kTokenBits | ((uint32_t)k & kTokenMask)});
        k = after;
      }
    }
  };
  // n lanes of some wave reach its bound: only what reaches the largest bound counts
  const auto threshold_of = [&](uint32_t most) {
    const uint32_t b = reached_by<8>(most, n);
    if (lane == 0) bound[wave] = b;
    __syncthreads();
    uint32_t t = 0;
#pragma unroll
    for (uint32_t w = 0; w < kJoinWaves; ++w) t = bound[w] > t ? bound[w] : t;
    return t;
  };
  const auto put = [&](uint32_t place, const Key2 &k) {
    const size_t o = (size_t)g * n + place;
    const bool there = k.a > kNoCandidate;
    const uint32_t w = kMaxBeams - 1 - (uint32_t)(k.b >> 59), token = ~(uint32_t)k.b & kTokenMask;
    out_score[o] = there ? (float)unorder(k.a) : -INFINITY;
    out_parent[o] = there ? w : place < beams ? place : beams - 1;
    out_token[o] = there && !over[w] ? token : eos;
  };
  if (beams <= kJoinWaves && each <= parts * 64) {
    // a candidate a lane: kept in a register, the few that count ranked by counting those over each
    Key2 mine = none;
    every([&](const Key2 &k) { mine = k; });
    const uint32_t threshold = threshold_of((uint32_t)(mine.a >> 32));
    const bool in = mine.a > kNoCandidate && (uint32_t)(mine.a >> 32) >= threshold;
    const uint64_t who = __ballot(in);
    uint32_t to = 0;
    if (lane == 0 && who) to = atomicAdd(&count_, (uint32_t)__builtin_popcountll(who));
    to = __builtin_amdgcn_readfirstlane(to) + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
    if (in) list[to] = mine;
    __syncthreads();
    const uint32_t c = count_;
    if (threadIdx.x < c) {
      const Key2 k = list[threadIdx.x];
      uint32_t rank = 0;
#pragma unroll 4
      for (uint32_t i = 0; i < c; ++i) rank += list[i].over(k);
      if (rank < n) put(rank, k);
    } else if (threadIdx.x < n) {
      put(threadIdx.x, none);
    }
    return;
  }
  uint32_t most = 0;
  every([&](const Key2 &k) {
    const uint32_t h = (uint32_t)(k.a >> 32);
    most = h > most ? h : most;
  });
  const uint32_t threshold = threshold_of(most);
  every([&](const Key2 &k) {
    if ((uint32_t)(k.a >> 32) < threshold) return;
    const uint32_t at = atomicAdd(&count_, 1u);
    if (at < kHeld) list[at] = k;
  });
  __syncthreads();
  const uint32_t c = count_;
  Key2 mine = none;
  if (c <= kHeld) {
    const uint32_t held = keep_best<kJoinWaves>(list, c, n, none, waves, best);
    if (threadIdx.x < held) mine = list[threadIdx.x];
  } else {
    Key2 top{~0ull, ~0ull};
    for (uint32_t r = 0; r < n; ++r) {
      Key2 mine_best = none;
      every([&](const Key2 &k) {
        if (top.over(k) && k.over(mine_best)) mine_best = k;
      });
      top = largest<kJoinWaves>(mine_best, waves);
      if (threadIdx.x == r) mine = top;
    }
  }
  if (threadIdx.x < n) put(threadIdx.x, mine);
}

// How a selection is cut: `piece` logits per workgroup, whole tiles, at most 64 pieces a row; kWant workgroups in all
// (64 x 8 beams of 131072, the first kernel: 1024 or more, two pieces a row, 40 us; 512 47; 2048 43).
constexpr uint32_t kWant = 1024;
struct Cut {
  uint32_t piece, pieces;
};
Cut cut(uint32_t rows, uint32_t vocab) {
  const uint32_t tiles = (vocab + kTile - 1) / kTile;
  uint32_t want = kWant / rows;
  want = want < 1 ? 1 : want > kMaxPieces ? kMaxPieces : want;
  const uint32_t per = (tiles + want - 1) / want;
  return {per * kTile, (tiles + per - 1) / per};
}

bool beam_shape_ok(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t n) {
  return groups >= 1 && beams >= 1 && beams <= kMaxBeams && n >= 1 && n <= kMaxBest && vocab >= 1 &&
         vocab <= kTokenMask && (uint64_t)groups * beams <= 65535;
}

// ---------------------------------------------------------------- gather
struct States {
  uint8_t *dst[kMaxBeams];
  const uint8_t *src[kMaxBeams];
};

// Grid (columns / 256, groups, states): a thread has a column of U bytes of the states of all beams
// of a group, and reads every one that it writes from before it writes.  Bound by memory: 40 slots of 5 beams, 8 states
// of 448 rows of 5120 bytes, from one array to another 184 us, 733 MB written and what the distinct parents have read.
// Stores past the caches: what is written is not read again here, and the states fill them many times over (plain
// ones 278 us).  Loads without branches, a wave's rows or, where there is nothing to move, one address for all: behind
// branches each waited for those before (234 us, groups of 8 beams 333 instead of 205).
template <typename U, int W>
__global__ __launch_bounds__(256) void beam_gather_kernel(States st, size_t stride, size_t row_bytes, uint32_t rows,
                                                          const uint32_t *__restrict__ lens,
                                                          const uint32_t *__restrict__ parent, uint32_t ldp, uint32_t beams) {
  const uint32_t g = blockIdx.y;
  uint8_t *dst = st.dst[blockIdx.z] + (size_t)g * beams * stride;
  const uint8_t *src = st.src[blockIdx.z] + (size_t)g * beams * stride;
  const size_t off = ((size_t)blockIdx.x * 256 + threadIdx.x) * sizeof(U);
  uint32_t from[W];
  size_t end[W];  // bytes to move
#pragma unroll
  for (int i = 0; i < W; ++i) {
    uint32_t f = i < (int)beams ? parent[(size_t)g * ldp + i] : beams, n = rows;
    if (f >= beams || (f == (uint32_t)i && src == dst)) {
      f = 0;
      n = 0;
    } else if (lens && lens[g * beams + f] < n) {
      n = lens[g * beams + f];
    }
    from[i] = f;
    end[i] = n * row_bytes;
  }
  bool cut = rows * row_bytes < sizeof(U);
#pragma unroll
  for (int i = 0; i < W; ++i) cut |= off < end[i] && end[i] - off < sizeof(U);
  if (!cut) {
    U v[W];
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = *reinterpret_cast<const U *>(src + from[i] * stride + (off < end[i] ? off : 0));
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (off < end[i]) __builtin_nontemporal_store(v[i], reinterpret_cast<U *>(dst + i * stride + off));
  } else {  // a row ends inside U: word by word
    for (size_t at = off; at < off + sizeof(U); at += 4) {
      uint32_t v[W];
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (at < end[i]) v[i] = *reinterpret_cast<const uint32_t *>(src + from[i] * stride + at);
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (at < end[i]) *reinterpret_cast<uint32_t *>(dst + i * stride + at) = v[i];
    }
  }
}

template <typename U>
void gather(const States &st, const madi_beam_states *s, uint32_t columns, uint32_t n) {
  const dim3 grid(columns, s->groups, n);
  const auto go = [&](auto kernel) {
    kernel<<<grid, 256, 0, stream()>>>(st, s->stride, s->row_bytes, s->rows, s->lens, s->parent, s->ldp, s->beams);
  };
  if (s->beams <= 4) go(beam_gather_kernel<U, 4>);
  else if (s->beams <= 8) go(beam_gather_kernel<U, 8>);
  else if (s->beams <= 16) go(beam_gather_kernel<U, 16>);
  else go(beam_gather_kernel<U, 32>);
}

}  // namespace

extern "C" size_t madi_beam_bytes(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t n) {
  if (!beam_shape_ok(groups, beams, vocab, n)) return 0;
  const Cut c = cut(groups * beams, vocab);
  return (size_t)groups * beams * c.pieces * (sizeof(Stat) + (size_t)n * 8);
}

extern "C" int madi_beam_select(const madi_beam *s) {
  const char *what = "madi_beam_select";
  if (!s) return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (s->groups == 0 && s->beams >= 1 && s->beams <= kMaxBeams) return initialized() ? MADI_OK : fail(MADI_ERR_NOT_INIT, "%s: madi_init has not succeeded", what);
  if (!beam_shape_ok(s->groups, s->beams, s->vocab, s->n))
    return fail(MADI_ERR_SHAPE, "%s: %u groups of %u beams, vocab %u, n %u (65535 rows, beams to 32, vocab below 2^27, n to 64)",
                what, s->groups, s->beams, s->vocab, s->n);
  const uint32_t rows = s->groups * s->beams, words = (s->vocab + 31) / 32;
  if (s->dtype != MADI_F16 && s->dtype != MADI_F32) return fail(MADI_ERR_ARG, "%s: dtype %d", what, s->dtype);
  if (s->ld < s->vocab) return fail(MADI_ERR_SHAPE, "%s: rows of logits are %u apart but %u long", what, s->ld, s->vocab);
  if (s->ban && s->ban_ld && s->ban_ld < words)
    return fail(MADI_ERR_SHAPE, "%s: rows of ban are %u words apart but %u long", what, s->ban_ld, words);
  if (!s->logits || !s->score || !s->out_score || !s->out_parent || !s->out_token || !s->work)
    return fail(MADI_ERR_NULL, "%s: null pointer", what);
  const size_t es = s->dtype == MADI_F32 ? 4 : 2;
  if (!aligned(s->logits, es) || !aligned(s->work, 16)) return fail(MADI_ERR_ALIGN, "%s: logits must be aligned to their type, work to 16 bytes", what);
  for (const void *q : {(const void *)s->score, (const void *)s->ban, (const void *)s->out_score, (const void *)s->out_parent, (const void *)s->out_token})
    if (!aligned(q, 4)) return fail(MADI_ERR_ALIGN, "%s: arrays must be 4-byte aligned", what);
  const Cut c = cut(rows, s->vocab);
  const size_t need = madi_beam_bytes(s->groups, s->beams, s->vocab, s->n);
  if (s->work_bytes < need) return fail(MADI_ERR_SHAPE, "%s: %zu bytes of work, needs %zu", what, s->work_bytes, need);
  const size_t out = (size_t)s->groups * s->n * 4;
  const Extent x[] = {{s->logits, ((size_t)(rows - 1) * s->ld + s->vocab) * es, false},
                      {s->score, s->score == s->out_score && s->n == s->beams ? 0 : (size_t)rows * 4, false},
                      {s->done, s->done ? rows : 0, false},
                      {s->ban, s->ban ? ((size_t)(rows - 1) * s->ban_ld + words) * 4 : 0, false},
                      {s->out_score, out, true}, {s->out_parent, out, true}, {s->out_token, out, true}, {s->work, need, true}};
  if (int rc = disjoint(what, x)) return rc;
  if (!initialized()) return fail(MADI_ERR_NOT_INIT, "%s: madi_init has not succeeded", what);
  if (int rc = ready(x)) return rc;
  Stat *stats = static_cast<Stat *>(s->work);
  uint64_t *keys = reinterpret_cast<uint64_t *>(stats + (size_t)rows * c.pieces);
  const dim3 grid(c.pieces, rows);
  const auto go = [&](auto kernel, auto *logits) {
    kernel<<<grid, kThreads, 0, stream()>>>(logits, s->ld, s->vocab, c.piece, s->n, s->ban, s->ban_ld, s->score, s->done, keys, stats);
  };
  if (s->dtype == MADI_F32) {
    const float *logits = static_cast<const float *>(s->logits);
    s->ban ? go(beam_part_kernel<float, true>, logits) : go(beam_part_kernel<float, false>, logits);
  } else {
    const f16 *logits = static_cast<const f16 *>(s->logits);
    s->ban ? go(beam_part_kernel<f16, true>, logits) : go(beam_part_kernel<f16, false>, logits);
  }
  if (int rc = check_launch(what)) return rc;
  beam_join_kernel<<<s->groups, kJoin, 0, stream()>>>(keys, stats, s->score, s->done, s->beams, c.pieces, s->n, s->eos, s->out_score, s->out_parent, s->out_token);
  return check_launch(what);
}

extern "C" int madi_beam_gather(const madi_beam_states *s) {
  const char *what = "madi_beam_gather";
  if (!s) return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (s->beams < 1 || s->beams > kMaxBeams || (uint64_t)s->groups * s->beams > 65535)
    return fail(MADI_ERR_SHAPE, "%s: %u groups of %u beams (beams to 32, 65535 slots)", what, s->groups, s->beams);
  if (s->ldp < s->beams) return fail(MADI_ERR_SHAPE, "%s: rows of parent are %u apart but %u long", what, s->ldp, s->beams);
  if (s->n_states > kMaxBeams) return fail(MADI_ERR_SHAPE, "%s: %u states (at most 32)", what, s->n_states);
  if (s->row_bytes % 4 || s->stride % 4) return fail(MADI_ERR_ALIGN, "%s: stride and row_bytes must be multiples of 4", what);
  if (s->row_bytes > (1ull << 40) || s->stride > (1ull << 40) || (s->rows && s->row_bytes > s->stride / s->rows))
    return fail(MADI_ERR_SHAPE, "%s: %u rows of %zu bytes, states %zu bytes apart", what, s->rows, s->row_bytes, s->stride);
  const size_t bytes = (size_t)s->rows * s->row_bytes, slots = (size_t)s->groups * s->beams;
  if (!s->parent || (s->n_states && !s->dst)) return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (!aligned(s->parent, 4) || !aligned(s->lens, 4)) return fail(MADI_ERR_ALIGN, "%s: arrays must be 4-byte aligned", what);
  const size_t extent = slots ? (slots - 1) * s->stride + bytes : 0;
  bool wide = s->stride % 16 == 0;
  States st{};
  const Extent read[] = {{s->parent, slots ? ((size_t)(s->groups - 1) * s->ldp + s->beams) * 4 : 0, false}, {s->lens, s->lens ? slots * 4 : 0, false}};
  for (uint32_t j = 0; j < s->n_states; ++j) {
    st.dst[j] = static_cast<uint8_t *>(s->dst[j]);
    st.src[j] = s->src ? static_cast<const uint8_t *>(s->src[j]) : st.dst[j];
    if (slots && bytes && (!st.dst[j] || !st.src[j])) return fail(MADI_ERR_NULL, "%s: null pointer", what);
    if (!aligned(st.dst[j], 4) || !aligned(st.src[j], 4)) return fail(MADI_ERR_ALIGN, "%s: states must be 4-byte aligned", what);
    wide = wide && aligned(st.dst[j], 16) && aligned(st.src[j], 16);
    for (const Extent &e : read)
      if (kv4_overlap(st.dst[j], extent, e.p, e.bytes)) return fail(MADI_ERR_ARG, "%s: parent or lens lies in a state", what);
  }
  for (uint32_t j = 0; j < s->n_states; ++j)
    for (uint32_t i = 0; i < s->n_states; ++i)
      if ((i != j && kv4_overlap(st.dst[j], extent, st.dst[i], extent)) ||
          ((i != j || st.src[i] != st.dst[j]) && kv4_overlap(st.dst[j], extent, st.src[i], extent)))
        return fail(MADI_ERR_ARG, "%s: two states overlap", what);
  const size_t columns = (bytes + (wide ? 4095 : 1023)) / (wide ? 4096 : 1024);
  if (columns > 0xffffffu) return fail(MADI_ERR_SHAPE, "%s: states of %zu bytes", what, bytes);  // 2^32 threads
  if (!initialized()) return fail(MADI_ERR_NOT_INIT, "%s: madi_init has not succeeded", what);
  if (slots == 0 || s->n_states == 0 || bytes == 0) return MADI_OK;
  if (int rc = ready(read)) return rc;
  for (uint32_t j = 0; j < s->n_states; ++j) {
    const Extent x[] = {{st.src[j], extent, false}, {st.dst[j], extent, true}};
    if (int rc = ready(x)) return rc;
  }
  if (wide) gather<u32x4>(st, s, (uint32_t)columns, s->n_states);
  else gather<uint32_t>(st, s, (uint32_t)columns, s->n_states);
  return check_launch(what);
}
