// kv4_attn.hip -- attention over the 4-bit key/value cache (madi_kv4_attn; the
// format and the layout are in madi_q8.h).
//
// The query heads of a kv head and the rows of a sequence make the columns of
// the products: column c is row c / G, head c % G of the G = nh / nkv.  A wave
// takes 16 columns and walks the keys 32 at a time:
//   S^T = K Q^T, v_mfma_f32_16x16x32_f16 with 16 keys as rows and one 32-element
//     block as K: lane (g, r) passes row r's word (g, b) as eight f16 codes, and the
//     block's sum gets its key's scale in f32: S = sum_b s_b (Q K^T)_b.  (Codes
//     masked into f16 subnormals would need no bias taken off, but the matrix
//     core sums products of subnormals to 2^-18 only, against 2^-24.)
//   softmax over a running reference M that is raised only when a score passes the
//     largest at its last raise by 2^7 (in the exponents of 2), so most steps
//     exchange nothing between lanes.
//   O^T += V^T P^T, 32 keys as K and 16 elements as rows: P^T comes straight
//     from the S^T registers (lane (g, c) holds keys 4g..4g+3 of both tiles),
//     V as its codes from the words that hold four tokens, and the V scale of a
//     key and block goes into P: one rounding, of P s, instead of P's and V's.
//     P comes times 2^-e, e the exponent of the largest V scale that the column
//     has seen, so that P s stays within f16: 2^-e is part of the reference
//     M + e and costs nothing.
// A lane holds two of the 8 nb scales of its four keys and passes them to the
// other 15 through DPP broadcasts, which cost nothing in a multiplication.
// f32 rows: q and P s are each split in two f16 (22 bits).
//
// What it costs (us, f16 rows, d 128; one MI355X):
//   128 sequences of 8192, 32 heads over 8: 226 to 229, 1.21 GB at 5.3 TB/s of the 6.5
//     that a kernel which only reads reaches.  A step of 32 keys is 327 vector
//     instructions (144 make codes of nibbles, 48 apply the K scales, 48 make P s)
//     and 16 MFMAs: the vector pipe is busy 68 % of the time, the matrix pipe 13 %,
//     and 16 % of the waves' time is waiting for memory or barriers.
//   1 sequence of 131072: 40.5, 33 in the kernel (4.6 TB/s; eight steps per wave
//     do not hide a segment's beginning and end), 5.4 in the join.
//   1 token over 213 keys, 20 heads of 64, f32: 5.7, of which 3 are launch and
//     the rest five dependent memory latencies (length, pages, words, results in
//     LDS, store).
#include <type_traits>

#include "kv4.h"
#include "vmem.h"

using namespace madi;

namespace {

constexpr int kCols = 16;  // columns of a wave (MFMA columns)
constexpr int kKeys = 32;  // keys of a step
// A prompt's workgroup: waves, tiles of 16 columns per wave (two where the
// registers allow it), keys in a buffer (two buffers fit LDS).
constexpr int kPromptWaves = 8;
constexpr int prompt_tiles(int d, bool f32) { return d < 128 || (d == 128 && !f32) ? 2 : 1; }
constexpr int prompt_keys(int d) { return d == 256 ? 32 : 64; }
// What a prompt's workgroup takes for 64 keys, in tenths of the time in which a CU's
// sixteen waves of the other kernel take four steps.  Measured: 2048 rows of 4 heads of
// d over one over 8192 keys, 4 of those, us here and there, f16 rows 260 and 356, 316 and 346,
// 366 and 385, 525 and 653 (d 64, 96, 128, 256), f32 318 and 353, 413 and 396, 322 and 451.
constexpr uint32_t prompt_cost(int d, bool f32) {
  return f32 ? (d == 64 ? 36 : d == 96 ? 42 : 29) : d == 64 ? 29 : d == 96 ? 37 : d == 128 ? 38 : 31;
}
// f32 rows of 256 do not fit the registers (97 spilled): 1299 us there, 844 in the other kernel.
constexpr bool has_prompt_kernel(int d, bool f32) { return d < 256 || !f32; }
constexpr float kNever = -__FLT_MAX__;  // reference before any key was seen
// P is 2^(x - M) with M at first the largest x - 7, raised when an x passes M
// by 14: P at most 2^14, P s 2^-e at most 2^15 (f16 holds 2^16), and what
// rounds to nothing is 2^-32 of the largest P at the largest s.  (A reference that
// follows the largest score at each step would rescale 32 registers each time.)
constexpr float kLift = 7.0f, kRaise = 14.0f;
// Scores this far from 0 have f32 neighbours 2^-3 and more away (at 2^28 32, at 10^30 2^76),
// and M - 7 is no number there.  A column whose largest score is as far takes that
// score itself as the reference M, without e, and raises it with every larger one: P is at
// most 1, P s at most 9352.  A score is rounded before its reference is taken off, which
// is exact then: a multiply-add would leave in what the rounding of the reference
// took, 2^-24 of 10^10.  (327 vector instructions a step in place of 326, the same times.)
constexpr float kFar = 0x1p20f;
__device__ inline bool is_far(float limit) { return !(__builtin_fabsf(limit) < kFar); }

// What a segment costs beside its steps (finding it, its queries, the first
// words' latency, the waves' results put together), in steps.  (4, 8, 12 and 16 were
// timed on 48 ragged sequences and on 128 of 8192: 8 and 12 are the best of both.)
constexpr uint32_t kOverhead = 8;
// Workgroups that share the steps, at most.
constexpr uint32_t kMaxGroups = 1024;
// f32 numbers of a partial result: O [16][D], then the references and the sums.
template <int D>
constexpr size_t kShare = kCols * (D + 2);

// Workgroups of four waves that a CU holds at once, by registers (f32 rows: those of
// the low parts) and by LDS (the ring).
constexpr uint32_t resident(uint32_t d, bool f32) { return d == 256 ? 2 : f32 && d == 128 ? 3 : 4; }

// Waves of a workgroup that has a tile and head for itself and more than kFew steps:
// as many as fit a CU's registers.
constexpr uint32_t waves_alone(uint32_t d, bool f32) { return 4 * resident(d, f32) > 12 ? 16 : 8; }
constexpr uint32_t kFew = 8;

struct AttnArgs {
  Kv4Args kv;
  const void *q;
  void *out;
  float *work;         // partial results, two per workgroup
  uint32_t *starts;    // behind them: the items' starts, and the length of a share
  uint32_t ldq, ldo, group, window, causal;
  uint32_t tiles, items;  // column tiles of a sequence; tiles of all sequences
  float scale;
};

typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ inline f16x2 as_f16x2(uint32_t w) { return __builtin_bit_cast(f16x2, w); }
__device__ inline uint32_t as_u32(f16x2 v) { return __builtin_bit_cast(uint32_t, v); }
__device__ inline f16x8 as_f16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(f16x8, (u32x4){a, b, c, d});
}
__device__ inline f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// over the four lanes that share a column
__device__ inline void swap16(float v, float &x, float &y) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = __builtin_bit_cast(float, (uint32_t)s[0]);
  y = __builtin_bit_cast(float, (uint32_t)s[1]);
}
__device__ inline void swap32(float v, float &x, float &y) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  x = __builtin_bit_cast(float, (uint32_t)s[0]);
  y = __builtin_bit_cast(float, (uint32_t)s[1]);
}
__device__ inline float sum_across(float v) {
  float x, y;
  swap16(v, x, y);
  swap32(x + y, x, y);
  return x + y;
}
__device__ inline float max_across(float v) {
  float x, y;
  swap16(v, x, y);
  swap32(__builtin_fmaxf(x, y), x, y);
  return __builtin_fmaxf(x, y);
}
// over the wave
template <int CTRL>
__device__ inline float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ inline float wave_sum(float v) {
  v += dpp<0x121>(v);  // row_ror 1, 2, 4, 8
  v += dpp<0x122>(v);
  v += dpp<0x124>(v);
  v += dpp<0x128>(v);
  return sum_across(v);
}
__device__ inline float wave_max(float v) {
  v = __builtin_fmaxf(v, dpp<0x121>(v));
  v = __builtin_fmaxf(v, dpp<0x122>(v));
  v = __builtin_fmaxf(v, dpp<0x124>(v));
  v = __builtin_fmaxf(v, dpp<0x128>(v));
  return max_across(v);
}

// One step's 32 keys as they lie in the cache, and whether their pages exist.
// Scale i = x * 4 nb + 4 b + token (x 0 for K, 1 for V) of the four tokens of
// group g is half i % 2 of word i / 2, which lane i / 2 % 16 of the group holds.
template <int NB>
struct Step {
  static constexpr int kScaleWords = (NB + 3) / 4;
  uint32_t k[2][NB], v[2][NB], s[2][kScaleWords];
  bool there[2];
};

// Page numbers of the wave's next kListed steps, two per step, one per lane: `at`
// is the first step, the others come `stride` apart.  (A scalar load per step
// would be waited for with the step's LDS reads.)  Past the table's end any entry stands in.
constexpr int kListed = 32;
__device__ inline uint32_t list_pages(const Kv4Args &a, uint32_t seq, uint32_t at, uint32_t stride, uint32_t lane) {
  const uint32_t n = ((at + (lane >> 1) * stride) * kKeys + (lane & 1) * 16) >> a.shift;
  return kv4_const(a.table + (size_t)seq * a.max_pages + (n < a.max_pages ? n : 0));
}

// A wave's ring of steps in LDS.  Every lane reads back what it loaded itself,
// so a wave waits for its own loads only, and in registers there is one step.
// Words of K, V and scales of a tile as pieces of 16 (4 for what is left) bytes
// per lane; a piece's 64 lanes lie side by side.
template <int NB>
struct Ring {
  static constexpr int kWide = NB / 4, kNarrow = NB % 4;  // pieces of NB words
  static constexpr int kScales = Step<NB>::kScaleWords;
  static constexpr int kTile = 256 * (2 * NB + kScales), kBytes = 2 * kTile;
  static constexpr int kLoads = 2 * (2 * (kWide + kNarrow) + kScales);  // of a step
};
template <int NB>
__device__ inline void load_pieces(const uint8_t *from, uint32_t voff, uint32_t to) {
  constexpr int W = Ring<NB>::kWide, N = Ring<NB>::kNarrow;
  if constexpr (W > 0) global_dma<16>(from, voff, to);
  if constexpr (W > 1) global_dma<16, 16>(from, voff, to + 1024 - 16);
  if constexpr (N > 0) global_dma<4, 16 * W>(from, voff, to + 1024 * W - 16 * W);
  if constexpr (N > 1) global_dma<4, 16 * W + 4>(from, voff, to + 1024 * W + 256 - (16 * W + 4));
  if constexpr (N > 2) global_dma<4, 16 * W + 8>(from, voff, to + 1024 * W + 512 - (16 * W + 8));
}
template <int NB>
__device__ inline void read_pieces(uint32_t (&w)[NB], const uint8_t *from, uint32_t lane) {
#pragma unroll
  for (int n = 0; n < Ring<NB>::kWide; ++n) {
    const u32x4 v = *reinterpret_cast<const u32x4 *>(from + 1024 * n + 16 * lane);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[4 * n + i] = v[i];
  }
#pragma unroll
  for (int n = 0; n < Ring<NB>::kNarrow; ++n)
    w[4 * Ring<NB>::kWide + n] =
        *reinterpret_cast<const uint32_t *>(from + 1024 * Ring<NB>::kWide + 256 * n + 4 * lane);
}
// Starts the loads of the step at `key` into the ring's slot at LDS address
// `to`; returns which tiles have a page (bits 0 and 1).
template <int NB>
__device__ inline uint32_t fetch(const Kv4Args &a, const uint32_t (&pages)[2], uint32_t head, int32_t key, int32_t len,
                                 uint32_t lane, uint32_t to) {
  constexpr uint32_t D = NB * 32;
  const uint32_t r = lane & 15, g = lane >> 4;
  const uint32_t kv = r * (D / 2) + g * (4 * NB), vv = ((D / 2) << a.shift) + g * (2 * D) + r * (4 * NB);
  uint32_t there = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // a tile past the end or without a page: any valid one stands in
    const bool ok = key + 16 * i < len && pages[i] < a.n_pages;
    there |= ok ? 1u << i : 0;
    const uint32_t off = (uint32_t)(key + 16 * i) & ((1u << a.shift) - 1);
    const uint8_t *blk = kv4_block(a, ok ? pages[i] : 0, head, D);
    const uint32_t at = to + i * Ring<NB>::kTile;
    load_pieces<NB>(blk, kv + off * (D / 2), at);
    load_pieces<NB>(blk, vv + off * (D / 2), at + 256 * NB);
#pragma unroll
    for (uint32_t n = 0; n < Ring<NB>::kScales; ++n) {
      const uint32_t w = 16 * n + r;  // (nb < 4: lanes past the words hold the last one)
      global_dma<4>(blk, (D << a.shift) + g * (D / 2) + 4 * (w < 4 * NB ? w : 4 * NB - 1) + off * (D / 8),
                    at + 512 * NB + 256 * n);
    }
  }
  return there;
}
template <int NB>
__device__ inline void read_step(Step<NB> &t, const uint8_t *slot, uint32_t there, uint32_t lane) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t *at = slot + i * Ring<NB>::kTile;
    read_pieces<NB>(t.k[i], at, lane);
    read_pieces<NB>(t.v[i], at + 256 * NB, lane);
#pragma unroll
    for (int n = 0; n < Ring<NB>::kScales; ++n)
      t.s[i][n] = *reinterpret_cast<const uint32_t *>(at + 512 * NB + 256 * n + 4 * lane);
    t.there[i] = there >> i & 1;
  }
}

// The wave's state for its 16 columns.
template <int NB>
struct Acc {
  f32x4 o[2 * NB];     // O^T tiles, scaled like P
  float ref, sum;      // M + e (far: M), and this lane's part of the sum of P 2^-e
  float limit;         // M + kRaise (far, or no key seen: M)
  float e, most;       // the column's e, and the largest V scale that it serves
  float check;         // lanes of V scales: the least `most` of all columns; else infinity
};

// Q^T as B operands, P parts per block.
template <int NB, int P>
struct Query {
  f16x8 q[NB][P];
  float fac;  // score from the product: scale * log2(e) / 2^k
};

// q of the lane's column as it lies in memory: the 8 elements of each block that
// slot group g multiplies.
template <int NB, typename T>
struct RawQuery {
  typedef T vec8 __attribute__((ext_vector_type(8)));
  vec8 x[NB];
  __device__ inline RawQuery(const T *q) {
#pragma unroll
    for (int b = 0; b < NB; ++b) x[b] = *reinterpret_cast<const vec8 __attribute__((aligned(16))) *>(q + 32 * b);
  }
};
// A scale as the scores' factor.  Never 0, so that it leaves the - infinity of a key not
// seen what it is, and never infinite, also times a K scale or 2^9, so that a sum of 0 stays
// 0: sums are multiples of 2^-57, so with 2^100 as with any larger factor the largest
// decides alone.
__device__ inline float factor(float scale) {
  return __builtin_fminf(__builtin_fmaxf(scale * 1.4426950408889634f, 1e-37f), 0x1p100f);
}
// As operands.  An f32 row is brought to [2^10, 2^11) by a power of two 2^k, so
// that its low parts lose nothing that counts.
template <int NB, int P, typename T>
__device__ inline void make_query(Query<NB, P> &Q, const RawQuery<NB, T> &raw, bool there, float scale) {
  int k = 0;
  if (P == 2) {
    float top = 0;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = __builtin_fmaxf(top, __builtin_fabsf((float)raw.x[b][e]));
    top = max_across(top);
    k = top > 0 && top < __builtin_inff() ? 11 - __builtin_amdgcn_frexp_expf(top) : 0;
  }
  Q.fac = factor(__builtin_ldexpf(__builtin_fabsf(scale), -k));
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if constexpr (P == 1) {
      Q.q[b][0] = there ? (scale < 0 ? -raw.x[b] : raw.x[b]) : (f16x8){0, 0, 0, 0, 0, 0, 0, 0};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = there ? __builtin_ldexpf(scale < 0 ? -raw.x[b][e] : raw.x[b][e], k) : 0.0f;
        Q.q[b][0][e] = (f16)x;
        Q.q[b][1][e] = (f16)(x - (float)Q.q[b][0][e]);
      }
    }
  }
}

// Nibbles 0 and 4 (HIGH: 1 and 5) of w as the codes' values in f16, exactly: the
// numbers 1024 + n (64 + n for the high ones, four bits further up), less
// 1024 (64) and the codes' 8.  The masks are in VGPRs: an instruction reads one
// SGPR or literal, and v_and_or_b32 wants two constants.
struct Masks {
  uint32_t lo, hi;
  float minus1;
};
__device__ inline Masks masks() {
  Masks m = {0x000f000fu, 0x00f000f0u, -1.0f};
  asm("" : "+v"(m.lo), "+v"(m.hi), "+v"(m.minus1));
  return m;
}
template <bool HIGH>
__device__ inline f16x2 codes(const Masks &m, uint32_t w) {
  const f16 off = HIGH ? (f16)-72.0f : (f16)-1032.0f;
  return as_f16x2(HIGH ? (w & m.hi) | 0x54005400u : (w & m.lo) | 0x64006400u) + (f16x2){off, off};
}
// The same times 2^-9 (kCodeUnit), in two thirds of the time: masked, a nibble is the f16
// subnormal n 2^-24 (n 2^-20), and one multiply-add makes it (n - 8) 2^-9.  (A
// v_and_b32 takes half as long as a v_and_or_b32 or a packed f16 instruction.)
constexpr float kCodeUnit = 0x1p-9f;
template <bool HIGH>
__device__ inline f16x2 small_codes(uint32_t w) {
  const f16 mul = HIGH ? (f16)0x1p11f : (f16)0x1p15f, add = (f16)(-8 * kCodeUnit);
  return __builtin_elementwise_fma(as_f16x2(w & (HIGH ? 0x00f000f0u : 0x000f000fu)), (f16x2){mul, mul},
                                   (f16x2){add, add});
}

// Lane LANE's word, or number, for each of its 16 (row_newbcast).
template <int LANE>
__device__ inline uint32_t word_from_lane(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x150 + LANE, 0xf, 0xf, true);
}
template <int LANE>
__device__ inline float from_lane(float v) {
  return __builtin_bit_cast(float, word_from_lane<LANE>(__builtin_bit_cast(uint32_t, v)));
}
template <int N, typename F>
__device__ inline void each(F f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(std::integral_constant<int, N - 1>());
  }
}

// Scores of a step, without the factor: x[4i + j] is key 16i + 4g + j.
template <int NB, int P>
__device__ inline void scores(float (&x)[8], const Query<NB, P> &Q, const Step<NB> &t) {
  each<NB>([&](auto B) {
    constexpr int b = B();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w = t.k[i][b], y = w >> 8;
      const f16x8 kk = as_f16x8(as_u32(small_codes<false>(w)), as_u32(small_codes<true>(w)),
                                as_u32(small_codes<false>(y)), as_u32(small_codes<true>(y)));
      f32x4 d = {0, 0, 0, 0};
#pragma unroll
      for (int p = 0; p < P; ++p) d = mfma(kk, Q.q[b][p], d);
      // (as f16 pairs: a multiply-add takes a half of a word, but no DPP operand)
      each<2>([&](auto J) {
        constexpr int j = J(), word = 2 * b + j;
        const f16x2 s = as_f16x2(word_from_lane<word % 16>(t.s[i][word / 16]));
        x[4 * i + 2 * j] = __builtin_fmaf((float)s.x, d[2 * j], b ? x[4 * i + 2 * j] : 0.0f);
        x[4 * i + 2 * j + 1] = __builtin_fmaf((float)s.y, d[2 * j + 1], b ? x[4 * i + 2 * j + 1] : 0.0f);
      });
    }
    if (b % 2) __builtin_amdgcn_sched_barrier(0);
  });
}

// A step that some column does not see all of.  First the scales of what lies
// past the end or stands in for a page that is not there become 0, and the others
// finite (the bits of a key that is not seen may be anything, and 0 times an infinity is
// not 0), then the scores of the keys that the lane's column does not see, [lo, hi)
// it does, - infinity.
template <int NB>
__device__ inline void cut_scales(Step<NB> &t, int32_t key, int32_t len, uint32_t r, uint32_t g) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // (lanes past the words hold the last one, of tokens 2 and 3)
    const int32_t k = key + 16 * i + 4 * (int32_t)g + (r >= 4 * NB ? 2 : 2 * (int32_t)(r & 1));
    uint32_t keep = t.there[i] && k < len ? 0xffffu : 0;
    if (t.there[i] && k + 1 < len) keep |= 0xffff0000u;
#pragma unroll
    for (int n = 0; n < Step<NB>::kScaleWords; ++n) t.s[i][n] = kv4_finite(t.s[i][n]) & keep;
  }
}
template <int NB>
__device__ inline void cut_scores(float (&x)[8], const Step<NB> &t, int32_t key, int32_t lo, int32_t hi, uint32_t g) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int32_t k = key + 16 * (i / 4) + 4 * (int32_t)g + i % 4;
    x[i] = k >= lo && k < hi && t.there[i / 4] ? x[i] : -__builtin_inff();
  }
}

// Two f32 as f16 pairs: their roundings and what those leave (exact), rounded.
// (minus1: -1 in a register, which keeps x - hi one instruction that takes hi as f16.)
__device__ inline void split_pair(float minus1, float x, float y, uint32_t &hi, uint32_t &lo) {
  const f16x2 h = __builtin_convertvector(((f32x2){x, y}), f16x2);
  const f32x2 r = {__builtin_fmaf((float)h.x, minus1, x), __builtin_fmaf((float)h.y, minus1, y)};
  hi = as_u32(h);
  lo = as_u32(__builtin_convertvector(r, f16x2));
}

// The words from 2 nb on are V's: only these are looked at here, as f32 numbers
// (times 2^-e once that is known).
template <int NB>
struct VScales {
  static constexpr int kFirst = 2 * NB / 16, kLane = 2 * NB % 16;
  float s[2][Step<NB>::kScaleWords][2];  // [tile][word][half]
  template <int I>
  __device__ float of(int tile) const {  // V scale I = 4 b + token
    constexpr int i = 4 * NB + I;
    return from_lane<i / 2 % 16>(s[tile][i / 32][i % 2]);
  }
};

template <int NB>
__device__ inline void rescale(Acc<NB> &A, float f) {
#pragma unroll
  for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) A.o[n][j] *= f;
}

// A larger score or V scale than M and e serve: new ones, per column.  `big` is
// the lane's largest V scale, of which in a step that all columns see whole
// each is any column's; else a column takes those of the keys it sees (a key that
// a row does not see, an infinity's maybe, costs its P no bits).
template <int NB>
__device__ inline void raise(Acc<NB> &A, const VScales<NB> &c, const float (&x)[8], float top, float big, bool whole) {
  const bool mine = (threadIdx.x & 15) >= VScales<NB>::kLane;
  if (whole) {
    big = wave_max(mine ? big : 0.0f);
  } else {
    big = 0;
    each<2>([&](auto I) {
      each<4 * NB>([&](auto N) {
        constexpr int i = I(), n = N();
        const float s = c.template of<n>(i);
        big = __builtin_fmaxf(big, x[4 * i + n % 4] > -__builtin_inff() ? s : 0.0f);
      });
    });
    big = max_across(big);
  }
  top = max_across(top);
  // (a column whose M + kRaise would be far, M not: M = top - kRaise)
  if (top > A.limit) A.limit = is_far(top - kLift + kRaise) ? top : top - kLift + kRaise;
  if (big > A.most) {
    const int e = __builtin_amdgcn_frexp_expf(big);
    A.e = (float)e;
    A.most = __builtin_ldexpf(2.0f, e);
  }
  // (that of a column that has seen no key stays kNever)
  const float ref = is_far(A.limit) ? A.limit : A.limit - kRaise + A.e, f = __builtin_amdgcn_exp2f(A.ref - ref);
  A.ref = ref;
  A.sum *= f;
  rescale(A, f);
  const float least = -wave_max(-A.most);  // (with all lanes active: not inside the ?:)
  A.check = mine ? least : __builtin_inff();
}

// Softmax weights of a step and their product with V.
template <int NB, int P>
__device__ inline void add_values(Acc<NB> &A, float (&x)[8], float fac, const Step<NB> &t, const Masks &m, bool whole) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= fac;
  float top = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(x[0], x[1]), __builtin_fmaxf(x[2], x[3])),
                              __builtin_fmaxf(__builtin_fmaxf(x[4], x[5]), __builtin_fmaxf(x[6], x[7])));
  VScales<NB> c;
  float big = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = VScales<NB>::kFirst; n < Step<NB>::kScaleWords; ++n) {
      const f16x2 w = as_f16x2(t.s[i][n]);
      c.s[i][n][0] = (float)w.x;
      c.s[i][n][1] = (float)w.y;
      big = __builtin_fmaxf(big, __builtin_fmaxf(c.s[i][n][0], c.s[i][n][1]));
    }
  if (__any(top > A.limit || big > A.check)) raise<NB>(A, c, x, top, big, whole);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = __builtin_amdgcn_exp2f(x[i] - A.ref);
    A.sum += x[i];
  }
  each<NB>([&](auto B) {
    constexpr int b = B();
    uint32_t ph[4], pl[4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      each<2>([&](auto J) {
        constexpr int j = J(), first = 4 * b + 2 * j;
        const float p0 = c.template of<first>(i) * x[4 * i + 2 * j];
        const float p1 = c.template of<first + 1>(i) * x[4 * i + 2 * j + 1];
        if (P == 2) split_pair(m.minus1, p0, p1, ph[2 * i + j], pl[2 * i + j]);
        else ph[2 * i + j] = as_u32(__builtin_convertvector(((f32x2){p0, p1}), f16x2));
      });
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      // words hold tokens 0 2 1 3: (tok0, tok1) then (tok2, tok3)
      uint32_t v[4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t w = t.v[i][b] >> (8 * j);
          v[2 * i + j] = as_u32(half ? small_codes<true>(w) : small_codes<false>(w));
        }
      const f16x8 v8 = as_f16x8(v[0], v[1], v[2], v[3]);
      f32x4 d = A.o[2 * b + half];
      if (P == 2) d = mfma(v8, as_f16x8(pl[0], pl[1], pl[2], pl[3]), d);
      A.o[2 * b + half] = mfma(v8, as_f16x8(ph[0], ph[1], ph[2], ph[3]), d);
    }
    __builtin_amdgcn_sched_barrier(0);
  });
}

// A tile of 16 columns of a sequence, and the 32-key steps [first, first + steps)
// that some column of it sees.
struct Item {
  Kv4Seq s;
  uint32_t seq, cols, col0;  // the sequence's columns, the tile's first
  int32_t first, steps;
  bool none;                 // past the sequence's columns
};
template <uint32_t COLS = kCols>
__device__ inline Item item_of(const AttnArgs &a, uint32_t item) {
  Item t;
  t.seq = a.tiles == 1 ? item : item / a.tiles;
  t.col0 = (item - t.seq * a.tiles) * COLS;
  t.s = kv4_seq(a.kv, t.seq);
  t.cols = t.s.nrows * a.group;
  t.none = t.col0 >= t.cols;
  int32_t lo = 0, hi = t.s.len;
  if (a.causal) {
    const uint32_t last = (t.col0 + COLS < t.cols ? t.col0 + COLS : t.cols) - 1;
    const int32_t p0 = t.s.pos0 + (int32_t)(t.col0 / a.group), p1 = t.s.pos0 + (int32_t)(last / a.group);
    hi = p1 + 1 < hi ? p1 + 1 : hi;
    if (a.window && p0 >= (int32_t)a.window) lo = p0 - (int32_t)a.window + 1;
  }
  hi = hi > 0 && !t.none ? hi : 0;
  t.first = lo / kKeys;
  t.steps = (hi + kKeys - 1) / kKeys - t.first;
  t.steps = t.steps > 0 ? t.steps : 0;
  return t;
}
// Length of an item (all its heads) in the row of all items: a head's steps come
// after kOverhead places of none.
__device__ inline uint32_t item_length(const AttnArgs &a, const Item &t) {
  return t.none ? 0 : ((uint32_t)t.steps + kOverhead) * a.kv.nkv;
}

template <typename T>
__device__ inline void put(T *out, float v);
template <>
__device__ inline void put<float>(float *out, float v) { *out = v; }
template <>
__device__ inline void put<f16>(f16 *out, float v) { *out = (f16)v; }

// Sum over the wave's lanes up to and with the caller's.
template <int CTRL, int ROWS = 0xf>
__device__ inline uint32_t shifted(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ inline uint32_t wave_scan(uint32_t v) {
  v += shifted<0x111>(v);  // row_shr 1, 2, 4, 8
  v += shifted<0x112>(v);
  v += shifted<0x114>(v);
  v += shifted<0x118>(v);
  v += shifted<0x142, 0xa>(v);  // row_bcast 15: rows 0 and 2 into 1 and 3
  v += shifted<0x143, 0xc>(v);  // row_bcast 31: the lower half into the upper
  return v;
}

// W waves on the same 16 columns, wave w taking steps w, w + W, .. of the
// workgroup's segments.
//
// SHARED: the steps of all items and heads in a row (item by item, head by
// head, each after kOverhead empty places) are dealt out to the workgroups in
// equal shares, however long the sequences are; a share may hold several
// segments, and a segment that is not a whole item and head goes into the workspace
// for kv4_attn_join_kernel.  A workgroup has two places there: 0 for
// a segment that others began, 1 for one that it begins and does not end.
// Else: a workgroup per item and head.
//
// Dealt out because lengths differ and heads are few: 48 sequences of 1 to 8000
// tokens take 23.6 us with the join, 45.9 with a workgroup per item and head,
// one of 131072 40.6 and 665; 128 equal ones of 8192, 1024 items and heads, 229 and 228.
// With a workgroup alone there is no second launch (a join is 4.5 to 6 us).
template <int NB, int W, bool SHARED, typename T>
__global__ __launch_bounds__(64 * W, resident(NB * 32, sizeof(T) == 4)) void kv4_attn_kernel(KV4_PARAMS, AttnArgs a) {
  a.kv = KV4_GATHER;
  constexpr int P = sizeof(T) == 4 ? 2 : 1;
  constexpr int D = NB * 32;
  // as deep as LDS lets the resident waves be; a workgroup alone has few steps per wave
  constexpr int R = NB == 2 && SHARED ? 4 : 2;
  struct Results {
    float ref[kCols][W], sum[kCols][W], o[W][kCols][D + 4];
  };
  constexpr size_t kLds = sizeof(Results) > (size_t)W * R * Ring<NB>::kBytes ? sizeof(Results)
                                                                             : (size_t)W * R * Ring<NB>::kBytes;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kLds];
  Results &res = *reinterpret_cast<Results *>(lds);

  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t r = lane & 15, g = lane >> 4;
  const uint8_t *ring = lds + wave * (R * Ring<NB>::kBytes);
  const uint32_t ring_at = lds_addr(ring);
  const Masks m = masks();

  // The workgroup's part [at, end) of the row, from place `in` of item `item`
  uint32_t item, in, left;
  if (SHARED) {
    // The length of all items, then the one that holds place `from`; every wave
    // by itself, 64 items at a time (up to 64, both from one scan).
    uint32_t total = 0, upto = 0, len = 0;
    for (uint32_t i = 0; i < a.items; i += 64) {
      len = i + lane < a.items ? item_length(a, item_of(a, i + lane)) : 0;
      upto = wave_scan(len);
      total += __builtin_amdgcn_readlane(upto, 63);
    }
    uint32_t share = (total + gridDim.x - 1) / gridDim.x;
    share = share > kOverhead + W ? share : kOverhead + W;
    const uint32_t from = blockIdx.x * share;  // below total + share
    item = a.items;
    in = 0;
    for (uint32_t i = 0, base = 0; i < a.items; i += 64) {
      if (a.items > 64) {
        len = i + lane < a.items ? item_length(a, item_of(a, i + lane)) : 0;
        upto = wave_scan(len);
      }
      const uint32_t start = base + upto - len;
      const uint64_t here = __ballot(from >= start && from - start < len);
      if (here) {
        const int n = __builtin_ctzll(here);
        item = i + n;
        in = from - __builtin_amdgcn_readlane(start, n);
      }
      if (blockIdx.x == 0 && wave == 0 && i + lane < a.items) a.starts[1 + i + lane] = start;
      base += __builtin_amdgcn_readlane(upto, 63);
      if (here && blockIdx.x != 0) break;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.starts[0] = share;
    item = __builtin_amdgcn_readfirstlane(item);
    in = __builtin_amdgcn_readfirstlane(in);
    left = share;
  } else {
    item = blockIdx.x / a.kv.nkv;
    in = blockIdx.x % a.kv.nkv;  // of heads
    left = 1;
  }
  // (without a window the steps begin at 0: the pages are asked for beside the
  // length, not after it)
  uint32_t listed = 0;
  if (!SHARED && !a.window) listed = list_pages(a.kv, a.tiles == 1 ? item : item / a.tiles, wave, W, lane);

  for (; item < a.items && left; ++item, in = 0) {
    const Item t = item_of(a, item);
    const Kv4Seq &s = t.s;
    if (t.none) {
      if (SHARED) continue;
      return;
    }
    // keys every column of the tile sees
    int32_t all_lo = 0, all_hi = s.len;
    if (a.causal) {
      const uint32_t last = (t.col0 + kCols < t.cols ? t.col0 + kCols : t.cols) - 1;
      const int32_t p0 = s.pos0 + (int32_t)(t.col0 / a.group), p1 = s.pos0 + (int32_t)(last / a.group);
      all_hi = p0 + 1 < all_hi ? p0 + 1 : all_hi;
      if (a.window && p1 >= (int32_t)a.window) all_lo = p1 - (int32_t)a.window + 1;
    }
    // the lane's column: its row, head and keys [lo, hi)
    const uint32_t col = t.col0 + r;
    const bool mine = col < t.cols;
    const uint32_t row = mine ? col / a.group : 0, sub = mine ? col % a.group : 0;
    int32_t lo = 0, hi = s.len;
    if (a.causal) {
      const int32_t p = s.pos0 + (int32_t)row;
      hi = p + 1 < hi ? p + 1 : hi;
      if (a.window && p >= (int32_t)a.window) lo = p - (int32_t)a.window + 1;
    }
    if (!mine) hi = 0;

    const uint32_t length = (uint32_t)t.steps + kOverhead;
    uint32_t head = SHARED ? in / length : in, place = SHARED ? in - head * length : 0;
    for (; head < a.kv.nkv && left; ++head, place = 0) {
      // the segment: steps [begin, end) of the head's t.steps
      int32_t begin = 0, end = t.steps;
      bool last = true;  // of the head
      if (SHARED) {
        const uint32_t n = length - place < left ? length - place : left;
        last = place + n == length;
        begin = place > kOverhead ? (int32_t)(place - kOverhead) : 0;
        end = place + n > kOverhead ? (int32_t)(place + n - kOverhead) : 0;
        left -= n;
        if (begin >= end && !(last && t.steps == 0)) continue;
      } else {
        left = 0;
      }
      const bool whole_head = begin == 0 && end == t.steps;

      int32_t at = begin + (int32_t)wave, issued = at;
      uint32_t slot_in = 0, there_in = 0;  // next slot to load; which tiles of the ring's slots have pages
      int32_t next = 0;  // in the list of pages
      if (SHARED || a.window) listed = list_pages(a.kv, t.seq, (uint32_t)(t.first + at), W, lane);
      auto issue = [&]() {
        if (issued < end) {
          if (next == kListed) {
            listed = list_pages(a.kv, t.seq, (uint32_t)(t.first + issued), W, lane);
            asm volatile("" : "+v"(listed));  // (waited for here, not, with all loads of the ring, at each step)
            next = 0;
          }
          const uint32_t pages[2] = {(uint32_t)__builtin_amdgcn_readlane(listed, 2 * next),
                                     (uint32_t)__builtin_amdgcn_readlane(listed, 2 * next + 1)};
          ++next;
          const uint32_t ok = fetch<NB>(a.kv, pages, head, (t.first + issued) * kKeys, s.len, lane,
                                        ring_at + slot_in * Ring<NB>::kBytes);
          there_in = (there_in & ~(3u << (2 * slot_in))) | ok << (2 * slot_in);
          slot_in = slot_in + 1 == R ? 0 : slot_in + 1;
          issued += W;
        }
      };
      // (the queries are asked for first: theirs is the shorter way)
      const RawQuery<NB, T> raw(static_cast<const T *>(a.q) + (size_t)(s.row0 + row) * a.ldq +
                                (size_t)(head * a.group + sub) * D + 8 * g);
      asm volatile("" : "+v"(listed));
#pragma unroll 1
      for (int n = 0; n < R - 1; ++n) issue();

      Query<NB, P> Q;
      make_query<NB, P, T>(Q, raw, mine, a.scale);
      Q.fac /= kCodeUnit;
      Acc<NB> A;
      A.ref = kNever;
      A.sum = 0;
      A.limit = kNever;
      A.e = A.most = 0;
      A.check = r >= VScales<NB>::kLane ? 0.0f : __builtin_inff();
#pragma unroll
      for (int n = 0; n < 2 * NB; ++n) A.o[n] = (f32x4){0, 0, 0, 0};

      uint32_t slot = 0;
      while (at < end) {
        issue();
        // this step's loads are done when only those of the later ones are not
        const int32_t later = (issued - at) / W - 1;
        if (R > 3 && later == 3) wait_loads<3 * Ring<NB>::kLoads>();
        else if (R > 2 && later == 2) wait_loads<2 * Ring<NB>::kLoads>();
        else if (later == 1) wait_loads<Ring<NB>::kLoads>();
        else wait_loads<0>();
        Step<NB> st;
        read_step<NB>(st, ring + slot * Ring<NB>::kBytes, there_in >> (2 * slot), lane);
        slot = slot + 1 == R ? 0 : slot + 1;
        const int32_t key = (t.first + at) * kKeys;
        const bool whole = key >= all_lo && key + kKeys <= all_hi && st.there[0] && st.there[1];
        if (!whole) cut_scales<NB>(st, key, s.len, r, g);
        float x[8];
        scores<NB, P>(x, Q, st);
        if (!whole) cut_scores<NB>(x, st, key, lo, hi, g);
        add_values<NB, P>(A, x, Q.fac, st, m, whole);
        at += W;
      }
      A.sum = sum_across(A.sum);
      // the waves' results: brought to a common reference, then added up
      __syncthreads();
      if (g == 0) res.ref[r][wave] = A.ref;
      __syncthreads();
      float ref = kNever;
#pragma unroll
      for (int w = 0; w < W; ++w) ref = __builtin_fmaxf(ref, res.ref[r][w]);
      const float f = __builtin_amdgcn_exp2f(A.ref - ref), fo = f / kCodeUnit;
      if (g == 0) res.sum[r][wave] = A.sum * f;
      if (mine)
#pragma unroll
        for (int n = 0; n < 2 * NB; ++n) *reinterpret_cast<f32x4 *>(&res.o[wave][r][16 * n + 4 * g]) = A.o[n] * fo;
      __syncthreads();
      const uint32_t ncols = t.cols - t.col0 < kCols ? t.cols - t.col0 : kCols;
      float *part = a.work + (2 * (size_t)blockIdx.x + (begin == 0)) * kShare<D>;
      for (uint32_t i = threadIdx.x; i < ncols * D; i += 64 * W) {
        const uint32_t c = i / D, d = i % D;
        float o = 0, sum = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          sum += res.sum[c][w];
          o += res.o[w][c][d];
        }
        if (whole_head) {
          const uint32_t orow = s.row0 + (t.col0 + c) / a.group, oh = head * a.group + (t.col0 + c) % a.group;
          put<T>(static_cast<T *>(a.out) + (size_t)orow * a.ldo + (size_t)oh * D + d, sum == 0 ? 0.0f : o / sum);
        } else {
          part[i] = o;
          if (d == 0) {
            ref = kNever;
#pragma unroll
            for (int w = 0; w < W; ++w) ref = __builtin_fmaxf(ref, res.ref[c][w]);
            part[kCols * D + c] = ref;
            part[kCols * D + kCols + c] = sum;
          }
        }
      }
      __syncthreads();
    }
  }
}

// The segments of one column of an item and head, joined, where there are more
// than one: a workgroup per item and column, and head.  The segments' weights
// first, then D threads add up their O, TH / D groups of them every so many segments.
// Bound by two dependent memory latencies and the launch: 5.4 us for 128
// segments of 32 columns, 5.9 for two or three of 4096.
template <int NB, int TH, typename T>
__global__ __launch_bounds__(TH) void kv4_attn_join_kernel(KV4_PARAMS, AttnArgs a, uint32_t tile_cols) {
  a.kv = KV4_GATHER;
  constexpr int D = NB * 32, G = TH / D;
  const uint32_t item = blockIdx.x / tile_cols, c = blockIdx.x % tile_cols, head = blockIdx.y;
  const Item t = item_of(a, item);
  if (t.col0 + c >= t.cols || t.steps == 0) return;
  const uint32_t share = kv4_const(a.starts);
  const uint32_t from = kv4_const(a.starts + 1 + item) + head * ((uint32_t)t.steps + kOverhead) + kOverhead;
  const uint32_t w0 = from / share, count = (from + (uint32_t)t.steps - 1) / share - w0 + 1;
  if (count == 1) return;
  __shared__ float weight[kMaxGroups], sums[G][D], red[32];
  // the workgroup that began the head has it in its place 1, the others in their place 0
  const float *w = a.work + 2 * (size_t)w0 * kShare<D>;
  const uint32_t th = threadIdx.x, grp = th / D, d = th % D;
  auto part = [&](uint32_t n) { return w + (2 * (size_t)n + (n == 0)) * kShare<D>; };
  // the first O on their way before the weights are known
  constexpr int kAhead = 8;
  float ahead[kAhead];
#pragma unroll
  for (uint32_t i = 0; i < kAhead; ++i)
    ahead[i] = grp < G && grp + i * G < count ? part(grp + i * G)[c * D + d] : 0.0f;
  float top = kNever, sum = 0;
  for (uint32_t n = th; n < count; n += TH) top = __builtin_fmaxf(top, weight[n] = part(n)[kCols * D + c]);
  top = wave_max(top);
  if (th % 64 == 0) red[th / 64] = top;
  __syncthreads();
#pragma unroll
  for (int n = 0; n < TH / 64; ++n) top = __builtin_fmaxf(top, red[n]);
  for (uint32_t n = th; n < count; n += TH) {
    const float f = __builtin_amdgcn_exp2f(weight[n] - top);
    sum = __builtin_fmaf(part(n)[kCols * D + kCols + c], f, sum);
    weight[n] = f;
  }
  sum = wave_sum(sum);
  if (th % 64 == 0) red[16 + th / 64] = sum;
  __syncthreads();
  if (grp < G) {
    float o = 0;
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
      if (grp + i * G < count) o = __builtin_fmaf(ahead[i], weight[grp + i * G], o);
#pragma unroll 4
    for (uint32_t n = grp + kAhead * G; n < count; n += G) o = __builtin_fmaf(part(n)[c * D + d], weight[n], o);
    sums[grp][d] = o;
  }
  __syncthreads();
  if (th < D) {
    float o = 0, l = 0;
#pragma unroll
    for (int n = 0; n < G; ++n) o += sums[n][th];
#pragma unroll
    for (int n = 0; n < TH / 64; ++n) l += red[16 + n];
    const uint32_t orow = t.s.row0 + (t.col0 + c) / a.group, oh = head * a.group + (t.col0 + c) % a.group;
    put<T>(static_cast<T *>(a.out) + (size_t)orow * a.ldo + (size_t)oh * D + th, l == 0 ? 0.0f : o / l);
  }
}

// ---------------------------------------------------------------- prompts
// Many columns: NW waves with two tiles of 16 columns each walk the same keys,
// KC at a time, and share what turning the words into f16 operands costs: the
// next KC keys' operands go to LDS while these are multiplied (two buffers, one
// barrier per KC keys), the words of the ones after that are on their way in
// registers.  The operands lie in LDS as the MFMAs read them, 16 bytes per lane.
//   K as its codes (the block sums get their scales, f32 in LDS, afterwards);
//   V as (n - 8) s in two f16, which hold all of its 15 bits: rounded to one
//     it would add an error like P's own rounding, and so would K.  (V below 2^-14 is
//     f16 subnormals, whose products the matrix core sums to 2^-18 only: f32 rows over V of
//     3e-6 come out to 8e-7 where others do to 2.7e-7.  A common power of two as in
//     the other kernel would have to be agreed on by the waves before they write V.)
// For 64 keys and 16 columns at d 128 that is 48 MFMAs (768 cycles) and about 200
// vector instructions (800 cycles), which do not run beside each other in one
// wave, and the two waves of a SIMD meet at a barrier each 64 keys.  2048 rows
// over 16384 keys (causal, 32 heads of 128 over 8): 730 to 748 us, 689 to 706 TFLOP/s of the
// product's 2 x 2 operations, the high and low V's third MFMA not counted (a
// library f16 product of 8192^3 with a transposed operand sustains 1520).  Two groups of waves, one multiplying while the
// other does its softmax, took 860.
template <int NB, int KC>
struct Buffer {
  static constexpr int kTiles = KC / 16;
  u32x4 k[kTiles][NB][64];           // [lane]: key lane % 16, elements 8 (lane / 16) ..
  u32x4 v[2][KC / 32][2 * NB][64];   // [high, low][pair of tiles][16 elements][lane]
  float ks[kTiles][NB][16];          // [key], times the scores' factor
  uint32_t there[kTiles];
};

// A wave's share of the words of KC keys: of a tile of 16 keys, wave `part` of
// its kPer has blocks part, part + kPer, ..
template <int NB, int KC, int NW>
struct Words {
  static constexpr int kPer = NW / (KC / 16);
  static constexpr int kBlocks = (NB + kPer - 1) / kPer;
  uint32_t k[kBlocks], v[kBlocks], s[kBlocks][2], ks, there;
  static __device__ inline uint32_t block(int i, uint32_t part) {
    const uint32_t b = part + i * kPer;
    return NB % kPer == 0 || b < NB ? b : NB - 1;  // (the last one twice)
  }
  // [lo, hi): the keys that every column of the workgroup sees.
  __device__ inline void fetch(const Kv4Args &a, uint32_t page, uint32_t head, int32_t key, int32_t len, int32_t lo,
                               int32_t hi, uint32_t part, uint32_t lane) {
    constexpr uint32_t D = NB * 32;
    const uint32_t r = lane & 15, g = lane >> 4;
    there = key < len && page < a.n_pages;
    page = there ? page : 0;
    const uint32_t off = (uint32_t)key & ((1u << a.shift) - 1);
    const uint8_t *blk = kv4_block(a, page, head, D);
    const uint8_t *kp = blk + (size_t)off * (D / 2), *vp = kp + ((size_t)(D / 2) << a.shift);
    const uint8_t *sp = blk + ((size_t)D << a.shift) + (size_t)off * (D / 8) + g * (D / 2);
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const uint32_t b = block(i, part);
      k[i] = *reinterpret_cast<const uint32_t *>(kp + 4 * b + r * (D / 2) + g * (4 * NB));
      v[i] = *reinterpret_cast<const uint32_t *>(vp + 4 * b + g * (2 * D) + r * (4 * NB));
      const u32x2 w = *reinterpret_cast<const u32x2 *>(sp + 8 * NB + 8 * b);
      s[i][0] = w.x;
      s[i][1] = w.y;
    }
    ks = *reinterpret_cast<const uint32_t *>(sp + 4 * (r < 2 * NB ? r : 2 * NB - 1));
    // V past the end or of a page that is not there: scale 0; of a key that a column does
    // not see: a finite one (any bits may lie there)
    if (there && key >= lo && key + 16 <= hi) return;
    const int32_t at = key + 4 * (int32_t)g;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t keep = there && at + 2 * j < len ? (at + 2 * j + 1 < len ? 0xffffffffu : 0xffffu) : 0;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) s[i][j] = kv4_finite(s[i][j]) & keep;
    }
  }
  // Its i-th block as operands, for tile `tile` of a buffer.
  __device__ inline void put(int i, Buffer<NB, KC> &to, const Masks &m, float fac, uint32_t tile, uint32_t part,
                             uint32_t lane) const {
    const uint32_t r = lane & 15, g = lane >> 4, b = block(i, part), y = k[i] >> 8;
    to.k[tile][b][lane] = (u32x4){as_u32(codes<false>(m, k[i])), as_u32(codes<true>(m, k[i])),
                                  as_u32(codes<false>(m, y)), as_u32(codes<true>(m, y))};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      u32x2 hi, lo;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t w = v[i] >> (8 * j);
        const f16x2 n = half ? codes<true>(m, w) : codes<false>(m, w), sc = as_f16x2(s[i][j]), x = n * sc;
        hi[j] = as_u32(x);
        lo[j] = as_u32(__builtin_elementwise_fma(n, sc, -x));
      }
      reinterpret_cast<u32x2 *>(&to.v[0][tile / 2][2 * b + half][lane])[tile % 2] = hi;
      reinterpret_cast<u32x2 *>(&to.v[1][tile / 2][2 * b + half][lane])[tile % 2] = lo;
    }
    if (i) return;
    // (the same from each of the tile's waves, and from lanes past the words the last one)
    const f16x2 w = as_f16x2(ks);
    const uint32_t n = r < 2 * NB ? r : 2 * NB - 1;
    *reinterpret_cast<f32x2 *>(&to.ks[tile][n / 2][4 * g + 2 * (n & 1)]) = (f32x2){(float)w.x * fac, (float)w.y * fac};
    to.there[tile] = there;
  }
};

template <int NB, typename T>
__global__ __launch_bounds__(64 * kPromptWaves, 2) void kv4_prompt_kernel(KV4_PARAMS, AttnArgs a) {
#pragma clang fp contract(off)  // (a score is rounded before its reference is taken off, see kFar)
  a.kv = KV4_GATHER;
  constexpr int P = sizeof(T) == 4 ? 2 : 1, NW = kPromptWaves;
  constexpr int D = NB * 32, KC = prompt_keys(D), KT = KC / 16, CT = prompt_tiles(D, sizeof(T) == 4);
  constexpr uint32_t COLS = NW * CT * 16;
  typedef Words<NB, KC, NW> Wd;
  static_assert(NW % KT == 0, "whole waves per tile");
  __shared__ Buffer<NB, KC> buf[2];

  // the last rows of a sequence first: they see the most keys
  const uint32_t head = blockIdx.x % a.kv.nkv;
  const Item t = item_of<COLS>(a, a.items - 1 - blockIdx.x / a.kv.nkv);
  if (t.none) return;
  const Kv4Seq &s = t.s;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t r = lane & 15, g = lane >> 4;
  const uint32_t my_tile = wave / Wd::kPer, part = wave % Wd::kPer;
  const Masks m = masks();
  // (f32 rows: theirs comes with the row's power of two, of which K scales times one
  // for all rows would be too large or too small)
  const float fac = P == 2 ? 1.0f : factor(__builtin_fabsf(a.scale));

  const int32_t c_end = ((t.first + t.steps) * kKeys + KC - 1) / KC;
  int32_t c = t.first * kKeys / KC;
  Wd words;
  // (past the end the last keys again, into a buffer that nobody reads; the page
  // number is asked for one step before its words)
  auto key_of = [&](int32_t n) { return (n < c_end ? n : c_end - 1) * KC + 16 * (int32_t)my_tile; };
  auto page_of = [&](int32_t n) {
    const uint32_t i = (uint32_t)key_of(n) >> a.kv.shift;
    return kv4_const(a.kv.table + (size_t)t.seq * a.kv.max_pages + (i < a.kv.max_pages ? i : 0));
  };
  uint32_t page = page_of(c);
  // keys that every column of the workgroup sees
  int32_t every_lo = 0, every_hi = s.len;
  if (a.causal) {
    const uint32_t last = (t.col0 + COLS < t.cols ? t.col0 + COLS : t.cols) - 1;
    const int32_t p0 = s.pos0 + (int32_t)(t.col0 / a.group), p1 = s.pos0 + (int32_t)(last / a.group);
    every_hi = p0 + 1 < every_hi ? p0 + 1 : every_hi;
    if (a.window && p1 >= (int32_t)a.window) every_lo = p1 - (int32_t)a.window + 1;
  }
  auto fetch = [&](int32_t n) {
    words.fetch(a.kv, page, head, key_of(n), s.len, every_lo, every_hi, part, lane);
    page = page_of(n + 1);
  };
  auto put = [&](int i, int32_t n) { words.put(i, buf[n & 1], m, fac, my_tile, part, lane); };
  auto put_all = [&](int32_t n) {
#pragma unroll
    for (int i = 0; i < Wd::kBlocks; ++i) put(i, n);
  };
  fetch(c);

  // the wave's columns: what each sees, and what all of them see
  Query<NB, P> Q[CT];
  Acc<NB> A[CT];
  int32_t lo[CT], hi[CT], any_lo = s.len, any_hi = 0, all_lo = 0, all_hi = s.len;
  bool mine[CT];
  size_t at[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const uint32_t col = t.col0 + (wave * CT + ct) * 16 + r;
    mine[ct] = col < t.cols;
    const uint32_t row = mine[ct] ? col / a.group : 0, sub = mine[ct] ? col % a.group : 0;
    lo[ct] = 0;
    hi[ct] = s.len;
    if (a.causal) {
      const int32_t p = s.pos0 + (int32_t)row;
      hi[ct] = p + 1 < hi[ct] ? p + 1 : hi[ct];
      if (a.window && p >= (int32_t)a.window) lo[ct] = p - (int32_t)a.window + 1;
    }
    if (!mine[ct]) hi[ct] = 0;
    at[ct] = (size_t)(s.row0 + row) * a.ldo + (size_t)(head * a.group + sub) * D;
    const RawQuery<NB, T> raw(static_cast<const T *>(a.q) + (size_t)(s.row0 + row) * a.ldq +
                              (size_t)(head * a.group + sub) * D + 8 * g);
    make_query<NB, P, T>(Q[ct], raw, mine[ct], a.scale);
    A[ct].ref = kNever;
    A[ct].sum = 0;
#pragma unroll
    for (int n = 0; n < 2 * NB; ++n) A[ct].o[n] = (f32x4){0, 0, 0, 0};
  }
  {
    const uint32_t first = t.col0 + wave * CT * 16, past = first + CT * 16 < t.cols ? first + CT * 16 : t.cols;
    if (first < t.cols) {
      any_lo = 0;
      any_hi = s.len;
      if (a.causal) {
        const int32_t p0 = s.pos0 + (int32_t)(first / a.group), p1 = s.pos0 + (int32_t)((past - 1) / a.group);
        any_hi = p1 + 1 < any_hi ? p1 + 1 : any_hi;
        all_hi = p0 + 1 < all_hi ? p0 + 1 : all_hi;
        if (a.window && p0 >= (int32_t)a.window) any_lo = p0 - (int32_t)a.window + 1;
        if (a.window && p1 >= (int32_t)a.window) all_lo = p1 - (int32_t)a.window + 1;
      }
    }
  }

  put_all(c);
  fetch(c + 1);
  __syncthreads();
  for (; c < c_end; ++c) {
    const int32_t key = c * KC;
    const Buffer<NB, KC> &b_ = buf[c & 1];
    const bool seen = key < any_hi && key + KC > any_lo;
    uint32_t p[CT][P][2 * KT];
    if (seen) {
    // Scores in stages of up to two blocks of a tile of keys: a stage starts the LDS reads of
    // the second next one, multiplies, and scales the products of the one before.
    // (By itself the compiler waits for each read where it is used, and
    // puts the scales after the branch below, which the empty asm keeps them before.)
    constexpr int kHalf = (NB + 1) / 2, kStages = 2 * KT;
    float x[CT][4 * KT];
    f16x8 kk[3][kHalf];
    f32x4 sc[3][kHalf], d[2][kHalf][CT];
    auto read = [&](int st) {
#pragma unroll
      for (int h = 0; h < kHalf; ++h) {
        const int i = st / 2, b = st % 2 * kHalf + h;
        if (b >= NB) continue;
        kk[st % 3][h] = __builtin_bit_cast(f16x8, b_.k[i][b][lane]);
        sc[st % 3][h] = *reinterpret_cast<const f32x4 *>(&b_.ks[i][b][4 * g]);
      }
    };
    auto scaled = [&](int st) {
#pragma unroll
      for (int h = 0; h < kHalf; ++h) {
        const int i = st / 2, b = st % 2 * kHalf + h;
        if (b >= NB) continue;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float &y = x[ct][4 * i + j];
            y = b ? __builtin_fmaf(sc[st % 3][h][j], d[st % 2][h][ct][j], y) : sc[st % 3][h][j] * d[st % 2][h][ct][j];
          }
      }
    };
    read(0);
    read(1);
#pragma unroll
    for (int st = 0; st < kStages; ++st) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < kHalf; ++h) {
        const int b = st % 2 * kHalf + h;
        if (b >= NB) continue;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          f32x4 y = {0, 0, 0, 0};
#pragma unroll
          for (int p = 0; p < P; ++p) y = mfma(kk[st % 3][h], Q[ct].q[b][p], y);
          d[st % 2][h][ct] = y;
        }
      }
      if (st) scaled(st - 1);
      if (st + 2 < kStages) read(st + 2);
    }
    __builtin_amdgcn_sched_barrier(0);
    scaled(kStages - 1);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int n = 0; n < 4 * KT; ++n) asm volatile("" : "+v"(x[ct][n]));
    bool whole = key >= all_lo && key + KC <= all_hi;
#pragma unroll
    for (int i = 0; i < KT; ++i) whole = whole && __builtin_amdgcn_readfirstlane(b_.there[i]);
    if (!whole) {
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        const bool there = b_.there[i];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int32_t k = key + 16 * i + 4 * (int32_t)g + j;
            x[ct][4 * i + j] = k >= lo[ct] && k < hi[ct] && there ? x[ct][4 * i + j] : -__builtin_inff();
          }
      }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float top = -__builtin_inff();
#pragma unroll
      for (int n = 0; n < 4 * KT; ++n) {
        if (P == 2) x[ct][n] *= Q[ct].fac;
        top = __builtin_fmaxf(top, x[ct][n]);
      }
      // (their difference is exact where it decides; a sum of large numbers is not)
      if (__any(top - A[ct].ref > kRaise)) {
        top = max_across(top);
        const float ref = top - A[ct].ref > kRaise ? top - kLift : A[ct].ref;
        const float f = __builtin_amdgcn_exp2f(A[ct].ref - ref);
        A[ct].ref = ref;
        A[ct].sum *= f;
        rescale(A[ct], f);
      }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int n = 0; n < 2 * KT; ++n) {
        const float x0 = __builtin_amdgcn_exp2f(x[ct][2 * n] - A[ct].ref);
        const float x1 = __builtin_amdgcn_exp2f(x[ct][2 * n + 1] - A[ct].ref);
        if (P == 2) {
          A[ct].sum += x0;
          A[ct].sum += x1;
          split_pair(m.minus1, x0, x1, p[ct][0][n], p[ct][P - 1][n]);
        } else {
          // the sum of the weights as they are multiplied
          const f16x2 h = __builtin_convertvector(((f32x2){x0, x1}), f16x2);
          A[ct].sum = __builtin_amdgcn_fdot2(h, (f16x2){(f16)1.0f, (f16)1.0f}, A[ct].sum, false);
          p[ct][0][n] = as_u32(h);
        }
      }
    // Products in stages of two tiles of elements, two stages after their reads.
    constexpr int kV = KT / 2 * NB;  // stages: pairs of key tiles x pairs of element tiles
    f16x8 v8[3][2][2];
    auto read_v = [&](int st) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          v8[st % 3][h][e] = __builtin_bit_cast(f16x8, b_.v[h][st / NB][2 * (st % NB) + e][lane]);
    };
    read_v(0);
    read_v(1);
#pragma unroll
    for (int st = 0; st < kV; ++st) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 1; h >= 0; --h)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            const uint32_t *ph = p[ct][0] + 4 * (st / NB), *pl = p[ct][P - 1] + 4 * (st / NB);
            f32x4 &o = A[ct].o[2 * (st % NB) + e];
            o = mfma(v8[st % 3][h][e], as_f16x8(ph[0], ph[1], ph[2], ph[3]), o);
            if (P == 2 && h == 0) o = mfma(v8[st % 3][0][e], as_f16x8(pl[0], pl[1], pl[2], pl[3]), o);
          }
      if (st + 2 < kV) read_v(st + 2);
      if (st < Wd::kBlocks) put(st, c + 1);
      if (st == Wd::kBlocks) fetch(c + 2);
    }
    __builtin_amdgcn_sched_barrier(0);
    } else {
      put_all(c + 1);
      fetch(c + 2);
    }
    __syncthreads();
  }

#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const float sum = sum_across(A[ct].sum), inv = sum == 0 ? 0.0f : 1 / sum;
    if (!mine[ct]) continue;
    typedef T vec4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int e = 0; e < 2 * NB; ++e)
      *reinterpret_cast<vec4 *>(static_cast<T *>(a.out) + at[ct] + 16 * e + 4 * g) =
          __builtin_convertvector(A[ct].o[e] * inv, vec4);
  }
}

struct Plan {
  uint32_t tiles, groups;  // groups: workgroups that share the steps, 0: one per tile and head
  bool few;                // steps
  bool prompt;
  size_t part;             // bytes of a partial result
  size_t starts;           // bytes of the items' starts
  size_t bytes() const { return groups ? groups * 2 * part + starts : 0; }
};
// A cache of up to four steps per wave (2048 keys at d 64) stays with one workgroup
// per tile and head: eight sequences of 1500, 20 heads of 64, f32, take 13.1 us
// there and 16.7 dealt out and joined; from more steps per wave on the join is the
// smaller part.  Where that is eight waves, though (d 256, f32 rows of d 128), and half of the
// CUs have a workgroup each, they stay alone up to 64 steps: f32 rows, 8 heads of
// 128, 1500 keys, 16 sequences 16.0 us alone and 21.4 dealt out, 4 sequences 16.1 and 13.9; of
// 256 27.1 and 29.6, 26.7 and 19.2.  Longer ones are dealt out over as many workgroups as are
// resident at once.  most: without the prompts' kernel, whose place
// depends on the type and window.
Plan plan_of(const madi_kv4 *c, const madi_kv4_batch *b, uint32_t nh, int dtype, uint32_t window, uint32_t cus,
             bool most = false) {
  Plan p = {};
  const uint64_t reach = (uint64_t)b->max_pages * c->page;
  uint64_t len = b->len_max && b->len_max < reach ? b->len_max : reach;
  if (window && (uint64_t)window + b->rows + kKeys < len) len = (uint64_t)window + b->rows + kKeys;
  const uint64_t cols = (uint64_t)b->rows * (nh / c->nkv);
  // Prompts where their workgroups fill the device.  Times are counted in steps of a CU
  // with sixteen waves of the other kernel (four steps at once), tenths of them.
  const bool f32 = dtype == MADI_F32;
  const uint64_t pcols = (uint64_t)kPromptWaves * 16 * prompt_tiles(c->d, f32);
  const uint64_t ptiles = (cols + pcols - 1) / pcols, steps = (len + kKeys - 1) / kKeys;
  const uint64_t cost = (len + 63) / 64 * prompt_cost(c->d, f32);
  const uint64_t tiles16 = (cols + kCols - 1) / kCols * c->nkv * b->b;
  const uint64_t rounds = (ptiles * c->nkv * b->b + cus - 1) / cus;
  if (!most && has_prompt_kernel(c->d, f32) && rounds * cost < 10 * tiles16 * steps / (4 * cus)) {
    p.prompt = true;
    p.tiles = (uint32_t)ptiles;
    return p;
  }
  p.tiles = (uint32_t)((cols + kCols - 1) / kCols);
  p.part = (size_t)kCols * (c->d + 2) * 4;
  const uint64_t items = (uint64_t)p.tiles * b->b;
  p.starts = (size_t)(items + 1) * 4;
  p.few = steps <= kFew;
  if (steps <= 4 * waves_alone(c->d, dtype == MADI_F32)) return p;
  if (steps <= 64 && items * c->nkv >= cus / 2) return p;
  // (the row's places are counted in 32 bits)
  if (items * c->nkv * ((reach + kKeys - 1) / kKeys + kOverhead + 1) > 0x40000000u) return p;
  if (items > 0xfffffu) return p;  // (the join's threads, 4096 per item, likewise)
  p.groups = resident(c->d, dtype == MADI_F32) * cus;
  p.groups = p.groups < kMaxGroups ? p.groups : kMaxGroups;
  return p;
}

template <int NB, typename T>
void launch(const AttnArgs &a, const Plan &p, uint32_t cus) {
  if constexpr (has_prompt_kernel(NB * 32, sizeof(T) == 4)) {
    if (p.prompt) {
      kv4_prompt_kernel<NB, T><<<a.items * a.kv.nkv, 64 * kPromptWaves, 0, stream()>>>(KV4_ARGS(a.kv), a);
      return;
    }
  }
  if (!p.groups) {
    constexpr int W = waves_alone(NB * 32, sizeof(T) == 4);
    // few steps: four waves (20 heads over 213 keys 5.7 us, with eight 5.95, with
    // sixteen 6.7; prompts of 17 to 224 rows, four of them, 9.8, 11.0 and 19.2)
    if (p.few) kv4_attn_kernel<NB, 4, false, T><<<a.items * a.kv.nkv, 256, 0, stream()>>>(KV4_ARGS(a.kv), a);
    else kv4_attn_kernel<NB, W, false, T><<<a.items * a.kv.nkv, 64 * W, 0, stream()>>>(KV4_ARGS(a.kv), a);
    return;
  }
  kv4_attn_kernel<NB, 4, true, T><<<p.groups, 256, 0, stream()>>>(KV4_ARGS(a.kv), a);
  const uint64_t cols = (uint64_t)a.kv.rows * a.group;
  const uint32_t tile_cols = cols < kCols ? (uint32_t)cols : kCols;
  const dim3 grid(a.items * tile_cols, a.kv.nkv);
  // few columns are of long caches, many segments each: 131072 keys, 32 columns,
  // 40.6 us with 1024 threads, 43.7 with 256.  Of many most have one or two: 128
  // sequences of 8192 229 us with 256 threads, 240 with 1024; 48 ragged ones 23.6, 29.3.
  if ((uint64_t)grid.x * grid.y <= 2 * cus)
    kv4_attn_join_kernel<NB, 1024, T><<<grid, 1024, 0, stream()>>>(KV4_ARGS(a.kv), a, tile_cols);
  else
    kv4_attn_join_kernel<NB, 256, T><<<grid, 256, 0, stream()>>>(KV4_ARGS(a.kv), a, tile_cols);
}

}  // namespace

extern "C" size_t madi_kv4_attn_bytes(const madi_kv4 *cache, const madi_kv4_batch *batch, uint32_t nh) {
  Kv4Args a;
  if (kv4_args("madi_kv4_attn_bytes", cache, batch, &a) || nh == 0 || nh % cache->nkv) return 0;
  // the most that any type and window may take (f16 rows have more workgroups, f32 rows of
  // d 128 are split from shorter caches on)
  const uint32_t cus = initialized() ? (uint32_t)cu_count() : 256;
  const size_t h = plan_of(cache, batch, nh, MADI_F16, 0, cus, true).bytes();
  const size_t f = plan_of(cache, batch, nh, MADI_F32, 0, cus, true).bytes();
  return h > f ? h : f;
}

extern "C" int madi_kv4_attn(void *out, const void *q, const madi_kv4 *cache, const madi_kv4_batch *batch,
                             uint32_t nh, uint32_t ldo, uint32_t ldq, uint32_t window, int causal, int dtype,
                             float scale) {
  const char *what = "madi_kv4_attn";
  AttnArgs a;
  if (int rc = kv4_args(what, cache, batch, &a.kv)) return rc;
  if (nh == 0 || nh % cache->nkv)
    return fail(MADI_ERR_SHAPE, "%s: %u query heads over %u kv heads", what, nh, cache->nkv);
  const uint64_t width = (uint64_t)nh * cache->d;
  size_t qb, ob;
  if (int rc = kv4_rows(what, "q", q, batch->m, width, ldq, dtype, &qb)) return rc;
  if (int rc = kv4_rows(what, "out", out, batch->m, width, ldo, dtype, &ob)) return rc;
  if (causal != 0 && causal != 1) return fail(MADI_ERR_ARG, "%s: causal %d", what, causal);
  if (!causal && window) return fail(MADI_ERR_ARG, "%s: a window without causal", what);
  if (window > 0x7fffffffu) window = 0;  // wider than any cache
  if (!(__builtin_fabsf(scale) < __builtin_inff())) return fail(MADI_ERR_ARG, "%s: scale %g", what, scale);
  if (batch->work && !aligned(batch->work, 16)) return fail(MADI_ERR_ALIGN, "%s: work must be 16-byte aligned", what);
  const size_t cb = kv4_cache_bytes(cache), wb = batch->work ? batch->work_bytes : 0;
  if (kv4_overlap(out, ob, cache->data, cb) || (kv4_overlap(out, ob, q, qb) && !(out == q && ldo == ldq)) ||
      kv4_overlap(out, ob, batch->work, wb) || kv4_overlap(q, qb, batch->work, wb) ||
      kv4_overlap(cache->data, cb, batch->work, wb))
    return fail(MADI_ERR_ARG, "%s: out or work overlaps another operand", what);
  if (kv4_on_batch(batch, out, ob) || kv4_on_batch(batch, batch->work, wb))
    return fail(MADI_ERR_ARG, "%s: out or work overlaps table, lens or row_off", what);
  if ((uint64_t)batch->rows * (nh / cache->nkv) > 0x7fffffffu)
    return fail(MADI_ERR_SHAPE, "%s: %u rows of a sequence in one call", what, batch->rows);
  if (!initialized()) return fail(MADI_ERR_NOT_INIT, "%s: madi_init has not succeeded", what);
  if (batch->m == 0 || batch->b == 0 || batch->rows == 0) return MADI_OK;
  Plan p = plan_of(cache, batch, nh, dtype, window, (uint32_t)cu_count());
  // as many workgroups as the workspace has places for
  if (p.bytes() > wb) p.groups = wb > p.starts ? (uint32_t)((wb - p.starts) / (2 * p.part)) : 0;
  if (p.groups < 2) p.groups = 0;
  const uint64_t items = (uint64_t)p.tiles * batch->b;
  if (items * cache->nkv > 0x3fffffu)  // workgroups of up to 1024 threads, below 2^32 in all
    return fail(MADI_ERR_SHAPE, "%s: %u rows of %u sequences in one call", what, batch->rows, batch->b);
  if (int rc = deferred_before_read(q, qb)) return rc;
  if (int rc = deferred_before_read(cache->data, cb)) return rc;
  if (int rc = kv4_before_write(out, ob)) return rc;
  if (p.groups)
    if (int rc = deferred_before_write(batch->work, wb)) return rc;
  a.q = q;
  a.out = out;
  a.work = static_cast<float *>(batch->work);
  a.ldq = ldq;
  a.ldo = ldo;
  a.group = nh / cache->nkv;
  a.window = window;
  a.causal = (uint32_t)causal;
  a.tiles = p.tiles;
  a.items = (uint32_t)items;
  a.starts = reinterpret_cast<uint32_t *>(a.work + p.groups * 2 * (p.part / 4));
  a.scale = scale;
  const bool f = dtype == MADI_F32;
  const uint32_t cus = (uint32_t)cu_count();
  switch (cache->d) {
  case 64: f ? launch<2, float>(a, p, cus) : launch<2, f16>(a, p, cus); break;
  case 96: f ? launch<3, float>(a, p, cus) : launch<3, f16>(a, p, cus); break;
  case 128: f ? launch<4, float>(a, p, cus) : launch<4, f16>(a, p, cus); break;
  default: f ? launch<8, float>(a, p, cus) : launch<8, f16>(a, p, cus); break;
  }
  return check_launch(what);
}
