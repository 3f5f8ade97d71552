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
//   softmax over a running reference that is raised only when a score passes
//     it by 2^8, so most steps exchange nothing between lanes.
//   O^T += V^T P^T, 32 keys as K and 16 elements as rows: P^T comes straight
//     from the S^T registers (lane (g, c) holds keys 4g..4g+3 of both tiles),
//     V as its codes from the words that hold four tokens, and the V scale of a
//     key and block goes into P: one rounding, of P s, instead of P's and V's.
//     s comes times 2^-e, e the largest exponent among the wave's V scales so
//     far, so that P s stays within f16.
// A lane holds two of the 8 nb scales of its four keys and passes them to the
// other 15 through DPP broadcasts, which cost nothing in a multiplication.
// f32 rows: q and P s are each split in two f16 (22 bits).
#include <type_traits>

#include "kv4.h"

using namespace madi;

namespace {

constexpr int kCols = 16;  // columns of a wave (MFMA columns)
constexpr int kKeys = 32;  // keys of a step
constexpr float kNever = -1e30f;  // reference before any key was seen
// P is 2^(x - M) with M at first the largest x - 7, raised when an x passes M
// by 14: P at most 2^14, P s 2^-e at most 2^15 (f16 holds 2^16), and what
// rounds to nothing is 2^-32 of the largest P at the largest s.
constexpr float kLift = 7.0f, kRaise = 14.0f;

constexpr int kMaxSplits = 256;
// f32 numbers of a share: O [16][D], then the references and the sums.
template <int D>
constexpr size_t kShare = kCols * (D + 2);

struct AttnArgs {
  Kv4Args kv;
  const void *q;
  void *out;
  float *work;
  uint32_t ldq, ldo, group, window, causal, splits, min_steps;
  float scale;
};

typedef float f32x2 __attribute__((ext_vector_type(2)));

template <int N>
__device__ inline void load_words(const uint8_t *p, uint32_t (&w)[N]) {
  constexpr int A = N % 4 == 0 ? 16 : N % 2 == 0 ? 8 : 4;
  __builtin_memcpy(w, __builtin_assume_aligned(p, A), 4 * N);
}
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

// Pages of the tiles at key and key + 16 (none past the end).
__device__ inline void find_pages(uint32_t (&page)[2], const Kv4Args &a, uint32_t seq, int32_t key, int32_t len) {
#pragma unroll
  for (int i = 0; i < 2; ++i) page[i] = key + 16 * i < len ? kv4_page(a, seq, key + 16 * i) : 0xffffffffu;
}

template <int NB>
__device__ inline void fetch(Step<NB> &t, const Kv4Args &a, const uint32_t (&pages)[2], uint32_t head, int32_t key,
                             uint32_t lane) {
  constexpr uint32_t D = NB * 32;
  const uint32_t r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // a tile without a page: any valid one stands in
    t.there[i] = pages[i] < a.n_pages;
    const uint32_t page = t.there[i] ? pages[i] : 0;
    const uint32_t off = (uint32_t)(key + 16 * i) & ((1u << a.shift) - 1);
    const uint8_t *blk = kv4_block(a, page, head, D);
    const uint8_t *kp = blk + (size_t)off * (D / 2) + (r * (D / 2) + g * (4 * NB));
    const uint8_t *vp = blk + ((size_t)(D / 2) << a.shift) + (size_t)(off / 4) * (2 * D) + (g * (2 * D) + r * (4 * NB));
    const uint8_t *sp = blk + ((size_t)D << a.shift) + (size_t)(off / 4) * (D / 2) + g * (D / 2);
    constexpr uint32_t kWords = 4 * NB;  // of a group
    load_words<NB>(kp, t.k[i]);
    load_words<NB>(vp, t.v[i]);
#pragma unroll
    for (uint32_t n = 0; n < Step<NB>::kScaleWords; ++n) {
      const uint32_t w = 16 * n + r;  // (nb < 4: lanes past the words hold the last one)
      load_words<1>(sp + 4 * (w < kWords ? w : kWords - 1), *reinterpret_cast<uint32_t(*)[1]>(&t.s[i][n]));
    }
  }
}

// The wave's state for its 16 columns.
template <int NB>
struct Acc {
  f32x4 o[2 * NB];  // O^T tiles, scaled like P
  float ref, sum;   // M, and this lane's part of sum P
  float down, most; // 2^-e, and the largest V scale that it serves
};

// Q^T as B operands, P parts per block.
template <int NB, int P>
struct Query {
  f16x8 q[NB][P];
  float fac;  // score from the product: scale * log2(e) / 2^k
};

template <typename T>
__device__ inline void load8f(const T *p, float (&x)[8]);
template <>
__device__ inline void load8f<float>(const float *p, float (&x)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
}
template <>
__device__ inline void load8f<f16>(const f16 *p, float (&x)[8]) {
  const f16x8 a = *reinterpret_cast<const f16x8 *>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
}

// q of the lane's column (the 8 elements of each block that slot group g
// multiplies).  An f32 row is brought to [2^10, 2^11) by a power of two 2^k, so
// that its low parts lose nothing that counts.
template <int NB, int P, typename T>
__device__ inline void load_query(Query<NB, P> &Q, const T *q, bool there, uint32_t g, float scale) {
  float x[NB][8], top = 0;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if (there) {
      load8f<T>(q + 32 * b + 8 * g, x[b]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[b][e] = 0;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) top = __builtin_fmaxf(top, __builtin_fabsf(x[b][e]));
  }
  int k = 0;
  if (P == 2) {
    top = max_across(top);
    k = top > 0 && top < __builtin_inff() ? 11 - __builtin_amdgcn_frexp_expf(top) : 0;
    k = k < -100 ? -100 : k > 100 ? 100 : k;
  }
  // (never 0, so that it leaves the - infinity of a key not seen what it is)
  Q.fac = __builtin_fmaxf(__builtin_ldexpf(__builtin_fabsf(scale) * 1.4426950408889634f, -k), 1e-37f);
  const float sign = scale < 0 ? -1.0f : 1.0f;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int p = 0; p < P; ++p) {
      f16x8 h;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (p == 0) x[b][e] = __builtin_ldexpf(x[b][e], k) * sign;
        h[e] = (f16)x[b][e];
        x[b][e] -= (float)h[e];
      }
      Q.q[b][p] = h;
    }
}

// Nibbles 0 and 4 (HIGH: 1 and 5) of w as the codes' values: the f16 numbers
// 1024 + n (64 + n for the high ones, four bits further up), less 1024 (64) and
// the codes' 8.  Exact.  The masks are in VGPRs: an instruction reads one SGPR or
// literal, and v_and_or_b32 wants two constants.
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
__device__ inline void scores(float (&x)[8], const Query<NB, P> &Q, const Step<NB> &t, const Masks &m) {
  each<NB>([&](auto B) {
    constexpr int b = B();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w = t.k[i][b], y = w >> 8;
      const f16x8 kk = as_f16x8(as_u32(codes<false>(m, w)), as_u32(codes<true>(m, w)), as_u32(codes<false>(m, y)),
                                as_u32(codes<true>(m, y)));
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
// past the end or stands in for a page that is not there become 0 (those bits may be
// anything, and 0 times an infinity is not 0), then the scores of the keys that
// the lane's column does not see, [lo, hi) it does, - infinity.
template <int NB>
__device__ inline void cut_scales(Step<NB> &t, int32_t key, int32_t len, uint32_t r, uint32_t g) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int32_t k = key + 16 * i + 4 * (int32_t)g + 2 * (int32_t)(r & 1);
    uint32_t keep = t.there[i] && k < len ? 0xffffu : 0;
    if (t.there[i] && k + 1 < len) keep |= 0xffff0000u;
#pragma unroll
    for (int n = 0; n < Step<NB>::kScaleWords; ++n) t.s[i][n] &= keep;
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

// Softmax weights of a step and their product with V.
template <int NB, int P>
__device__ inline void add_values(Acc<NB> &A, float (&x)[8], float fac, const Step<NB> &t, const Masks &m) {
  float top = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(x[0], x[1]), __builtin_fmaxf(x[2], x[3])),
                              __builtin_fmaxf(__builtin_fmaxf(x[4], x[5]), __builtin_fmaxf(x[6], x[7])));
  top *= fac;
  if (__any(top > A.ref + kRaise)) {
    top = max_across(top);
    // the reference of a column that has seen no key stays
    const float ref = top > A.ref + kRaise ? top - kLift : A.ref;
    const float f = __builtin_amdgcn_exp2f(A.ref - ref);
    A.ref = ref;
    A.sum *= f;
    rescale(A, f);
  }
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
  if (__any(big > A.most)) {  // (a lane of K scales has an infinite `most`)
    const bool mine = (threadIdx.x & 15) >= VScales<NB>::kLane;
    big = wave_max(mine ? big : 0.0f);
    const float down = __builtin_ldexpf(1.0f, -__builtin_amdgcn_frexp_expf(big));
    rescale(A, down / A.down);
    A.down = down;
    A.most = mine ? 2 / down : __builtin_inff();
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], fac, -A.ref));
    A.sum += x[i];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = VScales<NB>::kFirst; n < Step<NB>::kScaleWords; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) c.s[i][n][h] *= A.down;
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
          v[2 * i + j] = as_u32(half ? codes<true>(m, w) : codes<false>(m, w));
        }
      const f16x8 v8 = as_f16x8(v[0], v[1], v[2], v[3]);
      f32x4 d = A.o[2 * b + half];
      if (P == 2) d = mfma(v8, as_f16x8(pl[0], pl[1], pl[2], pl[3]), d);
      A.o[2 * b + half] = mfma(v8, as_f16x8(ph[0], ph[1], ph[2], ph[3]), d);
    }
    __builtin_amdgcn_sched_barrier(0);
  });
}

// The 32-key steps [first, first + steps) that some column of the tile sees,
// and the split of them over workgroups: `per` steps each, `active` shares.
struct Range {
  int32_t first, steps, per, active;
};
__device__ inline Range key_range(const AttnArgs &a, const Kv4Seq &s, uint32_t col0, uint32_t cols) {
  Range r;
  int32_t lo = 0, hi = s.len;
  if (a.causal) {
    const uint32_t last = (col0 + kCols < cols ? col0 + kCols : cols) - 1;
    const int32_t p0 = s.pos0 + (int32_t)(col0 / a.group), p1 = s.pos0 + (int32_t)(last / a.group);
    hi = p1 + 1 < hi ? p1 + 1 : hi;
    if (a.window && p0 >= (int32_t)a.window) lo = p0 - (int32_t)a.window + 1;
  }
  hi = hi > 0 ? hi : 0;
  r.first = lo / kKeys;
  r.steps = (hi + kKeys - 1) / kKeys - r.first;
  r.steps = r.steps > 0 ? r.steps : 0;
  const int32_t even = (r.steps + (int32_t)a.splits - 1) / (int32_t)a.splits;
  r.per = even > (int32_t)a.min_steps ? even : (int32_t)a.min_steps;
  r.active = r.steps ? (r.steps + r.per - 1) / r.per : 1;
  return r;
}

template <typename T>
__device__ inline void put(T *out, float v);
template <>
__device__ inline void put<float>(float *out, float v) { *out = v; }
template <>
__device__ inline void put<f16>(f16 *out, float v) { *out = (f16)v; }

// Workgroup: W waves on the same 16 columns, wave w taking steps w, w + W, ..
// of the workgroup's share; their results meet in LDS.  Grid: tiles of columns x
// splits, kv heads, sequences.
template <int NB, int W, typename T>
__global__ __launch_bounds__(64 * W, NB == 8 ? 2 : 3) void kv4_attn_kernel(AttnArgs a) {
  constexpr int P = sizeof(T) == 4 ? 2 : 1;
  constexpr int D = NB * 32;
  const uint32_t tile = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const uint32_t head = blockIdx.y, seq = blockIdx.z;
  const Kv4Seq s = kv4_seq(a.kv, seq);
  const uint32_t cols = s.nrows * a.group, col0 = tile * kCols;
  if (col0 >= cols) return;
  const Range rg = key_range(a, s, col0, cols);
  if ((int32_t)split >= rg.active) return;

  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t r = lane & 15, g = lane >> 4, col = col0 + r;
  const bool mine = col < cols;
  const uint32_t row = mine ? col / a.group : 0, sub = mine ? col % a.group : 0;
  Query<NB, P> Q;
  load_query<NB, P, T>(Q, static_cast<const T *>(a.q) + (size_t)(s.row0 + row) * a.ldq +
                              (size_t)(head * a.group + sub) * D, mine, g, a.scale);
  // keys the lane's column sees
  int32_t lo = 0, hi = s.len;
  if (a.causal) {
    const int32_t p = s.pos0 + (int32_t)row;
    hi = p + 1 < hi ? p + 1 : hi;
    if (a.window && p >= (int32_t)a.window) lo = p - (int32_t)a.window + 1;
  }
  if (!mine) hi = 0;
  // keys every column of the wave sees
  int32_t all_lo = 0, all_hi = s.len;
  if (a.causal) {
    const uint32_t last = (col0 + kCols < cols ? col0 + kCols : cols) - 1;
    const int32_t p0 = s.pos0 + (int32_t)(col0 / a.group), p1 = s.pos0 + (int32_t)(last / a.group);
    all_hi = p0 + 1 < all_hi ? p0 + 1 : all_hi;
    if (a.window && p1 >= (int32_t)a.window) all_lo = p1 - (int32_t)a.window + 1;
  }

  Acc<NB> A;
  A.ref = kNever;
  A.sum = 0;
  A.down = 1;
  A.most = r >= 2 * NB % 16 ? 0.0f : __builtin_inff();
#pragma unroll
  for (int n = 0; n < 2 * NB; ++n) A.o[n] = (f32x4){0, 0, 0, 0};

  const int32_t end = rg.first + (((int32_t)split + 1) * rg.per < rg.steps ? ((int32_t)split + 1) * rg.per : rg.steps);
  int32_t at = rg.first + (int32_t)split * rg.per + (int32_t)wave;
  // Two steps' words in registers, one used while the other arrives, and the
  // page numbers one step further ahead.
  Step<NB> st[2];
  uint32_t pages[2];
  const Masks m = masks();
  find_pages(pages, a.kv, seq, at * kKeys, at < end ? s.len : 0);
  if (at < end) fetch<NB>(st[0], a.kv, pages, head, at * kKeys, lane);
  find_pages(pages, a.kv, seq, (at + W) * kKeys, at + W < end ? s.len : 0);
  while (at < end) {
    if (at + W < end) fetch<NB>(st[1], a.kv, pages, head, (at + W) * kKeys, lane);
    find_pages(pages, a.kv, seq, (at + 2 * W) * kKeys, at + 2 * W < end ? s.len : 0);
    const int32_t key = at * kKeys;
    const bool whole = key >= all_lo && key + kKeys <= all_hi && st[0].there[0] && st[0].there[1];
    if (!whole) cut_scales<NB>(st[0], key, s.len, r, g);
    float x[8];
    scores<NB, P>(x, Q, st[0], m);
    if (!whole) cut_scores<NB>(x, st[0], key, lo, hi, g);
    add_values<NB, P>(A, x, Q.fac, st[0], m);
    st[0] = st[1];
    at += W;
  }
  A.sum = sum_across(A.sum);
  const float up = 1 / A.down;  // a power of two

  // the waves' results: a common reference, then sums over the waves
  __shared__ float sh_ref[W][kCols], sh_sum[W][kCols];
  __shared__ float sh_o[W][kCols][D + 4];
  if (g == 0) {
    sh_ref[wave][r] = A.ref;
    sh_sum[wave][r] = A.sum;
  }
#pragma unroll
  for (int n = 0; n < 2 * NB; ++n) *reinterpret_cast<f32x4 *>(&sh_o[wave][r][16 * n + 4 * g]) = A.o[n] * up;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < kCols * D; i += 64 * W) {
    const uint32_t c = i / D, d = i % D;
    if (col0 + c >= cols) break;
    float ref = kNever, o = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) ref = __builtin_fmaxf(ref, sh_ref[w][c]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = __builtin_amdgcn_exp2f(sh_ref[w][c] - ref);
      sum = __builtin_fmaf(sh_sum[w][c], f, sum);
      o = __builtin_fmaf(sh_o[w][c][d], f, o);
    }
    if (rg.active == 1) {
      const uint32_t orow = s.row0 + (col0 + c) / a.group, oh = head * a.group + (col0 + c) % a.group;
      put<T>(static_cast<T *>(a.out) + (size_t)orow * a.ldo + (size_t)oh * D + d, sum == 0 ? 0.0f : o / sum);
    } else {
      const uint32_t tiles = gridDim.x / a.splits;
      float *w = a.work + ((((size_t)seq * gridDim.y + head) * tiles + tile) * a.splits + split) * kShare<D>;
      w[i] = o;
      if (d == 0) {
        w[kCols * D + c] = ref;
        w[kCols * D + kCols + c] = sum;
      }
    }
  }
}

// The shares' results of one column, joined: a workgroup per column, kv head
// and sequence.  The shares' references and sums first (a thread each), then
// D threads add up the shares' O, 256 / D groups of them every so many shares.
template <int NB, typename T>
__global__ __launch_bounds__(256) void kv4_attn_join_kernel(AttnArgs a, uint32_t tiles, uint32_t tile_cols) {
  constexpr int D = NB * 32, G = 256 / D;
  const uint32_t tile = blockIdx.x / tile_cols, c = blockIdx.x % tile_cols, head = blockIdx.y, seq = blockIdx.z;
  const Kv4Seq s = kv4_seq(a.kv, seq);
  const uint32_t cols = s.nrows * a.group, col0 = tile * kCols;
  if (col0 + c >= cols) return;
  const Range rg = key_range(a, s, col0, cols);
  if (rg.active == 1) return;
  const float *w = a.work + (((size_t)seq * gridDim.y + head) * tiles + tile) * a.splits * kShare<D>;
  __shared__ float weight[kMaxSplits], part[G][D], red[8];
  const uint32_t t = threadIdx.x;
  static_assert(kMaxSplits <= 256, "a thread per share");
  const bool mine = (int32_t)t < rg.active;
  const float ref = mine ? w[t * kShare<D> + kCols * D + c] : kNever;
  const float sum = mine ? w[t * kShare<D> + kCols * D + kCols + c] : 0;
  const float top = wave_max(ref);
  if (t % 64 == 0) red[t / 64] = top;
  __syncthreads();
  const float f = __builtin_amdgcn_exp2f(ref - __builtin_fmaxf(__builtin_fmaxf(red[0], red[1]),
                                                               __builtin_fmaxf(red[2], red[3])));
  const float all = wave_sum(sum * f);
  if (t % 64 == 0) red[4 + t / 64] = all;
  if (mine) weight[t] = f;
  __syncthreads();
  const uint32_t grp = t / D, d = t % D;
  if (grp < G) {
    float o = 0;
#pragma unroll 8
    for (int32_t n = grp; n < rg.active; n += G) o = __builtin_fmaf(w[n * kShare<D> + c * D + d], weight[n], o);
    part[grp][d] = o;
  }
  __syncthreads();
  if (t < D) {
    float o = 0;
#pragma unroll
    for (int g = 0; g < G; ++g) o += part[g][t];
    const float l = (red[4] + red[5]) + (red[6] + red[7]);
    const uint32_t orow = s.row0 + (col0 + c) / a.group, oh = head * a.group + (col0 + c) % a.group;
    put<T>(static_cast<T *>(a.out) + (size_t)orow * a.ldo + (size_t)oh * D + t, l == 0 ? 0.0f : o / l);
  }
}

struct Plan {
  uint32_t tiles, splits, min_steps;
  size_t share;  // bytes of one split of one tile
};
// How many workgroups may share the keys of a tile, and the fewest steps of a
// share: two workgroups per CU if every sequence had len_max keys, but shares
// of no more than 64 steps (a batch's lengths may differ; the long ones must
// not be what the call waits for) and of no less than 8 (two per wave).
Plan plan_of(const madi_kv4 *c, const madi_kv4_batch *b, uint32_t nh, uint32_t cus) {
  Plan p;
  const uint64_t reach = (uint64_t)b->max_pages * c->page;
  const uint64_t len = b->len_max && b->len_max < reach ? b->len_max : reach;
  const uint64_t cols = (uint64_t)b->rows * (nh / c->nkv);
  p.tiles = (uint32_t)((cols + kCols - 1) / kCols);
  p.share = (size_t)kCols * (c->d + 2) * 4;
  const uint64_t groups = (uint64_t)p.tiles * c->nkv * b->b, steps = (len + kKeys - 1) / kKeys;
  uint64_t per = groups * steps / (2 * cus);
  per = per > 64 ? 64 : per < 8 ? 8 : per;
  uint64_t want = (steps + per - 1) / per;
  if (groups >= 8ull * cus) want = 1;
  p.min_steps = (uint32_t)per;
  p.splits = (uint32_t)(want > kMaxSplits ? kMaxSplits : want < 1 ? 1 : want);
  return p;
}

template <int NB, typename T>
void launch(const AttnArgs &a, uint32_t tiles, uint32_t b) {
  kv4_attn_kernel<NB, 4, T><<<dim3(tiles * a.splits, a.kv.nkv, b), 256, 0, stream()>>>(a);
  const uint64_t cols = (uint64_t)a.kv.rows * a.group;
  const uint32_t tile_cols = cols < kCols ? (uint32_t)cols : kCols;
  if (a.splits > 1)
    kv4_attn_join_kernel<NB, T><<<dim3(tiles * tile_cols, a.kv.nkv, b), 256, 0, stream()>>>(a, tiles, tile_cols);
}

}  // namespace

extern "C" size_t madi_kv4_attn_bytes(const madi_kv4 *cache, const madi_kv4_batch *batch, uint32_t nh) {
  Kv4Args a;
  if (kv4_args("madi_kv4_attn_bytes", cache, batch, &a) || nh == 0 || nh % cache->nkv) return 0;
  const Plan p = plan_of(cache, batch, nh, initialized() ? (uint32_t)cu_count() : 256);
  return p.splits > 1 ? (size_t)p.tiles * cache->nkv * batch->b * p.splits * p.share : 0;
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
  if ((uint64_t)batch->rows * (nh / cache->nkv) > 0x7fffffffu)
    return fail(MADI_ERR_SHAPE, "%s: %u rows of a sequence in one call", what, batch->rows);
  if (!initialized()) return fail(MADI_ERR_NOT_INIT, "%s: madi_init has not succeeded", what);
  if (batch->m == 0 || batch->b == 0 || batch->rows == 0) return MADI_OK;
  Plan p = plan_of(cache, batch, nh, (uint32_t)cu_count());
  // as many splits as the workspace holds
  const size_t each = (size_t)p.tiles * cache->nkv * batch->b * p.share;
  if ((size_t)p.splits * each > wb) p.splits = wb / each > 1 ? (uint32_t)(wb / each) : 1;
  if ((uint64_t)p.tiles * p.splits > 0x7fffffffu)
    return fail(MADI_ERR_SHAPE, "%s: %u rows of a sequence in one call", what, batch->rows);
  if (int rc = deferred_before_read(q, qb)) return rc;
  if (int rc = deferred_before_read(cache->data, cb)) return rc;
  if (int rc = deferred_before_write(out, ob)) return rc;
  if (p.splits > 1)
    if (int rc = deferred_before_write(batch->work, wb)) return rc;
  a.q = q;
  a.out = out;
  a.work = static_cast<float *>(batch->work);
  a.ldq = ldq;
  a.ldo = ldo;
  a.group = nh / cache->nkv;
  a.window = window;
  a.causal = (uint32_t)causal;
  a.splits = p.splits;
  a.min_steps = p.min_steps;
  a.scale = scale;
  const bool f = dtype == MADI_F32;
  switch (cache->d) {
  case 64: f ? launch<2, float>(a, p.tiles, batch->b) : launch<2, f16>(a, p.tiles, batch->b); break;
  case 96: f ? launch<3, float>(a, p.tiles, batch->b) : launch<3, f16>(a, p.tiles, batch->b); break;
  case 128: f ? launch<4, float>(a, p.tiles, batch->b) : launch<4, f16>(a, p.tiles, batch->b); break;
  default: f ? launch<8, float>(a, p.tiles, batch->b) : launch<8, f16>(a, p.tiles, batch->b); break;
  }
  return check_launch(what);
}
