// kv4.hip -- K and V rows into the 4-bit cache and back (madi_kv4_store,
// madi_kv4_load; the format and the layout are in madi_q8.h).
//
// A unit of work is four consecutive tokens (4u..4u+3 of a sequence) of one
// block of one head, first of K, then of V: 2 x 128 elements, 16 lanes of 8, so
// that a V word (four tokens' bytes) is made in one place.  Lane l of the 16 has
// token l & 3 and elements 32b + 8g .. + 7, g = 2 (l >> 2 & 1) + (l >> 3): with
// this order the V words come out of two byte transposes between neighbouring lanes
// (DPP) instead of through LDS.  A border between two codes costs one
// multiply-add beside the estimate (see code()), no division.
//
// Both are bound by memory, K's and V's loads in flight together: 131072 rows
// of 8 heads of 128 in f16 read back in 137 us (0.69 GB at 5.0 TB/s, where a copy
// reaches 5.1 to 5.24), 16384 stored in 23.2 (3.7 TB/s: the codes'
// arithmetic is not all hidden behind the copy) and read back in
// 15.3, single rows of eight sequences in 3.3 and 2.7, which is the latencies of a
// length, a page number and the rows, one after the other.  (Two units per lane: 130
// us for the first, but 24 sequences' ragged prompts, stored and read, 17.8 where they
// took 13.8 then, 12.5 now.)
#include "kv4.h"

using namespace madi;

namespace madi {

namespace {
// (a page's offsets within a head are 32-bit: 2^20 tokens of 288 bytes)
bool kv4_shape_ok(uint32_t page, uint32_t nkv, uint32_t d) {
  return (d == 64 || d == 96 || d == 128 || d == 256) && page >= 16 && (page & (page - 1)) == 0 &&
         page <= (1u << 20) && nkv >= 1 && nkv <= 65535;
}
}  // namespace

int kv4_args(const char *what, const madi_kv4 *c, const madi_kv4_batch *b, Kv4Args *a) {
  if (!c || !b) return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (!kv4_shape_ok(c->page, c->nkv, c->d))
    return fail(MADI_ERR_SHAPE,
                "%s: page %u, nkv %u, d %u (page a power of two from 16 to 2^20, nkv 1 to 65535, d 64, 96, "
                "128 or 256)", what, c->page, c->nkv, c->d);
  if (kv4_cache_bytes(c) == 0)
    return fail(MADI_ERR_SHAPE, "%s: a cache of %u pages (1 to 2^48 bytes)", what, c->n_pages);
  if (b->b > 65535) return fail(MADI_ERR_SHAPE, "%s: %u sequences (at most 65535)", what, b->b);
  if (b->m > 0x7fffffffu || b->rows > 0x7fffffffu)
    return fail(MADI_ERR_SHAPE, "%s: m %u, rows %u (below 2^31)", what, b->m, b->rows);
  if (!b->row_off && (uint64_t)b->b * b->rows != b->m)
    return fail(MADI_ERR_SHAPE, "%s: m = %u is not b * rows = %u * %u", what, b->m, b->b, b->rows);
  if (b->b && b->max_pages == 0) return fail(MADI_ERR_SHAPE, "%s: max_pages is 0", what);
  // (positions are int32_t, and a kernel's steps and chunks end a little past the last one)
  if ((uint64_t)b->max_pages * c->page > 0x7ffff000u)
    return fail(MADI_ERR_SHAPE, "%s: max_pages * page = %u * %u positions (at most 2^31 - 4096)", what,
                b->max_pages, c->page);
  if (!c->data || (b->b && (!b->table || !b->lens)))
    return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (!aligned(c->data, 16) || !aligned(b->table, 4) || !aligned(b->lens, 4) ||
      !aligned(b->row_off, 4))
    return fail(MADI_ERR_ALIGN, "%s: data must be 16-byte, table, lens and row_off 4-byte aligned", what);
  a->data = static_cast<uint8_t *>(c->data);
  a->table = b->table;
  a->lens = b->lens;
  a->row_off = b->row_off;
  a->n_pages = c->n_pages;
  a->shift = (uint32_t)__builtin_ctz(c->page);
  a->nkv = c->nkv;
  a->max_pages = b->max_pages;
  a->rows = b->rows;
  a->m = b->m;
  return MADI_OK;
}

int kv4_rows(const char *what, const char *name, const void *p, uint32_t m, uint64_t width,
             uint32_t ld, int dtype, size_t *bytes) {
  const uint32_t es = dtype == MADI_F32 ? 4 : 2;
  *bytes = 0;
  if (dtype != MADI_F16 && dtype != MADI_F32) return fail(MADI_ERR_ARG, "%s: dtype %d", what, dtype);
  if (width > ld) return fail(MADI_ERR_SHAPE, "%s: rows of %s are %u apart but %llu long", what, name, ld,
                              (unsigned long long)width);
  if (!p && m) return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (!aligned(p, 16) || (uint64_t)ld * es % 16)
    return fail(MADI_ERR_ALIGN, "%s: rows of %s must be 16-byte aligned", what, name);
  if (m) *bytes = ((size_t)(m - 1) * ld + width) * es;
  return MADI_OK;
}

}  // namespace madi

namespace {

// a value from another lane of the 16 (a DPP row)
template <int CTRL>
__device__ inline uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kReverse4 = 0x1b;  // quad_perm
constexpr int kRor4 = 0x124, kRor8 = 0x128, kHalfMirror = 0x141;
__device__ inline uint32_t lane_xor4(uint32_t v) {  // 7 - i, then within the four
  return dpp<kReverse4>(dpp<kHalfMirror>(v));
}

// 4 x 4 bytes between four neighbouring lanes: lane j's byte i <-> lane i's byte j.
__device__ inline uint32_t transpose4(uint32_t w, uint32_t lane) {
  uint32_t o = dpp<kXor1>(w);  // bytes (a0 a1 a2 a3), (b0 ..): even a0 b0 a2 b2, odd a1 b1 a3 b3
  w = lane & 1 ? __builtin_amdgcn_perm(w, o, 0x07030501u) : __builtin_amdgcn_perm(w, o, 0x02060004u);
  o = dpp<kXor2>(w);
  return lane & 2 ? __builtin_amdgcn_perm(w, o, 0x07060302u) : __builtin_amdgcn_perm(w, o, 0x01000504u);
}
// bytes 0 1 2 3 <-> tokens 0 2 1 3
__device__ inline uint32_t token_order(uint32_t w) { return __builtin_amdgcn_perm(w, w, 0x03010200u); }

__device__ inline void load8(const float *p, float (&x)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = a[i];
    x[4 + i] = b[i];
  }
}
__device__ inline void load8(const f16 *p, float (&x)[8]) {
  const f16x8 a = *reinterpret_cast<const f16x8 *>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
}
// (not kept in the L2, which the rows mostly exceed: with ordinary stores 131072 rows of 8
// heads of 128 took 6 % longer to read back)
__device__ inline void store8(float *p, const float (&x)[8]) {
  __builtin_nontemporal_store((f32x4){x[0], x[1], x[2], x[3]}, reinterpret_cast<f32x4 *>(p));
  __builtin_nontemporal_store((f32x4){x[4], x[5], x[6], x[7]}, reinterpret_cast<f32x4 *>(p + 4));
}
__device__ inline void store8(f16 *p, const float (&x)[8]) {
  f16x8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (f16)x[i];
  __builtin_nontemporal_store(v, reinterpret_cast<f16x8 *>(p));
}

// The code of x plus 8, as a number, against scale s > 0: |x| / s to the nearest
// whole number, halves away from zero.  `inv` is 1 / s taken 2^-21 too small, more than
// rcp and the multiply-add are off (by 2^-23 and 2^-24 of |x| / s + 1/2), so the estimate
// is the code or one less.  The remainder a - q s is exact in f32 (s has 11 bits and
// q 4), so comparing it with s / 2, exact too, settles the code.  A NaN's is 0: the
// maximum drops it, and it compares with nothing.
constexpr float kBelow = 1 - 0x1p-21f;
__device__ inline float code(float x, float s, float inv, float half) {
  const float a = __builtin_fabsf(x);
  float q = __builtin_fminf(__builtin_fmaxf(__builtin_floorf(__builtin_fmaf(a, inv, 0.5f)), 0.0f), 7.0f);
  q += __builtin_fmaf(-q, s, a) >= half ? 1.0f : 0.0f;
  return 8.0f + __builtin_copysignf(__builtin_fminf(q, 7.0f), x);
}

struct Unit {
  uint32_t seq, h, b, g, tok, col;  // col: first of the lane's 8 elements in a row
  int32_t pos;    // of the lane's token
  int32_t first;  // of token 0
  bool mine;      // the lane's token is one of the call's rows
  size_t row;     // and that row
  Kv4Seq s;
};
// The calling lane's unit; false where the workgroup or the lane has none.
template <int NB>
__device__ inline bool unit_of(const Kv4Args &a, uint32_t per_quad, Unit &u) {
  const uint32_t quad = blockIdx.x / per_quad, part = blockIdx.x % per_quad;
  const uint32_t l = threadIdx.x & 15, hb = part * 16 + (threadIdx.x >> 4);
  u.seq = blockIdx.y;
  u.s = kv4_seq(a, u.seq);
  if (quad * 4 >= ((uint32_t)u.s.pos0 & 3) + u.s.nrows || hb >= a.nkv * NB) return false;
  u.first = ((u.s.pos0 >> 2) + (int32_t)quad) * 4;
  u.h = hb / NB;
  u.b = hb % NB;
  u.tok = l & 3;
  u.g = (l >> 2 & 1) * 2 + (l >> 3);
  u.col = hb * 32 + u.g * 8;
  u.pos = u.first + (int32_t)u.tok;
  u.mine = u.pos >= u.s.pos0 && u.pos < u.s.pos0 + (int32_t)u.s.nrows;
  u.row = u.s.row0 + (uint32_t)(u.pos - u.s.pos0);
  return true;
}

// The codes (plus 8, a byte each) of the lane's 8 elements and their block's scale.
__device__ inline f16 quantise(const float (&x)[8], uint32_t &lo, uint32_t &hi) {
  float top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    top = __builtin_fmaxf(top, __builtin_fabsf(x[i]));  // (of a NaN and a number the number)
  }
  // the four lanes of the token's block
  top = __builtin_fmaxf(top, __builtin_bit_cast(float, dpp<kRor4>(__builtin_bit_cast(uint32_t, top))));
  top = __builtin_fmaxf(top, __builtin_bit_cast(float, dpp<kRor8>(__builtin_bit_cast(uint32_t, top))));
  f16 sh = (f16)(top / 7.0f);
  if (!(sh <= (f16)9352.0f)) sh = (f16)9352.0f;
  const float s = (float)sh;
  lo = hi = 0x08080808u;
  if (s > 0) {
    const float inv = __builtin_amdgcn_rcpf(s) * kBelow, half = 0.5f * s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo = __builtin_amdgcn_cvt_pk_u8_f32(code(x[i], s, inv, half), i, lo);
      hi = __builtin_amdgcn_cvt_pk_u8_f32(code(x[4 + i], s, inv, half), i, hi);
    }
  }
  return sh;
}

template <int NB, typename T>
__global__ __launch_bounds__(256) void kv4_store_kernel(KV4_PARAMS, const T *__restrict__ k,
                                                        const T *__restrict__ v, uint32_t ldk,
                                                        uint32_t ldv, uint32_t per_quad) {
  const Kv4Args a = KV4_GATHER;
  Unit u;
  if (!unit_of<NB>(a, per_quad, u) || u.first < 0) return;
  constexpr uint32_t D = NB * 32;
  const uint32_t l = threadIdx.x & 15;
  // a unit of four tokens lies in one page; its number and the rows are asked for together
  const uint32_t page = kv4_page(a, u.seq, u.first);
  float x[8] = {0, 0, 0, 0, 0, 0, 0, 0}, y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (u.mine) {
    load8(k + u.row * ldk + u.col, x);
    load8(v + u.row * ldv + u.col, y);
  }
  if (page >= a.n_pages) return;
  uint8_t *blk = kv4_block(a, page, u.h, D);
  const uint32_t off = (uint32_t)u.pos & ((1u << a.shift) - 1), four = off >> 2;
  f16 *sc = reinterpret_cast<f16 *>(blk + ((size_t)D << a.shift) + (size_t)four * (D / 2)) + u.b * 4 + u.tok;

  uint32_t lo, hi;
  f16 s = quantise(x, lo, hi);
  // K: element 2j in nibble j, element 2j+1 in nibble 4+j
  const uint32_t ev = __builtin_amdgcn_perm(hi, lo, 0x06040200u);  // bytes e0 e2 e4 e6
  const uint32_t od = __builtin_amdgcn_perm(hi, lo, 0x07050301u);  // bytes e1 e3 e5 e7
  const uint32_t evn = ev | ev >> 4, odn = od | od >> 4;           // nibble pairs in bytes 0, 2
  if (u.mine) {
    if (u.g == 0) sc[0] = s;
    *reinterpret_cast<uint32_t *>(blk + (size_t)off * (D / 2) + (u.g * NB + u.b) * 4) =
        __builtin_amdgcn_perm(odn, evn, 0x06040200u);
  }

  s = quantise(y, lo, hi);
  if (u.mine && u.g == 0) sc[4 * NB] = s;
  // V: lanes 8i + 0..3 have the low nibbles of 8 words, lanes 8i + 4..7 the high
  // ones of the same 8: they exchange four words' worth, then four lanes (the
  // four tokens) transpose, and lane l has word (c = l, b).
  const uint32_t odd = l & 4;
  const uint32_t got = lane_xor4(odd ? lo : hi);
  uint32_t w = odd ? (got | hi << 4) : (lo | got << 4);
  w = token_order(transpose4(w, l));
  uint8_t *dst = blk + ((size_t)(D / 2) << a.shift) + (size_t)four * (2 * D) + (l * NB + u.b) * 4;
  // tokens of this store among the four
  const int32_t lo_t = u.s.pos0 - u.first, hi_t = lo_t + (int32_t)u.s.nrows;
  if (lo_t <= 0 && hi_t >= 4) {
    *reinterpret_cast<uint32_t *>(dst) = w;
  } else {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int byte = (t & 1) * 2 + (t >> 1);
      if (t >= lo_t && t < hi_t) dst[byte] = (uint8_t)(w >> (8 * byte));
    }
  }
}

// Codes (plus 8, a byte each) times the scale.
template <typename T>
__device__ inline void put_row(T *p, uint32_t lo, uint32_t hi, float s) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = (float)((int)(lo >> (8 * i) & 0xffu) - 8) * s;
    x[4 + i] = (float)((int)(hi >> (8 * i) & 0xffu) - 8) * s;
  }
  store8(p, x);
}

template <int NB, typename T>
__global__ __launch_bounds__(256) void kv4_load_kernel(KV4_PARAMS, T *__restrict__ k, T *__restrict__ v,
                                                       uint32_t ldk, uint32_t ldv, uint32_t per_quad) {
  const Kv4Args a = KV4_GATHER;
  Unit u;
  if (!unit_of<NB>(a, per_quad, u)) return;
  constexpr uint32_t D = NB * 32;
  const uint32_t l = threadIdx.x & 15;
  uint32_t page = 0xffffffffu;
  if (u.first >= 0) page = kv4_page(a, u.seq, u.first);  // below 0 there is none
  uint32_t kw = 0x88888888u, vw = 0x88888888u;
  float ks = 0, vs = 0;
  if (page < a.n_pages) {
    const uint8_t *blk = kv4_block(a, page, u.h, D);
    const uint32_t off = (uint32_t)u.first & ((1u << a.shift) - 1), four = off >> 2;
    const f16 *sc = reinterpret_cast<const f16 *>(blk + ((size_t)D << a.shift) + (size_t)four * (D / 2)) + u.b * 4 + u.tok;
    kw = *reinterpret_cast<const uint32_t *>(blk + (size_t)(off + u.tok) * (D / 2) + (u.g * NB + u.b) * 4);
    vw = *reinterpret_cast<const uint32_t *>(blk + ((size_t)(D / 2) << a.shift) + (size_t)four * (2 * D) +
                                             (l * NB + u.b) * 4);
    ks = (float)sc[0];
    vs = (float)sc[4 * NB];
  }
  const uint32_t a0 = kw & 0x0f0f0f0fu, a1 = (kw >> 4) & 0x0f0f0f0fu;  // e0 e4 e1 e5, e2 e6 e3 e7
  if (u.mine)
    put_row(k + u.row * ldk + u.col, __builtin_amdgcn_perm(a1, a0, 0x06040200u),
            __builtin_amdgcn_perm(a1, a0, 0x07050301u), ks);
  vw = transpose4(token_order(vw), l);  // the lane's token of words c = 4 (l >> 2) + 0..3
  const uint32_t low = vw & 0x0f0f0f0fu, high = (vw >> 4) & 0x0f0f0f0fu, odd = l & 4;
  const uint32_t got = lane_xor4(odd ? low : high);
  if (u.mine) put_row(v + u.row * ldv + u.col, odd ? got : low, odd ? high : got, vs);
}

template <bool STORE, int NB, typename T>
void launch(const Kv4Args &a, dim3 grid, void *k, void *v, uint32_t ldk, uint32_t ldv, uint32_t per_quad) {
  if constexpr (STORE)
    kv4_store_kernel<NB, T><<<grid, 256, 0, stream()>>>(KV4_ARGS(a), (const T *)k, (const T *)v, ldk, ldv, per_quad);
  else
    kv4_load_kernel<NB, T><<<grid, 256, 0, stream()>>>(KV4_ARGS(a), (T *)k, (T *)v, ldk, ldv, per_quad);
}

template <bool STORE>
int run(const char *what, const madi_kv4 *c, const madi_kv4_batch *b, void *k, void *v, uint32_t ldk,
        uint32_t ldv, int dtype) {
  Kv4Args a;
  if (int rc = kv4_args(what, c, b, &a)) return rc;
  const uint64_t width = (uint64_t)c->nkv * c->d;
  size_t kb, vb;
  if (int rc = kv4_rows(what, "k", k, b->m, width, ldk, dtype, &kb)) return rc;
  if (int rc = kv4_rows(what, "v", v, b->m, width, ldv, dtype, &vb)) return rc;
  const size_t cb = kv4_cache_bytes(c);
  if (kv4_overlap(k, kb, c->data, cb) || kv4_overlap(v, vb, c->data, cb))
    return fail(MADI_ERR_ARG, "%s: k or v lies in the cache", what);
  if (STORE ? kv4_on_batch(b, c->data, cb) : kv4_on_batch(b, k, kb) || kv4_on_batch(b, v, vb))
    return fail(MADI_ERR_ARG, "%s: %s on table, lens or row_off", what, STORE ? "the cache lies" : "k or v lie");
  // K and V rows may alternate in one buffer; the extents overlap then, the rows do not
  if (!STORE && kv4_overlap(k, kb, v, vb)) {
    const size_t es = dtype == MADI_F32 ? 4 : 2, row = (size_t)ldk * es, w = (size_t)width * es;
    const uintptr_t x = reinterpret_cast<uintptr_t>(k), y = reinterpret_cast<uintptr_t>(v);
    const size_t gap = (x < y ? y - x : x - y) % row;
    if (ldk != ldv || gap < w || row - gap < w)
      return fail(MADI_ERR_ARG, "%s: rows of k and v overlap", what);
  }
  // workgroups of 16 units for each four tokens a sequence's rows may touch (those of
  // shorter sequences end at once)
  const uint32_t per_quad = (uint32_t)((width / 32 + 15) / 16);
  const uint64_t quads = ((uint64_t)b->rows + 3) / 4 + 1, gx = quads * per_quad;
  if (gx > 0xffffffu)  // 2^32 threads
    return fail(MADI_ERR_SHAPE, "%s: %u rows of %llu elements in one call", what, b->rows, (unsigned long long)width);
  if (!initialized()) return fail(MADI_ERR_NOT_INIT, "%s: madi_init has not succeeded", what);
  if (b->m == 0 || b->b == 0 || b->rows == 0) return MADI_OK;
  if (STORE) {
    if (int rc = deferred_before_read(k, kb)) return rc;
    if (int rc = deferred_before_read(v, vb)) return rc;
    if (int rc = kv4_before_write(c->data, cb)) return rc;
  } else {
    if (int rc = deferred_before_read(c->data, cb)) return rc;
    if (int rc = kv4_before_write(k, kb)) return rc;
    if (int rc = kv4_before_write(v, vb)) return rc;
  }
  const dim3 grid((uint32_t)gx, b->b);
  const bool f = dtype == MADI_F32;
  switch (c->d) {
  case 64: f ? launch<STORE, 2, float>(a, grid, k, v, ldk, ldv, per_quad)
             : launch<STORE, 2, f16>(a, grid, k, v, ldk, ldv, per_quad); break;
  case 96: f ? launch<STORE, 3, float>(a, grid, k, v, ldk, ldv, per_quad)
             : launch<STORE, 3, f16>(a, grid, k, v, ldk, ldv, per_quad); break;
  case 128: f ? launch<STORE, 4, float>(a, grid, k, v, ldk, ldv, per_quad)
              : launch<STORE, 4, f16>(a, grid, k, v, ldk, ldv, per_quad); break;
  default: f ? launch<STORE, 8, float>(a, grid, k, v, ldk, ldv, per_quad)
             : launch<STORE, 8, f16>(a, grid, k, v, ldk, ldv, per_quad); break;
  }
  return check_launch(what);
}

}  // namespace

extern "C" size_t madi_kv4_bytes(uint32_t n_pages, uint32_t page, uint32_t nkv, uint32_t d) {
  if (!kv4_shape_ok(page, nkv, d)) return 0;
  const size_t one = (size_t)nkv * page * (d / 8) * 9;  // below 2^45
  return n_pages <= ((size_t)1 << 48) / one ? n_pages * one : 0;
}

extern "C" int madi_kv4_store(const madi_kv4 *cache, const madi_kv4_batch *batch, const void *k,
                              const void *v, uint32_t ldk, uint32_t ldv, int dtype) {
  return run<true>("madi_kv4_store", cache, batch, const_cast<void *>(k), const_cast<void *>(v), ldk, ldv,
                   dtype);
}

extern "C" int madi_kv4_load(void *k, void *v, uint32_t ldk, uint32_t ldv, int dtype, const madi_kv4 *cache,
                             const madi_kv4_batch *batch) {
  return run<false>("madi_kv4_load", cache, batch, k, v, ldk, ldv, dtype);
}
