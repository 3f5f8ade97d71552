// kv4.h -- the 4-bit key/value cache's layout (see madi_q8.h) and the checks
// that its entry points share.
#pragma once

#include "common.h"

namespace madi {

// What a kernel needs of a madi_kv4 and a madi_kv4_batch.
struct Kv4Args {
  uint8_t *data;
  const uint32_t *table, *lens, *row_off;
  uint32_t n_pages, shift, nkv, max_pages, rows, m;
};

// A kernel's leading arguments: the hardware preloads the first 16 dwords of scalar
// arguments into SGPRs, but none of a struct, and a kernel's first loads (a length, a
// page number) wait for these.  KV4_ARGS passes them, KV4_GATHER puts them back.
#define KV4_PARAMS                                                                                         \
  const uint32_t *kv_lens, const uint32_t *kv_row_off, const uint32_t *kv_table, uint8_t *kv_data,         \
      uint32_t kv_max_pages, uint32_t kv_shift, uint32_t kv_rows, uint32_t kv_m, uint32_t kv_nkv,          \
      uint32_t kv_n_pages
#define KV4_ARGS(a) \
  (a).lens, (a).row_off, (a).table, (a).data, (a).max_pages, (a).shift, (a).rows, (a).m, (a).nkv, (a).n_pages
#define KV4_GATHER \
  Kv4Args{kv_data, kv_table, kv_lens, kv_row_off, kv_n_pages, kv_shift, kv_nkv, kv_max_pages, kv_rows, kv_m}

// Checks of the structs, the same for every entry point; fills `a`.
int kv4_args(const char *what, const madi_kv4 *c, const madi_kv4_batch *b, Kv4Args *a);
// Checks rows of `width` elements of dtype `ld` apart at p, and tells their
// extent in bytes.
int kv4_rows(const char *what, const char *name, const void *p, uint32_t m, uint64_t width,
             uint32_t ld, int dtype, size_t *bytes);
// Of a cache that kv4_args took.
inline size_t kv4_cache_bytes(const madi_kv4 *c) {
  return madi_kv4_bytes(c->n_pages, c->page, c->nkv, c->d);
}
inline bool kv4_overlap(const void *a, size_t an, const void *b, size_t bn) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return an && bn && x < y + bn && y < x + an;
}
// Whether [a, a + an) has a part of the batch's table, lens or row_off, which kernels take
// for constant while they write there.
inline bool kv4_on_batch(const madi_kv4_batch *b, const void *a, size_t an) {
  return kv4_overlap(a, an, b->table, (size_t)b->b * b->max_pages * 4) || kv4_overlap(a, an, b->lens, (size_t)b->b * 4) ||
         (b->row_off && kv4_overlap(a, an, b->row_off, ((size_t)b->b + 1) * 4));
}
// deferred_before_write for an extent of which a call writes some rows: what a recorded
// dequantisation owes the rest is carried out first.
inline int kv4_before_write(const void *p, size_t bytes) {
  if (int rc = deferred_before_read(p, bytes)) return rc;
  return deferred_before_write(p, bytes);
}

// ---------------------------------------------------------------- device side
// A number that no kernel writes while others read it: at a uniform address one
// scalar load, whatever else the kernel stores.
__device__ inline uint32_t kv4_const(const uint32_t *p) {
  return *(const __attribute__((address_space(4))) uint32_t *)(uintptr_t)p;
}
// Two scales as the most that a store writes, 9352, where they are more, infinite or no
// numbers, or negative: bits that no store wrote, at positions that a row does not
// see, times a weight of 0 are 0 then.
__device__ inline uint32_t kv4_finite(uint32_t w) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  const u16x2 s = __builtin_bit_cast(u16x2, w), most = {0x7091, 0x7091};
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(s, most));
}
// One sequence of the batch: its length, its rows [row0, row0 + nrows) of the
// inputs and outputs, and the position of the first.
struct Kv4Seq {
  int32_t len, pos0;
  uint32_t row0, nrows;
};
__device__ inline Kv4Seq kv4_seq(const Kv4Args &a, uint32_t i) {
  Kv4Seq s;
  const uint32_t reach = a.max_pages << a.shift, len = kv4_const(a.lens + i);
  s.len = (int32_t)(len < reach ? len : reach);
  uint32_t lo = i * a.rows, hi = lo + a.rows;
  if (a.row_off) {
    lo = kv4_const(a.row_off + i);
    hi = kv4_const(a.row_off + i + 1);
  }
  // the first row's position by all of the sequence's rows, those past m included
  const uint32_t all = lo < hi ? hi - lo : 0;
  s.pos0 = s.len - (int32_t)(all < 0x7fffffffu ? all : 0x7fffffffu);
  hi = hi < a.m ? hi : a.m;
  lo = lo < hi ? lo : hi;
  s.row0 = lo;
  s.nrows = hi - lo < a.rows ? hi - lo : a.rows;
  return s;
}
// Page of position pos (0 <= pos < reach) of sequence i.
__device__ inline uint32_t kv4_page(const Kv4Args &a, uint32_t i, uint32_t pos) {
  return kv4_const(a.table + (size_t)i * a.max_pages + (pos >> a.shift));
}
// Bytes of one page and head, and the start of page p, head h.
__device__ inline size_t kv4_block_bytes(uint32_t shift, uint32_t d) {
  return ((size_t)d * 9 / 8) << shift;
}
__device__ inline uint8_t *kv4_block(const Kv4Args &a, uint32_t p, uint32_t h, uint32_t d) {
  return a.data + ((size_t)p * a.nkv + h) * kv4_block_bytes(a.shift, d);
}

}  // namespace madi
