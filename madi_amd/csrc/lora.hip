// lora.hip -- the batched projection with a low-rank adapter per row (madi_q8_pproj_lora):
// out = W x + scale[a] B[a] (A[a] x).
//
// Two launches: h = scale A x of every row, here, kept as lora.h says; then the projection's own
// kernels, whose sums start from B h.
#include "kv4.h"
#include "lora.h"
#include "lora_places.h"

using namespace madi;

namespace {

constexpr uint32_t kMaxRank = 128;
// A workgroup per row up to kRowKernel rows, two for each CU, whose x fits kRowLds bytes.  (Whole projections with rows
// of adapters against tiles of 16: 8 x 1280 8.0 / 11.6 us, 256 x 5120 32 / 43, 400 x 1280 16.4 / 17.7;
// 1000 x 5120 with rank 64 70 / 63, 1500 x 1280 34 / 25.)
constexpr uint32_t kRowKernel = 512, kRowLds = 63 << 10;

struct Adapters {
  const f16 *a;
  const float *scale;
  const uint32_t *adapter, *row_seq;
  uint32_t n, rank, seqs;
};
// The adapter of a row, kNoAdapter if it has none.
__device__ inline uint32_t adapter_of(const Adapters &l, uint32_t row) {
  uint32_t i = row;
  if (l.row_seq) {
    i = l.row_seq[row];
    if (i >= l.seqs) return kNoAdapter;
  }
  const uint32_t a = l.adapter[i];
  return a < l.n ? a : kNoAdapter;
}

// Sums over lanes and rows of 16 lanes by DPP and row exchanges.
template <int CTRL>
__device__ inline float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ inline float wave_sum(float v) {
  v += dpp<0xb1>(v);
  v += dpp<0x4e>(v);
  v += dpp<0x141>(v);
  v += dpp<0x140>(v);
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto x = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = __builtin_bit_cast(float, (uint32_t)x[0]) + __builtin_bit_cast(float, (uint32_t)x[1]);
  const uint32_t w = __builtin_bit_cast(uint32_t, v);
  const auto y = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __builtin_bit_cast(float, (uint32_t)y[0]) + __builtin_bit_cast(float, (uint32_t)y[1]);
}

// A row's h as two f16: the largest (of those that are finite) is scaled to 2^14 .. 2^15, where the low part of every
// value that counts is a normal f16.  An infinity is one in the high part alone: B h is what it is in f32.
__device__ inline float finite(float v) {
  v = __builtin_fabsf(v);
  return v < INFINITY ? v : 0.0f;
}
__device__ inline int exponent_of(float top) {
  if (!(top > 0)) return 0;
  const int e = __builtin_amdgcn_frexp_expf(top) - 15;
  return e < -126 ? -126 : e;
}
__device__ inline void halves(float v, int e, f16 &hi, f16 &lo) {
  v = __builtin_amdgcn_ldexpf(v, -e);
  hi = (f16)v;
  lo = __builtin_fabsf(v) < INFINITY ? (f16)(v - (float)hi) : (f16)0.0f;
}

// The XCDs take workgroups in turn: here each gets neighbours, whose rows mostly share an adapter that its L2 reads
// once (320 x 5120 with rank 64 38.7 -> 37.5 us).
__device__ inline uint32_t neighbours() {
  const uint32_t n = gridDim.x, x = blockIdx.x % 8, more = n % 8;
  return x * (n / 8) + (x < more ? x : more) + blockIdx.x / 8;
}

// A workgroup of 16 waves per row, wave w has ranks w, w + 16, ...: x rounded to f16 once, through LDS; the adapter's
// rows S loads of 512 elements at a time, the next ones always on their way, the first before x is there.  (Loads past
// the end of a row take its last elements: with a branch around each, every use waited for the newest load.)  Bound by
// waits for memory: 40 rows of 5120 with rank 32 7.4 us (10.0 with branches), 340 KB into each of 40 CUs, whose waves wait
// 55 % of their cycles (counters) and keep the vector pipes busy for a tenth; 8 of 1280 with 16 3.5.  Grid (m).
constexpr uint32_t kStep = 512;
template <int S>
__global__ __launch_bounds__(1024) void lora_row_kernel(Adapters l, const float *__restrict__ in, uint32_t k,
                                                        uint32_t tile_rows, f16 *__restrict__ h, float *__restrict__ factor,
                                                        uint32_t *__restrict__ id) {
  extern __shared__ __attribute__((aligned(16))) uint8_t dyn[];
  f16 *xs = reinterpret_cast<f16 *>(dyn);  // [k]
  __shared__ float hs[kMaxRank];
  const uint32_t row = neighbours(), lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float *x = in + (size_t)row * k;
  const uint32_t c0 = threadIdx.x * 4;
  const auto load_x = [&](uint32_t c) { return *reinterpret_cast<const f32x4 *>(x + (c < k ? c : 0)); };
  const f32x4 first = load_x(c0);
  f32x4 second = {};
  if (S * kStep > 4096) second = load_x(c0 + 4096);
  const uint32_t a = adapter_of(l, row);
  if (threadIdx.x == 0) id[row] = a;
  if (a == kNoAdapter) {
    if (threadIdx.x == 0) factor[row] = 0;
    return;
  }
  const float scale = l.scale[a];
  const f16 *w = l.a + (size_t)a * l.rank * k;
  const auto load = [&](uint32_t r, uint32_t c, f16x8 (&v)[S]) {
    const f16 *p = w + (size_t)(r < l.rank ? r : l.rank - 1) * k;
#pragma unroll
    for (uint32_t j = 0; j < S; ++j) {
      const uint32_t at = c + j * kStep + lane * 8;
      v[j] = *reinterpret_cast<const f16x8 *>(p + (at < k ? at : k - 8));
    }
  };
  f16x8 now[S], next[S];
  load(wave, 0, now);
  const auto keep = [&](uint32_t c, const f32x4 &u) {
    f16x4 v = {(f16)u.x, (f16)u.y, (f16)u.z, (f16)u.w};
    asm volatile("" : "+v"(v));  // waited for by all lanes
    if (c < k) *reinterpret_cast<f16x4 *>(xs + c) = v;
  };
  keep(c0, first);
  if (S * kStep > 4096) {
    keep(c0 + 4096, second);
    for (uint32_t c = c0 + 8192; c < k; c += 4096) keep(c, *reinterpret_cast<const f32x4 *>(x + c));
  }
  __syncthreads();
  float sum[2] = {0, 0};
  uint32_t r = wave, c = 0;  // of `now`
  const auto take = [&](f16x8 (&v)[S], f16x8 (&then)[S]) {  // false after the wave's last
    const bool ends = c + S * kStep >= k;
    const uint32_t nr = ends ? r + 16 : r, nc = ends ? 0 : c + S * kStep;
    load(nr, nc, then);
#pragma unroll
    for (uint32_t j = 0; j < S; ++j) {
      const uint32_t at = c + j * kStep + lane * 8;
      if (at >= k) continue;
      const f16x8 u = *reinterpret_cast<const f16x8 *>(xs + at);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e & 1] = __builtin_fmaf((float)u[e], (float)v[j][e], sum[e & 1]);
    }
    if (ends) {
      const float all = wave_sum(sum[0] + sum[1]);
      if (lane == 0) hs[r] = all * scale;
      sum[0] = sum[1] = 0;
    }
    r = nr;
    c = nc;
    return r < l.rank;
  };
  if (r < l.rank)
    while (take(now, next) && take(next, now)) {}
  __syncthreads();
  if (threadIdx.x < l.rank) {
    float top = 0;
#pragma unroll 8
    for (uint32_t r = 0; r < l.rank; ++r) top = __builtin_fmaxf(top, finite(hs[r]));
    const int e = exponent_of(top);
    const LoraShape shape = lora_shape(l.rank, tile_rows);
    halves(hs[threadIdx.x], e, h[lora_at(shape, row, threadIdx.x, false)], h[lora_at(shape, row, threadIdx.x, true)]);
    if (threadIdx.x == 0) factor[row] = __builtin_amdgcn_ldexpf(1.0f, e);
  }
}

// Many rows: a workgroup of 16 waves per 16 rows, v_mfma_f32_16x16x32_f16 with the adapter's rows as the first
// operand.  x goes through LDS in f16, kChunk elements of a row at a time (and to x16 where that is asked for); the
// waves deal out the 16-row tiles of the rank (RT) and the chunk's steps of 32.  Each adapter of the rows takes a pass;
// where CUs are left over, grid y of them deal the passes out.  Bound by waits for memory (57 % of the waves' cycles)
// and by too few workgroups: 2000 rows of 1280, 12 adapters of rank 64, 11.6 us on 125 CUs, and a second adapter's pass on few
// more (15.4 with branches around the loads and both passes of a tile with two adapters in one workgroup).  Grid (m / 16,
// 1 to 4).
constexpr uint32_t kTileWaves = 16, kChunk = 2048, kPitch = kChunk * 2 + 16;  // (rows 16 bytes off: other banks)
template <int RT>
__global__ __launch_bounds__(kTileWaves * 64) void lora_tile_kernel(Adapters l, const float *__restrict__ in, uint32_t m,
                                                                    uint32_t k, uint32_t tile_rows, f16 *__restrict__ h,
                                                                    float *__restrict__ factor, uint32_t *__restrict__ id,
                                                                    f16 *__restrict__ x16) {
  __shared__ __attribute__((aligned(16))) uint8_t xs[16 * kPitch];
  __shared__ f32x4 part[kTileWaves][64];
  __shared__ uint32_t tops[16];
  constexpr uint32_t kParts = kTileWaves / RT, kTogether = RT == 1 ? 4 : RT == 2 ? 8 : 10, kLoads = kChunk / 256;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t t = wave % RT, kp = wave / RT;
  const uint32_t g = lane >> 4, c = lane & 15, m0 = neighbours() * 16, row = m0 + c < m ? m0 + c : m - 1;
  // wave w takes row w of x, 1 KiB at a time; the first chunk is asked for before the adapters are known
  const uint32_t xr = m0 + wave < m ? m0 + wave : m - 1;
  const float *x = in + (size_t)xr * k;
  f32x4 v[kLoads];
  const auto load_x = [&](uint32_t k0) {  // (past the row's end its last elements again: a branch per load, and a wait
#pragma unroll                            //  for all loads and stores before each use, took 3 us more)
    for (uint32_t j = 0; j < kLoads; ++j)
      v[j] = *reinterpret_cast<const f32x4 *>(x + lora_x_place(k0 + j * 256 + lane * 4, k));
  };
  load_x(0);
  const uint32_t mine = m0 + c < m ? adapter_of(l, row) : kNoAdapter;
  const float scale = mine != kNoAdapter ? l.scale[mine] : 0.0f;
  const uint32_t r = t * 16 + c < l.rank ? t * 16 + c : l.rank - 1;  // (sums past the rank are not kept)
  // the rows' adapters are dealt out over blockIdx.y, the first of them to 0
  uint64_t some = __ballot(mine != kNoAdapter);
  if (gridDim.y > 1) {
    uint64_t own = 0;
    for (uint32_t turn = 0; some; turn = turn + 1 < gridDim.y ? turn + 1 : 0) {
      const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)mine, __builtin_ctzll(some));
      const uint64_t its = __ballot(mine == a);
      if (turn == blockIdx.y) own |= its;
      some &= ~its;
    }
    some = own;
    if (blockIdx.y && !some) return;
  }
  if (blockIdx.y) x16 = nullptr;
  const bool here = some >> lane & 1, none = mine == kNoAdapter && blockIdx.y == 0;  // the row is this workgroup's
  const auto put_x16 = [&](uint32_t k0, uint32_t kc) {  // (after the products: a barrier waits for stores before it)
    if (x16 && m0 + wave < m)
      for (uint32_t at = lane * 8; at < kc; at += 512)
        *reinterpret_cast<f16x8 *>(x16 + (size_t)xr * k + k0 + at) = *reinterpret_cast<const f16x8 *>(xs + wave * kPitch + at * 2);
  };
  f32x4 acc = {};
  for (uint32_t k0 = 0; k0 < k && (some || x16); k0 += kChunk) {
    const uint32_t kc = k - k0 < kChunk ? k - k0 : kChunk, steps = kc / 32;
    const uint32_t s0 = steps * kp / kParts, s1 = steps * (kp + 1) / kParts;
    const auto weights = [&](uint32_t a, uint32_t s, f16x8 (&w)[kTogether]) {
      const f16 *p = l.a + ((size_t)a * l.rank + r) * k + k0 + g * 8;
#pragma unroll
      for (uint32_t j = 0; j < kTogether; ++j) {
        const uint32_t at = s + j < s1 ? s + j : s0;  // (past the wave's last step: not used)
        w[j] = *reinterpret_cast<const f16x8 *>(p + at * 32);
      }
    };
    uint64_t who = some;
    uint32_t left = here ? mine : kNoAdapter, a = 0;
    f16x8 w[kTogether];
    if (k0) {
      load_x(k0);
      __syncthreads();  // the chunk before is read
    }
    if (who) {  // on their way while x is taken in
      a = (uint32_t)__builtin_amdgcn_readlane((int)left, __builtin_ctzll(who));
      weights(a, s0, w);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) {
      const uint32_t at = j * 256 + lane * 4;
      *reinterpret_cast<f16x4 *>(xs + wave * kPitch + at * 2) = (f16x4){(f16)v[j].x, (f16)v[j].y, (f16)v[j].z, (f16)v[j].w};
    }
    __syncthreads();
    while (who) {
      f32x4 sum = {};
      for (uint32_t s = s0; s < s1; s += kTogether) {
        if (s != s0) weights(a, s, w);
#pragma unroll
        for (uint32_t j = 0; j < kTogether; ++j)
          if (s + j < s1)
            sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                w[j], *reinterpret_cast<const f16x8 *>(xs + c * kPitch + ((s + j) * 32 + g * 8) * 2), sum, 0, 0, 0);
      }
      const bool its = mine == a;
      if (its) left = kNoAdapter;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = its ? acc[e] + sum[e] : acc[e];
      who = __ballot(left != kNoAdapter);
      if (who) {
        a = (uint32_t)__builtin_amdgcn_readlane((int)left, __builtin_ctzll(who));
        weights(a, s0, w);
      }
    }
    put_x16(k0, kc);
  }
  part[wave][lane] = acc;
  if (threadIdx.x < 16) {
    tops[threadIdx.x] = 0;
    if (m0 + threadIdx.x < m && (here || none)) id[m0 + threadIdx.x] = mine;
  }
  __syncthreads();
  // wave t sums tile t over the parts: lane (g, c) has ranks 16t + 4g .. + 3 of row c
  const uint32_t r0 = wave * 16 + g * 4;
  f32x4 sum = {};
  if (wave < RT) {
#pragma unroll
    for (uint32_t p = 0; p < kParts; ++p) sum += part[p * RT + wave][lane];
    sum *= scale;
    // (ranks come in eights; numbers at least 0 are in the order of their bits)
    float top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = __builtin_fmaxf(top, finite(sum[e]));
    if (r0 < l.rank) atomicMax(&tops[c], __builtin_bit_cast(uint32_t, top));
  }
  __syncthreads();
  if (wave >= RT || m0 + c >= m || !(here || none)) return;
  const int e = exponent_of(__builtin_bit_cast(float, tops[c]));
  if (r0 < l.rank) {
    f16x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f16 u, w;
      halves(sum[i], e, u, w);
      hi[i] = u;
      lo[i] = w;
    }
    const LoraShape shape = lora_shape(l.rank, tile_rows);
    *reinterpret_cast<f16x4 *>(h + lora_at(shape, row, r0, false)) = hi;
    *reinterpret_cast<f16x4 *>(h + lora_at(shape, row, r0, true)) = lo;
  }
  if (wave == 0 && g == 0) factor[row] = mine != kNoAdapter ? __builtin_amdgcn_ldexpf(1.0f, e) : 0.0f;
}

// h, factors and adapters of m rows; x in f16 behind them where there are kX16Rows or more.
// (whole tiles of 32 rows and the most slots that either tile has)
size_t h_rows(uint32_t m) { return ((size_t)m + 31) & ~(size_t)31; }
size_t h_slots(uint32_t rank) { return 2 * (((size_t)rank + 31) & ~(size_t)31); }
size_t h_bytes(uint32_t m, uint32_t rank) { return h_rows(m) * (h_slots(rank) * 2 + 8); }

}  // namespace

extern "C" size_t madi_lora_bytes(uint32_t m, uint32_t k, uint32_t rank) {
  if (rank < 8 || rank > kMaxRank || rank % 8) return 0;
  return h_bytes(m, rank) + (m >= kX16Rows ? (size_t)m * k * 2 : 0);
}

extern "C" int madi_q8_pproj_lora(float *out, const float *in, const void *qs, const void *scales, uint32_t m,
                                  uint32_t n, uint32_t k, const madi_lora *lora) {
  const char *what = "madi_q8_pproj_lora";
  if (!out || !in || !qs || !scales || !lora) return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (m == 0 || n == 0 || k == 0 || k % 64)
    return fail(MADI_ERR_SHAPE, "%s: m=%u n=%u k=%u (need m, n > 0, k a positive multiple of 64)", what, m, n, k);
  if (lora->rank < 8 || lora->rank > kMaxRank || lora->rank % 8)
    return fail(MADI_ERR_SHAPE, "%s: rank %u (a multiple of 8, 8 to 128)", what, lora->rank);
  if (m > 65535 * 32u) return fail(MADI_ERR_SHAPE, "%s: m=%u exceeds %u rows", what, m, 65535 * 32u);
  if ((uint64_t)n * k >= (1ull << 31) || (uint64_t)k * 128 >= (1ull << 31))
    return fail(MADI_ERR_SHAPE, "%s: n=%u k=%u exceeds the 2 GiB operand limit", what, n, k);
  if (lora->adapters > 0x7fffffffu) return fail(MADI_ERR_SHAPE, "%s: %u adapters", what, lora->adapters);
  if (!lora->adapter || !lora->work || (lora->adapters && (!lora->a || !lora->b || !lora->scale)))
    return fail(MADI_ERR_NULL, "%s: null pointer", what);
  if (!aligned(in, 16) || !aligned(qs, 16) || !aligned(scales, 2) || !aligned(out, 4) || !aligned(lora->a, 16) || !aligned(lora->b, 16) || !aligned(lora->work, 16))
    return fail(MADI_ERR_ALIGN, "%s: in, qs, a, b and work need 16-byte alignment", what);
  if (!aligned(lora->scale, 4) || !aligned(lora->adapter, 4) || !aligned(lora->row_seq, 4))
    return fail(MADI_ERR_ALIGN, "%s: arrays must be 4-byte aligned", what);
  const size_t need = madi_lora_bytes(m, k, lora->rank);
  if (lora->work_bytes < need) return fail(MADI_ERR_SHAPE, "%s: %zu bytes of work, needs %zu", what, lora->work_bytes, need);
  const size_t na = lora->adapters, r = lora->rank;
  const Extent x[] = {{in, (size_t)m * k * 4, false}, {qs, (size_t)n * k, false}, {scales, (size_t)n * (k / 32) * 2, false},
                      {lora->a, na * r * k * 2, false}, {lora->b, na * r * n * 2, false}, {lora->scale, na * 4, false},
                      {lora->adapter, (lora->row_seq ? (size_t)lora->seqs : m) * 4, false},
                      {lora->row_seq, lora->row_seq ? (size_t)m * 4 : 0, false},
                      {out, (size_t)m * n * 4, true}, {lora->work, need, true}};
  if (int rc = disjoint(what, x)) return rc;
  if (!initialized()) return fail(MADI_ERR_NOT_INIT, "%s: madi_init has not succeeded", what);
  if (int rc = ready(x)) return rc;
  const Adapters l{(const f16 *)lora->a, lora->scale, lora->adapter, lora->row_seq, lora->adapters, lora->rank, lora->seqs};
  f16 *h = static_cast<f16 *>(lora->work);
  float *factor = reinterpret_cast<float *>(h + h_rows(m) * h_slots(lora->rank));
  uint32_t *id = reinterpret_cast<uint32_t *>(factor + h_rows(m));
  const uint32_t tile_rows = pproj_tile_rows(m, n, k);
  const bool whole = aligned(out, 16) && q8_gemm_x16_suits(m, n, k);
  f16 *x16 = whole ? reinterpret_cast<f16 *>(static_cast<uint8_t *>(lora->work) + h_bytes(m, lora->rank)) : nullptr;
  if (!whole && m <= kRowKernel && k * 2 <= kRowLds) {
    // (10 loads for rows of 4, the rest of them in vain: 8 x 1280 9.7 us instead of 8.0, 128 x 1280 with rank 64 15.4
    // instead of 11.5)
    if (k <= 4 * kStep) lora_row_kernel<4><<<m, 1024, k * 2, stream()>>>(l, in, k, tile_rows, h, factor, id);
    else lora_row_kernel<10><<<m, 1024, k * 2, stream()>>>(l, in, k, tile_rows, h, factor, id);
  } else {
    const auto go = [&](auto kernel) {
      const uint32_t tiles = (m + 15) / 16, of = (uint32_t)cu_count() / tiles;
      kernel<<<dim3(tiles, of < 1 ? 1 : of < 4 ? of : 4), kTileWaves * 64, 0, stream()>>>(l, in, m, k, tile_rows, h, factor, id, x16);
    };
    if (l.rank <= 16) go(lora_tile_kernel<1>);
    else if (l.rank <= 32) go(lora_tile_kernel<2>);
    else if (l.rank <= 64) go(lora_tile_kernel<4>);
    else go(lora_tile_kernel<8>);
  }
  if (int rc = check_launch(what)) return rc;
  const Lora u{h, factor, id, (const f16 *)lora->b, lora->rank, x16};
  return whole ? q8_gemm_x16_lora(qs, scales, out, m, n, k, u) : q8_pproj_lora(out, in, qs, scales, m, n, k, u);
}
