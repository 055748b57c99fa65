// Paged KV cache: rows into pages and back, and the choice of the pages that a
// query reads.
//
// Append and read move each row once and are bound by HBM from some 30 MB on (16,384 rows
// x 32 heads of 128, K and V: fp16 with bounds 537 MB in 101 us, 5.3 TB/s, and 98 us back; int8
// 403 MB in 97 us and 84 us back); below it by the loads that wait for one another (sequence,
// page, row): 32 rows of 8 heads 3.5 us.
#include "paged.h"

namespace rfsn {

int paged_check(const rfsn_paged* p, const char* what) {
  const std::string w(what);
  RFSN_REQUIRE(p != nullptr, w + ": null parameters");
  RFSN_REQUIRE(p->head_dim == 64 || p->head_dim == 128 || p->head_dim == 256, w + ": head_dim must be 64, 128 or 256");
  RFSN_REQUIRE(p->page_size == 16 || p->page_size == 32 || p->page_size == 64 || p->page_size == 128 ||
                   p->page_size == 256,
               w + ": page_size must be 16, 32, 64, 128 or 256");
  RFSN_REQUIRE(p->type == RFSN_PAGE_FP16 || p->type == RFSN_PAGE_INT8 || p->type == RFSN_PAGE_E4M3,
               w + ": unknown page type");
  RFSN_REQUIRE(p->kv_heads > 0 && p->kv_heads <= 65535, w + ": kv_heads out of range");
  RFSN_REQUIRE(p->batch >= 0 && p->batch <= 65535, w + ": batch out of range");
  RFSN_REQUIRE(p->pages > 0, w + ": the pool has no pages");
  RFSN_REQUIRE(p->table_width >= 0 && (int64_t)p->table_width * p->page_size <= (1ll << 31) - 1024,
               w + ": the table's positions must stay below 2^31");
  RFSN_REQUIRE(p->table_width == 0 || p->batch == 0 || p->table != nullptr, w + ": null table");
  RFSN_REQUIRE(p->batch == 0 || p->lens != nullptr, w + ": null lens");
  RFSN_REQUIRE(p->k && p->v && ((uintptr_t)p->k & 15) == 0 && ((uintptr_t)p->v & 15) == 0,
               w + ": k and v must be 16-byte aligned");
  RFSN_REQUIRE(p->head_stride % 16 == 0 && p->page_stride % 16 == 0 &&
                   (p->kv_heads == 1 || p->head_stride >= (int64_t)p->page_size * p->head_dim) && p->page_stride >= 0,
               w + ": page and head strides must be multiples of 16 that leave room for a head's rows");
  RFSN_REQUIRE((p->type == RFSN_PAGE_FP16) == (p->k_scale == nullptr) &&
                   (p->type == RFSN_PAGE_FP16) == (p->v_scale == nullptr),
               w + ": 8-bit pages need both scales, fp16 pages none");
  RFSN_REQUIRE(((uintptr_t)p->bounds & 15) == 0 && ((uintptr_t)p->k_scale & 15) == 0 && ((uintptr_t)p->v_scale & 15) == 0,
               w + ": scales and bounds must be 16-byte aligned");
  return RFSN_OK;
}

namespace {

// Sequence of row n < cu[batch], or -1: the last b with cu[b] <= n.  Memory-safe
// whatever cu holds.
__device__ __forceinline__ int row_sequence(const int32_t* __restrict__ cu, int batch, int64_t n) {
  if (n >= cu[batch] || n < cu[0]) return -1;
  int lo = 0, hi = batch;  // cu[lo] <= n < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (n >= cu[mid]) lo = mid; else hi = mid;
  }
  return lo;
}

struct RowPlace {
  int page;   // of the pool, or -1
  int row;    // in the page
  int count;  // rows of this call in the same page from here on
  bool start; // the first of them
  bool rest;  // behind the last sequence, or before the first
};
// Where a wave's rows go: a lane's row i is n0 + i RS + lane / LANES of the call, RS = 64 / LANES.
// Up to 63 sequences lie in the wave's lanes, so that no load waits for another but the table's.
template <int LANES, int I>
__device__ __forceinline__ void place_rows(const rfsn_paged& p, int shift, const int32_t* __restrict__ cu, int64_t rows,
                                           int64_t n0, int lane, RowPlace (&r)[I]) {
  constexpr int RS = 64 / LANES;
  const int slot = lane / LANES;
  int b[I], len[I];
  int64_t at[I], left[I];
#pragma unroll
  for (int i = 0; i < I; ++i) b[i] = -1, len[i] = 0, at[i] = 0, left[i] = 0;
  if (cu == nullptr) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int64_t n = n0 + i * RS + slot;
      if (n < rows) b[i] = (int)n, left[i] = 1, len[i] = p.lens[n];
    }
  } else if (p.batch > 0 && p.batch < 64) {
    const int c = cu[min(lane, p.batch)], ln = p.lens[min(lane, p.batch - 1)];
    auto bounds_upto = [&](int64_t n) { return (int)__popcll(__ballot(lane <= p.batch && c <= n)); };
    int before[I];  // bounds at or below the lane's rows
    const int x0 = bounds_upto(n0);
#pragma unroll
    for (int i = 0; i < I; ++i) before[i] = x0;
    if (bounds_upto(n0 + I * RS - 1) != x0) {  // rows of several sequences
#pragma unroll
      for (int i = 0; i < I; ++i)
        for (int s = 0; s < RS; ++s) {
          const int x = bounds_upto(n0 + i * RS + s);
          if (s == slot) before[i] = x;
        }
    }
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int64_t n = n0 + i * RS + slot;
      const int seq = min(max(before[i] - 1, 0), p.batch - 1);
      const int64_t c0 = __shfl(c, seq, 64), c1 = __shfl(c, seq + 1, 64);
      len[i] = __shfl(ln, seq, 64);
      if (n < rows && n >= c0 && n < c1) b[i] = seq, at[i] = n - c0, left[i] = (c1 < rows ? c1 : rows) - n;
    }
  } else if (p.batch >= 64) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int64_t n = n0 + i * RS + slot;
      if (n >= rows) continue;
      const int seq = row_sequence(cu, p.batch, n);
      if (seq < 0) continue;
      const int64_t c0 = cu[seq], c1 = cu[seq + 1];
      if (n >= c0 && n < c1) b[i] = seq, at[i] = n - c0, left[i] = (c1 < rows ? c1 : rows) - n, len[i] = p.lens[seq];
    }
  }
#pragma unroll
  for (int i = 0; i < I; ++i) {
    r[i] = {-1, 0, 0, false, true};
    if (b[i] < 0) continue;
    const int64_t pos = (int64_t)max(len[i], 0) + at[i];
    r[i].rest = false;
    r[i].page = paged_page(p, b[i], pos >> shift);
    r[i].row = (int)(pos & (p.page_size - 1));
    r[i].count = (int)(left[i] < p.page_size - r[i].row ? left[i] : p.page_size - r[i].row);
    r[i].start = at[i] == 0 || r[i].row == 0;
  }
}

typedef unsigned short ushort8v __attribute__((ext_vector_type(8)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
typedef unsigned short ushort4v __attribute__((ext_vector_type(4)));

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_top(uint32_t x) {
  const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 15, 15, true);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, x), __builtin_bit_cast(ushort2v, y)));
}
// The largest |x| of a K and a V row as bits, K's in the low half: infinity and NaN are the largest.
template <int LANES>
__device__ __forceinline__ uint32_t row_tops(half8v k, half8v v) {
  const ushort8v a = __builtin_bit_cast(ushort8v, k) & (unsigned short)0x7fff;
  const ushort8v b = __builtin_bit_cast(ushort8v, v) & (unsigned short)0x7fff;
  const ushort4v a4 = __builtin_elementwise_max(a.lo, a.hi), b4 = __builtin_elementwise_max(b.lo, b.hi);
  const ushort2v a2 = __builtin_elementwise_max(a4.lo, a4.hi), b2 = __builtin_elementwise_max(b4.lo, b4.hi);
  const ushort2v even = {a2[0], b2[0]}, odd = {a2[1], b2[1]};
  uint32_t t = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(even, odd));
  t = dpp_top<0xb1>(t);   // lanes ^ 1, ^ 2, then mirrored halves of 8 and rows of 16
  t = dpp_top<0x4e>(t);
  t = dpp_top<0x141>(t);
  if constexpr (LANES >= 16) t = dpp_top<0x140>(t);
  if constexpr (LANES >= 32) {
    const uint32_t y = (uint32_t)__shfl_xor((int)t, 16, 64);
    t = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, t), __builtin_bit_cast(ushort2v, y)));
  }
  return t;
}

// 8 values of a row as codes, by the row's largest magnitude: one fp32 product, then
// the code's own rounding.  A row that is not finite: codes 0, scale NaN.
template <int TYPE>
__device__ __forceinline__ uint2v quantise(half8v x, uint32_t top, float& scale) {
  constexpr float kTop = TYPE == RFSN_PAGE_INT8 ? 127.f : 448.f;
  const bool finite = top < 0x7c00u;
  const float amax = h2f((uint16_t)top);
  scale = finite ? amax / kTop : __builtin_nanf("");
  const float inv = top ? kTop / amax : 0.f;
  uint2v c;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (float)x[4 * w + e] * inv;
    if constexpr (TYPE == RFSN_PAGE_INT8) {
      uint32_t u[4];  // 1.5 2^23 + y rounds y to the nearest integer, which its low byte then is
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = __builtin_bit_cast(uint32_t, y[e] + 12582912.f);
      const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
      c[w] = lo | hi;
    } else {
      const int q = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      c[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], q, true);
    }
    if (!finite) c[w] = 0;
  }
  return c;
}

// Smallest and largest keys of 8 coordinates, and their largest magnitude's bits, which are past infinity's where one is NaN.
struct Bounds {
  half8v lo, hi;
  ushort8v top;
  __device__ __forceinline__ void add(half8v x) {
    lo = __builtin_elementwise_min(lo, x), hi = __builtin_elementwise_max(hi, x);
    top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort8v, x) & (unsigned short)0x7fff);
  }
  // what a page holds already
  __device__ __forceinline__ void add(half8v l, half8v h) { add(l), add(h); }
  __device__ __forceinline__ void across(int o) {  // with the lanes o apart
    const uint4w l = __builtin_bit_cast(uint4w, lo), h = __builtin_bit_cast(uint4w, hi), t = __builtin_bit_cast(uint4w, top);
    uint4w l2, h2, t2;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      l2[w] = (uint32_t)__shfl_xor((int)l[w], o, 64);
      h2[w] = (uint32_t)__shfl_xor((int)h[w], o, 64);
      t2[w] = (uint32_t)__shfl_xor((int)t[w], o, 64);
    }
    lo = __builtin_elementwise_min(lo, __builtin_bit_cast(half8v, l2));
    hi = __builtin_elementwise_max(hi, __builtin_bit_cast(half8v, h2));
    top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort8v, t2));
  }
  __device__ __forceinline__ void store(half8v* l, half8v* h) const {
    ushort8v a = __builtin_bit_cast(ushort8v, lo), b = __builtin_bit_cast(ushort8v, hi);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (top[e] > 0x7c00) a[e] = b[e] = 0x7e00;
    *l = __builtin_bit_cast(half8v, a), *h = __builtin_bit_cast(half8v, b);
  }
};
__device__ __forceinline__ Bounds bounds_of(half8v x) {
  return {x, x, __builtin_bit_cast(ushort8v, x) & (unsigned short)0x7fff};
}

// Block number of a grid of x by y blocks so that each XCD takes a contiguous range of
// them (hardware deals consecutive blocks to the 8 XCDs in turn).
__device__ __forceinline__ uint2 xcd_block() {
  const uint32_t i = blockIdx.y * gridDim.x + blockIdx.x, all = gridDim.x * gridDim.y;
  const uint32_t x = i & 7, each = all >> 3, more = all & 7;
  const uint32_t g = x * each + min(x, more) + (i >> 3);
  return make_uint2(g % gridDim.x, g / gridDim.x);
}

// Long appends pass the caches by: with 8,191 rows of 8 heads of 64 they take 9.7 us against 11.0, and 22.7
// with the attention of a token behind them against 23.3; 2,048 rows, which attention finds in the
// caches, 4.8 against 5.0 alone and 20.7 against 19.2 with it.  (V was loaded through them then.)
template <bool PASS, typename V>
__device__ __forceinline__ void store_page(V x, V* at) {
  if constexpr (PASS) __builtin_nontemporal_store(x, at);
  else *at = x;
}

// A wave writes I RS rows of one head, K and V, RS = 64 / (D / 8); a lane holds 8
// coordinates of a row.  Bounds: the wave of a run's first row (rows of one
// sequence in one page) takes those of the run's keys that it holds and reads the others, and
// writes the page's bounds, so no two waves write the same ones and no order changes them.  Bounds
// take 2 us of 101 for 16,384 x 32 x 128 in fp16, 14 of 97 in int8, 1.8 of 8.4 for 8,191 x 8 x 64.
// V, which no other wave reads, is loaded past the caches in rows of 64 (32,768 x 8: fp16 30.7 -> 28.3 us, int8
// 29.4 -> 27.7, e4m3 29.2 -> 27.4; 65,536 x 32: 202 alike, 173 -> 171, 173 -> 172; 5,000 to 16,384 x 8 lose or gain 1 %:
// 8,191 fp16 9.15 -> 9.10, int8 10.5 -> 10.6; 8,192 x 8 rows of 128 or more lose 1 %: 16.3 -> 16.5).
template <int D, int TYPE, int I>
__global__ void __launch_bounds__(256)
paged_append_kernel(const rfsn_paged p, int shift, const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                    int64_t ts, int64_t hs, int64_t rows, const int32_t* __restrict__ cu) {
  constexpr int LANES = D / 8, RS = 64 / LANES, R = I * RS, U = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint2 block = xcd_block();  // the rows of a run are in the L2 of the wave that reads them for its bounds
  const int h = block.y * 4 + wave;
  if (h >= p.kv_heads) return;
  const int slot = lane / LANES, chunk = lane % LANES;
  const int64_t n0 = (int64_t)block.x * R;
  const uint16_t* const kh = k + h * hs + chunk * 8;
  const uint16_t* const vh = v + h * hs + chunk * 8;
  half8v kx[I], vx[I];
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int64_t n = n0 + i * RS + slot < rows ? n0 + i * RS + slot : rows - 1;
    kx[i] = *reinterpret_cast<const half8v*>(kh + n * ts);
    if constexpr (I > 1 && D == 64) vx[i] = __builtin_nontemporal_load(reinterpret_cast<const half8v*>(vh + n * ts));
    else vx[i] = *reinterpret_cast<const half8v*>(vh + n * ts);
  }
  RowPlace at[I];
  place_rows<LANES, I>(p, shift, cu, rows, n0, lane, at);
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const bool write = at[i].page >= 0;
    const int64_t off = (int64_t)(write ? at[i].page : 0) * p.page_stride + h * p.head_stride + (int64_t)at[i].row * D + chunk * 8;
    if constexpr (TYPE == RFSN_PAGE_FP16) {
      if (write) {
        store_page<(I > 1)>(kx[i], (half8v*)((uint16_t*)p.k + off));
        store_page<(I > 1)>(vx[i], (half8v*)((uint16_t*)p.v + off));
      }
    } else {
      const int64_t sc = ((int64_t)(write ? at[i].page : 0) * p.kv_heads + h) * p.page_size + at[i].row;
      const uint32_t tops = row_tops<LANES>(kx[i], vx[i]);
      float ks, vs;
      const uint2v kc = quantise<TYPE>(kx[i], tops & 0xffffu, ks), vc = quantise<TYPE>(vx[i], tops >> 16, vs);
      if (write) {
        store_page<(I > 1)>(kc, (uint2v*)((uint8_t*)p.k + off));
        store_page<(I > 1)>(vc, (uint2v*)((uint8_t*)p.v + off));
        if (chunk == 0) p.k_scale[sc] = ks, p.v_scale[sc] = vs;
      }
    }
  }
  if (p.bounds == nullptr) return;
  auto bounds_at = [&](int page) {
    return reinterpret_cast<half8v*>((uint16_t*)p.bounds + ((int64_t)page * p.kv_heads + h) * 2 * D + chunk * 8);
  };
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const bool leads = at[i].page >= 0 && at[i].start;
    // runs of one row: each row slot on its own; longer ones by the whole wave
    if (leads && at[i].count == 1) {
      half8v* bp = bounds_at(at[i].page);
      Bounds m = bounds_of(kx[i]);
      if (at[i].row > 0) m.add(bp[0], bp[D / 8]);
      m.store(bp, bp + D / 8);
    }
    uint64_t todo = __ballot(leads && at[i].count > 1);
    while (todo) {
      const int src = __ffsll((unsigned long long)todo) - 1;  // a lane of the run's first row
      todo &= ~(((1ull << LANES) - 1) << (src / LANES * LANES));
      const int page = __builtin_amdgcn_readlane(at[i].page, src), row = __builtin_amdgcn_readlane(at[i].row, src);
      const int count = __builtin_amdgcn_readlane(at[i].count, src);
      const int r0 = i * RS + src / LANES, r1 = r0 + count;  // the run's rows, from the wave's first
      half8v* bp = bounds_at(page);
      Bounds m = bounds_of(kx[i]);  // a lane whose row is not the run's takes the run's first instead
      if (i * RS + slot < r0 || i * RS + slot >= r1) m = bounds_of(*reinterpret_cast<const half8v*>(kh + (n0 + r0) * ts));
      if (row > 0) m.add(bp[0], bp[D / 8]);
#pragma unroll
      for (int j = i + 1; j < I; ++j)
        if (j * RS + slot < r1) m.add(kx[j]);
      for (int j = R + slot; j - slot < r1; j += U * RS) {
        half8v x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const half8v*>(kh + (n0 + min(j + u * RS, r1 - 1)) * ts);
#pragma unroll
        for (int u = 0; u < U; ++u) m.add(x[u]);
      }
#pragma unroll
      for (int o = LANES; o < 64; o <<= 1) m.across(o);
      if (slot == 0) m.store(bp, bp + D / 8);
    }
  }
}

// The reverse, RS rows to a wave.  Four sets of rows per wave are slower at every size
// (8 heads of 64, fp16: 512 rows 3.5 us against 2.5, 8,192 rows 7.9 against 7.1; 16,384 rows x 32 heads of 128:
// 128 against 124): nothing is read twice here, and fewer waves wait for their table entry.
// Blocks in XCD ranges read a page's head in one L2 (16,384 rows x 32 heads of 128: 124 -> 99 us).
// Non-temporal stores would take 7 % more off the read alone and cost the attention that takes the
// rows from the caches more (8,191 rows read and attended by 128 queries: 36.8 us against 38.9).
template <int D, int TYPE>
__global__ void __launch_bounds__(256)
paged_read_kernel(const rfsn_paged p, int shift, const int32_t* __restrict__ cu, int64_t rows,
                  uint16_t* __restrict__ out_k, uint16_t* __restrict__ out_v, int zero_rest) {
  constexpr int LANES = D / 8, RS = 64 / LANES;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint2 block = xcd_block();
  const int h = block.y * 4 + wave;
  if (h >= p.kv_heads) return;
  const int slot = lane / LANES, chunk = lane % LANES;
  const int64_t n = (int64_t)block.x * RS + slot;
  RowPlace place[1];
  place_rows<LANES, 1>(p, shift, cu, rows, (int64_t)block.x * RS, lane, place);
  const RowPlace at = place[0];
  if (n >= rows || (at.rest && !zero_rest)) return;
  half8v ko = {}, vo = {};
  if (at.page >= 0) {
    const int64_t off = (int64_t)at.page * p.page_stride + h * p.head_stride + (int64_t)at.row * D + chunk * 8;
    if constexpr (TYPE == RFSN_PAGE_FP16) {
      ko = *reinterpret_cast<const half8v*>((const uint16_t*)p.k + off);
      vo = *reinterpret_cast<const half8v*>((const uint16_t*)p.v + off);
    } else {
      const int64_t sc = ((int64_t)at.page * p.kv_heads + h) * p.page_size + at.row;
      const float ks = p.k_scale[sc], vs = p.v_scale[sc];
      const float8v kf = load_page8<TYPE>(p.k, off), vf = load_page8<TYPE>(p.v, off);
#pragma unroll
      for (int e = 0; e < 8; ++e) ko[e] = (f16)(kf[e] * ks), vo[e] = (f16)(vf[e] * vs);
    }
  }
  const int64_t o = (n * p.kv_heads + h) * D + chunk * 8;
  *reinterpret_cast<half8v*>(out_k + o) = ko;
  *reinterpret_cast<half8v*>(out_v + o) = vo;
}

// ---------------------------------------------------------------- page choice

// x + the value of the lane that `ctrl` (a DPP pattern) names.
template <int CTRL>
__device__ __forceinline__ double dpp_add(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, 15, 15, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 15, 15, true);
  return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum over groups of 8, 16 or 32 lanes: lanes ^ 1, ^ 2, then mirrored halves of 8 and rows of 16.
template <int LANES>
__device__ __forceinline__ double group_sum(double x) {
  x = dpp_add<0xb1>(x);   // quad_perm 1,0,3,2
  x = dpp_add<0x4e>(x);   // quad_perm 2,3,0,1
  x = dpp_add<0x141>(x);  // row_half_mirror
  if constexpr (LANES >= 16) x = dpp_add<0x140>(x);  // row_mirror
  if constexpr (LANES >= 32) x += __shfl_xor(x, 16, 64);
  return x;
}

// Score of every page held by (sequence, KV head): a lane takes 8 coordinates of a page's
// bounds, D / 8 lanes a page, a wave U sets of pages, whose loads are all in flight together.
// Sums are held in 64 bits; the bounds are converted once for all query heads, which leaves two
// fused multiply-adds per coordinate and head.  2,048 pages x 4 KV heads of 64, 8 query heads each:
// 5.3 us, latency; 32 x 2,048 pages x 8 KV heads, 4 query heads: 44 us for 134 MB, 63 % of the copy rate, with vector
// instructions in some 60 % of the SIMDs' issue cycles; 32 ragged sequences of up to 2,048 pages: 11.8 us for 17 MB,
// a third of them, and waves that wait in 56 % of their cycles.
constexpr int kScoreSets = 2;
template <int D>
__global__ void __launch_bounds__(256)
page_score_kernel(const rfsn_paged p, int shift, const uint16_t* __restrict__ q, int G, float* __restrict__ score) {
  constexpr int LANES = D / 8, RS = 64 / LANES, U = kScoreSets;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int PER = 4 * RS * U;  // pages of a block's round
  const int h = blockIdx.y;
  const int slot = lane / LANES, chunk = lane % LANES;
  auto rounds = [&](int b) {
    return b < p.batch ? (uint32_t)((((int64_t)paged_len(p, shift, b) + p.page_size - 1 >> shift) + PER - 1) / PER) : 0u;
  };
  const uint32_t n_first = rounds(lane), upto_first = wave_upto(n_first);  // of the first 64 sequences
#pragma unroll 1
  for (uint32_t item = blockIdx.x;; item += gridDim.x) {
    // the item's sequence and round
    int b = -1;
    uint32_t x = 0, seen = 0;
    for (int base = 0; base < p.batch; base += 64) {
      const uint32_t n = base ? rounds(base + lane) : n_first, upto = base ? wave_upto(n) : upto_first;
      const uint64_t in = __ballot(item < seen + upto);
      if (in) {
        const int src = __ffsll((unsigned long long)in) - 1;
        b = base + src;
        x = item - seen - (uint32_t)__builtin_amdgcn_readlane((int)upto, src) + (uint32_t)__builtin_amdgcn_readlane((int)n, src);
        break;
      }
      seen += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
    if (b < 0) return;
    const int held = (int)(((int64_t)paged_len(p, shift, b) + p.page_size - 1) >> shift);
    const int n0 = (int)(x * PER) + wave * (RS * U) + slot;
    if (n0 - slot >= held) continue;
    const uint16_t* const qh = q + ((int64_t)b * p.kv_heads + h) * G * D + chunk * 8;
    half8v qv = *reinterpret_cast<const half8v*>(qh);
    int page[U];
#pragma unroll
    for (int u = 0; u < U; ++u) page[u] = n0 + u * RS < held ? paged_page(p, b, n0 + u * RS) : -1;
    half8v lo[U], hi[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const half8v* bp = reinterpret_cast<const half8v*>(
          (const uint16_t*)p.bounds + ((int64_t)max(page[u], 0) * p.kv_heads + h) * 2 * D + chunk * 8);
      lo[u] = bp[0], hi[u] = bp[D / 8];
    }
    // max(q, 0) hi + min(q, 0) lo = q (hi + lo) / 2 + |q| (hi - lo) / 2: a product with q and one with |q|,
    // which needs no second copy of q; half sums and half differences of fp16 values are exact in 64 bits
    double mid[U][8], half[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double x = (double)lo[u][e], y = (double)hi[u][e];
        mid[u][e] = (y + x) * 0.5, half[u][e] = (y - x) * 0.5;
      }
    double best[U];
    bool nan[U];
#pragma unroll
    for (int u = 0; u < U; ++u) best[u] = -__builtin_inf(), nan[u] = false;
#pragma unroll 1
    for (int g = 0; g < G; ++g) {
      double x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (double)qv[e];
      qv = *reinterpret_cast<const half8v*>(qh + (int64_t)min(g + 1, G - 1) * D);  // the next head's
#pragma unroll
      for (int u = 0; u < U; ++u) {
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_fma(x[e], mid[u][e], __builtin_fma(__builtin_fabs(x[e]), half[u][e], s));
        s = group_sum<LANES>(s);
        nan[u] |= s != s;
        best[u] = s > best[u] ? s : best[u];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = n0 + u * RS;
      if (n < held && chunk == 0)
        score[((int64_t)b * p.kv_heads + h) * p.table_width + n] =
            page[u] < 0 ? -__builtin_inff() : nan[u] ? __builtin_nanf("") : (float)best[u];
    }
  }
}

// Order of the scores as unsigned keys: NaN as +infinity, -0 as +0.
__device__ __forceinline__ uint32_t page_key(float s) {
  if (s != s) s = __builtin_inff();
  const uint32_t u = __builtin_bit_cast(uint32_t, s + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

// The pages of a row's largest keys besides the kept ones, all in ascending order.  A block a row.
// The smallest key to keep is found by narrowing [lo, hi], at first the smallest and largest key: a histogram of
// 2,048 equal parts of it says which part holds the key wanted.  Scores share their exponent mostly, so parts
// of their range spread over the counters where their leading bits would meet in one; two rounds are the rule,
// three the most (leading bits as counters: 50 us for 128 of 2,048 pages, 256 rows; so 6.3, latency of
// some ten block barriers).  Then each of 16 waves counts what it keeps of its own run of pages and writes it
// behind the waves before it.  Keys past the LDS copy are read again from the scores.
constexpr int kChooseWaves = 16, kChooseBins = 2048, kChooseKeys = 8192;
__global__ void __launch_bounds__(kChooseWaves * 64)
page_choose_kernel(const rfsn_paged p, int shift, const float* __restrict__ score, int count, int first, int last,
                   int32_t* __restrict__ chosen) {
  constexpr int T = kChooseWaves * 64, PER = kChooseBins / T;
  __shared__ uint32_t s_key[kChooseKeys];
  __shared__ uint32_t hist[kChooseBins];
  __shared__ uint32_t s_wave[2][kChooseWaves], s_found[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.x, b = blockIdx.y;
  const int64_t row = (int64_t)b * p.kv_heads + h;
  const float* s = score + row * p.table_width;
  int32_t* out = chosen + row * count;
  const int held = (int)(((int64_t)paged_len(p, shift, b) + p.page_size - 1) >> shift);
  if (held <= count) {
    for (int i = tid; i < count; i += T) out[i] = i < held ? i : -1;
    return;
  }
  // held > count >= first + last: the kept pages are apart, the others lie between them
  const int begin = first, end = held - last;
  uint32_t left = (uint32_t)(count - first - last);
  auto key = [&](int n) { return n - begin < kChooseKeys ? s_key[n - begin] : page_key(s[n]); };
  uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll 4
  for (int n = begin + tid; n < end; n += T) {
    const uint32_t k = page_key(s[n]);
    if (n - begin < kChooseKeys) s_key[n - begin] = k;
    lo = min(lo, k), hi = max(hi, k);
  }
  lo = ~wave_most(~lo), hi = wave_most(hi);
  if (lane == 0) s_wave[0][wave] = lo, s_wave[1][wave] = hi;
  __syncthreads();
  lo = ~wave_most(lane < kChooseWaves ? ~s_wave[0][lane] : 0u), hi = wave_most(lane < kChooseWaves ? s_wave[1][lane] : 0u);
  // what the waves before this one have of s_wave[i]
  auto before_wave = [&](int i) { return wave_total(lane < wave ? s_wave[i][lane] : 0u); };
  uint32_t over = 0xffffffffu, tie = 0xffffffffu;  // keys from `over` on are kept, and `left` of those equal to `tie`
  while (left > 0) {
    if (lo == hi) {
      over = lo + 1, tie = lo;
      break;
    }
    const int bits = 32 - __builtin_clz(hi - lo), sh = bits > 11 ? bits - 11 : 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) hist[tid + i * T] = 0;
    __syncthreads();
    for (int n = begin + tid; n < end; n += T) {
      const uint32_t k = key(n);
      if (k >= lo && k <= hi) atomicAdd(&hist[(k - lo) >> sh], 1u);
    }
    __syncthreads();
    // keys in the parts above each thread's PER parts, from the top down
    uint32_t c[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) mine += c[i] = hist[kChooseBins - 1 - (tid * PER + i)];
    const uint32_t upto = wave_upto(mine);
    if (lane == 63) s_wave[0][wave] = upto;
    __syncthreads();
    uint32_t above = upto - mine + before_wave(0);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (above < left && above + c[i] >= left) {
        s_found[0] = (uint32_t)(kChooseBins - 1 - (tid * PER + i));
        s_found[1] = left - above;
        s_found[2] = c[i];
      }
      above += c[i];
    }
    __syncthreads();
    lo += s_found[0] << sh;
    hi = min(hi, lo + ((1u << sh) - 1u));
    left = s_found[1];
    if (s_found[2] == left) {  // the whole part
      over = lo, left = 0;
    }
  }
  __syncthreads();  // s_wave is written again
  const int seg = ((end - begin + kChooseWaves - 1) / kChooseWaves + 63) / 64 * 64;
  const int n0 = begin + wave * seg, n1 = min(end, n0 + seg);
  uint32_t kept = 0, ties = 0;
  for (int n = n0 + lane; n - lane < n1; n += 64) {
    const uint32_t k = n < n1 ? key(n) : 0;
    kept += (uint32_t)__popcll(__ballot(n < n1 && k >= over));
    ties += (uint32_t)__popcll(__ballot(n < n1 && left && k == tie));
  }
  if (lane == 0) s_wave[0][wave] = kept, s_wave[1][wave] = ties;
  __syncthreads();
  uint32_t before = before_wave(1), at = (uint32_t)first + before_wave(0);
  at += min(before, left);
  const uint64_t below = (1ull << lane) - 1;
  for (int n = n0 + lane; n - lane < n1; n += 64) {
    const uint32_t k = n < n1 ? key(n) : 0;
    const bool is_tie = n < n1 && left && k == tie;
    const uint64_t bt = __ballot(is_tie);
    const bool keep = (n < n1 && k >= over) || (is_tie && before + (uint32_t)__popcll(bt & below) < left);
    const uint64_t bk = __ballot(keep);
    if (keep) out[at + (uint32_t)__popcll(bk & below)] = n;
    at += (uint32_t)__popcll(bk), before += (uint32_t)__popcll(bt);
  }
  for (int i = tid; i < first; i += T) out[i] = i;
  for (int i = tid; i < last; i += T) out[count - last + i] = end + i;
}

#define RFSN_PAGED_DISPATCH(D, TYPE, ...)                                                       \
  do {                                                                                          \
    if (D == 64 && TYPE == RFSN_PAGE_FP16) { constexpr int DD = 64, TT = RFSN_PAGE_FP16; __VA_ARGS__ }        \
    else if (D == 64 && TYPE == RFSN_PAGE_INT8) { constexpr int DD = 64, TT = RFSN_PAGE_INT8; __VA_ARGS__ }   \
    else if (D == 64) { constexpr int DD = 64, TT = RFSN_PAGE_E4M3; __VA_ARGS__ }                             \
    else if (D == 128 && TYPE == RFSN_PAGE_FP16) { constexpr int DD = 128, TT = RFSN_PAGE_FP16; __VA_ARGS__ } \
    else if (D == 128 && TYPE == RFSN_PAGE_INT8) { constexpr int DD = 128, TT = RFSN_PAGE_INT8; __VA_ARGS__ } \
    else if (D == 128) { constexpr int DD = 128, TT = RFSN_PAGE_E4M3; __VA_ARGS__ }                           \
    else if (TYPE == RFSN_PAGE_FP16) { constexpr int DD = 256, TT = RFSN_PAGE_FP16; __VA_ARGS__ }             \
    else if (TYPE == RFSN_PAGE_INT8) { constexpr int DD = 256, TT = RFSN_PAGE_INT8; __VA_ARGS__ }             \
    else { constexpr int DD = 256, TT = RFSN_PAGE_E4M3; __VA_ARGS__ }                                         \
  } while (0)

}  // namespace
}  // namespace rfsn

using namespace rfsn;

extern "C" int rfsn_paged_append(const rfsn_paged* p, const void* k, const void* v, int64_t token_stride,
                                 int64_t head_stride, int64_t rows, const int32_t* cu, void* stream) {
  if (int st = paged_check(p, "paged_append")) return st;
  RFSN_REQUIRE(rows >= 0, "paged_append: negative row count");
  RFSN_REQUIRE(cu != nullptr || rows == p->batch, "paged_append: without cu there is one row per sequence");
  if (rows == 0 || p->batch == 0) return RFSN_OK;
  RFSN_REQUIRE(k && v && ((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0 && token_stride % 8 == 0 &&
                   head_stride % 8 == 0,
               "paged_append: k and v rows must be 16-byte aligned");
  const int rs = 512 / p->head_dim;
  RFSN_REQUIRE(ceil_div(rows, rs) < (1ll << 24) && ceil_div(rows, rs) * ceil_div(p->kv_heads, 4) < (1ll << 31),
               "paged_append: too many rows");
  const int shift = paged_shift(*p);
  // Four sets of rows per wave hold most of their pages' rows and read few again for the
  // bounds, but leave fewer waves.  With both storing alike, 8 heads of 64, fp16 pages of 16: 512 rows (512 sets) 6.0 us
  // against 4.1, 4,096 rows 7.1 against 7.3 (int8 7.9 against 7.4), 8,192 rows 11.1 against 11.8;
  // 16,384 rows x 32 heads of 128: 107 us against 135.
  const bool four = ceil_div(rows, rs) * p->kv_heads > 4096;
  const dim3 grid((unsigned)ceil_div(rows, four ? 4 * rs : rs), (unsigned)ceil_div(p->kv_heads, 4));
  RFSN_PAGED_DISPATCH(p->head_dim, p->type, {
    if (four)
      hipLaunchKernelGGL((paged_append_kernel<DD, TT, 4>), grid, dim3(256), 0, (hipStream_t)stream, *p, shift,
                         (const uint16_t*)k, (const uint16_t*)v, token_stride, head_stride, rows, cu);
    else
      hipLaunchKernelGGL((paged_append_kernel<DD, TT, 1>), grid, dim3(256), 0, (hipStream_t)stream, *p, shift,
                         (const uint16_t*)k, (const uint16_t*)v, token_stride, head_stride, rows, cu);
  });
  return check_launch("paged_append");
}

extern "C" int rfsn_paged_read(const rfsn_paged* p, const int32_t* cu, int64_t rows, void* out_k, void* out_v,
                               int32_t zero_rest, void* stream) {
  if (int st = paged_check(p, "paged_read")) return st;
  RFSN_REQUIRE(rows >= 0, "paged_read: negative row count");
  if (rows == 0) return RFSN_OK;
  RFSN_REQUIRE(cu != nullptr, "paged_read: null cu");
  RFSN_REQUIRE(out_k && out_v && ((uintptr_t)out_k & 15) == 0 && ((uintptr_t)out_v & 15) == 0,
               "paged_read: outputs must be 16-byte aligned");
  const int rs = 512 / p->head_dim;
  RFSN_REQUIRE(ceil_div(rows, rs) < (1ll << 24) && ceil_div(rows, rs) * ceil_div(p->kv_heads, 4) < (1ll << 31),
               "paged_read: too many rows");
  const int shift = paged_shift(*p);
  const dim3 grid((unsigned)ceil_div(rows, rs), (unsigned)ceil_div(p->kv_heads, 4));
  RFSN_PAGED_DISPATCH(p->head_dim, p->type, {
    hipLaunchKernelGGL((paged_read_kernel<DD, TT>), grid, dim3(256), 0, (hipStream_t)stream, *p, shift, cu, rows,
                       (uint16_t*)out_k, (uint16_t*)out_v, zero_rest);
  });
  return check_launch("paged_read");
}

extern "C" size_t rfsn_page_select_workspace_bytes(const rfsn_paged* p) {
  if (p == nullptr || p->batch <= 0 || p->kv_heads <= 0 || p->table_width <= 0) return 0;
  return (size_t)p->batch * p->kv_heads * p->table_width * sizeof(float);
}

extern "C" int rfsn_page_select(const rfsn_paged* p, const void* q, int32_t q_heads, int32_t count, int32_t first,
                                int32_t last, int32_t* chosen, void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = paged_check(p, "page_select")) return st;
  RFSN_REQUIRE(p->bounds != nullptr, "page_select: the pages hold no bounds");
  RFSN_REQUIRE(q_heads > 0 && q_heads % p->kv_heads == 0, "page_select: q_heads must be a multiple of kv_heads");
  RFSN_REQUIRE(count > 0 && first >= 0 && last >= 0 && (int64_t)first + last <= count,
               "page_select: count must be positive and have room for the first and last pages");
  RFSN_REQUIRE((int64_t)count * p->page_size <= (1ll << 31) - 1024, "page_select: too many pages");
  if (p->batch == 0) return RFSN_OK;
  RFSN_REQUIRE(q && ((uintptr_t)q & 15) == 0 && chosen, "page_select: null or misaligned q, or null output");
  RFSN_REQUIRE(workspace_bytes >= rfsn_page_select_workspace_bytes(p) && (workspace || p->table_width == 0),
               "page_select: workspace too small");
  const int shift = paged_shift(*p);
  const hipStream_t s = (hipStream_t)stream;
  const int G = q_heads / p->kv_heads;
  if (p->table_width > 0) {
    const int per = 4 * kScoreSets * (512 / p->head_dim);
    // Blocks take the rounds of all sequences in turn: a block for each that the table's width allows would
    // mostly find nothing (32 ragged sequences of up to 2,048 pages: 8,448 blocks, 17.3 us against 12.3).
    int64_t across = ceil_div(p->table_width, per) * p->batch;
    if (across > ceil_div(2048, p->kv_heads)) across = ceil_div(2048, p->kv_heads);
    const dim3 grid((unsigned)across, (unsigned)p->kv_heads);
#define RFSN_SCORE(DD) \
  hipLaunchKernelGGL(page_score_kernel<DD>, grid, dim3(256), 0, s, *p, shift, (const uint16_t*)q, G, (float*)workspace)
    if (p->head_dim == 64) RFSN_SCORE(64);
    else if (p->head_dim == 128) RFSN_SCORE(128);
    else RFSN_SCORE(256);
#undef RFSN_SCORE
    if (int st = check_launch("page_select")) return st;
  }
  hipLaunchKernelGGL(page_choose_kernel, dim3((unsigned)p->kv_heads, (unsigned)p->batch), dim3(kChooseWaves * 64), 0, s, *p,
                     shift, (const float*)workspace, count, first, last, chosen);
  return check_launch("page_select");
}
