// Paged KV cache: rows into pages and back, and the choice of the pages that a
// query reads.
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
// Where the lanes' rows go: row n0 + lane / LANES of the call, one wave, n0 the wave's.
// Up to 63 sequences lie in the wave's lanes, so that no load waits for another but the table's.
template <int LANES>
__device__ __forceinline__ RowPlace row_place(const rfsn_paged& p, int shift, const int32_t* __restrict__ cu,
                                              int64_t rows, int64_t n0, int lane) {
  const int64_t n = n0 + lane / LANES;
  RowPlace r = {-1, 0, 0, false, true};
  int64_t i = 0, left = 0;
  int b = -1, len = 0;
  if (cu == nullptr) {
    if (n < rows) b = (int)n, left = 1, len = p.lens[b];
  } else if (p.batch > 0 && p.batch < 64) {
    const int c = cu[min(lane, p.batch)], ln = p.lens[min(lane, p.batch - 1)];
    int before = 0;  // bounds at or below the lane's row
#pragma unroll
    for (int s = 0; s < 64 / LANES; ++s) {
      const int x = (int)__popcll(__ballot(lane <= p.batch && c <= n0 + s));
      if (s == lane / LANES) before = x;
    }
    const int at = min(max(before - 1, 0), p.batch - 1);
    const int64_t c0 = __shfl(c, at, 64), c1 = __shfl(c, at + 1, 64);
    len = __shfl(ln, at, 64);
    if (n < rows && n >= c0 && n < c1) b = at, i = n - c0, left = (c1 < rows ? c1 : rows) - n;
  } else if (p.batch >= 64 && n < rows) {
    b = row_sequence(cu, p.batch, n);
    if (b >= 0) {
      i = n - cu[b];
      left = (cu[b + 1] < rows ? cu[b + 1] : rows) - n;
      len = p.lens[b];
      if (i < 0 || left <= 0) b = -1;  // no prefix
    }
  }
  if (b < 0) return r;
  const int64_t pos = (int64_t)max(len, 0) + i;
  r.rest = false;
  r.page = paged_page(p, b, pos >> shift);
  r.row = (int)(pos & (p.page_size - 1));
  r.count = (int)(left < p.page_size - r.row ? left : p.page_size - r.row);
  r.start = i == 0 || r.row == 0;
  return r;
}

// A row's values by the row's largest: rounding is one fp32 product, then the code's own.
template <int TYPE, int LANES>
__device__ __forceinline__ void store_row(const rfsn_paged& p, void* base, float* scales, int64_t off, int64_t scale_at,
                                          half8v x, int chunk, bool write) {
  if constexpr (TYPE == RFSN_PAGE_FP16) {
    if (write) *reinterpret_cast<half8v*>((uint16_t*)base + off) = x;
  } else {
    uint32_t top = 0;  // |x| as bits: infinity and NaN are the largest
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, (uint32_t)__builtin_bit_cast(uint16_t, (f16)x[e]) & 0x7fffu);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    constexpr float kTop = TYPE == RFSN_PAGE_INT8 ? 127.f : 448.f;
    const bool finite = top < 0x7c00u;
    const float amax = h2f((uint16_t)top);
    const float scale = finite ? amax / kTop : __builtin_nanf("");
    const float inv = finite && top ? kTop / amax : 0.f;
    uint2v c;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = finite ? (float)x[4 * w + e] * inv : 0.f;
      if constexpr (TYPE == RFSN_PAGE_INT8) {
        c[w] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) c[w] |= ((uint32_t)(int)rintf(y[e]) & 255u) << (8 * e);
      } else {
        int q = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        c[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], q, true);
      }
    }
    if (write) {
      *reinterpret_cast<uint2v*>((uint8_t*)base + off) = c;
      if (chunk == 0) scales[scale_at] = scale;
    }
  }
}

typedef unsigned short ushort8v __attribute__((ext_vector_type(8)));

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

// A wave writes RS = 64 / (D / 8) rows of one head, K and V; a lane holds 8
// coordinates of a row.  Bounds: the wave of a run's first row (rows of one
// sequence in one page) reads the run's keys, eight rows of a lane in flight, and writes
// the page's bounds, so no two waves write the same ones and no order changes them.
template <int D, int TYPE>
__global__ void __launch_bounds__(256)
paged_append_kernel(const rfsn_paged p, int shift, const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                    int64_t ts, int64_t hs, int64_t rows, const int32_t* __restrict__ cu) {
  constexpr int LANES = D / 8, RS = 64 / LANES, U = 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int h = blockIdx.y * 4 + wave;
  if (h >= p.kv_heads) return;
  const int slot = lane / LANES, chunk = lane % LANES;
  const int64_t n0 = (int64_t)blockIdx.x * RS, nc = n0 + slot < rows ? n0 + slot : rows - 1;
  const half8v kx = *reinterpret_cast<const half8v*>(k + nc * ts + h * hs + chunk * 8);
  const half8v vx = *reinterpret_cast<const half8v*>(v + nc * ts + h * hs + chunk * 8);
  const RowPlace at = row_place<LANES>(p, shift, cu, rows, n0, lane);
  const bool write = at.page >= 0;
  const int64_t off = (int64_t)(write ? at.page : 0) * p.page_stride + h * p.head_stride + (int64_t)at.row * D + chunk * 8;
  const int64_t sc = ((int64_t)(write ? at.page : 0) * p.kv_heads + h) * p.page_size + at.row;
  store_row<TYPE, LANES>(p, p.k, p.k_scale, off, sc, kx, chunk, write);
  store_row<TYPE, LANES>(p, p.v, p.v_scale, off, sc, vx, chunk, write);
  if (p.bounds == nullptr) return;
  const bool leads = write && at.start;
  auto bounds_at = [&](int page) {
    return reinterpret_cast<half8v*>((uint16_t*)p.bounds + ((int64_t)page * p.kv_heads + h) * 2 * D + chunk * 8);
  };
  // runs of one row: each row slot on its own; longer ones by the whole wave
  if (leads && at.count == 1) {
    half8v* bp = bounds_at(at.page);
    Bounds m = bounds_of(kx);
    if (at.row > 0) m.add(bp[0], bp[D / 8]);
    m.store(bp, bp + D / 8);
  }
  uint64_t todo = __ballot(leads && at.count > 1);
  while (todo) {
    const int src = __ffsll((unsigned long long)todo) - 1;  // a lane of the run's first row
    todo &= ~(((1ull << LANES) - 1) << (src / LANES * LANES));
    const int page = __builtin_amdgcn_readlane(at.page, src), row = __builtin_amdgcn_readlane(at.row, src);
    const int count = __builtin_amdgcn_readlane(at.count, src);
    const uint16_t* run = k + (n0 + src / LANES) * ts + h * hs + chunk * 8;
    half8v* bp = bounds_at(page);
    const half8v x0 = *reinterpret_cast<const half8v*>(run + min(slot, count - 1) * ts);
    Bounds m = bounds_of(x0);
    if (row > 0) m.add(bp[0], bp[D / 8]);
    for (int i = slot + RS; i - slot < count; i += U * RS) {
      half8v x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const half8v*>(run + min(i + u * RS, count - 1) * ts);
#pragma unroll
      for (int u = 0; u < U; ++u) m.add(x[u]);
    }
#pragma unroll
    for (int o = LANES; o < 64; o <<= 1) m.across(o);
    if (slot == 0) m.store(bp, bp + D / 8);
  }
}

template <int D, int TYPE>
__global__ void __launch_bounds__(256)
paged_read_kernel(const rfsn_paged p, int shift, const int32_t* __restrict__ cu, int64_t rows,
                  uint16_t* __restrict__ out_k, uint16_t* __restrict__ out_v, int zero_rest) {
  constexpr int LANES = D / 8, RS = 64 / LANES;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int h = blockIdx.y * 4 + wave;
  if (h >= p.kv_heads) return;
  const int slot = lane / LANES, chunk = lane % LANES;
  const int64_t n = (int64_t)blockIdx.x * RS + slot;
  const RowPlace at = row_place<LANES>(p, shift, cu, rows, (int64_t)blockIdx.x * RS, lane);
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
// bounds, D / 8 lanes a page, a wave kScoreSets sets of pages, whose loads are all in
// flight together.  Products of fp16 values are exact in fp32, and of q+ hi and q- lo one
// is zero; sums are held in 64 bits.
constexpr int kScoreSets = 4;
template <int D>
__global__ void __launch_bounds__(256)
page_score_kernel(const rfsn_paged p, int shift, const uint16_t* __restrict__ q, int G, float* __restrict__ score) {
  constexpr int LANES = D / 8, RS = 64 / LANES, U = kScoreSets;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int h = blockIdx.y, b = blockIdx.z;
  const int slot = lane / LANES, chunk = lane % LANES;
  const int held = (int)(((int64_t)paged_len(p, shift, b) + p.page_size - 1) >> shift);
  const int n0 = (blockIdx.x * 4 + wave) * (RS * U) + slot;
  if (n0 - slot >= held) return;
  int page[U];
  half8v lo[U], hi[U];
#pragma unroll
  for (int u = 0; u < U; ++u) page[u] = n0 + u * RS < held ? paged_page(p, b, n0 + u * RS) : -1;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const half8v* bp = reinterpret_cast<const half8v*>(
        (const uint16_t*)p.bounds + ((int64_t)max(page[u], 0) * p.kv_heads + h) * 2 * D + chunk * 8);
    lo[u] = bp[0], hi[u] = bp[D / 8];
  }
  double best[U];
  bool nan[U];
#pragma unroll
  for (int u = 0; u < U; ++u) best[u] = -__builtin_inf(), nan[u] = false;
#pragma unroll 1
  for (int g = 0; g < G; ++g) {
    const half8v qv = *reinterpret_cast<const half8v*>(q + (((int64_t)b * p.kv_heads + h) * G + g) * D + chunk * 8);
    float up[8], down[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = (float)qv[e];
      up[e] = x < 0.f ? 0.f : x, down[e] = x > 0.f ? 0.f : x;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      double s = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) s += (double)fmaf(up[e], (float)hi[u][e], down[e] * (float)lo[u][e]);
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
// three the most.  Then each of 16 waves counts what it keeps of its own run of pages and writes it
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
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) lo = min(lo, (uint32_t)__shfl_xor((int)lo, o, 64)), hi = max(hi, (uint32_t)__shfl_xor((int)hi, o, 64));
  if (lane == 0) s_wave[0][wave] = lo, s_wave[1][wave] = hi;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kChooseWaves; ++w) lo = min(lo, s_wave[0][w]), hi = max(hi, s_wave[1][w]);
  __syncthreads();  // s_wave is written again
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
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t x = (uint32_t)__shfl_up((int)upto, o, 64);
      if (lane >= o) upto += x;
    }
    if (lane == 63) s_wave[0][wave] = upto;
    __syncthreads();
    uint32_t above = upto - mine;
    for (int w = 0; w < wave; ++w) above += s_wave[0][w];
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
    // s_found and hist are written again behind the next barriers
    __syncthreads();
  }
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
  uint32_t at = (uint32_t)first, before = 0;
  for (int w = 0; w < wave; ++w) at += s_wave[0][w], before += s_wave[1][w];
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
  RFSN_REQUIRE(ceil_div(rows, rs) < (1ll << 24), "paged_append: too many rows");
  const int shift = paged_shift(*p);
  const dim3 grid((unsigned)ceil_div(rows, rs), (unsigned)ceil_div(p->kv_heads, 4));
  RFSN_PAGED_DISPATCH(p->head_dim, p->type, {
    hipLaunchKernelGGL((paged_append_kernel<DD, TT>), grid, dim3(256), 0, (hipStream_t)stream, *p, shift,
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
  RFSN_REQUIRE(ceil_div(rows, rs) < (1ll << 24), "paged_read: too many rows");
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
  if (p->batch == 0) return RFSN_OK;
  RFSN_REQUIRE(q && ((uintptr_t)q & 15) == 0 && chosen, "page_select: null or misaligned q, or null output");
  RFSN_REQUIRE(workspace_bytes >= rfsn_page_select_workspace_bytes(p) && (workspace || p->table_width == 0),
               "page_select: workspace too small");
  const int shift = paged_shift(*p);
  const hipStream_t s = (hipStream_t)stream;
  const int G = q_heads / p->kv_heads;
  if (p->table_width > 0) {
    const int per = 4 * kScoreSets * (512 / p->head_dim);
    const dim3 grid((unsigned)ceil_div(p->table_width, per), (unsigned)p->kv_heads, (unsigned)p->batch);
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
