// Attention of one query per sequence over a paged KV cache (attention.py:39-105
// for a batch of paged windows), over all positions or a list of pages.
//
//   out_i = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),  s_t = scale q_i . k_t
//
// in one pass over K and V with a running maximum.  A block takes a chunk of
// positions of one (sequence, KV head) with up to 16 of its query heads, so K and
// V are read once for the group; chunks are cut by the lengths, which only the
// device knows (find_chunk), and a second kernel joins their (m, l, O).
//
// Bound: the HBM read of K and V where there is enough of it (32 x 32,768
// positions, 8 KV heads of 64: fp16 2.15 GB in 324 to 331 us, 6.5 TB/s, 1.001 of the bytes
// that there are, the matrix cores 6 % busy, VALU 15 %, no LDS conflicts; int8 205 us,
// 5.6 TB/s; 4 x 8,001, 32 KV heads of 128: 77 to 84 us, 6.2 to 6.8 TB/s).  Below some
// 50 MB the chain of dependent loads (length, page, rows), the launch and the merge:
// 1,021 positions x 8 KV heads 8.8 to 9.4 us, 8,192 of int8 8.5 us and 3 to 4 for the merge.
// One wave per head and chunk with fp32 FMAs (attend_row, now for sums that are not
// finite alone) took 4,104 us for the first and 88 us for 1,021 positions.
#include "paged.h"
#include "paged_plan.h"

namespace rfsn {
namespace {

struct Chunk {
  int b;       // sequence, -1: none
  int j, n;    // number in the sequence, and of how many
  int64_t t0, t1;
};

// ceil(len / size) for quotients below 2^20, by a product with the reciprocal (off by less than half then)
// and a correction of the one that its floor may be off by.
__device__ __forceinline__ uint32_t parts_of(uint32_t len, uint32_t size) {
  const uint32_t n = (uint32_t)((float)len * __builtin_amdgcn_rcpf((float)size));
  const int64_t left = (int64_t)len - (int64_t)n * size;
  if (left < 0) return left + size == 0 ? n - 1 : n;
  return left == 0 ? n : left <= (int64_t)size ? n + 1 : n + 2;
}

// Chunk number w of a batch that is cut by the lengths, by one wave.  Of three sizes, for 2, 3 or 4
// blocks per CU (1, 2 or 3 of many waves), the one whose fullest CU has the fewest positions: 24 x 5,000
// positions of 8 KV heads take 51 us as 768 blocks and 57 as 576; 131,072 of one 54 as 512 and 61 as 896.
__device__ __forceinline__ Chunk find_chunk(const rfsn_paged& p, int shift, const Cut& cut, int w, int lane) {
  const int len0 = lane < p.batch ? paged_len(p, shift, lane) : 0;  // of the first 64, which are most batches
  float total = 0.f;
  if (p.batch == 1) {
    total = (float)__builtin_amdgcn_readfirstlane(len0);
  } else {  // in 32 bits by wave: lengths below 2^31 in two halves
    uint64_t sum = ((uint64_t)wave_total((uint32_t)len0 >> 16) << 16) + wave_total((uint32_t)len0 & 0xffffu);
    for (int base = 64; base < p.batch; base += 64) {
      const uint32_t len = base + lane < p.batch ? (uint32_t)paged_len(p, shift, base + lane) : 0u;
      sum += ((uint64_t)wave_total(len >> 16) << 16) + wave_total(len & 0xffffu);
    }
    total = (float)sum;
  }
  auto about = [](uint32_t len, uint32_t n) { return (uint32_t)((float)len * __builtin_amdgcn_rcpf((float)max(n, 1u))); };
  uint32_t size = 0;
  float least = 0.f;
#pragma unroll
  for (int x = 0; x < kTries; ++x) {
    if (x > 0 && p.batch == 1) break;  // of one sequence the chunks are alike: the fewest
    const float each = total * cut.one_over[x] + 0.98f;  // rounded up, but for an excess that is fp32's
    uint32_t s = each < 2147483520.f ? (uint32_t)each : 2147483520u;
    s = s <= (uint32_t)cut.chunk ? (uint32_t)cut.chunk : (s + 127) & ~127u;
    if (s > cut.longest) s = (uint32_t)cut.longest;
    uint32_t n = parts_of((uint32_t)len0, s), most = about(len0, n);
    for (int b = 64 + lane; b < p.batch; b += 64) {
      const uint32_t len = (uint32_t)paged_len(p, shift, b), m = parts_of(len, s);
      n += m, most = max(most, about(len, m));
    }
    if (p.batch > 1) n = wave_total(n), most = wave_most(most);
    // positions on the fullest CU, each chunk costing as much as 128 more
    const float cost = (float)((n * (uint32_t)cut.units + kCUs - 1) / kCUs) * ((float)most + 128.f);
    if (x == 0 || cost < least) least = cost, size = s;
  }
  size = __builtin_amdgcn_readfirstlane(size);
  int seen = 0;
  for (int base = 0; base < p.batch; base += 64) {
    const int b = base + lane;
    const int len = base == 0 ? len0 : b < p.batch ? paged_len(p, shift, b) : 0;
    const int n = (int)parts_of((uint32_t)len, size);
    const int upto = p.batch > 1 ? (int)wave_upto((uint32_t)n) : n;
    const uint64_t in = __ballot(w < seen + upto && w >= seen + upto - n);
    if (in) {
      const int src = __ffsll((unsigned long long)in) - 1;
      const int of = __builtin_amdgcn_readlane(n, src), j = w - seen - __builtin_amdgcn_readlane(upto, src) + of;
      const int64_t end = __builtin_amdgcn_readlane(len, src);
      // the sequence's chunks are alike
      const int64_t part = (int64_t)(((uint32_t)end + (uint32_t)of - 1) / (uint32_t)of + 127) & ~127ll, t0 = j * part;
      return {base + src, j, of, t0 < end ? t0 : end, t0 + part < end ? t0 + part : end};
    }
    seen += __builtin_amdgcn_readlane(upto, 63);
  }
  return {-1, 0, 0, 0, 0};
}

// Where listed position t of (b, h) lies: t itself without a list, else row t %
// page_size of the list's page t / page_size.
struct Place {
  bool valid;
  int page, row;
};
__device__ __forceinline__ Place place(const rfsn_paged& p, int shift, const int32_t* list, int len, int b, int64_t t,
                                       int64_t end) {
  Place r = {false, 0, (int)(t & (p.page_size - 1))};
  if (t >= end) return r;
  const int64_t ord = list ? list[t >> shift] : t >> shift;
  if (ord < 0 || (ord << shift) + r.row >= len) return r;
  const int page = paged_page(p, b, ord);
  if (page < 0) return r;
  r.valid = true, r.page = page;
  return r;
}

// One head over positions t0 .. t1 by one wave: lane = position for the scores,
// lane = coordinate for P V, everything in fp32.
template <int D, int TYPE>
__device__ __forceinline__ void attend_row(const rfsn_paged& p, int shift, const int32_t* list, int b, int h, int64_t t0,
                                           int64_t t1, const uint16_t* __restrict__ q, float scale_log2, int lane,
                                           float& m, float& l, float (&acc)[D / 64]) {
  constexpr int E = D / 64;
  m = -__builtin_inff(), l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  const int len = paged_len(p, shift, b);
#pragma unroll 1
  for (int64_t base = t0; base < t1; base += 64) {
    const Place at = place(p, shift, list, len, b, base + lane, t1);
    const int64_t off = (int64_t)at.page * p.page_stride + h * p.head_stride + (int64_t)at.row * D;
    const int64_t sc = ((int64_t)at.page * p.kv_heads + h) * p.page_size + at.row;
    float s = -__builtin_inff(), vs = 1.f;
    if (at.valid) {
      float dot = 0.f;
#pragma unroll 2
      for (int c = 0; c < D / 8; ++c) {
        const float8v kv = load_page8<TYPE>(p.k, off + 8 * c);
        const half8v qv = reinterpret_cast<const half8v*>(q)[c];
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf((float)qv[e], kv[e], dot);
      }
      if constexpr (TYPE != RFSN_PAGE_FP16) dot *= p.k_scale[sc], vs = p.v_scale[sc];
      s = dot * scale_log2;
    }
    uint64_t todo = __ballot(at.valid);
    if (!todo) continue;
    const float top = wave_max(s);
    const bool odd = __any(s != s);  // a NaN score is no maximum
    const float mn = fmaxf(m, top), mref = mn > -__builtin_inff() ? mn : 0.f;
    const float w = at.valid ? (odd ? __builtin_nanf("") : exp2f(s - mref)) : 0.f;
    const float corr = m > -__builtin_inff() ? exp2f(m - mref) : 1.f;
    l = l * corr + wave_sum(w);
    m = mn;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= corr;
    while (todo) {
      const int i = __ffsll((unsigned long long)todo) - 1;
      todo &= todo - 1;
      const int64_t vo = ((int64_t)__builtin_amdgcn_readlane((int)(off >> 32), i) << 32) |
                         (uint32_t)__builtin_amdgcn_readlane((int)off, i);
      float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i));
      const float si = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vs), i));
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float x;
        const int64_t o = vo + lane * E + e;
        if constexpr (TYPE == RFSN_PAGE_FP16) x = h2f(((const uint16_t*)p.v)[o]);
        else if constexpr (TYPE == RFSN_PAGE_INT8) x = (float)((const int8_t*)p.v)[o] * si;
        else x = __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)p.v)[o], 0) * si;
        acc[e] = fmaf(wi, x, acc[e]);
      }
    }
  }
}

// ---- tiles on the matrix cores
//
// A wave takes two groups of 16 positions at a time (each inside one page; four groups, with half
// the waves' registers, changed no time by more than 3 % where they fit and cost 8 % with 8-bit rows of 128), a
// block's waves take them in turn, and a lane's 16 columns are the query heads of the KV
// head (the others repeat the last: the matrix cores are idle otherwise).
//   S = K Q^T      MFMA 16x16x32, A = 16 rows of K as they lie in memory (16 bytes a
//                  lane, the coordinates of Q in the same order), so K goes from
//                  memory to its operand without LDS; a lane holds 8 scores of one head;
//   O^T += V^T P^T with the weights' registers as the B operand as they are: k slot
//                  (lane group g, j) is position 16 (j >> 2) + 4 g + (j & 3).  V passes
//                  through LDS of the wave's own, and ds_read_b64_tr_b16 reads V^T from it
//                  in that order.
// Weights are rounded twice.  With 8-bit pages p times the row's scale is bf16 hi + lo, which has fp32's range, and
// off by 2^-16 of itself (codes are exact in bf16).  With fp16 pages p 2^8 is fp16 hi + lo: off by 2^-22 of itself
// or by 2^-33 of the largest weight that the wave has seen, whichever is more, because fp16 ends at 2^-24; what
// is under 2^-33 adds nothing to O and counts in l.  N positions of a wave are then off by at most N 2^-33 of the
// largest |v|, and no wave has more than 2^20 (kLongestChunk; tables for over 2^37 positions aside).  All of it is
// well under the 2^-11 of the result's own rounding; the second product costs matrix-core time that is idle.
// Scores, maxima, sums and O are fp32.
// Where V or a score is infinite or NaN, hi, lo and weights of 0 meet it apart; a block that
// finds a sum that is not finite takes its chunk again by attend_row.

typedef float float4v __attribute__((ext_vector_type(4)));
typedef _Float16 half2w __attribute__((ext_vector_type(2)));
typedef _Float16 half4w __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short short4w __attribute__((ext_vector_type(4)));
typedef short short8w __attribute__((ext_vector_type(8)));

constexpr int NG = 2;              // groups of a wave's step
constexpr float kPBias = 8.f;      // a weight is kept as p 2^8
constexpr float kPSum = 32768.f;   // a lane's sum below it: every weight is finite in fp16

// 16-byte chunk c of row t of a [32][D] 16-bit tile sits at chunk c ^ v_swz(t): the
// transposed reads take 32 bytes of 8 rows at once, which then lie in different banks.
template <int D>
__device__ __forceinline__ int v_swz(int t) { return D == 64 ? ((t >> 1) & 3) << 1 : (t & 7) << 1; }

// 8 codes as fp16 (exact).
template <int TYPE>
__device__ __forceinline__ half8v codes_f16(uint32_t a, uint32_t b) {
  half8v r;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint32_t c = w ? b : a;
    half2w lo, hi;
    if constexpr (TYPE == RFSN_PAGE_INT8) {
      const uint32_t u = c ^ 0x80808080u;  // code + 128 as the low bits of 1024 + code + 128
      lo = __builtin_bit_cast(half2w, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - (f16)1152.f;
      hi = __builtin_bit_cast(half2w, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - (f16)1152.f;
    } else {
      lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.f, false);
      hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.f, true);
    }
    r[4 * w] = lo[0], r[4 * w + 1] = lo[1], r[4 * w + 2] = hi[0], r[4 * w + 3] = hi[1];
  }
  return r;
}

// 8 codes as bf16 (exact), packed.
template <int TYPE>
__device__ __forceinline__ uint4w codes_bf16(uint32_t a, uint32_t b) {
  uint4w r;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint32_t c = w ? b : a;
    float f[4];
    if constexpr (TYPE == RFSN_PAGE_INT8) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = (float)(int8_t)(c >> (8 * e));
    } else {
      f[0] = __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
      f[1] = __builtin_amdgcn_cvt_f32_fp8((int)c, 1);
      f[2] = __builtin_amdgcn_cvt_f32_fp8((int)c, 2);
      f[3] = __builtin_amdgcn_cvt_f32_fp8((int)c, 3);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)  // the high halves
      r[2 * w + e] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[2 * e + 1]),
                                           __builtin_bit_cast(uint32_t, f[2 * e]), 0x07060302u);
  }
  return r;
}

// 16 bytes of a row, marked as not to be kept where the call reads more than the caches hold (Plan).
template <bool kOnce>
__device__ __forceinline__ uint4w load16(const uint8_t* a) {
  if constexpr (kOnce) return __builtin_nontemporal_load(reinterpret_cast<const uint4w*>(a));
  else return *reinterpret_cast<const uint4w*>(a);
}

// Partial results of a split call: (m, l) and O of each chunk and query head, and for each
// sequence that has any its first chunk and their number.
struct Parts {
  float* acc;   // [slots][q_heads][D]
  float* ml;    // [slots][q_heads][2]
  int32_t* seq; // [batch][2]
};

template <int D, int TYPE, int kWaves, bool kOnce>
__global__ void __launch_bounds__(kWaves * 64, kWaves > 4 ? 1 : D == 64 ? 4 : D == 128 ? 2 : 1)
paged_attn_kernel(const rfsn_paged p, int shift, const int32_t* __restrict__ table, const uint16_t* __restrict__ q, int G,
                  float scale_log2, const int32_t* __restrict__ chosen, int count, const Cut cut,
                  uint16_t* __restrict__ out, const Parts parts) {
  constexpr bool kCodes = TYPE != RFSN_PAGE_FP16;
  constexpr int E = D / 64;
  constexpr int ES = kCodes ? 1 : 2;                 // bytes of a stored value
  constexpr int KS = D / 32;                         // MFMA k steps of a score
  constexpr int KL = D * ES / 64;                    // 16-byte loads of a lane's share of a K row
  constexpr int DT = D / 16;                         // 16-coordinate tiles of O^T
  constexpr int VC = D * ES / 16;                    // 16-byte chunks of a stored row
  constexpr int kTile = 16 * NG;                     // positions per wave and step
  constexpr int GT = 64 / NG;                        // tiles whose groups fill a wave's lanes
  constexpr int VU = 16 * VC / 64;                   // V loads of a lane for a group
  constexpr int CH = D / 8;                          // 16-byte chunks of a row in LDS
  __shared__ uint4w smem[kWaves * kTile * CH];       // V tiles; then the waves' O, m, l
  __shared__ float s_ml[kWaves][2][16];
  __shared__ int s_odd[kWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int h = blockIdx.x, w = blockIdx.y, g0 = blockIdx.z * 16;
  const int heads = G - g0 < 16 ? G - g0 : 16;
  const int step = kWaves * kTile;
  int b, t0;
  int64_t t1_cut = 0;
  if (cut.per_seq) {
    b = w / cut.per_seq;
    t0 = (int)((w - b * cut.per_seq) * cut.chunk);
  } else {
    const Chunk c = find_chunk(p, shift, cut, w, lane);
    if (c.b < 0) return;
    if (c.j == 0 && h == 0 && g0 == 0 && threadIdx.x == 0) parts.seq[2 * c.b] = w, parts.seq[2 * c.b + 1] = c.n;
    b = __builtin_amdgcn_readfirstlane(c.b), t0 = __builtin_amdgcn_readfirstlane((int)c.t0), t1_cut = c.t1;
  }
  const int32_t* const list = chosen ? chosen + ((int64_t)b * p.kv_heads + h) * count : nullptr;
  const int32_t* const pages = table + (int64_t)b * p.table_stride;
  const int64_t row0 = ((int64_t)b * p.kv_heads + h) * G + g0;  // of q and out

  // The pages of 64 groups of 16 positions, those of this wave's next GT tiles, one group a lane:
  // lane NG k + u has group u of tile k.  Their loads wait for nothing but a list's.
  auto ordinal = [&](int tile) {
    const int64_t t = (int64_t)t0 + wave * kTile + (int64_t)(tile + lane / NG) * step + lane % NG * 16;
    const int64_t ord = t >> shift;
    if (list == nullptr) return ord;
    return ord < count ? (int64_t)list[ord] : -1;
  };
  auto entry = [&](int64_t ord) { return ord >= 0 && ord < p.table_width ? pages[ord] : -1; };
  int64_t ord_l = ordinal(0);
  int page_l = entry(ord_l);
  half8v qf[KS];
  {
    const uint16_t* qr = q + (row0 + (col < heads ? col : heads - 1)) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qf[s] = *reinterpret_cast<const half8v*>(qr + (kCodes ? (s >> 1) * 64 + grp * 16 + (s & 1) * 8 : s * 32 + grp * 8));
  }
  const int len = __builtin_amdgcn_readfirstlane(paged_len(p, shift, b));
  if (cut.per_seq) {
    const int64_t end = chosen ? (int64_t)count << shift : len;
    t1_cut = t0 + cut.chunk < end ? t0 + cut.chunk : end;
  }
  const int t1 = __builtin_amdgcn_readfirstlane((int)t1_cut);
  int rows_l;  // rows of the lane's group that are attended; page_l is a page of the pool from here on
  auto locate = [&](int tile) {
    const int64_t t = (int64_t)t0 + wave * kTile + (int64_t)(tile + lane / NG) * step + lane % NG * 16;
    int64_t n = t1 - t;
    if (list) {
      const int64_t left = (int64_t)len - ((ord_l << shift) + (t & (p.page_size - 1)));
      n = left < n ? left : n;
    }
    if (page_l < 0 || page_l >= p.pages || n <= 0) n = 0, page_l = 0;
    rows_l = (int)(n < 16 ? n : 16);
  };
  locate(0);

  float4v o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = float4v{0.f, 0.f, 0.f, 0.f};
  float m_run = -__builtin_inff(), l_run = 0.f;  // reference exponent of the head's weights, this lane's sum of them

  uint4w kr[NG][KL], vr[NG][VU];
  float4v ks[NG], vs[NG];
  int n_next[NG] = {};  // rows of the fetched groups that are attended
  // Rows past the last one attended re-read it: their weights are 0.  A group with none
  // reads page 0, and its V is not used.
  auto fetch = [&](int t, int tile) {
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      const int page = __builtin_amdgcn_readlane(page_l, NG * (tile % GT) + u);
      const int n = __builtin_amdgcn_readlane(rows_l, NG * (tile % GT) + u);
      const int row = (t + 16 * u) & (p.page_size - 1);
      n_next[u] = n;
      const int last = n > 0 ? n - 1 : 0;
      const int64_t base = ((int64_t)page * p.page_stride + (int64_t)h * p.head_stride + (int64_t)row * D) * ES;
      const uint8_t* kb = (const uint8_t*)p.k + base;
      const uint8_t* vb = (const uint8_t*)p.v + base;
      const uint32_t kl = (uint32_t)(min(col, last) * (D * ES) + grp * 16);
#pragma unroll
      for (int i = 0; i < KL; ++i) kr[u][i] = load16<kOnce>(kb + kl + i * 64);
#pragma unroll
      for (int i = 0; i < VU; ++i) {
        const int idx = i * 64 + lane, r = idx / VC, ch = idx % VC;
        vr[u][i] = load16<kOnce>(vb + (uint32_t)(min(r, last) * (D * ES) + ch * 16));
      }
      if constexpr (kCodes) {
        const int64_t sc = ((int64_t)page * p.kv_heads + h) * p.page_size + row;
        ks[u] = *reinterpret_cast<const float4v*>(p.k_scale + sc + (uint32_t)(grp * 4));
        vs[u] = *reinterpret_cast<const float4v*>(p.v_scale + sc + (uint32_t)(grp * 4));
      }
    }
  };
  uint4w* const sv = smem + wave * kTile * CH;
  int t = t0 + wave * kTile, tile = 0;
  if (t < t1) fetch(t, 0);
  for (; t < t1; t += step) {
    int n[NG];
#pragma unroll
    for (int u = 0; u < NG; ++u) n[u] = n_next[u];
    // V to LDS
#pragma unroll
    for (int u = 0; u < NG; ++u)
#pragma unroll
      for (int i = 0; i < VU; ++i) {
        const int idx = i * 64 + lane, r = u * 16 + idx / VC, ch = idx % VC;
        uint4w x = vr[u][i];
        if (n[u] == 0) x = uint4w{0, 0, 0, 0};
        if constexpr (!kCodes) {
          sv[r * CH + (ch ^ v_swz<D>(r))] = x;
        } else {
          sv[r * CH + ((2 * ch) ^ v_swz<D>(r))] = codes_bf16<TYPE>(x[0], x[1]);
          sv[r * CH + ((2 * ch + 1) ^ v_swz<D>(r))] = codes_bf16<TYPE>(x[2], x[3]);
        }
      }
    // scores in base 2
    float4v s[NG];
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      s[u] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        half8v kf;
        if constexpr (!kCodes) kf = __builtin_bit_cast(half8v, kr[u][k]);
        else kf = codes_f16<TYPE>(kr[u][k >> 1][2 * (k & 1)], kr[u][k >> 1][2 * (k & 1) + 1]);
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[k], s[u], 0, 0, 0);
      }
    }
    float4v vscale[NG];
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      if constexpr (kCodes) {
        s[u] *= ks[u];
        vscale[u] = vs[u];
      }
      s[u] *= scale_log2;
      if (n[u] < 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (grp * 4 + i >= n[u]) {
            s[u][i] = -__builtin_inff();
            if constexpr (kCodes) vscale[u][i] = 0.f;
          }
        }
      }
    }
    ++tile;
    if (t + step < t1) {
      if (tile % GT == 0) {  // the next GT tiles
        ord_l = ordinal(tile);
        page_l = entry(ord_l);
        locate(tile);
      }
      fetch(t + step, tile);
    }
    float pw[4 * NG], ls;
    auto weights = [&]() {
      const float mb = m_run > -__builtin_inff() ? m_run : 0.f;
      ls = 0.f;
#pragma unroll
      for (int i = 0; i < 4 * NG; ++i) {
        pw[i] = __builtin_amdgcn_exp2f(s[i >> 2][i & 3] - mb);
        ls += pw[i];
      }
    };
    weights();
    // The maximum is moved only when a lane's sum says that a weight may leave
    // fp16's range (or nothing was seen yet): no weight exceeds the sum.
    if (__any(!(ls < kPSum) || m_run == -__builtin_inff())) {
      float mx = s[0][0];
#pragma unroll
      for (int i = 1; i < 4 * NG; ++i) mx = fmaxf(mx, s[i >> 2][i & 3]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float m_new = fmaxf(m_run, mx - kPBias);
      const float corr = m_run > -__builtin_inff() ? __builtin_amdgcn_exp2f(m_run - m_new) : 0.f;
      l_run *= corr;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= corr;
      m_run = m_new;
      weights();
    }
    l_run += ls;
    uint32_t bh[2 * NG], bl[2 * NG];  // weights as B operands of 8, high and low parts
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i) {
      if constexpr (!kCodes) {
        const half2w hi = {(f16)pw[2 * i], (f16)pw[2 * i + 1]};
        const half2w lo = {(f16)(pw[2 * i] - (float)hi[0]), (f16)(pw[2 * i + 1] - (float)hi[1])};
        bh[i] = __builtin_bit_cast(uint32_t, hi), bl[i] = __builtin_bit_cast(uint32_t, lo);
      } else {
        const float a = pw[2 * i] * vscale[i >> 1][(2 * i) & 3], b = pw[2 * i + 1] * vscale[i >> 1][(2 * i + 1) & 3];
        const bf16x2 hi = {(__bf16)a, (__bf16)b};
        const bf16x2 lo = {(__bf16)(a - (float)hi[0]), (__bf16)(b - (float)hi[1])};
        bh[i] = __builtin_bit_cast(uint32_t, hi), bl[i] = __builtin_bit_cast(uint32_t, lo);
      }
    }
    // the tile was written by all lanes of this wave: LDS keeps a wave's order, the compiler has to as well
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int x = 0; x < NG / 2; ++x) {
      const uint4w hi = {bh[4 * x], bh[4 * x + 1], bh[4 * x + 2], bh[4 * x + 3]};
      const uint4w lo = {bl[4 * x], bl[4 * x + 1], bl[4 * x + 2], bl[4 * x + 3]};
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        typedef __attribute__((address_space(3))) short4w lds4;
        short4w a[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tv = 32 * x + 16 * e + 4 * grp + (col >> 2), cc = 2 * d + ((col & 3) >> 1);
          const int off = (tv * CH + (cc ^ v_swz<D>(tv))) * 16 + (col & 1) * 8;
          a[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)((__attribute__((address_space(3))) char*)sv + off));
        }
        const short8w av = {a[0][0], a[0][1], a[0][2], a[0][3], a[1][0], a[1][1], a[1][2], a[1][3]};
        if constexpr (!kCodes) {
          const half8v vf = __builtin_bit_cast(half8v, av);
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, __builtin_bit_cast(half8v, hi), o[d], 0, 0, 0);
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, __builtin_bit_cast(half8v, lo), o[d], 0, 0, 0);
        } else {
          const bf16x8 vf = __builtin_bit_cast(bf16x8, av);
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, __builtin_bit_cast(bf16x8, hi), o[d], 0, 0, 0);
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, __builtin_bit_cast(bf16x8, lo), o[d], 0, 0, 0);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
  }

  static_assert(kTile * CH * 16 >= DT * 64 * 16, "a wave's O fits its V tile");
  float zero = l_run * 0.f;  // NaN where a sum is infinite or NaN
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) zero = fmaf(o[d][i], 0.f, zero);
  const int odd = __any(zero != 0.f);
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  float* const so = reinterpret_cast<float*>(smem);
  if (lane == 0) s_odd[wave] = odd;
  if (grp == 0) s_ml[wave][0][col] = m_run, s_ml[wave][1][col] = l_run;
  // the waves' V tiles are done with: each wave's O lies over its own
#pragma unroll
  for (int d = 0; d < DT; ++d) *reinterpret_cast<float4v*>(so + wave * (kTile * CH * 4) + (d * 64 + lane) * 4) = o[d];
  __syncthreads();
  int any = s_odd[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) any |= s_odd[i];
  if (any) {  // block-uniform: the chunk again, a head at a time
    for (int g = wave; g < heads; g += kWaves) {
      const int64_t row = row0 + g;
      float m, l, acc[E];
      attend_row<D, TYPE>(p, shift, list, b, h, t0, t1, q + row * D, scale_log2, lane, m, l, acc);
      if (parts.ml == nullptr) {
#pragma unroll
        for (int e = 0; e < E; ++e) out[row * D + lane * E + e] = f2h(l == 0.f ? 0.f : acc[e] / l);
      } else {
        const int64_t slot = ((int64_t)w * p.kv_heads + h) * G + g0 + g;
        if (lane == 0) parts.ml[2 * slot] = m, parts.ml[2 * slot + 1] = l;
#pragma unroll
        for (int e = 0; e < E; ++e) parts.acc[slot * D + lane * E + e] = acc[e];
      }
    }
    return;
  }
  float m = s_ml[0][0][col], f[kWaves], l = 0.f;
#pragma unroll
  for (int i = 1; i < kWaves; ++i) m = fmaxf(m, s_ml[i][0][col]);
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const float mi = s_ml[i][0][col];
    f[i] = mi > -__builtin_inff() ? __builtin_amdgcn_exp2f(mi - m) : 0.f;
    l += f[i] * s_ml[i][1][col];
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const int64_t slot = ((int64_t)w * p.kv_heads + h) * G + g0 + col;
  if (parts.ml != nullptr && wave == 0 && grp == 0 && col < heads) parts.ml[2 * slot] = m, parts.ml[2 * slot + 1] = l;
  for (int d = wave; d < DT; d += kWaves) {
    float4v a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < kWaves; ++x) a += f[x] * *reinterpret_cast<const float4v*>(so + x * (kTile * CH * 4) + (d * 64 + lane) * 4);
    if (col >= heads) continue;
    if (parts.ml == nullptr) {
      const half4w r = {(f16)(a[0] * inv), (f16)(a[1] * inv), (f16)(a[2] * inv), (f16)(a[3] * inv)};
      *reinterpret_cast<half4w*>(out + (row0 + col) * D + d * 16 + grp * 4) = r;
    } else {
      *reinterpret_cast<float4v*>(parts.acc + slot * D + d * 16 + grp * 4) = a;
    }
  }
}

// out = sum_j w_j acc_j / sum_j w_j l_j over a sequence's chunks, w_j = 2^(m_j - max m).
// The (m, l) of 64 chunks are one load of a wave.  W waves share a row's chunks: 16 where few rows
// have many (131,072 positions of one sequence, 128 chunks: the call 64 -> 59 us), 4 for the rows of
// a batch (48 sequences x 32 heads: 25 us, and 27 with 16).
template <int D, int W>
__global__ void __launch_bounds__(W * 64)
paged_merge_kernel(const rfsn_paged p, int shift, int q_heads, int per_seq, const Parts parts, uint16_t* __restrict__ out) {
  constexpr int E = D / 64, U = 4;
  __shared__ float s_acc[W][D];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = blockIdx.x, b = blockIdx.y;
  int slot0 = b * per_seq, n = per_seq;
  if (!per_seq) {
    const int len = paged_len(p, shift, b);
    slot0 = parts.seq[2 * b], n = parts.seq[2 * b + 1];
    if (len == 0) slot0 = 0, n = 0;  // an empty sequence has no chunk, and nothing was written there
  }
  float m = -__builtin_inff(), l = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int base = 0; base < n; base += 64) {
    const int here = min(64, n - base);
    float mj = -__builtin_inff(), lj = 0.f;
    if (lane < here) {
      const int64_t s = (int64_t)(slot0 + base + lane) * q_heads + i;
      mj = parts.ml[2 * s], lj = parts.ml[2 * s + 1];
    }
    const float mn = fmaxf(m, wave_max(mj)), mref = mn > -__builtin_inff() ? mn : 0.f;
    const float corr = m > -__builtin_inff() ? exp2f(m - mref) : 1.f;
    const float wj = mj > -__builtin_inff() ? exp2f(mj - mref) : 1.f;  // with m -infinite the sums are 0 or NaN
    l = l * corr + wave_sum(lane < here ? wj * lj : 0.f);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= corr;
    for (int j0 = wave; j0 < here; j0 += W * U) {
      float x[U][E];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = min(j0 + W * u, here - 1);
        const float* a = parts.acc + ((int64_t)(slot0 + base + j) * q_heads + i) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = a[e];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (j0 + W * u >= here) break;
        const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wj), j0 + W * u));
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(w, x[u][e], acc[e]);
      }
    }
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_acc[wave][lane * E + e] = acc[e];
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += W * 64) {
    float a = s_acc[0][d];
#pragma unroll
    for (int x = 1; x < W; ++x) a += s_acc[x][d];
    out[((int64_t)b * q_heads + i) * D + d] = f2h(l == 0.f ? 0.f : a / l);
  }
}

size_t parts_bytes(const rfsn_paged& p, const Plan& c, int q_heads) {
  return (size_t)c.slots * q_heads * (p.head_dim + 2) * sizeof(float) + (size_t)p.batch * 2 * sizeof(int32_t);
}

}  // namespace
}  // namespace rfsn

using namespace rfsn;

extern "C" size_t rfsn_paged_attention_workspace_bytes(const rfsn_paged* p, int32_t q_heads, int32_t count) {
  if (p == nullptr || p->batch <= 0 || p->kv_heads <= 0 || p->page_size <= 0 || q_heads < p->kv_heads || count < 0) return 0;
  const Plan c = plan(*p, q_heads, count);
  return c.split() ? parts_bytes(*p, c, q_heads) : 0;
}

extern "C" int rfsn_paged_attention(const rfsn_paged* p, const void* q, int32_t q_heads, float scale,
                                    const int32_t* chosen, int32_t count, void* out, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (int st = paged_check(p, "paged_attention")) return st;
  RFSN_REQUIRE(q_heads > 0 && q_heads % p->kv_heads == 0 && q_heads <= 65535,
               "paged_attention: q_heads must be a multiple of kv_heads");
  RFSN_REQUIRE((chosen == nullptr) == (count == 0) && count >= 0, "paged_attention: chosen and count go together");
  RFSN_REQUIRE((int64_t)count * p->page_size <= (1ll << 31) - 1024, "paged_attention: too many chosen pages");
  const float sl2 = scale * 1.44269504088896340736f;
  RFSN_REQUIRE(sl2 == sl2 && sl2 < __builtin_inff() && sl2 > -__builtin_inff(),
               "paged_attention: scale must be finite, in base 2 as well");
  if (p->batch == 0) return RFSN_OK;
  RFSN_REQUIRE(q && out && ((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0,
               "paged_attention: q and out must be 16-byte aligned");
  const Plan c = plan(*p, q_heads, count);
  RFSN_REQUIRE(workspace_bytes >= rfsn_paged_attention_workspace_bytes(p, q_heads, count) && ((workspace && ((uintptr_t)workspace & 15) == 0) || !c.split()),
               "paged_attention: workspace too small or misaligned");
  RFSN_REQUIRE(c.slots <= 65535, "paged_attention: too many sequences");
  const hipStream_t s = (hipStream_t)stream;
  const int shift = paged_shift(*p), G = q_heads / p->kv_heads;
  Parts parts = {nullptr, nullptr, nullptr};
  if (c.split()) {
    parts.acc = (float*)workspace;
    parts.ml = parts.acc + c.slots * q_heads * p->head_dim;
    parts.seq = (int32_t*)(parts.ml + c.slots * q_heads * 2);
  }
  const dim3 grid((unsigned)p->kv_heads, (unsigned)c.slots, (unsigned)ceil_div(G, 16));
#define RFSN_ATTEND(DD, TT, NW, ONCE)                                                                               \
  hipLaunchKernelGGL((paged_attn_kernel<DD, TT, NW, ONCE>), grid, dim3(NW * 64), 0, s, *p, shift, p->table,           \
                     (const uint16_t*)q, G, sl2, chosen, count, c.cut, (uint16_t*)out, parts)
#define RFSN_ATTEND_D(DD, NW, ONCE)                                                \
  do {                                                                             \
    if (p->type == RFSN_PAGE_FP16) RFSN_ATTEND(DD, RFSN_PAGE_FP16, NW, ONCE);      \
    else if (p->type == RFSN_PAGE_INT8) RFSN_ATTEND(DD, RFSN_PAGE_INT8, NW, ONCE); \
    else RFSN_ATTEND(DD, RFSN_PAGE_E4M3, NW, ONCE);                                \
  } while (0)
  if (p->head_dim == 64 && c.wide) RFSN_ATTEND_D(64, 16, false);
  else if (p->head_dim == 64 && c.once) RFSN_ATTEND_D(64, 4, true);
  else if (p->head_dim == 64) RFSN_ATTEND_D(64, 4, false);
  else if (p->head_dim == 128 && c.wide) RFSN_ATTEND_D(128, 8, false);
  else if (p->head_dim == 128 && c.once) RFSN_ATTEND_D(128, 4, true);
  else if (p->head_dim == 128) RFSN_ATTEND_D(128, 4, false);
  else if (c.once) RFSN_ATTEND_D(256, 4, true);
  else RFSN_ATTEND_D(256, 4, false);
#undef RFSN_ATTEND_D
#undef RFSN_ATTEND
  if (int st = check_launch("paged_attention")) return st;
  if (c.split()) {
    const dim3 rows((unsigned)q_heads, (unsigned)p->batch);
    const bool many = (c.cut.per_seq ? c.cut.per_seq : c.slots - p->batch + 1) > 16 && (int64_t)q_heads * p->batch <= 256;
#define RFSN_MERGE(DD)                                                                                              \
  do {                                                                                                              \
    if (many)                                                                                                       \
      hipLaunchKernelGGL((paged_merge_kernel<DD, 16>), rows, dim3(1024), 0, s, *p, shift, q_heads, c.cut.per_seq,   \
                         parts, (uint16_t*)out);                                                                    \
    else                                                                                                            \
      hipLaunchKernelGGL((paged_merge_kernel<DD, 4>), rows, dim3(256), 0, s, *p, shift, q_heads, c.cut.per_seq,     \
                         parts, (uint16_t*)out);                                                                    \
  } while (0)
    if (p->head_dim == 64) RFSN_MERGE(64);
    else if (p->head_dim == 128) RFSN_MERGE(128);
    else RFSN_MERGE(256);
#undef RFSN_MERGE
  }
  return check_launch("paged_attention");
}
