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
// 5.6 TB/s; 4 x 8,001, 32 KV heads of 128: 77 to 84 us, 6.2 to 6.8 TB/s).  Of 4-bit pages
// the same 32 x 32,768 positions are 604 MB in 116 us, 5.2 TB/s, called again and again 130 to 150 at
// a lower clock (vector units 66 %, matrix cores 18 % busy; loads alone 107, arithmetic alone 83); with
// 32 KV heads of one query head, 24 of up to 12,001 positions of 128, 138 MB in 35 us.  Below some
// 50 MB the chain of dependent loads (length, page, rows), the launch and the merge:
// 1,021 positions x 8 KV heads 8.8 to 9.4 us, 8,192 of int8 8.5 us and 3 to 4 for the merge.
// One wave per head and chunk with fp32 FMAs (attend_row, now for sums that are not
// finite alone) took 4,104 us for the first and 88 us for 1,021 positions.
#pragma once

#include <type_traits>

#include "paged.h"
#include "paged_plan.h"

namespace rfsn {

// Partial results of a split call: (m, l) and O of each chunk and query head, and for each
// sequence that has any its first chunk and their number.
struct Parts {
  float* acc;   // [slots][q_heads][D]
  float* ml;    // [slots][q_heads][2]
  int32_t* seq; // [batch][2]
  // of a call that accumulates weights: each position's scores in base 2, and each query head's (m, l)
  float* score;     // [batch][kv_heads][positions / 16][G][16] (score_at)
  float* fin;       // [batch][q_heads][2]
  int64_t positions;
};

namespace {

// Where the scores of query head g of G lie for the 16 positions from t on (a multiple of 16), `from` = (b kv_heads + h) positions:
// what a wave writes at once, 16 positions of its heads, is one piece (a row of positions per head: 32 x 32,768 positions, 4 heads
// each, 479 us instead of 466).
__device__ __forceinline__ int64_t score_at(int64_t from, int G, int g, int64_t t) { return (from + t) * G + g * 16; }

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
    if (x > 0 && p.batch == 1 && cut.alike) break;  // of one sequence the chunks are alike: the fewest
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
    // positions on the fullest CU, each chunk costing as much as some more
    const float cost = (float)((n * (uint32_t)cut.units + kCUs - 1) / kCUs) * ((float)most + cut.start) * cut.each[x];
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
        float8v kv;
        if constexpr (TYPE == RFSN_PAGE_E2M1) {
          const half8v x = e2m1_f16(*reinterpret_cast<const uint32_t*>((const uint8_t*)p.k + (off + 8 * c) / 2),
                                    group_scale(((const uint8_t*)p.k_scale)[sc * (D / 16) + c / 2]));
#pragma unroll
          for (int e = 0; e < 8; ++e) kv[e] = (float)x[e];
        } else {
          kv = load_page8<TYPE>(p.k, off + 8 * c);
        }
        const half8v qv = reinterpret_cast<const half8v*>(q)[c];
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf((float)qv[e], kv[e], dot);
      }
      if constexpr (TYPE == RFSN_PAGE_INT8 || TYPE == RFSN_PAGE_E4M3)
        dot *= ((const float*)p.k_scale)[sc], vs = ((const float*)p.v_scale)[sc];
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
      const int64_t sci = ((int64_t)__builtin_amdgcn_readlane((int)(sc >> 32), i) << 32) |
                          (uint32_t)__builtin_amdgcn_readlane((int)sc, i);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float x;
        const int64_t o = vo + lane * E + e;
        if constexpr (TYPE == RFSN_PAGE_FP16) x = h2f(((const uint16_t*)p.v)[o]);
        else if constexpr (TYPE == RFSN_PAGE_INT8) x = (float)((const int8_t*)p.v)[o] * si;
        else if constexpr (TYPE == RFSN_PAGE_E2M1)
          x = (float)e2m1_f16((uint32_t)((const uint8_t*)p.v)[o / 2] >> (4 * (int)(o & 1)),
                              group_scale(((const uint8_t*)p.v_scale)[sci * (D / 16) + (lane * E + e) / 16]))[0];
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

// x - y[I], exact where y[I] is x rounded: one operation that takes y as fp16.
template <int I>
__device__ __forceinline__ float less(float x, half2w y) {
  float r;
  if constexpr (I == 0) asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(y), "v"(x));
  else asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(y), "v"(x));
  return r;
}

// 16 or 8 bytes of a row, marked as not to be kept where the call reads more than the caches hold (Plan).
template <bool kOnce, typename V>
__device__ __forceinline__ V load_piece(const uint8_t* a) {
  if constexpr (kOnce) return __builtin_nontemporal_load(reinterpret_cast<const V*>(a));
  else return *reinterpret_cast<const V*>(a);
}
template <int N>
__device__ __forceinline__ uint32_t load_scales(const uint8_t* a) {
  if constexpr (N == 1) return *a;
  else return *reinterpret_cast<const uint16_t*>(a);
}

// Blocks of 4 waves that registers are to leave room for (4-bit rows of 128: 139 registers, three blocks a CU; 127, four: 60
// ragged sequences of up to 9,000, 8 heads, 35.4 -> 33.3 us; with weights it would spill).
constexpr int blocks_per_cu(int D, int type, bool weigh) {
  return D == 64 || (D == 128 && type == RFSN_PAGE_E2M1 && !weigh) ? 4 : D == 128 || type == RFSN_PAGE_E2M1 ? 2 : 1;
}

template <int D, int TYPE, int kWaves, bool kOnce, bool kWeigh>
__global__ void __launch_bounds__(kWaves * 64, kWaves > 4 ? 1 : blocks_per_cu(D, TYPE, kWeigh))
paged_attn_kernel(const rfsn_paged p, int shift, const int32_t* __restrict__ table, const uint16_t* __restrict__ q, int G,
                  float scale_log2, const int32_t* __restrict__ chosen, int count, const Cut cut,
                  uint16_t* __restrict__ out, const Parts parts) {
  constexpr bool kCodes = TYPE == RFSN_PAGE_INT8 || TYPE == RFSN_PAGE_E4M3;
  constexpr bool kSmall = TYPE == RFSN_PAGE_E2M1;    // codes that are fp16 values by the time they are operands
  constexpr int E = D / 64;
  constexpr int RB = row_bytes<TYPE>(D);             // bytes of a stored row
  constexpr int LB = RB < 64 ? RB / 4 : 16;          // bytes of a lane's load
  constexpr int KS = D / 32;                         // MFMA k steps of a score
  constexpr int KL = RB / (4 * LB);                  // loads of a lane's share of a K row
  constexpr int DT = D / 16;                         // 16-coordinate tiles of O^T
  constexpr int VC = RB / LB;                        // such pieces of a stored row
  constexpr int kTile = 16 * NG;                     // positions per wave and step
  constexpr int GT = 64 / NG;                        // tiles whose groups fill a wave's lanes
  constexpr int VU = 16 * VC / 64;                   // V loads of a lane for a group
  constexpr int SB = LB / 8;                         // 4-bit codes: scale bytes that go with a load
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
      qf[s] = *reinterpret_cast<const half8v*>(qr + (kCodes   ? (s >> 1) * 64 + grp * 16 + (s & 1) * 8
                                                     : kSmall ? s / (LB / 4) * (LB * 8) + grp * (LB * 2) + s % (LB / 4) * 8
                                                              : s * 32 + grp * 8));
    // 4 bits: columns without a head stay 0, weights too (m_run below), which spares the matrix cores' power: 32 x 32,768
    // positions, 8 KV heads of 64, again and again 160 us, so 146
    if (kSmall && col >= heads)
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[s] = half8v{};
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
  float m_run = kSmall && col >= heads ? 0x1p100f : -__builtin_inff(), l_run = 0.f;  // reference exponent of the head's weights, this lane's sum of them

  typedef std::conditional_t<LB == 16, uint4w, uint2v> piece;
  piece kr[NG][KL], vr[NG][VU];
  float4v ks[NG], vs[NG];
  uint32_t kb8[NG][KL], vb8[NG][VU];  // scale bytes of 4-bit codes
  int n_next[NG] = {};  // rows of the fetched groups that are attended
  const int64_t page_bytes = p.page_stride * RB / D, head_bytes = p.head_stride * RB / D;
  const uint8_t* const k0 = (const uint8_t*)p.k + h * head_bytes;
  const uint8_t* const v0 = (const uint8_t*)p.v + h * head_bytes;
  constexpr int kScale = kSmall ? D / 16 : 4;  // bytes of a row's scales
  const int64_t scale_page = (int64_t)p.kv_heads * p.page_size * kScale;
  const uint8_t* const ks0 = (const uint8_t*)p.k_scale + (int64_t)h * p.page_size * kScale;
  const uint8_t* const vs0 = (const uint8_t*)p.v_scale + (int64_t)h * p.page_size * kScale;
  // Rows past the last one attended re-read it: their weights are 0.  A group with none
  // reads page 0, and its V is not used.  Of 4-bit pages all 16 rows are read, which are the
  // page's own, and the scales of those that are not attended taken as 0.
  auto fetch = [&](int t, int tile) {
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      const int page = __builtin_amdgcn_readlane(page_l, NG * (tile % GT) + u);
      const int n = __builtin_amdgcn_readlane(rows_l, NG * (tile % GT) + u);
      const int row = (t + 16 * u) & (p.page_size - 1);
      n_next[u] = n;
      const int last = n > 0 ? n - 1 : 0;
      const int64_t base = page * page_bytes + row * RB;
      const uint8_t* kb = k0 + base;
      const uint8_t* vb = v0 + base;
      const uint32_t kl = (uint32_t)((kSmall ? col : min(col, last)) * RB + grp * LB);
#pragma unroll
      for (int i = 0; i < KL; ++i) kr[u][i] = load_piece<kOnce, piece>(kb + kl + i * (4 * LB));
#pragma unroll
      for (int i = 0; i < VU; ++i) {
        const int idx = i * 64 + lane, r = idx / VC, ch = idx % VC;
        vr[u][i] = load_piece<kOnce, piece>(vb + (uint32_t)((kSmall ? r : min(r, last)) * RB + ch * LB));
      }
      if constexpr (kSmall) {
        const int64_t sc = page * scale_page + row * kScale;
#pragma unroll
        for (int i = 0; i < KL; ++i) kb8[u][i] = load_scales<SB>(ks0 + sc + (uint32_t)(col * kScale + (i * 4 + grp) * SB));
#pragma unroll
        for (int i = 0; i < VU; ++i) vb8[u][i] = load_scales<SB>(vs0 + sc + (uint32_t)((i * 64 + lane) * SB));
      }
      if constexpr (kCodes) {
        const int64_t sc = page * scale_page + row * kScale;
        ks[u] = *reinterpret_cast<const float4v*>(ks0 + sc + (uint32_t)(grp * 16));
        vs[u] = *reinterpret_cast<const float4v*>(vs0 + sc + (uint32_t)(grp * 16));
      }
    }
  };
  // 4 bits: a positive scale is left to the subtraction of the maximum (another would turn a masked score's infinity)
  const bool late = kSmall && scale_log2 > 0.f;
  const float factor = late ? scale_log2 : 1.f;
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
        piece x = vr[u][i];
        if (!kSmall && n[u] == 0) x = piece{};
        if constexpr (kSmall) {
          uint32_t sb = vb8[u][i];
          if (n[u] < 16 && idx / VC >= n[u]) sb = 0;  // (codes are finite)
#pragma unroll
          for (int c = 0; c < LB / 4; ++c)
            sv[r * CH + ((ch * (LB / 4) + c) ^ v_swz<D>(r))] =
                __builtin_bit_cast(uint4w, e2m1_f16(x[c], group_scale((sb >> (c / 2 * 8)) & 255u)));
        } else if constexpr (!kCodes) {
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
        if constexpr (kSmall) kf = e2m1_f16(kr[u][k / (LB / 4)][k % (LB / 4)], group_scale((kb8[u][k / (LB / 4)] >> (k % (LB / 4) / 2 * 8)) & 255u));
        else if constexpr (!kCodes) kf = __builtin_bit_cast(half8v, kr[u][k]);
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
      if (!late) s[u] *= scale_log2;
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
    // The scores of 32 x 32,768 positions, 134 MB, cost fp16 pages 140 us: what is read with them comes at 4.9 TB/s and not 6.5, as in a
    // copy.  Stored past the caches 480, without a branch (no wait for them, then) 466 as here.
    if constexpr (kWeigh) {
#pragma unroll
      for (int u = 0; u < NG; ++u)
        if (n[u] > 0 && col < heads)
          *reinterpret_cast<float4v*>(parts.score + score_at(((int64_t)b * p.kv_heads + h) * parts.positions, G, g0 + col, t + 16 * u) + grp * 4) =
              kSmall ? s[u] * factor : s[u];
    }
    float pw[4 * NG], ls;
    auto weights = [&]() {
      const float mb = m_run > -__builtin_inff() ? m_run : 0.f;
      ls = 0.f;
#pragma unroll
      for (int i = 0; i < 4 * NG; ++i) {
        pw[i] = __builtin_amdgcn_exp2f(kSmall ? fmaf(s[i >> 2][i & 3], factor, -mb) : s[i >> 2][i & 3] - mb);
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
      if constexpr (kSmall) mx *= factor;
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
        const half2w lo = {(f16)less<0>(pw[2 * i], hi), (f16)less<1>(pw[2 * i + 1], hi)};
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
        if constexpr (kWeigh)
          if (lane == 0) parts.fin[2 * row] = m, parts.fin[2 * row + 1] = l;
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
  if constexpr (kWeigh)
    if (parts.ml == nullptr && wave == 0 && grp == 0 && col < heads) parts.fin[2 * (row0 + col)] = m, parts.fin[2 * (row0 + col) + 1] = l;
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
__device__ __forceinline__ void merge_row(const rfsn_paged& p, int shift, int q_heads, int per_seq, const Parts& parts,
                                          uint16_t* __restrict__ out, int i, int b, float (&s_acc)[W][D]) {
  constexpr int E = D / 64, U = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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

template <int D, int W>
__global__ void __launch_bounds__(W * 64)
paged_merge_kernel(const rfsn_paged p, int shift, int q_heads, int per_seq, const Parts parts, uint16_t* __restrict__ out) {
  __shared__ float s_acc[W][D];
  merge_row<D, W>(p, shift, q_heads, per_seq, parts, out, blockIdx.x, blockIdx.y, s_acc);
}

// Whether 16 waves share a row's chunks, or 4.
inline bool merge_in_16(const rfsn_paged& p, const Plan& c, int q_heads) {
  return c.split() && (c.cut.per_seq ? c.cut.per_seq : c.slots - p.batch + 1) > 16 && (int64_t)q_heads * p.batch <= 256;
}

// The blocks of a checked call.
template <bool kWeigh>
int attend_launch(const rfsn_paged* p, const Plan& c, const void* q, int q_heads, float sl2, const int32_t* chosen, int count,
                  void* out, const Parts& parts, hipStream_t s) {
  const int shift = paged_shift(*p), G = q_heads / p->kv_heads;
  const dim3 grid((unsigned)p->kv_heads, (unsigned)c.slots, (unsigned)ceil_div(G, 16));
#define RFSN_ATTEND(DD, TT, NW, ONCE)                                                                               \
  hipLaunchKernelGGL((paged_attn_kernel<DD, TT, NW, ONCE, kWeigh>), grid, dim3(NW * 64), 0, s, *p, shift, p->table,           \
                     (const uint16_t*)q, G, sl2, chosen, count, c.cut, (uint16_t*)out, parts)
#define RFSN_ATTEND_D(DD, NW, ONCE)                                                \
  do {                                                                             \
    if (p->type == RFSN_PAGE_FP16) RFSN_ATTEND(DD, RFSN_PAGE_FP16, NW, ONCE);      \
    else if (p->type == RFSN_PAGE_INT8) RFSN_ATTEND(DD, RFSN_PAGE_INT8, NW, ONCE); \
    else if (p->type == RFSN_PAGE_E4M3) RFSN_ATTEND(DD, RFSN_PAGE_E4M3, NW, ONCE); \
    else RFSN_ATTEND(DD, RFSN_PAGE_E2M1, NW, ONCE);                                \
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
  return check_launch("paged_attention");
}

}  // namespace

// The call with accumulated weights, and then the weights (paged_weigh.hip).
int launch_weigh(const rfsn_paged* p, const Plan& c, const void* q, int q_heads, float sl2, void* out, const Parts& parts,
                 hipStream_t s);

}  // namespace rfsn
