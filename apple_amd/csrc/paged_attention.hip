// Attention of one query per sequence over a paged KV cache (attention.py:39-105
// for a batch of paged windows), over all positions or a list of pages.
//
//   out_i = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),  s_t = scale q_i . k_t
//
// A block takes a chunk of positions of one (sequence, KV head) with all of its
// query heads; chunks are cut by the sum of the lengths, which only the device
// knows (find_chunk), and a second kernel joins their (m, l, acc).
#include "paged.h"

namespace rfsn {
namespace {

constexpr int kUnit = 128;       // chunks are multiples of this many positions
constexpr int kMinChunk = 512;   // and no shorter
constexpr int kBlocks = 1024;    // blocks a launch aims at

__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((long long)v, o, 64);
  return v;
}

// Positions per chunk of a batch: at most `target` chunks over the sum of the
// lengths, one more per sequence for its last, shorter one.
__device__ __forceinline__ int64_t chunk_size(const rfsn_paged& p, int shift, int target, int lane) {
  int64_t total = 0;
  for (int b = lane; b < p.batch; b += 64) total += paged_len(p, shift, b);
  total = wave_sum64(total);
  int64_t c = (total + target - 1) / target;
  c = (c + kUnit - 1) / kUnit * kUnit;
  return c < kMinChunk ? kMinChunk : c;
}

// Chunks of the sequences before b.
__device__ __forceinline__ int chunks_before(const rfsn_paged& p, int shift, int64_t size, int b, int lane) {
  int64_t n = 0;
  for (int i = lane; i < b; i += 64) n += (paged_len(p, shift, i) + size - 1) / size;
  return (int)wave_sum64(n);
}

struct Chunk {
  int b;       // sequence, -1: none
  int64_t t0, t1;
};
// Chunk number w of the batch, by one wave.
__device__ __forceinline__ Chunk find_chunk(const rfsn_paged& p, int shift, int64_t size, int w, int lane) {
  int seen = 0;
  for (int base = 0; base < p.batch; base += 64) {
    const int b = base + lane;
    const int len = b < p.batch ? paged_len(p, shift, b) : 0;
    const int n = (int)((len + size - 1) / size);
    int upto = n;  // inclusive prefix over the wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o, 64);
      if (lane >= o) upto += x;
    }
    const uint64_t in = __ballot(w < seen + upto && w >= seen + upto - n);
    if (in) {
      const int src = __ffsll((unsigned long long)in) - 1;
      const int64_t t0 = (int64_t)(w - seen - __shfl(upto - n, src, 64)) * size;
      const int64_t end = __shfl(len, src, 64);
      return {base + src, t0, t0 + size < end ? t0 + size : end};
    }
    seen += __shfl(upto, 63, 64);
  }
  return {-1, 0, 0};
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

// per_seq > 0: every sequence has that many chunks of chunk_fixed listed
// positions (a list of pages, or one chunk); 0: cut by the lengths.
template <int D, int TYPE>
__global__ void __launch_bounds__(256)
paged_attn_kernel(const rfsn_paged p, int shift, const uint16_t* __restrict__ q, int G, float scale_log2,
                  const int32_t* __restrict__ chosen, int count, int per_seq, int64_t chunk_fixed, int target,
                  uint16_t* __restrict__ out, float* __restrict__ part_acc, float* __restrict__ part_ml) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.x, w = blockIdx.y;
  Chunk c;
  if (per_seq) {
    c.b = w / per_seq;
    c.t0 = (int64_t)(w % per_seq) * chunk_fixed;
    const int64_t end = chosen ? (int64_t)count << shift : paged_len(p, shift, c.b);
    c.t1 = c.t0 + chunk_fixed < end ? c.t0 + chunk_fixed : end;
  } else {
    c = find_chunk(p, shift, chunk_size(p, shift, target, lane), w, lane);
    if (c.b < 0) return;
  }
  const int32_t* list = chosen ? chosen + ((int64_t)c.b * p.kv_heads + h) * count : nullptr;
  for (int g = wave; g < G; g += 4) {
    const int64_t row = ((int64_t)c.b * p.kv_heads + h) * G + g;
    float m, l, acc[E];
    attend_row<D, TYPE>(p, shift, list, c.b, h, c.t0, c.t1, q + row * D, scale_log2, lane, m, l, acc);
    if (part_ml == nullptr) {
#pragma unroll
      for (int e = 0; e < E; ++e) out[row * D + lane * E + e] = f2h(l == 0.f ? 0.f : acc[e] / l);
    } else {
      const int64_t slot = ((int64_t)w * p.kv_heads + h) * G + g;
      if (lane == 0) part_ml[2 * slot] = m, part_ml[2 * slot + 1] = l;
#pragma unroll
      for (int e = 0; e < E; ++e) part_acc[slot * D + lane * E + e] = acc[e];
    }
  }
}

// out = sum_j w_j acc_j / sum_j w_j l_j over a sequence's chunks, w_j = 2^(m_j - max m).
template <int D>
__global__ void __launch_bounds__(256)
paged_merge_kernel(const rfsn_paged p, int shift, int q_heads, int per_seq, int target, const float* __restrict__ part_acc,
                   const float* __restrict__ part_ml, uint16_t* __restrict__ out) {
  constexpr int E = D / 64;
  __shared__ float s_l[4], s_acc[4][D];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = blockIdx.x, b = blockIdx.y;
  int slot0, n;
  if (per_seq) {
    slot0 = b * per_seq, n = per_seq;
  } else {
    const int64_t size = chunk_size(p, shift, target, lane);
    slot0 = chunks_before(p, shift, size, b, lane);
    n = (int)((paged_len(p, shift, b) + size - 1) / size);
  }
  float mx = -__builtin_inff();
  for (int j = lane; j < n; j += 64) mx = fmaxf(mx, part_ml[2 * ((int64_t)(slot0 + j) * q_heads + i)]);
  mx = wave_max(mx);
  float l = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int j = wave; j < n; j += 4) {
    const int64_t s = (int64_t)(slot0 + j) * q_heads + i;
    const float m = part_ml[2 * s];
    const float w = m > -__builtin_inff() ? exp2f(m - mx) : 1.f;  // with m -infinite the sums are 0 or NaN
    l += w * part_ml[2 * s + 1];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(w, part_acc[s * D + lane * E + e], acc[e]);
  }
  if (lane == 0) s_l[wave] = l;
#pragma unroll
  for (int e = 0; e < E; ++e) s_acc[wave][lane * E + e] = acc[e];
  __syncthreads();
  const float total = s_l[0] + s_l[1] + s_l[2] + s_l[3];
  for (int d = threadIdx.x; d < D; d += 256) {
    const float a = s_acc[0][d] + s_acc[1][d] + s_acc[2][d] + s_acc[3][d];
    out[((int64_t)b * q_heads + i) * D + d] = f2h(total == 0.f ? 0.f : a / total);
  }
}

// Chunks of a call: slots of partial results, chunks per sequence (0: cut by the
// lengths on the device), their size, and the number the device aims at.
struct Plan {
  int64_t slots;
  int per_seq;
  int64_t chunk;
  int target;
  bool split() const { return per_seq != 1; }
};
Plan plan(const rfsn_paged& p, int count) {
  const int64_t most = (int64_t)(count ? count : p.table_width) * p.page_size;
  const int64_t want = ceil_div(kBlocks, p.kv_heads);  // chunks that fill the chip
  if (most <= kMinChunk) return {p.batch, 1, kMinChunk, 0};
  if (count) {
    int64_t n = ceil_div(want, p.batch);
    if (n > ceil_div(most, kMinChunk)) n = ceil_div(most, kMinChunk);
    const int64_t chunk = ceil_div(ceil_div(most, n), kUnit) * kUnit;
    n = ceil_div(most, chunk);
    return {n * p.batch, (int)n, chunk, 0};
  }
  int64_t target = want;
  if (target > ceil_div(most, kMinChunk) * p.batch) target = ceil_div(most, kMinChunk) * p.batch;
  return {target + p.batch, 0, 0, (int)target};
}

}  // namespace
}  // namespace rfsn

using namespace rfsn;

extern "C" size_t rfsn_paged_attention_workspace_bytes(const rfsn_paged* p, int32_t q_heads, int32_t count) {
  if (p == nullptr || p->batch <= 0 || p->kv_heads <= 0 || p->page_size <= 0 || q_heads <= 0 || count < 0) return 0;
  const Plan c = plan(*p, count);
  return c.split() ? (size_t)c.slots * q_heads * (p->head_dim + 2) * sizeof(float) : 0;
}

extern "C" int rfsn_paged_attention(const rfsn_paged* p, const void* q, int32_t q_heads, float scale,
                                    const int32_t* chosen, int32_t count, void* out, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (int st = paged_check(p, "paged_attention")) return st;
  RFSN_REQUIRE(q_heads > 0 && q_heads % p->kv_heads == 0 && q_heads <= 65535,
               "paged_attention: q_heads must be a multiple of kv_heads");
  RFSN_REQUIRE((chosen == nullptr) == (count == 0) && count >= 0, "paged_attention: chosen and count go together");
  RFSN_REQUIRE((int64_t)count * p->page_size < (1ll << 31), "paged_attention: too many chosen pages");
  RFSN_REQUIRE(scale == scale && scale < __builtin_inff() && scale > -__builtin_inff(),
               "paged_attention: scale must be finite");
  if (p->batch == 0) return RFSN_OK;
  RFSN_REQUIRE(q && out && ((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0,
               "paged_attention: q and out must be 16-byte aligned");
  const Plan c = plan(*p, count);
  RFSN_REQUIRE(workspace_bytes >= rfsn_paged_attention_workspace_bytes(p, q_heads, count) && (workspace || !c.split()),
               "paged_attention: workspace too small");
  RFSN_REQUIRE(c.slots <= 65535, "paged_attention: too many sequences");
  const hipStream_t s = (hipStream_t)stream;
  const int shift = paged_shift(*p), G = q_heads / p->kv_heads;
  const float sl2 = scale * 1.44269504088896340736f;
  float* acc = c.split() ? (float*)workspace : nullptr;
  float* ml = c.split() ? acc + c.slots * q_heads * p->head_dim : nullptr;
#define RFSN_ATTEND(DD, TT)                                                                                            \
  hipLaunchKernelGGL((paged_attn_kernel<DD, TT>), dim3((unsigned)p->kv_heads, (unsigned)c.slots), dim3(256), 0, s, *p, \
                     shift, (const uint16_t*)q, G, sl2, chosen, count, c.per_seq, c.chunk, c.target, (uint16_t*)out,   \
                     acc, ml)
#define RFSN_ATTEND_D(DD)                                            \
  do {                                                               \
    if (p->type == RFSN_PAGE_FP16) RFSN_ATTEND(DD, RFSN_PAGE_FP16);  \
    else if (p->type == RFSN_PAGE_INT8) RFSN_ATTEND(DD, RFSN_PAGE_INT8); \
    else RFSN_ATTEND(DD, RFSN_PAGE_E4M3);                            \
  } while (0)
  if (p->head_dim == 64) RFSN_ATTEND_D(64);
  else if (p->head_dim == 128) RFSN_ATTEND_D(128);
  else RFSN_ATTEND_D(256);
#undef RFSN_ATTEND_D
#undef RFSN_ATTEND
  if (int st = check_launch("paged_attention")) return st;
  if (c.split()) {
    const dim3 grid((unsigned)q_heads, (unsigned)p->batch);
#define RFSN_MERGE(DD)                                                                                            \
  hipLaunchKernelGGL(paged_merge_kernel<DD>, grid, dim3(256), 0, s, *p, shift, q_heads, c.per_seq, c.target, acc, ml, \
                     (uint16_t*)out)
    if (p->head_dim == 64) RFSN_MERGE(64);
    else if (p->head_dim == 128) RFSN_MERGE(128);
    else RFSN_MERGE(256);
#undef RFSN_MERGE
  }
  return check_launch("paged_attention");
}
