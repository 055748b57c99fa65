// Attention over a paged KV cache that adds each position's softmax weight to its row's.
//
//   weight[row of t] += sum_i e^(s_it - m_i) / l_i   over the KV head's query heads i
//
// with the scores s as the attention's blocks had them (4 bytes per position and query head, written once and read
// once: 8 G bytes of G query heads, where K again would be 9/16 D to 2 D per position and its products once more; of 4-bit rows
// of 64 that is less from G = 8 on, and has not been built) and the (m, l) of whole sequences, which only the end of the attention
// knows: one launch behind it joins the chunks' results and adds the weights, each of its blocks joining the (m, l) that it
// needs by itself.  A position belongs to one thread, so that nothing depends on an order.
//
// Bound: HBM where there is enough of it (32 x 32,768 positions, 32 query heads over 8 of 64, fp16: 2.5 GB, the scores
// twice among them, in 500 us, 4.9 TB/s with reads and writes mixed; 333 without weights), below it the loads in turn of two launches
// (32 ragged sequences of up to 20,000, 32 query heads over 4: 14.5 + 8.6 us, K and V at 3.8 TB/s; 8,191 of one, 4 bits: 8.7 + 5.4).
// Calls with weights and without, us: 32 x 5,000 positions, 32 query heads over 8 of 64, int8 44.4 and 35.3, e4m3 44.2 and
// 33.7; 16 x 8,192 of 128 69.8 and 52.3, 69.0 and 51.9; 4 bits, 32 x 32,768 of 64, 4, 8 and 16 query heads of each of 8: 185,
// 241 and 362, and 135, 150 and 140.
#include "paged_attention.h"

namespace rfsn {
namespace {

constexpr int kWeighHeads = 64;  // query heads whose (m, 1 / l) a block holds at a time

// (m, 1 / l) of query heads first .. first + count - 1 of sequence b, each by one wave: (0, 0) without weights.
template <int W>
__device__ __forceinline__ void join_sums(const rfsn_paged& p, int shift, int q_heads, int per_seq, bool split, const Parts& parts,
                                          int b, int first, int count, float (&m_of)[kWeighHeads], float (&inv_of)[kWeighHeads]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int slot0 = 0, n = 0;
  if (split) {
    slot0 = per_seq ? b * per_seq : parts.seq[2 * b];
    n = per_seq ? per_seq : parts.seq[2 * b + 1];
  }
  constexpr int U = 4;  // heads whose loads a wave has in flight
  for (int g = wave * U; g < count; g += W * U) {
    float m[U], l[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = -__builtin_inff(), l[u] = 0.f;
      if (split) continue;
      const int64_t row = (int64_t)b * q_heads + first + min(g + u, count - 1);
      m[u] = parts.fin[2 * row], l[u] = parts.fin[2 * row + 1];
    }
    for (int base = 0; base < n; base += 64) {
      float2w x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t s = (int64_t)(slot0 + min(base + lane, n - 1)) * q_heads + first + min(g + u, count - 1);
        x[u] = *reinterpret_cast<const float2w*>(parts.ml + 2 * s);
        if (base + lane >= n) x[u] = float2w{-__builtin_inff(), 0.f};
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float mj = x[u][0], mn = fmaxf(m[u], wave_max(mj)), mref = mn > -__builtin_inff() ? mn : 0.f;
        const float corr = m[u] > -__builtin_inff() ? exp2f(m[u] - mref) : 1.f;
        const float wj = mj > -__builtin_inff() ? exp2f(mj - mref) : 1.f;  // with m -infinite the sums are 0 or NaN
        l[u] = l[u] * corr + wave_sum(wj * x[u][1]);
        m[u] = mn;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (lane == 0 && g + u < count) m_of[g + u] = l[u] == 0.f ? 0.f : m[u], inv_of[g + u] = l[u] == 0.f ? 0.f : 1.f / l[u];
  }
}

// Blocks 0 .. merges - 1 join a row of results each (as many waves as without weights: the same bits), the others take `across`
// blocks of 1,024 positions of each (sequence, head).
template <int D, int W>
__global__ void __launch_bounds__(W * 64)
paged_weigh_kernel(const rfsn_paged p, int shift, int q_heads, int per_seq, int split, int merges, int across, const Parts parts,
                   uint16_t* __restrict__ out) {
  constexpr int V = 16 / W;  // positions of a thread
  typedef float vec __attribute__((ext_vector_type(V)));
  __shared__ float s_acc[W][D];
  __shared__ float s_m[kWeighHeads], s_inv[kWeighHeads];
  if ((int)blockIdx.x < merges) {
    merge_row<D, W>(p, shift, q_heads, per_seq, parts, out, blockIdx.x % q_heads, blockIdx.x / q_heads, s_acc);
    return;
  }
  const int item = blockIdx.x - merges, G = q_heads / p.kv_heads;
  const int x = item % across, h = item / across % p.kv_heads, b = item / across / p.kv_heads;
  const int len = paged_len(p, shift, b);
  const int64_t from = ((int64_t)b * p.kv_heads + h) * parts.positions;
  const int64_t stride = (int64_t)across * 1024;
  // (block-uniform) rounds of the longest block of the sequence's
  for (int64_t t0 = (int64_t)x * 1024; t0 < len; t0 += stride) {
    const int64_t t = t0 + threadIdx.x * V;
    const int page = t < len ? paged_page(p, b, t >> shift) : -1;
    vec w = {};
    for (int g0 = 0; g0 < G; g0 += kWeighHeads) {
      const int count = min(kWeighHeads, G - g0);
      if (t0 == (int64_t)x * 1024 || G > kWeighHeads) {
        __syncthreads();
        join_sums<W>(p, shift, q_heads, per_seq, split, parts, b, h * G + g0, count, s_m, s_inv);
        __syncthreads();
      }
      if (page < 0) continue;
      const float* s = parts.score + score_at(from, G, g0, t & ~15ll) + (t & 15);
#pragma unroll 4
      for (int g = 0; g < count; ++g) {
        const vec sg = *reinterpret_cast<const vec*>(s + g * 16);
        const float m = s_m[g], inv = s_inv[g];
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] += __builtin_amdgcn_exp2f(sg[e] - m) * inv;
      }
    }
    if (page < 0) continue;
    float* at = p.weight + ((int64_t)page * p.kv_heads + h) * p.page_size + (t & (p.page_size - 1));
    if (t + V <= len) {
      *reinterpret_cast<vec*>(at) += w;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (t + e < len) at[e] += w[e];
    }
  }
}

}  // namespace

int launch_weigh(const rfsn_paged* p, const Plan& c, const void* q, int q_heads, float sl2, void* out, const Parts& parts,
                 hipStream_t s) {
  if (int st = attend_launch<true>(p, c, q, q_heads, sl2, nullptr, 0, out, parts, s)) return st;
  // blocks of 1,024 positions, as many as some 4,096 blocks in all leave to a (sequence, head)
  const int64_t heads = (int64_t)p->kv_heads * p->batch, merges = c.split() ? (int64_t)q_heads * p->batch : 0;
  int64_t across = ceil_div(4096, heads);
  if (across > ceil_div(parts.positions, 1024)) across = ceil_div(parts.positions, 1024);
  if (across * heads + merges == 0) return RFSN_OK;
  RFSN_REQUIRE(across * heads + merges < (1ll << 31), "paged_attention: too many sequences");
#define RFSN_WEIGH_W(DD, W)                                                                                              \
  hipLaunchKernelGGL((paged_weigh_kernel<DD, W>), dim3((unsigned)(across * heads + merges)), dim3(W * 64), 0, s, *p,     \
                     paged_shift(*p), q_heads, c.cut.per_seq, (int)c.split(), (int)merges, (int)(across > 0 ? across : 1), \
                     parts, (uint16_t*)out)
#define RFSN_WEIGH(DD)                             \
  do {                                             \
    if (merge_in_16(*p, c, q_heads)) RFSN_WEIGH_W(DD, 16); \
    else RFSN_WEIGH_W(DD, 4);                      \
  } while (0)
  if (p->head_dim == 64) RFSN_WEIGH(64);
  else if (p->head_dim == 128) RFSN_WEIGH(128);
  else RFSN_WEIGH(256);
#undef RFSN_WEIGH
#undef RFSN_WEIGH_W
  return check_launch("paged_attention");
}

}  // namespace rfsn
