// Attention over a paged KV cache that adds each position's softmax weight to its row's.
//
//   weight[row of t] += sum_i e^(s_it - m_i) / l_i   over the KV head's query heads i
//
// with the scores s as the attention's blocks had them (4 bytes per position and query head, written once
// and read once) and the (m, l) of whole sequences, which only the end of the attention knows.  A position belongs to one
// thread, so that nothing depends on an order.
#include "paged_attention.h"

namespace rfsn {
namespace {

__global__ void __launch_bounds__(256)
paged_weigh_kernel(const rfsn_paged p, int shift, int G, const Parts parts) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int len = paged_len(p, shift, b);
  const int64_t row0 = ((int64_t)b * p.kv_heads + h) * G;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < len; t += (int64_t)gridDim.x * 256) {
    const int page = paged_page(p, b, t >> shift);
    if (page < 0) continue;
    float w = 0.f;
    for (int g = 0; g < G; ++g) {
      const float m = parts.fin[2 * (row0 + g)], l = parts.fin[2 * (row0 + g) + 1];
      const float s = parts.score[(row0 + g) * parts.positions + t];
      if (l != 0.f) w += __builtin_amdgcn_exp2f(s - m) / l;
    }
    p.weight[((int64_t)page * p.kv_heads + h) * p.page_size + (t & (p.page_size - 1))] += w;
  }
}

}  // namespace

int launch_weigh(const rfsn_paged* p, const Plan& c, const void* q, int q_heads, float sl2, void* out, const Parts& parts,
                 hipStream_t s) {
  if (int st = attend_launch<true>(p, c, q, q_heads, sl2, nullptr, 0, out, parts, s)) return st;
  if (parts.positions == 0) return RFSN_OK;
  int64_t x = ceil_div(parts.positions, 256);
  if (x > 1024) x = 1024;
  hipLaunchKernelGGL(paged_weigh_kernel, dim3((unsigned)x, (unsigned)p->kv_heads, (unsigned)p->batch), dim3(256), 0, s, *p,
                     paged_shift(*p), q_heads / p->kv_heads, parts);
  return check_launch("paged_attention");
}

}  // namespace rfsn
