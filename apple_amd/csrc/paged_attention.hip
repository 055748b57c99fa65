// The entry points of the paged attention (kernels: paged_attention.h).
#include "paged_attention.h"

namespace rfsn {
namespace {

// Where a call's parts lie in its workspace, 16-byte aligned each; `end` is its size.
struct Room {
  size_t acc, ml, seq, score, fin, end;
};
Room room(const rfsn_paged& p, const Plan& c, int q_heads) {
  Room r = {};
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t from = at;
    at += (bytes + 15) & ~(size_t)15;
    return from;
  };
  if (c.split()) {
    r.acc = take((size_t)c.slots * q_heads * p.head_dim * sizeof(float));
    r.ml = take((size_t)c.slots * q_heads * 2 * sizeof(float));
    r.seq = take((size_t)p.batch * 2 * sizeof(int32_t));
  }
  if (p.weight) {
    r.score = take((size_t)p.batch * q_heads * p.table_width * p.page_size * sizeof(float));
    r.fin = take((size_t)p.batch * q_heads * 2 * sizeof(float));
  }
  r.end = at;
  return r;
}

}  // namespace
}  // namespace rfsn

using namespace rfsn;

extern "C" size_t rfsn_paged_attention_workspace_bytes(const rfsn_paged* p, int32_t q_heads, int32_t count) {
  if (p == nullptr || p->batch <= 0 || p->kv_heads <= 0 || p->page_size <= 0 || q_heads < p->kv_heads || count < 0) return 0;
  return room(*p, plan(*p, q_heads, count), q_heads).end;
}

extern "C" int rfsn_paged_attention(const rfsn_paged* p, const void* q, int32_t q_heads, float scale,
                                    const int32_t* chosen, int32_t count, void* out, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (int st = paged_check(p, "paged_attention")) return st;
  RFSN_REQUIRE(q_heads > 0 && q_heads % p->kv_heads == 0 && q_heads <= 65535,
               "paged_attention: q_heads must be a multiple of kv_heads");
  RFSN_REQUIRE((chosen == nullptr) == (count == 0) && count >= 0, "paged_attention: chosen and count go together");
  RFSN_REQUIRE((int64_t)count * p->page_size <= (1ll << 31) - 1024, "paged_attention: too many chosen pages");
  RFSN_REQUIRE(chosen == nullptr || p->weight == nullptr, "paged_attention: weights are of whole sequences, not of chosen pages");
  RFSN_REQUIRE(p->weight == nullptr || p->batch <= 1 || p->table_stride != 0,
               "paged_attention: weights of sequences that share a table");
  const float sl2 = scale * 1.44269504088896340736f;
  RFSN_REQUIRE(sl2 == sl2 && sl2 < __builtin_inff() && sl2 > -__builtin_inff(),
               "paged_attention: scale must be finite, in base 2 as well");
  if (p->batch == 0) return RFSN_OK;
  RFSN_REQUIRE(q && out && ((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0,
               "paged_attention: q and out must be 16-byte aligned");
  const Plan c = plan(*p, q_heads, count);
  const Room r = room(*p, c, q_heads);
  RFSN_REQUIRE(workspace_bytes >= r.end && ((workspace && ((uintptr_t)workspace & 15) == 0) || r.end == 0),
               "paged_attention: workspace too small or misaligned");
  RFSN_REQUIRE(c.slots <= 65535, "paged_attention: too many sequences");
  char* const w = (char*)workspace;
  Parts parts = {};
  if (c.split()) parts.acc = (float*)(w + r.acc), parts.ml = (float*)(w + r.ml), parts.seq = (int32_t*)(w + r.seq);
  if (p->weight == nullptr) {
    const hipStream_t s = (hipStream_t)stream;
    const int shift = paged_shift(*p);
    if (int st = attend_launch<false>(p, c, q, q_heads, sl2, chosen, count, out, parts, s)) return st;
    if (c.split()) {
      const dim3 rows((unsigned)q_heads, (unsigned)p->batch);
      const bool many = merge_in_16(*p, c, q_heads);
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
  parts.score = (float*)(w + r.score), parts.fin = (float*)(w + r.fin);
  parts.positions = (int64_t)p->table_width * p->page_size;
  return launch_weigh(p, c, q, q_heads, sl2, out, parts, (hipStream_t)stream);
}
