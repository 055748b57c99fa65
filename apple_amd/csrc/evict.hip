// Eviction from a paged KV cache by accumulated attention weight: per sequence and KV head the positions that
// stay, then their rows to the front of the sequence's own pages, then the pages' bounds.
#include "choose.h"
#include "paged.h"

namespace rfsn {
namespace {

// Table entry of a position below the sequence's length, which the table has room for: a load without a condition, so that many
// are in flight.  Outside [0, pages) it is no page.
__device__ __forceinline__ int entry_of(const rfsn_paged& p, int shift, int b, int n) {
  return p.table[(int64_t)b * p.table_stride + (n >> shift)];
}
__device__ __forceinline__ bool is_page(const rfsn_paged& p, int page) { return page >= 0 && page < p.pages; }

// The rows of the positions that (sequence, head) keeps, in their order, by their number in the pool (page times page_size + row; kNone:
// no page), and the sequences' new lengths.  A block a (sequence, head).
// Bound: latency (launch, table, weights, some eight block barriers): 2,111 positions of 8 heads 8.3 us; 32 sequences of up to
// 16,000 13.3, 1.9 MB from HBM (keys in LDS, counted and written by waves with ballots: 18.0).
__global__ void __launch_bounds__(kChooseWaves * 64)
evict_choose_kernel(const rfsn_paged p, int shift, int keep, int first, int last, uint32_t* __restrict__ kept,
                    int32_t* __restrict__ new_lens) {
  constexpr int T = kChooseWaves * 64;
  __shared__ ChooseBins room;
  const int tid = threadIdx.x;
  const int h = blockIdx.x, b = blockIdx.y;
  const int len = paged_len(p, shift, b);
  if (h == 0 && tid == 0) new_lens[b] = min(len, keep);
  if (len <= keep) return;
  uint32_t* out = kept + ((int64_t)b * p.kv_heads + h) * keep;
  const int end = len - last;
  auto name_of = [&](int page, int n) {
    return is_page(p, page) ? ((uint32_t)page << shift) + (uint32_t)(n & (p.page_size - 1)) : kNone;
  };
  struct Four {
    float4v score;
    uint32_t name;
  };
  auto load = [&](int n) {
    const int page = entry_of(p, shift, b, n);
    const int64_t row = ((int64_t)(is_page(p, page) ? page : 0) * p.kv_heads + h) * p.page_size + (n & (p.page_size - 1));
    const float4v w = *reinterpret_cast<const float4v*>(p.weight + row);
    const float none = -__builtin_inff();
    return Four{is_page(p, page) ? w : float4v{none, none, none, none}, name_of(page, n)};
  };
  for (int i = tid; i < first; i += T) out[i] = name_of(entry_of(p, shift, b, i), i);
  for (int i = tid; i < last; i += T) out[keep - last + i] = name_of(entry_of(p, shift, b, end + i), end + i);
  choose_fours(room, first, end, (uint32_t)(keep - first - last), first, load, out);
}

// The rows that the list names to positions 0, 1, ... of the sequence, in place.  Their positions ascend and none is below where its row
// goes, so rows that are read later lie behind all that is written now, and a set of them may be written once all of its reads are done: one
// barrier a set.  A thread moves `lanes`-th parts of T / lanes rows, U of them a set, at once.
// Bound: the loads in turn of a set (list, row), then HBM: 2,048 rows of 8 heads of 64, fp16, 11.0 us; 32 sequences to 4,096 rows
// of 8 heads of 128 in 4 bits 16.3 us, 79 MB, 4.8 TB/s.
template <typename V, int T, int U>
__device__ __forceinline__ void move_rows(const rfsn_paged& p, int shift, int b, const uint32_t* __restrict__ kept, int keep,
                                          uint8_t* base, int64_t page_bytes, int row_bytes, int lanes) {
  const int slot = threadIdx.x / lanes, rows = T / lanes;
  uint8_t* const at = base + (threadIdx.x % lanes) * sizeof(V);
  auto place = [&](uint32_t name) {
    return at + (int64_t)(name >> shift) * page_bytes + (int64_t)(name & (uint32_t)(p.page_size - 1)) * row_bytes;
  };
#pragma unroll 1
  for (uint32_t j0 = 0; j0 < (uint32_t)keep; j0 += rows * U) {
    uint32_t from[U], to[U];
    V x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t j = min(j0 + u * rows + slot, (uint32_t)keep - 1);
      from[u] = kept[j];
      to[u] = (uint32_t)entry_of(p, shift, b, (int)j);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t j = j0 + u * rows + slot;
      const bool there = j < (uint32_t)keep && slot < rows && is_page(p, (int)to[u]);
      to[u] = there ? (to[u] << shift) + (j & (uint32_t)(p.page_size - 1)) : kNone;
      if (from[u] == to[u]) to[u] = kNone;
      x[u] = V{};
      if (to[u] != kNone && is_page(p, (int)(from[u] >> shift))) x[u] = *reinterpret_cast<const V*>(place(from[u]));
    }
    // the set's loads have returned to every wave before any wave writes
#pragma unroll
    for (int u = 0; u < U; ++u) asm volatile("" ::"v"(x[u]) : "memory");
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (to[u] != kNone) *reinterpret_cast<V*>(place(to[u])) = x[u];
  }
}

// Blocks of a (sequence, head): `parts` slices of K rows, as many of V rows, one of weights and, with codes, two of scales.
constexpr int kMoveThreads = 1024;
template <int RB, int SB, int U>  // bytes of a row and of its scale
__global__ void __launch_bounds__(kMoveThreads)
evict_move_kernel(const rfsn_paged p, int shift, int parts, const uint32_t* __restrict__ kept_of, int keep) {
  const int x = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  if (paged_len(p, shift, b) <= keep) return;
  const uint32_t* kept = kept_of + ((int64_t)b * p.kv_heads + h) * keep;
  if (x < 2 * parts) {
    const int width = RB / parts;
    uint8_t* base = (uint8_t*)(x < parts ? p.k : p.v);
    const int64_t page_bytes = p.page_stride * RB / p.head_dim, head_bytes = p.head_stride * RB / p.head_dim;
    move_rows<uint4w, kMoveThreads, U>(p, shift, b, kept, keep, base + h * head_bytes + (x % parts) * width, page_bytes, RB, width / 16);
    return;
  }
  auto words = [&](void* base, int row) {
    const int64_t head = (int64_t)p.page_size * row;
    move_rows<uint32_t, kMoveThreads, 8>(p, shift, b, kept, keep, (uint8_t*)base + h * head, head * p.kv_heads, row, row / 4);
  };
  if (x == 2 * parts) words(p.weight, 4);
  else if constexpr (SB > 0) words(x == 2 * parts + 1 ? p.k_scale : p.v_scale, SB);
}

// Bounds of the pages that hold the kept rows, from the keys as they are read back.  A wave a (page, head).
// Bound: latency, a page's loads in turn (calls with bounds and without: 2,048 rows of 8 heads of 64, fp16, in pages of 16, 64
// and 256 rows 20.6, 22.3 and 28.5 us, and 17.2, 16.7 and 16.7; 32 sequences to 4,096 rows of 8 heads of 128, 4 bits, in
// pages of 32 and 256 rows 38.9 and 54.4, and 26.1 and 26.1).
template <int D, int TYPE>
__global__ void __launch_bounds__(64)
evict_bounds_kernel(const rfsn_paged p, int shift, int keep) {
  constexpr int LANES = D / 8, RS = 64 / LANES;
  const int lane = threadIdx.x, slot = lane / LANES, chunk = lane % LANES;
  const int o = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  if (paged_len(p, shift, b) <= keep) return;
  const int page = paged_page(p, b, o);
  if (page < 0) return;
  const int rows = min(p.page_size, keep - (o << shift));
  half8v x = read_page8<D, TYPE>(p, p.k, p.k_scale, page, h, min(slot, rows - 1), chunk);
  Bounds m = bounds_of(x);
  for (int r = RS + slot; r - slot < rows; r += RS) m.add(read_page8<D, TYPE>(p, p.k, p.k_scale, page, h, min(r, rows - 1), chunk));
#pragma unroll
  for (int w = LANES; w < 64; w <<= 1) m.across(w);
  half8v* bp = reinterpret_cast<half8v*>((uint16_t*)p.bounds + ((int64_t)page * p.kv_heads + h) * 2 * D + chunk * 8);
  if (slot == 0) m.store(bp, bp + D / 8);
}

}  // namespace
}  // namespace rfsn

using namespace rfsn;

extern "C" size_t rfsn_paged_evict_workspace_bytes(const rfsn_paged* p, int32_t keep) {
  if (p == nullptr || p->batch <= 0 || p->kv_heads <= 0 || keep <= 0) return 0;
  return (size_t)p->batch * p->kv_heads * keep * sizeof(uint32_t);
}

extern "C" int rfsn_paged_evict(const rfsn_paged* p, int32_t keep, int32_t first, int32_t last, int32_t* new_lens,
                                void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = paged_check(p, "paged_evict")) return st;
  RFSN_REQUIRE(p->weight != nullptr, "paged_evict: the pages hold no weights");
  RFSN_REQUIRE(keep > 0 && first >= 0 && last >= 0 && (int64_t)first + last <= keep,
               "paged_evict: keep must be positive and have room for the first and last positions");
  if (p->batch == 0) return RFSN_OK;
  RFSN_REQUIRE((int64_t)p->pages * p->page_size < (int64_t)kNone, "paged_evict: too many rows");
  RFSN_REQUIRE(p->batch == 1 || p->table_stride != 0, "paged_evict: sequences share a table");
  RFSN_REQUIRE(new_lens != nullptr, "paged_evict: null output");
  RFSN_REQUIRE((uintptr_t)new_lens >= (uintptr_t)(p->lens + p->batch) || (uintptr_t)p->lens >= (uintptr_t)(new_lens + p->batch),
               "paged_evict: new_lens overlaps lens, which the launches read");
  RFSN_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= rfsn_paged_evict_workspace_bytes(p, keep),
               "paged_evict: workspace too small or misaligned");
  const hipStream_t s = (hipStream_t)stream;
  const int shift = paged_shift(*p), D = p->head_dim;
  uint32_t* kept = (uint32_t*)workspace;
  hipLaunchKernelGGL(evict_choose_kernel, dim3((unsigned)p->kv_heads, (unsigned)p->batch), dim3(kChooseWaves * 64), 0, s, *p,
                     shift, keep, first, last, kept, new_lens);
  if (int st = check_launch("paged_evict")) return st;
  if ((int64_t)p->table_width * p->page_size <= keep) return RFSN_OK;  // nothing can be longer
  // Slices of a line of 128 bytes, narrower where that leaves blocks for the chip (2,048 rows of 8 heads of 64, fp16, one
  // sequence: 16 blocks of 128 bytes 13.8 us, 64 of 32 12.0).  Sets of 16 pieces a thread, or 4 where those hold all rows.
#define RFSN_EVICT_U(RB, SB, U)                                                                                     \
  hipLaunchKernelGGL((evict_move_kernel<RB, SB, U>), grid, dim3(kMoveThreads), 0, s, *p, shift, parts, kept, keep)
#define RFSN_EVICT(RB, SB)                                                                                          \
  do {                                                                                                              \
    int parts = RB > 128 ? RB / 128 : 1;                                                                            \
    while (RB / parts > 32 && (int64_t)2 * parts * p->kv_heads * p->batch < 256) parts *= 2;                        \
    const dim3 grid(2 * parts + 1 + (SB > 0 ? 2 : 0), (unsigned)p->kv_heads, (unsigned)p->batch);                   \
    if ((int64_t)keep * (RB / parts) <= 4 * 16 * kMoveThreads) RFSN_EVICT_U(RB, SB, 4);                             \
    else RFSN_EVICT_U(RB, SB, 16);                                                                                  \
  } while (0)
#define RFSN_EVICT_D(DD)                                    \
  do {                                                      \
    if (p->type == RFSN_PAGE_FP16) RFSN_EVICT(2 * DD, 0);   \
    else if (p->type == RFSN_PAGE_E2M1) RFSN_EVICT(DD / 2, DD / 16); \
    else RFSN_EVICT(DD, 4);                                 \
  } while (0)
  if (D == 64) RFSN_EVICT_D(64);
  else if (D == 128) RFSN_EVICT_D(128);
  else RFSN_EVICT_D(256);
#undef RFSN_EVICT_D
#undef RFSN_EVICT
#undef RFSN_EVICT_U
  if (int st = check_launch("paged_evict")) return st;
  if (p->bounds == nullptr) return RFSN_OK;
  const dim3 grid((unsigned)ceil_div(keep, p->page_size), (unsigned)p->kv_heads, (unsigned)p->batch);
  RFSN_PAGED_DISPATCH(D, p->type, {
    hipLaunchKernelGGL((evict_bounds_kernel<DD, TT>), grid, dim3(64), 0, s, *p, shift, keep);
  });
  return check_launch("paged_evict");
}
