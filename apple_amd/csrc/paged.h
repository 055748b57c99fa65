// What the paged KV cache's kernels share (paged.hip, paged_attention.hip).
#pragma once

#include "rfsn_common.h"

namespace rfsn {

typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float8v __attribute__((ext_vector_type(8)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4w __attribute__((ext_vector_type(4)));

// Checks every call makes of the pool, the table and the batch; 0 or a status.
int paged_check(const rfsn_paged* p, const char* what);

inline int paged_shift(const rfsn_paged& p) { return __builtin_ctz((unsigned)p.page_size); }

// 8 codes in fp32, where each is exact.
template <int TYPE>
__device__ __forceinline__ float8v page8(uint2v c) {
  float8v f;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if constexpr (TYPE == RFSN_PAGE_INT8) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * w + e] = (float)(int8_t)(c[w] >> (8 * e));
    } else {
      f[4 * w + 0] = __builtin_amdgcn_cvt_f32_fp8((int)c[w], 0);
      f[4 * w + 1] = __builtin_amdgcn_cvt_f32_fp8((int)c[w], 1);
      f[4 * w + 2] = __builtin_amdgcn_cvt_f32_fp8((int)c[w], 2);
      f[4 * w + 3] = __builtin_amdgcn_cvt_f32_fp8((int)c[w], 3);
    }
  }
  return f;
}

// 8 consecutive stored values of a row, without the row's scale.
template <int TYPE>
__device__ __forceinline__ float8v load_page8(const void* base, int64_t off) {
  if constexpr (TYPE == RFSN_PAGE_FP16) {
    const half8v h = *reinterpret_cast<const half8v*>((const uint16_t*)base + off);
    float8v f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)h[e];
    return f;
  } else {
    return page8<TYPE>(*reinterpret_cast<const uint2v*>((const uint8_t*)base + off));
  }
}

// Tokens of sequence b that the table can hold.
__device__ __forceinline__ int paged_len(const rfsn_paged& p, int shift, int b) {
  const int64_t most = (int64_t)p.table_width << shift;
  const int n = p.lens[b];
  return n < 0 ? 0 : (int)(n < most ? n : most);
}

// Page of ordinal ord of sequence b, or -1.
__device__ __forceinline__ int paged_page(const rfsn_paged& p, int b, int64_t ord) {
  if (ord < 0 || ord >= p.table_width) return -1;
  const int n = p.table[(int64_t)b * p.table_stride + ord];
  return n >= 0 && n < p.pages ? n : -1;
}

// Inclusive sums, or largest values, of the lanes up to each one, in data-parallel moves
// (rows of 16, then the rows' last lanes): lane 63 has the wave's.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp0(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 15, true);
}
__device__ __forceinline__ uint32_t wave_upto(uint32_t x) {
  x += dpp0<0x111, 15>(x), x += dpp0<0x112, 15>(x), x += dpp0<0x114, 15>(x), x += dpp0<0x118, 15>(x);
  x += dpp0<0x142, 10>(x), x += dpp0<0x143, 12>(x);
  return x;
}
__device__ __forceinline__ uint32_t wave_most(uint32_t x) {
  x = max(x, dpp0<0x111, 15>(x)), x = max(x, dpp0<0x112, 15>(x)), x = max(x, dpp0<0x114, 15>(x));
  x = max(x, dpp0<0x118, 15>(x)), x = max(x, dpp0<0x142, 10>(x)), x = max(x, dpp0<0x143, 12>(x));
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ uint32_t wave_total(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_readlane((int)wave_upto(x), 63);
}

}  // namespace rfsn
