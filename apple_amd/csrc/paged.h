// What the paged KV cache's kernels share: rows in pages, bounds and page choice (paged.hip, choose.h), attention and weights
// (paged_attention.h, paged_weigh.hip), eviction (evict.hip).
#pragma once

#include "rfsn_common.h"

namespace rfsn {

typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float8v __attribute__((ext_vector_type(8)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4w __attribute__((ext_vector_type(4)));
typedef _Float16 half2w __attribute__((ext_vector_type(2)));
typedef float float2w __attribute__((ext_vector_type(2)));

typedef unsigned short ushort8v __attribute__((ext_vector_type(8)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
typedef unsigned short ushort4v __attribute__((ext_vector_type(4)));

// The statements with the head size as DD and the page type as TT.
#define RFSN_PAGED_DISPATCH_D(D, TYPE, ...)                                              \
  do {                                                                                   \
    constexpr int DD = D;                                                                \
    if (TYPE == RFSN_PAGE_FP16) { constexpr int TT = RFSN_PAGE_FP16; __VA_ARGS__ }       \
    else if (TYPE == RFSN_PAGE_INT8) { constexpr int TT = RFSN_PAGE_INT8; __VA_ARGS__ }  \
    else if (TYPE == RFSN_PAGE_E4M3) { constexpr int TT = RFSN_PAGE_E4M3; __VA_ARGS__ }  \
    else { constexpr int TT = RFSN_PAGE_E2M1; __VA_ARGS__ }                              \
  } while (0)
#define RFSN_PAGED_DISPATCH(D, TYPE, ...)                         \
  do {                                                            \
    if (D == 64) RFSN_PAGED_DISPATCH_D(64, TYPE, __VA_ARGS__);    \
    else if (D == 128) RFSN_PAGED_DISPATCH_D(128, TYPE, __VA_ARGS__); \
    else RFSN_PAGED_DISPATCH_D(256, TYPE, __VA_ARGS__);           \
  } while (0)

// Bytes of a stored row of D coordinates.
template <int TYPE>
constexpr int row_bytes(int D) { return TYPE == RFSN_PAGE_FP16 ? 2 * D : TYPE == RFSN_PAGE_E2M1 ? D / 2 : D; }

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

// 4-bit pages: a scale byte as the number it stands for, 2^(e-15) (1 + m / 8) or, with e = 0, 2^-17 m.
__device__ __forceinline__ f16 group_scale(uint32_t byte) { return __builtin_bit_cast(f16, (uint16_t)(byte << 7)); }
// 8 codes (the low coordinate in the low bits) times their scale: a product of 2 and 4 significant bits, exact in fp16.
__device__ __forceinline__ half8v e2m1_f16(uint32_t codes, f16 scale) {
  const half2w s = {scale, scale};
  const half2w a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.f, 0) * s;
  const half2w b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.f, 1) * s;
  const half2w c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.f, 2) * s;
  const half2w d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.f, 3) * s;
  return half8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
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

// 8 coordinates of a row as they are read back: fp16, of codes one product rounded once.
template <int D, int TYPE>
__device__ __forceinline__ half8v read_page8(const rfsn_paged& p, const void* base, const void* scale, int page, int h, int row, int chunk) {
  const int64_t off = (int64_t)page * p.page_stride + h * p.head_stride + (int64_t)row * D + chunk * 8;
  const int64_t sc = ((int64_t)page * p.kv_heads + h) * p.page_size + row;
  if constexpr (TYPE == RFSN_PAGE_FP16) {
    return *reinterpret_cast<const half8v*>((const uint16_t*)base + off);
  } else if constexpr (TYPE == RFSN_PAGE_E2M1) {
    return e2m1_f16(*reinterpret_cast<const uint32_t*>((const uint8_t*)base + off / 2),
                    group_scale(((const uint8_t*)scale)[sc * (D / 16) + chunk / 2]));
  } else {
    const float x = ((const float*)scale)[sc];
    const float8v f = load_page8<TYPE>(base, off);
    half8v r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = (f16)(f[e] * x);
    return r;
  }
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
