// Rotary positions of the rows of a ragged batch (llama32_adapter.py:555-568, with the interleaved layout and
// parts of a head beside it):
//
//   (x1, x2) -> factor (x1 cos a - x2 sin a, x2 cos a + x1 sin a),  a = position * inv_freq[i]
//
// A block takes some rows with all of their heads, queries and keys, and makes each row's turns once in LDS.
#include "rfsn_common.h"

namespace rfsn {
namespace {

typedef uint32_t uint4w __attribute__((ext_vector_type(4)));
typedef __bf16 bf16;

template <int TYPE> struct Elem;
template <> struct Elem<RFSN_ROTARY_FP16> { typedef f16 type; };
template <> struct Elem<RFSN_ROTARY_BF16> { typedef bf16 type; };
template <> struct Elem<RFSN_ROTARY_FP32> { typedef float type; };

struct Turn {
  float c, s;
};

// cos and sin of a position's angle.  Angles of far positions have many turns: the part of one that counts is taken in
// 64 bits, to an eighth of a turn about the nearest quarter, which fp32 then holds to 2^-28 of a turn.
__device__ __forceinline__ Turn turn_of(double position, double inv_freq, float factor) {
  const double turns = position * inv_freq * 0.15915494309189533577;  // 1 / (2 pi)
  const double quarters = rint(turns * 4.0);
  const float r = (float)(turns * 4.0 - quarters);                    // quarter turns, -1/2 .. 1/2
  float s, c;
  sincospif(0.5f * r, &s, &c);
  const int q = (int)(quarters - 4.0 * floor(quarters * 0.25));       // 0 .. 3
  const float c1 = q & 1 ? s : c, s1 = q & 1 ? c : s;
  Turn t;
  t.c = factor * (q == 1 || q == 2 ? -c1 : c1);
  t.s = factor * (q & 2 ? -s1 : s1);
  return t;
}

__device__ __forceinline__ double position_of(const rfsn_rotary_params& p, int64_t n) {
  return p.wide_positions ? (double)((const int64_t*)p.positions)[n] : (double)((const int32_t*)p.positions)[n];
}

// Any sizes, strides and alignment: a thread a pair or a coordinate behind the rotated ones.
template <int TYPE>
__global__ void __launch_bounds__(256)
rotary_any_kernel(const rfsn_rotary_params p, int per) {
  typedef typename Elem<TYPE>::type T;
  extern __shared__ Turn turns[];
  const int half = p.rotary_dim / 2, units = half + p.head_dim - p.rotary_dim;
  const int64_t n0 = (int64_t)blockIdx.x * per;
  const int rows = (int)(p.rows - n0 < per ? p.rows - n0 : per);
  for (int i = threadIdx.x; i < rows * half; i += 256)
    turns[i] = turn_of(position_of(p, n0 + i / half), p.inv_freq[i % half], p.factor);
  __syncthreads();
#pragma unroll 1
  for (int w = 0; w < 2; ++w) {
    const int all = rows * p.heads[w] * units;
    for (int i = threadIdx.x; i < all; i += 256) {
      const int u = i % units, rh = i / units, h = rh % p.heads[w], r = rh / p.heads[w];
      const T* x = (const T*)p.x[w] + (n0 + r) * p.row_stride[w] + h * p.head_stride[w];
      T* y = (T*)p.out[w] + (n0 + r) * p.out_row_stride[w] + h * p.out_head_stride[w];
      if (u < half) {
        const int a = p.layout == RFSN_ROTARY_HALF ? u : 2 * u, b = p.layout == RFSN_ROTARY_HALF ? u + half : 2 * u + 1;
        const Turn t = turns[r * half + u];
        const float xa = (float)x[a], xb = (float)x[b];
        y[a] = (T)(xa * t.c - xb * t.s);
        y[b] = (T)(xb * t.c + xa * t.s);
      } else {
        y[u + half] = x[u + half];
      }
    }
  }
}

}  // namespace
}  // namespace rfsn

using namespace rfsn;

extern "C" int rfsn_rotary(const rfsn_rotary_params* p, void* stream) {
  RFSN_REQUIRE(p != nullptr, "rotary: null parameters");
  RFSN_REQUIRE(p->head_dim >= 2 && p->head_dim <= 1024, "rotary: head_dim must be 2 to 1024");
  RFSN_REQUIRE(p->rotary_dim >= 2 && p->rotary_dim <= p->head_dim && p->rotary_dim % 2 == 0,
               "rotary: rotary_dim must be even and at most head_dim");
  RFSN_REQUIRE(p->layout == RFSN_ROTARY_HALF || p->layout == RFSN_ROTARY_INTERLEAVED, "rotary: unknown layout");
  RFSN_REQUIRE(p->type == RFSN_ROTARY_FP16 || p->type == RFSN_ROTARY_BF16 || p->type == RFSN_ROTARY_FP32, "rotary: unknown type");
  RFSN_REQUIRE(p->heads[0] >= 0 && p->heads[1] >= 0 && p->heads[0] <= 65535 && p->heads[1] <= 65535, "rotary: heads out of range");
  RFSN_REQUIRE(p->rows >= 0 && p->rows < (1ll << 31), "rotary: row count out of range");
  if (p->rows == 0 || p->heads[0] + p->heads[1] == 0) return RFSN_OK;
  const int size = p->type == RFSN_ROTARY_FP32 ? 4 : 2;
  RFSN_REQUIRE(p->inv_freq && ((uintptr_t)p->inv_freq & 7) == 0 && p->positions &&
                   ((uintptr_t)p->positions & (p->wide_positions ? 7 : 3)) == 0,
               "rotary: null or misaligned positions or frequencies");
  for (int w = 0; w < 2; ++w)
    if (p->heads[w])
      RFSN_REQUIRE(p->x[w] && p->out[w] && (uintptr_t)p->x[w] % size == 0 && (uintptr_t)p->out[w] % size == 0,
                   "rotary: null or misaligned rows");
  const int per = 1;
  const unsigned blocks = (unsigned)ceil_div(p->rows, per);
  const size_t lds = (size_t)per * p->rotary_dim / 2 * sizeof(Turn);
  const hipStream_t s = (hipStream_t)stream;
#define RFSN_ROTARY(TT) hipLaunchKernelGGL(rotary_any_kernel<TT>, dim3(blocks), dim3(256), lds, s, *p, per)
  if (p->type == RFSN_ROTARY_FP16) RFSN_ROTARY(RFSN_ROTARY_FP16);
  else if (p->type == RFSN_ROTARY_BF16) RFSN_ROTARY(RFSN_ROTARY_BF16);
  else RFSN_ROTARY(RFSN_ROTARY_FP32);
#undef RFSN_ROTARY
  return check_launch("rotary");
}
