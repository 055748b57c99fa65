// Rotary positions of the rows of a ragged batch (llama32_adapter.py:555-568, with the interleaved layout and
// parts of a head beside it):
//
//   (x1, x2) -> factor (x1 cos a - x2 sin a, x2 cos a + x1 sin a),  a = position * inv_freq[i]
//
// A block takes some rows with all of their heads, queries and keys, and makes each row's turns once in LDS.
#include "rfsn_common.h"

namespace rfsn {
namespace {

typedef __bf16 bf16;

template <int TYPE> struct Elem;
template <> struct Elem<RFSN_ROTARY_FP16> { typedef f16 type; };
template <> struct Elem<RFSN_ROTARY_BF16> { typedef bf16 type; };
template <> struct Elem<RFSN_ROTARY_FP32> { typedef float type; };

template <typename T, int V> struct Vec { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T> struct Vec<T, 1> { typedef T type; };

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

template <bool kOnce, typename V, typename T>
__device__ __forceinline__ V load_vec(const T* a) {
  if constexpr (kOnce) return __builtin_nontemporal_load(reinterpret_cast<const V*>(a));
  else return *reinterpret_cast<const V*>(a);
}
template <bool kOnce, typename V, typename T>
__device__ __forceinline__ void store_vec(V x, T* a) {
  if constexpr (kOnce) __builtin_nontemporal_store(x, reinterpret_cast<V*>(a));
  else *reinterpret_cast<V*>(a) = x;
}

// Pieces of PB bytes: a thread keeps its place in the head, a piece of each half ("half"), a piece of pairs
// ("interleaved"; with pieces of one value the two of a pair), or a piece to copy, and goes through the block's
// (row, head) lines, U of them in flight.  The block's rows' turns are made once, while the first lines come.
//
// Bound: HBM.  8,191 rows of 40 heads of 64, fp16: 84 MB in 13.3 to 15.6 us, 5.4 to 6.3 TB/s; 16,384 of 64 of 128, bf16,
// interleaved: 537 MB in 82 us, 6.5 TB/s.  A thread a pair with divisions for its place took 32 and 269 us.
template <int TYPE, int LAYOUT, int PB, int U, bool kOnce>
__global__ void __launch_bounds__(1024)
rotary_kernel(const rfsn_rotary_params p, int per, int turning, int units, float over_heads) {
  typedef typename Elem<TYPE>::type T;
  constexpr int V = PB / sizeof(T);
  constexpr bool kSplit = LAYOUT == RFSN_ROTARY_HALF || V == 1;  // the pair's values in two pieces
  constexpr int P = kSplit ? V : V / 2;                          // pairs of a thread
  typedef typename Vec<T, V>::type vec;
  extern __shared__ Turn turns[];
  const int threads = blockDim.x;
  const int half = p.rotary_dim / 2, heads = p.heads[0] + p.heads[1];
  const int64_t n0 = (int64_t)blockIdx.x * per;
  const int rows = (int)(p.rows - n0 < per ? p.rows - n0 : per);
  const int slots = threads / units, slot = threadIdx.x / units, u = threadIdx.x % units, lines = rows * heads;
  const bool turn = u < turning;
  const int partner = !turn ? 0 : LAYOUT == RFSN_ROTARY_HALF ? half : 1;
  const int at = !turn ? p.rotary_dim + (u - turning) * V : LAYOUT == RFSN_ROTARY_HALF || !kSplit ? u * V : 2 * u;
  struct Line {
    const T* x;
    T* y;
    int row;
  };
  auto line = [&](int i) {
    const int r = (int)(((float)i + 0.5f) * over_heads), h = i - r * heads, w = h >= p.heads[0];
    const int hw = w ? h - p.heads[0] : h;
    return Line{(const T*)p.x[w] + (n0 + r) * p.row_stride[w] + hw * p.head_stride[w] + at,
                (T*)p.out[w] + (n0 + r) * p.out_row_stride[w] + hw * p.out_head_stride[w] + at, r};
  };
  Line l[U];
  vec a[U], b[U];
  auto load = [&](int i0) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = i0 + k * slots + slot;
      l[k] = line(i < lines ? i : lines - 1);
      a[k] = load_vec<kOnce, vec>(l[k].x);
      if constexpr (kSplit) b[k] = load_vec<kOnce, vec>(l[k].x + partner);
    }
  };
  if (slot < slots) load(0);
  for (int i = threadIdx.x; i < rows * half; i += threads) {
    const int r = i / half;
    turns[i] = turn_of(position_of(p, n0 + r), p.inv_freq[i - r * half], p.factor);
  }
  __syncthreads();
  if (slot >= slots) return;
  auto value = [](const vec& v, int e) -> float {
    if constexpr (V == 1) return (float)v;
    else return (float)v[e];
  };
  auto put = [](vec& v, int e, float y) {
    if constexpr (V == 1) v = (T)y;
    else v[e] = (T)y;
  };
  for (int i0 = 0;;) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (i0 + k * slots + slot >= lines) break;
      if (!turn) {
        store_vec<kOnce>(a[k], l[k].y);
        continue;
      }
      const Turn* t = turns + l[k].row * half + u * P;
      vec c, d;
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float x1 = value(a[k], kSplit ? e : 2 * e), x2 = kSplit ? value(b[k], e) : value(a[k], 2 * e + 1);
        put(c, kSplit ? e : 2 * e, x1 * t[e].c - x2 * t[e].s);
        put(kSplit ? d : c, kSplit ? e : 2 * e + 1, x2 * t[e].c + x1 * t[e].s);
      }
      store_vec<kOnce>(c, l[k].y);
      if constexpr (kSplit) store_vec<kOnce>(d, l[k].y + partner);
    }
    i0 += U * slots;
    if (i0 >= lines) break;
    load(i0);
  }
}

// Whether pieces of `bytes` are aligned, on one side of the border between turned and other coordinates and, of halves, of
// the one between them.
bool pieces(const rfsn_rotary_params& p, int size, int bytes) {
  const int v = bytes / size;
  if (p.rotary_dim % (p.layout == RFSN_ROTARY_HALF ? 2 * v : v) || p.head_dim % v) return false;
  for (int w = 0; w < 2; ++w) {
    if (p.heads[w] == 0) continue;
    if (((uintptr_t)p.x[w] | (uintptr_t)p.out[w]) % bytes) return false;
    if (p.rows > 1 && (p.row_stride[w] % v || p.out_row_stride[w] % v)) return false;
    if (p.heads[w] > 1 && (p.head_stride[w] % v || p.out_head_stride[w] % v)) return false;
  }
  return true;
}

template <int TYPE, int PB, int U>
void rotary_launch(const rfsn_rotary_params& p, bool same, hipStream_t s) {
  constexpr int size = (int)sizeof(typename Elem<TYPE>::type), V = PB / size;
  const int heads = p.heads[0] + p.heads[1];
  const int turning = p.rotary_dim / (p.layout == RFSN_ROTARY_HALF || V == 1 ? 2 * V : V);
  const int units = turning + (same ? 0 : (p.head_dim - p.rotary_dim) / V);  // what is not turned stays in place
  const int threads = units <= 256 ? 256 : 1024;
  int64_t per = (int64_t)(threads / units) * U / heads;
  if (per > ceil_div(p.rows, 1024)) per = ceil_div(p.rows, 1024);
  if (per * p.rotary_dim * 4 > 32768) per = 32768 / (p.rotary_dim * 4);  // bytes of LDS
  if (per < 1) per = 1;
  const dim3 grid((unsigned)ceil_div(p.rows, per));
  const size_t lds = (size_t)per * p.rotary_dim / 2 * sizeof(Turn);
  // Results of 256 MB, the size of the last-level cache, or more are gone from it before anything reads them: rows and
  // results pass the caches by (16,384 rows of 64 heads of 128, fp16: 101 -> 83 us interleaved, 102 -> 92 in halves; 8,191
  // of 72 of 256: 115 -> 103), where a wave's pieces are whole lines of 128 bytes (halves of 64: 100 -> 103).
  // Smaller ones stay (8,191 of 40 of 64: interleaved 14.9, so 17.0; fp32 25.4, so 28.4), as do rows turned in place (44, so 57).
  const bool once = PB == 16 && !same && (double)p.rows * heads * p.head_dim * size >= 256.0 * 1024 * 1024 &&
                    (p.layout == RFSN_ROTARY_INTERLEAVED || p.rotary_dim / 2 * size >= 128);
#define RFSN_ROTARY_LAUNCH(LL, ONCE)                                                                                  \
  hipLaunchKernelGGL((rotary_kernel<TYPE, LL, PB, U, ONCE>), grid, dim3(threads), lds, s, p, (int)per, turning, units, \
                     1.f / (float)heads)
  if constexpr (PB == 16)
    if (once) {
      if (p.layout == RFSN_ROTARY_HALF) RFSN_ROTARY_LAUNCH(RFSN_ROTARY_HALF, true);
      else RFSN_ROTARY_LAUNCH(RFSN_ROTARY_INTERLEAVED, true);
      return;
    }
  if (p.layout == RFSN_ROTARY_HALF) RFSN_ROTARY_LAUNCH(RFSN_ROTARY_HALF, false);
  else RFSN_ROTARY_LAUNCH(RFSN_ROTARY_INTERLEAVED, false);
#undef RFSN_ROTARY_LAUNCH
}

template <int TYPE>
void rotary_of(const rfsn_rotary_params& p, bool same, hipStream_t s) {
  constexpr int size = (int)sizeof(typename Elem<TYPE>::type);
  if (pieces(p, size, 16)) rotary_launch<TYPE, 16, 4>(p, same, s);
  else if (pieces(p, size, 2 * size)) rotary_launch<TYPE, 2 * size, 8>(p, same, s);
  else rotary_launch<TYPE, size, 8>(p, same, s);
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
  bool same = true;
  for (int w = 0; w < 2; ++w) same = same && (p->heads[w] == 0 || p->x[w] == p->out[w]);
  const hipStream_t s = (hipStream_t)stream;
  if (p->type == RFSN_ROTARY_FP16) rotary_of<RFSN_ROTARY_FP16>(*p, same, s);
  else if (p->type == RFSN_ROTARY_BF16) rotary_of<RFSN_ROTARY_BF16>(*p, same, s);
  else rotary_of<RFSN_ROTARY_FP32>(*p, same, s);
  return check_launch("rotary");
}
