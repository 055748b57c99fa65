// The largest of a row of scores, by one block: what page selection and eviction keep.
#pragma once

#include "paged.h"

namespace rfsn {
namespace {

typedef float float4v __attribute__((ext_vector_type(4)));

// Order of the scores as unsigned keys: NaN as +infinity, -0 as +0.
__device__ __forceinline__ uint32_t score_key(float s) {
  if (s != s) s = __builtin_inff();
  const uint32_t u = __builtin_bit_cast(uint32_t, s + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

constexpr int kChooseWaves = 16, kChooseBins = 2048;
template <int KEYS>
struct ChooseRoom {
  uint32_t key[KEYS];
  uint32_t hist[kChooseBins];
  uint32_t wave[2][kChooseWaves], found[3];
};

// The `left` numbers of begin .. end - 1 (left below their count) with the largest score(n), ties to the lower number,
// in ascending order to out[at], out[at + 1], ...  Scores that come in fours (kFours): score.four(n) has those of n .. n + 3, n a
// multiple of 4 at most `end`.
// The smallest key to keep is found by narrowing [lo, hi], at first the smallest and largest key: a histogram of
// 2,048 equal parts of it says which part holds the key wanted.  Scores share their exponent mostly, so parts
// of their range spread over the counters where their leading bits would meet in one; two rounds are the rule,
// three the most (leading bits as counters: 50 us for 128 of 2,048 pages, 256 rows; so 6.3, latency of
// some ten block barriers).  Then each of 16 waves counts what it keeps of its own run and writes it
// behind the waves before it.  Keys past the LDS copy are read again from the scores.
template <int KEYS, typename Score>
__device__ __forceinline__ void choose_largest(ChooseRoom<KEYS>& room, int begin, int end, uint32_t left, int at0,
                                               const Score& score, int32_t* __restrict__ out) {
  constexpr int T = kChooseWaves * 64, PER = kChooseBins / T;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int held = end - begin < KEYS ? end : begin + KEYS;  // of numbers below it the keys are in LDS
  // (Numbers past the last one are held in 32 bits without a sign: they may pass 2^31 by a few steps.)
  // Each number n, n + step, ... below `to` with its key to f, U keys read at a time.  f is called alike by all lanes of a
  // wave where `to` - n + lane is (numbers from `to` on come with `in` false).
  auto each = [&](uint32_t n, uint32_t to, uint32_t step, auto&& f) {
    constexpr int U = Score::kFours ? 4 : 1;  // (thousands of positions, or some hundred pages)
    for (; n - lane < to; n += U * step) {
      uint32_t k[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int m = (int)min(n + u * step, to - 1);
        k[u] = m < held ? room.key[m - begin] : score_key(score(m));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) f((int)(n + u * step), k[u], n + u * step < to);
    }
  };
  uint32_t lo = 0xffffffffu, hi = 0;
  auto take = [&](uint32_t n, float x) {
    const uint32_t k = score_key(x);
    if (n - (uint32_t)begin < KEYS) room.key[n - begin] = k;
    lo = min(lo, k), hi = max(hi, k);
  };
  if constexpr (Score::kFours) {
    constexpr int Q = 4;  // fours in flight
    for (uint32_t n4 = (begin & ~3) + 4 * tid; n4 < (uint32_t)end; n4 += Q * 4 * T) {
      float4v s[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) s[q] = score.four((int)min(n4 + q * 4 * T, (uint32_t)(end - 1) & ~3u));
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t n = n4 + q * 4 * T + e;
          if (n >= (uint32_t)begin && n < (uint32_t)end) take(n, s[q][e]);
        }
    }
  } else {
#pragma unroll 4
    for (int n = begin + tid; n < end; n += T) take(n, score(n));
  }
  lo = ~wave_most(~lo), hi = wave_most(hi);
  if (lane == 0) room.wave[0][wave] = lo, room.wave[1][wave] = hi;
  __syncthreads();
  lo = ~wave_most(lane < kChooseWaves ? ~room.wave[0][lane] : 0u), hi = wave_most(lane < kChooseWaves ? room.wave[1][lane] : 0u);
  // what the waves before this one have of room.wave[i]
  auto before_wave = [&](int i) { return wave_total(lane < wave ? room.wave[i][lane] : 0u); };
  uint32_t over = 0xffffffffu, tie = 0xffffffffu;  // keys from `over` on are kept, and `left` of those equal to `tie`
  while (left > 0) {
    if (lo == hi) {
      over = lo + 1, tie = lo;
      break;
    }
    const int bits = 32 - __builtin_clz(hi - lo), sh = bits > 11 ? bits - 11 : 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) room.hist[tid + i * T] = 0;
    __syncthreads();
    each(begin + tid, end, T, [&](int, uint32_t k, bool in) {
      if (in && k >= lo && k <= hi) atomicAdd(&room.hist[(k - lo) >> sh], 1u);
    });
    __syncthreads();
    // keys in the parts above each thread's PER parts, from the top down
    uint32_t c[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) mine += c[i] = room.hist[kChooseBins - 1 - (tid * PER + i)];
    const uint32_t upto = wave_upto(mine);
    if (lane == 63) room.wave[0][wave] = upto;
    __syncthreads();
    uint32_t above = upto - mine + before_wave(0);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (above < left && above + c[i] >= left) {
        room.found[0] = (uint32_t)(kChooseBins - 1 - (tid * PER + i));
        room.found[1] = left - above;
        room.found[2] = c[i];
      }
      above += c[i];
    }
    __syncthreads();
    lo += room.found[0] << sh;
    hi = min(hi, lo + ((1u << sh) - 1u));
    left = room.found[1];
    if (room.found[2] == left) {  // the whole part
      over = lo, left = 0;
    }
  }
  __syncthreads();  // room.wave is written again
  const uint32_t seg = ((end - begin + kChooseWaves - 1) / kChooseWaves + 63) / 64 * 64;
  const uint32_t n0 = min(begin + wave * seg, (uint32_t)end), n1 = min((uint32_t)end, n0 + seg);
  uint32_t kept = 0, ties = 0;
  each(n0 + lane, n1, 64, [&](int, uint32_t k, bool in) {
    kept += (uint32_t)__popcll(__ballot(in && k >= over));
    ties += (uint32_t)__popcll(__ballot(in && left && k == tie));
  });
  if (lane == 0) room.wave[0][wave] = kept, room.wave[1][wave] = ties;
  __syncthreads();
  uint32_t before = before_wave(1), at = (uint32_t)at0 + before_wave(0);
  at += min(before, left);
  const uint64_t below = (1ull << lane) - 1;
  each(n0 + lane, n1, 64, [&](int n, uint32_t k, bool in) {
    const bool is_tie = in && left && k == tie;
    const uint64_t bt = __ballot(is_tie);
    const bool keep = (in && k >= over) || (is_tie && before + (uint32_t)__popcll(bt & below) < left);
    const uint64_t bk = __ballot(keep);
    if (keep) out[at + (uint32_t)__popcll(bk & below)] = n;
    at += (uint32_t)__popcll(bk), before += (uint32_t)__popcll(bt);
  });
}

}  // namespace
}  // namespace rfsn
