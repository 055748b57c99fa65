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
struct ChooseBins {
  uint32_t hist[kChooseBins];
  uint32_t wave[2][kChooseWaves], found[3], few;
  uint32_t total[64];
};
template <int KEYS>
struct ChooseRoom : ChooseBins {
  uint32_t key[KEYS];
};

// Which keys are the `left` largest of a block's: those from `over` on, and of those equal to `tie` the first `left`.
struct Largest {
  uint32_t over, tie, left;
};

// lo, hi: this thread's smallest and largest key; visit(f) calls f(key) for each of its keys (keys below all of
// [lo, hi] are not counted).  left is below the keys' number.
// The smallest key to keep is found by narrowing [lo, hi], at first the smallest and largest key: a histogram of
// 2,048 equal parts of it says which part holds the key wanted.  Scores share their exponent mostly, so parts
// of their range spread over the counters where their leading bits would meet in one; two rounds are the rule, the second
// between at most 64 keys mostly, three the most (leading bits as counters: 50 us for 128 of 2,048 pages, 256 rows; so 5.8, latency of
// some eight block barriers).
template <typename Visit>
__device__ __forceinline__ Largest find_largest(ChooseBins& room, uint32_t lo, uint32_t hi, uint32_t left, const Visit& visit) {
  constexpr int T = kChooseWaves * 64, PER = kChooseBins / T;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // a thread clears and reads the same PER counters, parts from the top down
  auto part = [&](int i) { return kChooseBins - 1 - (tid * PER + i); };
#pragma unroll
  for (int i = 0; i < PER; ++i) room.hist[part(i)] = 0;
  if (tid == 0) room.few = 0;
  lo = ~wave_most(~lo), hi = wave_most(hi);
  if (lane == 0) room.wave[0][wave] = lo, room.wave[1][wave] = hi;
  __syncthreads();
  lo = ~wave_most(lane < kChooseWaves ? ~room.wave[0][lane] : 0u), hi = wave_most(lane < kChooseWaves ? room.wave[1][lane] : 0u);
  for (int round = 0; left > 0 && round < 3; ++round) {  // (11 of 32 bits each)
    if (lo == hi) return {lo + 1, lo, left};
    const int bits = 32 - __builtin_clz(hi - lo), sh = bits > 11 ? bits - 11 : 0;
    visit([&](uint32_t k) {
      if (k >= lo && k <= hi) atomicAdd(&room.hist[(k - lo) >> sh], 1u);
    });
    __syncthreads();
    // keys in the parts above each thread's
    uint32_t c[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) mine += c[i] = room.hist[part(i)];
#pragma unroll
    for (int i = 0; i < PER; ++i) room.hist[part(i)] = 0;
    const uint32_t upto = wave_upto(mine);
    if (lane == 63) room.wave[0][wave] = upto;
    __syncthreads();
    uint32_t above = upto - mine + wave_total(lane < wave ? room.wave[0][lane] : 0u);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (above < left && above + c[i] >= left) {
        room.found[0] = (uint32_t)part(i);
        room.found[1] = left - above;
        room.found[2] = c[i];
      }
      above += c[i];
    }
    __syncthreads();
    lo += room.found[0] << sh;
    hi = min(hi, lo + ((1u << sh) - 1u));
    left = room.found[1];
    const uint32_t n = room.found[2];
    if (n == left) return {lo, 0xffffffffu, 0};  // the whole part
    if (n <= 64) {  // each wave compares them with one another
      visit([&](uint32_t k) {
        if (k >= lo && k <= hi) room.hist[atomicAdd(&room.few, 1u) & (kChooseBins - 1)] = k;
      });
      __syncthreads();
      const uint32_t k = room.hist[lane];
      uint32_t more = 0, same = 0;
      for (uint32_t j = 0; j < n; ++j) {
        const uint32_t kj = (uint32_t)__builtin_amdgcn_readlane((int)k, (int)j);
        more += kj > k, same += kj == k;
      }
      const int at = __ffsll((unsigned long long)__ballot(lane < (int)n && more < left && more + same >= left)) - 1;
      const uint32_t tie = (uint32_t)__builtin_amdgcn_readlane((int)k, at);
      return {tie + 1, tie, left - (uint32_t)__builtin_amdgcn_readlane((int)more, at)};
    }
  }
  return {left > 0 ? lo + 1 : 0xffffffffu, left > 0 ? lo : 0xffffffffu, left};
}

// The `left` numbers of begin .. end - 1 (left below their count) with the largest score(n), ties to the lower number,
// in ascending order to out[at0], out[at0 + 1], ...: each of 16 waves counts what it keeps of its own run and writes it
// behind the waves before it.  Keys past the LDS copy are read again from the scores.
template <int KEYS, typename Score>
__device__ __forceinline__ void choose_largest(ChooseRoom<KEYS>& room, int begin, int end, uint32_t left, int at0,
                                               const Score& score, int32_t* __restrict__ out) {
  constexpr int T = kChooseWaves * 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int held = end - begin < KEYS ? end : begin + KEYS;  // of numbers below it the keys are in LDS
  // (Numbers past the last one are held in 32 bits without a sign: they may pass 2^31 by a few steps.)
  // Each number n, n + step, ... below `to` with its key to f, which is called alike by all lanes of a
  // wave where `to` - n + lane is (numbers from `to` on come with `in` false).
  auto each = [&](uint32_t n, uint32_t to, uint32_t step, auto&& f) {
    for (; n - lane < to; n += step) {
      const int m = (int)min(n, to - 1);
      f((int)n, m < held ? room.key[m - begin] : score_key(score(m)), n < to);
    }
  };
  uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll 4
  for (int n = begin + tid; n < end; n += T) {
    const uint32_t k = score_key(score(n));
    if (n - (uint32_t)begin < KEYS) room.key[n - begin] = k;
    lo = min(lo, k), hi = max(hi, k);
  }
  const Largest c = find_largest(room, lo, hi, left, [&](auto&& f) {
    each(begin + tid, end, T, [&](int, uint32_t k, bool in) { if (in) f(k); });
  });
  const uint32_t seg = ((end - begin + kChooseWaves - 1) / kChooseWaves + 63) / 64 * 64;
  const uint32_t n0 = min(begin + wave * seg, (uint32_t)end), n1 = min((uint32_t)end, n0 + seg);
  uint32_t kept = 0, ties = 0;
  each(n0 + lane, n1, 64, [&](int, uint32_t k, bool in) {
    kept += (uint32_t)__popcll(__ballot(in && k >= c.over));
    ties += (uint32_t)__popcll(__ballot(in && c.left && k == c.tie));
  });
  if (lane == 0) room.total[wave] = kept, room.total[kChooseWaves + wave] = ties;
  __syncthreads();
  uint32_t before = wave_total(lane < wave ? room.total[kChooseWaves + lane] : 0u);
  uint32_t at = (uint32_t)at0 + wave_total(lane < wave ? room.total[lane] : 0u) + min(before, c.left);
  const uint64_t below = (1ull << lane) - 1;
  each(n0 + lane, n1, 64, [&](int n, uint32_t k, bool in) {
    const bool is_tie = in && c.left && k == c.tie;
    const uint64_t bt = __ballot(is_tie);
    const bool keep = (in && k >= c.over) || (is_tie && before + (uint32_t)__popcll(bt & below) < c.left);
    const uint64_t bk = __ballot(keep);
    if (keep) out[at + (uint32_t)__popcll(bk & below)] = n;
    at += (uint32_t)__popcll(bk), before += (uint32_t)__popcll(bt);
  });
}

// The same of thousands of numbers whose scores come in fours: load(n) has those of n .. n + 3, n a multiple of 4 at most
// `end`, and the name of n, and writes name + e for number n + e (kNone: kNone).  Scores that change meanwhile may leave places
// unwritten, but none outside is written.  Each thread holds the keys of 16 numbers, in
// which it counts, and the block's places come from one prefix sum; the numbers past the block's 16,384 are read again.
constexpr uint32_t kNone = 0xffffffffu;
template <typename Load>
__device__ __forceinline__ void choose_fours(ChooseBins& room, int begin, int end, uint32_t left, int at0, const Load& load,
                                             uint32_t* __restrict__ out) {
  constexpr int T = kChooseWaves * 64, Q = 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t first4 = (uint32_t)begin & ~3u, last4 = (uint32_t)(end - 1) & ~3u;
  uint32_t key[Q][4], name[Q], from = first4;  // of the numbers from `from` on
  auto any = [&](int q) { return from + q * 4 * T < (uint32_t)end; };
  // (in 32 bits without a sign: numbers past the last one may pass 2^31)
  auto take = [&](uint32_t slab) {
    from = slab;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const uint32_t n4 = slab + (uint32_t)(q * T + tid) * 4;
      const auto x = load((int)min(n4, last4));
      name[q] = x.name;
#pragma unroll
      for (int e = 0; e < 4; ++e) key[q][e] = n4 + e >= (uint32_t)begin && n4 + e < (uint32_t)end ? score_key(x.score[e]) : 0;  // below all keys
    }
  };
  auto rest = [&](auto&& f) {
    for (uint32_t slab = first4 + Q * 4 * T; slab < (uint32_t)end; slab += Q * 4 * T) {
      take(slab);
      f();
    }
  };
  auto each = [&](auto&& f) {
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (any(q))
#pragma unroll
        for (int e = 0; e < 4; ++e) f(key[q][e]);
  };
  const bool one = first4 + Q * 4 * T >= (uint32_t)end;
  uint32_t lo = 0xffffffffu, hi = 0;
  auto bound = [&](uint32_t k) { lo = min(lo, k ? k : 0xffffffffu), hi = max(hi, k); };
  take(first4);
  each(bound);
  rest([&] { each(bound); });
  const Largest c = find_largest(room, lo, hi, left, [&](auto&& f) {
    if (!one) take(first4);
    each(f);
    rest([&] { each(f); });
  });
  uint32_t kept = 0, ties = 0;  // of the numbers so far
  if (!one) take(first4);
  auto write = [&] {
    uint32_t n[Q], upto[Q];  // kept in the low half, ties in the high one: a slab has 16,384 at most
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      n[q] = upto[q] = 0;
      if (any(q)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) n[q] += (key[q][e] >= c.over ? 1u : 0u) + (key[q][e] == c.tie ? 0x10000u : 0u);
        upto[q] = wave_upto(n[q]);
      }
      if (lane == 63) room.total[q * kChooseWaves + wave] = upto[q];
    }
    __syncthreads();
    const uint32_t all = room.total[lane], sum = wave_upto(all);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (!any(q)) continue;
      const uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)(sum - all), q * kChooseWaves + wave) + upto[q] - n[q];
      uint32_t k = kept + (at & 0xffffu), t = ties + (at >> 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool more = key[q][e] >= c.over, tie = key[q][e] == c.tie;
        const uint32_t to = k + min(t, c.left);
        if ((more || (tie && t < c.left)) && to < left) out[at0 + to] = name[q] == kNone ? kNone : name[q] + e;
        k += more, t += tie;
      }
    }
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    kept += total & 0xffffu, ties += total >> 16;
  };
  write();
  rest([&] {
    __syncthreads();  // room.total is written again
    write();
  });
}

}  // namespace
}  // namespace rfsn
