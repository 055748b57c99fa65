// How a call of the paged attention is cut into blocks, as far as the host knows.  Plain C++.
#pragma once

#include <stdint.h>

#include "rfsn_abi.h"

namespace rfsn {

inline int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// What the kernels take of it.  per_seq > 0: every sequence into that many chunks of `chunk`
// listed positions (a list of pages, or one chunk).  0: by the lengths, which only the device
// knows, into chunks of at least `chunk` positions.
constexpr int kCUs = 256, kTries = 3;
struct Cut {
  int per_seq;
  int units;                // blocks of a chunk (KV heads, and sets of 16 query heads)
  int64_t chunk;
  int64_t longest;          // positions that a chunk has at most
  float one_over[kTries];   // 1 / chunks aimed at, for so many blocks per CU
};
// Chunks aimed at with k blocks on each CU: each sequence adds half of one on average, and a batch
// that fills the chip by itself is cut where a sequence is longer than the mean.
inline int aim(int k, int units, int batch) {
  const int n = k * kCUs / units - batch / 2;
  return n > batch ? n : batch;
}

constexpr double kLastLevelCache = 256 * 1024 * 1024;
// Of fp16 pages a wave drops weights below 2^-33 of the largest that it sees from its products with V, and
// rounds others by as much (paged_attention.hip), so a chunk of four waves is off by at most 2^20 2^-33 of the
// largest |v|, a quarter of fp16's half step.
constexpr int64_t kLongestChunk = 1 << 22;
constexpr int kWideTiles = 8192;   // tiles of 32 positions of a call up to which blocks have many waves

// By sizes and the sequences' capacity; paged_attention.hip cuts by the lengths within it.
struct Plan {
  int64_t slots;  // of partial results
  Cut cut;
  bool wide;      // blocks of many waves
  bool once;      // rows are loaded past the caches
  bool split() const { return cut.per_seq != 1; }
};
inline int waves_of(int D, bool wide) { return !wide || D == 256 ? 4 : D == 64 ? 16 : 8; }  // (256: 8 would spill)
inline Plan plan(const rfsn_paged& p, int q_heads, int count) {
  const int64_t most = (int64_t)(count ? count : p.table_width) * p.page_size;
  const int units = (int)(p.kv_heads * div_up(q_heads / p.kv_heads, 16));
  Plan r;
  // Blocks of many waves have all of a short call's loads in flight (8,192 positions x 8 KV heads of 64: 17 us in
  // blocks of 4 waves, 12 so; 8 x 8,000: 31 in blocks of 4 and 37 so).  They also take a sequence without a
  // merge where its steps cost less than one: 8 steps (4,096 positions of 64, 2,048 of 128) with blocks for most CUs
  // (fp16, 8 KV heads: 24 x 4,000 of 64 43.6 -> 39.7 us, 32 x 1,900 of 128 53.3 -> 47.8, while 16 x 4,000, 128
  // blocks, goes from 31 to 34), 4 with 64 (8 x 2,000: 14.2 -> 13.7), else 3 (1,021: 10.0 -> 8.6; 2,000 as 4: 10.3 ->
  // 12.7).  Blocks of 4 waves take 512 positions so (1,024 x 300: 117 us, in wide blocks 193).
  const int64_t blocks = (int64_t)p.batch * units, tiles = blocks * div_up(most, 32);
  const int most_steps = blocks >= 192 ? 8 : blocks >= 64 ? 4 : 3;
  r.wide = tiles <= kWideTiles ||
           (most > 512 && blocks >= 192 && most <= most_steps * waves_of(p.head_dim, true) * 32);
  // K and V of 256 MB or more, the size of the last-level cache, are gone from it before the next call reads them
  // again: loaded as data that is used once they displace nothing and arrive sooner (32 x 32,768 positions, 8 KV heads
  // of 64: fp16 374 -> 344 us, int8 220 -> 205; 4 x 8,000, 32 of 128: 99 -> 90, 16 x 8,192, 8 of 256: 196 -> 180).
  // What fits stays for the next call (245 MB read again at once: 43 us, loaded so
  // 47), blocks of many waves have less than that, and a list of pages reads few of them.
  // What counts is what the call reads, as far as the host knows it: the pages that the caller says are held, else what
  // the tables have room for, one table once, however many sequences go over it (512 queries over 8,192 positions, 2 KV
  // heads of 256, fp16, took 650 us and 897 loaded so; 48 ragged sequences with 98 MB in a pool of 2.7 GB 24.8 and 27.0).
  double pages = (p.table_stride == 0 ? 1.0 : (double)p.batch) * p.table_width;
  if (pages > p.pages) pages = p.pages;
  if (p.held_pages > 0 && pages > p.held_pages) pages = p.held_pages;
  r.once = !r.wide && count == 0 &&
           pages * p.page_size * p.kv_heads * p.head_dim * (p.type == RFSN_PAGE_FP16 ? 4 : 2) >= kLastLevelCache;
  const int per_step = waves_of(p.head_dim, r.wide) * 32;
  const int64_t least = r.wide ? per_step : 4 * per_step;  // positions of a chunk
  int64_t longest = kLongestChunk;
  while (longest < most && div_up(most, longest) * p.batch > 32768) longest *= 2;  // the grid ends at 65,535 chunks
  if (most <= (r.wide ? most_steps : 4) * per_step) {
    r.slots = p.batch, r.cut = {1, units, most > 0 ? most : 1, longest, {}};
  } else if (count) {
    int64_t n = div_up(r.wide ? kCUs : 4 * kCUs, (int64_t)units * p.batch);
    if (n > div_up(most, least)) n = div_up(most, least);
    if (n < div_up(most, longest)) n = div_up(most, longest);
    const int64_t chunk = div_up(div_up(most, n), per_step) * per_step;
    n = div_up(most, chunk);
    r.slots = n * p.batch, r.cut = {(int)n, units, chunk, longest, {}};
  } else {
    const int first = r.wide ? 1 : 2;
    r.cut = {0, units, least, longest, {}};
    int64_t most_chunks = 0;
    for (int x = 0; x < kTries; ++x) {
      const int n = aim(first + x, units, p.batch);
      r.cut.one_over[x] = 1.f / (float)n;
      most_chunks = n > most_chunks ? n : most_chunks;
    }
    // The sum of ceil(len / size) is at most total / size + batch, and size at least total / target - 0.02
    // (find_chunk) and `least`: below 32767 (0.02 / 512 + 2^-21) < 2 chunks over the target (wide blocks
    // have a `least` of 128 to 512, and at most 8,192 tiles of sequences longer than it).  Chunks of `longest`
    // positions are as many as the sequences' capacity has.
    r.slots = most_chunks + 2 + p.batch;
    if (r.slots < div_up(most, longest) * p.batch) r.slots = div_up(most, longest) * p.batch;
    if (r.slots > div_up(most, least) * p.batch) r.slots = div_up(most, least) * p.batch;
  }
  return r;
}

}  // namespace rfsn
