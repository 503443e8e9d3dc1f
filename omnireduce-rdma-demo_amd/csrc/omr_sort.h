// omr_sort.h — groups tokens by the table row that they name (omr_embed.hip, omr_loss.hip).
#ifndef OMR_SORT_H
#define OMR_SORT_H

#include "omr_elem.h"

namespace omr_elem {

template <class I>
__device__ __forceinline__ bool id_ok(I id, uint32_t rows) {
  return id >= 0 && static_cast<uint64_t>(id) < rows;
}

// Groups the tokens by row in ONE launch without any exchange between workgroups: workgroup p owns the rows
// [p R, p R + R) and reads ALL ids itself (they sit in the L2s: 64 KiB for 8192 int64 ids), counting its own and how
// many are below its range, which is where its piece of the sorted list begins.
//   pass 1  wave w counts the ids of its contiguous part of the tokens in hist[w][id - lo], and notes the tokens it
//           counted, in order, in a list of its own
//   scan    start[v] = ids below v; hist[w][.] = where wave w's first token of that row goes
//   pass 2  the waves walk their lists (or, where a list is full, their tokens again) and place them: within 64 tokens
//           the lanes of equal ids rank themselves by lane (match by ballots over the bits of the local id), so the
//           order within a row is token order; named[i], where it is wanted, is the row of the i-th of the sorted list
// Every workgroup reads T ids: hidden in the L2 up to some 100 k tokens, where a radix sort would take three launches
// for each of three digits.  8192 ids of 65536 rows: 6.9 us; 20011 of 1009: 10.5, whether 8 or 20 loads are in flight and
// 16 or 4 rows are a workgroup's.
constexpr uint32_t kNoRow = ~0u;
constexpr uint32_t kSortList = 512;  // tokens a wave notes

// of a workgroup of WAVES waves: 96 KiB for 16, 12 KiB for 4
template <int WAVES>
struct SortSpace {
  static constexpr uint32_t kRange = 64 * WAVES;  // rows at most: one a thread
  static constexpr int kBits = WAVES == 16 ? 10 : 8;
  static_assert(kRange == 1u << kBits, "a local id's bits");
  uint32_t hist[WAVES * kRange];
  uint32_t list[WAVES][kSortList];  // (token - the wave's first) << kBits | local id
  uint32_t wsum[WAVES], below_w[WAVES], valid;
};

// rows per workgroup of 16 waves: one workgroup a CU where the table is small enough for that
inline uint32_t sort_range(uint32_t rows) {
  const uint32_t each = (rows + 255) / 256;
  return each < 16 ? 16 : each > SortSpace<16>::kRange ? SortSpace<16>::kRange : each;
}

// Workgroup `block` of WAVES waves: the positions of the ids that name one of its rows, by row and in order
// within it: those of row v at perm[start[v] .. start[v + 1]).  start: rows + 1, perm and named (or null): one an id.
template <class I, int WAVES>
__device__ __forceinline__ void sort_by_row(SortSpace<WAVES>& space, uint32_t block, const I* ids, uint32_t tokens, uint32_t rows,
                                            uint32_t range, uint32_t* start, uint32_t* perm, uint32_t* named) {
  constexpr int kSortWaves = WAVES, kSortBits = SortSpace<WAVES>::kBits;
  auto& hist = space.hist;
  auto& list = space.list;
  auto &wsum = space.wsum, &below_w = space.below_w;
  uint32_t& valid = space.valid;
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint32_t lo = block * range, n = min(range, rows - lo);
  for (uint32_t i = tid; i < kSortWaves * range; i += 64 * kSortWaves) hist[i] = 0;
  const uint32_t span = (tokens + 64 * kSortWaves - 1) / (64 * kSortWaves) * 64;  // tokens of a wave
  const uint32_t t0 = min(wave * span, tokens), t1 = min(t0 + span, tokens);
  uint32_t* mine = hist + wave * range;
  uint32_t below = 0, noted = 0;
  __syncthreads();
  constexpr int K = 8;  // loads in flight
  for (uint32_t t = t0; t < t1; t += 64 * K) {
    I id[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t at = t + 64 * k + lane;
      id[k] = at < t1 ? ids[at] : static_cast<I>(-1);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t v = id_ok(id[k], rows) ? static_cast<uint32_t>(id[k]) : ~0u;
      below += v < lo;
      const bool in = v - lo < n;
      const uint64_t who = __ballot(in);
      if (who == 0) continue;
      const uint32_t at = noted + __popcll(who & ((1ull << lane) - 1));
      if (in) {
        atomicAdd(&mine[v - lo], 1u);
        if (at < kSortList) list[wave][at] = (t + 64 * k + lane - t0) << kSortBits | (v - lo);
      }
      noted += static_cast<uint32_t>(__popcll(who));
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) below += __shfl_xor(below, d);
  if (lane == 0) below_w[wave] = below;
  __syncthreads();
  // exclusive scan over the range's rows of their totals, then over the waves within a row
  uint32_t total = 0;
  if (tid < n) {
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) total += hist[w * range + tid];
  }
  uint32_t incl = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t up = __shfl_up(incl, d);
    if (lane >= static_cast<uint32_t>(d)) incl += up;
  }
  if (lane == 63) wsum[wave] = incl;
  __syncthreads();
  uint32_t at = incl - total;
#pragma unroll
  for (uint32_t w = 0; w < kSortWaves; ++w) {
    at += below_w[w];
    if (w < wave) at += wsum[w];
  }
  if (tid < n) {
    start[lo + tid] = at;
    if (lo + tid == rows - 1) start[rows] = valid = at + total;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = hist[w * range + tid];
      hist[w * range + tid] = at;
      at += c;
    }
  }
  __syncthreads();
  // (a list holds token distances of 32 - kBits bits)
  const bool listed = noted <= kSortList && span <= 1u << (32 - kSortBits);
  const uint32_t steps = listed ? noted : t1 - t0;
  for (uint32_t i = 0; i < steps; i += 64) {
    uint32_t v = ~0u, t = t0 + i + lane;
    if (i + lane < steps) {
      if (listed) {
        const uint32_t e = list[wave][i + lane];
        v = e & (SortSpace<WAVES>::kRange - 1);
        t = t0 + (e >> kSortBits);
      } else if (id_ok(ids[t], rows)) {
        v = static_cast<uint32_t>(ids[t]) - lo;
      }
    }
    const bool in = v < n;
    uint64_t same = __ballot(in);
    if (same == 0) continue;
#pragma unroll
    for (int b = 0; b < kSortBits; ++b) {
      const bool bit = (v >> b) & 1;
      const uint64_t m = __ballot(bit);
      same &= bit ? m : ~m;
    }
    const uint32_t leader = in ? static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(same))) - 1 : lane;
    uint32_t base = 0;
    if (in && lane == leader) base = atomicAdd(&mine[v], static_cast<uint32_t>(__popcll(same)));
    base = __shfl(base, static_cast<int>(leader));
    if (in) {
      const uint32_t to = base + __popcll(same & ((1ull << lane) - 1));
      perm[to] = t;
      if (named != nullptr) named[to] = lo + v;
    }
  }
  if (named != nullptr && lo + n == rows)  // behind the last
    for (uint32_t i = valid + tid; i < tokens; i += 64 * kSortWaves) named[i] = kNoRow;
}

}  // namespace omr_elem

#endif
