// omr_embed.hip — embedding lookup with scaling, and the table's gradient by sorted tokens.
//
//   forward   out[t, :] = scale * table[ids[t], :]
//   backward  grad[v, :] (+)= scale * sum over the tokens t with ids[t] = v, in token order, of grad_out[t, :]
//
// An id outside [0, num_rows) names no row (padding): a zero row forward, no contribution backward, whatever values
// the token's row of grad_out holds.  The gradient is the fp32 tensor the sparse all-reduce takes: rows of tokens the
// step did not see are zero blocks.
//
// Every sum has a fixed order, so the same inputs give the same bits: tokens are grouped by a stable sort instead of
// meeting in floating-point atomics.
#include "omr_sort.h"

#include <algorithm>
#include <type_traits>

using namespace omr_elem;

namespace {

// ---------------------------------------------------------------- lookup
//
// Bound by HBM: each looked-up row is read once and each output row written once.  The outputs are swept as one list
// of VEC-element pieces (16 bytes of the table a lane), so a row of any length fills whole waves; a thread takes kLook
// pieces, a workgroup apart, and has all their loads in flight before its first store.  16384 rows of 4096 bf16 take 43
// us, 5.5 TB/s (54 with ordinary stores; a large copy reaches 5.1).
constexpr int kLook = 4;

template <class T, class O, class I, int VEC, class U>
__global__ __launch_bounds__(256) void k_embed(const T* table, uint32_t rows, uint64_t tstride, const I* ids, U pieces,
                                               U per_row, uint32_t dim, float scale, O* out, uint64_t ostride) {
  const U first = static_cast<U>(blockIdx.x) * (256 * kLook) + threadIdx.x;
  U tok[kLook], col[kLook];
  I id[kLook];
#pragma unroll
  for (int j = 0; j < kLook; ++j) {
    const U p = first + static_cast<U>(j) * 256;
    tok[j] = p / per_row;
    col[j] = (p - tok[j] * per_row) * VEC;
    id[j] = p < pieces ? ids[tok[j]] : static_cast<I>(-1);
  }
  float v[kLook][VEC];
#pragma unroll
  for (int j = 0; j < kLook; ++j) {
    if (id_ok(id[j], rows)) {
      load_some<T, VEC>(table + static_cast<uint64_t>(id[j]) * tstride + col[j], dim - static_cast<uint32_t>(col[j]),
                        v[j]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = 0.0f;
    }
  }
#pragma unroll
  for (int j = 0; j < kLook; ++j) {
    if (first + static_cast<U>(j) * 256 >= pieces) break;
    if (id_ok(id[j], rows)) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] *= scale;
    }
    stream_some<O, VEC>(out + static_cast<uint64_t>(tok[j]) * ostride + col[j], dim - static_cast<uint32_t>(col[j]), v[j]);
  }
}

constexpr int kSortWaves = 16;

template <class I>
__global__ __launch_bounds__(64 * kSortWaves) void k_embed_sort(const I* ids, uint32_t tokens, uint32_t rows,
                                                               uint32_t range, uint32_t* start, uint32_t* perm,
                                                               uint32_t* named) {
  __shared__ SortSpace<kSortWaves> space;
  sort_by_row<I>(space, blockIdx.x, ids, tokens, rows, range, start, perm, named);
}

// ---------------------------------------------------------------- sums
//
// Bound by HBM: grad_out is read once and the table's gradient written once (65536 x 1024 fp32: 256 MiB), most of it
// zeros.  Two kinds of workgroups of one launch share the rows:
//   - chunk workgroups take the sorted list in chunks of 16 positions and add up the rows that lie there, all their
//     loads in flight at once.  A row within its chunk is done; of one that goes on (a frequent
//     word) the chunk's piece goes to `partial`, and k_embed_join adds its pieces up in order, a launch later;
//   - fill workgroups store the zeros of the rows that no token names.
// Of every four rows of zeros one is stored as any store and three non-temporally.  The scan of the all-reduce reads the
// table next, and finds some of it in the last-level cache (256 MiB); but a table that fills that cache with dirty lines
// pays for their way out.  8192 tokens of 65536 x 1024 (256 MiB), two tables in turn, with the sort and the join, and
// then together with the scan: 54 us and 100; all stores ordinary 64 and 98, all non-temporal 53 and 110, every second
// one 55 and 97.  32768 tokens: 76 and 129, against 93 and 135, 73 and 134, 82 and 129.  131072 x 1024: 111 and 189,
// against 115 and 194, 100 and 209, 113 and 180.  8192 tokens of 49152 x 1024: 39 and 82, against 48 and 80, 41 and 87,
// 39 and 81.  (Torch's fill of 256 MiB alone takes 40 us.)
// Other forms.  Chunks of 32 in two flights of 16: 8 us more at 65536 x 1024.  Lane groups that sum or zero four rows each:
// 30 more, every row with tokens two dependent loads behind the stores around it.  The zeros, or the chunks, in a launch
// of their own, beside or behind the sort: 1 to 3 more.
constexpr uint32_t kChunk = 16;

struct SumArgs {
  const void* grad_out;
  uint64_t gstride;
  const uint32_t* start;  // [rows + 1]
  const uint32_t* perm;   // the valid tokens by row
  const uint32_t* named;  // their rows, kNoRow behind the last
  uint32_t tokens;
  float* partial;         // [2 * chunks][dim]: the piece of the row that began before the chunk; of the one that goes on
  float* out;
  uint64_t ostride;
  uint32_t rows, dim, chunks, tiles;  // tiles of columns of a chunk workgroup
  float scale;
  int accumulate;
  uint32_t fill;  // rows of a fill workgroup's wave
};

constexpr int VEC = 4;  // columns a lane: 16 bytes of the table

__device__ __forceinline__ void put(const SumArgs& a, uint32_t row, uint32_t c, float (&v)[VEC]) {
  float* o = a.out + static_cast<uint64_t>(row) * a.ostride + c;
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] *= a.scale;
  if (a.accumulate) {
    float old[VEC];
    load_some<float, VEC>(o, a.dim - c, old);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = old[i] + v[i];
  }
  store_some<float, VEC>(o, a.dim - c, v);
}

// blocks [0, chunk_blocks): chunks, 256 VEC columns each; behind them: zeros, `fill` rows a wave
template <class T>
__global__ __launch_bounds__(256) void k_embed_sum(SumArgs a, uint32_t chunk_blocks) {
  const uint32_t lane = threadIdx.x & 63;
  if (blockIdx.x < chunk_blocks) {
    const uint32_t k = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles;
    const uint32_t p0 = k * kChunk, p1 = min(p0 + kChunk, a.tokens);
    const uint32_t c = (tile * 256 + threadIdx.x) * VEC;
    // lane l: the token at position p0 + l, its row and its neighbours', all at once: a load that waits for another one
    // waits behind the zero fills' stores each time
    const uint32_t pos = min(p0 + lane % kChunk, p1 - 1);
    const uint32_t held = a.perm[pos], row = a.named[pos];
    const uint32_t next = pos + 1 < a.tokens ? a.named[pos + 1] : kNoRow;
    const uint32_t before = p0 != 0 ? a.named[p0 - 1] : kNoRow;
    const bool real = p0 + lane < p1 && row != kNoRow;
    const uint32_t here = static_cast<uint32_t>(__popcll(__ballot(real)));
    // its row's tokens here end with it, or go on behind the chunk
    const uint64_t ends = __ballot(real && (row != next || pos + 1 == p1)), on = __ballot(real && row == next);
    const T* g = static_cast<const T*>(a.grad_out) + c;
    float acc[VEC] = {};
    float v[kChunk][VEC];
#pragma unroll
    for (uint32_t i = 0; i < kChunk; ++i) {
      const uint32_t t = __builtin_amdgcn_readlane(held, i);
      if (i < here && c < a.dim) load_some<T, VEC>(g + static_cast<uint64_t>(t) * a.gstride, a.dim - c, v[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < kChunk; ++i) {
      if (i < here) {
#pragma unroll
        for (int x = 0; x < VEC; ++x) acc[x] += v[i][x];
        if (ends >> i & 1) {
          const uint32_t r = __builtin_amdgcn_readlane(row, i);
          const bool began = r == before, goes = on >> i & 1;
          if (c < a.dim) {
            if (!began && !goes)
              put(a, r, c, acc);
            else
              store_some<float, VEC>(a.partial + static_cast<uint64_t>(2 * k + (began ? 0 : 1)) * a.dim + c, a.dim - c, acc);
          }
#pragma unroll
          for (int x = 0; x < VEC; ++x) acc[x] = 0.0f;
        }
      }
    }
    return;
  }
  const uint64_t first = (static_cast<uint64_t>(blockIdx.x - chunk_blocks) * 4 + (threadIdx.x >> 6)) * a.fill;
  for (uint64_t row = first; row < min(first + a.fill, static_cast<uint64_t>(a.rows)); ++row) {
    if (a.start[row] != a.start[row + 1]) continue;
    float* o = a.out + row * a.ostride;
    const float zero[VEC] = {};
    for (uint32_t c = lane * VEC; c < a.dim; c += 64 * VEC) {
      if (row % 4 != 0)
        stream_some<float, VEC>(o + c, a.dim - c, zero);
      else
        store_some<float, VEC>(o + c, a.dim - c, zero);
    }
  }
}

// The row that begins in chunk k and goes on behind it, 64 VEC columns; the four waves each take a quarter of its pieces
// (in order), and wave 0 adds the quarters up.
__global__ __launch_bounds__(256) void k_embed_join(SumArgs a, uint32_t tiles) {
  __shared__ float sums[4][64 * VEC];
  const uint32_t k = blockIdx.x / tiles, tile = blockIdx.x % tiles;
  const uint32_t p0 = k * kChunk, p1 = p0 + kChunk;
  if (p1 >= a.tokens) return;  // nothing goes on behind the last chunk
  const uint32_t row = a.named[p1 - 1];
  if (row == kNoRow || a.named[p1] != row || (p0 != 0 && a.named[p0 - 1] == row)) return;
  const uint32_t e = a.start[row + 1];
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t c = (tile * 64 + lane) * VEC;
  const uint32_t pieces = (e - 1) / kChunk - k + 1, quarter = (pieces + 3) / 4;
  const uint32_t q0 = min(wave * quarter, pieces), q1 = min(q0 + quarter, pieces);
  float acc[VEC] = {};
  if (c < a.dim) {
    for (uint32_t q = q0; q < q1; q += 8) {  // eight pieces in flight, added in order
      float v[8][VEC];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t slot = 2 * (k + q + i) + (q + i == 0 ? 1 : 0);
        if (q + i < q1) load_some<float, VEC>(a.partial + static_cast<uint64_t>(slot) * a.dim + c, a.dim - c, v[i]);
      }
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        if (q + i < q1)
#pragma unroll
          for (int x = 0; x < VEC; ++x) acc[x] += v[i][x];
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) sums[wave][lane * VEC + i] = acc[i];
  __syncthreads();
  if (wave != 0 || c >= a.dim) return;
#pragma unroll
  for (int w = 1; w < 4; ++w)
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] += sums[w][lane * VEC + i];
  put(a, row, c, acc);
}

uint64_t round16(uint64_t b) { return (b + 15) / 16 * 16; }

constexpr uint64_t kMaxBlocks = (1u << 24) - 1;  // of 256 threads: a launch holds fewer than 2^32 threads

}  // namespace

extern "C" {

int omr_embed(const void* table, int table_dtype, uint64_t num_rows, uint32_t dim, uint64_t row_stride,
              const void* ids, int ids64, uint64_t num_ids, float scale, void* out, int out_dtype, uint64_t out_stride,
              omr_stream_t stream) {
  if (!dtype_ok(table_dtype) || !dtype_ok(out_dtype)) return efail("embed: unknown element type");
  if (dim == 0 || dim > OMR_MAX_DIM || num_rows >= (1ull << 31) || num_ids >= (1ull << 31))
    return efail("embed: dim must be 1..%u, rows and ids below 2^31", OMR_MAX_DIM);
  if (out_stride < dim) return efail("embed: the output's row stride is shorter than dim %u", dim);
  if (num_ids == 0) return 0;
  if (ids == nullptr || out == nullptr || (table == nullptr && num_rows != 0)) return efail("embed: NULL pointer");
  return with_dtype(table_dtype, [&](auto t) {
    using T = decltype(t);
    return with_dtype(out_dtype, [&](auto o) {
      using O = decltype(o);
      auto go = [&](auto i) {
        using I = decltype(i);
        constexpr int VEC = 16 / sizeof(T);
        const uint64_t per_row = ceil_div(dim, VEC), pieces = per_row * num_ids;
        const uint64_t grid = ceil_div(pieces, 256 * kLook);
        if (grid > kMaxBlocks) return efail("embed: %llu outputs are too many for one call",
                                               static_cast<unsigned long long>(num_ids * dim));
        const auto* tp = static_cast<const T*>(table);
        auto* op = static_cast<O*>(out);
        const auto* ip = static_cast<const I*>(ids);
        if (pieces + 256 * kLook < (1ull << 32))
          k_embed<T, O, I, VEC, uint32_t><<<static_cast<unsigned>(grid), 256, 0, S(stream)>>>(
              tp, static_cast<uint32_t>(num_rows), row_stride, ip, static_cast<uint32_t>(pieces),
              static_cast<uint32_t>(per_row), dim, scale, op, out_stride);
        else
          k_embed<T, O, I, VEC, uint64_t><<<static_cast<unsigned>(grid), 256, 0, S(stream)>>>(
              tp, static_cast<uint32_t>(num_rows), row_stride, ip, pieces, per_row, dim, scale, op, out_stride);
        return elaunch("omr_embed");
      };
      return ids64 ? go(int64_t{}) : go(int32_t{});
    });
  });
}

size_t omr_embed_grad_workspace_bytes(uint64_t num_ids, uint64_t num_rows, uint32_t dim) {
  if (dim == 0 || dim > OMR_MAX_DIM || num_rows >= (1ull << 31) || num_ids >= (1ull << 31)) return 0;
  const uint64_t chunks = num_ids != 0 ? ceil_div(num_ids, kChunk) : 0;
  return round16(4 * (num_rows + 1)) + 2 * round16(4 * num_ids) + 2 * chunks * round16(4ull * dim);
}

int omr_embed_grad_f32(const void* grad_out, int grad_dtype, uint64_t grad_stride, const void* ids, int ids64,
                       uint64_t num_ids, uint64_t num_rows, uint32_t dim, float scale, float* grad_table,
                       uint64_t table_stride, int accumulate, void* workspace, size_t workspace_bytes,
                       omr_stream_t stream) {
  if (!dtype_ok(grad_dtype)) return efail("embed_grad: unknown element type");
  if (dim == 0 || dim > OMR_MAX_DIM || num_rows >= (1ull << 31) || num_ids >= (1ull << 31))
    return efail("embed_grad: dim must be 1..%u, rows and ids below 2^31", OMR_MAX_DIM);
  if (table_stride < dim) return efail("embed_grad: the table's row stride is shorter than dim %u", dim);
  if (num_rows == 0) return 0;
  if (grad_table == nullptr || workspace == nullptr || (num_ids != 0 && (grad_out == nullptr || ids == nullptr)))
    return efail("embed_grad: NULL pointer");
  if (!aligned(workspace, 16)) return efail("embed_grad: the workspace must be 16-byte aligned");
  if (workspace_bytes < omr_embed_grad_workspace_bytes(num_ids, num_rows, dim))
    return efail("embed_grad: workspace of %zu bytes, %zu needed", workspace_bytes,
                 omr_embed_grad_workspace_bytes(num_ids, num_rows, dim));
  SumArgs a;
  char* ws = static_cast<char*>(workspace);
  a.grad_out = grad_out;
  a.gstride = grad_stride;
  uint32_t* start = reinterpret_cast<uint32_t*>(ws);
  uint32_t* perm = reinterpret_cast<uint32_t*>(ws + round16(4 * (num_rows + 1)));
  a.start = start;
  a.perm = perm;
  uint32_t* named = perm + round16(4 * num_ids) / 4;
  a.named = named;
  a.tokens = static_cast<uint32_t>(num_ids);
  a.partial = reinterpret_cast<float*>(ws + round16(4 * (num_rows + 1)) + 2 * round16(4 * num_ids));
  a.out = grad_table;
  a.ostride = table_stride;
  a.rows = static_cast<uint32_t>(num_rows);
  a.dim = dim;
  a.chunks = num_ids != 0 ? static_cast<uint32_t>(ceil_div(num_ids, kChunk)) : 0;
  a.scale = scale;
  a.accumulate = accumulate != 0;
  a.fill = static_cast<uint32_t>(ceil_div(num_rows, 1u << 25));  // one, but for a table of more than 2^25 rows
  a.tiles = static_cast<uint32_t>(ceil_div(dim, 256 * VEC));
  const uint64_t chunk_blocks = static_cast<uint64_t>(a.chunks) * a.tiles, join_tiles = ceil_div(dim, 64 * VEC),
                 blocks = chunk_blocks + (accumulate ? 0 : ceil_div(num_rows, 4 * a.fill));
  if (blocks > kMaxBlocks || a.chunks * join_tiles > kMaxBlocks)
    return efail("embed_grad: too many tokens or rows for one call");
  const uint32_t range = sort_range(a.rows);
  const unsigned sorters = static_cast<unsigned>(ceil_div(a.rows, range));
  if (ids64)
    k_embed_sort<int64_t><<<sorters, 64 * kSortWaves, 0, S(stream)>>>(static_cast<const int64_t*>(ids), a.tokens, a.rows,
                                                                     range, start, perm, named);
  else
    k_embed_sort<int32_t><<<sorters, 64 * kSortWaves, 0, S(stream)>>>(static_cast<const int32_t*>(ids), a.tokens, a.rows,
                                                                     range, start, perm, named);
  if (const int rc = elaunch("omr_embed_grad_f32 (sort)")) return rc;
  return with_dtype(grad_dtype, [&](auto t) {
    using T = decltype(t);
    if (blocks == 0) return 0;
    k_embed_sum<T><<<static_cast<unsigned>(blocks), 256, 0, S(stream)>>>(a, static_cast<uint32_t>(chunk_blocks));
    if (const int rc = elaunch("omr_embed_grad_f32")) return rc;
    if (a.chunks <= 1) return 0;
    k_embed_join<<<static_cast<unsigned>(a.chunks * join_tiles), 256, 0, S(stream)>>>(
        a, static_cast<uint32_t>(join_tiles));
    return elaunch("omr_embed_grad_f32 (join)");
  });
}

}  // extern "C"
