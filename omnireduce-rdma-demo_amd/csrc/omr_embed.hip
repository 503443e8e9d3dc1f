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
#include "omr_elem.h"

#include <algorithm>
#include <type_traits>

using namespace omr_elem;

namespace {

template <class I>
__device__ __forceinline__ bool id_ok(I id, uint32_t rows) {
  return id >= 0 && static_cast<uint64_t>(id) < rows;
}

// ---------------------------------------------------------------- lookup
//
// Bound by HBM: each looked-up row is read once and each output row written once.  The outputs are swept as one list
// of VEC-element pieces (16 bytes of the table a lane), so a row of any length fills whole waves; a thread takes kLook
// pieces, a workgroup apart, and has all their loads in flight before its first store.
constexpr int kLook = 4;

template <class T, class O, class I, int VEC, class U>
__global__ __launch_bounds__(256) void k_embed(const T* table, uint32_t rows, uint64_t tstride, const I* ids, U pieces,
                                               U per_row, float scale, O* out, uint64_t ostride) {
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
      load_f32<T, VEC>(table + static_cast<uint64_t>(id[j]) * tstride + col[j], v[j]);
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
    store_f32<O, VEC>(out + static_cast<uint64_t>(tok[j]) * ostride + col[j], v[j]);
  }
}

// ---------------------------------------------------------------- sort
//
// Groups the tokens by row in ONE launch without any exchange between workgroups: workgroup p owns the rows
// [p R, p R + R) and reads ALL ids itself (they sit in the L2s: 64 KiB for 8192 int64 ids), counting its own and how
// many are below its range, which is where its piece of the sorted list begins.
//   pass 1  wave w counts the ids of its contiguous sixteenth of the tokens in hist[w][id - lo]
//   scan    start[v] = ids below v; hist[w][.] = where wave w's first token of that row goes
//   pass 2  the waves walk their tokens again and place them: within 64 tokens the lanes of equal ids rank themselves
//           by lane (match by ballots over the bits of the local id), so the order within a row is token order
// A radix sort by 8 bits took the launches of three passes (about nine); this is one, and its work, T ids per
// workgroup, is hidden in the L2 up to some 100 k tokens.
constexpr int kSortWaves = 16;
constexpr int kSortRange = 1024;      // rows per workgroup at most: 64 KiB of histogram, two workgroups a CU
constexpr int kSortBits = 10;

template <class I>
__global__ __launch_bounds__(64 * kSortWaves) void k_embed_sort(const I* ids, uint32_t tokens, uint32_t rows,
                                                               uint32_t range, uint32_t* start, uint32_t* perm) {
  __shared__ uint32_t hist[kSortWaves * kSortRange];
  __shared__ uint32_t wsum[kSortWaves], below_w[kSortWaves];
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint32_t lo = blockIdx.x * range, n = min(range, rows - lo);
  for (uint32_t i = tid; i < kSortWaves * kSortRange; i += 64 * kSortWaves) hist[i] = 0;
  const uint32_t span = (tokens + 64 * kSortWaves - 1) / (64 * kSortWaves) * 64;  // tokens of a wave
  const uint32_t t0 = min(wave * span, tokens), t1 = min(t0 + span, tokens);
  uint32_t* mine = hist + wave * kSortRange;
  uint32_t below = 0;
  __syncthreads();
#pragma unroll 4
  for (uint32_t t = t0 + lane; t < t1; t += 64) {
    const I id = ids[t];
    if (id_ok(id, rows)) {
      const uint32_t v = static_cast<uint32_t>(id);
      below += v < lo;
      if (v - lo < n) atomicAdd(&mine[v - lo], 1u);
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) below += __shfl_xor(below, d);
  if (lane == 0) below_w[wave] = below;
  __syncthreads();
  // exclusive scan over the range's rows of their totals, then over the waves within a row
  uint32_t total = 0;
  for (int w = 0; w < kSortWaves; ++w) total += hist[w * kSortRange + tid];
  uint32_t incl = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t up = __shfl_up(incl, d);
    if (lane >= static_cast<uint32_t>(d)) incl += up;
  }
  if (lane == 63) wsum[wave] = incl;
  __syncthreads();
  uint32_t at = incl - total;
  for (uint32_t w = 0; w < kSortWaves; ++w) {
    at += below_w[w];
    if (w < wave) at += wsum[w];
  }
  if (tid < n) start[lo + tid] = at;
  if (lo + n == rows && tid == n - 1) start[rows] = at + total;
  for (int w = 0; w < kSortWaves; ++w) {
    const uint32_t c = hist[w * kSortRange + tid];
    hist[w * kSortRange + tid] = at;
    at += c;
  }
  __syncthreads();
  for (uint32_t t = t0; t < t1; t += 64) {
    uint32_t v = ~0u;
    if (t + lane < t1) {
      const I id = ids[t + lane];
      if (id_ok(id, rows)) v = static_cast<uint32_t>(id) - lo;
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
    if (in) perm[base + __popcll(same & ((1ull << lane) - 1))] = t + lane;
  }
}

// ---------------------------------------------------------------- sums
//
// Bound by HBM: grad_out is read once and the table's gradient written once (65536 x 1024 fp32: 256 MiB), most of it
// zeros.  k_embed_rows gives a group of lanes one row and lets it add the row's tokens up, or store zeros.  A row with
// more than `chunk` tokens (a frequent word) would hold its wave for long, so such rows are summed in pieces: the
// sorted list is cut into chunks, k_embed_partial adds up each chunk's tokens of such rows (at most two: one that began
// earlier and one that goes on), and a workgroup of k_embed_rows's launch adds the row's pieces up in order.
struct SumArgs {
  const void* grad_out;
  uint64_t gstride;
  const void* ids;
  const uint32_t* start;  // [rows + 1]
  const uint32_t* perm;   // the valid tokens by row
  float* partial;         // [2 * chunks][dim]
  float* out;
  uint64_t ostride;
  uint32_t rows, dim, chunk, chunks, tiles;  // tiles of columns
  float scale;
  int accumulate;
};

template <class I>
__device__ __forceinline__ uint32_t row_at(const SumArgs& a, uint32_t pos) {
  return static_cast<uint32_t>(static_cast<const I*>(a.ids)[a.perm[pos]]);
}

// acc += the rows of grad_out of the sorted positions [p0, p1), in order, at columns c + j * step
template <class T, int VEC, int NJ>
__device__ __forceinline__ void add_tokens(const SumArgs& a, uint32_t p0, uint32_t p1, uint32_t c, uint32_t step,
                                           float (&acc)[NJ][VEC]) {
  const T* g = static_cast<const T*>(a.grad_out) + c;
  constexpr int K = NJ >= 4 ? 2 : 8;  // tokens in flight
  uint32_t p = p0;
  for (; p + K <= p1; p += K) {
    float v[K][NJ][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const T* r = g + static_cast<uint64_t>(a.perm[p + k]) * a.gstride;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        if (c + j * step < a.dim) load_f32<T, VEC>(r + j * step, v[k][j]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        if (c + j * step < a.dim)
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[j][i] += v[k][j][i];
  }
  for (; p < p1; ++p) {
    const T* r = g + static_cast<uint64_t>(a.perm[p]) * a.gstride;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if (c + j * step < a.dim) {
        float v[VEC];
        load_f32<T, VEC>(r + j * step, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[j][i] += v[i];
      }
  }
}

// one wave: columns [wave tile), one chunk's piece(s)
template <class T, class I, int VEC>
__global__ __launch_bounds__(256) void k_embed_partial(SumArgs a) {
  const uint32_t valid = a.start[a.rows];
  const uint32_t k = blockIdx.x;
  const uint32_t p0 = k * a.chunk, p1 = min(p0 + a.chunk, valid);
  if (p0 >= p1) return;
  const uint32_t c = (blockIdx.y * 256 + threadIdx.x) * VEC;
  const uint32_t r0 = row_at<I>(a, p0), r1 = row_at<I>(a, p1 - 1);
  const uint32_t s0 = a.start[r0], e0 = a.start[r0 + 1], s1 = a.start[r1], e1 = a.start[r1 + 1];
  if (c >= a.dim) return;
  if (e0 - s0 > a.chunk) {  // the row at the chunk's first position
    float acc[1][VEC] = {};
    add_tokens<T, VEC, 1>(a, p0, min(e0, p1), c, 0, acc);
    store_f32<float, VEC>(a.partial + static_cast<uint64_t>(2 * k) * a.dim + c, acc[0]);
  }
  if (r1 != r0 && e1 - s1 > a.chunk) {  // the row that goes on behind it
    float acc[1][VEC] = {};
    add_tokens<T, VEC, 1>(a, s1, p1, c, 0, acc);
    store_f32<float, VEC>(a.partial + static_cast<uint64_t>(2 * k + 1) * a.dim + c, acc[0]);
  }
}

template <int VEC>
__device__ __forceinline__ void put(const SumArgs& a, uint32_t row, uint32_t c, float (&v)[VEC]) {
  float* o = a.out + static_cast<uint64_t>(row) * a.ostride + c;
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] *= a.scale;
  if (a.accumulate) {
    float old[VEC];
    load_f32<float, VEC>(o, old);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = old[i] + v[i];
  }
  store_f32<float, VEC>(o, v);
}

constexpr int kRowsNJ = 4;

// blocks [0, chunks * tiles): the rows of many tokens; behind them: `lpr` lanes a row, every other row
template <class T, class I, int VEC>
__global__ __launch_bounds__(256) void k_embed_rows(SumArgs a, uint32_t join_blocks, uint32_t lpr_log) {
  if (blockIdx.x < join_blocks) {
    // The row that begins in chunk k and goes on behind it, columns of this tile; the four waves each take a quarter
    // of its pieces (in order), and wave 0 adds the quarters up.
    __shared__ float sums[4][64 * VEC];
    const uint32_t valid = a.start[a.rows];
    const uint32_t k = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles;
    const uint32_t p0 = k * a.chunk, p1 = min(p0 + a.chunk, valid);
    if (p0 >= p1) return;
    const uint32_t row = row_at<I>(a, p1 - 1), s = a.start[row], e = a.start[row + 1];
    if (e - s <= a.chunk || s < p0) return;
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t c = (tile * 64 + lane) * VEC;
    const uint32_t pieces = (e - 1) / a.chunk - k + 1, quarter = (pieces + 3) / 4;
    const uint32_t q0 = min(wave * quarter, pieces), q1 = min(q0 + quarter, pieces);
    float acc[VEC] = {};
    if (c < a.dim) {
      for (uint32_t q = q0; q < q1; q += 8) {  // eight pieces in flight, added in order
        float v[8][VEC];
#pragma unroll
        for (uint32_t k8 = 0; k8 < 8; ++k8) {
          const uint32_t at = q + k8;
          const uint32_t slot = 2 * (k + at) + (at == 0 && s != p0 ? 1 : 0);
          if (at < q1) load_f32<float, VEC>(a.partial + static_cast<uint64_t>(slot) * a.dim + c, v[k8]);
        }
#pragma unroll
        for (uint32_t k8 = 0; k8 < 8; ++k8)
          if (q + k8 < q1)
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] += v[k8][i];
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) sums[wave][lane * VEC + i] = acc[i];
    __syncthreads();
    if (wave == 0 && c < a.dim) {
#pragma unroll
      for (int w = 1; w < 4; ++w)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += sums[w][lane * VEC + i];
      put<VEC>(a, row, c, acc);
    }
    return;
  }
  const uint32_t lpr = 1u << lpr_log;
  const uint64_t unit = (static_cast<uint64_t>(blockIdx.x - join_blocks) * 256 + threadIdx.x) >> lpr_log;
  const uint32_t sub = threadIdx.x & (lpr - 1), step = lpr * VEC;
  const uint32_t tiles = (a.dim + step * kRowsNJ - 1) / (step * kRowsNJ);
  const uint64_t row64 = unit / tiles;
  if (row64 >= a.rows) return;
  const uint32_t row = static_cast<uint32_t>(row64);
  const uint32_t c = static_cast<uint32_t>(unit - row64 * tiles) * step * kRowsNJ + sub * VEC;
  const uint32_t s = a.start[row], e = a.start[row + 1];
  if (e - s > a.chunk || (a.accumulate && s == e)) return;
  float acc[kRowsNJ][VEC] = {};
  if (s != e) add_tokens<T, VEC, kRowsNJ>(a, s, e, c, step, acc);
#pragma unroll
  for (int j = 0; j < kRowsNJ; ++j)
    if (c + j * step < a.dim) put<VEC>(a, row, c + j * step, acc[j]);
}

// Tokens of a chunk: a row of n tokens is added up by one wave until n > chunk, and by n / chunk pieces of chunk
// tokens and then one chain of n / chunk pieces beyond, so the longest chain is about chunk + tokens / chunk.
uint32_t chunk_tokens(uint64_t tokens) {
  uint32_t c = 64;
  while (c < 1024 && static_cast<uint64_t>(c) * c < tokens) c *= 2;
  return c;
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
      constexpr int W = 16 / sizeof(T);
      // whole 16-byte pieces of the table where every row begins on one (and the output's rows on its own 16 bytes, or
      // less where its pieces are shorter)
      constexpr size_t OB = W * sizeof(O) < 16 ? W * sizeof(O) : 16;
      const bool wide = dim % W == 0 && row_stride % W == 0 && aligned(table, 16) &&
                        out_stride * sizeof(O) % OB == 0 && aligned(out, OB);
      auto go = [&](auto i, auto vec) {
        using I = decltype(i);
        constexpr int VEC = decltype(vec)::value;
        const uint64_t per_row = dim / VEC, pieces = per_row * num_ids;
        const uint64_t grid = ceil_div(pieces, 256 * kLook);
        if (grid > kMaxBlocks) return efail("embed: %llu outputs are too many for one call",
                                               static_cast<unsigned long long>(num_ids * dim));
        const auto* tp = static_cast<const T*>(table);
        auto* op = static_cast<O*>(out);
        const auto* ip = static_cast<const I*>(ids);
        if (pieces + 256 * kLook < (1ull << 32))
          k_embed<T, O, I, VEC, uint32_t><<<static_cast<unsigned>(grid), 256, 0, S(stream)>>>(
              tp, static_cast<uint32_t>(num_rows), row_stride, ip, static_cast<uint32_t>(pieces),
              static_cast<uint32_t>(per_row), scale, op, out_stride);
        else
          k_embed<T, O, I, VEC, uint64_t><<<static_cast<unsigned>(grid), 256, 0, S(stream)>>>(
              tp, static_cast<uint32_t>(num_rows), row_stride, ip, pieces, per_row, scale, op, out_stride);
        return elaunch("omr_embed");
      };
      if (wide)
        return ids64 ? go(int64_t{}, std::integral_constant<int, W>{}) : go(int32_t{}, std::integral_constant<int, W>{});
      return ids64 ? go(int64_t{}, std::integral_constant<int, 1>{}) : go(int32_t{}, std::integral_constant<int, 1>{});
    });
  });
}

size_t omr_embed_grad_workspace_bytes(uint64_t num_ids, uint64_t num_rows, uint32_t dim) {
  // (a call of fewer tokens may take smaller chunks, and more of them: the space is for any call of up to num_ids)
  uint64_t chunks = 0;
  for (uint64_t c = 64; c <= 1024; c *= 2) {
    const uint64_t n = num_ids < c * c || c == 1024 ? num_ids : c * c;
    if (n > chunk_tokens(n)) chunks = std::max(chunks, ceil_div(n, chunk_tokens(n)));
  }
  return round16(4 * (num_rows + 1)) + round16(4 * num_ids) + 2 * chunks * round16(4ull * dim);
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
  a.ids = ids;
  uint32_t* start = reinterpret_cast<uint32_t*>(ws);
  uint32_t* perm = reinterpret_cast<uint32_t*>(ws + round16(4 * (num_rows + 1)));
  a.start = start;
  a.perm = perm;
  a.partial = reinterpret_cast<float*>(ws + round16(4 * (num_rows + 1)) + round16(4 * num_ids));
  a.out = grad_table;
  a.ostride = table_stride;
  a.rows = static_cast<uint32_t>(num_rows);
  a.dim = dim;
  a.chunk = chunk_tokens(num_ids);
  a.chunks = num_ids > a.chunk ? static_cast<uint32_t>(ceil_div(num_ids, a.chunk)) : 0;
  a.scale = scale;
  a.accumulate = accumulate != 0;
  const uint32_t tokens = static_cast<uint32_t>(num_ids);
  // rows per sorting workgroup: one workgroup a CU where the table is small enough for that
  uint64_t range = ceil_div(num_rows, 256);
  if (range > kSortRange) range = kSortRange;
  if (range < 16) range = 16;
  const unsigned sorters = static_cast<unsigned>(ceil_div(num_rows, range));
  if (ids64)
    k_embed_sort<int64_t><<<sorters, 64 * kSortWaves, 0, S(stream)>>>(
        static_cast<const int64_t*>(ids), tokens, a.rows, static_cast<uint32_t>(range), start, perm);
  else
    k_embed_sort<int32_t><<<sorters, 64 * kSortWaves, 0, S(stream)>>>(
        static_cast<const int32_t*>(ids), tokens, a.rows, static_cast<uint32_t>(range), start, perm);
  if (const int rc = elaunch("omr_embed_grad_f32 (sort)")) return rc;
  return with_dtype(grad_dtype, [&](auto t) {
    using T = decltype(t);
    const bool wide = dim % 4 == 0 && grad_stride % 4 == 0 && table_stride % 4 == 0 &&
                      aligned(grad_out, 4 * sizeof(T)) && aligned(grad_table, 16);
    auto go = [&](auto i, auto vec) {
      using I = decltype(i);
      constexpr int VEC = decltype(vec)::value;
      if (a.chunks != 0) {
        const dim3 grid(a.chunks, static_cast<unsigned>(ceil_div(dim, 256 * VEC)));
        k_embed_partial<T, I, VEC><<<grid, 256, 0, S(stream)>>>(a);
        if (const int rc = elaunch("omr_embed_grad_f32 (partial)")) return rc;
      }
      a.tiles = static_cast<uint32_t>(ceil_div(dim, 64 * VEC));
      uint32_t lpr_log = 6;
      while (lpr_log > 2 && (1u << (lpr_log - 1)) * VEC * kRowsNJ >= dim) --lpr_log;
      const uint64_t join = static_cast<uint64_t>(a.chunks) * a.tiles;
      const uint64_t units = num_rows * ceil_div(dim, (static_cast<uint64_t>(VEC) << lpr_log) * kRowsNJ);
      const uint64_t blocks = join + ceil_div(units, 256u >> lpr_log);
      if (blocks > kMaxBlocks) return efail("embed_grad: the table is too large for one call");
      k_embed_rows<T, I, VEC><<<static_cast<unsigned>(blocks), 256, 0, S(stream)>>>(a, static_cast<uint32_t>(join),
                                                                                   lpr_log);
      return elaunch("omr_embed_grad_f32");
    };
    if (wide)
      return ids64 ? go(int64_t{}, std::integral_constant<int, 4>{}) : go(int32_t{}, std::integral_constant<int, 4>{});
    return ids64 ? go(int64_t{}, std::integral_constant<int, 1>{}) : go(int32_t{}, std::integral_constant<int, 1>{});
  });
}

}  // extern "C"
