// omr_loss.hip — softmax cross entropy over a large vocabulary, in pieces of the vocabulary, without the logits.
//
//   z = hidden weight^T                     [tokens, vocab]
//   lse[n] = log sum_v exp z[n, v],  loss[n] = lse[n] - z[n, target[n]]     (0 where the target names no row)
//   G[n, v] = exp(z[n, v] - lse[n]) - (v == target[n])
//   grad_hidden[n] = grad_loss[n] sum_v G[n, v] weight[v],  grad_weight[v] (+)= sum_n G[n, v] grad_loss[n] hidden[n]
//
// Everything is matrix products on the 16-bit matrix instructions, bound by them from some 256 tokens on (below that by
// reading the weight).  The forward product keeps no logits: a wave folds its piece of the vocabulary into a running
// maximum and sum of exponentials a token, and k_merge joins the pieces.  The backward recomputes a piece of the logits
// (2 T V D of 8 T V D operations), stores G of that piece in 16 bits, and multiplies it with the weight and with the
// hidden states.
//
// 8192 tokens of 2048 against 32768 bf16 rows: 870 us forward (1.26 PFLOP/s; a library product of these sizes that stores
// its result takes 890), then 480 for each half of the vocabulary's G, 427 for its part of grad_weight and as much for that of
// grad_hidden (the library, on these layouts, 470 to 510 and 440 to 460): 3.4 ms in all, 1.3 PFLOP/s.  2048 tokens of 4096
// against 131072 rows forward: 1.57 ms, 1.40 PFLOP/s, as the library's product.  What bounds them is the power: the clock
// falls to 1.6 to 1.9 GHz of 2.4, with the matrix units busy 66 to 74 % of it.  The passes over few tiles (333 tokens of
// 520 against 5003 rows: 14 us forward, 33 to 35 back) are bound by their two and three (in fp16 four) launches, each too
// short to fill the CUs' pipelines.
//
// Roundings to 16 bits, besides the outputs':
//   - G, times 2^12 so that fp16 keeps the small probabilities normal (2^-26 and up).  The targets' entries, exp(..) - 1,
//     outweigh the others together: what their rounding loses (`lost`, one value a token) is added to both products, to
//     grad_hidden in fp32, to grad_weight as a product of its own in 16 bits (2^-18 of the entry remains in bf16).  Without
//     that a target's row was off by up to 2^-9 in bf16, however many tokens share it: 2^12 (p - 1) rounds to -2^12 for
//     every p below 2^-9, always to the same side.
//   - hidden[n] * (grad_loss[n] / max |grad_loss|) for grad_weight's sum over tokens: exact where grad_loss is the same
//     for every token (the mean and the sum), else one rounding.  In fp16 these products are scaled by the power of two that
//     brings the largest of them to 2^13 or more: the one rounding then holds down to 2^-27 of the largest (without it, one
//     of 1e-6 of the largest |grad_loss| was off by 2 %, and one of 1e-8 lost).
// Sums are in fp32 throughout.
#include "omr_sort.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

using namespace omr_elem;

namespace {

constexpr float kGScale = 4096.0f, kLog2E = 1.44269504f;
constexpr uint32_t kMaxStride = 1u << 22;  // elements: a tile's 32-bit byte offsets hold 256 rows of it

// 16 zero bytes: what lanes past the end of a product's inner dimension load
__device__ __attribute__((aligned(16))) uint32_t g_zero[4];

template <class T>
using frag = vec_t<T, 8>;

__device__ __forceinline__ v4f mma(const frag<__bf16>& a, const frag<__bf16>& b, const v4f& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mma(const frag<_Float16>& a, const frag<_Float16>& b, const v4f& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// ---------------------------------------------------------------- operand tiles
//
// C[m, n] = sum_k A(m, k) B(n, k).  An operand is stored with its inner dimension k consecutive (a "row" operand, element
// (m, k) at p[m ld + k]) or with m consecutive (a "column" operand, p[k ld + m]); neither is transposed in memory.  A
// workgroup's tile of ROWS x 64 goes from global memory straight into LDS in 16-byte pieces, which fill LDS in lane
// order; which piece a lane fetches is permuted so that the reads below spread over the banks:
//   row operand     LDS row m: 8 pieces, piece c at place c ^ (m & 7); a lane reads 8 consecutive k of its row (b128)
//   column operand  LDS row k: ROWS / 8 pieces in pairs, pair p at p ^ h(k), h = bits 0, 1, 3, 4 of k: the 16 rows that a
//                   transposing read (ds_read_b64_tr_b16: 4 k of one m a lane) touches at once lie in different banks
constexpr int kBK = 64;

__device__ __forceinline__ uint32_t pair_hash(uint32_t k) { return (k & 3) | ((k >> 3) & 3) << 2; }

template <class T>
struct Operand {
  const T* p;
  uint64_t ld;
  uint32_t rows;  // m (or n) extent; a column operand's is a multiple of 8
};

template <class T, int ROWS, int NT, bool COL>
struct Tile {
  static constexpr int kPieces = ROWS * 8 / NT;
  const char* base;          // this step's tile
  uint32_t off[kPieces];     // bytes from there
  uint64_t inc;

  // the piece's first k within a step
  __device__ __forceinline__ uint32_t kfirst(int i) const {
    const uint32_t q = i * NT + threadIdx.x;
    return COL ? q / (ROWS / 8) : ((q & 7) ^ (q >> 3 & 7)) * 8;
  }

  __device__ __forceinline__ void init(const Operand<T>& o, uint32_t row0, uint64_t kbegin) {
    const uint32_t t = threadIdx.x;
    row0 = min(row0, o.rows - 1);  // (a tile that lies past the end altogether)
    if constexpr (!COL) {
      base = reinterpret_cast<const char*>(o.p + row0 * o.ld + kbegin);
      inc = kBK * sizeof(T);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const uint32_t q = i * NT + t, m = q >> 3, c = (q & 7) ^ (m & 7);
        // rows past the end repeat the last one: they reach only results that are not stored
        const uint32_t row = min(row0 + m, o.rows - 1) - row0;
        off[i] = static_cast<uint32_t>((row * o.ld + c * 8) * sizeof(T));
      }
    } else {
      base = reinterpret_cast<const char*>(o.p + kbegin * o.ld + row0);
      inc = kBK * o.ld * sizeof(T);
      constexpr uint32_t kRow = ROWS / 8;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const uint32_t q = i * NT + t, k = q / kRow, c = q % kRow;
        uint32_t m = ((c >> 1) ^ (pair_hash(k) % (kRow / 2))) * 16 + (c & 1) * 8;
        if (row0 + m >= o.rows) m = 0;
        off[i] = static_cast<uint32_t>((k * o.ld + m) * sizeof(T));
      }
    }
  }

  __device__ __forceinline__ uint32_t place(const T* lds) const {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) T*)(lds))) +
           wave * 1024;
  }

  // This lane's piece i of a whole step's tile into `lds` (place() of it).
  // In inline assembly, and not as the builtin, because the compiler waits for all such loads in flight before any
  // transposing read from LDS; the product's own wait stands in front of the barrier behind which a tile is read.  The
  // loads write no register, and m0 (the LDS address) is set in the same block, with the wait state it needs.
  __device__ __forceinline__ void load(int i, uint32_t to) const {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(to + i * NT * 16), "v"(off[i]), "s"(base)
                 : "memory");
  }
  __device__ __forceinline__ void advance() { base += inc; }

  // a column operand's tile whose k-th row is row which[k] of the operand, k < left; zeros behind them
  __device__ __forceinline__ void load_rows(const Operand<T>& o, uint32_t row0, const uint32_t* which, uint32_t left,
                                            uint32_t to) const {
    static_assert(COL, "rows of k");
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const uint32_t k = kfirst(i), at = off[i] - static_cast<uint32_t>(k * o.ld * sizeof(T));
      const char* src = k < left ? reinterpret_cast<const char*>(o.p + which[k] * o.ld + row0) + at
                                 : reinterpret_cast<const char*>(g_zero);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                   :
                   : "s"(to + i * NT * 16), "v"(src)
                   : "memory");
    }
  }

  // a tile of `left` k, zeros behind them
  __device__ __forceinline__ void load_end(uint32_t to, uint32_t left) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const char* src = kfirst(i) < left ? base + off[i] : reinterpret_cast<const char*>(g_zero);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                   :
                   : "s"(to + i * NT * 16), "v"(src)
                   : "memory");
    }
  }
};

// A wave's fragments of NF times 16 rows from row `row0` (a multiple of 16 NF) on.  Their places differ by an exclusive
// or with a constant: one register holds the first, and the others are formed at each read (kept from being formed once
// and spilled).
template <class T, int ROWS, int NF, bool COL>
struct Frags {
  uint32_t at;

  __device__ __forceinline__ void init(uint32_t row0) {
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    if constexpr (!COL) {
      at = ((row0 + r) * 8 + (g ^ (r & 7))) * 8;
    } else {
      const uint32_t k = 8 * g + (r >> 2), h = pair_hash(k) % (ROWS / 16);
      at = k * ROWS + ((row0 >> 4) ^ h) * 16 + (r & 3) * 4;
    }
  }

  __device__ __forceinline__ frag<T> get(const T* lds, int half, int i) const {
    if constexpr (!COL) {
      return *reinterpret_cast<const frag<T>*>(lds + (at ^ (half * 4 * 8)) + i * 16 * kBK);
    } else {
      typedef short s4 __attribute__((ext_vector_type(4)));
      using lp = __attribute__((address_space(3))) s4*;
      const T* p = lds + (at ^ (i * 16)) + half * 32 * ROWS;
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(uintptr_t)(p));
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(uintptr_t)(p + 4 * ROWS));
      return __builtin_bit_cast(frag<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }

  // hides the place from the compiler, which would form all the others ahead of the loop and spill them
  __device__ __forceinline__ void touch() { asm volatile("" : "+v"(at)); }
};

// ---------------------------------------------------------------- the product
//
// The workgroup's tile is BM x BN, WM x WN waves of (BM / WM) x (BN / WN); a ring of R LDS buffers, one barrier a step of
// 64: behind it the tile R steps on starts on its way into the buffer that the step has done with.
enum { kStats, kGrad, kHidden, kWeight };

template <class T>
struct GemmArgs {
  Operand<T> a, b;
  uint32_t k;               // inner extent
  uint32_t mt, nt, splits;  // tiles; the inner dimension in `splits` parts of ksplit
  uint32_t ksplit;
  // kStats, kGrad: m = vocabulary rows of the piece (from v0 on), n = tokens
  const void* targets;
  int targets64;
  uint32_t v0, vocab, tokens;
  float* stats;             // [tokens][2 * pieces]: maximum and sum of each wave's part of the vocabulary
  uint32_t pieces;
  float* ztarget;           // [tokens]
  const float* lse;
  T* g;                     // [tokens][ldg]
  uint32_t ldg;
  // kHidden: m = columns, n = tokens; kWeight: m = columns, n = vocabulary rows of the piece
  uint32_t dim;
  float* acc;               // [splits][tokens][dim]
  int first, last;          // the sum over the pieces begins; is complete and goes to `out`
  const float* up;          // grad_loss, upstride apart
  uint64_t upstride;
  const float* amax;        // [2] the largest |grad_loss| of the tokens with a target; the scale of the hidden states' copy
  float* lost;              // [tokens] what the target's entry of G lost in rounding
  Operand<T> w;             // kHidden: the whole weight
  const uint32_t *start, *perm;  // kWeight: the tokens by target
  void* out;
  uint64_t ostride;
  int out_f32, accumulate;
};

template <class T>
__device__ __forceinline__ int target_of(const GemmArgs<T>& a, uint32_t n) {
  const int64_t t = a.targets64 ? static_cast<const int64_t*>(a.targets)[n] : static_cast<const int32_t*>(a.targets)[n];
  return t >= 0 && t < a.vocab ? static_cast<int>(t) : -1;
}

// a token's factor: its grad_loss, 0 without a target (whatever grad_loss holds)
template <class T>
__device__ __forceinline__ float factor_of(const GemmArgs<T>& a, uint32_t n) {
  return target_of(a, n) >= 0 ? a.up[n * a.upstride] : 0.0f;
}

// (maximum, sum of exp(. - maximum)) of two parts together; a part of nothing is (-inf, 0)
__device__ __forceinline__ float2 join(float2 p, float2 q) {
  const float top = fmaxf(p.x, q.x), from = top == -INFINITY ? 0.0f : top;
  return make_float2(top, p.y * expf(p.x - from) + q.y * expf(q.x - from));
}

// out[0..3] (+)= v, of which the first `n` exist
template <class O>
__device__ __forceinline__ void put4(O* out, v4f v, uint32_t n, int accumulate) {
  float f[4] = {};
  if (accumulate) load_some<O, 4>(out, n, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = accumulate ? f[i] + v[i] : v[i];
  store_some<O, 4>(out, n, f);
}

// A wave's MW x NW results as 16-bit elements, stored in whole 16-byte pieces by way of its own part of LDS: the matrix
// instruction leaves a lane four consecutive m of one n, and stores of those are segments of 32 bytes.  quad(i, j): the
// four at m = 16 i + 4 (lane / 16), n = 16 j + lane % 16; row(n, m, piece): eight consecutive m of an n.  (The pieces of a
// row of LDS are permuted by its number, for the banks.)
template <class T, int MW, int NW, class Q, class R>
__device__ __forceinline__ void put_tile(T* stage, Q&& quad, R&& row) {
  constexpr int CH = MW / 8;
  const uint32_t lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
  for (int j = 0; j < NW / 16; ++j)
#pragma unroll
    for (int i = 0; i < MW / 16; ++i) {
      const uint32_t n = 16 * j + (lane & 15), c = (2 * i + (g >> 1)) ^ (n & (CH - 1));
      *reinterpret_cast<vec_t<T, 4>*>(stage + (n * CH + c) * 8 + (g & 1) * 4) = quad(i, j);
    }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 4
  for (int q = 0; q < NW * CH / 64; ++q) {
    const uint32_t n = (q * 64 + lane) / CH, c = lane % CH;
    row(n, c * 8, *reinterpret_cast<const vec_t<T, 8>*>(stage + (n * CH + (c ^ (n & (CH - 1)))) * 8));
  }
}

// Eight elements of which the first n exist, in rows `stride` apart; they are not read here again.  Whole pieces go out
// non-temporally (128 x 131072 x 1024: 266 us backward, 295 else; 2048 x 32000 x 1024: 427, 430); where rows end inside
// one, by the L2, which joins the two rows that share a line (1 x 49855 x 667: 90 us, 101 non-temporally).
template <class T>
__device__ __forceinline__ void stream8(T* p, uint32_t n, uint64_t stride, const vec_t<T, 8>& v) {
  if (n >= 8 && stride % 8 == 0) {
    __builtin_nontemporal_store(v, reinterpret_cast<any_vec<T, 8>*>(p));
  } else if (n >= 8) {
    *reinterpret_cast<any_vec<T, 8>*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (static_cast<uint32_t>(i) < n) p[i] = v[i];
  }
}

// tile number `id` of a product, by the whole workgroup; lds: R (BM + BN) 64 elements
template <class T, int EPI, int BM, int BN, int WM, int WN, int R>
__device__ __forceinline__ void gemm_tile(const GemmArgs<T>& a, uint32_t id, T* lds) {
  constexpr int NT = 64 * WM * WN, MF = BM / WM / 16, NF = BN / WN / 16;
  constexpr bool AC = EPI == kHidden || EPI == kWeight, BC = EPI == kWeight;
  static_assert((R & (R - 1)) == 0, "step t's buffers are those at t mod R");
  auto la = [&](uint32_t t) { return lds + (t & (R - 1)) * (BM * kBK); };
  auto lb = [&](uint32_t t) { return lds + R * BM * kBK + (t & (R - 1)) * (BN * kBK); };
  static_assert(BM * BN <= R * (BM + BN) * kBK, "the results pass through LDS as 16-bit elements");
  // Workgroup ids go round the 8 XCDs: give each XCD a contiguous stretch of tiles, and walk the stretch in groups of 8
  // tile rows, so the tiles that run together on an XCD share operands in its L2.
  const uint32_t all = a.mt * a.nt * a.splits, per = all / 8, rem = all % 8, xcd = id % 8;
  id = xcd * per + min(xcd, rem) + id / 8;
  const uint32_t split = id / (a.mt * a.nt);
  id -= split * (a.mt * a.nt);
  const uint32_t group = id / (8 * a.nt), gm = min(8u, a.mt - group * 8), in = id - group * 8 * a.nt;
  const uint32_t m0 = (group * 8 + in % gm) * BM, n0 = in / gm * BN;
  const uint64_t kbegin = static_cast<uint64_t>(split) * a.ksplit;
  const uint32_t left = min(a.ksplit, static_cast<uint32_t>(a.k - kbegin));

  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t wm = wave % WM, wn = wave / WM;
  Tile<T, BM, NT, AC> ta;
  Tile<T, BN, NT, BC> tb;
  ta.init(a.a, m0, kbegin);
  tb.init(a.b, n0, kbegin);
  Frags<T, BM, MF, AC> fa;
  Frags<T, BN, NF, BC> fb;
  fa.init(wm * (BM / WM));
  fb.init(wn * (BN / WN));
  v4f acc[MF][NF] = {};

  // A step's 64 k are two halves.  The fragments of a half are read while the half before is multiplied: x[0], y[0] hold
  // the first half of a step, x[1], y[1] the second.  Between them lies the step's one barrier: in front of it every wave
  // has read its last from the step's buffer, into which the tile R steps on may then be loaded, and has waited for its
  // own pieces of the next tile.  Reads and loads are issued a few at a time between the matrix instructions: eight
  // loads behind each other, from eight waves at once, held every wave's products for about 1000 of a step's 3600 clocks.
  frag<T> x[2][MF], y[2][NF];
  constexpr int kLoads = Tile<T, BM, NT, AC>::kPieces + Tile<T, BN, NT, BC>::kPieces;
  static_assert(kLoads <= 2 * MF, "two loads a group at most");
  const uint32_t steps = (left + kBK - 1) / kBK, full = left / kBK;
  auto meet = [&]() {  // (the scheduler would move the products behind it)
    __builtin_amdgcn_sched_barrier(0);
    // (the tiles behind the next one, R - 2 of them, may still be on their way)
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"((R - 2) * kLoads) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // A whole tile at once.  Past the last step (R > 2) these are loads of zeros that nothing reads, so that the wait above
  // always has as many behind the one it is for.
  auto fetch = [&](uint32_t t) {
    const uint32_t toa = ta.place(la(t)), tob = tb.place(lb(t));
    if (t < full) {
#pragma unroll
      for (int i = 0; i < Tile<T, BM, NT, AC>::kPieces; ++i) ta.load(i, toa);
#pragma unroll
      for (int i = 0; i < Tile<T, BN, NT, BC>::kPieces; ++i) tb.load(i, tob);
    } else {
      const uint32_t n = t < steps ? left - t * kBK : 0;
      ta.load_end(toa, n);
      tb.load_end(tob, n);
    }
    ta.advance();
    tb.advance();
  };
  // The products of one half, with the reads of the other from step t's buffer; with `loads` also the loads of step
  // t + R - 1's tile.  (The reads end two groups early: the barrier behind waits for them.)
  auto half = [&](int h, uint32_t t, bool loads) {
    const T *ca = la(t), *cb = lb(t);
    const uint32_t toa = ta.place(la(t + R - 1)), tob = tb.place(lb(t + R - 1));
    constexpr int kReads = MF + NF, kOver = MF > 2 ? MF - 2 : 1;
    fa.touch();
    fb.touch();
#pragma unroll
    for (int i = 0; i < MF; ++i) {
#pragma unroll
      for (int j = 0; j < NF; ++j) acc[i][j] = mma(x[h][i], y[h][j], acc[i][j]);
      if (loads) {
#pragma unroll
        for (int l = i * kLoads / MF; l < (i + 1) * kLoads / MF; ++l) {
          if (l < Tile<T, BM, NT, AC>::kPieces)
            ta.load(l, toa);
          else
            tb.load(l - Tile<T, BM, NT, AC>::kPieces, tob);
        }
      }
#pragma unroll
      for (int r = i * kReads / kOver; r < (i + 1) * kReads / kOver && r < kReads; ++r) {
        if (r < NF)
          y[h ^ 1][r] = fb.get(cb, h ^ 1, r);
        else
          x[h ^ 1][r - NF] = fa.get(ca, h ^ 1, r - NF);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (loads) {
      ta.advance();
      tb.advance();
    }
  };
  if constexpr (R == 2) {
    fetch(0);
    meet();
    if (steps > 1) fetch(1);
  } else {
#pragma unroll
    for (uint32_t t = 0; t < R; ++t) fetch(t);
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"((R - 1) * kLoads) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
  uint32_t t = 0;
  if (full > R) {
#pragma unroll
    for (int j = 0; j < NF; ++j) y[0][j] = fb.get(lb(0), 0, j);
#pragma unroll
    for (int i = 0; i < MF; ++i) x[0][i] = fa.get(la(0), 0, i);
    do {
      half(0, t, false);
      meet();
      half(1, t + 1, true);
    } while (++t + R < full);
  }
  // the last steps, whose tiles may be cut short: read and multiply in turn
  for (; t < steps; ++t) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      fa.touch();
      fb.touch();
#pragma unroll
      for (int j = 0; j < NF; ++j) y[0][j] = fb.get(lb(t), h, j);
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        x[0][i] = fa.get(la(t), h, i);
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] = mma(x[0][i], y[0][j], acc[i][j]);
      }
    }
    meet();
    if (R > 2 || t + R < steps) fetch(t + R);
  }
  if constexpr (R > 2) {  // LDS is free when the zeros have come, too
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }

  // acc[i][j][r] = C[m + 16 i + r, n + 16 j]
  constexpr int MW = BM / WM, NW = BN / WN;
  const uint32_t mw = m0 + wm * MW, nw = n0 + wn * NW;
  const uint32_t m = mw + 4 * (lane >> 4), n = nw + (lane & 15);
  T* const stage = lds + wave * (MW * NW);
  if constexpr (EPI == kStats) {
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      const uint32_t tok = n + 16 * j;
      const int target = tok < a.tokens ? target_of(a, tok) : -1;
      const int at = target - static_cast<int>(m);  // the target's place among this lane's rows
      if (m0 + BM > a.vocab) {  // rows past the vocabulary do not count
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (m + 16 * i + r >= a.vocab) acc[i][j][r] = -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[i][j][r]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float from = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += __expf(acc[i][j][r] - from);
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      const bool here = target >= 0 && at >= 0 && at < 16 * MF && (at & 15) < 4;
      if (__ballot(here)) {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (at == 16 * i + r) z = acc[i][j][r];
        if (here) a.ztarget[tok] = z;
      }
      if (tok < a.tokens && lane < 16) {
        float* s = a.stats + (static_cast<uint64_t>(tok) * a.pieces + mw / MW) * 2;
        *reinterpret_cast<float2*>(s) = make_float2(top, sum);
      }
    }
  } else if constexpr (EPI == kGrad) {
    const bool tail = a.v0 + m0 + BM > a.vocab;
    int at[NF];
    float shift[NF];
    bool keep[NF], here[NF], any[NF];
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      const uint32_t tok = n + 16 * j;
      const int target = tok < a.tokens ? target_of(a, tok) : -1;
      keep[j] = target >= 0;
      at[j] = target - static_cast<int>(a.v0 + m);
      // 2^12 exp(z - lse) as one power of two: 2^(z log2 e + shift); the argument's rounding, 2^-24 of some tens, is far
      // below the result's
      shift[j] = keep[j] ? 12.0f - a.lse[tok] * kLog2E : 0.0f;
      here[j] = keep[j] && at[j] >= 0 && at[j] < 16 * MF && (at[j] & 15) < 4;
      any[j] = __ballot(here[j]) != 0;
    }
    put_tile<T, MW, NW>(
        stage,
        [&](int i, int j) {
          float p[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], kLog2E, shift[j]));
          if (any[j]) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (at[j] == 16 * i + r) p[r] -= kGScale;
          }
          if (tail) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (a.v0 + m + 16 * i + r >= a.vocab) p[r] = 0.0f;
          }
          vec_t<T, 4> o;
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = static_cast<T>(p[r]);
          if (any[j] && here[j]) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (at[j] == 16 * i + r) a.lost[n + 16 * j] = p[r] - static_cast<float>(o[r]);
          }
          return keep[j] ? o : vec_t<T, 4>{};  // (zeros without a target, whatever its hidden state holds)
        },
        [&](uint32_t row, uint32_t c, const vec_t<T, 8>& v) {
          if (nw + row < a.tokens)
            *reinterpret_cast<vec_t<T, 8>*>(a.g + static_cast<uint64_t>(nw + row) * a.ldg + mw + c) = v;
        });
  } else if constexpr (EPI == kHidden) {
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      const uint32_t tok = n + 16 * j;
      const bool real = tok < a.tokens;
      const float scale = real && a.last ? factor_of(a, tok) * (1.0f / kGScale) : 0.0f;
      const int target = real && a.last ? target_of(a, tok) : -1;
      const float lost = target >= 0 ? a.lost[tok] : 0.0f;
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        const uint32_t c = m + 16 * i;
        if (!real || c >= a.dim) continue;
        float* sum = a.acc + (static_cast<uint64_t>(split) * a.tokens + tok) * a.dim + c;
        const uint32_t have = a.dim - c;
        if (!a.first) {
          float f[4];
          load_some<float, 4>(sum, have, f);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] += f[r];
        }
        if (!a.last) {
          put4<float>(sum, acc[i][j], have, 0);
          continue;
        }
        if (target >= 0) {
          float f[4];
          load_f32<T, 4>(a.w.p + target * a.w.ld + c, f);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] += lost * f[r];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = scale == 0.0f ? 0.0f : acc[i][j][r] * scale;
      }
    }
    if (a.last)
      put_tile<T, MW, NW>(
          stage,
          [&](int i, int j) {
            vec_t<T, 4> o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = static_cast<T>(acc[i][j][r]);
            return o;
          },
          [&](uint32_t row, uint32_t c, const vec_t<T, 8>& v) {
            if (nw + row < a.tokens && mw + c < a.dim)
              stream8<T>(static_cast<T*>(a.out) + static_cast<uint64_t>(nw + row) * a.ostride + mw + c, a.dim - mw - c,
                         a.ostride, v);
          });
  } else {
    const float most = a.amax[0], unscale = 1.0f / (kGScale * a.amax[1]);  // (a power of two: exact, and first)
    const bool direct = a.out_f32 || a.accumulate;  // (a sum with what is there is rounded once, behind the addition)
    // What rounding took from the targets' entries: a product with the tokens whose target is one of the tile's rows, which
    // lie together in perm, 64 of them at a time.  A token's entry is in one row; its place and value wait in LDS.
    T* const lv = lds + R * BM * kBK;
    uint16_t* const lr = reinterpret_cast<uint16_t*>(lv + kBK);
    const uint32_t s1 = a.start[min(a.v0 + n0 + BN, a.vocab)];
    for (uint32_t s = a.start[min(a.v0 + n0, a.vocab)]; s < s1; s += kBK) {
      ta.load_rows(a.a, m0, a.perm + s, s1 - s, ta.place(lds));
      if (threadIdx.x < kBK) {
        const bool real = s + threadIdx.x < s1;
        const uint32_t tok = real ? a.perm[s + threadIdx.x] : 0;
        lv[threadIdx.x] = real ? static_cast<T>(a.lost[tok]) : static_cast<T>(0.0f);
        lr[threadIdx.x] = real ? static_cast<uint16_t>(target_of(a, tok) - static_cast<int>(a.v0 + n0)) : 0;
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      const uint32_t g = lane >> 4;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        fa.touch();
        const frag<T> value = *reinterpret_cast<const frag<T>*>(lv + 32 * h + 8 * g);
        const vec_t<uint16_t, 8> place = *reinterpret_cast<const vec_t<uint16_t, 8>*>(lr + 32 * h + 8 * g);
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            y[0][j][e] = place[e] == wn * NW + 16 * j + (lane & 15) ? value[e] : static_cast<T>(0.0f);
#pragma unroll
        for (int i = 0; i < MF; ++i) {
          x[0][i] = fa.get(lds, h, i);
#pragma unroll
          for (int j = 0; j < NF; ++j) acc[i][j] = mma(x[0][i], y[0][j], acc[i][j]);
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; direct && j < NF; ++j) {
      const uint32_t row = n + 16 * j;
      if (a.v0 + row >= a.vocab) continue;
      const uint64_t o = static_cast<uint64_t>(a.v0 + row) * a.ostride;
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        const uint32_t c = m + 16 * i;
        if (c >= a.dim) continue;
        const v4f v = acc[i][j] * unscale * most;
        if (a.out_f32)
          put4<float>(static_cast<float*>(a.out) + o + c, v, a.dim - c, a.accumulate);
        else
          put4<T>(static_cast<T*>(a.out) + o + c, v, a.dim - c, a.accumulate);
      }
    }
    if (!direct)
      put_tile<T, MW, NW>(
          stage,
          [&](int i, int j) {
            vec_t<T, 4> o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = static_cast<T>(acc[i][j][r] * unscale * most);
            return o;
          },
          [&](uint32_t row, uint32_t c, const vec_t<T, 8>& v) {
            if (a.v0 + nw + row < a.vocab && mw + c < a.dim)
              stream8<T>(static_cast<T*>(a.out) + static_cast<uint64_t>(a.v0 + nw + row) * a.ostride + mw + c,
                         a.dim - mw - c, a.ostride, v);
          });
  }
}

template <class T, int EPI, int BM, int BN, int WM, int WN, int R>
__global__ __launch_bounds__(64 * WM * WN) void k_gemm(GemmArgs<T> a) {
  __shared__ __attribute__((aligned(1024))) T lds[R * (BM + BN) * kBK];
  gemm_tile<T, EPI, BM, BN, WM, WN, R>(a, blockIdx.x, lds);
}

// Both products of a piece's G side by side: blocks [0, xtiles) are grad_hidden's.
template <class T, int BM, int BN, int WM, int WN, int R>
__global__ __launch_bounds__(64 * WM * WN) void k_both(GemmArgs<T> x, GemmArgs<T> y, uint32_t xtiles) {
  __shared__ __attribute__((aligned(1024))) T lds[R * (BM + BN) * kBK];
  if (blockIdx.x < xtiles)
    gemm_tile<T, kHidden, BM, BN, WM, WN, R>(x, blockIdx.x, lds);
  else
    gemm_tile<T, kWeight, BM, BN, WM, WN, R>(y, blockIdx.x - xtiles, lds);
}

// ---------------------------------------------------------------- what the products need

// The largest |grad_loss| of the tokens with a target, in every thread of a workgroup of WAVES waves.  (A NaN counts as the
// largest: the gradient shall have it.)
template <class T, int WAVES>
__device__ __forceinline__ float largest(const GemmArgs<T>& a, float* lds) {
  float m = 0.0f;
  auto more = [&](float g) { m = m != m || g <= m ? m : g; };
  for (uint64_t n0 = threadIdx.x; n0 < a.tokens; n0 += 4 * 64 * WAVES) {  // four tokens in flight
    float g[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t n = n0 + i * 64 * WAVES;
      g[i] = n < a.tokens ? fabsf(factor_of(a, static_cast<uint32_t>(n))) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) more(g[i]);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) more(__shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
  __syncthreads();
  m = lds[0];
  for (int w = 1; w < WAVES; ++w) more(lds[w]);
  return m;
}

// What of the hidden states' copy has to fit fp16, by a workgroup: the largest |grad_loss| of some tokens with a target, and
// the least e with |grad_loss[n] hidden[n, c]| < 2^e for all of them (from the factors' exponents: the product may pass
// fp32's range).  A launch of its own, 3 us at 333 x 520, 12 at 8192 x 2048 (27 by 256 workgroups), where fp16 takes a
// factor for each token.  One factor for all needs none: every share is 1.
struct Reach {
  float most;
  int e;
};
constexpr int kNoReach = -1000;
constexpr uint32_t kReachBlocks = 1024;

template <class T>
__global__ __launch_bounds__(256) void k_reach(GemmArgs<T> a, const T* hidden, uint64_t stride, uint32_t lpr_log, Reach* out) {
  __shared__ Reach part[4];
  Reach r{0.0f, kNoReach};
  const uint64_t step = gridDim.x * (256u >> lpr_log);
  for (uint64_t row = (static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x) >> lpr_log; row < a.tokens; row += step) {
    const float g = fabsf(factor_of(a, static_cast<uint32_t>(row)));
    if (g == 0.0f) continue;
    r.most = r.most != r.most || g <= r.most ? r.most : g;
    float top = 0.0f;
    for (uint32_t c = (threadIdx.x & ((1u << lpr_log) - 1)) * 8; c < a.dim; c += 8u << lpr_log) {
      float v[8];
      load_some<T, 8>(hidden + row * stride + c, a.dim - c, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(v[k]));
    }
    const float m = __builtin_amdgcn_frexp_mantf(g) * __builtin_amdgcn_frexp_mantf(top);
    if (top != 0.0f)
      r.e = max(r.e, __builtin_amdgcn_frexp_expf(g) + __builtin_amdgcn_frexp_expf(top) + __builtin_amdgcn_frexp_expf(m));
  }
  auto more = [&](float most, int e) {
    r.most = r.most != r.most || most <= r.most ? r.most : most;
    r.e = max(r.e, e);
  };
#pragma unroll
  for (int d = 32; d; d >>= 1) more(__shfl_xor(r.most, d), __shfl_xor(r.e, d));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = r;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 4; ++w) more(part[w].most, part[w].e);
  out[blockIdx.x] = r;
}

// The parts of all of k_reach's workgroups together, in every lane of a wave: the largest |grad_loss|, and the power of two
// that the shares are scaled by: |grad_loss[n] / most hidden[n, c]| < 2^(e - exponent of most + 1), which goes to 2^15.
// (Not below 1: a share is no larger than the hidden state itself.)
__device__ __forceinline__ float2 reach_of(const Reach* parts, uint32_t n) {
  Reach r{0.0f, kNoReach};
  auto more = [&](float most, int e) {
    r.most = r.most != r.most || most <= r.most ? r.most : most;
    r.e = max(r.e, e);
  };
#pragma unroll 4
  for (uint32_t i = threadIdx.x & 63; i < n; i += 64) more(parts[i].most, parts[i].e);
#pragma unroll
  for (int d = 32; d; d >>= 1) more(__shfl_xor(r.most, d), __shfl_xor(r.e, d));
  const int up = r.e == kNoReach ? 0 : 14 - r.e + __builtin_amdgcn_frexp_expf(r.most);
  return make_float2(r.most, __builtin_ldexpf(1.0f, min(max(up, 0), 40)));
}

// What grad_weight's product needs besides G, by workgroups of WAVES waves: blocks [0, sorters) sort the tokens by target;
// the others copy the hidden states into whole 16-byte pieces, zeros behind dim, each row times its share of the largest
// grad_loss, and zeros for tokens without a target, whatever they hold.  Up to kFindHere tokens each of these finds the
// largest itself: a launch less, 3 to 4 us of a backward pass up to 2048 tokens, nothing at 6000 to 8192, and 12 us lost
// at 16384, where every block would read that many.
constexpr uint32_t kFindHere = 4096;

template <class T>
struct PrepareArgs {
  uint32_t blocks, sorters, range;
  uint32_t *start, *perm;
  const T* src;  // hidden
  uint64_t stride;
  uint32_t pdim, lpr_log;  // 2^lpr_log lanes a row
  float* amax;
  const Reach* parts;      // fp16 with a factor for each token, else null: every token's scale is 1
  uint32_t nparts;
  T* dst;
};

template <class T, class I, int WAVES>
__device__ __forceinline__ void prepare(const GemmArgs<T>& a, const PrepareArgs<T>& p, uint32_t block,
                                        SortSpace<WAVES>& space) {
  if (block < p.sorters) {
    sort_by_row<I, WAVES>(space, block, static_cast<const I*>(a.targets), a.tokens, a.vocab, p.range, p.start, p.perm,
                          nullptr);
    return;
  }
  block -= p.sorters;
  float most, scale = 1.0f;
  if (p.parts != nullptr) {
    const float2 r = reach_of(p.parts, p.nparts);
    most = r.x;
    scale = r.y;
  } else if (a.tokens <= kFindHere) {
    most = largest<T, WAVES>(a, reinterpret_cast<float*>(space.wsum));
  } else {
    most = *p.amax;
  }
  if (block == 0 && threadIdx.x == 0) {
    if (p.parts != nullptr || a.tokens <= kFindHere) p.amax[0] = most;  // (else it is there)
    p.amax[1] = scale;
  }
  const uint64_t row = (static_cast<uint64_t>(block) * 64 * WAVES + threadIdx.x) >> p.lpr_log;
  if (row >= a.tokens) return;
  const float g = factor_of(a, static_cast<uint32_t>(row)), by = g == 0.0f ? 0.0f : g / most * scale;
  for (uint32_t c = (threadIdx.x & ((1u << p.lpr_log) - 1)) * 8; c < p.pdim; c += 8u << p.lpr_log) {
    float v[8] = {};
    if (by != 0.0f) {
      load_some<T, 8>(p.src + row * p.stride + c, a.dim - c, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= by;
    }
    store_f32<T, 8>(p.dst + row * p.pdim + c, v);
  }
}

template <class T, class I>
__global__ __launch_bounds__(1024) void k_prepare(GemmArgs<T> a, PrepareArgs<T> p) {
  __shared__ SortSpace<16> space;
  prepare<T, I, 16>(a, p, blockIdx.x, space);
}

// The same beside the first piece's G, where that has few tiles: blocks [0, p.blocks) prepare.
template <class T, class I, int BM, int BN, int WM, int WN, int R>
__global__ __launch_bounds__(64 * WM * WN) void k_grad_prepare(GemmArgs<T> a, PrepareArgs<T> p) {
  __shared__ __attribute__((aligned(1024))) T lds[R * (BM + BN) * kBK];
  static_assert(sizeof(SortSpace<WM * WN>) <= sizeof(lds), "they share LDS");
  if (blockIdx.x < p.blocks)
    prepare<T, I, WM * WN>(a, p, blockIdx.x, *reinterpret_cast<SortSpace<WM * WN>*>(lds));
  else
    gemm_tile<T, kGrad, BM, BN, WM, WN, R>(a, blockIdx.x - p.blocks, lds);
}

// ---------------------------------------------------------------- few tokens
//
// The forward of up to 32 tokens is bound by reading the weight.  The tiles above keep one step of it in flight a CU
// (16 KiB, 17 us for 16 tokens x 32000 x 1024 bf16); here each wave streams 16 rows of the vocabulary through a ring of
// its own in LDS, kRing steps of 64 columns (2 KiB) deep, and waits for nobody: 80 KiB in flight a CU, 14.5 us.  The hidden
// states lie in LDS, 1024 / NF columns of them at a time.  (Rows loaded straight into the matrix instructions' registers
// come in halves of a cache line: 19 us.)
constexpr uint32_t kFewTokens = 32;
constexpr int kRing = 5;

template <class T, int NF>
__global__ __launch_bounds__(256) void k_few(GemmArgs<T> a) {
  constexpr uint32_t KC = 1024 / NF, kSteps = KC / kBK;  // columns of the hidden states in LDS; steps of them
  __shared__ __attribute__((aligned(1024))) T ring[4][kRing][16 * kBK];
  __shared__ __attribute__((aligned(1024))) T hid[kSteps][16 * NF * kBK];
  __shared__ float2 part[4][16 * NF];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4,
                 r16 = lane & 15;
  const uint32_t row0 = blockIdx.x * 64 + wave * 16;
  // a load instruction's lane: row lane / 8 of eight, piece lane % 8 of its step's line, permuted as in Tile
  const uint32_t lr = lane >> 3, lc = (lane & 7) ^ lr;
  const char* w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = reinterpret_cast<const char*>(a.a.p + min(row0 + 8 * i + lr, a.vocab - 1) * a.a.ld + lc * 8);
  auto load = [&](const char* src, const T* lds) {
    const uint32_t to = __builtin_amdgcn_readfirstlane(
        static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) T*)(lds))));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(src) : "memory");
  };
  const uint32_t steps = (a.k + kBK - 1) / kBK;
  auto fetch = [&](uint32_t t) {  // step t into its place in the ring; past the end zeros, which nothing multiplies
#pragma unroll
    for (int i = 0; i < 2; ++i)
      load(t * kBK + lc * 8 < a.k ? w[i] + static_cast<uint64_t>(t) * kBK * sizeof(T)
                                  : reinterpret_cast<const char*>(g_zero),
           ring[wave][t % kRing] + 8 * i * kBK);
  };
  v4f acc[NF] = {};
  for (uint32_t t = 0; t < kRing; ++t) fetch(t);
  for (uint32_t t0 = 0; t0 < steps; t0 += kSteps) {
    __syncthreads();  // (every wave is done with the columns before)
    for (uint32_t q = wave; q < kSteps * 2 * NF; q += 4) {  // eight rows of a step each
      const uint32_t t = t0 + q / (2 * NF), row = q % (2 * NF) * 8 + lr, k = t * kBK + lc * 8;
      if (t >= steps) break;
      load(k < a.k ? reinterpret_cast<const char*>(a.b.p + min(row, a.tokens - 1) * a.b.ld + k)
                   : reinterpret_cast<const char*>(g_zero),
           hid[q / (2 * NF)] + q % (2 * NF) * 8 * kBK);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (uint32_t t = t0; t < min(t0 + kSteps, steps); ++t) {
      // two loads a step, kRing steps: this one's are there when those of the kRing - 1 behind it are all that is out
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"(2 * (kRing - 1)) : "memory");
      const T* x = ring[wave][t % kRing];
      const T* y = hid[t - t0];
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const uint32_t at = (r16 * 8 + ((sub * 4 + g) ^ (r16 & 7))) * 8;
        const frag<T> f = *reinterpret_cast<const frag<T>*>(x + at);
#pragma unroll
        for (int j = 0; j < NF; ++j)
          acc[j] = mma(f, *reinterpret_cast<const frag<T>*>(y + j * 16 * kBK + at), acc[j]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the step is read: its place may be loaded into
      fetch(t + kRing);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    const uint32_t tok = 16 * j + r16;
    const int target = tok < a.tokens ? target_of(a, tok) : -1;
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t v = row0 + 4 * g + r;
      if (v >= a.vocab) acc[j][r] = -INFINITY;
      if (target >= 0 && static_cast<uint32_t>(target) == v) a.ztarget[tok] = acc[j][r];
      top = fmaxf(top, acc[j][r]);
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float from = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) sum += __expf(acc[j][r] - from);
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (g == 0) part[wave][tok] = make_float2(top, sum);
  }
  __syncthreads();
  if (threadIdx.x >= 16 * NF || threadIdx.x >= a.tokens) return;
  float2 all = part[0][threadIdx.x];
#pragma unroll
  for (int v = 1; v < 4; ++v) all = join(all, part[v][threadIdx.x]);
  reinterpret_cast<float2*>(a.stats)[static_cast<uint64_t>(threadIdx.x) * a.pieces + blockIdx.x] = all;
}

// ---------------------------------------------------------------- the small kernels around it

// Joins the pieces' maxima and sums: WAVES waves a token, four pieces a lane in flight.
template <class T, int WAVES>
__global__ __launch_bounds__(256) void k_merge(GemmArgs<T> a, float* loss, float* lse) {
  __shared__ float2 part[4];
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t tok = blockIdx.x * (4 / WAVES) + wave / WAVES;
  float2 all = make_float2(-INFINITY, 0.0f);
  if (tok < a.tokens) {
    const float2* s = reinterpret_cast<const float2*>(a.stats) + static_cast<uint64_t>(tok) * a.pieces;
    for (uint32_t p = (wave % WAVES) * 64 + lane; p < a.pieces; p += 4 * 64 * WAVES) {
      float2 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = p + i * 64 * WAVES < a.pieces ? s[p + i * 64 * WAVES] : make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int i = 0; i < 4; ++i) all = join(all, v[i]);
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) all = join(all, make_float2(__shfl_xor(all.x, d), __shfl_xor(all.y, d)));
  if constexpr (WAVES > 1) {
    if (lane == 0) part[wave] = all;
    __syncthreads();
    if (wave % WAVES != 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) all = join(all, part[wave + w]);
  }
  if (lane != 0 || tok >= a.tokens) return;
  const float l = all.x + logf(all.y);
  lse[tok] = l;
  loss[tok] = target_of(a, tok) >= 0 ? l - a.ztarget[tok] : 0.0f;
}

template <class T>
__global__ __launch_bounds__(1024) void k_largest(GemmArgs<T> a, float* amax) {
  __shared__ float lds[16];
  const float m = largest<T, 16>(a, lds);
  if (threadIdx.x == 0) *amax = m;
}

// Rows copied into whole 16-byte pieces [rows][pdim], zeros behind dim; 2^lpr_log lanes a row.  Two matrices, either of
// which may have no rows: a launch less (4 us).
template <class T>
struct PackArgs {
  const T* src;
  uint64_t stride, rows;
  T* dst;
};

template <class T>
__global__ __launch_bounds__(256) void k_pack(PackArgs<T> x, PackArgs<T> y, uint32_t dim, uint32_t pdim,
                                              uint32_t lpr_log) {
  uint64_t row = (static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x) >> lpr_log;
  if (row >= x.rows + y.rows) return;
  const bool first = row < x.rows;
  if (!first) row -= x.rows;
  const T* src = (first ? x.src : y.src) + row * (first ? x.stride : y.stride);
  T* dst = (first ? x.dst : y.dst) + row * pdim;
  for (uint32_t c = (threadIdx.x & ((1u << lpr_log) - 1)) * 8; c < pdim; c += 8u << lpr_log) {
    float v[8];
    load_some<T, 8>(src + c, dim - c, v);
    store_f32<T, 8>(dst + c, v);
  }
}

// grad_hidden = factor * (the parts' sums, in order)
template <class T>
__global__ __launch_bounds__(256) void k_join(GemmArgs<T> a) {
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x, all = static_cast<uint64_t>(a.tokens) * a.dim;
  if (i >= all) return;
  const uint32_t tok = static_cast<uint32_t>(i / a.dim), c = static_cast<uint32_t>(i - static_cast<uint64_t>(tok) * a.dim);
  float v = 0.0f;
  for (uint32_t s = 0; s < a.splits; ++s) v += a.acc[s * all + i];
  const int target = target_of(a, tok);
  if (target >= 0) v += a.lost[tok] * static_cast<float>(a.w.p[target * a.w.ld + c]);
  const float scale = factor_of(a, tok) * (1.0f / kGScale);
  static_cast<T*>(a.out)[tok * a.ostride + c] = static_cast<T>(scale == 0.0f ? 0.0f : v * scale);
}

template <class O>
__global__ __launch_bounds__(256) void k_zero(O* out, uint64_t rows, uint32_t dim, uint64_t stride) {
  for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; i < rows * dim;
       i += static_cast<uint64_t>(gridDim.x) * 256) {
    const uint64_t row = i / dim;
    out[row * stride + (i - row * dim)] = static_cast<O>(0.0f);
  }
}

// ---------------------------------------------------------------- launches

uint64_t up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// Tile shapes: big ones do more work for each byte that goes through LDS, small ones fill the CUs with less.  Big from one
// tile a CU on (8192 x 32768 x 2048: 871 us, small ones 1192); small ones two a CU while there are enough, else one with a
// deeper ring; tiny ones where even those leave half the CUs idle (33 tokens x 5003 x 520: forward 10.7 us, small ones
// 14.1).
constexpr uint32_t kBig = 256, kSmall = 128, kTiny = 64;
enum { kTileBig, kTileSmall, kTileSmallDeep, kTileTiny };
int tile_of(uint64_t m, uint64_t n, uint64_t splits) {
  auto tiles = [&](uint32_t t) { return ceil_div(m, t) * ceil_div(n, t) * splits; };
  return tiles(kBig) >= 256 ? kTileBig : tiles(kSmall) > 256 ? kTileSmall : tiles(kSmall) > 128 ? kTileSmallDeep : kTileTiny;
}
uint32_t tile_rows(int tile) { return tile == kTileBig ? kBig : tile == kTileTiny ? kTiny : kSmall; }

// A launch holds fewer than 2^32 threads.  The calls look at all of theirs before the first.
constexpr uint64_t kMaxTiles = 1u << 22, kMaxBlocks = (1u << 24) - 1;
bool tiles_fit(uint64_t m, uint64_t n, uint64_t splits) {
  const uint32_t t = tile_rows(tile_of(m, n, splits));
  return ceil_div(m, t) * ceil_div(n, t) * splits < kMaxTiles;
}

template <class T, int EPI>
int launch(GemmArgs<T>& a, uint32_t m, uint32_t n, int tile, hipStream_t stream) {
  const uint32_t t = tile_rows(tile);
  a.mt = static_cast<uint32_t>(ceil_div(m, t));
  a.nt = static_cast<uint32_t>(ceil_div(n, t));
  const unsigned g = a.mt * a.nt * a.splits;
  switch (tile) {
    case kTileBig: k_gemm<T, EPI, 256, 256, 2, 4, 2><<<g, 512, 0, stream>>>(a); break;
    case kTileSmall: k_gemm<T, EPI, 128, 128, 2, 2, 2><<<g, 256, 0, stream>>>(a); break;
    case kTileSmallDeep: k_gemm<T, EPI, 128, 128, 2, 2, 4><<<g, 256, 0, stream>>>(a); break;
    default: k_gemm<T, EPI, 64, 64, 2, 2, 4><<<g, 256, 0, stream>>>(a); break;
  }
  return elaunch("omr_vocab_loss");
}

// G's product (of fewer than kTileBig's tiles) and, in front of it, what grad_weight's needs
template <class T, class I>
int launch_grad_prepare(GemmArgs<T>& a, const PrepareArgs<T>& p, uint32_t cols, int tile, hipStream_t stream) {
  const uint32_t t = tile_rows(tile);
  a.mt = static_cast<uint32_t>(ceil_div(cols, t));
  a.nt = static_cast<uint32_t>(ceil_div(a.tokens, t));
  const uint32_t g = p.blocks + a.mt * a.nt;
  if (tile == kTileSmall)
    k_grad_prepare<T, I, 128, 128, 2, 2, 2><<<g, 256, 0, stream>>>(a, p);
  else if (tile == kTileSmallDeep)
    k_grad_prepare<T, I, 128, 128, 2, 2, 4><<<g, 256, 0, stream>>>(a, p);
  else
    k_grad_prepare<T, I, 64, 64, 2, 2, 4><<<g, 256, 0, stream>>>(a, p);
  return elaunch("omr_vocab_loss_grad");
}

// x (grad_hidden) and y (grad_weight) in one launch, by the rule above for their tiles together
template <class T>
int launch_both(GemmArgs<T>& x, GemmArgs<T>& y, uint32_t dim, uint32_t cols, hipStream_t stream) {
  auto tiles = [&](GemmArgs<T>& a, uint32_t n, uint32_t t) {
    a.mt = static_cast<uint32_t>(ceil_div(dim, t));
    a.nt = static_cast<uint32_t>(ceil_div(n, t));
    return a.mt * a.nt * a.splits;
  };
  const uint32_t small = tiles(x, x.tokens, kSmall) + tiles(y, cols, kSmall), t = small > 128 ? kSmall : kTiny;
  const uint32_t xtiles = tiles(x, x.tokens, t), g = xtiles + tiles(y, cols, t);
  if (small > 256)
    k_both<T, 128, 128, 2, 2, 2><<<g, 256, 0, stream>>>(x, y, xtiles);
  else if (small > 128)
    k_both<T, 128, 128, 2, 2, 4><<<g, 256, 0, stream>>>(x, y, xtiles);
  else
    k_both<T, 64, 64, 2, 2, 4><<<g, 256, 0, stream>>>(x, y, xtiles);
  return elaunch("omr_vocab_loss_grad");
}

// The piece of the vocabulary whose G is held at a time: about 256 MiB of it (what the last-level cache holds), at least
// 1024 rows, in equal pieces of whole tiles.
constexpr uint64_t kPieceBytes = 256ull << 20;
uint32_t piece_rows(uint64_t tokens, uint64_t vocab) {
  const uint64_t most = std::max<uint64_t>(1024, kPieceBytes / (2 * std::max<uint64_t>(1, tokens)) / 256 * 256);
  const uint64_t pieces = ceil_div(vocab, most);
  return static_cast<uint32_t>(up(ceil_div(vocab, pieces), 256));
}
uint64_t piece_bytes_most(uint64_t tokens, uint64_t vocab) {
  return std::min(std::max(kPieceBytes, tokens * 1024 * 2), tokens * up(vocab, 256) * 2);
}

// Parts of grad_hidden's inner dimension (the vocabulary piece) where its tiles do not fill the CUs, of no less than 512
// rows each; the parts' sums are written and read again.
//   - where grad_weight's product goes beside it (launch_both): tiles for one a CU, and parts no shorter than that product's
//     inner dimension, the tokens (2048 x 4096 x 2048: 137 us backward, 153 with two a CU; 1500 x 3000 x 512: 50 both ways)
//   - else up to one row of tiles, where it is bound by reading the weight: for half the CUs (100 x 32000 x 1024: 70 us, 81
//     with two a CU; 64 x 49152 x 1024: 76, 101; 128 x 131072 x 1024: 266, 264)
//   - else for two a CU (256 x 32000 x 2048: 155 us, 165 with half; 200 x 65536 x 1024: 161, 165; 1024 x 32000 x 1024: 240,
//     263 with one a CU)
uint32_t hidden_splits(uint64_t tokens, uint64_t dim, uint32_t piece) {
  if (tile_of(dim, tokens, 1) == kTileBig) return 1;
  const bool both = tile_of(dim, piece, 1) != kTileBig;
  const uint64_t tiles = ceil_div(dim, kSmall) * ceil_div(tokens, kSmall), most = both ? 256 : tokens <= kSmall ? 128 : 512;
  return static_cast<uint32_t>(std::max<uint64_t>(
      1, std::min<uint64_t>(most / std::min(tiles, most), piece / std::max<uint64_t>(512, both ? tokens : 0))));
}
uint64_t acc_bytes_most(uint64_t tokens, uint64_t dim) {
  // splits * tokens * dim * 4 with splits <= 512 / tiles and tokens * dim <= tiles * 128^2
  return std::max<uint64_t>(tokens * dim * 4, 512ull * kSmall * kSmall * 4);
}

// The forward's pieces: two of each token a tile. Tiles of 64 rows are taken up to 2^21 logits, of 128 up to 2^24, and of 64
// by k_few; else of 256.
uint64_t stats_bytes_most(uint64_t tokens, uint64_t vocab) {
  return tokens * (ceil_div(vocab, 128) + 4) * 8 + std::min<uint64_t>(tokens, kFewTokens) * (ceil_div(vocab, 64) + 1) * 8 +
         (4ull << 20);
}

struct Space {
  uint64_t w, h, rest, bytes;  // packed weight, packed hidden states, then the pass's own
};
Space layout(uint64_t tokens, uint64_t vocab, uint64_t dim, bool pack, bool grads) {
  Space s;
  const uint64_t pdim = up(dim, 8);
  s.w = 0;
  s.h = s.w + (pack ? up(vocab * pdim * 2, 256) : 0);
  s.rest = s.h + (pack ? up(tokens * pdim * 2, 256) : 0);
  uint64_t fwd = up(tokens * 4, 256) + stats_bytes_most(tokens, vocab);
  uint64_t bwd = 256 + kReachBlocks * sizeof(Reach) + 2 * up(tokens * 4, 256) + up(4 * vocab + 4, 256) +
                 up(tokens * pdim * 2, 256) + up(piece_bytes_most(tokens, vocab), 256) + acc_bytes_most(tokens, dim);
  s.bytes = s.rest + (grads ? std::max(fwd, bwd) : fwd) + 256;
  return s;
}

bool rows_ok(const void* p, uint64_t stride) { return aligned(p, 16) && stride % 8 == 0 && stride < kMaxStride; }

constexpr uint32_t kMaxDim = 1u << 20;
constexpr uint64_t kMaxVocab = (1ull << 31) - 257, kMaxTokens = (1ull << 26) - 1;

int check(const char* what, int dtype, uint64_t tokens, uint64_t vocab, uint32_t dim) {
  if (dtype != OMR_BF16 && dtype != OMR_F16) return efail("%s: hidden and weight are bf16 or fp16", what);
  if (dim == 0 || dim > kMaxDim) return efail("%s: dim must be 1..%u", what, kMaxDim);
  if (vocab == 0 || vocab > kMaxVocab) return efail("%s: vocab must be 1..2^31 - 257", what);
  if (tokens > kMaxTokens) return efail("%s: tokens must be below 2^26", what);
  return 0;
}

uint32_t lanes_log(uint32_t pdim) {  // lanes that a row of pdim elements fills, a power of two up to a wave
  uint32_t l = 0;
  while (l < 6 && (8u << l) < pdim) ++l;
  return l;
}

// which of weight and hidden are laid out again, and by how many workgroups
struct Pack {
  bool w, h;
  uint64_t blocks;
};
Pack pack_of(const void* hidden, uint64_t hstride, const void* weight, uint64_t wstride, uint64_t tokens, uint64_t vocab,
             uint32_t dim) {
  Pack p{dim % 8 != 0 || !rows_ok(weight, wstride), dim % 8 != 0 || !rows_ok(hidden, hstride), 0};
  p.blocks = ceil_div((p.w ? vocab : 0) + (p.h ? tokens : 0), 256u >> lanes_log(static_cast<uint32_t>(up(dim, 8))));
  return p;
}

// hidden and weight as row operands of whole 16-byte pieces: the caller's, or copies in the workspace
template <class T>
int operands(const void* hidden, uint64_t hstride, const void* weight, uint64_t wstride, uint64_t tokens, uint64_t vocab,
             uint32_t dim, const Pack& pack, const Space& sp, char* ws, Operand<T>* h, Operand<T>* w, hipStream_t stream) {
  const uint32_t pdim = static_cast<uint32_t>(up(dim, 8)), lpr_log = lanes_log(pdim);
  *h = {static_cast<const T*>(hidden), hstride, static_cast<uint32_t>(tokens)};
  *w = {static_cast<const T*>(weight), wstride, static_cast<uint32_t>(vocab)};
  PackArgs<T> x{w->p, wstride, 0, reinterpret_cast<T*>(ws + sp.w)}, y{h->p, hstride, 0, reinterpret_cast<T*>(ws + sp.h)};
  if (pack.w) {
    x.rows = vocab;
    w->p = x.dst;
    w->ld = pdim;
  }
  if (pack.h) {
    y.rows = tokens;
    h->p = y.dst;
    h->ld = pdim;
  }
  if (pack.blocks == 0) return 0;
  k_pack<T><<<static_cast<unsigned>(pack.blocks), 256, 0, stream>>>(x, y, dim, pdim, lpr_log);
  return elaunch("omr_vocab_loss (layout)");
}

int check_space(const char* what, bool pack, uint64_t tokens, uint64_t vocab, uint32_t dim, bool grads,
                const void* workspace, size_t bytes, Space* sp) {
  *sp = layout(tokens, vocab, dim, pack, grads);
  if (workspace == nullptr || !aligned(workspace, 16)) return efail("%s: the workspace must be 16-byte aligned", what);
  if (bytes < sp->bytes)
    return efail("%s: workspace of %zu bytes, %llu needed%s", what, bytes, static_cast<unsigned long long>(sp->bytes),
                 pack ? " (rows that are not whole 16-byte pieces are laid out again: ask for it with pack)" : "");
  return 0;
}

}  // namespace

extern "C" {

size_t omr_vocab_loss_workspace_bytes(uint64_t max_tokens, uint64_t vocab, uint32_t dim, int pack, int grads) {
  if (dim == 0 || dim > kMaxDim || vocab == 0 || vocab > kMaxVocab || max_tokens > kMaxTokens) return 0;
  return layout(max_tokens, vocab, dim, pack || dim % 8 != 0, grads).bytes;
}

int omr_vocab_loss(const void* hidden, uint64_t hidden_stride, const void* weight, uint64_t weight_stride, int dtype,
                   uint64_t tokens, uint64_t vocab, uint32_t dim, const void* targets, int targets64, float* loss,
                   float* lse, void* workspace, size_t workspace_bytes, omr_stream_t stream) {
  if (const int rc = check("vocab_loss", dtype, tokens, vocab, dim)) return rc;
  if (tokens == 0) return 0;
  if (hidden == nullptr || weight == nullptr || targets == nullptr || loss == nullptr || lse == nullptr)
    return efail("vocab_loss: NULL pointer");
  Space sp;
  const Pack pack = pack_of(hidden, hidden_stride, weight, weight_stride, tokens, vocab, dim);
  if (const int rc = check_space("vocab_loss", pack.w || pack.h, tokens, vocab, dim, false, workspace, workspace_bytes, &sp))
    return rc;
  const bool few = tokens <= kFewTokens;
  if (pack.blocks > kMaxBlocks || (few ? ceil_div(vocab, 64) > kMaxBlocks : !tiles_fit(vocab, tokens, 1)) ||
      ceil_div(tokens, 4) > kMaxBlocks)
    return efail("vocab_loss: too many tokens or rows for one call");
  char* ws = static_cast<char*>(workspace);
  auto go = [&](auto t) {
    using T = decltype(t);
    GemmArgs<T> a{};
    if (const int rc = operands<T>(hidden, hidden_stride, weight, weight_stride, tokens, vocab, dim, pack, sp, ws, &a.b,
                                   &a.a, S(stream)))
      return rc;
    const int tile = tile_of(vocab, tokens, 1);
    a.k = dim;
    a.splits = 1;
    a.ksplit = dim;
    a.targets = targets;
    a.targets64 = targets64;
    a.vocab = static_cast<uint32_t>(vocab);
    a.tokens = static_cast<uint32_t>(tokens);
    a.ztarget = reinterpret_cast<float*>(ws + sp.rest);
    a.stats = reinterpret_cast<float*>(ws + sp.rest + up(tokens * 4, 256));
    if (few) {
      a.pieces = static_cast<uint32_t>(ceil_div(vocab, 64));
      if (tokens <= 16)
        k_few<T, 1><<<a.pieces, 256, 0, S(stream)>>>(a);
      else
        k_few<T, 2><<<a.pieces, 256, 0, S(stream)>>>(a);
      if (const int rc = elaunch("omr_vocab_loss")) return rc;
    } else {
      a.pieces = static_cast<uint32_t>(ceil_div(vocab, tile_rows(tile)) * 2);  // two waves' parts a tile
      if (const int rc = launch<T, kStats>(a, a.vocab, a.tokens, tile, S(stream))) return rc;
    }
    // four waves a token where there are not enough tokens to fill the CUs
    if (tokens <= 1024)
      k_merge<T, 4><<<static_cast<unsigned>(tokens), 256, 0, S(stream)>>>(a, loss, lse);
    else
      k_merge<T, 1><<<static_cast<unsigned>(ceil_div(tokens, 4)), 256, 0, S(stream)>>>(a, loss, lse);
    return elaunch("omr_vocab_loss");
  };
  return dtype == OMR_BF16 ? go(__bf16{}) : go(_Float16{});
}

int omr_vocab_loss_grad(const void* hidden, uint64_t hidden_stride, const void* weight, uint64_t weight_stride,
                        int dtype, uint64_t tokens, uint64_t vocab, uint32_t dim, const void* targets, int targets64,
                        const float* lse, const float* grad_loss, uint64_t grad_loss_stride, void* grad_hidden,
                        uint64_t grad_hidden_stride, void* grad_weight, int grad_weight_dtype,
                        uint64_t grad_weight_stride, int accumulate, void* workspace, size_t workspace_bytes,
                        omr_stream_t stream) {
  if (const int rc = check("vocab_loss_grad", dtype, tokens, vocab, dim)) return rc;
  if (grad_weight != nullptr && grad_weight_dtype != OMR_F32 && grad_weight_dtype != dtype)
    return efail("vocab_loss_grad: grad_weight is fp32 or of the weight's type");
  if ((grad_hidden != nullptr && grad_hidden_stride < dim) || (grad_weight != nullptr && grad_weight_stride < dim))
    return efail("vocab_loss_grad: an output's row stride is shorter than dim %u", dim);
  if (tokens != 0 && (hidden == nullptr || weight == nullptr || targets == nullptr || lse == nullptr ||
                      grad_loss == nullptr))
    return efail("vocab_loss_grad: NULL pointer");
  if (tokens == 0) {  // a sum over no tokens
    if (grad_weight == nullptr || accumulate) return 0;
    const uint64_t blocks = std::min<uint64_t>(ceil_div(vocab * dim, 256), 1u << 16);
    if (grad_weight_dtype == OMR_F32)
      k_zero<float><<<static_cast<unsigned>(blocks), 256, 0, S(stream)>>>(static_cast<float*>(grad_weight), vocab, dim,
                                                                          grad_weight_stride);
    else  // (a zero has the same bits in both 16-bit types)
      k_zero<__bf16><<<static_cast<unsigned>(blocks), 256, 0, S(stream)>>>(static_cast<__bf16*>(grad_weight), vocab, dim,
                                                                           grad_weight_stride);
    return elaunch("omr_vocab_loss_grad");
  }
  Space sp;
  const Pack pack = pack_of(hidden, hidden_stride, weight, weight_stride, tokens, vocab, dim);
  if (const int rc = check_space("vocab_loss_grad", pack.w || pack.h, tokens, vocab, dim, true, workspace, workspace_bytes,
                                 &sp))
    return rc;
  const uint32_t pdim = static_cast<uint32_t>(up(dim, 8)), piece = piece_rows(tokens, vocab);
  const uint32_t whole = static_cast<uint32_t>(std::min<uint64_t>(piece, vocab));  // rows of a piece but the last
  const uint32_t first_cols = static_cast<uint32_t>(up(whole, 256));
  // (a piece's columns of G that are written: zeros behind the vocabulary)
  const uint32_t ksplit = static_cast<uint32_t>(up(ceil_div(whole, hidden_splits(tokens, dim, piece)), kBK));
  const uint32_t splits = static_cast<uint32_t>(ceil_div(whole, ksplit));  // of a whole piece; the last may have fewer
  const bool beside = tokens <= kFindHere && tile_of(first_cols, tokens, 1) != kTileBig;
  // (beside the product few sorters: they hold places of its tiles)
  const uint32_t lpr_log = lanes_log(pdim), sort_rows = beside ? SortSpace<4>::kRange : sort_range(static_cast<uint32_t>(vocab));
  const uint64_t sorters = ceil_div(vocab, sort_rows),
                 prepare_blocks = sorters + ceil_div(tokens, (beside ? 256u : 1024u) >> lpr_log);
  if (pack.blocks > kMaxBlocks || !tiles_fit(first_cols, tokens, 1) ||
      (grad_hidden != nullptr && !tiles_fit(dim, tokens, splits)) ||
      (grad_weight != nullptr && (!tiles_fit(dim, first_cols, 1) || prepare_blocks >= kMaxTiles)))
    return efail("vocab_loss_grad: too many tokens or rows for one call");
  char* ws = static_cast<char*>(workspace);
  auto go = [&](auto t) {
    using T = decltype(t);
    Operand<T> h, w;
    if (const int rc = operands<T>(hidden, hidden_stride, weight, weight_stride, tokens, vocab, dim, pack, sp, ws, &h, &w,
                                   S(stream)))
      return rc;
    uint64_t at = sp.rest;
    auto take = [&](uint64_t bytes) {
      char* p = ws + at;
      at += up(bytes, 256);
      return p;
    };
    float* amax = reinterpret_cast<float*>(take(8));
    Reach* reach = reinterpret_cast<Reach*>(take(kReachBlocks * sizeof(Reach)));
    float* lost = reinterpret_cast<float*>(take(tokens * 4));
    uint32_t* perm = reinterpret_cast<uint32_t*>(take(tokens * 4));
    uint32_t* start = reinterpret_cast<uint32_t*>(take(4 * vocab + 4));
    T* clean = reinterpret_cast<T*>(take(tokens * pdim * 2));
    T* g = reinterpret_cast<T*>(take(piece_bytes_most(tokens, vocab)));
    float* acc = reinterpret_cast<float*>(take(acc_bytes_most(tokens, dim)));
    GemmArgs<T> a{};
    a.targets = targets;
    a.targets64 = targets64;
    a.vocab = static_cast<uint32_t>(vocab);
    a.tokens = static_cast<uint32_t>(tokens);
    a.dim = dim;
    a.up = grad_loss;
    a.upstride = grad_loss_stride;
    a.amax = amax;
    PrepareArgs<T> p{};
    if (grad_weight != nullptr) {
      p.lpr_log = lpr_log;
      p.range = sort_rows;
      p.sorters = static_cast<uint32_t>(sorters);
      p.blocks = static_cast<uint32_t>(prepare_blocks);
      p.start = start;
      p.perm = perm;
      p.src = static_cast<const T*>(hidden);
      p.stride = hidden_stride;
      p.pdim = pdim;
      p.amax = amax;
      p.dst = clean;
      if (dtype == OMR_F16 && grad_loss_stride != 0) {
        p.parts = reach;
        p.nparts = static_cast<uint32_t>(std::min<uint64_t>(ceil_div(tokens, 256u >> p.lpr_log), kReachBlocks));
        k_reach<T><<<p.nparts, 256, 0, S(stream)>>>(a, p.src, p.stride, p.lpr_log, reach);
        if (const int rc = elaunch("omr_vocab_loss_grad (reach)")) return rc;
      }
      if (!beside) {
        if (p.parts == nullptr && tokens > kFindHere) {
          k_largest<T><<<1, 1024, 0, S(stream)>>>(a, amax);
          if (const int rc = elaunch("omr_vocab_loss_grad (largest)")) return rc;
        }
        if (targets64)
          k_prepare<T, int64_t><<<p.blocks, 1024, 0, S(stream)>>>(a, p);
        else
          k_prepare<T, int32_t><<<p.blocks, 1024, 0, S(stream)>>>(a, p);
        if (const int rc = elaunch("omr_vocab_loss_grad (prepare)")) return rc;
      }
    }
    a.lse = lse;
    a.g = g;
    a.ldg = piece;
    a.acc = acc;
    a.lost = lost;
    a.w = w;
    a.start = start;
    a.perm = perm;
    for (uint64_t v0 = 0; v0 < vocab; v0 += piece) {
      const uint32_t rows = static_cast<uint32_t>(std::min<uint64_t>(piece, vocab - v0));
      const uint32_t cols = static_cast<uint32_t>(up(rows, 256));
      a.v0 = static_cast<uint32_t>(v0);
      GemmArgs<T> z = a;
      z.a = {w.p + v0 * w.ld, w.ld, rows};
      z.b = h;
      z.k = dim;
      z.ksplit = dim;
      z.splits = 1;
      const int zt = tile_of(cols, tokens, 1);
      if (grad_weight != nullptr && beside && v0 == 0) {
        if (const int rc = targets64 ? launch_grad_prepare<T, int64_t>(z, p, cols, zt, S(stream))
                                     : launch_grad_prepare<T, int32_t>(z, p, cols, zt, S(stream)))
          return rc;
      } else if (const int rc = launch<T, kGrad>(z, cols, z.tokens, zt, S(stream))) {
        return rc;
      }
      GemmArgs<T> x = a, y = a;
      x.a = {w.p + v0 * w.ld, w.ld, pdim};
      x.b = {g, piece, x.tokens};
      x.k = rows;
      x.ksplit = ksplit;
      x.splits = static_cast<uint32_t>(ceil_div(rows, ksplit));
      x.first = v0 == 0;
      const bool done = v0 + piece >= vocab;
      x.last = done && splits == 1;
      x.out = grad_hidden;
      x.ostride = grad_hidden_stride;
      y.a = {clean, pdim, pdim};
      y.b = {g, piece, cols};
      y.k = y.tokens;
      y.ksplit = y.tokens;
      y.splits = 1;
      y.out = grad_weight;
      y.ostride = grad_weight_stride;
      y.out_f32 = grad_weight_dtype == OMR_F32;
      y.accumulate = accumulate != 0;
      const int xt = tile_of(dim, x.tokens, x.splits), yt = tile_of(dim, cols, 1);
      if (grad_hidden != nullptr && grad_weight != nullptr && xt != kTileBig && yt != kTileBig) {
        if (const int rc = launch_both<T>(x, y, dim, cols, S(stream))) return rc;
      } else {
        if (grad_hidden != nullptr)
          if (const int rc = launch<T, kHidden>(x, dim, x.tokens, xt, S(stream))) return rc;
        if (grad_weight != nullptr)
          if (const int rc = launch<T, kWeight>(y, dim, cols, yt, S(stream))) return rc;
      }
      if (grad_hidden != nullptr && done && splits > 1) {
        x.splits = splits;
        k_join<T><<<static_cast<unsigned>(ceil_div(tokens * dim, 256)), 256, 0, S(stream)>>>(x);
        if (const int rc = elaunch("omr_vocab_loss_grad (join)")) return rc;
      }
    }
    return 0;
  };
  return dtype == OMR_BF16 ? go(__bf16{}) : go(_Float16{});
}

}  // extern "C"
