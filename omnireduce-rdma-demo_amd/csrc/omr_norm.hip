// omr_norm.hip — layer norm, forward and backward, with the reduction of the weight's and bias's gradients.
//
//   forward   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), y = (x - mu) r w + b
//   backward  xh = (x - mu) r, g = dy w:
//             dx = r (g - mean(g) - xh mean(g xh)),  dw (+)= sum over rows of dy xh,  db (+)= sum over rows of dy
//
// Both are bound by HBM (the forward reads and writes each element once, the backward reads two and writes one), so a
// row is read once and held in registers: WPR waves hold a row, 16 columns a lane, and statistics are two-pass sums over
// the registers: the mean first, then the distances d from it and their squares.  A mean far from zero is off by some of its
// own roundings, which the distances' mean c shows: mean + c, d - c and mean(d^2) - c^2 lose nothing to it (without that
// a row of 1000 times 10000.1 gave -0.3 for each, where it gives 0).  Workgroups walk
// several rows, so the parameters are loaded once, the next row is loaded while one is worked on, and the backward keeps
// its part of dw and db in registers until its last row: one partial row a workgroup, which a second launch adds up in a
// fixed order.  16384 rows of 4096 bf16 forward: 49 us, 5.5 TB/s (62 without the row ahead; a large copy reaches 5.1);
// 16384 of 2048 backward: 42 us, 4.8 TB/s, 4.6 of it the second launch; 65536 of 1024: 75 us, 5.4 TB/s.
// Rows of more than 16384 columns take the *_any kernels, which read a row again instead of holding it.
#include "omr_elem.h"

#include <type_traits>

using namespace omr_elem;

namespace {

constexpr int kCols = 16;  // columns a lane holds

struct NormArgs {
  const void* x;
  uint64_t xstride;
  const void* w;  // or null: ones
  const void* b;  // or null: zeros
  void* out;      // y, or dx
  uint64_t ostride;
  float* mean;
  float* rstd;
  const void* dy;
  uint64_t dystride;
  float* partial;  // [blocks][2][dim]: dw, db; or null
  uint64_t rows;
  uint32_t dim;
  float eps, inv_dim;
};

// Sum over the WPR waves of a row, in every lane.  Each call site has LDS of its own, and between two uses of one there
// is another's barrier (or, where a kernel has one call site, two alternating buffers).
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* lds) {
  v = wave_sum(v);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < WPR; ++w) v += lds[w];
  }
  return v;
}

__device__ __forceinline__ float lane_of(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// Two such sums behind one barrier, and for the exchanges of one: behind the first, lanes 0..31 carry v's and 32..63 q's.
// (16384 x 2048 bf16 read from the last-level cache: 23.5 us, 24.0 with 12 exchanges, 22.4 without the distances' sum, which
// is hidden where rows come from HBM.)
template <int WPR>
__device__ __forceinline__ float2 row_sum2(float v, float q, float2* lds) {
  const uint32_t lane = threadIdx.x & 63;
  float s = (lane < 32 ? v : q) + __shfl_xor(lane < 32 ? q : v, 32);
#pragma unroll
  for (int d = 16; d; d >>= 1) s += __shfl_xor(s, d);
  if constexpr (WPR == 1) {
    return make_float2(lane_of(s, 0), lane_of(s, 32));
  } else {
    if (lane % 32 == 0) reinterpret_cast<float*>(lds)[2 * (threadIdx.x >> 6) + lane / 32] = s;
    __syncthreads();
    float2 sums = lds[0];
#pragma unroll
    for (int w = 1; w < WPR; ++w) {
      sums.x += lds[w].x;
      sums.y += lds[w].y;
    }
    return sums;
  }
}

// The mean's first estimate, rounded: one value for the distances and for what their mean is added to (a product joined to
// the subtraction behind it, as the compiler may, would give the distances from another one).
__device__ __forceinline__ float estimate(float sum, float inv_dim) {
  float near = sum * inv_dim;
  asm volatile("" : "+v"(near));
  return near;
}

// 1 / sqrt(variance + eps) from the means of the distances and of their squares (which round to less than nothing at times)
__device__ __forceinline__ float rstd_of(float c, float squares, float eps) {
  const float var = squares - c * c;
  return 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + eps);
}

// VEC elements as they lie in memory, at any alignment; of a row's last piece the first n
template <class T, int VEC>
struct Piece {
  vec_t<T, VEC> v;

  __device__ __forceinline__ void load(const T* p, uint32_t n) {
    if (n >= VEC) {
      v = *reinterpret_cast<const any_vec<T, VEC>*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = static_cast<uint32_t>(i) < n ? p[i] : static_cast<T>(0.0f);
    }
  }

  __device__ __forceinline__ void arrive() { asm volatile("" : "+v"(v)); }  // it is waited for here
};

// Columns there are from c on: all VEC of them where rows are whole pieces (END false), known when compiling.
// Lanes behind the end of such a row (in() false) hold its last piece once more (at()), write the same results to the same
// place, and count in no sum: so neither loads nor stores need a branch.
template <int VEC, bool END>
__device__ __forceinline__ uint32_t have(uint32_t dim, uint32_t c) {
  return END ? dim - c : VEC;
}

template <class T, class P, int WPR, bool END>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void k_norm(NormArgs a) {
  constexpr int VEC = 16 / sizeof(T), NV = kCols / VEC, RPB = WPR == 1 ? 4 : 1;
  __shared__ float lds[WPR];
  __shared__ float2 lds2[WPR];
  // a lane's columns: VEC consecutive ones of every piece j
  const uint32_t t = WPR == 1 ? (threadIdx.x & 63) : threadIdx.x;
  auto col = [&](int j) { return (static_cast<uint32_t>(j) * 64 * WPR + t) * VEC; };
  auto in = [&](int j) { return col(j) < a.dim; };
  auto at = [&](int j) { return END ? col(j) : min(col(j), a.dim - VEC); };
  float w[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      w[j][i] = 1.0f;
      b[j][i] = 0.0f;
    }
    if (END && !in(j)) continue;
    const uint32_t n = have<VEC, END>(a.dim, at(j));
    if (a.w != nullptr) load_some<P, VEC>(static_cast<const P*>(a.w) + at(j), n, w[j]);
    if (a.b != nullptr) load_some<P, VEC>(static_cast<const P*>(a.b) + at(j), n, b[j]);
  }
  // The next row is on its way while this one is worked on: loads and stores without a branch (a register that a branch
  // may leave as it was is waited for and copied at once), and waited for behind this row's stores, whose number is known
  // there, so that the stores need not be done.
  Piece<T, VEC> ahead[NV];
  auto arrive = [&]() {
    if constexpr (!END) {
#pragma unroll
      for (int j = 0; j < NV; ++j) ahead[j].arrive();
    }
  };
  auto fetch = [&](uint64_t row) {
    const T* p = static_cast<const T*>(a.x) + (row < a.rows ? row : a.rows - 1) * a.xstride;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (!END || in(j)) ahead[j].load(p + at(j), have<VEC, END>(a.dim, at(j)));
  };
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * RPB;
  uint64_t row = static_cast<uint64_t>(blockIdx.x) * RPB + (WPR == 1 ? threadIdx.x >> 6 : 0);
  if (!END || row < a.rows) fetch(row);
  arrive();
  for (; row < a.rows; row += step) {
    float v[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = !END || in(j) ? static_cast<float>(ahead[j].v[i]) : 0.0f;
    if (!END || row + step < a.rows) fetch(row + step);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float piece = 0.0f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) piece += v[j][i];
      s += in(j) ? piece : 0.0f;
    }
    const float near = estimate(row_sum<WPR>(s, lds), a.inv_dim);
    float d = 0.0f, q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float piece = 0.0f, squares = 0.0f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[j][i] = !END || col(j) + i < a.dim ? v[j][i] - near : 0.0f;
        piece += v[j][i];
        squares += v[j][i] * v[j][i];
      }
      d += in(j) ? piece : 0.0f;
      q += in(j) ? squares : 0.0f;
    }
    const float2 sums = row_sum2<WPR>(d, q, lds2);
    const float c = sums.x * a.inv_dim, mean = near + c, rstd = rstd_of(c, sums.y * a.inv_dim, a.eps), shift = -c * rstd;
    T* out = static_cast<T*>(a.out) + row * a.ostride;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (END && !in(j)) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = __builtin_fmaf(v[j][i], rstd, shift) * w[j][i] + b[j][i];
      stream_some<T, VEC>(out + at(j), have<VEC, END>(a.dim, at(j)), v[j]);
    }
    if (WPR == 1 ? (threadIdx.x & 63) == 0 : threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    arrive();
  }
}

// A workgroup of 8 waves holds 8 / WPR rows at a time (WPR 16: one row of 16 waves), in lockstep where a row is more
// than a wave.  Registers for one workgroup a CU (see grad_blocks), or for two where rows end inside a piece.
template <class T, class P, int WPR, bool END>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 512, WPR == 16 || END ? 4 : 2) void k_norm_grad(NormArgs a) {
  constexpr int VEC = 16 / sizeof(T), NV = kCols / VEC, RPB = WPR == 16 ? 1 : 8 / WPR, WAVES = RPB * WPR, NT = 64 * WAVES;
  __shared__ float lds[2][2][WAVES];
  __shared__ float sum[RPB > 1 ? WAVES * 64 * kCols : 1];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slot = wave / WPR,
                 t = threadIdx.x - slot * 64 * WPR;
  auto col = [&](int j) { return (static_cast<uint32_t>(j) * 64 * WPR + t) * VEC; };
  auto in = [&](int j) { return col(j) < a.dim; };
  auto at = [&](int j) { return END ? col(j) : min(col(j), a.dim - VEC); };
  float dw[NV][VEC] = {}, db[NV][VEC] = {};
  // The next row is on its way while this one is worked on, where there are registers for it (8192 x 2048 fp32: 41 us
  // against 46).  The weight waits in LDS (a lane's columns together).
  constexpr bool kAhead = WPR <= 8 && (sizeof(T) == 2 || !END);
  __shared__ __attribute__((aligned(16))) float w[64 * WPR * kCols];
  if (slot == 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] = 1.0f;
      if (a.w != nullptr && (!END || in(j)))
        load_some<P, VEC>(static_cast<const P*>(a.w) + at(j), have<VEC, END>(a.dim, at(j)), f);
      store_f32<float, VEC>(&w[(j * 64 * WPR + t) * VEC], f);
    }
  }
  __syncthreads();
  Piece<T, VEC> xa[NV], da[NV];
  float mean_a, rstd_a;
  auto arrive = [&]() {
    if constexpr (kAhead && !END) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        xa[j].arrive();
        da[j].arrive();
      }
      asm volatile("" : "+v"(mean_a), "+v"(rstd_a));
    }
  };
  auto fetch = [&](uint64_t row) {
    row = row < a.rows ? row : a.rows - 1;
    const T* x = static_cast<const T*>(a.x) + row * a.xstride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dystride;
    mean_a = a.mean[row];
    rstd_a = a.rstd[row];
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (!END || in(j)) {
        xa[j].load(x + at(j), have<VEC, END>(a.dim, at(j)));
        da[j].load(dy + at(j), have<VEC, END>(a.dim, at(j)));  // (zeros behind a row's end add nothing below)
      }
  };
  int flip = 0;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * RPB;
  if (kAhead) fetch(static_cast<uint64_t>(blockIdx.x) * RPB + slot);
  arrive();
  for (uint64_t first = static_cast<uint64_t>(blockIdx.x) * RPB; first < a.rows; first += step) {
    const uint64_t row = first + slot;
    const bool real = row < a.rows;
    float v[NV][VEC], g[NV][VEC];
    float s1 = 0.0f, s2 = 0.0f;
    if (!kAhead) fetch(row);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[j][i] = static_cast<float>(xa[j].v[i]);
        g[j][i] = static_cast<float>(da[j].v[i]);
      }
    const float mean = mean_a, rstd = rstd_a;
    if (kAhead) fetch(row + step);
    if (real) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (END && !in(j)) continue;
        float wj[VEC], p1 = 0.0f, p2 = 0.0f;
        load_f32<float, VEC>(&w[(j * 64 * WPR + t) * VEC], wj);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xh = (v[j][i] - mean) * rstd;
          v[j][i] = xh;
          dw[j][i] += g[j][i] * xh;
          db[j][i] += g[j][i];
          g[j][i] *= wj[i];
          p1 += g[j][i];
          p2 += g[j][i] * xh;
        }
        s1 += in(j) ? p1 : 0.0f;
        s2 += in(j) ? p2 : 0.0f;
      }
    }
    // both sums behind one barrier; the buffers alternate, so a wave that is a row ahead writes the other one
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if constexpr (WPR > 1) {
      if ((threadIdx.x & 63) == 0) {
        lds[flip][0][wave] = s1;
        lds[flip][1][wave] = s2;
      }
      __syncthreads();
      s1 = lds[flip][0][slot * WPR];
      s2 = lds[flip][1][slot * WPR];
#pragma unroll
      for (int k = 1; k < WPR; ++k) {
        s1 += lds[flip][0][slot * WPR + k];
        s2 += lds[flip][1][slot * WPR + k];
      }
      flip ^= 1;
    }
    if (!real) {
      arrive();
      break;
    }
    s1 *= a.inv_dim;
    s2 *= a.inv_dim;
    T* out = static_cast<T*>(a.out) + row * a.ostride;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (END && !in(j)) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) g[j][i] = (g[j][i] - s1 - v[j][i] * s2) * rstd;
      stream_some<T, VEC>(out + at(j), have<VEC, END>(a.dim, at(j)), g[j]);
    }
    arrive();  // (behind the stores, as in k_norm)
  }
  if (a.partial == nullptr) return;
  float* part = a.partial + static_cast<uint64_t>(blockIdx.x) * 2 * a.dim;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&mine)[NV][VEC] = which == 0 ? dw : db;
    if constexpr (RPB > 1) {  // the slots' sums, in slot order
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[((slot * NV + j) * VEC + i) * 64 * WPR + t] = mine[j][i];
      __syncthreads();
      constexpr uint32_t kWidth = 64 * WPR * kCols;  // entry e of a slot: piece j, element i, lane
      for (uint32_t e = threadIdx.x; e < kWidth; e += NT) {
        const uint32_t ji = e / (64 * WPR), c = (ji / VEC * 64 * WPR + e % (64 * WPR)) * VEC + ji % VEC;
        float s = sum[e];
#pragma unroll
        for (int r = 1; r < RPB; ++r) s += sum[r * kWidth + e];
        if (c < a.dim) part[which * a.dim + c] = s;
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (col(j) < a.dim)
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (!END || col(j) + i < a.dim) part[which * a.dim + col(j) + i] = mine[j][i];
    }
  }
}

// ---------------------------------------------------------------- rows longer than the registers hold

constexpr int kAnyWaves = 16;

template <class T, class P>
__global__ __launch_bounds__(64 * kAnyWaves) void k_norm_any(NormArgs a) {
  __shared__ float lds[kAnyWaves];
  __shared__ float2 lds2[kAnyWaves];
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.xstride;
    T* out = static_cast<T*>(a.out) + row * a.ostride;
    float s = 0.0f;
    for (uint32_t c = threadIdx.x; c < a.dim; c += 64 * kAnyWaves) s += static_cast<float>(x[c]);
    const float near = estimate(row_sum<kAnyWaves>(s, lds), a.inv_dim);
    float d = 0.0f, q = 0.0f;
    for (uint32_t c = threadIdx.x; c < a.dim; c += 64 * kAnyWaves) {
      const float v = static_cast<float>(x[c]) - near;
      d += v;
      q += v * v;
    }
    const float2 sums = row_sum2<kAnyWaves>(d, q, lds2);
    const float off = sums.x * a.inv_dim, rstd = rstd_of(off, sums.y * a.inv_dim, a.eps);
    for (uint32_t c = threadIdx.x; c < a.dim; c += 64 * kAnyWaves) {
      const float w = a.w != nullptr ? static_cast<float>(static_cast<const P*>(a.w)[c]) : 1.0f;
      const float b = a.b != nullptr ? static_cast<float>(static_cast<const P*>(a.b)[c]) : 0.0f;
      out[c] = static_cast<T>((static_cast<float>(x[c]) - near - off) * rstd * w + b);
    }
    if (threadIdx.x == 0) {
      a.mean[row] = near + off;
      a.rstd[row] = rstd;
    }
  }
}

template <class T, class P>
__global__ __launch_bounds__(64 * kAnyWaves) void k_norm_dx_any(NormArgs a) {
  __shared__ float lds[2][kAnyWaves];
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.xstride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dystride;
    T* out = static_cast<T*>(a.out) + row * a.ostride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (uint32_t c = threadIdx.x; c < a.dim; c += 64 * kAnyWaves) {
      const float w = a.w != nullptr ? static_cast<float>(static_cast<const P*>(a.w)[c]) : 1.0f;
      const float g = static_cast<float>(dy[c]) * w;
      s1 += g;
      s2 += g * ((static_cast<float>(x[c]) - mean) * rstd);
    }
    s1 = row_sum<kAnyWaves>(s1, lds[0]) * a.inv_dim;
    s2 = row_sum<kAnyWaves>(s2, lds[1]) * a.inv_dim;
    for (uint32_t c = threadIdx.x; c < a.dim; c += 64 * kAnyWaves) {
      const float w = a.w != nullptr ? static_cast<float>(static_cast<const P*>(a.w)[c]) : 1.0f;
      const float xh = (static_cast<float>(x[c]) - mean) * rstd;
      out[c] = static_cast<T>((static_cast<float>(dy[c]) * w - s1 - xh * s2) * rstd);
    }
  }
}

// 64 columns a workgroup, its 16 waves a row each in turn
template <class T>
__global__ __launch_bounds__(64 * kAnyWaves) void k_norm_params_any(NormArgs a) {
  __shared__ float sum[2][kAnyWaves][64];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t c = blockIdx.x * 64 + lane;
  float dw = 0.0f, db = 0.0f;
  if (c < a.dim)
    for (uint64_t row = static_cast<uint64_t>(blockIdx.y) * kAnyWaves + wave; row < a.rows;
         row += static_cast<uint64_t>(gridDim.y) * kAnyWaves) {
      const float g = static_cast<float>(static_cast<const T*>(a.dy)[row * a.dystride + c]);
      const float x = static_cast<float>(static_cast<const T*>(a.x)[row * a.xstride + c]);
      dw += g * ((x - a.mean[row]) * a.rstd[row]);
      db += g;
    }
  sum[0][wave][lane] = dw;
  sum[1][wave][lane] = db;
  __syncthreads();
  if (wave < 2 && c < a.dim) {
    float s = 0.0f;
    for (int w = 0; w < kAnyWaves; ++w) s += sum[wave][w][lane];
    a.partial[(static_cast<uint64_t>(blockIdx.y) * 2 + wave) * a.dim + c] = s;
  }
}

// ---------------------------------------------------------------- the partial rows' sum
//
// 64 columns a workgroup; wave w adds the partial rows w, w + 16, ..., and wave 0 the sixteen sums in wave order.
__global__ __launch_bounds__(64 * kAnyWaves) void k_norm_params(const float* partial, uint32_t blocks, uint32_t dim,
                                                                float* dw, float* db, int accumulate) {
  __shared__ float sum[kAnyWaves][64];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t c = static_cast<uint64_t>(blockIdx.x) * 64 + lane, width = 2ull * dim;
  float s = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (uint32_t k = wave; k < blocks; k += kAnyWaves) s += partial[k * width + c];
  }
  sum[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= width) return;
  for (int w = 1; w < kAnyWaves; ++w) s += sum[w][lane];
  float* out = c < dim ? dw : db;
  if (out == nullptr) return;
  out += c < dim ? c : c - dim;
  *out = accumulate ? *out + s : s;
}

__global__ __launch_bounds__(256) void k_zero(float* p, uint64_t n) {
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) p[i] = 0.0f;
}

int waves_per_row(uint32_t dim) {
  int w = 1;
  while (w <= 16 && static_cast<uint32_t>(w) * 64 * kCols < dim) w *= 2;
  return w;  // 32: too long for registers
}

// Workgroups of the backward: one a CU.  Each ends in a partial row of 2 dim floats, written and read again; a second
// workgroup a CU hides nothing that the row ahead does not, and doubles them (8192 x 4096 bf16: 50 us against 45, 4096 x
// 8192: 56 against 48, 65536 x 1024: 81 against 75).  Rows that end inside a piece have branches between their loads, and
// are held by one wave up to 1024 columns: there two hide more (16384 x 777 bf16: 24 us against 26).
uint32_t grad_blocks(uint64_t rows, uint32_t dim, bool end) {
  const int wpr = waves_per_row(dim);
  const uint64_t want = wpr > 16 ? ceil_div(rows, kAnyWaves) : wpr == 16 ? rows : ceil_div(rows, 8 / wpr);
  const uint64_t most = end && wpr == 1 ? 512 : 256;
  return static_cast<uint32_t>(want < most ? want : most);
}

// fn(WPR, whether rows end inside a piece) as integral constants
template <class F>
int with_shape(bool end, int wpr, F&& fn) {
  auto ends = [&](auto p) { return end ? fn(p, std::true_type{}) : fn(p, std::false_type{}); };
  switch (wpr) {
    case 1: return ends(std::integral_constant<int, 1>{});
    case 2: return ends(std::integral_constant<int, 2>{});
    case 4: return ends(std::integral_constant<int, 4>{});
    case 8: return ends(std::integral_constant<int, 8>{});
    default: return ends(std::integral_constant<int, 16>{});
  }
}

constexpr uint64_t kMaxRows = 1ull << 40;

int check_args(const char* what, int dtype, int param_dtype, uint64_t rows, uint32_t dim) {
  if (!dtype_ok(dtype) || (param_dtype != OMR_F32 && param_dtype != dtype))
    return efail("%s: elements are fp32, bf16 or fp16, and parameters fp32 or of the elements' type", what);
  if (dim == 0 || dim > OMR_MAX_DIM) return efail("%s: dim must be 1..%u", what, OMR_MAX_DIM);
  if (rows >= kMaxRows) return efail("%s: too many rows", what);
  return 0;
}

}  // namespace

extern "C" {

int omr_layer_norm(const void* x, int dtype, uint64_t rows, uint32_t dim, uint64_t x_stride, const void* weight,
                   const void* bias, int param_dtype, float eps, void* out, uint64_t out_stride, float* mean,
                   float* rstd, omr_stream_t stream) {
  if (const int rc = check_args("layer_norm", dtype, param_dtype, rows, dim)) return rc;
  if (out_stride < dim) return efail("layer_norm: the output's row stride is shorter than dim %u", dim);
  if (!(eps >= 0.0f)) return efail("layer_norm: eps must not be negative");
  if (rows == 0) return 0;
  if (x == nullptr || out == nullptr || mean == nullptr || rstd == nullptr) return efail("layer_norm: NULL pointer");
  NormArgs a{};
  a.x = x;
  a.xstride = x_stride;
  a.w = weight;
  a.b = bias;
  a.out = out;
  a.ostride = out_stride;
  a.mean = mean;
  a.rstd = rstd;
  a.rows = rows;
  a.dim = dim;
  a.eps = eps;
  a.inv_dim = 1.0f / static_cast<float>(dim);
  const int wpr = waves_per_row(dim);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto params = [&](auto p) {
      using P = decltype(p);
      if (wpr > 16) {
        const unsigned grid = static_cast<unsigned>(rows < 2048 ? rows : 2048);
        k_norm_any<T, P><<<grid, 64 * kAnyWaves, 0, S(stream)>>>(a);
        return elaunch("omr_layer_norm");
      }
      return with_shape(dim % (16 / sizeof(T)) != 0, wpr, [&](auto waves, auto end) {
        constexpr int WPR = decltype(waves)::value;
        const uint64_t want = WPR == 1 ? ceil_div(rows, 4) : rows;
        const uint64_t most = WPR <= 4 ? 1024 : 4096 / WPR;
        k_norm<T, P, WPR, decltype(end)::value><<<static_cast<unsigned>(want < most ? want : most), WPR == 1 ? 256 : 64 * WPR, 0,
                                 S(stream)>>>(a);
        return elaunch("omr_layer_norm");
      });
    };
    return param_dtype == OMR_F32 ? params(float{}) : params(T{});
  });
}

size_t omr_layer_norm_grad_workspace_bytes(uint64_t rows, uint32_t dim) {
  if (dim == 0 || dim > OMR_MAX_DIM || rows >= kMaxRows) return 0;
  return static_cast<size_t>(grad_blocks(rows, dim, true)) * 2 * dim * sizeof(float) + 16;
}

int omr_layer_norm_grad(const void* grad_out, uint64_t grad_stride, const void* x, int dtype, uint64_t rows,
                        uint32_t dim, uint64_t x_stride, const float* mean, const float* rstd, const void* weight,
                        int param_dtype, void* grad_x, uint64_t grad_x_stride, float* grad_weight, float* grad_bias,
                        int accumulate, void* workspace, size_t workspace_bytes, omr_stream_t stream) {
  if (const int rc = check_args("layer_norm_grad", dtype, param_dtype, rows, dim)) return rc;
  if (grad_x_stride < dim) return efail("layer_norm_grad: grad_x's row stride is shorter than dim %u", dim);
  const bool params = grad_weight != nullptr || grad_bias != nullptr;
  if (rows == 0) {  // sums over no rows
    for (float* p : {grad_weight, grad_bias})
      if (p != nullptr && !accumulate) k_zero<<<static_cast<unsigned>(ceil_div(dim, 256)), 256, 0, S(stream)>>>(p, dim);
    return elaunch("omr_layer_norm_grad");
  }
  if (grad_out == nullptr || x == nullptr || mean == nullptr || rstd == nullptr || grad_x == nullptr)
    return efail("layer_norm_grad: NULL pointer");
  if (params && (workspace == nullptr || !aligned(workspace, 16)))
    return efail("layer_norm_grad: the parameters' gradients need a 16-byte aligned workspace");
  if (params && workspace_bytes < omr_layer_norm_grad_workspace_bytes(rows, dim))
    return efail("layer_norm_grad: workspace of %zu bytes, %zu needed", workspace_bytes,
                 omr_layer_norm_grad_workspace_bytes(rows, dim));
  NormArgs a{};
  a.x = x;
  a.xstride = x_stride;
  a.dy = grad_out;
  a.dystride = grad_stride;
  a.w = weight;
  a.out = grad_x;
  a.ostride = grad_x_stride;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.partial = params ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows;
  a.dim = dim;
  a.inv_dim = 1.0f / static_cast<float>(dim);
  const int wpr = waves_per_row(dim);
  const bool end = dim % (16 / elem_bytes(dtype)) != 0;
  const uint32_t blocks = grad_blocks(rows, dim, end);
  const int rc = with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto p) {
      using P = decltype(p);
      if (wpr > 16) {  // (the parameters first: grad_x may be grad_out or x)
        if (params) {
          const dim3 grid(static_cast<unsigned>(ceil_div(dim, 64)), blocks);
          k_norm_params_any<T><<<grid, 64 * kAnyWaves, 0, S(stream)>>>(a);
          if (const int rc = elaunch("omr_layer_norm_grad (parameters)")) return rc;
        }
        k_norm_dx_any<T, P><<<static_cast<unsigned>(rows < 2048 ? rows : 2048), 64 * kAnyWaves, 0, S(stream)>>>(a);
        return elaunch("omr_layer_norm_grad");
      }
      return with_shape(end, wpr, [&](auto waves, auto ends) {
        constexpr int WPR = decltype(waves)::value;
        k_norm_grad<T, P, WPR, decltype(ends)::value><<<blocks, WPR == 16 ? 1024 : 512, 0, S(stream)>>>(a);
        return elaunch("omr_layer_norm_grad");
      });
    };
    return param_dtype == OMR_F32 ? go(float{}) : go(T{});
  });
  if (rc != 0 || !params) return rc;
  k_norm_params<<<static_cast<unsigned>(ceil_div(2ull * dim, 64)), 64 * kAnyWaves, 0, S(stream)>>>(
      a.partial, blocks, dim, grad_weight, grad_bias, accumulate != 0);
  return elaunch("omr_layer_norm_grad (sum)");
}

}  // extern "C"
