// What the forward and the backward of the fused block norms share: a row spread over a group of
// threads, its reductions and statistics, and the choice of a kernel for a width.
#pragma once

#include <stdexcept>

#include "kernels.h"
#include "typed_io.cuh"

namespace mmf {

namespace {

// `tpr` threads of the block that share one row (a power of two from 32 up).  Every thread of the
// block takes part in every reduction.
struct RowGroup {
  int tpr, row, lane, warp0, warps;
  float* red;  // [2][3 * 32], used in turn so that one barrier a reduction is enough
  int turn = 0;
  __device__ RowGroup(int tpr_, float* red_) : tpr(tpr_), red(red_) {
    row = threadIdx.x / tpr;
    lane = threadIdx.x - row * tpr;
    warps = tpr >> 5;
    warp0 = row * warps;
  }
  // The sum of a (and of b) over the row's threads, the same bits in each of them.
  __device__ __forceinline__ void sum(float& a, float* b = nullptr) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      if (b) *b += __shfl_xor_sync(0xffffffffu, *b, o);
    }
    if (warps == 1) return;
    float* r = red + 96 * turn;
    turn ^= 1;
    const int w = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
      r[w] = a;
      if (b) r[32 + w] = *b;
    }
    __syncthreads();
    a = 0.f;
    if (b) *b = 0.f;
    for (int i = 0; i < warps; ++i) {
      a += r[warp0 + i];
      if (b) *b += r[32 + warp0 + i];
    }
  }
  // Joins (count, mean, sum of squared distances from the mean) over the row's threads.
  __device__ __forceinline__ void join(float& n, float& mean, float& m2) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      merge(n, mean, m2, __shfl_xor_sync(0xffffffffu, n, o), __shfl_xor_sync(0xffffffffu, mean, o),
            __shfl_xor_sync(0xffffffffu, m2, o));
    if (warps == 1) return;
    float* r = red + 96 * turn;
    turn ^= 1;
    const int w = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
      r[w] = n;
      r[32 + w] = mean;
      r[64 + w] = m2;
    }
    __syncthreads();
    n = mean = m2 = 0.f;
    for (int i = 0; i < warps; ++i) merge(n, mean, m2, r[warp0 + i], r[32 + warp0 + i], r[64 + warp0 + i]);
  }
  static __device__ __forceinline__ void merge(float& n, float& mean, float& m2, float n2, float mean2, float m22) {
    const float t = n + n2;
    const float f = t > 0.f ? n2 / t : 0.f;
    const float d = mean2 - mean;
    m2 += m22 + d * d * n * f;
    mean = fmaf(d, f, mean);
    n = t;
  }
};

struct Stat {
  float rstd, mean;
  template <bool LN>
  __device__ __forceinline__ void store(float* p, int64_t row) const {
    if (LN) {
      p[2 * row] = rstd;
      p[2 * row + 1] = mean;
    } else {
      p[row] = rstd;
    }
  }
  template <bool LN>
  static __device__ __forceinline__ Stat load(const float* p, int64_t row) {
    return LN ? Stat{p[2 * row], p[2 * row + 1]} : Stat{p[row], 0.f};
  }
};

// 1 / sqrt(mean square + eps), or with LN the mean and 1 / sqrt(variance + eps), of a row.
template <int VEC, int NV, bool LN>
__device__ __forceinline__ Stat row_stat(RowGroup& g, const float (&v)[NV][VEC], int cols, float eps) {
  if constexpr (!LN) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s = fmaf(v[k][e], v[k][e], s);  // zeros behind the row's end
    g.sum(s);
    return {rsqrtf(s / cols + eps), 0.f};
  } else {
    float n = 0.f, mean = 0.f, m2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if ((g.lane + k * g.tpr) * VEC < cols) {
        n += VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) mean += v[k][e];
      }
    }
    if (n > 0.f) mean /= n;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if ((g.lane + k * g.tpr) * VEC < cols) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float d = v[k][e] - mean;
          m2 = fmaf(d, d, m2);
        }
      }
    }
    g.join(n, mean, m2);
    return {rsqrtf(m2 / cols + eps), mean};
  }
}

constexpr int kMaxCols = 8192;
constexpr int kMaxThreads = 512;

// Calls go.run<T, VEC, NV, LN>(threads a row) for the widest access that divides the rows' width and
// their starts (16 bytes, else 4, else one value), with as few vectors a thread as the width allows.
template <typename T, bool LN, typename Go>
void dispatch_row_vec(const Go& go, const void* const* rows, int n, int cols) {
  constexpr int E = static_cast<int>(sizeof(T));
  auto fits = [&](int vec) {
    if (cols % vec) return false;
    for (int i = 0; i < n; ++i)
      if (reinterpret_cast<uintptr_t>(rows[i]) % (vec * E)) return false;
    return true;
  };
  auto threads = [&](int per_thread) {
    int t = 32;
    while (t * per_thread < cols) t *= 2;
    return t;
  };
  constexpr int W = 16 / E;
  constexpr int kNarrow = Go::kOneVector, kMiddle = Go::kTwoVectors;  // in threads a row
  if (fits(W)) {
    if (cols <= W * kNarrow) return go.template run<T, W, 1, LN>(threads(W));
    if constexpr (W * 2 * kMiddle < kMaxCols) {
      if (cols > W * 2 * kMiddle) return go.template run<T, W, 4, LN>(threads(4 * W));
    }
    return go.template run<T, W, 2, LN>(threads(2 * W));
  }
  if constexpr (E == 2) {
    if (fits(2)) {
      if (cols <= 2048) return go.template run<T, 2, 4, LN>(threads(8));
      return go.template run<T, 2, 8, LN>(threads(16));
    }
  }
  if (cols <= 1024) return go.template run<T, 1, 4, LN>(threads(4));
  return go.template run<T, 1, 16, LN>(threads(16));
}

template <typename Go>
void dispatch_row_kernel(const Go& go, const void* const* rows, int n, int cols, DType dtype, bool layer) {
  if (cols < 1 || cols > kMaxCols) throw std::runtime_error("mmf: block_norm: rows of 1 to 8192 values are supported");
  auto typed = [&](auto t) {
    using T = decltype(t);
    if (layer)
      dispatch_row_vec<T, true>(go, rows, n, cols);
    else
      dispatch_row_vec<T, false>(go, rows, n, cols);
  };
  if (dtype == DType::BF16)
    typed(__nv_bfloat16());
  else if (dtype == DType::F16)
    typed(__half());
  else
    typed(float());
}

}  // namespace

}  // namespace mmf
