// What the forward and the backward of the fused block norms share: a row spread over a group of
// threads, its reductions and statistics, and the choice of a kernel for a width.
#pragma once

#include <stdexcept>

#include "kernels.h"
#include "tc_common.cuh"
#include "typed_io.cuh"

namespace mmf {

namespace {

// `tpr` threads of the block that share one row (whole warps).  Every thread of the block takes part in
// every reduction.
struct RowGroup {
  int tpr, row, lane, warp0, warps;
  float* red;  // [2][4][32], used in turn so that one barrier a reduction is enough; 16-byte aligned
  int turn = 0;
  __device__ RowGroup(int tpr_, float* red_) : tpr(tpr_), red(red_) {
    row = threadIdx.x / tpr;
    lane = threadIdx.x - row * tpr;
    warps = tpr >> 5;
    warp0 = row * warps;
  }
  // Each of v summed over the row's threads, the same bits in each of them.
  template <int M>
  __device__ __forceinline__ void sum(float (&v)[M]) {
    static_assert(M <= 4, "");
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < M; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (warps == 1) return;
    float* r = red + 128 * turn;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < M; ++i) r[32 * i + (threadIdx.x >> 5)] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < M; ++i) v[i] = over_warps(r + 32 * i + warp0);
  }
  __device__ __forceinline__ float sum(float v) {
    float w[1] = {v};
    sum(w);
    return w[0];
  }

 private:
  __device__ __forceinline__ float over_warps(const float* r) const {
    float t = 0.f;
    if (warps % 4 == 0) {  // then every row's part of r is on a 16-byte boundary
      for (int i = 0; i < warps; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(r + i);
        t += (v.x + v.y) + (v.z + v.w);
      }
    } else {
      for (int i = 0; i < warps; ++i) t += r[i];
    }
    return t;
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

// Rows on their way into shared memory, each thread's vectors at places of its own, so that a thread has
// nothing but its own copies to wait for.
template <typename T, int VEC>
__device__ __forceinline__ void copy_ahead(Raw<T, VEC>* to, const T* from) {
  constexpr int BYTES = VEC * static_cast<int>(sizeof(T));
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  else if constexpr (BYTES == 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  else
    *to = ld_raw<T, VEC>(from);
}
// Ends a group of copies, and waits until at most `left` groups are under way.
__device__ __forceinline__ void end_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void wait_copies(int left) {
  if (left == 2)
    asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (left == 1)
    asm volatile("cp.async.wait_group 1;" ::: "memory");
  else
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// A thread's values of a row, as pairs: NV vectors of VEC, the k-th at column (lane + k tpr) VEC.
template <int N>
struct Values {
  float2 p[N / 2];
  __device__ __forceinline__ void fill(float v) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) p[i] = make_float2(v, v);
  }
  template <typename T, int VEC>
  __device__ __forceinline__ void put(int k, const Raw<T, VEC>& r) {
    float v[VEC];
    unpack<T, VEC>(r, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) at(k * VEC + e) = v[e];
  }
  template <typename T, int VEC>
  __device__ __forceinline__ Raw<T, VEC> get(int k) const {
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (k * VEC + e) % 2 ? p[(k * VEC + e) / 2].y : p[(k * VEC + e) / 2].x;
    return pack<T, VEC>(v);
  }

 private:
  __device__ __forceinline__ float& at(int i) { return i % 2 ? p[i / 2].y : p[i / 2].x; }
};
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// 1 / sqrt(mean square + eps), or with LN the mean and 1 / sqrt(variance + eps), of a row whose values
// behind its end are 0; inv = 1 / cols.  The variance is taken around the mean in a second reduction: a mean that is large
// against the deviation cancels nothing.
template <int N, int VEC, bool LN>
__device__ __forceinline__ Stat row_stat(RowGroup& g, const Values<N>& v, int cols, float inv, float eps) {
  float2 s = both(0.f);
  float mean = 0.f;
  if constexpr (LN) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) s = fadd2(s, v.p[i]);
    mean = g.sum(s.x + s.y) * inv;
    s = both(0.f);
  }
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    if constexpr (LN) {
      // the values behind the row's end are no distance from the mean; a pair is of one vector or (VEC 1) two
      const bool first = (g.lane + 2 * i / VEC * g.tpr) * VEC < cols, second = (g.lane + (2 * i + 1) / VEC * g.tpr) * VEC < cols;
      const float2 d = fadd2(v.p[i], both(-mean));
      s = ffma2(make_float2(first ? d.x : 0.f, second ? d.y : 0.f), d, s);
    } else {
      s = ffma2(v.p[i], v.p[i], s);
    }
  }
  return {rsqrtf(fmaf(g.sum(s.x + s.y), inv, eps)), mean};
}

constexpr int kMaxCols = 8192;
constexpr int kMaxThreads = 512;

// The columns of each of the blocks that share a row (the last has what is left).
__host__ __device__ __forceinline__ int share_of(int cols, int blocks, int vec) {
  return (cols + blocks * vec - 1) / (blocks * vec) * vec;
}

// Calls go.run<T, VEC, NV, LN>(threads a row) for the widest access that divides the rows' width and
// their starts (16 bytes, else 4, else one value), with Go::kValues values a thread (VEC at least); where
// kMaxThreads threads are too few for that, go.run<T, VEC, NV, LN, B>(threads of a block's share) with B
// blocks a row, 2 or 4.
template <typename T, bool LN, int VEC, typename Go>
void dispatch_row_width(const Go& go, int cols) {
  constexpr int NV = Go::kValues > VEC ? Go::kValues / VEC : 1;
  auto threads = [&](int n) { return ((n + NV * VEC - 1) / (NV * VEC) + 31) / 32 * 32; };
  constexpr int most = kMaxThreads * NV * VEC;
  if (cols <= most) return go.template run<T, VEC, NV, LN>(threads(cols));
  if constexpr (most < kMaxCols) {
    if (Go::four_blocks(cols)) return go.template run<T, VEC, NV, LN, 4>(threads(share_of(cols, 4, VEC)));
    go.template run<T, VEC, NV, LN, 2>(threads(share_of(cols, 2, VEC)));
  }
}
template <typename T, bool LN, typename Go>
void dispatch_row_vec(const Go& go, const void* const* rows, int n, int cols) {
  constexpr int E = static_cast<int>(sizeof(T));
  auto fits = [&](int vec) {
    if (cols % vec) return false;
    for (int i = 0; i < n; ++i)
      if (reinterpret_cast<uintptr_t>(rows[i]) % (vec * E)) return false;
    return true;
  };
  if (fits(16 / E)) return dispatch_row_width<T, LN, 16 / E>(go, cols);
  if constexpr (E == 2) {
    if (fits(2)) return dispatch_row_width<T, LN, 2>(go, cols);
  }
  dispatch_row_width<T, LN, 1>(go, cols);
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
