// The norms before and after a block fused with its gate and residual scale, forward:
//
//   p = norm_post(y),  h = residual_scale x + branch_scale g p,  n = norm_pre(h)
//
// norm is RMS (v / sqrt(mean v^2 + eps) * w) or Layer ((v - mean) / sqrt(var + eps) * w + b).
//
// Bound by memory: x and y are read once, h and n written once, the row stays in registers in
// between.  A row is shared by `tpr` threads (a warp up to the whole block) that hold NV vectors
// of VEC values each; every load of the row (the weights' too) is issued before the first
// reduction.  A layer norm's mean and variance come from one reduction: each thread's own mean and
// sum of squared distances, joined pairwise (Chan, Golub, LeVeque), which does not cancel where
// the mean is large against the deviation.  n is formed from h before its rounding.
#include <stdexcept>
#include <string>

#include "block_norm.cuh"

namespace mmf {

namespace {

template <typename T, int VEC, int NV, bool LN>
__global__ void __launch_bounds__(kMaxThreads) block_norm_fwd_kernel(const BlockNormArgs a, int tpr) {
  __shared__ float red[2 * 3 * 32];
  RowGroup g(tpr, red);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / tpr) + g.row;
  const bool live = row < a.rows;
  const int cols = a.cols;
  const int64_t off = row * cols;
  const T* x = static_cast<const T*>(a.x) + off;
  const T* y = static_cast<const T*>(a.y) + off;
  const T* pw = static_cast<const T*>(a.post_w);
  const T* pb = static_cast<const T*>(a.post_b);
  const T* gate = a.gate ? static_cast<const T*>(a.gate) + (live ? row / a.rows_per_gate : 0) * cols : nullptr;
  const T* nw = static_cast<const T*>(a.pre_w);
  const T* nb = static_cast<const T*>(a.pre_b);

  using R = Raw<T, VEC>;
  R rx[NV], ry[NV], rpw[NV], rg[NV], rnw[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (g.lane + k * tpr) * VEC;
    if (live && c < cols) {
      ry[k] = ld_raw<T, VEC>(y + c);
      rx[k] = ld_raw<T, VEC>(x + c);
    }
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (g.lane + k * tpr) * VEC;
    if (live && c < cols) {
      if (pw) rpw[k] = ld_raw<T, VEC>(pw + c);
      if (gate) rg[k] = ld_raw<T, VEC>(gate + c);
      if (nw) rnw[k] = ld_raw<T, VEC>(nw + c);
    }
  }

  float v[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (g.lane + k * tpr) * VEC;
    if (live && c < cols) {
      unpack<T, VEC>(ry[k], v[k]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k][e] = 0.f;
    }
  }
  if (pw) {
    const Stat s = row_stat<VEC, NV, LN>(g, v, cols, a.eps);
    if (a.stat_y && live && g.lane == 0) s.store<LN>(a.stat_y, row);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (g.lane + k * tpr) * VEC;
      if (live && c < cols) {
        float w[VEC];
        unpack<T, VEC>(rpw[k], w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[k][e] = (v[k][e] - s.mean) * s.rstd * w[e];
        if (LN && pb) {
          unpack<T, VEC>(ld_raw<T, VEC>(pb + c), w);
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[k][e] += w[e];
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (g.lane + k * tpr) * VEC;
    if (live && c < cols) {
      float u[VEC];
      if (gate) {
        unpack<T, VEC>(rg[k], u);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[k][e] *= u[e];
      }
      unpack<T, VEC>(rx[k], u);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k][e] = fmaf(a.residual_scale, u[e], a.branch_scale * v[k][e]);
      st_raw<T, VEC>(static_cast<T*>(a.h) + off + c, pack<T, VEC>(v[k]));
    }
  }
  if (nw == nullptr) return;
  const Stat s = row_stat<VEC, NV, LN>(g, v, cols, a.eps);
  if (a.stat_h && live && g.lane == 0) s.store<LN>(a.stat_h, row);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (g.lane + k * tpr) * VEC;
    if (live && c < cols) {
      float w[VEC];
      unpack<T, VEC>(rnw[k], w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k][e] = (v[k][e] - s.mean) * s.rstd * w[e];
      if (LN && nb) {
        unpack<T, VEC>(ld_raw<T, VEC>(nb + c), w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[k][e] += w[e];
      }
      st_raw<T, VEC>(static_cast<T*>(a.n) + off + c, pack<T, VEC>(v[k]));
    }
  }
}

struct Forward {
  static constexpr int kOneVector = 128, kTwoVectors = 256;
  const BlockNormArgs& a;
  cudaStream_t stream;
  template <typename T, int VEC, int NV, bool LN>
  void run(int tpr) const {
    const int block = tpr < 128 ? 128 : tpr;  // narrow rows: several to a block
    const int64_t blocks = (a.rows + block / tpr - 1) / (block / tpr);
    if (blocks > 0x7fffffff) throw std::runtime_error("mmf: block_norm: too many rows");
    block_norm_fwd_kernel<T, VEC, NV, LN><<<static_cast<unsigned>(blocks), block, 0, stream>>>(a, tpr);
  }
};

}  // namespace

void block_norm_fwd(const BlockNormArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return;
  const void* rows[] = {a.x, a.y, a.h, a.n, a.post_w, a.post_b, a.gate, a.pre_w, a.pre_b};
  dispatch_row_kernel(Forward{a, stream}, rows, 9, a.cols, a.dtype, a.layer);
  count_launch();
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("mmf: block_norm launch failed: ") + cudaGetErrorString(e));
}

}  // namespace mmf
