// The norms before and after a block fused with its gate and residual scale, forward:
//
//   p = norm_post(y),  h = residual_scale x + branch_scale g p,  n = norm_pre(h)
//
// norm is RMS (v / sqrt(mean v^2 + eps) * w) or Layer ((v - mean) / sqrt(var + eps) * w + b).
//
// Bound by memory: x and y are read once, h and n written once, the row stays in registers in
// between.  Blocks stay for many rows: the weights stay in registers (they are as many bytes as a row's x
// and y, and came from the second-level cache row by row before), and the next rows' x and y (and gates,
// where each row has its own) are copied ahead into shared memory.  A row is shared by few threads, 16
// values each: fewer take part in its reductions (8192 x 4096 bf16: 59 us, 69 with 8 values a thread; a
// block for each row 64).  A layer norm's variance is taken around its mean, in a reduction of its own.
// n is formed from h before its rounding.
#include <stdexcept>
#include <string>

#include "block_norm.cuh"
#include "launch_info.h"

namespace mmf {

namespace {

enum { IN_Y, IN_X, IN_GATE, INPUTS };

template <typename T, int VEC, int NV, bool LN>
__global__ void __launch_bounds__(kMaxThreads) block_norm_fwd_kernel(const BlockNormArgs a, int tpr, int inputs,
                                                                     int stages) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(16) float red[2 * 4 * 32];
  using R = Raw<T, VEC>;
  RowGroup g(tpr, red);
  const int cols = a.cols, threads = static_cast<int>(blockDim.x), groups = threads / tpr;
  const bool pw = a.post_w != nullptr, nw = a.pre_w != nullptr;
  const T* in[INPUTS] = {static_cast<const T*>(a.y), static_cast<const T*>(a.x), static_cast<const T*>(a.gate)};
  auto col = [&](int k) { return (g.lane + k * tpr) * VEC; };
  // stage s's vector k of input i is place(s)[(i * NV + k) * threads]
  auto place = [&](int stage) { return reinterpret_cast<R*>(smem) + threadIdx.x + stage * (inputs * NV) * threads; };
  const int rows = static_cast<int>(a.rows), rows_per_gate = static_cast<int>(a.rows_per_gate);
  const int first = static_cast<int>(blockIdx.x) * groups + g.row, step = static_cast<int>(gridDim.x) * groups;
  const int turns = (rows - static_cast<int>(blockIdx.x) * groups + step - 1) / step;  // the block's
  const float inv = 1.f / cols;
  int put = 0, get = 0;  // stages
  int64_t ahead = first;
  auto copy = [&]() {
    if (ahead < rows) {
      const int64_t off = ahead * cols + g.lane * VEC;
      R* to = place(put);
#pragma unroll
      for (int i = 0; i < INPUTS; ++i) {
        if (i < inputs) {
#pragma unroll
          for (int k = 0; k < NV; ++k)
            if (col(k) < cols) copy_ahead<T, VEC>(to + (i * NV + k) * threads, in[i] + off + k * tpr * VEC);
        }
      }
    }
    ahead += step;
    if (++put == stages) put = 0;
    end_copies();  // one group a turn, empty or not
  };
  for (int i = 0; i < stages - 1; ++i) copy();
  // the weights stay in registers, as they came; the gate for as long as rows share it
  auto columns = [&](const void* p, R (&r)[NV]) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (p && col(k) < cols) r[k] = ld_raw<T, VEC>(static_cast<const T*>(p) + col(k));
  };
  R post[NV], post_b[NV], pre[NV], pre_b[NV], gate[NV];
  columns(a.post_w, post);
  columns(a.pre_w, pre);
  if (LN) {
    columns(a.post_b, post_b);
    columns(a.pre_b, pre_b);
  }
  int gate_at = -1;
  for (int turn = 0; turn < turns; ++turn) {
    copy();
    wait_copies(stages - 1);
    const int64_t row = first + static_cast<int64_t>(turn) * step, off = row * cols;
    const bool live = row < rows;
    const R* here = place(get);
    if (++get == stages) get = 0;
    auto input = [&](int i, int k, float (&v)[VEC]) { unpack<T, VEC>(here[(i * NV + k) * threads], v); };
    if (a.gate && inputs < INPUTS) {
      const int its = live && rows_per_gate < rows ? static_cast<int>(row) / rows_per_gate : 0;
      if (its != gate_at) {
        gate_at = its;
        columns(in[IN_GATE] + static_cast<int64_t>(its) * cols, gate);
      }
    }
    float v[NV][VEC];
    auto normalise = [&](const Stat& s, const R (&weight)[NV], const R (&bias)[NV], bool biased) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (col(k) < cols) {
          float w[VEC];
          unpack<T, VEC>(weight[k], w);
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[k][e] = (LN ? v[k][e] - s.mean : v[k][e]) * s.rstd * w[e];
          if (LN && biased) {
            unpack<T, VEC>(bias[k], w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[k][e] += w[e];
          }
        }
      }
    };
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (live && col(k) < cols) {
        input(IN_Y, k, v[k]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[k][e] = 0.f;
      }
    }
    if (pw) {
      const Stat s = row_stat<VEC, NV, LN>(g, v, cols, inv, a.eps);
      if (a.stat_y && live && g.lane == 0) s.store<LN>(a.stat_y, row);
      normalise(s, post, post_b, a.post_b != nullptr);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (live && col(k) < cols) {
        float u[VEC];
        if (a.gate) {
          if (inputs < INPUTS)
            unpack<T, VEC>(gate[k], u);
          else
            input(IN_GATE, k, u);
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[k][e] *= u[e];
        }
        input(IN_X, k, u);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[k][e] = fmaf(a.residual_scale, u[e], a.branch_scale * v[k][e]);
        st_raw<T, VEC>(static_cast<T*>(a.h) + off + col(k), pack<T, VEC>(v[k]));
      }
    }
    if (nw) {
      const Stat s = row_stat<VEC, NV, LN>(g, v, cols, inv, a.eps);
      if (a.stat_h && live && g.lane == 0) s.store<LN>(a.stat_h, row);
      normalise(s, pre, pre_b, a.pre_b != nullptr);
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (live && col(k) < cols) st_raw<T, VEC>(static_cast<T*>(a.n) + off + col(k), pack<T, VEC>(v[k]));
    }
  }
}

struct Forward {
  static constexpr int kValues = 16;  // a thread, while the row needs no more than kMaxThreads
  const BlockNormArgs& a;
  cudaStream_t stream;
  template <typename T, int VEC, int NV, bool LN>
  void run(int tpr) const {
    auto kernel = block_norm_fwd_kernel<T, VEC, NV, LN>;
    const int block = tpr < 128 ? 128 : tpr, groups = block / tpr;  // narrow rows: several to a block
    const int inputs = a.gate && a.rows_per_gate == 1 ? INPUTS : INPUTS - 1;
    // two rows ahead where four blocks an SM can have that, one where two can
    const int stage = inputs * NV * VEC * static_cast<int>(sizeof(T)) * block;
    const int stages = 3 * stage <= (56 << 10) ? 3 : 2 * stage <= (112 << 10) ? 2 : 1;
    const int smem = stages * stage;
    const int64_t want = (a.rows + groups - 1) / groups;
    const int per_sm = resident_blocks(reinterpret_cast<const void*>(kernel), block, smem);
    const unsigned blocks = static_cast<unsigned>(want < 148LL * per_sm ? want : 148LL * per_sm);
    kernel<<<blocks, block, smem, stream>>>(a, tpr, inputs, stages);
  }
};

}  // namespace

void block_norm_fwd(const BlockNormArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return;
  if (a.rows > 0x3fffffff) throw std::runtime_error("mmf: block_norm: too many rows");
  const void* rows[] = {a.x, a.y, a.h, a.n, a.post_w, a.post_b, a.gate, a.pre_w, a.pre_b};
  dispatch_row_kernel(Forward{a, stream}, rows, 9, a.cols, a.dtype, a.layer);
  count_launch();
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("mmf: block_norm launch failed: ") + cudaGetErrorString(e));
}

}  // namespace mmf
