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
// values each: fewer take part in its reductions.  8192 x 4096 bf16 with both norms and a gate: 51 us
// (268 MB, 80 % of the copy rate); 59 with unpacked arithmetic, 69 with 8 values a thread, 64 with a block
// for each row.  A layer norm's variance is taken around its mean, in a reduction of its own.  n is formed
// from h before its rounding.
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
  constexpr int N = NV * VEC, H = N / 2;
  using R = Raw<T, VEC>;
  using V = Values<N>;
  RowGroup g(tpr, red);
  const int cols = a.cols, threads = static_cast<int>(blockDim.x), groups = threads / tpr;
  const bool pw = a.post_w != nullptr, nw = a.pre_w != nullptr;
  auto col = [&](int k) { return (g.lane + k * tpr) * VEC; };
  // stage s's vector k of input i is place(s)[(i * NV + k) * threads]; what is not copied there is 0
  auto place = [&](int stage) { return reinterpret_cast<R*>(smem) + threadIdx.x + stage * (inputs * NV) * threads; };
  const int rows = static_cast<int>(a.rows), rows_per_gate = static_cast<int>(a.rows_per_gate);
  const int first = static_cast<int>(blockIdx.x) * groups + g.row, step = static_cast<int>(gridDim.x) * groups;
  const int turns = (rows - static_cast<int>(blockIdx.x) * groups + step - 1) / step;  // the block's
  const float inv = 1.f / cols;
  auto clear = [&](int stage) {
    for (int i = 0; i < inputs * NV; ++i) place(stage)[i * threads] = R{};
  };
  for (int i = 0; i < stages; ++i) clear(i);
  int put = 0, get = 0;  // stages
  int64_t ahead = first;
  auto copy = [&]() {
    if (ahead < rows) {
      const int64_t off = ahead * cols + g.lane * VEC;
      R* to = place(put);
      auto fetch = [&](int i, const void* from) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
          if (col(k) < cols)
            copy_ahead<T, VEC>(to + (i * NV + k) * threads, static_cast<const T*>(from) + off + k * tpr * VEC);
      };
      fetch(IN_Y, a.y);
      fetch(IN_X, a.x);
      if (inputs == INPUTS) fetch(IN_GATE, a.gate);
    } else {
      clear(put);
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
      r[k] = p && col(k) < cols ? ld_raw<T, VEC>(static_cast<const T*>(p) + col(k)) : R{};
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
    auto widen = [&](const R (&r)[NV], V& v) {
#pragma unroll
      for (int k = 0; k < NV; ++k) v.template put<T, VEC>(k, r[k]);
    };
    auto input = [&](int i, V& v) {  // 0 behind the row's end (and for no row)
#pragma unroll
      for (int k = 0; k < NV; ++k) v.template put<T, VEC>(k, here[(i * NV + k) * threads]);
    };
    auto store = [&](void* to, const V& v) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (live && col(k) < cols) st_raw<T, VEC>(static_cast<T*>(to) + off + col(k), v.template get<T, VEC>(k));
    };
    if (a.gate && inputs < INPUTS) {
      const int its = live && rows_per_gate < rows ? static_cast<int>(row) / rows_per_gate : 0;
      if (its != gate_at) {
        gate_at = its;
        columns(static_cast<const T*>(a.gate) + static_cast<int64_t>(its) * cols, gate);
      }
    }
    V v, w;
    auto normalise = [&](const Stat& s, const R (&weight)[NV], const R (&bias)[NV], bool biased) {
      widen(weight, w);
      const float2 r = both(s.rstd), m = both(-s.mean * s.rstd);
#pragma unroll
      for (int i = 0; i < H; ++i) v.p[i] = fmul2(LN ? ffma2(v.p[i], r, m) : fmul2(v.p[i], r), w.p[i]);
      if (LN && biased) {
        widen(bias, w);
#pragma unroll
        for (int i = 0; i < H; ++i) v.p[i] = fadd2(v.p[i], w.p[i]);
      }
    };
    input(IN_Y, v);
    if (pw) {
      const Stat s = row_stat<N, VEC, LN>(g, v, cols, inv, a.eps);
      if (a.stat_y && live && g.lane == 0) s.store<LN>(a.stat_y, row);
      normalise(s, post, post_b, a.post_b != nullptr);
    }
    if (a.gate) {
      if (inputs < INPUTS)
        widen(gate, w);
      else
        input(IN_GATE, w);
#pragma unroll
      for (int i = 0; i < H; ++i) v.p[i] = fmul2(v.p[i], w.p[i]);
    }
    input(IN_X, w);
#pragma unroll
    for (int i = 0; i < H; ++i) v.p[i] = ffma2(both(a.residual_scale), w.p[i], fmul2(both(a.branch_scale), v.p[i]));
    store(a.h, v);
    if (nw) {
      const Stat s = row_stat<N, VEC, LN>(g, v, cols, inv, a.eps);
      if (a.stat_h && live && g.lane == 0) s.store<LN>(a.stat_h, row);
      normalise(s, pre, pre_b, a.pre_b != nullptr);
      store(a.n, v);
    }
  }
}

struct Forward {
  static constexpr int kValues = 16;  // a thread: kMaxThreads take the widest row
  const BlockNormArgs& a;
  cudaStream_t stream;
  template <typename T, int VEC, int NV, bool LN>
  void run(int tpr) const {
    auto kernel = block_norm_fwd_kernel<T, VEC, NV, LN>;
    const int groups = tpr < 128 ? 128 / tpr : 1, block = groups * tpr;  // narrow rows: several to a block
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
