// The backward of the fused block norms (block_norm.cu):
//
//   a  = dn w_pre,  dH = dh + r_h (a - h^ mean(a h^) [- mean(a)]),  dx = residual_scale dH
//   dp = branch_scale gate dH,  b = dp w_post,  dy = r_y (b - y^ mean(b y^) [- mean(b)])
//   dw_pre = sum dn h^, db_pre = sum dn, dw_post = sum dp y^, db_post = sum dp,
//   dgate = branch_scale sum dH p over the rows that share the gate
//
// with h^, y^ the normalised rows (recomputed from h, y and the forward's statistics) and the means
// in [] for layer norms alone.
//
// Bound by memory: dh, dn, h and y are read once, dx and dy written once.  A worker (a group of
// threads that shares a row) walks over a run of rows; its sums over rows stay in shared memory,
// each thread's columns its own, and leave once, as one partial row a worker (one a run for the
// gate).  A second kernel adds the partials in a fixed order, so that equal calls give equal bits.
#include <algorithm>
#include <stdexcept>
#include <string>

#include "block_norm.cuh"

namespace mmf {

namespace {

// Rows are dealt out in chunks of `chunk_rows` that do not cross a gate's group of rows.
struct Plan {
  int64_t groups, group_rows;  // rows that share a gate (one group where no sum over rows is asked)
  int64_t per_group, chunk_rows, chunks;
};

struct BwdParts {
  float *post_w, *post_b, *pre_w, *pre_b;  // [workers][cols] each, or null
  float* gate;                              // [chunks][cols], or null
};

template <typename T, int VEC>
__device__ __forceinline__ void load_or_zero(const T* p, float* v) {
  if (p) {
    unpack<T, VEC>(ld_raw<T, VEC>(p), v);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = 0.f;
  }
}

// The columns' sums of one thread, in shared memory: array i's vector k of thread `lane`.  Vectors
// of 8 are split into two of 4 so that a warp's accesses cover whole lines of banks.
template <int VEC, int NV>
struct Sums {
  static constexpr int P = VEC < 4 ? VEC : 4;  // values an access
  float* base;
  int tpr, lane;
  __device__ __forceinline__ float* at(int i, int k, int part) const {
    return base + (((i * NV + k) * (VEC / P) + part) * tpr + lane) * P;
  }
  __device__ __forceinline__ void add(int i, int k, const float* v) const {
#pragma unroll
    for (int q = 0; q < VEC / P; ++q) {
      float* s = at(i, k, q);
      float t[P];
      *reinterpret_cast<Raw<float, P>*>(t) = *reinterpret_cast<const Raw<float, P>*>(s);
#pragma unroll
      for (int e = 0; e < P; ++e) t[e] += v[q * P + e];
      *reinterpret_cast<Raw<float, P>*>(s) = *reinterpret_cast<const Raw<float, P>*>(t);
    }
  }
  __device__ __forceinline__ void zero(int i, int cols) const {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int q = 0; q < VEC / P; ++q)
#pragma unroll
        for (int e = 0; e < P; ++e) at(i, k, q)[e] = 0.f;
  }
  __device__ __forceinline__ void flush(int i, float* dst, int cols) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (lane + k * tpr) * VEC;
      if (c < cols) {
#pragma unroll
        for (int q = 0; q < VEC / P; ++q)
          *reinterpret_cast<Raw<float, P>*>(dst + c + q * P) = *reinterpret_cast<const Raw<float, P>*>(at(i, k, q));
      }
    }
  }
};

enum { S_POST_W, S_PRE_W, S_GATE, S_POST_B, S_PRE_B };

template <typename T, int VEC, int NV, bool LN>
__global__ void __launch_bounds__(kMaxThreads) block_norm_bwd_kernel(const BlockNormBwdArgs a, const Plan plan,
                                                                     const BwdParts parts, int tpr) {
  extern __shared__ __align__(16) float smem[];
  __shared__ float red[2 * 3 * 32];
  RowGroup g(tpr, red);
  const int cols = a.cols;
  const int groups = blockDim.x / tpr;
  const int64_t worker = static_cast<int64_t>(blockIdx.x) * groups + g.row;
  const int64_t workers = static_cast<int64_t>(gridDim.x) * groups;
  const Sums<VEC, NV> sums{smem + static_cast<int64_t>(g.row) * (LN ? 5 : 3) * NV * VEC * tpr, tpr, g.lane};
#pragma unroll
  for (int i = 0; i < (LN ? 5 : 3); ++i) sums.zero(i, cols);

  const T* pw = static_cast<const T*>(a.post_w);
  const T* pb = static_cast<const T*>(a.post_b);
  const T* nw = static_cast<const T*>(a.pre_w);
  const T* gate0 = static_cast<const T*>(a.gate);
  const float inv = 1.f / cols;
  const int64_t rounds = (plan.chunks + workers - 1) / workers;
  for (int64_t round = 0; round < rounds; ++round) {
    const int64_t chunk = round * workers + worker;
    const int64_t group = chunk / plan.per_group;
    const int64_t r0 = (chunk - group * plan.per_group) * plan.chunk_rows;  // within the group
    for (int64_t i = 0; i < plan.chunk_rows; ++i) {  // the same count for every worker of the block
      const bool live = chunk < plan.chunks && r0 + i < plan.group_rows;
      const int64_t row = live ? group * plan.group_rows + r0 + i : 0;
      const int64_t off = row * cols;
      const T* gate = gate0 ? gate0 + row / a.rows_per_gate * cols : nullptr;
      const Stat sh = (live && nw) ? Stat::load<LN>(a.stat_h, row) : Stat{0.f, 0.f};
      const Stat sy = (live && pw) ? Stat::load<LN>(a.stat_y, row) : Stat{0.f, 0.f};
      using R = Raw<T, VEC>;
      R rn[NV], rh[NV], ry[NV];
      float d[NV][VEC];  // dH
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (g.lane + k * tpr) * VEC;
        if (live && c < cols) {
          if (nw) {
            rn[k] = ld_raw<T, VEC>(static_cast<const T*>(a.dn) + off + c);
            rh[k] = ld_raw<T, VEC>(static_cast<const T*>(a.h) + off + c);
          }
          if (pw || gate) ry[k] = ld_raw<T, VEC>(static_cast<const T*>(a.y) + off + c);
          load_or_zero<T, VEC>(a.dh ? static_cast<const T*>(a.dh) + off + c : nullptr, d[k]);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[k][e] = 0.f;
        }
      }
      if (nw) {
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int c = (g.lane + k * tpr) * VEC;
          if (live && c < cols) {
            float w[VEC], n[VEC], h[VEC], t[VEC];
            unpack<T, VEC>(ld_raw<T, VEC>(nw + c), w);
            unpack<T, VEC>(rn[k], n);
            unpack<T, VEC>(rh[k], h);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float u = (h[e] - sh.mean) * sh.rstd;
              t[e] = n[e] * u;
              s1 = fmaf(n[e], w[e], s1);
              s2 = fmaf(t[e], w[e], s2);
            }
            if (parts.pre_w) sums.add(S_PRE_W, k, t);
            if (LN && parts.pre_b) sums.add(S_PRE_B, k, n);
          }
        }
        g.sum(s2, LN ? &s1 : nullptr);
        s1 *= inv;
        s2 *= inv;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int c = (g.lane + k * tpr) * VEC;
          if (live && c < cols) {
            float w[VEC], n[VEC], h[VEC];
            unpack<T, VEC>(ld_raw<T, VEC>(nw + c), w);
            unpack<T, VEC>(rn[k], n);
            unpack<T, VEC>(rh[k], h);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float u = (h[e] - sh.mean) * sh.rstd;
              d[k][e] += sh.rstd * (n[e] * w[e] - u * s2 - (LN ? s1 : 0.f));
            }
          }
        }
      }
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (g.lane + k * tpr) * VEC;
        if (live && c < cols) {
          float t[VEC], u[VEC], w[VEC], gt[VEC];
          if (a.dx) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) t[e] = a.residual_scale * d[k][e];
            st_raw<T, VEC>(static_cast<T*>(a.dx) + off + c, pack<T, VEC>(t));
          }
          if (pw || gate) unpack<T, VEC>(ry[k], u);
          if (gate) unpack<T, VEC>(ld_raw<T, VEC>(gate + c), gt);
          if (pw) unpack<T, VEC>(ld_raw<T, VEC>(pw + c), w);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            d[k][e] *= a.branch_scale;
            if (pw) u[e] = (u[e] - sy.mean) * sy.rstd;
          }
          if (gate && a.dgate) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) t[e] = pw ? u[e] * w[e] : u[e];
            if (LN && pb) {
              float bb[VEC];
              unpack<T, VEC>(ld_raw<T, VEC>(pb + c), bb);
#pragma unroll
              for (int e = 0; e < VEC; ++e) t[e] += bb[e];
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) t[e] *= d[k][e];
            if (parts.gate)
              sums.add(S_GATE, k, t);
            else
              st_raw<T, VEC>(static_cast<T*>(a.dgate) + off + c, pack<T, VEC>(t));
          }
          if (gate) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[k][e] *= gt[e];
          }
          if (pw) {
            if (LN && parts.post_b) sums.add(S_POST_B, k, d[k]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) t[e] = d[k][e] * u[e];
            if (parts.post_w) sums.add(S_POST_W, k, t);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              d[k][e] *= w[e];
              s1 += d[k][e];
              s2 = fmaf(t[e], w[e], s2);
            }
          }
        }
      }
      if (pw) {
        g.sum(s2, LN ? &s1 : nullptr);
        s1 *= inv;
        s2 *= inv;
      }
      if (a.dy) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int c = (g.lane + k * tpr) * VEC;
          if (live && c < cols) {
            if (pw) {
              float u[VEC];
              unpack<T, VEC>(ry[k], u);
#pragma unroll
              for (int e = 0; e < VEC; ++e)
                d[k][e] = sy.rstd * (d[k][e] - (u[e] - sy.mean) * sy.rstd * s2 - (LN ? s1 : 0.f));
            }
            st_raw<T, VEC>(static_cast<T*>(a.dy) + off + c, pack<T, VEC>(d[k]));
          }
        }
      }
    }
    if (parts.gate && chunk < plan.chunks) {
      sums.flush(S_GATE, parts.gate + chunk * cols, cols);
      sums.zero(S_GATE, cols);
    }
  }
  const int64_t at = worker * cols;
  if (parts.post_w) sums.flush(S_POST_W, parts.post_w + at, cols);
  if (parts.pre_w) sums.flush(S_PRE_W, parts.pre_w + at, cols);
  if (LN && parts.post_b) sums.flush(S_POST_B, parts.post_b + at, cols);
  if (LN && parts.pre_b) sums.flush(S_PRE_B, parts.pre_b + at, cols);
}

// out[g][c] = sum over i of part[g * n + i][c], in the order of i within each of 8 lanes, then of the
// lanes.  blockIdx.y: which array and group.
struct SumJob {
  const float* part;
  void* out;
  int64_t n;
};
struct SumJobs {
  SumJob job[4];
  SumJob gate;
  int count;
};

template <typename T>
__global__ void __launch_bounds__(256) block_norm_sum_kernel(const SumJobs jobs, int cols) {
  __shared__ float s[8][33];
  SumJob j;
  int64_t group = 0;
  if (static_cast<int>(blockIdx.y) < jobs.count) {
    j = jobs.job[blockIdx.y];
  } else {
    j = jobs.gate;
    group = blockIdx.y - jobs.count;
  }
  const int c = blockIdx.x * 32 + threadIdx.x;
  float t = 0.f;
  if (c < cols) {
    const float* p = j.part + group * j.n * cols + c;
#pragma unroll 4
    for (int64_t i = threadIdx.y; i < j.n; i += 8) t += p[i * cols];
  }
  s[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) t += s[i][threadIdx.x];
    static_cast<T*>(j.out)[group * cols + c] = from_f32<T>(t);
  }
}

// The launch of a width: what it needs of the device, and how rows are dealt out.
struct Backward {
  static constexpr int kOneVector = 128, kTwoVectors = 512;
  const BlockNormBwdArgs& a;
  cudaStream_t stream;
  int64_t* need;  // non-null: only count the scratch values

  template <typename T, int VEC, int NV, bool LN>
  void run(int tpr) const {
    auto kernel = block_norm_bwd_kernel<T, VEC, NV, LN>;
    const int block = tpr < 128 ? 128 : tpr;
    const int groups = block / tpr;
    const int smem = (LN ? 5 : 3) * NV * VEC * tpr * groups * static_cast<int>(sizeof(float));
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    int per_sm = 0;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, block, smem);
    if (e != cudaSuccess || per_sm < 1)
      throw std::runtime_error(std::string("mmf: block_norm_bwd: ") + cudaGetErrorString(e));
    const int64_t most = 148LL * per_sm * groups;  // workers on the device at once
    Plan p;
    const bool gate_sum = a.dgate && a.rows_per_gate > 1;
    p.groups = gate_sum ? a.rows / a.rows_per_gate : 1;
    p.group_rows = gate_sum ? a.rows_per_gate : a.rows;
    // one chunk a worker while the groups are few; with many groups several smaller ones, so that
    // the last round is not mostly idle
    p.per_group = p.groups * 4 <= most ? most / p.groups : (4 * most + p.groups - 1) / p.groups;
    p.per_group = std::min(p.per_group, p.group_rows);
    p.chunk_rows = (p.group_rows + p.per_group - 1) / p.per_group;
    p.per_group = (p.group_rows + p.chunk_rows - 1) / p.chunk_rows;
    p.chunks = p.groups * p.per_group;
    const int64_t workers = std::min(most, (p.chunks + groups - 1) / groups * groups);

    int64_t used = 0;
    auto take = [&](bool want, int64_t rows) {
      float* at = want && !need ? a.parts + used : nullptr;
      if (want) used += rows * a.cols;
      return at;
    };
    BwdParts parts;
    parts.post_w = take(a.dpost_w, workers);
    parts.pre_w = take(a.dpre_w, workers);
    parts.post_b = take(a.dpost_b, workers);
    parts.pre_b = take(a.dpre_b, workers);
    parts.gate = take(gate_sum, p.chunks);
    if (need) {
      *need = used;
      return;
    }
    kernel<<<static_cast<unsigned>(workers / groups), block, smem, stream>>>(a, p, parts, tpr);
    check("block_norm_bwd");

    SumJobs jobs{};
    auto add = [&](const float* part, void* out) {
      if (part) jobs.job[jobs.count++] = {part, out, workers};
    };
    add(parts.post_w, a.dpost_w);
    add(parts.pre_w, a.dpre_w);
    add(parts.post_b, a.dpost_b);
    add(parts.pre_b, a.dpre_b);
    jobs.gate = {parts.gate, a.dgate, p.per_group};
    // grid.y: the arrays, then the gate's groups; past its limit the gate goes on in more launches
    int64_t gates = gate_sum ? p.groups : 0;
    if (jobs.count + gates == 0) return;
    const dim3 threads(32, 8);
    while (true) {
      const int64_t now = std::min<int64_t>(gates, 32768);
      block_norm_sum_kernel<T>
          <<<dim3((a.cols + 31) / 32, static_cast<unsigned>(jobs.count + now)), threads, 0, stream>>>(jobs, a.cols);
      check("block_norm_bwd (sums)");
      gates -= now;
      if (gates == 0) return;
      jobs.count = 0;
      jobs.gate.part += now * p.per_group * a.cols;
      jobs.gate.out = static_cast<T*>(jobs.gate.out) + now * a.cols;
    }
  }
  static void check(const char* what) {
    count_launch();
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess)
      throw std::runtime_error(std::string("mmf: ") + what + " launch failed: " + cudaGetErrorString(e));
  }
};

void go(const Backward& b) {
  const BlockNormBwdArgs& a = b.a;
  const void* rows[] = {a.dh, a.dn, a.h, a.y, a.post_w, a.post_b, a.gate, a.pre_w, a.dx, a.dy, a.dgate};
  dispatch_row_kernel(b, rows, 11, a.cols, a.dtype, a.layer);
}

}  // namespace

int64_t block_norm_bwd_parts(const BlockNormBwdArgs& a) {
  int64_t need = 0;
  if (a.rows > 0) go(Backward{a, nullptr, &need});
  return need;
}

void block_norm_bwd(const BlockNormBwdArgs& a, cudaStream_t stream) {
  if (a.rows > 0) go(Backward{a, stream, nullptr});
}

}  // namespace mmf
