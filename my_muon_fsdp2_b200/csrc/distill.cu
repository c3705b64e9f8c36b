// Distillation from a teacher's top logits (kernels.h has the formulas), loss and gradient of one
// row of logits after another:
//
//   dz_v = alpha tau wk (q_tau(v) - sum over slots j with id_j = v of p_j)
//          + (1 - alpha) wc (q_1(v) - [v = target]),      q_t = softmax(z / t)
//
// Bound by memory: the logits are read once and, with the gradient, written once.  A row is spread
// over a cluster of blocks, each holding its slice in shared memory (a 128256 wide bf16 row has 250
// KB, one block's shared memory 227): one asynchronous copy in, the maximum and the sums over the
// slice, one exchange of (maximum, sums) through distributed shared memory, and the gradient
// straight out of the slice.  Several blocks an SM overlap one another's copies and arithmetic.
//
// The maximum is joined first within a thread, then sums are scaled to the common maximum as they
// are joined, so nothing overflows.  exp(z - max) is exp2((z - max) log2 e): the difference is taken
// before the product, which keeps its rounding relative to the distance from the maximum.
#include <cooperative_groups.h>

#include <algorithm>
#include <stdexcept>
#include <string>
#include <type_traits>
#include <utility>

#include "kernels.h"
#include "tc_common.cuh"
#include "typed_io.cuh"

namespace mmf {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 1024;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float teacher_value(const DistillArgs& a, int64_t i) {
  if (a.teacher_dtype == DType::F32) return static_cast<const float*>(a.teacher)[i];
  if (a.teacher_dtype == DType::BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(a.teacher)[i]);
  return __half2float(static_cast<const __half*>(a.teacher)[i]);
}
__device__ __forceinline__ int64_t slot_id(const DistillArgs& a, int64_t i) {
  return a.ids_32 ? static_cast<const int*>(a.ids)[i] : static_cast<const int64_t*>(a.ids)[i];
}
// The slot's id, or -1 for an empty slot; an id behind the vocabulary is empty and recorded.
__device__ __forceinline__ int valid_id(const DistillArgs& a, int64_t i, int* err) {
  const int64_t id = slot_id(a, i);
  if (id >= a.vocab) {
    atomicCAS(err, 0, ERR_BAD_ARGUMENT);
    return -1;
  }
  return id < 0 ? -1 : static_cast<int>(id);
}
// The row's target, or -1 where it is ignored; one outside the vocabulary is ignored and recorded.
__device__ __forceinline__ int valid_target(const DistillArgs& a, int64_t row, int* err) {
  if (a.targets == nullptr) return -1;
  const int64_t y = a.targets[row];
  if (y == a.ignore_index) return -1;
  if (y < 0 || y >= a.vocab) {
    atomicCAS(err, 0, ERR_BAD_ARGUMENT);
    return -1;
  }
  return static_cast<int>(y);
}

// max with the sums at tau (s) and at 1 (h), as joined over any two disjoint parts of a row
struct Part {
  float m, s, h;
};
__device__ __forceinline__ Part join(const Part& a, const Part& b, float c_tau) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s, a.h + b.h};  // nothing but -inf (or NaN, which the sums carry)
  const float da = a.m - m, db = b.m - m;
  return {m, a.s * ex2(da * c_tau) + b.s * ex2(db * c_tau), a.h * ex2(da * kLog2e) + b.h * ex2(db * kLog2e)};
}

// Rows of one tensor start anywhere on the type's own boundary: a row is a head of up to 7 values, a
// body of 16-byte vectors and a tail.
template <typename T>
struct RowSplit {
  static constexpr int V = 16 / static_cast<int>(sizeof(T));
  int head, vecs, tail;
  __device__ RowSplit(const T* p, int vocab) {
    head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(T));
    head = min(head, vocab);
    vecs = (vocab - head) / V;
    tail = vocab - head - vecs * V;
  }
};

// The teacher's distribution over a row's slots, in shared memory: p and id (-1: empty).
struct TeacherRow {
  float* p;
  int* id;
};
__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < kWarps; ++i) v = fmaxf(v, red[i]);
  return v;
}
__device__ __forceinline__ float block_add(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < kWarps; ++i) v += red[i];
  return v;
}
// Fills t; returns whether the row has a slot.  All threads of the block call it.
__device__ __forceinline__ bool teacher_row(const DistillArgs& a, int64_t row, const TeacherRow& t, float* red,
                                            int* err) {
  const float c = kLog2e / a.tau;
  float best = -INFINITY;
  int any = 0;
  for (int j = threadIdx.x; j < a.top; j += kThreads) {
    const int64_t i = row * a.top + j;
    int id = valid_id(a, i, err);
    const float v = id >= 0 ? teacher_value(a, i) : -INFINITY;
    if (v == -INFINITY) id = -1;
    t.id[j] = id;
    t.p[j] = v;
    best = fmaxf(best, v);
    any |= id >= 0;
  }
  any = __syncthreads_or(any);
  if (!any) return false;
  best = block_max(best, red);
  float s = 0.f;
  for (int j = threadIdx.x; j < a.top; j += kThreads) s += t.id[j] >= 0 ? ex2((t.p[j] - best) * c) : 0.f;
  const float inv = 1.f / block_add(s, red);
  for (int j = threadIdx.x; j < a.top; j += kThreads) t.p[j] = t.id[j] >= 0 ? ex2((t.p[j] - best) * c) * inv : 0.f;
  __syncthreads();
  return true;
}

// One row's softmaxes and its gradient.  dense(z) = k_a q_a(z) + k_b q_b(z), where a is the softmax
// at `c_a` / log2 e and b, when both temperatures are wanted, the one at 1; the slots take
// sub_p * p_j off, the target sub_y.
struct RowGrad {
  bool soft, hard;  // whether the row has a slot / a target that counts
  float m, c_a, l_a, l_b, k_a, k_b, sub_p, sub_y;

  __device__ __forceinline__ RowGrad(const DistillArgs& a, bool has_slot, bool has_target)
      : soft(has_slot && a.alpha > 0.f), hard(has_target && a.alpha < 1.f), m(0.f), l_a(0.f), l_b(0.f) {
    c_a = soft ? kLog2e / a.tau : kLog2e;
    sub_p = soft ? a.alpha * a.tau * (a.counts ? 1.f / max(1, a.counts[0]) : 1.f) : 0.f;
    sub_y = hard ? (1.f - a.alpha) * (a.counts ? 1.f / max(1, a.counts[1]) : 1.f) : 0.f;
    k_a = sub_p;
    k_b = sub_y;
    if (!two(a)) k_a += k_b;
  }
  // whether the row needs exponentials at two temperatures
  __device__ __forceinline__ bool two(const DistillArgs& a) const { return soft && hard && a.tau != 1.f; }
  template <bool TWO>
  __device__ __forceinline__ float dense(float z) const {
    const float d = z - m;
    float g = k_a * ex2(fmaf(d, c_a, -l_a));
    if (TWO) g = fmaf(k_b, ex2(fmaf(d, kLog2e, -l_b)), g);
    return g;
  }
};

// Rewrites the gradient at this block's slots and target, where the dense part alone was stored.
// get(v, z): whether position v of the row is this block's, and its logit.  The first slot of an id
// answers for all slots of that id, and for the target when it is that id.
template <typename T, bool TWO, typename Get>
__device__ __forceinline__ void put_slots(const RowGrad& r, const TeacherRow& t, int top, int target, T* grad,
                                          const Get& get) {
  for (int j = threadIdx.x; j <= top; j += kThreads) {
    const int id = j < top ? (r.soft ? t.id[j] : -1) : (r.hard ? target : -1);
    float z;
    if (id < 0 || !get(id, z)) continue;
    bool first = true;
    float p = 0.f;
    if (r.soft) {
      for (int i = 0; i < top; ++i) {
        if (t.id[i] != id) continue;
        if (i < j) {
          first = false;
          break;
        }
        p += t.p[i];
      }
    }
    if (!first) continue;
    float g = r.dense<TWO>(z) - r.sub_p * p;
    if (r.hard && id == target) g -= r.sub_y;
    grad[id] = from_f32<T>(g);
  }
}

// max and sums of a slice in shared memory (and of at most one more value of this thread)
template <typename T, bool TWO>
__device__ __forceinline__ Part slice_part(const uint4* slice, int n, bool has_edge, float edge, float c_a) {
  constexpr int V = RowSplit<T>::V;
  Part part{has_edge ? edge : -INFINITY, 0.f, 0.f};
  for (int i = threadIdx.x; i < n; i += kThreads) {
    float v[V];
    unpack<T, V>(slice[i], v);
#pragma unroll
    for (int e = 0; e < V; ++e) part.m = fmaxf(part.m, v[e]);
  }
  const float m = part.m == -INFINITY ? 0.f : part.m;  // nothing but -inf: every term is 0
  auto term = [&](float x) {
    const float d = x - m;
    part.s += ex2(d * c_a);
    if (TWO) part.h += ex2(d * kLog2e);
  };
  if (has_edge) term(edge);
  for (int i = threadIdx.x; i < n; i += kThreads) {
    float v[V];
    unpack<T, V>(slice[i], v);
#pragma unroll
    for (int e = 0; e < V; ++e) term(v[e]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Part q;
    q.m = __shfl_xor_sync(0xffffffffu, part.m, o);
    q.s = __shfl_xor_sync(0xffffffffu, part.s, o);
    q.h = __shfl_xor_sync(0xffffffffu, part.h, o);
    part = join(part, q, c_a);
  }
  return part;
}

template <typename T, bool TWO>
__device__ __forceinline__ void store_dense(const RowGrad& r, const uint4* from, uint4* to, int n) {
  constexpr int V = RowSplit<T>::V;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    float v[V];
    unpack<T, V>(from[i], v);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = r.dense<TWO>(v[e]);
    to[i] = pack<T, V>(v);
  }
}

// One row a cluster.  Shared memory: the block's slice of the row, p and id of the slots.
template <typename T>
__global__ void __launch_bounds__(kThreads) distill_rows_kernel(const DistillArgs a, int* err) {
  constexpr int V = RowSplit<T>::V;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float red[kWarps];
  __shared__ Part warp_part[kWarps];
  __shared__ Part block_part[kMaxCluster];  // every block's part, as each block of the cluster has it
  __shared__ float edge[2 * V];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), blocks = static_cast<int>(cluster.num_blocks());
  auto started = cluster.barrier_arrive();  // waited for before the first write to another block's memory
  const int64_t row = blockIdx.x / blocks;
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;

  const RowSplit<T> split(z, a.vocab);
  const int v0 = static_cast<int>(static_cast<int64_t>(split.vecs) * rank / blocks);
  const int n = static_cast<int>(static_cast<int64_t>(split.vecs) * (rank + 1) / blocks) - v0;
  const int head = rank == 0 ? split.head : 0, tail = rank == blocks - 1 ? split.tail : 0;
  const int behind = split.head + split.vecs * V;  // where the tail starts
  uint4* slice = reinterpret_cast<uint4*>(smem);
  TeacherRow t;
  t.p = reinterpret_cast<float*>(slice + a.vocab / V / blocks + 1);
  t.id = reinterpret_cast<int*>(t.p + a.top);

  const uint4* body = reinterpret_cast<const uint4*>(z + split.head) + v0;
  for (int i = threadIdx.x; i < n; i += kThreads)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(slice + i)), "l"(body + i) : "memory");
  asm volatile("cp.async.commit_group;" ::: "memory");
  const int tid = static_cast<int>(threadIdx.x);
  const bool has_edge = tid < head + tail;
  const int edge_at = tid < head ? tid : behind + tid - head;
  const float edge_z = has_edge ? to_f32(z[edge_at]) : 0.f;
  if (has_edge) edge[tid] = edge_z;

  const int target = valid_target(a, row, err);
  RowGrad r(a, teacher_row(a, row, t, red, err), target >= 0);
  const bool two = r.two(a), any = r.soft || r.hard;
  // the first block has the loss: it gathers the logits of the slots and of the target before any
  // block of the cluster can have written a gradient over them
  float slot_z[kMaxTop / kThreads], target_z = 0.f;
  if (rank == 0) {
#pragma unroll
    for (int k = 0; k < kMaxTop / kThreads; ++k) {
      const int j = tid + k * kThreads;
      slot_z[k] = r.soft && j < a.top && t.id[j] >= 0 ? to_f32(z[t.id[j]]) : 0.f;
    }
    if (r.hard) target_z = to_f32(z[target]);
  }

  asm volatile("cp.async.wait_all;" ::: "memory");
  if (any) {
    const Part p = two ? slice_part<T, true>(slice, n, has_edge, edge_z, r.c_a)
                       : slice_part<T, false>(slice, n, has_edge, edge_z, r.c_a);
    if ((tid & 31) == 0) warp_part[tid >> 5] = p;
  }
  __syncthreads();  // also: slices and edges are there for the other threads
  if (any) {
    Part p = warp_part[0];
    for (int w = 1; w < kWarps; ++w) p = join(p, warp_part[w], r.c_a);
    cluster.barrier_wait(std::move(started));
    if (tid < blocks) *cluster.map_shared_rank(&block_part[rank], tid) = p;
    cluster.sync();
    p = block_part[0];
    for (int b = 1; b < blocks; ++b) p = join(p, block_part[b], r.c_a);
    r.m = p.m;
    r.l_a = log2f(p.s);
    r.l_b = two ? log2f(p.h) : r.l_a;
  } else {
    cluster.barrier_wait(std::move(started));
  }

  if (rank == 0) {
    float kd = 0.f;  // sum p_j (log2 p_j - log2 q_tau(id_j))
    if (r.soft) {
#pragma unroll
      for (int k = 0; k < kMaxTop / kThreads; ++k) {
        const int j = tid + k * kThreads;
        if (j < a.top && t.id[j] >= 0 && t.p[j] > 0.f)
          kd = fmaf(t.p[j], log2f(t.p[j]) - fmaf(slot_z[k] - r.m, r.c_a, -r.l_a), kd);
      }
      kd = block_add(kd, red);
    }
    if (tid == 0) {
      const float ce = r.hard ? fmaf(r.l_b, kLn2, r.m - target_z) : 0.f;
      // sub_p = alpha tau / count; the loss has another tau
      a.loss[row] = r.sub_p * a.tau * kLn2 * kd + r.sub_y * ce;
      if (a.stats) {
        a.stats[3 * row] = r.m;
        a.stats[3 * row + 1] = r.l_a;
        a.stats[3 * row + 2] = r.l_b;
      }
    }
  }
  if (a.grad == nullptr) return;

  T* grad = static_cast<T*>(a.grad) + row * a.grad_ld;
  uint4* to = reinterpret_cast<uint4*>(grad + split.head) + v0;
  if (!any) {
    for (int i = tid; i < n; i += kThreads) to[i] = make_uint4(0u, 0u, 0u, 0u);
    if (has_edge) grad[edge_at] = from_f32<T>(0.f);
    return;
  }
  // position v of the row, if this block has it
  auto get = [&](int v, float& x) {
    if (v < split.head || v >= behind) {
      if (rank != (v < split.head ? 0 : blocks - 1)) return false;
      x = edge[v < split.head ? v : head + v - behind];
      return true;
    }
    const int i = (v - split.head) / V - v0;
    if (i < 0 || i >= n) return false;
    x = to_f32(reinterpret_cast<const T*>(slice + i)[(v - split.head) % V]);
    return true;
  };
  auto write = [&](auto mode) {
    constexpr bool TWO = decltype(mode)::value;
    store_dense<T, TWO>(r, slice, to, n);
    if (has_edge) grad[edge_at] = from_f32<T>(r.dense<TWO>(edge_z));
    __syncthreads();  // the slots' rewrites come after the dense stores
    put_slots<T, TWO>(r, t, a.top, target, grad, get);
  };
  if (two)
    write(std::true_type());
  else
    write(std::false_type());
}

// The gradient alone, from the statistics of an earlier pass and the incoming gradient: blocks of
// `segment` vectors of a row, straight from and to global memory.
template <typename T>
__global__ void __launch_bounds__(kThreads) distill_grad_kernel(const DistillArgs a, int segments, int segment,
                                                                int* err) {
  constexpr int V = RowSplit<T>::V;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float red[kWarps];
  const int64_t row = blockIdx.x / segments;
  const int seg = static_cast<int>(blockIdx.x - row * segments);
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  T* grad = static_cast<T*>(a.grad) + row * a.grad_ld;
  const RowSplit<T> split(z, a.vocab);
  const int v0 = min(seg * segment, split.vecs), n = min(segment, split.vecs - v0);
  const int behind = split.head + split.vecs * V;
  const int head = seg == 0 ? split.head : 0, tail = seg == segments - 1 ? split.tail : 0;
  const int tid = static_cast<int>(threadIdx.x);
  const bool has_edge = tid < head + tail;
  const int edge_at = tid < head ? tid : behind + tid - head;
  const uint4* from = reinterpret_cast<const uint4*>(z + split.head) + v0;
  uint4* to = reinterpret_cast<uint4*>(grad + split.head) + v0;

  TeacherRow t;
  t.p = reinterpret_cast<float*>(smem);
  t.id = reinterpret_cast<int*>(t.p + a.top);
  const int target = valid_target(a, row, err);
  RowGrad r(a, teacher_row(a, row, t, red, err), target >= 0);
  const bool two = r.two(a);
  if (!r.soft && !r.hard) {
    for (int i = tid; i < n; i += kThreads) to[i] = make_uint4(0u, 0u, 0u, 0u);
    if (has_edge) grad[edge_at] = from_f32<T>(0.f);
    return;
  }
  const float up = a.upstream[a.upstream_rows ? row : 0];
  r.k_a *= up;
  r.k_b *= up;
  r.sub_p *= up;
  r.sub_y *= up;
  r.m = a.stats[3 * row];
  r.l_a = a.stats[3 * row + 1];
  r.l_b = a.stats[3 * row + 2];
  auto get = [&](int v, float& x) {
    if (v < split.head || v >= behind) {
      if (seg != (v < split.head ? 0 : segments - 1)) return false;
    } else {
      const int i = (v - split.head) / V - v0;
      if (i < 0 || i >= n) return false;
    }
    x = to_f32(z[v]);
    return true;
  };
  auto write = [&](auto mode) {
    constexpr bool TWO = decltype(mode)::value;
    store_dense<T, TWO>(r, from, to, n);
    if (has_edge) grad[edge_at] = from_f32<T>(r.dense<TWO>(to_f32(z[edge_at])));
    __syncthreads();
    put_slots<T, TWO>(r, t, a.top, target, grad, get);
  };
  if (two)
    write(std::true_type());
  else
    write(std::false_type());
}

// counts[0]: rows with a slot, counts[1]: rows with a target.  One block: a thread mostly reads its
// rows' first slot alone.
__global__ void __launch_bounds__(1024) distill_count_kernel(const DistillArgs a, int* counts, int* err) {
  int slots = 0, targets = 0;
  for (int64_t row = threadIdx.x; row < a.rows; row += blockDim.x) {
    for (int j = 0; j < a.top; ++j) {
      const int64_t i = row * a.top + j;
      if (valid_id(a, i, err) >= 0 && !(teacher_value(a, i) == -INFINITY)) {
        ++slots;
        break;
      }
    }
    targets += valid_target(a, row, err) >= 0;
  }
  __shared__ int s[2];
  if (threadIdx.x < 2) s[threadIdx.x] = 0;
  __syncthreads();
  slots = __reduce_add_sync(0xffffffffu, slots);
  targets = __reduce_add_sync(0xffffffffu, targets);
  if ((threadIdx.x & 31) == 0) {  // whole numbers: the order does not matter
    atomicAdd(&s[0], slots);
    atomicAdd(&s[1], targets);
  }
  __syncthreads();
  if (threadIdx.x < 2) counts[threadIdx.x] = s[threadIdx.x];
}

__global__ void __launch_bounds__(512) distill_sum_kernel(const float* loss, int64_t rows, float* out) {
  __shared__ double s[512];
  double t = 0.0;
  for (int64_t i = threadIdx.x; i < rows; i += 512) t += loss[i];
  s[threadIdx.x] = t;
  for (int o = 256; o > 0; o >>= 1) {
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < o) s[threadIdx.x] += s[threadIdx.x + o];
  }
  if (threadIdx.x == 0) *out = static_cast<float>(s[0]);
}

template <typename T>
__global__ void __launch_bounds__(256) distill_scale_kernel(T* x, const float* s, int64_t n) {
  const float f = *s;
  if (f == 1.f) return;
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  const int64_t vecs = n / V, step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t i = first; i < vecs; i += step) {
    float v[V];
    unpack<T, V>(ld_raw<T, V>(x + i * V), v);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] *= f;
    st_raw<T, V>(x + i * V, pack<T, V>(v));
  }
  for (int64_t i = vecs * V + first; i < n; i += step) x[i] = from_f32<T>(to_f32(x[i]) * f);
}

void check(const char* what) {
  count_launch();
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    throw std::runtime_error(std::string("mmf: ") + what + " launch failed: " + cudaGetErrorString(e));
}

int* error_word() {
  int dev = 0;
  cudaGetDevice(&dev);
  return device_error_word(dev);
}

template <typename Go>
void typed(DType d, const Go& go) {
  if (d == DType::BF16)
    go(__nv_bfloat16());
  else if (d == DType::F16)
    go(__half());
  else
    go(float());
}

constexpr int kSliceGoal = 64 << 10;  // bytes: three blocks an SM
constexpr int kSliceMost = 200 << 10;
constexpr int kSliceLeast = 8 << 10;

}  // namespace

int64_t distill_max_vocab(DType dtype) { return kSliceMost / (dtype == DType::F32 ? 4 : 2) * kMaxCluster; }
int distill_max_top() { return kMaxTop; }

void distill_count(const DistillArgs& a, int* counts, cudaStream_t stream) {
  distill_count_kernel<<<1, 1024, 0, stream>>>(a, counts, error_word());
  check("distill_count");
}

void distill_rows(const DistillArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return;
  if (a.top < 1 || a.top > kMaxTop || a.vocab < 1 || a.vocab > distill_max_vocab(a.dtype))
    throw std::runtime_error("mmf: distill: vocabulary or number of slots out of range");
  typed(a.dtype, [&](auto tag) {
    using T = decltype(tag);
    const int64_t bytes = static_cast<int64_t>(a.vocab) * sizeof(T);
    // blocks a row: slices that fit three to an SM; with few rows more, down to 8 KB each, so that
    // every SM has one
    int blocks = 1;
    while (blocks < kMaxCluster && bytes / blocks > kSliceGoal) blocks *= 2;
    while (blocks < kMaxCluster && a.rows * blocks < 148 && bytes / blocks > kSliceLeast) blocks *= 2;
    if (a.rows * blocks > 0x7fffffff) throw std::runtime_error("mmf: distill: too many rows");
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const int smem = (a.vocab / V / blocks + 1) * 16 + a.top * 8;
    auto kernel = distill_rows_kernel<T>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) throw std::runtime_error(std::string("mmf: distill: ") + cudaGetErrorString(e));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.rows * blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(blocks);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, a, error_word());
  });
  check("distill_rows");
}

void distill_grad(const DistillArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return;
  if (a.top < 1 || a.top > kMaxTop) throw std::runtime_error("mmf: distill: number of slots out of range");
  typed(a.dtype, [&](auto tag) {
    using T = decltype(tag);
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const int segment = kThreads * 4;  // vectors
    const int segments = std::max(1, (a.vocab / V + segment - 1) / segment);
    if (a.rows * segments > 0x7fffffff) throw std::runtime_error("mmf: distill: too many rows");
    distill_grad_kernel<T><<<static_cast<unsigned>(a.rows * segments), kThreads, a.top * 8, stream>>>(
        a, segments, segment, error_word());
  });
  check("distill_grad");
}

void distill_sum(const float* loss, int64_t rows, float* out, cudaStream_t stream) {
  distill_sum_kernel<<<1, 512, 0, stream>>>(loss, rows, out);
  check("distill_sum");
}

void distill_scale(void* x, const float* s, int64_t n, DType dtype, cudaStream_t stream) {
  if (n == 0) return;
  typed(dtype, [&](auto tag) {
    using T = decltype(tag);
    distill_scale_kernel<T><<<148 * 8, 256, 0, stream>>>(static_cast<T*>(x), s, n);
  });
  check("distill_scale");
}

}  // namespace mmf
