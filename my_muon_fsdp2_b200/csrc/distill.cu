// Distillation from a teacher's top logits (kernels.h has the formulas), loss and gradient of one
// row of logits after another:
//
//   dz_v = alpha tau wk (q_tau(v) - sum over slots j with id_j = v of p_j)
//          + (1 - alpha) wc (q_1(v) - [v = target]),      q_t = softmax(z / t)
//
// Bound by memory: the logits are read once and, with the gradient, written once.  A row is spread
// over a cluster of blocks, each holding its slice in shared memory (a 128256 wide bf16 row has 250
// KB, one block's shared memory 227): one asynchronous copy in, the maximum and the sums over the
// slice, one exchange of (maximum, sums) between the blocks, and the gradient straight out of the
// slice.  Slices of about 32 KB and 256 threads let six blocks share an SM and overlap one another's
// copies, exchanges and stores.  Measured, 4096 x 128256 bf16, 64 slots, tau 2 with hard targets: 426 us (2.1
// GB, 75 % of the copy rate), with 8 slots 416, with 256 513 (their rewrites go to as many sectors of their own).
// The SMs issue in 81 % of the cycles and their pipe for exponentials is 63 % busy: the arithmetic takes nearly
// as long as the copies, and one exponential less or more a value shows (tau 1 397 us, tau 1.5 594).  Tried at
// a time when it took 405 us: slices of 64 KB 445; the exchange by a barrier of the cluster, whose release
// waits for every store before it, and five blocks an SM 510; blocks that stay for many rows, two an SM, with
// copies ahead and the exponentials kept in registers between the two passes 500.
//
// The arithmetic goes through packed fp32 instructions, the maximum of 16-bit types is taken without
// widening them, and at tau = 2 the softmax at 1 comes from the one at tau as its square (one
// exponential a value instead of two).
//
// Every exponential is 2^(c (z - m)), m the largest logit of a thread, later of the row.  The difference comes
// first: it is exactly 0 at the maximum, however far that is from 0 (a row whose words are all at the type's
// lowest value is uniform).  2^(c z - R) with R = c m rounded beforehand is one packed instruction less (1.5 %
// of the case above), but has R's rounding in its exponent: 440 at z = -1e10, and infinities behind it; with
// both forms, chosen by |c m|, the case took 1.1 % more all the same.  Sums are scaled by 2^(c (m - m')) as they
// are joined, so nothing overflows.
#include <cooperative_groups.h>

#include <algorithm>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "kernels.h"
#include "launch_info.h"
#include "tc_common.cuh"
#include "typed_io.cuh"

namespace mmf {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 1024;
constexpr int kWarpSlots = 128;  // up to which one warp sums the row's loss
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Which exponentials a launch needs: one (one of the two losses, or tau = 1), those at 1 as the squares
// of those at tau = 2, or two of their own.
enum Mode { ONE, SQUARE, TWO };

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A slot as it lies in memory: loading several and looking at them later lets their latencies overlap.
struct RawSlot {
  uint2 id;
  uint32_t value;
};
__device__ __forceinline__ RawSlot load_slot(const DistillArgs& a, int64_t i) {
  RawSlot r{make_uint2(0u, 0u), 0u};
  if (a.ids_32)
    r.id.x = static_cast<const uint32_t*>(a.ids)[i];
  else
    r.id = static_cast<const uint2*>(a.ids)[i];
  if (a.teacher_dtype == DType::F32)
    r.value = static_cast<const uint32_t*>(a.teacher)[i];
  else
    r.value = static_cast<const uint16_t*>(a.teacher)[i];
  return r;
}
// (id, value): -1 and -inf for an empty slot; an id behind the vocabulary is empty, and bad.
__device__ __forceinline__ void look_at(const DistillArgs& a, const RawSlot& r, int& id, float& v, bool& bad) {
  const int64_t wide = a.ids_32 ? static_cast<int64_t>(static_cast<int>(r.id.x))
                                : static_cast<int64_t>(static_cast<uint64_t>(r.id.y) << 32 | r.id.x);
  if (a.teacher_dtype == DType::F32)
    v = __uint_as_float(r.value);
  else if (a.teacher_dtype == DType::BF16)
    v = __uint_as_float(r.value << 16);
  else
    v = __half2float(__ushort_as_half(static_cast<uint16_t>(r.value)));
  bad |= wide >= a.vocab;
  const bool empty = wide < 0 || wide >= a.vocab || v == -INFINITY;
  id = empty ? -1 : static_cast<int>(wide);
  if (empty) v = -INFINITY;
}
__device__ __forceinline__ int64_t load_target(const DistillArgs& a, int64_t row) {
  return a.targets ? a.targets[row] : a.ignore_index;
}
// The target, or -1 where it is ignored; one outside the vocabulary is ignored and recorded.
__device__ __forceinline__ int look_at(const DistillArgs& a, int64_t y, int* err) {
  if (y == a.ignore_index) return -1;
  if (y < 0 || y >= a.vocab) {
    atomicCAS(err, 0, ERR_BAD_ARGUMENT);
    return -1;
  }
  return static_cast<int>(y);
}

// The largest of some logits, and the sums of their exponentials at the temperature of c_a (s) and, in
// the modes that have them, at 1 (h), relative to that maximum.
struct Part {
  float m, s, h;
  // What is taken off a logit: the maximum, or 0 where there is nothing but -inf (or NaN, which the sums
  // carry), so that every term is 0.
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
};
// Over groups of `W` lanes, the same bits in each of them.
template <int MODE, int W>
__device__ __forceinline__ Part warp_join(Part p, float c_a) {
  float m = p.m;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  // without a finite logit of its own a part is 0 (or NaN) against any maximum
  const float down = p.m == -INFINITY ? 0.f : p.m - m;
  p.s *= ex2(down * c_a);
  if (MODE != ONE) p.h *= ex2(down * kLog2e);
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    p.s += __shfl_xor_sync(0xffffffffu, p.s, o);
    if (MODE != ONE) p.h += __shfl_xor_sync(0xffffffffu, p.h, o);
  }
  p.m = m;
  return p;
}

__device__ __forceinline__ float2 exp2_2(float2 a) { return make_float2(ex2(a.x), ex2(a.y)); }
// 16 bytes of a row as pairs
template <typename T>
struct Vec {
  static constexpr int N = 16 / static_cast<int>(sizeof(T));
  static __device__ __forceinline__ void pairs(const uint4& w, float2 (&p)[N / 2]) {
    float v[N];
    unpack<T, N>(w, v);
#pragma unroll
    for (int e = 0; e < N / 2; ++e) p[e] = make_float2(v[2 * e], v[2 * e + 1]);
  }
  static __device__ __forceinline__ uint4 from_pairs(const float2 (&p)[N / 2]) {
    float v[N];
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      v[2 * e] = p[e].x;
      v[2 * e + 1] = p[e].y;
    }
    return pack<T, N>(v);
  }
};

// The largest value of several vectors; NaN is left out (the sums carry it).
template <typename T>
struct MaxOf {
  float m = -INFINITY;
  __device__ __forceinline__ void put(const uint4& w) {
    m = fmaxf(fmaxf(fmaxf(m, __uint_as_float(w.x)), __uint_as_float(w.y)),
              fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  __device__ __forceinline__ float get() const { return m; }
};
template <typename T2>
struct MaxOfHalves {
  T2 m;
  static __device__ __forceinline__ T2 as(uint32_t w) { return *reinterpret_cast<const T2*>(&w); }
  __device__ __forceinline__ void put(const uint4& w) {
    m = __hmax2(m, __hmax2(__hmax2(as(w.x), as(w.y)), __hmax2(as(w.z), as(w.w))));
  }
};
template <>
struct MaxOf<__nv_bfloat16> : MaxOfHalves<__nv_bfloat162> {
  __device__ __forceinline__ MaxOf() { m = as(0xff80ff80u); }  // -inf
  __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};
template <>
struct MaxOf<__half> : MaxOfHalves<__half2> {
  __device__ __forceinline__ MaxOf() { m = as(0xfc00fc00u); }
  __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};

// The positions of a row that a block has.  Rows start anywhere on the type's own boundary: a row is
// a head of up to 7 values, a body of 16-byte vectors and a tail; a row's first block has the head, its
// last the tail, and each `each` vectors (the last what is left).
template <typename T>
struct Share {
  static constexpr int V = Vec<T>::N;
  int first, vecs;  // the block's vectors: the position of the first, how many
  int lo, hi;       // all its positions
  int edges;        // how many of them are head and tail
  int behind;       // where the row's tail starts
  __device__ __forceinline__ Share(const T* row, int vocab, int each, int part, int parts) {
    const int head = min(static_cast<int>(-reinterpret_cast<uintptr_t>(row) & 15) / static_cast<int>(sizeof(T)), vocab);
    const int all = (vocab - head) / V;
    const int v0 = min(each * part, all);
    vecs = min(each, all - v0);
    first = head + v0 * V;
    behind = head + all * V;
    lo = part == 0 ? 0 : first;
    hi = part == parts - 1 ? vocab : first + vecs * V;
    edges = (hi - lo) - vecs * V;
  }
  __device__ __forceinline__ bool has(int v) const { return v >= lo && v < hi; }
  // the i-th of the head's and the tail's positions
  __device__ __forceinline__ int edge(int i) const { return i < first - lo ? lo + i : behind + i - (first - lo); }
};

// A row's slots in shared memory.  The teacher's values become exponentials e_j against the largest one
// (p_j = e_j / their sum); `z` are the logits there where those are wanted; own_id and own_p are id and e_j
// of the slots at the block's own positions, in the order of the slots.
constexpr int kSlotBytes = 20;
struct Slots {
  float *p, *z, *own_p;
  int *id, *own_id;
  __device__ __forceinline__ Slots(void* at, int top) {
    const int room = (top + 3) & ~3;  // read four at a time
    p = static_cast<float*>(at);
    z = p + room;
    own_p = z + room;
    id = reinterpret_cast<int*>(own_p + room);
    own_id = id + room;
  }
};
__device__ __forceinline__ float over_warps(const float* v, bool largest) {
  static_assert(kWarps == 8, "");
  const float4 a = *reinterpret_cast<const float4*>(v), b = *reinterpret_cast<const float4*>(v + 4);
  return largest ? fmaxf(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)), fmaxf(fmaxf(b.x, b.y), fmaxf(b.z, b.w)))
                 : ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
}
// What the warps tell one another about the slots: each thread has every kThreads-th.
struct __align__(16) SlotNotes {
  float best[kWarps], sum[kWarps];
  int any[kWarps];
  int own[kMaxTop / 32];  // slots at the block's own positions, among each 32
  // 1 / the sum of the slots' exponentials
  __device__ __forceinline__ float inverse() const { return __fdividef(1.f, over_warps(sum, false)); }
};
// Step 1, all threads: the teacher's ids and values, and (z not null) the logits there, into shared
// memory.  The id and the value of a slot are loaded side by side: what a block waits for here are two
// latencies at most, beside that of its slice.
template <typename T>
__device__ __forceinline__ void load_slots(const DistillArgs& a, int64_t row, const T* z, const Slots& t, SlotNotes& notes,
                                           const Share<T>& share, int* err) {
  bool bad = false, any = false;
  float best = -INFINITY;
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = threadIdx.x & 31;
  for (int j0 = 0; j0 < a.top; j0 += kThreads) {
    const int j = j0 + static_cast<int>(threadIdx.x);
    int id = -1;
    float v = -INFINITY;
    if (j < a.top) {
      look_at(a, load_slot(a, row * a.top + j), id, v, bad);
      if (z && id >= 0) t.z[j] = to_f32(z[id]);
      t.id[j] = id;
      t.p[j] = v;
    }
    any |= id >= 0;
    best = fmaxf(best, v);
    const unsigned mine = __ballot_sync(0xffffffffu, id >= 0 && share.has(id));
    if (lane == 0) notes.own[(j0 >> 5) + warp] = __popc(mine);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
  any = __any_sync(0xffffffffu, any);
  if (lane == 0) {
    notes.best[warp] = best;
    notes.any[warp] = any;
  }
  if (bad) atomicCAS(err, 0, ERR_BAD_ARGUMENT);
}
// Step 2, all threads behind a barrier: the values become exponentials.  Returns how many slots are the
// block's own, -1 for a row without a slot.
template <typename T>
__device__ __forceinline__ int fill_slots(const DistillArgs& a, float c_tau, const Slots& t, SlotNotes& notes,
                                           const Share<T>& share) {
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (!__any_sync(0xffffffffu, notes.any[lane % kWarps])) return -1;
  const float best = over_warps(notes.best, true);
  const int own = lane < (a.top + kThreads - 1) / kThreads * kWarps ? notes.own[lane] : 0;
  float s = 0.f;
  for (int j0 = 0; j0 < a.top; j0 += kThreads) {
    const int j = j0 + static_cast<int>(threadIdx.x);
    const int id = j < a.top ? t.id[j] : -1;
    const float e = id >= 0 ? ex2((t.p[j] - best) * c_tau) : 0.f;
    if (j < a.top) t.p[j] = e;
    s += e;
    const bool mine = id >= 0 && share.has(id);
    const unsigned ballot = __ballot_sync(0xffffffffu, mine);
    if (ballot) {
      const int before = __reduce_add_sync(0xffffffffu, lane < (j0 >> 5) + warp ? own : 0);
      if (mine) {
        const int at = before + __popc(ballot & ((1u << lane) - 1u));
        t.own_id[at] = id;
        t.own_p[at] = e;
      }
    }
  }
  s = warp_sum(s);
  if (lane == 0) notes.sum[warp] = s;
  return __reduce_add_sync(0xffffffffu, own);
}

// What a launch has in common, formed on the host.
struct Scales {
  float c_tau;       // log2 e / tau
  float c_a;         // the same, or log2 e where the soft loss has no weight
  float soft, hard;  // alpha tau, 1 - alpha
};
Scales scales(const DistillArgs& a) {
  const float c = static_cast<float>(1.4426950408889634 / a.tau);
  return {c, a.alpha > 0.f ? c : kLog2e, a.alpha * a.tau, 1.f - a.alpha};
}

// A row's coefficients: its gradient is k_a q_a + k_b q_b, with sub_p p_j off at the slots and sub_y
// off at the target; q_a is the softmax at tau (at 1 where only the target counts), q_b the one at 1.
struct Coefficients {
  float k_a, k_b, sub_p, sub_y;
  template <int MODE>
  static __device__ __forceinline__ Coefficients of(const Scales& s, const int* counts, bool soft, bool hard, float up) {
    Coefficients c;
    c.sub_p = soft ? s.soft * up : 0.f;
    c.sub_y = hard ? s.hard * up : 0.f;
    if (counts) {
      c.sub_p = __fdividef(c.sub_p, static_cast<float>(max(1, counts[0])));
      c.sub_y = __fdividef(c.sub_y, static_cast<float>(max(1, counts[1])));
    }
    c.k_a = MODE == ONE ? c.sub_p + c.sub_y : c.sub_p;
    c.k_b = c.sub_y;
    return c;
  }
};

// The gradient before the slots' and the target's own terms, from the row's joined part: the sums'
// reciprocals are in the factors.
template <int MODE>
struct Dense {
  float2 c, off, log2e, f_a, f_b;
  __device__ __forceinline__ Dense(const Coefficients& k, float c_a, const Part& p) {
    c = make_float2(c_a, c_a);
    off = make_float2(-p.base(), -p.base());
    log2e = make_float2(kLog2e, kLog2e);
    const float a = __fdividef(k.k_a, p.s), b = MODE == ONE ? 0.f : __fdividef(k.k_b, p.h);
    f_a = make_float2(a, a);
    f_b = make_float2(b, b);
  }
  __device__ __forceinline__ float2 operator()(float2 z) const {
    const float2 d = fadd2(z, off), e = exp2_2(fmul2(d, c));
    if (MODE == ONE) return fmul2(e, f_a);
    if (MODE == SQUARE) return fmul2(e, ffma2(e, f_b, f_a));
    return ffma2(exp2_2(fmul2(d, log2e)), f_b, fmul2(e, f_a));
  }
  __device__ __forceinline__ float one(float z) const { return (*this)(make_float2(z, z)).x; }
};

// Rewrites the gradient at this block's `owned` slots and at its target, where the dense part alone was
// stored.  A lane a slot; the first slot of an id answers for all slots of that id, and for the target
// when it is that id.  All slots of an id are the same block's, which is where they are looked for.
// get(v): the logit at the block's position v.
template <typename T, int MODE, typename Get>
__device__ __forceinline__ void put_slots(const Dense<MODE>& dense, const Coefficients& k, const Slots& t, int owned,
                                          const SlotNotes& notes, int target, const Share<T>& share, T* grad, const Get& get) {
  const bool has_target = target >= 0 && share.has(target);
  owned = max(owned, 0);
  for (int i = threadIdx.x; i < owned + has_target; i += kThreads) {
    const int id = i < owned ? t.own_id[i] : target;  // the target comes behind the slots
    float p = 0.f;
    bool earlier = false;
#pragma unroll 4
    for (int o = 0; o < owned; o += 4) {
      const int4 other = *reinterpret_cast<const int4*>(t.own_id + o);
      if (other.x == id || other.y == id || other.z == id || other.w == id) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (o + e < owned && t.own_id[o + e] == id) {
            p += t.own_p[o + e];
            earlier |= o + e < i;
          }
        }
      }
    }
    if (earlier) continue;
    float g = dense.one(get(id)) - k.sub_p * (owned ? p * notes.inverse() : 0.f);
    if (id == target) g -= k.sub_y;
    grad[id] = from_f32<T>(g);
  }
}

template <typename T, int MODE>
__device__ __forceinline__ void store_dense(const Dense<MODE>& dense, const uint4* from, uint4* to, int n) {
  constexpr int P = Vec<T>::N / 2;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += kThreads) {
    float2 p[P];
    Vec<T>::pairs(from[i], p);
#pragma unroll
    for (int e = 0; e < P; ++e) p[e] = dense(p[e]);
    to[i] = Vec<T>::from_pairs(p);
  }
}

// Maximum and sums of a slice in shared memory, and of one more value of the first threads.
template <typename T, int MODE>
__device__ __forceinline__ Part slice_part(const uint4* slice, int n, bool has_edge, float edge, float c_a) {
  constexpr int P = Vec<T>::N / 2;
  MaxOf<T> most;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += kThreads) most.put(slice[i]);
  Part part{most.get(), 0.f, 0.f};
  if (has_edge) part.m = fmaxf(part.m, edge);
  const float2 off = make_float2(-part.base(), -part.base()), c = make_float2(c_a, c_a);
  const float2 log2e = make_float2(kLog2e, kLog2e);
  float2 s = make_float2(0.f, 0.f), h = s;
  auto term = [&](float2 z) {
    const float2 d = fadd2(z, off), e = exp2_2(fmul2(d, c));
    s = fadd2(s, e);
    if (MODE == SQUARE) h = ffma2(e, e, h);
    if (MODE == TWO) h = fadd2(h, exp2_2(fmul2(d, log2e)));
  };
  if (has_edge) term(make_float2(edge, -INFINITY));
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += kThreads) {
    float2 p[P];
    Vec<T>::pairs(slice[i], p);
#pragma unroll
    for (int e = 0; e < P; ++e) term(p[e]);
  }
  part.s = s.x + s.y;
  part.h = h.x + h.y;
  return warp_join<MODE, 32>(part, c_a);
}

// One row a cluster.  Shared memory: the block's slice of the row, then the row's slots.
template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads, 6) distill_rows_kernel(const DistillArgs a, const Scales sc, int each, int* err) {
  constexpr int V = Vec<T>::N;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Part warp_part[kWarps];
  __shared__ float4 block_part[kMaxCluster];  // every block's part, as each block of the cluster has it
  __shared__ __align__(8) uint64_t received;
  __shared__ SlotNotes notes;
  __shared__ __align__(16) float loss_part[kWarps];
  __shared__ float target_z;
  __shared__ float edge_value[2 * V];  // the head's and the tail's logits
  // Parts travel as asynchronous stores that count their bytes on the receiver's barrier; every block
  // of the cluster has to have that before the first is sent.
  if (threadIdx.x == 0) {
    mbar_init(&received, 1);
    fence_mbar_init();
    mbar_arrive_expect_tx(&received, gridDim.y * static_cast<uint32_t>(sizeof(float4)));
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int rank = static_cast<int>(blockIdx.y), blocks = static_cast<int>(gridDim.y);
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  const Share<T> share(z, a.vocab, each, rank, blocks);
  const int n = share.vecs, tid = static_cast<int>(threadIdx.x), lane = tid & 31;
  uint4* slice = reinterpret_cast<uint4*>(smem);
  const Slots t(slice + each, a.top);

  const uint4* body = reinterpret_cast<const uint4*>(z + share.first);
#pragma unroll 4
  for (int i = tid; i < n; i += kThreads)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(slice + i)), "l"(body + i) : "memory");
  asm volatile("cp.async.commit_group;" ::: "memory");
  const bool has_edge = tid < share.edges;
  const int edge_at = share.edge(tid);
  const float edge_z = has_edge ? to_f32(z[edge_at]) : 0.f;

  // The first block has the loss: it gathers the logits of the slots and of the target before any
  // block of the cluster can have written a gradient over them.  Without a gradient the others are done
  // when they have sent it their parts (2047 x 50257 fp16: 52 us, 61 where all stay to the end).
  const bool whole = a.grad != nullptr;
  if (sc.soft > 0.f && (whole || rank == 0)) load_slots(a, row, rank == 0 ? z : nullptr, t, notes, share, err);
  const int target = sc.hard > 0.f ? look_at(a, load_target(a, row), err) : -1;
  if (rank == 0 && tid == 0 && target >= 0) target_z = to_f32(z[target]);
  const float c_a = sc.c_a;
  asm volatile("cp.async.wait_all;" ::: "memory");
  const Part wp = slice_part<T, MODE>(slice, n, has_edge, edge_z, c_a);
  if (lane == 0) warp_part[tid >> 5] = wp;
  if (has_edge) edge_value[tid] = edge_z;
  __syncthreads();  // also: the slice, the edges and the slots are there for the other threads
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (tid < 32) {
    const Part p = warp_join<MODE, kWarps>(warp_part[lane % kWarps], c_a);
    if (lane < (whole ? blocks : 1)) cluster_send(&block_part[rank], &received, lane, make_float4(p.m, p.s, p.h, 0.f));
  }
  if (!whole && rank != 0) return;
  const int owned = sc.soft > 0.f ? fill_slots(a, sc.c_tau, t, notes, share) : -1;
  __syncthreads();  // the slots and their notes
  const bool soft = owned >= 0, hard = target >= 0;
  mbar_wait(&received, 0, err, ERR_PEER_FLAG_TIMEOUT, MMF_WAIT_TIMEOUT_NS, false);
  const float4 part = lane % kMaxCluster < blocks ? block_part[lane % kMaxCluster] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
  const Part p = warp_join<MODE, kMaxCluster>(Part{part.x, part.y, part.z}, c_a);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the counts, where this kernel was let start before them
  const Coefficients k = Coefficients::of<MODE>(sc, a.counts, soft, hard, 1.f);

  auto put_loss = [&]() {
    const bool many = a.top > kWarpSlots;  // one warp has few; more are shared by all, which costs a barrier
    if (rank != 0 || (!many && tid >= 32)) return;
    const float base = p.base(), l_a = log2f(p.s);
    float kd = 0.f;  // sum p_j (log2 p_j - log2 q_tau(id_j))
    if (soft) {
      const float inv = notes.inverse();
      for (int j = tid; j < a.top; j += many ? kThreads : 32) {
        const float p_j = t.p[j] * inv;
        if (p_j != 0.f) kd = fmaf(p_j, log2f(p_j) - fmaf(t.z[j] - base, c_a, -l_a), kd);  // a teacher's NaN goes through
      }
      kd = warp_sum(kd);
      if (many) {
        if (lane == 0) loss_part[tid >> 5] = kd;
        __syncthreads();
        kd = over_warps(loss_part, false);
      }
    }
    if (tid == 0) {
      const float ce = kLn2 * (MODE == ONE ? l_a - (target_z - base) * c_a : log2f(p.h) - (target_z - base) * kLog2e);
      // sub_p = alpha tau / count; the loss has another tau
      a.loss[row] = (soft ? k.sub_p * a.tau * kLn2 * kd : 0.f) + (hard ? k.sub_y * ce : 0.f);
      if (a.stats) reinterpret_cast<float4*>(a.stats)[row] = make_float4(p.m, p.s, p.h, soft ? 1.f : 0.f);
    }
  };
  if (!whole) return put_loss();

  T* grad = static_cast<T*>(a.grad) + row * a.grad_ld;
  uint4* to = reinterpret_cast<uint4*>(grad + share.first);
  if (!soft && !hard) {  // takes no part, whatever its logits are
    for (int i = tid; i < n; i += kThreads) to[i] = make_uint4(0u, 0u, 0u, 0u);
    if (has_edge) grad[edge_at] = from_f32<T>(0.f);
    return put_loss();
  }
  const Dense<MODE> dense(k, c_a, p);
  store_dense<T, MODE>(dense, slice, to, n);
  if (has_edge) grad[edge_at] = from_f32<T>(dense.one(edge_z));
  __syncthreads();  // the slots' rewrites come after the dense stores
  put_slots<T, MODE>(dense, k, t, owned, notes, target, share, grad, [&](int v) {
    if (v < share.first) return edge_value[v - share.lo];
    const int at = v - share.first;
    return at < n * V ? to_f32(reinterpret_cast<const T*>(slice)[at])
                      : edge_value[share.first - share.lo + v - share.behind];
  });
  put_loss();
}

// The gradient alone, from the statistics of an earlier pass and the incoming gradient: blocks of
// `kSegment` vectors of a row, straight from and to global memory.
constexpr int kSegment = kThreads * 8;

template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads) distill_grad_kernel(const DistillArgs a, const Scales sc, int* err) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  T* grad = static_cast<T*>(a.grad) + row * a.grad_ld;
  const Share<T> share(z, a.vocab, kSegment, static_cast<int>(blockIdx.y), static_cast<int>(gridDim.y));
  const int tid = static_cast<int>(threadIdx.x);
  const bool has_edge = tid < share.edges;
  const int edge_at = share.edge(tid);
  const uint4* from = reinterpret_cast<const uint4*>(z + share.first);
  uint4* to = reinterpret_cast<uint4*>(grad + share.first);
  const Slots t(smem, a.top);
  const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
  const bool soft = st.w != 0.f;
  const int target = sc.hard > 0.f ? look_at(a, load_target(a, row), err) : -1;
  const bool hard = target >= 0;
  if (!soft && !hard) {
    for (int i = tid; i < share.vecs; i += kThreads) to[i] = make_uint4(0u, 0u, 0u, 0u);
    if (has_edge) grad[edge_at] = from_f32<T>(0.f);
    return;
  }
  const float up = a.upstream[a.upstream_rows ? row : 0];
  const Coefficients k = Coefficients::of<MODE>(sc, a.counts, soft, hard, up);
  const Dense<MODE> dense(k, sc.c_a, Part{st.x, st.y, st.z});
  __shared__ SlotNotes notes;
  if (soft) load_slots<T>(a, row, nullptr, t, notes, share, err);
  __syncthreads();
  const int owned = soft ? fill_slots(a, sc.c_tau, t, notes, share) : -1;
  store_dense<T, MODE>(dense, from, to, share.vecs);
  if (has_edge) grad[edge_at] = from_f32<T>(dense.one(to_f32(z[edge_at])));
  __syncthreads();  // the slots are there; their rewrites come after the dense stores
  put_slots<T, MODE>(dense, k, t, owned, notes, target, share, grad, [&](int v) { return to_f32(z[v]); });
}

// counts[0]: rows with a slot, counts[1]: rows with a target.  One cluster: a lane looks at its row's
// first slot, and the warp together at the rows where that one is empty.
__global__ void __cluster_dims__(kMaxCluster, 1, 1) __launch_bounds__(1024)
    distill_count_kernel(const DistillArgs a, int* counts, int* err) {
  __shared__ int s[2];
  // what comes behind may start: it waits for this kernel's end before it looks at the counts
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), lane = threadIdx.x & 31;
  if (threadIdx.x < 2) s[threadIdx.x] = 0;
  cluster.sync();
  int slots = 0, targets = 0;
  bool bad = false;
  auto filled = [&](int64_t row, int j) {
    int id;
    float v;
    look_at(a, load_slot(a, row * a.top + j), id, v, bad);
    return id >= 0;
  };
  for (int64_t base = (rank * 32 + (threadIdx.x >> 5)) * 32; base < a.rows; base += kMaxCluster * 1024) {
    const int64_t mine = base + lane;
    const bool live = mine < a.rows;
    const int64_t y = live ? load_target(a, mine) : a.ignore_index;
    const bool first = live && filled(mine, 0);
    targets += look_at(a, y, err) >= 0;
    slots += first;
    // four rows at a time, their loads on their way together
    for (unsigned rest = __ballot_sync(0xffffffffu, live && !first); rest;) {
      int64_t row[4];
      bool any[4], mine_too[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        mine_too[k] = rest != 0;
        row[k] = base + (rest ? __ffs(static_cast<int>(rest)) - 1 : 0);
        rest &= rest - 1;
        any[k] = false;
      }
      for (int j = 1 + lane; j < a.top; j += 32) {
#pragma unroll
        for (int k = 0; k < 4; ++k) any[k] |= mine_too[k] && filled(row[k], j);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) slots += __any_sync(0xffffffffu, any[k]) && lane == 0;
    }
  }
  if (bad) atomicCAS(err, 0, ERR_BAD_ARGUMENT);
  slots = __reduce_add_sync(0xffffffffu, slots);
  targets = __reduce_add_sync(0xffffffffu, targets);
  if (lane == 0) {  // whole numbers: the order does not matter
    atomicAdd(cluster.map_shared_rank(&s[0], 0), slots);
    atomicAdd(cluster.map_shared_rank(&s[1], 0), targets);
  }
  cluster.sync();
  if (rank == 0 && threadIdx.x < 2) counts[threadIdx.x] = s[threadIdx.x];
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

// Calls go(type, mode) with both as compile-time values.
template <typename Go>
void typed_mode(const DistillArgs& a, const Go& go) {
  const bool both = a.alpha > 0.f && a.alpha < 1.f && a.targets && a.tau != 1.f;
  typed(a.dtype, [&](auto t) {
    if (!both)
      go(t, std::integral_constant<int, ONE>());
    else if (a.tau == 2.f)
      go(t, std::integral_constant<int, SQUARE>());
    else
      go(t, std::integral_constant<int, TWO>());
  });
}

constexpr int kInFlight = 180 << 10;  // bytes of rows on an SM at once
// With few rows a row goes over more blocks, down to slices of this size, so that every SM has one: 8 rows
// of 50257 bf16 4.4 us, 4.7 with blocks_of_row's three.
constexpr int kSliceMost = 200 << 10;
constexpr int kSliceLeast = 8 << 10;
int slot_bytes(int top) { return ((top + 3) & ~3) * kSlotBytes; }

// Blocks for a row of `bytes`.  What an SM gets through goes by the bytes that it holds at once (a block
// takes about as long with 64 KB as with 32): the most blocks, hence the smallest slices, that still
// hold kInFlight of an SM's 228 KB, and where no number of blocks does, the number that holds most.  1 GB of
// bf16 logits, against slices of the next power of two below 32 KB: 50257 wide (three blocks instead of
// four) 441 instead of 509 us, 20000 wide (one instead of two) 442 instead of 534.
int blocks_of_row(int64_t bytes, int slots) {
  int best = 1;
  int64_t most = 0;
  for (int b = kMaxCluster; b >= 1; --b) {
    const int64_t slice = bytes / b;
    if (slice > kSliceMost) break;
    const int64_t held = slice * std::min<int64_t>(6, (228 << 10) / (slice + slots + 2048));  // 2 KB: a block's own
    if (held >= kInFlight) return b;
    if (held > most) {
      most = held;
      best = b;
    }
  }
  return best;
}

}  // namespace

int64_t distill_max_vocab(DType dtype) { return kSliceMost / (dtype == DType::F32 ? 4 : 2) * kMaxCluster; }
int distill_max_top() { return kMaxTop; }

void distill_count(const DistillArgs& a, int* counts, cudaStream_t stream) {
  distill_count_kernel<<<kMaxCluster, 1024, 0, stream>>>(a, counts, error_word());
  check("distill_count");
}

void distill_rows(const DistillArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return;
  if (a.top < 1 || a.top > kMaxTop || a.vocab < 1 || a.vocab > distill_max_vocab(a.dtype))
    throw std::runtime_error("mmf: distill: vocabulary or number of slots out of range");
  typed_mode(a, [&](auto tag, auto mode) {
    using T = decltype(tag);
    const int64_t bytes = static_cast<int64_t>(a.vocab) * sizeof(T);
    int blocks = blocks_of_row(bytes, slot_bytes(a.top));
    while (blocks < kMaxCluster && a.rows * blocks < 148 && bytes / blocks > kSliceLeast) ++blocks;
    if (a.rows > 0x7fffffff) throw std::runtime_error("mmf: distill: too many rows");
    const int each = (a.vocab / Vec<T>::N + blocks - 1) / blocks;
    const int smem = each * 16 + slot_bytes(a.top);
    auto kernel = distill_rows_kernel<T, decltype(mode)::value>;
    allow_shared(reinterpret_cast<const void*>(kernel), smem, /*carveout=*/true);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.rows), static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.z = 1;
    attr[0].val.clusterDim.y = static_cast<unsigned>(blocks);
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.behind_count ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, a, scales(a), each, error_word());
  });
  check("distill_rows");
}

void distill_grad(const DistillArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return;
  if (a.top < 1 || a.top > kMaxTop) throw std::runtime_error("mmf: distill: number of slots out of range");
  typed_mode(a, [&](auto tag, auto mode) {
    using T = decltype(tag);
    const int segments = std::max(1, (a.vocab / Vec<T>::N + kSegment - 1) / kSegment);
    if (a.rows > 0x7fffffff || segments > 65535) throw std::runtime_error("mmf: distill: too many rows");
    distill_grad_kernel<T, decltype(mode)::value>
        <<<dim3(static_cast<unsigned>(a.rows), static_cast<unsigned>(segments)), kThreads, slot_bytes(a.top), stream>>>(
            a, scales(a), error_word());
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
