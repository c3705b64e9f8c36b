// The backward of the fused block norms (block_norm.cu):
//
//   a  = dn w_pre,  dH = dh + r_h (a - h^ mean(a h^) [- mean(a)]),  dx = residual_scale dH
//   dp = branch_scale gate dH,  b = dp w_post,  dy = r_y (b - y^ mean(b y^) [- mean(b)])
//   dw_pre = sum dn h^, db_pre = sum dn, dw_post = sum dp y^, db_post = sum dp,
//   dgate = branch_scale sum dH p over the rows that share the gate
//
// with the means in [] for layer norms alone.  y^ and h^ are the normalised rows, from y, x and the
// forward's statistics: h is formed again from x and y rather than read back, the same bytes without
// the rounding of the stored h.
//
// Where rows share a gate, its gradient and that of the post norm come from the same column sums A =
// sum dH y^ and B = sum dH over those rows: dgate = branch_scale (w_post A + b_post B), dw_post +=
// branch_scale gate A, db_post += branch_scale gate B.
//
// Bound by memory: dh, dn, x and y are read once, dx and dy written once.  A worker (a group of
// threads that shares a row) walks over a run of rows, whose data are copied ahead into shared memory,
// each thread its own vectors, so that others are on their way while it is at one or two rows' two
// reductions.  Sums over rows stay in registers, 8 columns a thread, and leave once, as one partial row a
// worker (one a run for the gate).  Rows of more than 8 x 512 columns are shared by the blocks of a
// cluster, which exchange the sums of their shares: 8192 x 8192 bf16 233 us (gate for each token 281),
// where one block with 16 columns a thread had no registers left for the weights, 330 (303).  Narrower rows
// are not: at 4096 columns two blocks took 126 us, the exchange being slower than one block's barrier.  A
// second kernel adds the partials in a fixed order, so that equal calls give equal bits.  8192 x 4096 bf16
// with both norms and a gate: 93 us (403 MB, 66 % of the copy rate), and 5.5 for the sums.  One block fills an
// SM's registers (128 a thread); its warps issue in 57 % of the cycles, the fp32 pipe is 29 % busy, and what
// they wait for is mostly their own arithmetic and shared memory, two reductions a turn with little else to
// do beside them.  Layer norms, one row a turn, 143 us; fp32 146, layer 162.  With one row a turn 5 us more;
// unpacked arithmetic, sums in shared memory and no copies ahead 152; 16 columns a thread and two blocks an SM,
// weights loaded again for each row, 140.
#include <algorithm>
#include <stdexcept>
#include <string>

#include "block_norm.cuh"
#include "launch_info.h"
#include "tc_common.cuh"

namespace mmf {

namespace {

// Rows are dealt out in chunks of `chunk_rows` that do not cross a gate's group of rows.
struct Plan {
  int groups, group_rows;  // of rows that share a gate (one group of all rows where none is shared)
  int per_group, chunk_rows, chunks;
};

struct BwdParts {
  float *post_w, *post_b, *pre_w, *pre_b;  // [workers][cols] each, or null
  float* gate;                              // [chunks][cols], or null
};

// What a stage of the copies holds.
enum { IN_DN, IN_DH, IN_X, IN_Y, IN_GATE, INPUTS };

// Rows that a worker takes in one turn (with a layer norm's sums there is no room for two).
template <bool LN>
constexpr int kRows = LN ? 1 : 2;

// What blocks that share a row tell one another: the sums of their shares, asynchronous stores that
// count their bytes on the receiver's barrier.  Two places in turn: a block that is one reduction ahead
// has the others' parts of that one, which they send when all their threads have read the last.
template <int BLOCKS>
struct Shares {
  float2 part[2][BLOCKS];
  uint64_t bar[2];
};

// BLOCKS: of a cluster that shares each row, as many columns each (1: a row has one block, or less).
template <typename T, int VEC, int NV, bool LN, int BLOCKS>
__global__ void __launch_bounds__(kMaxThreads, 1) block_norm_bwd_kernel(const BlockNormBwdArgs a, const Plan plan,
                                                                        const BwdParts parts, int tpr, int inputs,
                                                                        int stages, int* err) {
  constexpr int N = NV * VEC, H = N / 2;
  constexpr int ROWS = kRows<LN>;  // in one turn, so that they share its barriers
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(16) float red[2 * 4 * 32];
  using R = Raw<T, VEC>;
  using V = Values<N>;
  RowGroup g(tpr, red);
  const int cols = a.cols, threads = static_cast<int>(blockDim.x);
  const int groups = threads / tpr;
  const int rank = BLOCKS > 1 ? static_cast<int>(blockIdx.y) : 0;
  const int worker = static_cast<int>(blockIdx.x) * groups + g.row, workers = static_cast<int>(gridDim.x) * groups;
  // the block's columns
  const int share = BLOCKS > 1 ? share_of(cols, BLOCKS, VEC) : cols, base = rank * share, end = min(base + share, cols);
  __shared__ Shares<BLOCKS> notes;
  [[maybe_unused]] constexpr uint32_t kBytes = (BLOCKS - 1) * sizeof(float2);  // of the others' parts
  [[maybe_unused]] uint32_t reductions = 0;
  if constexpr (BLOCKS > 1) {
    if (threadIdx.x == 0) {
      mbar_init(&notes.bar[0], 1);
      mbar_init(&notes.bar[1], 1);
      fence_mbar_init();
      mbar_arrive_expect_tx(&notes.bar[0], kBytes);
      mbar_arrive_expect_tx(&notes.bar[1], kBytes);
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  // sums over a row, the same bits in every thread that has it
  auto total = [&](auto& t) {
    g.sum(t);
    if constexpr (BLOCKS > 1) {
      constexpr int M = sizeof(t) / sizeof(float);
      const uint32_t at = reductions & 1, phase = reductions >> 1 & 1;
      ++reductions;
      static_assert(M <= 2, "");
      const float2 mine = make_float2(t[0], t[M - 1]);
      if (threadIdx.x < BLOCKS && static_cast<int>(threadIdx.x) != rank)
        cluster_send(&notes.part[at][rank], &notes.bar[at], static_cast<int>(threadIdx.x), mine);
      mbar_wait(&notes.bar[at], phase, err, ERR_PEER_FLAG_TIMEOUT, MMF_WAIT_TIMEOUT_NS, false);
      float2 sum = make_float2(0.f, 0.f);  // in the order of the blocks, the same in each of them
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i) sum = fadd2(sum, i == rank ? mine : notes.part[at][i]);
      t[0] = sum.x;
      if constexpr (M > 1) t[1] = sum.y;
      if (threadIdx.x == 0) mbar_arrive_expect_tx(&notes.bar[at], kBytes);
    }
  };
  const T* pw = static_cast<const T*>(a.post_w);
  const T* pb = static_cast<const T*>(a.post_b);
  const T* nw = static_cast<const T*>(a.pre_w);
  const bool gated = a.gate != nullptr, token_gate = gated && a.rows_per_gate == 1;
  // stage s's vector k of row r's input i is place(s, r)[(i * NV + k) * threads]; what is not copied there
  // is 0
  auto place = [&](int stage, int r) {
    return reinterpret_cast<R*>(smem) + threadIdx.x + (stage * ROWS + r) * (inputs * NV) * threads;
  };
  auto clear = [&](int stage, int r) {
    for (int i = 0; i < inputs * NV; ++i) place(stage, r)[i * threads] = R{};
  };
  for (int i = 0; i < stages; ++i)
    for (int r = 0; r < ROWS; ++r) clear(i, r);
  auto col = [&](int k) { return base + (g.lane + k * tpr) * VEC; };

  // the worker's rows: chunk after chunk, as many turns for every worker of the block
  const int rounds = (plan.chunks + workers - 1) / workers;
  const int turns = rounds * ((plan.chunk_rows + ROWS - 1) / ROWS);
  struct Cursor {
    int chunk, i, first, rows;  // row first + i of the chunk's `rows`; none behind the last chunk
  };
  auto start = [&](int chunk) {
    const int group = chunk / plan.per_group;
    const int at = (chunk - group * plan.per_group) * plan.chunk_rows;  // within the group
    return Cursor{chunk, 0, group * plan.group_rows + at,
                  chunk < plan.chunks ? min(plan.chunk_rows, plan.group_rows - at) : 0};
  };
  auto step = [&](Cursor& c) {
    if ((c.i += ROWS) >= plan.chunk_rows) c = start(c.chunk + workers);
  };
  Cursor ahead = start(worker), now = ahead;
  int put = 0, get = 0;  // stages
  auto copy = [&](int turn) {
    if (turn < turns) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (ahead.i + r < ahead.rows) {
          const int64_t off = static_cast<int64_t>(ahead.first + ahead.i + r) * cols + col(0);
          R* to = place(put, r);
          auto fetch = [&](int i, const void* from) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
              if (col(k) < end)
                copy_ahead<T, VEC>(to + (i * NV + k) * threads, static_cast<const T*>(from) + off + k * tpr * VEC);
          };
          if (nw) {
            fetch(IN_DN, a.dn);
            fetch(IN_X, a.x);
          }
          if (a.dh) fetch(IN_DH, a.dh);
          if (pw || gated || nw) fetch(IN_Y, a.y);
          if (token_gate) fetch(IN_GATE, a.gate);
        } else {
          clear(put, r);
        }
      }
      step(ahead);
      if (++put == stages) put = 0;
    }
    end_copies();  // one group a turn, empty or not
  };
  // a column vector (1 where there is none), 0 behind the row's end
  auto column = [&](const void* p, V& v) {
    v.fill(1.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (col(k) >= end)
        v.template put<T, VEC>(k, R{});
      else if (p)
        v.template put<T, VEC>(k, ld_raw<T, VEC>(static_cast<const T*>(p) + col(k)));
    }
  };
  auto flush = [&](const V& v, float* to) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (col(k) < end) {
        constexpr int P = VEC < 4 ? VEC : 4;
#pragma unroll
        for (int e = 0; e < VEC; e += P) {
          float f[P];
#pragma unroll
          for (int o = 0; o < P; ++o) f[o] = (k * VEC + e + o) % 2 ? v.p[(k * VEC + e + o) / 2].y : v.p[(k * VEC + e + o) / 2].x;
          st_raw<float, P>(to + col(k) + e, pack<float, P>(f));
        }
      }
    }
  };

  V sum_a, sum_n, sum_pw;
  [[maybe_unused]] V sum_b, sum_nb, sum_pb;
  sum_a.fill(0.f);
  sum_n.fill(0.f);
  sum_pw.fill(0.f);
  if constexpr (LN) {
    sum_b.fill(0.f);
    sum_nb.fill(0.f);
    sum_pb.fill(0.f);
  }
  // branch_scale gate times the post norm's weight (d h / d y^), or times its bias (0 where there is none)
  auto times = [&](const V& gate, const T* p, V& to) {
    column(p, to);
#pragma unroll
    for (int i = 0; i < H; ++i) to.p[i] = fmul2(both(a.branch_scale), fmul2(gate.p[i], to.p[i]));
  };
  [[maybe_unused]] V kept_pre, kept_scale, kept_shift;
  column(nw, kept_pre);
  const float inv = 1.f / cols;
  const int rows_per_gate = static_cast<int>(a.rows_per_gate);
  auto load_stats = [&](const Cursor& c, Stat (&y)[ROWS], Stat (&h)[ROWS]) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const bool there = c.i + r < c.rows;
      y[r] = there && pw ? Stat::load<LN>(a.stat_y, c.first + c.i + r) : Stat{1.f, 0.f};
      h[r] = there && nw ? Stat::load<LN>(a.stat_h, c.first + c.i + r) : Stat{0.f, 0.f};
    }
  };
  Stat next_y[ROWS], next_h[ROWS];
  load_stats(now, next_y, next_h);
  // with one stage rows' copies start when those before have been read, else a turn or two earlier
  for (int i = 0; i < stages - 1; ++i) copy(i);
  for (int turn = 0; turn < turns; ++turn) {
    copy(turn + stages - 1);
    wait_copies(stages - 1);
    auto input = [&](int r, int i, V& v) {
      const R* here = place(get, r);
#pragma unroll
      for (int k = 0; k < NV; ++k) v.template put<T, VEC>(k, here[(i * NV + k) * threads]);
    };
    auto store = [&](int r, void* to, const V& v) {
      const int64_t off = static_cast<int64_t>(now.first + now.i + r) * cols;
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (now.i + r < now.rows && col(k) < end)
          st_raw<T, VEC>(static_cast<T*>(to) + off + col(k), v.template get<T, VEC>(k));
    };
    if (now.i == 0) {  // of a chunk; where each row has its own gate that comes in with the row
      V gate;
      column(gated && !token_gate
                 ? static_cast<const T*>(a.gate) + static_cast<int64_t>(now.rows > 0 ? now.first / rows_per_gate : 0) * cols
                 : nullptr, gate);
      times(gate, pw, kept_scale);
      if constexpr (LN) times(gate, pb, kept_shift);
    }
    auto with_gate = [&](int r, const V& kept, V& v) {
      v = kept;
      if (token_gate) {
        V gate;
        input(r, IN_GATE, gate);
#pragma unroll
        for (int i = 0; i < H; ++i) v.p[i] = fmul2(gate.p[i], v.p[i]);
      }
    };
    // the next rows' statistics are on their way while these are used
    Stat sy[ROWS], sh[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      sy[r] = next_y[r];
      sh[r] = next_h[r];
    }
    {
      Cursor after = now;
      step(after);
      load_stats(after, next_y, next_h);
    }
    auto load_y = [&](int r, V& u) {  // y^ (y without a post norm)
      input(r, IN_Y, u);
      if (pw) {
        const float2 s = both(sy[r].rstd), m = both(-sy[r].mean * sy[r].rstd);
#pragma unroll
        for (int i = 0; i < H; ++i) u.p[i] = LN ? ffma2(u.p[i], s, m) : fmul2(u.p[i], s);
      }
    };
    auto load_h = [&](int r, const V& u, V& h) {  // h^
      V w;
      with_gate(r, kept_scale, w);
#pragma unroll
      for (int i = 0; i < H; ++i) h.p[i] = fmul2(u.p[i], w.p[i]);
      if (LN && pb) {
        with_gate(r, kept_shift, w);
#pragma unroll
        for (int i = 0; i < H; ++i) h.p[i] = fadd2(h.p[i], w.p[i]);
      }
      input(r, IN_X, w);
      const float2 s = both(sh[r].rstd), m = both(-sh[r].mean * sh[r].rstd), rho = both(a.residual_scale);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        h.p[i] = ffma2(rho, w.p[i], h.p[i]);
        h.p[i] = LN ? ffma2(h.p[i], s, m) : fmul2(h.p[i], s);
      }
    };
    constexpr int SUMS = LN ? 2 : 1;
    float t[ROWS * SUMS];
    V u[ROWS], d[ROWS];  // y^; dn w_pre, then dH, then d h / d (y^)
    if (nw) {
      V h[ROWS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        load_y(r, u[r]);
        load_h(r, u[r], h[r]);
        input(r, IN_DN, d[r]);
        float2 s1 = both(0.f), s2 = both(0.f);
#pragma unroll
        for (int i = 0; i < H; ++i) {
          sum_n.p[i] = ffma2(d[r].p[i], h[r].p[i], sum_n.p[i]);
          if constexpr (LN) sum_nb.p[i] = fadd2(d[r].p[i], sum_nb.p[i]);
          d[r].p[i] = fmul2(d[r].p[i], kept_pre.p[i]);
          if (LN) s1 = fadd2(d[r].p[i], s1);
          s2 = ffma2(d[r].p[i], h[r].p[i], s2);
        }
        t[r * SUMS] = s2.x + s2.y;
        if constexpr (LN) t[r * SUMS + 1] = s1.x + s1.y;
      }
      total(t);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        V dh;
        input(r, IN_DH, dh);
        const float k = -sh[r].rstd * inv;
        const float2 s = both(sh[r].rstd), c2 = both(k * t[r * SUMS]);
#pragma unroll
        for (int i = 0; i < H; ++i) {
          d[r].p[i] = ffma2(s, d[r].p[i], dh.p[i]);
          d[r].p[i] = ffma2(c2, h[r].p[i], d[r].p[i]);
          if constexpr (LN) d[r].p[i] = fadd2(both(k * t[r * SUMS + 1]), d[r].p[i]);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        load_y(r, u[r]);
        input(r, IN_DH, d[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (a.dx) {
        V x;
#pragma unroll
        for (int i = 0; i < H; ++i) x.p[i] = fmul2(both(a.residual_scale), d[r].p[i]);
        store(r, a.dx, x);
      }
      if (token_gate) {
        // each row's own gate: its gradient goes out with the row, A and B take it in
        V gate, x;
        input(r, IN_GATE, gate);
        if (a.dgate) {
#pragma unroll
          for (int i = 0; i < H; ++i) x.p[i] = fmul2(kept_scale.p[i], u[r].p[i]);
          if (LN && pb) {
#pragma unroll
            for (int i = 0; i < H; ++i) x.p[i] = fadd2(x.p[i], kept_shift.p[i]);
          }
#pragma unroll
          for (int i = 0; i < H; ++i) x.p[i] = fmul2(x.p[i], d[r].p[i]);
          store(r, a.dgate, x);
        }
#pragma unroll
        for (int i = 0; i < H; ++i) {
          const float2 x = fmul2(d[r].p[i], gate.p[i]);
          sum_a.p[i] = ffma2(x, u[r].p[i], sum_a.p[i]);
          if constexpr (LN) sum_b.p[i] = fadd2(x, sum_b.p[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < H; ++i) {
          sum_a.p[i] = ffma2(d[r].p[i], u[r].p[i], sum_a.p[i]);
          if constexpr (LN) sum_b.p[i] = fadd2(d[r].p[i], sum_b.p[i]);
        }
      }
      V scale;
      with_gate(r, kept_scale, scale);
      float2 s1 = both(0.f), s2 = both(0.f);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        d[r].p[i] = fmul2(d[r].p[i], scale.p[i]);
        if (LN) s1 = fadd2(d[r].p[i], s1);
        s2 = ffma2(d[r].p[i], u[r].p[i], s2);
      }
      t[r * SUMS] = s2.x + s2.y;
      if constexpr (LN) t[r * SUMS + 1] = s1.x + s1.y;
    }
    if (pw) total(t);
    if (a.dy) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (pw) {
          const float k = -sy[r].rstd * inv;
          const float2 s = both(sy[r].rstd), c2 = both(k * t[r * SUMS]);
#pragma unroll
          for (int i = 0; i < H; ++i) {
            d[r].p[i] = ffma2(c2, u[r].p[i], fmul2(s, d[r].p[i]));
            if constexpr (LN) d[r].p[i] = fadd2(both(k * t[r * SUMS + 1]), d[r].p[i]);
          }
        }
        store(r, a.dy, d[r]);
      }
    }

    if (now.i + ROWS >= plan.chunk_rows) {  // the chunk's sums
      V gate, w;
      if (token_gate) {
        gate.fill(1.f);
      } else {
        const int64_t at = static_cast<int64_t>(now.rows > 0 ? now.first / rows_per_gate : 0) * cols;
        column(gated ? static_cast<const T*>(a.gate) + at : nullptr, gate);
      }
      if (parts.gate && now.chunk < plan.chunks) {
        V t;
        column(pw, w);
#pragma unroll
        for (int i = 0; i < H; ++i) t.p[i] = fmul2(w.p[i], sum_a.p[i]);
        if constexpr (LN) {
          if (pb) {
            column(pb, w);
#pragma unroll
            for (int i = 0; i < H; ++i) t.p[i] = ffma2(w.p[i], sum_b.p[i], t.p[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < H; ++i) t.p[i] = fmul2(both(a.branch_scale), t.p[i]);
        flush(t, parts.gate + static_cast<int64_t>(now.chunk) * cols);
      }
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float2 k = fmul2(both(a.branch_scale), gate.p[i]);
        sum_pw.p[i] = ffma2(k, sum_a.p[i], sum_pw.p[i]);
        if constexpr (LN) sum_pb.p[i] = ffma2(k, sum_b.p[i], sum_pb.p[i]);
      }
      sum_a.fill(0.f);
      if constexpr (LN) sum_b.fill(0.f);
    }
    step(now);
    if (++get == stages) get = 0;
  }
  const int64_t at = static_cast<int64_t>(worker) * cols;
  if (parts.post_w) flush(sum_pw, parts.post_w + at);
  if (parts.pre_w) flush(sum_n, parts.pre_w + at);
  if constexpr (LN) {
    if (parts.post_b) flush(sum_pb, parts.post_b + at);
    if (parts.pre_b) flush(sum_nb, parts.pre_b + at);
  }
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
#pragma unroll 8
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

constexpr int kSharedMost = 224 << 10;

// The launch of a width: what it needs of the device, and how rows are dealt out.
struct Backward {
  static constexpr int kValues = 8;  // a thread
  // Whether four blocks take a row that is too wide for one: four with up to 5 warps each, of which an SM holds three,
  // else two.  8192 x 5120 bf16 157 us with four and 198 with two (layer norms 232 and 316), 8192 x 6144, where an
  // SM holds two of four, 224 and 202.
  static bool four_blocks(int cols) { return cols <= 4 * 160 * kValues; }
  const BlockNormBwdArgs& a;
  cudaStream_t stream;
  int64_t* need;  // non-null: only count the scratch values

  template <typename T, int VEC, int NV, bool LN, int BLOCKS = 1>
  void run(int tpr) const {
    auto kernel = block_norm_bwd_kernel<T, VEC, NV, LN, BLOCKS>;
    const int groups = BLOCKS == 1 && tpr < 128 ? 128 / tpr : 1, block = groups * tpr;  // narrow rows: several to a block
    // two turns' rows copied ahead, one or none where they are too wide for that; small blocks leave room for
    // a second one on the SM (8192 x 2048 bf16 with a gate for each token: 56 us, 80 with one and three stages)
    const int inputs = a.gate && a.rows_per_gate == 1 ? INPUTS : INPUTS - 1;
    const int stage = kRows<LN> * inputs * NV * VEC * static_cast<int>(sizeof(T)) * block;
    const int stages = std::max(1, std::min(3, kSharedMost / (block <= 256 ? 2 : 1) / stage));
    const int smem = stages * stage;
    // workers on the device at once
    const void* k = reinterpret_cast<const void*>(kernel);
    const int most = BLOCKS > 1 ? resident_clusters(k, block, smem, BLOCKS) : 148 * resident_blocks(k, block, smem) * groups;
    Plan p;
    const bool shared_gate = a.gate && a.rows_per_gate > 1, gate_sum = shared_gate && a.dgate;
    p.groups = static_cast<int>(shared_gate ? a.rows / a.rows_per_gate : 1);
    p.group_rows = static_cast<int>(shared_gate ? a.rows_per_gate : a.rows);
    // one chunk a worker while the groups are few; with many groups several smaller ones, so that
    // the last round is not mostly idle
    p.per_group = p.groups <= most / 4 ? most / p.groups : (4 * most - 1) / p.groups + 1;
    p.per_group = std::min(p.per_group, p.group_rows);
    p.chunk_rows = (p.group_rows + p.per_group - 1) / p.per_group;
    p.per_group = (p.group_rows + p.chunk_rows - 1) / p.chunk_rows;
    p.chunks = p.groups * p.per_group;
    const int workers = std::min(most, (p.chunks + groups - 1) / groups * groups);

    int64_t used = 0;
    auto take = [&](bool want, int rows) {
      float* at = want && !need ? a.parts + used : nullptr;
      if (want) used += static_cast<int64_t>(rows) * a.cols;
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
    int device = 0;
    cudaGetDevice(&device);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(workers / groups), BLOCKS);
    cfg.blockDim = dim3(static_cast<unsigned>(block));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = attr.val.clusterDim.z = 1;
    attr.val.clusterDim.y = BLOCKS;
    cfg.attrs = &attr;
    cfg.numAttrs = BLOCKS > 1 ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, a, p, parts, tpr, inputs, stages, device_error_word(device));
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
    int gates = gate_sum ? p.groups : 0;
    if (jobs.count + gates == 0) return;
    const dim3 threads(32, 8);
    while (true) {
      const int now = std::min(gates, 32768);
      block_norm_sum_kernel<T>
          <<<dim3((a.cols + 31) / 32, static_cast<unsigned>(jobs.count + now)), threads, 0, stream>>>(jobs, a.cols);
      check("block_norm_bwd (sums)");
      gates -= now;
      if (gates == 0) return;
      jobs.count = 0;
      jobs.gate.part += static_cast<int64_t>(now) * p.per_group * a.cols;
      jobs.gate.out = static_cast<T*>(jobs.gate.out) + static_cast<int64_t>(now) * a.cols;
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
  if (a.rows > 0x3fffffff) throw std::runtime_error("mmf: block_norm_bwd: too many rows");
  const void* rows[] = {a.dh, a.dn, a.x, a.y, a.post_w, a.post_b, a.gate, a.pre_w, a.dx, a.dy, a.dgate};
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
