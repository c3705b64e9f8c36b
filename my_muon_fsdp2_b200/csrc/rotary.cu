// Rotary positions of q and k in one launch: neighbouring or half-apart pairs, the whole head or
// its first rotary_dim values, any frequencies, forward, backward (the transpose) and in place.
//
//   (x1, x2) -> m (x1 cos a - x2 sin a, x2 cos a + x1 sin a),   a = position * frequency_i
//
// The angle.  At far positions a = position * frequency loses its fraction of a turn in fp32 (at
// 10^5 radians one ulp is 0.008).  The frequencies therefore come as turns per position in 64-bit
// fixed point (frequency / 2 pi * 2^64); position * turns modulo 2^64 is the fraction of a turn,
// exact but for the rounding of the table (2^-53 of the frequency), one integer multiply, no range
// reduction.  Its upper 32 bits, as a signed fraction of half a turn, go to sincospi.  From there on all is
// fp32: the fraction is rounded to it (2^-25 of half a turn, 1e-7 in the angle), cos and sin and their product with
// the magnitude are.  That is enough for 16 bits and shows in fp32 outputs alone: with a magnitude their error
// is 5.6e-8 of the values' size, against 4.6e-8 for cos and sin formed in 64 bits and rounded once.
//
// Bound by memory: q and k are read once and written once, 3 flops a value.  A block takes a few
// tokens; its threads first compute each token's cos and sin once (a head's worth, shared by all
// heads) into shared memory, then each thread keeps one vector position of one token in registers
// and walks over about ten heads, so that sincos is paid once for all heads.  Two heads in flight a
// thread and four blocks an SM: 8192 tokens x 40 heads x 128 bf16 take 31.6 us (81 % of the copy rate;
// with four heads in flight and two blocks an SM 43.7), 32768 x 20 x 128 fp32 105 us (97 %).  Where part of
// the head passes through, the threads that copy it have one load in flight: 3069 tokens x 40 heads x 64
// fp16, half rotated, 12.3 us (39 %).
#include <stdexcept>
#include <string>

#include "kernels.h"
#include "typed_io.cuh"

namespace mmf {

namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 10;  // about as many for each thread
constexpr int kUnroll = 2;  // of them in flight

template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(const RotaryArgs a, int units, int head_lanes,
                                                          int block_tokens) {
  extern __shared__ float cs[];  // [block_tokens][half] cos, then the same of sin
  const int half = a.rotary_dim >> 1;
  const uint32_t first = blockIdx.x * block_tokens;  // the launcher keeps batch * seq below 2^31
  const int here = min(block_tokens, static_cast<int>(a.batch * a.seq - first));
  float* sn = cs + block_tokens * half;
  for (int e = threadIdx.x; e < here * half; e += kThreads) {
    const int j = e / half, i = e - j * half;
    const int64_t b = (first + j) / a.seq, t = (first + j) % a.seq;
    int64_t pos = t;
    if (a.positions)
      pos = a.positions_32 ? static_cast<const int*>(a.positions)[b * a.pos_stride_b + t * a.pos_stride_t]
                           : static_cast<const int64_t*>(a.positions)[b * a.pos_stride_b + t * a.pos_stride_t];
    const uint64_t turn = static_cast<uint64_t>(pos) * a.turns[i];  // modulo one turn
    float s, c;
    sincospif(static_cast<float>(static_cast<int>(turn >> 32)) * 0x1p-31f, &s, &c);
    cs[e] = c * a.magnitude;
    sn[e] = s * (a.inverse ? -a.magnitude : a.magnitude);
  }
  __syncthreads();

  const int unit = threadIdx.x % units;
  const int rest = threadIdx.x / units;
  const int lane = rest % head_lanes, j = rest / head_lanes;
  if (j >= here) return;
  const int64_t b = (first + j) / a.seq, t = (first + j) % a.seq;
  const T* qi = static_cast<const T*>(a.q_in) + b * a.q_in_s[0] + t * a.q_in_s[1];
  const T* ki = static_cast<const T*>(a.k_in) + b * a.k_in_s[0] + t * a.k_in_s[1];
  T* qo = static_cast<T*>(a.q_out) + b * a.q_out_s[0] + t * a.q_out_s[1];
  T* ko = static_cast<T*>(a.k_out) + b * a.k_out_s[0] + t * a.k_out_s[1];
  const int heads = a.q_heads + a.k_heads;
  const int step = head_lanes * gridDim.y;
  const int rot_units = (INTERLEAVED ? a.rotary_dim : half) / VEC;
  // a head's place, q's heads before k's
  auto src = [&](int h) {
    return h < a.q_heads ? qi + h * a.q_in_s[2] : ki + (h - a.q_heads) * a.k_in_s[2];
  };
  auto dst = [&](int h) {
    return h < a.q_heads ? qo + h * a.q_out_s[2] : ko + (h - a.q_heads) * a.k_out_s[2];
  };
  const int h0 = lane + blockIdx.y * head_lanes;

  if (unit >= rot_units) {  // the part of the head that passes through (out of place only)
    const int off = a.rotary_dim + (unit - rot_units) * VEC;
    for (int h = h0; h < heads; h += step) st_raw<T, VEC>(dst(h) + off, ld_raw<T, VEC>(src(h) + off));
    return;
  }
  if constexpr (INTERLEAVED) {
    constexpr int P = VEC / 2;
    const int off = unit * VEC;
    float c[P], s[P];
#pragma unroll
    for (int e = 0; e < P; ++e) {
      c[e] = cs[j * half + unit * P + e];
      s[e] = sn[j * half + unit * P + e];
    }
    for (int h = h0; h < heads; h += step * kUnroll) {
      Raw<T, VEC> r[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (h + u * step < heads) r[u] = ld_raw<T, VEC>(src(h + u * step) + off);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (h + u * step < heads) {
          float v[VEC], o[VEC];
          unpack<T, VEC>(r[u], v);
#pragma unroll
          for (int e = 0; e < P; ++e) {
            o[2 * e] = v[2 * e] * c[e] - v[2 * e + 1] * s[e];
            o[2 * e + 1] = v[2 * e + 1] * c[e] + v[2 * e] * s[e];
          }
          st_raw<T, VEC>(dst(h + u * step) + off, pack<T, VEC>(o));
        }
      }
    }
  } else {
    const int off = unit * VEC;
    float c[VEC], s[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      c[e] = cs[j * half + off + e];
      s[e] = sn[j * half + off + e];
    }
    for (int h = h0; h < heads; h += step * kUnroll) {
      Raw<T, VEC> r1[kUnroll], r2[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (h + u * step < heads) {
          r1[u] = ld_raw<T, VEC>(src(h + u * step) + off);
          r2[u] = ld_raw<T, VEC>(src(h + u * step) + half + off);
        }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (h + u * step < heads) {
          float v1[VEC], v2[VEC], o1[VEC], o2[VEC];
          unpack<T, VEC>(r1[u], v1);
          unpack<T, VEC>(r2[u], v2);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            o1[e] = v1[e] * c[e] - v2[e] * s[e];
            o2[e] = v2[e] * c[e] + v1[e] * s[e];
          }
          st_raw<T, VEC>(dst(h + u * step) + off, pack<T, VEC>(o1));
          st_raw<T, VEC>(dst(h + u * step) + half + off, pack<T, VEC>(o2));
        }
      }
    }
  }
}

// Whether every row that the kernel touches starts and steps on `bytes` boundaries.
bool rows_on(const RotaryArgs& a, int elem, int bytes) {
  auto ok = [&](const void* p, const int64_t* s, int heads) {
    if (heads == 0) return true;
    if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
    for (int i = 0; i < 3; ++i)
      if (s[i] * elem % bytes) return false;
    return true;
  };
  return ok(a.q_in, a.q_in_s, a.q_heads) && ok(a.k_in, a.k_in_s, a.k_heads) && ok(a.q_out, a.q_out_s, a.q_heads) &&
         ok(a.k_out, a.k_out_s, a.k_heads);
}

template <typename T, int VEC, bool INTERLEAVED>
void launch(const RotaryArgs& a, cudaStream_t stream) {
  const int half = a.rotary_dim / 2;
  const int tail = a.in_place ? 0 : (a.head_dim - a.rotary_dim) / VEC;
  const int units = (INTERLEAVED ? a.rotary_dim : half) / VEC + tail;
  if (units > kThreads)
    throw std::runtime_error("mmf: rotary: head_dim is too large for its alignment");
  const int heads = a.q_heads + a.k_heads;
  const int64_t tokens = static_cast<int64_t>(a.batch) * a.seq;
  // about kHeads heads for each thread; the rest of the block takes more tokens
  int lanes = (heads + kHeads - 1) / kHeads;
  if (lanes * units > kThreads) lanes = kThreads / units;
  int block_tokens = kThreads / (lanes * units);
  if (block_tokens > tokens) block_tokens = static_cast<int>(tokens);
  const int64_t blocks = (tokens + block_tokens - 1) / block_tokens;
  if (tokens > 0x7fffffff) throw std::runtime_error("mmf: rotary: too many tokens");
  const size_t smem = static_cast<size_t>(block_tokens) * half * 2 * sizeof(float);
  // few tokens: the heads are split over blocks too, each computing the angles for itself (1 token of
  // 40 heads x 128: 2.1 us, 5.1 unsplit; 128 tokens 3.2, 6.4 unsplit)
  int splits = 1;
  while (blocks * splits < 148 && lanes * splits < heads) splits *= 2;
  rotary_kernel<T, VEC, INTERLEAVED>
      <<<dim3(static_cast<unsigned>(blocks), splits), kThreads, smem, stream>>>(a, units, lanes, block_tokens);
}

template <typename T, bool INTERLEAVED>
void dispatch_vec(const RotaryArgs& a, cudaStream_t stream) {
  constexpr int E = static_cast<int>(sizeof(T));
  const int part = INTERLEAVED ? a.rotary_dim : a.rotary_dim / 2;
  // the widest access that divides the rotated part, the rest of the head, and every row's start
  auto fits = [&](int vec) {
    return part % vec == 0 && (a.in_place || (a.head_dim - a.rotary_dim) % vec == 0) && rows_on(a, E, vec * E);
  };
  if (fits(16 / E)) return launch<T, 16 / E, INTERLEAVED>(a, stream);
  if (E == 2 && fits(4)) return launch<T, 4, INTERLEAVED>(a, stream);
  if (fits(2)) return launch<T, 2, INTERLEAVED>(a, stream);
  if constexpr (!INTERLEAVED) return launch<T, 1, INTERLEAVED>(a, stream);
  throw std::runtime_error("mmf: rotary: neighbouring pairs need rows that start on a pair's boundary");
}

}  // namespace

void rotary(const RotaryArgs& a, cudaStream_t stream) {
  if (a.batch == 0 || a.seq == 0 || a.q_heads + a.k_heads == 0) return;
  auto go = [&](auto t) {
    using T = decltype(t);
    if (a.interleaved)
      dispatch_vec<T, true>(a, stream);
    else
      dispatch_vec<T, false>(a, stream);
  };
  if (a.dtype == DType::BF16)
    go(__nv_bfloat16());
  else if (a.dtype == DType::F16)
    go(__half());
  else
    go(float());
  count_launch();
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("mmf: rotary launch failed: ") + cudaGetErrorString(e));
}

}  // namespace mmf
