// RMS norm per head, then rotary positions with several axes (time, height, width), on queries and keys in one launch, and
// the gradient.  Pair i of the P pairs of channels belongs to one axis and turns by the angle
//
//   a_i = position[axis(i)] * 2 pi * turns_i          (turns_i: the pair's frequency in full turns per unit of position)
//   (u, v) -> (u cos a_i - v sin a_i, v cos a_i + u sin a_i)
//
// with u, v the channels i and i + P, or 2 i and 2 i + 1; channels behind 2 P are passed on.  The norm before it is
// n_j = x_j * r * w_j, r = 1 / sqrt(mean x^2 + eps), as in producer.cu (the reference's fused qk-norm and rotary kernel,
// anemoi/models/minimax_h3/solengine/models/minimax_h3/optimized/fusions.py:208-274, which takes tables of cosines and
// sines).  Gradient: g = the output's, turned back (angle -a); w's is sum g_j x_j r; with b = g w the input's is
// r (b - x r mean(b x r)).
//
// The angle is reduced to a fraction of a turn before it is rounded to fp32, where a product in fp32 has no bits left beyond
// positions of 2^24.  Whole positions: the frequency is a 64-bit fraction of a turn, and the low 64 bits of its product with
// the position are the angle's fraction (a position of 2^31 is 2^-22 of a turn off, as the frequency is a double's 53 bits).
// Fractional positions: the same in double precision.  Of the fraction, within half
// a turn, the fast cosine and sine are good to 2^-20.
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/anemoi_sm100.h"
#include "layer.cuh"
#include "rows.cuh"

namespace {

using namespace rows;

constexpr int kThreads = 256;

struct RopeParams {
  const void *q, *k, *dq_out, *dk_out, *q_weight, *k_weight, *positions;
  void *q_out, *k_out;
  float* weight_partial;  // [blocks of queries, then of keys][D]
  int64_t position_batch;
  uint32_t batch, tokens;
  int64_t strides[6][3];  // forward: q, k, q_out, k_out; gradient: dq_out, dk_out, q, k, dq, dk
  int q_heads, k_heads, axes, pairs, interleaved, positions_type, q_blocks;
  float eps;
  int ends[4];       // of the axes' pairs
  double rates[64];    // frequencies in turns
  uint64_t turns[64];  // the frequencies' fractions of a turn times 2^64
};

// The position of a sample's token on the axis of a pair, as it lies in memory (32 bits of whatever type, or 64).
__device__ __forceinline__ int64_t position_of(const RopeParams& p, uint32_t token, int pair) {
  int axis = 0;
#pragma unroll
  for (int a = 0; a < 3; ++a) axis += pair >= p.ends[a];
  const int64_t at = blockIdx.y * p.position_batch + (int64_t)token * p.axes + axis;
  if (p.positions_type == 1) return static_cast<const int64_t*>(p.positions)[at];
  return static_cast<const int32_t*>(p.positions)[at];
}
// Cosine and sine of the pair's angle.
__device__ __forceinline__ float2 angle_of(const RopeParams& p, int64_t position, int pair) {
  float turn;
  if (p.positions_type == 2) {
    const double exact = (double)__int_as_float((int)position) * p.rates[pair];
    turn = (float)(exact - rint(exact));
  } else {
    const uint64_t fraction = (uint64_t)position * p.turns[pair];
    turn = (float)(int32_t)(uint32_t)(fraction >> 32) * 0x1p-32f;
  }
  const float radians = 6.283185307f * turn;
  return make_float2(__cosf(radians), __sinf(radians));
}

// What a lane has of a head: two pieces of 4 channels, which are 4 whole pairs where they turn.  Halves: channels 4 l ... and
// their partners P channels on; neighbours: 8 channels in a row.  No pair crosses lanes, so that turning needs no shuffles
// (with 8 channels in a row for both, 8 shuffles per row and half the arithmetic idle: 430 us for 33,272 tokens of 112 heads
// of 128).
struct Span {
  int first, second;  // channels
  bool in;
  __device__ __forceinline__ Span(int lane, int pairs, bool interleaved) {
    in = 4 * lane < pairs;
    first = interleaved ? 8 * lane : in ? 4 * lane : 2 * pairs + 8 * (lane - pairs / 4);
    second = interleaved || !in ? first + 4 : first + pairs;
  }
};

// The lane's 4 pairs' cosines and sines; 1 and 0 where its channels do not turn, or for a token that does not exist (whose
// place in the table nobody has written).
__device__ __forceinline__ void load_angles(const float* row, int lane, const Span& span, bool exists, int pairs, float4& c,
                                            float4& s) {
  c = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
  s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (span.in && exists) {
    c = *reinterpret_cast<const float4*>(row + 4 * lane);
    s = *reinterpret_cast<const float4*>(row + pairs + 4 * lane);
  }
}

// A lane's 8 channels as the first and the second of each of its 4 pairs: u[0] = (u_0, u_1), u[1] = (u_2, u_3), v alike.
template <typename T>
__device__ __forceinline__ void open_pairs(uint2 a, uint2 b, bool interleaved, float2 (&u)[2], float2 (&v)[2]) {
  const float2 a0 = Pair<T>::open(a.x), a1 = Pair<T>::open(a.y), b0 = Pair<T>::open(b.x), b1 = Pair<T>::open(b.y);
  u[0] = interleaved ? make_float2(a0.x, a1.x) : a0;
  v[0] = interleaved ? make_float2(a0.y, a1.y) : b0;
  u[1] = interleaved ? make_float2(b0.x, b1.x) : a1;
  v[1] = interleaved ? make_float2(b0.y, b1.y) : b1;
}
template <typename T>
__device__ __forceinline__ void store_pairs(T* a, T* b, bool interleaved, const float2 (&u)[2], const float2 (&v)[2]) {
  if (interleaved) {
    *reinterpret_cast<uint2*>(a) = make_uint2(Pair<T>::round(u[0].x, v[0].x), Pair<T>::round(u[0].y, v[0].y));
    *reinterpret_cast<uint2*>(b) = make_uint2(Pair<T>::round(u[1].x, v[1].x), Pair<T>::round(u[1].y, v[1].y));
  } else {
    *reinterpret_cast<uint2*>(a) = make_uint2(Pair<T>::round(u[0].x, u[0].y), Pair<T>::round(u[1].x, u[1].y));
    *reinterpret_cast<uint2*>(b) = make_uint2(Pair<T>::round(v[0].x, v[0].y), Pair<T>::round(v[1].x, v[1].y));
  }
}
__device__ __forceinline__ float2 negative(float2 a) { return make_float2(-a.x, -a.y); }

// Sums of N rows over kLanes lanes, each in the lanes that shuffle `row * (kLanes / N)` names; the lanes first share the rows
// out, half of them per step.
template <int kLanes, int N>
__device__ __forceinline__ float shared_out_sum(const float (&v)[N]) {
  static_assert(N == 1 || N == 2 || N == 4, "shared out by halves");
  const int lane = threadIdx.x;
  float mine = v[0];
  int off = kLanes / 2;
  if constexpr (N == 4) {
    const bool high = lane & (kLanes / 2), next = lane & (kLanes / 4);
    const float a = (high ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, high ? v[0] : v[2], kLanes / 2);
    const float b = (high ? v[3] : v[1]) + __shfl_xor_sync(0xffffffffu, high ? v[1] : v[3], kLanes / 2);
    mine = (next ? b : a) + __shfl_xor_sync(0xffffffffu, next ? a : b, kLanes / 4);
    off = kLanes / 8;
  } else if constexpr (N == 2) {
    const bool high = lane & (kLanes / 2);
    mine = (high ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, high ? v[0] : v[1], kLanes / 2);
    off = kLanes / 4;
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1)
    if (o <= off) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  return mine;
}

// Groups of D/8 lanes take kRows heads of one token of sample blockIdx.y: a unit.  A warp's units are of one token or of
// neighbours.
struct Unit {
  uint32_t first, into;   // the warp's first token, its first unit's place there
  uint32_t t, token;      // the group's token, from the first one and from the sample's
  uint32_t place;         // of the unit among its token's
};
template <int kUnits>
__device__ __forceinline__ uint32_t token_in_warp(uint32_t local, uint32_t per_token) {
  return per_token >= kUnits ? (uint32_t)(local >= per_token) : local / per_token;
}
template <int kUnits>
__device__ __forceinline__ Unit unit_at(uint32_t warp_unit, int group, uint32_t per_token) {
  Unit u;
  u.first = warp_unit / per_token;
  u.into = warp_unit - u.first * per_token;
  const uint32_t local = u.into + group;
  u.t = token_in_warp<kUnits>(local, per_token);
  u.token = u.first + u.t;
  u.place = local - u.t * per_token;
  return u;
}
// The angles of the warp's tokens, each once: [token][cosines of all pairs, then sines], in shared memory of the warp's own.
template <int kUnits>
__device__ __forceinline__ void warp_angles(const RopeParams& p, const Unit& u, uint32_t per_token, float* table) {
  const uint32_t last = token_in_warp<kUnits>(u.into + kUnits - 1, per_token);
  for (uint32_t n = 0; n <= last; ++n)
    if (u.first + n < p.tokens)
      for (int pair = threadIdx.x % 32; pair < p.pairs; pair += 32) {
        const float2 cs = angle_of(p, position_of(p, u.first + n, pair), pair);
        table[2 * n * p.pairs + pair] = cs.x;
        table[(2 * n + 1) * p.pairs + pair] = cs.y;
      }
}

// HBM bound: two bytes in and two out per channel; what comes next is issue slots, hence packed arithmetic, with the weights
// multiplied into the cosines and sines once for all rows: out = r (u w_u c - v w_v s), r (v w_v c + u w_u s).  The angles are
// formed while the heads' loads are in flight.  33,272 tokens of 112 heads of 128: 304 us, 6.3 TB/s (one table per
// block, behind a barrier: 377; 16 heads per group, two blocks per SM: 330).
__host__ __device__ constexpr int forward_blocks(int rows) { return rows == 8 ? 3 : 4; }
template <typename T, int D, int kRows, bool interleaved>
__global__ void __launch_bounds__(kThreads, forward_blocks(kRows)) forward_kernel(const __grid_constant__ RopeParams p) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes, kUnits = 32 / kLanes;
  __shared__ __align__(16) float tables[kThreads / 32][kUnits * D];
  float* table = tables[threadIdx.x / 32];
  const int lane = threadIdx.x % kLanes;
  const uint32_t q_units = (p.q_heads + kRows - 1) / kRows, per_token = q_units + (p.k_heads + kRows - 1) / kRows;
  const Unit u = unit_at<kUnits>(blockIdx.x * kGroups + threadIdx.x / 32 * kUnits, threadIdx.x % 32 / kLanes, per_token);
  const bool is_q = u.place < q_units;
  const int head = (int)(is_q ? u.place : u.place - q_units) * kRows;
  const int heads = u.token < p.tokens ? min(kRows, (is_q ? p.q_heads : p.k_heads) - head) : 0;
  const int64_t *in = p.strides[is_q ? 0 : 1], *out = p.strides[is_q ? 2 : 3];
  const Span span(lane, p.pairs, interleaved);
  const T* src = static_cast<const T*>(is_q ? p.q : p.k) + blockIdx.y * in[0] + u.token * in[1] + head * in[2];
  uint2 raw[kRows][2];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    raw[i][0] = raw[i][1] = make_uint2(0, 0);
    if (i < heads) {
      raw[i][0] = load_stream8(src + span.first);
      raw[i][1] = load_stream8(src + span.second);
    }
    src += in[2];
  }
  warp_angles<kUnits>(p, u, per_token, table);
  const bool normed = p.q_weight != nullptr;
  float2 wu[2] = {both(1.0f), both(1.0f)}, wv[2] = {both(1.0f), both(1.0f)};
  if (normed) {
    const T* weight = static_cast<const T*>(is_q ? p.q_weight : p.k_weight);
    open_pairs<T>(__ldg(reinterpret_cast<const uint2*>(weight + span.first)),
                  __ldg(reinterpret_cast<const uint2*>(weight + span.second)), interleaved, wu, wv);
  }
  __syncwarp();
  float4 c4, s4;
  load_angles(table + 2 * u.t * p.pairs, lane, span, heads > 0, p.pairs, c4, s4);
  const float2 c[2] = {make_float2(c4.x, c4.y), make_float2(c4.z, c4.w)};
  const float2 s[2] = {make_float2(s4.x, s4.y), make_float2(s4.z, s4.w)};
  float2 uc[2], us[2], vc[2], vs[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uc[j] = fmul2(wu[j], c[j]);
    us[j] = fmul2(wu[j], s[j]);
    vc[j] = fmul2(wv[j], c[j]);
    vs[j] = negative(fmul2(wv[j], s[j]));
  }
  T* dst = static_cast<T*>(is_q ? p.q_out : p.k_out) + blockIdx.y * out[0] + u.token * out[1] + head * out[2];
  constexpr int kShared = kRows < 4 ? kRows : 4;  // rows that share a sum over the lanes
#pragma unroll
  for (int i0 = 0; i0 < kRows; i0 += kShared) {
    float r_mine = 1.0f;
    if (normed) {
      float squares[kShared];
#pragma unroll
      for (int i = 0; i < kShared; ++i) {
        float2 x[2], y[2];
        open_pairs<T>(raw[i0 + i][0], raw[i0 + i][1], false, x, y);
        float2 sum = fmul2(x[0], x[0]);
        sum = ffma2(x[1], x[1], sum);
        sum = ffma2(y[0], y[0], sum);
        sum = ffma2(y[1], y[1], sum);
        squares[i] = sum.x + sum.y;
      }
      r_mine = rsqrtf(fmaf(shared_out_sum<kLanes, kShared>(squares), 1.0f / D, p.eps));
    }
#pragma unroll
    for (int i = 0; i < kShared; ++i) {
      float2 x[2], y[2];
      open_pairs<T>(raw[i0 + i][0], raw[i0 + i][1], interleaved, x, y);
      const float2 r = both(normed ? __shfl_sync(0xffffffffu, r_mine, i * (kLanes / kShared), kLanes) : 1.0f);
      float2 a[2], e[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        a[j] = fmul2(ffma2(y[j], vs[j], fmul2(x[j], uc[j])), r);
        e[j] = fmul2(ffma2(x[j], us[j], fmul2(y[j], vc[j])), r);
      }
      if (i0 + i < heads) store_pairs<T>(dst + span.first, dst + span.second, interleaved, a, e);
      dst += out[2];
    }
  }
}

// The gradient, the same way.  A block has queries or keys and walks units a grid apart, so that a thread's 8 sums of the
// weight stay in registers; they are added over its groups at the end, and the blocks' by sums_kernel.  Blocks are many more
// than fit at once: loads of one are in flight under the arithmetic of others (a ring of copies ahead, in blocks that stay,
// cost more instructions than it hid: 150 us for 32,256 tokens of 32 heads of 64; loads of the next unit ahead in registers:
// 117 to 142; three blocks per SM at 80 registers, which spill: 129; two: 98, 4.0 TB/s).
constexpr int kBackwardRows = 4;
template <typename T, int D, bool interleaved>
__global__ void __launch_bounds__(kThreads, 2) backward_kernel(const __grid_constant__ RopeParams p) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes, kUnits = 32 / kLanes, kRows = kBackwardRows;
  __shared__ __align__(16) float tables[kThreads / 32][kUnits * D];
  __shared__ float sums[kGroups][D];
  float* table = tables[threadIdx.x / 32];
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const bool keys = (int)blockIdx.x >= p.q_blocks, normed = p.q_weight != nullptr;
  const int block = keys ? blockIdx.x - p.q_blocks : blockIdx.x, blocks = keys ? gridDim.x - p.q_blocks : p.q_blocks;
  const int all_heads = keys ? p.k_heads : p.q_heads, which = keys ? 1 : 0;
  const uint32_t per_token = (all_heads + kRows - 1) / kRows, units = p.tokens * per_token;
  const Span span(lane, p.pairs, interleaved);
  const T* weight = static_cast<const T*>(keys ? p.k_weight : p.q_weight);
  const int64_t *ds = p.strides[which], *xs = p.strides[2 + which], *os = p.strides[4 + which];
  float2 wu[2] = {both(1.0f), both(1.0f)}, wv[2] = {both(1.0f), both(1.0f)};
  if (normed)
    open_pairs<T>(__ldg(reinterpret_cast<const uint2*>(weight + span.first)),
                  __ldg(reinterpret_cast<const uint2*>(weight + span.second)), interleaved, wu, wv);
  float2 sum_u[2] = {both(0.0f), both(0.0f)}, sum_v[2] = {both(0.0f), both(0.0f)};
#pragma unroll 1
  for (uint32_t unit = block * kGroups; unit < units; unit += blocks * kGroups) {
    const Unit u = unit_at<kUnits>(unit + threadIdx.x / 32 * kUnits, threadIdx.x % 32 / kLanes, per_token);
    const int head = (int)u.place * kRows, heads = u.token < p.tokens ? min(kRows, all_heads - head) : 0;
    const T* d = static_cast<const T*>(keys ? p.dk_out : p.dq_out) + blockIdx.y * ds[0] + u.token * ds[1] + head * ds[2];
    const T* x = static_cast<const T*>(keys ? p.k : p.q) + blockIdx.y * xs[0] + u.token * xs[1] + head * xs[2];
    uint2 d_raw[kRows][2], x_raw[kRows][2];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      d_raw[i][0] = d_raw[i][1] = x_raw[i][0] = x_raw[i][1] = make_uint2(0, 0);
      if (i < heads) {
        d_raw[i][0] = load_stream8(d + span.first);
        d_raw[i][1] = load_stream8(d + span.second);
        if (normed) {
          x_raw[i][0] = load_stream8(x + span.first);
          x_raw[i][1] = load_stream8(x + span.second);
        }
      }
      d += ds[2];
      x += xs[2];
    }
    // (everybody in the warp has read the angles of the units before)
    __syncwarp();
    warp_angles<kUnits>(p, u, per_token, table);
    __syncwarp();
    float4 c4, s4;
    load_angles(table + 2 * u.t * p.pairs, lane, span, heads > 0, p.pairs, c4, s4);
    const float2 c[2] = {make_float2(c4.x, c4.y), make_float2(c4.z, c4.w)};
    const float2 s[2] = {make_float2(s4.x, s4.y), make_float2(s4.z, s4.w)};
    const float2 minus_s[2] = {negative(s[0]), negative(s[1])};
    T* out = static_cast<T*>(keys ? p.k_out : p.q_out) + blockIdx.y * os[0] + u.token * os[1] + head * os[2];
    // two rows at a time
#pragma unroll
    for (int i0 = 0; i0 < kRows; i0 += 2) {
      float2 gu[2][2], gv[2][2], xu[2][2], xv[2][2];
      float row_sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float2 a[2], e[2];
        open_pairs<T>(d_raw[i0 + i][0], d_raw[i0 + i][1], interleaved, a, e);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          // turned back
          gu[i][j] = ffma2(e[j], s[j], fmul2(a[j], c[j]));
          gv[i][j] = ffma2(a[j], minus_s[j], fmul2(e[j], c[j]));
        }
        if (!normed) continue;
        open_pairs<T>(x_raw[i0 + i][0], x_raw[i0 + i][1], interleaved, xu[i], xv[i]);
        float2 square = both(0.0f), along = both(0.0f);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          square = ffma2(xu[i][j], xu[i][j], square);
          square = ffma2(xv[i][j], xv[i][j], square);
          along = ffma2(fmul2(gu[i][j], wu[j]), xu[i][j], along);
          along = ffma2(fmul2(gv[i][j], wv[j]), xv[i][j], along);
        }
        row_sums[2 * i] = square.x + square.y;
        row_sums[2 * i + 1] = along.x + along.y;
      }
      const float mine = normed ? shared_out_sum<kLanes, 4>(row_sums) : 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (normed) {
          const float square = __shfl_sync(0xffffffffu, mine, 2 * i * (kLanes / 4), kLanes);
          const float with_x = __shfl_sync(0xffffffffu, mine, (2 * i + 1) * (kLanes / 4), kLanes);
          // (a head that does not exist is zeros, and stays so with eps = 0)
          const float r = i0 + i < heads ? rsqrtf(fmaf(square, 1.0f / D, p.eps)) : 0.0f;
          const float2 r2 = both(r), back = both(-with_x * r * r * (1.0f / D));
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            sum_u[j] = ffma2(gu[i][j], fmul2(xu[i][j], r2), sum_u[j]);
            sum_v[j] = ffma2(gv[i][j], fmul2(xv[i][j], r2), sum_v[j]);
            gu[i][j] = fmul2(ffma2(xu[i][j], back, fmul2(gu[i][j], wu[j])), r2);
            gv[i][j] = fmul2(ffma2(xv[i][j], back, fmul2(gv[i][j], wv[j])), r2);
          }
        }
        if (i0 + i < heads) store_pairs<T>(out + span.first, out + span.second, interleaved, gu[i], gv[i]);
        out += os[2];
      }
    }
  }
  if (p.weight_partial == nullptr) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = i & 1 ? sum_u[i / 2].y : sum_u[i / 2].x, e = i & 1 ? sum_v[i / 2].y : sum_v[i / 2].x;
    const int at = interleaved ? (i < 2 ? span.first + 2 * i : span.second + 2 * (i - 2)) : span.first + i;
    const int partner = interleaved ? at + 1 : span.second + i;
    sums[group][at] = a;
    sums[group][partner] = e;
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float total = 0.0f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) total += sums[g][threadIdx.x];
    // (all samples' parts of queries first)
    const int64_t part = keys ? (int64_t)gridDim.y * p.q_blocks + blockIdx.y * blocks + block : blockIdx.y * blocks + block;
    p.weight_partial[part * D + threadIdx.x] = total;
  }
}

constexpr int kSumThreads = 1024;  // (few columns, many parts)
// blockIdx.y: queries', keys' weight; its blocks' parts.
template <typename T>
__global__ void __launch_bounds__(kSumThreads) sums_kernel(const float* partial, int q_parts, int k_parts, int d,
                                                           void* dq_weight, void* dk_weight) {
  layer::grid_dependency_wait();
  void* out = blockIdx.y ? dk_weight : dq_weight;
  const int parts = blockIdx.y ? k_parts : q_parts, across = sum_columns(parts), first = blockIdx.x * across;
  if (out == nullptr || first >= d) return;
  const float v = column_sum<kSumThreads>(partial + (blockIdx.y ? (int64_t)q_parts * d : 0), d, parts, first, d);
  if (threadIdx.x < across && first + (int)threadIdx.x < d) store1(static_cast<T*>(out) + first + threadIdx.x, v);
}

// Heads per group of lanes: eight (that many loads in flight, one read of weights and angles for them) where heads fill them
// and the groups fill the SMs, four where one of the two is half so, else one.
int rows_of(const anemoi_sm100_axial_rope_shape* s) {
  const int64_t groups = (int64_t)kSms * 2 * kThreads / (s->head_dim / 8);
  const int heads = std::max(s->q_heads, s->k_heads);
  const int64_t rows = s->batch * s->tokens * (s->q_heads + s->k_heads);
  return heads > 4 && rows >= 8 * groups ? 8 : heads > 2 && rows >= 2 * groups ? 4 : 1;
}

// The gradient's blocks of a sample: as many as its units fill, or as few as leave every SM 16 of them in all (a sum of the
// weights has that many parts), each of as many turns.
struct BackwardPlan {
  int q_blocks, k_blocks;
};
BackwardPlan plan_of(const anemoi_sm100_axial_rope_shape* s) {
  const int64_t groups = kThreads / (s->head_dim / 8);
  const int64_t q = (s->tokens * ((s->q_heads + kBackwardRows - 1) / kBackwardRows) + groups - 1) / groups;
  const int64_t k = (s->tokens * ((s->k_heads + kBackwardRows - 1) / kBackwardRows) + groups - 1) / groups;
  const int64_t turns = ((q + k) * s->batch + kSms * 16 - 1) / (kSms * 16);
  return {(int)((q + turns - 1) / turns), (int)((k + turns - 1) / turns)};
}

int check(const anemoi_sm100_axial_rope_shape* s) {
  if (s == nullptr || s->batch < 0 || s->tokens < 0 || s->q_heads <= 0 || s->k_heads < 0 || !(s->eps >= 0.0f))
    return ANEMOI_SM100_EINVAL;
  if ((s->head_dim != 64 && s->head_dim != 128) || s->axes < 1 || s->axes > 4 || s->positions_type < 0 ||
      s->positions_type > 2)
    return ANEMOI_SM100_EINVAL;
  int64_t pairs = 0;
  for (int a = 0; a < s->axes; ++a) {
    if (s->sections[a] < 0) return ANEMOI_SM100_EINVAL;
    pairs += s->sections[a];
  }
  if (2 * pairs > s->head_dim || pairs % (s->interleaved ? 4 : 8)) return ANEMOI_SM100_EINVAL;
  // (a sample's heads are counted in 32 bits, samples by the grid)
  if (s->q_heads > 4096 || s->k_heads > 4096 || s->batch > 65535 || s->tokens > 0x7fffffffLL / (s->q_heads + s->k_heads))
    return ANEMOI_SM100_ELIMIT;
  return ANEMOI_SM100_OK;
}

void fill(RopeParams& p, const anemoi_sm100_axial_rope_shape* s, const double* turns, const int64_t* strides, int tensors) {
  p.batch = (uint32_t)s->batch;
  p.tokens = (uint32_t)s->tokens;
  p.q_heads = s->q_heads;
  p.k_heads = s->k_heads;
  p.axes = s->axes;
  p.interleaved = s->interleaved != 0;
  p.positions_type = s->positions_type;
  p.eps = s->eps;
  p.pairs = 0;
  for (int a = 0; a < 4; ++a) p.ends[a] = p.pairs += a < s->axes ? s->sections[a] : 0;
  for (int i = 0; i < p.pairs; ++i) {
    p.rates[i] = turns[i];
    // (a double below 1 times 2^64 is whole from 2^-11 on, and rounds by less than one below)
    p.turns[i] = (uint64_t)((turns[i] - floor(turns[i])) * 0x1p64);
  }
  for (int i = 0; i < tensors; ++i)
    for (int j = 0; j < 3; ++j) p.strides[i][j] = strides[3 * i + j];
}

template <typename T, int D, int kRows>
int forward_launch(const RopeParams& p, cudaStream_t st) {
  constexpr int64_t kGroups = kThreads / (D / 8);
  const int64_t units = (int64_t)p.tokens * ((p.q_heads + kRows - 1) / kRows + (p.k_heads + kRows - 1) / kRows);
  const dim3 grid((unsigned)((units + kGroups - 1) / kGroups), p.batch);
  auto kernel = p.interleaved ? forward_kernel<T, D, kRows, true> : forward_kernel<T, D, kRows, false>;
  kernel<<<grid, kThreads, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? ANEMOI_SM100_OK : ANEMOI_SM100_ELAUNCH;
}

template <typename T, int D>
int forward_rows(const RopeParams& p, int rows, cudaStream_t st) {
  return rows == 8 ? forward_launch<T, D, 8>(p, st) : rows == 4 ? forward_launch<T, D, 4>(p, st) : forward_launch<T, D, 1>(p, st);
}

template <typename T, int D>
int backward_launch(RopeParams& p, const BackwardPlan& plan, void* dq_weight, void* dk_weight, cudaStream_t st) {
  p.q_blocks = plan.q_blocks;
  auto kernel = p.interleaved ? backward_kernel<T, D, true> : backward_kernel<T, D, false>;
  kernel<<<dim3(plan.q_blocks + plan.k_blocks, p.batch), kThreads, 0, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return ANEMOI_SM100_ELAUNCH;
  if (p.weight_partial == nullptr) return ANEMOI_SM100_OK;
  return layer::launch(sums_kernel<T>, dim3(D / 8, 2), dim3(kSumThreads), 0, st, p.weight_partial, plan.q_blocks * (int)p.batch,
                       plan.k_blocks * (int)p.batch, D, dq_weight, dk_weight) == cudaSuccess ? ANEMOI_SM100_OK : ANEMOI_SM100_ELAUNCH;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

extern "C" int anemoi_sm100_axial_rope(const anemoi_sm100_axial_rope_shape* s, const void* q, const void* k,
                                       const void* q_weight, const void* k_weight, const void* positions,
                                       int64_t position_batch, const double* turns, const int64_t* strides, void* q_out,
                                       void* k_out, void* stream) {
  const int bad = check(s);
  if (bad != ANEMOI_SM100_OK) return bad;
  if (!strides || position_batch < 0) return ANEMOI_SM100_EINVAL;
  for (int i = 0; i < 12; ++i)
    if (strides[i] % 8) return ANEMOI_SM100_EINVAL;
  for (const void* t : {q, k, q_weight, k_weight, (const void*)q_out, (const void*)k_out})
    if (!aligned(t)) return ANEMOI_SM100_EINVAL;
  if (s->batch == 0 || s->tokens == 0) return ANEMOI_SM100_OK;
  if (!q || !q_out || !positions || !turns || (s->k_heads > 0 && (!k || !k_out))) return ANEMOI_SM100_EINVAL;
  if (s->k_heads > 0 && !q_weight != !k_weight) return ANEMOI_SM100_EINVAL;
  RopeParams p{};
  p.q = q;
  p.k = k;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.positions = positions;
  p.position_batch = position_batch;
  p.q_out = q_out;
  p.k_out = k_out;
  fill(p, s, turns, strides, 4);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (s->is_bf16)
    return s->head_dim == 64 ? forward_rows<__nv_bfloat16, 64>(p, rows_of(s), st)
                             : forward_rows<__nv_bfloat16, 128>(p, rows_of(s), st);
  return s->head_dim == 64 ? forward_rows<__half, 64>(p, rows_of(s), st) : forward_rows<__half, 128>(p, rows_of(s), st);
}

extern "C" int64_t anemoi_sm100_axial_rope_backward_workspace(const anemoi_sm100_axial_rope_shape* s) {
  const int bad = check(s);
  if (bad != ANEMOI_SM100_OK) return bad;
  if (s->batch == 0 || s->tokens == 0) return 0;
  const BackwardPlan plan = plan_of(s);
  return (int64_t)(plan.q_blocks + plan.k_blocks) * s->batch * s->head_dim * (int64_t)sizeof(float);
}

extern "C" int anemoi_sm100_axial_rope_backward(const anemoi_sm100_axial_rope_shape* s, const void* dq_out,
                                                const void* dk_out, const void* q, const void* k, const void* q_weight,
                                                const void* k_weight, const void* positions, int64_t position_batch,
                                                const double* turns, const int64_t* strides, void* dq, void* dk,
                                                void* dq_weight, void* dk_weight, void* workspace, int64_t workspace_bytes,
                                                void* stream) {
  const int bad = check(s);
  if (bad != ANEMOI_SM100_OK) return bad;
  if (!strides || position_batch < 0 || s->batch == 0 || s->tokens == 0) return ANEMOI_SM100_EINVAL;
  for (int i = 0; i < 18; ++i)
    if (strides[i] % 8) return ANEMOI_SM100_EINVAL;
  for (const void* t : {dq_out, dk_out, q, k, q_weight, k_weight, (const void*)dq, (const void*)dk, (const void*)workspace})
    if (!aligned(t)) return ANEMOI_SM100_EINVAL;
  if (!dq_out || !dq || !positions || !turns || (s->k_heads > 0 && (!dk_out || !dk))) return ANEMOI_SM100_EINVAL;
  if (s->k_heads > 0 && !q_weight != !k_weight) return ANEMOI_SM100_EINVAL;
  if (q_weight != nullptr && (!q || (s->k_heads > 0 && !k))) return ANEMOI_SM100_EINVAL;
  const bool weights = dq_weight != nullptr || dk_weight != nullptr;
  if (weights && (!q_weight || !workspace || workspace_bytes < anemoi_sm100_axial_rope_backward_workspace(s)))
    return ANEMOI_SM100_EINVAL;
  RopeParams p{};
  p.dq_out = dq_out;
  p.dk_out = dk_out;
  p.q = q;
  p.k = k;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.positions = positions;
  p.position_batch = position_batch;
  p.q_out = dq;
  p.k_out = dk;
  p.weight_partial = weights ? static_cast<float*>(workspace) : nullptr;
  fill(p, s, turns, strides, 6);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const BackwardPlan plan = plan_of(s);
  if (s->is_bf16) {
    using T = __nv_bfloat16;
    return s->head_dim == 64 ? backward_launch<T, 64>(p, plan, dq_weight, dk_weight, st)
                             : backward_launch<T, 128>(p, plan, dq_weight, dk_weight, st);
  }
  using T = __half;
  return s->head_dim == 64 ? backward_launch<T, 64>(p, plan, dq_weight, dk_weight, st)
                           : backward_launch<T, 128>(p, plan, dq_weight, dk_weight, st);
}
