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
// The angle is formed in double precision and reduced to a fraction of a turn there: position * turns has 2^-53 relative,
// so that positions of 2^31 still have angles good to 2^-22 of a turn, where a product in fp32 has none beyond 2^24.  Cosine
// and sine of the fraction are fp32 (sincospif).
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/anemoi_sm100.h"
#include "rows.cuh"

namespace {

using namespace rows;

constexpr int kThreads = 256;

struct RopeParams {
  const void *q, *k, *dq_out, *dk_out, *q_weight, *k_weight, *positions;
  void *q_out, *k_out;
  float* weight_partial;  // [blocks of queries, then of keys][D]
  int64_t position_batch, batch, tokens;
  int64_t strides[6][3];  // forward: q, k, q_out, k_out; gradient: dq_out, dk_out, q, k, dq, dk
  int q_heads, k_heads, axes, pairs, interleaved, positions_type, block_tokens, q_blocks;
  float eps;
  int ends[4];       // of the axes' pairs
  double turns[64];
};

// Cosines and sines of `count` tokens from `first` on: [token][cosines of all pairs, then sines].
__device__ __forceinline__ void angles(const RopeParams& p, int64_t first, int count, float* table) {
  for (int i = threadIdx.x; i < count * p.pairs; i += kThreads) {
    const int t = i / p.pairs, pair = i - t * p.pairs;
    int axis = 0;
    while (axis < p.axes - 1 && pair >= p.ends[axis]) ++axis;
    const int64_t token = first + t, b = quotient(token, p.tokens);
    const int64_t at = b * p.position_batch + (token - b * p.tokens) * p.axes + axis;
    const double position = p.positions_type == 0   ? (double)static_cast<const int32_t*>(p.positions)[at]
                            : p.positions_type == 1 ? (double)static_cast<const int64_t*>(p.positions)[at]
                                                    : (double)static_cast<const float*>(p.positions)[at];
    const double turn = position * p.turns[pair];
    float s, c;
    sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
    table[2 * t * p.pairs + pair] = c;
    table[(2 * t + 1) * p.pairs + pair] = s;
  }
}

// What a lane has of a head: 8 consecutive channels.
struct Span {
  bool in, first;
  int partner, pair;
  __device__ __forceinline__ Span(int lane, int pairs, int interleaved) {
    const int c0 = lane * 8;
    in = c0 < 2 * pairs;
    first = c0 < pairs;
    partner = in && !interleaved ? (first ? lane + pairs / 8 : lane - pairs / 8) : lane;
    pair = interleaved ? c0 / 2 : first ? c0 : c0 - pairs;
  }
};

// A lane's cosines and sines (of its 8 channels' pairs, or of its 4 pairs of neighbours).  Halves: the sines of the first
// one's channels change sign here.  kBack: of the opposite angles.
template <bool kBack>
__device__ __forceinline__ void load_angles(const float* row, const Span& span, int pairs, bool interleaved, float (&c)[8],
                                            float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = 1.0f;
    s[i] = 0.0f;
  }
  if (!span.in) return;
  *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(row + span.pair);
  *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(row + pairs + span.pair);
  if (!interleaved) {
    *reinterpret_cast<float4*>(c + 4) = *reinterpret_cast<const float4*>(row + span.pair + 4);
    *reinterpret_cast<float4*>(s + 4) = *reinterpret_cast<const float4*>(row + pairs + span.pair + 4);
  }
  const bool minus = interleaved ? kBack : span.first != kBack;
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = minus ? -s[i] : s[i];
}

// Turns a lane's 8 channels.  All lanes of the warp take part.
template <int kLanes>
__device__ __forceinline__ void turn8(float (&n)[8], const Span& span, bool interleaved, const float (&c)[8],
                                      const float (&s)[8]) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = n[2 * i], v = n[2 * i + 1];
      n[2 * i] = fmaf(-v, s[i], u * c[i]);
      n[2 * i + 1] = fmaf(u, s[i], v * c[i]);
    }
    return;
  }
  float other[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(0xffffffffu, n[i], span.partner, kLanes);
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = fmaf(other[i], s[i], n[i] * c[i]);
}

template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// Groups of D/8 lanes take kRows heads of one token: a unit.  A block has as many units as groups, of one token or of
// neighbours, whose angles it forms once in shared memory while the heads' loads are in flight.  HBM bound: two bytes in and
// two out per channel.  One unit per group: several in turn, whose loads only start when the one before is done, took 430 us
// for 33,272 tokens of 112 heads of 128.
template <typename T, int D, int kRows>
__global__ void __launch_bounds__(kThreads, 4) forward_kernel(const __grid_constant__ RopeParams p) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes;
  __shared__ __align__(16) float table[(kGroups + 1) * D];
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const uint32_t all = (uint32_t)(p.batch * p.tokens);
  const uint32_t q_units = (p.q_heads + kRows - 1) / kRows, per_token = q_units + (p.k_heads + kRows - 1) / kRows;
  const uint64_t unit0 = (uint64_t)blockIdx.x * kGroups;
  const uint32_t first = (uint32_t)quotient(unit0, per_token);
  const uint32_t local = (uint32_t)(unit0 - (uint64_t)first * per_token) + group, t = local / per_token;
  const uint32_t token = first + t, u = local - t * per_token;
  const bool is_q = u < q_units;
  const int head = (int)(is_q ? u : u - q_units) * kRows;
  const int heads = token < all ? min(kRows, (is_q ? p.q_heads : p.k_heads) - head) : 0;
  const uint32_t b = token / (uint32_t)p.tokens, at = token - b * (uint32_t)p.tokens;
  const int64_t *in = p.strides[is_q ? 0 : 1], *out = p.strides[is_q ? 2 : 3];
  const T* src = static_cast<const T*>(is_q ? p.q : p.k) + b * in[0] + at * in[1] + head * in[2] + lane * 8;
  uint4 raw[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    raw[i] = make_uint4(0, 0, 0, 0);
    if (i < heads) raw[i] = load_stream(src + i * in[2]);
  }
  const uint32_t last = (uint32_t)(unit0 - (uint64_t)first * per_token + kGroups - 1) / per_token;
  angles(p, first, (int)(min(all, first + last + 1) - first), table);
  const T* weight = static_cast<const T*>(is_q ? p.q_weight : p.k_weight);
  const bool normed = p.q_weight != nullptr;
  float w[8];
  if (normed) shared8(weight + lane * 8, w);
  __syncthreads();
  const Span span(lane, p.pairs, p.interleaved);
  float cs[8], sn[8];
  load_angles<false>(table + 2 * t * p.pairs, span, p.pairs, p.interleaved, cs, sn);
  T* dst = static_cast<T*>(is_q ? p.q_out : p.k_out) + b * out[0] + at * out[1] + head * out[2] + lane * 8;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    float n[8];
    open8<T>(raw[i], n);
    if (normed) {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf(n[j], n[j], s);
      const float r = rsqrtf(fmaf(row_sum<kLanes>(s), 1.0f / D, p.eps));
#pragma unroll
      for (int j = 0; j < 8; ++j) n[j] = n[j] * r * w[j];
    }
    turn8<kLanes>(n, span, p.interleaved, cs, sn);
    if (i < heads) *reinterpret_cast<uint4*>(dst + i * out[2]) = round8<T>(n);
  }
}

// The gradient.  A block has queries or keys, and walks sets of block_tokens tokens a grid apart, so that a thread's 8 sums
// of the weight stay in registers; they are added over its groups at the end, and the blocks' by sums_kernel.  The next
// units are copied into a ring of shared memory meanwhile (a thread's own channels).
constexpr int kBackwardRows = 2, kRing = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 3) backward_kernel(const __grid_constant__ RopeParams p) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes, kRows = kBackwardRows;
  extern __shared__ __align__(16) uint4 ring_all[];  // [kRing][d, x][kRows][thread]
  __shared__ __align__(16) float table[16 * 128];
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const bool keys = (int)blockIdx.x >= p.q_blocks;
  const int block = keys ? blockIdx.x - p.q_blocks : blockIdx.x, blocks = keys ? gridDim.x - p.q_blocks : p.q_blocks;
  const int all_heads = keys ? p.k_heads : p.q_heads, which = keys ? 1 : 0;
  const uint32_t all = (uint32_t)(p.batch * p.tokens), per_token = (all_heads + kRows - 1) / kRows;
  const uint32_t sets = (all + p.block_tokens - 1) / p.block_tokens, units = p.block_tokens * per_token;
  const uint32_t steps = (units + kGroups - 1) / kGroups;
  const Span span(lane, p.pairs, p.interleaved);
  const bool normed = p.q_weight != nullptr;
  const T* weight = static_cast<const T*>(keys ? p.k_weight : p.q_weight);
  const int64_t *ds = p.strides[which], *xs = p.strides[2 + which], *os = p.strides[4 + which];
  const T* d_all = static_cast<const T*>(keys ? p.dk_out : p.dq_out) + lane * 8;
  const T* x_all = static_cast<const T*>(keys ? p.k : p.q) + lane * 8;
  T* out_all = static_cast<T*>(keys ? p.k_out : p.q_out) + lane * 8;
  float w[8];
  if (normed) shared8(weight + lane * 8, w);
  float weight_sum[8] = {};
  struct Unit {
    uint32_t b, at, t;
    int head, heads;
  };
  auto unit_of = [&](uint32_t set, uint32_t step) {
    const uint32_t unit = step * kGroups + group;
    Unit u;
    u.t = unit / per_token;
    const uint32_t token = set * p.block_tokens + u.t;
    u.head = (int)(unit - u.t * per_token) * kRows;
    u.heads = unit < units && token < all ? min(kRows, all_heads - u.head) : 0;
    u.b = token / (uint32_t)p.tokens;
    u.at = token - u.b * (uint32_t)p.tokens;
    if (u.heads == 0) u.t = 0;
    return u;
  };
  uint4* ring = ring_all + threadIdx.x;
  uint32_t ahead_set = block, ahead_step = 0;
  int ahead_place = 0;
  auto copy_next = [&]() {
    if (ahead_set < sets) {
      const Unit u = unit_of(ahead_set, ahead_step);
      uint4* to = ring + ahead_place * (2 * kRows * kThreads);
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (i < u.heads) {
          copy_async16(to + i * kThreads, d_all + u.b * ds[0] + u.at * ds[1] + (u.head + i) * ds[2]);
          if (normed) copy_async16(to + (kRows + i) * kThreads, x_all + u.b * xs[0] + u.at * xs[1] + (u.head + i) * xs[2]);
        }
    }
    copy_commit();
    ahead_place = ahead_place + 1 == kRing ? 0 : ahead_place + 1;
    if (++ahead_step == steps) {
      ahead_step = 0;
      ahead_set += blocks;
    }
  };
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) copy_next();
  int place = 0;
  for (uint32_t set = block; set < sets; set += blocks) {
    const uint32_t first = set * p.block_tokens;
    __syncthreads();
    angles(p, first, (int)min((uint32_t)p.block_tokens, all - first), table);
    __syncthreads();
    for (uint32_t step = 0; step < steps; ++step) {
      const Unit u = unit_of(set, step);
      // (into the place that was read in the step before, by this thread alone)
      copy_next();
      copy_wait<kRing - 1>();
      const uint4* from = ring + place * (2 * kRows * kThreads);
      place = place + 1 == kRing ? 0 : place + 1;
      float cs[8], sn[8];
      load_angles<true>(table + 2 * u.t * p.pairs, span, p.pairs, p.interleaved, cs, sn);
      T* out = out_all + u.b * os[0] + u.at * os[1] + u.head * os[2];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        float g[8];
        open8<T>(i < u.heads ? from[i * kThreads] : make_uint4(0, 0, 0, 0), g);
        turn8<kLanes>(g, span, p.interleaved, cs, sn);
        if (normed) {
          float v[8];
          float2 s = make_float2(0.0f, 0.0f);
          open8<T>(i < u.heads ? from[(kRows + i) * kThreads] : make_uint4(0, 0, 0, 0), v);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            s.x = fmaf(v[j], v[j], s.x);
            s.y = fmaf(g[j] * w[j], v[j], s.y);
          }
          s = make_float2(row_sum<kLanes>(s.x), row_sum<kLanes>(s.y));
          const float r = rsqrtf(fmaf(s.x, 1.0f / D, p.eps)), along = s.y * r * (1.0f / D);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[j] *= r;
            weight_sum[j] = fmaf(g[j], v[j], weight_sum[j]);
            g[j] = r * fmaf(-v[j], along, g[j] * w[j]);
          }
        }
        if (i < u.heads) *reinterpret_cast<uint4*>(out + i * os[2]) = round8<T>(g);
      }
    }
  }
  copy_wait<0>();
  if (p.weight_partial == nullptr) return;
  // [group][D] over the ring, which nobody reads any more
  float* sums = reinterpret_cast<float*>(ring_all);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) sums[group * D + lane * 8 + j] = weight_sum[j];
  __syncthreads();
  if (threadIdx.x < D) {
    float total = 0.0f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) total += sums[g * D + threadIdx.x];
    p.weight_partial[(int64_t)blockIdx.x * D + threadIdx.x] = total;
  }
}

template <typename T>
__global__ void sums_kernel(const float* partial, int q_blocks, int k_blocks, int d, void* dq_weight, void* dk_weight) {
  const int column = blockIdx.x * 32 + threadIdx.x;
  void* out = blockIdx.y ? dk_weight : dq_weight;
  if (out == nullptr) return;
  const float v = column_sum(partial + (blockIdx.y ? (int64_t)q_blocks * d : 0), d, blockIdx.y ? k_blocks : q_blocks, column,
                             true);
  if (threadIdx.y == 0) store1(static_cast<T*>(out) + column, v);
}

// Four heads per group of lanes (four loads in flight, one read of weights for them) where heads fill them and the groups
// fill the SMs, one else.
int rows_of(const anemoi_sm100_axial_rope_shape* s) {
  const int64_t groups = (int64_t)kSms * kThreads / (s->head_dim / 8);
  return std::max(s->q_heads, s->k_heads) > 2 && s->batch * s->tokens * (s->q_heads + s->k_heads) > groups ? 4 : 1;
}

// The gradient's blocks: three per SM, shared by queries and keys as their heads are; tokens of a set: up to 16, whose units
// leave the fewest groups of lanes without one in the last step.
struct BackwardPlan {
  int q_blocks, k_blocks, block_tokens;
};
BackwardPlan plan_of(const anemoi_sm100_axial_rope_shape* s) {
  const int64_t tokens = s->batch * s->tokens;
  const int groups = kThreads / (s->head_dim / 8), blocks = kSms * 3;
  const int heads = s->q_heads + s->k_heads, per_token = (s->q_heads + kBackwardRows - 1) / kBackwardRows;
  BackwardPlan p{1, 0, 1};
  if (s->k_heads > 0) p.k_blocks = std::max(1, (int)((int64_t)blocks * s->k_heads / heads));
  p.q_blocks = blocks - p.k_blocks;
  double best = 0.0;
  for (int t = 1; t <= 16; ++t) {
    if (t > 1 && tokens / t < 4 * p.q_blocks) break;  // (few tokens: a set for every block first)
    const int steps = (t * per_token + groups - 1) / groups;
    const double share = (double)t * per_token / ((double)steps * groups);
    if (share > best + 0.02) {
      best = share;
      p.block_tokens = t;
    }
  }
  const int64_t sets = (tokens + p.block_tokens - 1) / p.block_tokens;
  p.q_blocks = (int)std::min<int64_t>(p.q_blocks, sets);
  p.k_blocks = (int)std::min<int64_t>(p.k_blocks, sets);
  return p;
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
  if (s->q_heads > 65536 || s->k_heads > 65536 || (s->batch > 0 && s->tokens > 0x7fffffffLL / s->batch))
    return ANEMOI_SM100_ELIMIT;
  return ANEMOI_SM100_OK;
}

void fill(RopeParams& p, const anemoi_sm100_axial_rope_shape* s, const double* turns, const int64_t* strides, int tensors) {
  p.batch = s->batch;
  p.tokens = s->tokens;
  p.q_heads = s->q_heads;
  p.k_heads = s->k_heads;
  p.axes = s->axes;
  p.interleaved = s->interleaved != 0;
  p.positions_type = s->positions_type;
  p.eps = s->eps;
  p.pairs = 0;
  for (int a = 0; a < s->axes; ++a) p.ends[a] = p.pairs += s->sections[a];
  for (int i = 0; i < p.pairs; ++i) p.turns[i] = turns[i];
  for (int i = 0; i < tensors; ++i)
    for (int j = 0; j < 3; ++j) p.strides[i][j] = strides[3 * i + j];
}

template <typename T, int D, int kRows>
int forward_launch(const RopeParams& p, cudaStream_t st) {
  constexpr int64_t kGroups = kThreads / (D / 8);
  const int64_t units = p.batch * p.tokens * ((p.q_heads + kRows - 1) / kRows + (p.k_heads + kRows - 1) / kRows);
  const int64_t blocks = (units + kGroups - 1) / kGroups;
  if (blocks > 0x7fffffffLL) return ANEMOI_SM100_ELIMIT;
  forward_kernel<T, D, kRows><<<(unsigned)blocks, kThreads, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? ANEMOI_SM100_OK : ANEMOI_SM100_ELAUNCH;
}

template <typename T, int D>
int backward_launch(RopeParams& p, const BackwardPlan& plan, void* dq_weight, void* dk_weight, cudaStream_t st) {
  p.block_tokens = plan.block_tokens;
  p.q_blocks = plan.q_blocks;
  auto kernel = backward_kernel<T, D>;
  constexpr int kSmem = kRing * 2 * kBackwardRows * kThreads * 16;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
    return ANEMOI_SM100_ELAUNCH;
  kernel<<<plan.q_blocks + plan.k_blocks, kThreads, kSmem, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return ANEMOI_SM100_ELAUNCH;
  if (p.weight_partial == nullptr) return ANEMOI_SM100_OK;
  sums_kernel<T><<<dim3(D / 32, 2), dim3(32, kSlices), 0, st>>>(p.weight_partial, plan.q_blocks, plan.k_blocks, D, dq_weight,
                                                                dk_weight);
  return cudaGetLastError() == cudaSuccess ? ANEMOI_SM100_OK : ANEMOI_SM100_ELAUNCH;
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
  const bool four = rows_of(s) == 4;
  if (s->is_bf16) {
    using T = __nv_bfloat16;
    if (s->head_dim == 64) return four ? forward_launch<T, 64, 4>(p, st) : forward_launch<T, 64, 1>(p, st);
    return four ? forward_launch<T, 128, 4>(p, st) : forward_launch<T, 128, 1>(p, st);
  }
  using T = __half;
  if (s->head_dim == 64) return four ? forward_launch<T, 64, 4>(p, st) : forward_launch<T, 64, 1>(p, st);
  return four ? forward_launch<T, 128, 4>(p, st) : forward_launch<T, 128, 1>(p, st);
}

extern "C" int64_t anemoi_sm100_axial_rope_backward_workspace(const anemoi_sm100_axial_rope_shape* s) {
  const int bad = check(s);
  if (bad != ANEMOI_SM100_OK) return bad;
  if (s->batch == 0 || s->tokens == 0) return 0;
  const BackwardPlan plan = plan_of(s);
  return (int64_t)(plan.q_blocks + plan.k_blocks) * s->head_dim * (int64_t)sizeof(float);
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
