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
constexpr int kMostTokens = 16;  // of a block

struct RopeParams {
  const void *q, *k, *dq_out, *dk_out, *q_weight, *k_weight, *positions;
  void *q_out, *k_out;
  float* weight_partial;  // [blocks][2][D]
  int64_t position_batch, batch, tokens;
  int64_t strides[6][3];  // forward: q, k, q_out, k_out; gradient: dq_out, dk_out, q, k, dq, dk
  int q_heads, k_heads, axes, pairs, interleaved, positions_type, block_tokens, splits;
  float eps;
  int ends[4];       // of the axes' pairs
  double turns[64];
};

// Cosines and sines of `count` tokens from `first` on.
__device__ __forceinline__ void angles(const RopeParams& p, int64_t first, int count, float2* table) {
  for (int i = threadIdx.x; i < count * p.pairs; i += kThreads) {
    const int t = i / p.pairs, pair = i - t * p.pairs;
    int axis = 0;
    while (axis < p.axes - 1 && pair >= p.ends[axis]) ++axis;
    const int64_t token = first + t, b = token / p.tokens;
    const int64_t at = b * p.position_batch + (token - b * p.tokens) * p.axes + axis;
    const double position = p.positions_type == 0   ? (double)static_cast<const int32_t*>(p.positions)[at]
                            : p.positions_type == 1 ? (double)static_cast<const int64_t*>(p.positions)[at]
                                                    : (double)static_cast<const float*>(p.positions)[at];
    const double turn = position * p.turns[pair];
    float s, c;
    sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
    table[i] = make_float2(c, s);
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

// Turns a lane's 8 channels by the token's angles (kBack: by the opposite ones).  All lanes of the warp take part.
template <int kLanes, bool kBack>
__device__ __forceinline__ void turn8(float (&n)[8], const Span& span, const float2* table, bool interleaved) {
  if (interleaved) {
    if (!span.in) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 cs = table[span.pair + i];
      const float s = kBack ? -cs.y : cs.y, u = n[2 * i], v = n[2 * i + 1];
      n[2 * i] = fmaf(-v, s, u * cs.x);
      n[2 * i + 1] = fmaf(u, s, v * cs.x);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float other = __shfl_sync(0xffffffffu, n[i], span.partner, kLanes);
    if (span.in) {
      const float2 cs = table[span.pair + i];
      n[i] = fmaf(other, span.first == kBack ? cs.y : -cs.y, n[i] * cs.x);
    }
  }
}

template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// A block takes block_tokens tokens (or a share of one token's heads): their angles once, in shared memory, for all heads
// of queries and keys.  Groups of D/8 lanes take kRows heads of one token at a time; the first ones' loads are in flight
// while the angles are formed.  HBM bound: two bytes in and two out per channel.
template <typename T, int D, int kRows>
__global__ void __launch_bounds__(kThreads) forward_kernel(const __grid_constant__ RopeParams p) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes;
  __shared__ float2 table[kMostTokens * 64];
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int64_t all = p.batch * p.tokens, first = (int64_t)(blockIdx.x / p.splits) * p.block_tokens;
  const int count = (int)min((int64_t)p.block_tokens, all - first);
  const int q_units = (p.q_heads + kRows - 1) / kRows, k_units = (p.k_heads + kRows - 1) / kRows;
  const int per_token = q_units + k_units, units = count * per_token, step = kGroups * p.splits;
  const Span span(lane, p.pairs, p.interleaved);
  const bool normed = p.q_weight != nullptr;
  uint4 raw[kRows];
  const T* src;
  T* dst;
  int64_t src_head, dst_head;
  int heads, t;
  const T* weight;
  auto fetch = [&](int unit) {
    t = unit / per_token;
    const int u = unit - t * per_token;
    const bool is_q = u < q_units;
    const int head = (is_q ? u : u - q_units) * kRows;
    heads = unit < units ? min(kRows, (is_q ? p.q_heads : p.k_heads) - head) : 0;
    t = unit < units ? t : 0;
    const int64_t token = first + t, b = token / p.tokens, at = token - b * p.tokens;
    const int64_t *in = p.strides[is_q ? 0 : 1], *out = p.strides[is_q ? 2 : 3];
    src = static_cast<const T*>(is_q ? p.q : p.k) + b * in[0] + at * in[1] + head * in[2] + lane * 8;
    dst = static_cast<T*>(is_q ? p.q_out : p.k_out) + b * out[0] + at * out[1] + head * out[2] + lane * 8;
    src_head = in[2];
    dst_head = out[2];
    weight = static_cast<const T*>(is_q ? p.q_weight : p.k_weight);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      raw[i] = make_uint4(0, 0, 0, 0);
      if (i < heads) raw[i] = load_stream(src + i * src_head);
    }
  };
  const int unit0 = (int)(blockIdx.x % p.splits) * kGroups + group;
  fetch(unit0);
  angles(p, first, count, table);
  __syncthreads();
  // (all groups take the same number of steps: they meet in the warp's shuffles)
  for (int base = unit0 - group; base < units; base += step) {
    if (base + group != unit0) fetch(base + group);
    const float2* row = table + t * p.pairs;
    float w[8];
    if (normed) shared8(weight + lane * 8, w);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float n[8];
      open8<T>(raw[i], n);
      if (normed) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(n[j], n[j], s);
        const float r = 1.0f / sqrtf(fmaf(row_sum<kLanes>(s), 1.0f / D, p.eps));
#pragma unroll
        for (int j = 0; j < 8; ++j) n[j] = n[j] * r * w[j];
      }
      turn8<kLanes, false>(n, span, row, p.interleaved);
      if (i < heads) *reinterpret_cast<uint4*>(dst + i * dst_head) = round8<T>(n);
    }
  }
}

// The gradient.  Blocks walk token groups a grid apart, queries' heads and then keys' heads, so that a thread's 8 sums of
// either weight stay in registers; a block's are added over its groups at the end, the blocks' by sums_kernel.
template <typename T, int D, int kRows>
__global__ void __launch_bounds__(kThreads) backward_kernel(const __grid_constant__ RopeParams p) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes;
  __shared__ float2 table[kMostTokens * 64];
  __shared__ float sums[kGroups][D + 4];
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int64_t all = p.batch * p.tokens;
  const Span span(lane, p.pairs, p.interleaved);
  const bool normed = p.q_weight != nullptr;
  float weight_sum[2][8] = {};
  for (int64_t first = (int64_t)blockIdx.x * p.block_tokens; first < all; first += (int64_t)gridDim.x * p.block_tokens) {
    const int count = (int)min((int64_t)p.block_tokens, all - first);
    __syncthreads();
    angles(p, first, count, table);
    __syncthreads();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int all_heads = which ? p.k_heads : p.q_heads, per_token = (all_heads + kRows - 1) / kRows;
      const int units = count * per_token;
      const T* weight = static_cast<const T*>(which ? p.k_weight : p.q_weight);
      float w[8];
      if (normed && units > 0) shared8(weight + lane * 8, w);
      const int64_t *ds = p.strides[which], *xs = p.strides[2 + which], *os = p.strides[4 + which];
      for (int base = 0; base < units; base += kGroups) {
        const int unit = base + group, t = unit < units ? unit / per_token : 0;
        const int head = unit < units ? (unit - t * per_token) * kRows : 0;
        const int heads = unit < units ? min(kRows, all_heads - head) : 0;
        const int64_t token = first + t, b = token / p.tokens, at = token - b * p.tokens;
        const T* d = static_cast<const T*>(which ? p.dk_out : p.dq_out) + b * ds[0] + at * ds[1] + head * ds[2] + lane * 8;
        const T* x = normed ? static_cast<const T*>(which ? p.k : p.q) + b * xs[0] + at * xs[1] + head * xs[2] + lane * 8
                            : nullptr;
        T* out = static_cast<T*>(which ? p.k_out : p.q_out) + b * os[0] + at * os[1] + head * os[2] + lane * 8;
        uint4 d_raw[kRows], x_raw[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          d_raw[i] = x_raw[i] = make_uint4(0, 0, 0, 0);
          if (i < heads) {
            d_raw[i] = load_stream(d + i * ds[2]);
            if (normed) x_raw[i] = load_stream(x + i * xs[2]);
          }
        }
        const float2* row = table + t * p.pairs;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          float g[8];
          open8<T>(d_raw[i], g);
          turn8<kLanes, true>(g, span, row, p.interleaved);
          if (normed) {
            float v[8], s = 0.0f;
            open8<T>(x_raw[i], v);
#pragma unroll
            for (int j = 0; j < 8; ++j) s = fmaf(v[j], v[j], s);
            const float r = 1.0f / sqrtf(fmaf(row_sum<kLanes>(s), 1.0f / D, p.eps));
            float along = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              v[j] *= r;
              weight_sum[which][j] = fmaf(g[j], v[j], weight_sum[which][j]);
              g[j] *= w[j];
              along = fmaf(g[j], v[j], along);
            }
            along = row_sum<kLanes>(along) * (1.0f / D);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = r * fmaf(-v[j], along, g[j]);
          }
          if (i < heads) *reinterpret_cast<uint4*>(out + i * os[2]) = round8<T>(g);
        }
      }
    }
  }
  if (p.weight_partial == nullptr) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[group][lane * 8 + j] = weight_sum[which][j];
    __syncthreads();
    if (threadIdx.x < D) {
      float total = 0.0f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) total += sums[g][threadIdx.x];
      p.weight_partial[((int64_t)blockIdx.x * 2 + which) * D + threadIdx.x] = total;
    }
  }
}

template <typename T>
__global__ void sums_kernel(const float* partial, int parts, int d, void* dq_weight, void* dk_weight) {
  const int column = blockIdx.x * 32 + threadIdx.x;
  void* out = blockIdx.y ? dk_weight : dq_weight;
  if (out == nullptr) return;
  const float v = column_sum(partial + blockIdx.y * d, 2 * d, parts, column, true);
  if (threadIdx.y == 0) store1(static_cast<T*>(out) + column, v);
}

// Four heads per group of lanes (four loads in flight, one read of weights for them) where heads fill them, one else.
int rows_of(const anemoi_sm100_axial_rope_shape* s) { return std::max(s->q_heads, s->k_heads) > 2 ? 4 : 1; }
int units_of(const anemoi_sm100_axial_rope_shape* s) {
  const int rows = rows_of(s);
  return (s->q_heads + rows - 1) / rows + (s->k_heads + rows - 1) / rows;
}

// Tokens of a block: the fewest, up to 16, whose units leave the fewest groups of lanes without one in the last step.
int block_tokens(const anemoi_sm100_axial_rope_shape* s, int64_t tokens, int units) {
  const int groups = kThreads / (s->head_dim / 8);
  int best = 1;
  double best_share = 0.0;
  for (int t = 1; t <= kMostTokens; ++t) {
    // (few tokens: a block for every SM first)
    if (t > 1 && tokens / t < kSms * 4) break;
    const int steps = (t * units + groups - 1) / groups;
    const double share = (double)t * units / ((double)steps * groups);
    if (share > best_share + 0.02) {
      best_share = share;
      best = t;
    }
  }
  return best;
}

constexpr int kBackwardBlocks = kSms * 4;

int backward_blocks(const anemoi_sm100_axial_rope_shape* s) {
  const int64_t tokens = s->batch * s->tokens;
  const int each = block_tokens(s, tokens, units_of(s));
  return (int)std::min<int64_t>(kBackwardBlocks, (tokens + each - 1) / each);
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
  p.splits = 1;
}

template <typename T, int D, int kRows>
int forward_launch(RopeParams& p, const anemoi_sm100_axial_rope_shape* s, cudaStream_t st) {
  constexpr int kGroups = kThreads / (D / 8);
  const int64_t tokens = s->batch * s->tokens;
  const int units = units_of(s);
  p.block_tokens = block_tokens(s, tokens, units);
  // few tokens of many heads: several blocks share a token
  if (p.block_tokens == 1)
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>((units + kGroups - 1) / kGroups, kSms * 2 / tokens));
  const int64_t blocks = (tokens + p.block_tokens - 1) / p.block_tokens * p.splits;
  forward_kernel<T, D, kRows><<<(unsigned)blocks, kThreads, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? ANEMOI_SM100_OK : ANEMOI_SM100_ELAUNCH;
}

template <typename T, int D, int kRows>
int backward_launch(RopeParams& p, const anemoi_sm100_axial_rope_shape* s, void* dq_weight, void* dk_weight,
                    cudaStream_t st) {
  p.block_tokens = block_tokens(s, s->batch * s->tokens, units_of(s));
  const int blocks = backward_blocks(s);
  backward_kernel<T, D, kRows><<<blocks, kThreads, 0, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return ANEMOI_SM100_ELAUNCH;
  if (p.weight_partial == nullptr) return ANEMOI_SM100_OK;
  sums_kernel<T><<<dim3(D / 32, 2), dim3(32, kSlices), 0, st>>>(p.weight_partial, blocks, D, dq_weight, dk_weight);
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
    if (s->head_dim == 64) return four ? forward_launch<T, 64, 4>(p, s, st) : forward_launch<T, 64, 1>(p, s, st);
    return four ? forward_launch<T, 128, 4>(p, s, st) : forward_launch<T, 128, 1>(p, s, st);
  }
  using T = __half;
  if (s->head_dim == 64) return four ? forward_launch<T, 64, 4>(p, s, st) : forward_launch<T, 64, 1>(p, s, st);
  return four ? forward_launch<T, 128, 4>(p, s, st) : forward_launch<T, 128, 1>(p, s, st);
}

extern "C" int64_t anemoi_sm100_axial_rope_backward_workspace(const anemoi_sm100_axial_rope_shape* s) {
  const int bad = check(s);
  if (bad != ANEMOI_SM100_OK) return bad;
  if (s->batch == 0 || s->tokens == 0) return 0;
  return (int64_t)backward_blocks(s) * 2 * s->head_dim * (int64_t)sizeof(float);
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
  const bool four = rows_of(s) == 4;
  if (s->is_bf16) {
    using T = __nv_bfloat16;
    if (s->head_dim == 64)
      return four ? backward_launch<T, 64, 4>(p, s, dq_weight, dk_weight, st)
                  : backward_launch<T, 64, 1>(p, s, dq_weight, dk_weight, st);
    return four ? backward_launch<T, 128, 4>(p, s, dq_weight, dk_weight, st)
                : backward_launch<T, 128, 1>(p, s, dq_weight, dk_weight, st);
  }
  using T = __half;
  if (s->head_dim == 64)
    return four ? backward_launch<T, 64, 4>(p, s, dq_weight, dk_weight, st)
                : backward_launch<T, 64, 1>(p, s, dq_weight, dk_weight, st);
  return four ? backward_launch<T, 128, 4>(p, s, dq_weight, dk_weight, st)
              : backward_launch<T, 128, 1>(p, s, dq_weight, dk_weight, st);
}
