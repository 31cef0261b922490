// Pieces shared by the kernels that walk rows of channels (modulation.cu, axial_rope.cu): 8 channels per thread as one
// 16-byte access, sums over the lanes of a row, and sums of partial columns in a fixed order.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace rows {

constexpr int kSms = 148;

// Streamed once: past L1, whose lines are for what the rows share (modulation, weights).
__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// The same into shared memory, without registers: per thread, in groups that complete in order.  (A thread reads back what
// it copied itself, so that no barrier is needed.)
__device__ __forceinline__ void copy_async16(void* smem, const void* p) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(smem))),
               "l"(p)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLater>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLater) : "memory");
}

// a / b without a 64-bit division where both are below 2^32.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((uint64_t)a | (uint64_t)b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  static __device__ __forceinline__ float2 open(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  static __device__ __forceinline__ uint32_t round(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 open(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t round(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

template <typename T>
__device__ __forceinline__ void open8(const uint4& raw, float (&f)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = Pair<T>::open(w[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 round8(const float (&f)[8]) {
  return make_uint4(Pair<T>::round(f[0], f[1]), Pair<T>::round(f[2], f[3]), Pair<T>::round(f[4], f[5]),
                    Pair<T>::round(f[6], f[7]));
}

// 8 values that many rows share, in 16 or 32 bits.
template <typename M>
__device__ __forceinline__ void shared8(const M* p, float (&f)[8]) {
  open8<M>(__ldg(reinterpret_cast<const uint4*>(p)), f);
}
template <>
__device__ __forceinline__ void shared8<float>(const float* p, float (&f)[8]) {
  *reinterpret_cast<float4*>(f) = __ldg(reinterpret_cast<const float4*>(p));
  *reinterpret_cast<float4*>(f + 4) = __ldg(reinterpret_cast<const float4*>(p) + 1);
}
template <typename M>
__device__ __forceinline__ void store8(M* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = round8<M>(f);
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&f)[8]) {
  *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(f);
  *reinterpret_cast<float4*>(p + 4) = *reinterpret_cast<const float4*>(f + 4);
}
template <typename M>
__device__ __forceinline__ void store1(M* p, float v);
template <>
__device__ __forceinline__ void store1<float>(float* p, float v) {
  *p = v;
}
template <>
__device__ __forceinline__ void store1<__half>(__half* p, float v) {
  *p = __float2half_rn(v);
}
template <>
__device__ __forceinline__ void store1<__nv_bfloat16>(__nv_bfloat16* p, float v) {
  *p = __float2bfloat16_rn(v);
}
template <typename M>
__device__ __forceinline__ float load1(const M* p);
template <>
__device__ __forceinline__ float load1<float>(const float* p) {
  return *p;
}
template <>
__device__ __forceinline__ float load1<__half>(const __half* p) {
  return __half2float(*p);
}
template <>
__device__ __forceinline__ float load1<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}

// Sum of `parts` rows of `columns` fp32 partial sums, `stride` values apart, by a block of 32 x kSlices threads: slice y
// takes the parts y, y + kSlices, ..., the slices are added in order.  The order depends on `parts` alone, so that equal
// calls give equal bits.  Thread (x, 0) returns the sum of column `column`.
constexpr int kSlices = 16;
__device__ __forceinline__ float column_sum(const float* partial, int64_t stride, int parts, int column, bool in) {
  __shared__ float part[kSlices][33];
  float sum = 0.0f;
  if (in) {
#pragma unroll 4
    for (int i = threadIdx.y; i < parts; i += kSlices) sum += partial[(int64_t)i * stride + column];
  }
  part[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  float total = 0.0f;
  if (threadIdx.y == 0)
#pragma unroll
    for (int y = 0; y < kSlices; ++y) total += part[y][threadIdx.x];
  return total;
}

}  // namespace rows
