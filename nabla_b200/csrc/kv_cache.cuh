// What the kernels around a key / value cache in 8 bits share: where a token lies, and how a block's codes stand for numbers.
//
// The cache holds `blocks` blocks of N tokens (N a power of two, 16 to 128). For the keys and for the values there are codes
// [blocks][heads][N][D] (int8) and scales [blocks][heads] (fp32); code c of a block stands for c * scale. Position t of sequence b lies in
// row t % N of block table[b][t / N]. An entry of the table that names no block (negative, or too large) is a place without tokens:
// writes to it are dropped, reads give zeros, attention sees no key there. So no content of a table leads out of the cache.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "launch.cuh"
#include "nb_debug.cuh"

namespace nbc {

constexpr float LEAST_SCALE = 7.888609052210118e-31f;      // 2^-100: its reciprocal and its logarithm are finite

// A vector of whole numbers in 32 or 64 bits, one or the other as the caller has it.
struct Whole {
  const void* p;
  int wide;
  __device__ __forceinline__ long long at(long long i) const {
    long long v;
    int w;
    if (wide) {
      asm volatile("ld.global.s64 %0, [%1];" : "=l"(v) : "l"(static_cast<const long long*>(p) + i));      // volatile: behind the wait for the grid ahead
      return v;
    }
    asm volatile("ld.global.s32 %0, [%1];" : "=r"(w) : "l"(static_cast<const int*>(p) + i));
    return w;
  }
};
// Numbers i, i + step ... below `end` at once, -1 for the others and for what no int holds.
template <int N>
__device__ __forceinline__ void several(const Whole& w, long long base, int i, int step, int end, int (&out)[N]) {
  if (w.wide) {
    long long v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = -1;
      if (i + k * step < end) asm volatile("ld.global.s64 %0, [%1];" : "=l"(v[k]) : "l"(static_cast<const long long*>(w.p) + base + i + k * step));
    }
#pragma unroll
    for (int k = 0; k < N; ++k) out[k] = v[k] >= 0 && v[k] <= 0x7fffffff ? static_cast<int>(v[k]) : -1;
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      out[k] = -1;
      if (i + k * step < end) asm volatile("ld.global.s32 %0, [%1];" : "=r"(out[k]) : "l"(static_cast<const int*>(w.p) + base + i + k * step));
    }
  }
}
__device__ __forceinline__ float scale_at(const float* p, long long i) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p + i));
  return v;
}

struct Table {
  Whole ids;          // [batch][columns]
  int columns;
  int blocks;         // of the cache
  __device__ __forceinline__ int block(int b, int column) const {      // -1: none
    if (column >= columns || column < 0) return -1;
    const long long id = ids.at((long long)b * columns + column);
    return id >= 0 && id < blocks ? static_cast<int>(id) : -1;
  }
};

// Tokens that a sequence has, from 0 to what its row of the table has room for (below 2^30).
__device__ __forceinline__ int clamp_tokens(long long n, long long most) { return static_cast<int>(n < 0 ? 0 : n > most ? most : n); }

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
// Codes are read once by a block, past L1. (The address comes from the table, so these cannot move ahead of the wait for the grid ahead.)
__device__ __forceinline__ uint4 ldg16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ldg8(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// Eight numbers as they lie in memory.
template <typename T>
struct Eight;
template <>
struct Eight<__nv_bfloat16> {
  uint4 w;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void clear() { w = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ uint32_t top() const {              // of the magnitudes, which order as their bits do
    const uint32_t m = 0x7fff7fffu, x = __vmaxu2(__vmaxu2(w.x & m, w.y & m), __vmaxu2(w.z & m, w.w & m));
    return max(x & 0xffff0000u, x << 16);
  }
  __device__ __forceinline__ float2 pair(int i) const {
    const uint32_t x = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  }
};
template <>
struct Eight<float> {
  uint4 w, v;
  __device__ __forceinline__ void load(const float* p) { w = reinterpret_cast<const uint4*>(p)[0], v = reinterpret_cast<const uint4*>(p)[1]; }
  __device__ __forceinline__ void clear() { w = v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ uint32_t top() const {
    const uint32_t m = 0x7fffffffu;
    return max(max(max(w.x & m, w.y & m), max(w.z & m, w.w & m)), max(max(v.x & m, v.y & m), max(v.z & m, v.w & m)));
  }
  __device__ __forceinline__ float2 pair(int i) const {
    return i == 0 ? make_float2(__uint_as_float(w.x), __uint_as_float(w.y)) : i == 1 ? make_float2(__uint_as_float(w.z), __uint_as_float(w.w))
         : i == 2 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y)) : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
};
template <typename T>
__device__ __forceinline__ T round_to(float x);
template <>
__device__ __forceinline__ float round_to<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

}  // namespace nbc
