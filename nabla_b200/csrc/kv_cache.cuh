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
    return wide ? static_cast<const long long*>(p)[i] : static_cast<long long>(static_cast<const int*>(p)[i]);
  }
};

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
template <typename T>
__device__ __forceinline__ T round_to(float x);
template <>
__device__ __forceinline__ float round_to<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

}  // namespace nbc
