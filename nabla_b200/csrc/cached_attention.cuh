// What the kernels of attention over a key / value cache in 8 bits share (the operation: cached_attention.cu).
#pragma once
#include "kv_cache.cuh"

namespace nbc {

struct AttendArgs {
  const void* q;                 // [batch][new][heads][D]
  long long q_sb, q_st, q_sh;        // its strides in elements
  const int8_t* codes[2];        // keys, values
  const float* scales[2];
  Table table;
  Whole past, count;             // count.p null: all of them
  void* out;                     // [batch][new][heads][D], dense
  int batch, fresh, heads, kv_heads, block_log, causal;
  float scale_log2;              // softmax scale * log2(e)
  int splits;                    // ranges of keys, one block each; or blocks that share all keys
  int tile_rows;
  // fp32 results of parts, and log2 of the sum of their weights: [splits][batch][kv_heads][new * group] rows, or two tiles of rows for each block
  float *part_o, *part_w;
  int* lines;                    // see attend_few_kernel
};

// Few rows: a block's warps take steps of STEP keys of its range in turn. The keys of a range, and the row of its block at which the loads of 16 keys start,
// half i of a step. Loads have no condition, so every row that comes out of this lies in the block, with the 15 behind it: also those of a warp that
// has no step (`mine` up to 0).
constexpr int FEW_WARPS = 4, STEP = 32;
struct Keys {
  int k0, k1;
};
__host__ __device__ __forceinline__ Keys keys_of(int keys, int from, int length) {
  Keys k = {0, 0};                                    // empty: at the first key, where 16 keys start (at the last one, they do not)
  if (from < keys) k.k0 = from, k.k1 = keys - from < length ? keys : from + length;
  return k;
}
__host__ __device__ __forceinline__ int steps_of(const Keys& k, int warp) { return ((k.k1 - k.k0 + STEP - 1) / STEP - warp + FEW_WARPS - 1) / FEW_WARPS; }
__host__ __device__ __forceinline__ int key_of(const Keys& k, int warp, int mine, int step) {
  const int last = step < mine - 1 ? step : mine - 1;
  return k.k0 + ((last > 0 ? last : 0) * FEW_WARPS + warp) * STEP;
}
__host__ __device__ __forceinline__ int row_of(int key, int i, int block) { return (key + 16 * i) & (block - 1); }

// Checked build: do the 16 keys from row `row` of a block and head lie in that block, and it in the cache?
__device__ __forceinline__ bool holds_keys(const AttendArgs& a, long long unit, int row) {
  return NB_IN_BOUNDS(NB_SITE_CACHE_CODE, unit, (long long)a.table.blocks * a.kv_heads) && NB_IN_BOUNDS(NB_SITE_CACHE_ROW, row, (1 << a.block_log) - 15);
}

// Four neighbouring numbers of row r (token r / group, head r % group) of cache head h.
template <typename T, int D>
__device__ __forceinline__ void store_out(const AttendArgs& a, int b, int h, int r, int c, float4 x) {
  const int group = a.heads / a.kv_heads;
  if (!NB_IN_BOUNDS(NB_SITE_CACHE_ROW, r, a.fresh * group)) return;
  T* p = static_cast<T*>(a.out) + (((long long)b * a.fresh + r / group) * a.heads + h * group + r % group) * D + 4 * c;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = x;
  } else {
    __nv_bfloat162 u = __floats2bfloat162_rn(x.x, x.y), w = __floats2bfloat162_rn(x.z, x.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&u), *reinterpret_cast<uint32_t*>(&w));
  }
}

template <int D>
__device__ __forceinline__ void store_part(const AttendArgs& a, int part, int b, int h, int r, int c, float4 x, float weight) {
  const long long at = (((long long)part * a.batch + b) * a.kv_heads + h) * a.fresh * (a.heads / a.kv_heads) + r;
  reinterpret_cast<float4*>(a.part_o)[at * (D / 4) + c] = x;
  if (c == 0) a.part_w[at] = weight;
}

// ---------------------------------------------------------------- matrix instructions on codes
// A code c becomes the 16-bit float 1024 + (c + 128) by placing its byte under the exponent of 1024; less 1152 that is c, exactly. So
// keys and values go into products of 16-bit floats (fp32 sums) without a rounding. What is rounded is the other operand:
//  - queries, to 11 bits after a power of two that brings a row's largest to [2^8, 2^9); bf16 has 8 bits, so those are exact (down to 2^-23 of the largest),
//  - weights, to 11 bits. fp32 calls carry queries and weights as two such parts (22 bits) and take two products.
// Scales never meet a rounding: a key's goes into its score, and a value's into the exponent of its weight. With
//     t_j = scale * log2(e) * s_k(j) * (q . k_j) + log2 s_v(j),   m = max t_j,   P_j = 2^(t_j - m)
// the output is sum P_j v_j / sum (P_j / s_v(j)), and the largest P is near 1 however the scales differ. Where they differ so much that a P which counts in
// the lower sum falls out of the range of fp32, P_j / s_v(j) is taken as an exponential of its own.
// The m that weights are taken against is the largest t so far or up to 8 below it, and they are taken 2^ROOM larger: they stay below 2^15, and small ones, and
// the second parts of those of fp32 calls, keep their bits (16-bit floats have none below 2^-24). What is lost of a weight is at most 2^-32 of
// the largest: with 2^-25, a million keys that have 2 % of the sum together gave nothing to the output.
constexpr float ROOM = 7.f;
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_minus(uint32_t x, uint32_t y) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
  return d;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// 1024 + 128 + codes 0, 1 (sel 0x4140) or 2, 3 (sel 0x4342) of a word of biased codes
__device__ __forceinline__ uint32_t widen(uint32_t biased, uint32_t sel) { return __byte_perm(biased, 0x64646464u, sel); }
constexpr uint32_t BIAS2 = 0x64806480u;      // 1152 twice
// Many rows: tiles of 128 rows on the tensor cores (cached_attention_tcgen05.cu), bf16 only.
template <int D>
cudaError_t launch_many(const AttendArgs& a, int* status, cudaStream_t stream);

}  // namespace nbc
