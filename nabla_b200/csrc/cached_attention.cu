// Attention over a key / value cache in 8 bits (layout: kv_cache.cuh).
//
//   o = sum_j softmax_j(scale * s_k(j) * (q . k_j)) * s_v(j) * v_j       codes k, v and scales s_k, s_v of the block that holds key j
//
// Query i of a sequence with `past` tokens in front and `count` new ones sees keys 0 ... past + i (causal) or past + count - 1. Rows from
// `count` on, and rows that see no key, are zero. `group` query heads share a head of the cache.
#include <cooperative_groups.h>

#include "kv_cache.cuh"

namespace nbc {
using nb::follow_grid;
using nb::launch_following;

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
  int splits;                    // ranges of keys
  float *part_o, *part_w;        // of ranges that no cluster joins: [splits][batch][kv_heads][new * group] output, and log2 of the sum of its weights
};

// Four neighbouring numbers of row r (token r / group, head r % group) of cache head h.
template <typename T, int D>
__device__ __forceinline__ void store_out(const AttendArgs& a, int b, int h, int r, int c, float4 x) {
  const int group = a.heads / a.kv_heads;
  T* p = static_cast<T*>(a.out) + (((long long)b * a.fresh + r / group) * a.heads + h * group + r % group) * D + 4 * c;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = x;
  } else {
    __nv_bfloat162 u = __floats2bfloat162_rn(x.x, x.y), w = __floats2bfloat162_rn(x.z, x.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&u), *reinterpret_cast<uint32_t*>(&w));
  }
}

// ---------------------------------------------------------------- matrix instructions on codes
// A code c becomes the 16-bit float 1024 + (c + 128) by placing its byte under the exponent of 1024; less 1152 that is c, exactly. So
// keys and values go into products of 16-bit floats (fp32 sums) without a rounding. What is rounded is the other operand:
//  - queries, to 11 bits after a power of two that brings a row's largest to [2^8, 2^9); bf16 has 8 bits, so those are exact (down to 2^-23 of the largest),
//  - weights, to 11 bits. fp32 calls carry queries and weights as two such parts (22 bits) and take two products.
// Scales never meet a rounding: a key's goes into its score, and a value's into the exponent of its weight. With
//     t_j = scale * log2(e) * s_k(j) * (q . k_j) + log2 s_v(j),   m = max t_j,   P_j = 2^(t_j - m)
// the output is sum P_j v_j / sum (P_j / s_v(j)), and the largest P is 1 however the scales differ. Where they differ so much that a P which counts in
// the lower sum falls out of the range of fp32, P_j / s_v(j) is taken as an exponential of its own.
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
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy16_async(uint32_t smem, const void* p) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(p) : "memory");
}
__device__ __forceinline__ void copy4_async(uint32_t smem, const void* p) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem), "l"(p) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}

// ---------------------------------------------------------------- few rows
// Up to 16 rows (tokens times heads of a group) of one sequence and cache head, over one of `splits` ranges of its keys. Each of the four warps
// takes every fourth step of 32 keys: it fetches codes and scales some steps ahead into a ring of its own, so warps never wait for one
// another, and keeps its own maximum, sum and output until the end. Bound by memory: every code is read once from HBM, and per 16 codes
// some 20 arithmetic and 2 matrix instructions are issued, whatever the number of rows.
constexpr int FEW_ROWS = 16, FEW_WARPS = 4, STEP = 32;
template <int D>
struct Few {
  static constexpr int STAGES = D == 128 ? 3 : 5;
  static constexpr int STAGE = 2 * STEP * D;                     // bytes: keys, then values
  static constexpr int RING = STAGES * (STAGE + 16);             // and the scales of two halves: keys', values'
  static constexpr int JOIN = FEW_WARPS * FEW_ROWS * (D + 2) * 4 + FEW_ROWS * (D + 1) * 4;
  static constexpr int SMEM = RING * FEW_WARPS > JOIN ? RING * FEW_WARPS : JOIN;
};
// Byte of 16-byte piece c of row r in a tile of codes. Rows of 128: keys are read 8 rows x 4 pieces at a time, values rows 2t at piece g; rows of 64
// lie in pairs. The pieces of a 128-byte line are turned so that the 8 (16) lanes that a shared-memory access serves at once meet different banks.
template <int D>
__device__ __forceinline__ int key_at(int r, int c) { return D == 128 ? r * 128 + ((c ^ ((r & 1) << 2)) << 4) : r * 64 + (c << 4); }
template <int D>
__device__ __forceinline__ int value_at(int r, int c) {
  return D == 128 ? r * 128 + ((c ^ (((r >> 1) & 3) << 1)) << 4) : (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (((r >> 1) & 3) << 1)) << 4);
}
// Four-float piece c of a row of outputs in shared memory, turned likewise.
template <int D>
__device__ __forceinline__ int out_at(int r, int c) {
  return D == 128 ? r * 32 + (c ^ (r & 7) ^ ((c >> 3) << 1)) : r * 16 + (c ^ (r & 1) ^ (((c >> 3) & 1) << 1));
}

template <typename T, int D, bool CLUSTER>
__global__ void __launch_bounds__(32 * FEW_WARPS, 2) attend_few_kernel(const AttendArgs a) {
  using L = Few<D>;
  constexpr bool EXACT = sizeof(T) == 4;              // fp32: two parts, codes less their offset before the product
  constexpr int PARTS = EXACT ? 2 : 1, KSTEPS = D / 16, PIECES = D / 64, NT = D / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  follow_grid();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int group = a.heads / a.kv_heads, tiles = (a.fresh * group + FEW_ROWS - 1) / FEW_ROWS;
  const int sp = blockIdx.x % a.splits, h = blockIdx.x / a.splits % a.kv_heads, tile = blockIdx.x / a.splits / a.kv_heads % tiles,
            b = blockIdx.x / a.splits / a.kv_heads / tiles;
  const int room = a.table.columns << a.block_log, past = clamp_tokens(a.past.at(b), room);
  const int count = clamp_tokens(a.count.p == nullptr ? a.fresh : a.count.at(b), a.fresh);
  const int row0 = tile * FEW_ROWS, rows = min(FEW_ROWS, a.fresh * group - row0);       // row r: token r / group, head r % group
  const int live = min(rows, count * group - row0);                                     // rows from here on are zero
  const int first = row0 / group, last = (row0 + live - 1) / group;
  // keys that the last row sees
  const int keys = live <= 0 ? 0 : static_cast<int>(min((long long)room, (long long)past + (a.causal ? last + 1 : count)));
  const int per = (keys + a.splits * STEP - 1) / (a.splits * STEP) * STEP;
  const int k0 = min(keys, sp * per), k1 = min(keys, k0 + per);
  const int steps = (k1 - k0 + STEP - 1) / STEP, mine = (steps - warp + FEW_WARPS - 1) / FEW_WARPS;
  // rows g and g + 8 of this lane: the last key that each sees
  int lim[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) lim[i] = a.causal ? min(keys - 1, past + (row0 + g + 8 * i) / group) : keys - 1;
  const int all_see = a.causal ? min(keys - 1, past + first) : keys - 1;     // keys up to here are seen by every row

  // ---- the ring: step n of this warp holds keys k0 + (n * 4 + warp) * 32 ...
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * L::RING;
  uint32_t there = 0;                                 // two bits per stage: is there a block behind each half
  int ids[2] = {-1, -1};
  const int n = 1 << a.block_log;
  auto find = [&](int step) {                         // blocks of a step, one step before its codes are asked for
    const int at = k0 + (step * FEW_WARPS + warp) * STEP;
#pragma unroll
    for (int i = 0; i < 2; ++i) ids[i] = step < mine && at + 16 * i < k1 ? a.table.block(b, (at + 16 * i) >> a.block_log) : -1;
  };
  auto fetch = [&](int step, int stage) {
    const uint32_t to = ring + stage * (L::STAGE + 16);
    const int at = k0 + (step * FEW_WARPS + warp) * STEP;
    there = (there & ~(3u << (2 * stage))) | ((ids[0] >= 0 ? 1u : 0u) | (ids[1] >= 0 ? 2u : 0u)) << (2 * stage);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (ids[i] < 0) continue;
      const long long unit = (long long)ids[i] * a.kv_heads + h;
      const long long from = ((unit << a.block_log) + ((at + 16 * i) & (n - 1))) * D;
#pragma unroll
      for (int u = 0; u < 16 * D / 512; ++u) {
        const int piece = u * 32 + lane, r = piece / (D / 16), c = piece % (D / 16);
        copy16_async(to + key_at<D>(16 * i + r, c), a.codes[0] + from + piece * 16);
        copy16_async(to + STEP * D + value_at<D>(16 * i + r, c), a.codes[1] + from + piece * 16);
      }
      if (lane < 2) copy4_async(to + L::STAGE + (lane * 2 + i) * 4, (lane ? a.scales[1] : a.scales[0]) + unit);
    }
  };
  find(0);
#pragma unroll
  for (int s = 0; s < L::STAGES - 1; ++s) {
    fetch(s, s);
    copies_commit();
    find(s + 1);
  }

  // ---- queries: lane (g, t) holds dims 16 (t + 4 p) + 4 s + {0, 1} and {2, 3} of rows g and g + 8 for k-step 4 p + s
  uint32_t qa[PARTS][KSTEPS][4];
  float mul[2], offset[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = row0 + g + 8 * i;
    float x[KSTEPS][4];
    const T* q = static_cast<const T*>(a.q) + b * a.q_sb + (long long)(r / group) * a.q_st + (long long)(h * group + r % group) * a.q_sh;
    float top = 0.f;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      float y[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (g + 8 * i < live) {
          load8(q + 16 * (t + 4 * p) + 8 * u, y);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[4 * p + 2 * u + e / 4][e % 4] = y[e], top = fmaxf(top, fabsf(y[e]));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^(8 - exponent of the largest); a row of zeros, of infinities or with a NaN is left as it is
    int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    ex = ex == 128 || top == 0.f ? 8 : max(ex, -110);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + (8 - ex)) << 23);
    mul[i] = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - (8 - ex)) << 23);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float u = x[k][2 * e] * up, w = x[k][2 * e + 1] * up;
        const uint32_t hi = pack_half2(u, w);
        qa[0][k][2 * e + i] = hi;
        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        if (EXACT) qa[PARTS - 1][k][2 * e + i] = pack_half2(u - back.x, w - back.y);
        sum += back.x + back.y;
      }
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (!EXACT) offset[i] = 1152.f * sum;
  }

  float o[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  int stage = 0;
#pragma unroll 1
  for (int step = 0; step < mine; ++step) {
    copies_wait<L::STAGES - 2>();
    __syncwarp();                                     // all lanes' copies of this step, and all lanes are through with the step before
    {
      const int ahead = step + L::STAGES - 1, into = stage == 0 ? L::STAGES - 1 : stage - 1;
      fetch(ahead, into);
      copies_commit();
      find(ahead + 1);
    }
    const uint32_t at = ring + stage * (L::STAGE + 16);
    const uint32_t blocks = there >> (2 * stage) & 3;
    stage = stage == L::STAGES - 1 ? 0 : stage + 1;
    if (blocks == 0) continue;
    const int key0 = k0 + (step * FEW_WARPS + warp) * STEP;
    float s[4][4];                                    // [8 keys each][row g: keys 2t, 2t + 1; row g + 8: the same]
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const uint4 w4 = lds16(at + key_at<D>(8 * j + g, t + 4 * p));
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t c = w[k] ^ 0x80808080u;
          uint32_t b0 = widen(c, 0x4140), b1 = widen(c, 0x4342);
          if (EXACT) b0 = half2_minus(b0, BIAS2), b1 = half2_minus(b1, BIAS2);
#pragma unroll
          for (int u = 0; u < PARTS; ++u) mma16816(s[j], qa[u][4 * p + k], b0, b1);
        }
      }
    }
    const uint4 sc = lds16(at + L::STAGE);
    float per_value[2], lg[2];                        // 1 / s_v, log2 s_v
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool is = blocks >> i & 1;
      const float sk = __uint_as_float(i ? sc.y : sc.x);
      float sv = __uint_as_float(i ? sc.w : sc.z);
      if (sv < LEAST_SCALE) sv = LEAST_SCALE;
      lg[i] = __log2f(sv);
      per_value[i] = is ? __fdividef(1.f, sv) : 0.f;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float f = mul[r] * sk, c = EXACT ? lg[i] : fmaf(-offset[r], f, lg[i]);
#pragma unroll
        for (int j = 2 * i; j < 2 * i + 2; ++j)
#pragma unroll
          for (int e = 2 * r; e < 2 * r + 2; ++e) s[j][e] = is ? fmaf(s[j][e], f, c) : -INFINITY;
      }
    }
    if (key0 + STEP - 1 > all_see) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key0 + 8 * j + 2 * t + (e & 1) > lim[e >> 1]) s[j][e] = -INFINITY;
    }
    // the reference that weights are taken against follows the maximum only when that has grown by 2^8: weights stay below 2^8
    bool grow = false;
    float top[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1])),
                     fmaxf(fmaxf(s[2][2 * r], s[2][2 * r + 1]), fmaxf(s[3][2 * r], s[3][2 * r + 1])));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      grow |= top[r] > m[r] + 8.f || (m[r] == -INFINITY && top[r] > -INFINITY);
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        // in two steps: the factor alone may fall out of the range of fp32
        const float now = fmaxf(m[r], top[r]), f = m[r] == now ? 1.f : ex2(0.5f * (m[r] - now));
        m[r] = now;
        l[r] = l[r] * f * f;
#pragma unroll
        for (int j = 0; j < NT; ++j) o[j][2 * r] = o[j][2 * r] * f * f, o[j][2 * r + 1] = o[j][2 * r + 1] * f * f;
      }
    }
    const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
    uint32_t pa[PARTS][2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float u = ex2(s[2 * i + j][2 * r] - base[r]), w = ex2(s[2 * i + j][2 * r + 1] - base[r]);
          sum[r] += u + w;
          const uint32_t hi = pack_half2(u, w);
          pa[0][i][2 * j + r] = hi;
          if (EXACT) {
            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            pa[PARTS - 1][i][2 * j + r] = pack_half2(u - back.x, w - back.y);
          }
        }
      bool small = false;                             // weights that are lost in fp32 may count once their value's scale is taken out
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float most = fmaxf(fmaxf(s[2 * i][2 * r], s[2 * i][2 * r + 1]), fmaxf(s[2 * i + 1][2 * r], s[2 * i + 1][2 * r + 1]));
        small |= most < base[r] - 100.f && most > -INFINITY;
      }
      if (__any_sync(0xffffffffu, small)) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = s[2 * i + e / 2][2 * r + e % 2];
            if (x != -INFINITY) l[r] += ex2(x - base[r] - lg[i]);
          }
      } else {
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (sum[r] != 0.f) l[r] = fmaf(sum[r], per_value[i], l[r]);     // a row that sees none of these keys does not see their scale either
      }
    }
    // lane (g, t): dims g * D / 8 ... of keys 2t, 2t + 1, 2t + 8, 2t + 9; the tile of 8 dims number j takes dims j, D / 8 + j, 2 D / 8 + j ...
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!(blocks >> i & 1)) continue;               // what lies there was never written: not even times zero
      uint32_t w[4][D / 32];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * i + 2 * t + (r & 1) + 8 * (r >> 1);
        if (D == 128) {
          const uint4 x = lds16(at + STEP * D + value_at<D>(row, g));
          w[r][0] = x.x, w[r][1] = x.y, w[r][D / 32 - 2] = x.z, w[r][D / 32 - 1] = x.w;
        } else {
          const uint2 x = lds8(at + STEP * D + value_at<D>(row, g >> 1) + 8 * (g & 1));
          w[r][0] = x.x, w[r][1] = x.y;
        }
      }
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {                 // dims 4 k + 2 e and + 1
          const uint32_t sel = e ? 0x7362 : 0x5140;
          const uint32_t x = __byte_perm(w[0][k], w[1][k], sel) ^ 0x80808080u, y = __byte_perm(w[2][k], w[3][k], sel) ^ 0x80808080u;
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            const uint32_t b0 = half2_minus(widen(x, f ? 0x4342 : 0x4140), BIAS2), b1 = half2_minus(widen(y, f ? 0x4342 : 0x4140), BIAS2);
#pragma unroll
            for (int u = 0; u < PARTS; ++u) mma16816(o[4 * k + 2 * e + f], pa[u][i], b0, b1);
          }
        }
      }
    }
  }

  // ---- join the warps in a fixed order, as ranges are joined: by the sums of their weights
  copies_wait<0>();
  __syncthreads();
  float4* so = reinterpret_cast<float4*>(smem);                                   // [warp][row][D]
  float* sm = reinterpret_cast<float*>(smem) + FEW_WARPS * FEW_ROWS * D;           // [warp][row] log2 of the sum of weights (over s_v)
  float* sl = sm + FEW_WARPS * FEW_ROWS;                                           //             one over their sum
  float* to = sl + FEW_WARPS * FEW_ROWS;                                           // CLUSTER: [row][D] of this block
  float* tl = to + FEW_ROWS * D;                                                   //          [row] log2 of the sum of weights
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int row = g + 8 * r;
    if (t == 0) {
      sm[warp * FEW_ROWS + row] = l[r] == 0.f ? -INFINITY : m[r] + __log2f(l[r]);
      sl[warp * FEW_ROWS + row] = l[r] == 0.f ? 0.f : 1.f / l[r];
    }
    if (row < live)
#pragma unroll
      for (int e = 0; e < 2; ++e)                     // dims (2 t + e) * D / 8 ...
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
          so[warp * FEW_ROWS * (D / 4) + out_at<D>(row, (2 * t + e) * (D / 32) + c)] =
              make_float4(o[4 * c][2 * r + e], o[4 * c + 1][2 * r + e], o[4 * c + 2][2 * r + e], o[4 * c + 3][2 * r + e]);
  }
  __syncthreads();
  constexpr int PER = FEW_ROWS * (D / 4) / (32 * FEW_WARPS);
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int i = u * 32 * FEW_WARPS + threadIdx.x, row = i / (D / 4), c = i % (D / 4);
    if (row >= rows) break;
    float top = -INFINITY, sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < live) {
#pragma unroll
      for (int w = 0; w < FEW_WARPS; ++w) top = fmaxf(top, sm[w * FEW_ROWS + row]);
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < FEW_WARPS; ++w) {
        float f = ex2(sm[w * FEW_ROWS + row] - ref);
        const float4 y = so[w * FEW_ROWS * (D / 4) + out_at<D>(row, c)];
        sum += f;
        f *= sl[w * FEW_ROWS + row];
        x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
      }
    }
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;       // NaN stays
    x.x *= inverse, x.y *= inverse, x.z *= inverse, x.w *= inverse;
    const float weight = sum == 0.f ? -INFINITY : top + __log2f(sum);
    if (CLUSTER) {
      reinterpret_cast<float4*>(to)[i] = x;
      if (c == 0) tl[row] = weight;
    } else if (a.splits > 1) {
      const long long at = (((long long)sp * a.batch + b) * a.kv_heads + h) * a.fresh * group + row0 + row;
      reinterpret_cast<float4*>(a.part_o)[at * (D / 4) + c] = x;
      if (c == 0) a.part_w[at] = weight;
    } else {
      store_out<T, D>(a, b, h, row0 + row, c, x);
    }
  }
  if (CLUSTER) {
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    cluster.sync();
    for (int i = sp * 32 * FEW_WARPS + threadIdx.x; i < rows * (D / 4); i += a.splits * 32 * FEW_WARPS) {
      const int row = i / (D / 4), c = i % (D / 4);
      float top = -INFINITY, sum = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int r = 0; r < a.splits; ++r) top = fmaxf(top, *cluster.map_shared_rank(&tl[row], r));
      const float ref = top == -INFINITY ? 0.f : top;
      for (int r = 0; r < a.splits; ++r) {
        const float f = ex2(*cluster.map_shared_rank(&tl[row], r) - ref);
        const float4 y = *cluster.map_shared_rank(&reinterpret_cast<float4*>(to)[i], r);
        sum += f;
        x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
      }
      const float inverse = sum == 0.f ? 0.f : 1.f / sum;
      x.x *= inverse, x.y *= inverse, x.z *= inverse, x.w *= inverse;
      store_out<T, D>(a, b, h, row0 + row, c, x);
    }
    cluster.sync();                                   // a block's shared memory is read until here
  }
}

// Joins the ranges of keys: one warp per row, in the order of the ranges.
template <typename T, int D>
__global__ void __launch_bounds__(128) attend_join_kernel(const AttendArgs a) {
  follow_grid();
  const int group = a.heads / a.kv_heads, lane = threadIdx.x & 31;
  const long long rows = (long long)a.batch * a.kv_heads * a.fresh * group, at = (long long)blockIdx.x * 4 + threadIdx.x / 32;
  if (at >= rows) return;
  float top = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) top = fmaxf(top, a.part_w[s * rows + at]);
#pragma unroll
  for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
  const float ref = top == -INFINITY ? 0.f : top;
  constexpr int C = D / 4, LANES = C < 32 ? 32 / C : 1;      // ranges that a warp reads at once
  float sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = lane / C; s < a.splits; s += LANES) {
    const float w = a.part_w[s * rows + at];
    const float4 y = reinterpret_cast<const float4*>(a.part_o)[(s * rows + at) * C + lane % C];
    const float f = ex2(w - ref);
    sum += f;
    x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
  }
  if (LANES == 2) {
    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
    x.x += __shfl_xor_sync(0xffffffffu, x.x, 16), x.y += __shfl_xor_sync(0xffffffffu, x.y, 16);
    x.z += __shfl_xor_sync(0xffffffffu, x.z, 16), x.w += __shfl_xor_sync(0xffffffffu, x.w, 16);
  }
  const float inverse = sum == 0.f ? 0.f : 1.f / sum;
  x.x *= inverse, x.y *= inverse, x.z *= inverse, x.w *= inverse;
  const int r = static_cast<int>(at % (a.fresh * group)), h = static_cast<int>(at / (a.fresh * group) % a.kv_heads),
            b = static_cast<int>(at / (a.fresh * group) / a.kv_heads);
  if (lane < C) store_out<T, D>(a, b, h, r, lane, x);
}


// Ranges of keys for each (sequence, head, 16 rows), by sizes alone. A cluster of up to 8 blocks joins its ranges in distributed shared memory; more
// go through memory and a second kernel.
static int few_splits(int batch, int fresh, int heads, int kv_heads, long long room) {
  const long long units = (long long)batch * kv_heads * ((fresh * (heads / kv_heads) + FEW_ROWS - 1) / FEW_ROWS);
  const long long most = (room + FEW_WARPS * STEP - 1) / (FEW_WARPS * STEP);           // a step for each warp at least
  long long want = (296 + units - 1) / units;
  if (want <= 8) want = 8;
  if (units * want > 4 * 296) want = 4;
  if (units * want > 4 * 296) want = 2;
  if (units * want > 4 * 296) want = 1;
  if (want > most) want = most;
  if (want < 8) want = want >= 4 ? 4 : want >= 2 ? 2 : 1;
  return static_cast<int>(want < 1 ? 1 : want > 128 ? 128 : want);
}

template <typename T, int D>
static cudaError_t launch_few(const AttendArgs& a, cudaStream_t stream) {
  const bool cluster = a.splits > 1 && a.splits <= 8;
  const auto kernel = cluster ? attend_few_kernel<T, D, true> : attend_few_kernel<T, D, false>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<D>::SMEM);
  if (e != cudaSuccess) return e;
  const long long grid = (long long)a.splits * a.kv_heads * a.batch * ((a.fresh * (a.heads / a.kv_heads) + FEW_ROWS - 1) / FEW_ROWS);
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(32 * FEW_WARPS);
  cfg.dynamicSmemBytes = Few<D>::SMEM;
  cfg.stream = stream;
  cfg.attrs = attr;
  if (cluster) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(a.splits);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  nb::set_following(cfg);
  e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess || cluster || a.splits == 1) return e;
  const long long rows = (long long)a.batch * a.fresh * a.heads;
  return launch_following(attend_join_kernel<T, D>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0, stream, a);
}

}  // namespace nbc

// Ranges of keys that nb_cached_attention is to be called with for these sizes. From 9 on it needs scratch: splits * batch * new * heads * (head_dim + 1)
// floats.
extern "C" int nb_cached_attention_splits(int batch, int fresh, int heads, int kv_heads, int head_dim, int block, int columns, int fp32) {
  return nbc::few_splits(batch, fresh, heads, kv_heads, (long long)columns * block);
}

extern "C" int nb_cached_attention(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, void* out,
                                   const void* table, const void* past, const void* count, int wide, int batch, int fresh, int heads, int kv_heads,
                                   int head_dim, int block, int blocks, int columns, long long q_sb, long long q_st, long long q_sh, float scale,
                                   int causal, int splits, float* scratch, int fp32, void* stream) {
  using namespace nbc;
  AttendArgs a = {};
  a.q = q, a.q_sb = q_sb, a.q_st = q_st, a.q_sh = q_sh;
  a.codes[0] = static_cast<const int8_t*>(k_codes), a.codes[1] = static_cast<const int8_t*>(v_codes);
  a.scales[0] = static_cast<const float*>(k_scales), a.scales[1] = static_cast<const float*>(v_scales);
  a.table = Table{Whole{table, wide & 1}, columns, blocks};
  a.past = Whole{past, wide >> 1 & 1};
  a.count = Whole{count, wide >> 2 & 1};
  a.out = out;
  a.batch = batch, a.fresh = fresh, a.heads = heads, a.kv_heads = kv_heads, a.causal = causal;
  a.block_log = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : block == 128 ? 7 : -1;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.splits = splits, a.part_o = scratch, a.part_w = scratch + (long long)splits * batch * fresh * heads * head_dim;
  if (a.block_log < 0 || (head_dim != 64 && head_dim != 128)) return -1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (fp32) return head_dim == 64 ? launch_few<float, 64>(a, s) : launch_few<float, 128>(a, s);
  return head_dim == 64 ? launch_few<__nv_bfloat16, 64>(a, s) : launch_few<__nv_bfloat16, 128>(a, s);
}

NB_DEBUG_DEFINE(cached_attention)
