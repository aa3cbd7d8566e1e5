// Attention over a key / value cache in 8 bits for few rows, and the joining of parts (the operation: cached_attention.cu).
#pragma once
#include <cooperative_groups.h>

#include "cached_attention.cuh"

namespace nbc {
using nb::follow_grid;
using nb::launch_following;

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The transpose of an 8 x 8 tile of 16-bit numbers, lane (g, t) with numbers 2t and 2t + 1 of row g.
__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
// ---------------------------------------------------------------- few rows
// Up to 8 * RT rows (tokens times heads of a group) of one sequence and cache head, over one of `splits` ranges of its keys. The codes are the
// large operand of the products: S^T = K Q^T (16 keys by 8 rows) and O^T = V^T P^T (16 dims by 8 rows), so no part of a product is padding when
// there are 8 rows, and what is made of a code serves all rows. Fragments are read from global memory as the instruction wants them, whole
// sectors at a time; a product's reduction may run in any order, so a lane's 16 bytes of a key are the four dims each of four k-steps, and
// its 16 bytes of four values are rows of eight output tiles. Each of the four warps takes every fourth step of 32 keys and keeps its own
// reference, sum and output until the end; keys of the next step are on their way from when this step's are used up, so are values. No load
// stands behind a condition: it would be waited for where the paths meet.
//
// What bounds it: latency, then instructions. 2 x 120001 tokens, 16 heads over 2 of 128: 29.6 us for 123 MB, 4.15 TB/s, 64 % of a plain copy's rate; some 800
// instructions for 32 tokens, of which 320 make 16-bit floats of codes, at 12 warps an SM. 32 sequences of 200 to 4001, 16 heads over 4: 25 us
// for 69 MB, of which 8 are starts, the joining kernel and the way from the table to the first code. One sequence of 700 with 16 heads: 6 us.
// Slower were copies through shared memory (37 us for the first), and products of whole numbers with the weights in fixed point, which need no 16-bit floats
// but the maximum first and then more registers (35 to 43 us).
// Four-float piece c of a row of outputs in shared memory: pieces are turned so that the 8 lanes that an access serves at once meet different banks
// (lane (g, t) writes pieces g * D / 32 ... of rows 2t and 2t + 1).
template <int D>
__device__ __forceinline__ int out_at(int r, int c) { return r * (D / 4) + (c ^ (D == 128 ? r >> 1 & 3 : (r >> 1 & 1) | (r & 4))); }
template <int D, int RT>
struct Few {
  static constexpr int ROWS = 8 * RT;
  static constexpr int SMEM = (FEW_WARPS * ROWS * (D + 2) + ROWS * (D + 1)) * 4;
};

// How the keys are shared out:
//  ONE      a block for all keys of a sequence, head and tile of rows (FIRST: for one of `splits` ranges of them)
//  CLUSTER  a cluster of blocks for them, which joins its ranges in distributed shared memory (few sequences and heads: no second launch)
//  FLAT     all keys of all sequences and heads in one line, of which every block takes the same length, whatever the lengths of the sequences; a block
//           writes what it has for the (at most two) lines it does not hold whole, and attend_join_kernel joins them
enum Share { ONE, CLUSTER, FLAT };
constexpr int UNIT = FEW_WARPS * STEP, FLAT_BATCH = 1024;      // keys that a line is cut in multiples of; sequences that FLAT takes

// lines[b] = units of sequences in front of b, for b up to the batch, in shared memory. All threads.
template <bool PAST>
__device__ __forceinline__ void number_lines(const AttendArgs& a, int tiles, int* lines) {
  __shared__ int sums[FEW_WARPS];
  const int each = (a.batch + 32 * FEW_WARPS - 1) / (32 * FEW_WARPS), b0 = min(a.batch, static_cast<int>(threadIdx.x) * each), b1 = min(a.batch, b0 + each);
  const int room = a.table.columns << a.block_log;
  int own = 0;
  for (int b = b0; b < b1; ++b) {
    const int count = clamp_tokens(a.count.p == nullptr ? a.fresh : a.count.at<PAST>(b), a.fresh);
    const int keys = count == 0 ? 0 : min(room, clamp_tokens(a.past.at<PAST>(b), room) + count);
    const int units = (keys + UNIT - 1) / UNIT * a.kv_heads * tiles;
    lines[b + 1] = units;
    own += units;
  }
  int sum = own;                 // of the threads up to this one
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, sum, w);
    if ((threadIdx.x & 31) >= w) sum += x;
  }
  if ((threadIdx.x & 31) == 31) sums[threadIdx.x >> 5] = sum;
  __syncthreads();
  for (int w = 0; w < static_cast<int>(threadIdx.x >> 5); ++w) sum += sums[w];
  sum -= own;
  for (int b = b0; b < b1; ++b) sum += lines[b + 1], lines[b + 1] = sum;
  if (threadIdx.x == 0) lines[0] = 0;
  __syncthreads();
}

template <typename T, int D, int RT, Share SHARE, Role ROLE>
__global__ void __launch_bounds__(32 * FEW_WARPS, RT == 1 ? 3 : 2) attend_few_kernel(const AttendArgs a) {
  static_assert(ROLE != FIRST || SHARE == ONE, "the keys of a prefix are one sequence's: ranges of the same length");
  constexpr bool EXACT = sizeof(T) == 4;              // fp32: two parts, codes less their offset before the product
  constexpr int PARTS = EXACT ? 2 : 1, KSTEPS = D / 16, PIECES = D / 64, MT = D / 16, ROWS = 8 * RT;
  extern __shared__ __align__(16) uint8_t smem[];
  // SECOND works while the prefix is still being worked on, and waits before it stores results (launch.cuh says on what grounds): what it reads until then goes past L1
  constexpr bool PAST = ROLE == SECOND;
  if (!PAST) follow_grid();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int group = a.heads / a.kv_heads, tiles = (a.fresh * group + ROWS - 1) / ROWS;
  int sp = 0, h = 0, tile = 0, b = 0, line_from = 0, line_to = 0, line = 0;
  int* lines = reinterpret_cast<int*>(smem) + Few<D, RT>::SMEM / 4;
  if (SHARE == FLAT) {
    number_lines<PAST>(a, tiles, lines);
    const int all = lines[a.batch];
    // no more blocks than units, so that each has one: the joining kernel reads what every block between a line's first and last has written
    const int blocks = min(static_cast<int>(gridDim.x), all), c = blockIdx.x;
    if (c < blocks) line_from = static_cast<int>((long long)c * all / blocks), line_to = static_cast<int>((c + 1ll) * all / blocks);
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i <= a.batch; i += 32 * FEW_WARPS) a.lines[i] = lines[i];
  } else {
    sp = blockIdx.x % a.splits, h = blockIdx.x / a.splits % a.kv_heads, tile = blockIdx.x / a.splits / a.kv_heads % tiles,
    b = blockIdx.x / a.splits / a.kv_heads / tiles;
  }
  for (line = line_from; SHARE != FLAT || line < line_to;) {
  int piece = 0, slot = 0;             // FLAT: units of this piece, where it goes (-1: it is whole)
  int unit0 = 0;
  if (SHARE == FLAT) {
    int lo = 0, hi = a.batch;          // lines[lo] <= line < lines[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (lines[mid] <= line) lo = mid; else hi = mid;
    }
    b = lo;
    const int units = (lines[b + 1] - lines[b]) / (a.kv_heads * tiles), at = line - lines[b], pair = at / units;
    h = pair % a.kv_heads, tile = pair / a.kv_heads;
    unit0 = at - pair * units;
    piece = min(line_to - line, units - unit0);
    slot = piece == units ? -1 : 2 * static_cast<int>(blockIdx.x) + (unit0 == 0 ? 1 : 0);
    line += piece;
  }
  const int room = a.table.columns << a.block_log, past = ROLE == FIRST ? 0 : clamp_tokens(a.past.at<PAST>(b), room);
  const int count = clamp_tokens(ROLE == FIRST || a.count.p == nullptr ? a.fresh : a.count.at<PAST>(b), a.fresh);
  const int row0 = tile * ROWS, rows = min(ROWS, a.fresh * group - row0);       // row r: token r / group, head r % group
  const int live = min(rows, count * group - row0);                             // rows from here on are zero
  // keys that the last row sees
  const int keys = live <= 0 ? 0 : ROLE == FIRST ? clamp_tokens(a.limit.at(0), room) : static_cast<int>(min((long long)room, (long long)past + (a.causal ? (row0 + live - 1) / group + 1 : count)));
  const int per = SHARE == FLAT ? piece * UNIT : (keys + a.splits * STEP - 1) / (a.splits * STEP) * STEP;
  const Keys range = keys_of(keys, SHARE == FLAT ? unit0 * UNIT : sp * per, per);
  const int k0 = range.k0, k1 = range.k1, mine = steps_of(range, warp);
  const int all_see = a.causal ? min(keys - 1, past + row0 / group) : keys - 1;     // keys up to here are seen by every row
  const int n = 1 << a.block_log, last_key = max(k1 - 1, 0);

  // ---- where a step's codes lie
  // (of no block: the cache's first, so that loads need no condition: behind one they would be waited for where the paths meet. The step
  // behind the last is the last again.)
  struct Place { int id[2], there; };
  auto find = [&](int step) {
    const int at = key_of(range, warp, mine, step);
    const int x = a.table.block<PAST>(b, min(at, last_key) >> a.block_log), y = n == 16 ? a.table.block<PAST>(b, min(at + 16, last_key) >> a.block_log) : x;
    const Place p = {{max(x, 0), max(y, 0)}, (x >= 0 ? 1 : 0) | (y >= 0 && at + 16 < k1 ? 2 : 0)};
    return p;
  };
  auto unit = [&](const Place& p, int i) { return (long long)p.id[i] * a.kv_heads + h; };
  auto row = [&](int i, int step) { return row_of(key_of(range, warp, mine, step), i, n); };
  auto from = [&](const Place& p, int i, int step) { return ((unit(p, i) << a.block_log) + row(i, step)) * D; };
  uint4 kr[2][2][PIECES], vr[2][4];                   // [16 keys each][keys g and g + 8], [keys 2t, 2t + 1, 2t + 8, 2t + 9]
  float ks[2] = {0.f, 0.f}, vs[2] = {0.f, 0.f};
  auto get_keys = [&](const Place& p, int step) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!holds_keys(a, unit(p, i), row(i, step))) continue;
      const int8_t* at = a.codes[0] + from(p, i, step) + g * D + t * 16;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < PIECES; ++c) kr[i][u][c] = ldg16<PAST>(at + u * 8 * D + c * 64);
      ks[i] = scale_at<PAST>(a.scales[0], unit(p, i));
    }
  };
  auto get_values = [&](const Place& p, int step) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!holds_keys(a, unit(p, i), row(i, step))) continue;
      const int8_t* at = a.codes[1] + from(p, i, step) + 2 * t * D + g * (D / 8);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int8_t* codes = at + ((r & 1) + 8 * (r >> 1)) * D;
        if (D == 128) {
          vr[i][r] = ldg16<PAST>(codes);
        } else {
          const uint2 x = ldg8<PAST>(codes);
          vr[i][r].x = x.x, vr[i][r].y = x.y;
        }
      }
    }
  };
  Place now = find(0);
  get_keys(now, 0);
  get_values(now, 0);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    vs[i] = scale_at<PAST>(a.scales[1], unit(now, i));
  Place next = find(1);

  // ---- queries as the small operand: lane (g, t) holds dims 16 (t + 4 p) + 4 s + {0, 1} and {2, 3} of row g for k-step 4 p + s
  uint32_t qb[RT][PARTS][KSTEPS][2];
  float mul[RT][2], offset[RT][2];                    // of rows 2t and 2t + 1
  int lim[RT][2];                                     // the last key that they see
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    const int r = row0 + 8 * u + g;
    float x[KSTEPS][4], top = 0.f;
    const T* q = static_cast<const T*>(a.q) + b * a.q_sb + (long long)(r / group) * a.q_st + (long long)(h * group + r % group) * a.q_sh;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (8 * u + g < live) {
          if constexpr (PAST) load8_past(q + 16 * (t + 4 * p) + 8 * w, y); else load8(q + 16 * (t + 4 * p) + 8 * w, y);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[4 * p + 2 * w + e / 4][e % 4] = y[e], top = fmaxf(top, fabsf(y[e]));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^(8 - exponent of the largest); a row of zeros, of infinities or with a NaN is left as it is
    int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    ex = ex == 128 || top == 0.f ? 8 : max(ex, -110);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + (8 - ex)) << 23);
    const float back = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - (8 - ex)) << 23);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float y = x[k][2 * e] * up, z = x[k][2 * e + 1] * up;
        const uint32_t hi = pack_half2(y, z);
        qb[u][0][k][e] = hi;
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        if (EXACT) qb[u][PARTS - 1][k][e] = pack_half2(y - f.x, z - f.y);
        sum += f.x + f.y;
      }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
    for (int e = 0; e < 2; ++e) {                     // row 2t + e is that of lanes (2t + e, .)
      mul[u][e] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * e);
      offset[u][e] = EXACT ? 0.f : 1152.f * __shfl_sync(0xffffffffu, sum, 8 * t + 4 * e);
      lim[u][e] = a.causal ? min(keys - 1, past + (row0 + 8 * u + 2 * t + e) / group) : keys - 1;
    }
  }

  float o[RT][MT][4];                                 // [16 dims each][dim 2j, row 2t; row 2t + 1; dim 2j + 1 likewise] of lane g's dims
  float m[RT][2], l[RT][2];
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    m[u][0] = m[u][1] = -INFINITY, l[u][0] = l[u][1] = 0.f;
#pragma unroll
    for (int j = 0; j < MT; ++j) o[u][j][0] = o[u][j][1] = o[u][j][2] = o[u][j][3] = 0.f;
  }
#pragma unroll 1
  for (int step = 0; step < mine; ++step) {
    float s[RT][2][4];                                // [16 keys each][key g: rows 2t, 2t + 1; key g + 8: the same]
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) s[u][i][0] = s[u][i][1] = s[u][i][2] = s[u][i][3] = 0.f;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {                 // (two chains of products, in turn)
          const uint4 &kx = kr[i][0][p], &ky = kr[i][1][p];
          const uint32_t x = (k == 0 ? kx.x : k == 1 ? kx.y : k == 2 ? kx.z : kx.w) ^ 0x80808080u,
                         y = (k == 0 ? ky.x : k == 1 ? ky.y : k == 2 ? ky.z : ky.w) ^ 0x80808080u;
          uint32_t c[4] = {widen(x, 0x4140), widen(y, 0x4140), widen(x, 0x4342), widen(y, 0x4342)};
          if (EXACT)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = half2_minus(c[e], BIAS2);
#pragma unroll
          for (int u = 0; u < RT; ++u)
#pragma unroll
            for (int f = 0; f < PARTS; ++f) mma16816(s[u][i], c, qb[u][f][4 * p + k][0], qb[u][f][4 * p + k][1]);
        }
      }
    }
    const float sk[2] = {ks[0], ks[1]};
    get_keys(next, step + 1);

    const int key0 = k0 + (step * FEW_WARPS + warp) * STEP;
    float per_value[2], lg[2];                        // 1 / s_v, log2 s_v
    bool grow = false, small = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool is = now.there >> i & 1;
      const float sv = vs[i] < LEAST_SCALE ? LEAST_SCALE : vs[i];
      lg[i] = __log2f(sv);
      per_value[i] = __fdividef(1.f, sv);
#pragma unroll
      for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float f = mul[u][r] * sk[i], c = EXACT ? lg[i] : fmaf(-offset[u][r], f, lg[i]);
          s[u][i][r] = is ? fmaf(s[u][i][r], f, c) : -INFINITY;
          s[u][i][2 + r] = is ? fmaf(s[u][i][2 + r], f, c) : -INFINITY;
        }
    }
    if (key0 + STEP - 1 > all_see) {
#pragma unroll
      for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + 16 * i + 8 * (e >> 1) + g > lim[u][e & 1]) s[u][i][e] = -INFINITY;
    }
    // the reference that weights are taken against follows the maximum only when that has grown by 2^8
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float x = fmaxf(s[u][0][r], s[u][0][2 + r]), y = fmaxf(s[u][1][r], s[u][1][2 + r]), top = fmaxf(x, y), low = m[u][r] - 100.f;
        grow |= top > m[u][r] + 8.f;                  // (of nothing to something too)
        small |= (x < low && x > -INFINITY) || (y < low && y > -INFINITY);
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top = fmaxf(fmaxf(s[u][0][r], s[u][0][2 + r]), fmaxf(s[u][1][r], s[u][1][2 + r]));
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
          // in two steps: the factor alone may fall out of the range of fp32
          const float to = fmaxf(m[u][r], top), f = m[u][r] == to ? 1.f : ex2(0.5f * (m[u][r] - to));
          m[u][r] = to;
          l[u][r] = l[u][r] * f * f;
#pragma unroll
          for (int j = 0; j < MT; ++j) o[u][j][r] = o[u][j][r] * f * f, o[u][j][2 + r] = o[u][j][2 + r] * f * f;
        }
      small = true;                                   // (looked at under the reference before)
    }
    uint32_t pb[RT][PARTS][2][2];
    const bool apart = __any_sync(0xffffffffu, small);
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      const float base[2] = {m[u][0] == -INFINITY ? 0.f : m[u][0] - ROOM, m[u][1] == -INFINITY ? 0.f : m[u][1] - ROOM};
      if (apart) {                                    // weights that are lost in fp32 may count once their value's scale is taken out
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (s[u][i][e] != -INFINITY) l[u][e & 1] += ex2(s[u][i][e] - base[e & 1] - lg[i]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][i][e] = ex2(s[u][i][e] - base[e & 1]);
        if (!apart)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float sum = s[u][i][r] + s[u][i][2 + r];
            if (sum != 0.f) l[u][r] = fmaf(sum, per_value[i], l[u][r]);     // a row that sees none of these keys does not see their scale either
          }
#pragma unroll
        for (int k = 0; k < 2; ++k) {                 // keys g + 8 k of rows 2t, 2t + 1, turned to keys 2t, 2t + 1 (+ 8 k) of row g
          const uint32_t hi = pack_half2(s[u][i][2 * k], s[u][i][2 * k + 1]);
          pb[u][0][i][k] = turn8x8(hi);
          if (EXACT) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            pb[u][PARTS - 1][i][k] = turn8x8(pack_half2(s[u][i][2 * k] - f.x, s[u][i][2 * k + 1] - f.y));
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t w[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r) w[r][0] = vr[i][r].x, w[r][1] = vr[i][r].y, w[r][2] = vr[i][r].z, w[r][3] = vr[i][r].w;
#pragma unroll
      for (int j = 0; j < MT; ++j) {                  // dims 2 j and 2 j + 1 of this lane's
        const uint32_t sel = j & 1 ? 0x7362 : 0x5140;
        const uint32_t x = __byte_perm(w[0][j / 2], w[1][j / 2], sel) ^ 0x80808080u, y = __byte_perm(w[2][j / 2], w[3][j / 2], sel) ^ 0x80808080u;
        const uint32_t c[4] = {half2_minus(widen(x, 0x4140), BIAS2), half2_minus(widen(x, 0x4342), BIAS2), half2_minus(widen(y, 0x4140), BIAS2),
                               half2_minus(widen(y, 0x4342), BIAS2)};
#pragma unroll
        for (int u = 0; u < RT; ++u)
#pragma unroll
          for (int f = 0; f < PARTS; ++f) mma16816(o[u][j], c, pb[u][f][i][0], pb[u][f][i][1]);
      }
    }
    get_values(next, step + 1);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      vs[i] = scale_at<PAST>(a.scales[1], unit(next, i));
    now = next;
    next = find(step + 2);
  }

  // ---- join the warps in a fixed order, as ranges are joined: by the sums of their weights
  float4* so = reinterpret_cast<float4*>(smem);                                   // [warp][row][D]
  float* sm = reinterpret_cast<float*>(smem) + FEW_WARPS * ROWS * D;               // [warp][row] log2 of the sum of weights (over s_v)
  float* sl = sm + FEW_WARPS * ROWS;                                               //             one over their sum
  float* to = sl + FEW_WARPS * ROWS;                                               // CLUSTER: [row][D] of this block
  float* tl = to + ROWS * D;                                                       //          [row] log2 of the sum of weights
#pragma unroll
  for (int u = 0; u < RT; ++u)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l[u][r] += __shfl_xor_sync(0xffffffffu, l[u][r], w);
      const int row = 8 * u + 2 * t + r;
      if (g == 0) {
        sm[warp * ROWS + row] = l[u][r] == 0.f ? -INFINITY : m[u][r] - ROOM + __log2f(l[u][r]);
        sl[warp * ROWS + row] = l[u][r] == 0.f ? 0.f : 1.f / l[u][r];
      }
      if (row < live)
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
          so[warp * ROWS * (D / 4) + out_at<D>(row, g * (D / 32) + c)] =
              make_float4(o[u][2 * c][r], o[u][2 * c][2 + r], o[u][2 * c + 1][r], o[u][2 * c + 1][2 + r]);
    }
  if (PAST) follow_grid();
  __syncthreads();
  constexpr int PER = ROWS * (D / 4) / (32 * FEW_WARPS);
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int i = u * 32 * FEW_WARPS + threadIdx.x, row = i / (D / 4), c = i % (D / 4);
    if (row >= rows) break;
    float top = -INFINITY, sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < live) {
#pragma unroll
      for (int w = 0; w < FEW_WARPS; ++w) top = fmaxf(top, sm[w * ROWS + row]);
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < FEW_WARPS; ++w) {
        float f = ex2(sm[w * ROWS + row] - ref);
        const float4 y = so[w * ROWS * (D / 4) + out_at<D>(row, c)];
        sum += f;
        f *= sl[w * ROWS + row];
        x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
      }
    }
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;       // NaN stays
    x.x *= inverse, x.y *= inverse, x.z *= inverse, x.w *= inverse;
    const float weight = sum == 0.f ? -INFINITY : top + __log2f(sum);
    if (SHARE == CLUSTER) {
      reinterpret_cast<float4*>(to)[i] = x;
      if (c == 0) tl[row] = weight;
    } else if (SHARE == FLAT && slot >= 0) {
      reinterpret_cast<float4*>(a.part_o)[((long long)slot * ROWS + row) * (D / 4) + c] = x;
      if (c == 0) a.part_w[slot * ROWS + row] = weight;
    } else if (ROLE == FIRST) {
      store_part<D>(a, sp, b, h, row0 + row, c, x, weight);
    } else {
      store_result<T, D, ROLE>(a, b, h, row0 + row, c, x, weight, row < live);
    }
  }
  if (SHARE == CLUSTER) {
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    cluster.sync();
    for (int i = sp % a.splits * 32 * FEW_WARPS + threadIdx.x; i < rows * (D / 4); i += a.splits * 32 * FEW_WARPS) {
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
      store_result<T, D, ROLE>(a, b, h, row0 + row, c, x, sum == 0.f ? -INFINITY : top + __log2f(sum), row < live);
    }
    cluster.sync();                                   // a block's shared memory is read until here
  }
  if (SHARE != FLAT) break;
  __syncthreads();                                    // before the next piece's results
  }
  if (PAST && SHARE == FLAT) follow_grid();             // also of a block that has no share
}

// Joins the parts of each row in their order: those of ranges of keys (tiles of 128 rows), or of the pieces of a line (FLAT). One block per row; side s of its
// threads takes every SIDES-th part.
constexpr int JOIN_THREADS = 256;
template <typename T, int D, bool LINES, Role ROLE>
__global__ void __launch_bounds__(JOIN_THREADS) attend_join_kernel(const AttendArgs a) {
  constexpr int C = D / 4, SIDES = JOIN_THREADS / C;
  __shared__ float4 other[SIDES][C];
  __shared__ float others[SIDES], tops[SIDES];
  follow_grid();
  const int group = a.heads / a.kv_heads, c = threadIdx.x % C, side = threadIdx.x / C;
  const long long at = blockIdx.x;
  const int r = static_cast<int>(at % (a.fresh * group)), h = static_cast<int>(at / (a.fresh * group) % a.kv_heads),
            b = static_cast<int>(at / (a.fresh * group) / a.kv_heads);
  // part s of this row is number first + s * stride of the rows of parts; FLAT: behind the first, which ends its block's share, those that begin one
  long long first = at, stride = (long long)a.batch * a.kv_heads * a.fresh * group;
  int parts = a.splits;
  bool begins = false;
  if (LINES) {
    const int tile = r / a.tile_rows, tiles = (a.fresh * group + a.tile_rows - 1) / a.tile_rows, all = a.lines[a.batch];
    const int units = (a.lines[b + 1] - a.lines[b]) / (a.kv_heads * tiles), from = a.lines[b] + (tile * a.kv_heads + h) * units, to = from + units - 1;
    if (units == 0) {                                  // no keys: nobody has written it
      if (side == 0) store_result<T, D, ROLE>(a, b, h, r, c, make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, false);       // (a live row has its own key)
      return;
    }
    const long long n = min(a.splits, all);            // blocks that have a share
    const int c0 = static_cast<int>(((from + 1ll) * n - 1) / all), c1 = static_cast<int>(((to + 1ll) * n - 1) / all);
    if (c0 == c1) return;                              // one block had it whole
    parts = c1 - c0 + 1;
    begins = true;
    first = 2ll * c0 * a.tile_rows + r - tile * a.tile_rows;
    stride = 2ll * a.tile_rows;
  }
  auto place = [&](int s) { return first + s * stride + (begins && s == 0 ? a.tile_rows : 0); };
  // each side over its parts, eight under way at once, against the largest weight of the eights so far
  constexpr int AHEAD = 8;
  float top = -INFINITY, sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = side; s0 < parts; s0 += SIDES * AHEAD) {
    float w[AHEAD];
    float4 y[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int s = s0 + k * SIDES;
      w[k] = -INFINITY, y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s < parts) w[k] = a.part_w[place(s)], y[k] = reinterpret_cast<const float4*>(a.part_o)[place(s) * C + c];
    }
    float now = top;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) now = fmaxf(now, w[k]);
    const float ref = now == -INFINITY ? 0.f : now, f = ex2(top - ref);
    top = now;
    sum *= f, x.x *= f, x.y *= f, x.z *= f, x.w *= f;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const float e = ex2(w[k] - ref);
      sum += e;
      x.x = fmaf(e, y[k].x, x.x), x.y = fmaf(e, y[k].y, x.y), x.z = fmaf(e, y[k].z, x.z), x.w = fmaf(e, y[k].w, x.w);
    }
  }
  other[side][c] = x;
  if (c == 0) others[side] = sum, tops[side] = top;
  __syncthreads();
  if (side > 0) return;
#pragma unroll
  for (int s = 0; s < SIDES; ++s) top = fmaxf(top, tops[s]);
  const float ref = top == -INFINITY ? 0.f : top;
  x = make_float4(0.f, 0.f, 0.f, 0.f), sum = 0.f;
#pragma unroll
  for (int s = 0; s < SIDES; ++s) {
    const float4 y = other[s][c];
    const float f = ex2(tops[s] - ref);
    sum = fmaf(f, others[s], sum);
    x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
  }
  const float inverse = sum == 0.f ? 0.f : 1.f / sum;
  x.x *= inverse, x.y *= inverse, x.z *= inverse, x.w *= inverse;
  if (ROLE == ALONE) {
    store_out<T, D>(a, b, h, r, c, x);
  } else {
    const int count = clamp_tokens(a.count.p == nullptr ? a.fresh : a.count.at(b), a.fresh);
    store_result<T, D, ROLE>(a, b, h, r, c, x, sum == 0.f ? -INFINITY : top + __log2f(sum), r / group < count);
  }
}

// bf16 calls of more than 32 rows of a sequence and cache head go to tiles of 128 rows (cached_attention_tcgen05.cu), up to 128 rows where they are more tiles of
// 16 than 32, or than run at once where keys are few: the pass over the codes for each tile of 16 is then quicker than the longer start. us, tiles of 16 and of
// 128, 4 heads of 128: 4 pairs of sequence and head with 48 to 128 rows 9 to 11 and 18 to 20 for 1000 tokens, 20 to 21 and 20 to 24 for 8000; 32 pairs
// with 64 rows 15.5 and 26.1 for 1000, 27.4 and 27.5 for 2000, 69 and 55 for 8000; 64 pairs with 64 rows 32 and 43 for 2000, 131 and 97 for 8000, with 96
// rows (384 tiles) 59 and 50 for 2000; 128 pairs with 48 rows 36 and 29 for 1000.
static bool many(int rows, int fp32, long long pairs, long long room) {
  return !fp32 && rows > 32 && (rows > 128 || pairs * ((rows + 15) / 16) > (room <= 2048 ? 296 : 32));
}

// How a call is cut, by its sizes alone. (Both sides of each rule below were measured in bf16 with heads of 128. Heads of 64 and fp32 calls follow the same lines.
// fp32 calls of more than 128 rows are whole lines beyond what clusters take: a few long ones leave SMs without a block.)
struct Cut {
  Share share;
  int splits;                    // ranges of keys (tiles of 128 rows, CLUSTER), blocks (FLAT)
  int rows;                      // of a tile
  long long scratch;             // floats
};
static int few_rows(int rows) { return rows <= 8 ? 8 : 16; }
static Cut cut(int batch, int rows, long long heads_rows, int kv_heads, int head_dim, long long room, int fp32) {
  const bool wide = many(rows, fp32, (long long)batch * kv_heads, room);
  Cut c = {ONE, 1, wide ? 128 : few_rows(rows), 0};
  const long long units = (long long)batch * kv_heads * ((rows + c.rows - 1) / c.rows);
  if (wide) {
    const long long most = (room + 511) / 512, want = 148 / units;           // four tiles of keys at least
    c.splits = static_cast<int>(want < 2 || most < 2 ? 1 : want < most ? want : most);
    if (c.splits > 1) c.scratch = c.splits * heads_rows * (head_dim + 1);
    return c;
  }
  const long long most = (room + UNIT - 1) / UNIT;
  if (most < 2) return c;                                                    // a step for each warp
  // Lines that are short or many are not shared: a block that ends and begins within lines of 500 tokens has more to join than to read. us, shared and whole, with
  // 4 rows: 64 lines of 500 12.2 and 7.9, of 62 to 938 12.8 and 12.1, of 2000 20.6 and 23.8, of 250 to 3750 20.5 and 36.8; 256 of 500 22.5 and 13.9, of 2000
  // 36.8 and 35.4, of 250 to 3750 40.7 and 51.5; 1024 of 250 to 3750 127 and 111. With 16 rows: 64 lines of 500 15.4 and 11.0, of 2000 27.0 and 28.1; 256 of
  // 2000 57.8 and 35.2, of 250 to 3750 68.9 and 53.3, of 8000 131 and 114, of 1000 to 15000 143 and 191.
  const bool whole = room <= (c.rows == 16 && 24 * units > 1024 ? 24 * units : units < 1024 ? 1024 : 4 * units);
  // us, a cluster of 8 and a line for 4 query heads to each of 1, 8, 16, 32, 64 pairs: 2000 tokens 7.0 and 8.1, 7.7 and 9.2, 8.4 and 9.8, 11.3 and 16.2, 21.2 and
  // 20.7; 8000 tokens 12.7 and 8.9, 16.0 and 13.0, 18.4 and 18.0, 23.1 and 24.4, 42.5 and 34.1
  if (units * 8 <= 296 && room <= 4096 + 256 * units) {
    c.share = CLUSTER;
    c.splits = room >= 512 ? 8 : room >= 256 ? 4 : 2;
  } else if (!whole && rows <= 128 && batch <= FLAT_BATCH && units * most < (1ll << 31)) {
    c.share = FLAT;
    const long long blocks = 148 * (c.rows == 8 ? 3 : 2);
    c.splits = static_cast<int>(blocks < units * most ? blocks : units * most);
    c.scratch = 2ll * c.splits * c.rows * (head_dim + 1) + batch + 1;
  }
  return c;
}

static void set_parts(AttendArgs& a, const Cut& c, float* scratch, int head_dim) {
  a.splits = c.splits, a.tile_rows = c.rows;
  a.part_o = scratch;
  a.part_w = scratch + c.scratch / (head_dim + 1) * head_dim;
  if (c.share == FLAT) {
    a.part_w = scratch + 2ll * c.splits * c.rows * head_dim;
    a.lines = reinterpret_cast<int*>(a.part_w + 2ll * c.splits * c.rows);
  }
}

template <typename T, int D, bool LINES, Role ROLE>
static cudaError_t join(const AttendArgs& a, cudaStream_t stream) {
  return launch_following(attend_join_kernel<T, D, LINES, ROLE>, dim3(static_cast<unsigned>((long long)a.batch * a.fresh * a.heads)), dim3(JOIN_THREADS), 0, stream, a);
}

template <typename T, int D, int RT, Role ROLE>
static cudaError_t launch_few(const AttendArgs& a, const Cut& c, cudaStream_t stream) {
  const auto kernel = c.share == CLUSTER ? attend_few_kernel<T, D, RT, CLUSTER, ROLE> : c.share == FLAT ? attend_few_kernel<T, D, RT, FLAT, ROLE> : attend_few_kernel<T, D, RT, ONE, ROLE>;
  const long long grid = c.share == FLAT ? c.splits : (long long)c.splits * a.kv_heads * a.batch * ((a.fresh * (a.heads / a.kv_heads) + 8 * RT - 1) / (8 * RT));
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  static_assert(Few<D, RT>::SMEM + (FLAT_BATCH + 1) * 4 <= 48 * 1024, "no more than a kernel has without asking");
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(32 * FEW_WARPS);
  cfg.dynamicSmemBytes = Few<D, RT>::SMEM + (c.share == FLAT ? (a.batch + 1) * 4 : 0);
  cfg.stream = stream;
  cfg.attrs = attr;
  if (c.share == CLUSTER) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(c.splits);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  nb::set_following(cfg);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  return e != cudaSuccess || c.share != FLAT ? e : join<T, D, true, ROLE>(a, stream);
}

template <typename T, int D, Role ROLE>
static cudaError_t launch_attend(const AttendArgs& a, const Cut& c, int* status, cudaStream_t stream) {
  if (c.rows == 128) {
    const cudaError_t e = launch_many<D, ROLE>(a, 0, status, stream);
    return e != cudaSuccess || c.splits == 1 ? e : join<T, D, false, ROLE>(a, stream);
  }
  return c.rows == 8 ? launch_few<T, D, 1, ROLE>(a, c, stream) : launch_few<T, D, 2, ROLE>(a, c, stream);
}

}  // namespace nbc
