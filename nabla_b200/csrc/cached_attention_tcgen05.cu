// Attention over a key / value cache in 8 bits for many rows (the operation and its terms: cached_attention.cu, cached_attention.cuh).
//
// A block of threads takes two tiles of 128 rows (tokens times the heads of a group, so that all heads that share a cache head share its
// codes) and walks over tiles of 128 keys. 12 warps:
//   warps 0-2   make 16-bit floats of codes: 16 bytes at a time from global memory, a tile ahead in registers, into the swizzled operand tiles
//   warps 4-11  two groups of 128 threads, one per row tile, thread r owns row r (lane r of tensor memory): queries, softmax, output
//   warp 3      allocates tensor memory and issues the products (one elected thread)
// Scores S (fp32) of row tile t are in columns t * 128 ..., the weights (16-bit floats, two in a column) take the place of the scores just read and
// feed the second product from there, the outputs are in columns 256 + t * D.
//
// Scales are one per 16 keys or more, so a row's 128 scores have 8 of them: the maximum is taken over each 16 scores first, then with the scales.
// Scores of keys that a row does not see are put out of sight before that, and whole groups of them are taken without their scale, which may be NaN.
// Keys keep the offset of their codes (1152 each), and the product's part of it, 1152 times the sum of the query's numbers, is taken from the
// scores; values do not, their offset would cancel against far smaller sums.
//
// 2 x 2048 new tokens behind 2048, 16 heads over 4 of 128: 144 us for 93 GFLOP, 645 TFLOP/s, 40 % of the library's rate for a plain product. What bounds it: the
// exponentials (2048 clocks of some 4600 for a tile of 128 keys and two of 128 rows) and the way from a product to its weights to the next product, which only
// the other group's work covers. Making the codes costs 12 us of it. Two threads for a row (219 us), groups that take turns (186), weights without the
// maximum first (153) and scores of 64 keys at a time (162) were slower.
#include "sm100_ptx.cuh"

#include "cached_attention.cuh"

namespace nbc {
using namespace nb;

constexpr int BT = 128, MANY_THREADS = 384, CONVERT = 96, ISSUER = 3, GROUPS = BT / 16;

struct ManyArgs {
  AttendArgs a;
  int q_tiles;                   // row tiles of a block: 2, or 1 where those of 2 would leave SMs without a block
  int* status;
};

template <int D>
struct ManySmem {
  static constexpr int TILE = BT * D * 2;
  static constexpr int Q = 0, K = 2 * TILE, V = 4 * TILE;                  // two of each
  static constexpr int SCALES = 6 * TILE;                                  // [4][key scale, log2 of the value scale, its reciprocal][8]
  static constexpr int BARS = SCALES + 4 * 3 * GROUPS * 4;
  static constexpr int RAW = BARS + 16 * 8 + 16 + 1024;
  static constexpr int TOTAL = RAW < 120 * 1024 ? 120 * 1024 : RAW;        // one block per SM (it takes all of tensor memory)
};

__host__ __device__ constexpr uint32_t idesc_f16(int n, int b_mn) {       // 16-bit floats, fp32 sums, 128 rows
  return (1u << 4) | (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}
// D[128 x 128] = A[128 x HD] B[128 x HD]^T, both tiles of HD / 64 swizzled chunks of 64 columns
template <int HD>
__device__ __forceinline__ void product_scores(uint32_t d, uint32_t a0, uint32_t b0) {
#pragma unroll
  for (int k = 0; k < HD / 16; ++k) {
    const uint32_t at = (k >> 2) * (BT * 128) + (k & 3) * 32;
    umma_f16_ss(d, make_smem_desc_sw128(a0 + at, 16, 1024), make_smem_desc_sw128(b0 + at, 16, 1024), idesc_f16(BT, 0), k != 0);
  }
}
// D[128 x HD] (+)= A[128 x 128] B[128 x HD]: A in tensor memory, B with the keys as rows
template <int HD>
__device__ __forceinline__ void product_values(uint32_t d, uint32_t a, uint32_t b0, bool accumulate) {
#pragma unroll
  for (int k = 0; k < BT / 16; ++k)
    umma_f16_ts(d, a + 8 * k, make_smem_desc_sw128(b0 + k * (16 * 128), BT * 128, 1024), idesc_f16(HD, 1), (accumulate || k != 0) ? 1u : 0u);
}
__device__ __forceinline__ void st_tmem16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
      "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void sts16(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// 16 codes as 16-bit floats, less the offset of 1152 or not
__device__ __forceinline__ void widen16(uint4 c, bool offset, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {c.x ^ 0x80808080u, c.y ^ 0x80808080u, c.z ^ 0x80808080u, c.w ^ 0x80808080u};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    o[i] = widen(w[i / 2], i & 1 ? 0x4342 : 0x4140);
    if (!offset) o[i] = half2_minus(o[i], BIAS2);
  }
  lo = make_uint4(o[0], o[1], o[2], o[3]);
  hi = make_uint4(o[4], o[5], o[6], o[7]);
}
__device__ __forceinline__ float2 two(uint32_t a, uint32_t b) { return make_float2(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ float top3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int D>
__global__ void __launch_bounds__(MANY_THREADS, 1) attend_many_kernel(const ManyArgs args) {
  using L = ManySmem<D>;
  const AttendArgs& a = args.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scales = reinterpret_cast<float*>(smem + L::SCALES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* q_full = bars + 0;     // [2] per row tile (128 arrivals)
  uint64_t* k_full = bars + 2;     // [2] (96 arrivals)
  uint64_t* k_empty = bars + 4;    // [2]
  uint64_t* v_full = bars + 6;     // [2] (96 arrivals)
  uint64_t* v_empty = bars + 8;    // [2]
  uint64_t* s_full = bars + 10;    // [2] per row tile: the scores of the next key tile are there, and the last product of weights has retired
  uint64_t* p_full = bars + 12;    // [2] per row tile: the weights are there (128 arrivals)
  uint64_t* o_done = bars + 14;    // [2] per row tile: the last product has retired
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // an earlier bounded wait on this device already failed, as far as is known before the grid ahead has ended: leave (uniformly)
  if (__syncthreads_or(threadIdx.x == 0 ? *reinterpret_cast<volatile int*>(args.status) : 0)) return follow_grid();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 128);
      mbar_init(&k_full[i], CONVERT);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], CONVERT);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_done[i], 1);
    }
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == ISSUER) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  follow_grid();

  const int group = a.heads / a.kv_heads, rows = a.fresh * group;
  const int nqt = (rows + args.q_tiles * BT - 1) / (args.q_tiles * BT), pairs = a.batch * a.kv_heads * a.splits;
  const int qt = nqt - 1 - static_cast<int>(blockIdx.x) / pairs;        // the late tiles of a causal problem see the most keys: first
  int at_ = static_cast<int>(blockIdx.x) % pairs;
  const int sp = at_ % a.splits;
  at_ /= a.splits;
  const int h = at_ % a.kv_heads, b = at_ / a.kv_heads;
  const int room = a.table.columns << a.block_log, past = clamp_tokens(a.past.at(b), room);
  const int count = clamp_tokens(a.count.p == nullptr ? a.fresh : a.count.at(b), a.fresh);
  const int all_keys = min(room, past + count);
  const int row0 = qt * args.q_tiles * BT;
  int n_t[2], first_t[2];          // key tiles of a row tile, the last key that its first row sees
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int r0 = row0 + t * BT, r1 = min(min(r0 + BT, rows), count * group);        // rows [r0, r1) are live
    const bool any = t < args.q_tiles && r0 < r1;
    const int keys = !any ? 0 : a.causal ? min(room, past + (r1 - 1) / group + 1) : all_keys;
    n_t[t] = (keys + BT - 1) / BT;
    first_t[t] = a.causal ? min(all_keys - 1, past + r0 / group) : all_keys - 1;
  }
  const int per = (max(n_t[0], n_t[1]) + a.splits - 1) / a.splits, kt0 = sp * per;       // this block's key tiles: [kt0, kt0 + n_t[t])
  n_t[0] = min(max(n_t[0] - kt0, 0), per);
  n_t[1] = min(max(n_t[1] - kt0, 0), per);
  const int n_max = max(n_t[0], n_t[1]);

  if (warp < ISSUER) {
    // ---- codes: a unit is 8 keys by 64 codes, lane takes piece (lane & 3) of key lane / 4, so that 8 lanes write two keys' pieces to all banks. The warps take
    // units in turn
    constexpr int PER_KEYS = D / 64, UNITS = BT / 8 * PER_KEYS, MINE = (UNITS + ISSUER - 1) / ISSUER;
    const int key = lane >> 2, c = lane & 3, n = 1 << a.block_log;
    // lane i < 8 knows where the i-th 16 keys of a tile lie (those of no block: the cache's first, so that loads need no condition: behind one they
    // would be waited for where the paths meet)
    struct Place { long long codes, unit; bool there, in; };
    auto find = [&](int j) {
      const int at = (kt0 + j) * BT + 16 * (lane & 7);
      const int id = j < n_max && at < all_keys ? a.table.block(b, at >> a.block_log) : -1;
      const long long unit = (long long)max(id, 0) * a.kv_heads + h;
      return Place{((unit << a.block_log) + (at & (n - 1))) * D, unit, id >= 0, holds_keys(a, unit, at & (n - 1))};
    };
    auto get = [&](int which, const Place& place, uint4 (&x)[MINE]) {
      const int8_t* codes = which ? a.codes[1] : a.codes[0];
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const int u = min(warp + i * ISSUER, UNITS - 1), k = u / PER_KEYS;
        const long long at = __shfl_sync(0xffffffffu, place.codes, k >> 1);
#ifdef NB_DEBUG_CHECKS
        if (!__shfl_sync(0xffffffffu, place.in, k >> 1)) continue;
#endif
        x[i] = ldg16(codes + at + ((k & 1) * 8 + key) * D + (u % PER_KEYS) * 64 + c * 16);
      }
    };
    auto put = [&](uint32_t tile, const uint4 (&x)[MINE], bool offset) {
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const int u = warp + i * ISSUER, k = u / PER_KEYS;
        uint4 lo, hi;
        widen16(x[i], offset, lo, hi);
        const uint32_t row = tile + (u % PER_KEYS) * (BT * 128) + (k * 8 + key) * 128;
        if (u < UNITS) {
          sts16(row + (((2 * c) ^ key) << 4), lo);
          sts16(row + (((2 * c + 1) ^ key) << 4), hi);
        }
      }
    };
    uint4 kr[MINE], vr[MINE];
    Place now = find(0), next = find(1);
    get(0, now, kr);
    get(1, now, vr);
    float sk = scale_at(a.scales[0], now.unit), sv = scale_at(a.scales[1], now.unit);
    bool ok = true;
    for (int j = 0; j < n_max; ++j) {
      const int st = j & 1;
      const uint32_t ph = ((j >> 1) & 1) ^ 1;
      ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[st], ph));      // (the warp exchanges below)
      if (!ok) break;
      put(smem_u32(smem + L::K + st * L::TILE), kr, true);
      if (threadIdx.x < GROUPS) {
        // (the softmax of the tile three ahead has let this one's place go)
        float* s = scales + (j & 3) * 3 * GROUPS + threadIdx.x;
        const float v = sv < LEAST_SCALE ? LEAST_SCALE : sv;
        s[0] = !now.there ? 1.f : sk < LEAST_SCALE ? LEAST_SCALE : sk;
        s[GROUPS] = !now.there ? -INFINITY : __log2f(v);
        s[2 * GROUPS] = !now.there ? 0.f : __fdividef(1.f, v);
      }
      fence_proxy_async_smem();
      mbar_arrive(&k_full[st]);
      get(0, next, kr);
      ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[st], ph));
      if (!ok) break;
      put(smem_u32(smem + L::V + st * L::TILE), vr, false);
      fence_proxy_async_smem();
      mbar_arrive(&v_full[st]);
      get(1, next, vr);
      sk = scale_at(a.scales[0], next.unit), sv = scale_at(a.scales[1], next.unit);
      now = next;
      next = find(j + 2);
    }
    if (!ok) atomicExch(args.status, NB_ERR_TIMEOUT_PRODUCER);
  } else if (warp == ISSUER) {
    if (n_max > 0 && elect_one()) {
      const uint32_t q = smem_u32(smem + L::Q), k = smem_u32(smem + L::K), v = smem_u32(smem + L::V);
      bool ok = true;
      auto qk = [&](int t, int j) {
        product_scores<D>(tmem + t * BT, q + t * L::TILE, k + (j & 1) * L::TILE);
        umma_commit(&s_full[t]);
      };
      auto pv = [&](int t, int j) {
        product_values<D>(tmem + 256 + t * D, tmem + t * BT, v + (j & 1) * L::TILE, j != 0);
        if (j == n_t[t] - 1) umma_commit(&o_done[t]);
      };
      for (int t = 0; t < 2 && ok; ++t)
        if (n_t[t] > 0) ok = mbar_wait(&q_full[t], 0);
      ok = ok && mbar_wait(&k_full[0], 0);
      if (ok) {
        tc_fence_after();
        if (n_t[0] > 0) qk(0, 0);
        if (n_t[1] > 0) qk(1, 0);
        umma_commit(&k_empty[0]);
      }
      for (int j = 0; j < n_max && ok; ++j) {
        const bool more = j + 1 < n_max;
        if (!mbar_wait(&v_full[j & 1], (j >> 1) & 1)) { ok = false; break; }
        if (more && !mbar_wait(&k_full[(j + 1) & 1], ((j + 1) >> 1) & 1)) { ok = false; break; }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (j < n_t[t]) {
            if (!mbar_wait(&p_full[t], j & 1)) { ok = false; break; }
            tc_fence_after();
            pv(t, j);
          }
          if (t == 1) umma_commit(&v_empty[j & 1]);
          if (j + 1 < n_t[t]) qk(t, j + 1);
        }
        if (!ok) break;
        if (more) umma_commit(&k_empty[(j + 1) & 1]);
      }
      if (!ok) atomicExch(args.status, NB_ERR_TIMEOUT_MMA);
    }
  } else {
    const int t = (warp - 4) >> 2, wq = warp & 3, r = wq * 32 + lane;
    const int row = row0 + t * BT + r, token = row / group, n = n_t[t];
    const bool live = t < args.q_tiles && row < rows && token < count;
    const uint32_t lane_at = static_cast<uint32_t>(wq * 32) << 16, t_s = tmem + t * BT + lane_at, t_o = tmem + 256 + t * D + lane_at;
    float row_mul = 0.f, offset = 0.f;
    if (n > 0) {
      // the row as 16-bit floats, its largest brought to [2^8, 2^9) by a power of two; its 128 bytes of 64 numbers lie in turned 16-byte pieces
      const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + b * a.q_sb + (long long)token * a.q_st + (long long)(h * group + row % group) * a.q_sh;
      float top = 0.f;
      if (live)
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          float x[8];
          load8(q + 8 * c, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
        }
      int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
      ex = ex == 128 || top == 0.f ? 8 : max(ex, -110);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + (8 - ex)) << 23);
      row_mul = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - (8 - ex)) << 23);
      const uint32_t to = smem_u32(smem + L::Q + t * L::TILE) + r * 128;
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (live) load8(q + 8 * c, x);
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = pack_half2(x[2 * e] * up, x[2 * e + 1] * up);
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
          sum += f.x + f.y;
        }
        sts16(to + (c >> 3) * (BT * 128) + (((c & 7) ^ (r & 7)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
      }
      offset = 1152.f * sum;
      fence_proxy_async_smem();
      mbar_arrive(&q_full[t]);
    }
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    const int last = a.causal ? min(all_keys - 1, past + token) : all_keys - 1;      // this row's last visible key
    for (int j = 0; j < n; ++j) {
      const int kv0 = (kt0 + j) * BT;
      if (!mbar_wait(&s_full[t], j & 1)) {
        atomicExch(args.status, NB_ERR_TIMEOUT_EPILOGUE);
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      uint32_t va[32], vb[32];
      if (kv0 + BT - 1 > first_t[t]) {
        // a tile on the diagonal or the last one: scores of hidden keys are put out of sight, so that the passes below know nothing of them
#pragma unroll 1
        for (int c = 0; c < BT / 32; ++c) {
          tmem_ld_32x32(t_s + c * 32, va);
          tmem_ld_wait_regs(va);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (kv0 + c * 32 + i > last) va[i] = __float_as_uint(-INFINITY);
          tmem_st_32x32(t_s + c * 32, va);
        }
        tmem_st_wait();
      }
      // pass 1: the maximum of each 16 scores, then with their scales. The next 32 columns are under way while these are worked on
      const float* sc = scales + (j & 3) * 3 * GROUPS;
      float gt[GROUPS], fs[GROUPS], adds[GROUPS];      // of 16 keys: the largest exponent; an exponent is a score times fs plus adds
      tmem_ld_32x32(t_s, va);
#pragma unroll
      for (int c = 0; c < BT / 32; ++c) {
        uint32_t (&v)[32] = (c & 1) ? vb : va;
        uint32_t (&nx)[32] = (c & 1) ? va : vb;
        tmem_ld_wait_regs(v);
        tmem_ld_32x32(t_s + ((c + 1) & 3) * 32, nx);       // after the last: the first again, for pass 2
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float x = __uint_as_float(v[16 * k]), y = __uint_as_float(v[16 * k + 1]);
#pragma unroll
          for (int i = 2; i < 16; i += 4) x = top3(x, __uint_as_float(v[16 * k + i]), __uint_as_float(v[16 * k + i + 1]));
#pragma unroll
          for (int i = 4; i < 16; i += 4) y = top3(y, __uint_as_float(v[16 * k + i]), __uint_as_float(v[16 * k + i + 1]));
          const float f = sc[2 * c + k] * row_mul;
          fs[2 * c + k] = f < 1e-37f ? 1e-37f : f;     // so that what is out of sight stays there
          adds[2 * c + k] = fmaf(-offset, fs[2 * c + k], sc[GROUPS + 2 * c + k]);
          gt[2 * c + k] = fmaf(fmaxf(x, y), fs[2 * c + k], adds[2 * c + k]);
        }
      }
      if (kv0 + BT - 1 > first_t[t]) {     // the scale of 16 keys that a row does not see may be NaN
#pragma unroll
        for (int k = 0; k < GROUPS; ++k)
          if (kv0 + 16 * k > last) fs[k] = 1.f, adds[k] = 0.f, gt[k] = -INFINITY;
      }
      const float mx = fmaxf(fmaxf(fmaxf(gt[0], gt[1]), fmaxf(gt[2], gt[3])), fmaxf(fmaxf(gt[4], gt[5]), fmaxf(gt[6], gt[7])));
      // the reference follows the maximum only when that has grown by 2^8
      float half = 1.f;                    // the root of what the sums so far are multiplied by (the factor may fall out of the range of fp32)
      bool grow = false;
      if (m == -INFINITY) {
        m = mx;                            // may stay: every key so far is hidden from this row
      } else if (mx > m + 8.f) {
        half = ex2(0.5f * (m - mx));
        m = mx;
        grow = true;
      }
      const float base = m == -INFINITY ? 0.f : m - ROOM;
      if (__any_sync(0xffffffffu, grow)) {
        // the output is not being written now: s_full also tracks the product of the weights before
        l = l * half * half;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32(t_o + c * 32, o);
          tmem_ld_wait_regs(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * half * half);
          tmem_st_32x32(t_o + c * 32, o);
        }
      }
      // weights that are lost in fp32 may count once their value's scale is taken out: exponentials of their own (rare)
      uint32_t small = 0;
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) small |= (gt[k] < base - 100.f && gt[k] > -INFINITY ? 1u : 0u) << k;
      if (__any_sync(0xffffffffu, small != 0)) {
#pragma unroll 1
        for (int k = 0; k < GROUPS; ++k) {
          uint32_t x[16];
          tmem_ld_32x16(t_s + 16 * k, x);
          tmem_ld_wait();
          float f = sc[k] * row_mul;
          f = f < 1e-37f ? 1e-37f : f;
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            asm volatile("" : "+r"(x[i]));
            sum += ex2(fmaf(__uint_as_float(x[i]), f, fmaf(-offset, f, sc[GROUPS + k])) - base - sc[GROUPS + k]);
          }
          if (small >> k & 1) l += sum;
        }
      }
      // Scores far from 0: an exponent is rounded as that of the maximum was, and less that then, so that the largest weight is 2^ROOM however far they are. It
      // takes the score's place (rare). Near 0 the rounding of the sum of the two constants does not count (2^-15 at 512)
      float far = fabsf(base);
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) far = fmaxf(far, adds[k] > -INFINITY ? fabsf(adds[k]) : 0.f);
      if (__any_sync(0xffffffffu, !(far < 512.f))) {
        tmem_ld_wait_regs(va);
#pragma unroll
        for (int c = 0; c < BT / 32; ++c) {
          if (c > 0) {
            tmem_ld_32x32(t_s + c * 32, va);
            tmem_ld_wait_regs(va);
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) va[i] = __float_as_uint(fmaf(__uint_as_float(va[i]), fs[2 * c + i / 16], adds[2 * c + i / 16]) - base);
          tmem_st_32x32(t_s + c * 32, va);
        }
        tmem_st_wait();
        tmem_ld_32x32(t_s, va);
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) fs[k] = 1.f, adds[k] = 0.f;
      } else {
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) adds[k] -= base;
      }
      // pass 2: weights over the first 64 columns of the scores
#pragma unroll
      for (int c = 0; c < BT / 32; ++c) {
        uint32_t (&v)[32] = (c & 1) ? vb : va;
        uint32_t (&nx)[32] = (c & 1) ? va : vb;
        tmem_ld_wait_regs(v);
        if (c + 1 < BT / 32) tmem_ld_32x32(t_s + (c + 1) * 32, nx);
        uint32_t pk[16];
        float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int k = 0; k < 2; ++k) {    // two groups of 16 in turn
            const int gi = 2 * c + k;
            const float2 x = __ffma2_rn(two(v[16 * k + 2 * i], v[16 * k + 2 * i + 1]), make_float2(fs[gi], fs[gi]), make_float2(adds[gi], adds[gi]));
            const float2 p = make_float2(ex2(x.x), ex2(x.y));
            acc[k] = __fadd2_rn(acc[k], p);
            pk[8 * k + i] = pack_half2(p.x, p.y);
          }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int gi = 2 * c + k;
          const float sum = acc[k].x + acc[k].y;
          l = fmaf(sum, sum != 0.f && !(small >> gi & 1) ? sc[2 * GROUPS + gi] : 0.f, l);      // a row that sees none of these keys does not see their scale either
        }
        st_tmem16(t_s + c * 16, pk);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[t]);
    }
    if (ok && n > 0) {
      if (!mbar_wait(&o_done[t], 0)) {
        atomicExch(args.status, NB_ERR_TIMEOUT_EPILOGUE);
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok && t < args.q_tiles) {
      tc_fence_after();
      const bool none = l == 0.f || !live;
      const float inverse = none ? 0.f : 1.f / l;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        if (n > 0) {
          tmem_ld_32x32(t_o + c * 32, v);
          tmem_ld_wait_regs(v);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0;
        }
        if (row >= rows) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float4 x = make_float4(__uint_as_float(v[4 * i]) * inverse, __uint_as_float(v[4 * i + 1]) * inverse, __uint_as_float(v[4 * i + 2]) * inverse,
                                 __uint_as_float(v[4 * i + 3]) * inverse);
          if (none) x = make_float4(0.f, 0.f, 0.f, 0.f);
          if (a.splits > 1) {
            store_part<D>(a, sp, b, h, row, 8 * c + i, x, none ? -INFINITY : m - ROOM + __log2f(l));
          } else {
            store_out<__nv_bfloat16, D>(a, b, h, row, 8 * c + i, x);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == ISSUER) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D>
cudaError_t launch_many(const AttendArgs& a, int* status, cudaStream_t stream) {
  ManyArgs args = {a, 2, status};
  const long long rows = (long long)a.fresh * (a.heads / a.kv_heads), pairs = (long long)a.batch * a.kv_heads * a.splits;
  if ((rows + 255) / 256 * pairs < 148) args.q_tiles = 1;
  const long long grid = (rows + args.q_tiles * BT - 1) / (args.q_tiles * BT) * pairs;
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const cudaError_t e = cudaFuncSetAttribute(attend_many_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, ManySmem<D>::TOTAL);
  if (e != cudaSuccess) return e;
  return launch_following(attend_many_kernel<D>, dim3(static_cast<unsigned>(grid)), dim3(MANY_THREADS), ManySmem<D>::TOTAL, stream, args);
}
template cudaError_t launch_many<64>(const AttendArgs&, int*, cudaStream_t);
template cudaError_t launch_many<128>(const AttendArgs&, int*, cudaStream_t);

}  // namespace nbc

NB_DEBUG_DEFINE(cached_attention_tcgen05)
