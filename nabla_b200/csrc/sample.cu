// The draw of tokens from logits. Per row, with T its temperature:
//   order     by logit, the largest first, equal ones by their ids
//   w_v       = exp((z_v - max z) / T); those below 2^-44 are left out
//   top-k     keeps the first k
//   top-p     keeps those in front of which less than p of the sum of the w so far kept lies
//   min-p     keeps those with w >= m
//   token     the first, by id, with which the sum of the kept w exceeds u times all of it
// T <= 0: the first in order. A row without a token (-inf or NaN everywhere): -1.
//
// Borders have to be met exactly, and sums must not depend on the order in which threads add: weights are whole multiples of 2^-43, computed in 64 bits (a draw
// differs from one in exact arithmetic about once in 2^30), and their sums are sums of whole numbers. What the first k or a share p cut off is
// found by selection, not by a sort: a histogram of the logits by their distance from the largest, in 2048 steps of a 45th of an octave of w, says where
// the border lies, up to a step for p. Where all that is kept is some hundreds of tokens (a usual k) they are put into a list in shared memory, which is all
// that the rest works on. Else a pass makes the sums exact and checks the border; the tokens of its steps, some tens, are ranked in a list, and another
// pass makes the draw. Where too many are left (equal logits, flat rows) steps are cut into 2048 finer ones of the order, down to single tokens.
//
// What bounds it is neither memory nor the number of instructions but rows that wait. 256 rows of 32001 in bf16 with filters of their own take 54 to 75 us with the
// seed (85 seen), of which issue is 16: 17.9 million of a warp, four to a clock (1.9 were reached). The time is that of the slowest rows, those with top-p alone,
// each with the block or cluster that its index gave it, when rows with top-k alone (33 us for a call of them) are long done and their SMs idle; and a row waits at
// barriers, at some 15 rounds of exchange between its threads (a row of 1000 takes 8 us) and for loads, with 24 warps to an SM. 32 rows of 131072 with top-p 59 to 76;
// 512 rows of 8192 without filters 19, in 1.15 waves of blocks (floors of memory 2.5, 2.6, 1.3). Slower were, in turn on one box and seed, a list of all that a bin of the
// threads' largest logits lets through in place of the histogram (61 us for the first, against 56) and three steps around the border of top-p in place of one (65).
//
// A row is read two to four times, all but the first from the caches, by one block of threads or by a cluster of up to eight, which exchange sums,
// histograms and lists over distributed shared memory. Warps own stretches of ids.
#include <cooperative_groups.h>

#include "kv_cache.cuh"

namespace nbc {
using nb::follow_grid;

using u64 = unsigned long long;

struct SampleArgs {
  const void* in;                // [batch][vocab]
  const float *uniform, *temperature, *top_p, *min_p;        // [batch], null: temperature 1, no filter
  Whole top_k;                   // p null: no filter
  long long* out;                // [batch]
  int vocab, blocks;             // blocks of a row
};

constexpr int SAMPLE_THREADS = 512, SAMPLE_WARPS = SAMPLE_THREADS / 32, BINS = 2048, LIST = SAMPLE_THREADS, MOST_BLOCKS = 8;
constexpr float FAR = 45.f;      // octaves that the histogram covers: weights end at 44
constexpr double UNIT_WEIGHT = 8796093022208.0;              // 2^43

// Where a token stands in the order: larger is earlier. 0: nowhere (-inf, NaN). Keys order as numbers do.
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t u = __float_as_uint(z + 0.f);               // (-0 as 0)
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float number_of(uint32_t key) { return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ u64 order_of(float z, int v) { return z > -INFINITY ? (static_cast<u64>(key_of(z)) << 32) | (0xffffffffu - static_cast<uint32_t>(v)) : 0; }
__device__ __forceinline__ int token_of(u64 order) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(order)); }

struct Weigher {
  float top, half_top, per_half; // the largest logit, half of it (two logits may be further apart than the largest number); octaves of w for half a unit of logit
  double top64, rate;            // 32 octaves
  const double* roots;           // 2^(-i / 32), in shared memory
  bool alone;                    // the largest logit, or what a unit of logit is worth, is infinite: only tokens with that logit have a weight

  __device__ __forceinline__ Weigher(float largest, float temperature, const double* table) : top(largest), half_top(0.5f * largest), top64(largest), roots(table) {
    rate = 46.166241308446828 / static_cast<double>(temperature);                        // 32 log2(e)
    per_half = static_cast<float>(rate / 16.0);
    alone = top == INFINITY || per_half == INFINITY;
  }
  __device__ __forceinline__ float octaves(float z) const { return fmaf(z, -0.5f, half_top) * per_half; }
  // The step of the histogram that a logit falls into, BINS: behind its end, or nowhere. Monotone.
  __device__ __forceinline__ int bin(float z) const {
    if (alone) return z == top ? 0 : BINS;
    const float x = octaves(z);
    return x < FAR ? __float_as_int(fmaf(x, (BINS - 1) / FAR, 8388608.f)) & 0xfff : BINS;        // + 2^23: the nearest whole number is in the low bits
  }
  __device__ __forceinline__ float about(float z) const { return alone ? (z == top ? 1.f : 0.f) : exp2f(-octaves(z)); }
  // w in multiples of 2^-43. With t in 32nds of octaves and n the whole number next to it: exp(-(t - n) ln 2 / 32) by its series (the term behind the last is
  // below 2^-48), times a root of 2, put where its last bit is 2^-43 by adding 2^52. A logit of -inf and NaN have none.
  __device__ __forceinline__ u64 fixed(float z) const {
    if (alone) return z == top ? 1ull << 43 : 0;
    const double t = (top64 - static_cast<double>(z)) * rate, whole = t + 6755399441055744.0;       // 1.5 * 2^52
    const int n = __double2loint(whole);
    const double x = t - (whole - 6755399441055744.0);
    constexpr double U = -0.021660849392498290;              // -ln 2 / 32
    double e = fma(x, U * U * U * U * U / 120.0, U * U * U * U / 24.0);
    e = fma(x, e, U * U * U / 6.0), e = fma(x, e, U * U / 2.0), e = fma(x, e, U), e = fma(x, e, 1.0);
    const double unit = __hiloint2double((1023 + 43 - (n >> 5)) << 20, 0);                 // 2^(43 - n / 32)
    const double w = fma(e * roots[n & 31], unit, 4503599627370496.0);
    return t <= 32.0 * 44.0 ? static_cast<u64>(__double_as_longlong(w)) & 0xfffffffffffffull : 0;
  }
};

// A row, eight tokens at a time from where memory is aligned; each warp has a stretch of ids.
template <typename T>
struct LogitRow {
  const T* in;
  int vocab, shift, from, to, per_warp;                      // groups of eight of this warp, of each
  __device__ __forceinline__ LogitRow(const T* p, int n, int rank, int blocks) : in(p), vocab(n) {
    shift = static_cast<int>(reinterpret_cast<uintptr_t>(p) / sizeof(T) & 7);
    const int groups = (vocab + shift + 7) / 8, warps = blocks * SAMPLE_WARPS, each = ((groups + warps - 1) / warps + 31) / 32 * 32;
    per_warp = each;
    from = min(groups, (rank * SAMPLE_WARPS + static_cast<int>(threadIdx.x >> 5)) * each), to = min(groups, from + each);
  }
  __device__ __forceinline__ bool whole(int v) const { return v >= 0 && v + 8 <= vocab && NB_IN_BOUNDS(NB_SITE_LOGITS_TOKEN, v + 7, vocab); }
  // The eight logits from token v on, -inf where there is none
  __device__ __forceinline__ void get(int v, float (&z)[8]) const {
    if (whole(v)) {
      Eight<T> w;
      w.load(in + v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = w.pair(e);
        z[2 * e] = x.x, z[2 * e + 1] = x.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = v + e >= 0 && v + e < vocab ? static_cast<float>(in[v + e]) : -INFINITY;
    }
  }
  // f(token, logit) for all, the next group under way while one is worked on
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    int g = from + static_cast<int>(threadIdx.x & 31);
    Eight<T> next;
    if (g < to && whole(g * 8 - shift)) next.load(in + g * 8 - shift);
#pragma unroll 1
    for (; g < to; g += 32) {
      const Eight<T> now = next;
      const int v = g * 8 - shift, w = v + 256;
      if (g + 32 < to && whole(w)) next.load(in + w);
      float z[8];
      if (whole(v)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = now.pair(e);
          z[2 * e] = x.x, z[2 * e + 1] = x.y;
        }
      } else {
        get(v, z);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) f(v + e, z[e]);
    }
  }
  // The warp of the row's that owns token v
  __device__ __forceinline__ int warp_of(int v) const { return (v + shift) / 8 / per_warp; }
};

struct SampleShared {
  double roots[32];
  uint32_t bins[BINS], own_bins[BINS];     // of the row, of this block (blocks == 1: the row's are counted at once)
  u64 order[LIST], weights[LIST];
  u64 own_order[LIST];                     // of this block's part of the row
  u64 exchange[2][MOST_BLOCKS][3];         // what the blocks tell each other, in turn
  u64 joined[3][SAMPLE_WARPS];
  u64 edges[2];
  int found, before, entries, total;
};

__device__ __forceinline__ u64 over_warp_max(u64 x) {
#pragma unroll
  for (int w = 16; w; w >>= 1) x = max(x, __shfl_xor_sync(0xffffffffu, x, w));
  return x;
}
__device__ __forceinline__ u64 over_warp_sum(u64 x) {
#pragma unroll
  for (int w = 16; w; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
  return x;
}

// The threads of a row: a block, or the blocks of a cluster.
template <bool CLUSTER>
struct Team {
  SampleShared& s;
  int rank, blocks;
  int turn = 0;
  __device__ __forceinline__ Team(SampleShared& shared, int n) : s(shared), rank(CLUSTER ? static_cast<int>(blockIdx.x) % n : 0), blocks(CLUSTER ? n : 1) {}
  __device__ __forceinline__ void sync() const {
    if constexpr (CLUSTER) cooperative_groups::this_cluster().sync(); else __syncthreads();
  }
  template <typename P>
  __device__ __forceinline__ P* of(P* mine, int other) const { return cooperative_groups::this_cluster().map_shared_rank(mine, other); }

  // Numbers that each block has, by rank: s.exchange[turn][rank][...]. All threads; `x` counts where threadIdx.x < N of every block
  template <int N>
  __device__ __forceinline__ const u64 (*told(u64 x))[3] {
    turn ^= 1;
    if constexpr (CLUSTER) {
      if (threadIdx.x < N)
        for (int r = 0; r < blocks; ++r) *of(&s.exchange[turn][rank][threadIdx.x], r) = x;
    } else {
      if (threadIdx.x < N) s.exchange[turn][0][threadIdx.x] = x;
    }
    sync();
    return s.exchange[turn];
  }
  __device__ __forceinline__ u64 max_of(u64 x) {
    x = over_warp_max(x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.joined[0][threadIdx.x >> 5] = x;
    __syncthreads();
    const auto all = told<1>(over_warp_max(s.joined[0][threadIdx.x & (SAMPLE_WARPS - 1)]));
    x = all[0][0];
    for (int r = 1; r < blocks; ++r) x = max(x, all[r][0]);
    return x;
  }
  __device__ __forceinline__ void sums_of(u64& x, u64& y, u64& z) {
    x = over_warp_sum(x), y = over_warp_sum(y), z = over_warp_sum(z);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.joined[0][threadIdx.x >> 5] = x, s.joined[1][threadIdx.x >> 5] = y, s.joined[2][threadIdx.x >> 5] = z;
    __syncthreads();
    u64 part = 0;
    if (threadIdx.x < 3)
      for (int w = 0; w < SAMPLE_WARPS; ++w) part += s.joined[threadIdx.x][w];
    const auto all = told<3>(part);
    x = y = z = 0;
    for (int r = 0; r < blocks; ++r) x += all[r][0], y += all[r][1], z += all[r][2];
  }
  __device__ __forceinline__ void clear() const {
    for (int i = threadIdx.x; i < BINS / 4; i += SAMPLE_THREADS) {
      reinterpret_cast<uint4*>(s.bins)[i] = make_uint4(0, 0, 0, 0);
      if (CLUSTER) reinterpret_cast<uint4*>(s.own_bins)[i] = make_uint4(0, 0, 0, 0);
    }
  }
  // s.bins counts the tokens of the row for which `f` (token, logit) names a bin below BINS
  template <typename T, typename F>
  __device__ __forceinline__ void count(const LogitRow<T>& row, F&& f, bool again = true) {
    uint32_t* bins = CLUSTER ? s.own_bins : s.bins;
    if (again) {
      sync();                              // (others have read the ones before)
      clear();
      __syncthreads();
    }
    row.each([&](int v, float z) {
      const int i = f(v, z);
      if (i < BINS) atomicAdd(&bins[i], 1u);
    });
    sync();
    if constexpr (CLUSTER) {
      for (int i = threadIdx.x; i < BINS / 4; i += SAMPLE_THREADS) {
        uint4 sum = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < MOST_BLOCKS; ++r)
          if (r < blocks) {
            const uint4 x = of(reinterpret_cast<uint4*>(s.own_bins), r)[i];
            sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
          }
        reinterpret_cast<uint4*>(s.bins)[i] = sum;
      }
      __syncthreads();
    }
  }
  // s.order and s.weights (1 for `counted`) list the tokens of the row that `f` wants; their number. Where that is more than LIST, some LIST of them.
  template <typename T, typename F>
  __device__ __forceinline__ int list(const LogitRow<T>& row, const Weigher& weigh, bool counted, F&& f) {
    u64* own = CLUSTER ? s.own_order : s.order;
    sync();
    if (threadIdx.x == 0) s.entries = 0;
    __syncthreads();
    row.each([&](int v, float z) {
      if (!f(v, z)) return;
      const int i = atomicAdd(&s.entries, 1);
      if (i < LIST) own[i] = order_of(z, v);
    });
    __syncthreads();
    int n = s.entries;
    if constexpr (CLUSTER) {
      const auto all = told<1>(static_cast<u64>(n));
      n = 0;
      for (int r = 0; r < blocks; ++r) {
        const int m = static_cast<int>(all[r][0]);
        const u64* from = of(s.own_order, r);
        for (int i = threadIdx.x; i < m && n + i < LIST; i += SAMPLE_THREADS) s.order[n + i] = from[i];
        n += m;
      }
      __syncthreads();
    }
    if (static_cast<int>(threadIdx.x) < n) s.weights[threadIdx.x] = counted ? 1 : weigh.fixed(number_of(static_cast<uint32_t>(s.order[threadIdx.x] >> 32)));
    __syncthreads();
    return n;
  }
};
// Over the threads of a block
__device__ __forceinline__ u64 block_max(SampleShared& s, u64 x) {
  x = over_warp_max(x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.joined[0][threadIdx.x >> 5] = x;
  __syncthreads();
  return over_warp_max(s.joined[0][threadIdx.x & (SAMPLE_WARPS - 1)]);
}
__device__ __forceinline__ u64 block_sum(SampleShared& s, u64 x) {
  x = over_warp_sum(x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.joined[0][threadIdx.x >> 5] = x;
  __syncthreads();
  x = threadIdx.x % 32 < SAMPLE_WARPS ? s.joined[0][threadIdx.x % 32] : 0;
  return over_warp_sum(x);
}

// The last bin that holds a token and in front of which the sum of f(bin) (counts or weights) is below `want`, or below that share of all of it: s.found
// (-1: none), s.before the tokens in front of it; s.total: tokens of all bins. All threads.
template <typename N, bool SHARE, typename F>
__device__ __forceinline__ void find_bin(SampleShared& s, N want, F&& f) {
  constexpr int PER = BINS / SAMPLE_THREADS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  N part[PER], sum = 0;
  int n[PER], count = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    n[i] = static_cast<int>(s.bins[threadIdx.x * PER + i]), part[i] = f(static_cast<int>(threadIdx.x) * PER + i);
    sum += part[i], count += n[i];
  }
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const N x = __shfl_up_sync(0xffffffffu, sum, w);
    const int y = __shfl_up_sync(0xffffffffu, count, w);
    if (lane >= w) sum += x, count += y;
  }
  N x = __shfl_up_sync(0xffffffffu, sum, 1);
  int y = __shfl_up_sync(0xffffffffu, count, 1);
  if (lane == 0) x = 0, y = 0;
  N* sums = reinterpret_cast<N*>(s.joined[0]);
  int* counts = reinterpret_cast<int*>(s.joined[1]);
  __syncthreads();
  if (lane == 31) sums[warp] = sum, counts[warp] = count;
  if (threadIdx.x == 0) s.found = -1;
  __syncthreads();
  N all = 0;
  int all_count = 0;
  for (int w = 0; w < SAMPLE_WARPS; ++w) {
    if (w == warp) x += all, y += all_count;                 // in front of this thread's bins
    all += sums[w], all_count += counts[w];
  }
  if (SHARE) want *= all;
  int found = -1, before = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (n[i] > 0 && x < want) found = threadIdx.x * PER + i, before = y;
    x += part[i], y += n[i];
  }
  if (found >= 0) atomicMax(&s.found, found);
  if (threadIdx.x == 0) s.total = all_count;
  __syncthreads();
  if (found >= 0 && found == s.found) s.before = before;
  __syncthreads();
}
// Tokens in bins [0, b). All threads.
__device__ __forceinline__ int tokens_before(SampleShared& s, int b) {
  u64 x = 0;
  for (int i = threadIdx.x; i < b && i < BINS; i += SAMPLE_THREADS) x += s.bins[i];
  return static_cast<int>(block_sum(s, x));
}

// A stretch of the order that holds a border: tokens with low <= order <= high, n of them at most, `sum` of weights (or tokens) in front.
struct Stretch {
  u64 low, high, sum;
  int n;
};

// The place in the order of the last token in front of which less than `want` lies; the stretch holds it. COUNT: tokens are counted, not weighed.
// `entries`: the tokens of the stretch, which are in the list then; -1 where it was cut finer first.
template <typename T, bool CLUSTER, bool COUNT>
__device__ __noinline__ u64 last_kept(Team<CLUSTER>& team, const LogitRow<T>& row, const Weigher& weigh, Stretch at, double want, int& entries) {
  SampleShared& s = team.s;
  const bool whole = at.n <= LIST;
  for (int level = 0; at.n > LIST && level < 64; ++level) {   // (a few levels: each is one of some 2000 bins, or what is left beside it)
    // finer bins of the order
    const u64 range = at.high - at.low;
    const int shift = max(0, 64 - __clzll(static_cast<long long>(range)) - 11);
    team.count(row, [&](int v, float z) {
      const u64 q = order_of(z, v);
      return q >= at.low && q <= at.high ? static_cast<int>((at.high - q) >> shift) : BINS;
    });
    const auto cut = [&](int first, int last) {              // the stretch of bins [first, last]
      Stretch x = at;
      x.high = at.high - (static_cast<u64>(first) << shift);
      x.low = static_cast<u64>(last) >= range >> shift ? at.low : at.high - ((static_cast<u64>(last) + 1) << shift) + 1;
      return x;
    };
    if (COUNT) {
      find_bin<int, false>(s, static_cast<int>(want) - static_cast<int>(at.sum), [&](int i) { return static_cast<int>(s.bins[i]); });
      const int c = s.found;
      Stretch x = cut(c, c);
      x.sum = at.sum + s.before, x.n = static_cast<int>(s.bins[c]);
      at = x;
      continue;
    }
    const float missing = static_cast<float>((want - static_cast<double>(at.sum)) / UNIT_WEIGHT);
    find_bin<float, false>(s, missing, [&](int i) {
      const u64 n = s.bins[i], middle = at.high - (static_cast<u64>(i) << shift) - (shift ? 1ull << (shift - 1) : 0);
      return n ? static_cast<float>(n) * weigh.about(number_of(static_cast<uint32_t>(middle >> 32))) : 0.f;
    });
    const int named = max(s.found, 0);                        // (the estimate is seldom off by a bin: what it names is checked)
    Stretch x = cut(named, named);
    u64 above = 0, within = 0, none = 0;
    row.each([&](int v, float z) {
      const u64 q = order_of(z, v);
      if (q > at.high || q < x.low) return;
      const u64 w = weigh.fixed(z);
      if (q > x.high) above += w; else within += w;
    });
    team.sums_of(above, within, none);
    above += at.sum;
    if (static_cast<double>(above) >= want) {                // it lies in front
      x = cut(0, named - 1);
      x.sum = at.sum, x.n = tokens_before(s, named);
    } else if (static_cast<double>(above + within) < want) {
      x = cut(named + 1, BINS - 1);
      x.sum = above + within, x.n = at.n - tokens_before(s, named + 1);
    } else {
      x.sum = above, x.n = static_cast<int>(s.bins[named]);
    }
    at = x;
  }
  // (as numbers first: above the largest there is no number, nothing is at least that)
  const float z_low = number_of(static_cast<uint32_t>(at.low >> 32)), z_above = number_of(static_cast<uint32_t>(at.high >> 32) + 1);
  const int listed = team.list(row, weigh, COUNT, [&](int v, float z) {
    if (!(z >= z_low) || z >= z_above) return false;
    const u64 q = order_of(z, v);
    return q >= at.low && q <= at.high;
  });
  const int n = min(listed, LIST);         // (more only where the levels ran out)
  entries = whole && listed <= LIST ? n : -1;
  u64 kept = ~0ull;
  if (static_cast<int>(threadIdx.x) < n) {
    const u64 q = s.order[threadIdx.x];
    u64 sum = at.sum;
    for (int j = 0; j < n; ++j) sum += s.order[j] > q ? s.weights[j] : 0;
    if (static_cast<double>(sum) < want) kept = q;
  }
  return ~block_max(s, ~kept);
}

// The multiple of a weight's unit that the sum up to the drawn token exceeds: whole numbers exceed u * all where they exceed the whole part of that.
__device__ __forceinline__ u64 target_of(float u, u64 all) {
  const double to = u > 0.f ? static_cast<double>(u) * static_cast<double>(all) : 0.0;
  return to < static_cast<double>(all) ? min(static_cast<u64>(to), all - 1) : all - 1;
}

// FILTERED: with top-k or top-p.
template <typename T, bool CLUSTER, bool FILTERED>
__global__ void __launch_bounds__(SAMPLE_THREADS, FILTERED ? 2 : 3) sample_kernel(const SampleArgs a) {
  __shared__ __align__(16) SampleShared s;
  if (threadIdx.x < 32) s.roots[threadIdx.x] = exp2(-static_cast<double>(threadIdx.x) / 32.0);
  Team<CLUSTER> team(s, a.blocks);
  if (FILTERED) team.clear();
  if constexpr (CLUSTER) team.sync();      // every block of the cluster runs before another writes to it
  follow_grid();
  const int b = CLUSTER ? blockIdx.x / a.blocks : blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const LogitRow<T> row(static_cast<const T*>(a.in) + (long long)b * a.vocab, a.vocab, team.rank, team.blocks);
  const float temperature = a.temperature == nullptr ? 1.f : a.temperature[b], p = a.top_p == nullptr ? 1.f : a.top_p[b],
              least = a.min_p == nullptr ? 0.f : a.min_p[b], u = a.uniform[b];
  const long long asked = a.top_k.p == nullptr ? 0 : a.top_k.at(b);
  float largest = -INFINITY;
  row.each([&](int v, float z) { largest = fmaxf(largest, z); });      // (passes over NaN)
  const float top = number_of(static_cast<uint32_t>(team.max_of(key_of(largest))));
  if (!(top > -INFINITY) || !(temperature > 0.f) || asked == 1) {
    u64 first = 0;                         // the first in order
    if (top > -INFINITY) {
      row.each([&](int v, float z) { if (z == top) first = max(first, order_of(z, v)); });
      first = team.max_of(first);
    }
    if (threadIdx.x == 0 && team.rank == 0) a.out[b] = first == 0 ? -1ll : token_of(first);
    return;
  }
  const bool by_count = FILTERED && asked > 0 && asked < a.vocab, by_share = FILTERED && p < 1.f;
  const Weigher weigh(top, temperature, s.roots);
  // the least key in (lo, hi] for which `good` holds, which holds from some key on and at hi. A warp tries 32 keys at once
  const auto least_key = [&](uint32_t lo, uint32_t hi, auto&& good) {
    while (hi - lo > 1) {
      const uint32_t step = (hi - lo + 31) / 32, mid = lo + min(hi - lo, step * (lane + 1));
      const int k = __ffs(static_cast<int>(__ballot_sync(0xffffffffu, mid >= hi || good(number_of(mid))))) - 1;      // (the last lane is at hi)
      hi = lo + min(hi - lo, step * (k + 1));
      lo += step * k;
    }
    return static_cast<u64>(hi) << 32;
  };
  // min-p: a whole number of w counts as w >= m where it is at least that of m, rounded up (m is no whole number but by chance). Its border in the order:
  const u64 least_kept = least > 0.f ? static_cast<u64>(ceil(fmin(static_cast<double>(least), 1.0) * UNIT_WEIGHT)) : 0;
  const auto least_border = [&] {
    if (least_kept == 0) return 0ull;
    __syncthreads();
    if (warp == 0) {
      const u64 at = least_key(key_of(-INFINITY), key_of(top), [&](float z) { return weigh.fixed(z) >= least_kept; });
      if (lane == 0) s.edges[0] = at;
    }
    __syncthreads();
    return s.edges[0];
  };
  u64 last = 0;                            // of the order, the last that is kept
  // top-p: what this warp has above the bin that holds the border, where that begins, how many tokens of it are in the list (-1: not known); what it has up to the
  // border of min-p
  u64 above_mine = 0, least_mine = 0, bin_high = 0;
  int listed = -1;
  u64 least_order = 0;
  if (FILTERED && (by_count || by_share)) {
    const auto in_bins = [&](int v, float z) { return weigh.bin(z); };
    // ---- all that may be kept is in the list, one entry for each thread: the first `asked` of these, all where that is 0
    const auto finish = [&](int n, long long asked) {
      if constexpr (CLUSTER) {
        team.sync();                       // (its lists have been read)
        if (team.rank != 0) return;
      }
      const bool mine = static_cast<int>(threadIdx.x) < n;
      const u64 q = mine ? s.order[threadIdx.x] : 0, w = mine ? s.weights[threadIdx.x] : 0;
      u64 sum = 0;
      int place = 0;
      if (mine)
        for (int j = 0; j < n; ++j)
          if (s.order[j] > q) ++place, sum += s.weights[j];
      bool kept = mine && (asked == 0 || place < asked);
      if (by_share) {
        const double want = static_cast<double>(p) * static_cast<double>(block_sum(s, kept ? w : 0));
        kept = kept && (place == 0 || static_cast<double>(sum) < want);
      }
      kept = kept && w >= least_kept;
      const u64 all = block_sum(s, kept ? w : 0);            // (all threads are behind their reads of the weights)
      if (mine) s.weights[threadIdx.x] = kept ? w : 0;
      __syncthreads();
      if (!kept || w == 0) return;
      u64 front = 0;                       // of smaller ids
      for (int j = 0; j < n; ++j) front += static_cast<uint32_t>(s.order[j]) > static_cast<uint32_t>(q) ? s.weights[j] : 0;
      const u64 target = target_of(u, all);
      if (target >= front && target < front + w) a.out[b] = token_of(q);
    };
    const auto bin_count = [&](int i) { return static_cast<int>(s.bins[i]); };
    team.count(row, in_bins, false);
    // how far the first k, or all of weight, reach
    find_bin<int, false>(s, by_count ? static_cast<int>(asked) : 0x7fffffff, bin_count);
    const int c = s.found, before = s.before, total = s.total;
    const bool cut = by_count && total > asked;
    if (before + static_cast<int>(s.bins[c]) <= LIST)
      return finish(team.list(row, weigh, false, [&](int v, float z) { return weigh.bin(z) <= c; }), cut ? asked : 0);
    const auto stretch = [&](int first_bin, int last_bin) {  // of bins [first_bin, last_bin]: bins fall as keys grow
      __syncthreads();
      if (warp < 2) {
        const int b = warp ? last_bin + 1 : first_bin;
        const u64 at = least_key(key_of(-INFINITY), key_of(top) + 1, [&](float z) { return weigh.bin(z) < b; });
        if (lane == 0) s.edges[warp] = at;
      }
      __syncthreads();
      return Stretch{s.edges[1], s.edges[0] - 1, 0, 0};
    };
    const auto about = [&](int i) { return exp2f(static_cast<float>(i) * (-FAR / (BINS - 1))); };
    int end = BINS, end_tokens = 0;        // the bin that top-k ends in, and how many of it are kept
    if (cut) {
      end = c, end_tokens = static_cast<int>(asked) - before;
      Stretch x = stretch(c, c);
      x.sum = before, x.n = static_cast<int>(s.bins[c]);
      int entries;
      last = last_kept<T, CLUSTER, true>(team, row, weigh, x, static_cast<double>(asked), entries);
      if (by_share && x.n > LIST) team.count(row, in_bins);  // finer bins took the histogram's place
    }
    if (by_share) {
      find_bin<float, true>(s, p, [&](int i) { return i > end ? 0.f : static_cast<float>(i == end ? end_tokens : static_cast<int>(s.bins[i])) * about(i); });
      const int named = max(s.found, 0);                       // (the estimate is seldom off by a bin: what it names is checked)
      Stretch x = stretch(named, named);
      least_order = least_border();
      // the border of top-k as a number and an id, and the stretch as numbers (above the largest: no number, nothing is at least that)
      const float z_last = last ? number_of(static_cast<uint32_t>(last >> 32)) : -INFINITY, z_low = number_of(static_cast<uint32_t>(x.low >> 32)),
                  z_above = number_of(static_cast<uint32_t>(x.high >> 32) + 1), z_least = least_order ? number_of(static_cast<uint32_t>(least_order >> 32)) : INFINITY;
      bin_high = x.high;
      const int v_last = last ? token_of(last) : -1;
      u64 all = 0, above = 0, within = 0;
      row.each([&](int v, float z) {
        if (!(z > z_last || (z == z_last && v <= v_last))) return;
        const u64 w = weigh.fixed(z);
        all += w;
        if (z >= z_least) least_mine += w;
        if (z >= z_above) above += w;
        else if (z >= z_low) within += w;
      });
      above_mine = over_warp_sum(above), least_mine = over_warp_sum(least_mine);
      team.sums_of(all, above, within);
      const double want = fmax(static_cast<double>(p) * static_cast<double>(all), 0.5);     // (the first is kept)
      bool here = false;
      if (static_cast<double>(above) >= want) {
        x = stretch(0, named - 1);
        x.sum = 0, x.n = tokens_before(s, named);
      } else if (static_cast<double>(above + within) < want) {
        x = stretch(named + 1, BINS - 1);
        x.sum = above + within, x.n = total - tokens_before(s, named + 1);
      } else {
        x.sum = above, x.n = static_cast<int>(s.bins[named]);
        here = true;
      }
      x.low = max(x.low, last);
      last = last_kept<T, CLUSTER, false>(team, row, weigh, x, want, listed);
      if (!here) listed = -1, bin_high = 0;
    }
  }
  // ---- the draw
  if (!by_share) least_order = least_border();
  const u64 border = last;
  last = max(last, least_order);
  const float z_last = last ? number_of(static_cast<uint32_t>(last >> 32)) : -INFINITY;
  const int v_last = last ? (last > border ? 0x7fffffff : token_of(last)) : -1;      // (min-p keeps all with the logit of its border)
  const auto drawn = [&](int v, float z) { return z > z_last || (z == z_last && v <= v_last) ? weigh.fixed(z) : 0ull; };
  u64 sum = 0;
  if (FILTERED && bin_high && last > bin_high) {             // the sums are known: up to the border of min-p,
    sum = least_mine;
  } else if (FILTERED && listed >= 0) {    // or those above the bin of the border and what the list has of that
    const int me = team.rank * SAMPLE_WARPS + warp;
    for (int i = lane; i < listed; i += 32) {
      const u64 q = s.order[i];
      if (q >= last && row.warp_of(token_of(q)) == me) sum += s.weights[i];
    }
    sum = over_warp_sum(sum) + above_mine;
  } else {
    row.each([&](int v, float z) { sum += drawn(v, z); });
    sum = over_warp_sum(sum);
  }
  __syncthreads();
  if (lane == 0) s.joined[0][warp] = sum;
  __syncthreads();
  u64 all = 0, before = 0;
  for (int w = 0; w < SAMPLE_WARPS; ++w) {
    if (w == warp) before = all;
    all += s.joined[0][w];
  }
  if constexpr (CLUSTER) {
    const auto parts = team.template told<1>(all);
    all = 0;
    for (int r = 0; r < team.blocks; ++r) {
      if (r == team.rank) before += all;
      all += parts[r][0];
    }
    team.sync();                           // no block leaves while another still reads its bins or its list
  }
  const u64 target = target_of(u, all);
  if (target < before || target >= before + sum) return;
#pragma unroll 1
  for (int g = row.from; g < row.to; g += 32) {              // the warp that holds it
    float z[8];
    u64 w[8], mine = 0;
    const int v = (g + lane) * 8 - row.shift;
    if (g + lane < row.to) row.get(v, z);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = g + lane < row.to ? drawn(v + e, z[e]) : 0, mine += w[e];
    u64 upto = mine;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const u64 x = __shfl_up_sync(0xffffffffu, upto, k);
      if (lane >= k) upto += x;
    }
    const u64 here = __shfl_sync(0xffffffffu, upto, 31);
    if (target >= before + here) {
      before += here;
      continue;
    }
    u64 x = before + upto - mine;
    if (target >= x && target < x + mine) {
      int e = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (target >= x + w[i]) ++e, x += w[i]; else break;
      }
      a.out[b] = v + e;
    }
    return;
  }
}

template <typename T>
static cudaError_t launch_sample(SampleArgs a, int batch, cudaStream_t stream) {
  // Blocks of a row: as many as the chip has room for twice over, of 8192 tokens each (a cluster's exchanges cost 3 us). us with 1, 2, 4, 8 blocks: one row of
  // 32000 19.0, 16.9, 14.2, 14.9, of 8192 9.5, 11.7, 12.4, 14.0; 64 rows of 32001 82, 66, 55, 57; 128 rows 51, 44, 54, 96; 256 rows 62, 64, 85, 168; 32 rows of
  // 131072 158, 97, 70, 59.
  a.blocks = 1;
  while (a.blocks < MOST_BLOCKS && (long long)batch * a.blocks * 2 <= 296 && a.vocab > 8192 * a.blocks) a.blocks *= 2;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(static_cast<unsigned>(batch) * a.blocks);
  cfg.blockDim = dim3(SAMPLE_THREADS);
  cfg.stream = stream;
  cfg.attrs = attr;
  if (a.blocks > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(a.blocks);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  nb::set_following(cfg);
  if (a.top_k.p == nullptr && a.top_p == nullptr) return cudaLaunchKernelEx(&cfg, a.blocks > 1 ? sample_kernel<T, true, false> : sample_kernel<T, false, false>, a);
  return cudaLaunchKernelEx(&cfg, a.blocks > 1 ? sample_kernel<T, true, true> : sample_kernel<T, false, true>, a);
}

}  // namespace nbc

// wide: top_k holds 64-bit numbers. -1: more tokens than sums of weights have room for.
extern "C" int nb_sample_tokens(const void* in, const float* uniform, const float* temperature, const void* top_k, const float* top_p, const float* min_p,
                                void* out, int wide, int batch, int vocab, int fp32, void* stream) {
  using namespace nbc;
  if (vocab < 1 || vocab > 1 << 20 || batch < 1) return -1;
  SampleArgs a = {};
  a.in = in, a.uniform = uniform, a.temperature = temperature, a.top_p = top_p, a.min_p = min_p;
  a.top_k = Whole{top_k, wide}, a.out = static_cast<long long*>(out);
  a.vocab = vocab;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return fp32 ? launch_sample<float>(a, batch, s) : launch_sample<__nv_bfloat16>(a, batch, s);
}

NB_DEBUG_DEFINE(sample)
