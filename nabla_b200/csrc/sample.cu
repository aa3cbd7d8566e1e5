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
// the border lies, up to a step for p; a pass makes the sums there exact and checks it; what is left, some tens of tokens, is ranked in
// shared memory. Where too many are left (equal logits, flat rows) steps are cut into 2048 finer ones of the order, down to single tokens.
//
// One block of threads for each row; its warps own stretches of ids. The row is read four to six times, all but the first from the caches.
#include "kv_cache.cuh"

namespace nbc {
using nb::follow_grid;
using nb::launch_following;

using u64 = unsigned long long;

struct SampleArgs {
  const void* in;                // [batch][vocab]
  const float *uniform, *temperature, *top_p, *min_p;        // [batch], null: temperature 1, no filter
  Whole top_k;                   // p null: no filter
  long long* out;                // [batch]
  int batch, vocab;
};

constexpr int SAMPLE_THREADS = 512, SAMPLE_WARPS = SAMPLE_THREADS / 32, BINS = 2048, LIST = SAMPLE_THREADS;
constexpr float FAR = 45.f;      // octaves that the histogram covers: weights end at 44
constexpr double UNIT_WEIGHT = 8796093022208.0;              // 2^43

// Where a token stands in the order: larger is earlier. 0: nowhere (-inf, NaN). Keys order as numbers do.
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t u = __float_as_uint(z + 0.f);               // (-0 as 0)
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float number_of(uint32_t key) { return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ u64 order_of(float z, int v) { return z > -INFINITY ? (static_cast<u64>(key_of(z)) << 32) | (0xffffffffu - static_cast<uint32_t>(v)) : 0; }

struct Weigher {
  float top, per_octave;         // the largest logit; octaves of w for a unit of logit
  double rate;                   // 32 octaves
  const double* roots;           // 2^(-i / 32), in shared memory

  // The step of the histogram that a logit falls into, BINS: behind its end. Monotone.
  __device__ __forceinline__ int bin(float z) const {
    const float x = z == top ? 0.f : (top - z) * per_octave;
    return x < FAR ? static_cast<int>(x * ((BINS - 1) / FAR)) : BINS;
  }
  __device__ __forceinline__ float about(float z) const { return z == top ? 1.f : exp2f((z - top) * per_octave); }
  // w, as a number and in multiples of 2^-43
  __device__ __forceinline__ double weight(float z) const {
    if (z == top) return 1.0;
    const double t = (static_cast<double>(top) - static_cast<double>(z)) * rate;             // 32nds of octaves
    if (!(t <= 32.0 * 44.0)) return 0.0;
    const double whole = t + 6755399441055744.0;             // 1.5 * 2^52: the nearest whole number is in the low bits
    const int n = __double2loint(whole);
    const double r = (t - (whole - 6755399441055744.0)) * -0.021660849392498290;            // ln 2 / 32
    double e = fma(r, 1.0 / 120.0, 1.0 / 24.0);              // exp(r) for |r| <= ln 2 / 64: the next term is below 2^-48
    e = fma(r, e, 1.0 / 6.0), e = fma(r, e, 0.5), e = fma(r, e, 1.0), e = fma(r, e, 1.0);
    e *= roots[n & 31];
    return __hiloint2double(__double2hiint(e) - ((n >> 5) << 20), __double2loint(e));
  }
  static __device__ __forceinline__ u64 whole(double w) {
    return static_cast<u64>(__double_as_longlong(fma(w, UNIT_WEIGHT, 4503599627370496.0))) & 0xfffffffffffffull;      // + 2^52
  }
  __device__ __forceinline__ u64 fixed(float z) const { return whole(weight(z)); }
};

// A row, eight tokens at a time from where memory is aligned; each warp has a stretch of ids.
template <typename T>
struct LogitRow {
  const T* in;
  int vocab, shift, from, to;                                // groups of eight of this warp
  __device__ __forceinline__ LogitRow(const T* p, int n) : in(p), vocab(n) {
    shift = static_cast<int>(reinterpret_cast<uintptr_t>(p) / sizeof(T) & 7);
    const int groups = (vocab + shift + 7) / 8, each = ((groups + SAMPLE_WARPS - 1) / SAMPLE_WARPS + 31) / 32 * 32;
    from = min(groups, static_cast<int>(threadIdx.x >> 5) * each), to = min(groups, from + each);
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
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll 2
    for (int g = from + (threadIdx.x & 31); g < to; g += 32) {
      float z[8];
      get(g * 8 - shift, z);
      f(g * 8 - shift, z);
    }
  }
};

struct SampleShared {
  double roots[32];
  uint32_t bins[BINS];
  u64 order[LIST], weights[LIST];
  u64 joined[3][SAMPLE_WARPS];
  u64 edges[2];
  int found, before, entries, total;
  float mass;
};

__device__ __forceinline__ u64 over_warp_max(u64 x) {
#pragma unroll
  for (int w = 16; w; w >>= 1) x = max(x, __shfl_xor_sync(0xffffffffu, x, w));
  return x;
}
template <typename N>
__device__ __forceinline__ N over_warp_sum(N x) {
#pragma unroll
  for (int w = 16; w; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
  return x;
}
// All threads get the result.
__device__ __forceinline__ u64 over_block_max(SampleShared& s, u64 x) {
  x = over_warp_max(x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.joined[0][threadIdx.x >> 5] = x;
  __syncthreads();
  return over_warp_max(s.joined[0][threadIdx.x & (SAMPLE_WARPS - 1)]);
}
__device__ __forceinline__ void over_block_sums(SampleShared& s, u64& x, u64& y, u64& z) {
  x = over_warp_sum(x), y = over_warp_sum(y), z = over_warp_sum(z);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.joined[0][threadIdx.x >> 5] = x, s.joined[1][threadIdx.x >> 5] = y, s.joined[2][threadIdx.x >> 5] = z;
  __syncthreads();
  x = y = z = 0;
#pragma unroll
  for (int w = 0; w < SAMPLE_WARPS; ++w) x += s.joined[0][w], y += s.joined[1][w], z += s.joined[2][w];
}

// The last bin that holds a token and in front of which the sum of f(bin) (counts or weights) is below `want`: s.found (-1: none), s.before the tokens in
// front of it; s.total: tokens of all bins, s.mass: the sum over all bins. All threads.
template <typename N, typename F>
__device__ __forceinline__ void find_bin(SampleShared& s, N want, F&& f) {
  constexpr int PER = BINS / SAMPLE_THREADS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  N sum = 0;
  int count = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) sum += f(static_cast<int>(threadIdx.x) * PER + i), count += static_cast<int>(s.bins[threadIdx.x * PER + i]);
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
  int found = -1, before = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int n = static_cast<int>(s.bins[threadIdx.x * PER + i]);
    if (n > 0 && x < want) found = threadIdx.x * PER + i, before = y;
    x += f(static_cast<int>(threadIdx.x) * PER + i), y += n;
  }
  if (found >= 0) atomicMax(&s.found, found);
  if (threadIdx.x == 0) s.total = all_count, s.mass = static_cast<float>(all);
  __syncthreads();
  if (found >= 0 && found == s.found) s.before = before;
  __syncthreads();
}
// Tokens in bins [0, b). All threads.
__device__ __forceinline__ int tokens_before(SampleShared& s, int b) {
  u64 x = 0, y = 0, z = 0;
  for (int i = threadIdx.x; i < b && i < BINS; i += SAMPLE_THREADS) x += s.bins[i];
  over_block_sums(s, x, y, z);
  return static_cast<int>(x);
}

// A stretch of the order that holds a border: tokens with low <= order <= high, n of them at most, `sum` of weights (or tokens) in front.
struct Stretch {
  u64 low, high, sum;
  int n;
};

// The place in the order of the last token in front of which less than `want` lies; the stretch holds it. COUNT: tokens are counted, not weighed.
template <typename T, bool COUNT>
__device__ __noinline__ u64 last_kept(SampleShared& s, const LogitRow<T>& row, const Weigher& weigh, Stretch at, double want) {
  for (int level = 0; at.n > LIST && level < 64; ++level) {   // (a few levels: each is at most 3 of some 2000 bins, or what is left beside them)
    // finer bins of the order
    const u64 range = at.high - at.low;
    const int shift = max(0, 64 - __clzll(static_cast<long long>(range)) - 11);
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) s.bins[i] = 0;
    __syncthreads();
    row.each([&](int v, const float (&z)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const u64 q = order_of(z[e], v + e);
        if (q >= at.low && q <= at.high) atomicAdd(&s.bins[(at.high - q) >> shift], 1u);
      }
    });
    __syncthreads();
    const auto cut = [&](int first, int last) {              // the stretch of bins [first, last]
      Stretch x = at;
      x.high = at.high - (static_cast<u64>(first) << shift);
      x.low = static_cast<u64>(last) >= range >> shift ? at.low : at.high - ((static_cast<u64>(last) + 1) << shift) + 1;
      return x;
    };
    if (COUNT) {
      find_bin<int>(s, static_cast<int>(want) - static_cast<int>(at.sum), [&](int i) { return static_cast<int>(s.bins[i]); });
      const int c = s.found;
      Stretch x = cut(c, c);
      x.sum = at.sum + s.before, x.n = static_cast<int>(s.bins[c]);
      at = x;
      continue;
    }
    const float missing = static_cast<float>((want - static_cast<double>(at.sum)) / UNIT_WEIGHT);
    find_bin<float>(s, missing, [&](int i) {
      const u64 n = s.bins[i], middle = at.high - (static_cast<u64>(i) << shift) - (shift ? 1ull << (shift - 1) : 0);
      return n ? static_cast<float>(n) * weigh.about(number_of(static_cast<uint32_t>(middle >> 32))) : 0.f;
    });
    const int c = max(s.found, 0), first = max(c - 1, 0), last = min(c + 1, BINS - 1);
    Stretch x = cut(first, last);
    u64 above = 0, within = 0, none = 0;
    row.each([&](int v, const float (&z)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const u64 q = order_of(z[e], v + e);
        if (q > at.high || q < x.low) continue;
        const u64 w = weigh.fixed(z[e]);
        if (q > x.high) above += w; else within += w;
      }
    });
    over_block_sums(s, above, within, none);
    above += at.sum;
    if (static_cast<double>(above) >= want) {                // it lies in front
      x = cut(0, first - 1);
      x.sum = at.sum, x.n = tokens_before(s, first);
    } else if (static_cast<double>(above + within) < want) {
      x = cut(last + 1, BINS - 1);
      x.sum = above + within, x.n = at.n - tokens_before(s, last + 1);
    } else {
      x.sum = above, x.n = tokens_before(s, last + 1) - tokens_before(s, first);
    }
    at = x;
  }
  __syncthreads();
  if (threadIdx.x == 0) s.entries = 0;
  __syncthreads();
  row.each([&](int v, const float (&z)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const u64 q = order_of(z[e], v + e);
      if (q < at.low || q > at.high) continue;
      const int i = atomicAdd(&s.entries, 1);
      if (i < LIST) s.order[i] = q, s.weights[i] = COUNT ? 1 : weigh.fixed(z[e]);
    }
  });
  __syncthreads();
  const int n = min(s.entries, LIST);
  u64 kept = ~0ull;
  if (static_cast<int>(threadIdx.x) < n) {
    const u64 q = s.order[threadIdx.x];
    u64 sum = at.sum;
    for (int j = 0; j < n; ++j) sum += s.order[j] > q ? s.weights[j] : 0;
    if (static_cast<double>(sum) < want) kept = q;
  }
  return ~over_block_max(s, ~kept);
}

template <typename T>
__global__ void __launch_bounds__(SAMPLE_THREADS) sample_kernel(const SampleArgs a) {
  __shared__ SampleShared s;
  if (threadIdx.x < 32) s.roots[threadIdx.x] = exp2(-static_cast<double>(threadIdx.x) / 32.0);
  follow_grid();
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const LogitRow<T> row(static_cast<const T*>(a.in) + (long long)b * a.vocab, a.vocab);
  u64 best = 0;
  row.each([&](int v, const float (&z)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) best = max(best, order_of(z[e], v + e));
  });
  best = over_block_max(s, best);
  const float temperature = a.temperature == nullptr ? 1.f : a.temperature[b];
  const long long asked = a.top_k.p == nullptr ? 0 : a.top_k.at(b);
  if (best == 0 || !(temperature > 0.f) || asked == 1) {
    if (threadIdx.x == 0) a.out[b] = best == 0 ? -1ll : static_cast<long long>(0xffffffffu - static_cast<uint32_t>(best));
    return;
  }
  const float p = a.top_p == nullptr ? 1.f : a.top_p[b], least = a.min_p == nullptr ? 0.f : a.min_p[b], u = a.uniform[b];
  const bool by_count = asked > 0 && asked < a.vocab, by_share = p < 1.f;
  const double rate = 46.166241308446828 / static_cast<double>(temperature);              // 32 log2(e)
  const Weigher weigh = {number_of(static_cast<uint32_t>(best >> 32)), static_cast<float>(rate / 32.0), rate, s.roots};
  u64 last = 0;                            // of the order, the last that is kept
  if (by_count || by_share) {
    const auto count_bins = [&] {
      __syncthreads();
      for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) s.bins[i] = 0;
      __syncthreads();
      row.each([&](int v, const float (&z)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = z[e] > -INFINITY ? weigh.bin(z[e]) : BINS;
          if (i < BINS) atomicAdd(&s.bins[i], 1u);
        }
      });
      __syncthreads();
    };
    count_bins();
    // the order of the first token of a bin is at most this: keys whose bin is below `b` begin there (bins fall as keys grow)
    const auto edge = [&](int b) {
      u64 lo = key_of(-INFINITY), hi = static_cast<u64>(key_of(weigh.top)) + 1;              // the least key in (lo, hi] with a bin below b
      while (hi - lo > 1) {
        const u64 mid = (lo + hi) >> 1;
        if (weigh.bin(number_of(static_cast<uint32_t>(mid))) < b) hi = mid; else lo = mid;
      }
      return hi << 32;
    };
    const auto stretch = [&](int first, int last_bin) {      // of bins [first, last_bin]
      __syncthreads();
      if (warp == 0 && lane < 2) s.edges[lane] = edge(lane ? last_bin + 1 : first);
      __syncthreads();
      return Stretch{s.edges[1], s.edges[0] - 1, 0, 0};
    };
    const auto about = [&](int i) { return exp2f((static_cast<float>(i) + 0.5f) * (-FAR / (BINS - 1))); };
    int end = BINS, end_tokens = 0;        // the bin that top-k ends in, and how many of it are kept
    if (by_count) {
      find_bin<int>(s, static_cast<int>(asked), [&](int i) { return static_cast<int>(s.bins[i]); });
      const int c = s.found, before = s.before;
      if (s.total > asked) {
        end = c, end_tokens = static_cast<int>(asked) - before;
        Stretch x = stretch(c, c);
        x.sum = before, x.n = static_cast<int>(s.bins[c]);
        last = last_kept<T, true>(s, row, weigh, x, static_cast<double>(asked));
        if (by_share && x.n > LIST) count_bins();              // finer bins took the histogram's place
      }
    }
    if (by_share) {
      const auto mass = [&](int i) { return i > end ? 0.f : static_cast<float>(i == end ? end_tokens : static_cast<int>(s.bins[i])) * about(i); };
      find_bin<float>(s, INFINITY, mass);
      find_bin<float>(s, p * s.mass, mass);
      const int c = max(s.found, 0), first = max(c - 1, 0), last_bin = min(c + 1, BINS - 1);
      Stretch x = stretch(first, last_bin);
      u64 all = 0, above = 0, within = 0;
      row.each([&](int v, const float (&z)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const u64 q = order_of(z[e], v + e);
          if (q < last || q == 0) continue;
          const u64 w = weigh.fixed(z[e]);
          all += w;
          if (q > x.high) above += w; else if (q >= x.low) within += w;
        }
      });
      over_block_sums(s, all, above, within);
      const double want = fmax(static_cast<double>(p) * static_cast<double>(all), 0.5);     // (the first is kept)
      if (static_cast<double>(above) >= want) {
        x = stretch(0, first - 1);
        x.sum = 0, x.n = tokens_before(s, first);
      } else if (static_cast<double>(above + within) < want) {
        x = stretch(last_bin + 1, BINS - 1);
        x.sum = above + within, x.n = tokens_before(s, BINS) - tokens_before(s, last_bin + 1);
      } else {
        x.sum = above, x.n = tokens_before(s, last_bin + 1) - tokens_before(s, first);
      }
      x.low = max(x.low, last);
      last = last_kept<T, false>(s, row, weigh, x, want);
    }
  }
  // ---- the draw
  const double floor_of = least > 0.f ? fmin(static_cast<double>(least), 1.0) : 0.0;
  const auto drawn = [&](float z, int v) {
    const u64 q = order_of(z, v);
    if (q < last || q == 0) return 0ull;
    const double w = weigh.weight(z);
    return w >= floor_of ? Weigher::whole(w) : 0ull;
  };
  u64 sum = 0;
  row.each([&](int v, const float (&z)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += drawn(z[e], v + e);
  });
  sum = over_warp_sum(sum);
  __syncthreads();
  if (lane == 0) s.joined[0][warp] = sum;
  __syncthreads();
  u64 all = 0, before = 0;
  for (int w = 0; w < SAMPLE_WARPS; ++w) {
    if (w == warp) before = all;
    all += s.joined[0][w];
  }
  // whole numbers: the sum with a token exceeds u * all where it is more than the whole part of that
  const double to = u > 0.f ? static_cast<double>(u) * static_cast<double>(all) : 0.0;
  const u64 target = to < static_cast<double>(all) ? min(static_cast<u64>(to), all - 1) : all - 1;
  if (target < before || target >= before + sum) return;
  for (int g = row.from; g < row.to; g += 32) {              // the warp that holds it
    float z[8];
    u64 w[8], mine = 0;
    const int v = (g + lane) * 8 - row.shift;
    if (g + lane < row.to) row.get(v, z);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = g + lane < row.to ? drawn(z[e], v + e) : 0, mine += w[e];
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

}  // namespace nbc

// wide: top_k holds 64-bit numbers. -1: more tokens than sums of weights have room for.
extern "C" int nb_sample_tokens(const void* in, const float* uniform, const float* temperature, const void* top_k, const float* top_p, const float* min_p,
                                void* out, int wide, int batch, int vocab, int fp32, void* stream) {
  using namespace nbc;
  if (vocab < 1 || vocab > 1 << 20) return -1;
  SampleArgs a = {};
  a.in = in, a.uniform = uniform, a.temperature = temperature, a.top_p = top_p, a.min_p = min_p;
  a.top_k = Whole{top_k, wide}, a.out = static_cast<long long*>(out);
  a.batch = batch, a.vocab = vocab;
  return launch_following(fp32 ? sample_kernel<float> : sample_kernel<__nv_bfloat16>, dim3(static_cast<unsigned>(batch)), dim3(SAMPLE_THREADS), 0,
                          static_cast<cudaStream_t>(stream), a);
}

NB_DEBUG_DEFINE(sample)
