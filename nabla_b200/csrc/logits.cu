// Adjusting logits before a token is chosen. Per row b and token v, in fp32, rounded to the type of the logits at the end:
//   z' = z / r or z * r       (z > 0 or not) where v stands in the row's history            repetition (z / r as z * (1 / r), two roundings of fp32)
//   z' -= frequency * n + presence * [n > 0]          n: times that v stands in the history behind the prompt
//   z' += bias[v]
//   z' = -inf                 where the grammar's bit of v is 0
//
// Bound by memory: logits are read and written once, 8 at a time and asked for before the history is gone over. A row is cut into slices, one block of
// threads each; the counts of a slice's tokens are in shared memory, and every block of a row goes over its whole history. Counts are sums of
// whole numbers: their order does not matter.
// 256 rows of 32001 with histories of up to 2001, an odd row length, a bias and a grammar: 18.5 us in bf16, 21.6 in fp32; 13.9 and 17.5 without the bias, whose
// rows start off boundaries, 10.9 and 14.7 without the histories, 5.6 in bf16 without any of the three (6.1 TB/s). One row of 32000 with 300 tokens: 2.8.
// What bounds it are loads that wait for loads (4 of 11 cycles between a warp's instructions) and going over the history for each slice: 12 million
// instructions, 2.3 a clock. Blocks of 512 threads, and five or six resident blocks were slower (20 to 24 us in bf16).
#include "kv_cache.cuh"

namespace nbc {
using nb::follow_grid;
using nb::launch_following;

struct LogitsArgs {
  const void* in;                // [batch][vocab]
  void* out;
  Whole history;                 // [batch][longest], p null: none
  Whole length, prompt;          // tokens of a row's history, and how many of them are the prompt's. p null: all, none
  const float *repetition, *presence, *frequency;      // [batch], null: 1, 0, 0
  const float* bias;             // [vocab], or with bias_sb one row each; null: none
  long long bias_sb;
  const uint32_t* allowed;       // [batch][words], bit v % 32 of word v / 32; null: all
  int words;
  int batch, vocab, longest, slice_log;      // 2^slice_log slices
};

constexpr int THREADS = 256;

// PER: groups of 8 tokens of a thread. A slice takes every 2^slice_log-th run of 32 groups: the tokens that stand in a history most often have ids close to
// each other, and so fall to all slices alike.
template <typename T, int PER, bool GRAMMAR>
__global__ void __launch_bounds__(THREADS) adjust_kernel(const LogitsArgs a) {
  constexpr int SLICE = THREADS * PER * 8;
  extern __shared__ __align__(16) uint32_t times[];        // per token of the slice: how often in the prompt, how often behind it
  // 16 bits for each where no history is longer than that; else one bit and 31
  const bool packed = a.longest < 65536;
  const uint32_t one = packed ? 65536u : 2u;
  follow_grid();
  const int b = blockIdx.x >> a.slice_log, s = blockIdx.x & ((1 << a.slice_log) - 1);
  // groups of 8 tokens start where 8 logits of memory do: `shift` tokens of the row's first group belong to the row before. (in and out lie
  // alike, which the entry checks)
  const T* in = static_cast<const T*>(a.in) + (long long)b * a.vocab;
  T* out = static_cast<T*>(a.out) + (long long)b * a.vocab;
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(in) / sizeof(T) & 7);
  auto token = [&](int u) {                // the first of this thread's group u
    const int run = ((u * THREADS + threadIdx.x) >> 5 << a.slice_log) + s;
    return (run * 32 + (threadIdx.x & 31)) * 8 - shift;
  };
  if (s * 256 - shift >= a.vocab) return;
  Eight<T> raw[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int v = token(u);
    raw[u].clear();
    if (v >= 0 && v + 8 <= a.vocab && NB_IN_BOUNDS(NB_SITE_LOGITS_TOKEN, v + 7, a.vocab)) raw[u].load(in + v);
  }
  // the grammar's words are read ahead of the history; biases are not: registers for them cost blocks (21 to 23 us)
  uint32_t bits[GRAMMAR ? PER : 1];
  if (GRAMMAR)
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int v = token(u), w = v < 0 ? 0 : v >> 5;
      const uint32_t* allowed = a.allowed + (long long)b * a.words;
      uint32_t lo = 0u, hi = 0u;
      if (v < a.vocab) lo = allowed[w], hi = allowed[w + 1 < a.words ? w + 1 : w];
      bits[u] = v < 0 ? lo << -v : __funnelshift_r(lo, hi, v & 31);
    }
  const bool counted = a.history.p != nullptr;
  if (counted) {
    constexpr int AHEAD = 8;               // ids under way at once; the first of them before it is known how many count
    int id[AHEAD];
    several(a.history, (long long)b * a.longest, threadIdx.x, THREADS, a.longest, id);
    const int length = a.length.p == nullptr ? a.longest : clamp_tokens(a.length.at(b), a.longest);
    const int prompt = a.prompt.p == nullptr ? 0 : clamp_tokens(a.prompt.at(b), length);
    for (int i = threadIdx.x; i < SLICE / 4; i += THREADS) reinterpret_cast<uint4*>(times)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int i0 = threadIdx.x; i0 < length; i0 += THREADS * AHEAD) {
      if (i0 != threadIdx.x) several(a.history, (long long)b * a.longest, i0, THREADS, length, id);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int i = i0 + k * THREADS;
        if (i >= length || id[k] < 0 || id[k] >= a.vocab) continue;
        const int at = id[k] + shift, run = at >> 8;
        if ((run & ((1 << a.slice_log) - 1)) != s) continue;
        uint32_t* t = &times[(run >> a.slice_log) * 256 + (at & 255)];
        if (!packed && i < prompt) atomicOr(t, 1u); else atomicAdd(t, i < prompt ? 1u : one);
      }
    }
    __syncthreads();
  }
  const float r = a.repetition == nullptr ? 1.f : a.repetition[b], over = 1.f / r, presence = a.presence == nullptr ? 0.f : a.presence[b],
              frequency = a.frequency == nullptr ? 0.f : a.frequency[b];
  const float* bias = a.bias == nullptr ? nullptr : a.bias + b * a.bias_sb;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int at = (u * THREADS + threadIdx.x) * 8, v = token(u);
    if (v >= a.vocab || v + 8 <= 0) continue;
    const bool whole = v >= 0 && v + 8 <= a.vocab;
    float z[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 x = raw[u].pair(e);
      z[2 * e] = x.x, z[2 * e + 1] = x.y;
    }
    if (!whole)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v + e >= 0 && v + e < a.vocab) z[e] = static_cast<float>(in[v + e]);
    if (counted) {
      const uint4 x = *reinterpret_cast<const uint4*>(times + at), y = *reinterpret_cast<const uint4*>(times + at + 4);
      if (x.x | x.y | x.z | x.w | y.x | y.y | y.z | y.w) {
        const uint32_t t[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (t[e]) z[e] *= z[e] > 0.f ? over : r;
          if (t[e] >= one) z[e] -= frequency * static_cast<float>(t[e] >> (packed ? 16 : 1)) + presence;
        }
      }
    }
    if (bias != nullptr) {
      const float* p = bias + v;
      const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 2 & 3);         // the same for all groups of the row
      if (whole && v + 12 <= a.vocab) {      // three vectors that hold the eight numbers
        const float4 *q = reinterpret_cast<const float4*>(p - off), c0 = q[0], c1 = q[1], c2 = off ? q[2] : c1;
        const float c[12] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w, c2.x, c2.y, c2.z, c2.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] += off == 0 ? c[e] : off == 1 ? c[e + 1] : off == 2 ? c[e + 2] : c[e + 3];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (v + e >= 0 && v + e < a.vocab) z[e] += p[e];
      }
    }
    if (GRAMMAR)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!(bits[u] >> e & 1u)) z[e] = -INFINITY;
    T o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = round_to<T>(z[e]);
    if (whole) {
#pragma unroll
      for (int e = 0; e < static_cast<int>(sizeof(o) / 16); ++e) reinterpret_cast<uint4*>(out + v)[e] = reinterpret_cast<const uint4*>(o)[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v + e >= 0 && v + e < a.vocab) out[v + e] = o[e];
    }
  }
}

template <typename T, int PER>
static cudaError_t launch_adjust(LogitsArgs a, cudaStream_t stream) {
  constexpr int SLICE = THREADS * PER * 8;
  const long long tokens = a.vocab + 7ll;      // with the 7 that a row may start in front of a group's end
  while (tokens > (long long)SLICE << a.slice_log) ++a.slice_log;
  const long long grid = (long long)a.batch << a.slice_log;
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  return launch_following(a.allowed == nullptr ? adjust_kernel<T, PER, false> : adjust_kernel<T, PER, true>, dim3(static_cast<unsigned>(grid)), dim3(THREADS), a.history.p == nullptr ? 0 : SLICE * sizeof(uint32_t),
                          stream, a);
}
// Slices of 8192 tokens go over a row's history fewer times; where they are fewer than two for each SM, of 2048. fp32 rows are twice as long: slices of 4096
// have more loads under way (256 x 32001 with a history of 2001: 21.6 us, 22.9 in slices of 8192; bf16 19.7 and 18.5).
template <typename T>
static cudaError_t launch_adjust(const LogitsArgs& a, cudaStream_t stream) {
  return (long long)a.batch * ((a.vocab + 8191) / 8192) >= 296 ? launch_adjust<T, sizeof(T) == 4 ? 2 : 4>(a, stream) : launch_adjust<T, 1>(a, stream);
}

}  // namespace nbc

// wide: bit 0 the history, bit 1 `length`, bit 2 `prompt` are 64-bit numbers. -1: in and out do not start equally far from a boundary of 16 bytes.
extern "C" int nb_adjust_logits(const void* in, void* out, const void* history, const void* length, const void* prompt, const float* repetition,
                                const float* presence, const float* frequency, const float* bias, long long bias_sb, const void* allowed, int wide,
                                int batch, int vocab, int longest, int words, int fp32, void* stream) {
  using namespace nbc;
  if ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) return -1;
  LogitsArgs a = {};
  a.in = in, a.out = out;
  a.history = Whole{history, wide & 1}, a.length = Whole{length, wide >> 1 & 1}, a.prompt = Whole{prompt, wide >> 2 & 1};
  a.repetition = repetition, a.presence = presence, a.frequency = frequency, a.bias = bias, a.bias_sb = bias_sb;
  a.allowed = static_cast<const uint32_t*>(allowed), a.words = words;
  a.batch = batch, a.vocab = vocab, a.longest = longest;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return fp32 ? launch_adjust<float>(a, s) : launch_adjust<__nv_bfloat16>(a, s);
}

NB_DEBUG_DEFINE(logits)
