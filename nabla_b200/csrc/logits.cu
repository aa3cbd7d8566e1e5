// Adjusting logits before a token is chosen. Per row b and token v, in fp32, rounded once:
//   z' = z / r or z * r       (z > 0 or not) where v stands in the row's history            repetition
//   z' -= frequency * n + presence * [n > 0]          n: times that v stands in the history behind the prompt
//   z' += bias[v]
//   z' = -inf                 where the grammar's bit of v is 0
//
// Bound by memory: logits are read and written once. A row is cut into slices, one block of threads each; the counts of a slice's tokens
// are in shared memory, and every block of a row goes over its whole history. Counts are sums of whole numbers: their order does not matter.
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
  int batch, vocab, longest, slice, slices;      // slice: groups of 8 tokens of a block
};

constexpr int THREADS = 256;

template <typename T>
__global__ void __launch_bounds__(THREADS) adjust_kernel(const LogitsArgs a) {
  extern __shared__ uint32_t times[];        // per token of the slice: bit 0 in the prompt, the rest how often behind it
  follow_grid();
  const int b = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
  // groups of 8 tokens start on 16-byte boundaries of memory; `shift` tokens of the row's first group belong to the row before
  const T* in = static_cast<const T*>(a.in) + (long long)b * a.vocab;
  T* out = static_cast<T*>(a.out) + (long long)b * a.vocab;
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(in) / sizeof(T) & 7);
  const int v0 = s * a.slice * 8 - shift, v1 = min(a.vocab, v0 + a.slice * 8);
  if (v1 <= v0) return;
  if (a.history.p != nullptr) {
    for (int i = threadIdx.x; i < a.slice * 8; i += THREADS) times[i] = 0;
    __syncthreads();
    const int length = a.length.p == nullptr ? a.longest : clamp_tokens(a.length.at(b), a.longest);
    const int prompt = a.prompt.p == nullptr ? 0 : clamp_tokens(a.prompt.at(b), length);
    for (int i = threadIdx.x; i < length; i += THREADS) {
      const long long id = a.history.at((long long)b * a.longest + i);
      if (id < max(v0, 0) || id >= v1) continue;
      if (i < prompt) atomicOr(&times[id - v0], 1u); else atomicAdd(&times[id - v0], 2u);
    }
    __syncthreads();
  }
  const float r = a.repetition == nullptr ? 1.f : a.repetition[b], presence = a.presence == nullptr ? 0.f : a.presence[b],
              frequency = a.frequency == nullptr ? 0.f : a.frequency[b];
  const float* bias = a.bias == nullptr ? nullptr : a.bias + b * a.bias_sb;
  const uint32_t* allowed = a.allowed == nullptr ? nullptr : a.allowed + (long long)b * a.words;
  for (int i = threadIdx.x; i < v1 - v0; i += THREADS) {
    const int v = v0 + i;
    if (v < 0) continue;
    float z = static_cast<float>(in[v]);
    const uint32_t t = a.history.p == nullptr ? 0u : times[i];
    if (t) z = z > 0.f ? z / r : z * r;
    if (t > 1) z -= frequency * static_cast<float>(t >> 1) + presence;
    if (bias != nullptr) z += bias[v];
    if (allowed != nullptr && !(allowed[v >> 5] >> (v & 31) & 1u)) z = -INFINITY;
    out[v] = round_to<T>(z);
  }
}

}  // namespace nbc

// wide: bit 0 the history, bit 1 `length`, bit 2 `prompt` are 64-bit numbers.
extern "C" int nb_adjust_logits(const void* in, void* out, const void* history, const void* length, const void* prompt, const float* repetition,
                                const float* presence, const float* frequency, const float* bias, long long bias_sb, const void* allowed, int wide,
                                int batch, int vocab, int longest, int words, int fp32, void* stream) {
  using namespace nbc;
  LogitsArgs a = {};
  a.in = in, a.out = out;
  a.history = Whole{history, wide & 1}, a.length = Whole{length, wide >> 1 & 1}, a.prompt = Whole{prompt, wide >> 2 & 1};
  a.repetition = repetition, a.presence = presence, a.frequency = frequency, a.bias = bias, a.bias_sb = bias_sb;
  a.allowed = static_cast<const uint32_t*>(allowed), a.words = words;
  a.batch = batch, a.vocab = vocab, a.longest = longest;
  a.slice = 512;
  a.slices = (vocab + 7 + 7) / 8 / a.slice + 1;
  const long long grid = (long long)a.slices * batch;
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const size_t smem = history == nullptr ? 0 : static_cast<size_t>(a.slice) * 8 * 4;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (fp32) return launch_following(adjust_kernel<float>, dim3(static_cast<unsigned>(grid)), dim3(THREADS), smem, s, a);
  return launch_following(adjust_kernel<__nv_bfloat16>, dim3(static_cast<unsigned>(grid)), dim3(THREADS), smem, s, a);
}

NB_DEBUG_DEFINE(logits)
