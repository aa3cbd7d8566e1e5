// Attention over a key / value cache in 8 bits (layout: kv_cache.cuh).
//
//   o = sum_j softmax_j(scale * s_k(j) * (q . k_j)) * s_v(j) * v_j       codes k, v and scales s_k, s_v of the block that holds key j
//
// Query i of a sequence with `past` tokens in front and `count` new ones sees keys 0 ... past + i (causal) or past + count - 1. Rows from
// `count` on, and rows that see no key, are zero. `group` query heads share a head of the cache.
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
};

// One warp per row: the lanes share its head_dim.
template <typename T, int D>
__global__ void __launch_bounds__(128) attend_rows_kernel(const AttendArgs a) {
  constexpr int E = D / 32;
  follow_grid();
  const long long row = (long long)blockIdx.x * 4 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (row >= (long long)a.batch * a.fresh * a.heads) return;
  const int hq = static_cast<int>(row % a.heads), i = static_cast<int>(row / a.heads % a.fresh), b = static_cast<int>(row / a.heads / a.fresh);
  const int h = hq / (a.heads / a.kv_heads);
  const long long room = (long long)a.table.columns << a.block_log;
  const int past = clamp_tokens(a.past.at(b), room);
  const int count = clamp_tokens(a.count.p == nullptr ? a.fresh : a.count.at(b), a.fresh);
  const long long keys = i >= count ? 0 : min(room, a.causal ? past + (long long)i + 1 : past + (long long)count);
  const T* q = static_cast<const T*>(a.q) + b * a.q_sb + i * a.q_st + hq * a.q_sh + lane * E;
  float x[E], o[E] = {};
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = static_cast<float>(q[e]);
  float m = -INFINITY, l = 0.f;
  for (long long j0 = 0; j0 < keys; j0 += 1 << a.block_log) {
    const int block = a.table.block(b, static_cast<int>(j0 >> a.block_log));
    if (block < 0) continue;
    const long long unit = (long long)block * a.kv_heads + h;
    const float sk = a.scales[0][unit] * a.scale_log2, sv = a.scales[1][unit];
    const int8_t* k = a.codes[0] + (unit << a.block_log) * D + lane * E;
    const int8_t* v = a.codes[1] + (unit << a.block_log) * D + lane * E;
    const int n = static_cast<int>(min(keys - j0, 1ll << a.block_log));
    for (int r = 0; r < n; ++r) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(x[e], static_cast<float>(k[r * D + e]), s);
#pragma unroll
      for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      s *= sk;
      if (!(s <= m)) {           // NaN comes through here too
        const float f = exp2f(m - s);
        l *= f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= f;
        m = s;
      }
      const float p = exp2f(s - m);
      l += p;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(p * sv, static_cast<float>(v[r * D + e]), o[e]);
    }
  }
  T* out = static_cast<T*>(a.out) + row * D + lane * E;
  const float inverse = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = round_to<T>(o[e] * inverse);
}

template <typename T, int D>
static cudaError_t launch_attend(const AttendArgs& a, cudaStream_t stream) {
  const long long grid = ((long long)a.batch * a.fresh * a.heads + 3) / 4;
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  return launch_following(attend_rows_kernel<T, D>, dim3(static_cast<unsigned>(grid)), dim3(128), 0, stream, a);
}

}  // namespace nbc

extern "C" int nb_cached_attention(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, void* out,
                                   const void* table, const void* past, const void* count, int wide, int batch, int fresh, int heads, int kv_heads,
                                   int head_dim, int block, int blocks, int columns, long long q_sb, long long q_st, long long q_sh, float scale,
                                   int causal, int fp32, void* stream) {
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
  if (a.block_log < 0 || (head_dim != 64 && head_dim != 128)) return -1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (fp32) return head_dim == 64 ? launch_attend<float, 64>(a, s) : launch_attend<float, 128>(a, s);
  return head_dim == 64 ? launch_attend<__nv_bfloat16, 64>(a, s) : launch_attend<__nv_bfloat16, 128>(a, s);
}

NB_DEBUG_DEFINE(cached_attention)
