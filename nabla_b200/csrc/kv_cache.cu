// Writing keys and values into a cache of 8 bits, and reading them back (layout: kv_cache.cuh).
//
// Writing. New rows of a sequence stand behind `past` tokens. Per block and head that gets rows f ... of them:
//     scale' = max(scale if f > 0, max |new| / 127, 2^-100)
//     kept rows (in front of f)   code' = round(code * (scale * (1 / scale')))
//     new rows                    code' = round(x * (1 / scale'))
// so a block's scale only grows until its first row is written anew, and the rows in front are rounded again only when it does. A new
// value that is not finite makes the scale NaN: all that the block holds reads as NaN, as the product with that value would be.
//
// Both kernels are bound by memory. One block of threads takes the rows of one cache block and head: it holds the new values in
// registers between the maximum and the codes, so they are read once.
#include "kv_cache.cuh"

namespace nbc {
using nb::follow_grid;
using nb::launch_following;

struct WriteArgs {
  int8_t* codes[2];              // keys, values
  float* scales[2];
  const void* in[2];             // [batch][new][heads][D]
  long long sb[2], st[2], sh[2];     // their strides in elements
  Table table;
  Whole past, count;             // count.p null: all of them
  int batch, fresh, heads, block_log, columns;     // fresh: new tokens, columns: table columns that a sequence may touch
};

__device__ __forceinline__ float scale_for(float top) {      // top: the largest magnitude, NaN kept
  const float s = top * (1.0f / 127.0f);
  return s < INFINITY ? fmaxf(s, LEAST_SCALE) : __int_as_float(0x7fc00000);
}

template <typename T, int D, int THREADS, int VECS>
__global__ void __launch_bounds__(THREADS) kv_write_kernel(const WriteArgs a) {
  constexpr int PER_ROW = D / 8;
  follow_grid();
  int id = blockIdx.x;
  const int which = id & 1;
  id >>= 1;
  const int h = id % a.heads;
  id /= a.heads;
  const int j = id % a.columns, b = id / a.columns;
  const int n = 1 << a.block_log;
  const long long room = (long long)a.table.columns << a.block_log;
  const int past = clamp_tokens(a.past.at(b), room);
  const int count = clamp_tokens(a.count.p == nullptr ? a.fresh : a.count.at(b), a.fresh);
  const int column = (past >> a.block_log) + j;
  const long long first = (long long)column << a.block_log;       // position of the block's first row
  const int f = static_cast<int>(max(past - first, 0ll));                  // rows [f, e) are new
  const int e = static_cast<int>(min((long long)n, past + (long long)count - first));
  if (e <= f) return;
  const int block = a.table.block(b, column);
  if (block < 0) return;
  const long long unit = (long long)block * a.heads + h;
  int8_t* codes = a.codes[which] + unit * n * D;
  float* scale = a.scales[which] + unit;
  const float before = f > 0 ? *scale : 0.f;

  const T* in = static_cast<const T*>(a.in[which]) + b * a.sb[which] + h * a.sh[which];
  float x[VECS][8];
  float top = 0.f;
  bool odd = false;              // something that is not finite
#pragma unroll
  for (int u = 0; u < VECS; ++u) {
    const int i = u * THREADS + threadIdx.x, r = i / PER_ROW, c = i % PER_ROW;
    if (r >= f && r < e) {
      load8(in + (first + r - past) * a.st[which] + c * 8, x[u]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[u][k] = 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < VECS; ++u)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      top = fmaxf(top, fabsf(x[u][k]));
      odd |= !(fabsf(x[u][k]) < INFINITY);
    }
  top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(odd ? INFINITY : top)));     // magnitudes order as their bits do
  __shared__ float tops[THREADS / 32];
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) top = fmaxf(top, tops[w]);
  float now = scale_for(top);
  now = before > now || before != before ? before : now;
  const float inverse = 1.0f / now;
  if (threadIdx.x == 0) *scale = now;
  const bool known = now == now;
#pragma unroll
  for (int u = 0; u < VECS; ++u) {
    const int i = u * THREADS + threadIdx.x, r = i / PER_ROW, c = i % PER_ROW;
    if (r < f || r >= e) continue;
    uint32_t w[2] = {0u, 0u};
    if (known) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int q = max(-127, min(127, __float2int_rn(x[u][k] * inverse)));
        w[k / 4] |= (static_cast<uint32_t>(q) & 0xffu) << (8 * (k & 3));
      }
    }
    *reinterpret_cast<uint2*>(codes + r * D + c * 8) = make_uint2(w[0], w[1]);
  }
  if (f == 0 || now == before || !known) return;
  const float ratio = before * inverse;
  for (int i = threadIdx.x; i < f * PER_ROW; i += THREADS) {
    uint2 v = *reinterpret_cast<const uint2*>(codes + i * 8);
    uint32_t w[2] = {v.x, v.y}, o[2] = {0u, 0u};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int q = static_cast<int8_t>(w[k / 4] >> (8 * (k & 3)));
      const int t = max(-127, min(127, __float2int_rn(static_cast<float>(q) * ratio)));
      o[k / 4] |= (static_cast<uint32_t>(t) & 0xffu) << (8 * (k & 3));
    }
    *reinterpret_cast<uint2*>(codes + i * 8) = make_uint2(o[0], o[1]);
  }
}

// Reading: rows [start, start + count) of each sequence as numbers, zeros behind them up to `most`.
struct ReadArgs {
  const int8_t* codes[2];
  const float* scales[2];
  void* out[2];                  // [batch][most][heads][D]
  Table table;
  Whole start, count;
  int batch, most, heads, block_log, columns;      // columns: table columns that the rows of a sequence may touch
  long long vectors;             // of 16 codes, of one of keys and values: batch * columns * heads * N * D / 16
};

template <typename T, int D>
__global__ void __launch_bounds__(256) kv_read_kernel(const ReadArgs a) {
  constexpr int PER_ROW = D / 16;
  follow_grid();
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= a.vectors) return;
  const int which = blockIdx.y;
  const int n = 1 << a.block_log;
  const int c = static_cast<int>(at % PER_ROW);
  long long rest = at / PER_ROW;
  const int r = static_cast<int>(rest & (n - 1));
  rest >>= a.block_log;
  const int h = static_cast<int>(rest % a.heads);
  rest /= a.heads;
  const int j = static_cast<int>(rest % a.columns), b = static_cast<int>(rest / a.columns);
  const long long room = (long long)a.table.columns << a.block_log;
  const int start = clamp_tokens(a.start.at(b), room);
  const int count = clamp_tokens(a.count.at(b), a.most);
  const int column = (start >> a.block_log) + j;
  const long long i = ((long long)column << a.block_log) + r - start;        // row of the result
  if (i < 0 || i >= a.most) return;
  T o[16];
  const int block = i < count ? a.table.block(b, column) : -1;
  if (block >= 0) {
    const long long unit = (long long)block * a.heads + h;
    const int4 v = *reinterpret_cast<const int4*>(a.codes[which] + (unit * n + r) * D + c * 16);
    const float s = a.scales[which][unit];
    const int w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = round_to<T>(static_cast<float>(static_cast<int8_t>(w[k / 4] >> (8 * (k & 3)))) * s);
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = round_to<T>(0.f);
  }
  T* out = static_cast<T*>(a.out[which]) + (((long long)b * a.most + i) * a.heads + h) * D + c * 16;
#pragma unroll
  for (int k = 0; k < static_cast<int>(sizeof(o) / 16); ++k) reinterpret_cast<uint4*>(out)[k] = reinterpret_cast<const uint4*>(o)[k];
}

template <typename T, int D>
static cudaError_t launch_write(const WriteArgs& a, cudaStream_t stream) {
  const long long grid = 2ll * a.heads * a.columns * a.batch;
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const dim3 g(static_cast<unsigned>(grid));
  switch ((D / 8) << a.block_log) {      // vectors of a block
    case 128: return launch_following(kv_write_kernel<T, D, 128, 1>, g, dim3(128), 0, stream, a);
    case 256: return launch_following(kv_write_kernel<T, D, 128, 2>, g, dim3(128), 0, stream, a);
    case 512: return launch_following(kv_write_kernel<T, D, 256, 2>, g, dim3(256), 0, stream, a);
    case 1024: return launch_following(kv_write_kernel<T, D, 256, 4>, g, dim3(256), 0, stream, a);
    case 2048: return launch_following(kv_write_kernel<T, D, 256, 8>, g, dim3(256), 0, stream, a);
  }
  return cudaErrorInvalidValue;
}

template <typename T, int D>
static cudaError_t launch_read(const ReadArgs& a, cudaStream_t stream) {
  const long long grid = (a.vectors + 255) / 256;
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  return launch_following(kv_read_kernel<T, D>, dim3(static_cast<unsigned>(grid), 2), dim3(256), 0, stream, a);
}

static int block_log(int n) { return n == 16 ? 4 : n == 32 ? 5 : n == 64 ? 6 : n == 128 ? 7 : -1; }

}  // namespace nbc

// wide: bit 0 the table, bit 1 `past` / `start`, bit 2 `count` are 64-bit numbers. fp32: 0 bf16, 1 fp32. Codes of an error: cudaError_t, or -1 for
// what no kernel takes.
extern "C" int nb_kv_write(void* k_codes, void* k_scales, void* v_codes, void* v_scales, const void* k, const void* v, const void* table,
                           const void* past, const void* count, int wide, int batch, int fresh, int heads, int head_dim, int block, int blocks,
                           int columns, long long k_sb, long long k_st, long long k_sh, long long v_sb, long long v_st, long long v_sh, int fp32,
                           void* stream) {
  using namespace nbc;
  WriteArgs a = {};
  a.codes[0] = static_cast<int8_t*>(k_codes), a.codes[1] = static_cast<int8_t*>(v_codes);
  a.scales[0] = static_cast<float*>(k_scales), a.scales[1] = static_cast<float*>(v_scales);
  a.in[0] = k, a.in[1] = v;
  a.sb[0] = k_sb, a.st[0] = k_st, a.sh[0] = k_sh, a.sb[1] = v_sb, a.st[1] = v_st, a.sh[1] = v_sh;
  a.table = Table{Whole{table, wide & 1}, columns, blocks};
  a.past = Whole{past, wide >> 1 & 1};
  a.count = Whole{count, wide >> 2 & 1};
  a.batch = batch, a.fresh = fresh, a.heads = heads, a.block_log = block_log(block);
  if (a.block_log < 0 || (head_dim != 64 && head_dim != 128)) return -1;
  a.columns = (fresh + block - 2) / block + 1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (fp32) return head_dim == 64 ? launch_write<float, 64>(a, s) : launch_write<float, 128>(a, s);
  return head_dim == 64 ? launch_write<__nv_bfloat16, 64>(a, s) : launch_write<__nv_bfloat16, 128>(a, s);
}

extern "C" int nb_kv_read(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, void* k, void* v, const void* table,
                          const void* start, const void* count, int wide, int batch, int most, int heads, int head_dim, int block, int blocks,
                          int columns, int fp32, void* stream) {
  using namespace nbc;
  ReadArgs a = {};
  a.codes[0] = static_cast<const int8_t*>(k_codes), a.codes[1] = static_cast<const int8_t*>(v_codes);
  a.scales[0] = static_cast<const float*>(k_scales), a.scales[1] = static_cast<const float*>(v_scales);
  a.out[0] = k, a.out[1] = v;
  a.table = Table{Whole{table, wide & 1}, columns, blocks};
  a.start = Whole{start, wide >> 1 & 1};
  a.count = Whole{count, wide >> 2 & 1};
  a.batch = batch, a.most = most, a.heads = heads, a.block_log = block_log(block);
  if (a.block_log < 0 || (head_dim != 64 && head_dim != 128)) return -1;
  a.columns = (most + block - 2) / block + 1;
  a.vectors = (long long)batch * a.columns * heads * block * (head_dim / 16);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (fp32) return head_dim == 64 ? launch_read<float, 64>(a, s) : launch_read<float, 128>(a, s);
  return head_dim == 64 ? launch_read<__nv_bfloat16, 64>(a, s) : launch_read<__nv_bfloat16, 128>(a, s);
}

NB_DEBUG_DEFINE(kv_cache)
