// Writing keys and values into a cache of 8 bits, and reading them back (layout: kv_cache.cuh).
//
// Writing. New rows of a sequence stand behind `past` tokens. Per block and head that gets rows f ... of them:
//     scale' = max(scale if f > 0, max |new| / 127, 2^-100)
//     kept rows (in front of f)   code' = round(code * (scale * (1 / scale')))
//     new rows                    code' = round(x * (1 / scale'))
// so a block's scale only grows until its first row is written anew, and the rows in front are rounded again only when it does. A new
// value that is not finite makes the scale NaN: all that the block holds reads as NaN, as the product with that value would be.
//
// One block of threads takes the rows of one cache block and head: it holds the new values in registers between the maximum and the codes, so they
// are read once. Codes are made and read by adding numbers whose low bits they then are (two or three instructions a code; with conversions and
// 64-bit divisions for the places the kernels were bound by instructions: writing 26.8, reading 36.6 us).
// Reading is bound by memory: 16 sequences of up to 4001, 4 heads, 32.3 us for 180 MB, 5.6 TB/s. Writing by memory and nearly as much by
// instructions (the pipe for whole numbers 68 % busy): 4 x 2048 tokens of 16 heads of 128, bf16, 20 us for 101 MB, 5.0 TB/s. One token
// for each of 64 sequences: 3.7 us, a launch and five accesses one after the other.
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

__device__ __forceinline__ float scale_for(uint32_t top) {      // bits of the largest magnitude; those of infinities and NaN are the largest
  return top < 0x7f800000u ? fmaxf(__uint_as_float(top) * (1.0f / 127.0f), LEAST_SCALE) : __int_as_float(0x7fc00000);
}
// x * y, rounded, and z added to that, rounded again. Not by the two-wide functions: their pair was made one operation with one rounding here, and codes
// halfway between two differed from what the definition's two operations give.
__device__ __forceinline__ float2 multiply_then_add(float2 x, float2 y, float2 z) {
  return make_float2(__fadd_rn(__fmul_rn(x.x, y.x), z.x), __fadd_rn(__fmul_rn(x.y, y.y), z.y));
}
// Codes of four numbers. The product with 1 / scale is at most 127.00002 in magnitude; with 1.5 * 2^23 added its nearest whole number stands in
// the low byte.
__device__ __forceinline__ uint32_t codes4(float2 a, float2 b, float2 inverse) {
  const float2 magic = make_float2(12582912.f, 12582912.f);
  a = multiply_then_add(a, inverse, magic);
  b = multiply_then_add(b, inverse, magic);
  return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040),
                     0x5410);
}
// Code i of a word, exactly: its byte, with 128 added, under the exponent of 2^23.
__device__ __forceinline__ float code_value(uint32_t biased, int i) {
  return __uint_as_float(__byte_perm(biased, 0x4b000000u, 0x7440 | i)) - 8388736.f;
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
  const int room = a.table.columns << a.block_log;
  const int past = clamp_tokens(a.past.at(b), room);
  const int count = clamp_tokens(a.count.p == nullptr ? a.fresh : a.count.at(b), a.fresh);
  const int column = (past >> a.block_log) + j;
  const int first = column << a.block_log;              // position of the block's first row
  const int f = max(past - first, 0), e = min(n, past + count - first);       // rows [f, e) are new
  if (e <= f || column >= a.table.columns) return;
  const int block = a.table.block(b, column);

  const T* in = static_cast<const T*>((which ? a.in[1] : a.in[0])) + b * (which ? a.sb[1] : a.sb[0]) + h * (which ? a.sh[1] : a.sh[0]);
  Eight<T> x[VECS];
  uint32_t top = 0;
#pragma unroll
  for (int u = 0; u < VECS; ++u) {
    const int i = u * THREADS + threadIdx.x, r = i / PER_ROW, c = i % PER_ROW;
    if (r >= f && r < e && NB_IN_BOUNDS(NB_SITE_CACHE_ROW, first + r - past, a.fresh)) x[u].load(in + (first + r - past) * (which ? a.st[1] : a.st[0]) + c * 8); else x[u].clear();
  }
  if (block < 0) return;
  const long long unit = (long long)block * a.heads + h;
  int8_t* codes = (which ? a.codes[1] : a.codes[0]) + unit * n * D;
  float* scale = (which ? a.scales[1] : a.scales[0]) + unit;
  const float before = f > 0 ? scale_at(scale, 0) : 0.f;
#pragma unroll
  for (int u = 0; u < VECS; ++u) top = max(top, x[u].top());
  top = __reduce_max_sync(0xffffffffu, top);
  __shared__ uint32_t tops[THREADS / 32];
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) top = max(top, tops[w]);
  float now = scale_for(top);
  now = before > now || before != before ? before : now;
  const float inverse = 1.0f / now;
  if (threadIdx.x == 0) *scale = now;
  const bool known = now == now;
  const float2 inverse2 = make_float2(inverse, inverse);
#pragma unroll
  for (int u = 0; u < VECS; ++u) {
    const int i = u * THREADS + threadIdx.x, r = i / PER_ROW;
    if (r < f || r >= e || !NB_IN_BOUNDS(NB_SITE_CACHE_CODE, unit * n + r, (long long)a.table.blocks * a.heads * n)) continue;
    uint2 w = make_uint2(codes4(x[u].pair(0), x[u].pair(1), inverse2), codes4(x[u].pair(2), x[u].pair(3), inverse2));
    if (!known) w = make_uint2(0, 0);
    *reinterpret_cast<uint2*>(codes + i * 8) = w;
  }
  if (f == 0 || now == before || !known) return;
  const float ratio = before * inverse;
  const float2 ratio2 = make_float2(ratio, ratio);
  for (int i = threadIdx.x; i < f * PER_ROW; i += THREADS) {
    const uint2 v = *reinterpret_cast<const uint2*>(codes + i * 8);
    const uint32_t p = v.x ^ 0x80808080u, q = v.y ^ 0x80808080u;
    *reinterpret_cast<uint2*>(codes + i * 8) =
        make_uint2(codes4(make_float2(code_value(p, 0), code_value(p, 1)), make_float2(code_value(p, 2), code_value(p, 3)), ratio2),
                   codes4(make_float2(code_value(q, 0), code_value(q, 1)), make_float2(code_value(q, 2), code_value(q, 3)), ratio2));
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
};

// Sixteen codes times a scale: each product is rounded once to fp32, as a code is exact there, and to bf16 where that is asked for.
__device__ __forceinline__ float2 two_values(uint32_t biased, int i, float2 s) {
  return __fmul2_rn(make_float2(code_value(biased, i), code_value(biased, i + 1)), s);
}
template <typename T>
__device__ __forceinline__ void put16(T* p, uint4 v, float s) {
  const uint32_t w[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
  const float2 s2 = make_float2(s, s);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 x = two_values(w[k], 0, s2), y = two_values(w[k], 2, s2);
      reinterpret_cast<float4*>(p)[k] = make_float4(x.x, x.y, y.x, y.y);
    }
  } else {
    uint32_t o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float2 x = two_values(w[k / 2], 2 * (k & 1), s2);
      const __nv_bfloat162 y = __floats2bfloat162_rn(x.x, x.y);
      o[k] = *reinterpret_cast<const uint32_t*>(&y);
    }
    reinterpret_cast<uint4*>(p)[0] = make_uint4(o[0], o[1], o[2], o[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

// One block of threads takes one cache block and head, keys or values.
constexpr int READ_THREADS = 128;
template <typename T, int D>
__global__ void __launch_bounds__(READ_THREADS) kv_read_kernel(const ReadArgs a) {
  constexpr int PER_ROW = D / 16;
  follow_grid();
  int id = blockIdx.x;
  const int which = id & 1;
  id >>= 1;
  const int h = id % a.heads;
  id /= a.heads;
  const int j = id % a.columns, b = id / a.columns;
  const int n = 1 << a.block_log;
  const int room = a.table.columns << a.block_log;
  const int start = clamp_tokens(a.start.at(b), room), count = clamp_tokens(a.count.at(b), a.most);
  const int column = (start >> a.block_log) + j, first = (column << a.block_log) - start;       // the block's first row in the result
  // rows [from, to) of the block lie in the result, those from `end` on are zero
  const int from = max(-first, 0), to = static_cast<int>(min((long long)n, (long long)a.most - first));
  const int block = first + from < count ? a.table.block(b, column) : -1;
  const int end = block < 0 ? 0 : static_cast<int>(min((long long)to, (long long)count - first));
  const long long unit = (long long)max(block, 0) * a.heads + h;
  const int8_t* codes = (which ? a.codes[1] : a.codes[0]) + unit * n * D;
  const float s = block < 0 ? 0.f : scale_at((which ? a.scales[1] : a.scales[0]), unit);
  T* out = static_cast<T*>((which ? a.out[1] : a.out[0])) + (((long long)b * a.most + first) * a.heads + h) * D;
  const long long row = (long long)a.heads * D;
  for (int i0 = from * PER_ROW + threadIdx.x; i0 < to * PER_ROW; i0 += READ_THREADS * 4) {
    // four vectors under way at once
    const int i1 = i0 + READ_THREADS, i2 = i1 + READ_THREADS, i3 = i2 + READ_THREADS;
    const uint4 none = make_uint4(0, 0, 0, 0), v0 = i0 < end * PER_ROW ? ldg16(codes + i0 * 16) : none, v1 = i1 < end * PER_ROW ? ldg16(codes + i1 * 16) : none,
                v2 = i2 < end * PER_ROW ? ldg16(codes + i2 * 16) : none, v3 = i3 < end * PER_ROW ? ldg16(codes + i3 * 16) : none;
    auto put = [&](int i, uint4 v) {
      if (i < to * PER_ROW && NB_IN_BOUNDS(NB_SITE_CACHE_ROW, first + i / PER_ROW, a.most)) put16<T>(out + (i / PER_ROW) * row + (i % PER_ROW) * 16, v, i < end * PER_ROW ? s : 0.f);
    };
    put(i0, v0), put(i1, v1), put(i2, v2), put(i3, v3);
  }
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
  const long long grid = 2ll * a.heads * a.columns * a.batch;
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  return launch_following(kv_read_kernel<T, D>, dim3(static_cast<unsigned>(grid)), dim3(READ_THREADS), 0, stream, a);
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (fp32) return head_dim == 64 ? launch_read<float, 64>(a, s) : launch_read<float, 128>(a, s);
  return head_dim == 64 ? launch_read<__nv_bfloat16, 64>(a, s) : launch_read<__nv_bfloat16, 128>(a, s);
}

NB_DEBUG_DEFINE(kv_cache)
