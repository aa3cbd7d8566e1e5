// Norms of the heads of queries and keys and their rotation by the position, in one pass, and the gradient.
//
//   n = x * rsqrt(mean x^2 + eps),  z = n * g,  y = R z        over the D numbers of a head; without a gain: z = x
// R turns the pairs (z_i, z_i + rotary / 2), or neighbours (z_2i, z_2i + 1), of the first `rotary` numbers by position * base^(-2 i / rotary).
// Given dy:  dz = R^T dy,  dg = sum over all heads of dz n,  dx = r (dz g - n mean(dz g n))  with r the reciprocal root of above. Without a gain dx = dz.
//
// A head is held by D / 16 lanes (rounded up to a power of two), 16 numbers each: both halves of eight pairs, so a rotation needs no exchange and the means
// take two to four. The angles of a token are the same for all its heads: a block takes a few tokens and puts their cosines and sines into shared
// memory first. An angle is taken in turns, in 64 bits, and only what is left of a whole turn goes into 32 (a position of 10^6 would be off by
// 0.06 in 32 bits); that remainder is carried in two parts, so cosines and sines are off by about a unit in the last place.
#include "kv_cache.cuh"

namespace nbc {
using nb::follow_grid;
using nb::launch_following;

constexpr int ROTARY_THREADS = 256, MOST_DIM = 256, MOST_TOKENS = 4;

// Some heads of each token, all with the same gain: [batch][tokens][heads][D] by strides (in elements).
struct Heads {
  const void *x, *dy;
  void* out;
  const void* gain;              // null: no norm
  long long x_s[3], dy_s[3], out_s[3];
  int heads;
};
struct RotaryArgs {
  Heads part[3];
  int parts, copied;             // the last `copied` parts are copied as they are (backward: their dy)
  int batch, tokens, dim, rotary, all_heads, per_block;
  Whole positions;
  int positions_shared;          // one row of positions for the whole batch
  double log2_base;
  float eps;
  float* sums;                   // backward: [blocks][2][dim] parts of the gradients of the gains
};

__device__ __forceinline__ void fill_turns(const RotaryArgs& a, double* turns) {
  const double rate = -2.0 * a.log2_base / a.rotary;
  for (int i = threadIdx.x; i < a.rotary / 2; i += ROTARY_THREADS) turns[i] = exp2(rate * i) * 0.15915494309189535;        // 1 / (2 pi)
}
// cosines and sines of the block's tokens, [token][rotary / 2]
__device__ __forceinline__ void fill_angles(const RotaryArgs& a, const double* turns, float2* angles, int first, int n) {
  const int half = a.rotary / 2;
  for (int i = threadIdx.x; i < n * half; i += ROTARY_THREADS) {
    const int at = first + i / half;
    const double turn = static_cast<double>(a.positions.at(a.positions_shared ? at % a.tokens : at)) * turns[i % half];
    const double rest = 2.0 * (turn - rint(turn));                     // of half turns, from -1 to 1
    const float hi = static_cast<float>(rest), lo = static_cast<float>(rest - hi) * 3.14159265f;
    float s, c;
    sincospif(hi, &s, &c);
    angles[i] = make_float2(fmaf(-lo, s, c), fmaf(lo, c, s));
  }
}

template <typename T>
__device__ __forceinline__ void unpack(const Eight<T>& w, float (&x)[16], int at) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 v = w.pair(e);
    x[at + 2 * e] = v.x, x[at + 2 * e + 1] = v.y;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[16], int at) {
  __align__(16) T o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = round_to<T>(x[at + e]);
#pragma unroll
  for (int e = 0; e < static_cast<int>(sizeof(o) / 16); ++e) reinterpret_cast<uint4*>(p)[e] = reinterpret_cast<const uint4*>(o)[e];
}
// Sum over the LANES neighbouring lanes that hold a head.
template <int LANES>
__device__ __forceinline__ float over_head(float x) {
#pragma unroll
  for (int w = 1; w < LANES; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
  return x;
}
// The numbers of pairs (x_e, x_e + 8), or of neighbours, turned by the angles at cs[0 ... 7], or back.
template <bool NEIGHBOURS, bool BACK>
__device__ __forceinline__ void turn(float (&x)[16], const float2* cs) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 t = cs[e];
    const float c = t.x, s = BACK ? -t.y : t.y;
    float &a = x[NEIGHBOURS ? 2 * e : e], &b = x[NEIGHBOURS ? 2 * e + 1 : e + 8];
    const float u = a * c - b * s, w = a * s + b * c;
    a = u, b = w;
  }
}

// Where the 16 numbers of lane c of a head begin: two runs of eight.
template <bool NEIGHBOURS>
__device__ __forceinline__ void runs_of(const RotaryArgs& a, int c, int& first, int& second) {
  if (NEIGHBOURS || 16 * c >= a.rotary) {
    first = 16 * c, second = first + 8;
  } else {
    first = 8 * c, second = a.rotary / 2 + 8 * c;
  }
}

template <typename T, int LANES, bool NEIGHBOURS, bool BACK>
__global__ void __launch_bounds__(ROTARY_THREADS) norm_rotary_kernel(const RotaryArgs a) {
  constexpr int GROUPS = ROTARY_THREADS / LANES;
  __shared__ double turns[MOST_DIM / 2];
  __shared__ __align__(16) float2 angles[MOST_TOKENS * MOST_DIM / 2];
  __shared__ __align__(16) float gains[2][MOST_DIM];
  fill_turns(a, turns);
  follow_grid();
  for (int i = threadIdx.x; i < 2 * a.dim; i += ROTARY_THREADS) {
    const int p = i / a.dim;
    if (p < a.parts - a.copied && a.part[p].gain != nullptr) gains[p][i % a.dim] = static_cast<float>(static_cast<const T*>(a.part[p].gain)[i % a.dim]);
  }
  const int c = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const bool mine = 16 * c < a.dim, turned = 16 * c < a.rotary;
  int first, second;
  runs_of<NEIGHBOURS>(a, c, first, second);
  const float over_dim = 1.f / static_cast<float>(a.dim);
  const int tokens = a.batch * a.tokens;             // (the entry keeps it below 2^31, with the grid's last step)
  float sums[BACK ? 2 : 1][16];            // of the gradients of the gains
  if (BACK)
#pragma unroll
    for (int e = 0; e < 16; ++e) sums[0][e] = sums[BACK][e] = 0.f;

  for (int t0 = blockIdx.x * a.per_block; t0 < tokens; t0 += gridDim.x * a.per_block) {
    const int n = min(tokens - t0, a.per_block);
    __syncthreads();
    fill_angles(a, turns, angles, t0, n);
    __syncthreads();
    for (int row0 = 0; row0 < n * a.all_heads; row0 += GROUPS) {
      const int row = row0 + group, token = row / a.all_heads;
      int h = row - token * a.all_heads, p = 0;
      while (p + 1 < a.parts && h >= a.part[p].heads) h -= a.part[p].heads, ++p;
      const Heads& part = a.part[p];
      const bool there = mine && row < n * a.all_heads && NB_IN_BOUNDS(NB_SITE_ROW_INDEX, t0 + token, tokens);
      const int b_ = (t0 + token) / a.tokens;
      const long long b = b_, t = t0 + token - b_ * a.tokens;
      const T* x = static_cast<const T*>(part.x) + b * part.x_s[0] + t * part.x_s[1] + h * part.x_s[2];
      T* out = static_cast<T*>(part.out) + b * part.out_s[0] + t * part.out_s[1] + h * part.out_s[2];
      const bool copied = p >= a.parts - a.copied, normed = !copied && part.gain != nullptr;
      float v[16], d[16];
      Eight<T> w0, w1, u0, u1;
      w0.clear(), w1.clear(), u0.clear(), u1.clear();
      if (there && (!BACK || normed)) w0.load(x + first), w1.load(x + second);
      if (BACK && there) {
        const T* dy = static_cast<const T*>(part.dy) + b * part.dy_s[0] + t * part.dy_s[1] + h * part.dy_s[2];
        u0.load(dy + first), u1.load(dy + second);
      }
      unpack(w0, v, 0), unpack(w1, v, 8);
      const float2* cs = angles + token * (a.rotary / 2) + 8 * c;
      float squares = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) squares = fmaf(v[e], v[e], squares);
      const float r = rsqrtf(fmaf(over_head<LANES>(squares), over_dim, a.eps));
      if (!BACK) {
        if (normed)
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] *= r * gains[p][(e < 8 ? first : second) + (e & 7)];
        if (there && turned && !copied) turn<NEIGHBOURS, false>(v, cs);
        if (there) store8(out + first, v, 0), store8(out + second, v, 8);
        continue;
      }
      unpack(u0, d, 0), unpack(u1, d, 8);
      if (there && turned && !copied) turn<NEIGHBOURS, true>(d, cs);
      float dot = 0.f;
      if (normed && there) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          v[e] *= r;
          const float s = d[e] * v[e];
          if (p == 0) sums[0][e] += s; else sums[BACK][e] += s;
          d[e] *= gains[p][(e < 8 ? first : second) + (e & 7)];
          dot = fmaf(d[e], v[e], dot);
        }
      }
      const float mean = over_head<LANES>(dot) * over_dim;
      if (normed)
#pragma unroll
        for (int e = 0; e < 16; ++e) d[e] = r * fmaf(-v[e], mean, d[e]);
      if (there) store8(out + first, d, 0), store8(out + second, d, 8);
    }
  }
  if (!BACK || a.sums == nullptr) return;
  // the block's sums: groups of a warp by exchanges, then the warps one after the other in shared memory
  __shared__ float joined[ROTARY_THREADS / 32][2][MOST_DIM];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float s = sums[p ? BACK : 0][e];
#pragma unroll
      for (int w = LANES; w < 32; w <<= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      if (mine && (threadIdx.x & 31) < LANES) joined[threadIdx.x >> 5][p][(e < 8 ? first : second) + (e & 7)] = s;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.dim; i += ROTARY_THREADS) {
    const int p = i / a.dim, at = i - p * a.dim;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < ROTARY_THREADS / 32; ++w) s += joined[w][p][at];
    a.sums[(long long)blockIdx.x * 2 * a.dim + i] = s;
  }
}

// Sums of the blocks' parts, a warp for each number, in an order that depends on their count alone.
template <typename T>
__global__ void __launch_bounds__(256) gain_sums_kernel(const float* parts, int blocks, int dim, T* q_gain, T* k_gain) {
  follow_grid(parts, q_gain, k_gain);
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= 2 * dim) return;
  float s = 0.f;
  for (int b = threadIdx.x & 31; b < blocks; b += 32) s += parts[(long long)b * 2 * dim + i];
  s = over_head<32>(s);
  T* to = i < dim ? q_gain : k_gain;
  if ((threadIdx.x & 31) == 0 && to != nullptr) to[i < dim ? i : i - dim] = round_to<T>(s);
}

// Blocks that the backward pass runs with: their sums are joined by a second kernel.
static int blocks_of(long long tokens, int per_block, bool back) {
  const long long want = (tokens + per_block - 1) / per_block, most = back ? 148 * 3 : 1ll << 30;
  return static_cast<int>(want < most ? want : most);
}
static int per_block_of(long long tokens) { return tokens >= 148 * 8 * MOST_TOKENS ? MOST_TOKENS : 1; }

template <typename T, int LANES, bool BACK>
static cudaError_t launch_rotary(const RotaryArgs& a, bool neighbours, int blocks, cudaStream_t stream) {
  return launch_following(neighbours ? norm_rotary_kernel<T, LANES, true, BACK> : norm_rotary_kernel<T, LANES, false, BACK>,
                          dim3(static_cast<unsigned>(blocks)), dim3(ROTARY_THREADS), 0, stream, a);
}
template <typename T, bool BACK>
static cudaError_t launch_rotary(const RotaryArgs& a, bool neighbours, int blocks, cudaStream_t stream) {
  return a.dim <= 64 ? launch_rotary<T, 4, BACK>(a, neighbours, blocks, stream)
       : a.dim <= 128 ? launch_rotary<T, 8, BACK>(a, neighbours, blocks, stream) : launch_rotary<T, 16, BACK>(a, neighbours, blocks, stream);
}

}  // namespace nbc

// Floats of scratch of a backward call with gains.
extern "C" long long nb_norm_rotary_scratch(int batch, int tokens, int dim) {
  const long long n = (long long)batch * tokens;
  return 2ll * dim * nbc::blocks_of(n, nbc::per_block_of(n), true);
}

// Parts q, k and, where v_heads > 0, v, which is copied. strides: in elements, [x, dy][q, k, v][batch, token, head]. Results are dense (batch, tokens, heads,
// dim) each or, `packed`, one (batch, tokens, heads, {q, k, v}, dim). Backward where dy of q is given: results are gradients then. -1: sizes that the
// kernels do not take.
extern "C" int nb_norm_rotary(const void* q, const void* k, const void* v, const void* q_dy, const void* k_dy, const void* v_dy, void* q_out, void* k_out,
                              void* v_out, const void* q_gain, const void* k_gain, void* q_gain_grad, void* k_gain_grad, const void* positions, int wide,
                              int positions_shared, int batch, int tokens, int q_heads, int k_heads, int v_heads, int dim, int rotary, int neighbours,
                              double log2_base, float eps, const long long* strides, int packed, float* scratch, int fp32, void* stream) {
  using namespace nbc;
  const long long n = (long long)batch * tokens;
  if (n < 1 || n >= 1ll << 30 || dim < 16 || dim > MOST_DIM || dim % 16 || rotary < 16 || rotary > dim || rotary % 16) return -1;
  RotaryArgs a = {};
  const void* xs[3] = {q, k, v};
  const void* dys[3] = {q_dy, k_dy, v_dy};
  void* outs[3] = {q_out, k_out, v_out};
  const void* gains[3] = {q_gain, k_gain, nullptr};
  const int heads[3] = {q_heads, k_heads, v_heads};
  a.parts = v_heads > 0 ? 3 : 2, a.copied = v_heads > 0 ? 1 : 0;
  for (int p = 0; p < 3; ++p) {
    Heads& h = a.part[p];
    h.x = xs[p], h.dy = dys[p], h.out = outs[p], h.gain = gains[p], h.heads = heads[p];
    const long long row = packed ? 3ll * dim : dim, token = row * heads[p];
    h.out_s[0] = token * tokens, h.out_s[1] = token, h.out_s[2] = row;
    for (int i = 0; i < 3; ++i) h.x_s[i] = strides[3 * p + i], h.dy_s[i] = strides[9 + 3 * p + i];
  }
  a.batch = batch, a.tokens = tokens, a.dim = dim, a.rotary = rotary, a.all_heads = q_heads + k_heads + v_heads;
  a.positions = Whole{positions, wide}, a.positions_shared = positions_shared, a.log2_base = log2_base, a.eps = eps;
  const bool back = q_dy != nullptr, sums = back && (q_gain_grad != nullptr || k_gain_grad != nullptr);
  if (sums && scratch == nullptr) return -1;
  a.sums = sums ? scratch : nullptr;
  a.per_block = per_block_of(n);
  const int blocks = blocks_of(n, a.per_block, back);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (fp32) e = back ? launch_rotary<float, true>(a, neighbours, blocks, s) : launch_rotary<float, false>(a, neighbours, blocks, s);
  else e = back ? launch_rotary<__nv_bfloat16, true>(a, neighbours, blocks, s) : launch_rotary<__nv_bfloat16, false>(a, neighbours, blocks, s);
  if (e != cudaSuccess || !sums) return e;
  const dim3 grid((2 * dim + 7) / 8);
  if (fp32)
    return launch_following(gain_sums_kernel<float>, grid, dim3(256), 0, s, static_cast<const float*>(scratch), blocks, dim,
                            static_cast<float*>(q_gain_grad), static_cast<float*>(k_gain_grad));
  return launch_following(gain_sums_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, static_cast<const float*>(scratch), blocks, dim,
                          static_cast<__nv_bfloat16*>(q_gain_grad), static_cast<__nv_bfloat16*>(k_gain_grad));
}

NB_DEBUG_DEFINE(norm_rotary)
