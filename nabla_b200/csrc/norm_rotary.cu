// Norms of the heads of queries and keys and their rotation by the position, in one pass, and the gradient.
//
//   n = x * rsqrt(mean x^2 + eps),  z = n * g,  y = R z        over the D numbers of a head; without a gain: z = x
// R turns the pairs (z_i, z_i + rotary / 2), or neighbours (z_2i, z_2i + 1), of the first `rotary` numbers by position * base^(-2 i / rotary).
// Given dy:  dz = R^T dy,  dg = sum over all heads of dz n,  dx = r (dz g - n mean(dz g n))  with r the reciprocal root of above. Without a gain dx = dz.
//
// A head is held by D / 16 lanes (rounded up to a power of two), 16 numbers each: both halves of eight pairs, so a rotation needs no exchange and the means
// take two to four. A group of lanes keeps its head, and so its gain, for all tokens of its block; what it reads next is on its way into a ring in shared
// memory, each lane's own, so that no lane waits for another and no registers hold it. The angles of a token are the same for all its heads: the block
// puts their cosines and sines into shared memory first. An angle is a fraction of a turn in whole numbers of 2^-64, which the caller has rounded from more bits
// (an exponential in 64 bits is off by 2^-54 and more, a position of 2^33 by 10^-6 then), and only what is left of a whole turn becomes a number of 32 bits
// (a position of 10^6 would be off by 0.06 in 32 bits); that remainder is carried in two parts, so cosines and sines are off by two units in the last place, those
// of small angles too, and by 2^-62 for each position.
//
// Bound by memory: 8 x 2048 tokens of 16 heads of 128 with their values in bf16 take 73 us forward, 403 MB, 5.5 TB/s, and 103 us backward, 537 MB, 5.2 TB/s (a plain
// copy 6.5); 4 x 2048 tokens of 16 + 16 heads in fp32 54 and 83, 4.9 TB/s. Before the ring, with 2 or 4 tokens in registers, 90 to 108 and 165 to 378 (spilled). Three
// to eight stages of the ring are alike. Small calls are bound by the start of the launches, 6 us each way on the device.
#include "kv_cache.cuh"

namespace nbc {
using nb::follow_grid;
using nb::launch_following;

constexpr int MOST_THREADS = 256, MOST_DIM = 256, ANGLES = 2048, MOST_TOKENS = ANGLES / 8;

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
  int batch, tokens, dim, rotary, all_heads;
  int heads, abreast, chunk, chunks;       // of a block: heads, tokens at once; tokens of a chunk, chunks of a sequence
  Whole positions;
  int positions_shared;          // one row of positions for the whole batch
  float eps;
  float* sums;                   // backward: [blocks][2][dim] parts of the gradients of the gains
  unsigned long long turns[MOST_DIM / 2];        // of pairs, for a position, in 2^-64 of a turn: products with positions are taken modulo whole turns by themselves
};

__device__ __forceinline__ void fill_turns(const RotaryArgs& a, unsigned long long* turns) {
  for (int i = threadIdx.x; i < a.rotary / 2; i += blockDim.x) turns[i] = a.turns[i];
}
// cosines and, ANGLES behind them, sines of n tokens from the first, [token][rotary / 2]. All threads.
__device__ __forceinline__ void fill_angles(const RotaryArgs& a, const unsigned long long* turns, float* angles, long long* at, int first, int n) {
  const int half = a.rotary / 2;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) at[i] = a.positions.at(first + i);
  __syncthreads();
  const int more_t = blockDim.x / half, more_k = blockDim.x - more_t * half;
  int t = threadIdx.x / half, k = threadIdx.x - t * half;
  for (int i = threadIdx.x; t < n; i += blockDim.x) {
    // the fraction, from -2^63 to 2^63, in half turns: all of it, for the angle of a slow pair is in its lower bits. What a float does not hold goes into the second
    // part (2^63 itself, which the float may be, comes back as the number below it)
    const long long rest = static_cast<long long>(static_cast<unsigned long long>(at[t]) * turns[k]);
    const float hi = __ll2float_rn(rest), lo = __ll2float_rn(rest - __float2ll_rn(hi)) * (3.14159265f / 9223372036854775808.f);
    float s, c;
    sincospif(hi * (1.f / 9223372036854775808.f), &s, &c);
    angles[i] = fmaf(-lo, s, c), angles[ANGLES + i] = fmaf(lo, c, s);
    t += more_t, k += more_k;
    if (k >= half) k -= half, ++t;
  }
  __syncthreads();
}

// Sum over the LANES neighbouring lanes that hold a head.
template <int LANES>
__device__ __forceinline__ float over_head(float x) {
#pragma unroll
  for (int w = 1; w < LANES; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
  return x;
}
__device__ __forceinline__ float2 twice(float x) { return make_float2(x, x); }

// The 16 numbers of a lane as eight pairs (x, y), two pairs to an element: x[e] are the first numbers of pairs 2e and 2e + 1.
struct Pairs {
  float2 x[4], y[4];
};
// They lie in PIECES runs of 16 bytes, `step` apart, so that a run of all lanes of a head is one stretch of memory (lanes that read 32 bytes in a row, 16 at
// a time, fetch every sector twice: 4 x 2048 tokens of 32 heads of 128 in fp32 70 us). What is turned and what is not are shared out apart.
template <typename T>
struct Runs {
  static constexpr int PIECES = 2 * static_cast<int>(sizeof(T)) / 2, VEC = 16 / static_cast<int>(sizeof(T));
  int base, step;                          // in numbers of the head
  int angle, angle_step;                   // the first angle of a run, of runs of Q
  __device__ __forceinline__ int at(int piece) const { return base + piece * step; }
};
template <bool NEIGHBOURS, typename T>
constexpr int RUN = Runs<T>::VEC / (NEIGHBOURS ? 2 : 1);       // angles in a row
template <typename T, bool NEIGHBOURS>
__device__ __forceinline__ Runs<T> runs_of(const RotaryArgs& a, int lane) {
  constexpr int VEC = Runs<T>::VEC, Q = RUN<NEIGHBOURS, T>;
  const int turned = a.rotary / 16, n = lane < turned ? turned : a.dim / 16 - turned, l = lane < turned ? lane : lane - turned;
  return Runs<T>{(lane < turned ? 0 : a.rotary) + VEC * l, n * VEC, Q * l, n * Q};
}
// Number i of the 16 as they lie in the runs: halves have the eight first numbers in front of the second ones, neighbours alternate.
template <bool NEIGHBOURS>
__device__ __forceinline__ float& number(Pairs& v, int i) {
  const int pair = NEIGHBOURS ? i / 2 : i & 7;
  float2& e = (NEIGHBOURS ? i & 1 : i >> 3) ? v.y[pair / 2] : v.x[pair / 2];
  return pair & 1 ? e.y : e.x;
}
template <typename T>
__device__ __forceinline__ void numbers_of(uint4 w, float (&x)[Runs<T>::VEC]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(u[i]);
    else x[2 * i] = __uint_as_float(u[i] << 16), x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
template <typename T, bool NEIGHBOURS>
__device__ __forceinline__ Pairs unpack(const uint4 (&w)[Runs<T>::PIECES]) {
  Pairs v;
#pragma unroll
  for (int p = 0; p < Runs<T>::PIECES; ++p) {
    float x[Runs<T>::VEC];
    numbers_of<T>(w[p], x);
#pragma unroll
    for (int i = 0; i < Runs<T>::VEC; ++i) number<NEIGHBOURS>(v, p * Runs<T>::VEC + i) = x[i];
  }
  return v;
}
template <typename T, bool NEIGHBOURS>
__device__ __forceinline__ void store(T* out, const Runs<T>& r, Pairs& v) {
#pragma unroll
  for (int p = 0; p < Runs<T>::PIECES; ++p) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        u[i] = __float_as_uint(number<NEIGHBOURS>(v, p * 4 + i));
      } else {
        const __nv_bfloat162 o = __floats2bfloat162_rn(number<NEIGHBOURS>(v, p * 8 + 2 * i), number<NEIGHBOURS>(v, p * 8 + 2 * i + 1));
        u[i] = *reinterpret_cast<const uint32_t*>(&o);
      }
    }
    *reinterpret_cast<uint4*>(out + r.at(p)) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}
// Pairs turned by the angles whose cosines begin at cs, or back.
template <typename T, bool NEIGHBOURS, bool BACK>
__device__ __forceinline__ void turn(Pairs& v, const float* cs, const Runs<T>& r) {
  constexpr int Q = RUN<NEIGHBOURS, T>;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float* at = cs + r.angle + 2 * e / Q * r.angle_step + 2 * e % Q;
    const float2 c = *reinterpret_cast<const float2*>(at), s = *reinterpret_cast<const float2*>(at + ANGLES);
    float2 &x = v.x[e], &y = v.y[e];
    const float2 u = make_float2(BACK ? fmaf(y.x, s.x, x.x * c.x) : fmaf(-y.x, s.x, x.x * c.x), BACK ? fmaf(y.y, s.y, x.y * c.y) : fmaf(-y.y, s.y, x.y * c.y));
    y = make_float2(BACK ? fmaf(-x.x, s.x, y.x * c.x) : fmaf(x.x, s.x, y.x * c.x), BACK ? fmaf(-x.y, s.y, y.y * c.y) : fmaf(x.y, s.y, y.y * c.y));
    x = u;
  }
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }

template <typename T, bool BACK>
struct Ring {                              // of a lane: STAGES heads of PIECES times 16 bytes. (More stages gave nothing: 73 to 78 us for 73.7)
  static constexpr int PIECES = (BACK ? 2 : 1) * Runs<T>::PIECES, STAGES = PIECES == 2 ? 4 : PIECES == 4 ? 3 : 2;
};

template <typename T, int LANES, bool NEIGHBOURS, bool BACK>
__global__ void __launch_bounds__(MOST_THREADS, BACK ? 2 : 3) norm_rotary_kernel(const RotaryArgs a) {
  constexpr int PIECES = Ring<T, BACK>::PIECES, STAGES = Ring<T, BACK>::STAGES, RUNS = Runs<T>::PIECES;
  __shared__ unsigned long long turns[MOST_DIM / 2];
  __shared__ long long positions[MOST_TOKENS];
  __shared__ __align__(16) float angles[2 * ANGLES];
  extern __shared__ __align__(16) uint8_t ring[];          // [stage][piece][thread] 16 bytes; at the end the sums of the groups
  fill_turns(a, turns);
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, abreast = group / a.heads;
  int h = blockIdx.y * a.heads + group - abreast * a.heads, p = 0;
  const bool mine = 16 * lane < a.dim && h < a.all_heads && abreast < a.abreast;
  while (p + 1 < a.parts && h >= a.part[p].heads) h -= a.part[p].heads, ++p;
  const Heads& part = a.part[p];
  const bool copied = p >= a.parts - a.copied, normed = !copied && part.gain != nullptr, turned = 16 * lane < a.rotary && !copied;
  const Runs<T> runs = runs_of<T, NEIGHBOURS>(a, lane);
  const float over_dim = 1.f / static_cast<float>(a.dim);
  follow_grid();
  Pairs gain, sums;                        // sums: of the gradient of the gain
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    number<NEIGHBOURS>(gain, i) = mine && normed ? static_cast<float>(static_cast<const T*>(part.gain)[runs.at(i / Runs<T>::VEC) + i % Runs<T>::VEC]) : 1.f;
    number<NEIGHBOURS>(sums, i) = 0.f;
  }
  const uint32_t slot = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + threadIdx.x * 16, row = blockDim.x * 16;

  // The block's units: chunks of tokens of sequences. Where positions are shared, those of all sequences for a chunk come after each other, with the same angles
  const int units = a.batch * a.chunks, unit0 = static_cast<int>((long long)blockIdx.x * units / gridDim.x),
            unit1 = static_cast<int>((blockIdx.x + 1ll) * units / gridDim.x);
  struct Place { int b, t0; };
  auto next = [&](Place& q) {
    if (a.positions_shared) {
      if (++q.b == a.batch) q.b = 0, q.t0 += a.chunk;
    } else if ((q.t0 += a.chunk) >= a.tokens) {
      q.t0 = 0, ++q.b;
    }
  };
  Place now;
  if (a.positions_shared) now = Place{unit0 % a.batch, unit0 / a.batch * a.chunk}; else now = Place{unit0 / a.chunks, unit0 % a.chunks * a.chunk};
  const int steps = (a.chunk + a.abreast - 1) / a.abreast;   // of a unit, the same for all groups, which exchange
  const long long x_step = a.abreast * part.x_s[1], dy_step = a.abreast * part.dy_s[1], out_step = a.abreast * part.out_s[1];
  // the reader, STAGES - 1 steps ahead (units that are over have no tokens)
  const T *x = nullptr, *dy = nullptr;
  Place ahead = now;
  int ahead_unit = unit0 - 1, ahead_n = 0, ahead_steps = 0, ahead_slot = 0;          // ahead_n: tokens from this group's on
  auto get = [&] {
    if (ahead_steps == 0) {
      ahead_steps = steps;
      if (ahead_unit >= unit0) next(ahead);
      if (++ahead_unit < unit1) {
        x = static_cast<const T*>(part.x) + ahead.b * part.x_s[0] + (ahead.t0 + abreast) * part.x_s[1] + h * part.x_s[2];
        dy = static_cast<const T*>(part.dy) + ahead.b * part.dy_s[0] + (ahead.t0 + abreast) * part.dy_s[1] + h * part.dy_s[2];
        ahead_n = min(a.tokens - ahead.t0, a.chunk) - abreast;
      } else {
        ahead_n = 0;
      }
    }
    const uint32_t to = slot + ahead_slot * PIECES * row;
    if (mine && ahead_n > 0 && NB_IN_BOUNDS(NB_SITE_ROW_INDEX, ahead_unit, units)) {
      if (!BACK || normed)
#pragma unroll
        for (int i = 0; i < RUNS; ++i) copy16(to + i * row, x + runs.at(i));
      if (BACK)
#pragma unroll
        for (int i = 0; i < RUNS; ++i) copy16(to + (RUNS + i) * row, dy + runs.at(i));
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    x += x_step, dy += dy_step, ahead_n -= a.abreast, --ahead_steps;
    ahead_slot = ahead_slot + 1 == STAGES ? 0 : ahead_slot + 1;
  };
#pragma unroll 1
  for (int i = 0; i < STAGES - 1; ++i) get();
  int now_slot = 0, angles_of = -1;
  for (int unit = unit0; unit < unit1; ++unit, next(now)) {
    const int n = min(a.tokens - now.t0, a.chunk), which = a.positions_shared ? now.t0 : unit;
    if (which != angles_of) fill_angles(a, turns, angles, positions, a.positions_shared ? now.t0 : now.b * a.tokens + now.t0, n);
    angles_of = which;
    T* to = static_cast<T*>(part.out) + now.b * part.out_s[0] + (now.t0 + abreast) * part.out_s[1] + h * part.out_s[2];
    int t = abreast;
#pragma unroll 1
    for (int step = 0; step < steps; ++step, t += a.abreast, to += out_step) {
      const bool there = mine && t < n;
      get();
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      const uint8_t* from = ring + threadIdx.x * 16 + now_slot * PIECES * row;
      now_slot = now_slot + 1 == STAGES ? 0 : now_slot + 1;
      uint4 w[RUNS], u[RUNS];
#pragma unroll
      for (int i = 0; i < RUNS; ++i) {
        w[i] = *reinterpret_cast<const uint4*>(from + i * row);
        if (BACK) u[i] = *reinterpret_cast<const uint4*>(from + (RUNS + i) * row);
      }
      const float* cs = angles + (there && turned ? t * (a.rotary / 2) : 0);
      Pairs v = unpack<T, NEIGHBOURS>(w);
      float2 squares = twice(0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) squares = __ffma2_rn(v.x[e], v.x[e], squares), squares = __ffma2_rn(v.y[e], v.y[e], squares);
      const float r = rsqrtf(fmaf(over_head<LANES>(there ? squares.x + squares.y : 0.f), over_dim, a.eps));
      if (!BACK) {
        if (normed)
#pragma unroll
          for (int e = 0; e < 4; ++e) v.x[e] = __fmul2_rn(v.x[e], __fmul2_rn(gain.x[e], twice(r))), v.y[e] = __fmul2_rn(v.y[e], __fmul2_rn(gain.y[e], twice(r)));
        if (turned) turn<T, NEIGHBOURS, false>(v, cs, runs);
        if (there) store<T, NEIGHBOURS>(to, runs, v);
        continue;
      }
      Pairs d = unpack<T, NEIGHBOURS>(u);
      if (turned) turn<T, NEIGHBOURS, true>(d, cs, runs);
      float2 dot = twice(0.f);
      if (normed && there)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v.x[e] = __fmul2_rn(v.x[e], twice(r)), v.y[e] = __fmul2_rn(v.y[e], twice(r));
          const float2 s = __fmul2_rn(d.x[e], v.x[e]), z = __fmul2_rn(d.y[e], v.y[e]);
          sums.x[e] = __fadd2_rn(sums.x[e], s), sums.y[e] = __fadd2_rn(sums.y[e], z);
          dot = __ffma2_rn(s, gain.x[e], dot), dot = __ffma2_rn(z, gain.y[e], dot);
          d.x[e] = __fmul2_rn(d.x[e], gain.x[e]), d.y[e] = __fmul2_rn(d.y[e], gain.y[e]);
        }
      const float2 mean = twice(-over_head<LANES>(dot.x + dot.y) * over_dim);
      if (normed)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          d.x[e] = __fmul2_rn(__ffma2_rn(v.x[e], mean, d.x[e]), twice(r)), d.y[e] = __fmul2_rn(__ffma2_rn(v.y[e], mean, d.y[e]), twice(r));
      if (there) store<T, NEIGHBOURS>(to, runs, d);
    }
  }
  if (!BACK || a.sums == nullptr) return;
  // the block's sums: every group's in shared memory, then one thread for each number adds the groups of its part up in their order
  float* joined = reinterpret_cast<float*>(ring);          // [groups][dim]
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  if (mine)
#pragma unroll
    for (int i = 0; i < 16; ++i) joined[group * a.dim + runs.at(i / Runs<T>::VEC) + i % Runs<T>::VEC] = number<NEIGHBOURS>(sums, i);
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.dim; i += blockDim.x) {
    const int q = i / a.dim, at = i - q * a.dim, from = q ? a.part[0].heads : 0, to = from + a.part[q].heads;
    float s = 0.f;
    const int low = max(from - static_cast<int>(blockIdx.y) * a.heads, 0), high = min(to - static_cast<int>(blockIdx.y) * a.heads, a.heads);
    for (int g = 0; g < a.abreast; ++g)
      for (int k = low; k < high; ++k) s += joined[(g * a.heads + k) * a.dim + at];
    a.sums[((long long)blockIdx.y * gridDim.x + blockIdx.x) * 2 * a.dim + i] = s;
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

// How a call is cut. Heads of a block: all of them, or as many as MOST_THREADS hold; where they are few, several tokens abreast, so that a block has
// some 256 threads.
struct RotaryCut {
  int lanes, heads, abreast, chunk, chunks, across, blocks, threads;
};
static RotaryCut cut_rotary(int batch, int tokens, int all_heads, int dim, int rotary, int positions_shared, bool back) {
  RotaryCut c;
  c.lanes = dim <= 64 ? 4 : dim <= 128 ? 8 : 16;
  const int most = MOST_THREADS / c.lanes;
  c.across = (all_heads + most - 1) / most;
  c.heads = (all_heads + c.across - 1) / c.across;
  c.abreast = 256 / (c.heads * c.lanes);
  if (c.abreast < 1) c.abreast = 1;
  if (c.abreast > tokens) c.abreast = tokens;
  c.threads = (c.heads * c.abreast * c.lanes + 31) / 32 * 32;
  // A group of a block has 16 tokens (backward, where every block leaves a row of sums: what two blocks to an SM have), or less where there are too few for
  // three blocks to an SM. Where the angles serve several sequences, those of up to four take turns with a quarter of the tokens each.
  const int turns = positions_shared ? (batch < 4 ? batch : 4) : 1, room = ANGLES / (rotary / 2), each = (back ? 32 : 16) / turns;
  const long long resident = (148 * (back ? 2 : 3) + c.across - 1) / c.across, share = ((long long)batch * tokens + resident - 1) / resident;
  long long per = (share + c.abreast - 1) / c.abreast * c.abreast;
  if (per > each * c.abreast) per = each * c.abreast;
  c.chunk = static_cast<int>(per < room ? per : room);
  if (c.chunk > tokens) c.chunk = tokens;
  c.chunks = (tokens + c.chunk - 1) / c.chunk;
  const long long all = (long long)batch * c.chunks, want = back || all / turns < resident ? resident : (all + turns - 1) / turns;
  c.blocks = static_cast<int>(all < want ? all : want);
  return c;
}

template <typename T, int LANES, bool BACK>
static cudaError_t launch_rotary(const RotaryArgs& a, bool neighbours, const RotaryCut& c, cudaStream_t stream) {
  const auto kernel = neighbours ? norm_rotary_kernel<T, LANES, true, BACK> : norm_rotary_kernel<T, LANES, false, BACK>;
  constexpr size_t STAGE = Ring<T, BACK>::PIECES * 16;
  const size_t need = Ring<T, BACK>::STAGES * STAGE * c.threads, sums = a.sums == nullptr ? 0 : static_cast<size_t>(c.heads) * c.abreast * a.dim * 4, smem = need > sums ? need : sums;
  if (smem > 48 * 1024 - (2 * ANGLES * 4 + MOST_DIM * 4 + MOST_TOKENS * 8)) {            // with the static part
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  return launch_following(kernel, dim3(static_cast<unsigned>(c.blocks), static_cast<unsigned>(c.across)), dim3(static_cast<unsigned>(c.threads)), smem, stream, a);
}
template <typename T, bool BACK>
static cudaError_t launch_rotary(const RotaryArgs& a, bool neighbours, const RotaryCut& c, cudaStream_t stream) {
  return c.lanes == 4 ? launch_rotary<T, 4, BACK>(a, neighbours, c, stream)
       : c.lanes == 8 ? launch_rotary<T, 8, BACK>(a, neighbours, c, stream) : launch_rotary<T, 16, BACK>(a, neighbours, c, stream);
}

}  // namespace nbc

// Floats of scratch of a backward call with gains.
extern "C" long long nb_norm_rotary_scratch(int batch, int tokens, int all_heads, int dim, int rotary, int positions_shared) {
  const nbc::RotaryCut c = nbc::cut_rotary(batch, tokens, all_heads, dim, rotary, positions_shared, true);
  return 2ll * dim * c.blocks * c.across;
}

// Parts q, k and, where v_heads > 0, v, which is copied. turns: see RotaryArgs. strides: in elements, [x, dy][q, k, v][batch, token, head]. Results are dense (batch, tokens, heads,
// dim) each or, `packed`, one (batch, tokens, heads, {q, k, v}, dim). Backward where dy of q is given: results are gradients then. -1: sizes that the
// kernels do not take.
extern "C" int nb_norm_rotary(const void* q, const void* k, const void* v, const void* q_dy, const void* k_dy, const void* v_dy, void* q_out, void* k_out,
                              void* v_out, const void* q_gain, const void* k_gain, void* q_gain_grad, void* k_gain_grad, const void* positions, int wide,
                              int positions_shared, int batch, int tokens, int q_heads, int k_heads, int v_heads, int dim, int rotary, int neighbours,
                              const unsigned long long* turns, float eps, const long long* strides, int packed, float* scratch, int fp32, void* stream) {
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
  a.positions = Whole{positions, wide}, a.positions_shared = positions_shared, a.eps = eps;
  for (int i = 0; i < rotary / 2; ++i) a.turns[i] = turns[i];
  const bool back = q_dy != nullptr, sums = back && (q_gain_grad != nullptr || k_gain_grad != nullptr);
  if (sums && scratch == nullptr) return -1;
  a.sums = sums ? scratch : nullptr;
  const RotaryCut c = cut_rotary(batch, tokens, a.all_heads, dim, rotary, positions_shared, back);
  a.heads = c.heads, a.abreast = c.abreast, a.chunk = c.chunk, a.chunks = c.chunks;
  const int blocks = c.blocks * c.across;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (fp32) e = back ? launch_rotary<float, true>(a, neighbours, c, s) : launch_rotary<float, false>(a, neighbours, c, s);
  else e = back ? launch_rotary<__nv_bfloat16, true>(a, neighbours, c, s) : launch_rotary<__nv_bfloat16, false>(a, neighbours, c, s);
  if (e != cudaSuccess || !sums) return e;
  const dim3 grid((2 * dim + 7) / 8);
  if (fp32)
    return launch_following(gain_sums_kernel<float>, grid, dim3(256), 0, s, static_cast<const float*>(scratch), blocks, dim,
                            static_cast<float*>(q_gain_grad), static_cast<float*>(k_gain_grad));
  return launch_following(gain_sums_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, static_cast<const float*>(scratch), blocks, dim,
                          static_cast<__nv_bfloat16*>(q_gain_grad), static_cast<__nv_bfloat16*>(k_gain_grad));
}

NB_DEBUG_DEFINE(norm_rotary)
