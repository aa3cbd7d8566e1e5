// Attention over a key / value cache in 8 bits whose sequences begin with the same tokens (the operation and its terms: cached_attention.cu).
//
//   o = sum over the prefix and the own keys j of softmax_j(scale * s_k(j) * (q . k_j)) * s_v(j) * v_j
//
// Every query sees all `limit` keys of the prefix, and of its sequence's own ones what it would see without it. The prefix is read once for all
// sequences: their queries are the rows of one problem (FIRST), 128 to a tile of the tensor cores or 8 or 16 to a tile of the form for few rows, whose keys
// are cut into ranges so that the chip is full. A row's result over a range, and log2 of the sum of its weights, is a part. The own keys follow as in
// cached_attention (SECOND), and where a row's result is stored it is joined with the row's parts, in their order: a sum of numbers of a few ranges
// each, in fp32, that does not depend on which block was first. Where sequences have so many rows that tiles of 128 are full with each alone, a
// block walks over the keys of the prefix and then over the own ones (WHOLE), and there are no parts.
//
// 64 sequences of 50 to 1000 behind 8001 tokens, 16 heads over 4 of 128: 27 us (each over its whole text 71); 16 of up to 2000 behind 60001, 16 over 2: 43;
// 4 behind 1000: 9 on the device. What bounds it: the start and end of blocks (7 us of those of 128-row tiles) and the chain of product, exponentials and product
// of few tiles of keys for each block; for the last, starts. Prompts of 32 x 200 behind 2048: 193 us, exponentials (cached_attention_tcgen05.cu). Far from
// their floors are many sequences with some tokens each behind a short prefix, whose blocks pay their start and end for one or two steps of keys (81 x 10 behind 50, 24
// heads over 8, 74 us; 27 x 301 behind 50, 119), and fp32 of more than 32 rows, which widens the codes again for every 16 rows (32 x 200 behind 2048 1187 us).
#include "cached_attention_few.cuh"

namespace nbc {

// How the prefix is cut: rows of a tile, tiles of 128 rows to a block, ranges of its keys.
struct FirstCut {
  int rows, q_tiles, splits;
};
// `c`: how the own keys are cut, in lines of at most `room` keys. That is the rule of cached_attention, whose borders were measured for a kernel that has the chip to itself;
// here it shares the chip with the prefix. The times below are those of bf16 and heads of 128, of one step of keys and of a block's start and end; heads of 64 and
// fp32 go by them too, which was not measured for itself (results do not depend on the cut but by the order of sums).
static FirstCut cut_first(int rows, int kv_heads, long long prefix_room, int fp32, const Cut& c, int batch, int own_rows, long long room) {
  // Tiles of 128 rows start late and are soon quicker. us, tiles of 16 and of 128, behind 500, 2001 and 8001 tokens: 2 heads with 40 rows 10.8 and 15.6, 11.3 and
  // 16.0, 20.0 and 17.1, with 128 rows 9.2 and 14.8, 15.3 and 15.0, 20.0 and 16.6; 4 heads with 96 rows 9.5 and 14.6, 17.3 and 15.0, 22.6 and 19.3; 16 heads with
  // 64 rows 16.7 and 15.1, 21.5 and 22.3, 38.9 and 33.2.
  const bool wide = !fp32 && rows > 32 && (rows > 128 || (long long)kv_heads * ((rows + 15) / 16) * prefix_room > 32768);
  FirstCut f = {wide ? 128 : few_rows(rows), wide && rows > 128 ? 2 : 1, 1};
  const long long units = (long long)kv_heads * ((rows + f.rows * f.q_tiles - 1) / (f.rows * f.q_tiles)), least = wide ? 256 : UNIT,
                  most = (prefix_room + least - 1) / least;
  long long want = (wide ? 148 : 148 * (f.rows == 8 ? 3 : 2)) / units;
  if (wide && c.rows != 128) {
    // Blocks of 128-row tiles take an SM each, those of the own keys a third or half of one. Either the prefix has the chip for itself and the own keys follow, or it
    // takes the SMs that the own keys leave when all of their blocks run at once. us of the parts, measured: 7 for a block's start and end and 3.3 for a
    // tile of 128 keys with 256 rows, 2.2 with 128; 9 and 1.6 for each step of 128 keys of a line of own keys; 0.08 to join a part. Both together, behind 8001
    // tokens 64 sequences of up to 1000 with 16 heads over 4 27.2 beside each other (64 blocks) and 35.8 after each other (148), with up to 60 26.4 and 24.3; 16 of
    // up to 2000 with 16 heads over 2 behind 60001 49.5 and 41.1; 32 of up to 1000 behind 16001 26.7 (120 blocks) and 38.4.
    const long long lines = (long long)batch * kv_heads * ((own_rows + c.rows - 1) / c.rows);
    const long long blocks = c.share == FLAT ? c.splits : lines * c.splits, left = 148 - (blocks + (c.rows == 8 ? 2 : 1)) / (c.rows == 8 ? 3 : 2);
    const auto splits = [&](long long n) { return n / units < 1 ? 1 : n / units < most ? n / units : most; };
    const auto time = [&](long long n) {
      const long long tiles = (prefix_room + 127) / 128;
      return 7.0 + (f.q_tiles == 2 ? 3.3 : 2.2) * static_cast<double>((tiles + splits(n) - 1) / splits(n)) * static_cast<double>((units * splits(n) + n - 1) / n);
    };
    const double own = 9.0 + 1.6 * static_cast<double>(room) / UNIT / (c.share == ONE ? 1.0 : c.share == CLUSTER ? c.splits : static_cast<double>(c.splits) / lines);
    if (left >= units && left >= 16 && (time(left) > own ? time(left) : own) + 3.0 + 0.08 * splits(left) < time(148) + own + 0.08 * splits(148)) want = left / units;
  }
  f.splits = static_cast<int>(want < 2 || most < 2 ? 1 : want < most ? want : most);
  return f;
}

template <typename T, int D, int RT>
static cudaError_t first_few(const AttendArgs& a, cudaStream_t stream) {
  const long long grid = (long long)a.splits * a.kv_heads * ((a.fresh * (a.heads / a.kv_heads) + 8 * RT - 1) / (8 * RT));
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  return launch_following(attend_few_kernel<T, D, RT, ONE, FIRST>, dim3(static_cast<unsigned>(grid)), dim3(32 * FEW_WARPS), Few<D, RT>::SMEM, stream, a);
}
template <typename T, int D>
static cudaError_t launch_both(const AttendArgs& first, const FirstCut& f, const AttendArgs& second, const Cut& c, int* status, cudaStream_t stream) {
  if (f.splits == 0) {                     // WHOLE
    const cudaError_t e = launch_many<D, WHOLE>(second, 0, status, stream);
    return e != cudaSuccess || c.splits == 1 ? e : join<T, D, false, ALONE>(second, stream);
  }
  const cudaError_t e = f.rows == 128 ? launch_many<D, FIRST>(first, f.q_tiles, status, stream)
                      : f.rows == 8 ? first_few<T, D, 1>(first, stream) : first_few<T, D, 2>(first, stream);
  return e != cudaSuccess ? e : launch_attend<T, D, SECOND>(second, c, status, stream);
}

// Floats of the parts; what follows them starts on a boundary of 16 bytes.
static long long first_floats(long long rows, int splits, int head_dim) { return (rows * splits * (head_dim + 1) + 3) / 4 * 4; }
struct Cuts {
  bool whole;
  FirstCut first;
  Cut second;                    // whole: of all keys
};
static Cuts cut_both(int batch, int fresh, int heads, int kv_heads, int head_dim, long long prefix_room, long long room, int fp32) {
  const long long rows = (long long)batch * fresh * heads;
  const int own_rows = fresh * (heads / kv_heads);
  const Cut c = cut(batch, own_rows, rows, kv_heads, head_dim, room, fp32);
  const Cuts both = {false, cut_first(static_cast<int>(rows / kv_heads), kv_heads, prefix_room, fp32, c, batch, own_rows, room), c};
  if (c.rows != 128 || both.first.rows != 128) return both;
  // Two kernels pack the rows of all sequences densely for the prefix; one does not leave and join parts, and starts its blocks once. SM * us for each head and
  // sequence, from the times at cut_first: blocks of 256 rows, the last of 128 or fewer.
  const double tiles = static_cast<double>((prefix_room + 127) / 128), own = static_cast<double>((room + 127) / 128);
  const int full = own_rows / 256, left = (own_rows - full * 256 + 127) / 128;
  const double for_tile = 3.3 * full + (left == 2 ? 3.3 : left == 1 ? 2.2 : 0.0), blocks = full + (left > 0);
  const double two = own_rows / 256.0 * (3.3 * tiles + 9.0) + for_tile * own + 13.0 * blocks, one = for_tile * (tiles + own) + 9.0 * blocks;
  if (two <= one) return both;
  return Cuts{true, FirstCut{128, 0, 0}, cut(batch, own_rows, rows, kv_heads, head_dim, prefix_room + room, fp32)};
}
}  // namespace nbc

// Scratch of a call with these sizes, in floats (0: none).
extern "C" long long nb_shared_prefix_scratch(int batch, int fresh, int heads, int kv_heads, int head_dim, int block, int prefix_columns, int columns, int fp32) {
  using namespace nbc;
  const long long rows = (long long)batch * fresh * heads;
  if (rows > 0x7fffffffll) return -1;
  const Cuts c = cut_both(batch, fresh, heads, kv_heads, head_dim, (long long)prefix_columns * block, (long long)columns * block, fp32);
  return first_floats(rows, c.first.splits, head_dim) + c.second.scratch;
}
// Kernels that a call launches.
extern "C" int nb_shared_prefix_launches(int batch, int fresh, int heads, int kv_heads, int head_dim, int block, int prefix_columns, int columns, int fp32) {
  using namespace nbc;
  const Cuts c = cut_both(batch, fresh, heads, kv_heads, head_dim, (long long)prefix_columns * block, (long long)columns * block, fp32);
  return (c.whole ? 1 : 2) + (c.second.scratch > 0);
}

// Strides of q as the rows of one sequence: q_sb = fresh * q_st, or fresh is 1. wide: bit 0 prefix_table, 1 prefix_length, 2 table, 3 past, 4 count are
// 64-bit numbers.
extern "C" int nb_shared_prefix_attention(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, void* out,
                                          const void* prefix_table, const void* prefix_length, const void* table, const void* past, const void* count,
                                          int wide, int batch, int fresh, int heads, int kv_heads, int head_dim, int block, int blocks, int prefix_columns,
                                          int columns, long long q_sb, long long q_st, long long q_sh, float scale, int causal, float* scratch, int fp32,
                                          int* status, void* stream) {
  using namespace nbc;
  AttendArgs a = {};
  a.q = q, a.q_sb = q_sb, a.q_st = q_st, a.q_sh = q_sh;
  a.codes[0] = static_cast<const int8_t*>(k_codes), a.codes[1] = static_cast<const int8_t*>(v_codes);
  a.scales[0] = static_cast<const float*>(k_scales), a.scales[1] = static_cast<const float*>(v_scales);
  a.out = out;
  a.heads = heads, a.kv_heads = kv_heads;
  a.block_log = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : block == 128 ? 7 : -1;
  a.scale_log2 = scale * 1.4426950408889634f;
  const long long rows = (long long)batch * fresh * heads;
  if (a.block_log < 0 || (head_dim != 64 && head_dim != 128) || rows > 0x7fffffffll) return -1;
  if (batch > 1 && fresh > 1 && q_sb != fresh * q_st) return -1;
  const Cuts cuts = cut_both(batch, fresh, heads, kv_heads, head_dim, (long long)prefix_columns * block, (long long)columns * block, fp32);
  const FirstCut& f = cuts.first;
  const Cut& c = cuts.second;
  if ((f.splits > 0 || c.scratch > 0) && scratch == nullptr) return -1;
  AttendArgs first = a;
  first.table = Table{Whole{prefix_table, wide & 1}, prefix_columns, blocks};
  first.limit = Whole{prefix_length, wide >> 1 & 1};
  first.batch = 1, first.fresh = batch * fresh, first.causal = 0;
  first.q_st = fresh == 1 ? q_sb : q_st;
  first.splits = f.splits, first.tile_rows = f.rows;
  first.part_o = scratch, first.part_w = scratch + rows * f.splits * head_dim;
  scratch += first_floats(rows, f.splits, head_dim);
  a.table = Table{Whole{table, wide >> 2 & 1}, columns, blocks};
  a.past = Whole{past, wide >> 3 & 1}, a.count = Whole{count, wide >> 4 & 1};
  a.batch = batch, a.fresh = fresh, a.causal = causal;
  a.first_o = first.part_o, a.first_w = first.part_w, a.first_parts = f.splits;
  a.limit = first.limit, a.first_table = first.table;
  set_parts(a, c, scratch, head_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (fp32) return head_dim == 64 ? launch_both<float, 64>(first, f, a, c, status, s) : launch_both<float, 128>(first, f, a, c, status, s);
  return head_dim == 64 ? launch_both<__nv_bfloat16, 64>(first, f, a, c, status, s) : launch_both<__nv_bfloat16, 128>(first, f, a, c, status, s);
}

NB_DEBUG_DEFINE(shared_prefix)
