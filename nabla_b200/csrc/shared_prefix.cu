// Attention over a key / value cache in 8 bits whose sequences begin with the same tokens (the operation and its terms: cached_attention.cu).
//
//   o = sum over the prefix and the own keys j of softmax_j(scale * s_k(j) * (q . k_j)) * s_v(j) * v_j
//
// Every query sees all `limit` keys of the prefix, and of its sequence's own ones what it would see without it. The prefix is read once for all
// sequences: their queries are the rows of one problem (FIRST), 128 to a tile of the tensor cores or 8 or 16 to a tile of the form for few rows, whose keys
// are cut into ranges so that the chip is full. A row's result over a range, and log2 of the sum of its weights, is a part. The own keys follow as in
// cached_attention (SECOND), and where a row's result is stored it is joined with the row's parts, in their order: a sum of numbers of a few ranges
// each, in fp32, that does not depend on which block was first.
#include "cached_attention_few.cuh"

namespace nbc {

// How the prefix is cut: rows of a tile, ranges of its keys.
struct FirstCut {
  int rows, splits;
};
static FirstCut cut_first(int rows, int kv_heads, long long room, int fp32) {
  const bool wide = !fp32 && rows > 32;
  FirstCut c = {wide ? 128 : few_rows(rows), 1};
  const long long units = (long long)kv_heads * ((rows + c.rows - 1) / c.rows), blocks = wide ? 148 : 148 * (c.rows == 8 ? 3 : 2);
  const long long least = wide ? 512 : UNIT, most = (room + least - 1) / least, want = blocks / units;
  c.splits = static_cast<int>(want < 2 || most < 2 ? 1 : want < most ? want : most);
  return c;
}

template <typename T, int D, int RT>
static cudaError_t first_few(const AttendArgs& a, cudaStream_t stream) {
  const long long grid = (long long)a.splits * a.kv_heads * ((a.fresh * (a.heads / a.kv_heads) + 8 * RT - 1) / (8 * RT));
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  return launch_following(attend_few_kernel<T, D, RT, ONE, FIRST>, dim3(static_cast<unsigned>(grid)), dim3(32 * FEW_WARPS), Few<D, RT>::SMEM, stream, a);
}
template <typename T, int D>
static cudaError_t launch_both(const AttendArgs& first, const FirstCut& f, const AttendArgs& second, const Cut& c, int* status, cudaStream_t stream) {
  const cudaError_t e = f.rows == 128 ? launch_many<D, FIRST>(first, status, stream)
                      : f.rows == 8 ? first_few<T, D, 1>(first, stream) : first_few<T, D, 2>(first, stream);
  return e != cudaSuccess ? e : launch_attend<T, D, SECOND>(second, c, status, stream);
}

// Floats of the parts; what follows them starts on a boundary of 16 bytes.
static long long first_floats(long long rows, int splits, int head_dim) { return (rows * splits * (head_dim + 1) + 3) / 4 * 4; }
static Cut cut_second(int batch, int fresh, int heads, int kv_heads, int head_dim, long long room, int fp32) {
  return cut(batch, fresh * (heads / kv_heads), (long long)batch * fresh * heads, kv_heads, head_dim, room, fp32);
}
}  // namespace nbc

// Scratch of a call with these sizes, in floats.
extern "C" long long nb_shared_prefix_scratch(int batch, int fresh, int heads, int kv_heads, int head_dim, int block, int prefix_columns, int columns, int fp32) {
  using namespace nbc;
  const long long rows = (long long)batch * fresh * heads;
  if (rows > 0x7fffffffll) return -1;
  return first_floats(rows, cut_first(static_cast<int>(rows / kv_heads), kv_heads, (long long)prefix_columns * block, fp32).splits, head_dim)
         + cut_second(batch, fresh, heads, kv_heads, head_dim, (long long)columns * block, fp32).scratch;
}
// Kernels that a call launches.
extern "C" int nb_shared_prefix_launches(int batch, int fresh, int heads, int kv_heads, int head_dim, int block, int columns, int fp32) {
  return nbc::cut_second(batch, fresh, heads, kv_heads, head_dim, (long long)columns * block, fp32).scratch > 0 ? 3 : 2;
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
  if (a.block_log < 0 || (head_dim != 64 && head_dim != 128) || rows > 0x7fffffffll || scratch == nullptr) return -1;
  if (batch > 1 && fresh > 1 && q_sb != fresh * q_st) return -1;
  const FirstCut f = cut_first(static_cast<int>(rows / kv_heads), kv_heads, (long long)prefix_columns * block, fp32);
  AttendArgs first = a;
  first.table = Table{Whole{prefix_table, wide & 1}, prefix_columns, blocks};
  first.limit = Whole{prefix_length, wide >> 1 & 1};
  first.batch = 1, first.fresh = batch * fresh, first.causal = 0;
  first.q_st = fresh == 1 ? q_sb : q_st;
  first.splits = f.splits, first.tile_rows = f.rows;
  first.part_o = scratch, first.part_w = scratch + rows * f.splits * head_dim;
  const Cut c = cut_second(batch, fresh, heads, kv_heads, head_dim, (long long)columns * block, fp32);
  scratch += first_floats(rows, f.splits, head_dim);
  a.table = Table{Whole{table, wide >> 2 & 1}, columns, blocks};
  a.past = Whole{past, wide >> 3 & 1}, a.count = Whole{count, wide >> 4 & 1};
  a.batch = batch, a.fresh = fresh, a.causal = causal;
  a.first_o = first.part_o, a.first_w = first.part_w, a.first_parts = f.splits;
  set_parts(a, c, scratch, head_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (fp32) return head_dim == 64 ? launch_both<float, 64>(first, f, a, c, status, s) : launch_both<float, 128>(first, f, a, c, status, s);
  return head_dim == 64 ? launch_both<__nv_bfloat16, 64>(first, f, a, c, status, s) : launch_both<__nv_bfloat16, 128>(first, f, a, c, status, s);
}

NB_DEBUG_DEFINE(shared_prefix)
