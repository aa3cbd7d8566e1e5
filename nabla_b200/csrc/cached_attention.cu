// Attention over a key / value cache in 8 bits (layout: kv_cache.cuh).
//
//   o = sum_j softmax_j(scale * s_k(j) * (q . k_j)) * s_v(j) * v_j       codes k, v and scales s_k, s_v of the block that holds key j
//
// Query i of a sequence with `past` tokens in front and `count` new ones sees keys 0 ... past + i (causal) or past + count - 1. Rows from
// `count` on, and rows that see no key, are zero. `group` query heads share a head of the cache.
#include "cached_attention_few.cuh"

// The last row of a block of `block` tokens that the few-row kernel's loads touch for the range [from, from + length) of a sequence's keys.
extern "C" int nb_cached_attention_last_row(int keys, int from, int length, int block) {
  using namespace nbc;
  const Keys k = keys_of(keys, from, length);
  int last = 0;
  for (int warp = 0; warp < FEW_WARPS; ++warp)
    for (int mine = steps_of(k, warp), step = 0; step < (mine > 0 ? mine : 0) + 2; ++step)
      for (int i = 0; i < 2; ++i) {
        const int row = row_of(key_of(k, warp, mine, step), i, block) + 15;
        last = row > last ? row : last;
      }
  return last;
}

// Scratch of a call with these sizes, in floats.
extern "C" long long nb_cached_attention_scratch(int batch, int fresh, int heads, int kv_heads, int head_dim, int block, int columns, int fp32) {
  return nbc::cut(batch, fresh * (heads / kv_heads), (long long)batch * fresh * heads, kv_heads, head_dim, (long long)columns * block, fp32).scratch;
}

extern "C" int nb_cached_attention(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, void* out,
                                   const void* table, const void* past, const void* count, int wide, int batch, int fresh, int heads, int kv_heads,
                                   int head_dim, int block, int blocks, int columns, long long q_sb, long long q_st, long long q_sh, float scale,
                                   int causal, float* scratch, int fp32, int* status, void* stream) {
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
  const Cut c = cut(batch, fresh * (heads / kv_heads), (long long)batch * fresh * heads, kv_heads, head_dim, (long long)columns * block, fp32);
  if (c.scratch > 0 && scratch == nullptr) return -1;
  set_parts(a, c, scratch, head_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (fp32) return head_dim == 64 ? launch_attend<float, 64, ALONE>(a, c, status, s) : launch_attend<float, 128, ALONE>(a, c, status, s);
  return head_dim == 64 ? launch_attend<__nv_bfloat16, 64, ALONE>(a, c, status, s) : launch_attend<__nv_bfloat16, 128, ALONE>(a, c, status, s);
}

NB_DEBUG_DEFINE(cached_attention)
