// paged_prefill_q.hip -- causal prefill attention over 8-bit pools with one scale
// a tile (rkv_prefill_attention_q): the mfma kernel of prefill_kernel.hpp, whose
// tiles become fp16 as they are staged.
#include "block_quant.hpp"
#include "prefill_kernel.hpp"

namespace rkv {
namespace {

template <int FORMAT, int D>
PrefillCfg pick_q(int G) {
  switch (G) {
    case 1: return cfg_g<uint8_t, D, 1, kWaves, false, FORMAT>();
    case 2: return cfg_g<uint8_t, D, 2, kWaves, false, FORMAT>();
    case 4: return cfg_g<uint8_t, D, 4, kWaves, false, FORMAT>();
    case 8: return cfg_g<uint8_t, D, 8, kWaves, false, FORMAT>();
    default: return {nullptr, 0, 0, false};
  }
}

template <int FORMAT>
PrefillCfg pick_qd(int D, int G) {
  switch (D) {
    case 64: return pick_q<FORMAT, 64>(G);
    case 128: return pick_q<FORMAT, 128>(G);
    default: return {nullptr, 0, 0, false};
  }
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_prefill_attention_q(float* out, const float* q, const void* k_pool,
                                       const void* v_pool, const float* k_scale,
                                       const float* v_scale, const int32_t* block_tables,
                                       int max_blocks_per_seq, const int32_t* q_start,
                                       const int32_t* ctx_lens, int num_seqs, int num_q_heads,
                                       int num_kv_heads, int head_dim, int block_size,
                                       int64_t num_blocks, int max_q_len, float scale, int dtype,
                                       void* stream) {
  clear_error();
  if (num_seqs < 0 || max_blocks_per_seq < 0 || num_blocks < 0 || max_q_len < 0)
    return fail(RKV_ERR_INVALID_ARG, "rkv_prefill_attention_q: negative size argument");
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads)
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_prefill_attention_q: num_q_heads must be a positive multiple of num_kv_heads");
  if (dtype == RKV_I8 || dtype == RKV_FP8)
    return fail(RKV_ERR_UNSUPPORTED,
                "rkv_prefill_attention_q: row-scaled pools have no prefill (rkv_gather_q reads "
                "them back); block-scaled ones do");
  if (!block_scaled(dtype))
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_prefill_attention_q: dtype must be RKV_I8_BLOCK or RKV_FP8_BLOCK");
  if (block_size != kBS)
    return fail(RKV_ERR_UNSUPPORTED, "rkv_prefill_attention_q: block_size must be 16");
  const int G = num_q_heads / num_kv_heads;
  const PrefillCfg cfg = dtype == RKV_I8_BLOCK ? pick_qd<RKV_I8_BLOCK>(head_dim, G)
                                               : pick_qd<RKV_FP8_BLOCK>(head_dim, G);
  if (!cfg.fn)
    return fail(RKV_ERR_UNSUPPORTED,
                "rkv_prefill_attention_q: head_dim must be 64 or 128 and num_q_heads / "
                "num_kv_heads 1, 2, 4 or 8");
  if (num_seqs > 65535 || num_kv_heads > 65535)
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_prefill_attention_q: num_seqs and num_kv_heads must be <= 65535");
  if (num_seqs == 0 || max_q_len == 0 || max_blocks_per_seq == 0) return RKV_OK;
  if ((int64_t)max_blocks_per_seq * kBS > 0x7fffffff)
    return fail(RKV_ERR_INVALID_ARG, "rkv_prefill_attention_q: max_blocks_per_seq too large");
  if (num_blocks < 1) return fail(RKV_ERR_INVALID_ARG, "rkv_prefill_attention_q: num_blocks < 1");
  if (!out || !q || !k_pool || !v_pool || !k_scale || !v_scale || !block_tables || !q_start ||
      !ctx_lens)
    return fail(RKV_ERR_INVALID_ARG, "rkv_prefill_attention_q: null pointer argument");
  if (!aligned16(out) || !aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool))
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_prefill_attention_q: out, q and pools must be 16-byte aligned");
  const int64_t n_tiles = ((int64_t)max_q_len + cfg.tile - 1) / cfg.tile;
  const int64_t n_heads = (int64_t)num_seqs * num_kv_heads;
  const int heavy = n_tiles <= 65535 && n_heads <= 0x7fffffff;
  const dim3 grid = heavy ? dim3((unsigned)n_heads, (unsigned)n_tiles, 1)
                          : dim3((unsigned)n_tiles, (unsigned)num_kv_heads, (unsigned)num_seqs);
  hipLaunchKernelGGL(cfg.fn, grid, dim3(64 * cfg.waves), 0, static_cast<hipStream_t>(stream), out,
                     q, k_pool, v_pool, block_tables, max_blocks_per_seq, q_start, ctx_lens,
                     num_kv_heads, num_blocks, max_q_len, scale * kLog2e, heavy, 0, 0, k_scale,
                     v_scale);
  return check_launch("rkv_prefill_attention_q");
}
