// paged_prefill.hip -- causal prefill attention over fp32 and bf16 pools
// (rkv_prefill_attention): the builds of the mfma kernel of prefill_kernel.hpp, and
// which one a call takes.
#include "prefill_kernel.hpp"

namespace rkv {
namespace {

// When the 4-wave build is taken: 2 on every call, 1 when the sequences
// hold at most as many cached keys as new tokens, 0 never.  fp32 pools (us
// per call, the four shapes of the table in prefill_kernel.hpp; 8-wave -> 4-wave): G = 1, D = 32
// 6.2 -> 5.8 / 14.5 -> 13.2 / 25.2 -> 23.2 / 95 -> 83; G = 1, D = 128 15.4
// -> 14.8 / 32.4 -> 30.7 / 57.2 = 58.4 / 219 -> 242; elsewhere slower or
// even (G = 4, D = 32: 11.6 = 11.6 / 25.0 -> 23.3 / 50.9 -> 52.2 / 209 ->
// 226; at D = 64 slower on all four; at D = 128 and G >= 4 the 4-wave form
// spills into AGPRs at one wave per SIMD).
constexpr int short_build_use(bool f32, int G, int D) {
  if (f32) return G == 1 && D == 32 ? 2 : G == 1 && D == 128 ? 1 : 0;
  return D == 64 ? 2 : G == 1 ? 2 : (D == 128 && G == 2) ? 0 : 1;
}

template <typename T>
constexpr int kFormat = sizeof(T) == 4 ? RKV_F32 : RKV_BF16;

template <typename T, int D, int G>
PrefillCfg cfg_pick(bool short_prefix) {
  constexpr int use = short_build_use(sizeof(T) == 4, G, D);
  if constexpr (use > 0)
    if (use == 2 || short_prefix) return cfg_g<T, D, G, kShortWaves, RKV_PREFILL_PREFETCH != 0, kFormat<T>>();
  return cfg_g<T, D, G, kWaves, false, kFormat<T>>();
}

template <typename T, int D>
PrefillCfg pick_g(int G, bool short_prefix) {
  switch (G) {
    case 1: return cfg_pick<T, D, 1>(short_prefix);
    case 2: return cfg_pick<T, D, 2>(short_prefix);
    case 4: return cfg_pick<T, D, 4>(short_prefix);
    case 8: return cfg_pick<T, D, 8>(short_prefix);
    default: return {nullptr, 0, 0, false};
  }
}

template <typename T>
PrefillCfg pick_d(int D, int G, bool short_prefix) {
  switch (D) {
    case 32: return pick_g<T, 32>(G, short_prefix);
    case 64: return pick_g<T, 64>(G, short_prefix);
    case 128: return pick_g<T, 128>(G, short_prefix);
    default: return {nullptr, 0, 0, false};
  }
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_prefill_attention(float* out, const float* q, const void* k_pool,
                                     const void* v_pool, const int32_t* block_tables,
                                     int max_blocks_per_seq, const int32_t* q_start,
                                     const int32_t* ctx_lens, int num_seqs, int num_q_heads,
                                     int num_kv_heads, int head_dim, int block_size,
                                     int64_t num_blocks, int max_q_len, float scale, int dtype,
                                     void* stream) {
  clear_error();
  if (num_seqs < 0 || max_blocks_per_seq < 0 || num_blocks < 0 || max_q_len < 0)
    return fail(RKV_ERR_INVALID_ARG, "rkv_prefill_attention: negative size argument");
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads)
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_prefill_attention: num_q_heads must be a positive multiple of num_kv_heads");
  if (dtype != RKV_F32 && dtype != RKV_BF16)
    return fail(RKV_ERR_INVALID_ARG, "rkv_prefill_attention: dtype must be RKV_F32 or RKV_BF16");
  if (block_size != kBS)
    return fail(RKV_ERR_UNSUPPORTED, "rkv_prefill_attention: block_size must be 16");
  const int G = num_q_heads / num_kv_heads;
  // at most as many cached keys as new tokens, judged by the table width
  // (the keys a sequence can hold) against the longest new-token run
  const bool short_prefix = (int64_t)max_blocks_per_seq * kBS <= 2 * (int64_t)max_q_len;
  const PrefillCfg cfg = dtype == RKV_BF16 ? pick_d<uint16_t>(head_dim, G, short_prefix)
                                           : pick_d<float>(head_dim, G, short_prefix);
  if (!cfg.fn)
    return fail(RKV_ERR_UNSUPPORTED,
                "rkv_prefill_attention: head_dim must be 32, 64 or 128 and num_q_heads / "
                "num_kv_heads 1, 2, 4 or 8");
  if (num_seqs > 65535 || num_kv_heads > 65535)
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_prefill_attention: num_seqs and num_kv_heads must be <= 65535");
  if (num_seqs == 0 || max_q_len == 0 || max_blocks_per_seq == 0) return RKV_OK;
  if ((int64_t)max_blocks_per_seq * kBS > 0x7fffffff)
    return fail(RKV_ERR_INVALID_ARG, "rkv_prefill_attention: max_blocks_per_seq too large");
  if (num_blocks < 1) return fail(RKV_ERR_INVALID_ARG, "rkv_prefill_attention: num_blocks < 1");
  if (!out || !q || !k_pool || !v_pool || !block_tables || !q_start || !ctx_lens)
    return fail(RKV_ERR_INVALID_ARG, "rkv_prefill_attention: null pointer argument");
  if (!aligned16(out) || !aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool))
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_prefill_attention: out, q and pools must be 16-byte aligned");
  const int64_t n_tiles = (max_q_len + cfg.tile - 1) / cfg.tile;
  const int64_t n_heads = (int64_t)num_seqs * num_kv_heads;
  const int heavy = RKV_PREFILL_HEAVY_FIRST && n_tiles <= 65535 && n_heads <= 0x7fffffff;
  const dim3 grid = heavy ? dim3((unsigned)n_heads, (unsigned)n_tiles, 1)
                          : dim3((unsigned)n_tiles, (unsigned)num_kv_heads, (unsigned)num_seqs);
  // Of R resident workgroups and T in all, the later ones (from R on) start
  // as slots free up.  The touches go to the last min(R, T - R) workgroups
  // of the first round (its lightest: the grid runs heaviest first), each
  // for the workgroup that many places later; the heaviest, which end the
  // first round, touch nothing.  25 admissions of a serving step (us per call, one
  // box, interleaved): 26.7 against 28.6 when the first T - R workgroups
  // touch and 27.4 when the first R - (T - R) touch workgroups of the first
  // round (8 x 512 square: the same workgroups either way, 52.6).
  int pf_stride = 0, pf_first = 0;
  if (cfg.next && heavy) {
    const int64_t R = resident_workgroups(cfg.fn, 64 * cfg.waves), T = n_heads * n_tiles;
    if (R > 0 && T > R) {
      pf_stride = (int)(T - R < R ? T - R : R);
      pf_first = (int)(R - pf_stride);
    }
  }
  hipLaunchKernelGGL(cfg.fn, grid, dim3(64 * cfg.waves), 0, static_cast<hipStream_t>(stream), out, q, k_pool,
                     v_pool, block_tables, max_blocks_per_seq, q_start, ctx_lens, num_kv_heads,
                     num_blocks, max_q_len, scale * kLog2e, heavy, pf_stride, pf_first, nullptr, nullptr);
  return check_launch("rkv_prefill_attention");
}
