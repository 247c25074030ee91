// block_quant.hip -- append into the 8-bit pools with one scale for each
// (block, KV head) tile (rkv_append_block_q).
//
// A wave owns one tile of one pool (K or V): it reads the call's new rows that
// fall in the tile, takes their maximum, settles the tile's scale with the one
// it had for older rows, and writes the new rows' bytes; older rows are read
// and rounded to the new scale only where that grew.  The rows of a tile are
// settled by one wave, so no two writers meet on its scale.
// Bound by one chain of round trips (lengths, table, rows, store) for a decode step: 64
// sequences of one row, 8 KV heads of 128, 4.7 us, one sequence 3.9; by HBM for a
// prompt: 8 x 512 rows 13.5 us (42 MB, 3.1 TB/s).
// Lane l of pass i holds elements 4 (l % U) .. + 3 of row (64 / U) i + l / U, U
// = D / 4 words a row: 16-byte loads, 4-byte stores, contiguous over a row.
#include "block_quant.hpp"

namespace rkv {
namespace {

constexpr int kBS = 16;

template <int D, int DT>
__global__ __launch_bounds__(256) void append_block_q_kernel(
    uint8_t* __restrict__ k_pool, uint8_t* __restrict__ v_pool, float* __restrict__ k_scale,
    float* __restrict__ v_scale, int64_t pool_layer_stride, int64_t scale_layer_stride,
    const float* __restrict__ k_new, const float* __restrict__ v_new, int64_t src_layer_stride,
    int64_t src_tok_stride, int64_t src_head_stride, const int32_t* __restrict__ new_start,
    const int32_t* __restrict__ block_tables, int max_blocks_per_seq,
    const int32_t* __restrict__ ctx_lens, int num_kv_heads, int64_t num_blocks, int max_new) {
  constexpr int U = D / 4;          // words a row
  constexpr int RPP = 64 / U;       // rows a pass
  constexpr int NP = kBS / RPP;     // passes a tile
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = (int64_t)blockIdx.x * 4 + w;  // (touched block, head, K | V)
  const int per = 2 * num_kv_heads;
  const int j = (int)(unit / per), rem = (int)(unit - (int64_t)j * per);
  const int h = rem >> 1;
  const bool is_v = rem & 1;
  const int b = blockIdx.y, layer = blockIdx.z;
  const int s0 = new_start[b], n = new_start[b + 1] - s0;
  const int64_t pos0 = (int64_t)ctx_lens[b] - n;  // of the first new row
  const int take = n < max_new ? n : max_new;
  const int64_t first = pos0 < 0 ? 0 : pos0;
  const int64_t lb = first / kBS + j;  // the tile's block in the sequence
  if (take <= 0 || lb >= max_blocks_per_seq) return;
  const int64_t lo64 = first > lb * kBS ? first : lb * kBS;
  const int64_t hi64 = pos0 + take < (lb + 1) * kBS ? pos0 + take : (lb + 1) * kBS;
  if (lo64 >= hi64) return;
  const int32_t blk = block_tables[(int64_t)b * max_blocks_per_seq + lb];
  if (blk < 0 || blk >= num_blocks) return;
  const int lo = (int)(lo64 - lb * kBS), hi = (int)(hi64 - lb * kBS);  // rows lo .. hi - 1 are new
  const int64_t tile = (int64_t)blk * num_kv_heads + h;
  float* const sp = (is_v ? v_scale : k_scale) + layer * scale_layer_stride + tile;
  const float s_old = lo > 0 ? *sp : 0.0f;

  const int sub = lane / U, c = lane - sub * U;
  const float* src = (is_v ? v_new : k_new) + layer * src_layer_stride + h * src_head_stride + 4 * c;
  const int64_t row0 = s0 + lb * kBS - pos0;  // source row of the tile's row 0
  float4 x[NP];
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = RPP * i + sub;
    x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r >= lo && r < hi)
      x[i] = *reinterpret_cast<const float4*>(src + (row0 + r) * src_tok_stride);
  }
#pragma unroll
  for (int i = 0; i < NP; ++i)
    m = fmaxf(m, fmaxf(fmaxf(finite_abs(x[i].x), finite_abs(x[i].y)),
                       fmaxf(finite_abs(x[i].z), finite_abs(x[i].w))));
  const float need = tile_scale<DT>(wave_max(m));
  const float s = fmaxf(s_old, need);
  const float inv = s > 0.0f ? 1.0f / s : 0.0f;
  const bool grew = lo > 0 && s > s_old;  // wave-uniform
  const float ratio = grew ? s_old / s : 1.0f;
  uint32_t* dst = reinterpret_cast<uint32_t*>((is_v ? v_pool : k_pool) +
                                              layer * pool_layer_stride + tile * (kBS * D));
  if (grew) {
    uint32_t old[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = RPP * i + sub;
      old[i] = r < lo ? dst[r * U + c] : 0u;
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = RPP * i + sub;
      if (r < lo) dst[r * U + c] = tile_reword<DT>(old[i], s_old, s, ratio);
    }
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = RPP * i + sub;
    if (r >= lo && r < hi)
      dst[r * U + c] = tile_word<DT>(x[i], s, inv);
  }
  if (lane == 0 && (lo == 0 || grew)) *sp = s;
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_append_block_q(void* k_pool, void* v_pool, float* k_scale, float* v_scale,
                                  int64_t pool_layer_stride, const float* k_new,
                                  const float* v_new, int64_t src_layer_stride,
                                  int64_t src_tok_stride, int64_t src_head_stride,
                                  const int32_t* new_start, const int32_t* block_tables,
                                  int max_blocks_per_seq, const int32_t* ctx_lens, int num_seqs,
                                  int n_layers, int num_kv_heads, int head_dim, int block_size,
                                  int64_t num_blocks, int max_new, int dtype, void* stream) {
  clear_error();
  if (num_kv_heads <= 0 || num_blocks < 0 || num_seqs < 0 || n_layers < 0 || max_new < 0 ||
      max_blocks_per_seq < 0)
    return fail(RKV_ERR_INVALID_ARG, "rkv_append_block_q: bad size argument");
  if (!block_scaled(dtype))
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_append_block_q: dtype must be RKV_I8_BLOCK or RKV_FP8_BLOCK");
  if (block_size != kBS)
    return fail(RKV_ERR_UNSUPPORTED, "rkv_append_block_q: block_size must be 16");
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(RKV_ERR_UNSUPPORTED, "rkv_append_block_q: head_dim must be 32, 64 or 128");
  if (num_seqs > 65535 || n_layers > 65535)
    return fail(RKV_ERR_INVALID_ARG, "rkv_append_block_q: num_seqs and n_layers must be <= 65535");
  if (num_seqs == 0 || n_layers == 0 || max_new == 0 || max_blocks_per_seq == 0) return RKV_OK;
  if (!k_pool || !v_pool || !k_scale || !v_scale || !k_new || !v_new || !new_start ||
      !block_tables || !ctx_lens)
    return fail(RKV_ERR_INVALID_ARG, "rkv_append_block_q: null pointer argument");
  if ((src_layer_stride | src_tok_stride | src_head_stride) & 3)
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_append_block_q: source strides must be multiples of 4 elements");
  if (!aligned16(k_new) || !aligned16(v_new) || !aligned16(k_pool) || !aligned16(v_pool))
    return fail(RKV_ERR_INVALID_ARG, "rkv_append_block_q: pointers must be 16-byte aligned");
  if (n_layers > 1 && pool_layer_stride % (kBS * head_dim))
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_append_block_q: pool_layer_stride must be a multiple of 16 * head_dim");
  // n rows from any row of a block on touch at most (n + 14) / 16 + 1 blocks
  int64_t touched = ((int64_t)max_new + kBS - 2) / kBS + 1;
  if (touched > max_blocks_per_seq) touched = max_blocks_per_seq;
  const int64_t wgs = (touched * 2 * num_kv_heads + 3) / 4;
  if (wgs > 0x7fffffff)
    return fail(RKV_ERR_INVALID_ARG, "rkv_append_block_q: max_new too large for one launch");
  const dim3 grid((unsigned)wgs, (unsigned)num_seqs, (unsigned)n_layers);
  const int64_t scale_ls = n_layers > 1 ? pool_layer_stride / (kBS * head_dim) : 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
#define RKV_APPEND_B(D, T)                                                                     \
  append_block_q_kernel<D, T><<<grid, 256, 0, st>>>(                                           \
      static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool), k_scale, v_scale,          \
      pool_layer_stride, scale_ls, k_new, v_new, src_layer_stride, src_tok_stride,             \
      src_head_stride, new_start, block_tables, max_blocks_per_seq, ctx_lens, num_kv_heads,    \
      num_blocks, max_new)
#define RKV_APPEND_BD(T)                        \
  do {                                          \
    if (head_dim == 32) RKV_APPEND_B(32, T);    \
    else if (head_dim == 64) RKV_APPEND_B(64, T); \
    else RKV_APPEND_B(128, T);                  \
  } while (0)
  if (dtype == RKV_I8_BLOCK) RKV_APPEND_BD(RKV_I8_BLOCK);
  else RKV_APPEND_BD(RKV_FP8_BLOCK);
#undef RKV_APPEND_BD
#undef RKV_APPEND_B
  return check_launch("rkv_append_block_q");
}
