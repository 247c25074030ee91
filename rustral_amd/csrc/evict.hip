// evict.hip -- eviction by accumulated attention weight: which rows of a
// sequence each KV head keeps (rkv_evict_select), and their move to the blocks
// of a new table (rkv_evict_compact).  The sums come from
// rkv_decode_attention_weights (paged_decode.hip).
#include "block_quant.hpp"

#include <type_traits>

namespace rkv {
namespace {

constexpr int kBS = 16;

// ---- select --------------------------------------------------------------------
// One workgroup per (layer, sequence, KV head).  Every position becomes a 32-bit
// key that orders like (class, weight): 0 absent, 1 a NaN sum, then the sums in
// float order, all ones the first and last positions, which are always kept.
// The n-th largest key is found by digits of 11, 11 and 10 bits from the top: a
// histogram in LDS of the keys that share the digits found so far, a sum over its
// bins from the top, and the bin where it passes what is still wanted.  Counts are
// integers, so their order does not matter.  It ends early where a bin is wanted
// whole.  The first digit is counted as the keys are formed; the keys of its bin are
// then listed in LDS, if they are at most LIST, and the later digits are taken from the
// list (else from all keys again).  Keys are kept in LDS for up to kKeysMax positions
// (KEYS); a longer context is read again by each of the passes.
// A wave owns a contiguous run of positions, so the kept ones' places need one
// exchange of the waves' totals; inside a wave they come from ballots: with the
// keys above the threshold and those that equal it counted apart, the place of a
// position is  (above before it) + min(equal before it, equal wanted),  so ties go
// to the lower position.
// Lane l of a step holds 4 positions, a float4 of one block.  The loops stay rolled:
// a grid of few workgroups runs each instruction about once.
// Bound by the round trips of its passes (loads 5 us, a pass over 32,768 keys in LDS
// 2 to 4), far from its bytes.  us for 8 layers x 16 sequences of U[1500, 4096] / 2
// layers x 1 of 32,768, 8 KV heads: 29.5 / 66 with keys in registers (unrolled) and 32
// counts of the keys above a candidate; 29.6 / 44.7 with keys in LDS and counts at
// candidates on a line between the last two; 17.1 / 26.1 with every digit taken from all
// keys (23.8 / 42.8 without keys in LDS); 15.1 / 22.2 with the list.

__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 and +0 are one weight
  const uint32_t k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return w == w ? k : 1u;
}

constexpr uint32_t kHeld = 0xffffffffu;
constexpr int kBins = 2048;
constexpr int kKeysMax = 32768;  // positions whose keys fit in LDS beside the bins

// Inclusive prefix sum over the wave: row_shr 1, 2, 4, 8 inside each 16-lane row
// (0 past its start), then the last lane of row 0 added to row 1 and of row 2 to row
// 3 (row_bcast:15), and of row 1 to rows 2 and 3 (row_bcast:31).
__device__ __forceinline__ uint32_t wave_prefix(uint32_t x) {
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);
  return x;
}

template <int NT, bool KEYS>
__global__ __launch_bounds__(NT) void evict_select_kernel(
    int32_t* __restrict__ keep, int32_t* __restrict__ new_lens,
    const float* __restrict__ weights, int64_t weights_layer_stride,
    const int32_t* __restrict__ block_tables, int max_blocks_per_seq,
    const int32_t* __restrict__ ctx_lens, int num_kv_heads, int64_t num_blocks, int budget,
    int sinks, int recent, int cap) {
  constexpr int NW = NT / 64;
  constexpr int BPT = kBins / NT;  // bins a thread
  constexpr int LIST = 4 * NT < 2048 ? 2048 : 4 * NT;
  extern __shared__ __align__(16) uint4 s_key[];  // KEYS: four positions each
  __shared__ __align__(16) uint32_t s_bin[kBins];
  __shared__ uint32_t s_sum[NW];
  __shared__ uint32_t s_found[3];  // the bin, its count, the count above it
  __shared__ uint32_t s_list[LIST];
  __shared__ int s_above[NW], s_equal[NW];
  __shared__ int s_listed;
  const int h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  int L = ctx_lens[b];
  L = L < 0 ? 0 : (L > cap ? cap : L);
  const int32_t* __restrict__ tab = block_tables + (int64_t)b * max_blocks_per_seq;
  const float* __restrict__ wl = weights + layer * weights_layer_stride;
  const int groups = (L + 3) / 4;
  const int steps = ((groups + 63) / 64 + NW - 1) / NW;  // of a wave
  const int g0 = w * steps * 64 + lane;                  // this lane's group of step 0

  auto form = [&](int g) __attribute__((always_inline)) {
    uint4 k = make_uint4(0u, 0u, 0u, 0u);
    const int p = 4 * g;
    if (g < groups) {
      const int32_t blk = tab[p / kBS];
      if (blk >= 0 && blk < num_blocks) {
        const float4 v = *reinterpret_cast<const float4*>(
            wl + ((int64_t)blk * num_kv_heads + h) * kBS + p % kBS);
        auto one = [&](float x, int q) -> uint32_t {
          const bool held = q < sinks || q >= L - recent;
          return q < L ? (held ? kHeld : weight_key(x)) : 0u;
        };
        k = make_uint4(one(v.x, p), one(v.y, p + 1), one(v.z, p + 2), one(v.w, p + 3));
      }
    }
    return k;
  };
  // Keys of this lane's group of a step.  A lane reads back only what it wrote.
  auto keys = [&](int j) __attribute__((always_inline)) {
    const int g = g0 + 64 * j;
    if constexpr (KEYS) return g < groups ? s_key[g] : make_uint4(0u, 0u, 0u, 0u);
    else return form(g);
  };
  auto clear_bins = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < BPT; ++i) s_bin[tid + NT * i] = 0u;
    __syncthreads();
  };
  // Adds four keys' digits (key >> shift) % 2^bits to the bins: those of non-zero keys
  // whose bits above are `top`.
  auto add4 = [&](const uint4& k4, int shift, int bits, uint32_t top) __attribute__((always_inline)) {
    const uint32_t mask = (1u << bits) - 1u;
    const int above = shift + bits;  // 32 for the first digit: no bits above
    const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
    uint32_t d[4];
    bool in[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      in[e] = k[e] != 0u && (above >= 32 || (k[e] >> (above & 31)) == top);
      d[e] = (k[e] >> shift) & mask;
    }
    // one add for a wave whose 256 keys fall in one bin (equal sums, where every
    // lane's add would wait for the others')
    const uint32_t d0 = __builtin_amdgcn_readfirstlane(d[0]);
    const bool same = in[0] && in[1] && in[2] && in[3] && d[0] == d0 && d[1] == d0 &&
                      d[2] == d0 && d[3] == d0;
    if (__builtin_amdgcn_ballot_w64(!same) == 0) {
      if (lane == 0) atomicAdd(&s_bin[d0], 256u);
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (in[e]) atomicAdd(&s_bin[d[e]], 1u);
  };
  // The bin from the top where the bins' count reaches `want`: s_found.  Returns the
  // bins' total.
  auto find = [&](uint32_t want) __attribute__((always_inline)) {
    __syncthreads();
    // thread t has bins kBins - 1 - BPT t downwards: prefix sums from the top
    uint32_t c[BPT], mine = 0;
#pragma unroll
    for (int i = 0; i < BPT; ++i) {
      c[i] = s_bin[kBins - 1 - (BPT * tid + i)];
      mine += c[i];
    }
    const uint32_t run = wave_prefix(mine);  // inclusive over the wave
    if (lane == 63) s_sum[w] = run;
    __syncthreads();
    uint32_t before = run - mine, total = 0;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const uint32_t v = s_sum[x];
      if (x < w) before += v;
      total += v;
    }
    if (want > 0 && before < want && want <= before + mine) {  // one thread
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        if (before < want && want <= before + c[i]) {
          s_found[0] = (uint32_t)(kBins - 1 - (BPT * tid + i));
          s_found[1] = c[i];
          s_found[2] = before;
          break;
        }
        before += c[i];
      }
    }
    __syncthreads();
    return total;
  };
  // A later digit over all keys.
  auto digit_all = [&](int shift, int bits, uint32_t top, uint32_t want) __attribute__((always_inline)) {
    clear_bins();
#pragma unroll 2
    for (int j = 0; j < steps; ++j) add4(keys(j), shift, bits, top);
    find(want);
  };

  // The first digit, as the keys are formed.
  if (tid == 0) s_listed = 0;
  clear_bins();
#pragma unroll 4
  for (int j = 0; j < steps; ++j) {
    const int g = g0 + 64 * j;
    const uint4 k = form(g);
    if constexpr (KEYS)
      if (g < groups) s_key[g] = k;
    add4(k, 21, 11, 0u);
  }
  const uint32_t present = find((uint32_t)budget);
  // thr and equal: a key is kept above thr, and `equal` of those that equal it
  uint32_t thr = 0u;
  int equal = 0;
  bool counted = false;  // s_above, s_equal hold the waves' totals
  const int n = present < (uint32_t)budget ? (int)present : budget;
  if (present > (uint32_t)n) {
    const uint32_t t1 = s_found[0], held = s_found[1];
    uint32_t top = t1, want = (uint32_t)n - s_found[2];
    int shift = 21;
    bool whole = held == want;
    if (!whole && held <= (uint32_t)LIST) {
      // list the bin's keys (their low 21 bits, the wave above) and count those above
      // the bin, then go on with the list
      int na = 0;
#pragma unroll 4
      for (int j = 0; j < steps; ++j) {
        const uint4 k4 = keys(j);
        const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
        uint64_t in[4];
        int count = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          na += __popcll(__builtin_amdgcn_ballot_w64((k[e] >> 21) > t1));
          in[e] = __builtin_amdgcn_ballot_w64((k[e] >> 21) == t1 && k[e] != 0u);
          count += __popcll(in[e]);
        }
        if (count == 0) continue;
        int at = 0;
        if (lane == 0) at = atomicAdd(&s_listed, count);
        at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int mine = __builtin_amdgcn_mbcnt_hi(
              (uint32_t)(in[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in[e], at));
          if ((in[e] >> lane) & 1u) s_list[mine] = (k[e] & 0x1fffffu) | (uint32_t)w << 21;
          at += __popcll(in[e]);
        }
      }
      if (lane == 0) s_above[w] = na, s_equal[w] = 0;
      auto digit_list = [&](int shift_, int bits, uint32_t low) __attribute__((always_inline)) {
        clear_bins();
        for (uint32_t i = tid; i < held; i += NT) {
          const uint32_t k = s_list[i] & 0x1fffffu;
          if (bits == 11 || k >> 10 == low) atomicAdd(&s_bin[(k >> shift_) & ((1u << bits) - 1u)], 1u);
        }
        find(want);
      };
      digit_list(10, 11, 0u);
      top = t1 << 11 | s_found[0], want -= s_found[2], shift = 10;
      whole = s_found[1] == want;
      if (!whole) {
        digit_list(0, 10, s_found[0]);
        top = top << 10 | s_found[0], want -= s_found[2], shift = 0;
      }
      counted = true;
    } else if (!whole) {
      digit_all(10, 11, top, want);
      top = top << 11 | s_found[0], want -= s_found[2], shift = 10;
      whole = s_found[1] == want;
      if (!whole) {
        digit_all(0, 10, top, want);
        top = top << 10 | s_found[0], want -= s_found[2], shift = 0;
      }
    }
    // a whole bin: everything from its first key on
    if (whole) thr = top ? (top << shift) - 1u : 0u;
    else thr = top, equal = (int)want;
    if (counted) {
      for (uint32_t i = tid; i < held; i += NT) {
        const uint32_t e = s_list[i], k = t1 << 21 | (e & 0x1fffffu);
        if (k > thr) atomicAdd(&s_above[e >> 21], 1);
        else if (k == thr) atomicAdd(&s_equal[e >> 21], 1);
      }
    }
  }
  if (h == 0 && layer == 0 && tid == 0) new_lens[b] = n;

  // Places, with the keys that equal the threshold (EQ) or, as usual, without: this
  // wave's totals, everybody's before it, then its positions in order.
  int32_t* __restrict__ out =
      keep + (((int64_t)layer * gridDim.y + b) * num_kv_heads + h) * budget;
  auto place = [&](auto with) __attribute__((always_inline)) {
    constexpr bool EQ = decltype(with)::value;
    if (!counted) {
      int na = 0, ne = 0;
#pragma unroll 4
      for (int j = 0; j < steps; ++j) {
        const uint4 k4 = keys(j);
        const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          na += __popcll(__builtin_amdgcn_ballot_w64(k[e] > thr));
          if constexpr (EQ) ne += __popcll(__builtin_amdgcn_ballot_w64(k[e] == thr));
        }
      }
      if (lane == 0) s_above[w] = na, s_equal[w] = ne;
    }
    __syncthreads();
    int xa = 0, xe = 0;
#pragma unroll
    for (int x = 0; x < NW; ++x)
      if (x < w) xa += s_above[x], xe += s_equal[x];
#pragma unroll 2
    for (int j = 0; j < steps; ++j) {
      const uint4 k4 = keys(j);
      const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
      int la = xa, le = xe;  // before this lane's four
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t ba = __builtin_amdgcn_ballot_w64(k[e] > thr);
        la = __builtin_amdgcn_mbcnt_hi((uint32_t)(ba >> 32),
                                       __builtin_amdgcn_mbcnt_lo((uint32_t)ba, la));
        xa += __popcll(ba);
        if constexpr (EQ) {
          const uint64_t be = __builtin_amdgcn_ballot_w64(k[e] == thr);
          le = __builtin_amdgcn_mbcnt_hi((uint32_t)(be >> 32),
                                         __builtin_amdgcn_mbcnt_lo((uint32_t)be, le));
          xe += __popcll(be);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool up = k[e] > thr, eq = EQ && k[e] == thr;
        if (up || (eq && le < equal)) {
          const int at = EQ ? la + (le < equal ? le : equal) : la;
          out[at] = 4 * (g0 + 64 * j) + e;
        }
        la += up ? 1 : 0;
        if constexpr (EQ) le += eq ? 1 : 0;
      }
    }
  };
  if (equal > 0) place(std::true_type{});  // workgroup-uniform
  else place(std::false_type{});
  for (int i = n + tid; i < budget; i += NT) out[i] = -1;
}

// ---- compact --------------------------------------------------------------------
// One wave per (layer, sequence, KV head, destination block): lanes 0 .. 15 look
// up where the block's 16 rows come from, then the wave moves the rows of K and
// V 16 bytes a lane, all loads issued before the first store.  UPR: 16-byte
// units a row (template for the unrolled builds, 0: any).  Rows are 128 to 512
// bytes at scattered places, so whole rows are what memory is asked for.
// Bound by HBM: 8 layers x 16 sequences x 1,024 bf16 rows of 8 x 128, 1.07 GB, 214 us
// (5.0 TB/s); 2 layers x 8,192 int8 rows with a scale a tile, 67 MB, 19.0 us, 5 of
// them the launch and the three round trips to the first row.
template <int DT>
constexpr bool row_scales() { return DT == RKV_I8 || DT == RKV_FP8; }
template <int DT>
constexpr bool tile_scales() { return DT == RKV_I8_BLOCK || DT == RKV_FP8_BLOCK; }

template <int DT, int UPR>
__global__ __launch_bounds__(256) void evict_compact_kernel(
    uint8_t* __restrict__ k_pool, uint8_t* __restrict__ v_pool, float* __restrict__ k_scale,
    float* __restrict__ v_scale, float* __restrict__ weights, int64_t layer_bytes,
    int64_t scale_layer_stride, int64_t weights_layer_stride, const int32_t* __restrict__ keep,
    const int32_t* __restrict__ new_lens, int budget, const int32_t* __restrict__ src_tables,
    int src_blocks, const int32_t* __restrict__ dst_tables, int dst_blocks, int num_kv_heads,
    int upr_any, int64_t num_blocks) {
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = (int64_t)blockIdx.x * 4 + w;
  const int j = (int)(unit / num_kv_heads), h = (int)(unit - (int64_t)j * num_kv_heads);
  const int b = blockIdx.y, layer = blockIdx.z;
  if (j >= dst_blocks) return;
  // One round trip for what the arguments alone place (keep past new_lens is within its
  // row of the array), then the source table, then the rows.
  const int row = lane & 15;
  const int at = j * kBS + row;
  int32_t p = at < budget
                  ? keep[(((int64_t)layer * gridDim.y + b) * num_kv_heads + h) * budget + at]
                  : -1;
  const int32_t dst = dst_tables[(int64_t)b * dst_blocks + j];
  int n = new_lens[b];
  n = n > budget ? budget : n;
  if (at >= n) p = -1;
  if ((int64_t)j * kBS >= n || dst < 0 || dst >= num_blocks) return;
  // source row (in rows of the layer's pool) of destination row lane, or -1
  int64_t from = -1;
  int32_t sblk = -1;
  if (p >= 0 && p < src_blocks * kBS) {
    sblk = src_tables[(int64_t)b * src_blocks + p / kBS];
    if (sblk >= 0 && sblk < num_blocks)
      from = ((int64_t)sblk * num_kv_heads + h) * kBS + p % kBS;
  }
  const bool live = from >= 0;
  const int64_t to = ((int64_t)dst * num_kv_heads + h) * kBS;
  if (weights && lane < kBS && live) {
    float* wl = weights + layer * weights_layer_stride;
    wl[to + row] = wl[from];
  }
  float ks = 0.0f, vs = 0.0f, kt = 0.0f, vt = 0.0f;  // source row's scale, the tile's
  if constexpr (row_scales<DT>()) {
    if (lane < kBS && live) {
      float* kl = k_scale + layer * scale_layer_stride;
      float* vl = v_scale + layer * scale_layer_stride;
      kl[to + row] = kl[from];
      vl[to + row] = vl[from];
    }
  } else if constexpr (tile_scales<DT>()) {
    float* kl = k_scale + layer * scale_layer_stride;
    float* vl = v_scale + layer * scale_layer_stride;
    if (live) {
      const int64_t tile = (int64_t)sblk * num_kv_heads + h;
      ks = kl[tile];
      vs = vl[tile];
    }
    kt = group_max<16>(ks);  // every 16-lane row holds the same 16 rows
    vt = group_max<16>(vs);
    const bool any = __builtin_amdgcn_ballot_w64(live) != 0;
    if (lane == 0 && any) {
      const int64_t tile = (int64_t)dst * num_kv_heads + h;
      kl[tile] = kt;
      vl[tile] = vt;
    }
  }
  const int upr = UPR ? UPR : upr_any;  // 16-byte units a row
  const int64_t rb = (int64_t)upr * 16;
  uint8_t* kp = k_pool + layer * layer_bytes;
  uint8_t* vp = v_pool + layer * layer_bytes;
  auto convert = [&](uint4 x, float s, float t) {
    if constexpr (tile_scales<DT>()) {
      if (s != t) {
        const float ratio = s / t;  // t > s >= 0
        x.x = tile_reword<DT>(x.x, s, t, ratio);
        x.y = tile_reword<DT>(x.y, s, t, ratio);
        x.z = tile_reword<DT>(x.z, s, t, ratio);
        x.w = tile_reword<DT>(x.w, s, t, ratio);
      }
    }
    return x;
  };
  auto shfl64 = [&](int64_t v, int src) {
    const int lo = __shfl((int)(uint32_t)v, src), hi = __shfl((int)(v >> 32), src);
    return ((int64_t)hi << 32) | (uint32_t)lo;
  };
  if constexpr (UPR > 0) {
    constexpr int NU = kBS * UPR;                 // units of a tile
    constexpr int NP = NU >= 64 ? NU / 64 : 1;    // passes
    uint4 xk[NP], xv[NP];
    int64_t src[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int u = lane + 64 * i;
      const int r = u / UPR < kBS ? u / UPR : kBS - 1;
      src[i] = shfl64(from, r);
      if (u >= NU) src[i] = -1;
      if (src[i] >= 0) {
        xk[i] = load_stream(kp + src[i] * rb + (u % UPR) * 16);
        xv[i] = load_stream(vp + src[i] * rb + (u % UPR) * 16);
      }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int u = lane + 64 * i;
      const int r = u / UPR < kBS ? u / UPR : kBS - 1;
      float sk = 0.0f, sv = 0.0f;
      if constexpr (tile_scales<DT>()) {
        sk = __shfl(ks, r);
        sv = __shfl(vs, r);
      }
      if (src[i] >= 0) {
        store_stream(kp + (to + r) * rb + (u % UPR) * 16, convert(xk[i], sk, kt));
        store_stream(vp + (to + r) * rb + (u % UPR) * 16, convert(xv[i], sv, vt));
      }
    }
  } else {
    for (int r = 0; r < kBS; ++r) {
      const int64_t src = shfl64(from, r);
      if (src < 0) continue;  // wave-uniform
      for (int u = lane; u < upr; u += 64) {
        const uint4 a = load_stream(kp + src * rb + u * 16);
        const uint4 c = load_stream(vp + src * rb + u * 16);
        store_stream(kp + (to + r) * rb + u * 16, a);
        store_stream(vp + (to + r) * rb + u * 16, c);
      }
    }
  }
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_evict_select(int32_t* keep, int32_t* new_lens, const float* weights,
                                int64_t weights_layer_stride, const int32_t* block_tables,
                                int max_blocks_per_seq, const int32_t* ctx_lens, int num_seqs,
                                int n_layers, int num_kv_heads, int block_size,
                                int64_t num_blocks, int budget, int sinks, int recent,
                                int max_context, void* stream) {
  clear_error();
  if (num_seqs < 0 || n_layers < 0 || num_kv_heads <= 0 || num_blocks < 0 ||
      max_blocks_per_seq < 0 || max_context < 0)
    return fail(RKV_ERR_INVALID_ARG, "rkv_evict_select: bad size argument");
  if (block_size != kBS)
    return fail(RKV_ERR_UNSUPPORTED, "rkv_evict_select: block_size must be 16");
  if (budget <= 0 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_evict_select: budget must be > 0 and hold sinks + recent rows");
  if (num_seqs > 65535 || n_layers > 65535)
    return fail(RKV_ERR_INVALID_ARG, "rkv_evict_select: num_seqs and n_layers must be <= 65535");
  if ((int64_t)max_blocks_per_seq * kBS > 0x7fffff00)
    return fail(RKV_ERR_INVALID_ARG, "rkv_evict_select: max_blocks_per_seq too large");
  if (num_seqs == 0 || n_layers == 0) return RKV_OK;
  if (!keep || !new_lens || !ctx_lens || (max_blocks_per_seq > 0 && (!weights || !block_tables)))
    return fail(RKV_ERR_INVALID_ARG, "rkv_evict_select: null pointer argument");
  if (!aligned16(weights) || (n_layers > 1 && (weights_layer_stride & 3)))
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_evict_select: weights must be 16-byte aligned, its layer stride a multiple of 4");
  const int table = max_blocks_per_seq * kBS;
  const int cap = max_context < table ? max_context : table;
  const dim3 grid((unsigned)num_kv_heads, (unsigned)num_seqs, (unsigned)n_layers);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define RKV_SELECT(NT, K)                                                                      \
  evict_select_kernel<NT, K><<<grid, NT, K ? (size_t)(cap + 3) / 4 * 16 : 0, s>>>(             \
      keep, new_lens, weights, weights_layer_stride, block_tables, max_blocks_per_seq, ctx_lens, \
      num_kv_heads, num_blocks, budget, sinks, recent, cap)
  // Threads: where the workgroups leave CUs idle each runs wide, where several share a
  // CU fewer threads wait for each other's barriers.  us with 256 / 512 / 1,024 threads:
  //   128 workgroups, 700 positions 5.1 / 5.0 / 6.0; 2,000 7.2 / 6.0 / 7.3; 4,000 9.8 /
  //   7.6 / 7.8; 8,000 16.5 / 10.8 / 10.0; 32,000 61 / 35 / 26
  //   1,024 workgroups, 2,000 9.2 / 10.7 / 21.8; 4,000 15.0 / 16.6 / 26.0; 8,000 36.6 /
  //   26.8 / 35.9; 16,000 68 / 48 / 58; 32,000 232 / 133 / 99
  const bool crowded = (int64_t)num_kv_heads * num_seqs * n_layers > 512;
  const int narrow = crowded ? 4096 : 1024;
  if (cap <= narrow) RKV_SELECT(256, true);
  else if (cap <= 4 * narrow) RKV_SELECT(512, true);
  else if (cap <= kKeysMax) RKV_SELECT(1024, true);
  else RKV_SELECT(1024, false);
#undef RKV_SELECT
  return check_launch("rkv_evict_select");
}

extern "C" int rkv_evict_compact(void* k_pool, void* v_pool, float* k_scale, float* v_scale,
                                 float* weights, int64_t pool_layer_stride,
                                 int64_t weights_layer_stride, const int32_t* keep,
                                 const int32_t* new_lens, int budget, const int32_t* src_tables,
                                 int src_blocks_per_seq, const int32_t* dst_tables,
                                 int dst_blocks_per_seq, int num_seqs, int n_layers,
                                 int num_kv_heads, int head_dim, int block_size,
                                 int64_t num_blocks, int dtype, void* stream) {
  clear_error();
  if (num_seqs < 0 || n_layers < 0 || num_kv_heads <= 0 || num_blocks < 0 || budget <= 0 ||
      src_blocks_per_seq < 0 || dst_blocks_per_seq < 0)
    return fail(RKV_ERR_INVALID_ARG, "rkv_evict_compact: bad size argument");
  if (dtype < RKV_F32 || dtype > RKV_FP8_BLOCK)
    return fail(RKV_ERR_INVALID_ARG, "rkv_evict_compact: unknown dtype");
  const bool q8 = dtype >= RKV_I8;
  if (block_size != kBS)
    return fail(RKV_ERR_UNSUPPORTED, "rkv_evict_compact: block_size must be 16");
  if (q8 ? head_dim != 32 && head_dim != 64 && head_dim != 128 : head_dim <= 0 || head_dim % 8)
    return fail(RKV_ERR_UNSUPPORTED,
                "rkv_evict_compact: head_dim must be a multiple of 8 (1-byte pools: 32, 64, 128)");
  if (num_seqs > 65535 || n_layers > 65535)
    return fail(RKV_ERR_INVALID_ARG, "rkv_evict_compact: num_seqs and n_layers must be <= 65535");
  if ((int64_t)src_blocks_per_seq * kBS > 0x7fffff00)
    return fail(RKV_ERR_INVALID_ARG, "rkv_evict_compact: src_blocks_per_seq too large");
  if (num_seqs == 0 || n_layers == 0 || src_blocks_per_seq == 0 || dst_blocks_per_seq == 0)
    return RKV_OK;
  if (!k_pool || !v_pool || !keep || !new_lens || !src_tables || !dst_tables ||
      (q8 && (!k_scale || !v_scale)))
    return fail(RKV_ERR_INVALID_ARG, "rkv_evict_compact: null pointer argument");
  if (!aligned16(k_pool) || !aligned16(v_pool))
    return fail(RKV_ERR_INVALID_ARG, "rkv_evict_compact: pools must be 16-byte aligned");
  const int elem = dtype == RKV_F32 ? 4 : dtype == RKV_BF16 ? 2 : 1;
  const int64_t row_bytes = (int64_t)head_dim * elem;
  const int64_t layer_bytes = n_layers > 1 ? pool_layer_stride * elem : 0;
  if (layer_bytes % 16)
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_evict_compact: a layer must start on a multiple of 16 bytes");
  const int64_t per_scale = dtype == RKV_I8 || dtype == RKV_FP8 ? head_dim : kBS * head_dim;
  const int64_t scale_ls = n_layers > 1 && q8 ? pool_layer_stride / per_scale : 0;
  if (n_layers > 1 && q8 && pool_layer_stride % per_scale)
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_evict_compact: pool_layer_stride must be a whole number of scales");
  int64_t blocks = (budget + (int64_t)kBS - 1) / kBS;
  if (blocks > dst_blocks_per_seq) blocks = dst_blocks_per_seq;
  const int64_t wgs = (blocks * num_kv_heads + 3) / 4;
  if (wgs > 0x7fffffff)
    return fail(RKV_ERR_INVALID_ARG, "rkv_evict_compact: budget too large for one launch");
  const dim3 grid((unsigned)wgs, (unsigned)num_seqs, (unsigned)n_layers);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int upr = (int)(row_bytes / 16);
#define RKV_COMPACT(T, U)                                                                      \
  evict_compact_kernel<T, U><<<grid, 256, 0, s>>>(                                             \
      static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool), k_scale, v_scale, weights, \
      layer_bytes, scale_ls, weights_layer_stride, keep, new_lens, budget, src_tables,         \
      src_blocks_per_seq, dst_tables, dst_blocks_per_seq, num_kv_heads, upr, num_blocks)
#define RKV_COMPACT_Q(T)                   \
  do {                                     \
    if (upr == 2) RKV_COMPACT(T, 2);       \
    else if (upr == 4) RKV_COMPACT(T, 4);  \
    else RKV_COMPACT(T, 8);                \
  } while (0)
  switch (dtype) {
    case RKV_F32:
    case RKV_BF16:  // rows of bytes: the element type does not matter
      if (upr == 4) RKV_COMPACT(RKV_F32, 4);
      else if (upr == 8) RKV_COMPACT(RKV_F32, 8);
      else if (upr == 16) RKV_COMPACT(RKV_F32, 16);
      else if (upr == 32) RKV_COMPACT(RKV_F32, 32);
      else RKV_COMPACT(RKV_F32, 0);
      break;
    case RKV_I8:
    case RKV_FP8: RKV_COMPACT_Q(RKV_I8); break;
    case RKV_I8_BLOCK: RKV_COMPACT_Q(RKV_I8_BLOCK); break;
    default: RKV_COMPACT_Q(RKV_FP8_BLOCK); break;
  }
#undef RKV_COMPACT_Q
#undef RKV_COMPACT
  return check_launch("rkv_evict_compact");
}
