// rope.hip -- rotary positions for gfx950: rotation of q / k rows, alone
// (rkv_rope) and fused with the KV append (rkv_rope_append), and the
// frequency tables of the usual long-context scalings (host).
//
// Pair i < rotary_dim / 2 of a row at position p turns by the angle p f_i:
//   y0 = g (x0 cos - x1 sin),  y1 = g (x1 cos + x0 sin)
// with (x0, x1) = elements (i, i + rotary_dim / 2) or, interleaved, (2 i,
// 2 i + 1); elements from rotary_dim on pass unchanged.
//
// The angle is formed in 64 bits as turns, p f / (2 pi), and reduced to its
// fraction before it is rounded to 32: in 32 bits the product alone is off by
// p f 2^-24 rad, 0.06 rad at a million positions.  A float fraction of a turn
// in [-1/2, 1/2] is off by 2^-26 turns at most, 1e-7 rad.
//
// Every element is read and written once, a lane's in 16-byte pieces.  Bound by HBM for
// a prompt: 8,192 tokens of 32 query and 8 KV heads of 128 into a bf16 pool 69 us (368
// MB, 5.3 TB/s; a copy reaches 5.1), 16,384 x 16 half-rotated heads of 64 alone 27 us (4.9 TB/s);
// by its launch for a decode step: 64 tokens 3.9 us.
#include "common.hpp"

#include <cmath>

namespace rkv {
namespace {

constexpr double kTurnsPerRad = 0.15915494309189535;  // 1 / (2 pi)

// Where the four pairs a lane owns sit in its row, and how it reads them.  A
// row of D elements belongs to D / 8 lanes; lane c owns pairs 4 c .. 4 c + 3 of
// the D / 2 "pairs" (the rotated ones first, then the unrotated elements two at
// a time).
//   kHalf:   half layout, rotary_dim a multiple of 8: two 16-byte pieces.
//   kPairs:  interleaved: 8 consecutive elements, two 16-byte pieces.
//   kSingle: half layout with another rotary_dim: one element at a time (the
//            second elements of the pairs start off a 16-byte boundary).
enum Layout { kHalf, kPairs, kSingle };

struct RopeRows {
  const float* x;          // [n_tokens] rows of `heads` heads
  int64_t tok_stride, head_stride;
  int heads;
};

// The fused append's pools; a row is its head's D elements in the pool's format
// (bytes as rkv_append_q forms them).
struct RopePool {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  const int64_t* slots;
  int64_t num_slots;
  int block_size;
};

// cos and sin of the lane's four pairs, times g.
__device__ __forceinline__ void turn(const double* __restrict__ inv_freq, int c, int half,
                                     double pos, float g, float (&co)[4], float (&si)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int i = 4 * c + e;
    co[e] = 1.0f;
    si[e] = 0.0f;
    if (i < half) {
      const double t = pos * (inv_freq[i] * kTurnsPerRad);
      const float frac = (float)(t - rint(t));
      float s, cs;
      sincospif(2.0f * frac, &s, &cs);
      co[e] = cs * g;
      si[e] = s * g;
    }
  }
}

// The lane's pairs of a row as a[e] (first elements) and b[e] (second).
template <Layout LAY>
__device__ __forceinline__ void load_pairs(const float* row, int c, int half, float (&a)[4],
                                           float (&b)[4]) {
  if constexpr (LAY == kPairs) {
    const float4 u = *reinterpret_cast<const float4*>(row + 8 * c);
    const float4 v = *reinterpret_cast<const float4*>(row + 8 * c + 4);
    a[0] = u.x, b[0] = u.y, a[1] = u.z, b[1] = u.w;
    a[2] = v.x, b[2] = v.y, a[3] = v.z, b[3] = v.w;
  } else if constexpr (LAY == kHalf) {
    const bool turned = 4 * c < half;  // half % 4 == 0: all four pairs or none
    const int i = turned ? 4 * c : 8 * c, j = turned ? i + half : i + 4;
    const float4 u = *reinterpret_cast<const float4*>(row + i);
    const float4 v = *reinterpret_cast<const float4*>(row + j);
    a[0] = u.x, a[1] = u.y, a[2] = u.z, a[3] = u.w;
    b[0] = v.x, b[1] = v.y, b[2] = v.z, b[3] = v.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 4 * c + e;
      a[e] = row[i < half ? i : 2 * i];
      b[e] = row[i < half ? i + half : 2 * i + 1];
    }
  }
}

// Elements e .. e + 3 of the lane's first piece (q = 0) or second (q = 1), as
// they lie in memory for the 16-byte layouts.
template <Layout LAY>
__device__ __forceinline__ void piece(const float (&a)[4], const float (&b)[4], int q,
                                      float (&o)[4]) {
  if constexpr (LAY == kPairs) {
    o[0] = q ? a[2] : a[0], o[1] = q ? b[2] : b[0];
    o[2] = q ? a[3] : a[1], o[3] = q ? b[3] : b[1];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = q ? b[e] : a[e];
  }
}

template <Layout LAY>
__device__ __forceinline__ int piece_at(int c, int half, int q) {
  if constexpr (LAY == kPairs) return 8 * c + 4 * q;
  const bool turned = 4 * c < half;
  return turned ? 4 * c + (q ? half : 0) : 8 * c + 4 * q;
}

template <Layout LAY>
__device__ __forceinline__ void store_pairs(float* row, int c, int half, const float (&a)[4],
                                            const float (&b)[4]) {
  if constexpr (LAY == kSingle) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 4 * c + e;
      row[i < half ? i : 2 * i] = a[e];
      row[i < half ? i + half : 2 * i + 1] = b[e];
    }
  } else {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float o[4];
      piece<LAY>(a, b, q, o);
      *reinterpret_cast<float4*>(row + piece_at<LAY>(c, half, q)) =
          make_float4(o[0], o[1], o[2], o[3]);
    }
  }
}

// Pairs past `half` are left alone (a select: an infinity there times a zero
// sine would be a NaN).
__device__ __forceinline__ void rotate4(float (&a)[4], float (&b)[4], int c, int half,
                                        const float (&co)[4], const float (&si)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x0 = a[e], x1 = b[e];
    const bool turned = 4 * c + e < half;
    a[e] = turned ? fmaf(x0, co[e], -(x1 * si[e])) : x0;
    b[e] = turned ? fmaf(x1, co[e], x0 * si[e]) : x1;
  }
}

// rkv_rope: grid (n_tokens, row splits), lpr = D / 8 lanes a row; the workgroup
// is a whole number of rows wide, so a thread keeps its place in the row and
// takes its sines once for all its rows.  out may be x (a thread reads what it
// writes, and nobody else does).
template <Layout LAY>
__global__ __launch_bounds__(256) void rope_kernel(float* out, int64_t out_tok_stride,
                                                   int64_t out_head_stride, RopeRows in,
                                                   const int32_t* __restrict__ positions,
                                                   const double* __restrict__ inv_freq, int lpr,
                                                   int half, float g) {
  const int64_t t = blockIdx.x;
  const int rows_wg = blockDim.x / lpr;
  const int r0 = threadIdx.x / lpr, c = threadIdx.x - r0 * lpr;
  float co[4], si[4];
  turn(inv_freq, c, half, (double)positions[t], g, co, si);
  for (int h = blockIdx.y * rows_wg + r0; h < in.heads; h += gridDim.y * rows_wg) {
    float a[4], b[4];
    load_pairs<LAY>(in.x + t * in.tok_stride + h * in.head_stride, c, half, a, b);
    rotate4(a, b, c, half, co, si);
    store_pairs<LAY>(out + t * out_tok_stride + h * out_head_stride, c, half, a, b);
  }
}

// Stores one row into a pool in its format (amax over the row's lanes for the
// 1-byte ones, every lane of the group present).
template <Layout LAY, int DT, int LPR>
__device__ __forceinline__ void store_row(void* pool, float* scale, int64_t row, int D, int c,
                                          int half, const float (&a)[4], const float (&b)[4]) {
  if constexpr (DT == RKV_F32) {
    store_pairs<LAY>(static_cast<float*>(pool) + row * D, c, half, a, b);
  } else if constexpr (DT == RKV_BF16) {
    uint16_t* p = static_cast<uint16_t*>(pool) + row * D;
    if constexpr (LAY == kSingle) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * c + e;
        p[i < half ? i : 2 * i] = (uint16_t)bf16_rne(a[e]);
        p[i < half ? i + half : 2 * i + 1] = (uint16_t)bf16_rne(b[e]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float o[4];
        piece<LAY>(a, b, q, o);
        *reinterpret_cast<uint2*>(p + piece_at<LAY>(c, half, q)) =
            make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
      }
    }
  } else {
    constexpr float kTop = DT == RKV_I8 ? 127.0f : 448.0f;
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) m = fmaxf(m, fmaxf(fabsf(a[e]), fabsf(b[e])));
    m = group_max<LPR>(m);
    const float inv = m > 0.0f ? kTop / m : 0.0f;
    auto byte = [&](float x) -> uint32_t {
      return DT == RKV_I8 ? i8_quant(x, inv) : e4m3_from_f32(x * inv);
    };
    uint8_t* p = static_cast<uint8_t*>(pool) + row * D;
    if constexpr (LAY == kSingle) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * c + e;
        p[i < half ? i : 2 * i] = (uint8_t)byte(a[e]);
        p[i < half ? i + half : 2 * i + 1] = (uint8_t)byte(b[e]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float o[4];
        piece<LAY>(a, b, q, o);
        *reinterpret_cast<uint32_t*>(p + piece_at<LAY>(c, half, q)) =
            byte(o[0]) | byte(o[1]) << 8 | byte(o[2]) << 16 | byte(o[3]) << 24;
      }
    }
    if (c == 0) scale[row] = m / kTop;
  }
}

// rkv_rope_append: grid (n_tokens, row splits); rows 0 .. Hq - 1 of a token are
// its query heads (rotated into q_out), the next Hkv its keys (rotated into the
// pool), the last Hkv its values (into the pool as they are).  LPR > 0 is D / 8
// for the 1-byte formats, whose row maximum needs it; 0 takes it from D.
template <Layout LAY, int DT, int LPR>
__global__ __launch_bounds__(256) void rope_append_kernel(
    float* q_out, int64_t out_tok_stride, int64_t out_head_stride, RopeRows q, RopeRows k,
    RopeRows v, RopePool pool, const int32_t* __restrict__ positions,
    const double* __restrict__ inv_freq, int D, int half, float g) {
  const int64_t t = blockIdx.x;
  const int lpr = LPR ? LPR : D / 8;
  const int rows_wg = blockDim.x / lpr;
  const int r0 = threadIdx.x / lpr, c = threadIdx.x - r0 * lpr;
  const int64_t slot = pool.slots[t];
  const bool on = slot >= 0 && slot < pool.num_slots;
  const int64_t blk = on ? slot / pool.block_size : 0;
  const int64_t in_blk = slot - blk * pool.block_size;
  const int n_rows = q.heads + 2 * k.heads;
  float co[4], si[4];
  turn(inv_freq, c, half, (double)positions[t], g, co, si);
  for (int r = blockIdx.y * rows_wg + r0; r < n_rows; r += gridDim.y * rows_wg) {
    float a[4], b[4];
    if (r < q.heads) {
      load_pairs<LAY>(q.x + t * q.tok_stride + r * q.head_stride, c, half, a, b);
      rotate4(a, b, c, half, co, si);
      store_pairs<LAY>(q_out + t * out_tok_stride + r * out_head_stride, c, half, a, b);
      continue;
    }
    if (!on) continue;  // padding or out-of-range slot
    const bool is_k = r < q.heads + k.heads;
    const int h = r - q.heads - (is_k ? 0 : k.heads);
    const RopeRows& src = is_k ? k : v;
    load_pairs<LAY>(src.x + t * src.tok_stride + h * src.head_stride, c, half, a, b);
    if (is_k) rotate4(a, b, c, half, co, si);
    const int64_t row = (blk * k.heads + h) * pool.block_size + in_blk;
    store_row<LAY, DT, LPR>(is_k ? pool.k : pool.v, is_k ? pool.k_scale : pool.v_scale, row, D, c,
                            half, a, b);
  }
}

int check_rope(const char* who, int64_t n_tokens, int num_heads, int head_dim, int rotary_dim) {
  const auto bad = [&](int rc, const char* what) { return fail(rc, std::string(who) + what); };
  if (n_tokens < 0 || num_heads <= 0)
    return bad(RKV_ERR_INVALID_ARG, ": n_tokens must be >= 0 and the head counts > 0");
  if (n_tokens > 0x7fffffff)
    return bad(RKV_ERR_INVALID_ARG, ": n_tokens too large for one launch");
  if (head_dim <= 0 || head_dim % 8 || head_dim > 1024)
    return bad(RKV_ERR_UNSUPPORTED, ": head_dim must be a multiple of 8 up to 1024");
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim)
    return bad(RKV_ERR_INVALID_ARG, ": rotary_dim must be even, > 0 and <= head_dim");
  return RKV_OK;
}

Layout layout_of(int interleaved, int rotary_dim) {
  return interleaved ? kPairs : rotary_dim % 8 == 0 ? kHalf : kSingle;
}

// Threads of a workgroup (whole rows) and workgroups a token's rows are split
// over: one row a thread while that leaves fewer workgroups than kFill, so that
// a decode step's few tokens spread over the chip; then every row of a token in
// one workgroup, which takes the sines once.  us for 64 tokens of 32 + 2 x 8 rows of 128:
// split 3.9, one workgroup a token 4.3; for 8,192 tokens: split three ways 70.3, one
// workgroup 69.1.
constexpr int64_t kFill = 2048;
void shape_of(int64_t n_tokens, int rows, int lpr, unsigned& threads, unsigned& splits) {
  const int most = 256 / lpr;
  const int rows_wg = rows < most ? rows : most;
  threads = (unsigned)(rows_wg * lpr);
  const int64_t all = (rows + rows_wg - 1) / rows_wg;
  int64_t s = n_tokens >= kFill ? 1 : (kFill + n_tokens - 1) / n_tokens;
  splits = (unsigned)(s < all ? s : all);
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_rope(float* out, const float* x, const int32_t* positions,
                        const double* inv_freq, int64_t n_tokens, int num_heads, int head_dim,
                        int rotary_dim, int64_t out_tok_stride, int64_t out_head_stride,
                        int64_t tok_stride, int64_t head_stride, int interleaved, float magnitude,
                        void* stream) {
  clear_error();
  if (int rc = check_rope("rkv_rope", n_tokens, num_heads, head_dim, rotary_dim)) return rc;
  if (n_tokens == 0) return RKV_OK;
  if (!out || !x || !positions || !inv_freq)
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope: null pointer argument");
  if ((out_tok_stride | out_head_stride | tok_stride | head_stride) & 3)
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope: strides must be multiples of 4 elements");
  if (!aligned16(out) || !aligned16(x))
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope: pointers must be 16-byte aligned");
  if (out == x && (out_tok_stride != tok_stride || out_head_stride != head_stride))
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope: in place, both sides need the same strides");
  const int lpr = head_dim / 8;
  unsigned threads, splits;
  shape_of(n_tokens, num_heads, lpr, threads, splits);
  const dim3 grid((unsigned)n_tokens, splits);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const RopeRows in{x, tok_stride, head_stride, num_heads};
#define RKV_ROPE(L)                                                                            \
  rope_kernel<L><<<grid, threads, 0, s>>>(out, out_tok_stride, out_head_stride, in, positions, \
                                          inv_freq, lpr, rotary_dim / 2, magnitude)
  switch (layout_of(interleaved, rotary_dim)) {
    case kHalf: RKV_ROPE(kHalf); break;
    case kPairs: RKV_ROPE(kPairs); break;
    default: RKV_ROPE(kSingle); break;
  }
#undef RKV_ROPE
  return check_launch("rkv_rope");
}

extern "C" int rkv_rope_append(float* q_out, void* k_pool, void* v_pool, float* k_scale,
                               float* v_scale, const float* q, const float* k_new,
                               const float* v_new, int64_t out_tok_stride,
                               int64_t out_head_stride, int64_t q_tok_stride,
                               int64_t q_head_stride, int64_t src_tok_stride,
                               int64_t src_head_stride, const int32_t* positions,
                               const double* inv_freq, const int64_t* slot_mapping,
                               int64_t n_tokens, int num_q_heads, int num_kv_heads, int head_dim,
                               int rotary_dim, int interleaved, float magnitude, int block_size,
                               int64_t num_blocks, int dtype, void* stream) {
  clear_error();
  if (int rc = check_rope("rkv_rope_append", n_tokens, num_q_heads, head_dim, rotary_dim))
    return rc;
  if (num_kv_heads <= 0 || block_size <= 0 || num_blocks < 0)
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope_append: num_kv_heads, block_size must be > 0");
  const bool q8 = dtype == RKV_I8 || dtype == RKV_FP8;
  if (dtype != RKV_F32 && dtype != RKV_BF16 && !q8)
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_rope_append: dtype must be RKV_F32, RKV_BF16, RKV_I8 or RKV_FP8");
  if (q8 && head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(RKV_ERR_UNSUPPORTED,
                "rkv_rope_append: 1-byte pools: head_dim must be 32, 64 or 128");
  if (n_tokens == 0) return RKV_OK;
  if (!q_out || !k_pool || !v_pool || !q || !k_new || !v_new || !positions || !inv_freq ||
      !slot_mapping || (q8 && (!k_scale || !v_scale)))
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope_append: null pointer argument");
  if ((out_tok_stride | out_head_stride | q_tok_stride | q_head_stride | src_tok_stride |
       src_head_stride) & 3)
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope_append: strides must be multiples of 4 elements");
  if (!aligned16(q_out) || !aligned16(q) || !aligned16(k_new) || !aligned16(v_new) ||
      !aligned16(k_pool) || !aligned16(v_pool))
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope_append: pointers must be 16-byte aligned");
  if (q_out == q && (out_tok_stride != q_tok_stride || out_head_stride != q_head_stride))
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope_append: in place, both sides need the same strides");
  const int lpr = head_dim / 8;
  unsigned threads, splits;
  shape_of(n_tokens, num_q_heads + 2 * num_kv_heads, lpr, threads, splits);
  const dim3 grid((unsigned)n_tokens, splits);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const RopeRows qr{q, q_tok_stride, q_head_stride, num_q_heads};
  const RopeRows kr{k_new, src_tok_stride, src_head_stride, num_kv_heads};
  const RopeRows vr{v_new, src_tok_stride, src_head_stride, num_kv_heads};
  const RopePool pool{k_pool, v_pool, k_scale, v_scale, slot_mapping, num_blocks * block_size,
                      block_size};
#define RKV_ROPE_L(L, T, P)                                                                  \
  rope_append_kernel<L, T, P><<<grid, threads, 0, s>>>(q_out, out_tok_stride, out_head_stride, \
                                                       qr, kr, vr, pool, positions, inv_freq,  \
                                                       head_dim, rotary_dim / 2, magnitude)
#define RKV_ROPE(T, P)                                    \
  do {                                                    \
    switch (layout_of(interleaved, rotary_dim)) {         \
      case kHalf: RKV_ROPE_L(kHalf, T, P); break;         \
      case kPairs: RKV_ROPE_L(kPairs, T, P); break;       \
      default: RKV_ROPE_L(kSingle, T, P); break;          \
    }                                                     \
  } while (0)
#define RKV_ROPE_Q(T)                      \
  do {                                     \
    if (head_dim == 32) RKV_ROPE(T, 4);    \
    else if (head_dim == 64) RKV_ROPE(T, 8); \
    else RKV_ROPE(T, 16);                  \
  } while (0)
  if (dtype == RKV_F32) RKV_ROPE(RKV_F32, 0);
  else if (dtype == RKV_BF16) RKV_ROPE(RKV_BF16, 0);
  else if (dtype == RKV_I8) RKV_ROPE_Q(RKV_I8);
  else RKV_ROPE_Q(RKV_FP8);
#undef RKV_ROPE_Q
#undef RKV_ROPE
#undef RKV_ROPE_L
  return check_launch("rkv_rope_append");
}

extern "C" int rkv_rope_frequencies(double* inv_freq, float* magnitude, int rotary_dim,
                                    double base, int scaling, double factor,
                                    int64_t original_context, double low, double high) {
  clear_error();
  const double kPi = 3.14159265358979323846;
  if (rotary_dim <= 0 || rotary_dim % 2 || !(base > 1.0))
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_rope_frequencies: rotary_dim must be even and > 0, base > 1");
  if (!inv_freq || !magnitude)
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope_frequencies: null pointer argument");
  if (scaling < RKV_ROPE_PLAIN || scaling > RKV_ROPE_BANDS)
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope_frequencies: unknown scaling");
  if (scaling != RKV_ROPE_PLAIN && !(factor >= 1.0 && std::isfinite(factor)))
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope_frequencies: factor must be >= 1");
  const bool parts = scaling == RKV_ROPE_PARTS || scaling == RKV_ROPE_BANDS;
  if (parts && (original_context <= 0 || !(low > 0.0) || !(high > low)))
    return fail(RKV_ERR_INVALID_ARG,
                "rkv_rope_frequencies: original_context > 0 and 0 < low < high are needed");
  if (scaling == RKV_ROPE_BASE && rotary_dim == 2)
    return fail(RKV_ERR_INVALID_ARG, "rkv_rope_frequencies: base scaling needs rotary_dim > 2");
  const int n = rotary_dim / 2;
  *magnitude = 1.0f;
  if (scaling == RKV_ROPE_BASE) base *= std::pow(factor, rotary_dim / (rotary_dim - 2.0));
  // the pair whose wave makes r turns within original_context
  const auto pair_of = [&](double r) {
    return rotary_dim * std::log(original_context / (r * 2.0 * kPi)) / (2.0 * std::log(base));
  };
  double first = 0.0, last = 0.0;
  if (scaling == RKV_ROPE_PARTS) {
    first = std::fmax(0.0, std::floor(pair_of(high)));
    last = std::fmin(rotary_dim - 1.0, std::ceil(pair_of(low)));
    if (last <= first) last = first + 0.001;
    *magnitude = (float)(0.1 * std::log(factor) + 1.0);
  }
  for (int i = 0; i < n; ++i) {
    const double f = std::pow(base, -2.0 * i / rotary_dim);
    double share = 1.0;  // of the unstretched frequency
    if (scaling == RKV_ROPE_LINEAR) {
      share = 0.0;
    } else if (scaling == RKV_ROPE_PARTS) {
      share = 1.0 - std::fmin(1.0, std::fmax(0.0, (i - first) / (last - first)));
    } else if (scaling == RKV_ROPE_BANDS) {
      const double turns = original_context * f / (2.0 * kPi);
      share = std::fmin(1.0, std::fmax(0.0, (turns - low) / (high - low)));
    }
    inv_freq[i] = share * f + (1.0 - share) * f / (parts || scaling == RKV_ROPE_LINEAR ? factor : 1.0);
  }
  return RKV_OK;
}
