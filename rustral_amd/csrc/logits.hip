// logits.hip -- penalties, biases and masks on logits with the greedy pick
// (rkv_process_logits, include/rustral_model.h).
//
// A workgroup owns kSlice columns of one row.  It requests its logits, counts
// the row's history and finds the row's biases that fall in the slice in LDS
// (integer atomics: a count, and the largest entry index of a bias, do not
// depend on their order), then makes one pass over its columns and keeps its
// best (value, index).  A row's slices meet in a second small launch, which only
// a pick needs.  Bound by the read and write of the logits for large batches,
// by the two launches for single rows.  us for 1 x 32,000 / 64 x 128,256 columns
// (histories of 300 / 2,048 at most) by columns and threads a workgroup: 4,096 with
// 512 7.6 / 22.3 (with the mask and the history requested only after the first barrier
// 7.8 / 22.8); 2,048 with 256 7.4 / 23.2; 8,192 with 1,024 8.4 / 23.1.  With streaming
// stores 7.7 / 21.3; streaming loads as well 22.9 (a caller's logits are often cached).
// One workgroup of 1,024 threads for a whole row (no second launch): 1 x 5,000 6.9 for
// 7.6, 1 x 16,384 9.7 for 7.7, 1 x 32,000 15.0 for 7.7: not for a vocabulary's length.
#include "../../include/rustral_model.h"
#include "common.hpp"

#include <cmath>

namespace rkv {
namespace {

constexpr int kSlice = 4096;  // columns a workgroup
constexpr int kThreads = 512;
// History ids a thread has in flight: us with 1 / 4 / 8 / 16 for 1 x 32,000 (history 300)
// 7.8 / 8.0 / 8.2 / 8.8, for 64 x 128,256 (up to 2,048) 23.8 / 22.8 / 23.3 / 23.9.
constexpr int kAhead = 4;
constexpr uint32_t kPrompt = 0x80000000u;  // the token stands in the prompt

struct Best {
  float v;
  int i;
};

// The better of two: the larger value, the later index among equals; an index
// of -1 stands for a row (part) with nothing but -infinity.
__device__ __forceinline__ Best better(Best a, Best b) {
  return b.v > a.v || (b.v == a.v && b.i > a.i) ? b : a;
}

__device__ __forceinline__ Best wave_best(Best x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x = better(x, Best{__shfl_xor(x.v, o), __shfl_xor(x.i, o)});
  return x;
}

struct LogitsArgs {
  float* out;
  int64_t out_stride;
  const float* logits;
  int64_t row_stride;
  int n;
  const int32_t *history, *history_start, *prompt_lens;
  const float *repetition, *frequency, *presence;
  const int32_t* bias_ids;
  const float* bias;
  const int32_t* bias_start;
  const int32_t* allowed;
  int64_t allowed_stride;
  int32_t* pick;   // written here when the row is one slice
  Best* part;      // else [rows][slices]
};

// VEC: columns a load (4 where the rows are 16-byte aligned, else 1).
template <int VEC>
__global__ __launch_bounds__(kThreads) void process_logits_kernel(LogitsArgs p) {
  constexpr int NL = kSlice / (kThreads * VEC);
  __shared__ __align__(16) uint32_t s_count[kSlice];
  __shared__ __align__(16) uint32_t s_bias[kSlice];
  __shared__ Best s_best[kThreads / 64];
  const int r = blockIdx.y, tid = threadIdx.x;
  const int c0 = blockIdx.x * kSlice;
  const int cols = p.n - c0 < kSlice ? p.n - c0 : kSlice;
  const float* x = p.logits + (int64_t)r * p.row_stride + c0;
  float v[NL][VEC];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int c = VEC * (tid + kThreads * i);
    if constexpr (VEC == 4) {
      if (c + 3 < cols) {
        const float4 f = *reinterpret_cast<const float4*>(x + c);
        v[i][0] = f.x, v[i][1] = f.y, v[i][2] = f.z, v[i][3] = f.w;
        continue;
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[i][e] = c + e < cols ? x[c + e] : 0.0f;
  }
  // Everything that does not wait for the LDS counters is requested before the first
  // barrier: the mask's words and the first of the history and of the biases.
  const uint32_t* mask = p.allowed ? reinterpret_cast<const uint32_t*>(p.allowed) +
                                         (int64_t)r * p.allowed_stride
                                   : nullptr;
  uint32_t bits[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    // c0 and c are multiples of VEC: one word of the mask holds all VEC bits
    const int c = VEC * (tid + kThreads * i);
    bits[i] = mask && c < cols ? mask[(c0 + c) >> 5] >> ((c0 + c) & 31) : 0xffffffffu;
  }
  const bool counts = p.repetition || p.frequency || p.presence;
  const int h0 = counts ? p.history_start[r] : 0, h1 = counts ? p.history_start[r + 1] : 0;
  const int made = h0 + (counts && p.prompt_lens ? p.prompt_lens[r] : 0);
  const int b0 = p.bias_ids ? p.bias_start[r] : 0, b1 = p.bias_ids ? p.bias_start[r + 1] : 0;
  const float rep = p.repetition ? p.repetition[r] : 1.0f;
  const float freq = p.frequency ? p.frequency[r] : 0.0f;
  const float pres = p.presence ? p.presence[r] : 0.0f;
  const bool use_h = h1 > h0, use_b = b1 > b0;  // workgroup-uniform
  if (use_h || use_b) {
    // kAhead ids a thread requested together: a row's history is read by every
    // slice, and one id at a time each wait is a round trip
    int id[kAhead];
    auto ids = [&](int at) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = at + tid + kThreads * u;
        id[u] = i < h1 ? p.history[i] : -1;
      }
    };
    ids(h0);
    int bias_id = b0 + tid < b1 ? p.bias_ids[b0 + tid] : -1;
    for (int i = tid; i < kSlice / 4; i += kThreads) {
      if (use_h) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0u, 0u, 0u, 0u);
      if (use_b) reinterpret_cast<uint4*>(s_bias)[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __syncthreads();
    for (int at = h0; at < h1; at += kAhead * kThreads) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (id[u] >= c0 && id[u] - c0 < cols) {
          if (at + tid + kThreads * u < made) atomicOr(&s_count[id[u] - c0], kPrompt);
          else atomicAdd(&s_count[id[u] - c0], 1u);
        }
      }
      if (at + kAhead * kThreads < h1) ids(at + kAhead * kThreads);
    }
    for (int i = b0 + tid; i < b1; i += kThreads) {
      if (bias_id >= c0 && bias_id - c0 < cols)
        atomicMax(&s_bias[bias_id - c0], (uint32_t)(i - b0) + 1u);
      bias_id = i + kThreads < b1 ? p.bias_ids[i + kThreads] : -1;
    }
    __syncthreads();
  }
  float* out = p.out ? p.out + (int64_t)r * p.out_stride + c0 : nullptr;
  Best best{-INFINITY, -1};
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int c = VEC * (tid + kThreads * i);
    if (c >= cols) continue;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (c + e >= cols) continue;
      float y = v[i][e];
      if (use_h) {
        const uint32_t n = s_count[c + e];
        if (n) {
          y = y > 0.0f ? y / rep : y * rep;
          const uint32_t times = n & ~kPrompt;
          if (times) y -= fmaf(freq, (float)times, pres);
        }
      }
      if (use_b) {
        const uint32_t at = s_bias[c + e];
        if (at) y += p.bias[b0 + (int)at - 1];
      }
      y = (bits[i] >> e) & 1u ? y : -INFINITY;
      v[i][e] = y;
      if (y > -INFINITY) best = better(best, Best{y, c0 + c + e});  // a NaN is not
    }
    if (out) {
      if constexpr (VEC == 4) {
        if (c + 3 < cols) {
          store_stream(out + c, __builtin_bit_cast(uint4, make_float4(v[i][0], v[i][1], v[i][2],
                                                                      v[i][3])));
          continue;
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (c + e < cols) out[c + e] = v[i][e];
    }
  }
  if (!p.pick) return;
  best = wave_best(best);
  if ((tid & 63) == 0) s_best[tid >> 6] = best;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) best = better(best, s_best[w]);
    if (gridDim.x == 1) p.pick[r] = best.i;
    else p.part[(int64_t)r * gridDim.x + blockIdx.x] = best;
  }
}

// One wave a row: the best of its slices.
__global__ __launch_bounds__(64) void pick_kernel(int32_t* __restrict__ pick,
                                                  const Best* __restrict__ part, int slices) {
  const int r = blockIdx.x;
  Best best{-INFINITY, -1};
  for (int i = threadIdx.x; i < slices; i += 64)
    best = better(best, part[(int64_t)r * slices + i]);
  best = wave_best(best);
  if (threadIdx.x == 0) pick[r] = best.i;
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" size_t rkv_process_logits_workspace_bytes(int rows, int n) {
  if (rows <= 0 || n <= kSlice) return 0;
  return (size_t)rows * (((size_t)n + kSlice - 1) / kSlice) * sizeof(Best);
}

extern "C" int rkv_process_logits(float* out, int64_t out_stride, int32_t* pick,
                                  const float* logits, int64_t row_stride, int rows, int n,
                                  const int32_t* history, const int32_t* history_start,
                                  const int32_t* prompt_lens, const float* repetition,
                                  const float* frequency, const float* presence,
                                  const int32_t* bias_ids, const float* bias,
                                  const int32_t* bias_start, const int32_t* allowed,
                                  int64_t allowed_stride, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  clear_error();
  if (rows < 0 || n <= 0 || rows > 65535)
    return fail(RKV_ERR_INVALID_ARG, "rkv_process_logits: bad size argument");
  if (n > 0x7fffffff - kSlice) return fail(RKV_ERR_INVALID_ARG, "rkv_process_logits: n too large");
  if (rows == 0) return RKV_OK;
  if (!logits || (!out && !pick))
    return fail(RKV_ERR_INVALID_ARG, "rkv_process_logits: null pointer argument");
  if ((repetition || frequency || presence) && (!history || !history_start))
    return fail(RKV_ERR_INVALID_ARG, "rkv_process_logits: penalties need the history");
  if (bias_ids && (!bias || !bias_start))
    return fail(RKV_ERR_INVALID_ARG, "rkv_process_logits: bias_ids needs bias and bias_start");
  if (row_stride < n || (out && out_stride < n) ||
      (allowed && allowed_stride < (n + (int64_t)31) / 32))
    return fail(RKV_ERR_INVALID_ARG, "rkv_process_logits: a stride is shorter than its row");
  if (out == logits && out_stride != row_stride)
    return fail(RKV_ERR_INVALID_ARG, "rkv_process_logits: in place, both sides need the same stride");
  const int slices = (n + kSlice - 1) / kSlice;
  const size_t need = pick ? rkv_process_logits_workspace_bytes(rows, n) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(RKV_ERR_WORKSPACE,
                "rkv_process_logits: workspace missing or smaller than "
                "rkv_process_logits_workspace_bytes()");
  if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 7u))
    return fail(RKV_ERR_INVALID_ARG, "rkv_process_logits: workspace must be 8-byte aligned");
  LogitsArgs a{out, out_stride, logits, row_stride, n, history, history_start, prompt_lens,
               repetition, frequency, presence, bias_ids, bias, bias_start, allowed,
               allowed_stride, pick, static_cast<Best*>(workspace)};
  const dim3 grid((unsigned)slices, (unsigned)rows);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool wide = aligned16(logits) && row_stride % 4 == 0 &&
                    (!out || (aligned16(out) && out_stride % 4 == 0));
  if (wide) process_logits_kernel<4><<<grid, kThreads, 0, s>>>(a);
  else process_logits_kernel<1><<<grid, kThreads, 0, s>>>(a);
  if (int rc = check_launch("rkv_process_logits")) return rc;
  if (pick && slices > 1) {
    pick_kernel<<<(unsigned)rows, 64, 0, s>>>(pick, a.part, slices);
    return check_launch("rkv_process_logits: pick");
  }
  return RKV_OK;
}
