// Log probabilities of given tokens, entropy and top alternatives of each row of logits, on
// MI355X. With M the row's maximum, S = sum e^(x-M) and U = sum (x-M) e^(x-M) (f32):
//   log p_i = (x_i - M) - log S,  H = log S - U / S.
// Alternatives: the largest logits, larger value first, then lower index; NaN and -inf are
// never one. A row with nothing above -inf has no distribution: -inf, entropy 0, no
// alternatives. A NaN or +inf makes S, so the row's log probabilities and entropy, NaN.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/yaxus_hip.h"
#include "step_after.hpp"

namespace yx {

static constexpr int kLpThreads = 256;

struct LogprobsOut {
  float* logprob;          // [rows][given] (null: none)
  float* entropy;          // [rows] (null: none)
  uint32_t* top_ids;       // [rows][top]
  float* top_logprobs;     // [rows][top]
};

// Key of a logit as a candidate: as argmax_key, and 0 (none) for -inf too.
__device__ __forceinline__ unsigned long long top_key(float v, uint32_t i) {
  return v > -INFINITY ? argmax_key(v, i) : 0ull;
}

// The value a key was made of (-0 comes back as +0).
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

// One workgroup per row: the sums in one pass, then a pass for each alternative.
__global__ __launch_bounds__(kLpThreads) void logprobs_rows(const float* __restrict__ logits, uint32_t cols,
                                                            size_t ld, const uint32_t* __restrict__ tokens,
                                                            uint32_t given, uint32_t top, LogprobsOut out) {
  __shared__ float ws[3][kLpThreads / 64];
  __shared__ unsigned long long wk[kLpThreads / 64];
  const uint32_t row = blockIdx.x;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const float* lr = logits + row * ld;
  float m = -INFINITY, s = 0.0f, u = 0.0f;
  for (uint32_t i = threadIdx.x; i < cols; i += kLpThreads) m = fmaxf(m, lr[i]);
  for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
  if (lane == 0) ws[0][wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(ws[0][0], ws[0][1]), fmaxf(ws[0][2], ws[0][3]));
  if (m == -INFINITY) m = 0.0f;
  for (uint32_t i = threadIdx.x; i < cols; i += kLpThreads) {
    const float d = lr[i] - m, e = __expf(d);
    s += e;
    u = fmaf(fmaxf(d, -200.0f), e, u);
  }
  for (int off = 32; off > 0; off >>= 1) {
    s += __shfl_xor(s, off);
    u += __shfl_xor(u, off);
  }
  if (lane == 0) {
    ws[1][wave] = s;
    ws[2][wave] = u;
  }
  __syncthreads();
  s = (ws[1][0] + ws[1][1]) + (ws[1][2] + ws[1][3]);
  u = (ws[2][0] + ws[2][1]) + (ws[2][2] + ws[2][3]);
  const float log_s = s == 0.0f ? 0.0f : logf(s);
  if (out.logprob)
    for (uint32_t i = threadIdx.x; i < given; i += kLpThreads) {
      const uint32_t tok = tokens[static_cast<size_t>(row) * given + i];
      out.logprob[static_cast<size_t>(row) * given + i] = (tok < cols ? lr[tok] - m : -INFINITY) - log_s;
    }
  if (out.entropy && threadIdx.x == 0) out.entropy[row] = s == 0.0f ? 0.0f : log_s - u / s;
  unsigned long long prev = ~0ull;
  for (uint32_t j = 0; j < top; ++j) {
    unsigned long long best = 0;
    for (uint32_t i = threadIdx.x; i < cols; i += kLpThreads) {
      const unsigned long long k = top_key(lr[i], i);
      if (k < prev && k > best) best = k;
    }
    for (int off = 32; off > 0; off >>= 1) {
      const unsigned long long o = __shfl_xor(best, off);
      best = o > best ? o : best;
    }
    __syncthreads();
    if (lane == 0) wk[wave] = best;
    __syncthreads();
    for (int wv = 0; wv < kLpThreads / 64; ++wv) best = wk[wv] > best ? wk[wv] : best;
    if (threadIdx.x == 0) {
      out.top_ids[static_cast<size_t>(row) * top + j] = best ? ~static_cast<uint32_t>(best) : YX_NO_TOKEN;
      out.top_logprobs[static_cast<size_t>(row) * top + j] = best ? (key_value(best) - m) - log_s : -INFINITY;
    }
    prev = best ? best : 1;  // 1: below every key
  }
}

}  // namespace yx
