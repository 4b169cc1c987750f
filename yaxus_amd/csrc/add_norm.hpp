// The seam between two blocks of a model: residual addition and RMSNorms of rows, on MI355X:
//   u = norm(x; post_w, post_offset) or x,  h' = h + u or u,  out = norm(h'; w, offset),
//   norm(v; w, o)_i = v_i / sqrt(mean v^2 + eps) * (o + w_i)
// (all f32). h_out and out may each be x or h itself: a thread writes only columns that it
// alone reads.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace yx {

struct AddNorm {
  const float* x;
  const float* post_w;  // null: u = x
  const float* h;       // null: h' = u
  float* h_out;         // null: not stored
  const float* w;       // null: no out
  float* out;
  float post_offset, offset, eps;
};

static constexpr int kNormThreads = 256;

// The workgroup's sum of v, to all its threads.
__device__ __forceinline__ float norm_sum(float v, float* ws) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = v;
  __syncthreads();
  return (ws[0] + ws[1]) + (ws[2] + ws[3]);
}

// One workgroup per row.
__global__ __launch_bounds__(kNormThreads) void add_norm_rows(AddNorm a, uint32_t cols) {
  __shared__ float ws[kNormThreads / 64];
  const size_t base = static_cast<size_t>(blockIdx.x) * cols;
  float ru = 1.0f, sum = 0.0f;
  if (a.post_w) {
    for (uint32_t i = threadIdx.x; i < cols; i += kNormThreads) sum = fmaf(a.x[base + i], a.x[base + i], sum);
    ru = 1.0f / sqrtf(norm_sum(sum, ws) / static_cast<float>(cols) + a.eps);
  }
  const auto stream = [&](uint32_t i) {
    float v = a.x[base + i];
    if (a.post_w) v = v * ru * (a.post_offset + a.post_w[i]);
    return a.h ? a.h[base + i] + v : v;
  };
  sum = 0.0f;
  for (uint32_t i = threadIdx.x; i < cols; i += kNormThreads) {
    const float v = stream(i);
    sum = fmaf(v, v, sum);
    if (!a.w) a.h_out[base + i] = v;
  }
  if (!a.w) return;
  const float r = 1.0f / sqrtf(norm_sum(sum, ws) / static_cast<float>(cols) + a.eps);
  for (uint32_t i = threadIdx.x; i < cols; i += kNormThreads) {
    const float v = stream(i);
    if (a.h_out) a.h_out[base + i] = v;
    a.out[base + i] = v * r * (a.offset + a.w[i]);
  }
}

}  // namespace yx
