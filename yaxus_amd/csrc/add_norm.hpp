// The seam between two blocks of a model: residual addition and RMSNorms of rows, on MI355X:
//   u = norm(x; post_w, post_offset) or x,  h' = h + u or u,  out = norm(h'; w, offset),
//   norm(v; w, o)_i = v_i / sqrt(mean v^2 + eps) * (o + w_i)
// (all f32; sums of squares f32 in a fixed order). Bound by reading x and h and writing h' and out
// once: rows of up to 16384 columns stay in a workgroup's registers between the sums and the
// stores; with few rows by the chain load, sum, sum, store, so the weights' loads go out with the
// rows'. h_out and out may each be x or h itself: a thread writes only columns that it alone
// reads, after it has read them.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "epilogue.hpp"

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

// The workgroup's sum of v (TH threads), to all of them. ws: TH / 64 floats.
template <int TH>
__device__ __forceinline__ float norm_sum(float v, float* ws) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = (ws[0] + ws[1]) + (ws[2] + ws[3]);
#pragma unroll
  for (int i = 4; i < TH / 64; i += 4) s += (ws[i] + ws[i + 1]) + (ws[i + 2] + ws[i + 3]);
  return s;
}

// Columns 4q .. 4q + 3 of a row whose length and address may be any.
__device__ __forceinline__ f32x4 norm_load(const float* p, uint32_t q, uint32_t cols) {
  if (4 * q + 4 <= cols) return reinterpret_cast<const f32x4_any*>(p)[q];
  f32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (4 * q + j < cols) v[j] = p[4 * q + j];
  return v;
}
__device__ __forceinline__ void norm_store(float* p, uint32_t q, uint32_t cols, const f32x4& v) {
  if (4 * q + 4 <= cols) {
    reinterpret_cast<f32x4_any*>(p)[q] = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (4 * q + j < cols) p[4 * q + j] = v[j];
}

// One workgroup of TH threads per row, V pieces of four columns per thread: at most 4 TH V columns.
// Eight pieces take 490 registers, one wave per SIMD; four in twice the threads: 2048 x 5000 85 -> 35
// us, 2048 x 8192 118 -> 53 (5.1 TB/s). 4096 x 2048 24 us (5.6 TB/s), 16 x 2048 4.0.
template <int TH, int V>
__global__ __launch_bounds__(TH) void add_norm_rows(AddNorm a, uint32_t cols) {
  __shared__ float ws[2][TH / 64];
  const size_t base = static_cast<size_t>(blockIdx.x) * cols;
  f32x4 x[V], h[V], pw[V], w[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint32_t q = i * TH + threadIdx.x;
    x[i] = h[i] = pw[i] = w[i] = f32x4{0, 0, 0, 0};
    if (4 * q >= cols) continue;
    x[i] = norm_load(a.x + base, q, cols);
    if (a.h) h[i] = norm_load(a.h + base, q, cols);
    if (a.post_w) pw[i] = norm_load(a.post_w, q, cols);
    if (a.w) w[i] = norm_load(a.w, q, cols);
  }
  const auto rms = [&](const f32x4 (&v)[V], float* s) {  // 1 / sqrt(mean v^2 + eps)
    f32x4 sum = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < V; ++i) sum = sum + v[i] * v[i];
    return 1.0f / sqrtf(norm_sum<TH>((sum.x + sum.y) + (sum.z + sum.w), s) / static_cast<float>(cols) + a.eps);
  };
  if (a.post_w) {
    const float r = rms(x, ws[0]);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = x[i] * r * (a.post_offset + pw[i]);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint32_t q = i * TH + threadIdx.x;
    if (a.h) x[i] = h[i] + x[i];
    if (a.h_out && 4 * q < cols) norm_store(a.h_out + base, q, cols, x[i]);
  }
  if (!a.w) return;
  const float r = rms(x, ws[1]);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint32_t q = i * TH + threadIdx.x;
    if (4 * q < cols) norm_store(a.out + base, q, cols, x[i] * r * (a.offset + w[i]));
  }
}

static constexpr int kNormLongThreads = 1024;

// The same for rows of any length, which are read again after each sum, in 4-byte accesses. 2048 x
// 20000 with an addition 182 us, 3.6 TB/s of the values read and written once (16384 columns in
// registers 105, 5.1); 16 x 20000 12.
__global__ __launch_bounds__(kNormLongThreads) void add_norm_long_rows(AddNorm a, uint32_t cols) {
  __shared__ float ws[kNormLongThreads / 64];
  const size_t base = static_cast<size_t>(blockIdx.x) * cols;
  float ru = 1.0f, sum = 0.0f;
  if (a.post_w) {
    for (uint32_t i = threadIdx.x; i < cols; i += kNormLongThreads) sum = fmaf(a.x[base + i], a.x[base + i], sum);
    ru = 1.0f / sqrtf(norm_sum<kNormLongThreads>(sum, ws) / static_cast<float>(cols) + a.eps);
  }
  const auto stream = [&](uint32_t i) {
    float v = a.x[base + i];
    if (a.post_w) v = v * ru * (a.post_offset + a.post_w[i]);
    return a.h ? a.h[base + i] + v : v;
  };
  sum = 0.0f;
  for (uint32_t i = threadIdx.x; i < cols; i += kNormLongThreads) {
    const float v = stream(i);
    sum = fmaf(v, v, sum);
    if (!a.w) a.h_out[base + i] = v;
  }
  if (!a.w) return;
  const float r = 1.0f / sqrtf(norm_sum<kNormLongThreads>(sum, ws) / static_cast<float>(cols) + a.eps);
  for (uint32_t i = threadIdx.x; i < cols; i += kNormLongThreads) {
    const float v = stream(i);
    if (a.h_out) a.h_out[base + i] = v;
    a.out[base + i] = v * r * (a.offset + a.w[i]);
  }
}

}  // namespace yx
