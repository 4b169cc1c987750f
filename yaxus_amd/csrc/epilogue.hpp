// What a weight product does with its sums before they leave the registers: nothing
// (yx_matmul_bf16_dev), or bias, activation, gate and residual (yx_linear_bf16_dev):
//   out = act(y + bias) + residual,  gated: act(y_gate + bias_gate) * (y_up + bias_up) + residual.
// On its own each of these would read and write the rows once more (134 MB each way for 4096 x 8192).
// Everything is f32; the activations' e^x and 1/x are the hardware's (within 1 ulp, e^x of an
// argument rounded to f32), written so that no term cancels: silu and gelu_tanh divide by
// 1 + e^-z, gelu uses erfc. 4096 x 2048 x 8192 with bias: none 344 us, silu 348, gelu_tanh 350,
// gelu 373.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/yaxus_hip.h"
#include "attn_decode.hpp"

namespace yx {

typedef float f32x4 __attribute__((ext_vector_type(4)));
// Four floats at any float's address: the hardware takes 16-byte accesses there.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// Four values at once (one branch on act, which is uniform). NaN stays NaN in every one of
// them; -inf gives NaN where the formula is -inf * 0 (all but none and relu).
__device__ __forceinline__ f32x4 activate(f32x4 y, uint32_t act) {
  switch (act) {
    case YX_ACT_RELU:
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = y[i] < 0.0f ? 0.0f : y[i];
      break;
    case YX_ACT_SILU:
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] *= __builtin_amdgcn_rcpf(1.0f + __expf(-y[i]));
      break;
    case YX_ACT_GELU:
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] *= 0.5f * erfcf(y[i] * -0.70710678f);
      break;
    case YX_ACT_GELU_TANH:  // y (1 + tanh u) / 2 = y / (1 + e^-2u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float u2 = y[i] * fmaf(0.07135481f * y[i], y[i], 1.5957691f);
        y[i] *= __builtin_amdgcn_rcpf(1.0f + __expf(-u2));
      }
      break;
    default: break;
  }
  return y;
}

struct NoEpilogue {
  static constexpr bool kGated = false, kFused = false;
};

// residual may be the output itself: a lane reads the four values it then writes. Gated:
// bias holds the n gate rows' values, then the n up rows'.
template <bool kGated_>
struct Epilogue {
  static constexpr bool kGated = kGated_, kFused = true;
  const float* bias;      // null: none
  const float* residual;  // null: none
  uint32_t act;
};

// A lane's outputs at columns col .. col + 3 of one row; y holds the sums (of the gate rows),
// up those of the up rows (gated only). wide (without an epilogue): wide_out.
template <class E>
__device__ __forceinline__ void store_out4(const E& e, float* out, uint32_t row, uint32_t col, uint32_t n,
                                           bool wide, const f32x4& y, const f32x4& up) {
  if (col >= n) return;
  float* o = out + static_cast<size_t>(row) * n + col;
  if constexpr (!E::kFused) {
    if (wide) {
      *reinterpret_cast<f32x4*>(o) = y;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col + i < n) o[i] = y[i];
    }
  } else {
    f32x4 v = y, u = up, a = {0, 0, 0, 0};
    const float* r = e.residual + static_cast<size_t>(row) * n + col;
    const bool whole = col + 4 <= n;  // 16-byte accesses, at any float's address
    if (whole) {
      if (e.residual) a = *reinterpret_cast<const f32x4_any*>(r);
      if (e.bias) {
        v = v + *reinterpret_cast<const f32x4_any*>(e.bias + col);
        if (E::kGated) u = u + *reinterpret_cast<const f32x4_any*>(e.bias + static_cast<size_t>(n) + col);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        if (col + i >= n) continue;
        if (e.residual) a[i] = r[i];
        if (e.bias) {
          v[i] += e.bias[col + i];
          if (E::kGated) u[i] += e.bias[static_cast<size_t>(n) + col + i];
        }
      }
    }
    v = activate(v, e.act);
    if (E::kGated) v = v * u;
    if (e.residual) v = v + a;
    if (whole) {
      *reinterpret_cast<f32x4_any*>(o) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (col + i < n) o[i] = v[i];
    }
  }
}

// Whether store_out4 may use 16-byte accesses without an epilogue.
__device__ __forceinline__ bool wide_out(const float* out, uint32_t n) {
  return (n & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
}

}  // namespace yx
