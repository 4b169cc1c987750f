// Products of at most 32 rows with an epilogue: bound by reading the weight once.
// out[t][n] = x[t][:] . w[n][:] as in matmul_bf16.hpp (x in three bf16 parts, every product
// exact, f32 sums), then the epilogue.
//
// A workgroup's 8 waves own NT tiles of 16 weight rows each (gated: 16 gate rows and their 16 up
// rows) against all R tiles of 16 rows of x. x is cut up once per workgroup, KC of k at a time,
// into LDS (two slots, one barrier per KC), in the order in which lanes read it; the weight goes
// straight from memory to the registers of the wave that multiplies it, a whole chunk of KC
// ahead, so that nothing waits for it but its own product. No sums meet between waves; a chunk's
// products are added to the result in f32, so chains stay short.
// Workgroups start at different chunks and go round: rows are 2 k bytes apart, and workgroups in
// step would ask the same memory channels for their rows' same columns (k 8192, 262 MB 61 -> 52
// us, 524 MB 126 -> 104; k 2048 28.4 -> 27.9).
// Layouts as in step_after.hpp (A: 16 weight rows, B: 16 rows of a part of x).
// With ks > 1 (grid y) the workgroups of a column group take consecutive chunks of k and hand
// their tiles over as matmul_bf16_rows does.
// Measured, 16 rows, weights from HBM: k 2048, n 8192 gated (67 MB) 17.7 us, k 8192, n 2048 14.1 (33.5
// MB), k 4096, n 14336 gated 52 (4.6 TB/s), k 8192, n 16000 gated 104 (5.1 TB/s). Tried: a wave streaming
// tiles past x in registers (16 rows of 2 KiB at a time, no LDS) 100 us for the last, but 18-29%
// slower up to 34 MB, where each part of x is cut up for too few tiles.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "epilogue.hpp"
#include "matmul_bf16.hpp"

namespace yx {

static constexpr int kFewThreads = 512;

template <int R>
constexpr int few_chunk() {
  return R == 1 ? 256 : 128;
}

template <int R, int NT, class E>
__global__ __launch_bounds__(kFewThreads, 4) void matmul_bf16_few(
    const float* __restrict__ x, const uint16_t* __restrict__ w, float* out, uint32_t t, uint32_t k,
    uint32_t n, f32x4* __restrict__ part, uint32_t part_bytes, uint32_t* __restrict__ counters, E epi) {
  constexpr int KC = few_chunk<R>(), STEPS = KC / 32, TH = kFewThreads;
  constexpr int XC = R * 16 * KC / 8 / TH;  // pieces of 8 k of x per thread
  static_assert(XC * TH == R * 16 * KC / 8, "whole rounds of pieces");
  constexpr uint32_t COLS = E::kGated ? 128 : 128 * NT;
  constexpr int kOutside = 0x7ffffff0;  // beyond every resource: reads zeros
  static_assert(!E::kGated || NT == 2, "a gate and an up tile");
  __shared__ u16x8 xs[2][STEPS][R][3][64];
  __shared__ uint32_t last;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int c = lane & 15, g = lane >> 4, sw = c * 4 + (g ^ ((c >> 1) & 3));
  const uint32_t n0 = blockIdx.x * COLS, ks = gridDim.y, kp = blockIdx.y;
  const uint32_t chunks = (k + KC - 1) / KC, c0 = chunks * kp / ks, c1 = chunks * (kp + 1) / ks;

  const uint32_t len = c1 - c0, rot = blockIdx.x % len;
  const auto chunk = [&](uint32_t i) { return i < len ? c0 + (i + rot >= len ? i + rot - len : i + rot) : c1; };
  const uint32_t wbytes = min(n - n0, COLS) * k * 2;
  const __amdgpu_buffer_rsrc_t rw = make_rsrc(const_cast<uint16_t*>(w + static_cast<size_t>(n0) * k), wbytes);
  const __amdgpu_buffer_rsrc_t ru =
      make_rsrc(const_cast<uint16_t*>(w + (static_cast<size_t>(n0) + (E::kGated ? n : 0)) * k), wbytes);
  int wo[NT];
#pragma unroll
  for (int a = 0; a < NT; ++a)
    wo[a] = ((E::kGated ? wave : wave * NT + a) * 16 + c) * static_cast<int>(k) * 2 + 16 * g;
  u16x8 wv[STEPS][NT];
  // (A resource's range counts from its scalar offset, so that stays inside it where nothing is
  // read too: k - 8 is the last piece of a row.)
  const auto load_w = [&](int s, uint32_t ch) {  // past this part: zeros, nothing read
    const uint32_t kb = ch * KC + s * 32, at = min(kb, k - 8) * 2;
    const bool ok = (ch < c1) & (kb + 8 * g < k);
#pragma unroll
    for (int a = 0; a < NT; ++a)
      wv[s][a] = __builtin_bit_cast(
          u16x8, __builtin_amdgcn_raw_buffer_load_b128(E::kGated && a ? ru : rw, ok ? wo[a] : kOutside, at, 0));
  };

  const __amdgpu_buffer_rsrc_t rx = make_rsrc(const_cast<float*>(x), t * k * 4);  // rows past t: zeros
  int xo[XC], xd[XC];
  uint32_t xk[XC];
#pragma unroll
  for (int i = 0; i < XC; ++i) {
    const int id = i * TH + tid, row = id / (KC / 8), kc = id % (KC / 8), r = row % 16;
    xk[i] = kc * 8;
    xo[i] = (row * static_cast<int>(k) + kc * 8) * 4;
    xd[i] = ((kc / 4) * R + row / 16) * 3 * 64 + r * 4 + ((kc & 3) ^ ((r >> 1) & 3));
  }
  struct XRegs {
    f32x4 a[XC], b[XC];
  };
  const auto load_x = [&](XRegs& r, uint32_t ch) {
    const uint32_t kb = ch * KC, at = min(kb, k - 8) * 4;
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      const bool ok = (ch < c1) & (kb + xk[i] < k);
      const int o = ok ? xo[i] : kOutside;
      r.a[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rx, o, at, 0));
      r.b[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rx, o, at + 16, 0));
    }
  };
  const auto write_x = [&](const XRegs& r, int slot) {
    u16x8* d = &xs[slot][0][0][0][0];
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      const float v[8] = {r.a[i].x, r.a[i].y, r.a[i].z, r.a[i].w, r.b[i].x, r.b[i].y, r.b[i].z, r.b[i].w};
      u32x4 p[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t h, m, l;
        split_bf16x3<true>(v[2 * e], v[2 * e + 1], h, m, l);
        p[0][e] = h;
        p[1][e] = m;
        p[2][e] = l;
      }
#pragma unroll
      for (int q = 0; q < 3; ++q) d[xd[i] + q * 64] = __builtin_bit_cast(u16x8, p[q]);
    }
  };

  f32x4 sum[NT][R];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int b = 0; b < R; ++b) sum[a][b] = f32x4{0, 0, 0, 0};
  // Loads in the loop's order, the next chunk's x before the weight's: a wait for x, then and in
  // the loop, lets the weight's loads fly on.
  XRegs xr;
  {
    XRegs first;
    load_x(first, chunk(0));
    load_x(xr, chunk(1));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) load_w(s, chunk(0));
    __builtin_amdgcn_sched_barrier(0);
    write_x(first, 0);
  }
  lds_barrier();
  int slot = 0;
  for (uint32_t i = 0; i < len; ++i, slot ^= 1) {
    const uint32_t next = chunk(i + 1);
    // The other slot was last read before the barrier that ended the previous chunk.
    write_x(xr, slot ^ 1);
    load_x(xr, chunk(i + 2));
    __builtin_amdgcn_sched_barrier(0);
    f32x4 acc[NT][R];
    bf16x8 xf[2][R][3];
    const auto read_x = [&](int s) {
#pragma unroll
      for (int b = 0; b < R; ++b)
#pragma unroll
        for (int q = 0; q < 3; ++q) xf[s & 1][b][q] = __builtin_bit_cast(bf16x8, xs[slot][s][b][q][sw]);
    };
    read_x(0);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (s + 1 < STEPS) read_x(s + 1);
#pragma unroll
      for (int b = 0; b < R; ++b)
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
          for (int a = 0; a < NT; ++a)
            acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv[s][a]), xf[s & 1][b][q],
                                                                s == 0 && q == 0 ? f32x4{0, 0, 0, 0} : acc[a][b], 0, 0, 0);
      load_w(s, next);
      __builtin_amdgcn_sched_barrier(0);  // this step's registers are filled again here, not at the chunk's end
    }
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int b = 0; b < R; ++b) sum[a][b] = sum[a][b] + acc[a][b];
    lds_barrier();
  }

  if (ks > 1) {  // as matmul_bf16_rows: write-through partial tiles, an arrival count
    const __amdgpu_buffer_rsrc_t rp = make_rsrc(part, part_bytes);
    constexpr uint32_t kTile = 8 * NT * R * 64;  // in f32x4
    const uint32_t base = blockIdx.x * ks * kTile + wave * NT * R * 64 + lane;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int b = 0; b < R; ++b)
        st4_coherent(rp, (base + kp * kTile + (a * R + b) * 64) * 16, __builtin_bit_cast(float4, sum[a][b]));
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
      uint32_t* cnt = counters + static_cast<size_t>(blockIdx.x) * kCounterStride;
      const uint32_t arrived = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = arrived == ks - 1;
      if (last) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int b = 0; b < R; ++b) sum[a][b] = f32x4{0, 0, 0, 0};
    for (uint32_t q = 0; q < ks; ++q)  // the parts in k order
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < R; ++b)
          sum[a][b] = sum[a][b] + __builtin_bit_cast(f32x4, ld4_coherent(rp, (base + q * kTile + (a * R + b) * 64) * 16));
  }
  const bool wide = wide_out(out, n);
#pragma unroll
  for (int b = 0; b < R; ++b) {
    const uint32_t row = b * 16 + c;
    if (row >= t) continue;
    if constexpr (E::kGated) {
      store_out4(epi, out, row, n0 + wave * 16 + 4 * g, n, wide, sum[0][b], sum[1][b]);
    } else {
#pragma unroll
      for (int a = 0; a < NT; ++a)
        store_out4(epi, out, row, n0 + (wave * NT + a) * 16 + 4 * g, n, wide, sum[a][b], sum[a][b]);
    }
  }
}

}  // namespace yx
