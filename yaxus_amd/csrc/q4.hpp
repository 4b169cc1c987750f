// The 4-bit form of K and V, its store and its read-back.
//
// Of a group of 32 consecutive values of a head vector, m is the one of the largest magnitude
// (the first of equals). The step s = m / -8 rounded to binary16 (nearest even, limited to the
// largest finite value); the code of x is x / s rounded to the nearest whole number, ties to
// even, + 8, limited to 0 .. 15; it stands for s (code - 8), exact in f32. The value farthest
// from zero thus gets the code 0, the only one of magnitude 8, so the 16 codes are all in use
// whichever its sign (N(0, 1): 7.6% of the values' root mean square; with a magnitude of at most
// 7 on both sides 8.7%). A group of zeros, or below binary16's smallest: step 0, codes 8. A
// group that holds an infinity or NaN: step NaN, codes 8, so each of its values reads NaN and
// no code ever stands for anything but a small whole number. (Groups, signed step and offset 8 are those
// of the published block format Q4_0; ties, limits and byte order are this arena's.)
//
// A head vector is 72 bytes (64 of codes, 4 steps; 256 in binary16). Arena layout per layer:
// `[page][kv_head][block of 16 keys]`, 1152 bytes a block, codes first, steps at 1024. Both
// orders are what one 16-byte load per lane gives the attention kernels (lane l, c = l % 16,
// g = l / 16; e = 0..7, p = 0..3, n = 0..7):
//   K: byte 16 l + 4 p: a dword of the 8 codes of key c, dims 32 p + 8 g + e, code e in the
//      nibble (e / 2) + 4 (e % 2);
//   V: byte 16 l + 4 i: a dword of the 8 codes of key 4 g + i, dims 16 n + c, code n in nibble n;
//   steps, binary16: K `[key][4 groups]`, V `[g][4 groups][4 keys]`.
// Masks of 0x000f000f and 0x00f000f0 over a dword and over the dword shifted by 8 leave two codes
// each in the halves of a register, a few bits from being a binary16 matrix operand.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_kernels.hpp"

namespace yx {

struct q4_t {  // an arena's bytes
  uint8_t b;
};

static constexpr uint32_t kQ4Block = 1152;   // bytes of 16 keys of one head
static constexpr uint32_t kQ4Steps = 1024;   // offset of their steps
static constexpr uint32_t kQ4Row = 72;       // bytes of one head vector
static constexpr float kQ4MaxStep = 65504.0f;

// Byte of a block that holds the dword of K's dims 32 p + 8 g .. + 7 of key c, and of V's dims
// c, 16 + c, .. of key k.
__host__ __device__ inline uint32_t q4_k_word(uint32_t c, uint32_t g, uint32_t p) { return (g * 16 + c) * 16 + p * 4; }
__host__ __device__ inline uint32_t q4_v_word(uint32_t k, uint32_t c) { return ((k / 4) * 16 + c) * 16 + (k % 4) * 4; }
// Index of the step of key k, group p, behind kQ4Steps.
__host__ __device__ inline uint32_t q4_k_step(uint32_t k, uint32_t p) { return k * 4 + p; }
__host__ __device__ inline uint32_t q4_v_step(uint32_t k, uint32_t p) { return (k / 4) * 16 + p * 4 + k % 4; }
__host__ __device__ inline uint32_t q4_k_nibble(uint32_t e) { return e / 2 + 4 * (e % 2); }

// Another lane's value within a row of 16 by a data-parallel-primitive control (register moves, where
// a shuffle goes through LDS): 0xb1 lanes 1, 0, 3, 2; 0x4e lanes 2, 3, 0, 1; 0x141 mirrored in eights;
// 0x140 in the row. One after the other they bring a value to all lanes of the row.
template <int kCtrl>
__device__ __forceinline__ uint32_t q4_lanes(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(v), static_cast<int>(v), kCtrl, 0xf, 0xf, false));
}

// A wave's 32-lane halves hold one group each: the group's step and this lane's code.
__device__ __forceinline__ void q4_quantise(float x, int lane, _Float16& step, uint32_t& code) {
  const uint32_t mag = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  uint32_t most = max(mag, q4_lanes<0xb1>(mag));
  most = max(most, q4_lanes<0x4e>(most));
  most = max(most, q4_lanes<0x141>(most));
  most = max(most, q4_lanes<0x140>(most));
  most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16)));
  const uint64_t at = __builtin_amdgcn_ballot_w64(mag == most);
  const int first = __builtin_ctz(static_cast<uint32_t>(lane & 32 ? at >> 32 : at)) + (lane & 32);
  const float top = __shfl(x, first) * -0.125f;
  const bool finite = most < 0x7f800000u;
  step = finite ? static_cast<_Float16>(fminf(fmaxf(top, -kQ4MaxStep), kQ4MaxStep)) : static_cast<_Float16>(__builtin_nanf(""));
  const float s = static_cast<float>(step);
  // The quotient by an approximate reciprocal is off by less than one; what is left of x beside
  // it (exact: both are multiples of x's last bit and it is no longer than x) sets it right.
  float r = fminf(fmaxf(__builtin_rintf(x * __builtin_amdgcn_rcpf(s)), -9.0f), 8.0f);
  const float e = __builtin_fmaf(-r, s, x), half = 0.5f * fabsf(s);
  const bool odd = (static_cast<int>(r) & 1) != 0;
  if (fabsf(e) > half || (fabsf(e) == half && odd)) r += (e > 0.0f) == (s > 0.0f) ? 1.0f : -1.0f;
  r = fminf(fmaxf(r, -8.0f), 7.0f);
  code = finite && s != 0.0f ? static_cast<uint32_t>(static_cast<int>(r) + 8) : 8u;
}

__device__ __forceinline__ uint32_t or_xor(uint32_t v, int o) {
  return v | static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o));
}

// One key vector (or value vector) of key `k` of the block at `blk`, by a whole wave: the lane's
// dims are lane and lane + 64.
__device__ __forceinline__ void q4_store_k(float x0, float x1, uint32_t k, int lane, q4_t* blk) {
  _Float16 s0, s1;
  uint32_t c0, c1;
  q4_quantise(x0, lane, s0, c0);
  q4_quantise(x1, lane, s1, c1);
  const uint32_t sh = 4 * q4_k_nibble(lane & 7);
  c0 <<= sh;
  c1 <<= sh;
  for (uint32_t* c : {&c0, &c1}) {  // of 8 lanes
    *c |= q4_lanes<0xb1>(*c);
    *c |= q4_lanes<0x4e>(*c);
    *c |= q4_lanes<0x141>(*c);
  }
  const uint32_t p = lane >> 5, g = (lane >> 3) & 3;
  if ((lane & 7) == 0) {
    *reinterpret_cast<uint32_t*>(blk + q4_k_word(k, g, p)) = c0;
    *reinterpret_cast<uint32_t*>(blk + q4_k_word(k, g, p + 2)) = c1;
  }
  if ((lane & 31) == 0) {
    _Float16* st = reinterpret_cast<_Float16*>(blk + kQ4Steps);
    st[q4_k_step(k, p)] = s0;
    st[q4_k_step(k, p + 2)] = s1;
  }
}

__device__ __forceinline__ void q4_store_v(float x0, float x1, uint32_t k, int lane, q4_t* blk) {
  _Float16 s0, s1;
  uint32_t c0, c1;
  q4_quantise(x0, lane, s0, c0);
  q4_quantise(x1, lane, s1, c1);
  const uint32_t n = lane >> 4;
  const uint32_t w = or_xor(or_xor((c0 << (4 * n)) | (c1 << (4 * n + 16)), 16), 32);
  if (lane < 16) *reinterpret_cast<uint32_t*>(blk + q4_v_word(k, lane)) = w;
  if ((lane & 31) == 0) {
    _Float16* st = reinterpret_cast<_Float16*>(blk + kQ4Steps);
    st[q4_v_step(k, lane >> 5)] = s0;
    st[q4_v_step(k, (lane >> 5) + 2)] = s1;
  }
}

// The block of a slot (pages of 1 << page_shift slots) in a layer's arena.
__device__ __forceinline__ size_t q4_block_of(uint32_t slot, uint32_t kh, uint32_t hkv, uint32_t page_shift) {
  const uint32_t blk = (slot & ((1u << page_shift) - 1u)) >> 4;
  return ((((static_cast<size_t>(slot >> page_shift) * hkv + kh) << page_shift) >> 4) + blk) * kQ4Block;
}

// As the other arenas' (see qk_rope.hpp): a key head, normalised and rotated, and its raw value
// head, by a whole wave.
__device__ __forceinline__ void store_kv_head(float k0, float k1, const float* __restrict__ vsrc,
                                              uint32_t slot, uint32_t kh, uint32_t hkv,
                                              uint32_t page_shift, uint32_t lane, q4_t* kc, q4_t* vc) {
  const size_t blk = q4_block_of(slot, kh, hkv, page_shift);
  q4_store_k(k0, k1, slot & 15, static_cast<int>(lane), kc + blk);
  q4_store_v(vsrc[lane], vsrc[lane + 64], slot & 15, static_cast<int>(lane), vc + blk);
}

// The K/V store of write_rows into a 4-bit arena: one wave per vector, K (blockIdx.y 0) or V. 65536
// rows of 4 heads: 143 us, 2.1 TB/s (151 with the group's maximum by shuffles); bound by the
// instructions of a vector (two groups' maxima, codes with their exact ties, their gathering), not memory.
// 16 rows: 2.6 us.
__global__ __launch_bounds__(256) void kv_append_q4(const float* __restrict__ k, const float* __restrict__ v,
                                                    const uint32_t* __restrict__ kv_slot, q4_t* __restrict__ kc,
                                                    q4_t* __restrict__ vc, uint32_t vecs, uint32_t hkv,
                                                    uint32_t page_shift) {
  const uint32_t vec = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (vec >= vecs) return;  // uniform over the wave
  const uint32_t row = vec / hkv, kh = vec % hkv, slot = kv_slot[row];
  const float* src = (blockIdx.y == 0 ? k : v) + static_cast<size_t>(vec) * 128;
  const float x0 = src[lane], x1 = src[lane + 64];
  const size_t blk = q4_block_of(slot, kh, hkv, page_shift);
  if (blockIdx.y == 0) q4_store_k(x0, x1, slot & 15, lane, kc + blk);
  else q4_store_v(x0, x1, slot & 15, lane, vc + blk);
}

// What an arena holds of the pass's rows, as f32 `[rows][hkv][128]`: 16 threads per vector, 8
// dims each; blockIdx.y: 0 = K, 1 = V. Bound by the f32 stores (4096 rows of 4 heads, 17 MB: 5.9 us),
// one row by the trip to memory (1.4).
__device__ __forceinline__ void kv_row_piece(const q4_t* kc, const q4_t* vc, bool is_k, uint32_t slot, uint32_t kh,
                                             uint32_t hkv, uint32_t page_shift, uint32_t ch, float* x) {
  const q4_t* blk = (is_k ? kc : vc) + q4_block_of(slot, kh, hkv, page_shift);
  const uint32_t key = slot & 15;
  const float s = static_cast<float>(reinterpret_cast<const _Float16*>(blk + kQ4Steps)[is_k ? q4_k_step(key, ch / 4) : q4_v_step(key, ch / 4)]);
  if (is_k) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(blk + q4_k_word(key, ch & 3, ch >> 2));
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) x[e] = s * (static_cast<float>((w >> (4 * q4_k_nibble(e))) & 15u) - 8.0f);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {  // dim 8 ch + e = 16 (ch / 2) + 8 (ch % 2) + e
      const uint32_t w = *reinterpret_cast<const uint32_t*>(blk + q4_v_word(key, 8 * (ch & 1) + e));
      x[e] = s * (static_cast<float>((w >> (4 * (ch >> 1))) & 15u) - 8.0f);
    }
  }
}

__device__ __forceinline__ void kv_row_piece(const _Float16* kc, const _Float16* vc, bool is_k, uint32_t slot,
                                             uint32_t kh, uint32_t hkv, uint32_t page_shift, uint32_t ch, float* x) {
  const uint32_t off = slot & ((1u << page_shift) - 1u);
  const size_t region = ((static_cast<size_t>(slot >> page_shift) * hkv + kh) * 128) << page_shift;
  const _Float16* src = is_k ? kc + region + k_offset(off, ch) : vc + region + off * 128 + ch * 8;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(src[e]);
}

__device__ __forceinline__ void kv_row_piece(const float* kc, const float* vc, bool is_k, uint32_t slot, uint32_t kh,
                                             uint32_t hkv, uint32_t page_shift, uint32_t ch, float* x) {
  const size_t row = (((static_cast<size_t>(slot >> page_shift) * hkv + kh) << page_shift) +
                      (slot & ((1u << page_shift) - 1u))) * 128;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (is_k ? kc : vc)[row + ch * 8 + e];
}

template <typename T>
__global__ __launch_bounds__(256) void kv_rows(const T* __restrict__ kc, const T* __restrict__ vc,
                                               const uint32_t* __restrict__ kv_slot, float* __restrict__ k_out,
                                               float* __restrict__ v_out, uint32_t vecs, uint32_t hkv,
                                               uint32_t page_shift) {
  const uint32_t vec = blockIdx.x * 16 + (threadIdx.x >> 4), ch = threadIdx.x & 15;
  if (vec >= vecs) return;
  float* out = blockIdx.y == 0 ? k_out : v_out;
  if (out == nullptr) return;
  float x[8];
  kv_row_piece(kc, vc, blockIdx.y == 0, kv_slot[vec / hkv], vec % hkv, hkv, page_shift, ch, x);
  float4* dst = reinterpret_cast<float4*>(out + static_cast<size_t>(vec) * 128 + ch * 8);
  dst[0] = float4{x[0], x[1], x[2], x[3]};
  dst[1] = float4{x[4], x[5], x[6], x[7]};
}

}  // namespace yx
