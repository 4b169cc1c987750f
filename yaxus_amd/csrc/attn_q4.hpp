// Paged attention over a 4-bit arena (q4.hpp) for gfx950: decode and verify items, and prefill
// tiles.
//
// out = softmax(q K^T scale) V with K, V = s (code - 8), s the binary16 step of 32 dims: up to 15
// bits, more than a binary16 holds.
//   S[key] = sum_p s_p[key] sum_d q_d (code_d - 8)          p: a group of 32 dims
//     one v_mfma_f32_16x16x32_f16 per group and part of q, the codes as binary16 (below); then
//     one fused multiply-add per score and group;
//   O_d = sum_key P V_d
//     V as a binary16 hi part (the rounded product of step and code) and a lo part (what that left,
//     exact: one packed fused multiply-add), P as hi and lo too; all products but lo lo.
// K's steps stay apart since a score needs one multiply-add per group where K's lo part would need
// a third matrix product per group; V's go in since they would cost a cut of P per group and row.
// q is scaled by a power of two of its row (its largest value near 2^12) before it is cut, so its
// size does not matter; the cuts keep ~2^-22. A binary16 holds V's parts (and 16 times them) below
// 4096: a wave whose result is not finite runs again, once for the steps from 1 up, scaled down,
// and once for the others, with steps of NaN (or infinite) left out and noted where a row sees them.
// So does a wave with scores beyond 2^16, whose weights need another form (q4_is_far).
// Outputs are 3-4e-7 off 64 bits (1500 keys), also of small V down to 1e-5, whose products with codes
// are subnormal binary16 numbers, of which the matrix unit drops bits: 7e-7 at 3e-6, 2-4e-6 at 1e-6.
// Steps of keys that no row of the wave sees are cleared at once. So a masked key never has an
// effect, whatever it holds.
//
// Operands (lane l, c = l % 16, g = l / 16): columns are logical rows ((row, q head) pairs), 16 a
// tile. S^T and P^T: keys 4 g + i of column c. O^T: dims 16 n + 4 g + i of column c (n: tile of V).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "attn_decode.hpp"
#include "attn_prefill.hpp"
#include "q4.hpp"

namespace yx {

typedef _Float16 half2_q4 __attribute__((ext_vector_type(2)));

// K of a 16-key block as a lane holds it: codes, and the steps of keys 4 g .. 4 g + 3. V likewise.
struct Q4Half {
  u32x4 codes, steps[2];
};

template <int kPolicy>
__device__ __forceinline__ void q4_load(Q4Half& r, const q4_t* blk, bool valid, int lane) {
  const __amdgpu_buffer_rsrc_t rs =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<q4_t*>(blk), 0, valid ? static_cast<int>(kQ4Block) : 0, 0x00020000);
  const int st = static_cast<int>(kQ4Steps) + (lane >> 4) * 32;
  r.codes = __builtin_amdgcn_raw_buffer_load_b128(rs, lane * 16, 0, kPolicy);
  r.steps[0] = __builtin_amdgcn_raw_buffer_load_b128(rs, st, 0, kPolicy);
  r.steps[1] = __builtin_amdgcn_raw_buffer_load_b128(rs, st, 16, kPolicy);
}

// Two codes in the low nibbles of w's halves (kOdd: the second nibbles) less 8 (kOdd: 16 times
// that) as binary16: or-ed under the exponent of 1024 they read 1024 + code (1024 + 16 code), and
// the difference is exact. (As they lie, read as subnormals code * 2^-24, they would need no
// exponent, but the matrix unit aligns a subnormal's products by its nominal exponent and drops
// up to 7 of their bits: outputs 6e-6 off after 600 keys and 1.3e-5 after 4000, against 3e-7.)
// The exponent comes in a register: with two literals the and-or would be two instructions.
template <bool kOdd>
__device__ __forceinline__ half2_q4 q4_codes(uint32_t w, uint32_t exponent) {
  const half2_q4 c = __builtin_bit_cast(half2_q4, (w & (kOdd ? 0x00f000f0u : 0x000f000fu)) | exponent);
  const _Float16 base = static_cast<_Float16>(kOdd ? 1152.0f : 1032.0f);
  return c - half2_q4{base, base};
}

// The codes of a K dword as a matrix operand (dims 32 p + 8 g + 0 .. 7; 2, 3, 6, 7 times 16).
__device__ __forceinline__ half8 q4_k_codes(uint32_t w, uint32_t e) {
  const half2_q4 a = q4_codes<false>(w, e), b = q4_codes<true>(w, e), c = q4_codes<false>(w >> 8, e), d = q4_codes<true>(w >> 8, e);
  return half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Two values as a binary16 hi part and a lo part each. The values and the hi parts are pinned: the
// compiler would otherwise take hi from the unrounded product a value comes from in one place and
// from the value in the other, which differ by a last bit now and then (outputs up to 1e-5 off).
__device__ __forceinline__ void q4_cut(float y0, float y1, uint32_t& hi, uint32_t& lo) {
  pin(y0);
  pin(y1);
  hi = __builtin_bit_cast(uint32_t, half2_q4{static_cast<_Float16>(y0), static_cast<_Float16>(y1)});
  pin(hi);
  float r0, r1;  // y - hi, the half read where it lies
  __asm__("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(hi), "v"(y0));
  __asm__("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(hi), "v"(y1));
  lo = __builtin_bit_cast(uint32_t, half2_q4{static_cast<_Float16>(r0), static_cast<_Float16>(r1)});
}

// Weights are 2^(kQ4Room + x - m), x and m in log2, and x > m + kQ4Lazy moves m: as high as
// binary16 allows, since parts of weights below its smallest normal value lose bits.
static constexpr float kQ4Lazy = 2.0f;
static constexpr float kQ4Room = 13.0f;

// What one wave attends: NT tiles of 16 logical rows over the blocks [b0, b0 + nblk) of a page
// table.
template <int NT>
struct Q4Wave {
  float m[NT], l[NT];      // maximum (log2) and sum
  floatx4 o[NT][8];        // unnormalised, dims 16 n + 4 g + i
};

// The rows of a wave: this lane's column of each tile.
template <int NT>
struct Q4Rows {
  bool has[NT];            // there is a row
  int pos[NT], lo[NT];     // its last (-1: no row) and first key
  float fac[NT];           // from products to log2 scores
  int all_lo, all_pos;     // keys that every row of the wave sees,
  int any_lo, any_pos;     // and from the first to the last that some row does
};

// A tile's q (this lane's dims 32 p + 8 g + 0 .. 7 of its column) as operands: hi and lo parts
// scaled by a power of two; returns the factor from products to log2 scores. The scale's sign goes
// into q, and a factor of 0 becomes one without effect, so that it is positive: the maximum
// may be looked for before it, and a masked -inf stays one.
__device__ __forceinline__ float q4_cut_q(float4 (&raw)[8], float scale_log2, u32x4 (&hi)[4], u32x4 (&lo)[4]) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float4 a = raw[j];
    top = fmaxf(top, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))));
  }
  top = max_xor32(max_xor16(top));
  const int ex = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;  // top < 2^ex
  if (scale_log2 < 0.0f) {
    __asm__ volatile("");  // a branch: no select per value
#pragma unroll
    for (int j = 0; j < 8; ++j) raw[j] = float4{-raw[j].x, -raw[j].y, -raw[j].z, -raw[j].w};
  }
#pragma unroll
  for (int p = 0; p < 4; ++p)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 a = raw[2 * p + j];
      uint32_t h0, l0, h1, l1;  // elements 2, 3 meet codes 16 times as large
      q4_cut(__builtin_ldexpf(a.x, 13 - ex), __builtin_ldexpf(a.y, 13 - ex), h0, l0);
      q4_cut(__builtin_ldexpf(a.z, 9 - ex), __builtin_ldexpf(a.w, 9 - ex), h1, l1);
      hi[p][2 * j] = h0;
      hi[p][2 * j + 1] = h1;
      lo[p][2 * j] = l0;
      lo[p][2 * j + 1] = l1;
    }
  // At least 2^-126, never 0, which a masked -inf would make NaN: products are below 2^40, so such a
  // score is 2^-86 at most, as good as 0. A scale of 0 is that whatever q's size.
  const float fac = scale_log2 == 0.0f ? 0.0f : __builtin_ldexpf(fabsf(scale_log2), ex - 13);
  return fac < 0x1p-126f ? 0x1p-126f : fac;
}

// Scores this large need the second form below. 2^(x + (kQ4Room - m)) is one multiply-add a score,
// with a sum in brackets that is rounded, and x exact where m is a rounded product: up to 2^16 both
// are off by 2^-8, so weights stay below 2^(kQ4Room + kQ4Lazy + 2^-7), in binary16's range; from
// 2^26 on kQ4Room would round to 16 or to nothing. (Scores of ordinary models are some hundreds.)
static constexpr float kQ4Far = 0x1p16f;
__device__ __forceinline__ bool q4_is_far(float m) { return fabsf(m) > kQ4Far && m > -INFINITY; }

// A weight in the slow runs: a row's is made by the same form in every wave. Where the maximum is
// far, the product is rounded as the maximum's was, so their difference is exact near it and at most
// kQ4Lazy whatever their size.
__device__ __forceinline__ float q4_slow_weight(float score, float fac, float m) {
  float x = score * fac;
  pin(x);  // no multiply-add with the difference
  const float far = (x - fmaxf(m, kLowest)) + kQ4Room, near = __builtin_fmaf(score, fac, kQ4Room - fmaxf(m, kLowest));
  return __builtin_amdgcn_exp2f(q4_is_far(m) ? far : near);
}

// Whether the wave runs again: a result is an infinity or NaN, or a row's maximum is far.
template <int NT>
__device__ __forceinline__ bool q4_again(const floatx4 (&acc)[NT][8], const float (&m)[NT]) {
  float bad = 0.0f;
  bool far = false;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    far |= q4_is_far(m[t]);
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) bad += acc[t][n][i] * 0.0f;
  }
  return __builtin_amdgcn_ballot_w64(far | (bad != 0.0f)) != 0;
}

// The wave's results and sums, without the operands' powers of two.
template <int NT>
__device__ __forceinline__ void q4_done(Q4Wave<NT>& w, const floatx4 (&acc)[NT][8]) {
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    w.l[t] = sum_xor32(sum_xor16(w.l[t])) * __builtin_amdgcn_exp2f(-kQ4Room);
#pragma unroll
    for (int n = 0; n < 8; ++n) w.o[t][n] = acc[t][n] * ((n & 1 ? 0.0625f : 1.0f) * __builtin_amdgcn_exp2f(-kQ4Room));
  }
}

// kSlots: pairs of blocks a wave holds; each half (K, V) is loaded again as soon as it is used up.
// q(t, p, part): the operand of tile t.
// begin(): the wave's q and rows, made ready while the first blocks are on their way.
// kFast false: only the two runs of a wave whose fast one, made elsewhere, does not do (q4_again).
template <int NT, int kSlots, bool kLong, int kPolicy, bool kFast, typename Q, typename Begin>
__device__ __forceinline__ void q4_attend(Q4Wave<NT>& w, const q4_t* __restrict__ kc, const q4_t* __restrict__ vc,
                                          const uint32_t* __restrict__ pt, uint32_t b0, uint32_t nblk,
                                          uint32_t bpp_shift, uint32_t kh, uint32_t hkv, const Q4Rows<NT>& rows, int lane,
                                          Q q, Begin begin) {
  const uint32_t bpp_mask = (1u << bpp_shift) - 1u;
  const size_t head_bytes = static_cast<size_t>(kQ4Block) << bpp_shift;

  // Page ids: kLong false, at most 64 blocks, a lane per block; else read a pair ahead of its use.
  int pid = 0;
  uint32_t ahead[2] = {0, 0};
  auto page_at = [&](uint32_t b) -> uint32_t {
    return pt[__builtin_amdgcn_readfirstlane((b0 + (b < nblk ? b : nblk - 1)) >> bpp_shift)];
  };
  struct Where {
    size_t off;
    bool valid;
  };
  auto where = [&](uint32_t b, int h) -> Where {
    const bool valid = b < nblk;
    uint32_t page;
    if constexpr (kLong) {
      page = ahead[h];
      ahead[h] = page_at(b + 2);
    } else {
      page = static_cast<uint32_t>(__builtin_amdgcn_readlane(pid, static_cast<int>(b & 63)));
    }
    return {(static_cast<size_t>(page) * hkv + kh) * head_bytes + ((b0 + b) & bpp_mask) * kQ4Block, valid};
  };
  Q4Half k[kSlots][2], v[kSlots][2];
  Where at[kSlots][2];  // of the blocks whose V is to be loaded
  auto load_k = [&](int s, uint32_t b) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      at[s][h] = where(b + h, h);
      q4_load<kPolicy>(k[s][h], kc + at[s][h].off, at[s][h].valid, lane);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto load_v = [&](int s) {
#pragma unroll
    for (int h = 0; h < 2; ++h) q4_load<kPolicy>(v[s][h], vc + at[s][h].off, at[s][h].valid, lane);
    __builtin_amdgcn_sched_barrier(0);
  };
  const int key_end = static_cast<int>((b0 + nblk) * 16);
  uint32_t exponent = 0x64006400u;
  __asm__("" : "+v"(exponent));
  floatx4 acc[NT][8];
  uint32_t poison[NT];  // groups in which a row sees a step of NaN (slow runs)
#pragma unroll
  for (int t = 0; t < NT; ++t) poison[t] = 0;

  // One run over the blocks: all steps (kSlow false), or those from 1 up (scaled 2^-12), or the others,
  // onto the first's results and with its maxima.
  auto pass = [&](auto slow, bool small) {
    constexpr bool kSlow = decltype(slow)::value;
    if (nblk) {
      if constexpr (kLong) {
        ahead[0] = page_at(0);
        ahead[1] = page_at(1);
      } else {
        pid = static_cast<uint32_t>(lane) < nblk ? static_cast<int>(pt[(b0 + lane) >> bpp_shift]) : 0;
      }
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        load_k(s, 2 * s);
        load_v(s);
      }
    }
    if constexpr (!kSlow) begin();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (!small) w.m[t] = -INFINITY;
      w.l[t] = 0.0f;
#pragma unroll
      for (int n = 0; n < 8; ++n) acc[t][n] = small ? acc[t][n] * 0x1p12f : floatx4{0, 0, 0, 0};
    }
    // A pair of blocks; false: the maxima moved, once more (kSlots 1: so the loop's own path has one
    // set of registers for the results; a branch around the scaling within it costs a move each).
    auto compute = [&](int s, uint32_t b, bool masked) -> bool {  // masked: uniform
      const int key0 = static_cast<int>((b0 + b) * 16) + 4 * (lane >> 4);
      u32x4 ph[NT], pl[NT];
      floatx4 sc[NT][2];
      float top[NT];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[t][h] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const half8 ka = q4_k_codes(k[s][h].codes[p], exponent);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            floatx4 d = {0, 0, 0, 0};
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q(t, p, 0), d, 0, 0, 0);
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q(t, p, 1), d, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float step = static_cast<float>(__builtin_bit_cast(half8, k[s][h].steps[i >> 1])[(i & 1) * 4 + p]);
              sc[t][h][i] = __builtin_fmaf(step, d[i], sc[t][h][i]);
            }
          }
        }
      }
      if (masked) {
        int first = key0;  // known here only: a branch, with no comparison of it in every pair
        pin(first);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int key = first + (e >> 2) * 16 + (e & 3);
            if (!((key >= rows.lo[t]) & (key <= rows.pos[t]) & (key < key_end))) sc[t][e >> 2][e & 3] = -INFINITY;
          }
      }
      bool moved = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        top[t] = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) top[t] = fmaxf(top[t], sc[t][e >> 2][e & 3]);
        top[t] *= rows.fac[t];
        moved |= top[t] > w.m[t] + kQ4Lazy;
      }
      if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float mn = fmaxf(w.m[t], max_xor32(max_xor16(top[t])));
          const float corr = __builtin_amdgcn_exp2f(w.m[t] - fmaxf(mn, kLowest));
          w.m[t] = mn;
          w.l[t] *= corr;
#pragma unroll
          for (int n = 0; n < 8; ++n) acc[t][n] *= corr;
        }
        if constexpr (kSlots == 1) return false;
      }
      load_k(s, b + 2 * kSlots);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[8];
        const float base = kQ4Room - fmaxf(w.m[t], kLowest);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (kSlow) x[e] = q4_slow_weight(sc[t][e >> 2][e & 3], rows.fac[t], w.m[t]);
          else x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][e >> 2][e & 3], rows.fac[t], base));
          w.l[t] += x[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t hi, lo;
          q4_cut(x[2 * e], x[2 * e + 1], hi, lo);
          ph[t][e] = hi;
          pl[t][e] = lo;
        }
        if constexpr (kSlow) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              const float step = static_cast<float>(__builtin_bit_cast(half8, v[s][e >> 2].steps[p >> 1])[(p & 1) * 4 + (e & 3)]);
              const int key = key0 + (e >> 2) * 16 + (e & 3);
              const bool ok = (key >= rows.lo[t]) & (key <= rows.pos[t]) & (key < key_end);
              if (!(fabsf(step) < INFINITY) && ok) poison[t] |= 1u << p;
            }
        }
      }
      if constexpr (kSlow) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            half8 st = __builtin_bit_cast(half8, v[s][h].steps[j]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float f = fabsf(static_cast<float>(st[e]));
              const _Float16 big = st[e] * static_cast<_Float16>(0x1p-12f);
              st[e] = small ? (f < 1.0f ? st[e] : static_cast<_Float16>(0.0f))
                            : (f >= 1.0f && f < INFINITY ? big : static_cast<_Float16>(0.0f));
            }
            v[s][h].steps[j] = __builtin_bit_cast(u32x4, st);
          }
      }
      if (masked) {  // keys no row sees
        int first = key0;
        pin(first);
        u32x2 seen[2];        // [block][keys 2 h, 2 h + 1]
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const int key = first + (e >> 2) * 16 + (e & 3);
          const auto in = [&](int x) { return x >= rows.any_lo && x <= rows.any_pos; };
          seen[e >> 2][(e >> 1) & 1] = (in(key) ? 0xffffu : 0u) | (in(key + 1) ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[s][h].steps[j >> 2][j & 3] &= seen[h][j & 1];
      }
      // V: halves of the four keys' dwords brought together, [block][keys 2 h, 2 h + 1][tiles 0-3, 4-7].
      uint32_t vr[2][2][2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          vr[j][h][0] = __builtin_amdgcn_perm(v[s][j].codes[2 * h + 1], v[s][j].codes[2 * h], 0x05040100u);
          vr[j][h][1] = __builtin_amdgcn_perm(v[s][j].codes[2 * h + 1], v[s][j].codes[2 * h], 0x07060302u);
        }
      auto tile = [&](auto nc) {
        constexpr int n = decltype(nc)::value, p = n >> 1;
        u32x4 hi, lo;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t word = vr[j][h][n >> 2];
            const half2_q4 c = q4_codes<(n & 1) != 0>((n & 2) ? word >> 8 : word, exponent);
            const half2_q4 st = __builtin_bit_cast(half2_q4, static_cast<uint32_t>(v[s][j].steps[p >> 1][(p & 1) * 2 + h]));
            uint32_t product = __builtin_bit_cast(uint32_t, c * st);
            pin(product);
            hi[2 * j + h] = product;
            lo[2 * j + h] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c, st, -__builtin_bit_cast(half2_q4, product)));
          }
        const half8 vh = __builtin_bit_cast(half8, hi), vl = __builtin_bit_cast(half8, lo);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const half8 a = __builtin_bit_cast(half8, ph[t]), b2 = __builtin_bit_cast(half8, pl[t]);
          acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, a, acc[t][n], 0, 0, 0);
          acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, b2, acc[t][n], 0, 0, 0);
          acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, a, acc[t][n], 0, 0, 0);
        }
      };
      tile(std::integral_constant<int, 0>{});
      tile(std::integral_constant<int, 1>{});
      tile(std::integral_constant<int, 2>{});
      tile(std::integral_constant<int, 3>{});
      tile(std::integral_constant<int, 4>{});
      tile(std::integral_constant<int, 5>{});
      tile(std::integral_constant<int, 6>{});
      tile(std::integral_constant<int, 7>{});
      load_v(s);
      return true;
    };
    auto whole = [&](uint32_t b) {  // every row sees every key of the pair
      const int key0 = static_cast<int>((b0 + b) * 16);
      return key0 >= rows.all_lo && key0 + 31 <= rows.all_pos && key0 + 32 <= key_end;
    };
    if constexpr (kSlots == 1) {
      for (uint32_t b = 0; b < nblk;)
        if (compute(0, b, !whole(b))) b += 2;
    } else {
      for (uint32_t b = 0; b < nblk; b += 2 * kSlots) {
#pragma unroll
        for (int s = 0; s < kSlots; ++s) compute(s, b + 2 * s, !whole(b + 2 * s));
      }
    }
  };
  if constexpr (kFast) pass(std::false_type{}, false);
  if (!kFast || q4_again<NT>(acc, w.m)) {
    pass(std::true_type{}, false);
    pass(std::true_type{}, true);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      uint32_t seen = poison[t];
      seen |= static_cast<uint32_t>(__shfl_xor(static_cast<int>(seen), 16));
      seen |= static_cast<uint32_t>(__shfl_xor(static_cast<int>(seen), 32));
#pragma unroll
      for (int n = 0; n < 8; ++n)
        if (seen >> (n >> 1) & 1) acc[t][n] = floatx4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
    }
  }
  q4_done<NT>(w, acc);
}

// This lane's part of a wave's rows: tile t's column is logical row lr0 + 16 t + c. First the loads
// of its position and q (dims 32 p + 8 g + 0 .. 7), unconditional, of a valid row.
template <int NT>
struct Q4Raw {
  int pos[NT];
  float4 q[NT][8];
};
template <int NT>
__device__ __forceinline__ void q4_rows_load(Q4Raw<NT>& raw, uint32_t lr0, uint32_t r0, uint32_t nlog, uint32_t kh,
                                             uint32_t G, uint32_t hq, const uint32_t* pos, const float* q, int lane) {
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const uint32_t lr = lr0 + t * 16 + (lane & 15), lrc = lr < nlog ? lr : 0;
    const uint32_t rr = r0 + lrc / G, h = kh * G + lrc % G;
    raw.pos[t] = static_cast<int>(pos[rr]);
    const float* src = q + (static_cast<size_t>(rr) * hq + h) * kD + (lane >> 4) * 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      raw.q[t][2 * j] = *reinterpret_cast<const float4*>(src + j * 32);
      raw.q[t][2 * j + 1] = *reinterpret_cast<const float4*>(src + j * 32 + 4);
    }
  }
  // Issued here (q and pos are not declared __restrict__ and the empty asm may write memory), so
  // that waiting for them waits for nothing issued after.
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// The least value of a row of 16 lanes, in each of them.
__device__ __forceinline__ int row16_min(int v) {
  v = min(v, __builtin_amdgcn_update_dpp(v, v, 0xb1, 0xf, 0xf, false));   // lanes 1, 0, 3, 2
  v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x4e, 0xf, 0xf, false));   // 2, 3, 0, 1
  v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xf, 0xf, false));  // mirrored in eights
  return min(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xf, 0xf, false));  // in the row
}

// Then the rows' keys, and q cut, a tile at a time: keep(t, hi, lo). A column without a row has the
// item's first row's q and sees no key.
template <int NT, typename Keep>
__device__ __forceinline__ void q4_rows(Q4Rows<NT>& rows, Q4Raw<NT>& raw, uint32_t lr0, uint32_t nlog,
                                        uint32_t window, float scale_log2, int lane, Keep keep) {
  int all_lo = 0, all_pos = 0x7fffffff, any_lo = 0x7fffffff, any_pos = -1;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const bool has = lr0 + t * 16 + (lane & 15) < nlog;
    const int p = raw.pos[t];
    rows.has[t] = has;
    rows.pos[t] = has ? p : -1;
    rows.lo[t] = (window > 0 && p + 1 > static_cast<int>(window)) ? p + 1 - static_cast<int>(window) : 0;
    u32x4 hi[4], lo[4];
    rows.fac[t] = q4_cut_q(raw.q[t], scale_log2, hi, lo);
    keep(t, hi, lo);
    if (has) {
      all_lo = max(all_lo, rows.lo[t]);
      any_lo = min(any_lo, rows.lo[t]);
      all_pos = min(all_pos, p);
      any_pos = max(any_pos, p);
    }
  }
  rows.all_lo = -__builtin_amdgcn_readfirstlane(row16_min(-all_lo));
  rows.any_lo = __builtin_amdgcn_readfirstlane(row16_min(any_lo));
  rows.all_pos = __builtin_amdgcn_readfirstlane(row16_min(all_pos));
  rows.any_pos = -__builtin_amdgcn_readfirstlane(row16_min(-any_pos));
}

// Decode and verify: a work item's blocks dealt evenly over W waves: 8, one item to a CU, or 4, two
// (build_plan chooses). Items, hand-off and merge are those of the binary16 arena's 16-row-tile kernel. q lies in LDS, since its parts of two
// tiles are 64 registers, and is cut while the first blocks are on their way.
// 16 x 4096 keys, 16/4 heads: 15.4 us, of which 2.3 to q and the first blocks, 0.9 q's cut, 6.5 the blocks (four
// pairs a wave, two waves a SIMD: about 300 vector instructions a pair bind them, not the 2.4 TB/s), 2 until
// the slowest wave's results are in LDS, 1.2 the hand-off. 4 x 131072, 32/8 heads: 145 us, 4.2 TB/s. Two
// tiles (16 x 5 rows): 27.8 us.
template <int NT, int W>
struct Q4Shared {
  float m[W][NT * 16];
  float l[W][NT * 16];
  float4 o[W][NT * 16][kD / 4];
  uint32_t last;
};

template <int NT, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_attn_decode_q4(
    const AttnItem* __restrict__ items, const uint32_t* pos, const uint32_t* __restrict__ pages,
    const q4_t* __restrict__ kc, const q4_t* __restrict__ vc, const float* q, float* __restrict__ out,
    float* __restrict__ part_o, float2* __restrict__ part_ml, uint32_t* __restrict__ counters, uint32_t part_o_bytes,
    uint32_t part_ml_bytes, uint32_t hq, uint32_t hkv, uint32_t bpp_shift, uint32_t window, float scale_log2,
    const SubRef* __restrict__ members, uint32_t by_item) {
  __shared__ Q4Shared<NT, W> sh;
  const AttnItem it = items[by_item ? blockIdx.y : blockIdx.x];
  const uint32_t kh = by_item ? blockIdx.x : blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const uint32_t G = hq / hkv;
  const uint32_t nlog = it.nrows * G;  // at most NT * 16
  const uint32_t nall = it.blk1 - it.blk0;
  const uint32_t wb0 = it.blk0 + nall * wave / W;
  const uint32_t wb1 = it.blk0 + nall * (wave + 1) / W;

  Q4Rows<NT> rows;
  Q4Wave<NT> w;
  // q in LDS, in the space of the waves' results.
  half8* const qs = reinterpret_cast<half8*>(&sh.o[0][0][0]);
  static_assert(sizeof(sh.o) >= NT * 8 * 64 * sizeof(half8), "q fits");
  Q4Raw<NT> raw;
  q4_rows_load<NT>(raw, 0, it.r0, nlog, kh, G, hq, pos, q, lane);
  q4_attend<NT, NT == 1 ? 2 : 1, false, kNontemporal, true>(
      w, kc, vc, pages + it.pt_off, wb0, wb1 - wb0, bpp_shift, kh, hkv, rows, lane,
      [&](int t, int p, int part) { return qs[(t * 8 + part * 4 + p) * 64 + lane]; },
      [&]() {
        q4_rows<NT>(rows, raw, 0, nlog, window, scale_log2, lane, [&](int t, const u32x4* hi, const u32x4* lo) {
          if (wave == t)
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              qs[(t * 8 + p) * 64 + lane] = __builtin_bit_cast(half8, hi[p]);
              qs[(t * 8 + 4 + p) * 64 + lane] = __builtin_bit_cast(half8, lo[p]);
            }
        });
        lds_barrier();
      });
  __syncthreads();  // every wave is done with q before any writes its result over it
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int lr = t * 16 + c;
    if (g == 0) {
      sh.m[wave][lr] = w.m[t];
      sh.l[wave][lr] = w.l[t];
    }
    if (rows.has[t])
#pragma unroll
      for (int n = 0; n < 8; ++n) sh.o[wave][lr][n * 4 + g] = __builtin_bit_cast(float4, w.o[t][n]);
  }
  __syncthreads();
  finish_item<64 * W, NT * 16, true>(it, kh, G, hq, hkv, nlog, out, part_o, part_ml, counters, part_o_bytes,
                                              part_ml_bytes, sh.last,
                                              [&](uint32_t lr, uint32_t qi, float& mt, float& lt, float4& o) {
    mt = -INFINITY;
#pragma unroll
    for (int v = 0; v < W; ++v) mt = fmaxf(mt, sh.m[v][lr]);
    lt = 0.0f;
    o = float4{0, 0, 0, 0};
    const float mf = fmaxf(mt, kLowest);
#pragma unroll
    for (int v = 0; v < W; ++v) {
      const float wt = __builtin_amdgcn_exp2f(sh.m[v][lr] - mf);  // 0 for an empty wave
      lt += sh.l[v][lr] * wt;
      const float4 ow = sh.o[v][lr][qi];
      o.x += ow.x * wt;
      o.y += ow.y * wt;
      o.z += ow.z * wt;
      o.w += ow.w * wt;
    }
  }, members);
}

// Prefill: a tile of kQ4TileRows logical rows, NT tiles of 16 to each of 4 waves, over the item's
// blocks. A pair of blocks is made into operands once for the four waves: K's codes (a dword of each
// lane, group p by wave p) and V's hi and lo parts (tiles 2 w, 2 w + 1, which share group w's steps),
// through LDS, two pairs deep with one barrier a pair. q is in registers.
// 512 rows after 24000 keys, 20/4 heads: 318 us (each wave by itself converting, q in LDS: 360). What bounds it is
// the waves' own order of instructions: 80 matrix instructions (1280 cycles), 256 vector and 28 LDS
// ones a pair take a wave 4000 cycles alone and two of a SIMD 5000 each. Four tiles a wave spill.
static constexpr int kQ4TileWaves = 4;
static constexpr int kQ4WaveTiles = 2;
static constexpr int kQ4TileRows = kQ4TileWaves * kQ4WaveTiles * 16;

// A pair's operands.
struct Q4Stage {
  half8 k[2][4][64];       // [block][group][lane]
  half8 v[8][2][64];       // [tile][hi, lo][lane]
  u32x4 steps[2][8];       // K's, [block][two keys' four groups]
};

// What a wave loads of a pair to make its share of them.
struct Q4Share {
  u32x4 v[2];
  u32x2 vsteps[2];
  uint32_t k[2], ksteps;
};

// Of two waves of a SIMD the older goes first and leaves the other to run alone at the end (512 rows
// after 24000 keys: 225 and 295 us). A wave with fewer blocks left gives way, so both end close to
// each other (265 and 280).
__device__ __forceinline__ void q4_priority(uint32_t left) {
  if (left > 96) __builtin_amdgcn_s_setprio(3);
  else if (left > 32) __builtin_amdgcn_s_setprio(2);
  else if (left > 8) __builtin_amdgcn_s_setprio(1);
  else __builtin_amdgcn_s_setprio(0);
}

__global__ __launch_bounds__(64 * kQ4TileWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_attn_prefill_q4(
    const PrefillItem* __restrict__ items, const uint32_t* pos, const uint32_t* __restrict__ pages,
    const q4_t* __restrict__ kc, const q4_t* __restrict__ vc, const float* q, float* __restrict__ out,
    uint32_t hq, uint32_t hkv, uint32_t bpp_shift, uint32_t window, float scale_log2, float* __restrict__ part_o,
    float2* __restrict__ part_ml, uint32_t* __restrict__ counters, uint32_t part_o_bytes, uint32_t part_ml_bytes) {
  constexpr int NT = kQ4WaveTiles;
  __shared__ Q4Stage stages[2];
  __shared__ int seen_lo[kQ4TileWaves], seen_pos[kQ4TileWaves];
  const PrefillItem it = items[blockIdx.x / hkv];
  const uint32_t kh = blockIdx.x % hkv;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const uint32_t G = hq / hkv;
  const uint32_t nlog = it.nrows * G;  // at most kQ4TileRows
  const uint32_t* const pt = pages + it.pt_off;
  const uint32_t nblk = it.blk1 - it.blk0;
  const uint32_t bpp_mask = (1u << bpp_shift) - 1u;
  const size_t head_bytes = static_cast<size_t>(kQ4Block) << bpp_shift;

  // Page ids are read a pair ahead of their use.
  auto page_at = [&](uint32_t b) -> uint32_t {
    return pt[__builtin_amdgcn_readfirstlane((it.blk0 + (b < nblk ? b : nblk - 1)) >> bpp_shift)];
  };
  uint32_t ahead[2] = {page_at(0), page_at(1)};
  Q4Share share;
  size_t off[2];  // of the pair being loaded
  int bytes[2];
  auto locate = [&](uint32_t b) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t page = ahead[h];
      ahead[h] = page_at(b + h + 2);
      const bool valid = b + h < nblk;
      off[h] = (static_cast<size_t>(page) * hkv + kh) * head_bytes + ((it.blk0 + b + h) & bpp_mask) * kQ4Block;
      bytes[h] = valid ? static_cast<int>(kQ4Block) : 0;
    }
  };
  auto load_k = [&]() {
    __amdgpu_buffer_rsrc_t rs[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      rs[h] = __builtin_amdgcn_make_buffer_rsrc(const_cast<q4_t*>(kc + off[h]), 0, bytes[h], 0x00020000);
      share.k[h] = __builtin_amdgcn_raw_buffer_load_b32(rs[h], lane * 16, wave * 4, 0);
    }
    share.ksteps = __builtin_amdgcn_raw_buffer_load_b32((wave & 1) ? rs[1] : rs[0], static_cast<int>(kQ4Steps) + (lane & 31) * 4, 0, 0);
  };
  auto load_v = [&]() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<q4_t*>(vc + off[h]), 0, bytes[h], 0x00020000);
      share.v[h] = __builtin_amdgcn_raw_buffer_load_b128(rs, lane * 16, 0, 0);
      share.vsteps[h] = __builtin_amdgcn_raw_buffer_load_b64(rs, static_cast<int>(kQ4Steps) + g * 32, wave * 8, 0);
    }
  };
  auto load = [&](uint32_t b) {
    locate(b);
    load_k();
    load_v();
  };
  load(0);

  Q4Rows<NT> rows;
  half8 qa[NT][2][4];
  {
    Q4Raw<NT> raw;
    q4_rows_load<NT>(raw, wave * NT * 16, it.r0, nlog, kh, G, hq, pos, q, lane);
    q4_rows<NT>(rows, raw, wave * NT * 16, nlog, window, scale_log2, lane, [&](int t, const u32x4* hi, const u32x4* lo) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        qa[t][0][p] = __builtin_bit_cast(half8, hi[p]);
        qa[t][1][p] = __builtin_bit_cast(half8, lo[p]);
      }
    });
  }
  if (lane == 0) {
    seen_lo[wave] = rows.any_lo;
    seen_pos[wave] = rows.any_pos;
  }
  lds_barrier();
  int any_lo = seen_lo[0], any_pos = seen_pos[0];  // keys that some row of the tile sees
#pragma unroll
  for (int v = 1; v < kQ4TileWaves; ++v) {
    any_lo = min(any_lo, seen_lo[v]);
    any_pos = max(any_pos, seen_pos[v]);
  }
  any_lo = __builtin_amdgcn_readfirstlane(any_lo);
  any_pos = __builtin_amdgcn_readfirstlane(any_pos);

  uint32_t exponent = 0x64006400u;
  __asm__("" : "+v"(exponent));
  const uint32_t byte_sel = 0x0c000c00u | static_cast<uint32_t>(wave) | static_cast<uint32_t>(wave + 4) << 16;
  // This wave's share of a pair, made into operands: steps of keys no row sees cleared, then four
  // pieces (K's two blocks, V's two tiles).
  auto clear = [&](uint32_t b) {
    const int first = static_cast<int>((it.blk0 + b) * 16);
    if (first >= any_lo && first + 31 <= any_pos) return;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int key = first + h * 16 + 4 * g + 2 * j;
        const auto in = [&](int x) { return x >= any_lo && x <= any_pos; };
        share.vsteps[h][j] &= (in(key) ? 0xffffu : 0u) | (in(key + 1) ? 0xffff0000u : 0u);
      }
  };
  auto make = [&](auto piece, Q4Stage& st) {
    constexpr int kPiece = decltype(piece)::value;
    if constexpr (kPiece < 2) {
      st.k[kPiece][wave][lane] = q4_k_codes(share.k[kPiece], exponent);
      if constexpr (kPiece == 0) reinterpret_cast<uint32_t*>(st.steps)[(wave & 1) * 32 + (lane & 31)] = share.ksteps;
    } else {
      constexpr int n = kPiece - 2;
      u32x4 hi, lo;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t word = __builtin_amdgcn_perm(share.v[j][2 * h + 1], share.v[j][2 * h], byte_sel);
          const half2_q4 x = q4_codes<n != 0>(word, exponent);
          const half2_q4 step = __builtin_bit_cast(half2_q4, static_cast<uint32_t>(share.vsteps[j][h]));
          uint32_t product = __builtin_bit_cast(uint32_t, x * step);
          pin(product);
          hi[2 * j + h] = product;
          lo[2 * j + h] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(x, step, -__builtin_bit_cast(half2_q4, product)));
        }
      st.v[2 * wave + n][0][lane] = __builtin_bit_cast(half8, hi);
      st.v[2 * wave + n][1][lane] = __builtin_bit_cast(half8, lo);
    }
  };
  auto convert = [&](Q4Stage& st, uint32_t b) {
    clear(b);
    make(std::integral_constant<int, 0>{}, st);
    make(std::integral_constant<int, 1>{}, st);
    make(std::integral_constant<int, 2>{}, st);
    make(std::integral_constant<int, 3>{}, st);
  };

  Q4Wave<NT> w;
  floatx4 acc[NT][8];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    w.m[t] = -INFINITY;
    w.l[t] = 0.0f;
#pragma unroll
    for (int n = 0; n < 8; ++n) acc[t][n] = floatx4{0, 0, 0, 0};
  }
  const int key_end = static_cast<int>(it.blk1 * 16);
  u32x4 ph[NT], pl[NT];
  float corr[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) corr[t] = 1.0f;
  // A pair's weights; false: the maxima moved, the results are to be scaled by corr.
  auto weights = [&](const Q4Stage& st, int first, bool masked) -> bool {
    floatx4 sc[NT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const half8 steps[2] = {__builtin_bit_cast(half8, st.steps[h][2 * g]), __builtin_bit_cast(half8, st.steps[h][2 * g + 1])};
#pragma unroll
      for (int t = 0; t < NT; ++t) sc[t][h] = floatx4{0, 0, 0, 0};
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const half8 ka = st.k[h][p][lane];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          floatx4 d = {0, 0, 0, 0};
          d = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qa[t][0][p], d, 0, 0, 0);
          d = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qa[t][1][p], d, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sc[t][h][i] = __builtin_fmaf(static_cast<float>(steps[i >> 1][(i & 1) * 4 + p]), d[i], sc[t][h][i]);
        }
      }
    }
    if (masked) {
      int key0 = first + 4 * g;  // known here only: a branch, with no comparison of it in every pair
      pin(key0);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = key0 + (e >> 2) * 16 + (e & 3);
          if (!((key >= rows.lo[t]) & (key <= rows.pos[t]) & (key < key_end))) sc[t][e >> 2][e & 3] = -INFINITY;
        }
    }
    float top[NT];
    bool moved = false;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      top[t] = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) top[t] = fmaxf(top[t], sc[t][e >> 2][e & 3]);
      top[t] *= rows.fac[t];
      moved |= top[t] > w.m[t] + kQ4Lazy;
    }
    if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float mn = fmaxf(w.m[t], max_xor32(max_xor16(top[t])));
        corr[t] = __builtin_amdgcn_exp2f(w.m[t] - fmaxf(mn, kLowest));
        w.m[t] = mn;
        w.l[t] *= corr[t];
      }
      return false;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float x[8];
      const float base = kQ4Room - fmaxf(w.m[t], kLowest);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][e >> 2][e & 3], rows.fac[t], base));
        w.l[t] += x[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t hi, lo;
        q4_cut(x[2 * e], x[2 * e + 1], hi, lo);
        ph[t][e] = hi;
        pl[t][e] = lo;
      }
    }
    return true;
  };
  convert(stages[0], 0);
  load(2);
  lds_barrier();
  // The pairs some row of this wave sees; for the tile's others it makes operands alone.
  const bool some = rows.any_pos >= 0;
  const uint32_t b0 = some ? max(it.blk0, static_cast<uint32_t>(rows.any_lo) / 16) - it.blk0 : nblk;
  const uint32_t b1 = some ? min(it.blk1, max(it.blk0, static_cast<uint32_t>(rows.any_pos) / 16 + 1)) - it.blk0 : 0;
  const uint32_t p0 = min(b0, nblk) / 2 * 2;
  uint32_t b = 0;
  auto others = [&](uint32_t end) {
    for (; b < end; b += 2) {
      convert(stages[((b >> 1) & 1) ^ 1], b + 2);
      load(b + 4);
      lds_barrier();
    }
  };
  q4_priority(nblk);
  others(p0);
  // Where the maxima move, the inner loop ends, the results are scaled and the pair is looked at once
  // more: so the inner loop has one set of registers for the results, with no moves.
  for (bool moved = b < b1; moved;) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int n = 0; n < 8; ++n) acc[t][n] *= corr[t];
    moved = false;
    while (b < b1) {
      const Q4Stage& st = stages[(b >> 1) & 1];
      const int first = static_cast<int>((it.blk0 + b) * 16);
      moved = !weights(st, first, !(first >= rows.all_lo && first + 31 <= rows.all_pos && first + 32 <= key_end));
      if (moved) break;
      clear(b + 2);
      Q4Stage& next = stages[((b >> 1) & 1) ^ 1];
      // V's operands are read a tile ahead, the next pair's are made in the shadow of the products.
      half8 vh = st.v[0][0][lane], vl = st.v[0][1][lane];
      auto tile = [&](auto nc) {
        constexpr int n = decltype(nc)::value;
        __builtin_amdgcn_sched_barrier(0);
        const half8 h = vh, l = vl;
        if constexpr (n < 7) {
          vh = st.v[n + 1][0][lane];
          vl = st.v[n + 1][1][lane];
        }
        if constexpr ((n & 1) == 0) make(std::integral_constant<int, n / 2>{}, next);
        if constexpr (n == 1) locate(b + 4);
        if constexpr (n == 3) load_k();
        if constexpr (n == 7) load_v();
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, __builtin_bit_cast(half8, ph[t]), acc[t][n], 0, 0, 0);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, __builtin_bit_cast(half8, pl[t]), acc[t][n], 0, 0, 0);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l, __builtin_bit_cast(half8, ph[t]), acc[t][n], 0, 0, 0);
      };
      tile(std::integral_constant<int, 0>{});
      tile(std::integral_constant<int, 1>{});
      tile(std::integral_constant<int, 2>{});
      tile(std::integral_constant<int, 3>{});
      tile(std::integral_constant<int, 4>{});
      tile(std::integral_constant<int, 5>{});
      tile(std::integral_constant<int, 6>{});
      tile(std::integral_constant<int, 7>{});
      __builtin_amdgcn_sched_barrier(0);
      lds_barrier();
      b += 2;
      q4_priority(nblk - b);
    }
  }
  others(nblk);
  if (q4_again<NT>(acc, w.m)) {  // again, a tile at a time with q in LDS (the operands' space is free)
    half8 (*const qs)[64] = reinterpret_cast<half8 (*)[64]>(stages) + wave * 8;
    static_assert(sizeof(stages) >= kQ4TileWaves * 8 * sizeof(*qs), "q fits");
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        qs[p][lane] = qa[t][0][p];
        qs[4 + p][lane] = qa[t][1][p];
      }
      const Q4Rows<1> row = {{rows.has[t]}, {rows.pos[t]}, {rows.lo[t]}, {rows.fac[t]}, rows.all_lo, rows.all_pos, rows.any_lo, rows.any_pos};
      Q4Wave<1> one;
      q4_attend<1, 1, true, 0, false>(one, kc, vc, pt, it.blk0 + b0, b1 > b0 ? b1 - b0 : 0, bpp_shift, kh, hkv, row, lane,
                                      [&](int, int p, int part) { return qs[part * 4 + p][lane]; }, []() {});
      w.m[t] = one.m[0];
      w.l[t] = one.l[0];
#pragma unroll
      for (int n = 0; n < 8; ++n) w.o[t][n] = one.o[0][n];
    }
  } else {
    q4_done<NT>(w, acc);
  }
  const uint32_t nch = it.chunk_nch >> 16;
  if (nch <= 1) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (!rows.has[t]) continue;
      const uint32_t lr = (wave * NT + t) * 16 + c, rr = it.r0 + lr / G, h = kh * G + lr % G;
      float* o = out + (static_cast<size_t>(rr) * hq + h) * kD + g * 4;
      const float inv = 1.0f / w.l[t];
#pragma unroll
      for (int n = 0; n < 8; ++n) *reinterpret_cast<floatx4*>(o + n * 16) = w.o[t][n] * inv;
    }
    return;
  }
  // A tile split along keys: the hand-off of the other arenas' tiles (attn_prefill.hpp).
  const __amdgpu_buffer_rsrc_t ro = make_rsrc(part_o, part_o_bytes);
  const __amdgpu_buffer_rsrc_t rml = make_rsrc(part_ml, part_ml_bytes);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (!rows.has[t]) continue;
    const uint32_t lr = (wave * NT + t) * 16 + c;
    const size_t e = ((static_cast<size_t>(it.part_base) + (it.chunk_nch & 0xffffu)) * hkv + kh) * kQ4TileRows + lr;
#pragma unroll
    for (int n = 0; n < 8; ++n)
      st4_coherent(ro, static_cast<uint32_t>((e * kD + 16 * n + 4 * g) * 4), __builtin_bit_cast(float4, w.o[t][n]));
    if (g == 0) st2_coherent(rml, static_cast<uint32_t>(e * 8), float2{w.m[t], w.l[t]});
  }
  __builtin_amdgcn_s_waitcnt(0);
  __shared__ uint32_t last_chunk;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t* cnt = counters + (static_cast<size_t>(it.counter) * hkv + kh) * kCounterStride;
    const uint32_t arrived = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last_chunk = arrived == nch - 1;
    if (last_chunk) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last_chunk) return;
  merge_tile<64 * kQ4TileWaves, kQ4TileRows>(it.r0, it.nrows, it.part_base, nch, kh, G, hq, hkv, out, ro, rml);
}

}  // namespace yx
