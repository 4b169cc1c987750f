// Paged attention over a 4-bit arena (q4.hpp) for gfx950: decode and verify items, and prefill
// tiles.
//
// out = softmax(q K^T scale) V with K, V = s (code - 8), s the binary16 step of 32 dims. Codes and
// steps go into the matrix products apart, so that both stay exact (their product has 15 bits,
// more than a binary16 holds):
//   S[key] = sum_p s_p[key] sum_d q_d (code_d - 8)          p: a group of 32 dims
//     one v_mfma_f32_16x16x32_f16 per group and part of q, the codes as binary16 (below); then
//     one fused multiply-add per score and group;
//   O_d = sum_key (P s_p) (code_d - 8)
//     P s_p per group as a binary16 hi and lo part.
// q is scaled by a power of two of its row (its largest value near 2^12) before it is cut into hi
// and lo, so its size does not matter; both cuts keep ~2^-22. P s_p is cut at a fixed scale that
// holds steps below 8; where a larger one overflows it, the wave starts again at a scale that
// holds every binary16 (V beyond 64 in magnitude). A masked key has weight 0 and its step is left
// out, so whatever lies behind a sequence's last token has no effect, NaN steps included.
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

// One 16-key block of a lane: K and V codes, the steps of keys 4 g .. 4 g + 3 of both.
struct Q4Regs {
  u32x4 k, v, ks[2], vs[2];
};

template <int kPolicy>
__device__ __forceinline__ void q4_load(Q4Regs& r, const q4_t* kblk, const q4_t* vblk, bool valid, int lane) {
  const int bytes = valid ? static_cast<int>(kQ4Block) : 0;
  const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<q4_t*>(kblk), 0, bytes, 0x00020000);
  const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<q4_t*>(vblk), 0, bytes, 0x00020000);
  const int st = static_cast<int>(kQ4Steps) + (lane >> 4) * 32;
  r.k = __builtin_amdgcn_raw_buffer_load_b128(rk, lane * 16, 0, kPolicy);
  r.ks[0] = __builtin_amdgcn_raw_buffer_load_b128(rk, st, 0, kPolicy);
  r.ks[1] = __builtin_amdgcn_raw_buffer_load_b128(rk, st, 16, kPolicy);
  r.v = __builtin_amdgcn_raw_buffer_load_b128(rv, lane * 16, 0, kPolicy);
  r.vs[0] = __builtin_amdgcn_raw_buffer_load_b128(rv, st, 0, kPolicy);
  r.vs[1] = __builtin_amdgcn_raw_buffer_load_b128(rv, st, 16, kPolicy);
}

// Step of key 4 g + i, group p.
__device__ __forceinline__ float q4_step(const u32x4* s, int i, int p) {
  return static_cast<float>(__builtin_bit_cast(half8, s[i >> 1])[(i & 1) * 4 + p]);
}

// Two codes in the low nibbles of w's halves (kOdd: the second nibbles) less 8 (kOdd: 16 times
// that) as binary16: or-ed under the exponent of 1024 they read 1024 + code (1024 + 16 code), and
// the difference is exact. (As they lie, read as subnormals code * 2^-24, they would need no
// exponent, but the matrix unit aligns a subnormal's products by its nominal exponent and drops
// up to 7 of their bits: outputs 6e-6 off after 600 keys and 1.3e-5 after 4000, against 4e-7.)
template <bool kOdd>
__device__ __forceinline__ uint32_t q4_codes(uint32_t w) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  const h2 c = __builtin_bit_cast(h2, (w & (kOdd ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u);
  const _Float16 base = static_cast<_Float16>(kOdd ? 1152.0f : 1032.0f);
  return __builtin_bit_cast(uint32_t, c - h2{base, base});
}

// The codes of a K dword as a matrix operand (dims 32 p + 8 g + 0 .. 7; 2, 3, 6, 7 times 16).
__device__ __forceinline__ half8 q4_k_codes(uint32_t w) {
  return __builtin_bit_cast(half8, u32x4{q4_codes<false>(w), q4_codes<true>(w), q4_codes<false>(w >> 8), q4_codes<true>(w >> 8)});
}

// V dwords of four keys, halves brought together: r[h][0] has the dims of tiles 0 to 3 of keys
// 2 h and 2 h + 1, r[h][1] those of tiles 4 to 7.
__device__ __forceinline__ void q4_v_halves(const u32x4& v, uint32_t (&r)[2][2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    r[h][0] = __builtin_amdgcn_perm(v[2 * h + 1], v[2 * h], 0x05040100u);
    r[h][1] = __builtin_amdgcn_perm(v[2 * h + 1], v[2 * h], 0x07060302u);
  }
}

// Tile n's codes of keys 2 h and 2 h + 1 (odd n: times 16).
template <int n>
__device__ __forceinline__ uint32_t q4_v_codes(const uint32_t (&r)[2]) {
  return q4_codes<(n & 1) != 0>(r[n >> 2] >> (8 * ((n >> 1) & 1)));
}

// Two values as a binary16 hi part and a lo part each. The values and the hi parts are pinned: the
// compiler would otherwise take hi from the unrounded product y comes from in one place and from y
// in the other, which differ by a last bit now and then.
__device__ __forceinline__ void q4_cut(float y0, float y1, uint32_t& hi, uint32_t& lo) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  pin(y0);
  pin(y1);
  hi = __builtin_bit_cast(uint32_t, h2{static_cast<_Float16>(y0), static_cast<_Float16>(y1)});
  pin(hi);
  const h2 h = __builtin_bit_cast(h2, hi);
  lo = __builtin_bit_cast(uint32_t, h2{static_cast<_Float16>(y0 - static_cast<float>(h.x)), static_cast<_Float16>(y1 - static_cast<float>(h.y))});
}

// Weights are 2^(room + x - m), x and m in log2, and x > m + kQ4Lazy moves m. As high as binary16
// allows, since parts of weights below its smallest normal value lose bits: where one key
// outweighs 4000 others, outputs were 1e-5 off with the maximum moved by more than 8 only (and
// room 5), 2e-7 off like this.
static constexpr float kQ4Lazy = 2.0f;
static constexpr float kQ4Room = 11.0f;     // steps below 8 fit
static constexpr float kQ4RoomBig = -4.0f;  // any step fits

// What one wave attends: NT tiles of 16 logical rows over the blocks [b0, b0 + nblk) of a page
// table. rpos / rlo: the last and first key of this lane's column (rpos -1: no row).
template <int NT>
struct Q4Wave {
  float m[NT], l[NT];      // maximum (log2) and this lane's share of the sum
  floatx4 o[NT][8];        // unnormalised, dims 16 n + 4 g + i
};

template <int NT, int kPolicy>
__device__ __forceinline__ void q4_attend(Q4Wave<NT>& w, const q4_t* __restrict__ kc, const q4_t* __restrict__ vc,
                                          const uint32_t* __restrict__ pt, uint32_t b0, uint32_t nblk,
                                          uint32_t bpp_shift, uint32_t kh, uint32_t hkv, const float4 (&qraw)[NT][8],
                                          const bool (&has)[NT], const int (&rpos)[NT], const int (&rlo)[NT],
                                          float scale_log2, int lane) {
  const uint32_t bpp_mask = (1u << bpp_shift) - 1u;
  const size_t head_bytes = static_cast<size_t>(kQ4Block) << bpp_shift;

  // Page ids, a lane per block, 64 blocks at a time and the next 64 on their way.
  int pid = 0, pid_next = 0;
  uint32_t batch = 0;
  auto ids = [&](uint32_t k) -> int {
    const uint32_t b = 64 * k + static_cast<uint32_t>(lane);
    return b < nblk ? static_cast<int>(pt[(b0 + b) >> bpp_shift]) : 0;
  };
  auto load = [&](Q4Regs& r, uint32_t b) {
    const bool valid = b < nblk;
    if (valid && (b >> 6) != batch) {  // uniform
      pid = pid_next;
      batch = b >> 6;
      pid_next = ids(batch + 1);
    }
    const uint32_t page = static_cast<uint32_t>(__builtin_amdgcn_readlane(pid, static_cast<int>(b & 63)));
    const size_t off = valid ? (static_cast<size_t>(page) * hkv + kh) * head_bytes + ((b0 + b) & bpp_mask) * static_cast<size_t>(kQ4Block) : 0;
    q4_load<kPolicy>(r, kc + off, vc + off, valid, lane);
  };
  Q4Regs s0[2], s1[2];
  auto load_pair = [&](Q4Regs* r, uint32_t b) {
    load(r[0], b);
    load(r[1], b + 1);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto start = [&]() {
    batch = 0;
    pid = ids(0);
    pid_next = nblk > 64 ? ids(1) : 0;
    load_pair(s0, 0);
    load_pair(s1, 2);
  };
  if (nblk) start();

  // q as hi and lo parts, the factor from products to log2 scores.
  half8 qh[NT][4], ql[NT][4];
  float fac[NT];
  int wmin = 0x7fffffff, wlo = 0;  // keys that every row of this wave sees: [wlo, wmin]
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 a = qraw[t][j];
      top = fmaxf(top, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))));
    }
    top = max_xor32(max_xor16(top));
    const bool usable = has[t] && top > 0.0f && top < INFINITY;
    const int ex = usable ? __builtin_amdgcn_frexp_expf(top) : 0;  // top < 2^ex
    fac[t] = __builtin_ldexpf(scale_log2, ex - 13);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const float4 a = qraw[t][2 * p], b = qraw[t][2 * p + 1];
      const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = has[t] ? __builtin_ldexpf(x[e], 13 - ex) : 0.0f;
        const float part = (e & 2) ? v * 0.0625f : v;
        const _Float16 hi = static_cast<_Float16>(part);
        qh[t][p][e] = hi;
        ql[t][p][e] = static_cast<_Float16>(part - static_cast<float>(hi));
      }
    }
    int lo = has[t] ? rlo[t] : 0, hi = has[t] ? rpos[t] : 0x7fffffff;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      lo = max(lo, __shfl_xor(lo, o));
      hi = min(hi, __shfl_xor(hi, o));
    }
    wmin = min(wmin, __builtin_amdgcn_readfirstlane(hi));
    wlo = max(wlo, __builtin_amdgcn_readfirstlane(lo));
  }
  const int key_end = static_cast<int>((b0 + nblk) * 16);

  float room = kQ4Room;
  for (;;) {
    floatx4 acc[NT][8];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      w.m[t] = -INFINITY;
      w.l[t] = 0.0f;
#pragma unroll
      for (int n = 0; n < 8; ++n) acc[t][n] = floatx4{0, 0, 0, 0};
    }
    auto compute = [&](auto masked, const Q4Regs* r, int key0) {
      constexpr bool kMask = decltype(masked)::value;
      half8 ka[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int p = 0; p < 4; ++p) ka[h][p] = q4_k_codes(r[h].k[p]);
      uint32_t vr[2][2][2];
      q4_v_halves(r[0].v, vr[0]);
      q4_v_halves(r[1].v, vr[1]);
      auto v_tile = [&](auto n) -> half8 {
        constexpr int N = decltype(n)::value;
        return __builtin_bit_cast(half8, u32x4{q4_v_codes<N>(vr[0][0]), q4_v_codes<N>(vr[0][1]),
                                               q4_v_codes<N>(vr[1][0]), q4_v_codes<N>(vr[1][1])});
      };
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[8];
        bool ok[8];
        float top = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          floatx4 sc = {0, 0, 0, 0};
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            floatx4 d = {0, 0, 0, 0};
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[h][p], qh[t][p], d, 0, 0, 0);
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[h][p], ql[t][p], d, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[i] = __builtin_fmaf(q4_step(r[h].ks, i, p), d[i], sc[i]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = h * 4 + i;
            x[e] = sc[i] * fac[t];
            if constexpr (kMask) {
              const int key = key0 + h * 16 + 4 * (lane >> 4) + i;
              ok[e] = (key >= rlo[t]) & (key <= rpos[t]) & (key < key_end);
              x[e] = ok[e] ? x[e] : -INFINITY;
            }
            top = fmaxf(top, x[e]);
          }
        }
        if (__builtin_amdgcn_ballot_w64(top > w.m[t] + kQ4Lazy)) {
          const float mn = fmaxf(w.m[t], max_xor32(max_xor16(top)));
          const float corr = __builtin_amdgcn_exp2f(w.m[t] - fmaxf(mn, kLowest));
          w.m[t] = mn;
          w.l[t] *= corr;
#pragma unroll
          for (int n = 0; n < 8; ++n) acc[t][n] *= corr;
        }
        const float base = fmaxf(w.m[t], kLowest) - room;
        float pr[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          pr[e] = __builtin_amdgcn_exp2f(x[e] - base);
          w.l[t] += pr[e];
        }
        auto group = [&](auto pc) {
          constexpr int p = decltype(pc)::value;
          u32x4 hi, lo;
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            float y0 = pr[e] * q4_step(r[e >> 2].vs, e & 3, p), y1 = pr[e + 1] * q4_step(r[e >> 2].vs, (e & 3) + 1, p);
            if constexpr (kMask) {
              y0 = ok[e] ? y0 : 0.0f;
              y1 = ok[e + 1] ? y1 : 0.0f;
            }
            uint32_t a, b;
            q4_cut(y0, y1, a, b);
            hi[e / 2] = a;
            lo[e / 2] = b;
          }
          const half8 ph = __builtin_bit_cast(half8, hi), pl = __builtin_bit_cast(half8, lo);
          const half8 va = v_tile(std::integral_constant<int, 2 * p>{}), vb = v_tile(std::integral_constant<int, 2 * p + 1>{});
          acc[t][2 * p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph, acc[t][2 * p], 0, 0, 0);
          acc[t][2 * p + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb, ph, acc[t][2 * p + 1], 0, 0, 0);
          acc[t][2 * p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl, acc[t][2 * p], 0, 0, 0);
          acc[t][2 * p + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb, pl, acc[t][2 * p + 1], 0, 0, 0);
        };
        group(std::integral_constant<int, 0>{});
        group(std::integral_constant<int, 1>{});
        group(std::integral_constant<int, 2>{});
        group(std::integral_constant<int, 3>{});
      }
    };
    auto pair = [&](const Q4Regs* r, uint32_t b) {
      const int key0 = static_cast<int>((b0 + b) * 16);
      if (key0 >= wlo && key0 + 31 <= wmin && key0 + 32 <= key_end)  // uniform
        compute(std::false_type{}, r, key0);
      else
        compute(std::true_type{}, r, key0);
    };
    for (uint32_t b = 0; b < nblk; b += 4) {
      pair(s0, b);
      load_pair(s0, b + 4);
      pair(s1, b + 2);
      load_pair(s1, b + 6);
    }
    float bad = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w.o[t][n][i] = acc[t][n][i] * (n & 1 ? 0.0625f : 1.0f);
          bad += w.o[t][n][i] * 0.0f;
        }
    // An infinity or NaN: a step too large for the scale (or in the inputs). At most once.
    if (room != kQ4Room || !__builtin_amdgcn_ballot_w64(bad != 0.0f)) break;
    room = kQ4RoomBig;
    start();
  }
  // Weights relative to the maximum alike, whichever scale was taken.
  const float unit = __builtin_amdgcn_exp2f(-room);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    w.l[t] = sum_xor32(sum_xor16(w.l[t])) * unit;
#pragma unroll
    for (int n = 0; n < 8; ++n) w.o[t][n] *= unit;
  }
}

// q of a logical row, this lane's dims 32 p + 8 g + 0 .. 7.
__device__ __forceinline__ void q4_read_q(float4 (&raw)[8], const float* q, int g) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    raw[2 * p] = *reinterpret_cast<const float4*>(q + p * 32 + g * 8);
    raw[2 * p + 1] = *reinterpret_cast<const float4*>(q + p * 32 + g * 8 + 4);
  }
}

// Decode and verify: a work item's blocks dealt evenly over 8 waves, as the binary16 arena's
// 16-row-tile kernel, whose items, hand-off and merge these are.
template <int NT>
__global__ __launch_bounds__(64 * kWideWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_attn_decode_q4(
    const AttnItem* __restrict__ items, const uint32_t* __restrict__ pos, const uint32_t* __restrict__ pages,
    const q4_t* __restrict__ kc, const q4_t* __restrict__ vc, const float* __restrict__ q, float* __restrict__ out,
    float* __restrict__ part_o, float2* __restrict__ part_ml, uint32_t* __restrict__ counters, uint32_t part_o_bytes,
    uint32_t part_ml_bytes, uint32_t hq, uint32_t hkv, uint32_t bpp_shift, uint32_t window, float scale_log2,
    const SubRef* __restrict__ members, uint32_t by_item) {
  __shared__ WideShared<NT, false> sh;
  const AttnItem it = items[by_item ? blockIdx.y : blockIdx.x];
  const uint32_t kh = by_item ? blockIdx.x : blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const uint32_t G = hq / hkv;
  const uint32_t nlog = it.nrows * G;  // at most NT * 16
  const uint32_t nall = it.blk1 - it.blk0;
  const uint32_t wb0 = it.blk0 + nall * wave / kWideWaves;
  const uint32_t wb1 = it.blk0 + nall * (wave + 1) / kWideWaves;

  int rpos[NT], rlo[NT];
  bool has[NT];
  float4 qraw[NT][8];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const uint32_t lr = t * 16 + c;
    has[t] = lr < nlog;
    const uint32_t lrc = has[t] ? lr : 0;
    const uint32_t rr = it.r0 + lrc / G, h = kh * G + lrc % G;
    const int p = static_cast<int>(pos[rr]);
    rpos[t] = has[t] ? p : -1;
    rlo[t] = (window > 0 && p + 1 > static_cast<int>(window)) ? p + 1 - static_cast<int>(window) : 0;
    q4_read_q(qraw[t], q + (static_cast<size_t>(rr) * hq + h) * kD, g);
  }
  Q4Wave<NT> w;
  q4_attend<NT, kNontemporal>(w, kc, vc, pages + it.pt_off, wb0, wb1 - wb0, bpp_shift, kh, hkv, qraw, has, rpos, rlo,
                              scale_log2, lane);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int lr = t * 16 + c;
    if (g == 0) {
      sh.m[wave][lr] = w.m[t];
      sh.l[wave][lr] = w.l[t];
    }
    if (has[t])
#pragma unroll
      for (int n = 0; n < 8; ++n) sh.o[wave][lr][n * 4 + g] = __builtin_bit_cast(float4, w.o[t][n]);
  }
  __syncthreads();
  finish_item<64 * kWideWaves, NT * 16, true>(it, kh, G, hq, hkv, nlog, out, part_o, part_ml, counters, part_o_bytes,
                                              part_ml_bytes, sh.last,
                                              [&](uint32_t lr, uint32_t qi, float& mt, float& lt, float4& o) {
    mt = -INFINITY;
#pragma unroll
    for (int v = 0; v < kWideWaves; ++v) mt = fmaxf(mt, sh.m[v][lr]);
    lt = 0.0f;
    o = float4{0, 0, 0, 0};
    const float mf = fmaxf(mt, kLowest);
#pragma unroll
    for (int v = 0; v < kWideWaves; ++v) {
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

// Prefill: a tile of 64 logical rows, 16 to each of 4 waves, over the item's blocks; the waves
// read the blocks by themselves (the codes of a block are 2 KiB: they come from the CU's cache
// for all but the first).
static constexpr int kQ4TileWaves = 4;
static constexpr int kQ4TileRows = 64;

__global__ __launch_bounds__(64 * kQ4TileWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_attn_prefill_q4(
    const PrefillItem* __restrict__ items, const uint32_t* __restrict__ pos, const uint32_t* __restrict__ pages,
    const q4_t* __restrict__ kc, const q4_t* __restrict__ vc, const float* __restrict__ q, float* __restrict__ out,
    uint32_t hq, uint32_t hkv, uint32_t bpp_shift, uint32_t window, float scale_log2, float* __restrict__ part_o,
    float2* __restrict__ part_ml, uint32_t* __restrict__ counters, uint32_t part_o_bytes, uint32_t part_ml_bytes) {
  const PrefillItem it = items[blockIdx.x / hkv];
  const uint32_t kh = blockIdx.x % hkv;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const uint32_t G = hq / hkv;
  const uint32_t nlog = it.nrows * G;  // at most kQ4TileRows
  const uint32_t lr = wave * 16 + c;
  const bool has[1] = {lr < nlog};
  const uint32_t lrc = has[0] ? lr : 0;
  const uint32_t rr = it.r0 + lrc / G, h = kh * G + lrc % G;
  const int p = static_cast<int>(pos[rr]);
  const int rpos[1] = {has[0] ? p : -1};
  const int rlo[1] = {(window > 0 && p + 1 > static_cast<int>(window)) ? p + 1 - static_cast<int>(window) : 0};
  float4 qraw[1][8];
  q4_read_q(qraw[0], q + (static_cast<size_t>(rr) * hq + h) * kD, g);
  // The blocks some row of this wave sees.
  int first = has[0] ? rlo[0] : 0x7fffffff, last = rpos[0];
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    first = min(first, __shfl_xor(first, o));
    last = max(last, __shfl_xor(last, o));
  }
  first = __builtin_amdgcn_readfirstlane(first);
  last = __builtin_amdgcn_readfirstlane(last);
  const uint32_t b0 = last < 0 ? it.blk0 : max(it.blk0, static_cast<uint32_t>(first) / 16);
  const uint32_t b1 = last < 0 ? it.blk0 : min(it.blk1, static_cast<uint32_t>(last) / 16 + 1);
  Q4Wave<1> w;
  q4_attend<1, 0>(w, kc, vc, pages + it.pt_off, b0, b1 > b0 ? b1 - b0 : 0, bpp_shift, kh, hkv, qraw, has, rpos, rlo,
                  scale_log2, lane);
  const uint32_t nch = it.chunk_nch >> 16;
  if (nch <= 1) {
    if (!has[0]) return;
    float* o = out + (static_cast<size_t>(rr) * hq + h) * kD + g * 4;
    const float inv = 1.0f / w.l[0];
#pragma unroll
    for (int n = 0; n < 8; ++n) *reinterpret_cast<floatx4*>(o + n * 16) = w.o[0][n] * inv;
    return;
  }
  // A tile split along keys: the hand-off of the other arenas' tiles (attn_prefill.hpp).
  const __amdgpu_buffer_rsrc_t ro = make_rsrc(part_o, part_o_bytes);
  const __amdgpu_buffer_rsrc_t rml = make_rsrc(part_ml, part_ml_bytes);
  if (has[0]) {
    const size_t e = ((static_cast<size_t>(it.part_base) + (it.chunk_nch & 0xffffu)) * hkv + kh) * kQ4TileRows + lr;
#pragma unroll
    for (int n = 0; n < 8; ++n)
      st4_coherent(ro, static_cast<uint32_t>((e * kD + 16 * n + 4 * g) * 4), __builtin_bit_cast(float4, w.o[0][n]));
    if (g == 0) st2_coherent(rml, static_cast<uint32_t>(e * 8), float2{w.m[0], w.l[0]});
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
