// Verification of drafted tokens against the target's probabilities (speculative sampling), from
// given uniform numbers, on MI355X.
//
// A sequence has k drafts x_i and k + 1 rows of target logits. With temperature t,
// p(j) = w_j / W, w_j = e^((l_j - M) / t) (M the row's maximum, W the sum of w), and q likewise
// of the draft's logits; a draft without logits was certain, q(x) = 1. Draft i is accepted while
//   u_i q_i(x_i) < p_i(x_i).
// The next token is drawn from the first rejected draft's residual max(p - q, 0), or from
// p_{k+1}: the first token whose cumulative weight, in index order, exceeds v times the whole.
// At temperature 0 p is the most probable token (the first of equals).
//
// The draw's answer is a whole number that hangs on the order of cumulative sums, so weights and
// sums are 64-bit: with 150 thousand tokens of similar weight, f32's rounding (2^-24 of the whole)
// would cross the border of one in 50 draws, 64 bits' that of one in 10^10. e^x in 64 bits is a
// polynomial of 12 terms here, about 20 operations a logit: at 64-bit rates 4 us for 80 rows of
// 151936 logits, less than the 9 us that reading them takes.
//
// Launch 1: every chunk of 4096 logits (target and draft rows) gives its maximum M_c and
// sum e^((l - M_c) / t); a sequence's last chunk to arrive adds them up, decides, and draws where
// one row's chunk sums say enough (accepted all, certain drafts, temperature 0): the chunk by its
// cumulative sum, then the token within it. Launch 2 (drafts with logits, sequences with a
// rejected one): the residual's sum per chunk, the last to arrive draws from them. Chunk order
// fixes every sum's order: the same answer every time.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/yaxus_hip.h"
#include "attn_decode.hpp"
#include "epilogue.hpp"

namespace yx {

static constexpr int kVdThreads = 256;
static constexpr int kVdQuads = 4;                                     // 16-byte loads a thread and chunk
static constexpr uint32_t kVdChunk = kVdThreads * kVdQuads * 4;        // logits
static constexpr uint32_t kVdMaxChunks = 1024;
static constexpr uint32_t kVdSeqs = 256;                               // sequences of a launch

struct VerifyRows {  // the launch's sequences: first target row of each, in its logits
  uint32_t off[kVdSeqs + 1];
  uint32_t seqs;
};

struct VerifyIn {
  const float* logits;   // [rows][ld]
  const float* dlogits;  // [drafts][dld], null: certain drafts
  const uint32_t* drafts;
  const float* temperature;  // null: 1
  const float* u;
  const float* v;
  size_t ld, dld;
  uint32_t cols, nch;
};

struct VerifyPart {  // a chunk: sum of weights relative to its maximum, that maximum, its first index
  double s;
  float m;
  uint32_t at;
};

// Where a sequence stopped.
struct VerifyStop {
  double ip, iq;      // 1 / W of the row and of the draft's row
  double c;           // log2(e) / temperature (-1: temperature 0)
  float mp, mq;       // their maxima
  uint32_t row, drow;
  uint32_t drawn;     // the next token is drawn already
};

// 2^t, t <= 0, within 2^-50: 2^f by its series (|f| <= 1/2, the next term below 2^-51).
__device__ __forceinline__ double vd_exp2(double t) {
  t = fmax(t, -1100.0);  // (and NaN)
  const double n = __builtin_rint(t), f = t - n;
  constexpr double k[13] = {1.0,
                            6.93147180559945286e-01,
                            2.40226506959100694e-01,
                            5.55041086648215762e-02,
                            9.61812910762847687e-03,
                            1.33335581464284411e-03,
                            1.54035303933816061e-04,
                            1.52527338040598393e-05,
                            1.32154867901443053e-06,
                            1.01780860092396960e-07,
                            7.05491162080112188e-09,
                            4.44553827187081007e-10,
                            2.56784359934881958e-11};  // ln(2)^i / i!
  double p = k[12];
#pragma unroll
  for (int i = 11; i >= 0; --i) p = __builtin_fma(p, f, k[i]);
  return __builtin_ldexp(p, static_cast<int>(n));
}

// Weight of a logit relative to the maximum m (above -inf), c = log2(e) / temperature.
__device__ __forceinline__ double vd_weight(float x, float m, double c) {
  const double w = vd_exp2((static_cast<double>(x) - static_cast<double>(m)) * c);
  return x == m ? 1.0 : x > -INFINITY ? w : 0.0;  // (a NaN: 0)
}

// log2(e) / temperature; -1 for temperature 0 (and below, and NaN).
__device__ __forceinline__ double vd_c(const VerifyIn& in, uint32_t seq) {
  const float t = in.temperature ? in.temperature[seq] : 1.0f;
  return t > 0.0f ? 1.4426950408889634 / static_cast<double>(t) : -1.0;
}

// This thread's 16 logits of a chunk: quad i holds elements 4 (i * 256 + thread) of the chunk;
// -inf past the row's end and for NaN.
__device__ __forceinline__ void vd_load(f32x4 (&v)[kVdQuads], const float* row, uint32_t cols, uint32_t chunk) {
  const uint32_t e0 = chunk * kVdChunk;
  if (e0 + kVdChunk <= cols) {  // uniform
#pragma unroll
    for (int i = 0; i < kVdQuads; ++i)
      v[i] = *reinterpret_cast<const f32x4_any*>(row + e0 + 4 * (i * kVdThreads + threadIdx.x));
  } else {
#pragma unroll
    for (int i = 0; i < kVdQuads; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t e = e0 + 4 * (i * kVdThreads + threadIdx.x) + j;
        v[i][j] = e < cols ? row[e] : -INFINITY;
      }
  }
#pragma unroll
  for (int i = 0; i < kVdQuads; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[i][j] = v[i][j] == v[i][j] ? v[i][j] : -INFINITY;
}

__device__ __forceinline__ double vd_shfl_xor(double x, int o) { return __shfl_xor(x, o); }

struct VerifyShared {
  double mass[kVdMaxChunks];
  double sum[kVdQuads][4];  // [sub-block][wave]
  double row_w[2 * 64];     // W of a batch's target and draft rows
  float row_m[2 * 64];
  uint32_t row_at[2 * 64];
  double total;
  float m[4];
  uint32_t at[4];
  uint32_t chunk, first, last_pos, flag;
  VerifyStop stop;
};

// Sum over the workgroup, to all threads, in a fixed order.
__device__ __forceinline__ double vd_sum(VerifyShared& sh, double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += vd_shfl_xor(x, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.sum[0][threadIdx.x >> 6] = x;
  __syncthreads();
  return (sh.sum[0][0] + sh.sum[0][1]) + (sh.sum[0][2] + sh.sum[0][3]);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t vd_rsrc(void* p, size_t bytes) {
  return make_rsrc(p, static_cast<uint32_t>(bytes));
}
__device__ __forceinline__ VerifyPart vd_part(__amdgpu_buffer_rsrc_t r, uint32_t i) {
  return __builtin_bit_cast(VerifyPart, ld4_coherent(r, i * 16));
}

// What a draw weighs: p of a row, p without one token, or the residual of p and q.
struct VerifyDraw {
  const float* x;
  const float* y;  // null: p alone
  double c, ip, iq;
  float mp, mq;
  uint32_t without;  // a token left out (YX_NO_TOKEN: none)
  __device__ __forceinline__ double weight(float a, float b, uint32_t e) const {
#pragma clang fp contract(off)  // equal p and q leave nothing, not the rounding of one product
    const double p = vd_weight(a, mp, c);
    if (y == nullptr) return e == without ? 0.0 : p;
    return fmax(p * ip - (mq > -INFINITY ? vd_weight(b, mq, c) : 0.0) * iq, 0.0);
  }
};

// This thread's weights of a chunk.
__device__ __forceinline__ void vd_weights(double (&w)[kVdQuads][4], const VerifyDraw& d, uint32_t cols, uint32_t chunk) {
  f32x4 a[kVdQuads], b[kVdQuads];
  vd_load(a, d.x, cols, chunk);
  if (d.y) vd_load(b, d.y, cols, chunk);
#pragma unroll
  for (int i = 0; i < kVdQuads; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[i][j] = d.weight(a[i][j], d.y ? b[i][j] : 0.0f, chunk * kVdChunk + 4 * (i * kVdThreads + threadIdx.x) + j);
}

__device__ __forceinline__ double vd_chunk_sum(VerifyShared& sh, const VerifyDraw& d, uint32_t cols, uint32_t chunk) {
  double w[kVdQuads][4], s = 0.0;
  vd_weights(w, d, cols, chunk);
#pragma unroll
  for (int i = 0; i < kVdQuads; ++i) s += (w[i][0] + w[i][1]) + (w[i][2] + w[i][3]);
  return vd_sum(sh, s);
}

// The token at v among the weights of d, whose chunk sums lie in sh.mass[0 .. nch): the first
// whose cumulative sum exceeds v times the whole, the last with any weight where none does (v not
// below 1); YX_NO_TOKEN where there is no weight. All threads call it and have the result.
__device__ __forceinline__ uint32_t vd_draw(VerifyShared& sh, const VerifyDraw& d, uint32_t cols, uint32_t nch, float v) {
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    uint32_t last = YX_NO_TOKEN;
    for (uint32_t c = 0; c < nch; ++c) {
      total += sh.mass[c];
      if (sh.mass[c] > 0.0) last = c;
    }
    const double target = static_cast<double>(v) * total;
    uint32_t c = 0;
    double before = 0.0;  // the sum of the chunks before c
    if (last != YX_NO_TOKEN)
      for (; c < last && !(sh.mass[c] > 0.0 && before + sh.mass[c] > target); ++c) before += sh.mass[c];
    sh.chunk = last == YX_NO_TOKEN ? YX_NO_TOKEN : c;
    sh.total = target - before;
    sh.first = YX_NO_TOKEN;
    sh.last_pos = 0;
  }
  __syncthreads();
  const uint32_t chunk = sh.chunk;
  if (chunk == YX_NO_TOKEN) return YX_NO_TOKEN;  // uniform
  const double target = sh.total;                // within the chunk
  double w[kVdQuads][4];
  vd_weights(w, d, cols, chunk);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double own[kVdQuads], upto[kVdQuads];  // a thread's sum of a sub-block of 1024, and that of the wave's lanes up to it
#pragma unroll
  for (int i = 0; i < kVdQuads; ++i) {
    own[i] = (w[i][0] + w[i][1]) + (w[i][2] + w[i][3]);
    double x = own[i];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    upto[i] = x;
    if (lane == 63) sh.sum[i][wave] = x;
  }
  __syncthreads();
  double base = 0.0;
#pragma unroll
  for (int i = 0; i < kVdQuads; ++i) {
    double before = base;
    for (int k = 0; k < wave; ++k) before += sh.sum[i][k];
    double sum = before + (upto[i] - own[i]);
    uint32_t first = YX_NO_TOKEN, last = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t e = chunk * kVdChunk + 4 * (i * kVdThreads + threadIdx.x) + j;
      sum += w[i][j];
      if (w[i][j] > 0.0) {
        last = e + 1;
        if (sum > target && first == YX_NO_TOKEN) first = e;
      }
    }
    if (first != YX_NO_TOKEN) atomicMin(&sh.first, first);
    if (last) atomicMax(&sh.last_pos, last);
    base += (sh.sum[i][0] + sh.sum[i][1]) + (sh.sum[i][2] + sh.sum[i][3]);
  }
  __syncthreads();
  return sh.first != YX_NO_TOKEN ? sh.first : sh.last_pos - 1;
}

// Chunk masses of a row (relative to its maximum m) from its parts, into sh.mass.
__device__ __forceinline__ void vd_masses(VerifyShared& sh, __amdgpu_buffer_rsrc_t parts, uint32_t row, uint32_t nch,
                                          float m, double c) {
  for (uint32_t i = threadIdx.x; i < nch; i += kVdThreads) {
    const VerifyPart p = vd_part(parts, row * nch + i);
    sh.mass[i] = p.m > -INFINITY ? p.s * vd_weight(p.m, m, c) : 0.0;
  }
}

// Launch 1. Grid: (chunks, target rows + draft rows). parts: a VerifyPart per (row, chunk),
// target rows first; counters: one per sequence, zero on entry and left at zero.
__global__ __launch_bounds__(kVdThreads) void verify_sums(VerifyRows rows, VerifyIn in, VerifyPart* __restrict__ parts,
                                                          size_t part_bytes, VerifyStop* __restrict__ stops,
                                                          uint32_t* __restrict__ counters,
                                                          uint32_t* __restrict__ accepted, uint32_t* __restrict__ next) {
  __shared__ VerifyShared sh;
  const uint32_t chunk = blockIdx.x, r = blockIdx.y, nrows = rows.off[rows.seqs];
  const bool draft = r >= nrows;
  // The sequence of the row: target row off[s] + i; draft off[s] - s + i.
  uint32_t lo = 0, hi = rows.seqs;  // off[lo] <= row < off[hi]
  const uint32_t mine = draft ? r - nrows : r;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (rows.off[mid] - (draft ? mid : 0) <= mine) lo = mid;
    else hi = mid;
  }
  const uint32_t seq = lo, row0 = rows.off[seq], k = rows.off[seq + 1] - row0 - 1, draft0 = row0 - seq;
  const double c = vd_c(in, seq);
  const __amdgpu_buffer_rsrc_t pr = vd_rsrc(parts, part_bytes);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

  if (!draft || c >= 0.0) {  // uniform: a draft's own distribution does not count at temperature 0
    f32x4 v[kVdQuads];
    vd_load(v, draft ? in.dlogits + mine * in.dld : in.logits + mine * in.ld, in.cols, chunk);
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kVdQuads; ++i) m = fmaxf(m, fmaxf(fmaxf(v[i].x, v[i].y), fmaxf(v[i].z, v[i].w)));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (lane == 0) sh.m[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sh.m[0], sh.m[1]), fmaxf(sh.m[2], sh.m[3]));
    double s = 0.0;
    uint32_t at = YX_NO_TOKEN;
    if (c >= 0.0) {
      if (m > -INFINITY)
#pragma unroll
        for (int i = 0; i < kVdQuads; ++i) {
          double t[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) t[j] = vd_weight(v[i][j], m, c);
          s += (t[0] + t[1]) + (t[2] + t[3]);
        }
      s = vd_sum(sh, s);
    } else {  // the first of the largest
#pragma unroll
      for (int i = 0; i < kVdQuads; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (v[i][j] == m) at = min(at, chunk * kVdChunk + 4 * (i * kVdThreads + threadIdx.x) + j);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) at = min(at, static_cast<uint32_t>(__shfl_xor(static_cast<int>(at), o)));
      if (lane == 0) sh.at[wave] = at;
      __syncthreads();
      at = min(min(sh.at[0], sh.at[1]), min(sh.at[2], sh.at[3]));
    }
    if (threadIdx.x == 0) st4_coherent(pr, (r * in.nch + chunk) * 16, __builtin_bit_cast(float4, VerifyPart{s, m, at}));
  }
  // Arrival (the memory order of the attention's split-K hand-off, attn_decode.hpp).
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t* cnt = counters + static_cast<size_t>(seq) * kCounterStride;
    const uint32_t all = in.nch * (k + 1 + (in.dlogits ? k : 0));
    const uint32_t arrived = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sh.flag = arrived == all - 1;
    if (sh.flag) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!sh.flag) return;

  // The sequence's decision. A batch of up to 64 drafts: each wave adds up a row's chunks.
  uint32_t taken = 0;  // accepted
  bool stopped = false;
  double wp = 0.0, wq = 0.0;
  float mp = -INFINITY, mq = -INFINITY;
  uint32_t best = YX_NO_TOKEN;
  for (uint32_t b = 0; b <= k && !stopped; b += 64) {  // uniform
    const uint32_t n = min(64u, k + 1 - b);            // rows of this batch (the last may be the free one)
    __syncthreads();
    for (uint32_t i = wave; i < 2 * n; i += 4) {
      const bool q = i >= n;
      const uint32_t j = b + (q ? i - n : i);
      double w = 0.0;
      float m = -INFINITY;
      uint32_t at = YX_NO_TOKEN;
      if (!q || (in.dlogits && j < k && c >= 0.0)) {
        const uint32_t pr_row = q ? nrows + draft0 + j : row0 + j;
        for (uint32_t h = lane; h < in.nch; h += 64) {
          const VerifyPart p = vd_part(pr, pr_row * in.nch + h);
          if (p.m > m) at = p.at;
          if (c >= 0.0 && p.m > -INFINITY) {
            const float mn = fmaxf(m, p.m);
            w = (m > -INFINITY ? w * vd_weight(m, mn, c) : 0.0) + p.s * vd_weight(p.m, mn, c);
          }
          m = fmaxf(m, p.m);
        }
        float top = m;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        if (m != top || top == -INFINITY) at = YX_NO_TOKEN;
        w = m > -INFINITY ? w * vd_weight(m, top, c) : 0.0;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
          w += vd_shfl_xor(w, o);
          at = min(at, static_cast<uint32_t>(__shfl_xor(static_cast<int>(at), o)));
        }
        m = top;
      }
      if (lane == 0) {
        sh.row_w[i] = w;
        sh.row_m[i] = m;
        sh.row_at[i] = at;
      }
    }
    __syncthreads();
    for (uint32_t i = 0; i < n; ++i) {  // uniform
      const uint32_t j = b + i;
      wp = sh.row_w[i];
      mp = sh.row_m[i];
      best = sh.row_at[i];
      wq = sh.row_w[n + i];
      mq = sh.row_m[n + i];
      if (j == k) break;
      const uint32_t x = in.drafts[draft0 + j];
      bool ok = false;
      if (c < 0.0) {
        ok = x == best && best != YX_NO_TOKEN;
      } else if (x < in.cols && mp > -INFINITY) {
        const float a = in.logits[(row0 + j) * in.ld + x];
        const double p = vd_weight(a, mp, c) / wp;
        double q = 1.0;
        if (in.dlogits) q = mq > -INFINITY ? vd_weight(in.dlogits[(draft0 + j) * in.dld + x], mq, c) / wq : 0.0;
        ok = static_cast<double>(in.u[draft0 + j]) * q < p;
      }
      if (!ok) {
        stopped = true;
        break;
      }
      ++taken;
    }
  }
  const uint32_t row = row0 + taken, drow = draft0 + taken;
  const bool residual = stopped && in.dlogits != nullptr && c >= 0.0 && mp > -INFINITY && mq > -INFINITY;
  if (threadIdx.x == 0) {
    accepted[seq] = taken;
    stops[seq] = VerifyStop{mp > -INFINITY ? 1.0 / wp : 0.0, mq > -INFINITY ? 1.0 / wq : 0.0, c, mp, mq, row, drow, residual ? 0u : 1u};
  }
  if (residual) return;
  uint32_t token = best;  // temperature 0
  if (c >= 0.0) {
    token = YX_NO_TOKEN;
    if (mp > -INFINITY) {
      VerifyDraw d{in.logits + row * in.ld, nullptr, c, 1.0, 0.0, mp, mq, YX_NO_TOKEN};
      __syncthreads();
      vd_masses(sh, pr, row, in.nch, mp, c);
      __syncthreads();
      const uint32_t x = stopped ? in.drafts[drow] : YX_NO_TOKEN;
      if (stopped && in.dlogits == nullptr && x < in.cols) {
        // Without the rejected token: its chunk added up anew (taken away, it could leave only
        // rounding errors).
        d.without = x;
        const double s = vd_chunk_sum(sh, d, in.cols, x / kVdChunk);
        __syncthreads();
        const double kept = sh.mass[x / kVdChunk];
        __syncthreads();
        if (threadIdx.x == 0) sh.mass[x / kVdChunk] = s;
        token = vd_draw(sh, d, in.cols, in.nch, in.v[seq]);
        if (token == YX_NO_TOKEN) {  // nothing else has weight: p itself
          __syncthreads();
          if (threadIdx.x == 0) sh.mass[x / kVdChunk] = kept;
          d.without = YX_NO_TOKEN;
          token = vd_draw(sh, d, in.cols, in.nch, in.v[seq]);
        }
      } else {
        token = vd_draw(sh, d, in.cols, in.nch, in.v[seq]);
      }
    }
  }
  if (threadIdx.x == 0) next[seq] = token;
}

// Launch 2. Grid: (chunks, sequences). sums: a residual's sum per (sequence, chunk).
__global__ __launch_bounds__(kVdThreads) void verify_residual(VerifyRows rows, VerifyIn in, VerifyPart* __restrict__ parts,
                                                              size_t part_bytes, const VerifyStop* __restrict__ stops,
                                                              double* __restrict__ sums,
                                                              uint32_t* __restrict__ counters,
                                                              uint32_t* __restrict__ next) {
  __shared__ VerifyShared sh;
  const uint32_t chunk = blockIdx.x, seq = blockIdx.y;
  const VerifyStop st = stops[seq];
  if (st.drawn) return;  // uniform
  VerifyDraw d{in.logits + st.row * in.ld, in.dlogits + st.drow * in.dld, st.c, st.ip, st.iq, st.mp, st.mq, YX_NO_TOKEN};
  const double s = vd_chunk_sum(sh, d, in.cols, chunk);
  double* mine = sums + static_cast<size_t>(seq) * in.nch;
  if (threadIdx.x == 0) {
    __hip_atomic_store(mine + chunk, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_s_waitcnt(0);
    uint32_t* cnt = counters + static_cast<size_t>(seq) * kCounterStride;
    const uint32_t arrived = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sh.flag = arrived == in.nch - 1;
    if (sh.flag) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!sh.flag) return;
  for (uint32_t i = threadIdx.x; i < in.nch; i += kVdThreads)
    sh.mass[i] = __hip_atomic_load(mine + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  uint32_t token = vd_draw(sh, d, in.cols, in.nch, in.v[seq]);
  if (token == YX_NO_TOKEN) {  // p nowhere above q: p itself
    d.y = nullptr;
    __syncthreads();
    vd_masses(sh, vd_rsrc(parts, part_bytes), st.row, in.nch, st.mp, st.c);
    token = vd_draw(sh, d, in.cols, in.nch, in.v[seq]);
  }
  if (threadIdx.x == 0) next[seq] = token;
}

}  // namespace yx
