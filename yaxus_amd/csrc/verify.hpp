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
// would cross the border of one in 50 draws, weights within 2^-47 that of one in 4 x 10^8. e^x in 64 bits is a
// polynomial of 12 terms here, about 20 operations a logit: at 64-bit rates 4 us for 80 rows of
// 151936 logits, less than the 9 us that reading them takes.
//
// Launch 1 reads every chunk of 4096 logits (target and draft rows): its maximum M_c and
// sum e^((l - M_c) / t). Launch 2, a workgroup per sequence (where drafts have logits several, each
// with an equal share of the chunks, at most one a CU over all sequences): adds the chunks up and decides,
// every workgroup of a sequence by itself; then draws where one row's chunk sums say enough (accepted
// all, certain drafts, temperature 0): the chunk by its cumulative sum, then the token within it. Where
// they don't, each workgroup adds up its chunks of the residual and the last of the sequence to
// arrive draws. Chunk order fixes every sum's order: the same answer every time.
//
// Measured: launch 1 is bound by reading (249 rows of 151936: 38 us, 4.0 TB/s), launch 2 by its chain of
// trips to memory (sums, decision, residual, arrival, draw): 12 us for one sequence of 5 drafts, 18 for 16 of 4, 9
// where no residual of two rows is drawn from.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/yaxus_hip.h"
#include "attn_decode.hpp"
#include "epilogue.hpp"

namespace yx {

static constexpr int kVdSumThreads = 256, kVdSumQuads = 4;             // launch 1: 16-byte loads a thread
// Launch 2: one 16-byte load a thread. Four times the logits in a quarter of the threads is four
// times the code, which a launch this short fetches more slowly than it runs it (7 us a chunk of
// both rows' weights).
static constexpr int kVdThreads = 1024;
static constexpr int kVdWaves = kVdThreads / 64;
static constexpr uint32_t kVdChunk = kVdThreads * 4;                   // logits
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

// 2^t, t <= 0 (below -1000, and NaN: 2^-1000), within 2^-47: the whole part n of t goes into the
// exponent, 2^f by its series (|f| <= 1/2: the first term left out is below 2^-47). 17 operations,
// all at full rate: the rounding by a large addend instead of rndne, the exponent by an integer
// addition instead of ldexp.
__device__ __forceinline__ double vd_exp2(double t) {
  constexpr double kWhole = 6755399441055744.0;  // 1.5 * 2^52: the sum's last bit is worth 1
  t = fmax(t, -1000.0);
  const double r = t + kWhole, f = t - (r - kWhole);
  constexpr double k[12] = {1.0,
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
                            4.44553827187081007e-10};  // ln(2)^i / i!
  double p = k[11];
#pragma unroll
  for (int i = 10; i >= 0; --i) p = __builtin_fma(p, f, k[i]);
  const uint64_t bits = __builtin_bit_cast(uint64_t, p);
  const uint32_t n = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, r));
  const uint32_t hi = static_cast<uint32_t>(bits >> 32) + (n << 20);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | static_cast<uint32_t>(bits));
}

// Weight of a logit relative to the maximum m (above -inf), c = log2(e) / temperature. Below 2^-1000
// there is none: a token far below, beside +inf, of -inf or NaN (the differences -inf and NaN) is
// never accepted or drawn, at numbers of 0 either.
__device__ __forceinline__ double vd_weight(float x, float m, double c) {
  const double t = (static_cast<double>(x) - static_cast<double>(m)) * c, w = vd_exp2(t);
  return x == m ? 1.0 : t >= -1000.0 ? w : 0.0;
}

// log2(e) / temperature; -1 for temperature 0 (and below, and NaN).
__device__ __forceinline__ double vd_c(const VerifyIn& in, uint32_t seq) {
  const float t = in.temperature ? in.temperature[seq] : 1.0f;
  return t > 0.0f ? 1.4426950408889634 / static_cast<double>(t) : -1.0;
}

// This thread's 4 logits of a chunk; -inf past the row's end.
__device__ __forceinline__ f32x4 vd_load(const float* row, uint32_t cols, uint32_t chunk) {
  const uint32_t e = chunk * kVdChunk + 4 * threadIdx.x;
  if (e + 4 <= cols) return *reinterpret_cast<const f32x4_any*>(row + e);
  f32x4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  if (e < cols) v.x = row[e];
  if (e + 1 < cols) v.y = row[e + 1];
  if (e + 2 < cols) v.z = row[e + 2];
  return v;
}

// A lane's neighbour by a data-parallel-primitive control, 0 where it has none (or kRows leaves its
// row of 16 out). These are register moves, where a shuffle goes through LDS (100 cycles a step).
template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ double vd_dpp(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(b), kCtrl, kRows, 0xf, true));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), kCtrl, kRows, 0xf, true));
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// Inclusive sums over the lanes of a row of 16, and of the wave.
__device__ __forceinline__ double vd_scan16(double x) {
  x += vd_dpp<0x111>(x);  // row_shr:1, 2, 4, 8
  x += vd_dpp<0x112>(x);
  x += vd_dpp<0x114>(x);
  x += vd_dpp<0x118>(x);
  return x;
}
__device__ __forceinline__ double vd_scan(double x) {
  x = vd_scan16(x);
  x += vd_dpp<0x142, 0xa>(x);  // row_bcast:15 into rows 1 and 3
  x += vd_dpp<0x143, 0xc>(x);  // row_bcast:31 into rows 2 and 3
  return x;
}

__device__ __forceinline__ double vd_lane(double x, int lane) {  // uniform lane
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b), lane));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b >> 32), lane));
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// The wave's sum.
__device__ __forceinline__ double vd_wave_sum(double x) { return vd_lane(vd_scan(x), 63); }

static constexpr uint32_t kVdBatch = 64;  // drafts decided at once

struct VerifyShared {
  double mass[kVdMaxChunks];
  double sum[kVdWaves];
  double row_w[2 * kVdBatch + 2];  // W of a batch's target rows, then of its drafts'
  float row_m[2 * kVdBatch + 2];
  uint32_t row_at[kVdBatch + 1];
  double before;
  float m[kVdWaves];
  uint32_t at[kVdWaves], last[kVdWaves];
  uint32_t flag;
};

// Sum over the workgroup, to all threads, in a fixed order.
__device__ __forceinline__ double vd_sum(VerifyShared& sh, double x) {
  static_assert(kVdWaves == 16, "the waves' sums are a row of lanes");
  x = vd_wave_sum(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.sum[threadIdx.x >> 6] = x;
  __syncthreads();
  return vd_lane(vd_scan16(sh.sum[threadIdx.x & (kVdWaves - 1)]), kVdWaves - 1);
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

// This thread's logits of a chunk, and their weights.
struct VerifyLogits {
  f32x4 a, b;
};
__device__ __forceinline__ VerifyLogits vd_logits(const VerifyDraw& d, uint32_t cols, uint32_t chunk) {
  VerifyLogits l{vd_load(d.x, cols, chunk), f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
  if (d.y) l.b = vd_load(d.y, cols, chunk);
  return l;
}
__device__ __forceinline__ void vd_weights(double (&w)[4], const VerifyDraw& d, const VerifyLogits& l, uint32_t chunk) {
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = d.weight(l.a[j], l.b[j], chunk * kVdChunk + 4 * threadIdx.x + j);
}

// Of a wave whose lanes hold rising indexes: the first lane's that has one (YX_NO_TOKEN: none), and
// the last lane's. (Ballots: LDS atomics of divergent lanes become loops over the lanes, 20 us a draw.)
__device__ __forceinline__ uint32_t vd_first(uint32_t i) {
  const uint64_t has = __builtin_amdgcn_ballot_w64(i != YX_NO_TOKEN);
  return has ? static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(i), __builtin_ctzll(has))) : YX_NO_TOKEN;
}
__device__ __forceinline__ uint32_t vd_last(uint32_t i) {
  const uint64_t has = __builtin_amdgcn_ballot_w64(i != YX_NO_TOKEN);
  return has ? static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(i), 63 - __builtin_clzll(has))) : YX_NO_TOKEN;
}

// Of the workgroup, whose threads hold rising indexes: the first thread's that has one, else the
// last of `last` (YX_NO_TOKEN: neither), to all threads.
__device__ __forceinline__ uint32_t vd_choose(VerifyShared& sh, uint32_t first, uint32_t last) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  first = vd_first(first);
  last = vd_last(last);
  if (lane == 0) {
    sh.at[wave] = first;
    sh.last[wave] = last;
  }
  __syncthreads();
  first = vd_first(lane < kVdWaves ? sh.at[lane] : YX_NO_TOKEN);
  last = vd_last(lane < kVdWaves ? sh.last[lane] : YX_NO_TOKEN);
  return first != YX_NO_TOKEN ? first : last;
}

// The token at v among the weights of d, whose chunk sums lie in sh.mass[0 .. nch): the first
// whose cumulative sum exceeds v times the whole, the last with any weight where none does (v not
// below 1); YX_NO_TOKEN where there is no weight. All threads call it and have the result.
__device__ __forceinline__ uint32_t vd_draw(VerifyShared& sh, const VerifyDraw& d, uint32_t cols, uint32_t nch, float v) {
  static_assert(kVdMaxChunks <= kVdThreads, "a thread per chunk");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  __syncthreads();
  double mass = sh.mass[threadIdx.x & (kVdMaxChunks - 1)];
  mass = threadIdx.x < nch ? mass : 0.0;
  double upto = vd_scan(mass);
  if (lane == 63) sh.sum[wave] = upto;
  __syncthreads();
  double waves = vd_scan16(sh.sum[lane & (kVdWaves - 1)]);  // lane i: of waves 0 to i
  if (wave) upto += vd_lane(waves, wave - 1);
  double target = static_cast<double>(v) * vd_lane(waves, kVdWaves - 1);
  const bool some = mass > 0.0;
  const uint32_t chunk = vd_choose(sh, some && upto > target ? threadIdx.x : YX_NO_TOKEN, some ? threadIdx.x : YX_NO_TOKEN);
  if (chunk == YX_NO_TOKEN) return chunk;  // uniform: no weight
  if (threadIdx.x == chunk) sh.before = upto - mass;
  double w[4];
  vd_weights(w, d, vd_logits(d, cols, chunk), chunk);
  const double own = (w[0] + w[1]) + (w[2] + w[3]);
  upto = vd_scan(own);
  __syncthreads();  // (every wave has read the chunks' sums)
  if (lane == 63) sh.sum[wave] = upto;
  __syncthreads();
  target -= sh.before;  // within the chunk
  waves = vd_scan16(sh.sum[lane & (kVdWaves - 1)]);
  double sum = upto - own + (wave ? vd_lane(waves, wave - 1) : 0.0);
  uint32_t first = YX_NO_TOKEN, last = YX_NO_TOKEN;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t e = chunk * kVdChunk + 4 * threadIdx.x + j;
    sum += w[j];
    if (w[j] > 0.0) {
      last = e;
      if (sum > target && first == YX_NO_TOKEN) first = e;
    }
  }
  return vd_choose(sh, first, last);
}

// Chunk masses of a row (relative to its maximum m) from its parts, into sh.mass.
__device__ __forceinline__ void vd_masses(VerifyShared& sh, const VerifyPart* __restrict__ parts, uint32_t nch, float m,
                                          double c) {
  if (const uint32_t i = threadIdx.x; i < nch) {
    const VerifyPart p = parts[i];
    sh.mass[i] = p.m > -INFINITY ? p.s * vd_weight(p.m, m, c) : 0.0;
  }
}

// Launch 1. Grid: (chunks, target rows + draft rows). parts: a VerifyPart per (row, chunk),
// target rows first.
__global__ __launch_bounds__(kVdSumThreads) void verify_sums(VerifyRows rows, VerifyIn in, VerifyPart* __restrict__ parts) {
  constexpr int kWaves = kVdSumThreads / 64;
  static_assert(kVdSumThreads * kVdSumQuads * 4 == kVdChunk && kWaves == 4, "a chunk of logits a workgroup");
  __shared__ float ms[kWaves];
  __shared__ double ss[kWaves];
  __shared__ uint32_t ns[kWaves];
  const uint32_t chunk = blockIdx.x, r = blockIdx.y, nrows = rows.off[rows.seqs];
  const bool draft = r >= nrows;
  const uint32_t mine = draft ? r - nrows : r, e0 = chunk * kVdChunk;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* row = draft ? in.dlogits + mine * in.dld : in.logits + mine * in.ld;
  f32x4 v[kVdSumQuads];
#pragma unroll
  for (int i = 0; i < kVdSumQuads; ++i) {
    const uint32_t e = e0 + 4 * (i * kVdSumThreads + threadIdx.x);
    v[i] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (e + 4 <= in.cols) {
      v[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(row + e));
    } else {
      if (e < in.cols) v[i].x = row[e];
      if (e + 1 < in.cols) v[i].y = row[e + 1];
      if (e + 2 < in.cols) v[i].z = row[e + 2];
    }
  }
  // The sequence of the row: target row off[s] + i; draft off[s] - s + i. (Read as a lane per
  // sequence while the logits are on their way.)
  {
    const uint32_t s = threadIdx.x;
    const bool before = s < rows.seqs && rows.off[s] - (draft ? s : 0) <= mine;
    const uint32_t n = __popcll(__builtin_amdgcn_ballot_w64(before));
    if (lane == 0) ns[wave] = n;
  }
  static_assert(kVdSeqs <= kVdSumThreads, "a thread per sequence");
  __syncthreads();
  // (Of sequences without drafts, which share their draft offset with the next, the last.)
  const uint32_t seq = __builtin_amdgcn_readfirstlane(ns[0] + ns[1] + ns[2] + ns[3]) - 1;
  const double c = vd_c(in, seq);
  if (draft && c < 0.0) return;  // uniform: a draft's own distribution does not count at temperature 0
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kVdSumQuads; ++i) m = fmaxf(m, fmaxf(fmaxf(v[i].x, v[i].y), fmaxf(v[i].z, v[i].w)));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if (lane == 0) ms[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
  double s = 0.0;
  uint32_t at = YX_NO_TOKEN;
  const bool plain = c > 0x1p-100 && m > -INFINITY && m < INFINITY;  // tokens without weight then add 2^-1000 each, nothing beside 1
  if (c < 0.0 || !plain) {
    // Temperature 0: the first of the largest. A row of nothing, +inf, temperatures beyond 2^100: the exact form.
#pragma unroll
    for (int i = 0; i < 4 * kVdSumQuads; ++i) {
      const float x = v[i / 4][i % 4];
      if (c < 0.0) {
        if (x == m && m > -INFINITY) at = min(at, e0 + 4 * (i / 4 * kVdSumThreads + threadIdx.x) + i % 4);
      } else if (m == INFINITY) {
        s += x == m ? 1.0 : 0.0;
      } else if (m > -INFINITY) {
        s += vd_weight(x, m, c);
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) at = min(at, static_cast<uint32_t>(__shfl_xor(static_cast<int>(at), o)));
    if (lane == 0) ns[wave] = at;
  } else {
    const double md = static_cast<double>(m);
#pragma unroll 1
    for (int i = 0; i < kVdSumQuads; ++i) {
      double t[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = vd_exp2((static_cast<double>(v[0][j]) - md) * c);
      s += (t[0] + t[1]) + (t[2] + t[3]);
#pragma unroll
      for (int j = 0; j + 1 < kVdSumQuads; ++j) v[j] = v[j + 1];  // (a loop a quarter as long)
    }
  }
  s = vd_wave_sum(s);
  if (lane == 0) ss[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0)
    parts[static_cast<size_t>(r) * in.nch + chunk] =
        VerifyPart{(ss[0] + ss[1]) + (ss[2] + ss[3]), m, c < 0.0 ? min(min(ns[0], ns[1]), min(ns[2], ns[3])) : YX_NO_TOKEN};
}

// Launch 2. Grid: (shares of a sequence's chunks, `per` chunks each, where drafts have logits, else
// 1; sequences). sums: a residual's sum per (sequence, chunk); counters: one per sequence, zero on
// entry and left at zero.
__global__ __launch_bounds__(kVdThreads) void verify_pick(VerifyRows rows, VerifyIn in, const VerifyPart* __restrict__ parts,
                                                          uint32_t per, double* __restrict__ sums, uint32_t* __restrict__ counters,
                                                          uint32_t* __restrict__ accepted, uint32_t* __restrict__ next) {
  __shared__ VerifyShared sh;
  const uint32_t share = blockIdx.x, seq = blockIdx.y, nrows = rows.off[rows.seqs];
  const uint32_t row0 = rows.off[seq], k = rows.off[seq + 1] - row0 - 1, draft0 = row0 - seq;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double c = vd_c(in, seq);
  const bool dist = in.dlogits != nullptr && c >= 0.0;
  // The sequence's decision, up to 64 drafts at once: each wave adds up rows' chunks, two at a
  // time on their way, while a thread per draft has its token, number and logits brought.
  uint32_t taken = 0;  // accepted
  bool stopped = false;
  double wp = 0.0, wq = 0.0;
  float mp = -INFINITY, mq = -INFINITY;
  uint32_t best = YX_NO_TOKEN;
  for (uint32_t b = 0; b <= k && !stopped; b += kVdBatch) {  // uniform
    const uint32_t n = min(kVdBatch, k - b);                 // drafts of this batch
    const uint32_t nt = min(n + 1, k + 1 - b), all = nt + (dist ? n : 0);  // target rows, the free one's among them at the end
    uint32_t x = YX_NO_TOKEN;
    float u = 0.0f, a = -INFINITY, y = -INFINITY;
    if (threadIdx.x < n) {
      x = in.drafts[draft0 + b + threadIdx.x];
      u = in.u[draft0 + b + threadIdx.x];
      if (x < in.cols) {
        a = in.logits[(row0 + b + threadIdx.x) * in.ld + x];
        if (dist) y = in.dlogits[(draft0 + b + threadIdx.x) * in.dld + x];
      }
    }
    __syncthreads();
    for (uint32_t i0 = wave; i0 < all; i0 += 2 * kVdWaves) {
      double w[2];
      float m[2];
      uint32_t at[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint32_t i = i0 + kVdWaves * g, pr_row = i < nt ? row0 + b + i : nrows + draft0 + b + (i - nt);
        w[g] = 0.0;
        m[g] = -INFINITY;
        at[g] = YX_NO_TOKEN;
        if (i >= all) continue;  // uniform
        VerifyPart p{0.0, -INFINITY, YX_NO_TOKEN};
        if (static_cast<uint32_t>(lane) < in.nch) p = parts[static_cast<size_t>(pr_row) * in.nch + lane];
        w[g] = p.s;
        m[g] = p.m;
        at[g] = p.at;
      }
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint32_t i = i0 + kVdWaves * g, pr_row = i < nt ? row0 + b + i : nrows + draft0 + b + (i - nt);
        if (i >= all) continue;
        for (uint32_t h = lane + 64; h < in.nch; h += 64) {  // more than 64 chunks
          const VerifyPart p = parts[static_cast<size_t>(pr_row) * in.nch + h];
          if (p.m > m[g]) at[g] = p.at;
          const float mn = fmaxf(m[g], p.m);
          if (c >= 0.0 && mn > -INFINITY)
            w[g] = (m[g] > -INFINITY ? w[g] * vd_weight(m[g], mn, c) : 0.0) + (p.m > -INFINITY ? p.s * vd_weight(p.m, mn, c) : 0.0);
          m[g] = mn;
        }
        float top = m[g];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        if (c >= 0.0) {
          w[g] = vd_wave_sum(m[g] > -INFINITY ? w[g] * vd_weight(m[g], top, c) : 0.0);
        } else {
          uint32_t f = m[g] == top && top > -INFINITY ? at[g] : YX_NO_TOKEN;
#pragma unroll
          for (int o = 32; o > 0; o >>= 1) f = min(f, static_cast<uint32_t>(__shfl_xor(static_cast<int>(f), o)));
          at[g] = f;
        }
        if (lane == 0) {
          const uint32_t to = i < nt ? i : kVdBatch + 1 + (i - nt);
          sh.row_w[to] = w[g];
          sh.row_m[to] = top;
          if (i < nt) sh.row_at[i] = at[g];
        }
      }
    }
    __syncthreads();
    if (wave == 0) {
      bool ok = false;
      if (threadIdx.x < n) {
        const uint32_t i = threadIdx.x;
        const float m = sh.row_m[i];
        if (c < 0.0) {
          ok = x == sh.row_at[i] && x != YX_NO_TOKEN;
        } else if (x < in.cols && m > -INFINITY) {
          const double p = vd_weight(a, m, c) / sh.row_w[i];
          double q = 1.0;
          if (dist) {
            const float md = sh.row_m[kVdBatch + 1 + i];
            q = md > -INFINITY ? vd_weight(y, md, c) / sh.row_w[kVdBatch + 1 + i] : 0.0;
          }
          ok = static_cast<double>(u) * q < p;
        }
      }
      const uint64_t stand = __builtin_amdgcn_ballot_w64(ok);
      const uint32_t first = ~stand ? static_cast<uint32_t>(__builtin_ctzll(~stand)) : 64u;
      if (lane == 0) sh.flag = min(first, n);
    }
    __syncthreads();
    const uint32_t i = sh.flag;
    taken = b + i;
    stopped = i < n;
    if (!stopped && taken < k) continue;  // the next batch
    wp = sh.row_w[i];
    mp = sh.row_m[i];
    best = sh.row_at[i];
    if (dist && stopped) {
      wq = sh.row_w[kVdBatch + 1 + i];
      mq = sh.row_m[kVdBatch + 1 + i];
    }
    break;
  }
  const uint32_t row = row0 + taken, drow = draft0 + taken;
  if (share == 0 && threadIdx.x == 0) accepted[seq] = taken;
  const bool residual = stopped && dist && mp > -INFINITY && mq > -INFINITY;
  if (!residual && share != 0) return;  // uniform
  uint32_t token = best;                // temperature 0
  if (c >= 0.0) token = YX_NO_TOKEN;
  if (c >= 0.0 && mp > -INFINITY) {
    VerifyDraw d{in.logits + row * in.ld, nullptr, c, 1.0, 0.0, mp, mq, YX_NO_TOKEN};
    const VerifyPart* const row_parts = parts + static_cast<size_t>(row) * in.nch;
    if (residual) {
      d.y = in.dlogits + drow * in.dld;
      d.ip = 1.0 / wp;
      d.iq = 1.0 / wq;
    } else if (stopped && in.dlogits == nullptr) {
      const uint32_t x = in.drafts[drow];
      if (x < in.cols) d.without = x;
    }
    // The residual's sum in this chunk; or that of p without the rejected token in its chunk (added
    // up anew: taken away, it could leave only rounding errors).
    const bool without = d.without != YX_NO_TOKEN;
    double s = 0.0;
    double* const mine = sums + static_cast<size_t>(seq) * in.nch;
    if (residual || without) {
      const uint32_t first = residual ? share * per : d.without / kVdChunk, end = residual ? min(in.nch, first + per) : first + 1;
      VerifyLogits l = vd_logits(d, in.cols, first);
#pragma unroll 1
      for (uint32_t chunk = first; chunk < end; ++chunk) {
        const VerifyLogits now = l;
        if (chunk + 1 < end) l = vd_logits(d, in.cols, chunk + 1);
        double w[4];
        vd_weights(w, d, now, chunk);
        s = vd_sum(sh, (w[0] + w[1]) + (w[2] + w[3]));
        if (residual && threadIdx.x == 0) __hip_atomic_store(mine + chunk, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    if (residual) {
      // Arrival (the memory order of the attention's split-K hand-off, attn_decode.hpp).
      if (threadIdx.x == 0) {
        __builtin_amdgcn_s_waitcnt(0);
        uint32_t* cnt = counters + static_cast<size_t>(seq) * kCounterStride;
        const uint32_t arrived = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh.flag = arrived == gridDim.x - 1;
        if (sh.flag) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (!sh.flag) return;
      if (const uint32_t i = threadIdx.x; i < in.nch)
        sh.mass[i] = __hip_atomic_load(mine + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else {
      vd_masses(sh, row_parts, in.nch, mp, c);
      __syncthreads();
      if (without && threadIdx.x == 0) sh.mass[d.without / kVdChunk] = s;
    }
#pragma unroll 1
    for (int more = residual || without ? 1 : 0;; --more) {
      token = vd_draw(sh, d, in.cols, in.nch, in.v[seq]);
      if (token != YX_NO_TOKEN || more == 0) break;  // uniform
      // Nothing is left (p nowhere above q, or the rejected token is all): p itself.
      d.y = nullptr;
      d.without = YX_NO_TOKEN;
      __syncthreads();
      vd_masses(sh, row_parts, in.nch, mp, c);
    }
  }
  if (threadIdx.x == 0) next[seq] = token;
}

}  // namespace yx
