// Log probabilities of given tokens, entropy and top alternatives of each row of logits, on
// MI355X. With M the row's maximum, S = sum e^(x-M) and U = sum (x-M) e^(x-M) (f32):
//   log p_i = (x_i - M) - log S,  H = log S - U / S.
// Alternatives: the largest logits, larger value first, then lower index; NaN and -inf are
// never one. A row with nothing above -inf has no distribution: -inf, entropy 0, no
// alternatives. A NaN or +inf makes S, so the row's log probabilities and entropy, NaN.
//
// Bound by reading the logits once. A row is read by one workgroup or, where rows are few, by
// several (slices), in chunks of 8192 logits, each thread's 32 in registers; the other workgroups
// of a CU have theirs on the way. Sums: every thread keeps a maximum of its own (m, s, u rescaled when it rises); the
// threads meet once, at the slice's end.
// Alternatives: the `top` best keys so far (argmax_key: value, then lower index; unique) lie
// sorted in LDS; a chunk's logits at or above the last of them are appended and everything is
// ranked by counting (~20 of 8192 in a row's second chunk, fewer later; a chunk without any
// costs a barrier). A first chunk has no list: the top-th largest of 64 groups' maxima (a group:
// the 128 logits of one lane number) is a value that at least `top` logits reach. More than a
// list of 256 (many equal values, or large ones in few groups) takes `top` rounds of a maximum
// over the chunk instead.
// Slices hand their sums and sorted keys over through memory all XCDs share; the last of a row
// to arrive (a counter, left at zero) joins them in slice order: the same bits every time.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/yaxus_hip.h"
#include "step_after.hpp"

namespace yx {

static constexpr int kLpThreads = 256;
static constexpr int kLpQuads = 8;          // 16-byte loads of a thread per chunk
static constexpr int kLpMaxSlices = 64;
static constexpr uint32_t kLpList = 256;    // candidates ranked at once, the best so far included

struct LogprobsOut {
  float* logprob;       // [rows][given] (null: none)
  float* entropy;       // [rows] (null: none)
  uint32_t* top_ids;    // [rows][top]
  float* top_logprobs;  // [rows][top]
};

// Key of a logit as a candidate: as argmax_key, and 0 (none) for -inf too.
__device__ __forceinline__ unsigned long long top_key(float v, uint32_t i) {
  return v > -INFINITY ? argmax_key(v, i) : 0ull;
}

// The value of a key's upper half (-0 comes back as +0).
__device__ __forceinline__ float ord_value(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

// Sums of e^(x - m) and (x - m) log2(e) e^(x - m) over some logits and their maximum m.
struct LpSums {
  float m, s, u;
  // The same relative to a maximum r >= m (m -inf: no logits yet, s = u = 0).
  __device__ __forceinline__ void rebase(float r) {
    const float d = fmaxf((m - r) * 1.44269504f, -300.0f), e = __builtin_amdgcn_exp2f(d);
    u = e * fmaf(d, s, u);
    s = e * s;
    m = r;
  }
  __device__ __forceinline__ void add(const LpSums& o) {
    s += o.s;
    u += o.u;
  }
};

struct LpShared {
  unsigned long long list[kLpList];  // the best so far, then a chunk's candidates
  unsigned long long best[4];
  LpSums sums[4];
  uint32_t ord[kLpThreads];
  uint32_t count[3];
  uint32_t last;
};

// The workgroup's largest key, to all its threads.
__device__ __forceinline__ unsigned long long lp_max(LpShared& sh, unsigned long long k) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const unsigned long long o = __shfl_xor(k, off);
    k = o > k ? o : k;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.best[threadIdx.x >> 6] = k;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) k = sh.best[i] > k ? sh.best[i] : k;
  return k;
}

// list[0 .. n): its `top` largest keys to the front, sorted, zeros behind fewer. n <= kLpList.
__device__ __forceinline__ void lp_rank(LpShared& sh, uint32_t n, uint32_t top) {
  const uint32_t tid = threadIdx.x;
  const unsigned long long k = tid < n ? sh.list[tid] : 0ull;
  uint32_t rank = 0;
  if ((tid & ~63u) < n)  // this wave has some
    for (uint32_t i = 0; i < n; ++i) rank += sh.list[i] > k ? 1 : 0;
  __syncthreads();
  if (tid < top) sh.list[tid] = 0ull;
  __syncthreads();
  if (k && rank < top) sh.list[rank] = k;
  __syncthreads();
}

// Of the 64 lanes' values (order-preserving bits, 0: none) one that at least `top` of them reach,
// the largest or, found early, one between it and the next; 0 if fewer than `top` have one.
__device__ __forceinline__ uint32_t lp_reach(uint32_t o, uint32_t top) {
  uint32_t least = 0;
  for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
    const uint32_t n = __popcll(__ballot(o >= (least | bit)));
    if (n >= top) least |= bit;
    if (n == top) break;
  }
  return least;
}

// `top` rounds of a maximum over each thread's keys (best(below) gives its largest key under
// `below`), appended to list[top ..]: where there are more candidates than the list holds.
template <class F>
__device__ __forceinline__ uint32_t lp_rounds(LpShared& sh, uint32_t top, F best) {
  unsigned long long below = ~0ull;
  uint32_t n = top;
  for (; n < 2 * top; ++n) {
    const unsigned long long k = lp_max(sh, best(below));
    if (!k) break;
    if (threadIdx.x == 0) sh.list[n] = k;
    below = k;
  }
  __syncthreads();
  return n;
}

// Grid: (rows, slices), slices of `per` quads of logits (the last may be shorter). parts [rows][slices] sums and keys [rows][slices][top] are scratch,
// counters [rows] zero on entry and left at zero (slices > 1 only).
__global__ __launch_bounds__(kLpThreads, 4) void logprobs_rows(const float* __restrict__ logits, uint32_t cols,
                                                               size_t ld, const uint32_t* __restrict__ tokens,
                                                               uint32_t given, uint32_t top, LogprobsOut out,
                                                               uint32_t per, unsigned long long* __restrict__ keys,
                                                               float* __restrict__ parts,
                                                               uint32_t* __restrict__ counters) {
  __shared__ LpShared sh;
  const uint32_t row = blockIdx.x, slice = blockIdx.y, nsl = gridDim.y, tid = threadIdx.x;
  const int wave = tid >> 6, lane = tid & 63;
  const float* lr = logits + row * ld;
  constexpr uint32_t kChunk = kLpThreads * kLpQuads;  // in quads
  const uint32_t quads = (cols + 3) / 4;
  const uint32_t q0 = slice * per, q1 = min(quads, q0 + per);
  f32x4 v[kLpQuads];
  const auto load = [&](uint32_t qb) {  // past the slice's end: -inf
    if (qb + kChunk <= q1 && qb + kChunk <= cols / 4) {  // uniform
      const __amdgpu_buffer_rsrc_t r = make_rsrc(const_cast<float*>(lr + 4 * static_cast<size_t>(qb)), kChunk * 16);
#pragma unroll
      for (int i = 0; i < kLpQuads; ++i)
        v[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, tid * 16, i * kLpThreads * 16, 2));
    } else {
#pragma unroll
      for (int i = 0; i < kLpQuads; ++i) {
        const uint32_t q = qb + i * kLpThreads + tid;
        v[i] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (q < min(q1, cols / 4)) v[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(lr) + q);
      }
      const uint32_t end = cols / 4 - qb;  // the row's last, partial quad
      if (cols / 4 < q1 && tid == end % kLpThreads && end < kChunk) {
        const float* p = lr + 4 * static_cast<size_t>(cols / 4);
        const f32x4 x = {p[0], (cols & 3) > 1 ? p[1] : -INFINITY, (cols & 3) > 2 ? p[2] : -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kLpQuads; ++i)
          if (i == static_cast<int>(end / kLpThreads)) v[i] = x;
      }
    }
  };
  load(q0);
  // The first given tokens' logits, on their way while the row is read.
  uint32_t tok = 0;
  float tok_x = -INFINITY;
  if (tid < given) {
    tok = tokens[static_cast<size_t>(row) * given + tid];
    if (tok < cols) tok_x = lr[tok];
  }
  if (tid < 3) sh.count[tid] = top;
  if (tid < top) sh.list[tid] = 0ull;
  __syncthreads();

  LpSums a{-INFINITY, 0.0f, 0.0f};
  unsigned long long floor = 1ull;  // candidates have at least this key
  uint32_t turn = 0;                // chunk number modulo 3
  const auto chunk = [&](uint32_t qb) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kLpQuads; ++i)  // (the instruction itself: fmaxf would canonicalise its operands)
      asm("v_max3_f32 %0, %0, %1, %2\n\tv_max3_f32 %0, %0, %3, %4" : "+&v"(m) : "v"(v[i].x), "v"(v[i].y), "v"(v[i].z), "v"(v[i].w));
    const float ref = fmaxf(a.m, m), base = ref == -INFINITY ? 0.0f : ref;
    a.rebase(ref == -INFINITY ? a.m : ref);
    float s[4] = {0, 0, 0, 0}, u[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kLpQuads; ++i) {
      if (qb + i * kLpThreads >= q1) break;  // uniform
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float d = (v[i][j] - base) * 1.44269504f, e = __builtin_amdgcn_exp2f(d);
        s[j] += e;
        u[j] = fmaf(fmaxf(d, -300.0f), e, u[j]);
      }
    }
    const float chunk_s = (s[0] + s[1]) + (s[2] + s[3]);
    a.s += chunk_s;
    a.u += (u[0] + u[1]) + (u[2] + u[3]);
    if (top == 0) return;
    if (chunk_s != chunk_s) {  // a signalling NaN may have cost v_max3 the maximum so far
      m = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4 * kLpQuads; ++i) m = v[i / 4][i % 4] > m ? v[i / 4][i % 4] : m;
    }

    if (floor == 1ull) {  // fewer than `top` so far: a value that `top` logits reach, if that many are
      sh.ord[tid] = static_cast<uint32_t>(top_key(m, 0) >> 32);
      __syncthreads();
      const uint32_t o = max(max(sh.ord[lane], sh.ord[64 + lane]), max(sh.ord[128 + lane], sh.ord[192 + lane]));
      floor = max(1ull, static_cast<unsigned long long>(lp_reach(o, top)) << 32);
    }
    uint32_t* count = &sh.count[turn];
    // (-3.4e38: any number. -inf would let in every masked logit, 32 turns of the loop below for
    // each thread of a masked row.)
    const uint32_t fo = static_cast<uint32_t>(floor >> 32);
    const float reach = fo > 0x00800000u ? ord_value(fo) : -3.402823466e38f;
    if (m >= reach) {
      uint32_t hits = 0;  // bit 4 i + j: v[i][j]
#pragma unroll
      for (int i = 0; i < 4 * kLpQuads; ++i) hits |= v[i / 4][i % 4] >= reach ? 1u << i : 0u;
      while (hits) {
        const int at = __builtin_ctz(hits);
        hits &= hits - 1;
        float x = v[0][0];
#pragma unroll
        for (int i = 1; i < 4 * kLpQuads; ++i) x = at == i ? v[i / 4][i % 4] : x;
        const unsigned long long k = top_key(x, 4 * (qb + at / 4 * kLpThreads + tid) + at % 4);
        if (k >= floor) {
          const uint32_t p = atomicAdd(count, 1u);
          if (p < kLpList) sh.list[p] = k;
        }
      }
    }
    __syncthreads();
    uint32_t n = *count;
    turn = turn == 2 ? 0 : turn + 1;
    // The counter of the chunk after next: read before the barrier above, used after the next.
    if (tid == 0) sh.count[turn == 2 ? 0 : turn + 1] = top;
    if (n == top) return;  // uniform: no candidates
    if (n > kLpList)
      n = lp_rounds(sh, top, [&](unsigned long long below) {  // (from memory: in a cache, and no registers)
        unsigned long long best = 0;
        const uint32_t e1 = min(cols, 4 * min(q1, qb + kChunk));
        for (uint32_t e = 4 * qb + tid; e < e1; e += kLpThreads) {
          const unsigned long long k = top_key(lr[e], e);
          if (k < below && k > best) best = k;
        }
        return best;
      });
    lp_rank(sh, n, top);
    floor = sh.list[top - 1] + 1;  // a full list: above its last
  };
  for (uint32_t qb = q0; qb < q1; qb += kChunk) {
    if (qb != q0) load(qb);
    chunk(qb);
  }

  // The slice's sums, to all threads.
  const auto join = [&](LpSums& v) {  // over the lanes of a wave
    float m = v.m;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    if (m > -INFINITY) v.rebase(m);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v.add(LpSums{m, __shfl_xor(v.s, off), __shfl_xor(v.u, off)});
  };
  join(a);
  if (lane == 0) sh.sums[wave] = a;
  __syncthreads();
  a = lane < 4 ? sh.sums[lane] : LpSums{-INFINITY, 0.0f, 0.0f};
  join(a);

  if (nsl > 1) {
    const size_t at = static_cast<size_t>(row) * nsl + slice;
    if (tid < top) __hip_atomic_store(keys + at * top + tid, sh.list[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (tid < 3)
      __hip_atomic_store(parts + at * 4 + tid, tid == 0 ? a.m : tid == 1 ? a.s : a.u, __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
      uint32_t* cnt = counters + static_cast<size_t>(row) * kCounterStride;
      const uint32_t arrived = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      sh.last = arrived == nsl - 1;
      if (sh.last) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!sh.last) return;
    const size_t first = static_cast<size_t>(row) * nsl;
    a = LpSums{-INFINITY, 0.0f, 0.0f};
    if (lane < nsl) {
      const float* p = parts + (first + lane) * 4;
      a.m = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      a.s = __hip_atomic_load(p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      a.u = __hip_atomic_load(p + 2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (top) {
      // Candidates are the keys that `top` of the slices' first ones (64 of them: the best of each
      // of 64 slices, the best two of 32, ...) reach.
      constexpr int kMost = kLpMaxSlices * YX_MAX_TOP / kLpThreads;
      const auto key = [&](uint32_t s, uint32_t r) {
        return __hip_atomic_load(keys + (first + s) * top + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      };
      const unsigned long long head = lane / nsl < top ? key(lane % nsl, lane / nsl) : 0ull;
      unsigned long long k[kMost];
#pragma unroll
      for (int i = 0; i < kMost; ++i) {
        const uint32_t e = i * kLpThreads + tid;
        k[i] = e < nsl * top ? key(0, e) : 0ull;
      }
      if (tid == 0) sh.count[0] = top;
      if (tid < top) sh.list[tid] = 0ull;
      __syncthreads();
      const unsigned long long least = max(1ull, static_cast<unsigned long long>(lp_reach(static_cast<uint32_t>(head >> 32), top)) << 32);
#pragma unroll
      for (int i = 0; i < kMost; ++i)
        if (k[i] >= least) {
          const uint32_t p = atomicAdd(&sh.count[0], 1u);
          if (p < kLpList) sh.list[p] = k[i];
        }
      __syncthreads();
      uint32_t n = sh.count[0];
      if (n > kLpList)
        n = lp_rounds(sh, top, [&](unsigned long long below) {
          unsigned long long best = 0;
#pragma unroll
          for (int i = 0; i < kMost; ++i)
            if (k[i] < below && k[i] > best) best = k[i];
          return best;
        });
      lp_rank(sh, n, top);
    }
    join(a);
  }

  const float m = a.m == -INFINITY ? 0.0f : a.m;
  const float log_s = a.s == 0.0f ? 0.0f : logf(a.s);
  if (out.entropy && tid == 0) out.entropy[row] = a.s == 0.0f ? 0.0f : log_s - a.u * 0.693147181f / a.s;
  if (tid < given) out.logprob[static_cast<size_t>(row) * given + tid] = (tok_x - m) - log_s;
  for (uint32_t i = kLpThreads + tid; i < given; i += kLpThreads) {
    const uint32_t t = tokens[static_cast<size_t>(row) * given + i];
    out.logprob[static_cast<size_t>(row) * given + i] = ((t < cols ? lr[t] : -INFINITY) - m) - log_s;
  }
  if (tid < top) {
    const unsigned long long k = sh.list[tid];
    out.top_ids[static_cast<size_t>(row) * top + tid] = k ? ~static_cast<uint32_t>(k) : YX_NO_TOKEN;
    out.top_logprobs[static_cast<size_t>(row) * top + tid] =
        k ? (ord_value(static_cast<uint32_t>(k >> 32)) - m) - log_s : -INFINITY;
  }
}

}  // namespace yx
