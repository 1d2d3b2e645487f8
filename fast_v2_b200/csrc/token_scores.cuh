// Scores of tokens from a row of logits x [vocab]:
//   lse = m + ln z,  m = max_v x_v,  z = sum_v exp(x_v - m)
//   logprob = x_target - lse
//   entropy = ln z - sum_v exp(x_v - m) (x_v - m) / z
//   top[i]  = the k tokens of largest x, the lower index first among equals,
//             with x - lse
// A target below 0 scores 0 (a row without a target); one past the
// vocabulary scores NaN and is reported.  A row that is no distribution (a
// NaN, +inf, or nothing above -inf) gives NaN everywhere and tokens -1, and
// is reported.
//
// One CTA per row: one pass for the sums, then a pass per top token that
// finds the best entry behind the last one.
#pragma once
#include "common.cuh"
#include "norm_rope.cuh"

namespace fdl {

constexpr int kTokThreads = 512;
constexpr int kTokWarps = kTokThreads / 32;
constexpr int kTokMaxTop = 32;

struct TokScoreArgs {
  const void* x;
  int64_t rs;  // elements
  int V;
  const int64_t* targets;
  float* logprob;
  float* entropy;
  int top;
  float* top_lp;
  int64_t* top_tok;
};

// Whole number in the order of (value, lower index first): the larger wins.
__device__ __forceinline__ uint64_t score_key(float x, int idx) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 ranks as 0
  const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (static_cast<uint64_t>(o) << 32) | (0xffffffffu - static_cast<uint32_t>(idx));
}

template <typename T>
__global__ void __launch_bounds__(kTokThreads) token_scores_kernel(const __grid_constant__ TokScoreArgs a) {
  __shared__ float sh_m[kTokWarps], sh_z[kTokWarps], sh_t[kTokWarps];
  __shared__ uint64_t sh_key[kTokWarps];
  const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* x = static_cast<const T*>(a.x) + static_cast<int64_t>(row) * a.rs;
  float m = -INFINITY;
  bool bad = false;
  for (int v = threadIdx.x; v < a.V; v += kTokThreads) {
    const float f = static_cast<float>(x[v]);
    bad |= !(f < INFINITY);
    m = fmaxf(m, f);
  }
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if (lane == 0) sh_m[warp] = m;
  bad = __syncthreads_or(bad);
  for (int w = 0; w < kTokWarps; ++w) m = fmaxf(m, sh_m[w]);
  bad |= m == -INFINITY;
  if (bad) {
    if (threadIdx.x == 0) {
      report(FDL_DEV_INDEX, row);
      a.logprob[row] = NAN;
      a.entropy[row] = NAN;
    }
    for (int i = threadIdx.x; i < a.top; i += kTokThreads) {
      a.top_lp[static_cast<int64_t>(row) * a.top + i] = NAN;
      a.top_tok[static_cast<int64_t>(row) * a.top + i] = -1;
    }
    return;
  }
  float z = 0.f, t = 0.f;
  for (int v = threadIdx.x; v < a.V; v += kTokThreads) {
    const float d = static_cast<float>(x[v]) - m;
    const float e = expf(d);
    z += e;
    if (e > 0.f) t = fmaf(e, d, t);
  }
  for (int off = 16; off > 0; off >>= 1) {
    z += __shfl_xor_sync(0xffffffffu, z, off);
    t += __shfl_xor_sync(0xffffffffu, t, off);
  }
  if (lane == 0) {
    sh_z[warp] = z;
    sh_t[warp] = t;
  }
  __syncthreads();
  z = t = 0.f;
  for (int w = 0; w < kTokWarps; ++w) {
    z += sh_z[w];
    t += sh_t[w];
  }
  const float lz = logf(z);
  if (threadIdx.x == 0) {
    const int64_t tg = a.targets[row];
    float lp = 0.f;
    if (tg >= a.V) {
      report(FDL_DEV_INDEX, tg);
      lp = NAN;
    } else if (tg >= 0) {
      lp = static_cast<float>(x[tg]) - m - lz;
    }
    a.logprob[row] = lp;
    a.entropy[row] = lz - t / z;
  }
  uint64_t last = ~0ull;
  for (int i = 0; i < a.top; ++i) {
    uint64_t best = 0;
    for (int v = threadIdx.x; v < a.V; v += kTokThreads) {
      const uint64_t key = score_key(static_cast<float>(x[v]), v);
      if (key < last && key > best) best = key;
    }
    for (int off = 16; off > 0; off >>= 1) {
      const uint64_t o = __shfl_xor_sync(0xffffffffu, best, off);
      best = best > o ? best : o;
    }
    if (lane == 0) sh_key[warp] = best;
    __syncthreads();
    for (int w = 0; w < kTokWarps; ++w) best = best > sh_key[w] ? best : sh_key[w];
    __syncthreads();
    last = best;
    if (threadIdx.x == 0) {
      const int tok = static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
      a.top_tok[static_cast<int64_t>(row) * a.top + i] = tok;
      a.top_lp[static_cast<int64_t>(row) * a.top + i] = static_cast<float>(x[tok]) - m - lz;
    }
  }
}

}  // namespace fdl
