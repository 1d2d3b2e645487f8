// Attention of one new token per sequence over a paged KV cache:
//   o[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q[b,h].k_j - m),
//   m = max_j scale * q[b,h].k_j,  j < lens[b],
// with k_j, v_j row j % page of page table[b, j / page], head h / (hq / hkv).
// A sequence without a visible key gives zeros.  A page outside the pool
// hides its keys and is reported.
//
// One CTA per (sequence, query head): every warp walks its own keys with a
// running maximum and sum, lanes share the head's elements, and the warps'
// states are joined at the end.
#pragma once
#include "common.cuh"
#include "norm_rope.cuh"

namespace fdl {

struct PagedAttnArgs {
  const void* q;
  int64_t q_sb, q_sh;       // elements
  const char* k;
  const char* v;
  int64_t sp, ss, sh;       // bytes
  const int32_t* table;
  int64_t table_sb;
  const int32_t* lens;
  void* out;
  int64_t o_sb, o_sh;
  int B, hq, hkv, num_pages, max_pages;
  FastDiv page;
  float scale_log2;
};

constexpr int kPagedThreads = 128;

template <typename T, int D>
__global__ void __launch_bounds__(kPagedThreads) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
  constexpr int E = D / 32;  // elements per lane
  __shared__ float s_o[kPagedThreads / 32][D];
  __shared__ float s_m[kPagedThreads / 32], s_l[kPagedThreads / 32];
  const int b = blockIdx.y, h = blockIdx.x, kh = h / (a.hq / a.hkv);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int len = a.lens[b];
  const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page.d;
  if (len < 0 || len > cap) {
    if (threadIdx.x == 0) report(FDL_DEV_LENGTH, b);
    len = len < 0 ? 0 : static_cast<int>(cap);
  }
  const T* q = static_cast<const T*>(a.q) + b * a.q_sb + h * a.q_sh + lane * E;
  float qf[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qf[e] = static_cast<float>(q[e]) * a.scale_log2;
    o[e] = 0.f;
  }
  for (int j = warp; j < len; j += kPagedThreads / 32) {
    uint32_t i, r;
    a.page.divmod(j, i, r);
    const int page = a.table[b * a.table_sb + i];
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0) report(FDL_DEV_INDEX, page);
      continue;
    }
    const int64_t at = page * a.sp + r * a.ss + kh * a.sh;
    const T* k = reinterpret_cast<const T*>(a.k + at) + lane * E;
    const T* v = reinterpret_cast<const T*>(a.v + at) + lane * E;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(qf[e], static_cast<float>(k[e]), s);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    const float mn = fmaxf(m, s);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float p = exp2f(s - ref), c = exp2f(m - ref);
    l = l * c + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(p, static_cast<float>(v[e]), o[e] * c);
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  float M = -INFINITY, Lsum = 0.f;
  for (int w = 0; w < kPagedThreads / 32; ++w) M = fmaxf(M, s_m[w]);
  const float ref = M == -INFINITY ? 0.f : M;
  for (int w = 0; w < kPagedThreads / 32; ++w) Lsum += s_l[w] * exp2f(s_m[w] - ref);
  T* out = static_cast<T*>(a.out) + b * a.o_sb + h * a.o_sh;
  for (int d = threadIdx.x; d < D; d += kPagedThreads) {
    float x = 0.f;
    for (int w = 0; w < kPagedThreads / 32; ++w) x += s_o[w][d] * exp2f(s_m[w] - ref);
    out[d] = static_cast<T>(Lsum > 0.f || Lsum != Lsum ? x / Lsum : 0.f);
  }
}

}  // namespace fdl
