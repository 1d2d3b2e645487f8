// Scores of tokens from a row of logits x [vocab]:
//   lse = m + ln z,  m = max_v x_v,  z = sum_v exp(x_v - m)
//   logprob = x_target - lse
//   entropy = ln z - t / z,  t = sum_v exp(x_v - m) (x_v - m)
//   top[i]  = the k tokens of largest x, the lower index first among equals,
//             with x - lse
// A target below 0 scores 0 (a row without a target); one past the
// vocabulary scores NaN and is reported.  A row that is no distribution (a
// NaN, +inf, or nothing above -inf) gives NaN everywhere and tokens -1, and
// is reported.
//
// Bound by HBM (the special-function unit is at 70% of its rate at the copy
// rate in a 16-bit type), so the row is read once: a cluster of 1 to 8 CTAs
// takes a row, every thread walks 16-byte vectors of it with sums relative to
// a reference of its own (moved only when a logit passes it by kTokSlack) and
// remembers the largest logit it saw and where.
//
// The top k need no second pass over the row.  Order all entries by (logit,
// lower index first).  If each of W warps has r >= k / W threads whose largest
// entry is at or above tau, then at least k entries are, so every one of the
// top k is -- and lies with a thread whose largest entry is at or above tau.
// tau is the smallest over these warps of the r-th largest thread maximum;
// only the vectors of the threads at or above it are read again (some tens of
// the 512, from L2), the entries at or above tau are collected and sorted: in
// each warp by a bitonic network, then list by list in a tree that keeps the
// best 32.  Rows with very many entries above tau (long runs of equal logits,
// say) overflow the list; the k-th best of the entries caught is then a
// better tau.
#pragma once
#include "common.cuh"
#include "device_util.cuh"

namespace fdl {

constexpr int kTokThreads = 512;
constexpr int kTokWarps = kTokThreads / 32;
constexpr int kTokMaxTop = 32;
constexpr int kTokUnroll = 4;     // vectors in flight a thread
constexpr float kTokSlack = 10.f;
constexpr float kTokLog2e = 1.4426950408889634f;
constexpr float kTokFloor = -1000.f;  // exp() of it is 0 in fp32; keeps 0 * inf out of t

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
__device__ __forceinline__ uint64_t score_key(float x, uint32_t idx) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 ranks as 0
  const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (static_cast<uint64_t>(o) << 32) | (0xffffffffu - idx);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t min64(uint64_t a, uint64_t b) { return a < b ? a : b; }

// One compare-exchange step of a network over the warp's lanes: the lane
// whose bit `off` is clear keeps the larger key when `down`.
__device__ __forceinline__ uint64_t exchange(uint64_t key, int off, bool down) {
  const uint64_t o = __shfl_xor_sync(0xffffffffu, key, off);
  return ((threadIdx.x & off) == 0) == down ? max64(key, o) : min64(key, o);
}
// Sorts the warp's 32 keys, largest in lane 0.
__device__ __forceinline__ uint64_t warp_sort(uint64_t key) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int off = size / 2; off > 0; off >>= 1) key = exchange(key, off, (threadIdx.x & size & 31) == 0);
  return key;
}
// The best 32 of two sorted lists, sorted: lane i holds one, and is given
// entry 31 - i of the other.
__device__ __forceinline__ uint64_t warp_merge(uint64_t key, uint64_t other_reversed) {
  key = max64(key, other_reversed);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) key = exchange(key, off, true);
  return key;
}
// Warps 0 .. lists - 1 hold a sorted list each; warp 0 ends with the best 32.
// Every thread of the CTA calls it; sh is free again after the next barrier.
__device__ __forceinline__ uint64_t block_merge(uint64_t key, int lists, uint64_t (*sh)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int step = 1; step < lists; step <<= 1) {
    if (warp < lists && (warp & (2 * step - 1)) == step) sh[warp][lane] = key;
    __syncthreads();
    if ((warp & (2 * step - 1)) == 0 && warp + step < lists) key = warp_merge(key, sh[warp + step][31 - lane]);
  }
  return key;
}

template <typename T>
struct TokVec {  // 16 bytes of logits
  static constexpr int kN = 16 / sizeof(T);
  float f[kN];
  __device__ __forceinline__ explicit TokVec(uint4 u) {
    if constexpr (sizeof(T) == 4) {
      f[0] = __uint_as_float(u.x);
      f[1] = __uint_as_float(u.y);
      f[2] = __uint_as_float(u.z);
      f[3] = __uint_as_float(u.w);
    } else {
      unpack8<T>(u, f);
    }
  }
  __device__ __forceinline__ float max() const {
    float m = f[0];
#pragma unroll
    for (int e = 1; e < kN; ++e) m = fmaxf(m, f[e]);
    return m;
  }
};

// Sums relative to a reference: z = sum exp(x - ref), t = sum exp(x - ref) (x - ref).
struct TokSums {
  float ref, z, t;
  __device__ __forceinline__ void move(float to) {  // to >= ref
    const float d = fmaxf(ref - to, kTokFloor), f = ex2(d * kTokLog2e);
    t = f * fmaf(d, z, t);
    z *= f;
    ref = to;
  }
  __device__ __forceinline__ void add(float x) {
    float d = x - ref;
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(d) : "f"(kTokFloor));
    const float e = ex2(d * kTokLog2e);
    z += e;
    t = fmaf(e, d, t);
  }
};

template <typename T>
__global__ void __launch_bounds__(kTokThreads) token_scores_kernel(const __grid_constant__ TokScoreArgs a) {
  constexpr int kN = TokVec<T>::kN;
  __shared__ float sh_m[kTokWarps], sh_z[kTokWarps], sh_t[kTokWarps];
  __shared__ uint64_t sh_tau[kTokWarps];
  __shared__ uint64_t sh_list[kTokWarps][32];
  __shared__ uint64_t sh_cand[kTokThreads];
  __shared__ uint64_t sh_top[32];
  __shared__ float4 sh_sum;
  __shared__ int sh_n;
  await_stream();
  release_stream();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t ranks = cluster_size(), rank = cluster_rank();
  const int row = blockIdx.x / ranks;
  const T* x = static_cast<const T*>(a.x) + static_cast<int64_t>(row) * a.rs;
  // The row: `head` entries up to a 16-byte boundary, whole vectors shared out
  // over the CTAs of the cluster, and the rest.
  const int head = min(a.V, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
  const int nvec = (a.V - head) / kN, rest = a.V - head - nvec * kN;
  const int v0 = static_cast<int>(static_cast<int64_t>(nvec) * rank / ranks);
  const int nv = static_cast<int>(static_cast<int64_t>(nvec) * (rank + 1) / ranks) - v0;
  const char* vec = reinterpret_cast<const char*>(x + head) + static_cast<int64_t>(v0) * 16;
  const int first = head + v0 * kN;  // index of this CTA's first vector entry
  // The entry outside the vectors that this thread holds, or -1.
  int single = -1;
  if (rank == 0 && threadIdx.x < head) single = threadIdx.x;
  if (rank == ranks - 1 && threadIdx.x >= 32 && threadIdx.x - 32 < rest) single = a.V - rest + threadIdx.x - 32;

  // ---- the one pass
  TokSums s{-3.402823466e38f, 0.f, 0.f};
  float best = -INFINITY;  // largest entry in this thread's vectors, and the first vector that has it
  int at = threadIdx.x;
  auto take = [&](uint4 u, int v) {
    const TokVec<T> q(u);
    const float m = q.max();
    if (m > best) {
      best = m;
      at = v;
    }
    if (m > s.ref + kTokSlack) s.move(m);
#pragma unroll
    for (int e = 0; e < kN; ++e) s.add(q.f[e]);
  };
  int v = threadIdx.x;
  for (; v + (kTokUnroll - 1) * kTokThreads < nv; v += kTokUnroll * kTokThreads) {
    uint4 u[kTokUnroll];
#pragma unroll
    for (int i = 0; i < kTokUnroll; ++i) u[i] = ld_stream16(vec + static_cast<int64_t>(v + i * kTokThreads) * 16);
#pragma unroll
    for (int i = 0; i < kTokUnroll; ++i) take(u[i], v + i * kTokThreads);
  }
  for (; v < nv; v += kTokThreads) take(ld_stream16(vec + static_cast<int64_t>(v) * 16), v);
  float lone = -INFINITY;
  if (single >= 0) {
    lone = static_cast<float>(x[single]);
    if (lone > s.ref) s.move(lone);
    s.add(lone);
  }

  // ---- sums of the CTA, relative to its largest entry
  float m = fmaxf(best, lone);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if (lane == 0) sh_m[warp] = m;
  // the r-th largest thread maximum of the warp; a maximum counts as the last
  // entry of its vector, mine + kN - 1 is the first
  const uint64_t mine = threadIdx.x < nv ? score_key(best, first + at * kN + kN - 1) : 0;
  const int full = min(nv / 32, kTokWarps);  // warps with a vector for every thread
  if (a.top > 0 && warp < full) {
    const int r = (a.top + full - 1) / full;
    uint64_t big = 0;
    if (r <= 2) {
      uint64_t left = mine;
      for (int i = 0; i < r; ++i) {
        big = left;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) big = max64(big, __shfl_xor_sync(0xffffffffu, big, off));
        if (left == big) left = 0;
      }
    } else {
      big = __shfl_sync(0xffffffffu, warp_sort(mine), r - 1);
    }
    if (lane == 0) sh_tau[warp] = big;
  }
  if (threadIdx.x == 0) sh_n = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kTokWarps; ++w) m = fmaxf(m, sh_m[w]);
  // a CTA that has seen nothing above -inf keeps z = 0
  s.move(fmaxf(m, s.ref));
  const float ref = s.ref;  // threads without a larger entry agree on max(m, lowest)
  float z = s.z, t = s.t;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    z += __shfl_xor_sync(0xffffffffu, z, off);
    t += __shfl_xor_sync(0xffffffffu, t, off);
  }
  if (lane == 0) {
    sh_z[warp] = z;
    sh_t[warp] = t;
  }

  // ---- the top entries of the CTA
  uint64_t key = 0;
  if (a.top > 0) {
    uint64_t tau = full > 0 ? sh_tau[0] : 0;  // below 32 vectors all entries fit the list
    for (int w = 1; w < full; ++w) tau = min64(tau, sh_tau[w]);
    for (;;) {
      auto offer = [&](float f, int idx) {
        const uint64_t k = score_key(f, idx);
        if (k >= tau) {
          const int n = atomicAdd(&sh_n, 1);
          if (n < kTokThreads) sh_cand[n] = k;
        }
      };
      for (unsigned who = __ballot_sync(0xffffffffu, threadIdx.x < nv && mine + (kN - 1) >= tau); who; who &= who - 1) {
        const int owner = warp * 32 + __ffs(who) - 1;
        for (int i = owner + lane * kTokThreads; i < nv; i += 32 * kTokThreads) {
          const TokVec<T> q(*reinterpret_cast<const uint4*>(vec + static_cast<int64_t>(i) * 16));
#pragma unroll
          for (int e = 0; e < kN; ++e) offer(q.f[e], first + i * kN + e);
        }
      }
      if (single >= 0) offer(lone, single);
      __syncthreads();
      const int n = sh_n;
      // warps behind the last candidate hold empty lists
      key = threadIdx.x < min(n, kTokThreads) ? sh_cand[threadIdx.x] : 0;
      if (warp * 32 < n) key = warp_sort(key);
      key = block_merge(key, (min(n, kTokThreads) + 31) / 32, sh_list);
      if (n <= kTokThreads) break;
      if (threadIdx.x == a.top - 1) sh_tau[0] = key;
      __syncthreads();
      tau = sh_tau[0];
      if (threadIdx.x == 0) sh_n = 0;
      __syncthreads();
    }
  }
  __syncthreads();
  z = t = 0.f;
#pragma unroll
  for (int w = 0; w < kTokWarps; ++w) {
    z += sh_z[w];
    t += sh_t[w];
  }
  TokSums row_s{ref, z, t};
  if (ranks > 1) {
    if (warp == 0) sh_top[lane] = key;
    if (threadIdx.x == 0) sh_sum = make_float4(ref, z, t, 0.f);
    cluster_sync();
    if (rank == 0) {
      for (uint32_t r = 1; r < ranks; ++r) {
        const float4 o = ld_cluster4(smem_addr(&sh_sum), r);
        TokSums other{o.x, o.y, o.z};
        const float to = fmaxf(row_s.ref, other.ref);
        row_s.move(to);
        other.move(to);
        row_s.z += other.z;
        row_s.t += other.t;
      }
      if (a.top > 0) {
        if (warp > 0 && warp < ranks) {
          const float2 k2 = ld_cluster2(smem_addr(&sh_top[lane]), warp);
          key = static_cast<uint64_t>(__float_as_uint(k2.y)) << 32 | __float_as_uint(k2.x);
        }
        key = block_merge(key, ranks, sh_list);
      }
    }
    cluster_sync();  // no CTA leaves while its shared memory is read
    if (rank != 0) return;
  }
  const bool bad = !(row_s.z > 0.f && row_s.z < INFINITY);
  const float lz = logf(row_s.z);
  if (threadIdx.x == 0) {
    const int64_t tg = a.targets[row];
    float lp = 0.f;
    if (bad) {
      report(FDL_DEV_INDEX, row);
    } else if (tg >= a.V) {
      report(FDL_DEV_INDEX, tg);
      lp = NAN;
    } else if (tg >= 0) {
      lp = static_cast<float>(x[tg]) - row_s.ref - lz;
    }
    a.logprob[row] = bad ? NAN : lp;
    a.entropy[row] = bad ? NAN : lz - row_s.t / row_s.z;
  }
  if (threadIdx.x < a.top) {
    const int64_t to = static_cast<int64_t>(row) * a.top + threadIdx.x;
    a.top_lp[to] = bad ? NAN : key_value(key) - row_s.ref - lz;
    a.top_tok[to] = bad ? -1 : static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key));
  }
}

}  // namespace fdl
