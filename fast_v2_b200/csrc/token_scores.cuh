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
// Bound by HBM (with 16-bit logits the special-function unit is at 70% of its
// rate at the copy rate), so the row is read once: a warp, or a CTA, or a
// cluster of up to 8 CTAs takes a row, every thread walks 16-byte vectors of
// it with sums relative to a reference of its own (moved only when a logit
// passes it by kTokSlack) and remembers the largest logit it saw and where.
// The sums are kept for powers of two, 2^(x log2 e - ref'), one fused
// multiply-add an entry; ref' is the rounded ref * log2 e, and what the
// rounding is off is known exactly and put right at the end.  The power is the
// hardware's, off by about two steps of fp32: the results are 0.9e-7 to
// 1.3e-7 from 64 bits (512 rows of 152064; exp in full fp32 0.6e-7).
//
// The top k need no second pass over the row.  Order all entries by (logit,
// lower index first).  If there are k threads whose largest entry is at or
// above tau, then at least k entries are, so every one of the top k is -- and
// lies with a thread whose largest entry is at or above tau.  In a CTA tau is
// the k-th largest of the r = ceil(1.5 k / W) largest thread maxima of each of W
// warps (r = ceil(k / W) leaves more to rank: 512 rows, top 32, 49 us against
// 40), in a warp the k-th largest lane maximum; only the vectors of the
// threads at or above it are read again (k and a few, from L2 or L1), the
// entries at or above tau are collected and put in order.  Rows with very many
// entries above tau (long runs of equal logits, say) overflow the list; the
// k-th best of the entries caught is then a better tau.
//
// Measured: 512 rows of 152064 bf16 logits, top 20, 38 us (4.1 TB/s; 32 us
// without the top), 1500 rows of 50257 fp32, top 5, 52 us (5.8 TB/s), 8 rows of
// 152064 8.9 us.
#pragma once
#include <type_traits>

#include "common.cuh"
#include "device_util.cuh"
#include "sm100_ptx.cuh"

namespace fdl {

constexpr int kTokMaxTop = 32;
constexpr int kTokCta = 256;      // threads a row, or half of them
constexpr int kTokRowWarps = 8;   // rows a CTA of the warp form
constexpr int kTokRowList = 320;  // its lists (31 vectors of 8 entries and 14 more fit)
constexpr int kTokList = 512;  // entries above tau that are caught (a cluster of 8 brings 8 * 32)
constexpr int kTokUnroll = 3;  // vectors a batch
constexpr int kTokStages = 4;  // batches of a thread's ring
constexpr float kTokSlack = 10.f;
constexpr float kTokLog2e = 1.4426950408889634f;
constexpr float kTokBig = 1048576.f;  // 2^20: its product with log2 e rounds by 2^-4 at most
constexpr float kTokFloor = -1000.f;  // exp() of it is 0 in fp32; keeps 0 * inf out of t

struct TokScoreArgs {
  const void* x;
  int64_t rs;  // elements
  int V, rows;
  const int64_t* targets;
  float* logprob;
  float* entropy;
  int top;
  float* top_lp;
  int64_t* top_tok;
};

// Whole number in the order of the values (above 0 for all but NaN).
__device__ __forceinline__ uint32_t score_order(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 ranks as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// The same in the order of (value, lower index first): the larger wins.
__device__ __forceinline__ uint64_t order_key(uint32_t order, uint32_t idx) {
  return (static_cast<uint64_t>(order) << 32) | (0xffffffffu - idx);
}
__device__ __forceinline__ uint64_t score_key(float x, uint32_t idx) { return order_key(score_order(x), idx); }
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
// The CTA ranks n <= kTokList distinct keys by counting the larger ones and
// puts the best 32 in order; four threads a key where there are enough.
template <int NT>
__device__ __forceinline__ void block_rank(const uint64_t* cand, int n, uint64_t* best) {
  const int q = n * 4 <= NT ? 4 : 1, part = threadIdx.x % q;
  for (int i0 = 0; i0 < n; i0 += NT) {
    const int i = i0 + threadIdx.x / q;
    const uint64_t key = i < n ? cand[i] : 0;
    int above = 0;
    if (i < n)
      for (int j = part; j < n; j += q) above += cand[j] > key;
    if (q == 4) {
      above += __shfl_xor_sync(0xffffffffu, above, 1);
      above += __shfl_xor_sync(0xffffffffu, above, 2);
    }
    if (i < n && part == 0 && above < kTokMaxTop) best[above] = key;
  }
}

// The finite floor that -inf is raised to in the fast sums.
template <typename T>
constexpr float kTokLowest = std::is_same<T, __half>::value ? -65504.f : -1.2676506e30f;  // -2^100
// max(x, floor) that keeps a NaN, for the entries in a word of logits.
template <typename T>
__device__ __forceinline__ uint32_t clamp_word(uint32_t u) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(u) : "r"(0xf180f180u));  // -2^100
  else if constexpr (std::is_same<T, __half>::value)
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(u) : "r"(0xfbfffbffu));  // -65504
  else {
    float f = __uint_as_float(u);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(f) : "f"(kTokLowest<T>));
    u = __float_as_uint(f);
  }
  return u;
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
  // With -inf (and what is below a finite floor) raised to the floor, whose
  // exponential is 0 next to any reference that the fast sums allow.
  __device__ __forceinline__ static TokVec finite(uint4 u) {
    return TokVec(make_uint4(clamp_word<T>(u.x), clamp_word<T>(u.y), clamp_word<T>(u.z), clamp_word<T>(u.w)));
  }
  // Entry e of a vector, and the entries not below x as bits.
  __device__ __forceinline__ static float pick(uint4 u, int e) {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(e & 2 ? (e & 1 ? u.w : u.z) : (e & 1 ? u.y : u.x));
    } else {
      const float2 two = Pack2<T>::to(e & 4 ? (e & 2 ? u.w : u.z) : (e & 2 ? u.y : u.x));
      return e & 1 ? two.y : two.x;
    }
  }
  __device__ __forceinline__ unsigned reaching(float x) const {
    unsigned bits = 0;
#pragma unroll
    for (int e = 0; e < kN; ++e) bits |= !(f[e] < x) ? 1u << e : 0u;
    return bits;
  }
  __device__ __forceinline__ float max() const {
    float m = fmaxf(f[0], f[1]);
#pragma unroll
    for (int e = 2; e < kN; e += 2) m = ptx::fmax3(m, f[e], f[e + 1]);
    return m;
  }
};

// Sums relative to a reference: z = sum exp(x - ref), t = sum exp(x - ref) (x
// - ref).
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

// The same with powers of two, two finite entries at a time: y = x log2 e -
// refl, z = sum 2^y, t = sum 2^y y.  The reference starts at -kTokBig, below which every
// entry counts as 0; a row whose largest entry is outside +-kTokBig is summed
// again with TokSums.
struct TokSums2 {
  float ref, refl;
  uint64_t z, t;
  __device__ __forceinline__ void start() {
    ref = -kTokBig;
    refl = ref * kTokLog2e;
    z = t = 0;
  }
  __device__ __forceinline__ void move(float to) {
    const float l = to * kTokLog2e, d = fmaxf(refl - l, 2.f * kTokFloor), f = ex2(d);
    const uint64_t f2 = ptx::pack2(f, f);
    t = ptx::mul2(f2, ptx::fma2(ptx::pack2(d, d), z, t));
    z = ptx::mul2(f2, z);
    ref = to;
    refl = l;
  }
  __device__ __forceinline__ void add(float x0, float x1) {
    float y0, y1;
    const uint64_t y = ptx::fma2(ptx::pack2(x0, x1), ptx::pack2(kTokLog2e, kTokLog2e), ptx::pack2(-refl, -refl));
    ptx::unpack2(y, y0, y1);
    const uint64_t e = ptx::pack2(ex2(y0), ex2(y1));
    z = ptx::add2(z, e);
    t = ptx::fma2(e, y, t);
  }
  __device__ __forceinline__ TokSums natural() const {
    float z0, z1, t0, t1;
    ptx::unpack2(z, z0, z1);
    ptx::unpack2(t, t0, t1);
    const float r = fmaf(ref, kTokLog2e, -refl);  // exact: what refl is off
    const float zz = z0 + z1, f = ex2(-r);
    return TokSums{ref, zz * f, f * fmaf(-r, zz, t0 + t1) * 0.6931471805599453f};
  }
};

// One thread's part of the one pass over nv vectors: vectors tid, tid + NT, ..
// in batches of kTokUnroll (the last ones one by one).
template <typename T, int NT>
struct TokPass {
  static constexpr int kN = TokVec<T>::kN, kBatch = kTokUnroll * NT;
  TokSums2 sums;
  // largest entry of the thread's batches, the first batch that has it (its
  // first vector), and the largest entry of the others
  float best, second;
  int at, whole;

  __device__ __forceinline__ void note(float m, int v) {
    second = fmaxf(second, fminf(m, best));
    if (m > best) at = v;
    best = fmaxf(m, best);
    if (m > sums.ref + kTokSlack) sums.move(m);
  }
  __device__ __forceinline__ void add(const TokVec<T>& q) {
#pragma unroll
    for (int e = 0; e < kN; e += 2) sums.add(q.f[e], q.f[e + 1]);
  }
  __device__ __forceinline__ void start(int nv, int tid) {
    sums.start();
    best = second = -INFINITY;
    at = tid;
    whole = nv / kBatch * kBatch;
  }
  __device__ __forceinline__ void batch(const uint4 (&u)[kTokUnroll], int v) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kTokUnroll; ++i) m = fmaxf(m, TokVec<T>::finite(u[i]).max());
    note(m, v);
#pragma unroll
    for (int i = 0; i < kTokUnroll; ++i) add(TokVec<T>::finite(u[i]));
  }
  __device__ __forceinline__ void one(uint4 u, int v) {
    const TokVec<T> q = TokVec<T>::finite(u);
    note(q.max(), v);
    add(q);
  }
  // A CTA's threads: each has a ring of kTokStages batches in shared memory,
  // filled by its own asynchronous copies (nothing is shared, so nothing waits
  // for another thread).  ring: kTokStages * kBatch * 16 bytes of the CTA.
  __device__ __forceinline__ void run_ring(const char* vec, int nv, int tid, char* ring) {
    start(nv, tid);
    const char* src = vec + tid * 16;
    const uint32_t dst = smem_addr(ring) + tid * 16;
    int next = 0, fill = 0;  // first vector and slot of the next batch to load
    auto issue = [&]() {
      if (next < nv) {
#pragma unroll
        for (int i = 0; i < kTokUnroll; ++i)
          if (next < whole || next + tid + i * NT < nv)
            cp_async16(dst + (fill * kTokUnroll + i) * NT * 16, src + i * NT * 16);
        src += kBatch * 16;
        next += kBatch;
        fill = fill + 1 == kTokStages ? 0 : fill + 1;
      }
      cp_commit();
    };
#pragma unroll
    for (int i = 0; i < kTokStages - 1; ++i) issue();
    const uint4* mine = reinterpret_cast<const uint4*>(ring) + tid;
    int use = 0;
    for (int v = 0; v < nv; v += kBatch) {
      issue();
      cp_wait<kTokStages - 1>();
      const uint4* slot = mine + use * kTokUnroll * NT;
      use = use + 1 == kTokStages ? 0 : use + 1;
      if (v < whole) {
        uint4 u[kTokUnroll];
#pragma unroll
        for (int i = 0; i < kTokUnroll; ++i) u[i] = slot[i * NT];
        batch(u, v + tid);
      } else {
#pragma unroll
        for (int i = 0; i < kTokUnroll; ++i)
          if (v + tid + i * NT < nv) one(slot[i * NT], v + tid + i * NT);
      }
    }
  }
  // The warp form reads many vectors of its short row again, so it lets them
  // stay in L1.
  __device__ __forceinline__ static uint4 load(const char* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void run(const char* vec, int nv, int tid) {
    start(nv, tid);
    const char* p = vec + tid * 16;
    uint4 next[kTokUnroll];  // the next batch is on its way while one is summed
    auto fetch = [&](int v) {
      if (v < whole) {
#pragma unroll
        for (int i = 0; i < kTokUnroll; ++i) next[i] = load(p + i * NT * 16);
      } else {
#pragma unroll
        for (int i = 0; i < kTokUnroll; ++i)
          if (v + tid + i * NT < nv) next[i] = load(p + i * NT * 16);
      }
      p += kBatch * 16;
    };
    fetch(0);
    for (int v = 0; v < whole; v += kBatch) {
      uint4 u[kTokUnroll];
#pragma unroll
      for (int i = 0; i < kTokUnroll; ++i) u[i] = next[i];
      fetch(v + kBatch);
      batch(u, v + tid);
    }
#pragma unroll
    for (int i = 0; i < kTokUnroll; ++i) {
      const int v = whole + tid + i * NT;
      if (v < nv) one(next[i], v);
    }
  }
  // The largest entry lies between (least_order(), least_index(first)) -- the
  // last entry of its batch; -inf where the floor hides it -- and most(first),
  // the first one; `first` is the index of vector 0's first entry.
  __device__ __forceinline__ bool hidden() const { return !(best > kTokLowest<T>); }
  __device__ __forceinline__ int last() const { return at < whole ? at + (kTokUnroll - 1) * NT : at; }
  __device__ __forceinline__ uint32_t least_order() const { return score_order(hidden() ? -INFINITY : best); }
  __device__ __forceinline__ uint32_t least_index(int first) const { return first + last() * kN + kN - 1; }
  __device__ __forceinline__ uint64_t most(int first) const { return score_key(best, hidden() ? 0 : first + at * kN); }
  // Whether a batch other than `at` may have an entry at or above tau.
  __device__ __forceinline__ bool more(uint64_t tau) const { return hidden() || score_key(second, 0) >= tau; }
};

template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) token_scores_kernel(const __grid_constant__ TokScoreArgs a) {
  constexpr int kN = TokVec<T>::kN, kWarps = NT / 32;
  extern __shared__ __align__(16) char ring[];
  __shared__ float sh_m[kWarps], sh_z[kWarps], sh_t[kWarps];
  __shared__ uint64_t sh_max[kWarps + kTokMaxTop * 3 / 2];  // the largest thread maxima of each warp
  __shared__ uint64_t sh_tau;
  __shared__ __align__(16) uint64_t sh_cand[kTokList];
  __shared__ uint64_t sh_top[kTokMaxTop];
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

  // the target is read during the pass, its logit behind it
  const int64_t target = rank == 0 && threadIdx.x == 0 ? a.targets[row] : -1;

  // ---- the one pass
  TokPass<T, NT> pass;
  pass.run_ring(vec, nv, threadIdx.x, ring);
  const float target_x = target >= 0 && target < a.V ? static_cast<float>(x[target]) : 0.f;
  TokSums s = pass.sums.natural();
  float lone = -INFINITY;
  if (single >= 0) {
    lone = static_cast<float>(x[single]);
    if (lone > s.ref) s.move(lone);
    s.add(lone);
  }

  // ---- sums of the CTA, relative to its largest entry
  float m = fmaxf(pass.best, lone);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if (lane == 0) sh_m[warp] = m;
  // the r largest thread maxima of each warp
  const int full = min(nv / 32, kWarps);  // warps with a vector for every thread
  const int r = full > 0 ? min(32, (a.top * 3 / 2 + full - 1) / full) : 0;
  if (warp < full) {
    uint32_t order = pass.least_order();
    const uint32_t index = pass.least_index(first);
    for (int i = 0; i < r; ++i) {
      const uint32_t big = __reduce_max_sync(0xffffffffu, order);
      const uint32_t low = __reduce_min_sync(0xffffffffu, order == big ? index : 0xffffffffu);
      if (lane == 0) sh_max[warp * r + i] = order_key(big, low);
      if (index == low) order = 0;
    }
  }
  if (threadIdx.x == 0) {
    sh_n = 0;
    sh_tau = 0;  // below 32 vectors all entries fit the list
  }
  if (threadIdx.x < kTokMaxTop) sh_top[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sh_m[w]);
  if (fabsf(m) > kTokBig || m <= kTokLowest<T>) {
    // Sizes that the fast sums do not hold: again, with the true maximum.  (A
    // CTA that sees nothing above -inf keeps z = 0.)
    auto each = [&](auto f) {
      for (int i = threadIdx.x; i < nv; i += NT) {
        const TokVec<T> q(*reinterpret_cast<const uint4*>(vec + static_cast<int64_t>(i) * 16));
#pragma unroll
        for (int e = 0; e < kN; ++e) f(q.f[e]);
      }
      if (single >= 0) f(lone);
    };
    m = -INFINITY;
    each([&](float x) { m = fmaxf(m, x); });
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    __syncthreads();
    if (lane == 0) sh_m[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sh_m[w]);
    s = TokSums{fmaxf(m, -3.402823466e38f), 0.f, 0.f};
    each([&](float x) { s.add(x); });
  } else if (m > s.ref) {
    s.move(m);
  }
  const float ref = s.ref;
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
  if (threadIdx.x < full * r) {  // the k-th largest of them
    const uint64_t key = sh_max[threadIdx.x];
    int above = 0;
    for (int i = 0; i < full * r; ++i) above += sh_max[i] > key;
    if (above == a.top - 1) sh_tau = key;
  }
  __syncthreads();

  // ---- the top entries of the CTA
  if (a.top > 0) {
    for (;;) {
      const uint64_t tau = sh_tau;
      const float tau_x = tau ? key_value(tau) : -INFINITY;
      auto offer = [&](float f, int idx) {
        const uint64_t k = score_key(f, idx);
        if (k >= tau) {
          const int n = atomicAdd(&sh_n, 1);
          if (n < kTokList) sh_cand[n] = k;
        }
      };
      auto load_vector = [&](int i) { return *reinterpret_cast<const uint4*>(vec + static_cast<int64_t>(i) * 16); };
      auto offer_vector = [&](uint4 u, int i) {
        for (unsigned hits = TokVec<T>(u).reaching(tau_x); hits; hits &= hits - 1) {
          const int e = __ffs(hits) - 1;
          offer(TokVec<T>::pick(u, e), first + i * kN + e);
        }
      };
      const bool in = threadIdx.x < nv && pass.most(first) >= tau;
      const bool more = in && pass.more(tau);
      if (in && !more) {
        uint4 u[kTokUnroll];
        const int last = pass.last();
#pragma unroll
        for (int j = 0; j < kTokUnroll; ++j) u[j] = load_vector(min(pass.at + j * NT, last));
#pragma unroll
        for (int j = 0; j < kTokUnroll; ++j)
          if (pass.at + j * NT <= last) offer_vector(u[j], pass.at + j * NT);
      }
      if (single >= 0) offer(lone, single);
      // the warp reads all vectors of such threads, all lanes at work
      const unsigned who = __ballot_sync(0xffffffffu, more);
      const int each = (nv + NT - 1) / NT;
      for (int p = lane; p < __popc(who) * each; p += 32) {
        unsigned w = who;
        int i = p;
        for (; i >= each; i -= each) w &= w - 1;
        i = warp * 32 + __ffs(w) - 1 + i * NT;
        if (i < nv) offer_vector(load_vector(i), i);
      }
      __syncthreads();
      const int n = sh_n;
      block_rank<NT>(sh_cand, min(n, kTokList), sh_top);
      __syncthreads();
      if (n <= kTokList) break;
      if (threadIdx.x == 0) {
        sh_tau = sh_top[a.top - 1];
        sh_n = 0;
      }
      __syncthreads();
    }
  }
  z = t = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    z += sh_z[w];
    t += sh_t[w];
  }
  TokSums row_s{ref, z, t};
  if (ranks > 1) {
    if (threadIdx.x == 0) sh_sum = make_float4(ref, z, t, 0.f);
    cluster_sync();
    if (rank == 0) {
      // every warp joins the sums, lane by lane
      TokSums o{-3.402823466e38f, 0.f, 0.f};
      if (lane < ranks) {
        const float4 f = ld_cluster4(smem_addr(&sh_sum), lane);
        o = TokSums{f.x, f.y, f.z};
      }
      float to = o.ref;
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, off));
      to = __shfl_sync(0xffffffffu, to, 0);
      o.move(to);
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) {
        o.z += __shfl_xor_sync(0xffffffffu, o.z, off);
        o.t += __shfl_xor_sync(0xffffffffu, o.t, off);
      }
      row_s = TokSums{to, __shfl_sync(0xffffffffu, o.z, 0), __shfl_sync(0xffffffffu, o.t, 0)};
      if (a.top > 0) {
        // The largest of the CTAs' k-th best is a tau for the row; what is
        // below it need not be ranked.
        const int n = static_cast<int>(ranks) * a.top;
        uint64_t k = 0;
        if (threadIdx.x < n) {  // n <= 8 * 32 = NT
          const float2 k2 = ld_cluster2(smem_addr(&sh_top[threadIdx.x % a.top]), threadIdx.x / a.top);
          k = static_cast<uint64_t>(__float_as_uint(k2.y)) << 32 | __float_as_uint(k2.x);
          if (k == 0) k = threadIdx.x + 1;  // empty entries (a CTA with fewer than k entries) stay distinct
        }
        if (threadIdx.x == 0) {
          sh_tau = 0;
          sh_n = 0;
        }
        __syncthreads();
        if (threadIdx.x < n && threadIdx.x % a.top == a.top - 1)
          atomicMax(reinterpret_cast<unsigned long long*>(&sh_tau), static_cast<unsigned long long>(k));
        __syncthreads();
        if (threadIdx.x < n && k >= sh_tau) sh_cand[atomicAdd(&sh_n, 1)] = k;
        __syncthreads();
      }
    }
    cluster_sync();  // no CTA leaves (or ranks into sh_top) while its shared memory is read
    if (rank != 0) return;
    if (a.top > 0) {
      block_rank<NT>(sh_cand, sh_n, sh_top);
      __syncthreads();
    }
  }
  const uint64_t key = threadIdx.x < a.top ? sh_top[threadIdx.x] : 0;
  const bool bad = !(row_s.z > 0.f && row_s.z < INFINITY);
  const float lz = logf(row_s.z);
  if (threadIdx.x == 0) {
    float lp = 0.f;
    if (bad) {
      report(FDL_DEV_INDEX, row);
    } else if (target >= a.V) {
      report(FDL_DEV_INDEX, target);
      lp = NAN;
    } else if (target >= 0) {
      lp = target_x - row_s.ref - lz;
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

// The best 32 of two sorted lists, sorted: lane i holds one, and is given
// entry 31 - i of the other.
__device__ __forceinline__ uint64_t warp_merge(uint64_t key, uint64_t other_reversed) {
  key = max64(key, other_reversed);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) key = exchange(key, off, true);
  return key;
}

// Many rows of a small vocabulary: a warp takes a row, and nothing waits for
// another warp.  tau is the k-th largest lane maximum; the caught entries are
// sorted 32 at a time.
template <typename T>
__global__ void __launch_bounds__(kTokRowWarps * 32, 4) token_scores_warp_kernel(const __grid_constant__ TokScoreArgs a) {
  constexpr int kN = TokVec<T>::kN;
  __shared__ uint64_t sh_list[kTokRowWarps][kTokRowList];
  __shared__ int sh_n[kTokRowWarps];  // entries at or above tau
  await_stream();
  release_stream();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * kTokRowWarps + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  uint64_t* list = sh_list[threadIdx.x >> 5];
  const T* x = static_cast<const T*>(a.x) + static_cast<int64_t>(row) * a.rs;
  const int head = min(a.V, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
  const int nv = (a.V - head) / kN, rest = a.V - head - nv * kN;
  const char* vec = reinterpret_cast<const char*>(x + head);
  int single = -1;  // at most 7 entries in front of the vectors and 7 behind them
  if (lane < head) single = lane;
  if (lane >= 8 && lane - 8 < rest) single = a.V - rest + lane - 8;
  const int64_t target = a.targets[row];

  TokPass<T, 32> pass;
  pass.run(vec, nv, lane);
  TokSums s = pass.sums.natural();
  float lone = -INFINITY, target_x = 0.f;
  if (target >= 0 && target < a.V) target_x = static_cast<float>(x[target]);
  if (single >= 0) {
    lone = static_cast<float>(x[single]);
    if (lone > s.ref) s.move(lone);
    s.add(lone);
  }
  auto warp_max = [&](float m) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    return m;
  };
  float m = warp_max(fmaxf(pass.best, lone));
  if (fabsf(m) > kTokBig || m <= kTokLowest<T>) {  // as in token_scores_kernel
    auto each = [&](auto f) {
      for (int i = lane; i < nv; i += 32) {
        const TokVec<T> q(TokPass<T, 32>::load(vec + static_cast<int64_t>(i) * 16));
#pragma unroll
        for (int e = 0; e < kN; ++e) f(q.f[e]);
      }
      if (single >= 0) f(lone);
    };
    m = -INFINITY;
    each([&](float v) { m = fmaxf(m, v); });
    m = warp_max(m);
    s = TokSums{fmaxf(m, -3.402823466e38f), 0.f, 0.f};
    each([&](float v) { s.add(v); });
  } else if (m > s.ref) {
    s.move(m);
  }
  float z = s.z, t = s.t;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    z += __shfl_xor_sync(0xffffffffu, z, off);
    t += __shfl_xor_sync(0xffffffffu, t, off);
  }
  const bool bad = !(z > 0.f && z < INFINITY);
  const float lz = logf(z);
  if (lane == 0) {
    float lp = 0.f;
    if (bad) {
      report(FDL_DEV_INDEX, row);
    } else if (target >= a.V) {
      report(FDL_DEV_INDEX, target);
      lp = NAN;
    } else if (target >= 0) {
      lp = target_x - s.ref - lz;
    }
    a.logprob[row] = bad ? NAN : lp;
    a.entropy[row] = bad ? NAN : lz - t / z;
  }
  if (a.top == 0) return;

  uint64_t tau = 0;  // below 32 vectors all entries fit the list
  if (nv >= 32) {
    const uint32_t order = pass.least_order(), index = pass.least_index(head);
    uint32_t o = order;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
      for (int off = size / 2; off > 0; off >>= 1) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, o, off);
        o = ((lane & off) == 0) == ((lane & size & 31) == 0) ? max(o, other) : min(o, other);
      }
    const uint32_t kth = __shfl_sync(0xffffffffu, o, a.top - 1);
    // of the lanes whose maximum has that value, as many as are needed, the
    // lower indices first
    uint32_t mine = order == kth ? index : 0xffffffffu, low = 0;
    for (int need = a.top - __popc(__ballot_sync(0xffffffffu, order > kth)); need > 0; --need) {
      low = __reduce_min_sync(0xffffffffu, mine);
      if (mine == low) mine = 0xffffffffu;
    }
    tau = order_key(kth, low);
  }
  uint64_t key = 0;
  int* count = sh_n + (threadIdx.x >> 5);
  for (;;) {
    if (lane == 0) *count = 0;
    __syncwarp();
    const float tau_x = tau ? key_value(tau) : -INFINITY;
    auto offer = [&](float f, int idx) {
      const uint64_t k = score_key(f, idx);
      if (k >= tau) {
        const int to = atomicAdd(count, 1);
        if (to < kTokRowList) list[to] = k;
      }
    };
    // Which entries of four vectors at a time reach tau's value, as bits, and
    // then one by one: the lanes' few entries are spread over all places.
    const bool in = lane < nv && pass.most(head) >= tau, all = __any_sync(0xffffffffu, in && pass.more(tau));
    for (int i0 = all ? lane : pass.at; in && i0 < (all ? nv : pass.last() + 1); i0 += 4 * 32) {
      uint4 u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = TokPass<T, 32>::load(vec + static_cast<int64_t>(min(i0 + j * 32, nv - 1)) * 16);
      unsigned hits = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned some = TokVec<T>(u[j]).reaching(tau_x);
        if (i0 + j * 32 < nv) hits |= some << (j * kN);
      }
      for (; hits; hits &= hits - 1) {
        const int bit = __ffs(hits) - 1, idx = head + (i0 + bit / kN * 32) * kN + bit % kN;
        offer(static_cast<float>(x[idx]), idx);
      }
    }
    if (single >= 0) offer(lone, single);
    __syncwarp();
    const int n = *count;
    const int have = min(n, kTokRowList);
    key = warp_sort(lane < have ? list[lane] : 0);
    for (int c = 32; c < have; c += 32) {
      const uint64_t more_keys = warp_sort(c + lane < have ? list[c + lane] : 0);
      key = warp_merge(key, __shfl_sync(0xffffffffu, more_keys, 31 - lane));
    }
    __syncwarp();
    if (n <= kTokRowList) break;
    tau = __shfl_sync(0xffffffffu, key, a.top - 1);
  }
  if (lane < a.top) {
    const int64_t to = static_cast<int64_t>(row) * a.top + lane;
    a.top_lp[to] = bad ? NAN : key_value(key) - s.ref - lz;
    a.top_tok[to] = bad ? -1 : static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key));
  }
}

}  // namespace fdl
