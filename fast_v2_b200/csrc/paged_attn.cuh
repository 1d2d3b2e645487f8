// Attention of one new token per sequence over a paged KV cache:
//   o[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q[b,h].k_j - m),
//   m = max_j scale * q[b,h].k_j,  j < lens[b],
// with k_j, v_j row j % page of page table[b, j / page], head h / (hq / hkv).
// A sequence without a visible key gives zeros.  A page outside the pool
// hides its keys and is reported.
//
// Bound by HBM: every K and V row is read once for all query heads of its KV
// head (2 * 2 * D bytes for 4 * D * G operations: at G = 7, 7 operations a
// byte).  What has to be won is bytes in flight and an even share of them for
// every SM, whatever the lengths.
//
// Unit = (sequence, KV head, group of 8 * NH query heads); its keys come in
// tiles of 16 per warp.  Two ways to share the units out (chosen by
// paged_plan on sizes alone):
//   line     The tiles of all units form one line, and each CTA of a grid that
//            fits the GPU takes an equal piece of it (found with one scan of
//            the lengths, on the device: lengths may change under a captured
//            graph).  A unit that lies in one piece is finished by its CTA;
//            the pieces of the others go to the workspace -- at most two a
//            CTA, so it does not grow with the batch -- and a second kernel
//            joins them in order.
//   cluster  A thread-block cluster takes a unit, its CTAs equal parts of the
//            unit's tiles, joined through distributed shared memory -- or one
//            CTA of 1 to 4 warps where units are many: one launch, no
//            workspace.  For short caches, where the scan and the second
//            kernel cost more than an uneven share.
//
// Within a CTA every warp takes 16 keys of a tile and runs on its own: its
// rows arrive by cp.async in a ring of its own, no barrier between warps
// until a unit ends.  Scores are formed transposed, S^T = K Q^T (m16n8k16:
// 16 keys x 8 heads), and so is the output, O^T = V^T P^T: 8 query heads fill
// the short side of the instruction, where Q on the long side would leave
// half of it empty.  The matrix instructions are the warp-level ones: at 7
// operations a byte they are far from busy, and an M = 128 instruction of the
// tcgen05 kind would be 15/16 padding.
#pragma once
#include <type_traits>

#include "common.cuh"
#include "device_util.cuh"

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
  int B, hq, hkv, num_pages;
  int G, HG, NU;            // query heads a KV head, groups of them, units a sequence
  int cap;                  // keys the table can name
  FastDiv page;
  float scale_log2;
  // line
  float* part_o;            // [2 grid, 8 NH, D] sums relative to the piece's reference
  float2* part_ml;          // [2 grid, 8 NH] (reference, sum of p)
  int4* desc;               // [grid] (sequence, unit of it) whose first piece ends the CTA's part of the line, or -1;
                            // state of the CTA's first piece: 0 starts a unit, 1 middle of one, 2 end of one
};

constexpr int kPagedWarpKeys = 16;
constexpr int kPagedLineWarps = 4;
constexpr int kPagedLineTile = kPagedLineWarps * kPagedWarpKeys;
// A score may pass the running reference by 2^8 before the sums are scaled
// down to a new one.
constexpr float kPagedSlack = 8.f;
// fp16 has no numbers below 2^-24.  Its weights are lifted by 2^7 (p <= 2^15),
// which cancels in the quotient: a key behind a strong one loses at most 2^-32
// of the strong one's weight, 2^-24 for the 256 keys that a warp takes in the
// forms for short caches.  On the line it may take 2^15 and more.  There the
// reference also moves down, to the largest score of a tile that lies 2^12
// below it, and the weak keys keep their share; down to 2^40 below the largest
// score at most, so that the sums stay inside fp32.
constexpr float kPagedLift = 7.f;
constexpr float kPagedFar = 12.f;
constexpr float kPagedDepth = 40.f;

// Stages of a warp's ring.  On the line two CTAs a SM (D = 128) with three
// stages keep HBM busy (30.9 us for 65k keys against 31.4 us with three CTAs
// of two stages); CTAs with a unit of their own wait on their own arithmetic,
// and more of them with two stages win (200 rows of 1 to 1000 keys 22.8
// against 26.4 us).
template <int D, int NW, bool LINE>
struct PagedCfg {
  static constexpr int kStages = !LINE && (NW <= 2 || (NW == 4 && D == 128)) ? 2 : 3;
  static constexpr int kStage = 2 * kPagedWarpKeys * D * 2;  // bytes of a warp's tile: K rows, V rows
  static constexpr int kSmem = NW * kStages * kStage;
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ int paged_len(const PagedAttnArgs& a, int b) { return min(max(a.lens[b], 0), a.cap); }

// n / f.d for n < 2^31 (FastDiv::div with the 32-bit halves of the product
// spelled out: two multiplies).
__device__ __forceinline__ int paged_div(const FastDiv& f, int n) {
  if (f.d == 1) return n;
  const uint64_t lo = static_cast<uint64_t>(static_cast<uint32_t>(f.m)) * static_cast<uint32_t>(n);
  const uint64_t hi = (f.m >> 32) * static_cast<uint32_t>(n) + (lo >> 32);
  return static_cast<int>(hi >> 32);
}

// A place on the line of tiles of NW * 16 keys.
template <int TILE>
struct PagedPos {
  int b, kh, hg;  // sequence, KV head, group of its query heads
  int t, nt;      // tile of the unit, tiles of a unit of b
  int len;
  __device__ __forceinline__ void unit(const PagedAttnArgs& a, int n) {
    kh = n / a.HG;
    hg = n - kh * a.HG;
  }
  __device__ __forceinline__ void next(const PagedAttnArgs& a) {
    if (++t < nt) return;
    t = 0;
    if (++hg < a.HG) return;
    hg = 0;
    if (++kh < a.hkv) return;
    kh = 0;
    for (++b; b < a.B; ++b) {
      len = paged_len(a, b);
      nt = (len + TILE - 1) / TILE;
      if (nt > 0) return;
    }
  }
};

template <typename T, int D, int NH, int NW, bool LINE>
__global__ void __launch_bounds__(NW * 32) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
  using Cfg = PagedCfg<D, NW, LINE>;
  constexpr int kThreads = NW * 32, kTile = NW * kPagedWarpKeys;
  constexpr bool kNarrow = std::is_same<T, __half>::value, kFollow = kNarrow && LINE;
  constexpr int kStages = Cfg::kStages, kChunks = D / 8, kRowB = D * 2, H = 8 * NH;
  constexpr int kLoads = kPagedWarpKeys * kChunks / 32;  // 16-byte pieces of K (and of V) a lane and tile
  extern __shared__ __align__(128) char smem[];
  __shared__ int s_mask[NW][kStages];
  __shared__ float2 s_ml[NW][H];
  __shared__ float2 s_cta[H];  // cluster: (reference, sum) of this CTA
  __shared__ int s_pos[4];
  __shared__ long long s_scan[NW];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c4 = lane & 3;
  const uint32_t ring = smem_addr(smem) + warp * kStages * Cfg::kStage;
  T* const out = static_cast<T*>(a.out);

  // ---- this CTA's piece of the line
  PagedPos<kTile> p{};
  int left;  // tiles
  await_stream();
  release_stream();
  if constexpr (LINE) {
    const int per = (a.B + kThreads - 1) / kThreads;
    const int b0 = threadIdx.x * per, b1 = min(a.B, b0 + per);
    long long sum = 0;
    int one = 0;  // the length, where the thread has one sequence
    for (int b = b0; b < b1; ++b) {
      const int raw = a.lens[b];
      if (blockIdx.x == 0 && (raw < 0 || raw > a.cap)) report(FDL_DEV_LENGTH, b);
      one = min(max(raw, 0), a.cap);
      sum += (one + kTile - 1) / kTile;
    }
    long long incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += o;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < warp) incl += s_scan[w];
      total += s_scan[w];
    }
    total *= a.NU;
    // Equal pieces, the first ones a tile longer.  No CTA before the last
    // busy one is without tiles, so pieces of a unit lie on consecutive CTAs.
    long long first = 0;
    {
      long long q, r;
      if (total <= INT32_MAX) {  // 32-bit division: a tenth of the 64-bit one's instructions
        q = static_cast<uint32_t>(total) / gridDim.x;
        r = static_cast<uint32_t>(total) % gridDim.x;
      } else {
        q = total / gridDim.x;
        r = total % gridDim.x;
      }
      first = q * blockIdx.x + min(static_cast<long long>(blockIdx.x), r);
      left = static_cast<int>(q) + (blockIdx.x < r);
    }
    long long at = (incl - sum) * a.NU;
    if (left > 0 && first >= at && first < incl * a.NU) {
      for (int b = b0; b < b1; ++b) {
        const int len = per == 1 ? one : paged_len(a, b), nt = (len + kTile - 1) / kTile;
        const long long mine = static_cast<long long>(nt) * a.NU;
        if (first < at + mine) {
          const int local = static_cast<int>(first - at);
          s_pos[0] = b;
          s_pos[1] = local / nt;
          s_pos[2] = local % nt;
          s_pos[3] = len;
          break;
        }
        at += mine;
      }
    }
    // Sequences without keys: shared out over the grid.
    for (int b = blockIdx.x; b < a.B; b += gridDim.x)
      if (paged_len(a, b) == 0)
        for (int i = threadIdx.x; i < a.hq * kChunks; i += kThreads)
          *reinterpret_cast<uint4*>(out + b * a.o_sb + (i / kChunks) * a.o_sh + (i % kChunks) * 8) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (left == 0) {
      if (threadIdx.x == 0) a.desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
      return;
    }
    p.b = s_pos[0];
    p.unit(a, s_pos[1]);
    p.t = s_pos[2];
    p.len = s_pos[3];
  } else {
    const uint32_t ranks = cluster_size(), rank = cluster_rank(), unit = blockIdx.x / ranks;
    p.b = unit / a.NU;
    p.unit(a, unit % a.NU);
    const int raw = a.lens[p.b];
    if (rank == 0 && unit % a.NU == 0 && threadIdx.x == 0 && (raw < 0 || raw > a.cap)) report(FDL_DEV_LENGTH, p.b);
    p.len = min(max(raw, 0), a.cap);
    const int nt = (p.len + kTile - 1) / kTile;
    if (nt == 0) {  // no CTA of the cluster goes on
      const int h0 = p.kh * a.G + p.hg * H, hn = min(H, a.G - p.hg * H);
      if (rank == 0)
        for (int i = threadIdx.x; i < hn * kChunks; i += kThreads)
          *reinterpret_cast<uint4*>(out + p.b * a.o_sb + (h0 + i / kChunks) * a.o_sh + (i % kChunks) * 8) =
              make_uint4(0, 0, 0, 0);
      return;
    }
    p.t = nt * rank / ranks;
    left = nt * (rank + 1) / ranks - p.t;
  }
  p.nt = (p.len + kTile - 1) / kTile;
  // line: 0 this CTA's first piece starts its unit, 1 lies inside, 2 ends it
  int state = p.t == 0 ? 0 : (p.t + left >= p.nt ? 2 : 1);
  const int first_state = state;

  // ---- loads: the warp's 16 rows of tile `w`, with the pages looked up one tile ahead
  constexpr int kRows = 32 / kChunks;  // rows a warp-wide copy covers (D = 64: 4, 128: 2, 256: 1)
  PagedPos<kTile> w = p;  // next tile to load
  int w_left = left;
  const bool whole = a.page.d % kPagedWarpKeys == 0;  // the 16 keys lie in one page
  const int64_t lane_src = static_cast<int64_t>(lane / kChunks) * a.ss + (lane % kChunks) * 16;
  const int64_t step_src = a.ss * kRows;
  const int64_t v_minus_k = reinterpret_cast<int64_t>(a.v) - reinterpret_cast<int64_t>(a.k);
  // Row r holds its 16-byte piece ch at ch ^ (r & 7): eight rows of one piece
  // lie in different banks.  Offsets of this lane, by what they depend on.
  uint32_t to_off[8 / kRows], k_off[4], v_off[4];
#pragma unroll
  for (int i = 0; i < 8 / kRows; ++i) {
    const int r = i * kRows + lane / kChunks;
    to_off[i] = r * kRowB + (((lane % kChunks) ^ (r & 7)) * 16);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rk = lane & 15, rv = (lane & 7) | ((lane >> 4) << 3);
    k_off[i] = rk * kRowB + (((i * 2 + (lane >> 4)) ^ (rk & 7)) * 16);
    v_off[i] = kPagedWarpKeys * kRowB + rv * kRowB + (((i * 2 + ((lane >> 3) & 1)) ^ (rv & 7)) * 16);
  }
  int page = 0, in_page = 0;
  auto look_up = [&]() {  // the page of this lane's key of tile w
    if (w_left > 0) {
      const int key = w.t * kTile + warp * kPagedWarpKeys + (whole ? 0 : lane & 15);
      if (key < w.len) {
        const int i = paged_div(a.page, key);
        in_page = key - i * static_cast<int>(a.page.d);
        page = a.table[w.b * a.table_sb + i];
      }
    }
  };
  int fill = 0;
  auto load = [&]() {
    if (w_left > 0) {
      const int n = w.len - w.t * kTile - warp * kPagedWarpKeys;  // keys from the warp's first on
      if (n > 0) {
        const bool bad = static_cast<unsigned>(page) >= static_cast<unsigned>(a.num_pages);
        const int64_t off = static_cast<int64_t>(page) * a.sp + static_cast<int64_t>(in_page) * a.ss +
                            static_cast<int64_t>(w.kh) * a.sh;
        const uint32_t dst = ring + fill * Cfg::kStage;
        if (whole && n >= kPagedWarpKeys && !bad) {
          if (lane == 0) s_mask[warp][fill] = 0xffff;
          const char* src = a.k + off + lane_src;
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            const uint32_t to = dst + to_off[i % (8 / kRows)] + (i / (8 / kRows)) * 8 * kRowB;
            cp_async16(to, src);
            cp_async16(to + kPagedWarpKeys * kRowB, src + v_minus_k);
            src += step_src;
          }
        } else {
          // the last keys of a sequence, bad pages, pages that end inside
          // the 16 keys: row by row, zeros in place of what is not there
          const bool in = (lane & 15) < n;
          if (in && bad && lane < 16) report(FDL_DEV_INDEX, page);
          const unsigned mask = __ballot_sync(0xffffffffu, in && !bad) & 0xffffu;
          if (lane == 0) s_mask[warp][fill] = mask;
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            const int r = i * kRows + lane / kChunks;
            const int64_t row = whole ? off + r * a.ss : __shfl_sync(0xffffffffu, off, r);
            const bool get = (mask >> r) & 1;
            const int64_t at = get ? row + (lane % kChunks) * 16 : 0;
            const uint32_t to = dst + to_off[i % (8 / kRows)] + (i / (8 / kRows)) * 8 * kRowB;
            cp_async16(to, a.k + at, get ? 16 : 0);
            cp_async16(to + kPagedWarpKeys * kRowB, a.v + at, get ? 16 : 0);
          }
        }
      }
      if (--w_left > 0) w.next(a);
    }
    cp_commit();
    fill = fill + 1 == kStages ? 0 : fill + 1;
    look_up();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load();

  uint32_t qf[NH][D / 16][2];
  float o[NH][D / 16][4];
  float m[NH][2], l[NH][2];
  float deep[NH][2];  // kFollow: how far down the reference may move
  auto load_q = [&]() {  // the query heads of p's unit
    const int h0 = p.kh * a.G + p.hg * H, hn = min(H, a.G - p.hg * H);
    const T* q = static_cast<const T*>(a.q) + p.b * a.q_sb + h0 * a.q_sh;
#pragma unroll
    for (int x = 0; x < NH; ++x) {
      const int hh = x * 8 + g;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          qf[x][kk][e] = hh < hn ? *reinterpret_cast<const uint32_t*>(q + hh * a.q_sh + kk * 16 + e * 8 + c4 * 2) : 0u;
    }
  };
  auto clear = [&]() {
#pragma unroll
    for (int x = 0; x < NH; ++x) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[x][kk][e] = 0.f;
      m[x][0] = m[x][1] = deep[x][0] = deep[x][1] = -INFINITY;
      l[x][0] = l[x][1] = 0.f;
    }
  };
  // The warp's state goes to its part of `to` ([H, D] floats; the 8-float
  // pieces of a head are exchanged so that the four heads that a warp writes
  // at a time lie in different banks).
  auto put_state = [&](float* to) {
#pragma unroll
    for (int x = 0; x < NH; ++x) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[x][e] += __shfl_xor_sync(0xffffffffu, l[x][e], off);
      if (g == 0) {
        s_ml[warp][x * 8 + c4 * 2] = make_float2(m[x][0], l[x][0]);
        s_ml[warp][x * 8 + c4 * 2 + 1] = make_float2(m[x][1], l[x][1]);
      }
      float* mo = to + (x * 8 + c4 * 2) * D;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const int d0 = ((kk * 2) ^ c4) * 8 + g, d1 = ((kk * 2 + 1) ^ c4) * 8 + g;
        mo[d0] = o[x][kk][0];
        mo[D + d0] = o[x][kk][1];
        mo[d1] = o[x][kk][2];
        mo[D + d1] = o[x][kk][3];
      }
    }
  };
  // Eight elements of head hh, summed over the warps' states (`stride` floats
  // apart) relative to the largest reference M; L is the sum of p.
  auto take_state = [&](const float* from, int stride, int hh, int ch, float (&acc)[8], float& M, float& L) {
    M = -INFINITY;
    L = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) M = fmaxf(M, s_ml[x][hh].x);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float2 ml = s_ml[x][hh];
      const float f = ex2(ml.x - ref);
      L = fmaf(ml.y, f, L);
      const float4* src = reinterpret_cast<const float4*>(from + x * stride + hh * D + ((ch ^ ((hh >> 1) & 3)) * 8));
      const float4 u0 = src[0], u1 = src[1];
      acc[0] = fmaf(u0.x, f, acc[0]);
      acc[1] = fmaf(u0.y, f, acc[1]);
      acc[2] = fmaf(u0.z, f, acc[2]);
      acc[3] = fmaf(u0.w, f, acc[3]);
      acc[4] = fmaf(u1.x, f, acc[4]);
      acc[5] = fmaf(u1.y, f, acc[5]);
      acc[6] = fmaf(u1.z, f, acc[6]);
      acc[7] = fmaf(u1.w, f, acc[7]);
    }
  };
  auto finish = [&](int b, int h, int ch, float (&acc)[8], float L) {
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= inv;
    *reinterpret_cast<uint4*>(out + b * a.o_sb + h * a.o_sh + ch * 8) = pack8<T>(acc);
  };
  load_q();
  clear();
  int use = 0;
  while (left > 0) {
    __syncwarp();  // the slot that is loaded next has been read
    load();
    cp_wait<kStages - 1>();
    __syncwarp();
    if (p.t * kTile + warp * kPagedWarpKeys < p.len) {
      const uint32_t slot = ring + use * Cfg::kStage;
      const unsigned mask = s_mask[warp][use];
      float s[NH][2][4];
#pragma unroll
      for (int x = 0; x < NH; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[x][0][e] = s[x][1][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t f[4];
        ldsm4(f, slot + k_off[kk & 3] + (kk >> 2) * 128);
#pragma unroll
        for (int x = 0; x < NH; ++x) mma16816<T>(s[x][kk & 1], f, qf[x][kk][0], qf[x][kk][1]);
      }
      uint32_t pf[NH][2], pl[NH][2];
      float v[NH][4];  // keys g, g, g + 8, g + 8 of heads 2 c4, 2 c4 + 1
      bool above = false, near = true;
#pragma unroll
      for (int x = 0; x < NH; ++x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[x][e] = (s[x][0][e] + s[x][1][e]) * a.scale_log2;
        if (mask != 0xffffu) {
          if (!((mask >> g) & 1)) v[x][0] = v[x][1] = -INFINITY;
          if (!((mask >> (g + 8)) & 1)) v[x][2] = v[x][3] = -INFINITY;
        }
        const float t0 = fmaxf(v[x][0], v[x][2]), t1 = fmaxf(v[x][1], v[x][3]);
        above = above || t0 > m[x][0] + kPagedSlack || t1 > m[x][1] + kPagedSlack;
        near = near && t0 >= m[x][0] - kPagedFar && t1 >= m[x][1] - kPagedFar;
      }
      bool move = __any_sync(0xffffffffu, above);
      if constexpr (kFollow) {  // a lane's heads have to be near in one of the eight lanes that share them
        unsigned all = __ballot_sync(0xffffffffu, near);
        all |= all >> 16;
        all |= all >> 8;
        move = move || ((all | all >> 4) & 0xfu) != 0xfu;
      }
      if (move) {
#pragma unroll
        for (int x = 0; x < NH; ++x) {
          float t0 = fmaxf(v[x][0], v[x][2]), t1 = fmaxf(v[x][1], v[x][3]);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, off));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, off));
          }
          float n0 = fmaxf(m[x][0], t0), n1 = fmaxf(m[x][1], t1);
          if constexpr (kFollow) {
            deep[x][0] = fmaxf(deep[x][0], n0 - kPagedDepth);
            deep[x][1] = fmaxf(deep[x][1], n1 - kPagedDepth);
            if (t0 < m[x][0] - kPagedFar && t0 != -INFINITY) n0 = fminf(n0, fmaxf(t0, deep[x][0]));
            if (t1 < m[x][1] - kPagedFar && t1 != -INFINITY) n1 = fminf(n1, fmaxf(t1, deep[x][1]));
          }
          const float f0 = n0 == -INFINITY ? 1.f : ex2(m[x][0] - n0), f1 = n1 == -INFINITY ? 1.f : ex2(m[x][1] - n1);
          m[x][0] = n0;
          m[x][1] = n1;
          l[x][0] *= f0;
          l[x][1] *= f1;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            o[x][kk][0] *= f0;
            o[x][kk][1] *= f1;
            o[x][kk][2] *= f0;
            o[x][kk][3] *= f1;
          }
        }
      }
#pragma unroll
      for (int x = 0; x < NH; ++x) {
        constexpr float lift = kNarrow ? kPagedLift : 0.f;
        const float r0 = (m[x][0] == -INFINITY ? 0.f : m[x][0]) - lift, r1 = (m[x][1] == -INFINITY ? 0.f : m[x][1]) - lift;
        // A weight goes into the product as two numbers of V's type, its
        // rounded value and what that leaves: 2^-16 (bf16) or 2^-22 (fp16) of
        // it is lost.  One number would lose 2^-8 or 2^-11, as much as the
        // output's own rounding, and take 0.1 to 0.9 us less (200 rows of 1 to
        // 1000 keys 21.9 against 22.8 us, one row of 65k keys 30.6 against 30.7).
        const float p0 = ex2(v[x][0] - r0), p1 = ex2(v[x][1] - r1), p2 = ex2(v[x][2] - r0), p3 = ex2(v[x][3] - r1);
        l[x][0] += p0 + p2;
        l[x][1] += p1 + p3;
        const uint32_t h0 = Pack2<T>::from(p0, p1), h1 = Pack2<T>::from(p2, p3);
        const float2 q0 = Pack2<T>::to(h0), q1 = Pack2<T>::to(h1);
        pf[x][0] = movmatrix_t(h0);
        pf[x][1] = movmatrix_t(h1);
        pl[x][0] = movmatrix_t(Pack2<T>::from(p0 - q0.x, p1 - q0.y));
        pl[x][1] = movmatrix_t(Pack2<T>::from(p2 - q1.x, p3 - q1.y));
      }
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t f[4];
        ldsm4_t(f, slot + v_off[kk & 3] + (kk >> 2) * 128);
#pragma unroll
        for (int x = 0; x < NH; ++x) {
          mma16816<T>(o[x][kk], f, pf[x][0], pf[x][1]);
          mma16816<T>(o[x][kk], f, pl[x][0], pl[x][1]);
        }
      }
    }
    --left;
    const PagedPos<kTile> was = p;
    if (left > 0) p.next(a);
    if constexpr (LINE) {
      const bool ends = was.t + 1 == was.nt;
      if (ends || left == 0) {
        // ---- finish the unit, or leave the piece in the workspace.  The
        // slot that was read last is the warp's room: nothing is loaded into
        // it before the next tile.
        if (left > 0) load_q();  // on its way while the warps are joined
        const float* room = reinterpret_cast<const float*>(smem + use * Cfg::kStage);
        put_state(const_cast<float*>(room) + warp * (kStages * Cfg::kStage / 4));
        __syncthreads();
        const bool all = state == 0 && ends;
        const int piece = blockIdx.x * 2 + (state == 0 ? 1 : 0);
        const int h0 = was.kh * a.G + was.hg * H, hn = min(H, a.G - was.hg * H);
        for (int i = threadIdx.x; i < hn * kChunks; i += kThreads) {
          const int hh = i / kChunks, ch = i % kChunks;
          float acc[8], M, L;
          take_state(room, kStages * Cfg::kStage / 4, hh, ch, acc, M, L);
          if (all) {
            finish(was.b, h0 + hh, ch, acc, L);
          } else {
            float4* dst = reinterpret_cast<float4*>(a.part_o + (static_cast<int64_t>(piece) * H + hh) * D + ch * 8);
            dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
            dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
            if (ch == 0) a.part_ml[piece * H + hh] = make_float2(M, L);
          }
        }
        if (left == 0 && threadIdx.x == 0)
          a.desc[blockIdx.x] = make_int4(state == 0 && !ends ? was.b : -1, was.kh * a.HG + was.hg, first_state, 0);
        __syncthreads();  // the room and s_ml are free again
        clear();
        state = 0;
      }
    }
    use = use + 1 == kStages ? 0 : use + 1;
  }
  cp_wait<0>();
  if constexpr (!LINE) {
    __syncthreads();  // the whole ring is room
    float* room = reinterpret_cast<float*>(smem);
    put_state(room + warp * H * D);
    __syncthreads();
    const uint32_t ranks = cluster_size();
    const int h0 = p.kh * a.G + p.hg * H, hn = min(H, a.G - p.hg * H);
    if (ranks == 1) {
      for (int i = threadIdx.x; i < hn * kChunks; i += kThreads) {
        float acc[8], M, L;
        take_state(room, H * D, i / kChunks, i % kChunks, acc, M, L);
        finish(p.b, h0 + i / kChunks, i % kChunks, acc, L);
      }
      return;
    }
    // This CTA's sums, in the room of warp 0 (a thread overwrites only what it
    // alone has read), then all CTAs' for a share of the outputs each.
    for (int i = threadIdx.x; i < H * kChunks; i += kThreads) {
      const int hh = i / kChunks, ch = i % kChunks;
      float acc[8], M, L;
      take_state(room, H * D, hh, ch, acc, M, L);
      float4* dst = reinterpret_cast<float4*>(room + hh * D + ((ch ^ ((hh >> 1) & 3)) * 8));
      dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (ch == 0) s_cta[hh] = make_float2(M, L);
    }
    cluster_sync();
    for (int i = cluster_rank() * kThreads + threadIdx.x; i < hn * kChunks; i += ranks * kThreads) {
      const int hh = i / kChunks, ch = i % kChunks;
      float acc[8], M = -INFINITY, L = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.f;
      for (uint32_t r = 0; r < ranks; ++r) M = fmaxf(M, ld_cluster2(smem_addr(&s_cta[hh]), r).x);
      const float ref = M == -INFINITY ? 0.f : M;
      const uint32_t src = smem_addr(room + hh * D + ((ch ^ ((hh >> 1) & 3)) * 8));
      for (uint32_t r = 0; r < ranks; ++r) {
        const float2 ml = ld_cluster2(smem_addr(&s_cta[hh]), r);
        const float4 u0 = ld_cluster4(src, r), u1 = ld_cluster4(src + 16, r);
        const float f = ex2(ml.x - ref);
        L = fmaf(ml.y, f, L);
        acc[0] = fmaf(u0.x, f, acc[0]);
        acc[1] = fmaf(u0.y, f, acc[1]);
        acc[2] = fmaf(u0.z, f, acc[2]);
        acc[3] = fmaf(u0.w, f, acc[3]);
        acc[4] = fmaf(u1.x, f, acc[4]);
        acc[5] = fmaf(u1.y, f, acc[5]);
        acc[6] = fmaf(u1.z, f, acc[6]);
        acc[7] = fmaf(u1.w, f, acc[7]);
      }
      finish(p.b, h0 + hh, ch, acc, L);
    }
    cluster_sync();  // no CTA leaves while its shared memory is read
  }
}

// Joins the pieces of the units that lie on more than one CTA.  CTA (i, h)
// takes query head h of a unit that CTA c of the line leaves open -- c = i, or
// with few units the i-th such CTA: its pieces are the last one of CTA c and
// the first ones of the CTAs behind c, up to the one that ends the unit.  The
// warps take pieces in turn and are joined in order.
template <typename T, int D, int NH, bool FEW>
__global__ void __launch_bounds__(FEW ? 512 : 128) paged_join_kernel(const __grid_constant__ PagedAttnArgs a, int grid) {
  constexpr int NW = FEW ? 16 : 4, H = 8 * NH, E = D / 32;
  __shared__ float s_o[NW][D];
  __shared__ float2 s_ml[NW];
  await_stream();
  release_stream();
  const int hh = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int c, last = -1;
  int4 d;
  if constexpr (FEW) {
    // the i-th CTA that leaves a unit open, and the next one that ends one:
    // a warp reads all descriptors, eight a lane at a time
    c = -1;
    d = make_int4(-1, 0, 0, 0);
    int want = blockIdx.x;  // open units to pass
    for (int i0 = 0; i0 < grid && last < 0; i0 += 256) {
      int4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * 32 + lane;
        v[u] = i < grid ? a.desc[i] : make_int4(-1, 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        unsigned end = __ballot_sync(0xffffffffu, v[u].z == 2), open = __ballot_sync(0xffffffffu, v[u].x >= 0);
        if (last >= 0) continue;
        if (c < 0) {
          if (want >= __popc(open)) {
            want -= __popc(open);
            continue;
          }
          for (; want > 0; --want) open &= open - 1;
          const int at = __ffs(open) - 1;
          c = i0 + u * 32 + at;
          d.x = __shfl_sync(0xffffffffu, v[u].x, at);
          d.y = __shfl_sync(0xffffffffu, v[u].y, at);
          end &= at == 31 ? 0u : 0xffffffffu << (at + 1);
        }
        if (end) last = i0 + u * 32 + __ffs(end) - 1;
      }
    }
  } else {
    c = blockIdx.x;
    d = a.desc[c];
    if (d.x < 0) return;
    for (int i0 = c + 1; i0 < grid && last < 0; i0 += 32) {
      const unsigned end = __ballot_sync(0xffffffffu, i0 + lane < grid && a.desc[i0 + lane].z == 2);
      if (end) last = i0 + __ffs(end) - 1;
    }
  }
  if (last < 0) return;
  const int g0 = (d.y % a.HG) * H;
  if (hh >= min(H, a.G - g0)) return;
  // Each warp keeps a reference of its own, four pieces at a time.
  float acc[E], L = 0.f, M = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int i0 = c + warp; i0 <= last; i0 += 4 * NW) {
    float2 ml[4];
    float x[4][E];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * NW;
      ml[u] = make_float2(-INFINITY, 0.f);
      if (i <= last) {
        const int slot = (i * 2 + (i == c)) * H + hh;
        ml[u] = a.part_ml[slot];
        const float* src = a.part_o + static_cast<int64_t>(slot) * D + lane;
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = src[e * 32];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = 0.f;
      }
    }
    const float n = fmaxf(M, fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)));
    const float ref = n == -INFINITY ? 0.f : n;
    const float f = ex2(M - ref);
    M = n;
    L *= f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float g = ex2(ml[u].x - ref);
      L = fmaf(ml[u].y, g, L);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(x[u][e], g, acc[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][e * 32 + lane] = acc[e];
  if (lane == 0) s_ml[warp] = make_float2(M, L);
  __syncthreads();
  float top = -INFINITY, l = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) top = fmaxf(top, s_ml[w].x);
  const float ref = top == -INFINITY ? 0.f : top;
  float f[NW];
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    f[w] = ex2(s_ml[w].x - ref);
    l = fmaf(s_ml[w].y, f[w], l);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = static_cast<T*>(a.out) + d.x * a.o_sb + ((d.y / a.HG) * a.G + g0 + hh) * a.o_sh;
  for (int i = threadIdx.x; i < D / 2; i += NW * 32) {
    float x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      x0 = fmaf(s_o[w][2 * i], f[w], x0);
      x1 = fmaf(s_o[w][2 * i + 1], f[w], x1);
    }
    reinterpret_cast<uint32_t*>(out)[i] = Pack2<T>::from(x0 * inv, x1 * inv);
  }
}

}  // namespace fdl
