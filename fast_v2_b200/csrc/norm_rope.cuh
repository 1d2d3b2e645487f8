// Split of the fused q/k/v projection rows, RMS norm of each query and key
// head, rotary positions and the store of K and V into their pages, in one
// pass.  For row r (position p = pos[r]), head x of D elements:
//   x'  = x * rsqrt(mean(x^2) + eps) * w          (where a weight is given)
//   (a, b) -> f * (a cos t_j - b sin t_j,  b cos t_j + a sin t_j)
// over the first `rot` elements, pairs (a, b) = (x'_j, x'_{j + rot/2}) in the
// half layout and (x'_{2j}, x'_{2j+1}) in the interleaved one, t_j = p *
// inv_freq[j]; the other elements and the V heads pass unturned.  All
// arithmetic is fp32 and each output is rounded once.
//
// The angle of a far position has more bits than fp32 holds (p = 10^6 leaves
// 2^-4 of a radian), so p * inv_freq is formed and reduced to a fraction of a
// turn in fp64 -- three operations per pair and row, shared by all heads.
//
// Bound by HBM: each element is read once and written once.  A CTA takes a few
// rows (one where rows are few); a head takes GS lanes (D / 16 rounded up to a
// power of two), each with two 16-byte vectors, so that both elements of a
// pair sit in one thread in either layout and the norm is a shuffle over the
// head's lanes.  The cos / sin tables of all the CTA's rows are computed in
// one go, one pair a thread, while the first vectors are on their way, and the
// next head's vectors are loaded while one is turned.  The issue slots come
// next (339 instructions a warp and four heads kept them 67% busy), hence
// packed fp32 pairs, weights widened once per CTA, and addresses that move
// from head to head by additions.
#pragma once
#include "common.cuh"
#include "device_util.cuh"
#include "sm100_ptx.cuh"

namespace fdl {

constexpr int kNrThreads = 256;
constexpr int kNrMaxDim = 256;
constexpr int kNrMaxRows = 8;  // rows a CTA

struct NormRopeArgs {
  const void* y;
  int64_t y_rs;
  const int64_t* pos;
  const float* inv_freq;
  const void* qw;
  const void* kw;
  void* q;
  char* k;
  char* v;
  int64_t sp, ss, sh;  // page, slot, head strides (bytes)
  const int64_t* slots;
  int64_t n_slots;
  FastDiv page;
  FastDiv heads;  // hq + 2 hkv
  FastDiv pairs;  // rot / 2
  float eps, scale;
  int rows, hq, hkv, D, rot;
  int per;  // rows a CTA
};

// The 8 elements of a vector as four fp32 pairs.
template <typename T>
__device__ __forceinline__ void unpack_pairs(uint4 u, uint64_t (&x)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = Pack2<T>::to(w[i]);
    x[i] = ptx::pack2(t.x, t.y);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack_pairs(const uint64_t (&x)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    ptx::unpack2(x[i], lo, hi);
    w[i] = Pack2<T>::from(lo, hi);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint64_t sub2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <typename T, int GS, bool INTER>
__global__ void __launch_bounds__(kNrThreads, 4) norm_rope_kernel(const __grid_constant__ NormRopeArgs a) {
  // Per row, 16 bytes hold (cos, cos, sin, sin) of two neighbouring pairs,
  // ordered so that the lanes of a head read consecutive pieces; then the
  // weights of q and k heads, 16 bytes of a vector's halves ordered alike.
  extern __shared__ ulonglong2 s_cs[];
  __shared__ ulonglong2 s_w[2][2][kNrMaxDim / 8];
  __shared__ int64_t s_at[kNrMaxRows];  // byte offset of the row's slot, or -1
  await_stream();
  release_stream();
  const int row0 = blockIdx.x * a.per, nrows = min(a.per, a.rows - row0);
  const int L = a.D / 16;        // lanes that hold elements of a head
  const int RL = a.rot / 16;     // of these, lanes that turn pairs (half layout)
  const int lane = threadIdx.x % GS;
  // The two 16-byte vectors of this lane.
  int v0, v1;
  if (INTER) {
    v0 = lane;
    v1 = lane + L;
  } else if (lane < RL) {
    v0 = lane;
    v1 = lane + RL;
  } else {
    v0 = 2 * lane;
    v1 = 2 * lane + 1;
  }
  const bool mine = lane < L;
  const int heads = a.hq + 2 * a.hkv;
  // This lane group's heads: every kStep-th of the rows' heads.
  constexpr int kStep = kNrThreads / GS;
  uint32_t r0, h0, dr, dh;
  a.heads.divmod(threadIdx.x / GS, r0, h0);
  a.heads.divmod(kStep, dr, dh);
  int r = r0, h = h0;
  const int64_t head_b = a.D * 2, row_b = a.y_rs * 2;
  const int64_t move = static_cast<int64_t>(dr) * row_b + static_cast<int64_t>(dh) * head_b;
  const int64_t wrap = row_b - static_cast<int64_t>(heads) * head_b;
  const char* src = static_cast<const char*>(a.y) + (row0 + static_cast<int64_t>(r)) * row_b + h * head_b;
  int fr = r, fh = h;  // of the next vectors to load
  uint4 n0 = make_uint4(0, 0, 0, 0), n1 = n0;
  auto fetch = [&]() {
    if (mine && fr < nrows) {
      n0 = ld_stream16(src + v0 * 16);
      n1 = ld_stream16(src + v1 * 16);
    }
    src += move;
    fr += dr;
    fh += dh;
    if (fh >= heads) {
      fh -= heads;
      ++fr;
      src += wrap;
    }
  };
  fetch();
  if (threadIdx.x < nrows) {
    const int64_t slot = a.slots[row0 + threadIdx.x];
    int64_t at = -1;
    if (slot >= 0 && slot < a.n_slots) {
      uint32_t page, off;  // the host refuses pools of 2^31 slots
      a.page.divmod(static_cast<uint32_t>(slot), page, off);
      at = static_cast<int64_t>(page) * a.sp + static_cast<int64_t>(off) * a.ss;
    } else if (slot != -1) {
      report(FDL_DEV_INDEX, slot);
    }
    s_at[threadIdx.x] = at;
  }
  const bool norms = a.qw || a.kw;
  if (norms)
    for (int i = threadIdx.x; i < a.D / 4; i += kNrThreads) {  // (q or k, vector)
      const int k = i >= a.D / 8, v = i - k * (a.D / 8);
      const void* w = k ? a.kw : a.qw;
      if (w) {
        uint64_t f[4];
        unpack_pairs<T>(static_cast<const uint4*>(w)[v], f);
        s_w[k][0][v] = make_ulonglong2(f[0], f[1]);
        s_w[k][1][v] = make_ulonglong2(f[2], f[3]);
      }
    }
  const int pairs = a.rot / 2;
  for (int i = threadIdx.x; i < nrows * pairs; i += kNrThreads) {
    uint32_t rr, j;
    a.pairs.divmod(i, rr, j);
    double t = static_cast<double>(a.pos[row0 + rr]) * static_cast<double>(a.inv_freq[j]) * 0.15915494309189535;  // turns
    t -= rint(t);
    float sn, c;
    sincospif(2.f * static_cast<float>(t), &sn, &c);
    // half layout: piece (j % 8) / 2 of lane j / 8; interleaved: piece (j %
    // 4) / 2 of vector j / 4
    const int piece = INTER ? (j % 4) / 2 * (a.rot / 8) + j / 4 : (j % 8) / 2 * RL + j / 8;
    float* cs = reinterpret_cast<float*>(s_cs + rr * (pairs / 2) + piece);
    cs[j % 2] = c * a.scale;
    cs[2 + j % 2] = sn * a.scale;
  }
  __syncthreads();
  const float inv_d = 1.f / a.D;
  // every lane of a warp runs the same trips
  for (int left = (nrows * heads + kStep - 1) / kStep; left > 0; --left) {
    const uint4 u0 = n0, u1 = n1;
    fetch();
    const bool on = mine && r < nrows;
    const int kind = h < a.hq ? 0 : h < a.hq + a.hkv ? 1 : 2;  // q, k, v
    uint64_t x0[4], x1[4];
    unpack_pairs<T>(u0, x0);
    unpack_pairs<T>(u1, x1);
    if (norms) {
      uint64_t s2 = ptx::mul2(x0[0], x0[0]);
#pragma unroll
      for (int e = 1; e < 4; ++e) s2 = ptx::fma2(x0[e], x0[e], s2);
#pragma unroll
      for (int e = 0; e < 4; ++e) s2 = ptx::fma2(x1[e], x1[e], s2);
      float s, s_hi;
      ptx::unpack2(s2, s, s_hi);
      s += s_hi;
#pragma unroll
      for (int off = GS / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      if (on && (kind == 0 ? a.qw : kind == 1 ? a.kw : nullptr)) {
        const float inv = rsqrtf(fmaf(s, inv_d, a.eps));
        const uint64_t inv2 = ptx::pack2(inv, inv);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const ulonglong2 w0 = s_w[kind][half][v0], w1 = s_w[kind][half][v1];
          x0[2 * half] = ptx::mul2(x0[2 * half], ptx::mul2(inv2, w0.x));
          x0[2 * half + 1] = ptx::mul2(x0[2 * half + 1], ptx::mul2(inv2, w0.y));
          x1[2 * half] = ptx::mul2(x1[2 * half], ptx::mul2(inv2, w1.x));
          x1[2 * half + 1] = ptx::mul2(x1[2 * half + 1], ptx::mul2(inv2, w1.y));
        }
      }
    }
    if (on) {
      if (kind < 2) {
        const ulonglong2* cs = s_cs + r * (pairs / 2);
        if (INTER) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int vv = half ? v1 : v0;
            uint64_t(&x)[4] = half ? x1 : x0;
            if (vv < a.rot / 8) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const ulonglong2 c = cs[i * (a.rot / 8) + vv];
                float c0, c1, s0, s1;
                ptx::unpack2(c.x, c0, c1);
                ptx::unpack2(c.y, s0, s1);
                float xa, xb;
                ptx::unpack2(x[2 * i], xa, xb);
                x[2 * i] = ptx::pack2(xa * c0 - xb * s0, xb * c0 + xa * s0);
                ptx::unpack2(x[2 * i + 1], xa, xb);
                x[2 * i + 1] = ptx::pack2(xa * c1 - xb * s1, xb * c1 + xa * s1);
              }
            }
          }
        } else if (lane < RL) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const ulonglong2 c = cs[i * RL + lane];
            const uint64_t xa = x0[i], xb = x1[i];
            x0[i] = sub2(ptx::mul2(xa, c.x), ptx::mul2(xb, c.y));
            x1[i] = ptx::fma2(xb, c.x, ptx::mul2(xa, c.y));
          }
        }
      }
      char* dst;
      bool write = true;
      if (kind == 0) {
        dst = static_cast<char*>(a.q) + ((row0 + static_cast<int64_t>(r)) * a.hq + h) * head_b;
      } else {
        const int64_t at = s_at[r];
        dst = kind == 1 ? a.k + at + (h - a.hq) * a.sh : a.v + at + (h - a.hq - a.hkv) * a.sh;
        write = at >= 0;
      }
      if (write) {
        // V keeps its bits (a NaN's payload too)
        *reinterpret_cast<uint4*>(dst + v0 * 16) = kind == 2 ? u0 : pack_pairs<T>(x0);
        *reinterpret_cast<uint4*>(dst + v1 * 16) = kind == 2 ? u1 : pack_pairs<T>(x1);
      }
    }
    r += dr;
    h += dh;
    if (h >= heads) {
      h -= heads;
      ++r;
    }
  }
}

}  // namespace fdl
