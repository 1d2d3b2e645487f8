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
// next head's vectors are loaded while one is turned.
#pragma once
#include "common.cuh"
#include "device_util.cuh"

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

template <typename T, int GS, bool INTER>
__global__ void __launch_bounds__(kNrThreads, 4) norm_rope_kernel(const __grid_constant__ NormRopeArgs a) {
  // (cos, sin) of pair j of each row, ordered so that the lanes of a head
  // read consecutive 16-byte pieces.
  extern __shared__ float4 s_cs[];
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
  const int items = nrows * static_cast<int>(a.heads.d);
  const char* y0 = static_cast<const char*>(a.y) + static_cast<int64_t>(row0) * a.y_rs * 2;
  uint4 n0 = make_uint4(0, 0, 0, 0), n1 = n0;  // the next item's vectors
  auto fetch = [&](int i) {
    if (mine && i < items) {
      uint32_t r, h;
      a.heads.divmod(i, r, h);
      const char* p = y0 + static_cast<int64_t>(r) * a.y_rs * 2 + h * a.D * 2;
      n0 = ld_stream16(p + v0 * 16);
      n1 = ld_stream16(p + v1 * 16);
    }
  };
  int item = threadIdx.x / GS;
  constexpr int kStep = kNrThreads / GS;
  fetch(item);
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
  for (int i = threadIdx.x; i < nrows * (a.rot / 2); i += kNrThreads) {
    uint32_t r, j;
    a.pairs.divmod(i, r, j);
    double t = static_cast<double>(a.pos[row0 + r]) * static_cast<double>(a.inv_freq[j]) * 0.15915494309189535;  // turns
    t -= rint(t);
    float sn, c;
    sincospif(2.f * static_cast<float>(t), &sn, &c);
    // half layout: piece (j % 8) / 2 of lane j / 8; interleaved: piece (j %
    // 4) / 2 of vector j / 4
    const int at = INTER ? ((j % 4) / 2 * (a.rot / 8) + j / 4) * 2 + j % 2 : ((j % 8) / 2 * RL + j / 8) * 2 + j % 2;
    reinterpret_cast<float2*>(s_cs)[r * (a.rot / 2) + at] = make_float2(c * a.scale, sn * a.scale);
  }
  __syncthreads();
  for (int base = 0; base < items; base += kStep, item += kStep) {  // every lane runs the same trips
    const uint4 u0 = n0, u1 = n1;
    fetch(item + kStep);
    uint32_t r, hh;
    a.heads.divmod(min(item, items - 1), r, hh);
    const int h = hh;
    const bool on = mine && item < items;
    const void* w = h < a.hq ? a.qw : h < a.hq + a.hkv ? a.kw : nullptr;
    float x0[8], x1[8];
    unpack8<T>(u0, x0);
    unpack8<T>(u1, x1);
    if (a.qw || a.kw) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(x0[e], x0[e], s);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(x1[e], x1[e], s);
#pragma unroll
      for (int off = GS / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      if (w && on) {
        const float inv = rsqrtf(s / a.D + a.eps);
        float w0[8], w1[8];
        unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const char*>(w) + v0 * 16), w0);
        unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const char*>(w) + v1 * 16), w1);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x0[e] = x0[e] * inv * w0[e];
          x1[e] = x1[e] * inv * w1[e];
        }
      }
    }
    if (on) {
      const bool copied = h >= a.hq + a.hkv;  // V keeps its bits (a NaN's payload too)
      if (!copied) {
        const float4* cs = s_cs + r * (a.rot / 4);
        if (INTER) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int vv = half ? v1 : v0;
            float* x = half ? x1 : x0;
            if (vv < a.rot / 8) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float4 c = cs[i * (a.rot / 8) + vv];
                const float a0 = x[4 * i], b0 = x[4 * i + 1], a1 = x[4 * i + 2], b1 = x[4 * i + 3];
                x[4 * i] = a0 * c.x - b0 * c.y;
                x[4 * i + 1] = b0 * c.x + a0 * c.y;
                x[4 * i + 2] = a1 * c.z - b1 * c.w;
                x[4 * i + 3] = b1 * c.z + a1 * c.w;
              }
            }
          }
        } else if (lane < RL) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 c = cs[i * RL + lane];
            const float a0 = x0[2 * i], b0 = x1[2 * i], a1 = x0[2 * i + 1], b1 = x1[2 * i + 1];
            x0[2 * i] = a0 * c.x - b0 * c.y;
            x1[2 * i] = b0 * c.x + a0 * c.y;
            x0[2 * i + 1] = a1 * c.z - b1 * c.w;
            x1[2 * i + 1] = b1 * c.z + a1 * c.w;
          }
        }
      }
      char* dst;
      bool write = true;
      if (h < a.hq) {
        dst = static_cast<char*>(a.q) + ((static_cast<int64_t>(row0) + r) * a.hq + h) * a.D * 2;
      } else {
        const int kh = h - a.hq;
        const int64_t at = s_at[r];
        dst = kh < a.hkv ? a.k + at + kh * a.sh : a.v + at + (kh - a.hkv) * a.sh;
        write = at >= 0;
      }
      if (write) {
        *reinterpret_cast<uint4*>(dst + v0 * 16) = copied ? u0 : pack8<T>(x0);
        *reinterpret_cast<uint4*>(dst + v1 * 16) = copied ? u1 : pack8<T>(x1);
      }
    }
  }
}

}  // namespace fdl
