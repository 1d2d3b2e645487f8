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
// Bound by HBM: each element is read once and written once.  A CTA holds one
// row; a head takes GS lanes (D / 16 rounded up to a power of two), each with
// two 16-byte vectors, so that both elements of a pair sit in one thread in
// either layout and the norm is a shuffle over the head's lanes.  Both loads
// are in flight before the row's cos / sin table is computed.
#pragma once
#include "common.cuh"
#include "device_util.cuh"

namespace fdl {

constexpr int kNrMaxThreads = 512;
constexpr int kNrMaxDim = 256;

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
  float eps, scale;
  int rows, hq, hkv, D, rot;
};

template <typename T, int GS, bool INTER>
__global__ void __launch_bounds__(kNrMaxThreads) norm_rope_kernel(const __grid_constant__ NormRopeArgs a) {
  // (cos, sin) of pair j, ordered so that the lanes of a head read
  // consecutive 16-byte pieces.
  __shared__ float4 s_cs[kNrMaxDim / 4];
  await_stream();
  release_stream();
  const int row = blockIdx.x;
  const int L = a.D / 16;        // lanes that hold elements of a head
  const int RL = a.rot / 16;     // of these, lanes that turn pairs (half layout)
  const int heads = a.hq + 2 * a.hkv;
  const int lane = threadIdx.x % GS;
  const char* yr = static_cast<const char*>(a.y) + static_cast<int64_t>(row) * a.y_rs * 2;
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
  uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0;
  int h = threadIdx.x / GS;
  const int hstep = blockDim.x / GS;
  if (mine && h < heads) {
    u0 = ld_stream16(yr + (h * a.D + v0 * 8) * 2);
    u1 = ld_stream16(yr + (h * a.D + v1 * 8) * 2);
  }
  const int64_t slot = a.slots[row];
  {
    const double p = static_cast<double>(a.pos[row]);
    float2* cs = reinterpret_cast<float2*>(s_cs);
    for (int j = threadIdx.x; j < a.rot / 2; j += blockDim.x) {
      double t = p * static_cast<double>(a.inv_freq[j]) * 0.15915494309189535;  // turns
      t -= rint(t);
      float sn, c;
      sincospif(2.f * static_cast<float>(t), &sn, &c);
      // half layout: piece i = (j % 8) / 2 of lane j / 8; interleaved: piece
      // (j % 4) / 2 of vector j / 4
      const int at = INTER ? ((j % 4) / 2 * (a.rot / 8) + j / 4) * 2 + j % 2 : ((j % 8) / 2 * RL + j / 8) * 2 + j % 2;
      cs[at] = make_float2(c * a.scale, sn * a.scale);
    }
  }
  const bool store = slot >= 0 && slot < a.n_slots;
  if (!store && slot != -1 && threadIdx.x == 0) report(FDL_DEV_INDEX, slot);
  uint32_t pg = 0, po = 0;
  if (store) {
    // slots below 2^31 divide fast; the host refuses larger pools
    a.page.divmod(static_cast<uint32_t>(slot), pg, po);
  }
  const int64_t kv_at = static_cast<int64_t>(pg) * a.sp + static_cast<int64_t>(po) * a.ss;
  __syncthreads();
  for (; h - static_cast<int>(threadIdx.x / GS) < heads; h += hstep) {  // every lane of a warp runs the same trips
    const bool on = mine && h < heads;
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
      if (h < a.hq + a.hkv) {
        if (INTER) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int vv = half ? v1 : v0;
            float* x = half ? x1 : x0;
            if (vv < a.rot / 8) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float4 c = s_cs[i * (a.rot / 8) + vv];
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
            const float4 c = s_cs[i * RL + lane];
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
        dst = static_cast<char*>(a.q) + (static_cast<int64_t>(row) * a.hq + h) * a.D * 2;
      } else {
        const int kh = h - a.hq;
        dst = kh < a.hkv ? a.k + kv_at + kh * a.sh : a.v + kv_at + (kh - a.hkv) * a.sh;
        write = store;
      }
      if (write) {
        // heads that are only copied keep their bits (a NaN's payload too)
        const bool same = h >= a.hq + a.hkv;
        *reinterpret_cast<uint4*>(dst + v0 * 16) = same ? u0 : pack8<T>(x0);
        *reinterpret_cast<uint4*>(dst + v1 * 16) = same ? u1 : pack8<T>(x1);
      }
    }
    const int hn = h + hstep;
    if (mine && hn < heads) {
      u0 = ld_stream16(yr + (hn * a.D + v0 * 8) * 2);
      u1 = ld_stream16(yr + (hn * a.D + v1 * 8) * 2);
    }
  }
}

}  // namespace fdl
