// RMS norm of every head of q and k and the rotation of its position, in one pass, with its gradients.
//
// For a row x of D values (one head of one token), its weight w [D] and row pos of cos / sin [rows, R/2]:
//     r = 1 / sqrt(mean(x^2) + eps)        y = x r w
//     o[a_i] = y[a_i] cos_i - y[b_i] sin_i,  o[b_i] = y[b_i] cos_i + y[a_i] sin_i   for i < R/2,   o[j] = y[j] for j >= R
// with the pairs (a_i, b_i) = (i, i + R/2), or (2i, 2i + 1) when interleaved. Backward, with g the gradient turned back
// (the rotation's transpose):
//     dw = sum over rows of g x r          dx = r (g w - x r mean(g w x r))
// r is computed again from x, which the backward reads anyway.
//
// Everything is fp32 from the loads to the one rounding of each output; the products of the reference's separate passes
// (norm, then kernels/rotary/kernel.cpp:44-74) are rounded to bf16 in between.
//
// Bound by HBM: the forward reads x and writes o, the backward reads x and do and writes dx, once each. A row belongs to LPR
// lanes of 16 values, which a lane takes as two 16-byte pieces: the two halves of eight pairs, or 16 neighbours. Sums over a
// row are shuffles. The rows of q and those of k are counted apart, and a block has rows of one of them only: so a thread
// keeps its 16 weights in registers, and in the backward its 16 sums of dw.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_fwd_sm100.cuh"
#include "sm100_ptx.cuh"

namespace hk {

enum : int { kStatusBadPos = 5 };  // a position outside the tables

constexpr int kQknThreads = 256;
constexpr int kQknMaxD = 256;
constexpr int kQknMaxBlocks = 1184;  // of the backward, and rows of partial sums in its workspace: 8 on each of 148 SMs

// One of q and k.
struct QknSide {
  const __nv_bfloat16* x;
  const __nv_bfloat16* dy;      // backward: contiguous [tokens, heads, D]
  __nv_bfloat16* out;           // o, or dx: contiguous [tokens, heads, D]
  const void* w;                // [D], bf16 or fp32 (weight_f32); null: ones
  void* dw;                     // backward: [D] of w's type, or null
  long long stride_b, stride_n, stride_h;  // of x, elements
  int rows;                     // tokens * heads
  int heads;
  FastDiv fd_heads;
};
struct QknParams {
  QknSide side[2];              // q, k
  const void* cos;              // [table_rows, R/2]
  const void* sin;
  const int32_t* positions;     // [tokens], or null: token n of a sequence is at n + pos0
  float* partial;               // backward: [blocks][D] sums of dw, blocks of q before those of k; null: no dw wanted
  int N, D, R, table_rows, pos0, weight_f32;
  int blocks0;                  // blocks [0, blocks0) have rows of q
  float eps;
  FastDiv fd_n;
  int* status;
};

namespace qkn {

__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(ptx::pack_bf16x2(f[0], f[1]), ptx::pack_bf16x2(f[2], f[3]), ptx::pack_bf16x2(f[4], f[5]),
                    ptx::pack_bf16x2(f[6], f[7]));
}
// Eight values from `at` on, of a bf16 or fp32 array.
template <bool F32>
__device__ __forceinline__ void load8(const void* p, size_t at, float* f) {
  if constexpr (F32) {
    const float4* v = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 a = v[0], b = v[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + at), f);
  }
}

// What one lane has of a row: 16 values in two pieces of 8, at columns c0 and c1, and whether they are rotated pairs.
struct Lane {
  int c0, c1;
  bool active, turned;
};
template <bool INTER>
__device__ __forceinline__ Lane lane_of(int u, int D, int R) {
  Lane l;
  l.active = u * 16 < D;
  l.turned = u * 16 < R;
  l.c0 = (INTER || !l.turned) ? u * 16 : u * 8;
  l.c1 = (INTER || !l.turned) ? u * 16 + 8 : R / 2 + u * 8;
  return l;
}
// Turns the pairs of a lane's 16 values by the angles of cos and sin (sin negated: back).
template <bool INTER>
__device__ __forceinline__ void turn(float* y, const float* cos, const float* sin, float sign) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int a = INTER ? 2 * i : i, b = INTER ? 2 * i + 1 : i + 8;
    const float s = sign * sin[i], ya = y[a], yb = y[b];
    y[a] = ya * cos[i] - yb * s;
    y[b] = yb * cos[i] + ya * s;
  }
}
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// Where a row lies, and its row of the tables (-1: outside, which the caller reports).
struct Row {
  size_t x, dense;
  int pos;
};
__device__ __forceinline__ Row locate(const QknParams& p, const QknSide& s, int row) {
  int token, h, b, n;
  s.fd_heads.divmod(row, token, h);
  p.fd_n.divmod(token, b, n);
  Row r;
  r.x = static_cast<size_t>(b) * s.stride_b + static_cast<size_t>(n) * s.stride_n + static_cast<size_t>(h) * s.stride_h;
  r.dense = static_cast<size_t>(row) * p.D;
  r.pos = p.positions ? p.positions[token] : n + p.pos0;
  if (r.pos < 0 || r.pos >= p.table_rows) r.pos = -1;
  return r;
}

}  // namespace qkn

// A thread takes UN rows and requests all of them before it reduces the first. grid = blocks of q, then blocks of k;
// block = 256, kQknThreads / LPR * UN rows each.
template <int LPR, bool INTER, bool TF32, int UN>
__global__ void __launch_bounds__(kQknThreads) qk_norm_rotary_kernel(const __grid_constant__ QknParams p) {
  using namespace qkn;
  constexpr int kRows = kQknThreads / LPR;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const bool is_k = static_cast<int>(blockIdx.x) >= p.blocks0;
  const QknSide& s = p.side[is_k];
  const int row0 = (static_cast<int>(blockIdx.x) - (is_k ? p.blocks0 : 0)) * (kRows * UN) + threadIdx.x / LPR;
  const int u = threadIdx.x % LPR;
  const Lane l = lane_of<INTER>(u, p.D, p.R);

  Row at[UN];
  uint4 raw[UN][2];
#pragma unroll
  for (int i = 0; i < UN; ++i) {
    at[i] = locate(p, s, min(row0 + i * kRows, s.rows - 1));  // a row beyond the last: that one again, and not stored
    raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
    if (l.active) {
      raw[i][0] = __ldcs(reinterpret_cast<const uint4*>(s.x + at[i].x + l.c0));
      raw[i][1] = __ldcs(reinterpret_cast<const uint4*>(s.x + at[i].x + l.c1));
    }
  }
  float w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = 1.f;
  if (s.w && l.active) {
    if (p.weight_f32) {
      load8<true>(s.w, l.c0, w);
      load8<true>(s.w, l.c1, w + 8);
    } else {
      load8<false>(s.w, l.c0, w);
      load8<false>(s.w, l.c1, w + 8);
    }
  }
#pragma unroll
  for (int i = 0; i < UN; ++i) {
    float y[16], cos[8], sin[8];
    const size_t t = static_cast<size_t>(max(at[i].pos, 0)) * (p.R / 2) + u * 8;
    if (l.turned) {
      load8<TF32>(p.cos, t, cos);
      load8<TF32>(p.sin, t, sin);
    }
    unpack8(raw[i][0], y);
    unpack8(raw[i][1], y + 8);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) ss = fmaf(y[j], y[j], ss);
    const float r = rsqrtf(row_sum<LPR>(ss) / static_cast<float>(p.D) + p.eps);
#pragma unroll
    for (int j = 0; j < 16; ++j) y[j] = y[j] * r * w[j];
    if (l.turned) turn<INTER>(y, cos, sin, 1.f);
    if (row0 + i * kRows < s.rows && l.active) {
      uint4 a = pack8(y), b = pack8(y + 8);
      if (at[i].pos < 0) {
        a = b = make_uint4(0, 0, 0, 0);
        if (u == 0) atomicCAS(p.status, kStatusOk, kStatusBadPos);
      }
      *reinterpret_cast<uint4*>(s.out + at[i].dense + l.c0) = a;
      *reinterpret_cast<uint4*>(s.out + at[i].dense + l.c1) = b;
    }
  }
}

// The same rows, backwards: a block goes through its share of them, and leaves its sums of dw for the kernel behind.
template <int LPR, bool INTER, bool TF32>
__global__ void __launch_bounds__(kQknThreads) qk_norm_rotary_bwd_kernel(const __grid_constant__ QknParams p) {
  using namespace qkn;
  constexpr int kRows = kQknThreads / LPR, UN = 2;
  __shared__ float sums[kQknThreads / 32][LPR * 16];
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const bool is_k = static_cast<int>(blockIdx.x) >= p.blocks0;
  const QknSide& s = p.side[is_k];
  const int block = static_cast<int>(blockIdx.x) - (is_k ? p.blocks0 : 0);
  const int blocks = is_k ? static_cast<int>(gridDim.x) - p.blocks0 : p.blocks0;
  const int u = threadIdx.x % LPR;
  const Lane l = lane_of<INTER>(u, p.D, p.R);

  float w[16], dw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    w[i] = 1.f;
    dw[i] = 0.f;
  }
  if (s.w && l.active) {
    if (p.weight_f32) {
      load8<true>(s.w, l.c0, w);
      load8<true>(s.w, l.c1, w + 8);
    } else {
      load8<false>(s.w, l.c0, w);
      load8<false>(s.w, l.c1, w + 8);
    }
  }
  // the loop is uniform over the block: the sums over a row are shuffles of whole warps
  for (long long base = static_cast<long long>(block) * (kRows * UN); base < s.rows;
       base += static_cast<long long>(blocks) * (kRows * UN)) {
    const int row0 = static_cast<int>(base) + threadIdx.x / LPR;
    Row at[UN];
    uint4 raw[UN][2], rawg[UN][2];
    bool live[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      live[i] = row0 + i * kRows < s.rows;  // rows stay below 2^31 - 2^20
      at[i] = locate(p, s, live[i] ? row0 + i * kRows : s.rows - 1);
      raw[i][0] = raw[i][1] = rawg[i][0] = rawg[i][1] = make_uint4(0, 0, 0, 0);
      if (l.active) {
        raw[i][0] = __ldcs(reinterpret_cast<const uint4*>(s.x + at[i].x + l.c0));
        raw[i][1] = __ldcs(reinterpret_cast<const uint4*>(s.x + at[i].x + l.c1));
        rawg[i][0] = __ldcs(reinterpret_cast<const uint4*>(s.dy + at[i].dense + l.c0));
        rawg[i][1] = __ldcs(reinterpret_cast<const uint4*>(s.dy + at[i].dense + l.c1));
      }
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      float x[16], g[16], cos[8], sin[8];
      const size_t t = static_cast<size_t>(max(at[i].pos, 0)) * (p.R / 2) + u * 8;
      if (l.turned) {
        load8<TF32>(p.cos, t, cos);
        load8<TF32>(p.sin, t, sin);
      }
      unpack8(raw[i][0], x);
      unpack8(raw[i][1], x + 8);
      unpack8(rawg[i][0], g);
      unpack8(rawg[i][1], g + 8);
      if (l.turned) turn<INTER>(g, cos, sin, -1.f);
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        ss = fmaf(x[j], x[j], ss);
        dot = fmaf(g[j] * w[j], x[j], dot);
      }
      const float inv_d = 1.f / static_cast<float>(p.D);
      const float r = rsqrtf(row_sum<LPR>(ss) * inv_d + p.eps);
      const float m = row_sum<LPR>(dot) * r * inv_d;  // mean of (g w) (x r)
      const bool good = live[i] && at[i].pos >= 0;
      float dx[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float hat = x[j] * r;
        if (good) dw[j] = fmaf(g[j], hat, dw[j]);
        dx[j] = r * (g[j] * w[j] - hat * m);
      }
      if (live[i] && l.active) {
        uint4 a = pack8(dx), b = pack8(dx + 8);
        if (at[i].pos < 0) {
          a = b = make_uint4(0, 0, 0, 0);
          if (u == 0) atomicCAS(p.status, kStatusOk, kStatusBadPos);
        }
        *reinterpret_cast<uint4*>(s.out + at[i].dense + l.c0) = a;
        *reinterpret_cast<uint4*>(s.out + at[i].dense + l.c1) = b;
      }
    }
  }
  if (!p.partial) return;  // uniform over the grid
  // the block's sums, in a fixed order: lanes of a warp that have the same columns, then the warps
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int off = 16; off >= LPR; off >>= 1) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], off);
  if ((threadIdx.x & 31) < LPR && l.active) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sums[threadIdx.x / 32][l.c0 + i] = dw[i];
      sums[threadIdx.x / 32][l.c1 + i] = dw[8 + i];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.D; c += kQknThreads) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kQknThreads / 32; ++k) v += sums[k][c];
    p.partial[static_cast<size_t>(blockIdx.x) * p.D + c] = v;
  }
}

// dw of q and of k from the blocks' sums, added in a fixed order: a warp has 32 columns of every 32nd block, and the warps
// are added up. grid = (ceil(D / 32), 2), block = 1024.
__global__ void __launch_bounds__(1024) qk_norm_rotary_dw_kernel(const __grid_constant__ QknParams p, int blocks) {
  __shared__ float sums[32][33];
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const QknSide& s = p.side[blockIdx.y];
  const int first = blockIdx.y ? p.blocks0 : 0, end = blockIdx.y ? blocks : p.blocks0;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < p.D) {
#pragma unroll 4
    for (int b = first + warp; b < end; b += 32) v += p.partial[static_cast<size_t>(b) * p.D + c];
  }
  sums[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < p.D && s.dw) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += sums[k][lane];
    if (p.weight_f32) static_cast<float*>(s.dw)[c] = t;
    else static_cast<__nv_bfloat16*>(s.dw)[c] = __float2bfloat16(t);
  }
}

}  // namespace hk
