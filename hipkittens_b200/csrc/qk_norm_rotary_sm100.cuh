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
// A warp has a run of rows, so that the heads of one token share the angles in registers and the next row is an addition away;
// arithmetic is packed in pairs; the rows to come wait in a ring of cp.async stages and take no registers. Instructions are what
// would bound it otherwise: with four unrelated rows a thread, each with divisions for its place and angles of its own in scalar
// arithmetic, 16 values take 300 of them. us, B4 N4096 H32/8 D128, so / as it is: forward 73.7 / 55.4 (336 MB, 6.06 TB/s),
// backward 106 / 87 to 89 (503 MB, 5.7 TB/s).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_fwd_sm100.cuh"
#include "paged_decode_common.cuh"
#include "sm100_ptx.cuh"

namespace hk {


constexpr int kQknThreads = 128;
constexpr int kQknStages = 3;
constexpr int kQknMaxD = 256;
constexpr int kQknMaxBlocks = 1184;  // of the backward, each with a row of partial sums in its workspace

// One of q and k.
struct QknSide {
  const __nv_bfloat16* x;
  const __nv_bfloat16* dy;      // backward: contiguous [tokens, heads, D]
  __nv_bfloat16* out;           // o, or dx: contiguous [tokens, heads, D]
  const void* w;                // [D], bf16 or fp32 (weight_f32); null: ones
  void* dw;                     // backward: [D] of w's type, or null
  long long stride_b;           // of x, in units of 8 values
  int stride_n, stride_h;
  int rows;                     // tokens * heads
  int heads;
  int run_units, run_more;      // units of 32 / LPR rows that every warp takes, and how many warps take one more
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
  float eps, inv_d;
  FastDiv fd_n;
  int* status;
};

namespace qkn {

// The 16 values of a lane as packed fp32 pairs: with (a_i, b_i) the i-th of its rotated pairs, a[j] holds a_2j and a_2j+1,
// b[j] holds b_2j and b_2j+1, in either layout. (Values that are not rotated take the places of pairs as they come.)
struct Vals {
  uint64_t a[4], b[4];
};
__device__ __forceinline__ uint64_t lows(uint32_t v0, uint32_t v1) {
  return ptx::pack2(__uint_as_float(v0 << 16), __uint_as_float(v1 << 16));
}
__device__ __forceinline__ uint64_t highs(uint32_t v0, uint32_t v1) {
  return ptx::pack2(__uint_as_float(v0 & 0xffff0000u), __uint_as_float(v1 & 0xffff0000u));
}
__device__ __forceinline__ uint64_t both(uint32_t v) {
  return ptx::pack2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
// From the lane's two 16-byte pieces of bf16.
template <bool INTER>
__device__ __forceinline__ void unpack(const uint4& p0, const uint4& p1, Vals& v) {
  const uint32_t w[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v.a[j] = INTER ? lows(w[2 * j], w[2 * j + 1]) : both(w[j]);
    v.b[j] = INTER ? highs(w[2 * j], w[2 * j + 1]) : both(w[4 + j]);
  }
}
template <bool INTER>
__device__ __forceinline__ void pack(const Vals& v, uint4& p0, uint4& p1) {
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a0, a1, b0, b1;
    ptx::unpack2(v.a[j], a0, a1);
    ptx::unpack2(v.b[j], b0, b1);
    w[INTER ? 2 * j : j] = INTER ? ptx::pack_bf16x2(a0, b0) : ptx::pack_bf16x2(a0, a1);
    w[INTER ? 2 * j + 1 : 4 + j] = INTER ? ptx::pack_bf16x2(a1, b1) : ptx::pack_bf16x2(b0, b1);
  }
  p0 = make_uint4(w[0], w[1], w[2], w[3]);
  p1 = make_uint4(w[4], w[5], w[6], w[7]);
}
// Eight neighbours of a table, as four packed pairs.
template <bool F32>
__device__ __forceinline__ void load8(const void* p, size_t at, uint64_t* f) {
  if constexpr (F32) {
    const float4* v = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 x = v[0], y = v[1];
    f[0] = ptx::pack2(x.x, x.y), f[1] = ptx::pack2(x.z, x.w), f[2] = ptx::pack2(y.x, y.y), f[3] = ptx::pack2(y.z, y.w);
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + at);
    f[0] = both(v.x), f[1] = both(v.y), f[2] = both(v.z), f[3] = both(v.w);
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
template <bool INTER>
__device__ __forceinline__ void load_weight(const void* w, int f32, const Lane& l, Vals& v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v.a[j] = v.b[j] = ptx::pack2(1.f, 1.f);
  if (!w || !l.active) return;
  if (f32) {
    const float* p = static_cast<const float*>(w);
    float x[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = p[l.c0 + i];
      x[8 + i] = p[l.c1 + i];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v.a[j] = INTER ? ptx::pack2(x[4 * j], x[4 * j + 2]) : ptx::pack2(x[2 * j], x[2 * j + 1]);
      v.b[j] = INTER ? ptx::pack2(x[4 * j + 1], x[4 * j + 3]) : ptx::pack2(x[8 + 2 * j], x[8 + 2 * j + 1]);
    }
  } else {
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(w);
    unpack<INTER>(*reinterpret_cast<const uint4*>(p + l.c0), *reinterpret_cast<const uint4*>(p + l.c1), v);
  }
}
// Turns the pairs by the angles of cos and sin, or back.
template <bool BACK>
__device__ __forceinline__ void turn(Vals& v, const uint64_t* cos, const uint64_t* sin) {
  const uint64_t minus = ptx::pack2(-1.f, -1.f);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t neg = ptx::mul2(sin[j], minus), s_a = BACK ? sin[j] : neg, s_b = BACK ? neg : sin[j];
    const uint64_t a = ptx::fma2(v.b[j], s_a, ptx::mul2(v.a[j], cos[j]));
    v.b[j] = ptx::fma2(v.a[j], s_b, ptx::mul2(v.b[j], cos[j]));
    v.a[j] = a;
  }
}
__device__ __forceinline__ float sum2(uint64_t v) {
  float x, y;
  ptx::unpack2(v, x, y);
  return x + y;
}
__device__ __forceinline__ float dot(const Vals& x, const Vals& y) {
  uint64_t s = ptx::mul2(x.a[0], y.a[0]), t = ptx::mul2(x.b[0], y.b[0]);
#pragma unroll
  for (int j = 1; j < 4; ++j) {
    s = ptx::fma2(x.a[j], y.a[j], s);
    t = ptx::fma2(x.b[j], y.b[j], t);
  }
  return sum2(ptx::add2(s, t));
}
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// A row of a thread's run, and what comes kStep rows behind it: the next heads of the same token, mostly.
struct Walk {
  int b, n, h;
  __device__ __forceinline__ Walk(const QknParams& p, const QknSide& s, int row) {
    int token;
    s.fd_heads.divmod(row, token, h);
    p.fd_n.divmod(token, b, n);
  }
  // true: another token
  __device__ __forceinline__ bool next(const QknParams& p, const QknSide& s, int step) {
    h += step;
    if (h < s.heads) return false;
    int tokens, seqs;
    s.fd_heads.divmod(h, tokens, h);
    p.fd_n.divmod(n + tokens, seqs, n);
    b += seqs;
    return true;
  }
  // What `step` more heads of the same token are away. In 64 bits: a head's stride alone may be 2^30 units.
  static __device__ __forceinline__ long long heads_on(const QknSide& s, int step) { return static_cast<long long>(step) * s.stride_h; }
  __device__ __forceinline__ const uint4* place(const QknSide& s) const {
    return reinterpret_cast<const uint4*>(s.x) + (b * s.stride_b + static_cast<long long>(n) * s.stride_n + static_cast<long long>(h) * s.stride_h);
  }
};
// The angles of a token's position, as a lane needs them; false: the position lies outside the tables.
template <bool TF32>
__device__ __forceinline__ bool angles(const QknParams& p, const Walk& at, const Lane& l, int u, uint64_t* cos, uint64_t* sin) {
  const int pos = p.positions ? p.positions[static_cast<long long>(at.b) * p.N + at.n] : at.n + p.pos0;
  if (static_cast<unsigned>(pos) >= static_cast<unsigned>(p.table_rows)) return false;
  if (l.turned) {
    const size_t t = static_cast<size_t>(pos) * (p.R / 2) + u * 8;
    load8<TF32>(p.cos, t, cos);
    load8<TF32>(p.sin, t, sin);
  }
  return true;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

}  // namespace qkn

// The rows of a side are dealt to its warps in runs, kStep of them at a time, a row to LPR lanes. Each lane has a ring of stages of
// its own in shared memory, PIECES 16-byte pieces a row (x, or x and dy): what it has asked for takes no registers, and nobody
// waits for anybody. Heads of one token share their angles, which stay in registers until the token changes.
template <int LPR, int PIECES>
struct QknRing {
  static constexpr int kStep = 32 / LPR;
  static constexpr int kStageBytes = kQknThreads * 16 * PIECES;
  static constexpr int kBytes = kQknStages * kStageBytes;
};
struct QknRun {
  int row, end;  // rows [row, end) of this thread's warp, from this thread's first
  template <int STEP>
  static __device__ __forceinline__ QknRun of(const QknSide& s, int block, int lane_row) {
    const int w = block * (kQknThreads / 32) + threadIdx.x / 32;
    const int first = w * s.run_units + min(w, s.run_more);  // the first run_more warps have a unit more
    return {first * STEP + lane_row, (first + s.run_units + (w < s.run_more ? 1 : 0)) * STEP};
  }
};

template <int LPR, bool INTER, bool TF32>
__global__ void __launch_bounds__(kQknThreads, 6) qk_norm_rotary_kernel(const __grid_constant__ QknParams p) {
  using namespace qkn;
  using Ring = QknRing<LPR, 2>;
  constexpr int kStep = Ring::kStep;
  __shared__ __align__(16) uint8_t ring[Ring::kBytes];
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const bool is_k = static_cast<int>(blockIdx.x) >= p.blocks0;
  const QknSide& s = p.side[is_k];
  const int block = static_cast<int>(blockIdx.x) - (is_k ? p.blocks0 : 0);
  const int u = threadIdx.x % LPR;
  const Lane l = lane_of<INTER>(u, p.D, p.R);
  const uint32_t slot = ptx::smem_u32(ring) + threadIdx.x * 16;
  const QknRun run = QknRun::of<kStep>(s, block, (threadIdx.x & 31) / LPR);

  Walk ahead(p, s, run.row), at = ahead;
  const uint4* x = ahead.place(s);
  int ahead_row = run.row;
  auto fetch = [&](int stage) {
    if (ahead_row < run.end && ahead_row < s.rows && l.active) {
      cp_async16(slot + stage * Ring::kStageBytes, x + l.c0 / 8);
      cp_async16(slot + stage * Ring::kStageBytes + kQknThreads * 16, x + l.c1 / 8);
    }
    cp_async_commit();
    ahead_row += kStep;
    x += Walk::heads_on(s, kStep);
    if (ahead.next(p, s, kStep)) x = ahead.place(s);
  };
#pragma unroll
  for (int i = 0; i < kQknStages - 1; ++i) fetch(i);
  Vals w;
  load_weight<INTER>(s.w, p.weight_f32, l, w);
  uint4* out = reinterpret_cast<uint4*>(s.out) + static_cast<long long>(run.row) * (p.D / 8);
  uint64_t cos[4], sin[4];
  int stage = 0;
  bool fresh = true, good = false;
  // the loop is uniform over a warp: the sums over a row are shuffles
  for (int row = run.row; row < run.end; row += kStep, out += kStep * (p.D / 8)) {
    const bool live = row < s.rows && l.active;
    if (fresh && live) good = angles<TF32>(p, at, l, u, cos, sin);
    cp_async_wait<kQknStages - 2>();
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (live) {
      a = lds16(slot + stage * Ring::kStageBytes);
      b = lds16(slot + stage * Ring::kStageBytes + kQknThreads * 16);
    }
    fetch((stage + kQknStages - 1) % kQknStages);
    Vals y;
    unpack<INTER>(a, b, y);
    const float r = rsqrtf(fmaf(row_sum<LPR>(dot(y, y)), p.inv_d, p.eps));
    const uint64_t r2 = ptx::pack2(r, r);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      y.a[j] = ptx::mul2(ptx::mul2(y.a[j], r2), w.a[j]);
      y.b[j] = ptx::mul2(ptx::mul2(y.b[j], r2), w.b[j]);
    }
    if (l.turned) turn<false>(y, cos, sin);
    if (live) {
      pack<INTER>(y, a, b);
      if (!good) {
        a = b = make_uint4(0, 0, 0, 0);
        if (u == 0) atomicCAS(p.status, kStatusOk, kStatusBadPos);
      }
      out[l.c0 / 8] = a;
      out[l.c1 / 8] = b;
    }
    fresh = at.next(p, s, kStep);
    stage = stage + 1 == kQknStages ? 0 : stage + 1;
  }
  cp_async_wait<0>();
}

// The same rows, backwards: a block leaves its sums of dw for the kernel behind.
template <int LPR, bool INTER, bool TF32>
__global__ void __launch_bounds__(kQknThreads, 4) qk_norm_rotary_bwd_kernel(const __grid_constant__ QknParams p) {
  using namespace qkn;
  using Ring = QknRing<LPR, 4>;
  constexpr int kStep = Ring::kStep;
  __shared__ __align__(16) uint8_t ring[Ring::kBytes];
  __shared__ float sums[kQknThreads / 32][LPR * 16];
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const bool is_k = static_cast<int>(blockIdx.x) >= p.blocks0;
  const QknSide& s = p.side[is_k];
  const int block = static_cast<int>(blockIdx.x) - (is_k ? p.blocks0 : 0);
  const int u = threadIdx.x % LPR;
  const Lane l = lane_of<INTER>(u, p.D, p.R);
  const uint32_t slot = ptx::smem_u32(ring) + threadIdx.x * 16;
  const QknRun run = QknRun::of<kStep>(s, block, (threadIdx.x & 31) / LPR);

  Walk ahead(p, s, run.row), at = ahead;
  const uint4* x_ahead = ahead.place(s);
  const uint4* dy = reinterpret_cast<const uint4*>(s.dy) + static_cast<long long>(run.row) * (p.D / 8);
  int ahead_row = run.row;
  auto fetch = [&](int stage) {
    if (ahead_row < run.end && ahead_row < s.rows && l.active) {
      const uint32_t dst = slot + stage * Ring::kStageBytes;
      cp_async16(dst, x_ahead + l.c0 / 8);
      cp_async16(dst + kQknThreads * 16, x_ahead + l.c1 / 8);
      cp_async16(dst + kQknThreads * 32, dy + l.c0 / 8);
      cp_async16(dst + kQknThreads * 48, dy + l.c1 / 8);
    }
    cp_async_commit();
    ahead_row += kStep;
    dy += kStep * (p.D / 8);
    x_ahead += Walk::heads_on(s, kStep);
    if (ahead.next(p, s, kStep)) x_ahead = ahead.place(s);
  };
#pragma unroll
  for (int i = 0; i < kQknStages - 1; ++i) fetch(i);
  Vals w, dw;
  load_weight<INTER>(s.w, p.weight_f32, l, w);
#pragma unroll
  for (int j = 0; j < 4; ++j) dw.a[j] = dw.b[j] = ptx::pack2(0.f, 0.f);
  uint4* out = reinterpret_cast<uint4*>(s.out) + static_cast<long long>(run.row) * (p.D / 8);
  uint64_t cos[4], sin[4];
  int stage = 0;
  bool fresh = true, good = false;
  for (int row = run.row; row < run.end; row += kStep, out += kStep * (p.D / 8)) {
    const bool live = row < s.rows && l.active;
    if (fresh && live) good = angles<TF32>(p, at, l, u, cos, sin);
    cp_async_wait<kQknStages - 2>();
    uint4 a = make_uint4(0, 0, 0, 0), b = a, c = a, d = a;
    if (live) {
      const uint32_t src = slot + stage * Ring::kStageBytes;
      a = lds16(src);
      b = lds16(src + kQknThreads * 16);
      c = lds16(src + kQknThreads * 32);
      d = lds16(src + kQknThreads * 48);
    }
    fetch((stage + kQknStages - 1) % kQknStages);
    Vals x, g, gx;
    unpack<INTER>(a, b, x);
    unpack<INTER>(c, d, g);
    if (l.turned) turn<true>(g, cos, sin);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      gx.a[j] = ptx::mul2(g.a[j], x.a[j]);
      gx.b[j] = ptx::mul2(g.b[j], x.b[j]);
    }
    const float r = rsqrtf(fmaf(row_sum<LPR>(dot(x, x)), p.inv_d, p.eps));
    // mean of (g w) (x r), times r^2: what dx loses of x
    const float m = row_sum<LPR>(dot(gx, w)) * p.inv_d * r * r * r;
    const uint64_t r2 = ptx::pack2(r, r), m2 = ptx::pack2(-m, -m);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (live && good) {
        dw.a[j] = ptx::fma2(gx.a[j], r2, dw.a[j]);
        dw.b[j] = ptx::fma2(gx.b[j], r2, dw.b[j]);
      }
      g.a[j] = ptx::fma2(x.a[j], m2, ptx::mul2(ptx::mul2(g.a[j], w.a[j]), r2));
      g.b[j] = ptx::fma2(x.b[j], m2, ptx::mul2(ptx::mul2(g.b[j], w.b[j]), r2));
    }
    if (live) {
      pack<INTER>(g, a, b);
      if (!good) {
        a = b = make_uint4(0, 0, 0, 0);
        if (u == 0) atomicCAS(p.status, kStatusOk, kStatusBadPos);
      }
      out[l.c0 / 8] = a;
      out[l.c1 / 8] = b;
    }
    fresh = at.next(p, s, kStep);
    stage = stage + 1 == kQknStages ? 0 : stage + 1;
  }
  cp_async_wait<0>();
  if (!p.partial) return;  // uniform over the grid
  // the block's sums, in a fixed order: lanes of a warp that have the same columns, then the warps
  float v[16];  // piece 0, piece 1
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ptx::unpack2(dw.a[j], v[INTER ? 4 * j : 2 * j], v[INTER ? 4 * j + 2 : 2 * j + 1]);
    ptx::unpack2(dw.b[j], v[INTER ? 4 * j + 1 : 8 + 2 * j], v[INTER ? 4 * j + 3 : 8 + 2 * j + 1]);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int off = 16; off >= LPR; off >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
  if ((threadIdx.x & 31) < LPR && l.active) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sums[threadIdx.x / 32][l.c0 + i] = v[i];
      sums[threadIdx.x / 32][l.c1 + i] = v[8 + i];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.D; c += kQknThreads) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < kQknThreads / 32; ++k) t += sums[k][c];
    p.partial[static_cast<size_t>(blockIdx.x) * p.D + c] = t;
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
    for (int b0 = first + warp; b0 < end; b0 += 32 * 16) {  // 16 blocks' sums are asked for before the first is added
      float t[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) t[i] = b0 + 32 * i < end ? p.partial[static_cast<size_t>(b0 + 32 * i) * p.D + c] : 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) v += t[i];
    }
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
