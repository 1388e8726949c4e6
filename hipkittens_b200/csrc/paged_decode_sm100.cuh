// Paged-KV GQA decode for sm_100a: one query token per sequence, KV cache in 16-token pages that are
// reached through a block table. The reference has no such kernel; the math is the forward's
// (kernels/attn/gqa/kernel.cpp:569-573 for L) applied to one query row that sees its whole context.
//
// Split-K layout: a CTA owns part of the context of one (sequence, kv head) and all G = H / H_KV query heads of that kv
// head, so every K/V byte of the context is read exactly once. Inside the CTA each of the 4 or 8 warps streams its own
// pages through a private cp.async ring of 16-byte copies; scores and the PV product run on mma.sync m16n8k16 (bf16,
// fp32 accumulate) with the G heads in the 16-row M dimension, which is far more than an HBM-bound kernel needs and keeps
// the CUDA cores free for address generation and the exponentials.
// The CTAs of one (sequence, kv head) are a cluster, which splits the context evenly whatever its length and merges the
// partial results through distributed shared memory: one launch, nothing in the workspace. Where that would leave the GPU
// to a few CTAs (decode_pick_shape), a CTA takes a chunk of 512 or 1024 consecutive tokens instead; contexts of one chunk
// are finished in place, longer ones leave per-chunk (O, m, l) partials in the workspace, which
// `paged_decode_combine_kernel` merges.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "dependent_launch.cuh"
#include "paged_decode_common.cuh"
#include "sm100_ptx.cuh"

namespace hk {

// grid = (max_splits, H_KV, S), or (cluster size, H_KV, S) in clusters along x; block = 32 W threads, dynamic smem =
// decode_smem_bytes(W).
template <int G, bool CLUSTER, int W, int D = kDecodeD, bool WINDOW = false>
__global__ void __launch_bounds__(W * 32, W == 8 ? 1 : 2) paged_decode_split_kernel(const DecodeParams p) {
  using namespace dec;
  using Ring = DecodeRing<D>;
  constexpr int kDecodeStages = Ring::kStages, kSlabBytes = Ring::kSlabBytes, kStageBytes = Ring::kStageBytes;
  constexpr int kRowBytes = D * 2, kChunks = D / 8;  // of a token: its bytes, and 16-byte chunks
  extern __shared__ __align__(128) uint8_t dsmem[];
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int split = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  // A length beyond what the block-table row can address is clamped to the row's capacity and reported; nothing
  // past the row is read.
  int ctx = p.ctx_lens[seq];
  if (ctx > p.max_pages * kPageTokens) {
    ctx = p.max_pages * kPageTokens;
    if (threadIdx.x == 0) atomicCAS(p.status, 0, kStatusBadLen);
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const LivePages live(ctx, WINDOW ? p.window : 1, WINDOW ? p.sinks : 0);
  const int total_pages = WINDOW ? live.total : (ctx + kPageTokens - 1) / kPageTokens;
  // This warp's pages: page_first, page_first + page_step, ... below page_end. A CTA of a cluster takes every n_used-th
  // group of W pages, so that whatever the length the live CTAs of a cluster differ by a page per warp at most.
  int n_used, page_first, page_step, page_end;
  if constexpr (CLUSTER) {
    if (ctx <= 0) {  // defined output for an empty context
      if (split == 0) {
        for (int i = threadIdx.x; i < G * D; i += W * 32)
          p.o[(size_t(seq) * p.H + kvh * G) * D + i] = __float2bfloat16(0.f);
        if (threadIdx.x < G) p.lse[size_t(seq) * p.H + kvh * G + threadIdx.x] = -INFINITY;
      }
      return;
    }
    n_used = min(static_cast<int>(gridDim.x), (total_pages + W - 1) / W);  // a page for every warp of a live CTA
    if (split >= n_used) return;  // the cluster's barriers count the threads that are left
    page_first = split * W + warp;
    page_step = n_used * W;
    page_end = total_pages;
  } else {
    if (WINDOW ? ctx <= 0 || split * p.chunk_pages >= total_pages : split * p.chunk_pages * kPageTokens >= ctx) return;
    n_used = 1;
    page_first = split * p.chunk_pages + warp;
    page_step = W;
    page_end = min(split * p.chunk_pages + p.chunk_pages, total_pages);
  }
  const float c = p.scale_log2;

  // page ids of this warp, one per lane: no warp has more than 32 pages (decode_pick_shape and the chunk sizes see to it).
  // With a window, 32 at a time; pages without a key that the query sees are not looked up.
  int my_id = 0;
  auto look_up = [&](int i0) {
    if (const int page = page_first + (i0 + lane) * page_step; page < page_end) {
      my_id = p.block_table[size_t(seq) * p.max_pages + (WINDOW ? live.page(page) : page)];
      if (my_id < 0 || my_id >= p.num_pages) {
        atomicCAS(p.status, 0, kStatusBadPage);  // never dereference an id outside the pool
        my_id = 0;
      }
    }
  };
  look_up(0);

  // Q fragments: row g = head kvh*G+g (rows >= G are zero), k-steps of 16 columns
  uint32_t qa[D / 16][2];
  {
    const __nv_bfloat16* qrow = p.q + (size_t(seq) * p.H + kvh * G + (g < G ? g : 0)) * D;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t lo = *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + 2 * t);
      uint32_t hi = *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + 8 + 2 * t);
      qa[ks][0] = (g < G) ? lo : 0u;
      qa[ks][1] = (g < G) ? hi : 0u;
    }
  }

  const uint32_t ring = ptx::smem_u32(dsmem) + warp * (kDecodeStages * kStageBytes);
  const size_t row_elems = size_t(p.H_KV) * D;  // elements between consecutive tokens of a page

  auto sees = [&](int key) { return key < ctx && (key >= live.first_key || key < p.sinks); };
  // 16-byte gather of one page of this kv head: lane copies chunks lane, lane+32, ... of the
  // chunks (16 tokens x D / 8 chunks) of K and of V; chunk index is XOR-swizzled with the token so that
  // ldmatrix reads are bank-conflict free.
  auto fetch = [&](int i) {
    if (page_first + i * page_step < page_end) {
      if (WINDOW && i > 0 && (i & 31) == 0) look_up(i);
      const int id = __shfl_sync(0xffffffffu, my_id, WINDOW ? i & 31 : i);
      const size_t base = (size_t(id) * kPageTokens) * row_elems + size_t(kvh) * D;
      const uint32_t st = ring + (i % kDecodeStages) * kStageBytes;
#pragma unroll
      for (int r = 0; r < kChunks / 2; ++r) {
        const int ch_lin = r * 32 + lane;
        const int tok = ch_lin / kChunks, ch = ch_lin % kChunks;
        const size_t src = base + size_t(tok) * row_elems + ch * 8;
        const uint32_t dst = tok * kRowBytes + ((ch ^ (tok & 7)) << 4);
        if constexpr (WINDOW) {
          // keys that the query does not see are not read, and are zeros: whatever the cache holds there meets p = 0
          const bool seen = sees(live.page(page_first + i * page_step) * kPageTokens + tok);
          cp_async16_if(st + dst, p.k_pages + src, seen);
          cp_async16_if(st + kSlabBytes + dst, p.v_pages + src, seen);
        } else {
          cp_async16(st + dst, p.k_pages + src);
          cp_async16(st + kSlabBytes + dst, p.v_pages + src);
        }
      }
    }
    cp_async_commit();
  };

  float oacc[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) oacc[j][0] = oacc[j][1] = oacc[j][2] = oacc[j][3] = 0.f;
  float m = -INFINITY, l = 0.f;

#pragma unroll
  for (int i = 0; i < kDecodeStages - 1; ++i) fetch(i);

  for (int i = 0, page = page_first; page < page_end; ++i, page += page_step) {
    fetch(i + kDecodeStages - 1);
    cp_async_wait<kDecodeStages - 1>();
    __syncwarp();
    const uint32_t sK = ring + (i % kDecodeStages) * kStageBytes;
    const uint32_t sV = sK + kSlabBytes;

    // ---- S[16 x 16 tokens] = Q K^T, in two halves of the head dimension: a warp has one page at a time, and with one
    // accumulator per 8 tokens the eight products on it wait for one another
    float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    {
      float sd[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      const int mi = lane >> 3, r = lane & 7;
      const int tok = r + 8 * (mi >> 1);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int ch = ks * 2 + (mi & 1);
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4(sK + tok * kRowBytes + ((ch ^ (tok & 7)) << 4), b0, b1, b2, b3);
        mma_16816(ks & 1 ? sd[0] : sc[0], qa[ks][0], 0u, qa[ks][1], 0u, b0, b1);
        mma_16816(ks & 1 ? sd[1] : sc[1], qa[ks][0], 0u, qa[ks][1], 0u, b2, b3);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sc[0][e] += sd[0][e];
        sc[1][e] += sd[1][e];
      }
    }
    // ---- online softmax over this page (row g, tokens nt*8 + 2t + {0,1})
    const int tok_base = (WINDOW ? live.page(page) : page) * kPageTokens;
    float sv[4] = {sc[0][0], sc[0][1], sc[1][0], sc[1][1]};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int tok = tok_base + (e >> 1) * 8 + 2 * t + (e & 1);
      if (WINDOW ? !sees(tok) : tok >= ctx) sv[e] = -INFINITY;
    }
    float pm = fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]));
    pm = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, 1));
    pm = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, 2));
    const float m_new = fmaxf(m, pm);
    if (__any_sync(0xffffffffu, (m_new - m) * c > kRescaleThresholdLog2)) {
      const float alpha = ptx::ex2_approx((m - m_new) * c);  // m = -inf on the first page gives 0
      l *= alpha;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        oacc[j][0] *= alpha;
        oacc[j][1] *= alpha;
      }
      m = m_new;
    }
    const float mc = m * c;
    float pv[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      pv[e] = ptx::ex2_approx(fmaf(sv[e], c, -mc));
      l += pv[e];
    }
    const uint32_t pa0 = ptx::pack_bf16x2(pv[0], pv[1]);
    const uint32_t pa2 = ptx::pack_bf16x2(pv[2], pv[3]);
    // ---- O[16 x 128] += P[16 x 16 tokens] V[16 tokens x 128]
    {
      const int mi = lane >> 3, r = lane & 7;
      const int tok = r + 8 * (mi & 1);
#pragma unroll
      for (int jp = 0; jp < D / 16; ++jp) {
        const int ch = jp * 2 + (mi >> 1);
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4_trans(sV + tok * kRowBytes + ((ch ^ (tok & 7)) << 4), b0, b1, b2, b3);
        mma_16816(oacc[2 * jp], pa0, 0u, pa2, 0u, b0, b1);
        mma_16816(oacc[2 * jp + 1], pa0, 0u, pa2, 0u, b2, b3);
      }
    }
    __syncwarp();
  }
  cp_async_wait<0>();
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);

  // ---- merge the W warps through shared memory (the ring is idle now)
  __syncthreads();
  float* sm_o = reinterpret_cast<float*>(dsmem);  // [W][8][D]
  float* sm_m = sm_o + W * 8 * D;                // [W][8]
  float* sm_l = sm_m + W * 8;                     // [W][8]
#pragma unroll
  for (int j = 0; j < D / 8; ++j) {
    float2 v2 = make_float2(oacc[j][0], oacc[j][1]);
    *reinterpret_cast<float2*>(sm_o + (warp * 8 + g) * D + j * 8 + 2 * t) = v2;
  }
  if (t == 0) {
    sm_m[warp * 8 + g] = m;
    sm_l[warp * 8 + g] = l;
  }
  __syncthreads();
  // D threads <-> D output columns; where there are more threads, each D of them take every kHalves-th head of the group
  constexpr int kHalves = W * 32 / D, kHeads = (G + kHalves - 1) / kHalves;
  const int d = threadIdx.x & (D - 1), h0 = threadIdx.x / D;
  // per head of this thread: reference maximum, row sum and this thread's column of the CTA's share
  float M[kHeads], L[kHeads], acc[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = min(i * kHalves + h0, G - 1);
    M[i] = sm_m[h];
#pragma unroll
    for (int w = 1; w < W; ++w) M[i] = fmaxf(M[i], sm_m[w * 8 + h]);
    acc[i] = L[i] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float wgt = ptx::ex2_approx((sm_m[w * 8 + h] - M[i]) * c);
      acc[i] += wgt * sm_o[(w * 8 + h) * D + d];
      L[i] += wgt * sm_l[w * 8 + h];
    }
  }
  if constexpr (CLUSTER) {
    if (n_used > 1) {
      // ---- merge the CTAs of the cluster: each leaves its share in its own shared memory, and CTA r reads all of
      // head r, r + n_used, ... in the order of the ranks
      float* cl_o = sm_l + W * 8;          // [G][D]
      float* cl_ml = cl_o + 8 * D;         // [G][2]
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        const int h = i * kHalves + h0;
        if (h >= G) break;
        cl_o[h * D + d] = acc[i];
        if (d == 0) {
          cl_ml[2 * h] = M[i];
          cl_ml[2 * h + 1] = L[i];
        }
      }
      ptx::cluster_arrive();
      ptx::cluster_wait();
      for (int h = split * kHalves + h0; h < G; h += n_used * kHalves) {
        float m_r[kMaxCluster], l_r[kMaxCluster], o_r[kMaxCluster];
        const uint32_t a_ml = ptx::smem_u32(cl_ml + 2 * h), a_o = ptx::smem_u32(cl_o + h * D + d);
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
          m_r[r] = -INFINITY;
          l_r[r] = o_r[r] = 0.f;
          if (r < n_used) {
            const uint32_t ml = ptx::map_to_rank(a_ml, r);
            m_r[r] = ptx::ld_cluster(ml);
            l_r[r] = ptx::ld_cluster(ml + 4);
            o_r[r] = ptx::ld_cluster(ptx::map_to_rank(a_o, r));
          }
        }
        float Mc = m_r[0];
#pragma unroll
        for (int r = 1; r < kMaxCluster; ++r) Mc = fmaxf(Mc, m_r[r]);
        float sum = 0.f, out = 0.f;
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
          const float wgt = ptx::ex2_approx((m_r[r] - Mc) * c);
          sum += wgt * l_r[r];
          out += wgt * o_r[r];
        }
        const size_t row = size_t(seq) * p.H + kvh * G + h;
        p.o[row * D + d] = __float2bfloat16(out / sum);
        if (d == 0) p.lse[row] = Mc * p.scale + __logf(sum);
      }
      ptx::cluster_arrive();  // nobody leaves while its shared memory is being read
      ptx::cluster_wait();
      return;
    }
  }
  const int n_splits = CLUSTER ? 1 : (total_pages + p.chunk_pages - 1) / p.chunk_pages;
  const int max_splits = decode_max_splits(WINDOW ? p.span_pages : p.max_pages);
  float* ws_o = reinterpret_cast<float*>(p.workspace);
  const size_t o_bytes = (size_t(p.S) * p.H * max_splits * D * sizeof(float) + 255) & ~size_t(255);
  float* ws_ml = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(p.workspace) + o_bytes);
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = i * kHalves + h0;
    if (h >= G) break;
    const size_t row = size_t(seq) * p.H + kvh * G + h;
    if (n_splits == 1) {
      p.o[row * D + d] = __float2bfloat16(acc[i] / L[i]);
      if (d == 0) p.lse[row] = M[i] * p.scale + __logf(L[i]);
    } else {
      const size_t slot = row * max_splits + split;
      ws_o[slot * D + d] = acc[i];
      if (d == 0) {
        ws_ml[slot * 2] = M[i];
        ws_ml[slot * 2 + 1] = L[i];
      }
    }
  }
}

// grid = (H, S), block = D threads (one per output column). Merges the per-chunk partials of
// sequences that span more than one chunk.
template <int D, bool WINDOW>
__global__ void __launch_bounds__(D) paged_decode_combine_kernel(const DecodeParams p) {
  ptx::grid_dep_wait();  // from here on the split grid has completed and its partials are visible
  ptx::grid_dep_launch();
  const int head = blockIdx.x, seq = blockIdx.y;
  const int ctx = min(p.ctx_lens[seq], p.max_pages * kPageTokens);  // clamped as in the split kernel, which reports it
  const int d = threadIdx.x;
  if (ctx <= 0) {  // defined output for an empty context
    p.o[(size_t(seq) * p.H + head) * D + d] = __float2bfloat16(0.f);
    if (d == 0) p.lse[size_t(seq) * p.H + head] = -INFINITY;
    return;
  }
  const int chunk_tokens = p.chunk_pages * kPageTokens;
  const int n_splits = WINDOW ? (LivePages(ctx, p.window, p.sinks).total + p.chunk_pages - 1) / p.chunk_pages
                              : (ctx + chunk_tokens - 1) / chunk_tokens;
  if (n_splits == 1) return;  // finished by the split kernel
  const int max_splits = decode_max_splits(WINDOW ? p.span_pages : p.max_pages);
  const float* ws_o = reinterpret_cast<const float*>(p.workspace);
  const size_t o_bytes = (size_t(p.S) * p.H * max_splits * D * sizeof(float) + 255) & ~size_t(255);
  const float* ws_ml = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(p.workspace) + o_bytes);
  const size_t slot0 = (size_t(seq) * p.H + head) * max_splits;
  __shared__ float s_w[kMaxCombineSplits];
  __shared__ float s_M, s_L;
  if (threadIdx.x < 32) {
    float M = -INFINITY;
    for (int i = threadIdx.x; i < n_splits; i += 32) M = fmaxf(M, ws_ml[(slot0 + i) * 2]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    float L = 0.f;
    for (int i = threadIdx.x; i < n_splits; i += 32) {
      const float w = ptx::ex2_approx((ws_ml[(slot0 + i) * 2] - M) * p.scale_log2);
      s_w[i] = w;
      L += w * ws_ml[(slot0 + i) * 2 + 1];
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
    if (threadIdx.x == 0) {
      s_M = M;
      s_L = L;
    }
  }
  __syncthreads();
  float acc = 0.f;
#pragma unroll 4
  for (int i = 0; i < n_splits; ++i) acc += s_w[i] * ws_o[(slot0 + i) * D + d];
  p.o[(size_t(seq) * p.H + head) * D + d] = __float2bfloat16(acc / s_L);
  if (d == 0) p.lse[size_t(seq) * p.H + head] = s_M * p.scale + __logf(s_L);
}

template <int G, bool CLUSTER, int W, int D, bool WINDOW>
cudaError_t prepare_decode_kernel() {
  auto* fn = paged_decode_split_kernel<G, CLUSTER, W, D, WINDOW>;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, decode_smem_bytes(W));
  if (e != cudaSuccess || !CLUSTER) return e;
  return cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}
template <int G>
cudaError_t prepare_decode_kernels_of() {
  cudaError_t e = prepare_decode_kernel<G, false, 4, kDecodeD, false>();
  if (e == cudaSuccess) e = prepare_decode_kernel<G, true, 4, kDecodeD, false>();
  if (e == cudaSuccess) e = prepare_decode_kernel<G, true, 8, kDecodeD, false>();
  return e;
}
template <int G>
cudaError_t prepare_window_kernels_of() {
  cudaError_t e = prepare_decode_kernel<G, false, 4, 128, true>();
  if (e == cudaSuccess) e = prepare_decode_kernel<G, true, 4, 128, true>();
  if (e == cudaSuccess) e = prepare_decode_kernel<G, true, 8, 128, true>();
  if (e == cudaSuccess) e = prepare_decode_kernel<G, false, 4, 64, true>();
  if (e == cudaSuccess) e = prepare_decode_kernel<G, true, 4, 64, true>();
  if (e == cudaSuccess) e = prepare_decode_kernel<G, true, 8, 64, true>();
  return e;
}
// Those of calls with a window; the sizes of their clusters that fit are the others'.
inline int prepare_window_decode_kernels(char* err, size_t err_len) {
  for (auto* prepare : {prepare_window_kernels_of<1>, prepare_window_kernels_of<2>, prepare_window_kernels_of<3>,
                        prepare_window_kernels_of<4>, prepare_window_kernels_of<5>, prepare_window_kernels_of<6>,
                        prepare_window_kernels_of<7>, prepare_window_kernels_of<8>}) {
    const cudaError_t e = prepare();
    if (e != cudaSuccess) {
      snprintf(err, err_len, "window decode kernel attribute: %s", cudaGetErrorString(e));
      return -3;
    }
  }
  return 0;
}
inline int prepare_decode_kernels(char* err, size_t err_len, int sm_count, DecodeLimits* lim) {
  for (auto* prepare : {prepare_decode_kernels_of<1>, prepare_decode_kernels_of<2>, prepare_decode_kernels_of<3>,
                        prepare_decode_kernels_of<4>, prepare_decode_kernels_of<5>, prepare_decode_kernels_of<6>,
                        prepare_decode_kernels_of<7>, prepare_decode_kernels_of<8>}) {
    const cudaError_t e = prepare();
    if (e != cudaSuccess) {
      snprintf(err, err_len, "decode kernel attribute: %s", cudaGetErrorString(e));
      return -3;
    }
  }
  lim->sm_count = sm_count;
  for (int n = 2; n <= kMaxCluster; ++n) lim->clusters4[n] = clusters_held(paged_decode_split_kernel<8, true, 4>, 4 * 32, decode_smem_bytes(4), n);
  lim->clusters8 = clusters_held(paged_decode_split_kernel<8, true, 8>, 8 * 32, decode_smem_bytes(8), kMaxCluster);
  return 0;
}

template <int G, int D, bool WINDOW>
cudaError_t launch_decode_split(const DecodeParams& p, int splits, int cluster, int warps, cudaStream_t stream) {
  const dim3 grid(cluster ? cluster : splits, p.H_KV, p.S);
  if (cluster == 0)
    return launch_dependent(true, paged_decode_split_kernel<G, false, 4, D, WINDOW>, grid, 128, decode_smem_bytes(4), stream, p);
  auto* fn = warps == 8 ? paged_decode_split_kernel<G, true, 8, D, WINDOW> : paged_decode_split_kernel<G, true, 4, D, WINDOW>;
  return launch_dependent(true, fn, grid, warps * 32, decode_smem_bytes(warps), stream, ClusterX{unsigned(cluster)}, p);
}

template <int D, bool WINDOW>
cudaError_t launch_decode_shape(DecodeParams p, DecodeShape shape, int pages, int sm_count, cudaStream_t stream, int* launched) {
  const int cluster = shape.cluster, warps = shape.warps;
  p.chunk_pages = decode_pick_chunk_pages(p.S, p.H_KV, pages, sm_count);
  const int splits = (pages + p.chunk_pages - 1) / p.chunk_pages;
  if (splits > kMaxCombineSplits) return cudaErrorInvalidValue;
  cudaError_t e;
  switch (p.H / p.H_KV) {
#define HK_CASE(g) \
  case g: e = launch_decode_split<g, D, WINDOW>(p, splits, cluster, warps, stream); break;
    HK_CASE(1) HK_CASE(2) HK_CASE(3) HK_CASE(4) HK_CASE(5) HK_CASE(6) HK_CASE(7) HK_CASE(8)
#undef HK_CASE
    default: return cudaErrorInvalidValue;
  }
  *launched += 1;
  if (e != cudaSuccess || cluster) return e;
  e = launch_dependent(true, paged_decode_combine_kernel<D, WINDOW>, dim3(p.H, p.S), D, 0, stream, p);
  *launched += 1;
  return e;
}

inline cudaError_t launch_paged_decode(const DecodeParams& p, const DecodeLimits& lim, cudaStream_t stream, int* launched) {
  const DecodeShape shape = decode_pick_shape(p.S, p.H_KV, p.max_pages, lim);
  return launch_decode_shape<kDecodeD, false>(p, shape, p.max_pages, lim.sm_count, stream, launched);
}
// With p.window, p.sinks and p.span_pages set.
inline cudaError_t launch_window_decode(const DecodeParams& p, int D, const DecodeLimits& lim, cudaStream_t stream,
                                        int* launched) {
  const DecodeShape shape = decode_pick_window_shape(p.S, p.H_KV, p.span_pages, lim);
  auto* launch = D == 64 ? launch_decode_shape<64, true> : launch_decode_shape<128, true>;
  return launch(p, shape, p.span_pages, lim.sm_count, stream, launched);
}

}  // namespace hk
