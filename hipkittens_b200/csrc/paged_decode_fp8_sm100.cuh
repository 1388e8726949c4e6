// Paged decode against a cache of e4m3 codes with a scale for each page and head (paged_kv_fp8_sm100.cuh): one query token per
// sequence, optionally with a window and sinks. O = softmax(scale q K^T) V and L as in the bf16 decode.
//
// Half the bytes of the bf16 cache in the same time need twice the work per byte, and the work is what this kernel is arranged for.
// With s_K and s_V the scales of a page, q K^T = s_K (q codes^T) is scaled once per score, and s_V goes into P; the codes themselves
// meet the tensor cores as they are, widened in registers:
//  * S^T = K Q^T (16 tokens x the up to 8 heads of the group) and O^T += V^T P^T: with the heads in the 8-wide dimension no row of an
//    `mma.sync` m16n8k16 is idle but those of heads that a group lacks; the heads as rows would take twice the products and
//    accumulators. P^T of one product is the B operand of the next after a transposition of its two 8 x 8 tiles (`movmatrix`).
//  * K in fp16: `cvt` widens pairs of codes exactly. q goes to fp16 over its own power of two (of its largest value), so that its
//    8 significant bits survive but for values below 2^-17 of that.
//  * V in bf16: an e4m3 code's exponent and mantissa moved behind its sign are the bf16 of 2^-120 times its value (subnormals
//    included). V's codes are fetched transposed in pairs of neighbouring columns, and the two halves of such a pair are two
//    shifts and masks apart, where `cvt` would first have to bring the tokens of one column together. bf16, because P takes the
//    page's scale with it, which may be anything: p s_V / r with r the largest s_V so far keeps 8 bits whatever the scales, as 2^112
//    times that; the accumulators are O / (2^-8 ...) in fp32 until the end.
// How a context is spread over warps, CTAs and clusters is the bf16 kernel's scheme (paged_decode_sm100.cuh), in CTAs of half the
// shared memory.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include "attn_fwd_sm100.cuh"
#include "paged_decode_common.cuh"
#include "paged_kv_fp8_sm100.cuh"

namespace hk {

template <int D>
struct DecodeFp8Ring {
  static constexpr int kStages = 3 * (128 / D);         // pages in flight per warp
  static constexpr int kRowBytes = D;
  static constexpr int kSlabBytes = kPageTokens * D;    // one page of one head: 2 KB at D = 128
  static constexpr int kStageBytes = 2 * kSlabBytes;    // K and V
};
// The ring of every warp, and a barrier for each stage.
__host__ __device__ constexpr int decode_fp8_ring_bytes(int warps) { return warps * DecodeFp8Ring<128>::kStages * DecodeFp8Ring<128>::kStageBytes; }
constexpr int decode_fp8_smem_bytes(int warps) { return decode_fp8_ring_bytes(warps) + warps * DecodeFp8Ring<64>::kStages * 8 + 8; }

struct DecodeFp8Params : DecodeParams {  // k_pages and v_pages are not used; a call without a window has one that hides nothing
  const float *k_scales, *v_scales;      // [P, H_KV]
};

namespace fp8 {

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t widen(uint32_t codes) {  // the low two codes, as fp16
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<unsigned short>(codes)));
  return h;
}
// Codes 0 and 2 of a word, and 1 and 3, as bf16 of 2^-120 times their values.
__device__ __forceinline__ uint32_t even_bf16(uint32_t x) { return ((x << 4) & 0x07f007f0u) | ((x << 8) & 0x80008000u); }
__device__ __forceinline__ uint32_t odd_bf16(uint32_t x) { return ((x >> 4) & 0x07f007f0u) | (x & 0x80008000u); }
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

}  // namespace fp8

// grid = (max_splits, H_KV, S), or (cluster size, H_KV, S) in clusters along x; block = 32 W threads, dynamic smem =
// decode_fp8_smem_bytes(W).
template <bool CLUSTER, int W, int D>
__global__ void __launch_bounds__(W * 32, 16 / W)
paged_decode_fp8_split_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                              const __grid_constant__ DecodeFp8Params p) {
  using namespace dec;
  using Ring = DecodeFp8Ring<D>;
  constexpr int kStages = Ring::kStages, kSlabBytes = Ring::kSlabBytes, kStageBytes = Ring::kStageBytes, kRowBytes = Ring::kRowBytes;
  constexpr int kChunks = D / 16;  // 16-byte chunks of a token, of 16 dimensions
  extern __shared__ __align__(1024) uint8_t dsmem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* const full = reinterpret_cast<uint64_t*>(dsmem + decode_fp8_ring_bytes(W)) + warp * kStages;
  uint32_t* const abort_word = reinterpret_cast<uint32_t*>(dsmem + decode_fp8_ring_bytes(W) + W * DecodeFp8Ring<64>::kStages * 8);
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) ptx::mbar_init(full + s, 1);
    if (warp == 0) *abort_word = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmap_k);
    ptx::prefetch_tmap(&tmap_v);
  }
  __syncthreads();
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int split = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const int G = p.H / p.H_KV;
  int ctx = p.ctx_lens[seq];
  if (ctx > p.max_pages * kPageTokens) {  // clamped to what the block table's row can address
    ctx = p.max_pages * kPageTokens;
    if (threadIdx.x == 0) atomicCAS(p.status, 0, kStatusBadLen);
  }
  const int g = lane >> 2, t = lane & 3;
  const LivePages live(ctx, p.window, p.sinks);
  // this warp's pages: page_first, page_first + page_step, ... below page_end, of the live ones
  int n_used, page_first, page_step, page_end;
  if constexpr (CLUSTER) {
    if (ctx <= 0) {  // defined output for an empty context
      if (split == 0) {
        for (int i = threadIdx.x; i < G * D; i += W * 32) p.o[(size_t(seq) * p.H + kvh * G) * D + i] = __float2bfloat16(0.f);
        if (threadIdx.x < G) p.lse[size_t(seq) * p.H + kvh * G + threadIdx.x] = -INFINITY;
      }
      return;
    }
    n_used = min(static_cast<int>(gridDim.x), (live.total + W - 1) / W);  // a page for every warp of a live CTA
    if (split >= n_used) return;  // the cluster's barriers count the threads that are left
    page_first = split * W + warp;
    page_step = n_used * W;
    page_end = live.total;
  } else {
    if (ctx <= 0 || split * p.chunk_pages >= live.total) return;
    n_used = 1;
    page_first = split * p.chunk_pages + warp;
    page_step = W;
    page_end = min(split * p.chunk_pages + p.chunk_pages, live.total);
  }
  const float c = p.scale_log2;

  // A lane has one of 32 pages at a time: its id, for the fetches, which run ahead, and its scales, for the products.
  int my_id = 0;
  float next_ks = 0.f, next_vs = 0.f;
  auto look_up = [&](int i0) {
    next_ks = next_vs = 0.f;
    if (const int page = page_first + (i0 + lane) * page_step; page < page_end) {
      my_id = p.block_table[size_t(seq) * p.max_pages + live.page(page)];
      if (my_id < 0 || my_id >= p.num_pages) {
        atomicCAS(p.status, 0, kStatusBadPage);  // never dereference an id outside the pool
        my_id = 0;
      }
      next_ks = p.k_scales[size_t(my_id) * p.H_KV + kvh];
      next_vs = p.v_scales[size_t(my_id) * p.H_KV + kvh];
    }
  };
  look_up(0);

  uint8_t* const ring = dsmem + warp * (kStages * kStageBytes);
  auto sees = [&](int key) { return key < ctx && (key >= live.first_key || key < p.sinks); };
  // A page's tokens of this head are one box of the pool, swizzled so that ldmatrix finds a chunk of 8 consecutive tokens in 8 different
  // groups of banks. All 16 come, whether the query sees them or not: masked scores do not look at K, and p = 0 meets a finite V, since
  // the products take no code for a NaN.
  auto fetch = [&](int i) {
    if (page_first + i * page_step < page_end) {
      if (i > 0 && (i & 31) == 0) look_up(i);
      const int id = __shfl_sync(0xffffffffu, my_id, i & 31);
      if (lane == 0) {
        uint64_t* const bar = full + i % kStages;
        uint8_t* const st = ring + (i % kStages) * kStageBytes;
        ptx::mbar_expect_tx(bar, kStageBytes);
        ptx::tma_load_3d(st, &tmap_k, bar, 0, kvh, id * kPageTokens);
        ptx::tma_load_3d(st + kSlabBytes, &tmap_v, bar, 0, kvh, id * kPageTokens);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);

  // Q^T as B operand: lane (g, t) has the values 16 c + 4 t ... + 3 of head g, which the products take as its four places of the sum
  // over the dimension; K's lanes have the same places.
  uint32_t qb[kChunks][2];
  float qs0, qs1;  // powers of two of heads 2 t and 2 t + 1
  {
    const uint2* const qrow = reinterpret_cast<const uint2*>(p.q + (size_t(seq) * p.H + kvh * G + (g < G ? g : 0)) * D) + t;
    uint2 x[kChunks];
    uint32_t two = 0;
#pragma unroll
    for (int ch = 0; ch < kChunks; ++ch) {
      x[ch] = g < G ? qrow[ch * 4] : make_uint2(0, 0);
      two = __vmaxu2(two, __vmaxu2(x[ch].x & 0x7fff7fffu, x[ch].y & 0x7fff7fffu));
    }
    uint32_t top = max(two & 0xffffu, two >> 16);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = min(max(static_cast<int>(top >> 7), 1), 253);  // the exponent as bf16 has it
    const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23), up = __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
    for (int ch = 0; ch < kChunks; ++ch) {
      const float2 lo = fp8::bf16x2(x[ch].x), hi = fp8::bf16x2(x[ch].y);
      const __half2 a = __floats2half2_rn(lo.x * down, lo.y * down), b = __floats2half2_rn(hi.x * down, hi.y * down);
      qb[ch][0] = *reinterpret_cast<const uint32_t*>(&a);
      qb[ch][1] = *reinterpret_cast<const uint32_t*>(&b);
    }
    qs0 = __shfl_sync(0xffffffffu, up, 8 * t);
    qs1 = __shfl_sync(0xffffffffu, up, 8 * t + 4);
  }

  float oacc[kChunks][4];  // O^T: dimensions 16 c + 2 g (0, 1) and 16 c + 2 g + 1 (2, 3), heads 2 t (0, 2) and 2 t + 1 (1, 3)
#pragma unroll
  for (int j = 0; j < kChunks; ++j) oacc[j][0] = oacc[j][1] = oacc[j][2] = oacc[j][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  float my_ks = 0.f, my_w = 0.f, most_vs = 0.f;
  const uint32_t ring_at = ptx::smem_u32(ring);
  // where this lane's row of ldmatrix begins: tokens 0-7 and 8-15, of a chunk and the one behind it
  const int row = (lane & 7) + ((lane >> 3) & 1) * 8;
  const uint32_t mine = row * kRowBytes + (((lane >> 4) ^ (D == 128 ? row & 7 : (row >> 1) & 3)) << 4);
  constexpr float kUp = 5192296858534827628530496329220096.f;  // 2^112

  for (int i = 0, page = page_first; page < page_end; ++i, page += page_step) {
    if ((i & 31) == 0) {
      my_ks = next_ks;
      float most = next_vs;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
      if (most > most_vs) {
        if (i > 0) {
          const float less = most_vs / most;
#pragma unroll
          for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) oacc[j][e] *= less;
        }
        most_vs = most;
      }
      my_w = most_vs > 0.f ? next_vs / most_vs * kUp : next_vs * kUp;  // all zero, or NaN
    }
    fetch(i + kStages - 1);
    if (!__all_sync(0xffffffffu, ptx::mbar_wait(full + i % kStages, (i / kStages) & 1, abort_word, kWaitLimitCycles))) break;
    const uint32_t sK = ring_at + (i % kStages) * kStageBytes, sV = sK + kSlabBytes;
    const float ks = __shfl_sync(0xffffffffu, my_ks, i & 31), wv = __shfl_sync(0xffffffffu, my_w, i & 31);

    // ---- S^T[16 tokens x 8 heads] = K Q^T, even and odd chunks apart: one accumulator's products wait for one another
    float sc[4] = {0.f, 0.f, 0.f, 0.f}, sd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ch = 0; ch < kChunks; ch += 2) {
      uint32_t r0, r1, r2, r3;
      ldmatrix_x4((sK + mine) ^ (ch << 4), r0, r1, r2, r3);
      fp8::mma_f16(sc, fp8::widen(r0), fp8::widen(r1), fp8::widen(r0 >> 16), fp8::widen(r1 >> 16), qb[ch][0], qb[ch][1]);
      fp8::mma_f16(sd, fp8::widen(r2), fp8::widen(r3), fp8::widen(r2 >> 16), fp8::widen(r3 >> 16), qb[ch + 1][0], qb[ch + 1][1]);
    }
    const float f0 = ks * qs0, f1 = ks * qs1;
    float sv[4] = {(sc[0] + sd[0]) * f0, (sc[1] + sd[1]) * f1, (sc[2] + sd[2]) * f0, (sc[3] + sd[3]) * f1};
    // ---- online softmax over tokens g and g + 8 of this page, heads 2 t and 2 t + 1
    const int key = live.page(page) * kPageTokens;
    if (key + kPageTokens > ctx || (key < live.first_key && key + kPageTokens > p.sinks)) {  // a page that is not seen whole
      if (!sees(key + g)) sv[0] = sv[1] = -INFINITY;
      if (!sees(key + g + 8)) sv[2] = sv[3] = -INFINITY;
    }
    // The maximum is looked for only where some score is far above the one that the head has (the first page's is -inf)
    float pm0 = fmaxf(sv[0], sv[2]), pm1 = fmaxf(sv[1], sv[3]);
    if (__any_sync(0xffffffffu, (pm0 - m0) * c > kRescaleThresholdLog2 || (pm1 - m1) * c > kRescaleThresholdLog2)) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        pm0 = fmaxf(pm0, __shfl_xor_sync(0xffffffffu, pm0, off));
        pm1 = fmaxf(pm1, __shfl_xor_sync(0xffffffffu, pm1, off));
      }
      const float n0 = fmaxf(m0, pm0), n1 = fmaxf(m1, pm1);
      const float alpha0 = n0 == m0 ? 1.f : ptx::ex2_approx((m0 - n0) * c), alpha1 = n1 == m1 ? 1.f : ptx::ex2_approx((m1 - n1) * c);
      l0 *= alpha0, l1 *= alpha1;
#pragma unroll
      for (int j = 0; j < kChunks; ++j) oacc[j][0] *= alpha0, oacc[j][1] *= alpha1, oacc[j][2] *= alpha0, oacc[j][3] *= alpha1;
      m0 = n0, m1 = n1;
    }
    const float mc0 = m0 * c, mc1 = m1 * c;
    const float p0 = ptx::ex2_approx(fmaf(sv[0], c, -mc0)), p1 = ptx::ex2_approx(fmaf(sv[1], c, -mc1)),
                p2 = ptx::ex2_approx(fmaf(sv[2], c, -mc0)), p3 = ptx::ex2_approx(fmaf(sv[3], c, -mc1));
    l0 += p0 + p2, l1 += p1 + p3;
    const uint32_t b0 = fp8::transpose8x8(ptx::pack_bf16x2(p0 * wv, p1 * wv)), b1 = fp8::transpose8x8(ptx::pack_bf16x2(p2 * wv, p3 * wv));
    // ---- O^T[D x 8 heads] += V^T[D x 16 tokens] P^T
#pragma unroll
    for (int ch = 0; ch < kChunks; ch += 2) {
      uint32_t r0, r1, r2, r3;
      ldmatrix_x4_trans((sV + mine) ^ (ch << 4), r0, r1, r2, r3);
      mma_16816(oacc[ch], fp8::even_bf16(r0), fp8::odd_bf16(r0), fp8::even_bf16(r1), fp8::odd_bf16(r1), b0, b1);
      mma_16816(oacc[ch + 1], fp8::even_bf16(r2), fp8::odd_bf16(r2), fp8::even_bf16(r3), fp8::odd_bf16(r3), b0, b1);
    }
    __syncwarp();
  }
  __syncthreads();  // the ring is idle now, or a wait has run out
  if (*static_cast<volatile uint32_t*>(abort_word) != 0) {
    // copies that are still in flight get time to land before the shared memory goes away
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 2000000ull) {
    }
    if (threadIdx.x == 0) atomicCAS(p.status, kStatusOk, kStatusTimeout);
  }
#pragma unroll
  for (int off = 4; off < 32; off <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, off);
    l1 += __shfl_xor_sync(0xffffffffu, l1, off);
  }

  // ---- merge the W warps through shared memory
  float* sm_o = reinterpret_cast<float*>(dsmem);  // [W][8][D]
  float* sm_m = sm_o + W * 8 * D;                // [W][8]
  float* sm_l = sm_m + W * 8;                     // [W][8]
  const float out_scale = most_vs > 0.f ? most_vs * 256.f : 256.f;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    float* const dst = sm_o + (warp * 8 + 2 * t) * D + j * 16 + 2 * g;
    *reinterpret_cast<float2*>(dst) = make_float2(oacc[j][0] * out_scale, oacc[j][2] * out_scale);
    *reinterpret_cast<float2*>(dst + D) = make_float2(oacc[j][1] * out_scale, oacc[j][3] * out_scale);
  }
  if (g == 0) {
    sm_m[warp * 8 + 2 * t] = m0, sm_m[warp * 8 + 2 * t + 1] = m1;
    sm_l[warp * 8 + 2 * t] = l0, sm_l[warp * 8 + 2 * t + 1] = l1;
  }
  __syncthreads();
  // D threads <-> D output columns; where there are more threads, each D of them take every kHalves-th head of the group
  constexpr int kHalves = W * 32 / D, kHeads = 8 / kHalves;
  const int d = threadIdx.x & (D - 1), h0 = threadIdx.x / D;
  float M[kHeads], L[kHeads], acc[kHeads];  // per head of this thread: maximum, row sum and this thread's column of the CTA's share
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = i * kHalves + h0;
    M[i] = L[i] = acc[i] = 0.f;
    if (h >= G) break;
    M[i] = sm_m[h];
#pragma unroll
    for (int w = 1; w < W; ++w) M[i] = fmaxf(M[i], sm_m[w * 8 + h]);
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
      float* cl_o = sm_l + W * 8;          // [8][D]
      float* cl_ml = cl_o + 8 * D;         // [8][2]
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        const int h = i * kHalves + h0;
        if (h >= G) break;
        cl_o[h * D + d] = acc[i];
        if (d == 0) cl_ml[2 * h] = M[i], cl_ml[2 * h + 1] = L[i];
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
  const int n_splits = CLUSTER ? 1 : (live.total + p.chunk_pages - 1) / p.chunk_pages;
  const int max_splits = decode_max_splits(p.span_pages);
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
      if (d == 0) ws_ml[slot * 2] = M[i], ws_ml[slot * 2 + 1] = L[i];
    }
  }
}

template <bool CLUSTER, int W, int D>
cudaError_t prepare_decode_fp8_kernel() {
  auto* fn = paged_decode_fp8_split_kernel<CLUSTER, W, D>;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, decode_fp8_smem_bytes(W));
  if (e != cudaSuccess || !CLUSTER) return e;
  return cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}
inline int prepare_decode_fp8_kernels(char* err, size_t err_len, int sm_count, DecodeLimits* lim) {
  for (auto* prepare : {prepare_decode_fp8_kernel<false, 4, 128>, prepare_decode_fp8_kernel<true, 4, 128>,
                        prepare_decode_fp8_kernel<true, 8, 128>, prepare_decode_fp8_kernel<false, 4, 64>,
                        prepare_decode_fp8_kernel<true, 4, 64>, prepare_decode_fp8_kernel<true, 8, 64>}) {
    const cudaError_t e = prepare();
    if (e != cudaSuccess) {
      snprintf(err, err_len, "fp8 decode kernel attribute: %s", cudaGetErrorString(e));
      return -3;
    }
  }
  lim->sm_count = sm_count;
  for (int n = 2; n <= kMaxCluster; ++n)
    lim->clusters4[n] = clusters_held(paged_decode_fp8_split_kernel<true, 4, 128>, 4 * 32, decode_fp8_smem_bytes(4), n);
  lim->clusters8 = clusters_held(paged_decode_fp8_split_kernel<true, 8, 128>, 8 * 32, decode_fp8_smem_bytes(8), kMaxCluster);
  return 0;
}

inline DecodeShape decode_pick_fp8_shape(int S, int H_KV, int span, const DecodeLimits& lim) {
  return decode_pick_window_shape(S, H_KV, span, lim);
}

template <int D>
cudaError_t launch_decode_fp8(const CUtensorMap& tk, const CUtensorMap& tv, DecodeFp8Params p, DecodeShape shape, int chunk_pages,
                              cudaStream_t stream, int* launched) {
  p.chunk_pages = chunk_pages;
  const int splits = (p.span_pages + p.chunk_pages - 1) / p.chunk_pages;
  if (splits > kMaxCombineSplits) return cudaErrorInvalidValue;
  const dim3 grid(shape.cluster ? shape.cluster : splits, p.H_KV, p.S);
  cudaError_t e;
  if (shape.cluster == 0) {
    e = launch_dependent(true, paged_decode_fp8_split_kernel<false, 4, D>, grid, 128, decode_fp8_smem_bytes(4), stream, tk, tv, p);
  } else {
    auto* fn = shape.warps == 8 ? paged_decode_fp8_split_kernel<true, 8, D> : paged_decode_fp8_split_kernel<true, 4, D>;
    e = launch_dependent(true, fn, grid, shape.warps * 32, decode_fp8_smem_bytes(shape.warps), stream,
                         ClusterX{unsigned(shape.cluster)}, tk, tv, p);
  }
  *launched += 1;
  if (e != cudaSuccess || shape.cluster) return e;
  e = launch_window_combine(p, D, stream);
  *launched += 1;
  return e;
}

inline cudaError_t launch_paged_decode_fp8(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeFp8Params& p, int D, const DecodeLimits& lim, cudaStream_t stream,
                                           int* launched) {
  const DecodeShape shape = decode_pick_fp8_shape(p.S, p.H_KV, p.span_pages, lim);
  const int chunk_pages = decode_pick_chunk_pages(p.S, p.H_KV, p.span_pages, lim.sm_count);
  return (D == 64 ? launch_decode_fp8<64> : launch_decode_fp8<128>)(tk, tv, p, shape, chunk_pages, stream, launched);
}

}  // namespace hk
