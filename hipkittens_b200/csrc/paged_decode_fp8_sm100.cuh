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
//    shifts and masks apart, where `cvt` would first have to bring the tokens of one column together. A code that is NaN comes out as 480 and
//    is found beside that, by the largest size of a page's codes (one context of 12,006 tokens 0.6 of 15 us). bf16, because P takes the
//    page's scale with it, which may be anything: p s_V / r, with r the unit's largest s_V so far, keeps 8 bits whatever
//    the scales, as 2^117 times that, and the accumulators are 2^-3 O l / r in fp32 until the end. (What is 2^-146 of r is their smallest
//    step: values so far below the largest that the same query sees are lost, and no others.)
// How contexts are spread (decode_pick_fp8_cluster): with few (sequence, K/V head) units a cluster of CTAs shares each, as in the bf16 kernel
// (paged_decode_common.cuh). Otherwise the pages of all units are one row of work, of which every warp of the GPU takes an equal run,
// whatever the contexts' lengths, and a second kernel joins the units that more than one warp had a part of.
// Bound by HBM where contexts are many: 64 of 512 to 8192 tokens, H64/8 D128, in a loop 70 us, 71% of the copy rate; the row kernel
// takes 63 of them and is at 94% of it for equal contexts, the join the rest. One context of 12,006 tokens (H32/8) 14.7 us, of which its 25
// MB are 3.8: a launch, three dependent loads and the cluster's barriers are the rest. At D = 64 a TMA row is 64 bytes and their rate the bound.
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
constexpr int kFp8Warps = 4;  // of a CTA, of which an SM holds four
// Dynamic shared memory: the ring of every warp, a barrier for each stage, a word that says that a wait has run out.
constexpr int kFp8RingBytes = kFp8Warps * DecodeFp8Ring<128>::kStages * DecodeFp8Ring<128>::kStageBytes;
constexpr int kFp8SmemBytes = kFp8RingBytes + kFp8Warps * DecodeFp8Ring<64>::kStages * 8 + 8;

struct DecodeFp8Params : DecodeParams {  // k_pages and v_pages are not used; a call without a window has one that hides nothing
  const float *k_scales, *v_scales;      // [P, H_KV]
  int row_groups;                        // groups of H_KV warps that share the row of all pages
};
// A warp leaves at most two parts of units that it does not have whole: its first and its last. Workspace: their O as fp32 [part][8][D], then
// (m, l) pairs [part][8][2], l negative where O is 2^-64 times what it is, then for each unit which parts it has (DecodeFp8Parts).
constexpr int kRowWarps = 16 * 148;  // what a B200 holds at once
// No warp takes fewer pages, unless there are no more: what it leaves has to be joined. us, 2 / 4 / 8 / 16, a read of 256 MB before each: one
// context of 100,000 tokens H8/1 D128 44 / 38 / 30 / 30, of 40,000 30 / 24 / 22 / 28, of H32/8 30 / 30 / 30 / 32.
constexpr int kRowPages = 8;
inline int decode_fp8_row_groups(int H_KV, int warps = kRowWarps) { return H_KV < warps ? warps / H_KV : 1; }
struct __align__(16) DecodeFp8Parts {
  int first, group, last_group, unused;  // the part of its first group, that group and the last one; the same: none, the rows are finished
};
// Whether these lie in the workspace. The row kernel leaves them for every context that is not empty, unless a wait of its has run out: then
// the join finds whatever was there before.
__host__ __device__ inline bool decode_fp8_parts_valid(const DecodeFp8Parts& x, int row_groups, int H_KV) {
  return x.group >= 0 && x.group <= x.last_group && x.last_group < row_groups && x.first >= 0 && x.first < 2 * row_groups * H_KV;
}
inline size_t decode_fp8_workspace_bytes(int S, int H_KV, int D) {
  return size_t(decode_fp8_row_groups(H_KV)) * H_KV * 2 * 8 * (D + 2) * sizeof(float) + size_t(S) * H_KV * sizeof(DecodeFp8Parts);
}

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
// Codes 0 and 2 of a word, and 1 and 3, as bf16 of 2^-120 times their values, NaN as that of 480. `top` is the largest size so far of each
// half of the words: 0x07f0 for a NaN and below that for numbers.
struct Bf16Codes {
  uint32_t even, odd;
  __device__ __forceinline__ Bf16Codes(uint32_t x, uint32_t& top) {
    const uint32_t e = (x << 4) & 0x07f007f0u, o = (x >> 4) & 0x07f007f0u;
    top = __vimax3_u16x2(top, e, o);
    even = e | ((x << 8) & 0x80008000u);
    odd = o | (x & 0x80008000u);
  }
};
__device__ __forceinline__ bool has_nan(uint32_t top) { return ((top + 0x00100010u) & 0x08000800u) != 0; }
// The high bit of each code that is NaN.
__device__ __forceinline__ uint32_t nan_codes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// The largest number for what is above it (and above zero), so that a score of zero is one; NaN stays.
__device__ __forceinline__ float finite(float x) {
  float y;
  asm("min.NaN.f32 %0, %1, 0f7F7FFFFF;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

}  // namespace fp8

constexpr float kHugeScale = 0x1p-64f;

// One warp's state: its ring, up to 32 pages that are looked up ahead, and the attention of a unit's heads over the pages so far.
template <int D>
struct DecodeFp8Warp {
  using Ring = DecodeFp8Ring<D>;
  static constexpr int kChunks = D / 16;  // 16-byte chunks of a token, of 16 dimensions
  // bits beside a page's 16 for the tokens that the query sees: it is the unit's first page, or its last
  enum : uint32_t { kAll = 0xffffu, kBegins = 1u << 16, kEnds = 1u << 17 };

  const DecodeFp8Params& p;
  const CUtensorMap &tmap_k, &tmap_v;
  uint8_t* ring;
  uint64_t* full;
  volatile uint32_t* abort_word;
  int lane, g, t;
  uint32_t ring_at, mine;
  // a lane's page of those that are fetched, and what the products will need of it
  int my_id = 0, next_unit = 0;
  float next_ks = 0.f, next_vs = 0.f;
  uint32_t next_seen = 0;
  // ... of those that are worked on
  int my_unit = 0;
  float my_ks = 0.f, my_vs = 0.f;
  uint32_t my_seen = 0;
  float ref = 0.f;  // r of the unit; 0: it has no pages yet
  // Q^T as B operand: lane (g, t) has the values 16 c + 4 t ... + 3 of head g, which the products take as its four places of the sum
  // over the dimension; K's lanes have the same places
  uint32_t qb[kChunks][2];
  float qs0, qs1;          // powers of two of heads 2 t and 2 t + 1
  float oacc[kChunks][4];  // O^T: dimensions 16 c + 2 g (0, 1) and 16 c + 2 g + 1 (2, 3), heads 2 t (0, 2) and 2 t + 1 (1, 3)
  float m0, m1, l0, l1;

  __device__ __forceinline__ DecodeFp8Warp(const DecodeFp8Params& params, const CUtensorMap& k, const CUtensorMap& v, uint8_t* smem)
      : p(params), tmap_k(k), tmap_v(v) {
    const int warp = threadIdx.x >> 5;
    lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    ring = smem + warp * (Ring::kStages * Ring::kStageBytes);
    ring_at = ptx::smem_u32(ring);
    full = reinterpret_cast<uint64_t*>(smem + kFp8RingBytes) + warp * Ring::kStages;
    abort_word = reinterpret_cast<uint32_t*>(smem + kFp8SmemBytes - 8);
    // where this lane's row of ldmatrix begins: tokens 0-7 and 8-15, of a chunk and the one behind it
    const int row = (lane & 7) + ((lane >> 3) & 1) * 8;
    mine = row * Ring::kRowBytes + (((lane >> 4) ^ (D == 128 ? row & 7 : (row >> 1) & 3)) << 4);
    if (lane == 0) {
      for (int s = 0; s < Ring::kStages; ++s) ptx::mbar_init(full + s, 1);
      if (warp == 0) *abort_word = 0;
      ptx::fence_mbar_init();
      ptx::prefetch_tmap(&tmap_k);
      ptx::prefetch_tmap(&tmap_v);
    }
  }

  // This lane's page: the `page`-th live one of a sequence.
  __device__ __forceinline__ void look_up(int seq, int ctx, int page, int head, uint32_t ends) {
    const LivePages live(ctx, p.window, p.sinks);
    const int at = live.page(page), key = at * kPageTokens;
    my_id = p.block_table[size_t(seq) * p.max_pages + at];
    if (my_id < 0 || my_id >= p.num_pages) {
      atomicCAS(p.status, 0, kStatusBadPage);  // never dereference an id outside the pool
      my_id = 0;
    }
    next_ks = p.k_scales[size_t(my_id) * p.H_KV + head];
    next_vs = p.v_scales[size_t(my_id) * p.H_KV + head];
    next_seen = seen_bits(key, live.first_key, ctx - 1, min(p.sinks, ctx)) & kAll | ends;
    next_unit = seq * p.H_KV + head;
  }
  __device__ __forceinline__ void look_up_none() { next_ks = next_vs = 0.f; }

  // What is fetched is read once: it goes first when L2 needs room, so that the parts of units stay there until they are joined (64 contexts of
  // 512 to 8192 tokens H64/8 D128 in a loop 80.1 / 75.1 us).
  // A page's tokens of a head are one box of the pool, swizzled so that ldmatrix finds a chunk of 8 consecutive tokens in 8 different
  // groups of banks. All 16 come, whether the query sees them or not: masked scores do not look at K, and p = 0 meets a finite V, since
  // the products take no code for a NaN (add_nans has those of tokens that the query sees).
  __device__ __forceinline__ void fetch(int i, int head) {
    const int id = __shfl_sync(0xffffffffu, my_id, i & 31);
    if (lane == 0) {
      uint64_t* const bar = full + i % Ring::kStages;
      uint8_t* const st = ring + (i % Ring::kStages) * Ring::kStageBytes;
      ptx::mbar_expect_tx(bar, Ring::kStageBytes);
      ptx::tma_load_3d_once(st, &tmap_k, bar, 0, head, id * kPageTokens);
      ptx::tma_load_3d_once(st + Ring::kSlabBytes, &tmap_v, bar, 0, head, id * kPageTokens);
    }
  }

  __device__ __forceinline__ void begin_unit(int unit, int G) {
    const uint2* const qrow = reinterpret_cast<const uint2*>(p.q + (size_t(unit) * G + (g < G ? g : 0)) * D) + t;
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
#pragma unroll
    for (int j = 0; j < kChunks; ++j) oacc[j][0] = oacc[j][1] = oacc[j][2] = oacc[j][3] = 0.f;
    m0 = m1 = -INFINITY, l0 = l1 = 0.f;
    ref = 0.f;
  }

  // The pages looked up last are those that are worked on from here.
  __device__ __forceinline__ void take_pages() { my_ks = next_ks, my_vs = next_vs, my_seen = next_seen, my_unit = next_unit; }
  // r, where a unit begins or goes on to these pages, and what P takes of each of them: 2^117 s_V / r. Of pages of other units nothing is
  // taken. r is a number, and 2^-10 at least, so that 2^117 / r is one.
  __device__ __forceinline__ void refer(int unit) {
    constexpr float kUp = 0x1p117f;
    const uint32_t vs = __float_as_uint(my_vs);
    const uint32_t most = __reduce_max_sync(0xffffffffu, my_unit == unit && vs <= 0x7f800000u ? min(max(vs, 117u << 23), 0x7f7fffffu) : 117u << 23);
    const float to = fmaxf(ref, __uint_as_float(most));
    if (ref != 0.f && to > ref) {
      const float less = ref / to;
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) oacc[j][e] *= less;
    }
    ref = to;
    if (my_unit == unit) my_vs *= kUp / to;
  }
  __device__ __forceinline__ uint32_t seen_of(int i) const { return __shfl_sync(0xffffffffu, my_seen, i & 31); }

  // V has codes that are NaN on this page: columns where a token that the query sees has one become NaN, for all heads.
  __device__ __noinline__ static uint32_t nan_columns(uint32_t v_at, uint32_t seen) {
    const int t = threadIdx.x & 3;
    auto of = [&](int token) { return (seen >> token & 1 ? 0x8080u : 0u) | (seen >> (token + 1) & 1 ? 0x80800000u : 0u); };
    const uint32_t low = of(2 * t), high = of(2 * t + 8);
    uint32_t columns = 0;  // bits 2 c and 2 c + 1: the lane's two columns of chunk c
    auto note = [&](int ch, uint32_t codes) {
      columns |= (codes & 0x00800080u ? 1u : 0u) << 2 * ch | (codes & 0x80008000u ? 2u : 0u) << 2 * ch;
    };
    for (int ch = 0; ch < kChunks; ch += 2) {
      uint32_t r0, r1, r2, r3;
      dec::ldmatrix_x4_trans(v_at ^ (ch << 4), r0, r1, r2, r3);
      note(ch, (fp8::nan_codes(r0) & low) | (fp8::nan_codes(r1) & high));
      note(ch + 1, (fp8::nan_codes(r2) & low) | (fp8::nan_codes(r3) & high));
    }
    columns |= __shfl_xor_sync(0xffffffffu, columns, 1);
    return columns | __shfl_xor_sync(0xffffffffu, columns, 2);
  }
  __device__ __forceinline__ void add_nans(uint32_t sV, uint32_t seen) {
    const uint32_t columns = nan_columns(sV + mine, seen);
#pragma unroll
    for (int ch = 0; ch < kChunks; ++ch) {
      if (columns >> 2 * ch & 1) oacc[ch][0] = oacc[ch][1] = __int_as_float(0x7fffffff);
      if (columns >> 2 * ch & 2) oacc[ch][2] = oacc[ch][3] = __int_as_float(0x7fffffff);
    }
  }

  // Page i, which has been fetched. False: the wait for it has run out.
  __device__ __forceinline__ bool page(int i, uint32_t seen) {
    using namespace dec;
    if (!__all_sync(0xffffffffu, ptx::mbar_wait(full + i % Ring::kStages, (i / Ring::kStages) & 1, abort_word, kWaitLimitCycles))) return false;
    const uint32_t sK = ring_at + (i % Ring::kStages) * Ring::kStageBytes, sV = sK + Ring::kSlabBytes;
    const float ks = __shfl_sync(0xffffffffu, my_ks, i & 31), wv = __shfl_sync(0xffffffffu, my_vs, i & 31);
    const float c = p.scale_log2;
    // ---- S^T[16 tokens x 8 heads] = K Q^T, even and odd chunks apart: one accumulator's products wait for one another
    float sc[4] = {0.f, 0.f, 0.f, 0.f}, sd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ch = 0; ch < kChunks; ch += 2) {
      uint32_t r0, r1, r2, r3;
      ldmatrix_x4((sK + mine) ^ (ch << 4), r0, r1, r2, r3);
      fp8::mma_f16(sc, fp8::widen(r0), fp8::widen(r1), fp8::widen(r0 >> 16), fp8::widen(r1 >> 16), qb[ch][0], qb[ch][1]);
      fp8::mma_f16(sd, fp8::widen(r2), fp8::widen(r3), fp8::widen(r2 >> 16), fp8::widen(r3 >> 16), qb[ch + 1][0], qb[ch + 1][1]);
    }
    const float f0 = fp8::finite(ks * qs0), f1 = fp8::finite(ks * qs1);
    float sv[4] = {(sc[0] + sd[0]) * f0, (sc[1] + sd[1]) * f1, (sc[2] + sd[2]) * f0, (sc[3] + sd[3]) * f1};
    // ---- online softmax over tokens g and g + 8 of this page, heads 2 t and 2 t + 1
    if ((seen & kAll) != kAll) {
      if (!(seen >> g & 1)) sv[0] = sv[1] = -INFINITY;
      if (!(seen >> (g + 8) & 1)) sv[2] = sv[3] = -INFINITY;
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
    uint32_t top = 0;
#pragma unroll
    for (int ch = 0; ch < kChunks; ch += 2) {
      uint32_t r0, r1, r2, r3;
      ldmatrix_x4_trans((sV + mine) ^ (ch << 4), r0, r1, r2, r3);
      const fp8::Bf16Codes v0(r0, top), v1(r1, top), v2(r2, top), v3(r3, top);
      mma_16816(oacc[ch], v0.even, v0.odd, v1.even, v1.odd, b0, b1);
      mma_16816(oacc[ch + 1], v2.even, v2.odd, v3.even, v3.odd, b0, b1);
    }
    if (__any_sync(0xffffffffu, fp8::has_nan(top))) add_nans(sV, seen);
    __syncwarp();
    return true;
  }

  // Row sums over all tokens.
  __device__ __forceinline__ void end_unit() {
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, off);
      l1 += __shfl_xor_sync(0xffffffffu, l1, off);
    }
  }
  // What O^T is times. The sum of values near the end of fp32, as an infinity that was appended leaves one (448 x 2^119), is no number:
  // those are 2^-64 of theirs, and who adds them up to others takes these times 2^-64 too.
  __device__ __forceinline__ bool is_huge() const { return ref >= 1.f / kHugeScale; }
  __device__ __forceinline__ float sum_scale(bool huge) const { return ref * (huge ? 8.f * kHugeScale : 8.f); }
};

// Where a wait has run out, the status says so, and copies that are still in flight get time to land before the shared memory goes away.
// Returns whether `flag` holds for any thread of the CTA.
__device__ __forceinline__ bool decode_fp8_check_waits(const volatile uint32_t* abort_word, int* status, bool flag = false) {
  flag = __syncthreads_or(flag);
  if (*abort_word != 0) {
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 2000000ull) {
    }
    if (threadIdx.x == 0) atomicCAS(status, kStatusOk, kStatusTimeout);
  }
  return flag;
}

// grid = (cluster size, H_KV, S) in clusters along x; block = 128, dynamic smem = kFp8SmemBytes.
template <int D>
__global__ void __launch_bounds__(kFp8Warps * 32, 4)
paged_decode_fp8_cluster_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                                const __grid_constant__ DecodeFp8Params p) {
  using Warp = DecodeFp8Warp<D>;
  constexpr int kStages = DecodeFp8Ring<D>::kStages, W = kFp8Warps;
  extern __shared__ __align__(1024) uint8_t dsmem[];
  Warp a(p, tmap_k, tmap_v, dsmem);
  __syncthreads();
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int split = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z, warp = threadIdx.x >> 5;
  const int G = p.H / p.H_KV;
  int ctx = p.ctx_lens[seq];
  if (ctx > p.max_pages * kPageTokens) {  // clamped to what the block table's row can address
    ctx = p.max_pages * kPageTokens;
    if (threadIdx.x == 0) atomicCAS(p.status, 0, kStatusBadLen);
  }
  if (ctx <= 0) {  // defined output for an empty context
    if (split == 0) {
      for (int i = threadIdx.x; i < G * D; i += W * 32) p.o[(size_t(seq) * p.H + kvh * G) * D + i] = __float2bfloat16(0.f);
      if (threadIdx.x < G) p.lse[size_t(seq) * p.H + kvh * G + threadIdx.x] = -INFINITY;
    }
    return;
  }
  // a CTA takes every n_used-th group of W pages, so that whatever the length the live CTAs differ by a page per warp at most
  const int total = LivePages(ctx, p.window, p.sinks).total;
  const int n_used = min(static_cast<int>(gridDim.x), (total + W - 1) / W);  // a page for every warp of a live CTA
  if (split >= n_used) return;  // the cluster's barriers count the threads that are left
  const int page_first = split * W + warp, page_step = n_used * W;
  const float c = p.scale_log2;
  auto look_up = [&](int i0) {
    const int page = page_first + (i0 + a.lane) * page_step;
    if (page < total) a.look_up(seq, ctx, page, kvh, 0);
    else a.look_up_none();
  };
  auto fetch = [&](int i) {
    if (page_first + i * page_step >= total) return;
    if (i > 0 && (i & 31) == 0) look_up(i);
    a.fetch(i, kvh);
  };
  look_up(0);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  a.begin_unit(seq * p.H_KV + kvh, G);
  for (int i = 0; page_first + i * page_step < total; ++i) {
    if ((i & 31) == 0) {
      a.take_pages();
      a.refer(seq * p.H_KV + kvh);
    }
    fetch(i + kStages - 1);
    if (!a.page(i, a.seen_of(i))) break;
  }
  const bool huge = decode_fp8_check_waits(a.abort_word, p.status, a.is_huge());

  // ---- merge the W warps through shared memory (the ring is idle now)
  a.end_unit();
  const float out_scale = a.sum_scale(huge), up = huge ? 1.f / kHugeScale : 1.f;
  float* sm_o = reinterpret_cast<float*>(dsmem);  // [W][8][D]
  float* sm_m = sm_o + W * 8 * D;                // [W][8]
  float* sm_l = sm_m + W * 8;                     // [W][8]
#pragma unroll
  for (int j = 0; j < Warp::kChunks; ++j) {
    float* const dst = sm_o + (warp * 8 + 2 * a.t) * D + j * 16 + 2 * a.g;
    *reinterpret_cast<float2*>(dst) = make_float2(a.oacc[j][0] * out_scale, a.oacc[j][2] * out_scale);
    *reinterpret_cast<float2*>(dst + D) = make_float2(a.oacc[j][1] * out_scale, a.oacc[j][3] * out_scale);
  }
  if (a.g == 0) {
    sm_m[warp * 8 + 2 * a.t] = a.m0, sm_m[warp * 8 + 2 * a.t + 1] = a.m1;
    sm_l[warp * 8 + 2 * a.t] = a.l0, sm_l[warp * 8 + 2 * a.t + 1] = a.l1;
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
  if (n_used == 1) {
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int h = i * kHalves + h0;
      if (h >= G) break;
      const size_t row = size_t(seq) * p.H + kvh * G + h;
      p.o[row * D + d] = __float2bfloat16(acc[i] / L[i] * up);
      if (d == 0) p.lse[row] = M[i] * p.scale + __logf(L[i]);
    }
    return;
  }
  // ---- merge the CTAs of the cluster: each leaves its share in its own shared memory, and CTA r reads all of head r, r + n_used, ... in
  // the order of the ranks
  float* cl_o = sm_l + W * 8;          // [8][D]
  float* cl_ml = cl_o + 8 * D;         // [8][2]
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = i * kHalves + h0;
    if (h >= G) break;
    cl_o[h * D + d] = acc[i];
    if (d == 0) cl_ml[2 * h] = M[i], cl_ml[2 * h + 1] = huge ? -L[i] : L[i];
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
    uint32_t signs = __float_as_uint(l_r[0]);
#pragma unroll
    for (int r = 1; r < kMaxCluster; ++r) Mc = fmaxf(Mc, m_r[r]), signs |= __float_as_uint(l_r[r]);
    const bool any_huge = signs >> 31;
    if (any_huge) {
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        if (!signbit(l_r[r])) o_r[r] *= kHugeScale;
        l_r[r] = fabsf(l_r[r]);
      }
    }
    float sum = 0.f, out = 0.f;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      const float wgt = ptx::ex2_approx((m_r[r] - Mc) * c);
      sum += wgt * l_r[r];
      out += wgt * o_r[r];
    }
    const size_t row = size_t(seq) * p.H + kvh * G + h;
    p.o[row * D + d] = __float2bfloat16(out / sum * (any_huge ? 1.f / kHugeScale : 1.f));
    if (d == 0) p.lse[row] = Mc * p.scale + __logf(sum);
  }
  ptx::cluster_arrive();  // nobody leaves while its shared memory is being read
  ptx::cluster_wait();
}

// ------------------------------------------------------------------------------------ all pages as one row
// The live pages of sequence after sequence; group w of n has the places [T w / n, T (w + 1) / n), each of its H_KV warps for a head of its
// own. (With the heads' pages one head after the other, what the GPU reads at a time is 128 or 64 bytes here and there: 64 contexts of 4096
// tokens of H_KV 8 D128 155 us, against 148, when the kernel was slower in other ways.)
struct DecodeFp8Row {
  long long total = 0;  // T
  int groups = 0;       // n
  // the sequence that holds a place (find), and where it begins
  long long begin = 0;
  int seq = 0;
  static __device__ __forceinline__ int context(const DecodeFp8Params& p, int s) { return min(p.ctx_lens[s], p.max_pages * kPageTokens); }
  static __device__ __forceinline__ int pages(const DecodeFp8Params& p, int s) {
    const int ctx = context(p, s);
    return ctx <= 0 ? 0 : LivePages(ctx, p.window, p.sinks).total;
  }
  // Executed by whole warps, as what follows.
  __device__ __forceinline__ explicit DecodeFp8Row(const DecodeFp8Params& p) : total(begin_of(p, p.S)) {
    groups = static_cast<int>(min(static_cast<long long>(p.row_groups), (total + kRowPages - 1) / kRowPages));
  }
  __device__ __forceinline__ long long first(int w) const { return total * w / groups; }
  __device__ __forceinline__ int group_of(long long at) const { return static_cast<int>(((at + 1) * groups - 1) / total); }
  __device__ __forceinline__ void find(const DecodeFp8Params& p, long long at) {
    const int lane = threadIdx.x & 31;
    for (int base = 0; base < p.S; base += 32) {
      const int own = base + lane < p.S ? pages(p, base + lane) : 0;
      long long sum = own;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const long long other = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += other;
      }
      const unsigned behind = __ballot_sync(0xffffffffu, begin + sum > at);
      if (behind) {
        const int l = __ffs(behind) - 1;
        seq = base + l;
        begin += __shfl_sync(0xffffffffu, sum - own, l);
        return;
      }
      begin += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  // Where sequence s begins.
  static __device__ __forceinline__ long long begin_of(const DecodeFp8Params& p, int s) {
    long long sum = 0;
    for (int i = threadIdx.x & 31; i < s; i += 32) sum += pages(p, i);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    return sum;
  }
};
__device__ __forceinline__ float* part_o(const DecodeFp8Params& p, int part, int D) { return static_cast<float*>(p.workspace) + size_t(part) * 8 * D; }
__device__ __forceinline__ float* part_ml(const DecodeFp8Params& p, int part, int D) {
  return static_cast<float*>(p.workspace) + size_t(p.row_groups) * p.H_KV * 2 * 8 * D + size_t(part) * 16;
}
__device__ __forceinline__ DecodeFp8Parts* parts_of(const DecodeFp8Params& p, int unit, int D) {
  return reinterpret_cast<DecodeFp8Parts*>(part_ml(p, p.row_groups * p.H_KV * 2, D)) + unit;
}

// grid = warps / 4, block = 128, dynamic smem = kFp8SmemBytes. Warps work on their own: a unit's end leaves the finished rows,
// or a part of them in the workspace.
template <int D>
__global__ void __launch_bounds__(kFp8Warps * 32, 4)
paged_decode_fp8_row_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                            const __grid_constant__ DecodeFp8Params p) {
  using Warp = DecodeFp8Warp<D>;
  constexpr int kStages = DecodeFp8Ring<D>::kStages;
  extern __shared__ __align__(1024) uint8_t dsmem[];
  Warp a(p, tmap_k, tmap_v, dsmem);
  __syncthreads();
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int w = blockIdx.x * kFp8Warps + (threadIdx.x >> 5), G = p.H / p.H_KV;
  const int group = w / p.H_KV, head = w - group * p.H_KV;
  DecodeFp8Row row(p);
  if (group < row.groups) {
    const long long x0 = row.first(group);
    const int n = static_cast<int>(row.first(group + 1) - x0);  // pages
    row.find(p, x0);
    // a lane walks on from here to the sequences of its own pages
    int seq = row.seq, ctx = DecodeFp8Row::context(p, seq), pages = DecodeFp8Row::pages(p, seq);
    int rel = static_cast<int>(x0 - row.begin) + a.lane;  // of its next page, in the sequence
    auto look_up = [&](int i0) {
      if (i0 + a.lane < n) {
        while (rel >= pages) {
          rel -= pages;
          ctx = DecodeFp8Row::context(p, ++seq);
          pages = DecodeFp8Row::pages(p, seq);
        }
        a.look_up(seq, ctx, rel, head, (rel == 0 ? Warp::kBegins : 0u) | (rel == pages - 1 ? Warp::kEnds : 0u));
        rel += 32;
      } else {
        a.look_up_none();
      }
    };
    auto fetch = [&](int i) {
      if (i >= n) return;
      if (i > 0 && (i & 31) == 0) look_up(i);
      a.fetch(i, head);
    };
    look_up(0);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(i);
    bool fresh = true, begun = false;
    int part = 2 * w, unit_at = 0;
    for (int i = 0; i < n; ++i) {
      if ((i & 31) == 0) a.take_pages();
      const uint32_t seen = a.seen_of(i);
      const int unit = __shfl_sync(0xffffffffu, a.my_unit, i & 31);
      if (fresh) {
        a.begin_unit(unit, G);
        begun = seen & Warp::kBegins;
        unit_at = i;
      }
      if (fresh || (i & 31) == 0) a.refer(unit);
      fetch(i + kStages - 1);
      if (!a.page(i, seen)) break;
      fresh = (seen & Warp::kEnds) || i == n - 1;
      if (!fresh) continue;
      a.end_unit();
      const int h = 2 * a.t;
      const bool whole = begun && (seen & Warp::kEnds);
      if (begun) {
        const int last = whole ? group : row.group_of(x0 + unit_at + DecodeFp8Row::pages(p, unit / p.H_KV) - 1);
        if (a.lane == 0) *parts_of(p, unit, D) = DecodeFp8Parts{part, group, last, 0};
      }
      if (whole) {
        // a mean of values is a number where they are
        const bool huge = a.is_huge();
        const float out_scale = a.sum_scale(huge), up = huge ? 1.f / kHugeScale : 1.f, inv0 = out_scale / a.l0, inv1 = out_scale / a.l1;
        __nv_bfloat16* const dst = p.o + (size_t(unit) * G + h) * D + 2 * a.g;
#pragma unroll
        for (int j = 0; j < Warp::kChunks; ++j) {
          if (h < G) *reinterpret_cast<uint32_t*>(dst + j * 16) = ptx::pack_bf16x2(a.oacc[j][0] * inv0 * up, a.oacc[j][2] * inv0 * up);
          if (h + 1 < G) *reinterpret_cast<uint32_t*>(dst + D + j * 16) = ptx::pack_bf16x2(a.oacc[j][1] * inv1 * up, a.oacc[j][3] * inv1 * up);
        }
        if (a.g < 2 && h + a.g < G)
          p.lse[size_t(unit) * G + h + a.g] = a.g ? a.m1 * p.scale + __logf(a.l1) : a.m0 * p.scale + __logf(a.l0);
      } else {
        const bool huge = a.is_huge();
        const float out_scale = a.sum_scale(huge);
        float* const dst = part_o(p, part, D) + h * D + 2 * a.g;
#pragma unroll
        for (int j = 0; j < Warp::kChunks; ++j) {
          if (h < G) *reinterpret_cast<float2*>(dst + j * 16) = make_float2(a.oacc[j][0] * out_scale, a.oacc[j][2] * out_scale);
          if (h + 1 < G) *reinterpret_cast<float2*>(dst + D + j * 16) = make_float2(a.oacc[j][1] * out_scale, a.oacc[j][3] * out_scale);
        }
        if (a.g < 2) {
          const float l = a.g ? a.l1 : a.l0;
          *reinterpret_cast<float2*>(part_ml(p, part, D) + 2 * (h + a.g)) = make_float2(a.g ? a.m1 : a.m0, huge ? -l : l);
        }
      }
      part = 2 * w + 1;  // what is behind the first unit and not whole is the last one
    }
  }
  decode_fp8_check_waits(a.abort_word, p.status);
}

// grid = (H_KV x ceil(G / heads), S), block = 32 W, W = 8 or 32: a block has `heads` (8, 4, 2 or 1) heads of a unit, W / heads warps for each,
// every warp so many-th parts, and a lane D / 32 columns.
template <int D, int W>
__global__ void __launch_bounds__(W * 32) paged_decode_fp8_join_kernel(const __grid_constant__ DecodeFp8Params p, int heads) {
  constexpr int kCols = D / 32, kWarps = W;
  __shared__ float s_m[kWarps], s_l[kWarps], s_o[kWarps][D];
  ptx::grid_dep_wait();  // from here on the parts are visible
  ptx::grid_dep_launch();
  const int seq = blockIdx.y, G = p.H / p.H_KV, blocks = gridDim.x / p.H_KV, kvh = blockIdx.x / blocks, per_head = kWarps / heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % per_head;
  const int h = (blockIdx.x - kvh * blocks) * heads + warp / per_head;
  const int ctx = p.ctx_lens[seq];
  const DecodeFp8Parts parts = *parts_of(p, seq * p.H_KV + kvh, D);  // nothing wrote those of an empty context
  const size_t row = size_t(seq) * p.H + kvh * G;
  if (ctx <= 0) {  // defined output for an empty context
    if (h >= G || sub != 0) return;
    for (int i = lane; i < D; i += 32) p.o[(row + h) * D + i] = __float2bfloat16(0.f);
    if (lane == 0) p.lse[row + h] = -INFINITY;
    return;
  }
  if (ctx > p.max_pages * kPageTokens && threadIdx.x == 0) atomicCAS(p.status, 0, kStatusBadLen);
  if (!decode_fp8_parts_valid(parts, p.row_groups, p.H_KV)) {
    if (threadIdx.x == 0) atomicCAS(p.status, kStatusOk, kStatusTimeout);
    return;
  }
  if (parts.group == parts.last_group) return;
  const int n = h < G ? parts.last_group - parts.group + 1 : 0;
  auto part = [&](int i) { return i == 0 ? parts.first : 2 * ((parts.group + i) * p.H_KV + kvh); };
  // of a negative row sum O is 2^-64 times what it is: so are the sums from there on
  float m = -INFINITY, l = 0.f, acc[kCols] = {}, unit = 1.f;
  auto huge_too = [&] {
    if (unit == 1.f) {
      unit = kHugeScale;
#pragma unroll
      for (int k = 0; k < kCols; ++k) acc[k] *= kHugeScale;
    }
  };
#pragma unroll 4
  for (int i = sub; i < n; i += per_head) {
    const float2 ml = *reinterpret_cast<const float2*>(part_ml(p, part(i), D) + 2 * h);
    const float* const src = part_o(p, part(i), D) + h * D + lane * kCols;
    float x[kCols];
    if constexpr (kCols == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(src);
    else *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(src);
    const float top = fmaxf(m, ml.x), a = ptx::ex2_approx((m - top) * p.scale_log2), b = ptx::ex2_approx((ml.x - top) * p.scale_log2);
    const bool huge = signbit(ml.y);
    if (huge) huge_too();
    const float b_o = huge ? b : b * unit;
    m = top;
    l = l * a + fabsf(ml.y) * b;
#pragma unroll
    for (int k = 0; k < kCols; ++k) acc[k] = acc[k] * a + x[k] * b_o;
  }
  if (per_head > 1) {
    if (lane == 0) s_m[warp] = m, s_l[warp] = unit == 1.f ? l : -l;
#pragma unroll
    for (int k = 0; k < kCols; ++k) s_o[warp][lane * kCols + k] = acc[k];
    __syncthreads();
    if (sub == 0) {
      for (int w = warp + 1; w < warp + per_head; ++w) {  // a warp without a part has l = 0 and m = -inf, and this one has one
        const float top = fmaxf(m, s_m[w]), a = ptx::ex2_approx((m - top) * p.scale_log2), b = ptx::ex2_approx((s_m[w] - top) * p.scale_log2);
        const bool huge = signbit(s_l[w]);
        if (huge) huge_too();
        const float b_o = huge ? b : b * unit;
        m = top;
        l = l * a + fabsf(s_l[w]) * b;
#pragma unroll
        for (int k = 0; k < kCols; ++k) acc[k] = acc[k] * a + s_o[w][lane * kCols + k] * b_o;
      }
    }
  }
  if (h >= G || sub != 0) return;
  const float up = unit == 1.f ? 1.f : 1.f / kHugeScale;
  uint32_t out[kCols / 2];
#pragma unroll
  for (int k = 0; k < kCols / 2; ++k) out[k] = ptx::pack_bf16x2(acc[2 * k] / l * up, acc[2 * k + 1] / l * up);
  uint32_t* const dst = reinterpret_cast<uint32_t*>(p.o + (row + h) * D + lane * kCols);
#pragma unroll
  for (int k = 0; k < kCols / 2; ++k) dst[k] = out[k];
  if (lane == 0) p.lse[row + h] = m * p.scale + __logf(l);
}

template <int D>
cudaError_t prepare_decode_fp8() {
  auto* cluster = paged_decode_fp8_cluster_kernel<D>;
  cudaError_t e = cudaFuncSetAttribute(cluster, cudaFuncAttributeMaxDynamicSharedMemorySize, kFp8SmemBytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(cluster, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_decode_fp8_row_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFp8SmemBytes);
  return e;
}
inline int prepare_decode_fp8_kernels(char* err, size_t err_len, int sm_count, DecodeLimits* lim) {
  cudaError_t e = prepare_decode_fp8<128>();
  if (e == cudaSuccess) e = prepare_decode_fp8<64>();
  if (e != cudaSuccess) {
    snprintf(err, err_len, "fp8 decode kernel attribute: %s", cudaGetErrorString(e));
    return -3;
  }
  lim->sm_count = sm_count;
  for (int n = 2; n <= kMaxCluster; ++n)
    lim->clusters4[n] = clusters_held(paged_decode_fp8_cluster_kernel<128>, kFp8Warps * 32, kFp8SmemBytes, n);
  return 0;
}

// The size of the cluster that shares a unit; 0: all pages as one row.
//  * Few units: clusters as large as keeps all of them in one wave. One launch, but a long context is its cluster's alone, about 0.6 us a
//    page of a warp; and the row's parts take another kernel, the longer the more warps shared a unit. us, row / clusters (size), H64/8 D128
//    unless said, a read of 256 MB before each: 1 context of 12006 tokens H32/8 30.7 / 18.4 (16), 1 of 2019 H32/8 16.4 / 12.3 (16), 4 of
//    2000 to 4000 H32/8 22.5 / 16.4 (8), 8 of 4096 to 8192 30.7 / 26.6 (8), 64 of 512 to 8192 of H8/1 26.6 / 24.6 (8), 16 of 512 to 8192
//    34.8 / 36.9 (4), 32 of them 42.9 / 61.4 (3).
//  * Many units, each a CTA of its own while the longest a context can be does not hold up the rest: 64 of 300 to 1000 tokens 30.7 / 26.6
//    (1); windows, which most contexts fill: 64 of 2048 61.4 / 57.3 (1), 33 of H48/8 D64 500 20.4 / 14.3 (1). Otherwise the row: 64 of
//    512 to 8192 77.9 / 131 (1), 92 (4); of 4096 each 100.3 / 98.3 (1), 111 (4); D64 53.2 / 94 (1), 65.6 (2); 256 of 200 to 2000 of
//    H32/4 53.2 / 55.3 (1). Chunks of 64 pages and a combining kernel, as in the bf16 decode, took as long for 64 of 512 to 8192, and
//    leave a tail that the row does not have: D64 53.2 / 60.
inline int decode_pick_fp8_cluster(int S, int H_KV, int span, bool window, const DecodeLimits& lim) {
  const long long units = 1ll * S * H_KV;
  int cluster = kMaxCluster;
  while (cluster > 1 && lim.clusters4[cluster] < units) --cluster;
  const int useful = (span + kFp8Warps - 1) / kFp8Warps;  // a page per warp
  if (cluster >= 4 && span <= 128 * cluster) return cluster < useful ? cluster : useful;
  return units <= 4ll * lim.sm_count && span <= (window ? 160 : 64) ? 1 : 0;
}

template <int D>
cudaError_t launch_decode_fp8(const CUtensorMap& tk, const CUtensorMap& tv, DecodeFp8Params p, int cluster, int sm_count,
                              cudaStream_t stream, int* launched) {
  *launched += 1;
  if (cluster)
    return launch_dependent(true, paged_decode_fp8_cluster_kernel<D>, dim3(cluster, p.H_KV, p.S), kFp8Warps * 32, kFp8SmemBytes, stream,
                            ClusterX{unsigned(cluster)}, tk, tv, p);
  p.row_groups = decode_fp8_row_groups(p.H_KV, 16 * sm_count < kRowWarps ? 16 * sm_count : kRowWarps);
  const int warps = p.row_groups * p.H_KV;
  const cudaError_t e = launch_dependent(true, paged_decode_fp8_row_kernel<D>, (warps + kFp8Warps - 1) / kFp8Warps, kFp8Warps * 32,
                                         kFp8SmemBytes, stream, tk, tv, p);
  if (e != cudaSuccess) return e;
  *launched += 1;
  // as many warps for a head as leave two waves of blocks. us in a loop, 1 / 2 / 4 / 8 heads to a block, 64 contexts H64/8 D128 of 512 to 8192
  // 78.8 / 75.1 / 77.7 / 83.1, of 4096 108.7 / 105.1 / 105.2 / 119
  const int G = p.H / p.H_KV;
  int heads = 1;
  while (heads < G && 1ll * p.S * p.H_KV * ((G + heads - 1) / heads) > 16ll * sm_count) heads *= 2;
  // many parts to a unit: 32 warps (one context of 100,000 tokens H8/1 D128 107 / 44, of H32/8 54 / 46)
  const bool many = heads == 1 && p.row_groups > 16 * p.S;
  return launch_dependent(true, many ? paged_decode_fp8_join_kernel<D, 32> : paged_decode_fp8_join_kernel<D, 8>,
                          dim3(p.H_KV * ((G + heads - 1) / heads), p.S), many ? 1024 : 256, 0, stream, p, heads);
}

inline cudaError_t launch_paged_decode_fp8(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeFp8Params& p, int D, bool window,
                                           const DecodeLimits& lim, cudaStream_t stream, int* launched) {
  const int cluster = decode_pick_fp8_cluster(p.S, p.H_KV, p.span_pages, window, lim);
  return (D == 64 ? launch_decode_fp8<64> : launch_decode_fp8<128>)(tk, tv, p, cluster, lim.sm_count, stream, launched);
}

}  // namespace hk
