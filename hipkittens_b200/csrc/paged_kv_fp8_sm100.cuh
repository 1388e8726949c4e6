// The paged KV cache in 8 bits: appending new K/V tokens to it, and reading tokens back as bf16.
//
// A page holds 16 tokens of every K/V head as e4m3 codes; the 16 x D codes of one page and head are a block, with one fp32 scale for
// K and one for V: value = code * scale. An append picks the smallest power of two that brings the block's largest magnitude to 448
// (the largest e4m3 value) at most:
//     amax = m * 2^e, 1 <= m < 2:  scale = 2^(e - 8) if m <= 1.75, else 2^(e - 7)        (448 = 1.75 * 2^8)
// A code has an exponent of its own, so a power of two costs no relative precision against amax / 448, and where a later token needs a
// larger scale the block's other tokens move by a power of two: their codes change exactly, but for those that become subnormal
// (below 2^-14 of the block's largest value). With scales that are not powers of two every growth would round them once more.
// The arithmetic is fp32 with one rounding, to e4m3; the rotation of K is part of it, so that a rotated token is rounded once and not
// twice. Its products and sums are rounded one by one (no fused multiply-adds), the same in any order of evaluation.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "attn_fwd_sm100.cuh"
#include "paged_decode_common.cuh"
#include "sm100_ptx.cuh"

namespace hk {

constexpr int kFp8LeastExp = -120, kFp8MostExp = 119;  // exponents of the scales that an append picks

struct Fp8Cache {
  uint8_t *k_pages, *v_pages;   // [P, 16, H_KV, D] e4m3 codes
  float *k_scales, *v_scales;   // [P, H_KV]
  const int32_t* block_table;   // [S, max_pages]
  int S, H_KV, max_pages, num_pages;
  int* status;
};

// Where the tokens of sequence s are: [S, T, heads, D], or rows cu[s] .. cu[s + 1] - 1 of [T, heads, D] (T in all).
struct Fp8Rows {
  const int32_t* cu;  // [S + 1], or null
  int T;
  FastDiv fd_units;   // without cu: units of a sequence
};

namespace fp8 {

// Units of 16 tokens of ragged sequences: sequence s has those from cu[s] / 16 + PER * s on, which is room for whole pages from its
// first token on (PER = 1) or for pages that it enters and leaves in the middle (PER = 2).
template <int PER>
__device__ __forceinline__ int first_unit(const int32_t* cu, int s) { return (cu[s] >> 4) + PER * s; }
// The last sequence of `n` that starts at or before `unit`; all lanes of a warp look, at 32 sequences a turn. Whatever cu holds, it is
// one of them.
template <int PER>
__device__ __forceinline__ int sequence_of(const int32_t* cu, int n, int unit) {
  int lo = 0;
  while (n > 1) {
    const int step = (n + 31) >> 5, at = static_cast<int>(threadIdx.x & 31) * step;
    const uint32_t before = __ballot_sync(0xffffffffu, at < n && first_unit<PER>(cu, lo + at) <= unit) | 1u;
    const int skip = (31 - __clz(before)) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}
// Rows [first, first + n) of sequence s, kept inside [0, total) whatever cu holds.
__device__ __forceinline__ void ragged_rows(const int32_t* cu, int s, int total, int& first, int& n) {
  first = min(max(cu[s], 0), total);
  n = max(min(cu[s + 1], total) - first, 0);
}
// One block of threads looks the whole array over.
__device__ __forceinline__ void check_cu(const int32_t* cu, int S, int total, int* status) {
  for (int s = threadIdx.x; s < S; s += blockDim.x)
    if (cu[s] < 0 || cu[s + 1] < cu[s] || cu[s + 1] > total) atomicCAS(status, 0, kStatusBadLen);
}

__device__ __forceinline__ float2 decode2(uint32_t codes) {  // the low 16 bits
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<unsigned short>(codes)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  unsigned short lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return lo | static_cast<uint32_t>(hi) << 16;
}
__device__ __forceinline__ float2 bf16x2(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Loads from shared memory that stay where they are: moved up, eight rows of them would not fit in the registers.
__device__ __forceinline__ uint2 lds2(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void lds4(uint32_t at, uint64_t (&v)[2]) {
  asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(v[0]), "=l"(v[1]) : "r"(at) : "memory");
}

// Bits of the scale for a largest magnitude, given by its bits: NaN for NaN, which makes the whole block NaN for every reader.
__device__ __forceinline__ uint32_t scale_bits(uint32_t amax) {
  if (amax > 0x7f800000u) return 0x7fc00000u;
  const int e = static_cast<int>(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(min(max(e, kFp8LeastExp), kFp8MostExp) + 127) << 23;
}
// The larger of two magnitudes and a, NaN if one of them is.
__device__ __forceinline__ float max_size(float a, float x, float y) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(fabsf(x)), "f"(fabsf(y)));
  return d;
}
// x / scale for four values at a time, as codes. Exact through the reciprocal of a power of two (an append's own scales are powers, or
// NaN); a scale that another quantiser left behind divides.
struct ByPower {
  uint64_t inv2;
  __device__ __forceinline__ explicit ByPower(uint32_t bits) {
    const float inv = __uint_as_float(bits > 0x7f800000u ? bits : (254u << 23) - bits);
    inv2 = ptx::pack2(inv, inv);
  }
  __device__ __forceinline__ uint32_t operator()(float a, float b, float c, float d) const {
    return (*this)(ptx::pack2(a, b), ptx::pack2(c, d));
  }
  __device__ __forceinline__ uint32_t operator()(uint64_t ab, uint64_t cd) const {
    float a, b, c, d;
    ptx::unpack2(ptx::mul2(ab, inv2), a, b);
    ptx::unpack2(ptx::mul2(cd, inv2), c, d);
    return encode4(a, b, c, d);
  }
};
struct ByDivision {
  float scale;
  __device__ __forceinline__ uint32_t operator()(float a, float b, float c, float d) const {
    return encode4(__fdiv_rn(a, scale), __fdiv_rn(b, scale), __fdiv_rn(c, scale), __fdiv_rn(d, scale));
  }
  __device__ __forceinline__ uint32_t operator()(uint64_t ab, uint64_t cd) const {
    float a, b, c, d;
    ptx::unpack2(ab, a, b);
    ptx::unpack2(cd, c, d);
    return (*this)(a, b, c, d);
  }
};
template <typename Fn>
__device__ __forceinline__ void with_divisor(uint32_t bits, const Fn& fn) {
  const int e = static_cast<int>(bits >> 23);
  if ((bits & 0x807fffffu) == 0 && e > 0 && e < 254) fn(ByPower(bits));
  else fn(ByDivision{__uint_as_float(bits)});
}

}  // namespace fp8

enum Fp8Rotation : int { kFp8Plain = 0, kFp8TableBf16 = 1, kFp8TableF32 = 2 };

struct AppendFp8Params {
  Fp8Cache c;
  Fp8Rows rows;
  const __nv_bfloat16 *k_new, *v_new;
  long long k_stride[3], v_stride[3];  // sequence, token, head; elements
  const int32_t* start_pos;            // [S] position of the first new token of each sequence
  const void *cos, *sin;               // [table_rows, R / 2] bf16 or fp32
  int rotation;                        // Fp8Rotation
  int R, table_rows;
  int turns;                           // heads of a warp
  FastDiv fd_groups2, fd_groups;       // 2 * groups, groups of a CTA's warps x turns heads
};

constexpr int kFp8AppendWarps = 4;  // at most
constexpr int fp8_append_turns(int D) { return 256 / D; }  // at most: 8 KB of tokens a warp
// Dynamic shared memory: cos and sin [16, D / 2], then the tokens of each warp's turns.
constexpr int fp8_append_smem(int D, bool rotates, int warps, int turns) {
  return (rotates ? 2 * kPageTokens * (D / 2) * 4 : 0) + warps * turns * kPageTokens * D * 2;
}
static_assert(fp8_append_smem(128, true, kFp8AppendWarps, fp8_append_turns(128)) <= 48 * 1024, "what a kernel has without asking");

// A CTA has new tokens of a page, of K or of V, and its warps have a block at a time: a head's tokens of the page, and those of the
// next head already on their way. A warp finds the block's largest magnitude, settles the scale, and writes the codes; if the page had
// tokens already and the scale grows, it reads and rounds anew the rows that get none. Nothing else touches that block, so there is
// nothing to order. The rows of the tables that the page's tokens need are brought in once, as fp32, for all of the CTA's heads: with
// them read from L1 by every warp, and a warp's tokens in its registers from the start, prompts of 29,000 tokens at H_KV = 8 and D = 128
// took 66 us.
// Bound by HBM (3 bytes a value): those take 34 us, 80% of the copy rate, and 30 without a rotation; a token for each sequence is a
// launch and three dependent loads.
// grid = units x 2 x groups of heads; block = up to 32 * kFp8AppendWarps, dynamic smem = fp8_append_smem.
template <int D, bool ROT>
__global__ void __launch_bounds__(kFp8AppendWarps * 32, ROT ? 4 : 5) paged_kv_append_fp8_kernel(const __grid_constant__ AppendFp8Params p) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes, kSteps = kPageTokens / kRows;  // lanes of a row, rows of a step
  constexpr int kTile = kPageTokens * D * 2;
  constexpr int kTable = ROT ? kPageTokens * D / 2 : 0;  // values: [16, R / 2]
  extern __shared__ __align__(16) uint8_t append_smem[];
  float* const tables = reinterpret_cast<float*>(append_smem);  // cos, sin
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const Fp8Cache& c = p.c;
  const int32_t* const cu = p.rows.cu;
  if (cu && blockIdx.x == 0) fp8::check_cu(cu, c.S, p.rows.T, c.status);
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  int unit, rem, group, is_v;
  p.fd_groups2.divmod(blockIdx.x, unit, rem);
  p.fd_groups.divmod(rem, is_v, group);
  int s, block, n = p.rows.T, first = 0;
  if (cu) {
    s = fp8::sequence_of<2>(cu, c.S, unit);
    block = unit - fp8::first_unit<2>(cu, s);
    fp8::ragged_rows(cu, s, p.rows.T, first, n);
  } else {
    p.rows.fd_units.divmod(unit, s, block);
  }
  const long long start = p.start_pos[s], slot = (start >> 4) + block, base = slot * kPageTokens - start;  // row r has token base + r
  const int r0 = static_cast<int>(max(-base, 0ll));
  int r1 = static_cast<int>(min(n - base, static_cast<long long>(kPageTokens)));
  if (block < 0 || r1 <= r0) return;
  if (slot < 0 || slot >= c.max_pages) {
    if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusBadPage);
    return;
  }
  const int id = c.block_table[static_cast<size_t>(s) * c.max_pages + slot];
  if (ROT && slot * kPageTokens + r1 > p.table_rows) {  // tokens behind the tables are not written
    if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusBadPos);
    r1 = static_cast<int>(p.table_rows - slot * kPageTokens);
    if (r1 <= r0) return;
  }

  const int row0 = lane / kLanes, col = (lane % kLanes) * 8;
  const int head0 = group * p.turns * warps + warp, heads = min(p.turns, (c.H_KV - head0 + warps - 1) / warps);  // every warps-th from head0 on
  const long long* const stride = is_v ? p.v_stride : p.k_stride;
  const __nv_bfloat16* const src = (is_v ? p.v_new : p.k_new) + s * stride[0] + (first + base + row0) * stride[1] + col;
  uint8_t* const ring = append_smem + 2 * kTable * sizeof(float) + warp * p.turns * kTile;
  const uint32_t ring_u32 = ptx::smem_u32(ring) + (row0 * D + col) * 2;
  auto request = [&](int turn) {  // rows that are not new become zeros
    const __nv_bfloat16* at = src + (head0 + turn * warps) * stride[2];
    uint32_t to = ring_u32 + turn * kTile;
#pragma unroll
    for (int r = row0; r < kPageTokens; r += kRows, at += kRows * stride[1], to += kRows * D * 2)
      dec::cp_async16_if(to, at, r >= r0 && r < r1);
    dec::cp_async_commit();
  };
  if (heads > 0) request(0);
  if (ROT && !is_v) {
    const int quads = p.R / 8;  // of a row
    for (int i = r0 * quads + threadIdx.x; i < r1 * quads; i += blockDim.x) {
      const size_t at = static_cast<size_t>(slot) * kPageTokens * quads + i;
      float4 cs, sn;
      if (p.rotation == kFp8TableF32) {
        cs = static_cast<const float4*>(p.cos)[at], sn = static_cast<const float4*>(p.sin)[at];
      } else {
        const uint2 a = static_cast<const uint2*>(p.cos)[at], b = static_cast<const uint2*>(p.sin)[at];
        const float2 a0 = fp8::bf16x2(a.x), a1 = fp8::bf16x2(a.y), b0 = fp8::bf16x2(b.x), b1 = fp8::bf16x2(b.y);
        cs = make_float4(a0.x, a0.y, a1.x, a1.y), sn = make_float4(b0.x, b0.y, b1.x, b1.y);
      }
      reinterpret_cast<float4*>(tables)[i] = cs;
      reinterpret_cast<float4*>(tables + kTable)[i] = sn;
    }
    __syncthreads();
  }
  if (id < 0 || id >= c.num_pages) {  // never write through an id outside the pool
    if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusBadPage);
    dec::cp_async_wait<0>();
    return;
  }

  const size_t row_bytes = static_cast<size_t>(c.H_KV) * D;
  // FULL: all of the page's rows are new. TURN: these heads are rotated.
  auto work = [&](auto full_c, auto turn_c) {
    constexpr bool FULL = decltype(full_c)::value, TURN = decltype(turn_c)::value;
    // A lane has 8 neighbouring values of a row, or where they are turned 4 and their 4 partners, half the rotated columns further on.
    const bool turned = TURN && col < p.R;
    const int col0 = turned ? col / 2 : col, col1 = turned ? (col + p.R) / 2 : col + 4;
    auto is_new = [&](int i) { return FULL || (row0 + i * kRows >= r0 && row0 + i * kRows < r1); };
#pragma unroll 1
    for (int turn = 0; turn < heads; ++turn) {
      const int head = head0 + turn * warps;
      float* const scale_at = (is_v ? c.v_scales : c.k_scales) + static_cast<size_t>(id) * c.H_KV + head;
      uint8_t* const page = (is_v ? c.v_pages : c.k_pages) + static_cast<size_t>(id) * kPageTokens * row_bytes + head * D;
      const uint32_t before = !FULL && r0 > 0 ? __float_as_uint(*scale_at) : 0u;  // a page that starts anew has no scale yet
      // From the largest magnitude on: the scale, the codes of the new rows (`row(i, divide)`: those of a lane's 8 values in step i), and
      // where the scale has grown the other rows'.
      auto finish = [&](uint32_t amax, auto&& row) {
        uint32_t bits = fp8::scale_bits(__reduce_max_sync(0xffffffffu, amax));
        auto write = [&](auto divide) {
          uint8_t* at = page + row0 * row_bytes;
#pragma unroll
          for (int i = 0; i < kSteps; ++i, at += kRows * row_bytes) {
            if (!is_new(i)) continue;
            const uint2 codes = row(i, divide);
            if constexpr (TURN) {
              *reinterpret_cast<uint32_t*>(at + col0) = codes.x;
              *reinterpret_cast<uint32_t*>(at + col1) = codes.y;
            } else {
              *reinterpret_cast<uint2*>(at + col) = codes;
            }
          }
        };
        if (FULL) {
          write(fp8::ByPower(bits));
          if (lane == 0) *scale_at = __uint_as_float(bits);
          return;
        }
        if (r0 > 0) {
          if ((before & 0x7fffffffu) > 0x7f800000u) bits = 0x7fc00000u;
          else if (static_cast<int>(before) > static_cast<int>(bits)) bits = before;  // of floats above zero
        }
        fp8::with_divisor(bits, [&](auto divide) {
          write(divide);
          if (r0 > 0 && bits != before) {
            const float old = __uint_as_float(before);
#pragma unroll 1
            for (int r = row0; r < kPageTokens; r += kRows) {
              if (r >= r0 && r < r1) continue;
              uint2* const at = reinterpret_cast<uint2*>(page + r * row_bytes + col);
              const uint2 v = *at;
              auto anew = [&](uint32_t codes) {
                const float2 a = fp8::decode2(codes), b = fp8::decode2(codes >> 16);
                return divide(a.x * old, a.y * old, b.x * old, b.y * old);
              };
              *at = make_uint2(anew(v.x), anew(v.y));
            }
          }
        });
        if (lane == 0 && (r0 == 0 || bits != before)) *scale_at = __uint_as_float(bits);
      };

      if (turn + 1 < heads) {
        request(turn + 1);
        dec::cp_async_wait<1>();
      } else {
        dec::cp_async_wait<0>();
      }
      __syncwarp();
      const uint8_t* const tile = ring + turn * kTile + row0 * D * 2;
      if constexpr (!TURN) {
        auto values = [&](int i) { return *reinterpret_cast<const uint4*>(tile + (i * kRows * D + col) * 2); };
        uint32_t two = 0;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const uint4 x = values(i);
          for (uint32_t v : {x.x, x.y, x.z, x.w}) two = __vmaxu2(two, v & 0x7fff7fffu);
        }
        finish(max(two & 0xffff0000u, two << 16), [&](int i, auto divide) {
          const uint4 x = values(i);
          const float2 a = fp8::bf16x2(x.x), b = fp8::bf16x2(x.y), d = fp8::bf16x2(x.z), e = fp8::bf16x2(x.w);
          return make_uint2(divide(ptx::pack2(a.x, a.y), ptx::pack2(b.x, b.y)), divide(ptx::pack2(d.x, d.y), ptx::pack2(e.x, e.y)));
        });
      } else {
        // a pair (i, i + R / 2) becomes (a cos - b sin, b cos + a sin)
        uint64_t y[kSteps][4];
        float amax = 0.f;
        const float* const cs_at = tables + row0 * (p.R / 2) + col0;
        const uint32_t at0 = ptx::smem_u32(cs_at), step = kRows * (p.R / 2) * 4, x0 = ptx::smem_u32(tile);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const uint2 xa = fp8::lds2(x0 + (i * kRows * D + col0) * 2), xb = fp8::lds2(x0 + (i * kRows * D + col1) * 2);
          const uint32_t words[4] = {xa.x, xa.y, xb.x, xb.y};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 v = fp8::bf16x2(words[j]);
            y[i][j] = ptx::pack2(v.x, v.y);
          }
          if (turned && is_new(i)) {
            uint64_t cs[2], sn[2];
            fp8::lds4(at0 + i * step, cs);
            fp8::lds4(at0 + i * step + kTable * 4, sn);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint64_t a2 = y[i][j], b2 = y[i][j + 2];
              y[i][j] = ptx::fma2(ptx::mul2(b2, sn[j]), ptx::pack2(-1.f, -1.f), ptx::mul2(a2, cs[j]));
              y[i][j + 2] = ptx::add2(ptx::mul2(b2, cs[j]), ptx::mul2(a2, sn[j]));
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float lo, hi;
            ptx::unpack2(y[i][j], lo, hi);
            amax = fp8::max_size(amax, lo, hi);
          }
        }
        finish(__float_as_uint(amax), [&](int i, auto divide) { return make_uint2(divide(y[i][0], y[i][1]), divide(y[i][2], y[i][3])); });
      }
    }
  };
  const bool full = r0 == 0 && r1 == kPageTokens;
  if (!ROT || is_v) {
    full ? work(std::true_type{}, std::false_type{}) : work(std::false_type{}, std::false_type{});
  } else if constexpr (ROT) {
    full ? work(std::true_type{}, std::true_type{}) : work(std::false_type{}, std::true_type{});
  }
}

struct ReadFp8Params {
  Fp8Cache c;
  Fp8Rows rows;
  const int32_t* ctx_lens;        // [S], without rows.cu
  __nv_bfloat16 *k_out, *v_out;   // contiguous
  int zero_rest;                  // with rows.cu: rows in front of the first sequence and behind the last one become zeros
  int warps;                      // units x H_KV
  FastDiv fd_heads;
};

// A warp has 16 tokens of one head, K and V: all of their codes are requested before the first is used (8 x 16 bytes a lane at D =
// 128), scaled in fp32 and rounded once. Bound by HBM, 3 bytes a value: 4 sequences of 4,096 to 8,192 tokens, H_KV 8 D128, 31 us in a
// loop, 87% of the copy rate; 32-byte stores, where the output allows them, are one a lane in place of two.
template <int D>
__global__ void __launch_bounds__(256) paged_kv_read_fp8_kernel(const __grid_constant__ ReadFp8Params p) {
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const Fp8Cache& c = p.c;
  const int32_t* const cu = p.rows.cu;
  if (cu && blockIdx.x == 0) fp8::check_cu(cu, c.S, p.rows.T, c.status);
  const int w = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (w >= p.warps) return;
  int unit, head, s, block;
  p.fd_heads.divmod(w, unit, head);
  int len, there;       // tokens of the sequence, rows of this unit that are written
  long long out_row;
  if (cu) {
    s = fp8::sequence_of<1>(cu, c.S + 1, unit);
    block = unit - fp8::first_unit<1>(cu, s);
    if (s == 0 && block <= 0 && p.zero_rest) {  // the rows of this unit that are in front of the first sequence
      const int row = unit * kPageTokens, n = min(min(max(cu[0], 0), p.rows.T) - row, kPageTokens);
      for (int i = lane; i < n * (D / 8); i += 32) {
        const size_t at = (static_cast<size_t>(row + i / (D / 8)) * c.H_KV + head) * D + i % (D / 8) * 8;
        *reinterpret_cast<uint4*>(p.k_out + at) = *reinterpret_cast<uint4*>(p.v_out + at) = make_uint4(0, 0, 0, 0);
      }
    }
    if (block < 0) return;
    int first;
    if (s < c.S) {
      fp8::ragged_rows(cu, s, p.rows.T, first, len);
      there = len - block * kPageTokens;
    } else {
      if (!p.zero_rest) return;
      first = min(max(cu[s], 0), p.rows.T);
      len = 0;
      there = p.rows.T - first - block * kPageTokens;
    }
    out_row = first + block * kPageTokens;
  } else {
    p.rows.fd_units.divmod(unit, s, block);
    len = p.ctx_lens[s];
    there = p.rows.T - block * kPageTokens;
    out_row = static_cast<long long>(s) * p.rows.T + block * kPageTokens;
  }
  there = min(there, kPageTokens);
  if (there <= 0) return;
  if (len > static_cast<long long>(c.max_pages) * kPageTokens || (!cu && len > p.rows.T)) {
    if (lane == 0) atomicCAS(c.status, 0, kStatusBadLen);
    len = static_cast<int>(min(static_cast<long long>(len), static_cast<long long>(c.max_pages) * kPageTokens));
  }
  int valid = min(len - block * kPageTokens, there);  // what lies behind them comes back as zeros
  int id = 0;
  if (valid > 0) {
    id = c.block_table[static_cast<size_t>(s) * c.max_pages + block];
    if (id < 0 || id >= c.num_pages) {
      if (lane == 0) atomicCAS(c.status, 0, kStatusBadPage);
      id = valid = 0;
    }
  }
  constexpr int kLanes = D / 16, kRows = 32 / kLanes, kSteps = kPageTokens / kRows;
  const int col = (lane % kLanes) * 16, row0 = lane / kLanes;
  const size_t row_bytes = static_cast<size_t>(c.H_KV) * D, at = static_cast<size_t>(id) * kPageTokens * row_bytes + head * D + col;
  uint4 x[2][kSteps];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv)
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int r = row0 + i * kRows;
      x[kv][i] = make_uint4(0, 0, 0, 0);
      if (r < valid) x[kv][i] = __ldcs(reinterpret_cast<const uint4*>((kv ? c.v_pages : c.k_pages) + at + r * row_bytes));
    }
  const bool wide[2] = {(reinterpret_cast<uintptr_t>(p.k_out) & 31) == 0, (reinterpret_cast<uintptr_t>(p.v_out) & 31) == 0};
  const size_t scale_at = static_cast<size_t>(id) * c.H_KV + head;
  const float scales[2] = {valid > 0 ? c.k_scales[scale_at] : 0.f, valid > 0 ? c.v_scales[scale_at] : 0.f};
#pragma unroll
  for (int kv = 0; kv < 2; ++kv)
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int r = row0 + i * kRows;
      if (r >= there) continue;
      const uint32_t words[4] = {x[kv][i].x, x[kv][i].y, x[kv][i].z, x[kv][i].w};
      uint32_t o[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = fp8::decode2(words[j]), b = fp8::decode2(words[j] >> 16);
        o[2 * j] = ptx::pack_bf16x2(a.x * scales[kv], a.y * scales[kv]);
        o[2 * j + 1] = ptx::pack_bf16x2(b.x * scales[kv], b.y * scales[kv]);
      }
      if (r >= valid)
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = 0;  // and not a NaN of the block's scale
      uint4* const dst = reinterpret_cast<uint4*>((kv ? p.v_out : p.k_out) + ((out_row + r) * c.H_KV + head) * D + col);
      if (wide[kv]) {
        ptx::st_global_v8(dst, o);
      } else {
        dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
        dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
      }
    }
}

}  // namespace hk
