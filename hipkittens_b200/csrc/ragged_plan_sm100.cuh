// The work of a ragged attention call: which sequence and tile each work item is. The lengths lie on the device, so the list of them is
// made there, by a kernel in front of the call's others.
//
// A place of a list is a query tile, a pair of them, or a key block of one sequence, and stands for one item per K/V head (and head or pair
// of heads). Places come in the order of the tiles that their items meet, the most first, and are dealt to CTAs in a snake (planned_item):
// what a CTA gets is then as long as what any other gets, whatever the lengths. The order is a counting sort over 1024 classes, in
// one CTA per list; inside a class it is whatever the atomics make it, which changes no result, since every item owns its outputs.
// In the backward the lists are made beside delta, by the same launch.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_bwd_sm100.cuh"
#include "attn_fwd_sm100.cuh"
#include "paged_decode_common.cuh"
#include "sm100_ptx.cuh"

namespace hk {

enum RaggedList : int { kQueryTiles = 0, kQueryPairs = 1, kKeyBlocks = 2 };

// Rows of an output that no sequence has become zeros (fp32 rows of L: -inf).
struct RaggedRest {
  void* out;                          // null: none
  long long row_stride, head_stride;  // elements
  int heads, rows, units;             // units: of 8 values in a head's row; 0: fp32, one value, and row_stride 1
  int of_keys;                        // rows of k, and not of q
};

struct RaggedPlanParams {
  const int32_t *cu_q, *cu_k;  // [S + 1]
  int S, q_rows, k_rows, causal;
  int lists;
  int kind[2];
  int* count[2];
  int4* places[2];             // two words of four: q0, queries, k0, keys; tile
  int rests;
  RaggedRest rest[3];
  int* status;
};

constexpr int kPlanClasses = 1024, kPlanThreads = 1024, kPrepThreads = 256;  // of the plan alone, and of the backward's with delta
constexpr int kPlanRestThreads = 32 * 1024;                                       // that fill rows without a sequence

struct RaggedSequence {
  int q0, n_q, k0, n_k;
  RaggedSequence() = default;
  __device__ __forceinline__ RaggedSequence(const RaggedPlanParams& p, int s) {
    q0 = p.cu_q[s], n_q = p.cu_q[s + 1] - q0, k0 = p.cu_k[s], n_k = p.cu_k[s + 1] - k0;
  }
  __device__ __forceinline__ bool is_bad(const RaggedPlanParams& p) const {  // offsets that fall, or that lie outside the rows
    return q0 < 0 || k0 < 0 || n_q < 0 || n_k < 0 || n_q > p.q_rows - q0 || n_k > p.k_rows - k0;
  }
  __device__ __forceinline__ int places(int kind) const {
    return kind == kKeyBlocks ? (n_k + kBlockN - 1) / kBlockN : kind == kQueryTiles ? (n_q + kBlockM - 1) / kBlockM : (n_q + 2 * kBlockM - 1) / (2 * kBlockM);
  }
  // the tiles that an item of this place meets (in the kernels' terms: decode_item, decode_dkdv_item)
  __device__ __forceinline__ int cost(int kind, int place, bool causal) const {
    const int off = n_k - n_q, n_kv = (n_k + kBlockN - 1) / kBlockN, n_qt = (n_q + kBlockM - 1) / kBlockM;
    if (kind == kKeyBlocks) return max(n_qt - (causal ? max(place * kBlockN - off, 0) / kBlockM : 0), 0);
    const int tile = kind == kQueryTiles ? place : min(2 * place + 1, n_qt - 1);
    return causal ? min(max((tile * kBlockM + kBlockM + off + kBlockN - 1) / kBlockN, 0), n_kv) : n_kv;
  }
};

template <int THREADS>
struct RaggedPlanSmem {
  int classes[kPlanClasses];
  int starts[THREADS + 1];        // of the places of up to THREADS sequences
  RaggedSequence seq[THREADS];
  int sums[THREADS / 32], most;
};

// Of v over the CTA's threads up to this one.
template <int THREADS>
__device__ __forceinline__ int scan(int v, int (&sums)[THREADS / 32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += other;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  const int ahead = __reduce_add_sync(0xffffffffu, lane < warp ? sums[lane] : 0);
  return v + ahead;
}

template <int THREADS>
__device__ __forceinline__ bool any_bad_sequence(const RaggedPlanParams& p) {
  bool bad = false;
  for (int s = threadIdx.x; s < p.S; s += THREADS) bad |= RaggedSequence(p, s).is_bad(p);
  return __syncthreads_or(bad);
}

// One CTA makes a list. It takes THREADS sequences at a time, and of their places one to a thread, which finds its sequence by the sums of
// their numbers: two passes of a few hundred cycles. From cold caches, against a warp for each sequence (of 32 and more; fewer one after
// the other, by the whole CTA): 23 sequences of up to 400 tokens 6.1 us, against 16; 10 of up to 3,000 6.1, against 9.9.
template <int THREADS>
__device__ void ragged_plan_list(const RaggedPlanParams& p, int list, RaggedPlanSmem<THREADS>& m) {
  const int tid = threadIdx.x, kind = p.kind[list];
  bool bad = false;
  int longest = 0;
  RaggedSequence own{};
  for (int s = tid; s < p.S; s += THREADS) {
    own = RaggedSequence(p, s);
    bad |= own.is_bad(p);
    longest = max(longest, kind == kKeyBlocks ? own.n_q : own.n_k);
  }
  if (tid == 0) m.most = 0;
  for (int c = tid; c < kPlanClasses; c += THREADS) m.classes[c] = 0;
  if (__syncthreads_or(bad)) {
    if (tid == 0) {
      *p.count[list] = 0;
      atomicCAS(p.status, 0, kStatusBadLen);
    }
    return;
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  if ((tid & 31) == 0) atomicMax(&m.most, (longest + kBlockM - 1) / kBlockM);
  int total = 0;
  auto load = [&] {  // own is a sequence of these, or none
    m.seq[tid] = own;
    const int n = scan<THREADS>(own.places(kind), m.sums);
    m.starts[tid + 1] = n;
    if (tid == 0) m.starts[0] = 0;
    __syncthreads();
    total = m.starts[THREADS];
  };
  const bool once = p.S <= THREADS;
  if (once) load();
  else __syncthreads();
  int shift = 0;
  while ((m.most >> shift) >= kPlanClasses) ++shift;
  auto each = [&](auto&& fn) {
    for (int s0 = 0; s0 < p.S; s0 += THREADS) {
      if (!once) {
        own = s0 + tid < p.S ? RaggedSequence(p, s0 + tid) : RaggedSequence{};
        load();
      }
      for (int i = tid; i < total; i += THREADS) {
        int at = 0;
#pragma unroll
        for (int step = THREADS / 2; step > 0; step >>= 1)
          if (m.starts[at + step] <= i) at += step;
        const RaggedSequence x = m.seq[at];
        const int place = i - m.starts[at];
        fn(x, place, x.cost(kind, place, p.causal) >> shift);
      }
      __syncthreads();
    }
  };
  each([&](const RaggedSequence&, int, int c) { atomicAdd(&m.classes[c], 1); });
  // where each class begins: behind all higher ones
  constexpr int kOwn = kPlanClasses / THREADS;
  int n[kOwn], sum = 0;
#pragma unroll
  for (int c = 0; c < kOwn; ++c) sum += n[c] = m.classes[kPlanClasses - 1 - tid * kOwn - c];
  const int upto = scan<THREADS>(sum, m.sums);
  if (tid == THREADS - 1) *p.count[list] = upto;
  int at = upto - sum;
#pragma unroll
  for (int c = 0; c < kOwn; ++c) {
    m.classes[kPlanClasses - 1 - tid * kOwn - c] = at;
    at += n[c];
  }
  __syncthreads();
  int4* const places = p.places[list];
  each([&](const RaggedSequence& x, int place, int c) {
    const int at = atomicAdd(&m.classes[c], 1);
    places[2 * at] = make_int4(x.q0, x.n_q, x.k0, x.n_k);
    places[2 * at + 1] = make_int4(place, 0, 0, 0);
  });
}

// Rows that no sequence has, by kPlanRestThreads threads in all.
__device__ __forceinline__ void ragged_fill_rest(const RaggedPlanParams& p, int thread) {
  for (int i = 0; i < p.rests; ++i) {
    const RaggedRest& r = p.rest[i];
    const int32_t* const cu = r.of_keys ? p.cu_k : p.cu_q;
    const int front = cu[0], behind = cu[p.S];
    const long long width = static_cast<long long>(r.heads) * max(r.units, 1), n = (front + static_cast<long long>(r.rows - behind)) * width;
    for (long long at = thread; at < n; at += kPlanRestThreads) {
      const long long nth = at / width, row = nth < front ? nth : behind + nth - front;
      const int rem = static_cast<int>(at - nth * width);
      if (r.units) {
        const int head = rem / r.units, u = rem % r.units;
        reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(r.out) + row * r.row_stride + head * r.head_stride)[u] = make_uint4(0, 0, 0, 0);
      } else {
        static_cast<float*>(r.out)[row + rem * r.head_stride] = -INFINITY;
      }
    }
  }
}

// grid = lists, and kPlanRestThreads / kPlanThreads more where rows without a sequence are filled; block = kPlanThreads. Bad offsets are
// reported, and the call does nothing.
__global__ void __launch_bounds__(kPlanThreads) ragged_plan_kernel(const __grid_constant__ RaggedPlanParams p) {
  __shared__ RaggedPlanSmem<kPlanThreads> smem;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int block = blockIdx.x;
  if (block < p.lists) ragged_plan_list(p, block, smem);
  else if (!any_bad_sequence<kPlanThreads>(p)) ragged_fill_rest(p, (block - p.lists) * kPlanThreads + threadIdx.x);
}

// The backward's: beside the lists, delta. Of most rows that is rowsum(dO * O), as in attn_bwd_prep_kernel; of rows of few keys it is the
// sum of P dP over these, from the scores, as in attn_bwd_prep_window_kernel and for its reasons: those at the first kFewRows positions of
// a sequence under the causal rule, and without it all rows of sequences of up to kFewKeys keys. (With delta from O alone in all rows, dQ
// over 23 sequences of up to 400 tokens was off by 2.6e-3 of its size, D = 64; so by 2.4e-3, of which 2.35e-3 are the roundings of dS and
// of dQ itself.) 12,100 tokens of 32 heads of 128 take 35 us from cold caches; the plan and attn_bwd_prep_kernel one
// after the other took 41.
struct RaggedPrepParams {
  RaggedPlanParams plan;
  const __nv_bfloat16 *q, *k, *v, *o, *d_o;
  const float* lse;
  float* delta;                                     // [H, q_rows]
  long long q_stride[2], k_stride[2], v_stride[2];  // row, head; elements
  int H, rows;                                      // heads, rows of all heads
  int few_blocks, row_blocks;                       // few_blocks: 8 of ragged_few_tiles x H warps
  float scale_log2;
  FastDiv fd_h, fd_g;                               // H, H / H_KV
};

// Tiles of 16 rows that may be of few keys: causal, two of each sequence; otherwise sequence s has those from cu[s] / 16 + s on.
inline long long ragged_few_tiles(int S, int q_rows, bool causal) { return causal ? 2ll * S : q_rows / 16 + 1ll * S; }

// The last sequence whose `key` is not above `value`; all lanes of a warp look. Keys do not fall; whatever they do, it is one of them.
template <typename Key>
__device__ __forceinline__ int ragged_sequence_at(int S, int value, const Key& key) {
  int s = 0;
  for (int n = S; n > 1;) {
    const int step = (n + 31) >> 5, at = static_cast<int>(threadIdx.x & 31) * step;
    const uint32_t there = __ballot_sync(0xffffffffu, at < n && key(s + at) <= value) | 1u;
    const int skip = (31 - __clz(there)) * step;
    s += skip;
    n = min(step, n - skip);
  }
  return s;
}

// Is delta of the row at this position of a sequence taken from the scores?
__device__ __forceinline__ bool ragged_few(const RaggedSequence& x, bool causal, int row) {
  const int pos = row + x.n_k - x.n_q;
  return causal ? pos >= 0 && pos < kFewRows : x.n_k <= kFewKeys;
}

// One of those tiles, one head.
template <int D>
__device__ void ragged_few_rows(const RaggedPrepParams& p, int tile, int h) {
  const bool causal = p.plan.causal;
  int s = tile >> 1;
  if (causal) {
    if (s >= p.plan.S) return;
    tile &= 1;
  } else {
    auto first_tile = [&](int at) { return (p.plan.cu_q[at] >> 4) + at; };
    s = ragged_sequence_at(p.plan.S, tile, first_tile);
    tile -= first_tile(s);
  }
  const RaggedSequence x(p.plan, s);
  if (x.is_bad(p.plan) || tile < 0 || (!causal && x.n_k > kFewKeys)) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, kvh = p.fd_g.div(h);
  const int behind = causal ? x.n_k - x.n_q : 0;  // a row's position less its number
  const int rows = causal ? min(kFewRows - behind, x.n_q) : x.n_q;
  const __nv_bfloat16 *const k = p.k + x.k0 * p.k_stride[0] + kvh * p.k_stride[1] + t * 8,
                      *const v = p.v + x.k0 * p.v_stride[0] + kvh * p.v_stride[1] + t * 8;
  auto load = [](const __nv_bfloat16* at) { return *reinterpret_cast<const uint4*>(at); };
  if (const int first = max(-behind, 0) + tile * 16; first < rows) {
    const __nv_bfloat16 *q[2], *grad[2];  // rows g and g + 8
    float nl[2], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long n = x.q0 + min(first + g + 8 * i, x.n_q - 1);  // a row that is not there: the last one, and not stored
      q[i] = p.q + n * p.q_stride[0] + h * p.q_stride[1] + t * 8;
      grad[i] = p.d_o + (n * p.H + h) * D + t * 8;
      nl[i] = p.lse[h * static_cast<long long>(p.plan.q_rows) + n] * -1.4426950408889634f;
    }
    const int end = causal ? min(first + 16 + behind, x.n_k) : x.n_k;
#pragma unroll 1
    for (int key0 = 0; key0 < end; key0 += 8) {
      const long long key = min(key0 + g, x.n_k - 1);
      float sc[4] = {0.f, 0.f, 0.f, 0.f}, dp[4] = {0.f, 0.f, 0.f, 0.f};
      // A lane has 8 neighbouring columns of its rows and of its key at a time, in place of those that the products name
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        const uint4 kc = load(k + key * p.k_stride[0] + c), vc = load(v + key * p.v_stride[0] + c);
        const uint4 q0 = load(q[0] + c), q1 = load(q[1] + c), g0 = load(grad[0] + c), g1 = load(grad[1] + c);
        ptx::mma_16816(sc, q0.x, q1.x, q0.y, q1.y, kc.x, kc.y);
        ptx::mma_16816(dp, g0.x, g1.x, g0.y, g1.y, vc.x, vc.y);
        ptx::mma_16816(sc, q0.z, q1.z, q0.w, q1.w, kc.z, kc.w);
        ptx::mma_16816(dp, g0.z, g1.z, g0.w, g1.w, vc.z, vc.w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // rows g and g + 8, keys 2 t and 2 t + 1
        const int at = key0 + 2 * t + (e & 1), pos = first + g + 8 * (e >> 1) + behind;
        if (at < x.n_k && (!causal || at <= pos))
          sum[e >> 1] = fmaf(ptx::ex2_approx(fmaf(sc[e], p.scale_log2, nl[e >> 1])), dp[e], sum[e >> 1]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
      const int row = first + g + 8 * i;
      if (t == 0 && row < rows) p.delta[h * static_cast<long long>(p.plan.q_rows) + x.q0 + row] = sum[i];
    }
  }
}

// grid = lists, few_blocks, row_blocks, and the rest's; block = kPrepThreads.
template <int D>
__global__ void __launch_bounds__(kPrepThreads, 4) ragged_prep_kernel(const __grid_constant__ RaggedPrepParams p) {
  __shared__ RaggedPlanSmem<kPrepThreads> smem;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  int block = blockIdx.x;
  if (block < p.plan.lists) return ragged_plan_list(p.plan, block, smem);
  block -= p.plan.lists;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (block < p.few_blocks) {
    int tile, h;
    p.fd_h.divmod(block * 8 + warp, tile, h);
    return ragged_few_rows<D>(p, tile, h);
  }
  block -= p.few_blocks;
  if (block >= p.row_blocks) {
    if (!any_bad_sequence<kPrepThreads>(p.plan)) ragged_fill_rest(p.plan, (block - p.row_blocks) * kPrepThreads + threadIdx.x);
    return;
  }
  constexpr int kLanesPerRow = D / 8, kRowsPerWarp = 32 / kLanesPerRow;
  const int sub = lane % kLanesPerRow, warp0 = (block * 8 + warp) * (kRowsPerWarp * kRowPassUnroll), row0 = warp0 + lane / kLanesPerRow;
  uint4 a[kRowPassUnroll], b[kRowPassUnroll];
#pragma unroll
  for (int u = 0; u < kRowPassUnroll; ++u) {
    const int row = min(row0 + u * kRowsPerWarp, p.rows - 1);  // a row beyond the last: that one again, and not stored
    a[u] = __ldcs(reinterpret_cast<const uint4*>(p.o + static_cast<size_t>(row) * D) + sub);
    b[u] = __ldcs(reinterpret_cast<const uint4*>(p.d_o + static_cast<size_t>(row) * D) + sub);
  }
  // the sequence of the warp's first row, while they come in; the others' are its or next ones
  int s = ragged_sequence_at(p.plan.S, p.fd_h.div(min(warp0, p.rows - 1)), [&](int at) { return p.plan.cu_q[at]; });
  RaggedSequence x(p.plan, s);
#pragma unroll
  for (int u = 0; u < kRowPassUnroll; ++u) {
    const uint32_t aw[4] = {a[u].x, a[u].y, a[u].z, a[u].w}, bw[4] = {b[u].x, b[u].y, b[u].z, b[u].w};
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc = fmaf(__uint_as_float(aw[i] << 16), __uint_as_float(bw[i] << 16), acc);
      acc = fmaf(__uint_as_float(aw[i] & 0xffff0000u), __uint_as_float(bw[i] & 0xffff0000u), acc);
    }
#pragma unroll
    for (int off = kLanesPerRow / 2; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    const int row = row0 + u * kRowsPerWarp;
    if (row < p.rows && sub == 0) {
      int n, h;
      p.fd_h.divmod(row, n, h);
      while (n >= x.q0 + x.n_q && s + 1 < p.plan.S) x = RaggedSequence(p.plan, ++s);
      if (n < x.q0 || n >= x.q0 + x.n_q || !ragged_few(x, p.plan.causal, n - x.q0)) p.delta[h * static_cast<long long>(p.plan.q_rows) + n] = acc;
    }
  }
}

}  // namespace hk
