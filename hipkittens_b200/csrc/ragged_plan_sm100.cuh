// The work of a ragged attention call: which sequence and tile each work item is. The lengths lie on the device, so the list of them is
// made there, by a kernel in front of the call's others.
//
// A place of a list is a query tile, a pair of them, or a key block of one sequence, and stands for one item per K/V head (and head or pair
// of heads). Places come in the order of the tiles that their items meet, the most first, and are dealt to CTAs in a snake (planned_item):
// what a CTA gets is then as long as what any other gets, whatever the lengths. The order is a counting sort over 1024 classes, in
// one CTA per list; inside a class it is whatever the atomics make it, which changes no result, since every item owns its outputs.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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

constexpr int kPlanThreads = 1024, kPlanClasses = 1024, kPlanRestBlocks = 32;

struct RaggedSequence {
  int q0, n_q, k0, n_k;
  __device__ __forceinline__ RaggedSequence(const RaggedPlanParams& p, int s) {
    q0 = p.cu_q[s], n_q = p.cu_q[s + 1] - q0, k0 = p.cu_k[s], n_k = p.cu_k[s + 1] - k0;
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

// grid = lists, and kPlanRestBlocks more where rows without a sequence are filled; block = kPlanThreads. Offsets that fall, or that lie
// outside the rows, are reported, and the call does nothing.
__global__ void __launch_bounds__(kPlanThreads) ragged_plan_kernel(const __grid_constant__ RaggedPlanParams p) {
  __shared__ int classes[kPlanClasses], warp_sums[32], most;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int tid = threadIdx.x, list = blockIdx.x, kind = p.kind[min(list, 1)];
  bool bad = false;
  int longest = 0;
  for (int s = tid; s < p.S; s += kPlanThreads) {
    const RaggedSequence x(p, s);
    bad |= x.q0 < 0 || x.k0 < 0 || p.cu_q[s + 1] < x.q0 || p.cu_k[s + 1] < x.k0 || p.cu_q[s + 1] > p.q_rows || p.cu_k[s + 1] > p.k_rows;
    longest = max(longest, kind == kKeyBlocks ? x.n_q : x.n_k);
  }
  if (tid == 0) most = 0;
  classes[tid] = 0;
  bad = __syncthreads_or(bad);
  if (bad) {
    if (list < p.lists && tid == 0) {
      *p.count[list] = 0;
      atomicCAS(p.status, 0, kStatusBadLen);
    }
    return;
  }
  if (list >= p.lists) {
    for (int i = 0; i < p.rests; ++i) {
      const RaggedRest& r = p.rest[i];
      const int32_t* const cu = r.of_keys ? p.cu_k : p.cu_q;
      const int front = cu[0], behind = cu[p.S];
      const long long width = static_cast<long long>(r.heads) * max(r.units, 1), n = (front + static_cast<long long>(r.rows - behind)) * width;
      for (long long at = (list - p.lists) * static_cast<long long>(kPlanThreads) + tid; at < n; at += kPlanRestBlocks * static_cast<long long>(kPlanThreads)) {
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
    return;
  }
  atomicMax(&most, (longest + kBlockM - 1) / kBlockM);
  __syncthreads();
  int shift = 0;
  while ((most >> shift) >= kPlanClasses) ++shift;
  // a group of threads takes a sequence at a time: a warp, or where there are few sequences the CTA
  const int group = p.S >= 32 ? 32 : kPlanThreads, lane = tid & (group - 1);
  auto each = [&](auto&& fn) {
    for (int s = tid / group; s < p.S; s += kPlanThreads / group) {
      const RaggedSequence x(p, s);
      const int n = x.places(kind);
      for (int i = lane; i < n; i += group) fn(x, i, x.cost(kind, i, p.causal) >> shift);
    }
  };
  each([&](const RaggedSequence&, int, int c) { atomicAdd(&classes[c], 1); });
  __syncthreads();
  // where each class begins: behind all higher ones
  const int mine = kPlanClasses - 1 - tid, n = classes[mine];
  int sum = n;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, sum, off);
    if ((tid & 31) >= off) sum += other;
  }
  if ((tid & 31) == 31) warp_sums[tid >> 5] = sum;
  __syncthreads();
  if (tid < 32) {
    int w = warp_sums[tid];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, w, off);
      if (tid >= off) w += other;
    }
    warp_sums[tid] = w;
  }
  __syncthreads();
  if (tid >= 32) sum += warp_sums[(tid >> 5) - 1];
  classes[mine] = sum - n;
  if (tid == kPlanThreads - 1) *p.count[list] = sum;
  __syncthreads();
  int4* const places = p.places[list];
  each([&](const RaggedSequence& x, int i, int c) {
    const int at = atomicAdd(&classes[c], 1);
    places[2 * at] = make_int4(x.q0, x.n_q, x.k0, x.n_k);
    places[2 * at + 1] = make_int4(i, 0, 0, 0);
  });
}

}  // namespace hk
