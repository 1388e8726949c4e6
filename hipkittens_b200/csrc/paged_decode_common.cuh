// What the paged decode kernels share, and the host side of all of them: parameters, live pages, how contexts are spread over CTAs,
// the workspace, and copies and fragment loads.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "dependent_launch.cuh"
#include "sm100_ptx.cuh"

namespace hk {

constexpr int kPageTokens = 16;
constexpr int kDecodeD = 128;                         // of the calls without a window
constexpr int kChunkPagesMin = 32;                    // pages per CTA: 32 (512 tokens) or 64 (1024 tokens),
constexpr int kChunkPagesMax = 64;                    // chosen per launch by decode_pick_chunk_pages
template <int D>
struct DecodeRing {
  static constexpr int kStages = 3 * (128 / D);          // pages in flight per warp: as many bytes for either head dimension
  static constexpr int kSlabBytes = kPageTokens * D * 2;    // one page of one kv head: 4 KB at D = 128
  static constexpr int kStageBytes = 2 * kSlabBytes;     // K slab + V slab
};
constexpr int decode_smem_bytes(int warps) { return warps * DecodeRing<128>::kStages * DecodeRing<128>::kStageBytes; }  // 96 or 192 KB
constexpr int kMaxCombineSplits = 256;

// 3 is the backward kernels' kStatusSmemAlign; kStatusBadPos: a position outside rotary tables
enum : int { kStatusBadPage = 2, kStatusBadLen = 4, kStatusBadPos = 5 };

struct DecodeParams {
  const __nv_bfloat16* q;        // [S,1,H,D]
  const __nv_bfloat16* k_pages;  // [P,16,H_KV,D]
  const __nv_bfloat16* v_pages;
  const int32_t* block_table;    // [S,max_pages]
  const int32_t* ctx_lens;       // [S]
  __nv_bfloat16* o;              // [S,1,H,D]
  float* lse;                    // [S,H,1,1]
  int S, H, H_KV, max_pages, num_pages;
  int chunk_pages;               // pages per CTA (kChunkPagesMin or kChunkPagesMax)
  float scale, scale_log2;
  void* workspace;
  int* status;
  // With a window: the query, at position ctx - 1, sees the last `window` keys and the first `sinks`
  int window, sinks;
  int span_pages;                // the most pages that hold such keys
};

// The pages of a context that hold keys the query sees, counted without those between the sinks and the window.
struct LivePages {
  int sink_pages, skip;  // the first sink_pages are pages 0, 1, ...; those behind them are `skip` further on
  int total;
  int first_key;         // of the window
  __host__ __device__ LivePages(int ctx, int window, int sinks) {
    first_key = ctx > window ? ctx - window : 0;
    const int first_page = first_key / kPageTokens;
    sink_pages = (sinks + kPageTokens - 1) / kPageTokens;
    if (sink_pages > first_page) sink_pages = first_page;
    skip = first_page - sink_pages;
    total = (ctx + kPageTokens - 1) / kPageTokens - skip;
  }
  __host__ __device__ int page(int i) const { return i < sink_pages ? i : i + skip; }
};
// The most of them that any context in a table of max_pages has.
inline int decode_span_pages(int max_pages, int window, int sinks) {
  const long long most = (1ll * sinks + kPageTokens - 1) / kPageTokens + (1ll * window + kPageTokens - 2) / kPageTokens + 1;
  return most < max_pages ? int(most) : max_pages;
}

// The workspace is laid out for the smaller chunk size (the larger split count), whichever size a launch uses.
__host__ __device__ inline int decode_max_splits(int max_pages) {
  return (max_pages + kChunkPagesMin - 1) / kChunkPagesMin;
}
// Chunks: 1024-token chunks halve the partial results and were measured 4-5 % faster on the 64-sequence workload
// (94.5 % vs 90.7 % of the copy bandwidth); 512-token chunks keep more CTAs in flight when the batch is
// small. Take the large chunk when it still gives every SM two rounds of two CTAs.
inline int decode_pick_chunk_pages(int S, int H_KV, int max_pages, int sm_count) {
  const long long ctas = 1ll * S * H_KV * ((max_pages + kChunkPagesMax - 1) / kChunkPagesMax);
  return ctas >= 4ll * sm_count ? kChunkPagesMax : kChunkPagesMin;
}
// What the device holds at once of the split kernel, by the size of its clusters (filled by prepare_decode_kernels).
struct DecodeLimits {
  int sm_count = 0;
  int clusters4[kMaxCluster + 1] = {};  // clusters of so many CTAs of 4 warps (two per SM)
  int clusters8 = 0;                    // clusters of kMaxCluster CTAs of 8 warps (one per SM)
};

// How the context of one (sequence, kv head), a unit, is spread: over a cluster of CTAs of 4 or 8 warps, or, with
// cluster = 0, over chunks that a second kernel combines. The host knows the block table's width and not the contexts;
// clusters spread each context evenly, so the width matters only for the most that one CTA may meet.
//  * Clusters as large as keeps all units in one wave, and no larger: a cluster behind the first wave starts when a whole
//    one fits, and one size too many costs more than it gives. us, chunks / clusters of that size / of another, H_KV 8 unless
//    said: 1 x 3250 tokens 10.4 / 7.6 (16) / 8.0 (8); 4 x 750 10.1 / 6.3 (8) / 6.7 (4), 11.4 (16); 8 x 2500 20.6 / 17.0
//    (4) / 22.6 (2), 19.0 (8); 40 x 1650 of H_KV 1 13.3 / 10.9 (6) / 14.1 (7).
//  * How much of one context a CTA may meet is bounded: the table may be as wide as it is for one long context among short
//    ones, which its own cluster then reads alone (12.5 us per 1000 tokens of a CTA of 4 warps, 5.5 with 8), where chunks
//    would spread it over the GPU. The lines are where that costs the one long context about as much as batches of equal
//    lengths gain. us, chunks / this, one context as long as the table beside others of 100 tokens, then all that long, then
//    all a quarter of that:
//    CTAs of 4 warps in clusters, 64 pages each: 8 x 48 pages of H_KV 8 10.8 / 10.4, 22.3 / 16.6, 11.7 / 6.7; 8 x
//    4096 10.8 / 12.4, 30.5 / 25.3, 11.9 / 7.2; 64 x 4096 of H_KV 1 9.8 / 11.9, 30.2 / 25.1, 12.3 / 7.3; behind the line 8 x 8192
//    12.3 / 19.8, 53.7 / 45.2, 14.0 / 10.0.
//    CTAs of their own of 8 warps (units for more than a wave in clusters of 3), 96 pages: 16 x 1408 10.8 / 10.7, 20.1 /
//    15.3, 9.1 / 5.6; 32 x 1536 11.1 / 11.4, 43.2 / 36.7, 10.6 / 10.4; behind the line 12 x 2560 10.4 / 16.5, 29.1 / 24.5, 12.3 /
//    7.2, 32 x 2048 10.3 / 14.0, 52.7 / 45.9, 12.5 / 11.9.
//    Of 4 warps, while one wave of those with 8 is not enough, 64 pages: 24 x 1024 10.6 / 11.2, 22.8 / 19.7, 8.1 / 6.3; 32 x 1024
//    10.6 / 12.5, 30.7 / 24.8, 8.6 / 6.3 (8 warps 8.9, 27.6, 9.1).
//    With units for more than two waves of those of 8 they are the better ones throughout, and the chunks are slower with the one
//    long context too: 80 pages, 64 x 1152 15.2 / 12.8, 57.6 / 49.9, 16.3 / 12.9 (8 warps 13.4, 55.2, 19.0).
//    One wave of CTAs of 8 warps also serves 160 pages where the chunks need more than two waves: then all but the one long
//    context gain most (18 x 2560 10.8 / 16.5, 40.9 / 32.6, 13.7 / 7.1, lengths evenly up to 2560 21.5 / 18.4).
//  * Clusters of several waves gain up to 5 % on long contexts (64 x 4350: 182 / 174 in clusters of 4), but where most of the
//    table's width is empty their idle CTAs cost more than those of the chunks (64 x 300 tokens in tables for 8192: 24 / 47),
//    so those stay in chunks.
//  * Few units with long contexts: 16 CTAs of 4 warps fall behind the chunks from some 700 tokens each on (1 x 14000 13.5 /
//    14.7); up to 6 units the CTAs can have 8 warps (H_KV 1, 1 x 16000: 11.7 / 11.0, 4 warps 12.5; below 4096 tokens 4
//    warps are better, 1 x 2000: 9.4 / 5.4, 8 warps 6.2).
struct DecodeShape {
  int cluster, warps;
};
inline DecodeShape decode_pick_shape(int S, int H_KV, int max_pages, const DecodeLimits& lim) {
  const long long units = 1ll * S * H_KV;
  constexpr DecodeShape kChunks{0, 4};
  int cluster = kMaxCluster, warps = 4;
  while (cluster > 1 && lim.clusters4[cluster] < units) --cluster;
  if (cluster < 3) {
    cluster = 1;
    const bool one_wave = units <= lim.sm_count, two_waves = units <= 2ll * lim.sm_count;
    const bool many_chunks = units * max_pages > 4ll * lim.sm_count * kChunkPagesMin;
    warps = one_wave || (two_waves && max_pages > 64) ? 8 : 4;
    if (max_pages > (one_wave && many_chunks ? 160 : two_waves ? 96 : 80)) return kChunks;
  } else if (max_pages > 256 && units <= lim.clusters8) {
    cluster = kMaxCluster;
    warps = 8;
    if (max_pages > 64 * cluster) return kChunks;
  } else if (max_pages > (cluster == kMaxCluster ? 44 : 64) * cluster) {
    return kChunks;
  }
  const int useful = (max_pages + warps - 1) / warps;  // a page per warp
  return {cluster < useful ? cluster : useful, warps};
}
// With a window, `span` pages are the most that any context holds, and most contexts of a serving batch hold all of them: a CTA may
// meet up to 320 (5120 tokens), and what one long context beside short ones loses is bounded by the window (75 us there, in chunks
// 15). Otherwise as above; a unit of its own has 8 warps while all of them are one wave and 4 from there on.
// us, chunks of 64 pages / clusters or CTAs of 4 warps (size) / of 8, H64/8 D128 unless said, contexts longer than the window:
// 64 contexts, window 512 36.0 / 31.2 (1) / 39.2 (1); 2048 100.9 / 88.1 (1) / 96.5 (1); 4096 182 / 164 (1) / 172 (1); 32, 2048 55.0 / 46.7
// (1) / 48.2 (1); 16, 2048 33.0 / 29.1 (2) / 25.9 (1); 8, 4096 33.2 / 27.3 (4) / 27.7 (2); 8, 1024 21.0 / 12.3 (4) / 12.5 (2); 4, 1024 20.7 / 9.1
// (8) / 9.1 (4); H32/8, 1 context, 4096 20.4 / 10.2 (16) / 10.4 (8); D = 64, 33 contexts of H48/8, 500 12.7 / 10.3 (1) / 13.5 (1); H64/8,
// 64 contexts, 2048 61.4 / 51.2 (1) / 56.4 (1). Few units with long windows stay in chunks: H1, 1 context, 32768 17.1 (of 32 pages) /
// 33.2 (16) / 22.1 (16); H32/8 D = 64, 2 contexts, 16384 18.8 / 19.3 (12) / 19.7 (6).
inline DecodeShape decode_pick_window_shape(int S, int H_KV, int span, const DecodeLimits& lim) {
  const long long units = 1ll * S * H_KV;
  constexpr DecodeShape kChunks{0, 4};
  constexpr int kMost = 320;
  int cluster = kMaxCluster, warps = 4;
  while (cluster > 1 && lim.clusters4[cluster] < units) --cluster;
  if (cluster < 3) {
    cluster = 1;
    warps = units <= lim.sm_count ? 8 : 4;
    if (span > kMost) return kChunks;
  } else if (span > 256 && units <= lim.clusters8) {
    cluster = kMaxCluster;
    warps = 8;
    if (span > 64 * cluster) return kChunks;
  } else if (span > (cluster == kMaxCluster ? 44 : kMost) * cluster) {
    return kChunks;
  }
  const int useful = (span + warps - 1) / warps;  // a page per warp
  return {cluster < useful ? cluster : useful, warps};
}
// Shapes the two kernels can be launched for: the combine kernel holds one weight per split in shared memory
// (kMaxCombineSplits of them, counted for the smaller chunk size so that either chunk choice fits), and sequences
// and kv heads are grid dimensions y and z.
inline bool decode_shape_supported(int S, int H_KV, int max_pages) {
  return S > 0 && S <= 65535 && H_KV > 0 && H_KV <= 65535 && max_pages > 0 &&
         decode_max_splits(max_pages) <= kMaxCombineSplits;
}
// Workspace: partial O as fp32 [S][H][splits][D], then, from the next multiple of 256 bytes, (m, l) pairs as fp32 [S][H][splits][2].
inline size_t decode_workspace_bytes(int S, int H, int D, int max_pages, int page_size, bool any_d = false) {
  if (S <= 0 || S > 65535 || H <= 0 || page_size != kPageTokens || max_pages <= 0) return 0;
  if (D != kDecodeD && !(any_d && D == 64)) return 0;
  if (decode_max_splits(max_pages) > kMaxCombineSplits) return 0;
  const size_t splits = decode_max_splits(max_pages);
  const size_t o_bytes = size_t(S) * H * splits * D * sizeof(float);
  const size_t ml_bytes = size_t(S) * H * splits * 2 * sizeof(float);
  return ((o_bytes + 255) & ~size_t(255)) + ((ml_bytes + 255) & ~size_t(255));
}

namespace dec {

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The same, or 16 zero bytes and nothing read.
__device__ __forceinline__ void cp_async16_if(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2,
                                                  uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
using ptx::mma_16816;

}  // namespace dec

}  // namespace hk
