// Host side of libhk_attn's 8-bit paged cache: append, read back and decode. C ABI in include/hk_attn.h.
#include <algorithm>
#include <cmath>

#include "hk_host.cuh"
#include "paged_decode_fp8_sm100.cuh"
#include "paged_kv_fp8_sm100.cuh"

using namespace hk_host;

namespace {

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// Everything that the three entries have in common. `st` is entered only if all of it is right.
int fp8_cache(hk::Fp8Cache& c, const void* k_pages, const void* v_pages, const float* k_scales, const float* v_scales,
              const int32_t* block_table, int S, int H_KV, int D, int page_size, int max_pages, int num_pages) {
  if (!k_pages || !v_pages || !k_scales || !v_scales || !block_table) return HK_EINVAL;
  if (S <= 0 || H_KV <= 0 || D <= 0 || max_pages <= 0 || num_pages <= 0) return HK_EINVAL;
  if (page_size != hk::kPageTokens || (D != 64 && D != 128)) return HK_EUNSUPPORTED;
  if (S > 65535 || H_KV > 65535 || max_pages > 0x7fffffff / hk::kPageTokens || num_pages > 0x7fffffff / hk::kPageTokens) return HK_EINVAL;
  if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned4(k_scales) || !aligned4(v_scales) || !aligned4(block_table)) return HK_EINVAL;
  c.k_pages = static_cast<uint8_t*>(const_cast<void*>(k_pages));
  c.v_pages = static_cast<uint8_t*>(const_cast<void*>(v_pages));
  c.k_scales = const_cast<float*>(k_scales);
  c.v_scales = const_cast<float*>(v_scales);
  c.block_table = block_table;
  c.S = S, c.H_KV = H_KV, c.max_pages = max_pages, c.num_pages = num_pages;
  return HK_OK;
}

// The units of 16 tokens of a call, times what each takes; false if that is too many for an int.
bool fp8_units(long long units, int per_unit, int* count) {
  const long long n = units * per_unit;
  *count = static_cast<int>(n);
  return n <= 0x7ffffff0ll;
}

}  // namespace

extern "C" {

int hk_paged_kv_append_fp8(const void* k_new, const void* v_new, void* k_pages, void* v_pages, float* k_scales, float* v_scales,
                           const int32_t* block_table, const int32_t* start_pos, const int32_t* cu_seqlens, const void* sin,
                           const void* cos, int S, int T, int H_KV, int D, const long long* k_strides, const long long* v_strides,
                           int rotary_dim, int table_rows, int flags, int page_size, int max_pages_per_seq, int num_pages,
                           int device, void* cuda_stream) {
  hk::AppendFp8Params p = {};
  int rc = fp8_cache(p.c, k_pages, v_pages, k_scales, v_scales, block_table, S, H_KV, D, page_size, max_pages_per_seq, num_pages);
  if (rc != HK_OK) return rc;
  if (!k_new || !v_new || !start_pos || !k_strides || !v_strides || T <= 0 || (!sin) != (!cos)) return HK_EINVAL;
  if (flags & ~HK_FP8_TABLE_F32) return HK_EINVAL;
  if (!aligned16(k_new) || !aligned16(v_new) || !aligned4(start_pos) || !aligned4(cu_seqlens) || !aligned16(sin) || !aligned16(cos))
    return HK_EINVAL;
  for (int i = cu_seqlens ? 1 : 0; i < 3; ++i)
    for (const long long* st : {k_strides, v_strides})
      if (st[i] <= 0 || st[i] % 8 != 0 || st[i] >= (1ll << 39)) return HK_EINVAL;
  if (sin) {
    if (rotary_dim <= 0) rotary_dim = D;
    if (rotary_dim % 16 != 0 || rotary_dim > D) return HK_EUNSUPPORTED;
    if (table_rows <= 0) return HK_EINVAL;
  }
  const long long units = cu_seqlens ? T / hk::kPageTokens + 2ll * S : S * ((T + 30ll) / hk::kPageTokens);
  int warps = std::min(hk::kFp8AppendWarps, H_KV);
  int blocks;  // with a head a warp
  if (!fp8_units(units, 2 * ((H_KV + warps - 1) / warps), &blocks)) return HK_EINVAL;
  DeviceState* st = nullptr;
  DeviceScope scope;
  if ((rc = scope.enter(device, &st)) != HK_OK) return rc;
  // Several heads a warp where there is more than the device holds at once: the next head's tokens come in meanwhile, and a page's tables
  // serve as many. us, 1 / 2 / 4 heads of a warp, rotated prompts of as many bytes as 29,000 tokens of H_KV 8 D128: H_KV 8 D128 40.6 / 33.7 /
  // 38, H_KV 4 D128 40.2 / 35.4 / 41, H_KV 8 D64 - / 41 / 37, H_KV 4 D64 56 / 42 / 38; a token for each of 64 sequences, H_KV 8 D128: 3.6 /
  // 4.4. One head of 128 takes 52.
  if (blocks > 4 * st->sm_count) {
    p.turns = std::min(hk::fp8_append_turns(D), H_KV);
    warps = std::min(hk::kFp8AppendWarps, (H_KV + p.turns - 1) / p.turns);
  } else {
    p.turns = 1;
  }
  const int groups = (H_KV + p.turns * warps - 1) / (p.turns * warps);
  p.c.status = st->status;
  p.rows.cu = cu_seqlens;
  p.rows.T = T;
  p.rows.fd_units = hk::FastDiv(static_cast<int>((T + 30ll) / hk::kPageTokens));
  p.k_new = static_cast<const __nv_bfloat16*>(k_new);
  p.v_new = static_cast<const __nv_bfloat16*>(v_new);
  for (int i = 0; i < 3; ++i) p.k_stride[i] = k_strides[i], p.v_stride[i] = v_strides[i];
  if (cu_seqlens) p.k_stride[0] = p.v_stride[0] = 0;
  p.start_pos = start_pos;
  p.cos = cos, p.sin = sin;
  p.R = rotary_dim, p.table_rows = table_rows;
  p.fd_groups2 = hk::FastDiv(2 * groups);
  p.fd_groups = hk::FastDiv(groups);
  p.rotation = !sin ? hk::kFp8Plain : flags & HK_FP8_TABLE_F32 ? hk::kFp8TableF32 : hk::kFp8TableBf16;
  auto* fn = D == 128 ? sin ? hk::paged_kv_append_fp8_kernel<128, true> : hk::paged_kv_append_fp8_kernel<128, false>
                      : sin ? hk::paged_kv_append_fp8_kernel<64, true> : hk::paged_kv_append_fp8_kernel<64, false>;
  const int smem = hk::fp8_append_smem(D, sin, warps, p.turns);
  HK_CUDA(hk::launch_dependent(true, fn, unsigned(units * 2 * groups), warps * 32, smem, static_cast<cudaStream_t>(cuda_stream), p));
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return HK_OK;
}

int hk_paged_kv_read_fp8(const void* k_pages, const void* v_pages, const float* k_scales, const float* v_scales,
                         const int32_t* block_table, const int32_t* ctx_lens, const int32_t* cu_seqlens, void* k_out, void* v_out,
                         int S, int rows, int H_KV, int D, int zero_rest, int page_size, int max_pages_per_seq, int num_pages,
                         int device, void* cuda_stream) {
  hk::ReadFp8Params p = {};
  int rc = fp8_cache(p.c, k_pages, v_pages, k_scales, v_scales, block_table, S, H_KV, D, page_size, max_pages_per_seq, num_pages);
  if (rc != HK_OK) return rc;
  if (!k_out || !v_out || (!ctx_lens) == (!cu_seqlens) || rows <= 0) return HK_EINVAL;
  if (!aligned16(k_out) || !aligned16(v_out) || !aligned4(ctx_lens) || !aligned4(cu_seqlens)) return HK_EINVAL;
  const long long per_seq = (rows + 15ll) / hk::kPageTokens;
  if (!fp8_units(cu_seqlens ? rows / hk::kPageTokens + S + 1ll : S * per_seq, H_KV, &p.warps)) return HK_EINVAL;
  DeviceState* st = nullptr;
  DeviceScope scope;
  if ((rc = scope.enter(device, &st)) != HK_OK) return rc;
  p.c.status = st->status;
  p.rows.cu = cu_seqlens;
  p.rows.T = rows;
  p.rows.fd_units = hk::FastDiv(static_cast<int>(per_seq));
  p.ctx_lens = ctx_lens;
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.zero_rest = zero_rest;
  p.fd_heads = hk::FastDiv(H_KV);
  auto* fn = D == 128 ? hk::paged_kv_read_fp8_kernel<128> : hk::paged_kv_read_fp8_kernel<64>;
  HK_CUDA(hk::launch_dependent(true, fn, unsigned((p.warps + 7ll) / 8), 256, 0, static_cast<cudaStream_t>(cuda_stream), p));
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return HK_OK;
}

size_t hk_attn_paged_decode_fp8_workspace_bytes(int S, int H_KV, int D) {
  if (S <= 0 || S > 65535 || H_KV <= 0 || H_KV > 65535 || 1ll * S * H_KV > 0x3fffffff || (D != 64 && D != 128)) return 0;
  return hk::decode_fp8_workspace_bytes(S, H_KV, D);
}

int hk_attn_paged_decode_fp8(const void* q, const void* k_pages, const void* v_pages, const float* k_scales, const float* v_scales,
                             const int32_t* block_table, const int32_t* ctx_lens, void* o, float* lse, int S, int H, int H_KV, int D,
                             int page_size, int max_pages_per_seq, int num_pages, int window, int sinks, float softmax_scale,
                             void* workspace, size_t workspace_bytes, int device, void* cuda_stream) {
  hk::Fp8Cache c = {};
  int rc = fp8_cache(c, k_pages, v_pages, k_scales, v_scales, block_table, S, H_KV, D, page_size, max_pages_per_seq, num_pages);
  if (rc != HK_OK) return rc;
  if (!q || !ctx_lens || !o || !lse || H <= 0 || window < 0 || sinks < 0 || (window == 0 && sinks != 0)) return HK_EINVAL;
  if (H % H_KV != 0) return HK_EINVAL;
  if (H / H_KV > 8) return HK_EUNSUPPORTED;  // the heads of a group sit in the 8 columns of one product
  if (!aligned16(q) || !aligned16(o) || !aligned4(ctx_lens) || !aligned4(lse)) return HK_EINVAL;
  const size_t need = hk_attn_paged_decode_fp8_workspace_bytes(S, H_KV, D);
  if (need == 0) return HK_EINVAL;
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)) return HK_EWORKSPACE;
  DeviceState* st = nullptr;
  DeviceScope scope;
  if ((rc = scope.enter(device, &st)) != HK_OK) return rc;
  {
    std::lock_guard<std::mutex> lock(st->mu);
    if (!st->decode_fp8_ready) {
      rc = hk::prepare_decode_fp8_kernels(g_cuda_err, sizeof(g_cuda_err), st->sm_count, &st->decode_fp8);
      if (rc != HK_OK) return rc;
      st->decode_fp8_ready = true;
    }
  }
  CUtensorMap tk, tv;
  if ((rc = make_code_map(&tk, k_pages, num_pages, H_KV, D)) != HK_OK) return rc;
  if ((rc = make_code_map(&tv, v_pages, num_pages, H_KV, D)) != HK_OK) return rc;
  hk::DecodeFp8Params p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k_scales = c.k_scales, p.v_scales = c.v_scales;
  p.block_table = block_table;
  p.ctx_lens = ctx_lens;
  p.o = static_cast<__nv_bfloat16*>(o);
  p.lse = lse;
  p.S = S, p.H = H, p.H_KV = H_KV;
  p.max_pages = max_pages_per_seq, p.num_pages = num_pages;
  p.scale = softmax_scale > 0.f ? softmax_scale : 1.0f / std::sqrt(float(D));
  p.scale_log2 = p.scale * 1.4426950408889634f;
  p.workspace = workspace;
  p.status = st->status;
  const int capacity = max_pages_per_seq * hk::kPageTokens;  // no context is longer
  p.window = window == 0 ? capacity : std::min(window, capacity);
  p.sinks = std::min(sinks, capacity);
  p.span_pages = window == 0 ? max_pages_per_seq : hk::decode_span_pages(max_pages_per_seq, window, sinks);
  int launched = 0;
  const cudaError_t e = hk::launch_paged_decode_fp8(tk, tv, p, D, window != 0, st->decode_fp8, static_cast<cudaStream_t>(cuda_stream), &launched);
  g_launches.fetch_add(launched, std::memory_order_relaxed);
  if (e != cudaSuccess) return cuda_fail(e, "fp8 decode launch");
  return HK_OK;
}

int hk_selftest_decode_fp8_parts(int first, int group, int last_group, int row_groups, int H_KV) {
  if (row_groups <= 0 || H_KV <= 0 || H_KV > 65535 || 1ll * row_groups * H_KV > 0x3fffffff) return HK_EINVAL;
  return hk::decode_fp8_parts_valid({first, group, last_group, 0}, row_groups, H_KV) ? 1 : 0;
}

}  // extern "C"
