// Host side of libhk_attn's attention over ragged batches, forward and backward. C ABI in include/hk_attn.h.
#include <algorithm>
#include <cmath>

#include "hk_host.cuh"
#include "ragged_plan_sm100.cuh"

using namespace hk_host;

namespace {

constexpr long long kMostRows = 1ll << 30;

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
size_t list_bytes(long long places) { return (static_cast<size_t>(places) * 2 * sizeof(int4) + 255) & ~size_t(255); }
// At most so many places has a list over sequences of `rows` rows in all.
long long most_places(int rows, int per, int S) { return rows / per + static_cast<long long>(S); }

int init_ragged(DeviceState* st) {
  std::lock_guard<std::mutex> lock(st->mu);
  if (st->ragged_ready) return HK_OK;
  int rc;
  if ((rc = prepare_fwd_kernel<128, hk::kMaskRagged, true>()) != HK_OK) return rc;
  if ((rc = prepare_fwd_kernel<64, hk::kMaskRagged, true>()) != HK_OK) return rc;
  if ((rc = prepare_bwd_kernels<128, hk::kMaskRagged>()) != HK_OK) return rc;
  if ((rc = prepare_bwd_kernels<64, hk::kMaskRagged>()) != HK_OK) return rc;
  st->ragged_ready = true;
  return HK_OK;
}

// What both directions ask of their arguments. Rows may be none, and pointers to none null.
int check_ragged(std::initializer_list<const void*> q_rows, std::initializer_list<const void*> k_rows, const int32_t* cu_q, const int32_t* cu_k,
                 const float* lse, int S, int Tq, int Tk, int H, int H_KV, int D, std::initializer_list<const long long*> strides) {
  if (!cu_q || !cu_k || S <= 0 || Tq < 0 || Tk < 0 || H <= 0 || H_KV <= 0) return HK_EINVAL;
  if (D != 64 && D != 128) return HK_EUNSUPPORTED;
  if (H % H_KV != 0 || S > 65535 || Tq > kMostRows || Tk > kMostRows) return HK_EINVAL;
  if (!aligned4(cu_q) || !aligned4(cu_k) || (Tq > 0 && !lse) || !aligned4(lse)) return HK_EINVAL;
  for (const void* p : q_rows)
    if ((Tq > 0 && !p) || !aligned16(p)) return HK_EINVAL;
  for (const void* p : k_rows)
    if ((Tk > 0 && !p) || !aligned16(p)) return HK_EINVAL;
  for (const long long* st : strides) {
    if (!st) return HK_EINVAL;
    for (int i = 0; i < 2; ++i)
      if (st[i] <= 0 || st[i] % 8 != 0 || st[i] >= (1ll << 39)) return HK_EINVAL;
  }
  // work items are indexed with int
  if (most_places(Tq, hk::kBlockM, S) * H > 0x3fffffffll || most_places(Tk, hk::kBlockN, S) * H_KV > 0x3fffffffll) return HK_EINVAL;
  return HK_OK;
}

struct RowStrides {
  long long st[3];  // as make_bnhd_map takes them, of the one batch element that has all rows
  explicit RowStrides(const long long* s) : st{s[0], s[0], s[1]} {}
};

}  // namespace

extern "C" {

size_t hk_attn_fwd_ragged_workspace_bytes(int S, int q_rows) {
  return S > 0 && q_rows >= 0 ? 256 + list_bytes(most_places(q_rows, hk::kBlockM, S)) : 0;
}

int hk_attn_fwd_ragged(const void* q, const void* k, const void* v, void* o, float* lse, const int32_t* cu_seqlens_q,
                       const int32_t* cu_seqlens_k, int S, int q_rows, int k_rows, int H, int H_KV, int D, const long long* q_strides,
                       const long long* k_strides, const long long* v_strides, int causal, float softmax_scale, int fill_rest,
                       void* workspace, size_t workspace_bytes, int device, void* cuda_stream) {
  int rc = check_ragged({q, o}, {k, v}, cu_seqlens_q, cu_seqlens_k, lse, S, q_rows, k_rows, H, H_KV, D, {q_strides, k_strides, v_strides});
  if (rc != HK_OK) return rc;
  if (!workspace || workspace_bytes < hk_attn_fwd_ragged_workspace_bytes(S, q_rows) || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return HK_EWORKSPACE;
  if (q_rows == 0) return HK_OK;
  DeviceState* st = nullptr;
  DeviceScope scope;
  if ((rc = scope.enter(device, &st)) != HK_OK || (rc = init_ragged(st)) != HK_OK) return rc;
  const RowStrides qs(q_strides), ks(k_strides), vs(v_strides);
  const long long contiguous[2] = {1ll * H * D, D};
  const RowStrides os(contiguous);
  CUtensorMap tq, tk, tv, to;
  if ((rc = make_bnhd_map(&tq, q, 1, q_rows, H, D, qs.st)) != HK_OK) return rc;
  if ((rc = make_bnhd_map(&to, o, 1, q_rows, H, D, os.st)) != HK_OK) return rc;
  tk = tv = tq;  // of no keys nothing is loaded
  if (k_rows > 0 && (rc = make_bnhd_map(&tk, k, 1, k_rows, H_KV, D, ks.st)) != HK_OK) return rc;
  if (k_rows > 0 && (rc = make_bnhd_map(&tv, v, 1, k_rows, H_KV, D, vs.st)) != HK_OK) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const int G = H / H_KV;
  hk::RaggedPlanParams plan = {};
  hk::FwdParams p = {};
  p.pair_heads = G % 2 == 0 ? 1 : 0;
  plan.cu_q = cu_seqlens_q, plan.cu_k = cu_seqlens_k;
  plan.S = S, plan.q_rows = q_rows, plan.k_rows = k_rows, plan.causal = causal != 0;
  plan.lists = 1;
  plan.kind[0] = plan.kind[1] = p.pair_heads ? hk::kQueryTiles : hk::kQueryPairs;
  plan.count[0] = static_cast<int*>(workspace);
  plan.places[0] = reinterpret_cast<int4*>(static_cast<char*>(workspace) + 256);
  if (fill_rest) {
    plan.rests = 2;
    plan.rest[0] = {o, 1ll * H * D, D, H, q_rows, D / 8, 0};
    plan.rest[1] = {lse, 1, q_rows, H, q_rows, 0, 0};
  }
  plan.status = st->status;
  const int plan_grid = plan.lists + (plan.rests ? hk::kPlanRestThreads / hk::kPlanThreads : 0);
  HK_CUDA(hk::launch_dependent(true, hk::ragged_plan_kernel, unsigned(plan_grid), hk::kPlanThreads, 0, stream, plan));
  p.o = static_cast<__nv_bfloat16*>(o);
  p.lse = lse;
  p.B = 1, p.N = q_rows, p.NK = k_rows, p.H = H, p.H_KV = H_KV;
  p.group_units = p.group_items = p.rounds_per_group = 1;
  hk::set_item_decode(p);
  p.per_place = H_KV * p.inner;
  p.fd_per_place = hk::FastDiv(p.per_place);
  p.causal = causal != 0;
  p.plan_count = plan.count[0];
  p.plan = plan.places[0];
  p.scale = softmax_scale > 0.f ? softmax_scale : 1.0f / std::sqrt(float(D));
  p.scale_log2 = p.scale * 1.4426950408889634f;
  p.status = st->status;
  const long long most = most_places(q_rows, p.pair_heads ? hk::kBlockM : 2 * hk::kBlockM, S) * p.per_place;
  const int grid = int(std::min<long long>(most, st->sm_count));
  auto* fn = D == 128 ? hk::attn_fwd_kernel<128, hk::kMaskRagged, true> : hk::attn_fwd_kernel<64, hk::kMaskRagged, true>;
  const int smem = D == 128 ? hk::FwdSmem<128, true>::kDynBytes : hk::FwdSmem<64, true>::kDynBytes;
  HK_CUDA(hk::launch_dependent(true, fn, unsigned(grid), hk::kFwdThreads, smem, stream, tq, tk, tv, to, p));
  g_launches.fetch_add(2, std::memory_order_relaxed);
  return HK_OK;
}

size_t hk_attn_bwd_ragged_workspace_bytes(int S, int q_rows, int k_rows) {
  if (S <= 0 || q_rows < 0 || k_rows < 0) return 0;
  return 256 + list_bytes(most_places(q_rows, hk::kBlockM, S)) + list_bytes(most_places(k_rows, hk::kBlockN, S));
}

int hk_attn_bwd_ragged(const void* q, const void* k, const void* v, const void* o, const void* d_o, const float* lse, float* delta,
                       void* dq, void* dk, void* dv, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int S, int q_rows,
                       int k_rows, int H, int H_KV, int D, const long long* q_strides, const long long* k_strides,
                       const long long* v_strides, const long long* dq_strides, const long long* dk_strides, const long long* dv_strides,
                       int causal, float softmax_scale, int fill_rest, void* workspace, size_t workspace_bytes, int device,
                       void* cuda_stream) {
  int rc = check_ragged({q, o, d_o, dq}, {k, v, dk, dv}, cu_seqlens_q, cu_seqlens_k, lse, S, q_rows, k_rows, H, H_KV, D,
                        {q_strides, k_strides, v_strides, dq_strides, dk_strides, dv_strides});
  if (rc != HK_OK) return rc;
  if ((q_rows > 0 && !delta) || !aligned4(delta)) return HK_EINVAL;
  if (1ll * q_rows * H > 0x7fffffffll) return HK_EINVAL;  // rows are indexed with int
  if (!workspace || workspace_bytes < hk_attn_bwd_ragged_workspace_bytes(S, q_rows, k_rows) || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return HK_EWORKSPACE;
  if (q_rows == 0 && k_rows == 0) return HK_OK;
  DeviceState* st = nullptr;
  DeviceScope scope;
  if ((rc = scope.enter(device, &st)) != HK_OK || (rc = init_ragged(st)) != HK_OK) return rc;
  const RowStrides qs(q_strides), ks(k_strides), vs(v_strides), dqs(dq_strides), dks(dk_strides), dvs(dv_strides);
  const long long contiguous[2] = {1ll * H * D, D};
  const RowStrides os(contiguous);
  CUtensorMap tq, tk, tv, tdo;
  if (q_rows > 0 && (rc = make_bnhd_map(&tq, q, 1, q_rows, H, D, qs.st)) != HK_OK) return rc;
  if (q_rows > 0 && (rc = make_bnhd_map(&tdo, d_o, 1, q_rows, H, D, os.st)) != HK_OK) return rc;
  if (k_rows > 0 && (rc = make_bnhd_map(&tk, k, 1, k_rows, H_KV, D, ks.st)) != HK_OK) return rc;
  if (k_rows > 0 && (rc = make_bnhd_map(&tv, v, 1, k_rows, H_KV, D, vs.st)) != HK_OK) return rc;
  if (q_rows == 0) tq = tdo = tk;  // of no rows nothing is loaded
  if (k_rows == 0) tk = tv = tq;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  hk::RaggedPrepParams prep = {};
  hk::RaggedPlanParams& plan = prep.plan;
  plan.cu_q = cu_seqlens_q, plan.cu_k = cu_seqlens_k;
  plan.S = S, plan.q_rows = q_rows, plan.k_rows = k_rows, plan.causal = causal != 0;
  plan.lists = 2;
  plan.kind[0] = hk::kKeyBlocks, plan.kind[1] = hk::kQueryTiles;
  plan.count[0] = static_cast<int*>(workspace), plan.count[1] = plan.count[0] + 1;
  plan.places[0] = reinterpret_cast<int4*>(static_cast<char*>(workspace) + 256);
  const long long blocks = most_places(k_rows, hk::kBlockN, S), tiles = most_places(q_rows, hk::kBlockM, S);
  plan.places[1] = reinterpret_cast<int4*>(reinterpret_cast<char*>(plan.places[0]) + list_bytes(blocks));
  if (fill_rest) {
    plan.rests = 3;
    plan.rest[0] = {dq, dqs.st[1], dqs.st[2], H, q_rows, D / 8, 0};
    plan.rest[1] = {dk, dks.st[1], dks.st[2], H_KV, k_rows, D / 8, 1};
    plan.rest[2] = {dv, dvs.st[1], dvs.st[2], H_KV, k_rows, D / 8, 1};
  }
  plan.status = st->status;
  hk::BwdParams p = {};
  p.lse = lse;
  p.delta = delta;
  p.dq = static_cast<__nv_bfloat16*>(dq);
  p.dk = static_cast<__nv_bfloat16*>(dk);
  p.dv = static_cast<__nv_bfloat16*>(dv);
  p.dq_stride_b = dqs.st[0], p.dq_stride_n = dqs.st[1], p.dq_stride_h = dqs.st[2];
  p.dk_stride_b = dks.st[0], p.dk_stride_n = dks.st[1], p.dk_stride_h = dks.st[2];
  p.dv_stride_b = dvs.st[0], p.dv_stride_n = dvs.st[1], p.dv_stride_h = dvs.st[2];
  p.B = 1, p.N = q_rows, p.NK = k_rows, p.H = H, p.H_KV = H_KV;
  p.G = H / H_KV;
  p.split = 1;
  p.scale = softmax_scale > 0.f ? softmax_scale : 1.0f / std::sqrt(float(D));
  p.scale_log2 = p.scale * 1.4426950408889634f;
  p.causal = causal != 0;
  p.status = st->status;
  const bool d128 = D == 128;
  prep.q = static_cast<const __nv_bfloat16*>(q), prep.k = static_cast<const __nv_bfloat16*>(k), prep.v = static_cast<const __nv_bfloat16*>(v);
  prep.o = static_cast<const __nv_bfloat16*>(o), prep.d_o = static_cast<const __nv_bfloat16*>(d_o);
  prep.lse = lse, prep.delta = delta;
  for (int i = 0; i < 2; ++i) prep.q_stride[i] = qs.st[i + 1], prep.k_stride[i] = ks.st[i + 1], prep.v_stride[i] = vs.st[i + 1];
  prep.H = H, prep.rows = q_rows * H;
  prep.scale_log2 = p.scale_log2;
  prep.fd_h = hk::FastDiv(H), prep.fd_g = hk::FastDiv(p.G);
  const int per_block = hk::row_pass_rows(D / 8);
  if (q_rows > 0) {
    prep.few_blocks = int((hk::ragged_few_tiles(S, q_rows, causal != 0) * H + 7) / 8);
    prep.row_blocks = int((1ll * q_rows * H + per_block - 1) / per_block);
  }
  const long long prep_grid = plan.lists + 1ll * prep.few_blocks + prep.row_blocks + (plan.rests ? hk::kPlanRestThreads / hk::kPrepThreads : 0);
  HK_CUDA(hk::launch_dependent(true, d128 ? hk::ragged_prep_kernel<128> : hk::ragged_prep_kernel<64>, unsigned(prep_grid), hk::kPrepThreads,
                               0, stream, prep));
  g_launches.fetch_add(1, std::memory_order_relaxed);
  const int smem = d128 ? hk::BwdSmem<128>::kDynBytes : hk::BwdSmem<64>::kDynBytes;
  if (k_rows > 0) {
    p.plan_count = plan.count[0], p.plan = plan.places[0];
    p.per_place = H_KV;
    p.fd_per_place = hk::FastDiv(H_KV);
    auto* fn = d128 ? hk::attn_bwd_dkdv_kernel<128, hk::kMaskRagged, false> : hk::attn_bwd_dkdv_kernel<64, hk::kMaskRagged, false>;
    const int grid = int(std::min<long long>(blocks * H_KV, st->sm_count));
    HK_CUDA(hk::launch_dependent(true, fn, unsigned(grid), hk::kBwdThreads, smem, stream, tq, tk, tv, tdo, p));
    g_launches.fetch_add(1, std::memory_order_relaxed);
  }
  if (q_rows > 0) {
    p.plan_count = plan.count[1], p.plan = plan.places[1];
    p.per_place = H;
    p.fd_per_place = hk::FastDiv(H);
    p.fd_inner = hk::FastDiv(p.G);
    const Span out(dq, dqs.st, 1, q_rows, H, D);
    const long long stats = 4ll * H * q_rows;
    const bool beside = k_rows > 0 && !out.meets({q, qs.st, 1, q_rows, H, D}) && !out.meets({d_o, os.st, 1, q_rows, H, D}) &&
                        !out.meets({k, ks.st, 1, k_rows, H_KV, D}) && !out.meets({v, vs.st, 1, k_rows, H_KV, D}) &&
                        !out.meets({lse, stats}) && !out.meets({delta, stats});
    p.dq_waits = !beside;
    auto* fn = d128 ? hk::attn_bwd_dq_kernel<128, hk::kMaskRagged> : hk::attn_bwd_dq_kernel<64, hk::kMaskRagged>;
    const int grid = int(std::min<long long>(tiles * H, st->sm_count));
    HK_CUDA(hk::launch_dependent(true, fn, unsigned(grid), hk::kBwdThreads, smem, stream, tq, tk, tv, tdo, p));
    g_launches.fetch_add(1, std::memory_order_relaxed);
  }
  return HK_OK;
}

}  // extern "C"
