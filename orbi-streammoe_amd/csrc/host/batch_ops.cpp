// batch_ops.cpp -- routing to experts by a rule, rows grouped by key, and a
// q4 projection of many tokens with adapters: checks and dispatch. Arguments
// are checked before any device work; device arrays cannot be, so the kernels
// bound every index they read from one.
#include <cmath>
#include <limits>
#include <string>

#include "host_util.hpp"
#include "osm_hip.hpp"

namespace osm {
namespace {

// Kernel grids and the rows' indices stay below 2^31.
constexpr std::uint32_t kMaxTokens = 1U << 20;

std::size_t dtype_bytes(std::uint32_t dtype) { return osm_meta_bytes(dtype); }

bool aligned(const void* p, std::size_t bytes) { return reinterpret_cast<std::uintptr_t>(p) % bytes == 0U; }

HipDispatchResult refused(std::string why) {
  HipDispatchResult r;
  r.diagnostic = std::move(why);
  return r;
}

// `bytes` of the context's shared workspace, which does not grow while a
// capture is recording on its stream; nullptr with the reason in *why.
void* workspace(HipComputeContext& context, std::size_t bytes, const char* what, std::string* why) {
  int rc = 0;
  if (bytes > context.shared_workspace_bytes()) {
    int capturing = 0;
    rc = osmd_stream_capturing(context.stream(), &capturing);
    if (rc != 0) return *why = hip_error((std::string(what) + ": stream query failed").c_str(), rc), nullptr;
    if (capturing)
      return *why = std::string(what) + ": the context's workspace is too small for this call and cannot grow during a "
                                        "capture; make the call once before it",
             nullptr;
  }
  void* p = context.shared_workspace(bytes, &rc);
  if (p == nullptr) *why = hip_error((std::string(what) + ": workspace allocation failed").c_str(), rc);
  return p;
}

HipDispatchResult enqueued(int rc, const char* failed, const char* done) {
  HipDispatchResult r;
  r.executed = rc == 0;
  r.diagnostic = rc == 0 ? std::string(done) : hip_error(failed, rc);
  return r;
}

}  // namespace

bool check_route_rule(const HipRouteRule& rule, std::string* diagnostic) noexcept {
  const auto no = [&](const char* why) { return set_diag(diagnostic, why), false; };
  if (rule.expert_count == 0U || rule.expert_count > OSMD_MAX_EXPERTS)
    return no("routing rule: expert_count must be in [1, 1024]");
  if (rule.score > OSMD_SCORE_SIGMOID) return no("routing rule: score must be softmax or sigmoid");
  if (rule.groups == 0U || rule.groups > 64U || rule.expert_count % rule.groups != 0U)
    return no("routing rule: groups must be in [1, 64] and divide expert_count");
  if (rule.top_groups == 0U || rule.top_groups > rule.groups)
    return no("routing rule: top_groups must be in [1, groups]");
  const std::uint32_t per_group = rule.expert_count / rule.groups;
  if (rule.group_score == 0U || rule.group_score > 2U || rule.group_score > per_group)
    return no("routing rule: group_score must be 1 or 2 and at most the experts of a group");
  if (rule.top_k == 0U || rule.top_k > OSMD_ROUTE_MAX_TOP_K || rule.top_k > per_group * rule.top_groups)
    return no("routing rule: top_k must be in [1, 64] and at most the experts of top_groups groups");
  if (!std::isfinite(rule.scale)) return no("routing rule: scale must be finite");
  return true;
}

HipDispatchResult run_hip_route_experts(HipComputeContext& context, const HipRouteRule& rule, const void* logits,
                                        std::uint32_t logits_dtype, std::size_t logits_stride, const float* bias,
                                        std::uint32_t tokens, std::uint32_t* ids, float* weights,
                                        float* mass) noexcept {
  try {
    std::string d;
    if (!check_route_rule(rule, &d)) return refused(d);
    if (logits_dtype > OSM_META_BF16) return refused("routing: logits must be F32, F16 or BF16");
    if (logits_stride == 0U) logits_stride = rule.expert_count;
    if (logits_stride < rule.expert_count) return refused("routing: the logits' stride is below expert_count");
    if (tokens > kMaxTokens) return refused("routing: at most 2^20 tokens a call");
    if (tokens != 0U && (logits == nullptr || ids == nullptr || weights == nullptr))
      return refused("routing needs device logits, ids and weights");
    if (!aligned(logits, dtype_bytes(logits_dtype)) || !aligned(bias, 4U) || !aligned(ids, 4U) ||
        !aligned(weights, 4U) || !aligned(mass, 4U))
      return refused("routing: an array is not aligned to its elements");
    if (!context.activate(&d)) return refused(d);
    if (tokens == 0U) return enqueued(0, "", "HIP routing: no tokens.");
    osmd_route_rule r{};
    r.active = 1U;
    r.score = rule.score;
    r.groups = rule.groups;
    r.top_groups = rule.top_groups;
    r.group_score = rule.group_score;
    r.renormalize = rule.renormalize ? 1U : 0U;
    r.scale = rule.scale;
    r.bias = bias;
    return enqueued(osmd_route_experts(&r, logits, logits_dtype, logits_stride, tokens, rule.expert_count, rule.top_k,
                                       ids, weights, mass, context.stream()),
                    "routing launch failed", "HIP routing enqueued.");
  } catch (...) {
    return HipDispatchResult{};
  }
}

HipDispatchResult run_hip_group_rows(HipComputeContext& context, const std::int32_t* keys, std::uint32_t rows,
                                     std::uint32_t buckets, std::uint32_t* offsets, std::uint32_t* order) noexcept {
  try {
    if (buckets == 0U || buckets > OSMD_GROUP_MAX_BUCKETS) return refused("row grouping: buckets must be in [1, 65535]");
    if (rows > static_cast<std::uint32_t>(std::numeric_limits<std::int32_t>::max()))
      return refused("row grouping: at most 2^31 - 1 rows");
    if (offsets == nullptr || (rows != 0U && (keys == nullptr || order == nullptr)))
      return refused("row grouping needs device keys, offsets and order");
    if (!aligned(keys, 4U) || !aligned(offsets, 4U) || !aligned(order, 4U))
      return refused("row grouping: an array is not aligned to its elements");
    std::string d;
    if (!context.activate(&d)) return refused(d);
    const std::size_t bytes = osmd_group_rows_workspace(rows, buckets);
    void* work = bytes != 0U ? workspace(context, bytes, "row grouping", &d) : nullptr;
    if (bytes != 0U && work == nullptr) return refused(d);
    return enqueued(osmd_group_rows(keys, rows, buckets, offsets, order, work, context.stream()),
                    "row grouping launch failed", "HIP row grouping enqueued.");
  } catch (...) {
    return HipDispatchResult{};
  }
}

HipDispatchResult run_hip_q4_project(HipComputeContext& context, const HipQ4ProjectionWeights& weights, const void* x,
                                     std::uint32_t x_dtype, std::size_t x_stride, void* y, std::uint32_t y_dtype,
                                     std::size_t y_stride, std::uint32_t tokens, const osmd_adapters& adapters,
                                     const std::int32_t* adapter_ids) noexcept {
  try {
    if (!weights.valid()) return refused("Q4 projection weights are not valid");
    if (weights.device() != context.device()) return refused("Q4 projection weights belong to a different device");
    if (x_dtype > OSM_META_BF16 || y_dtype > OSM_META_BF16)
      return refused("Q4 projection: x and y must be F32, F16 or BF16");
    const std::size_t K = weights.in_dim(), N = weights.out_dim();
    if (x_stride == 0U) x_stride = K;
    if (y_stride == 0U) y_stride = N;
    if (x_stride < K || y_stride < N) return refused("Q4 projection: a row stride is below the row's length");
    if (tokens > kMaxTokens) return refused("Q4 projection: at most 2^20 tokens a call");
    if (tokens != 0U && (x == nullptr || y == nullptr)) return refused("Q4 projection needs device input and output");
    if (!aligned(x, dtype_bytes(x_dtype)) || !aligned(y, dtype_bytes(y_dtype)))
      return refused("Q4 projection: an array is not aligned to its elements");
    if (adapters.count != 0U) {
      if (adapters.dtype > OSM_META_BF16) return refused("Q4 projection: adapters must be F32, F16 or BF16");
      if (adapters.max_rank == 0U || adapters.max_rank > OSMD_MAX_ADAPTER_RANK)
        return refused("Q4 projection: adapter ranks must be in [1, 256]");
      if (adapters.count > static_cast<std::uint32_t>(std::numeric_limits<std::int32_t>::max()))
        return refused("Q4 projection: too many adapters");
      if (adapters.a == nullptr || adapters.b == nullptr || (tokens != 0U && adapter_ids == nullptr))
        return refused("Q4 projection: adapters need A, B and the tokens' adapter ids");
      if (!aligned(adapters.a, dtype_bytes(adapters.dtype)) || !aligned(adapters.b, dtype_bytes(adapters.dtype)) ||
          !aligned(adapters.scales, 4U) || !aligned(adapters.ranks, 4U) || !aligned(adapter_ids, 4U))
        return refused("Q4 projection: an adapter array is not aligned to its elements");
    }
    std::string d;
    if (!context.activate(&d)) return refused(d);
    if (tokens == 0U) return enqueued(0, "", "HIP Q4 projection: no tokens.");
    osmd_project_args a{};
    a.w = weights.view();
    a.x = x;
    a.y = y;
    a.x_stride = x_stride;
    a.y_stride = y_stride;
    a.x_dtype = x_dtype;
    a.y_dtype = y_dtype;
    a.tokens = tokens;
    a.adapters = adapters;
    a.adapter_ids = adapter_ids;
    if ((N + 3U) / 4U * ((tokens + 3U) / 4U) > (std::size_t{1} << 30))
      return refused("Q4 projection: out_dim x tokens exceeds the kernels' grids; split the call");
    const std::size_t bytes = osmd_q4_project_workspace(&a);
    void* work = bytes != 0U ? workspace(context, bytes, "Q4 projection", &d) : nullptr;
    if (bytes != 0U && work == nullptr) return refused(d);
    return enqueued(osmd_q4_project(&a, work, context.stream()), "Q4 projection launch failed",
                    "HIP Q4 projection enqueued.");
  } catch (...) {
    return HipDispatchResult{};
  }
}

}  // namespace osm
