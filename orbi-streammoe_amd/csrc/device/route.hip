// route.hip -- routing to experts by a rule (softmax or sigmoid scores, a
// balance bias, groups, top-k, renormalised weights), and rows grouped by a
// small key.
//
// Routing, token t with logits l_e (one wavefront per token, lane i holds the
// PER consecutive experts from i * PER on):
//   score   s_e = exp(l_e - max l) / sum exp(l - max l), or 1 / (1 + exp(-l_e))
//   choice  c_e = s_e + bias_e, in fp64
//   groups  of E / groups consecutive experts; a group's score is its best
//           choice or the sum of its best two; the best top_groups groups
//           stay (ties: the lower group)
//   picks   the top_k best choices of the groups that stay (ties: the lower
//           id); without a bias the logits themselves are ranked, which is
//           the same order in exact arithmetic
//   weights scale * s / (renormalize ? sum of the picks' s : 1)
// Choices are compared in fp64: two scores that differ by less than an fp32
// rounding still rank the way their values do.
#include "device_common.hpp"

namespace {

using namespace osmk;

enum : int { kSrcPlanes = 3, kSrcPlanes64 = 4 };  // after OSM_META_*: router GEMM planes

constexpr int kRouteRuleWaves = 4;  // tokens per workgroup
constexpr uint64_t kKeyMasked = 0x000FFFFFFFFFFFFFull;  // ordered key of -infinity
constexpr uint32_t kMaxGroups = 64;

struct RuleView {
  const void* logits;
  size_t stride;
  const float* planes;
  const double* planes64;
  uint32_t parts, tokens, experts, top_k;
  osmd_route_rule rule;
  uint32_t* ids;
  float* weights;
  float* mass;
  // Layer form: the rest of what a selection publishes.
  float* logits_out;
  float* gate_out;
  const uint8_t* const* expert_table;
  const uint8_t* shared_expert;
  const uint8_t* fallback;
  const uint8_t** slot_ptrs;
  uint32_t nslot;
  uint32_t* stats;
};

// Double bits as an unsigned key that orders like the value; -0 as +0.
__device__ __forceinline__ uint64_t ordered_key64(double d) {
  const uint64_t u = __builtin_bit_cast(uint64_t, d + 0.0);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

__device__ __forceinline__ double readlane_d(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u), lane));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane));
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}

// Token t's logits, experts base .. base + PER - 1 (clamped: every load in
// bounds).
template <int PER, int SRC>
__device__ __forceinline__ void load_logits(const RuleView& v, uint32_t t, uint32_t base, float (&l)[PER]) {
  const uint32_t E = v.experts;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint32_t e = base + j < E ? base + j : E - 1u;
    if constexpr (SRC == kSrcPlanes || SRC == kSrcPlanes64) {
      // The router GEMM's K ranges, added in plane order (fp64 planes: rounded once).
      const size_t ps = static_cast<size_t>(v.tokens) * (E + 1u);
      const size_t o = static_cast<size_t>(t) * (E + 1u) + e;
      if constexpr (SRC == kSrcPlanes64) {
        double s = 0.0;
        for (uint32_t p = 0; p < v.parts; ++p) s += v.planes64[p * ps + o];
        l[j] = static_cast<float>(s);
      } else {
        float s = v.planes[o];
        for (uint32_t p = 1; p < v.parts; ++p) s += v.planes[p * ps + o];
        l[j] = s;
      }
      if (base + j < E) v.logits_out[static_cast<size_t>(t) * E + e] = l[j];
    } else {
      l[j] = meta_at<SRC>(v.logits, t * v.stride + e);
    }
  }
}

template <int PER, int SRC>
__global__ __launch_bounds__(kRouteRuleWaves* kWave) void route_rule_kernel(RuleView v) {
  __shared__ double choice_lds[kRouteRuleWaves][PER * kWave];
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t t = blockIdx.x * kRouteRuleWaves + wave;
  if (t >= v.tokens) return;  // no barrier below: waves are on their own
  const uint32_t E = v.experts, k = v.top_k, base = lane * PER;
  const osmd_route_rule& rule = v.rule;
  float l[PER];
  load_logits<PER, SRC>(v, t, base, l);

  // An expert whose logit is NaN or -infinity is not available.
  bool avail[PER];
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    avail[j] = base + j < E && l[j] > -INFINITY;
    if (avail[j]) m = fmaxf(m, l[j]);
  }
  double s[PER];
  if (rule.score == OSMD_SCORE_SOFTMAX) {
    m = wave_max(m);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      // The largest logit's term is 1 also where it is infinite.
      s[j] = !avail[j] ? 0.0 : l[j] == m ? 1.0 : exp(static_cast<double>(l[j]) - static_cast<double>(m));
      sum += s[j];
    }
    sum = wave_sum_d(sum);
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] = avail[j] ? s[j] / sum : 0.0;
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] = avail[j] ? 1.0 / (1.0 + exp(-static_cast<double>(l[j]))) : 0.0;
  }

  uint64_t key[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const double c = rule.bias ? s[j] + static_cast<double>(rule.bias[base + j < E ? base + j : E - 1u])
                               : static_cast<double>(l[j]);
    key[j] = base + j >= E ? 0ull : avail[j] && c > -INFINITY ? ordered_key64(c) : kKeyMasked;
  }
  if (rule.groups > 1u) {
    const uint32_t per_group = E / rule.groups;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const double c = rule.bias && base + j < E ? s[j] + static_cast<double>(rule.bias[base + j]) : s[j];
      choice_lds[wave][base + j] = key[j] > kKeyMasked ? c : -INFINITY;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    double gs = -INFINITY;
    if (lane < rule.groups) {
      double first = -INFINITY, second = -INFINITY;
      for (uint32_t i = 0; i < per_group; ++i) {
        const double c = choice_lds[wave][lane * per_group + i];
        second = fmax(second, fmin(first, c));
        first = fmax(first, c);
      }
      gs = rule.group_score == 2u ? first + second : first;
      if (gs != gs) gs = -INFINITY;
    }
    uint32_t better = 0;
    for (uint32_t g = 0; g < rule.groups; ++g) {
      const double o = readlane_d(gs, static_cast<int>(g));
      better += (o > gs || (o == gs && g < lane)) ? 1u : 0u;
    }
    const uint64_t kept = __ballot(lane < rule.groups && better < rule.top_groups);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t g = (base + j < E ? base + j : E - 1u) / per_group;
      if (base + j < E && !((kept >> g) & 1ull)) key[j] = kKeyMasked;
    }
  }

  // One pick a round: the lane's best (the lowest of equal ones), then the
  // first lane that has the wavefront's best.
  uint32_t my_id = 0;
  double my_s = 0.0, sum = 0.0;
  for (uint32_t r = 0; r < k; ++r) {
    uint64_t best = key[0];
    int bj = 0;
#pragma unroll
    for (int j = 1; j < PER; ++j)
      if (key[j] > best) best = key[j], bj = j;
    const uint32_t hi = wave_max_u32(static_cast<uint32_t>(best >> 32));
    const bool at = static_cast<uint32_t>(best >> 32) == hi;
    const uint32_t lo = wave_max_u32(at ? static_cast<uint32_t>(best) : 0u);
    const uint64_t who = __ballot(at && static_cast<uint32_t>(best) == lo);
    const int owner = __builtin_ctzll(who);
    double ps = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (j == bj) {
        ps = key[j] > kKeyMasked ? s[j] : 0.0;
        if (static_cast<int>(lane) == owner) key[j] = 0ull;
      }
    const uint32_t id = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(base + bj), owner));
    ps = readlane_d(ps, owner);
    sum += ps;
    if (lane == r) my_id = id, my_s = ps;
  }
  if (lane < k) {
    const double w = rule.renormalize ? (sum > 0.0 ? my_s / sum : 0.0) : my_s;
    v.ids[static_cast<size_t>(t) * k + lane] = my_id;
    v.weights[static_cast<size_t>(t) * k + lane] = static_cast<float>(static_cast<double>(rule.scale) * w);
    if (v.slot_ptrs) {
      const uint8_t* b = v.expert_table ? v.expert_table[my_id] : nullptr;
      v.slot_ptrs[static_cast<size_t>(t) * v.nslot + lane] = b ? b : v.fallback;
    }
  }
  if (lane == 0) {
    if (v.mass) v.mass[t] = static_cast<float>(sum);
    if (v.slot_ptrs && v.nslot > k) v.slot_ptrs[static_cast<size_t>(t) * v.nslot + k] = v.shared_expert;
    if (v.stats) atomicAdd(v.stats, 1u);
    if constexpr (SRC == kSrcPlanes || SRC == kSrcPlanes64) {
      if (v.nslot > k) {  // the shared gate, column E of the planes
        const size_t ps = static_cast<size_t>(v.tokens) * (E + 1u), o = static_cast<size_t>(t) * (E + 1u) + E;
        double g = 0.0;
        for (uint32_t p = 0; p < v.parts; ++p)
          g += SRC == kSrcPlanes64 ? v.planes64[p * ps + o] : static_cast<double>(v.planes[p * ps + o]);
        v.gate_out[t] = 1.0f / (1.0f + expf(-static_cast<float>(g)));
      }
    }
  }
}

template <int SRC>
int launch_rule(const RuleView& v, hipStream_t st) {
  const unsigned grid = (v.tokens + kRouteRuleWaves - 1) / kRouteRuleWaves;
  const uint32_t per = (v.experts + kWave - 1) / kWave;
  auto go = [&](auto kernel) { kernel<<<grid, kRouteRuleWaves * kWave, 0, st>>>(v); };
  if (per <= 1)
    go(route_rule_kernel<1, SRC>);
  else if (per <= 2)
    go(route_rule_kernel<2, SRC>);
  else if (per <= 4)
    go(route_rule_kernel<4, SRC>);
  else if (per <= 8)
    go(route_rule_kernel<8, SRC>);
  else
    go(route_rule_kernel<16, SRC>);
  return launch_status();
}

bool rule_ok(const osmd_route_rule& r, uint32_t experts, uint32_t top_k) {
  return experts > 0 && experts <= OSMD_MAX_EXPERTS && r.score <= OSMD_SCORE_SIGMOID && r.groups > 0 &&
         r.groups <= kMaxGroups && experts % r.groups == 0 && r.top_groups > 0 && r.top_groups <= r.groups &&
         r.group_score > 0 && r.group_score <= 2u && r.group_score <= experts / r.groups && top_k > 0 &&
         top_k <= OSMD_ROUTE_MAX_TOP_K && top_k <= experts / r.groups * r.top_groups;
}

// ---- rows grouped by key -------------------------------------------------------
// A stable counting sort in one launch: every workgroup owns a run of
// buckets (the rows outside every bucket are one more) and reads all keys
// twice, so nothing is exchanged between workgroups. Each of its 16
// wavefronts takes a contiguous run of rows. First it counts the keys below
// the workgroup's buckets and, per bucket, its own; then, from the sums of
// the wavefronts before it, it places its rows in order. Among 64 rows the
// owned ones are taken bucket by bucket (a ballot each).
constexpr int kGroupWaves = 16;
constexpr uint32_t kGroupMaxOwn = 256;

__global__ __launch_bounds__(kGroupWaves* kWave) void group_rows_kernel(const int32_t* __restrict__ keys, uint32_t n,
                                                                        uint32_t buckets, uint32_t own,
                                                                        uint32_t* __restrict__ offsets,
                                                                        uint32_t* __restrict__ order) {
  __shared__ uint32_t cnt[kGroupWaves][kGroupMaxOwn];
  __shared__ uint32_t below_lds[kGroupWaves];
  __shared__ uint32_t start[kGroupMaxOwn];
  const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const uint32_t b0 = blockIdx.x * own;
  const uint32_t nb = b0 + own <= buckets + 1u ? own : buckets + 1u - b0;
  for (uint32_t i = tid; i < kGroupWaves * kGroupMaxOwn; i += blockDim.x) (&cnt[0][0])[i] = 0u;
  __syncthreads();
  const uint32_t run = ((n + kGroupWaves - 1u) / kGroupWaves + kWave - 1u) / kWave * kWave;
  const uint32_t r0 = wave * run < n ? wave * run : n;
  const uint32_t r1 = n - r0 < run ? n : r0 + run;
  volatile uint32_t* mine = cnt[wave];
  // Bucket of row r (buckets: outside); rows past the run own nothing.
  auto bucket = [&](uint32_t r) -> uint32_t {
    if (r >= r1) return 0xFFFFFFFFu;
    const uint32_t key = static_cast<uint32_t>(keys[r]);
    return key < buckets ? key : buckets;
  };
  uint32_t below = 0;
  for (uint32_t r = r0; r < r1; r += kWave) {
    const uint32_t b = bucket(r + lane);
    below += static_cast<uint32_t>(__popcll(__ballot(b < b0)));
    uint64_t left = __ballot(b - b0 < nb);
    while (left) {
      const uint32_t lb = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b), __builtin_ctzll(left)));
      const uint64_t same = __ballot(b == lb);
      if (lane == 0) mine[lb - b0] = mine[lb - b0] + static_cast<uint32_t>(__popcll(same));
      left &= ~same;
    }
  }
  if (lane == 0) below_lds[wave] = below;
  __syncthreads();
  if (tid < nb) {
    uint32_t s = 0;
    for (int w = 0; w < kGroupWaves; ++w) {
      const uint32_t c = cnt[w][tid];
      cnt[w][tid] = s;  // rows of this bucket in the wavefronts before
      s += c;
    }
    start[tid] = s;
  }
  __syncthreads();
  if (tid == 0) {
    uint32_t s = 0;
    for (int w = 0; w < kGroupWaves; ++w) s += below_lds[w];
    for (uint32_t i = 0; i < nb; ++i) {
      const uint32_t c = start[i];
      start[i] = s;
      s += c;
    }
  }
  __syncthreads();
  if (tid < nb) offsets[b0 + tid] = start[tid];
  for (uint32_t r = r0; r < r1; r += kWave) {
    const uint32_t b = bucket(r + lane);
    uint64_t left = __ballot(b - b0 < nb);
    while (left) {
      const uint32_t lb = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b), __builtin_ctzll(left)));
      const uint64_t same = __ballot(b == lb);
      const uint32_t first = mine[lb - b0];
      if (b == lb) order[start[lb - b0] + first + __popcll(same & ((1ull << lane) - 1ull))] = r + lane;
      if (lane == 0) mine[lb - b0] = first + static_cast<uint32_t>(__popcll(same));
      left &= ~same;
    }
  }
}

}  // namespace

extern "C" {

int osmd_route_experts(const osmd_route_rule* rule, const void* logits, uint32_t dtype, size_t stride, uint32_t tokens,
                       uint32_t experts, uint32_t top_k, uint32_t* ids, float* weights, float* mass, osmd_stream s) {
  if (!rule_ok(*rule, experts, top_k) || stride < experts) return static_cast<int>(hipErrorInvalidValue);
  RuleView v{};
  v.logits = logits;
  v.stride = stride;
  v.tokens = tokens;
  v.experts = experts;
  v.top_k = top_k;
  v.rule = *rule;
  v.ids = ids;
  v.weights = weights;
  v.mass = mass;
  const hipStream_t st = static_cast<hipStream_t>(s);
  switch (dtype) {
    case OSM_META_F32: return launch_rule<OSM_META_F32>(v, st);
    case OSM_META_F16: return launch_rule<OSM_META_F16>(v, st);
    case OSM_META_BF16: return launch_rule<OSM_META_BF16>(v, st);
    default: return static_cast<int>(hipErrorInvalidValue);
  }
}

int osmd_moe_select_rule(const osmd_moe_args* a, osmd_stream s) {
  if (!rule_ok(a->rule, a->expert_count, a->top_k)) return static_cast<int>(hipErrorInvalidValue);
  RuleView v{};
  v.logits = a->logits;
  v.stride = a->expert_count;
  v.planes = a->logit_planes;
  v.planes64 = a->logit_planes64;
  v.parts = a->logit_parts;
  v.tokens = a->tokens;
  v.experts = a->expert_count;
  v.top_k = a->top_k;
  v.rule = a->rule;
  v.ids = a->ids;
  v.weights = a->weights;
  v.mass = a->mass;
  v.logits_out = a->logits;
  v.gate_out = a->shared_gate;
  v.expert_table = a->expert_table;
  v.shared_expert = a->shared_expert;
  v.fallback = a->fallback_blob;
  v.slot_ptrs = a->slot_ptrs;
  v.nslot = a->top_k + ((a->flags & OSMD_MOE_SHARED) ? 1u : 0u);
  v.stats = a->route_stats;
  const hipStream_t st = static_cast<hipStream_t>(s);
  if (a->logit_planes64) return launch_rule<kSrcPlanes64>(v, st);
  if (a->logit_planes) return launch_rule<kSrcPlanes>(v, st);
  return launch_rule<OSM_META_F32>(v, st);
}

int osmd_group_rows(const int32_t* keys, uint32_t rows, uint32_t buckets, uint32_t* offsets, uint32_t* order,
                    osmd_stream s) {
  if (buckets == 0 || buckets > OSMD_GROUP_MAX_BUCKETS || rows > 0x7FFFFFFFu)
    return static_cast<int>(hipErrorInvalidValue);
  const uint32_t own = (buckets + 1u + 255u) / 256u;  // at most 256 workgroups
  const uint32_t grid = (buckets + 1u + own - 1u) / own;
  group_rows_kernel<<<grid, kGroupWaves * kWave, 0, static_cast<hipStream_t>(s)>>>(keys, rows, buckets, own, offsets, order);
  return launch_status();
}

}  // extern "C"
