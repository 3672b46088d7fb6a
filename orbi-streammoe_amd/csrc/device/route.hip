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
// What bounds it is issue: 16,383 tokens of 512 experts with a bias and 10
// picks take 30 us, 7 of them the 34 MB, 1.1 a pick (two instructions a key:
// the greatest of the wavefront is found from the high words of the keys, and
// taken out by the masks that found it), the rest exponentials. One token takes
// 5 us, a launch and the chain of picks.
#include "device_common.hpp"

namespace {

using namespace osmk;

enum : int { kSrcPlanes = 3, kSrcPlanes64 = 4 };  // after OSM_META_*: router GEMM planes

constexpr int kRouteRuleWaves = 4;  // tokens per workgroup
// High word of the key of an expert that may not be chosen: that of fp64
// -infinity, below that of fp32 -infinity.
constexpr uint32_t kHiMasked = 0x000FFFFFu;
constexpr uint32_t kMaxGroups = 64;

struct RuleView {
  const void* logits;
  size_t stride;
  const float* planes;
  const double* planes64;
  uint32_t parts, tokens, experts, top_k;
  osmd_route_rule rule;
  bool logits_wide, bias_wide;  // chunks of wide_chunk values can be read at once
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

__device__ __forceinline__ double readlane_d(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u), lane));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane));
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}

// e^x to an fp64 rounding or two, x a difference of two fp32 values; 0 and
// infinity beyond the range, no special values. With n the integer next to
// x / ln 2 and r = x - n ln 2 (|r| <= 0.35), the terms of the series of e^r
// up to r^12 / 12! leave out less than 2^-52. Straight-line, so that the terms
// of a lane's experts share their constants and fill each other's latency.
__device__ __forceinline__ double exp_d(double x) {
  constexpr double kLn2Hi = 0x1.62e42fefap-1;       // 36 bits: n * kLn2Hi is exact
  constexpr double kLn2Lo = 0x1.cf79abc9e3b3ap-40;  // ln 2 - kLn2Hi
  x = fmin(fmax(x, -1100.0), 1100.0);
  const double n = __builtin_rint(x * 1.4426950408889634);
  const double r = fma(n, -kLn2Lo, fma(n, -kLn2Hi, x));
  double p = 1.0 / 479001600.0;
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return __builtin_ldexp(p, static_cast<int>(n));
}

__device__ __forceinline__ double sigmoid_d(float l) { return 1.0 / (1.0 + exp_d(-static_cast<double>(l))); }

// LDS that other lanes of the wavefront wrote before is read after.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Values of a lane that one load can take: 16 bytes or all PER.
template <int SRC>
__host__ __device__ constexpr int wide_chunk(int per) {
  constexpr int most = SRC == OSM_META_F32 ? 4 : 8;
  return per < most ? per : most;
}

// Experts base .. base + PER - 1 of one row of E values (clamped: every load
// in bounds). Loads of one value cost as many cache lines each as wide ones:
// at 16,383 tokens of 512 experts the logits and the bias took 30 us that way
// and take 8 wide.
template <int PER, int SRC>
__device__ __forceinline__ void load_experts(const void* p, size_t row, uint32_t base, uint32_t E, bool wide,
                                             float (&l)[PER]) {
  constexpr int kChunk = wide_chunk<SRC>(PER), kWords = kChunk * (SRC == OSM_META_F32 ? 4 : 2) / 4;
  if constexpr (kChunk >= 4) {
    if (wide) {
      typedef uint32_t words __attribute__((ext_vector_type(kWords)));
      words w[PER / kChunk];
#pragma unroll
      for (int c = 0; c < PER / kChunk; ++c) {
        const uint32_t e = base + c * kChunk < E ? base + c * kChunk : E - kChunk;
        w[c] = *reinterpret_cast<const words*>(static_cast<const char*>(p) + (row + e) * (SRC == OSM_META_F32 ? 4u : 2u));
      }
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int c = j / kChunk, i = j % kChunk;
        if constexpr (SRC == OSM_META_F32)
          l[j] = __uint_as_float(w[c][i]);
        else
          l[j] = SRC == OSM_META_BF16 ? bf16_to_f32(static_cast<uint16_t>(w[c][i / 2] >> (i % 2 * 16)))
                                      : f16_to_f32(static_cast<uint16_t>(w[c][i / 2] >> (i % 2 * 16)));
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) l[j] = meta_at<SRC>(p, row + (base + j < E ? base + j : E - 1u));
}

// Token t's logits, experts base .. base + PER - 1.
template <int PER, int SRC>
__device__ __forceinline__ void load_logits(const RuleView& v, uint32_t t, uint32_t base, float (&l)[PER]) {
  const uint32_t E = v.experts;
  if constexpr (SRC != kSrcPlanes && SRC != kSrcPlanes64) {
    load_experts<PER, SRC>(v.logits, t * v.stride, base, E, v.logits_wide, l);
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t e = base + j < E ? base + j : E - 1u;
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
    }
  }
}

template <int PER, int SRC>
__global__ __launch_bounds__(kRouteRuleWaves* kWave) void route_rule_kernel(RuleView v) {
  __shared__ double lds[kRouteRuleWaves][PER * kWave];  // choices, then scores
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t t = blockIdx.x * kRouteRuleWaves + wave;
  if (t >= v.tokens) return;  // no barrier below: waves are on their own
  const uint32_t E = v.experts, k = v.top_k, base = lane * PER;
  const osmd_route_rule& rule = v.rule;
  float l[PER], bias[PER];
  load_logits<PER, SRC>(v, t, base, l);
  if (rule.bias) {
    load_experts<PER, OSM_META_F32>(rule.bias, 0u, base, E, v.bias_wide, bias);
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) bias[j] = 0.0f;
  }

  // An expert whose logit is NaN or -infinity is not available.
  bool avail[PER];
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    avail[j] = base + j < E && l[j] > -INFINITY;
    m = avail[j] && l[j] > m ? l[j] : m;
  }
  // Scores. Without a bias a softmax's are left unnormalised until its picks
  // are known, and a sigmoid's are not needed before, unless groups add them.
  double s[PER], inverse = 1.0;
  const bool late = rule.score == OSMD_SCORE_SIGMOID && !rule.bias && rule.groups == 1u;
  if (rule.score == OSMD_SCORE_SOFTMAX) {
    m = wave_max(m);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const double e = exp_d(static_cast<double>(l[j]) - static_cast<double>(m));
      s[j] = !avail[j] ? 0.0 : l[j] == m ? 1.0 : e;  // 1 also where the largest is infinite
      sum += s[j];
    }
    inverse = 1.0 / wave_sum_d(sum);
    if (rule.bias) {
#pragma unroll
      for (int j = 0; j < PER; ++j) s[j] = avail[j] ? s[j] * inverse : 0.0;
      inverse = 1.0;
    }
  } else if (late) {
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] = static_cast<double>(l[j]);
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const double one = sigmoid_d(l[j]);
      s[j] = avail[j] ? one : 0.0;
    }
  }

  // Keys that order like the choices (no choice is -0), or like the logits
  // where there is no bias (then all low words are 0).
  uint32_t hi[PER], lo[PER];
  if (rule.bias) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const double c = s[j] + static_cast<double>(bias[j]);
      const uint64_t u = __builtin_bit_cast(uint64_t, c);
      const uint32_t sign = static_cast<uint32_t>(static_cast<int32_t>(u >> 32) >> 31);
      const bool masked = !avail[j] || !(c > -INFINITY);
      hi[j] = masked ? kHiMasked : static_cast<uint32_t>(u >> 32) ^ (sign | 0x80000000u);
      lo[j] = masked ? 0u : static_cast<uint32_t>(u) ^ sign;
    }
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t u = __float_as_uint(l[j] + 0.0f);
      hi[j] = avail[j] ? u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u) : kHiMasked;
      lo[j] = 0u;
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) hi[j] = base + j < E ? hi[j] : 0u;
  double* const mine = lds[wave];
  if (rule.groups > 1u) {
    const uint32_t per_group = E / rule.groups;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      mine[base + j] = hi[j] > kHiMasked ? s[j] + static_cast<double>(bias[j]) : -INFINITY;
    wave_lds_fence();
    // 2^shift lanes take a group together, then all know its score.
    const uint32_t shift = static_cast<uint32_t>(__builtin_clz(rule.groups - 1u)) - 26u;
    const uint32_t g = lane >> shift, part = lane - (g << shift);
    double first = -INFINITY, second = -INFINITY;
    if (g < rule.groups)
      for (uint32_t i = part; i < per_group; i += 1u << shift) {
        const double c = mine[g * per_group + i];
        second = fmax(second, fmin(first, c));
        first = fmax(first, c);
      }
    for (int x = 1; x < 1 << shift; x <<= 1) {
      const double f2 = __shfl_xor(first, x, kWave), s2 = __shfl_xor(second, x, kWave);
      second = fmax(fmin(first, f2), fmax(second, s2));
      first = fmax(first, f2);
    }
    double gs = rule.group_score == 2u ? first + second : first;
    if (gs != gs) gs = -INFINITY;
    uint32_t better = 0;
    for (uint32_t o = 0; o < rule.groups; ++o) {
      const double other = readlane_d(gs, static_cast<int>(o << shift));
      better += (other > gs || (other == gs && o < g)) ? 1u : 0u;
    }
    const uint64_t kept = __ballot(g < rule.groups && better < rule.top_groups);
    uint32_t mg = base / per_group, left = (mg + 1u) * per_group - base;  // of the lane's first expert
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const bool masked = base + j < E && !((kept >> (mg << shift)) & 1ull);
      hi[j] = masked ? kHiMasked : hi[j];
      lo[j] = masked ? 0u : lo[j];
      const bool next = --left == 0u;
      mg += next ? 1u : 0u;
      left = next ? per_group : left;
    }
    wave_lds_fence();
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) mine[base + j] = s[j];
  wave_lds_fence();

  // One pick a round: the wavefront's greatest high word; where several
  // experts share it, the greatest low word and then the lowest id.
  uint32_t my_id = 0, my_top = 0;
  for (uint32_t r = 0; r < k; ++r) {
    uint32_t best = hi[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) best = max(best, hi[j]);
    const uint32_t top = wave_max_u32(best);
    uint64_t at[PER], any = 0, twice = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      at[j] = __ballot(hi[j] == top);
      twice |= any & at[j];
      any |= at[j];
    }
    if (twice | (any & (any - 1ull))) {
      if (rule.bias) {
        uint32_t low = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) low = max(low, hi[j] == top ? lo[j] : 0u);
        low = wave_max_u32(low);
        any = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) any |= at[j] = __ballot(hi[j] == top && lo[j] == low);
      }
      any &= ~any + 1ull;
      uint64_t one = any;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        at[j] &= one;
        one &= ~at[j];
      }
    }
    uint32_t id = base;
#pragma unroll
    for (int j = PER - 1; j >= 0; --j) {
      const bool mine_j = __builtin_amdgcn_inverse_ballot_w64(at[j]);
      id = mine_j ? base + j : id;
      hi[j] = mine_j ? 0u : hi[j];
    }
    id = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(id), __builtin_ctzll(any)));
    my_id = lane == r ? id : my_id;
    my_top = lane == r ? top : my_top;
  }
  double my_s = 0.0;
  if (my_top > kHiMasked) {  // pick `lane` is one that may be chosen
    my_s = mine[my_id];
    my_s = late ? sigmoid_d(static_cast<float>(my_s)) : my_s * inverse;
  }
  const double sum = wave_sum_d(my_s);
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

template <int PER, int SRC>
int launch_rule_per(RuleView v, hipStream_t st) {
  auto aligned = [](const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
  constexpr uint32_t kChunk = wide_chunk<SRC>(PER), kBias = wide_chunk<OSM_META_F32>(PER);
  v.logits_wide = v.experts % kChunk == 0 && v.stride % kChunk == 0 &&
                  aligned(v.logits, kChunk * (SRC == OSM_META_F32 ? 4u : 2u));
  v.bias_wide = v.experts % kBias == 0 && aligned(v.rule.bias, kBias * 4u);
  const unsigned grid = (v.tokens + kRouteRuleWaves - 1) / kRouteRuleWaves;
  route_rule_kernel<PER, SRC><<<grid, kRouteRuleWaves * kWave, 0, st>>>(v);
  return launch_status();
}

template <int SRC>
int launch_rule(const RuleView& v, hipStream_t st) {
  const uint32_t per = (v.experts + kWave - 1) / kWave;
  if (per <= 1) return launch_rule_per<1, SRC>(v, st);
  if (per <= 2) return launch_rule_per<2, SRC>(v, st);
  if (per <= 4) return launch_rule_per<4, SRC>(v, st);
  if (per <= 8) return launch_rule_per<8, SRC>(v, st);
  return launch_rule_per<16, SRC>(v, st);
}

bool rule_ok(const osmd_route_rule& r, uint32_t experts, uint32_t top_k) {
  return experts > 0 && experts <= OSMD_MAX_EXPERTS && r.score <= OSMD_SCORE_SIGMOID && r.groups > 0 &&
         r.groups <= kMaxGroups && experts % r.groups == 0 && r.top_groups > 0 && r.top_groups <= r.groups &&
         r.group_score > 0 && r.group_score <= 2u && r.group_score <= experts / r.groups && top_k > 0 &&
         top_k <= OSMD_ROUTE_MAX_TOP_K && top_k <= experts / r.groups * r.top_groups;
}

// ---- rows grouped by key -------------------------------------------------------
// A stable counting sort, in two forms. Up to kOneLaunchRows rows, or very
// many buckets: one launch, in which every workgroup owns a run of buckets
// (the rows outside every bucket are one more) and goes through all keys, so
// nothing is exchanged between workgroups. Each of its 16 wavefronts takes a
// contiguous run of rows: first it counts the keys below the workgroup's
// buckets and, per bucket, its own; then, from the sums of the wavefronts
// before it, it places its rows in order. Counts of up to 4 buckets are
// scalars, a ballot each; more are in LDS, a ballot for each owned bucket that
// 64 rows hold. kRowsAhead loads of 64 keys are in flight; up to
// 16 x 64 x kRowsAhead rows are read once and kept. What bounds it is a launch
// (3.2 us for 64 rows), then that every compute unit sees every key: 36 us for
// 81,920 rows of 256 buckets, which two launches do in 10.
constexpr int kGroupWaves = 16;
constexpr uint32_t kGroupMaxOwn = 256;
constexpr uint32_t kRowsAhead = 16;

// OWN: buckets of a workgroup where at most 4, else 0 (`own` of them).
template <int OWN>
__global__ __launch_bounds__(kGroupWaves* kWave) void group_rows_kernel(const int32_t* __restrict__ keys, uint32_t n,
                                                                        uint32_t buckets, uint32_t own,
                                                                        uint32_t* __restrict__ offsets,
                                                                        uint32_t* __restrict__ order) {
  constexpr uint32_t kOwn = OWN ? OWN : kGroupMaxOwn;
  __shared__ uint32_t cnt[kGroupWaves][kOwn];
  __shared__ uint32_t below_lds[kGroupWaves];
  __shared__ uint32_t start[kOwn];
  const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const uint32_t b0 = blockIdx.x * own;
  const uint32_t nb = b0 + own <= buckets + 1u ? own : buckets + 1u - b0;
  const uint32_t run = ((n + kGroupWaves - 1u) / kGroupWaves + kWave - 1u) / kWave * kWave;
  const uint32_t r0 = wave * run < n ? wave * run : n;
  const uint32_t r1 = n - r0 < run ? n : r0 + run;
  if constexpr (OWN == 0) {
    for (uint32_t i = lane; i < nb; i += kWave) cnt[wave][i] = 0u;  // this wavefront's own
  }
  volatile uint32_t* mine = cnt[wave];
  uint32_t key[kRowsAhead], next[kRowsAhead];
  auto fetch = [&](uint32_t (&k)[kRowsAhead], uint32_t r) {
#pragma unroll
    for (uint32_t i = 0; i < kRowsAhead; ++i) {
      const uint32_t at = r + i * kWave + lane;
      k[i] = static_cast<uint32_t>(keys[at < r1 ? at : r0 < n ? r0 : 0u]);
    }
  };
  // f(bucket, row) for 64 rows at a time in order; rows past the run have no bucket.
  const bool kept = run <= kRowsAhead * kWave;
  auto pass = [&](bool loaded, auto f) {
    if (r0 >= r1) return;
    if (!loaded) fetch(key, r0);
    for (uint32_t r = r0; r < r1; r += kRowsAhead * kWave) {
      const bool more = r1 - r > kRowsAhead * kWave;
      if (more) fetch(next, r + kRowsAhead * kWave);
#pragma unroll
      for (uint32_t i = 0; i < kRowsAhead; ++i) {
        const uint32_t row = r + i * kWave + lane;
        if (r + i * kWave >= r1) break;
        f(row < r1 ? (key[i] < buckets ? key[i] : buckets) : 0xFFFFFFFFu, row);
      }
      if (more) {
#pragma unroll
        for (uint32_t i = 0; i < kRowsAhead; ++i) key[i] = next[i];
      }
    }
  };
  uint32_t below = 0, count[kOwn < 4u ? kOwn : 4u] = {};
  pass(false, [&](uint32_t b, uint32_t) {
    below += static_cast<uint32_t>(__popcll(__ballot(b < b0)));
    if constexpr (OWN != 0) {
#pragma unroll
      for (int j = 0; j < OWN; ++j) count[j] += static_cast<uint32_t>(__popcll(__ballot(b == b0 + j)));
    } else {
      uint64_t left = __ballot(b - b0 < nb);
      while (left) {
        const uint32_t lb = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b), __builtin_ctzll(left)));
        const uint64_t same = __ballot(b == lb);
        if (lane == 0) mine[lb - b0] = mine[lb - b0] + static_cast<uint32_t>(__popcll(same));
        left &= ~same;
      }
    }
  });
  if (lane == 0) {
    below_lds[wave] = below;
    if constexpr (OWN != 0) {
#pragma unroll
      for (int j = 0; j < OWN; ++j) cnt[wave][j] = count[j];
    }
  }
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
  if (wave == 0) {
    // Exclusive sum of the buckets' counts, 64 at a time, from the rows below on.
    uint32_t base = lane < kGroupWaves ? below_lds[lane] : 0u;
#pragma unroll
    for (int m = 1; m < kGroupWaves; m <<= 1) base += __shfl_xor(base, m, kWave);
    base = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(base)));
    for (uint32_t i0 = 0; i0 < nb; i0 += kWave) {
      const uint32_t c = i0 + lane < nb ? start[i0 + lane] : 0u;
      uint32_t s = c;
#pragma unroll
      for (int m = 1; m < kWave; m <<= 1) {
        const uint32_t o = __shfl_up(s, m, kWave);
        s += lane >= static_cast<uint32_t>(m) ? o : 0u;
      }
      if (i0 + lane < nb) {
        start[i0 + lane] = base + s - c;
        offsets[b0 + i0 + lane] = base + s - c;
      }
      base += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(s), kWave - 1));
    }
  }
  __syncthreads();
  const uint64_t before = (1ull << lane) - 1ull;
  uint32_t at[kOwn < 4u ? kOwn : 4u];
  if constexpr (OWN != 0) {
#pragma unroll
    for (int j = 0; j < OWN; ++j)
      at[j] = static_cast<uint32_t>(j) < nb ? start[j] + cnt[wave][j] : 0u;
  }
  pass(kept, [&](uint32_t b, uint32_t row) {
    if constexpr (OWN != 0) {
#pragma unroll
      for (int j = 0; j < OWN; ++j) {
        const bool is = b == b0 + j && static_cast<uint32_t>(j) < nb;
        const uint64_t same = __ballot(is);
        if (same) {
          if (is) order[at[j] + __popcll(same & before)] = row;
          at[j] += static_cast<uint32_t>(__popcll(same));
        }
      }
    } else {
      uint64_t left = __ballot(b - b0 < nb);
      while (left) {
        const uint32_t lb = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b), __builtin_ctzll(left)));
        const uint64_t same = __ballot(b == lb);
        const uint32_t first = mine[lb - b0];
        if (b == lb) order[start[lb - b0] + first + __popcll(same & before)] = row;
        if (lane == 0) mine[lb - b0] = first + static_cast<uint32_t>(__popcll(same));
        left &= ~same;
      }
    }
  });
}

// Many rows: two launches. A workgroup of the first counts the keys of its
// run of rows; one of the second sums, per bucket, the counts of the runs
// before its own (and of all, whose exclusive sum is where buckets start) and
// places its rows, 1,024 at a time. Rows of one wavefront with equal keys find
// each other by a ballot per key bit; the wavefronts' counts are summed in LDS.
constexpr uint32_t kRoundRows = kGroupWaves * kWave;
constexpr uint32_t kManyMaxBuckets = 2047;  // the wavefronts' 16-bit counts fit 64 KB of LDS

__global__ __launch_bounds__(kRoundRows) void count_rows_kernel(const int32_t* __restrict__ keys, uint32_t n, uint32_t buckets,
                                                               uint32_t run, uint32_t* __restrict__ counts) {
  __shared__ uint32_t cnt[kManyMaxBuckets + 1u];
  for (uint32_t b = threadIdx.x; b <= buckets; b += kRoundRows) cnt[b] = 0u;
  __syncthreads();
  const uint32_t r0 = blockIdx.x * run, r1 = n - r0 < run ? n : r0 + run;
  for (uint32_t r = r0 + threadIdx.x; r < r1; r += kRoundRows) {
    const uint32_t key = static_cast<uint32_t>(keys[r]);
    atomicAdd(&cnt[key < buckets ? key : buckets], 1u);
  }
  __syncthreads();
  for (uint32_t b = threadIdx.x; b <= buckets; b += kRoundRows)
    counts[static_cast<size_t>(blockIdx.x) * (buckets + 1u) + b] = cnt[b];
}

__global__ __launch_bounds__(kRoundRows) void place_rows_kernel(const int32_t* __restrict__ keys, uint32_t n, uint32_t buckets,
                                                               uint32_t run, const uint32_t* __restrict__ counts,
                                                               uint32_t* __restrict__ offsets, uint32_t* __restrict__ order) {
  __shared__ uint32_t at[kManyMaxBuckets + 1u];  // where the bucket's next row of this run goes
  __shared__ uint16_t cnt[kGroupWaves][kManyMaxBuckets + 1u];
  __shared__ uint32_t sums[kGroupWaves];
  const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, nb = buckets + 1u;
  // Two neighbouring buckets a thread.
  uint32_t total[2] = {}, before[2] = {};
  constexpr uint32_t kRunsAhead = 16;
  const uint32_t last = gridDim.x - 1u;
  if (2u * tid < nb) {
    const uint32_t b0 = 2u * tid, b1 = b0 + 1u < nb ? b0 + 1u : b0;
    for (uint32_t w = 0; w <= last; w += kRunsAhead) {
      uint32_t c[kRunsAhead][2];
#pragma unroll
      for (uint32_t i = 0; i < kRunsAhead; ++i) {
        const uint32_t* row = counts + static_cast<size_t>(w + i < last ? w + i : last) * nb;
        c[i][0] = row[b0];
        c[i][1] = row[b1];
      }
#pragma unroll
      for (uint32_t i = 0; i < kRunsAhead; ++i)
#pragma unroll
        for (uint32_t j = 0; j < 2u; ++j) {
          const uint32_t one = w + i <= last && b0 + j < nb ? c[i][j] : 0u;
          total[j] += one;
          before[j] += w + i < blockIdx.x ? one : 0u;
        }
    }
  }
  const uint32_t pair = total[0] + total[1];
  uint32_t s = pair;
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const uint32_t o = __shfl_up(s, m, kWave);
    s += lane >= static_cast<uint32_t>(m) ? o : 0u;
  }
  if (lane == kWave - 1) sums[wave] = s;
  __syncthreads();
  for (uint32_t w = 0; w < wave; ++w) s += sums[w];
#pragma unroll
  for (uint32_t j = 0; j < 2u; ++j) {
    const uint32_t b = 2u * tid + j, first = s - pair + (j ? total[0] : 0u);
    if (b < nb) {
      at[b] = first + before[j];
      if (blockIdx.x == 0u) offsets[b] = first;
    }
  }
  const uint32_t r0 = blockIdx.x * run, r1 = n - r0 < run ? n : r0 + run;
  const uint32_t bits = 32u - static_cast<uint32_t>(__builtin_clz(nb));  // of a bucket's index, nb included
  for (uint32_t r = r0; r < r1; r += kRoundRows) {
    for (uint32_t b = lane; b < nb; b += kWave) cnt[wave][b] = 0u;  // this wavefront's own
    const uint32_t row = r + tid;
    const bool in = row < r1;
    const uint32_t key = in ? static_cast<uint32_t>(keys[row]) : 0u;
    const uint32_t b = !in ? nb : key < buckets ? key : buckets;
    uint64_t same = ~0ull;
    for (uint32_t i = 0; i < bits; ++i) {
      const uint64_t set = __ballot((b >> i) & 1u);
      same &= (b >> i) & 1u ? set : ~set;
    }
    const uint32_t rank = static_cast<uint32_t>(__popcll(same & ((1ull << lane) - 1ull)));
    if (in && rank == 0u) cnt[wave][b] = static_cast<uint16_t>(__popcll(same));
    __syncthreads();
    // Per bucket: each wavefront's count becomes the sum of those before it,
    // and the place for the next round moves on.
    for (uint32_t i = tid; i < nb; i += kRoundRows) {
      uint32_t sum = 0;
#pragma unroll
      for (int w = 0; w < kGroupWaves; ++w) {
        const uint32_t c = cnt[w][i];
        cnt[w][i] = static_cast<uint16_t>(sum);
        sum += c;
      }
      total[i != tid ? 1 : 0] = sum;
    }
    __syncthreads();
    if (in) order[at[b] + cnt[wave][b] + rank] = row;
    __syncthreads();
    for (uint32_t i = tid; i < nb; i += kRoundRows) at[i] += total[i != tid ? 1 : 0];
  }
}

// One launch up to the rows whose keys it keeps. Both sides at 8 / 257 / 2,047
// buckets: 16,384 rows take 6.8 / 7.3 / 9.7 us in one launch, one row more
// takes 6.8 / 7.9 / 16.0 in two.
constexpr uint32_t kOneLaunchRows = kRoundRows * kRowsAhead;
// Runs of a grouping in two launches (0: one launch does it): at least 1,024
// rows each, and as many as 256 or 1 MB of counts, since every workgroup of
// the second launch reads all counts.
uint32_t group_runs(uint32_t rows, uint32_t buckets, uint32_t& run) {
  if (rows <= kOneLaunchRows || buckets > kManyMaxBuckets) return 0u;
  uint32_t most = (1u << 18) / (buckets + 1u);
  most = most < 256u ? most : 256u;
  const uint32_t rounds = (rows + kRoundRows - 1u) / kRoundRows;
  run = (rounds + most - 1u) / most * kRoundRows;
  return (rows + run - 1u) / run;
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

size_t osmd_group_rows_workspace(uint32_t rows, uint32_t buckets) {
  uint32_t run = 0;
  return static_cast<size_t>(group_runs(rows, buckets, run)) * (buckets + 1u) * sizeof(uint32_t);
}

int osmd_group_rows(const int32_t* keys, uint32_t rows, uint32_t buckets, uint32_t* offsets, uint32_t* order,
                    void* workspace, osmd_stream s) {
  if (buckets == 0 || buckets > OSMD_GROUP_MAX_BUCKETS || rows > 0x7FFFFFFFu)
    return static_cast<int>(hipErrorInvalidValue);
  const hipStream_t st = static_cast<hipStream_t>(s);
  uint32_t run = 0;
  if (const uint32_t runs = group_runs(rows, buckets, run)) {
    uint32_t* counts = static_cast<uint32_t*>(workspace);
    count_rows_kernel<<<runs, kRoundRows, 0, st>>>(keys, rows, buckets, run, counts);
    place_rows_kernel<<<runs, kRoundRows, 0, st>>>(keys, rows, buckets, run, counts, offsets, order);
    return launch_status();
  }
  const uint32_t own = (buckets + 1u + 255u) / 256u;  // at most 256 workgroups
  const uint32_t grid = (buckets + 1u + own - 1u) / own;
  auto go = [&](auto kernel) {
    kernel<<<grid, kGroupWaves * kWave, 0, st>>>(keys, rows, buckets, own, offsets, order);
  };
  if (own == 1u)
    go(group_rows_kernel<1>);
  else if (own == 2u)
    go(group_rows_kernel<2>);
  else if (own <= 4u)
    go(group_rows_kernel<4>);
  else
    go(group_rows_kernel<0>);
  return launch_status();
}

}  // extern "C"
