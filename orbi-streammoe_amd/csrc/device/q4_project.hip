// q4_project.hip -- a q4 projection of many tokens with a low-rank adapter of
// each token's own beside it:
//   y_t = W x_t + scale_a B_a (A_a x_t),  a = adapter_ids[t]
// W [N, K] affine q4 (W = s q + b per group of columns), A_a [R, K], B_a
// [N, R]. Tokens whose id is outside [0, count) have no adapter. All sums are
// fp32; only y is rounded to its type.
#include "device_common.hpp"

namespace {

using namespace osmk;

__device__ __forceinline__ uint16_t bf16_rne(float f) {
  uint32_t u = __float_as_uint(f);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return static_cast<uint16_t>((u >> 16) | 0x40u);
  u += 0x7FFFu + ((u >> 16) & 1u);
  return static_cast<uint16_t>(u >> 16);
}

__device__ __forceinline__ void store_out(void* y, uint32_t dtype, size_t i, float v) {
  if (dtype == OSM_META_F32)
    static_cast<float*>(y)[i] = v;
  else if (dtype == OSM_META_BF16)
    static_cast<uint16_t*>(y)[i] = bf16_rne(v);
  else
    static_cast<_Float16*>(y)[i] = static_cast<_Float16>(v);
}

// The rank of token t's adapter (0: none), and the adapter.
__device__ __forceinline__ uint32_t token_rank(const osmd_adapters& ad, const int32_t* ids, uint32_t t, uint32_t& a) {
  if (ad.count == 0u) return 0u;
  a = static_cast<uint32_t>(ids[t]);
  if (a >= ad.count) return 0u;
  const uint32_t r = ad.ranks ? ad.ranks[a] : ad.max_rank;
  return r < ad.max_rank ? r : ad.max_rank;
}

constexpr int kShrinkWaves = 4;

// v[t, j] = scale_a (A_a x_t)_j: a wavefront per rank row and token.
template <int XT, int AT>
__global__ __launch_bounds__(kShrinkWaves* kWave) void shrink_kernel(osmd_project_args p, float* __restrict__ v) {
  const uint32_t R = p.adapters.max_rank, rows = (R + kShrinkWaves - 1u) / kShrinkWaves;
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t t = blockIdx.x / rows, j = blockIdx.x % rows * kShrinkWaves + wave;
  uint32_t a = 0;
  if (j >= token_rank(p.adapters, p.adapter_ids, t, a)) return;
  const uint32_t K = p.w.packed_cols * 8u;
  const size_t xo = t * p.x_stride, ao = (static_cast<size_t>(a) * R + j) * K;
  float s = 0.0f;
  for (uint32_t c = lane; c < K; c += kWave) s = fmaf(meta_at<XT>(p.x, xo + c), meta_at<AT>(p.adapters.a, ao + c), s);
  s = wave_sum(s);
  if (lane == 0) v[static_cast<size_t>(t) * R + j] = s * (p.adapters.scales ? p.adapters.scales[a] : 1.0f);
}

constexpr int kAnyWaves = 4;
constexpr uint32_t kAnyTokens = 4;

// Any geometry: a wavefront per row of W and kAnyTokens tokens, each weight
// dequantised once for them.
template <int META, int XT>
__global__ __launch_bounds__(kAnyWaves* kWave) void project_any_kernel(osmd_project_args p, const float* __restrict__ v) {
  const uint32_t N = p.w.out_dim, blocks = (N + kAnyWaves - 1u) / kAnyWaves;
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t n = blockIdx.x % blocks * kAnyWaves + wave, t0 = blockIdx.x / blocks * kAnyTokens;
  if (n >= N) return;
  const uint32_t words = p.w.packed_cols, G = p.w.group, groups = words * 8u / G;
  float acc[kAnyTokens] = {};
  size_t xo[kAnyTokens];
#pragma unroll
  for (uint32_t i = 0; i < kAnyTokens; ++i) xo[i] = (t0 + i < p.tokens ? t0 + i : t0) * p.x_stride;
  for (uint32_t w = lane; w < words; w += kWave) {
    const uint32_t word = p.w.packed[static_cast<size_t>(n) * words + w];
    for (uint32_t j = 0; j < 8u; ++j) {
      const uint32_t c = 8u * w + j;
      const size_t g = static_cast<size_t>(n) * groups + c / G;
      const float q = static_cast<float>((word >> (4u * j)) & 15u);
      const float value = fmaf(meta_at<META>(p.w.scales, g), q, meta_at<META>(p.w.biases, g));
#pragma unroll
      for (uint32_t i = 0; i < kAnyTokens; ++i) acc[i] = fmaf(value, meta_at<XT>(p.x, xo[i] + c), acc[i]);
    }
  }
  for (uint32_t i = 0; i < kAnyTokens && t0 + i < p.tokens; ++i) {
    const uint32_t t = t0 + i, R = p.adapters.max_rank;
    uint32_t a = 0;
    const uint32_t rank = token_rank(p.adapters, p.adapter_ids, t, a);
    float d = 0.0f;
    for (uint32_t j = lane; j < rank; j += kWave) {
      const size_t o = (static_cast<size_t>(a) * N + n) * R + j;
      const float b = p.adapters.dtype == OSM_META_F32    ? meta_at<OSM_META_F32>(p.adapters.b, o)
                      : p.adapters.dtype == OSM_META_BF16 ? meta_at<OSM_META_BF16>(p.adapters.b, o)
                                                          : meta_at<OSM_META_F16>(p.adapters.b, o);
      d = fmaf(b, v[static_cast<size_t>(t) * R + j], d);
    }
    const float y = wave_sum(acc[i] + d);
    if (lane == 0) store_out(p.y, p.y_dtype, t * p.y_stride + n, y);
  }
}

// f(integral_constant<dtype>) for one of the three element types.
template <typename F>
int by_dtype(uint32_t dtype, F f) {
  switch (dtype) {
    case OSM_META_F32: return f(std::integral_constant<int, OSM_META_F32>{});
    case OSM_META_F16: return f(std::integral_constant<int, OSM_META_F16>{});
    case OSM_META_BF16: return f(std::integral_constant<int, OSM_META_BF16>{});
    default: return static_cast<int>(hipErrorInvalidValue);
  }
}

}  // namespace

extern "C" {

size_t osmd_q4_project_workspace(const osmd_project_args* a) {
  return a->adapters.count ? static_cast<size_t>(a->tokens) * a->adapters.max_rank * sizeof(float) : 0u;
}

int osmd_q4_project(const osmd_project_args* a, void* workspace, osmd_stream s) {
  const hipStream_t st = static_cast<hipStream_t>(s);
  float* v = static_cast<float*>(workspace);
  if (a->adapters.count) {
    const uint32_t rows = (a->adapters.max_rank + kShrinkWaves - 1u) / kShrinkWaves;
    const int r = by_dtype(a->x_dtype, [&](auto xt) {
      return by_dtype(a->adapters.dtype, [&](auto at) {
        shrink_kernel<decltype(xt)::value, decltype(at)::value>
            <<<a->tokens * rows, kShrinkWaves * kWave, 0, st>>>(*a, v);
        return launch_status();
      });
    });
    if (r != 0) return r;
  }
  const uint32_t blocks = (a->w.out_dim + kAnyWaves - 1u) / kAnyWaves;
  const uint32_t tiles = (a->tokens + kAnyTokens - 1u) / kAnyTokens;
  return by_dtype(a->w.meta_dtype, [&](auto meta) {
    return by_dtype(a->x_dtype, [&](auto xt) {
      project_any_kernel<decltype(meta)::value, decltype(xt)::value>
          <<<blocks * tiles, kAnyWaves * kWave, 0, st>>>(*a, v);
      return launch_status();
    });
  });
}

}  // extern "C"
