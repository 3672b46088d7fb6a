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

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// ---- the prepared input --------------------------------------------------------
// The matrix instructions multiply f16 pairs: a nibble q masked in place is
// the f16 subnormal q 2^-24 (nibbles 0, 2, 4, 6 of a word) or q 2^-20 (1, 3,
// 5, 7; w & 0x00F000F0), so five instructions unpack eight nibbles, exactly.
// x is brought to f16 once per call: row t times 2^e, e such that its largest
// value lies in [2^14, 2^15), as one term (bf16 and f16 input: exact down to
// 2^-24 steps, 2^-35 of the row's largest value) or as two (fp32: 22 bits),
// columns that meet a q 2^-20 divided by 16. With D the fp32 sum of a group,
//   y = 2^(24 - e) sum over groups of (s D + b X),  X = 2^(e - 24) sum of x.
// Products are exact in fp32; nothing else is rounded to fewer bits.
//
// Layout: tiles of R tokens in the instructions' operand order. Lane l of an
// R x R instruction holds row l % R and the 8 columns of k-slot l / R; a step
// is one instruction's 8 * slots columns. A sub-group of SC columns (the
// quantisation group, or its largest part of 32, 64 or 128) gives slot h
// words h * GW .. h * GW + GW - 1, GW = SC / 8 / slots, one word a step, so a
// lane's words of W are contiguous. A fragment (64 lanes x 16 bytes) is 1 KB:
//   frag [tile][step][term][64][8] f16, sums [tile][K / SC][R], exps [token]
template <int R>
constexpr int kSlots = kWave / R;
template <int R>
constexpr int kAcc = R * R / kWave;  // accumulator registers of one tile

struct Prepared {
  _Float16* frag;
  float* sums;
  int32_t* exps;  // 24 - e
  float* v;       // [token][vr] scale_a A_a x, zero from the rank on
  uint32_t vr;    // max_rank rounded up to 16
};

template <int XT>
__device__ __forceinline__ void load8(const void* x, size_t o, bool wide, float (&v)[8]) {
  if (wide) {
    if constexpr (XT == OSM_META_F32) {
      const float* p = static_cast<const float*>(x) + o;
      const uint4 a = ldg16(p), b = ldg16(p + 4);
      const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u[i]);
    } else {
      const uint4 a = ldg16(static_cast<const uint16_t*>(x) + o);
      const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = meta_widen<XT>(u[i] & 0xFFFFu);
        v[2 * i + 1] = meta_widen<XT>(u[i] >> 16);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = meta_at<XT>(x, o + i);
  }
}

// Whether rows of `stride` elements from p on can be read 16 bytes at a time.
bool wide_rows(const void* p, size_t stride, uint32_t dtype) {
  return reinterpret_cast<uintptr_t>(p) % 16u == 0u && stride * osm_meta_bytes(dtype) % 16u == 0u;
}

struct PrepareParams {
  const void* x;
  size_t stride;
  uint32_t tokens, rows, words;  // rows: tokens rounded up to whole tiles (the rest is zero)
  uint32_t wide;
  const uint32_t* order;         // row i is token order[i], or null
  Prepared out;
};

// TPT threads per row, 256 / TPT rows per workgroup.
template <int XT, int R, int GW, int TPT>
__device__ __forceinline__ void prepare_rows(const PrepareParams& p, uint32_t block) {
  constexpr int NT = XT == OSM_META_F32 ? 2 : 1;
  constexpr uint32_t GWS = GW * kSlots<R>;  // words of a sub-group
  __shared__ float red[256 / kWave];
  const uint32_t i = threadIdx.x % TPT, row = block * (256u / TPT) + threadIdx.x / TPT;
  const bool live = row < p.tokens;
  const uint32_t t = !live ? 0u : p.order ? p.order[row] : row;
  const size_t xo = t * p.stride;
  float top = 0.0f;
  if (live)
    for (uint32_t w = i; w < p.words; w += TPT) {
      float v[8];
      load8<XT>(p.x, xo + 8u * w, p.wide, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(v[k]));
    }
  if constexpr (TPT == 256) {
    top = wave_max(top);
    if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  } else {
    static_assert(TPT == 32, "half a wavefront");
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, kWave));
  }
  if (row >= p.rows) return;
  const int e = 141 - static_cast<int>(__float_as_uint(top) >> 23);
  if (i == 0) p.out.exps[row] = 24 - e;
  const uint32_t tile = row / R, steps = p.words / kSlots<R>, subs = p.words / GWS;
  // Whole groups of GWS lanes stay in the loop together (words is a multiple of GWS).
  for (uint32_t w = i; w < p.words; w += TPT) {
    float v[8];
    if (live) {
      load8<XT>(p.x, xo + 8u * w, p.wide, v);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.0f;
    }
    float sum = 0.0f;
    f16x8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      constexpr int nibble[8] = {0, 4, 1, 5, 2, 6, 3, 7};
      const float s = ldexpf(v[nibble[k]], e);
      sum += s;
      const float o = (nibble[k] & 1) ? s * 0.0625f : s;
      hi[k] = static_cast<_Float16>(o);
      if constexpr (NT == 2) lo[k] = static_cast<_Float16>(o - static_cast<float>(hi[k]));
    }
    const uint32_t sub = w / GWS, iw = w % GWS;
    const uint32_t lane = iw / GW * R + row % R, step = sub * GW + iw % GW;
    _Float16* f = p.out.frag + ((static_cast<size_t>(tile) * steps + step) * NT * kWave + lane) * 8u;
    *reinterpret_cast<f16x8*>(f) = hi;
    if constexpr (NT == 2) *reinterpret_cast<f16x8*>(f + kWave * 8u) = lo;
    sum = row_sum<GWS < 16 ? GWS : 16>(sum);
    if (iw == 0) p.out.sums[(static_cast<size_t>(tile) * subs + sub) * R + row % R] = sum * 0x1p-24f;
  }
}

// v[row, j] = scale_a (A_a x_t)_j: a wavefront per rank row and token, for
// few tokens. Columns from the rank on are zero.
struct ShrinkParams {
  const void* x;
  size_t stride;
  uint32_t tokens, words, x_wide, a_wide;
  osmd_adapters ad;
  const int32_t* ids;
  float* v;
  uint32_t vr;
};
template <int XT, int AT>
__device__ __forceinline__ void shrink_rows(const ShrinkParams& p, uint32_t block) {
  const uint32_t blocks = p.vr / 4u;
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t t = block / blocks, j = block % blocks * 4u + wave;
  uint32_t a = 0;
  const uint32_t rank = token_rank(p.ad, p.ids, t, a);
  float s = 0.0f;
  if (j < rank) {
    const size_t xo = t * p.stride, ao = (static_cast<size_t>(a) * p.ad.max_rank + j) * p.words * 8u;
    for (uint32_t w = lane; w < p.words; w += kWave) {
      float x[8], c[8];
      load8<XT>(p.x, xo + 8u * w, p.x_wide, x);
      load8<AT>(p.ad.a, ao + 8u * w, p.a_wide, c);
#pragma unroll
      for (int k = 0; k < 8; ++k) s = fmaf(x[k], c[k], s);
    }
    s = wave_sum(s);
    if (p.ad.scales) s *= p.ad.scales[a];
  }
  if (lane == 0) p.v[static_cast<size_t>(t) * p.vr + j] = s;
}

// Few tokens: both in one launch, the workgroups past `prepare_blocks` shrink.
template <int XT, int R, int GW, int AT>
__global__ __launch_bounds__(256) void prepare_few_kernel(PrepareParams p, ShrinkParams s, uint32_t prepare_blocks) {
  if (blockIdx.x < prepare_blocks)
    prepare_rows<XT, R, GW, 256>(p, blockIdx.x);
  else
    shrink_rows<XT, AT>(s, blockIdx.x - prepare_blocks);
}

// ---- few tokens ------------------------------------------------------------------
// A workgroup owns R rows of W and all (at most MT * R) tokens; its wavefronts
// split the columns and their sums are added in LDS in wavefront order. The
// lanes of an instruction's D columns are rows of W, so a lane needs one
// scale and bias per sub-group.
template <int R>
struct Tile;
template <>
struct Tile<16> {
  typedef f32x4 acc;
  static __device__ __forceinline__ acc mfma(f16x8 a, f16x8 b, acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t row(uint32_t lane, int i) { return 4u * (lane / 16u) + i; }
};
template <>
struct Tile<32> {
  typedef f32x16 acc;
  static __device__ __forceinline__ acc mfma(f16x8 a, f16x8 b, acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t row(uint32_t lane, int i) {
    return 8u * (i / 4) + 4u * (lane / 32u) + i % 4;
  }
};

// Eight nibbles as the operand (see above).
__device__ __forceinline__ f16x8 nibble_operand(uint32_t w) {
  const uint32_t t = w >> 8;
  const u32x4 v = {w & 0x000F000Fu, w & 0x00F000F0u, t & 0x000F000Fu, t & 0x00F000F0u};
  return __builtin_bit_cast(f16x8, v);
}
__device__ __forceinline__ f16x8 load_frag(const _Float16* p) { return __builtin_bit_cast(f16x8, ldg<u32x4>(p)); }

template <int GW>
__device__ __forceinline__ void load_words(const uint32_t* p, uint32_t (&w)[GW]) {
  if constexpr (GW == 1) {
    w[0] = ldg<uint32_t>(p);
  } else if constexpr (GW == 2) {
    const uint2 v = ldg8(p);
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < GW / 4; ++i) {
      const uint4 v = ldg16(p + 4 * i);
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  }
}

struct ProjectParams {
  osmd_q4_proj w;
  uint32_t groups, per_group;  // groups of a row, sub-groups of a group
  Prepared in;
  void* y;
  size_t y_stride;
  uint32_t y_dtype, tokens;
  osmd_adapters ad;
  const int32_t* ids;
  uint32_t b_wide;
  const uint32_t* order;
};

__device__ __forceinline__ float adapter_element(const osmd_adapters& ad, size_t o) {
  return ad.dtype == OSM_META_F32    ? meta_at<OSM_META_F32>(ad.b, o)
         : ad.dtype == OSM_META_BF16 ? meta_at<OSM_META_BF16>(ad.b, o)
                                     : meta_at<OSM_META_F16>(ad.b, o);
}

// (B_a v_t)_n for one token and row.
__device__ __forceinline__ float expand_one(const ProjectParams& p, uint32_t t, uint32_t n) {
  uint32_t a = 0;
  const uint32_t rank = token_rank(p.ad, p.ids, t, a);
  const size_t o = (static_cast<size_t>(a) * p.w.out_dim + n) * p.ad.max_rank;
  const float* v = p.in.v + static_cast<size_t>(t) * p.in.vr;
  float s = 0.0f;
  uint32_t j = 0;
  if (p.b_wide) {
    for (; j + 8u <= rank; j += 8u) {
      float b[8], c[8];
      if (p.ad.dtype == OSM_META_BF16)
        load8<OSM_META_BF16>(p.ad.b, o + j, true, b);
      else if (p.ad.dtype == OSM_META_F16)
        load8<OSM_META_F16>(p.ad.b, o + j, true, b);
      else
        load8<OSM_META_F32>(p.ad.b, o + j, true, b);
      load8<OSM_META_F32>(v, j, true, c);
#pragma unroll
      for (int k = 0; k < 8; ++k) s = fmaf(b[k], c[k], s);
    }
  }
  for (; j < rank; ++j) s = fmaf(adapter_element(p.ad, o + j), v[j], s);
  return s;
}

constexpr int kFewWaves = 8;

template <int R, int NT, int MT, int GW, int META>
__global__ __launch_bounds__(kFewWaves* kWave) void project_few_kernel(ProjectParams p) {
  typedef typename Tile<R>::acc acc_t;
  constexpr int A = kAcc<R>;
  constexpr uint32_t GWS = GW * kSlots<R>;
  constexpr int U = 4;  // sub-groups in flight
  __shared__ float part[kFewWaves][MT][A][kWave];
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t N = p.w.out_dim, words = p.w.packed_cols, subs = words / GWS, steps = subs * GW;
  const uint32_t n0 = blockIdx.x * R;
  const uint32_t n = n0 + lane % R < N ? n0 + lane % R : N - 1u;
  const uint32_t s0 = subs * wave / kFewWaves, s1 = subs * (wave + 1u) / kFewWaves;
  const uint32_t* wrow = p.w.packed + static_cast<size_t>(n) * words + lane / R * GW;
  const size_t mrow = static_cast<size_t>(n) * p.groups;
  const _Float16* frag = p.in.frag + lane * 8u;
  acc_t total[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < A; ++i) total[m][i] = 0.0f;
  for (uint32_t s = s0; s < s1; s += U) {
    uint32_t w[U][GW];
    uint32_t sb[U], bb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t c = s + u < s1 ? s + u : s1 - 1u;
      load_words<GW>(wrow + c * GWS, w[u]);
      sb[u] = meta_bits<META>(p.w.scales, mrow + c / p.per_group);
      bb[u] = meta_bits<META>(p.w.biases, mrow + c / p.per_group);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u >= s1) break;
      const uint32_t c = s + u;
      f16x8 q[GW];
#pragma unroll
      for (int g = 0; g < GW; ++g) q[g] = nibble_operand(w[u][g]);
      const float sc = meta_widen<META>(sb[u]), bc = meta_widen<META>(bb[u]);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        acc_t d;
#pragma unroll
        for (int i = 0; i < A; ++i) d[i] = 0.0f;
        const _Float16* f = frag + (static_cast<size_t>(m) * steps + c * GW) * NT * kWave * 8u;
#pragma unroll
        for (int g = 0; g < GW; ++g)
#pragma unroll
          for (int k = 0; k < NT; ++k) d = Tile<R>::mfma(load_frag(f + (g * NT + k) * kWave * 8u), q[g], d);
        const float* xs = p.in.sums + (static_cast<size_t>(m) * subs + c) * R;
#pragma unroll
        for (int i = 0; i < A; ++i)
          total[m][i] = fmaf(sc, d[i], fmaf(bc, xs[Tile<R>::row(lane, i)], total[m][i]));
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < A; ++i) part[wave][m][i][lane] = total[m][i];
  __syncthreads();
  for (uint32_t o = threadIdx.x; o < MT * R * R; o += kFewWaves * kWave) {
    const uint32_t t = o / R, nn = n0 + o % R, tr = t % R, m = t / R;
    if (t >= p.tokens || nn >= N) continue;
    const uint32_t i = R == 16 ? tr % 4u : tr / 8u * 4u + tr % 4u;
    const uint32_t l = (R == 16 ? tr / 4u : tr / 4u % 2u) * R + o % R;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < kFewWaves; ++k) y += part[k][m][i][l];
    y = ldexpf(y, p.in.exps[t]);
    if (p.ad.count) y += expand_one(p, t, nn);
    store_out(p.y, p.y_dtype, t * p.y_stride + nn, y);
  }
}

constexpr int kShrinkWaves = 4;

// v[t, j] = scale_a (A_a x_t)_j: a wavefront per rank row and token.
template <int XT, int AT>
__global__ __launch_bounds__(kShrinkWaves* kWave) void shrink_kernel(ShrinkParams p) {
  shrink_rows<XT, AT>(p, blockIdx.x);
}

constexpr int kAnyWaves = 4;
constexpr uint32_t kAnyTokens = 4;

// Any geometry: a wavefront per row of W and kAnyTokens tokens, each weight
// dequantised once for them.
template <int META, int XT>
__global__ __launch_bounds__(kAnyWaves* kWave) void project_any_kernel(osmd_project_args p, const float* __restrict__ v,
                                                                       uint32_t vr) {
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
      d = fmaf(b, v[static_cast<size_t>(t) * vr + j], d);
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

constexpr uint32_t kFewTokens = 64;

uint32_t round_up(uint32_t n, uint32_t m) { return (n + m - 1u) / m * m; }
size_t align256(size_t n) { return (n + 255u) & ~static_cast<size_t>(255u); }

// What a call runs: the columns of a sub-group (0: a group that is no
// multiple of 32, one kernel for any) and the tile.
struct Plan {
  uint32_t sub_cols, tile, rows, terms, vr;
  size_t frag, sums, exps, v, total;  // workspace offsets
};
Plan plan_of(const osmd_project_args& a) {
  Plan p{};
  const uint32_t G = a.w.group, K = a.w.packed_cols * 8u;
  p.vr = a.adapters.count ? round_up(a.adapters.max_rank, 16u) : 0u;
  if (G % 32u == 0u && a.tokens <= kFewTokens) {
    p.sub_cols = G % 128u == 0u ? 128u : G % 64u == 0u ? 64u : 32u;
    p.tile = a.tokens <= 16u ? 16u : 32u;
    p.rows = round_up(a.tokens, p.tile);
    p.terms = a.x_dtype == OSM_META_F32 ? 2u : 1u;
    p.sums = align256(static_cast<size_t>(p.rows) * K * 2u * p.terms);
    p.exps = p.sums + align256(static_cast<size_t>(p.rows) * (K / p.sub_cols) * 4u);
    p.v = p.exps + align256(static_cast<size_t>(p.rows) * 4u);
  }
  p.total = p.v + static_cast<size_t>(a.tokens) * p.vr * sizeof(float);
  return p;
}

template <int R, int GW, int MT>
int launch_few(const osmd_project_args& a, const Plan& pl, uint8_t* work, hipStream_t st) {
  PrepareParams pp{};
  pp.x = a.x;
  pp.stride = a.x_stride;
  pp.tokens = a.tokens;
  pp.rows = pl.rows;
  pp.words = a.w.packed_cols;
  pp.wide = wide_rows(a.x, a.x_stride, a.x_dtype) ? 1u : 0u;
  pp.out.frag = reinterpret_cast<_Float16*>(work + pl.frag);
  pp.out.sums = reinterpret_cast<float*>(work + pl.sums);
  pp.out.exps = reinterpret_cast<int32_t*>(work + pl.exps);
  pp.out.v = reinterpret_cast<float*>(work + pl.v);
  pp.out.vr = pl.vr;
  ShrinkParams sp{};
  sp.x = a.x;
  sp.stride = a.x_stride;
  sp.tokens = a.tokens;
  sp.words = a.w.packed_cols;
  sp.x_wide = pp.wide;
  sp.a_wide = wide_rows(a.adapters.a, 8u * a.w.packed_cols, a.adapters.dtype) ? 1u : 0u;
  sp.ad = a.adapters;
  sp.ids = a.adapter_ids;
  sp.v = pp.out.v;
  sp.vr = pl.vr;
  const uint32_t shrink_blocks = a.tokens * (pl.vr / 4u);
  int r = by_dtype(a.x_dtype, [&](auto xt) {
    return by_dtype(a.adapters.dtype, [&](auto at) {
      prepare_few_kernel<decltype(xt)::value, R, GW, decltype(at)::value>
          <<<pl.rows + shrink_blocks, 256, 0, st>>>(pp, sp, pl.rows);
      return launch_status();
    });
  });
  if (r != 0) return r;
  ProjectParams p{};
  p.w = a.w;
  p.groups = a.w.packed_cols * 8u / a.w.group;
  p.per_group = a.w.group / pl.sub_cols;
  p.in = pp.out;
  p.y = a.y;
  p.y_stride = a.y_stride;
  p.y_dtype = a.y_dtype;
  p.tokens = a.tokens;
  p.ad = a.adapters;
  p.ids = a.adapter_ids;
  p.b_wide = wide_rows(a.adapters.b, a.adapters.max_rank, a.adapters.dtype) ? 1u : 0u;
  const uint32_t grid = (a.w.out_dim + R - 1u) / R;
  return by_dtype(a.w.meta_dtype, [&](auto meta) {
    constexpr int M = decltype(meta)::value;
    if (pl.terms == 2u)
      project_few_kernel<R, 2, MT, GW, M><<<grid, kFewWaves * kWave, 0, st>>>(p);
    else
      project_few_kernel<R, 1, MT, GW, M><<<grid, kFewWaves * kWave, 0, st>>>(p);
    return launch_status();
  });
}

}  // namespace

extern "C" {

size_t osmd_q4_project_workspace(const osmd_project_args* a) { return plan_of(*a).total; }

int osmd_q4_project(const osmd_project_args* a, void* workspace, osmd_stream s) {
  const hipStream_t st = static_cast<hipStream_t>(s);
  const Plan pl = plan_of(*a);
  uint8_t* work = static_cast<uint8_t*>(workspace);
  if (pl.sub_cols) {
    auto few = [&](auto gw16) {  // words of a slot with tiles of 16; of 32: twice
      constexpr int W = decltype(gw16)::value;
      if (pl.tile == 16u) return launch_few<16, W, 1>(*a, pl, work, st);
      if (pl.rows == 32u) return launch_few<32, 2 * W, 1>(*a, pl, work, st);
      return launch_few<32, 2 * W, 2>(*a, pl, work, st);
    };
    return pl.sub_cols == 128u  ? few(std::integral_constant<int, 4>{})
           : pl.sub_cols == 64u ? few(std::integral_constant<int, 2>{})
                                : few(std::integral_constant<int, 1>{});
  }
  float* v = reinterpret_cast<float*>(work + pl.v);
  if (a->adapters.count) {
    ShrinkParams sp{};
    sp.x = a->x;
    sp.stride = a->x_stride;
    sp.tokens = a->tokens;
    sp.words = a->w.packed_cols;
    sp.x_wide = wide_rows(a->x, a->x_stride, a->x_dtype) ? 1u : 0u;
    sp.a_wide = wide_rows(a->adapters.a, 8u * a->w.packed_cols, a->adapters.dtype) ? 1u : 0u;
    sp.ad = a->adapters;
    sp.ids = a->adapter_ids;
    sp.v = v;
    sp.vr = pl.vr;
    const int r = by_dtype(a->x_dtype, [&](auto xt) {
      return by_dtype(a->adapters.dtype, [&](auto at) {
        shrink_kernel<decltype(xt)::value, decltype(at)::value>
            <<<a->tokens * (pl.vr / kShrinkWaves), kShrinkWaves * kWave, 0, st>>>(sp);
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
          <<<blocks * tiles, kAnyWaves * kWave, 0, st>>>(*a, v, pl.vr);
      return launch_status();
    });
  });
}

}  // extern "C"
