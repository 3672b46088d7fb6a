// q4_project.hip -- a q4 projection of many tokens with a low-rank adapter of
// each token's own beside it:
//   y_t = W x_t + scale_a B_a (A_a x_t),  a = adapter_ids[t]
// W [N, K] affine q4 (W = s q + b per group of columns), A_a [R, K], B_a
// [N, R]. Tokens whose id is outside [0, count) have no adapter. All sums are
// fp32; only y is rounded to its type.
#include "device_common.hpp"

namespace {

using namespace osmk;

__device__ __forceinline__ void store_out(void* y, uint32_t dtype, size_t i, float v) {
  if (dtype == OSM_META_F32)
    static_cast<float*>(y)[i] = v;
  else if (dtype == OSM_META_BF16)
    static_cast<__bf16*>(y)[i] = static_cast<__bf16>(v);
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
// The matrix instructions multiply f16 pairs: a nibble q in the upper bits of
// the fraction, below an exponent of 0, is the f16 subnormal q 2^-18, so eight
// instructions unpack eight nibbles, exactly. (Lower in the fraction they need
// fewer shifts, but the instructions align products by the operands' exponent
// fields: a fraction that starts with zeros costs the sum as many bits. In
// place at q 2^-24 and q 2^-20, five instructions, fp32 outputs of 4,096
// columns were off by 1e-5.)
// x is brought to f16 once per call: row t times 2^e, e such that its largest
// value lies in [2^14, 2^15), as one term (bf16 and f16 input: exact down to
// 2^-24 steps, 2^-38 of the row's largest value) or as two (fp32: 22 bits).
// With D the fp32 sum of a group,
//   y = 2^(18 - e) sum over groups of (s D + b X),  X = 2^(e - 18) sum of x.
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
  int32_t* exps;  // 18 - e
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

// Eight elements as loaded.
template <int T>
struct Raw8 {
  uint32_t u[T == OSM_META_F32 ? 8 : 4];
  __device__ __forceinline__ float get(int i) const {
    if constexpr (T == OSM_META_F32)
      return __uint_as_float(u[i]);
    else
      return meta_widen<T>((u[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
  }
  __device__ __forceinline__ void clear(int i) {
    if constexpr (T == OSM_META_F32)
      u[i] = 0u;
    else
      u[i >> 1] &= i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
  }
};
template <int T>
__device__ __forceinline__ void load_raw8(const void* x, size_t o, bool wide, Raw8<T>& r) {
  if (wide) {
    const uint4 a = ldg16(static_cast<const uint8_t*>(x) + o * (T == OSM_META_F32 ? 4u : 2u));
    r.u[0] = a.x, r.u[1] = a.y, r.u[2] = a.z, r.u[3] = a.w;
    if constexpr (T == OSM_META_F32) {
      const uint4 b = ldg16(static_cast<const float*>(x) + o + 4u);
      r.u[4] = b.x, r.u[5] = b.y, r.u[6] = b.z, r.u[7] = b.w;
    }
  } else if constexpr (T == OSM_META_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.u[i] = meta_bits<T>(x, o + i);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.u[i] = meta_bits<T>(x, o + 2 * i) | (meta_bits<T>(x, o + 2 * i + 1) << 16);
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

constexpr int kSumTerms = 3;

// What the tiled kernel reads besides the fragments.
struct ManyPrepared {
  __bf16* sum_frag;   // [tile][16 sub-groups][term][64][8]
  float* scales;      // [sub-group][row of W, scale_row apart], then a row of zeros
  uint32_t scale_row;
  __bf16* bias_frag;  // [32 rows][16 sub-groups][term][64][8]
  uint32_t kgs;       // runs of 16 sub-groups
  __bf16* v_frag;     // [tile][16 rank rows][term][64][8]: v, scale_a A_a x
};

// The sum of a sub-group of a token as bf16 terms, each the nearest to what is left.
__device__ __forceinline__ void store_sum(const ManyPrepared& m, uint32_t tile, uint32_t sub, uint32_t row, float v) {
  const uint32_t lane = sub % 16u / 8u * 32u + row;
#pragma unroll
  for (int t = 0; t < kSumTerms; ++t) {
    const __bf16 b = static_cast<__bf16>(v);
    m.sum_frag[(((static_cast<size_t>(tile) * m.kgs + sub / 16u) * kSumTerms + t) * kWave + lane) * 8u + sub % 8u] = b;
    v -= static_cast<float>(b);
  }
}

// TPT threads a row, of a workgroup's THREADS.
template <int XT, int R, int GW, int TPT, int THREADS = 256, bool MANY = false>
__device__ __forceinline__ void prepare_rows(const PrepareParams& p, uint32_t block, const ManyPrepared* many = nullptr) {
  constexpr int NT = XT == OSM_META_F32 ? 2 : 1;
  constexpr uint32_t GWS = GW * kSlots<R>;  // words of a sub-group
  __shared__ float red[THREADS / kWave];
  const uint32_t i = threadIdx.x % TPT, row = block * (THREADS / TPT) + threadIdx.x / TPT;
  const bool live = row < p.tokens;
  const uint32_t t = !live ? 0u : p.order ? p.order[row] : row;
  const size_t xo = t * p.stride;
  // Up to kKeep units of 8 columns a thread are read once and kept; of longer
  // rows every batch is read again for the second pass.
  constexpr uint32_t kKeep = 8;
  Raw8<XT> keep[kKeep];
  auto batch = [&](uint32_t w0) {
#pragma unroll
    for (uint32_t u = 0; u < kKeep; ++u) {
      const uint32_t w = w0 + u * TPT;
      load_raw8<XT>(p.x, xo + 8u * (w < p.words ? w : p.words - 1u), p.wide, keep[u]);
    }
  };
  float top = 0.0f;
  for (uint32_t w0 = i; w0 < p.words; w0 += kKeep * TPT) {
    batch(w0);
#pragma unroll
    for (uint32_t u = 0; u < kKeep; ++u)
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(keep[u].get(k)));
  }
  if constexpr (TPT > kWave) {
    static_assert(TPT == THREADS, "a row is a wavefront's part or the workgroup's");
    top = wave_max(top);
    if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) top = fmaxf(top, red[w]);
  } else {
#pragma unroll
    for (int m = 1; m < TPT; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, kWave));
  }
  if (row >= p.rows) return;
  const int e = 141 - static_cast<int>(__float_as_uint(top) >> 23);
  if (i == 0) p.out.exps[row] = 18 - e;
  const uint32_t tile = row / R, steps = p.words / kSlots<R>, subs = p.words / GWS;
  for (uint32_t w0 = i; w0 < p.words; w0 += kKeep * TPT) {
    if (p.words > kKeep * TPT) batch(w0);
#pragma unroll
    for (uint32_t u = 0; u < kKeep; ++u) {
      const uint32_t w = w0 + u * TPT;
      if (w >= p.words) break;  // whole groups of GWS lanes leave together (words is a multiple of GWS)
      float sum = 0.0f;
      f16x8 hi, lo;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        constexpr int nibble[8] = {0, 4, 1, 5, 2, 6, 3, 7};
        const float s = live ? ldexpf(keep[u].get(nibble[k]), e) : 0.0f;
        sum += s;
        hi[k] = static_cast<_Float16>(s);
        if constexpr (NT == 2) lo[k] = static_cast<_Float16>(s - static_cast<float>(hi[k]));
      }
      const uint32_t sub = w / GWS, iw = w % GWS;
      const uint32_t lane = iw / GW * R + row % R, step = sub * GW + iw % GW;
      _Float16* f = p.out.frag + ((static_cast<size_t>(tile) * steps + step) * NT * kWave + lane) * 8u;
      *reinterpret_cast<f16x8*>(f) = hi;
      if constexpr (NT == 2) *reinterpret_cast<f16x8*>(f + kWave * 8u) = lo;
      sum = row_sum<GWS < 16 ? GWS : 16>(sum);
      if constexpr (MANY) {
        if (iw == 0) {
          store_sum(*many, tile, sub, row % R, sum * 0x1p-18f);
          if (sub + 1u == subs)
            for (uint32_t z = subs; z < many->kgs * 16u; ++z) store_sum(*many, tile, z, row % R, 0.0f);
        }
      } else {
        if (iw == 0) p.out.sums[(static_cast<size_t>(tile) * subs + sub) * R + row % R] = sum * 0x1p-18f;
      }
    }
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
  constexpr uint32_t kAhead = 4;  // pieces of 8 columns in flight
  const size_t xo = t * p.stride;
  Raw8<XT> x[kAhead];
  auto load_x = [&](uint32_t w0) {
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) {
      const uint32_t w = w0 + u * kWave < p.words ? w0 + u * kWave : p.words - 1u;
      load_raw8<XT>(p.x, xo + 8u * w, p.x_wide, x[u]);
    }
  };
  load_x(lane);  // while the adapter's id and rank are on their way
  uint32_t a = 0;
  const uint32_t rank = token_rank(p.ad, p.ids, t, a);
  float s = 0.0f;
  if (j < rank) {
    const float scale = p.ad.scales ? p.ad.scales[a] : 1.0f;
    const size_t ao = (static_cast<size_t>(a) * p.ad.max_rank + j) * p.words * 8u;
    for (uint32_t w0 = lane; w0 < p.words; w0 += kAhead * kWave) {
      if (w0 != lane) load_x(w0);
      Raw8<AT> c[kAhead];
#pragma unroll
      for (uint32_t u = 0; u < kAhead; ++u) {
        const uint32_t w = w0 + u * kWave < p.words ? w0 + u * kWave : p.words - 1u;
        load_raw8<AT>(p.ad.a, ao + 8u * w, p.a_wide, c[u]);
      }
#pragma unroll
      for (uint32_t u = 0; u < kAhead; ++u) {
        float d = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) d = fmaf(x[u].get(k), c[u].get(k), d);
        s += w0 + u * kWave < p.words ? d : 0.0f;
      }
    }
    s = wave_sum(s) * scale;
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
// A workgroup owns R rows of W and R tokens; its wavefronts split the columns
// and their sums are added in LDS in wavefront order. The lanes of an
// instruction's D columns are rows of W, so a lane needs one scale and bias
// per sub-group. What bounds it is the latency of one stage (words, then the
// sums, then the adapters' rows): 37 fp32 tokens through 2048 x 4096 take 5 us
// of preparation and 12 here, 64 bf16 ones through 12289 x 2048 take 5 and 23
// (35 MB, 25 of them B_a of 64 adapters: 1.5 TB/s).
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
  constexpr uint32_t kMask = 0x03C003C0u;
  const u32x4 v = {(w << 6) & kMask, (w << 2) & kMask, (w >> 2) & kMask, (w >> 6) & kMask};
  return __builtin_bit_cast(f16x8, v);
}
__device__ __forceinline__ f16x8 load_frag(const _Float16* p) { return __builtin_bit_cast(f16x8, ldg<u32x4>(p)); }

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
  uint32_t stage_subs, stage_log2;  // few tokens: sub-groups of a stage, log2 of its chunks rounded up
};

__device__ __forceinline__ float adapter_element(const osmd_adapters& ad, size_t o) {
  return ad.dtype == OSM_META_F32    ? meta_at<OSM_META_F32>(ad.b, o)
         : ad.dtype == OSM_META_BF16 ? meta_at<OSM_META_BF16>(ad.b, o)
                                     : meta_at<OSM_META_F16>(ad.b, o);
}

// Columns of B taken ahead of their use (16-bit adapters, rows of whole
// 16-byte pieces): up to 16.
struct ExpandAhead {
  uint32_t a, rank;
  uint4 b[2];
};
__device__ __forceinline__ void expand_ahead(const ProjectParams& p, uint32_t t, uint32_t n, ExpandAhead& x) {
  x.a = 0;
  x.rank = token_rank(p.ad, p.ids, t, x.a);
  if (p.b_wide && p.ad.dtype != OSM_META_F32 && x.rank != 0u) {
    const uint16_t* b = static_cast<const uint16_t*>(p.ad.b) + (static_cast<size_t>(x.a) * p.w.out_dim + n) * p.ad.max_rank;
    x.b[0] = ldg16(b);
    x.b[1] = ldg16(b + (p.ad.max_rank > 8u ? 8u : 0u));
  }
}

// s + the first `count` (at most 8) of b . v.
template <typename B>
__device__ __forceinline__ float dot8(const B& b, const float* v, uint32_t count, float s) {
  const float4 lo = *reinterpret_cast<const float4*>(v), hi = *reinterpret_cast<const float4*>(v + 4);
  const float c[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int k = 0; k < 8; ++k) s = static_cast<uint32_t>(k) < count ? fmaf(b[k], c[k], s) : s;
  return s;
}

// (B_a v_t)_n for one token and row.
__device__ __forceinline__ float expand_one(const ProjectParams& p, uint32_t t, uint32_t n, const ExpandAhead& x) {
  if (x.rank == 0u) return 0.0f;
  const size_t o = (static_cast<size_t>(x.a) * p.w.out_dim + n) * p.ad.max_rank;
  const float* v = p.in.v + static_cast<size_t>(t) * p.in.vr;
  float s = 0.0f;
  uint32_t j = 0;
  if (p.b_wide && p.ad.dtype != OSM_META_F32) {
    const bool bf = p.ad.dtype == OSM_META_BF16;
    for (; j < x.rank; j += 8u) {
      const uint4 q = j == 0u ? x.b[0] : j == 8u ? x.b[1] : ldg16(static_cast<const uint16_t*>(p.ad.b) + o + j);
      const uint32_t u[4] = {q.x, q.y, q.z, q.w};
      float b[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        b[2 * i] = bf ? bf16_to_f32(u[i] & 0xFFFFu) : f16_to_f32(u[i] & 0xFFFFu);
        b[2 * i + 1] = bf ? __uint_as_float(u[i] & 0xFFFF0000u) : f16_to_f32(u[i] >> 16);
      }
      s = dot8(b, v + j, x.rank - j, s);
    }
    return s;
  }
  for (; j < x.rank; ++j) s = fmaf(adapter_element(p.ad, o + j), v[j], s);
  return s;
}

constexpr int kFewWaves = 8;
constexpr int kWaitVmcnt0 = 0x0F70;  // s_waitcnt operand: vector memory counter 0, the others at their maximum
// Vector memory counter n and LDS counter 0.
constexpr int wait_vm_lgkm(int n) { return (n & 15) | (n >> 4 << 14) | 7 << 4; }

// 16 bytes per lane from global memory straight into LDS, lane l's at
// dst + 16 l (dst wave-uniform).
__device__ __forceinline__ void load_lds16(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(src, dst, 16, 0, 0);
}
__device__ __forceinline__ void load_lds4(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(src, dst, 4, 0, 0);
}

// A stage is what a workgroup holds in LDS at a time: its R rows' words of
// up to 4096 (R = 16) or 2048 columns, which are contiguous in memory row by
// row, so every load moves whole lines (read by the lanes in operand order
// they took several times as long, a wavefront touching 16 or 32 lines an
// instruction); with them the scales and biases widened to fp32 and the
// tokens' group sums. Chunk c of 16 bytes of row r sits at (r << lc) + (c ^ (r
// & 15)), which spreads the rows' equal chunks over the banks.
template <int R, int NT, int GW, int META>
__global__ __launch_bounds__(kFewWaves* kWave, 4) void project_few_kernel(ProjectParams p) {
  typedef typename Tile<R>::acc acc_t;
  constexpr int A = kAcc<R>;
  constexpr uint32_t GWS = GW * kSlots<R>;
  constexpr uint32_t kChunks = 2048u / R;          // of a row in a stage
  constexpr uint32_t kSubs = kChunks * 4u / GWS;   // sub-groups in a stage
  constexpr int P = (R * R + kFewWaves * kWave - 1) / (kFewWaves * kWave);  // outputs of a thread
  __shared__ __attribute__((aligned(16))) union {
    uint4 w[R * kChunks];
    float part[kFewWaves][A][kWave];
  } lds;
  __shared__ float scale[kSubs][R + 1], bias[kSubs][R + 1];
  __shared__ __attribute__((aligned(16))) float sums[kSubs * R];
  const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const uint32_t N = p.w.out_dim, words = p.w.packed_cols, subs = words / GWS, steps = subs * GW;
  const uint32_t n0 = blockIdx.x * R, tile = blockIdx.y, row = lane % R, slot = lane / R;
  const uint32_t lc = p.stage_log2, swizzle = (1u << lc) - 1u < 15u ? (1u << lc) - 1u : 15u;
  const _Float16* frag = p.in.frag + static_cast<size_t>(tile) * steps * NT * kWave * 8u + lane * 8u;
  const float* tile_sums = p.in.sums + static_cast<size_t>(tile) * subs * R;
  acc_t total;
#pragma unroll
  for (int i = 0; i < A; ++i) total[i] = 0.0f;
  ExpandAhead ahead[P];
#pragma unroll
  for (int o = 0; o < P; ++o) ahead[o].rank = 0u;
  for (uint32_t S0 = 0; S0 < subs; S0 += p.stage_subs) {
    const uint32_t S = subs - S0 < p.stage_subs ? subs - S0 : p.stage_subs;
    if (S0 != 0u) __syncthreads();  // the stage before is read
    const uint32_t chunks = S * GWS / 4u;
    for (uint32_t i0 = wave * kWave; i0 < R << lc; i0 += kFewWaves * kWave) {
      const uint32_t i = i0 + lane, r = i >> lc, c = (i & ((1u << lc) - 1u)) ^ (r & swizzle);
      const size_t n = n0 + r < N ? n0 + r : N - 1u;
      if (i < R << lc) load_lds16(p.w.packed + n * words + S0 * GWS + 4u * (c < chunks ? c : chunks - 1u), &lds.w[i0]);
    }
    for (uint32_t i0 = wave * kWave; i0 < S * R / 4u; i0 += kFewWaves * kWave)
      if (i0 + lane < S * R / 4u) load_lds16(tile_sums + S0 * R + 4u * (i0 + lane), sums + 4u * i0);
    for (uint32_t i = tid; i < R * S; i += kFewWaves * kWave) {
      const uint32_t r = i / S, s = i % S;
      const size_t o = static_cast<size_t>(n0 + r < N ? n0 + r : N - 1u) * p.groups + (S0 + s) / p.per_group;
      scale[s][r] = meta_at<META>(p.w.scales, o);
      bias[s][r] = meta_at<META>(p.w.biases, o);
    }
    const uint32_t s0 = S * wave / kFewWaves, s1 = S * (wave + 1u) / kFewWaves;
    // The next sub-group's operands are loaded while one computes; not in the
    // widest case, where two workgroups' registers (128 a lane) hold one.
    constexpr bool kNext = R == 16 || GW * NT < 8;
    f16x8 x[kNext ? 2 : 1][GW * NT];
    auto load = [&](f16x8 (&v)[GW * NT], uint32_t s) {
      const uint32_t c = S0 + (s < s1 ? s : s0 < s1 ? s1 - 1u : 0u);
#pragma unroll
      for (int k = 0; k < GW * NT; ++k) v[k] = load_frag(frag + (static_cast<size_t>(c) * GW * NT + k) * kWave * 8u);
    };
    load(x[0], s0);
    if (S0 == 0u && p.ad.count) {
#pragma unroll
      for (int o = 0; o < P; ++o) {
        const uint32_t i = tid + o * kFewWaves * kWave, t = tile * R + i / R, nn = n0 + i % R;
        if (i < R * R && t < p.tokens && nn < N) expand_ahead(p, t, nn, ahead[o]);
      }
    }
    __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
    __syncthreads();
    auto compute = [&](const f16x8 (&v)[GW * NT], uint32_t s) {
      const uint32_t word = s * GWS + slot * GW;
      const uint32_t* q = reinterpret_cast<const uint32_t*>(&lds.w[(row << lc) + ((word / 4u) ^ (row & swizzle))]) + word % 4u;
      uint32_t w[GW];
      if constexpr (GW == 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(q);
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
      } else if constexpr (GW == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(q);
        w[0] = u.x, w[1] = u.y;
      } else {
        w[0] = *q;
      }
      const float sc = scale[s][row], bc = bias[s][row];
      acc_t d;
#pragma unroll
      for (int i = 0; i < A; ++i) d[i] = 0.0f;
#pragma unroll
      for (int k = 0; k < GW; ++k) {
        const f16x8 b = nibble_operand(w[k]);
#pragma unroll
        for (int t = 0; t < NT; ++t) d = Tile<R>::mfma(v[k * NT + t], b, d);
      }
#pragma unroll
      for (int i = 0; i < A / 4; ++i) {
        const float4 xs = *reinterpret_cast<const float4*>(sums + s * R + Tile<R>::row(lane, 4 * i));
        total[4 * i] = fmaf(sc, d[4 * i], fmaf(bc, xs.x, total[4 * i]));
        total[4 * i + 1] = fmaf(sc, d[4 * i + 1], fmaf(bc, xs.y, total[4 * i + 1]));
        total[4 * i + 2] = fmaf(sc, d[4 * i + 2], fmaf(bc, xs.z, total[4 * i + 2]));
        total[4 * i + 3] = fmaf(sc, d[4 * i + 3], fmaf(bc, xs.w, total[4 * i + 3]));
      }
    };
    if constexpr (kNext) {
      for (uint32_t s = s0; s < s1; s += 2u) {
        load(x[1], s + 1u);
        compute(x[0], s);
        load(x[0], s + 2u);
        if (s + 1u < s1) compute(x[1], s + 1u);
      }
    } else {
      for (uint32_t s = s0; s < s1; ++s) {
        compute(x[0], s);
        load(x[0], s + 1u);
      }
    }
  }
  // The adapters' part of each output, while other wavefronts still sum.
  float e[P] = {};
  if (p.ad.count) {
#pragma unroll
    for (int o = 0; o < P; ++o) {
      const uint32_t i = tid + o * kFewWaves * kWave;
      e[o] = expand_one(p, tile * R + i / R, n0 + i % R, ahead[o]);
    }
  }
  __syncthreads();  // the words are read; their place holds the sums
#pragma unroll
  for (int i = 0; i < A; ++i) lds.part[wave][i][lane] = total[i];
  __syncthreads();
#pragma unroll
  for (int o = 0; o < P; ++o) {
    const uint32_t i = tid + o * kFewWaves * kWave, tr = i / R, t = tile * R + tr, nn = n0 + i % R;
    if (i >= R * R || t >= p.tokens || nn >= N) continue;
    const uint32_t r = R == 16 ? tr % 4u : tr / 8u * 4u + tr % 4u;
    const uint32_t l = (R == 16 ? tr / 4u : tr / 4u % 2u) * R + i % R;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < kFewWaves; ++k) y += lds.part[k][r][l];
    store_out(p.y, p.y_dtype, t * p.y_stride + nn, ldexpf(y, p.in.exps[t]) + e[o]);
  }
}

// ---- one to four tokens ----------------------------------------------------------
// A wavefront takes ROWS rows of W; a lane holds 32 consecutive columns of
// each token in registers (a chunk, within one quantisation group) and the
// chunk's sum for the bias. No preparation: one launch, after the shrink (2.4
// us; 4096 x 2048 for one token then takes 5.2 to 5.6, 4.9 MB).
constexpr int kVecWaves = 4;

template <int XT>
__device__ __forceinline__ void load32(const void* x, size_t o, bool wide, float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float u[8];
    load8<XT>(x, o + 8u * i, wide, u);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[8 * i + k] = u[k];
  }
}

struct VecParams {
  ProjectParams p;
  const void* x;
  size_t stride;
  uint32_t wide;
};

template <int META, int XT, int TV, int ROWS>
__global__ __launch_bounds__(kVecWaves* kWave) void project_vec_kernel(VecParams vp) {
  const ProjectParams& p = vp.p;
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t N = p.w.out_dim, words = p.w.packed_cols, chunks = words / 4u, G = p.w.group;
  const uint32_t n0 = (blockIdx.x * kVecWaves + wave) * ROWS, t0 = blockIdx.y * TV;
  if (n0 >= N) return;
  // The adapters' columns, one a lane, join the lanes' sums; the first 64 are
  // loaded before the weights.
  uint32_t a[TV] = {}, rank[TV];
  float column[ROWS][TV], v[TV];
  auto load_columns = [&](int t, uint32_t j) {
    v[t] = p.in.v[static_cast<size_t>(t0 + t) * p.in.vr + j];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const size_t n = n0 + r < N ? n0 + r : N - 1u;
      column[r][t] = adapter_element(p.ad, (a[t] * static_cast<size_t>(N) + n) * p.ad.max_rank + j);
    }
  };
#pragma unroll
  for (int t = 0; t < TV; ++t) {
    rank[t] = t0 + t < p.tokens ? token_rank(p.ad, p.ids, t0 + t, a[t]) : 0u;
    if (lane < rank[t]) load_columns(t, lane);
  }
  float acc[ROWS][TV] = {};
  for (uint32_t c = lane; c < chunks; c += kWave) {
    uint4 q[ROWS];
    uint32_t sb[ROWS], bb[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const size_t n = n0 + r < N ? n0 + r : N - 1u;
      q[r] = ldg16(p.w.packed + n * words + 4u * c);
      sb[r] = meta_bits<META>(p.w.scales, n * p.groups + 32u * c / G);
      bb[r] = meta_bits<META>(p.w.biases, n * p.groups + 32u * c / G);
    }
    float x[TV][32], sum[TV];
#pragma unroll
    for (int t = 0; t < TV; ++t) {
      load32<XT>(vp.x, (t0 + t < p.tokens ? t0 + t : t0) * vp.stride + 32u * c, vp.wide, x[t]);
      sum[t] = 0.0f;
#pragma unroll
      for (int k = 0; k < 32; ++k) sum[t] += x[t][k];
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int t = 0; t < TV; ++t)
        acc[r][t] = fmaf(meta_widen<META>(sb[r]), nib_dot32(q[r], x[t]), fmaf(meta_widen<META>(bb[r]), sum[t], acc[r][t]));
  }
#pragma unroll
  for (int t = 0; t < TV; ++t)
    for (uint32_t j = lane; j < rank[t]; j += kWave) {
      if (j != lane) load_columns(t, j);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) acc[r][t] = fmaf(column[r][t], v[t], acc[r][t]);
    }
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int t = 0; t < TV; ++t) {
      const float y = wave_sum(acc[r][t]);
      if (lane == 0 && n0 + r < N && t0 + t < p.tokens) store_out(p.y, p.y_dtype, (t0 + t) * p.y_stride + n0 + r, y);
    }
}

// ---- many tokens -------------------------------------------------------------------
// Tiles of 32 x 32 outputs, W unpacked in registers and used for MT tiles of
// tokens; the tokens' fragments and the packed words go straight from memory
// into LDS, a ring of stages ahead of the one that computes. Per output and
// sub-group of 64 columns that is 64 products on the matrix cores against one
// FMA (the scale) and 64 / (32 MT) unpacked nibbles on the vector units; the
// biases, a product of [tokens, sub-groups] by [sub-groups, rows], are on the
// matrix cores too. Their factors are split into bf16 terms (the sums into
// three; a bias into one, two or three by its type), products below 2^-24 of
// the whole left out. Before the main launch one prepares x (as above), the
// scales transposed to [sub-group][row] and the biases as operands.
// 4,096 bf16 tokens through 8192 x 4096, rank 64: 345 to 354 us here (281 GFLOP, 800
// TFLOP/s; the slope is 63 us per 1,024 columns, so some 80 are a tile's
// beginning and end, where a compute unit has nothing else to run) and 46 + 5
// before it, which are the first products' loads from L2 and x's round trip.
template <int AT>
constexpr int kTerms = AT == OSM_META_BF16 ? 1 : AT == OSM_META_F16 ? 2 : 3;  // exact in that many bf16 terms

// v = t[0] + t[1] + ..., each the bf16 nearest to what is left.
template <int NT>
__device__ __forceinline__ void split_terms(const float (&v)[8], bf16x8 (&t)[NT]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    float left = v[k];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      t[i][k] = static_cast<__bf16>(left);
      if (i + 1 < NT) left -= static_cast<float>(t[i][k]);
    }
  }
}

__device__ __forceinline__ f32x16 mfma_bf16(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_bf16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// c + a b, terms i and j with i + j < 3.
template <int NA, int NB, typename C>
__device__ __forceinline__ C mfma_terms(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], C c) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < 3) c = mfma_bf16(a[i], b[j], c);
  return c;
}

// The same of eight elements as loaded.
template <int T, int NT>
__device__ __forceinline__ void raw_terms(const Raw8<T>& r, bf16x8 (&t)[NT]) {
  if constexpr (T == OSM_META_BF16) {
    const u32x4 v = {r.u[0], r.u[1], r.u[2], r.u[3]};
    t[0] = __builtin_bit_cast(bf16x8, v);
  } else {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = r.get(k);
    split_terms(v, t);
  }
}

__device__ __forceinline__ bf16x8 load_bf16(const __bf16* p) { return __builtin_bit_cast(bf16x8, ldg<u32x4>(p)); }

// Scales and biases of W for sub-groups of which `per_group` make a group: a
// workgroup takes 16 sub-groups of 32 rows; what lies past the last is zero.
template <int META>
__device__ __forceinline__ void prepare_meta(const osmd_q4_proj& w, uint32_t groups, uint32_t per_group, uint32_t subs,
                                             const ManyPrepared& out, uint32_t block) {
  constexpr int NT = kTerms<META>;
  const uint32_t nb = block / out.kgs, kg = block % out.kgs;
  for (uint32_t i = threadIdx.x; i < 512u; i += blockDim.x) {
    const uint32_t r = i % 32u, s = i / 32u, n = nb * 32u + r, sub = kg * 16u + s;
    const bool in = n < w.out_dim && sub < subs;
    const size_t o = static_cast<size_t>(in ? n : 0u) * groups + (in ? sub / per_group : 0u);
    if (sub < subs) out.scales[static_cast<size_t>(sub) * out.scale_row + n] = in ? meta_at<META>(w.scales, o) : 0.0f;
    if (sub == 0u) out.scales[static_cast<size_t>(subs) * out.scale_row + n] = 0.0f;
    float left = in ? meta_at<META>(w.biases, o) : 0.0f;
    const uint32_t lane = s / 8u * 32u + r;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const __bf16 b = static_cast<__bf16>(left);
      out.bias_frag[(((static_cast<size_t>(nb) * out.kgs + kg) * NT + t) * kWave + lane) * 8u + s % 8u] = b;
      left -= static_cast<float>(b);
    }
  }
}

// v of tiles of 16 tokens (in `order`): x and A_a split into bf16 terms, the
// wavefronts taking the columns in turn, kSteps steps of loads in flight; one
// pass per adapter that the tile holds and 16 JB rank rows.
constexpr int kShrinkManyWaves = 8;
struct ShrinkManyParams {
  ShrinkParams s;
  const uint32_t* order;
  __bf16* v_frag;
};

template <int XT, int AT, int JB>
__device__ __forceinline__ void shrink_tile(const ShrinkManyParams& sp, uint32_t block) {
  const ShrinkParams& p = sp.s;
  constexpr int NX = kTerms<XT>, NA = kTerms<AT>;
  // Steps in flight, within some 180 registers: one workgroup a compute unit
  // (fewer in flight or spilled registers for two cost more: 46 us and 53 or
  // more for 4,096 tokens of 4,096 columns, rank 64).
  constexpr int kSteps = JB == 1 ? 8 : AT == OSM_META_F32 ? 2 : 4;
  __shared__ float part[kShrinkManyWaves][JB][4][kWave];
  const uint32_t lane = threadIdx.x % kWave, K = p.words * 8u;
  const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / kWave)));
  const uint32_t tiles = (p.tokens + 15u) / 16u, i0 = block % tiles * 16u, j0 = block / tiles * 16u * JB;
  const uint32_t i = i0 + lane % 16u, slot = lane / 16u;
  const uint32_t t = i < p.tokens ? (sp.order ? sp.order[i] : i) : 0u;
  const size_t xo = t * p.stride + 8u * slot;
  // The batch of x that the registers hold starts at column `held`; rows of
  // one batch are read once for all adapters, and before those are known.
  constexpr uint32_t kApart = kShrinkManyWaves * 32u;
  Raw8<XT> x[kSteps];
  uint32_t held = wave * 32u;
  auto load_x = [&](uint32_t k0) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const uint32_t k = k0 + s * kApart;
      load_raw8<XT>(p.x, xo + (k < K ? k : K - 32u), p.x_wide, x[s]);
    }
  };
  load_x(held);
  uint32_t a = 0;
  const uint32_t rank = i < p.tokens ? token_rank(p.ad, p.ids, t, a) : 0u;
  uint64_t left = __ballot(rank != 0u) & 0xFFFFull;
  while (left) {
    const int leader = __builtin_ctzll(left);
    const uint32_t aa = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(a), leader));
    const uint32_t rr = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(rank), leader));
    const uint64_t same = __ballot(rank != 0u && a == aa) & 0xFFFFull;
    left &= ~same;
    const float scale = p.ad.scales ? p.ad.scales[aa] : 1.0f;
    f32x4 acc[JB];
    size_t ao[JB];
#pragma unroll
    for (int b = 0; b < JB; ++b) {
      acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
      const uint32_t j = j0 + 16u * b + lane % 16u;  // rows past the rank repeat its last
      ao[b] = (static_cast<size_t>(aa) * p.ad.max_rank + (j < rr ? j : rr - 1u)) * K + 8u * slot;
    }
    Raw8<AT> c[kSteps][JB];
    for (uint32_t k0 = wave * 32u; k0 < K; k0 += kSteps * kApart) {
      if (held != k0) load_x(k0);
      held = k0;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t k = k0 + s * kApart;
#pragma unroll
        for (int b = 0; b < JB; ++b) load_raw8<AT>(p.ad.a, ao[b] + (k < K ? k : K - 32u), p.a_wide, c[s][b]);
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (k0 + s * kApart >= K) break;
        bf16x8 xt[NX];
        raw_terms(x[s], xt);
#pragma unroll
        for (int b = 0; b < JB; ++b) {
          bf16x8 at[NA];
          raw_terms(c[s][b], at);
          acc[b] = mfma_terms(xt, at, acc[b]);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < JB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[wave][b][e][lane] = acc[b][e];
    __syncthreads();
    for (uint32_t o = threadIdx.x; o < 16u * 16u * JB; o += kShrinkManyWaves * kWave) {
      const uint32_t r = o / (16u * JB), j = o % (16u * JB);
      if (!((same >> r) & 1u) || j0 + j >= p.vr) continue;
      const uint32_t l = r / 4u * 16u + j % 16u;
      float y = 0.0f;
#pragma unroll
      for (int w = 0; w < kShrinkManyWaves; ++w) y += part[w][j / 16u][r % 4u][l];
      // As the three bf16 terms that the tiled product reads.
      y = j0 + j < rr ? y * scale : 0.0f;
      const uint32_t it = i0 + r, jt = j0 + j, fl = jt % 16u / 8u * 32u + it % 32u;
      __bf16* f = sp.v_frag + ((static_cast<size_t>(it / 32u) * (p.vr / 16u) + jt / 16u) * 3u * kWave + fl) * 8u + jt % 8u;
#pragma unroll
      for (int t = 0; t < 3; ++t) {
        const __bf16 b = static_cast<__bf16>(y);
        f[t * kWave * 8u] = b;
        y -= static_cast<float>(b);
      }
    }
    __syncthreads();
  }
}

// One launch before the tiled product: workgroups that shrink, then those that
// prepare x, then W's scales and biases.
struct PrepareManyParams {
  ShrinkManyParams s;
  PrepareParams x;
  ManyPrepared many;
  osmd_q4_proj w;
  uint32_t groups, per_group, subs, shrink_blocks, x_blocks;
};
constexpr int kPrepareThreads = kShrinkManyWaves * kWave;

template <int XT, int GW, int TPT, int AT, int JB>
__global__ __launch_bounds__(kPrepareThreads) void prepare_many_kernel(PrepareManyParams p) {
  if (blockIdx.x < p.shrink_blocks) return shrink_tile<XT, AT, JB>(p.s, blockIdx.x);
  const uint32_t block = blockIdx.x - p.shrink_blocks;
  if (block < p.x_blocks) return prepare_rows<XT, 32, GW, TPT, kPrepareThreads, true>(p.x, block, &p.many);
  if (p.w.meta_dtype == OSM_META_F32)
    prepare_meta<OSM_META_F32>(p.w, p.groups, p.per_group, p.subs, p.many, block - p.x_blocks);
  else if (p.w.meta_dtype == OSM_META_F16)
    prepare_meta<OSM_META_F16>(p.w, p.groups, p.per_group, p.subs, p.many, block - p.x_blocks);
  else
    prepare_meta<OSM_META_BF16>(p.w, p.groups, p.per_group, p.subs, p.many, block - p.x_blocks);
}

struct ManyParams {
  ProjectParams p;
  ManyPrepared many;
  const uint32_t* order;
  uint32_t tiles;
  uint32_t y_wide;  // 16-bit rows of y that 16 bytes at a time can be stored to
};

// e += v of the tile's tokens times B_a of the rows nrow, over the a's rank;
// the loads of kDeep steps are in flight together.
template <int AT, int NB>
__device__ __forceinline__ void expand_tile(const ProjectParams& p, uint32_t a, uint32_t rank, const __bf16* v_frag,
                                            const uint32_t (&nrow)[NB], uint32_t slot, f32x16 (&e)[NB]) {
  struct Step {
    bf16x8 v[3];
    Raw8<AT> b[NB];
  };
  constexpr uint32_t kDeep = AT == OSM_META_F32 ? 2 : 4;
  Step step[kDeep];
  const uint32_t R = p.ad.max_rank;
  auto load = [&](Step& s, uint32_t j) {
#pragma unroll
    for (int t = 0; t < 3; ++t) s.v[t] = load_bf16(v_frag + (j / 16u * 3u + t) * kWave * 8u);
    const uint32_t c = j + 8u * slot;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const size_t o = (static_cast<size_t>(a) * p.w.out_dim + nrow[nb]) * R;
      if (p.b_wide && R % 8u == 0u) {
        load_raw8<AT>(p.ad.b, o + (c < R ? c : 0u), true, s.b[nb]);
      } else {
        // Rows that hold no whole pieces: element by element, the last one again past the end.
        auto at = [&](uint32_t k) { return meta_bits<AT>(p.ad.b, o + (c + k < R ? c + k : R - 1u)); };
        if constexpr (AT == OSM_META_F32) {
#pragma unroll
          for (int k = 0; k < 8; ++k) s.b[nb].u[k] = at(k);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) s.b[nb].u[k] = at(2 * k) | (at(2 * k + 1) << 16);
        }
      }
    }
  };
  auto compute = [&](const Step& s, uint32_t j) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      Raw8<AT> raw = s.b[nb];
      if (j + 16u > rank) {  // zero from the rank on
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (j + 8u * slot + k >= rank) raw.clear(k);
      }
      bf16x8 bt[kTerms<AT>];
      raw_terms(raw, bt);
      e[nb] = mfma_terms(s.v, bt, e[nb]);
    }
  };
  for (uint32_t j0 = 0; j0 < rank; j0 += 16u * kDeep) {
#pragma unroll
    for (uint32_t d = 0; d < kDeep; ++d)
      if (j0 + 16u * d < rank) load(step[d], j0 + 16u * d);
#pragma unroll
    for (uint32_t d = 0; d < kDeep; ++d)
      if (j0 + 16u * d < rank) compute(step[d], j0 + 16u * d);
  }
}

// SK columns a stage, sub-groups of 16 * GW columns. WM x WN wavefronts of MT
// token tiles and NB row blocks each, WK of them to a tile: they take a
// stage's sub-groups in turn. RING stages in LDS: one computes while the next
// are on their way into it, straight from memory. Each stage has an array of
// its own: the compiler then knows that a stage's reads need not wait for the
// loads into the others. The loop has no branch: it runs whole rounds of the
// ring, stages past the last with scales of 0 on data read again.
template <int META, int NT, int MT, int NB, int WM, int WN, int WK, int GW, int SK, int RING>
__global__ __launch_bounds__(WM* WN* WK* kWave, 2) void project_many_kernel(ManyParams mp) {
  const ProjectParams& p = mp.p;
  constexpr int kBiasTerms = kTerms<META>;
  constexpr uint32_t TH = WM * WN * WK * kWave;
  constexpr uint32_t SC = 16u * GW, STEPS = SK / 16, SUBS = SK / SC / WK;  // SUBS: a wavefront's, of a stage
  static_assert(SK % (SC * WK) == 0, "every wavefront takes as many sub-groups");
  constexpr uint32_t kTiles = WM * MT, kRows = WN * NB * 32u, kCh = SK / 32;  // kCh: 16-byte chunks of a row
  constexpr uint32_t kXUnits = kTiles * STEPS * NT * kWave, kWUnits = kRows * kCh;
  static_assert(kXUnits % TH == 0 && kWUnits % kWave == 0, "whole wavefronts");
  static_assert(kWUnits % TH == 0 || TH % kWUnits == 0, "a round of words is every wavefront's, or repeated");
  // Scales: a wavefront's own, 4 bytes a lane, two blocks of 32 rows a load.
  static_assert(SUBS * NB % 2 == 0, "whole wavefronts");
  constexpr uint32_t kWPer = (kWUnits + TH - 1u) / TH, kSPer = SUBS * NB / 2u;
  constexpr int kLoads = kXUnits / TH + kWPer + kSPer;  // of a wavefront, a stage
  constexpr uint32_t kStage = kXUnits + kWPer * TH + TH / kWave * kSPer * 16u;
  __shared__ uint4 l0[kStage], l1[kStage], l2[kStage], l3[RING == 4 ? kStage : 1];
  __shared__ uint32_t info[4][kTiles * 32u];
  const uint32_t tid = threadIdx.x, lane = tid % kWave;
  const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(tid / kWave)));
  const uint32_t wm = wave % WM, wn = wave / WM % WN, wk = wave / (WM * WN);
  const uint32_t row = lane % 32u, slot = lane / 32u;
  const uint32_t N = p.w.out_dim, words = p.w.packed_cols, steps = words / 2u, subs = words * 8u / SC;
  // Workgroups go to the 8 XCDs in turn: each XCD takes a run of the tiles, so
  // that its L2 holds what its compute units read. Of a run, 8 token tiles go
  // through the row blocks together.
  const uint32_t tgrid = (mp.tiles + kTiles - 1u) / kTiles, ngrid = (N + kRows - 1u) / kRows;
  uint32_t b = blockIdx.x;
  {
    const uint32_t total = tgrid * ngrid, per = total / 8u, rest = total % 8u, x = b % 8u, y = b / 8u;
    b = x * per + (x < rest ? x : rest) + y;
  }
  const uint32_t band = b / (8u * ngrid), width = tgrid - band * 8u < 8u ? tgrid - band * 8u : 8u, in_band = b - band * 8u * ngrid;
  const uint32_t tile0 = (band * 8u + in_band % width) * kTiles, n0 = in_band / width * kRows;
  const uint4* frag = reinterpret_cast<const uint4*>(p.in.frag);
  const uint32_t stages = (subs + SUBS * WK - 1u) / (SUBS * WK);
  // The lane's chunks of words: row pointers and place in a stage's chunks.
  const uint4* wrow[kWPer];
  uint32_t wchunk[kWPer];
#pragma unroll
  for (uint32_t i = 0; i < kWPer; ++i) {
    // Chunk c of row r sits at r kCh + (c ^ (r % kCh)), which spreads the rows' equal chunks over the banks.
    const uint32_t u = (tid + i * TH) % kWUnits, r = u / kCh;
    const uint32_t n = n0 + r < N ? n0 + r : N - 1u;
    wrow[i] = reinterpret_cast<const uint4*>(p.w.packed + static_cast<size_t>(n) * words);
    wchunk[i] = (u % kCh) ^ (r % kCh);
  }
  auto issue = [&](uint4* to, uint32_t st) {
    // Scales (their rows are padded to whole workgroups').
#pragma unroll
    for (uint32_t i = 0; i < kSPer; ++i) {
      // Block pair i: of NB = 2 sub-group i, of NB = 1 sub-groups 2 i and 2 i + 1.
      const uint32_t u = NB == 2 ? i : 2u * i + slot, sub = (st * SUBS + u) * WK + wk;
      const float* from = mp.many.scales + static_cast<size_t>(sub < subs ? sub : subs) * mp.many.scale_row + n0 +
                          (NB == 2 ? wn * 64u + lane : wn * 32u + row);
      load_lds4(from, to + (kXUnits + kWPer * TH + (wave * kSPer + i) * 16u));
    }
    // Fragments, 1 KB each; past a row's last step its last is read again.
#pragma unroll
    for (uint32_t i = 0; i < kXUnits / TH; ++i) {
      const uint32_t f = i * (TH / kWave) + wave, m = f / (STEPS * NT), o = f % (STEPS * NT);
      const uint32_t tile = tile0 + m < mp.tiles ? tile0 + m : mp.tiles - 1u;
      const uint32_t at = st * STEPS * NT + o < steps * NT ? st * STEPS * NT + o : steps * NT - 1u;
      load_lds16(frag + (static_cast<size_t>(tile) * steps * NT + at) * kWave + lane, to + f * kWave);
    }
#pragma unroll
    for (uint32_t i = 0; i < kWPer; ++i) {
      const uint32_t c = wchunk[i] + st * kCh, last = words / 4u - 1u;
      load_lds16(wrow[i] + (c < last ? c : last), to + (kXUnits + i * TH + wave * kWave));
    }
  };
  issue(l0, 0u);
  issue(l1, 1u);
  issue(l2, 2u);
  if constexpr (RING == 4) issue(l3, 3u);
  // What the end needs of the tiles' tokens: place in y, exponent, adapter, rank.
  for (uint32_t i = tid; i < kTiles * 32u; i += TH) {
    const uint32_t at = tile0 * 32u + i;
    uint32_t a = 0;
    const uint32_t token = at < p.tokens ? (mp.order ? mp.order[at] : at) : 0u;
    info[0][i] = token;
    info[1][i] = at < p.tokens ? static_cast<uint32_t>(p.in.exps[at]) : 0u;
    info[3][i] = p.ad.count && at < p.tokens ? token_rank(p.ad, p.ids, token, a) : 0u;
    info[2][i] = a;
  }
  f32x16 total[NB][MT];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) total[nb][m][i] = 0.0f;
  // The biases' part, a run of sub-groups' operands on their way while one's
  // products run.
  {
    struct Run {
      bf16x8 x[MT][kSumTerms], b[NB][kBiasTerms];
    } run[2];
    const __bf16* xf[MT];
    const __bf16* bf[NB];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const uint32_t tl = tile0 + wm * MT + m, tile = tl < mp.tiles ? tl : mp.tiles - 1u;
      xf[m] = mp.many.sum_frag + (static_cast<size_t>(tile) * mp.many.kgs * kSumTerms * kWave + lane) * 8u;
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      bf[nb] = mp.many.bias_frag + (static_cast<size_t>(n0 / 32u + wn * NB + nb) * mp.many.kgs * kBiasTerms * kWave + lane) * 8u;
    auto load = [&](Run& r, uint32_t kg) {
      const size_t at = kg < mp.many.kgs ? kg : mp.many.kgs - 1u;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < kSumTerms; ++t) r.x[m][t] = load_bf16(xf[m] + (at * kSumTerms + t) * kWave * 8u);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int t = 0; t < kBiasTerms; ++t) r.b[nb][t] = load_bf16(bf[nb] + (at * kBiasTerms + t) * kWave * 8u);
    };
    auto add = [&](const Run& r) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int m = 0; m < MT; ++m) total[nb][m] = mfma_terms(r.x[m], r.b[nb], total[nb][m]);
    };
    load(run[0], wk);
    for (uint32_t kg = wk; kg < mp.many.kgs; kg += 2u * WK) {
      load(run[1], kg + WK);
      add(run[0]);
      load(run[0], kg + 2u * WK);
      if (kg + WK < mp.many.kgs) add(run[1]);
    }
  }
  // Units of one sub-group and token tile: while one's matrix instructions
  // run, the next one's operands come from LDS and the block before is scaled
  // and added.
  constexpr uint32_t kUnits = SUBS * MT;
  static_assert(kUnits * NB % 2u == 0u, "blocks alternate between two sets of registers");
  f16x8 x[2][GW * NT], q[NB][GW];
  uint4 w[NB];
  float scale[NB];
  f32x16 d[2];
  float before = 0.0f;  // the scale of the block before
#pragma unroll
  for (int i = 0; i < 16; ++i) d[1][i] = 0.0f;
  auto load_unit = [&](const uint4* at, uint32_t j, f16x8 (&xx)[GW * NT]) {
    const uint32_t u = j / MT, m = j % MT;
    if (m == 0u) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const uint32_t r = (wn * NB + nb) * 32u + row, word = ((u * WK + wk) * 2u + slot) * GW;
        const uint32_t* from = reinterpret_cast<const uint32_t*>(at + kXUnits + r * kCh + ((word / 4u) ^ (r % kCh))) + word % 4u;
        if constexpr (GW == 4) {
          w[nb] = *reinterpret_cast<const uint4*>(from);
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(from);
          w[nb].x = v.x, w[nb].y = v.y;
        }
        scale[nb] = reinterpret_cast<const float*>(at + kXUnits + kWPer * TH + wave * kSPer * 16u)[(u * NB + nb) * 32u + row];
      }
    }
#pragma unroll
    for (int k = 0; k < GW * NT; ++k)
      xx[k] = __builtin_bit_cast(f16x8, at[((wm * MT + m) * STEPS + (u * WK + wk) * GW) * NT * kWave + k * kWave + lane]);
  };
  // Products of unit j (`words` and `scales` are its sub-group's), each block
  // of rows beside the sum of the block before.
  auto run_unit = [&](uint32_t j, const uint4 (&words)[NB], const float (&scales)[NB], const f16x8 (&xx)[GW * NT]) {
    const uint32_t m = j % MT;
    if (m == 0u) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        q[nb][0] = nibble_operand(words[nb].x), q[nb][1] = nibble_operand(words[nb].y);
        if constexpr (GW == 4) q[nb][2] = nibble_operand(words[nb].z), q[nb][3] = nibble_operand(words[nb].w);
      }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const uint32_t s = j * NB + nb, pm = (s + kUnits * NB - 1u) / NB % MT, pb = (s + NB - 1u) % NB;
      f32x16& to = d[s % 2u];
      const f32x16& from = d[(s + 1u) % 2u];
#pragma unroll
      for (int i = 0; i < 16; ++i) to[i] = 0.0f;
#pragma unroll
      for (int k = 0; k < GW; ++k)
#pragma unroll
        for (int t = 0; t < NT; ++t) to = Tile<32>::mfma(xx[k * NT + t], q[nb][k], to);
#pragma unroll
      for (int i = 0; i < 16; ++i) total[pb][pm][i] = fmaf(before, from[i], total[pb][pm][i]);
      before = scales[nb];
    }
  };
  // A stage ends where its last unit's operands are read: its place is then
  // filled anew, and the next stage read, before that unit's products. The
  // wait leaves at most the RING - 2 stages after next outstanding: loads
  // complete in order, so the next stage's are done, on every wavefront after
  // the barrier; this wavefront's LDS reads are done as well.
  auto arrive = [&](auto left) {
    constexpr int LEFT = decltype(left)::value;
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm(LEFT * kLoads));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto step = [&](uint4* at, const uint4* then, uint32_t st) {
#pragma unroll
    for (uint32_t j = 0; j < kUnits; ++j) {
      uint4 words[NB];
      float scales[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) words[nb] = w[nb], scales[nb] = scale[nb];
      if (j + 1u < kUnits) {
        load_unit(at, j + 1u, x[(j + 1u) % 2u]);
      } else {
        arrive(std::integral_constant<int, RING - 2>{});
        issue(at, st + RING);
        load_unit(then, 0u, x[(j + 1u) % 2u]);
      }
      __builtin_amdgcn_sched_barrier(0);
      run_unit(j, words, scales, x[j % 2u]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  arrive(std::integral_constant<int, RING - 1>{});
  load_unit(l0, 0u, x[0]);
  static_assert(kUnits % 2u == 0u, "units alternate between two sets of registers");
  for (uint32_t st = 0; st < stages; st += RING) {
    step(l0, l1, st);
    step(l1, l2, st + 1u);
    if constexpr (RING == 4) {
      step(l2, l3, st + 2u);
      step(l3, l0, st + 3u);
    } else {
      step(l2, l0, st + 2u);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) total[NB - 1][MT - 1][i] = fmaf(before, d[1][i], total[NB - 1][MT - 1][i]);
  __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);  // nothing is on its way into LDS when the workgroup ends or uses it anew
  uint32_t nrow[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const uint32_t n = n0 + (wn * NB + nb) * 32u + row;
    nrow[nb] = n < N ? n : N - 1u;
  }
  __syncthreads();  // the stages' places are free
  if constexpr (WK > 1) {
    // The wavefronts of a tile add up in the first's registers, in order.
    static_assert(WK == 2, "one other");
    static_assert(sizeof(float) * 16u * NB * MT * kWave * WM * WN <= sizeof(l0), "the sums fit a stage's place");
    float* part = reinterpret_cast<float*>(l0) + (wave % (WM * WN)) * 16u * NB * MT * kWave;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (wk == 1u) part[((nb * MT + m) * 16 + i) * kWave + lane] = total[nb][m][i];
    __syncthreads();
    if (wk == 1u) return;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) total[nb][m][i] += part[((nb * MT + m) * 16 + i) * kWave + lane];
  }
  // Outputs of 16 bits go through LDS (a place of the wavefront's own, in the
  // second and third stages') and leave as 16 bytes a lane, whole lines where
  // two lanes' halves of a line each would go out alone.
  constexpr uint32_t kPitch = NB * 32u + 8u;  // elements of a token's row there
  static_assert((WM * WN + 1u) / 2u * 32u * kPitch * 2u <= sizeof(l1), "the outputs fit two stages' places");
  uint16_t* mine = reinterpret_cast<uint16_t*>(wave % 2u ? l1 : l2) + wave % (WM * WN) / 2u * 32u * kPitch;
  const uint32_t nw = n0 + wn * NB * 32u;  // the wavefront's first row of W
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const uint32_t local = (wm * MT + m) * 32u, tile = tile0 + wm * MT + m;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int e = static_cast<int>(info[1][local + Tile<32>::row(lane, i)]);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) total[nb][m][i] = ldexpf(total[nb][m][i], e);
    }
    // One product per adapter that the tile's tokens have, added to its own
    // tokens' rows.
    const uint32_t a = info[2][local + row], rank = info[3][local + row];
    uint32_t left = static_cast<uint32_t>(__ballot(rank != 0u));
    while (left) {
      const int leader = __builtin_ctz(left);
      const uint32_t aa = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(a), leader));
      const uint32_t rr = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(rank), leader));
      const uint32_t same = static_cast<uint32_t>(__ballot(rank != 0u && a == aa));
      left &= ~same;
      f32x16 e[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int k = 0; k < 16; ++k) e[nb][k] = 0.0f;
      const __bf16* v = mp.many.v_frag + (static_cast<size_t>(tile < mp.tiles ? tile : 0u) * (p.in.vr / 16u) * 3u * kWave + lane) * 8u;
      if (p.ad.dtype == OSM_META_BF16)
        expand_tile<OSM_META_BF16, NB>(p, aa, rr, v, nrow, slot, e);
      else if (p.ad.dtype == OSM_META_F16)
        expand_tile<OSM_META_F16, NB>(p, aa, rr, v, nrow, slot, e);
      else
        expand_tile<OSM_META_F32, NB>(p, aa, rr, v, nrow, slot, e);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const bool own = (same >> Tile<32>::row(lane, k)) & 1u;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) total[nb][m][k] += own ? e[nb][k] : 0.0f;
      }
    }
    if (mp.y_wide && nw + NB * 32u <= N) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const float v = total[nb][m][i];
          mine[Tile<32>::row(lane, i) * kPitch + nb * 32u + row] =
              p.y_dtype == OSM_META_BF16 ? __builtin_bit_cast(uint16_t, static_cast<__bf16>(v))
                                         : __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      constexpr uint32_t kPieces = NB * 4u;  // 16-byte pieces of a token's row
#pragma unroll
      for (uint32_t i = 0; i < 32u * kPieces / kWave; ++i) {
        const uint32_t r = (i * kWave + lane) / kPieces, c = (i * kWave + lane) % kPieces;
        const uint4 v = *reinterpret_cast<const uint4*>(mine + r * kPitch + c * 8u);
        if (tile * 32u + r < p.tokens)
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.y) + info[0][local + r] * p.y_stride + nw + c * 8u) = v;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();  // the next tile's outputs take the same place
      continue;
    }
    auto store = [&](auto put) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t r = Tile<32>::row(lane, i);
        const size_t o = info[0][local + r] * p.y_stride;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const uint32_t n = nw + nb * 32u + row;
          if (tile * 32u + r < p.tokens && n < N) put(o + n, total[nb][m][i]);
        }
      }
    };
    if (p.y_dtype == OSM_META_F32)
      store([&](size_t o, float v) { static_cast<float*>(p.y)[o] = v; });
    else if (p.y_dtype == OSM_META_BF16)
      store([&](size_t o, float v) { static_cast<__bf16*>(p.y)[o] = static_cast<__bf16>(v); });
    else
      store([&](size_t o, float v) { static_cast<_Float16*>(p.y)[o] = static_cast<_Float16>(v); });
  }
}

constexpr int kShrinkWaves = 4;

// v[t, j] = scale_a (A_a x_t)_j: a wavefront per rank row and token.
template <int XT, int AT>
__global__ __launch_bounds__(kShrinkWaves* kWave) void shrink_kernel(ShrinkParams p) {
  for (uint32_t block = blockIdx.x; block < p.tokens * (p.vr / kShrinkWaves); block += gridDim.x) shrink_rows<XT, AT>(p, block);
}

constexpr int kAnyWaves = 4;
constexpr uint32_t kAnyTokens = 4;

// Any geometry: a wavefront per row of W and kAnyTokens tokens, each weight
// dequantised once for them.
template <int META, int XT>
__global__ __launch_bounds__(kAnyWaves* kWave) void project_any_kernel(osmd_project_args p, const float* __restrict__ v,
                                                                       uint32_t vr) {
  const uint32_t N = p.w.out_dim;
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t n = blockIdx.x * kAnyWaves + wave;
  if (n >= N) return;
  const uint32_t words = p.w.packed_cols, G = p.w.group, groups = words * 8u / G;
  for (uint32_t t0 = blockIdx.y * kAnyTokens; t0 < p.tokens; t0 += gridDim.y * kAnyTokens) {
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

constexpr uint32_t kVecTokens = 4;
constexpr uint32_t kFewTokens = 64;

uint32_t round_up(uint32_t n, uint32_t m) { return (n + m - 1u) / m * m; }
size_t align256(size_t n) { return (n + 255u) & ~static_cast<size_t>(255u); }

// What a call runs. sub_cols: columns of a sub-group, 0 where a group is no
// multiple of 32 (one kernel for any).
enum class Path { kAny, kVec, kFew, kMany };
struct Plan {
  Path path;
  bool sort;
  uint32_t sub_cols, tile, rows, terms, vr, kgs, bias_terms;
  size_t frag, sums, exps, scales, biases, order, offsets, counts, v, total;  // workspace offsets
};
Plan plan_of(const osmd_project_args& a) {
  Plan p{};
  const uint32_t G = a.w.group, K = a.w.packed_cols * 8u, N = a.w.out_dim;
  p.vr = a.adapters.count ? round_up(a.adapters.max_rank, 16u) : 0u;
  p.path = G % 32u != 0u             ? Path::kAny
           : a.tokens <= kVecTokens ? Path::kVec
           : a.tokens <= kFewTokens ? Path::kFew
                                    : Path::kMany;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += align256(bytes);
    return o;
  };
  if (p.path == Path::kFew || p.path == Path::kMany) {
    // Tiles of 16 up to 16 tokens, and where tiles of 32 would give fewer
    // workgroups than compute units (37 fp32 tokens through 2048 x 4096: 16
    // us with 32, 11.5 with 16; 64 bf16 ones through 12289 x 2048: 23 and 30).
    p.tile = p.path == Path::kMany || (a.tokens > 16u && (N + 31u) / 32u * ((a.tokens + 31u) / 32u) >= 256u) ? 32u : 16u;
    // Tiles of 32 have no registers for the operands of 128 columns.
    p.sub_cols = G % 128u == 0u && p.tile == 16u ? 128u : G % 64u == 0u ? 64u : 32u;
    p.rows = round_up(a.tokens, p.tile);
    p.terms = a.x_dtype == OSM_META_F32 ? 2u : 1u;
    p.frag = take(static_cast<size_t>(p.rows) * K * 2u * p.terms);
    const uint32_t subs = K / p.sub_cols;
    p.exps = take(static_cast<size_t>(p.rows) * 4u);
    if (p.path == Path::kFew) {
      p.sums = take(static_cast<size_t>(p.rows) * subs * 4u);
    } else {
      p.kgs = (subs + 15u) / 16u;
      p.bias_terms = a.w.meta_dtype == OSM_META_BF16 ? 1u : a.w.meta_dtype == OSM_META_F16 ? 2u : 3u;
      p.sums = take(static_cast<size_t>(p.rows) * p.kgs * 16u * kSumTerms * 2u);
      p.scales = take((static_cast<size_t>(subs) + 1u) * round_up(N, 256u) * 4u);
      p.biases = take(static_cast<size_t>(round_up(N, 256u)) * p.kgs * 16u * p.bias_terms * 2u);
      p.sort = a.adapters.count > 1u && a.adapters.count <= OSMD_GROUP_MAX_BUCKETS;
      if (p.sort) {
        p.order = take(static_cast<size_t>(a.tokens) * 4u);
        p.offsets = take((static_cast<size_t>(a.adapters.count) + 1u) * 4u);
        p.counts = take(osmd_group_rows_workspace(a.tokens, a.adapters.count));
      }
    }
  }
  // v: fp32 rows, or the three bf16 terms of whole tiles.
  p.v = take(p.path == Path::kMany ? static_cast<size_t>(p.rows) * p.vr * 6u : static_cast<size_t>(a.tokens) * p.vr * sizeof(float));
  p.total = at;
  return p;
}

Prepared prepared_of(const Plan& pl, uint8_t* work) {
  Prepared out;
  out.frag = reinterpret_cast<_Float16*>(work + pl.frag);
  out.sums = reinterpret_cast<float*>(work + pl.sums);
  out.exps = reinterpret_cast<int32_t*>(work + pl.exps);
  out.v = reinterpret_cast<float*>(work + pl.v);
  out.vr = pl.vr;
  return out;
}

ShrinkParams shrink_params(const osmd_project_args& a, const Plan& pl, uint8_t* work) {
  ShrinkParams sp{};
  sp.x = a.x;
  sp.stride = a.x_stride;
  sp.tokens = a.tokens;
  sp.words = a.w.packed_cols;
  sp.x_wide = wide_rows(a.x, a.x_stride, a.x_dtype) ? 1u : 0u;
  sp.a_wide = wide_rows(a.adapters.a, 8u * a.w.packed_cols, a.adapters.dtype) ? 1u : 0u;
  sp.ad = a.adapters;
  sp.ids = a.adapter_ids;
  sp.v = prepared_of(pl, work).v;
  sp.vr = pl.vr;
  return sp;
}

ProjectParams project_params(const osmd_project_args& a, const Plan& pl, uint8_t* work) {
  ProjectParams p{};
  p.w = a.w;
  p.groups = a.w.packed_cols * 8u / a.w.group;
  p.per_group = pl.sub_cols ? a.w.group / pl.sub_cols : 1u;
  p.in = prepared_of(pl, work);
  p.y = a.y;
  p.y_stride = a.y_stride;
  p.y_dtype = a.y_dtype;
  p.tokens = a.tokens;
  p.ad = a.adapters;
  p.ids = a.adapter_ids;
  p.b_wide = wide_rows(a.adapters.b, a.adapters.max_rank, a.adapters.dtype) ? 1u : 0u;
  return p;
}

int launch_shrink(const osmd_project_args& a, const Plan& pl, uint8_t* work, hipStream_t st) {
  const ShrinkParams sp = shrink_params(a, pl, work);
  const uint32_t blocks = a.tokens * (pl.vr / kShrinkWaves), grid = blocks < 1u << 20 ? blocks : 1u << 20;
  return by_dtype(a.x_dtype, [&](auto xt) {
    return by_dtype(a.adapters.dtype, [&](auto at) {
      shrink_kernel<decltype(xt)::value, decltype(at)::value><<<grid, kShrinkWaves * kWave, 0, st>>>(sp);
      return launch_status();
    });
  });
}

template <int GW>
int launch_many(const osmd_project_args& a, const Plan& pl, uint8_t* work, hipStream_t st) {
  ManyParams mp{};
  mp.p = project_params(a, pl, work);
  mp.tiles = pl.rows / 32u;
  mp.y_wide = a.y_dtype != OSM_META_F32 && wide_rows(a.y, a.y_stride, a.y_dtype) ? 1u : 0u;
  mp.many.sum_frag = reinterpret_cast<__bf16*>(work + pl.sums);
  mp.many.scales = reinterpret_cast<float*>(work + pl.scales);
  mp.many.bias_frag = reinterpret_cast<__bf16*>(work + pl.biases);
  mp.many.kgs = pl.kgs;
  mp.many.scale_row = round_up(a.w.out_dim, 256u);
  mp.many.v_frag = reinterpret_cast<__bf16*>(work + pl.v);
  int r = 0;
  if (pl.sort) {
    // Tokens by adapter: a tile then holds one, or the few whose runs meet in it.
    uint32_t* order = reinterpret_cast<uint32_t*>(work + pl.order);
    r = osmd_group_rows(a.adapter_ids, a.tokens, a.adapters.count, reinterpret_cast<uint32_t*>(work + pl.offsets), order, work + pl.counts,
                        st);
    if (r != 0) return r;
    mp.order = order;
  }
  PrepareManyParams pp{};
  pp.x.x = a.x;
  pp.x.stride = a.x_stride;
  pp.x.tokens = a.tokens;
  pp.x.rows = pl.rows;
  pp.x.words = a.w.packed_cols;
  pp.x.wide = wide_rows(a.x, a.x_stride, a.x_dtype) ? 1u : 0u;
  pp.x.order = mp.order;
  pp.x.out = mp.p.in;
  pp.many = mp.many;
  pp.w = a.w;
  pp.groups = mp.p.groups;
  pp.per_group = mp.p.per_group;
  pp.subs = a.w.packed_cols * 8u / pl.sub_cols;
  // A wavefront a row while it holds the row in registers, else the workgroup.
  const bool wave_rows = a.w.packed_cols <= 512u;
  pp.x_blocks = wave_rows ? pl.rows / kShrinkManyWaves : pl.rows;
  const uint32_t meta_blocks = round_up(a.w.out_dim, 256u) / 32u * pl.kgs;
  const uint32_t ranks = pl.vr <= 16u ? 16u : 64u;  // of a shrinking workgroup
  pp.shrink_blocks = a.adapters.count ? (a.tokens + 15u) / 16u * ((pl.vr + ranks - 1u) / ranks) : 0u;
  pp.s = ShrinkManyParams{shrink_params(a, pl, work), mp.order, mp.many.v_frag};
  r = by_dtype(a.x_dtype, [&](auto xt) {
    return by_dtype(a.adapters.dtype, [&](auto at) {
      constexpr int X = decltype(xt)::value, A = decltype(at)::value;
      auto go = [&](auto kernel) {
        kernel<<<pp.shrink_blocks + pp.x_blocks + meta_blocks, kPrepareThreads, 0, st>>>(pp);
        return launch_status();
      };
      if (ranks == 16u)
        return wave_rows ? go(prepare_many_kernel<X, GW, 64, A, 1>) : go(prepare_many_kernel<X, GW, kPrepareThreads, A, 1>);
      return wave_rows ? go(prepare_many_kernel<X, GW, 64, A, 4>) : go(prepare_many_kernel<X, GW, kPrepareThreads, A, 4>);
    });
  });
  if (r != 0) return r;
  auto go = [&](auto kernel, uint32_t tiles, uint32_t rows, uint32_t threads) {
    const uint32_t grid = (mp.tiles + tiles - 1u) / tiles * ((a.w.out_dim + rows - 1u) / rows);
    kernel<<<grid, threads, 0, st>>>(mp);
    return launch_status();
  };
  // The tile with the least time expected: microseconds of a round of
  // workgroups at 2,048 columns (the others' in proportion) times the rounds.
  // One term, tiles of 64 x 128 / 128 x 128 / 128 x 256, measured: 512 tokens
  // through 4,096 rows 17 / 27 / 35, 1,024: 32 / 30 / 38, 2,048: 65 / 47 / 44.
  // Two terms, 32 x 128 / 128 x 256: 32 / 84, 62 / 88, 132 / 105.
  auto groups = [&](uint32_t tiles, uint32_t rows) {
    return (mp.tiles + tiles - 1u) / tiles * ((a.w.out_dim + rows - 1u) / rows);
  };
  return by_dtype(a.w.meta_dtype, [&](auto meta) {
    constexpr int M = decltype(meta)::value;
    if (pl.terms == 2u) {
      if ((groups(1u, 128u) + 255u) / 256u * 16u <= (groups(4u, 256u) + 255u) / 256u * 102u)
        return go(project_many_kernel<M, 2, 1, 1, 1, 4, 2, GW, 256, 3>, 1u, 128u, 512u);
      return go(project_many_kernel<M, 2, 2, 2, 2, 4, 1, GW, 64, 3>, 4u, 256u, 512u);
    }
    const uint32_t small = (groups(2u, 128u) + 255u) / 256u * 16u;
    const uint32_t middle = groups(4u, 128u) <= 256u ? 28u : (groups(4u, 128u) + 511u) / 512u * 47u;
    const uint32_t large = (groups(4u, 256u) + 255u) / 256u * 43u;
    if (small <= middle && small <= large) return go(project_many_kernel<M, 1, 1, 1, 2, 4, 1, GW, 128, 4>, 2u, 128u, 512u);
    if (middle <= large) return go(project_many_kernel<M, 1, 2, 2, 2, 2, 1, GW, 64, 3>, 4u, 128u, 256u);
    return go(project_many_kernel<M, 1, 2, 2, 2, 4, 1, GW, 64, 3>, 4u, 256u, 512u);
  });
}

int launch_vec(const osmd_project_args& a, const Plan& pl, uint8_t* work, hipStream_t st) {
  VecParams vp{};
  vp.p = project_params(a, pl, work);
  vp.x = a.x;
  vp.stride = a.x_stride;
  vp.wide = wide_rows(a.x, a.x_stride, a.x_dtype) ? 1u : 0u;
  return by_dtype(a.w.meta_dtype, [&](auto meta) {
    return by_dtype(a.x_dtype, [&](auto xt) {
      constexpr int M = decltype(meta)::value, X = decltype(xt)::value;
      auto go = [&](auto kernel, uint32_t rows, uint32_t tokens) {
        const uint32_t per = kVecWaves * rows;
        kernel<<<dim3((a.w.out_dim + per - 1u) / per, (a.tokens + tokens - 1u) / tokens), kVecWaves * kWave, 0, st>>>(vp);
      };
      if (a.tokens == 1u)
        go(project_vec_kernel<M, X, 1, 4>, 4u, 1u);
      else
        go(project_vec_kernel<M, X, 2, 4>, 4u, 2u);
      return launch_status();
    });
  });
}

template <int R, int GW>
int launch_few(const osmd_project_args& a, const Plan& pl, uint8_t* work, hipStream_t st) {
  PrepareParams pp{};
  pp.x = a.x;
  pp.stride = a.x_stride;
  pp.tokens = a.tokens;
  pp.rows = pl.rows;
  pp.words = a.w.packed_cols;
  pp.wide = wide_rows(a.x, a.x_stride, a.x_dtype) ? 1u : 0u;
  pp.out = prepared_of(pl, work);
  const ShrinkParams sp = shrink_params(a, pl, work);
  const uint32_t shrink_blocks = a.tokens * (pl.vr / 4u);
  int r = by_dtype(a.x_dtype, [&](auto xt) {
    return by_dtype(a.adapters.dtype, [&](auto at) {
      prepare_few_kernel<decltype(xt)::value, R, GW, decltype(at)::value>
          <<<pl.rows + shrink_blocks, 256, 0, st>>>(pp, sp, pl.rows);
      return launch_status();
    });
  });
  if (r != 0) return r;
  ProjectParams p = project_params(a, pl, work);
  const uint32_t per_chunk = pl.sub_cols / 32u, subs = a.w.packed_cols * 8u / pl.sub_cols;
  const uint32_t most = 2048u / R / per_chunk;  // sub-groups that a stage holds
  const uint32_t stages = (subs + most - 1u) / most;
  p.stage_subs = (subs + stages - 1u) / stages;
  while ((1u << p.stage_log2) < p.stage_subs * per_chunk) ++p.stage_log2;
  const dim3 grid((a.w.out_dim + R - 1u) / R, pl.rows / R);
  return by_dtype(a.w.meta_dtype, [&](auto meta) {
    constexpr int M = decltype(meta)::value;
    if (pl.terms == 2u)
      project_few_kernel<R, 2, GW, M><<<grid, kFewWaves * kWave, 0, st>>>(p);
    else
      project_few_kernel<R, 1, GW, M><<<grid, kFewWaves * kWave, 0, st>>>(p);
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
  if (pl.path == Path::kMany)
    return pl.sub_cols == 64u ? launch_many<4>(*a, pl, work, st) : launch_many<2>(*a, pl, work, st);
  if (pl.path == Path::kFew) {
    if (pl.tile == 32u) return pl.sub_cols == 64u ? launch_few<32, 4>(*a, pl, work, st) : launch_few<32, 2>(*a, pl, work, st);
    return pl.sub_cols == 128u  ? launch_few<16, 4>(*a, pl, work, st)
           : pl.sub_cols == 64u ? launch_few<16, 2>(*a, pl, work, st)
                                : launch_few<16, 1>(*a, pl, work, st);
  }
  if (a->adapters.count) {
    const int r = launch_shrink(*a, pl, work, st);
    if (r != 0) return r;
  }
  if (pl.path == Path::kVec) return launch_vec(*a, pl, work, st);
  const float* v = reinterpret_cast<const float*>(work + pl.v);
  const uint32_t blocks = (a->w.out_dim + kAnyWaves - 1u) / kAnyWaves;
  const uint32_t tiles = (a->tokens + kAnyTokens - 1u) / kAnyTokens;
  return by_dtype(a->w.meta_dtype, [&](auto meta) {
    return by_dtype(a->x_dtype, [&](auto xt) {
      project_any_kernel<decltype(meta)::value, decltype(xt)::value>
          <<<dim3(blocks, tiles < 65535u ? tiles : 65535u), kAnyWaves * kWave, 0, st>>>(*a, v, pl.vr);
      return launch_status();
    });
  });
}

}  // extern "C"
