// Transformer-block operators for B200 (sm_100a): the gated feed-forward
// block with its backward, counter-based dropout, and the product in 8-bit
// integers.  C ABI: include/gfblock.h.
//
// All matrix products run on one persistent, warp-specialised tcgen05 kernel
// (gemm_kernel) whose epilogues hold the rest of each operator.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <nvtx3/nvToolsExt.h>

#include <atomic>
#include <type_traits>

#include "gfblock.h"
#include "tc100.cuh"

namespace gf {
gf_status fail(gf_status s, const char* fmt, ...) __attribute__((format(printf, 2, 3)));  // gfield.cu
}

namespace gfb {

using gf::fail;

struct Range {
  explicit Range(const char* name) { nvtxRangePushA(name); }
  ~Range() { nvtxRangePop(); }
};

constexpr int64_t kMaxDim = (int64_t(1) << 31) - 512;  // sizes stay in int32 after rounding up to a tile

template <typename I>
constexpr I round_up(I v, I m) {
  return (v + m - 1) / m * m;
}
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

__device__ uint32_t g_status;  // GF_FLAG_*, sticky (gf_block_status)

// Bounds checks of the debug build (-DGF_CHECK, libgfield_check.so): every
// access to global memory by an address of its own (TMA copies are clipped by
// their tensor maps) is tested against its extent; a failure sets
// GF_FLAG_BOUNDS and the access is skipped (never a trap).  In the release
// build the check is the constant true and compiles away.
#ifdef GF_CHECK
__device__ __forceinline__ bool bounds_ok(bool ok) {
  if (!ok) atomicOr(&g_status, GF_FLAG_BOUNDS);
  return ok;
}
#define GFB_IN_BOUNDS(cond) gfb::bounds_ok(cond)
#else
#define GFB_IN_BOUNDS(cond) ((void)sizeof(cond), true)  // unevaluated: names its operands, costs nothing
#endif
// v in [0, n), and the `count` elements from v within n
__device__ __forceinline__ bool within(int64_t v, int64_t n, int64_t count = 1) { return v >= 0 && v + count <= n; }

// ---------------------------------------------------------------------------
// element types

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(v);
  else return __half2float(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
  else return __float2half_rn(v);
}
// two 16-bit elements in a register, the first in the low half
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// ---------------------------------------------------------------------------
// Philox-4x32-10 (Salmon et al., SC 2011): ten rounds of two 32x32 -> 64-bit
// products, the words swapped and the two halves of the key xored in; the key
// steps by the two Weyl constants.

struct DropArgs {
  uint64_t seed;
  const uint64_t* seed_ptr;
  uint32_t site;
  uint32_t threshold;  // keep when the word is at least this
  float scale;
  int32_t on;
};

struct Philox {
  uint32_t k0, k1, site;
  __device__ __forceinline__ Philox(const DropArgs& d) {
    const uint64_t s = d.seed_ptr ? *d.seed_ptr : d.seed;
    k0 = (uint32_t)s;
    k1 = (uint32_t)(s >> 32);
    site = d.site;
  }
  // the four words of elements (row, 4 * block .. 4 * block + 3)
  __device__ __forceinline__ uint4 operator()(uint32_t block, uint64_t row) const {
    uint32_t c0 = block, c1 = (uint32_t)row, c2 = site, c3 = (uint32_t)(row >> 32);
    uint32_t a = k0, b = k1;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
      c0 = (uint32_t)(p1 >> 32) ^ c1 ^ a;
      c2 = (uint32_t)(p0 >> 32) ^ c3 ^ b;
      c1 = (uint32_t)p1;
      c3 = (uint32_t)p0;
      a += 0x9E3779B9u;
      b += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
  }
};

DropArgs drop_args(const gf_dropout_rule& r) {
  DropArgs d{};
  d.seed = r.seed;
  d.seed_ptr = r.seed_ptr;
  d.site = r.site;
  double t = r.p * 4294967296.0;
  t = __builtin_rint(t);
  d.threshold = t >= 4294967295.0 ? 0xFFFFFFFFu : (uint32_t)t;
  d.scale = (float)(1.0 / (1.0 - r.p));
  d.on = r.p > 0.0;
  return d;
}

gf_status check_rule(const char* who, const gf_dropout_rule& r) {
  if (!(r.p >= 0.0 && r.p < 1.0)) return fail(GF_ERR_INVALID_ARG, "%s: dropout p must be in [0, 1)", who);
  if (r.reserved != 0) return fail(GF_ERR_INVALID_ARG, "%s: reserved fields must be 0", who);
  if (reinterpret_cast<uintptr_t>(r.seed_ptr) & 7u)
    return fail(GF_ERR_INVALID_ARG, "%s: seed_ptr must be 8-byte aligned", who);
  return GF_OK;
}

// ---------------------------------------------------------------------------
// activations, two arguments at a time: value and slope.
//
// gelu: with z = |g| / sqrt(2), Phi(-|g|) = erfc(z) / 2 = t Q(t) exp(-z^2),
// t = 1 / (1 + 0.36 z), the form of Abramowitz and Stegun 7.1.26.  Their five
// coefficients bound the absolute error alone (half a step of fp16 relative to
// Phi at g = -4, 1 % at -8, 3 % at -12); these seven are a minimax fit by
// linear programming to both: 1.1e-8 absolute and 1.4e-5 relative.  In fp32
// steps, with the exponent's rounding, that is 1.8e-7 and 2.2e-5 down to
// g = -13, a twentieth of half a step of fp16; below -13.2 the exponential
// leaves fp32's normal range and Phi is 0.  The two further coefficients take
// 1 to 2 % of a training pass (16384 x 320 x 1280: 144.1 -> 145.4 us).
// exp(-z^2) is also the density in the slope Phi(g) + g phi(g).  silu:
// g / (1 + exp(-g)), within 2e-5 of itself down to g = -87, where the
// reciprocal becomes 0.
// Both take one base-2 exponential and one reciprocal of the special-function
// unit per argument, each a few 2^-22 relative.

template <int ACT, bool SLOPE>
__device__ __forceinline__ void activate(float g0, float g1, uint64_t& value, uint64_t& slope) {
  using namespace tc;
  const uint64_t g = pack_f2(g0, g1);
  if constexpr (ACT == GF_ACT_GELU) {
    constexpr float kP = 0.36f * 0.70710678118654752f;
    const uint64_t t = pack_f2(rcp(fmaf(fabsf(g0), kP, 1.0f)), rcp(fmaf(fabsf(g1), kP, 1.0f)));
    constexpr float kE = -0.72134752044448170f;  // -log2(e) / 2
    const float2 x = unpack_f2(mul_f2(mul_f2(g, pack_f2(kE, kE)), g));
    const uint64_t e = pack_f2(ex2(x.x), ex2(x.y));
    constexpr float kQ[7] = {0.101156034f,  0.107818983f, 0.055485018f, 0.211434215f,
                             -0.175171271f, 0.280878156f, -0.0816011503f};
    uint64_t q = pack_f2(kQ[6], kQ[6]);  // Horner's rule
#pragma unroll
    for (int i = 5; i >= 0; --i) q = fma_f2(q, t, pack_f2(kQ[i], kQ[i]));
    const float2 tail = unpack_f2(mul_f2(mul_f2(q, t), e));  // Phi(-|g|)
    const uint64_t cdf = pack_f2(g0 > 0.0f ? 1.0f - tail.x : tail.x, g1 > 0.0f ? 1.0f - tail.y : tail.y);
    value = mul_f2(g, cdf);
    if constexpr (SLOPE) slope = fma_f2(mul_f2(g, pack_f2(0.3989422804f, 0.3989422804f)), e, cdf);
  } else {
    constexpr float kE = -1.4426950408889634f;
    const float2 x = unpack_f2(mul_f2(g, pack_f2(kE, kE)));
    const uint64_t sig = pack_f2(rcp(1.0f + ex2(x.x)), rcp(1.0f + ex2(x.y)));
    value = mul_f2(g, sig);
    // sig (1 + g (1 - sig)) = sig + value - value sig
    if constexpr (SLOPE) slope = add_f2(sig, fma_f2(value, mul_f2(sig, pack_f2(-1.0f, -1.0f)), value));
  }
}

// ---------------------------------------------------------------------------
// The product kernel.  D[m, n] = sum_k A(m, k) B(n, k), persistent and
// warp-specialised, on tiles of 128 x bn for one CTA or 256 x bn for a pair:
//  warp 0      TMA producer: 64 k (128 bytes) of both operands per stage
//  warp 1      issues tcgen05.mma into one of two TMEM accumulators
//  the others  epilogue of the other accumulator: warp w reads TMEM lanes
//              32 * (w % 4) onwards, and the warps of a quarter take its
//              32-column chunks in turn
// Each CTA (or pair) walks over a run of tiles and K ranges.
//
// Why pairs: a CTA's tile of 128 x 256 takes (128 + 256) * 128 bytes of
// operands every 512 clocks of products, 96 bytes a clock, and the way from L2
// into an SM gave about 70; in a pair each CTA loads its own rows of A and
// half of B, 64 bytes a clock.

constexpr int kTileM = 128;   // rows of a CTA
constexpr int kMaxN = 256;
constexpr int kABytes = kTileM * 128;
constexpr int kRowsBytes = 32 * 64;     // staging block: 64 bytes of each of a warp's 32 rows
constexpr int kVectorBytes = 32 * 4;    // a warp's vector of 32 floats (bias, scale)
constexpr uint32_t kTmemCols = 512;
constexpr int kSmemLimit = 232448;

enum Epilogue { EPI_STORE, EPI_GATED, EPI_GATED_BWD, EPI_INT8 };

// Warps and shared memory of a variant.  A chunk's result leaves as staging
// blocks through TMA stores, which have the next chunk's arithmetic to be read
// in; what is left holds operand stages.  The gate's arithmetic hides behind
// 16 warps (16384 x 320 x 1280 forward: 34 us, with 8 warps 39), the integer
// results, a conversion each, behind 12 (16384 x 1280 x 10240: 160 us, with 8
// warps 171); the backward, whose products take longer, is no faster with more
// than 8 (1024 x 1280 x 5120: 37 us, with 16 warps and fewer stages 42).
template <int EPI>
struct Config {
  static constexpr int epi_warps = EPI == EPI_GATED ? 16 : EPI == EPI_INT8 ? 12 : 8;
  static constexpr int threads = 64 + 32 * epi_warps;
  static constexpr int blocks = EPI == EPI_GATED ? 1 : 2;
  static constexpr int vectors = EPI == EPI_STORE ? 1 : 2;
  static constexpr int side_bytes = epi_warps * (blocks * kRowsBytes + vectors * kVectorBytes) + 512;
  static constexpr int stage_room = (kSmemLimit - side_bytes) / 1024 * 1024;
};
constexpr int kMaxStages = 8;

struct alignas(64) GemmParams {
  CUtensorMap ma, mb;
  CUtensorMap ma2, mb2;          // GATED_BWD: operands of dh, dy (m, k) and w_out (k, n)
  CUtensorMap mo;                // tiles of 64 bytes x 32 rows of the result (or of the partial products)
  int32_t M, N;                // rows and columns of the result (gated: columns of h, without padding)
  int32_t tiles_m, tiles_n, splits, kb_total, kb_split;
  int32_t rows_m;              // rows of all tiles of M
  int32_t bn;                  // columns of the MMA
  int32_t cols;                // columns of the result per tile: bn, or bn / 2 (gated: value and gate side by side)
  int32_t a_mn, b_mn;          // operand is M/N-contiguous
  int32_t gate_row;            // gated: row of B where the gate half starts
  uint32_t idesc, tx_bytes;
  uint32_t idesc2, tx_bytes2;  // GATED_BWD: of dh
  int32_t kb2;                 // and its k steps
  int32_t stages, stage_bytes;
  int32_t seg_pad, seg;        // result rows come in two runs of `seg` rows, the second starting at seg_pad (0: one run)
  int32_t tma_out;             // the result is written through mo (its rows are 16-byte aligned, in one run)
  int64_t ld_out;
  void* out;                   // STORE, INT8: result
  float* partial;              // splits > 1: [splits][tiles_m * 128][ld_partial]
  int64_t ld_partial;
  const void* bias;            // [N] (gated, forward and backward: [2 N])
  int32_t hp;                  // gated: padded hidden size
  const float* a_scale;
  const float* b_scale;
  DropArgs drop;
};

struct Pipe {  // barriers and the abort flag, in shared memory
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], spare;
  uint32_t tmem, abort;
};
static_assert(sizeof(Pipe) <= 512, "the room behind the staging blocks");

// The tiles of one CTA or pair, columns first: with few column tiles a run of
// consecutive ones, so that its rows of A come from memory once and from L2
// after that; with many, every units-th, so that all units share the rows of
// a few row tiles and neighbouring columns at a time.  us in runs / interleaved,
// 8-bit products of 16384 x 1280 with 10 column tiles 45.8 / 48.5, 14 58.1 /
// 59.3, 16 64.1 / 65.3, 20 83.0 / 83.1, 24 96.5 / 95.5, 40 162.8 / 157.7;
// feed-forwards of 16384 rows with 10 46.9 / 47.5, 16 68.0 / 69.6, 20 125.3 /
// 122.7.  Going on is an addition: a division would stand in every role's way.
constexpr int kRunColumns = 16;
struct Tile {
  int n, m, split;       // tile coordinates
  int m0, n0, kb0, kb1;  // first row of this CTA, first column, range of k steps
  int left;              // tiles still to do, this one included
  int step_n, step_m;    // to the next one
};
template <bool PAIR>
__device__ __forceinline__ void place(const GemmParams& p, Tile& t, uint32_t rank) {
  t.m0 = (t.m * (PAIR ? 2 : 1) + (int)rank) * kTileM;
  t.n0 = t.n * p.cols;
  t.kb0 = t.split * p.kb_split;
  t.kb1 = min(t.kb0 + p.kb_split, p.kb_total);
}
template <bool PAIR>
__device__ __forceinline__ Tile first_tile(const GemmParams& p, uint32_t rank) {
  const uint32_t unit = PAIR ? blockIdx.x >> 1 : blockIdx.x, units = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int64_t items = (int64_t)p.tiles_m * p.tiles_n * p.splits;
  const int64_t each = items / units, more = items - each * units;  // the first `more` units take one more
  const bool run = p.tiles_n <= kRunColumns;
  const int64_t item = run ? unit * each + (unit < more ? unit : more) : unit;
  const int64_t rest = item / p.tiles_n;
  Tile t;
  t.n = (int)(item - rest * p.tiles_n);
  t.split = (int)(rest / p.tiles_m);
  t.m = (int)(rest - (int64_t)t.split * p.tiles_m);
  t.left = (int)(each + (unit < more));
  t.step_m = run ? 0 : (int)(units / p.tiles_n);
  t.step_n = run ? 1 : (int)(units % p.tiles_n);
  place<PAIR>(p, t, rank);
  return t;
}
template <bool PAIR>
__device__ __forceinline__ void next_tile(const GemmParams& p, Tile& t, uint32_t rank) {
  --t.left;
  t.n += t.step_n;
  t.m += t.step_m;
  if (t.n >= p.tiles_n) t.n -= p.tiles_n, ++t.m;
  while (t.m >= p.tiles_m) t.m -= p.tiles_m, ++t.split;
  place<PAIR>(p, t, rank);
}

template <int EPI, typename T, int ACT, bool DROP>
struct EpilogueWarp {
  const GemmParams& p;
  char* stage;
  float* vec0;  // two vectors of 32 floats
  float* vec1;
  const int lane;
  Philox rng;
  float row_scale = 0.0f;  // INT8: of this lane's row
  bool far_scale = false;  // and whether any of the warp's could take a sum past fp32's range

  __device__ __forceinline__ EpilogueWarp(const GemmParams& p_, char* stage_, char* vectors)
      : p(p_), stage(stage_), vec0(reinterpret_cast<float*>(vectors)), vec1(vec0 + 32), lane(threadIdx.x & 31),
        rng(p_.drop) {}

  // Bias and scale of this lane's column of a chunk, fetched ahead.
  struct Ahead {
    float a, b;
  };
  __device__ __forceinline__ void fetch(Ahead& x, int n) const {
    x.a = x.b = 0.0f;
    if (lane < p.N - n) {
      const T* bias = static_cast<const T*>(p.bias);
      if (!GFB_IN_BOUNDS(within(n + lane, p.N))) return;
      if (bias) x.a = to_float(bias[n + lane]);
      if ((EPI == EPI_GATED || EPI == EPI_GATED_BWD) && bias) x.b = to_float(bias[p.N + n + lane]);
      if (EPI == EPI_INT8) x.b = p.b_scale[n + lane];
    }
  }

  // One 32-column chunk at result column n of rows m .. m + 31, from the
  // accumulator columns at `acc` (dh: at `acc2`).  `release` runs once they
  // are read, `fetch_next` once `ahead` is.
  template <typename Release, typename Next>
  __device__ __forceinline__ void chunk(uint32_t acc, uint32_t acc2, const Tile& t, int m, int n, const Ahead& ahead,
                                        Release release, Next fetch_next) {
    uint32_t d[32];
    if constexpr (EPI == EPI_STORE || EPI == EPI_INT8) tc::tmem_load32(d, acc);
    if constexpr (EPI == EPI_STORE) {
      tc::tmem_wait();
      release();
      if (p.splits > 1) {
        const int row = t.split * p.rows_m + m;
        fetch_next();
        begin();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = d[16 * h + i];
          put(h, v);
        }
        send([&] {
          tc::tma_store(&p.mo, block(0), n, row);
          tc::tma_store(&p.mo, block(1), n + 16, row);
        });
        return;
      }
      vectors(ahead);
      fetch_next();
      uint32_t v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = pack2<T>(f(d[2 * i]) + vec0[2 * i], f(d[2 * i + 1]) + vec0[2 * i + 1]);
      begin();
      put(0, v);
      result<2>(1, m, n);
    } else if constexpr (EPI == EPI_INT8) {
      const float s = row_scale;
      vectors(ahead);
      fetch_next();
      tc::tmem_wait();
      release();
      // |sum| <= 2^31: one rounding to fp32, then the two scales and the bias;
      // the smaller scale first where the row's alone could overflow
      if (!far_scale) {
#pragma unroll
        for (int i = 0; i < 32; ++i) d[i] = __float_as_uint((float)(int)d[i] * s * vec1[i] + vec0[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const bool less = s < vec1[i];
          d[i] = __float_as_uint((float)(int)d[i] * (less ? s : vec1[i]) * (less ? vec1[i] : s) + vec0[i]);
        }
      }
      uint32_t v[16];
      begin();
      if constexpr (std::is_same_v<T, float>) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = d[16 * h + i];
          put(h, v);
        }
        result<4>(2, m, n);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = pack2<T>(f(d[2 * i]), f(d[2 * i + 1]));
        put(0, v);
        result<2>(1, m, n);
      }
    } else {
      vectors(ahead);
      fetch_next();
      gated(acc, acc2, m, n, release);
    }
  }

  // Every block must be out of shared memory before the CTA ends.
  __device__ __forceinline__ void finish() {
    if (lane == 0) tc::tma_store_drain();
    __syncwarp();
  }

 private:
  static __device__ __forceinline__ float f(uint32_t v) { return __uint_as_float(v); }

  __device__ __forceinline__ void vectors(const Ahead& x) {
    __syncwarp();
    vec0[lane] = x.a;
    if constexpr (C::vectors == 2) vec1[lane] = x.b;
    __syncwarp();
  }

  // The forward's chunk, h = keep * value * act(gate), or the backward's,
  // du_value = keep * dh * act(gate) and du_gate = keep * dh * value *
  // act'(gate), from the same value and gate in fp32: the backward computes
  // them again instead of reading them.  That is 4 * tokens * hidden *
  // in_features more operations against 8 bytes written and read for every
  // element of h, half the activation memory of the block, and one rounding
  // less in every gradient.  keep is 1 / (1 - p) or 0, 1 without dropout.
  template <typename Release>
  __device__ __forceinline__ void gated(uint32_t acc, uint32_t acc2, int m, int n, Release release) {
    constexpr bool kBack = EPI == EPI_GATED_BWD;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t a[16], g[16], dh[16], o0[8], o1[8];
      const int left = p.N - n - 16 * half;  // the padding columns of h and du are zeros
      tc::tmem_load16(a, acc + 16 * half);
      tc::tmem_load16(g, acc + p.cols + 16 * half);
      if constexpr (kBack) tc::tmem_load16(dh, acc2 + 16 * half);
      tc::tmem_wait();
      if (half == 1) release();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t keep[2];  // of two 16-bit results: ones where they are kept (a dropped one is 0 whatever it holds)
        if constexpr (DROP) {
          const uint4 w = rng((uint32_t)(n + 16 * half + 4 * q) >> 2, (uint32_t)(m + lane));
          const uint32_t th = p.drop.threshold;
          keep[0] = (w.x >= th ? 0xFFFFu : 0u) | (w.y >= th ? 0xFFFF0000u : 0u);
          keep[1] = (w.z >= th ? 0xFFFFu : 0u) | (w.w >= th ? 0xFFFF0000u : 0u);
        }
        const float4 b0 = *reinterpret_cast<const float4*>(vec0 + 16 * half + 4 * q);
        const float4 b1 = *reinterpret_cast<const float4*>(vec1 + 16 * half + 4 * q);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = 4 * q + 2 * i, o = 2 * q + i;
          const uint64_t x = tc::add_f2(tc::pack_f2(f(a[c]), f(a[c + 1])), i ? tc::pack_f2(b0.z, b0.w) : tc::pack_f2(b0.x, b0.y));
          const float2 y = tc::unpack_f2(
              tc::add_f2(tc::pack_f2(f(g[c]), f(g[c + 1])), i ? tc::pack_f2(b1.z, b1.w) : tc::pack_f2(b1.x, b1.y)));
          uint64_t value, slope = 0;
          activate<ACT, kBack>(y.x, y.y, value, slope);
          float2 r;
          if constexpr (kBack) {
            uint64_t d = tc::pack_f2(f(dh[c]), f(dh[c + 1]));
            if constexpr (DROP) d = tc::mul_f2(d, tc::pack_f2(p.drop.scale, p.drop.scale));
            r = tc::unpack_f2(tc::mul_f2(d, value));
            o0[o] = pack2<T>(r.x, r.y);
            r = tc::unpack_f2(tc::mul_f2(tc::mul_f2(d, x), slope));
            o1[o] = pack2<T>(r.x, r.y);
          } else {
            if constexpr (DROP) value = tc::mul_f2(value, tc::pack_f2(p.drop.scale, p.drop.scale));
            r = tc::unpack_f2(tc::mul_f2(x, value));
            o0[o] = pack2<T>(r.x, r.y);
          }
          if constexpr (DROP) {
            o0[o] &= keep[i];
            if constexpr (kBack) o1[o] &= keep[i];
          }
        }
      }
      if (left < 16) {
#pragma unroll
        for (int o = 0; o < 8; ++o) {
          const uint32_t mask = 2 * o + 1 < left ? 0xFFFFFFFFu : 2 * o < left ? 0xFFFFu : 0u;
          o0[o] &= mask;
          if constexpr (kBack) o1[o] &= mask;
        }
      }
      if (half == 0) begin();
      put_half(0, half, o0);
      if constexpr (kBack) put_half(1, half, o1);
    }
    send([&] {
      tc::tma_store(&p.mo, block(0), n, m);
      if constexpr (kBack) tc::tma_store(&p.mo, block(1), p.hp + n, m);
    });
  }

  // Results leave as blocks of 64 bytes of the 32 rows: begin() waits until
  // the last chunk's blocks are read, put() writes lane's row with its 16-byte
  // pieces swizzled as the tensor maps say (piece ^ (row / 2 % 4): eight lanes
  // then cover all banks), send() stores them.
  using C = Config<EPI>;
  __device__ __forceinline__ void begin() {
    if (lane == 0) tc::tma_store_wait<0>();
    __syncwarp();
  }
  __device__ __forceinline__ uint32_t block(int i) const { return tc::smem_addr(stage) + i * kRowsBytes; }
  __device__ __forceinline__ void put_piece(int b, int i, const uint32_t* v) {
    *reinterpret_cast<uint4*>(stage + b * kRowsBytes + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(v[0], v[1], v[2], v[3]);
  }
  __device__ __forceinline__ void put(int b, const uint32_t (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) put_piece(b, i, v + 4 * i);
  }
  __device__ __forceinline__ void put_half(int b, int half, const uint32_t (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) put_piece(b, 2 * half + i, v + 4 * i);
  }
  template <typename Stores>
  __device__ __forceinline__ void send(Stores stores) {
    tc::fence_proxy_async();
    __syncwarp();
    if (lane == 0) {
      stores();
      tc::tma_store_commit();
    }
  }

  // `blocks` blocks of the result, rows m .. m + 31 from column n.
  template <int ES>
  __device__ __forceinline__ void result(int blocks, int m, int n) {
    constexpr int per_row = 64 / ES;
    if (p.tma_out) {
      send([&] {
        tc::tma_store(&p.mo, block(0), n, m);
        if (blocks > 1 && n + per_row < p.N) tc::tma_store(&p.mo, block(1), n + per_row, m);
      });
      return;
    }
    // rows off the 16-byte grid, or in two runs (seg_pad is a multiple of 64:
    // 32 rows never straddle them): element by element, a row's together
    int rows = min(32, p.M - m);
    int64_t row = m;
    if (p.seg_pad) {
      const int in = m >= p.seg_pad ? m - p.seg_pad : m;
      rows = min(rows, p.seg - in);
      row = m >= p.seg_pad ? (int64_t)p.seg + in : in;
    }
    __syncwarp();
    for (int k = 0; k < blocks; ++k) {
      const int at = n + k * per_row, cols = min(per_row, p.N - at);
      char* dst = static_cast<char*>(p.out) + ES * (row * p.ld_out + at);
      for (int i = lane; i < 32 * per_row; i += 32) {
        const int r = i / per_row, c = i % per_row, b = c * ES;
        if (r < rows && c < cols && GFB_IN_BOUNDS(within(row + r, p.seg_pad ? 2 * (int64_t)p.seg : p.M) && within(at + c, p.N))) {
          const char* src = stage + k * kRowsBytes + r * 64 + (((b >> 4) ^ ((r >> 1) & 3)) << 4) + (b & 15);
          if constexpr (ES == 2)
            *reinterpret_cast<uint16_t*>(dst + ES * (r * p.ld_out + c)) = *reinterpret_cast<const uint16_t*>(src);
          else
            *reinterpret_cast<uint32_t*>(dst + ES * (r * p.ld_out + c)) = *reinterpret_cast<const uint32_t*>(src);
        }
      }
    }
  }
};

template <int EPI, typename T, int ACT, bool DROP, bool PAIR>
__global__ void __launch_bounds__(Config<EPI>::threads, 1) gemm_kernel(const __grid_constant__ GemmParams p) {
  using C = Config<EPI>;
  extern __shared__ __align__(1024) char smem[];
  char* staging = smem + C::stage_room;
  char* vectors = staging + C::epi_warps * C::blocks * kRowsBytes;
  Pipe* pipe = reinterpret_cast<Pipe*>(vectors + C::epi_warps * C::vectors * kVectorBytes);
  const uint32_t base = tc::smem_addr(smem);
  if (base & 1023u) {  // the operand tiles' swizzle needs it; the kernel has no other shared memory
    if (threadIdx.x == 0) atomicOr(&g_status, GF_FLAG_TIMEOUT);
    return;
  }
  const uint32_t full = tc::smem_addr(pipe->full), empty = tc::smem_addr(pipe->empty);
  const uint32_t acc_full = tc::smem_addr(pipe->acc_full), acc_empty = tc::smem_addr(pipe->acc_empty);
  volatile uint32_t* abort = &pipe->abort;
  const int warp = threadIdx.x >> 5;
  const uint32_t rank = PAIR ? tc::cluster_rank() : 0;

  if (threadIdx.x == 0) {
    tc::tma_prefetch(&p.ma);
    tc::tma_prefetch(&p.mb);
    if constexpr (EPI == EPI_GATED_BWD) {
      tc::tma_prefetch(&p.ma2);
      tc::tma_prefetch(&p.mb2);
    }
    for (int i = 0; i < p.stages; ++i) {
      tc::mbar_init(full + 8 * i, 1);
      tc::mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(acc_full + 8 * i, 1);
      tc::mbar_init(acc_empty + 8 * i, C::epi_warps * (PAIR ? 2 : 1));
    }
    tc::mbar_init(tc::smem_addr(&pipe->spare), 1);
    pipe->abort = 0;
    tc::fence_barrier_init();
    tc::fence_proxy_async();
  }
  if (warp == 1) tc::tmem_alloc<PAIR>(tc::smem_addr(&pipe->tmem), kTmemCols);
  __syncwarp();
  tc::fence_before();
  if constexpr (PAIR) tc::cluster_sync();
  else __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&pipe->tmem);
  tc::dependency_wait();  // everything up to here is the CTA's own
  tc::let_dependents();

  if (warp == 0) {
    // Both CTAs of a pair load; the copies of both count on the first one's barrier.
    if (tc::elect_one()) {
      uint32_t s = 0, phase = 0, n = 0;  // stage, its phase, stages filled
      bool ok = true;
      const uint32_t full0 = PAIR ? tc::peer_addr(full, 0) : full;
      const int b_cols = PAIR ? p.bn / 2 : p.bn;
      auto load = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
        if constexpr (PAIR) tc::tma_load_pair(dst, map, bar, x, y);
        else tc::tma_load(dst, map, bar, x, y);
      };
      // one stage: fill(its A, its B, the barrier) once the stage is free
      auto stage = [&](uint32_t bytes, auto fill) {
        ok = tc::mbar_wait(empty + 8 * s, phase ^ 1, abort);
        if (!ok) return;
        const uint32_t a = base + s * p.stage_bytes;
        if (rank == 0) tc::mbar_expect_tx(full + 8 * s, bytes);
        fill(a, a + kABytes, full0 + 8 * s);
        ++n;
        if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
      };
      for (Tile t = first_tile<PAIR>(p, rank); ok && t.left > 0; next_tile<PAIR>(p, t, rank)) {
        if constexpr (EPI == EPI_GATED_BWD) {
          const int half = PAIR ? p.cols / 2 : p.cols, n2 = t.n0 + (PAIR ? (int)rank * half : 0);
          for (int kb = 0; ok && kb < p.kb2; ++kb)
            stage(p.tx_bytes2, [&](uint32_t a, uint32_t b, uint32_t bar) {
              load(a, &p.ma2, bar, 64 * kb, t.m0);
              for (int i = 0; i < half; i += 64) load(b + 128 * i, &p.mb2, bar, n2 + i, 64 * kb);
            });
        }
        const int n0 = t.n0 + (PAIR ? (int)rank * b_cols : 0);
        for (int kb = t.kb0; ok && kb < t.kb1; ++kb)
          stage(p.tx_bytes, [&](uint32_t a, uint32_t b, uint32_t bar) {
            const int k0 = kb * (EPI == EPI_INT8 ? 128 : 64);
            if (p.a_mn) {
              load(a, &p.ma, bar, t.m0, k0);
              load(a + tc::kMnGroupBytes, &p.ma, bar, t.m0 + 64, k0);
            } else {
              load(a, &p.ma, bar, k0, t.m0);
            }
            if (EPI == EPI_GATED || EPI == EPI_GATED_BWD) {  // value rows, then gate rows: one half of B each
              if (!PAIR || rank == 0) load(b, &p.mb, bar, k0, t.n0);
              if (!PAIR || rank == 1) load(b + (PAIR ? 0 : p.cols * 128), &p.mb, bar, k0, p.gate_row + t.n0);
            } else if (p.b_mn) {
              for (int i = 0; i < b_cols; i += 64) load(b + 128 * i, &p.mb, bar, n0 + i, k0);
            } else {
              load(b, &p.mb, bar, k0, n0);
            }
          });
      }
      // The copies in flight must land before the CTA ends.  Every product
      // waits for its copies, so this matters after a wait that gave up only.
      // The second CTA's count on the first one's barriers, where the first
      // waits for those of the stages it has filled too; of one that the
      // second was ahead with nobody knows, so it stays for far longer than a
      // copy takes.
      if (!ok && rank == 0) {
        volatile uint32_t ignore = 0;
        const uint32_t from = n > (uint32_t)p.stages ? n - p.stages : 0;
        for (uint32_t i = from; i < n; ++i) tc::mbar_wait(full + 8 * (i % p.stages), (i / p.stages) & 1, &ignore);
      } else if (!ok) {
        for (int i = 0; i < 20; ++i) __nanosleep(1000000);  // at most a millisecond each
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && tc::elect_one()) {
      uint32_t s = 0, phase = 0, it = 0;
      bool ok = true;
      // one k step of products into the accumulator at d
      auto step = [&](uint32_t d, bool a_mn, bool b_mn, uint32_t idesc, bool fresh) {
        ok = tc::mbar_wait(full + 8 * s, phase, abort);
        if (!ok) return;
        tc::fence_after();
        const uint32_t a = base + s * p.stage_bytes;
        const uint32_t a_step = a_mn ? 2048 >> 4 : 32 >> 4, b_step = b_mn ? 2048 >> 4 : 32 >> 4;
        const uint64_t da = tc::operand_desc(a, a_mn), db = tc::operand_desc(a + kABytes, b_mn);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          tc::mma<PAIR, EPI == EPI_INT8>(d, da + i * a_step, db + i * b_step, idesc, !fresh || i > 0);
        tc::mma_commit<PAIR>(empty + 8 * s);
        if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
      };
      for (Tile t = first_tile<PAIR>(p, rank); ok && t.left > 0; next_tile<PAIR>(p, t, rank), ++it) {
        const uint32_t buf = it & 1;
        ok = tc::mbar_wait(acc_empty + 8 * buf, ((it >> 1) & 1) ^ 1, abort);
        if (!ok) break;
        tc::fence_after();
        uint32_t d = tmem + buf * kMaxN;
        if constexpr (EPI == EPI_GATED_BWD) {
          // dh in one of two buffers; value and gate, which need the rest of
          // TMEM, once the epilogue of the tile before is through
          for (int kb = 0; ok && kb < p.kb2; ++kb)
            step(tmem + kMaxN + buf * (kMaxN / 2), false, true, p.idesc2, kb == 0);
          if (ok && it > 0) {
            ok = tc::mbar_wait(acc_empty + 8 * (buf ^ 1), ((it - 1) >> 1) & 1, abort);
            tc::fence_after();
          }
          d = tmem;
        }
        for (int kb = t.kb0; ok && kb < t.kb1; ++kb) step(d, p.a_mn, p.b_mn, p.idesc, kb == t.kb0);
        if (!ok) break;
        tc::mma_commit<PAIR>(acc_full + 8 * buf);
      }
    }
  } else {
    constexpr int kSets = C::epi_warps / 4;  // warps of a quarter
    const int quarter = warp & 3, set = (warp - 2) >> 2;
    EpilogueWarp<EPI, T, ACT, DROP> epi(p, staging + (warp - 2) * C::blocks * kRowsBytes,
                                        vectors + (warp - 2) * C::vectors * kVectorBytes);
    const uint32_t empty0 = PAIR ? tc::peer_addr(acc_empty, 0) : acc_empty;
    // gated: the padding columns of h, u and du are written too (zeros)
    const int n_end = EPI == EPI_GATED || EPI == EPI_GATED_BWD ? p.hp : p.N;
    uint32_t it = 0;
    for (Tile t = first_tile<PAIR>(p, rank); t.left > 0; next_tile<PAIR>(p, t, rank), ++it) {
      const uint32_t buf = it & 1;
      const int m = t.m0 + 32 * quarter;
      const int c_end = m < p.M ? min(p.cols, n_end - t.n0) : 0;
      const uint32_t lanes = tmem + ((uint32_t)(32 * quarter) << 16);
      const uint32_t acc = lanes + (EPI == EPI_GATED_BWD ? 0 : buf * kMaxN), acc2 = lanes + kMaxN + buf * (kMaxN / 2);
      int c = 32 * set;
      if (EPI == EPI_INT8) {
        const int row = m + (int)(threadIdx.x & 31);
        epi.row_scale = row < p.M && GFB_IN_BOUNDS(within(row, p.M)) ? p.a_scale[row] : 0.0f;
        epi.far_scale = __any_sync(0xFFFFFFFFu, fabsf(epi.row_scale) >= 79228162514264337593543950336.0f);  // 2^96
      }
      typename decltype(epi)::Ahead ahead;
      if (c < c_end) epi.fetch(ahead, t.n0 + c);
      if (!__all_sync(0xFFFFFFFFu, tc::mbar_wait(acc_full + 8 * buf, (it >> 1) & 1, abort))) break;
      tc::fence_after();
      auto release = [&](bool last) {
        if (!last) return;
        tc::fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) {
          if constexpr (PAIR) tc::mbar_arrive_cluster(empty0 + 8 * buf);
          else tc::mbar_arrive(empty0 + 8 * buf);
        }
      };
      if (c >= c_end) release(true);  // no chunk of this tile is this warp's
      for (; c < c_end; c += 32 * kSets) {
        const int next = c + 32 * kSets;
        epi.chunk(acc + c, acc2 + c, t, m, t.n0 + c, ahead, [&] { release(next >= c_end); },
                  [&] { if (next < c_end) epi.fetch(ahead, t.n0 + next); });
      }
    }
    epi.finish();
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort) atomicOr(&g_status, GF_FLAG_TIMEOUT);
  if (warp == 1) {
    tc::fence_after();
    if (*abort && rank == 0) {
      // Products may still be running: their end is a commit away, by the lane
      // that issued them and, as every tcgen05 instruction of a kernel, with its
      // cta_group (a pair's commit arrives on both CTAs' barriers).
      if (tc::elect_one()) {
        volatile uint32_t ignore = 0;
        const uint32_t spare = tc::smem_addr(&pipe->spare);
        tc::mma_commit<PAIR>(spare);
        tc::mbar_wait(spare, 0, &ignore);
      }
      __syncwarp();
    }
  }
  if constexpr (PAIR) tc::cluster_sync();  // the peer still signals here, and reads this CTA's operands
  if (warp == 1) tc::tmem_free<PAIR>(tmem, kTmemCols);
}

// ---------------------------------------------------------------------------
// K ranges joined: out = sum of the partial products (in order) + bias

template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ GemmParams p) {
  tc::dependency_wait();
  tc::let_dependents();
  const int64_t groups = p.ld_partial / 4, total = (int64_t)p.M * groups;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t m = i / groups;
    const int n = (int)(i - m * groups) * 4;
    if (n >= p.N) continue;
    int64_t row = m;
    if (p.seg_pad) {
      const int64_t in = m >= p.seg_pad ? m - p.seg_pad : m;
      if (in >= p.seg) continue;
      row = m >= p.seg_pad ? p.seg + in : in;
    }
    float4 s = make_float4(0, 0, 0, 0);
    for (int k = 0; k < p.splits; ++k) {
      if (!GFB_IN_BOUNDS(within(m, p.rows_m) && within(n, p.ld_partial, 4))) continue;
      const float4 v = *reinterpret_cast<const float4*>(p.partial + ((int64_t)k * p.rows_m + m) * p.ld_partial + n);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    if (!GFB_IN_BOUNDS(within(row, p.seg_pad ? 2 * (int64_t)p.seg : p.M) && within(n, p.N))) continue;
    const float f[4] = {s.x, s.y, s.z, s.w};
    T* out = static_cast<T*>(p.out) + row * p.ld_out + n;
    const T* bias = static_cast<const T*>(p.bias);
    __align__(8) T r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = from_float<T>(f[j] + (bias && n + j < p.N ? to_float(bias[n + j]) : 0.0f));
    if (p.N % 8 == 0 && p.ld_out % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0) {
      *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(r);
    } else {
      for (int j = 0; j < 4 && n + j < p.N; ++j) out[j] = r[j];
    }
  }
}

// ---------------------------------------------------------------------------
// column sums (bias gradients): rows cut into runs, each summed in order, the
// runs then added in order.  One launch does up to two matrices (blockIdx.z).

struct SumJob {
  const void* src;
  int64_t ld;
  int32_t rows, cols, run, parts;
  int32_t seg_pad, seg;  // results: `seg` columns from 0 and from seg_pad (0: all columns)
  float* partial;        // [parts][cols]
  void* out;
};
struct SumJobs {
  SumJob job[2];
};

template <typename T>
__global__ void __launch_bounds__(256) column_sums_kernel(const __grid_constant__ SumJobs jobs) {
  tc::dependency_wait();
  tc::let_dependents();
  const SumJob& j = jobs.job[blockIdx.z];
  const int c = blockIdx.x * 32 + threadIdx.x % 32, w = threadIdx.x / 32;
  if ((int)blockIdx.x * 32 >= j.cols || (int)blockIdx.y >= j.parts) return;
  const T* src = static_cast<const T*>(j.src);
  const int64_t r0 = (int64_t)blockIdx.y * j.run, r1 = min((int64_t)j.rows, r0 + j.run);
  float s = 0.0f;
  if (c < j.cols)
    for (int64_t r = r0 + w; r < r1; r += 8)
      if (GFB_IN_BOUNDS(within(r, j.rows) && within(c, j.cols))) s += to_float(src[r * j.ld + c]);
  __shared__ float sums[8][32];
  sums[w][threadIdx.x % 32] = s;
  __syncthreads();
  if (w == 0 && c < j.cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sums[i][threadIdx.x];
    if (GFB_IN_BOUNDS(within(blockIdx.y, j.parts) && within(c, j.cols))) j.partial[(int64_t)blockIdx.y * j.cols + c] = s;
  }
}
template <typename T>
__global__ void __launch_bounds__(256) column_join_kernel(const __grid_constant__ SumJobs jobs) {
  tc::dependency_wait();
  tc::let_dependents();
  const SumJob& j = jobs.job[blockIdx.z];
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (j.seg_pad ? 2 * j.seg : j.cols)) return;
  const int c = j.seg_pad && i >= j.seg ? j.seg_pad + i - j.seg : i;
  float s = 0.0f;
  if (!GFB_IN_BOUNDS(within(c, j.cols))) return;
  for (int k = 0; k < j.parts; ++k) s += j.partial[(int64_t)k * j.cols + c];
  static_cast<T*>(j.out)[i] = from_float<T>(s);
}

// ---------------------------------------------------------------------------
// copies into 16-byte aligned rows, up to four in one launch (blockIdx.y): dst
// row r holds src row r (or, with two runs of rows, src rows 0 .. seg - 1 and
// seg .. 2 seg - 1 at 0 and seg_pad); everything else is zero

struct AlignJob {
  const void* src;
  void* dst;
  int64_t ld, src_rows, dst_rows;
  int32_t cols, ld_dst, seg_pad, seg;
};
struct AlignJobs {
  AlignJob job[4];
  int n;
};

template <typename E>
__global__ void __launch_bounds__(256) align_kernel(const __grid_constant__ AlignJobs jobs) {
  tc::dependency_wait();
  tc::let_dependents();
  const AlignJob& j = jobs.job[blockIdx.y];
  // a warp copies whole rows
  const int lane = threadIdx.x & 31;
  for (int64_t r = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; r < j.dst_rows; r += (int64_t)gridDim.x * 8) {
    int64_t from = r;
    if (j.seg_pad) {
      const int64_t in = r >= j.seg_pad ? r - j.seg_pad : r;
      from = in < j.seg ? (r >= j.seg_pad ? j.seg + in : in) : j.src_rows;
    }
    const E* src = static_cast<const E*>(j.src) + from * j.ld;
    E* dst = static_cast<E*>(j.dst) + r * j.ld_dst;
    const int cols = from < j.src_rows ? j.cols : 0;
    if (!GFB_IN_BOUNDS(within(r, j.dst_rows) && (cols == 0 || (within(from, j.src_rows) && cols <= j.ld)))) continue;
    for (int c = lane; c < j.ld_dst; c += 32) dst[c] = c < cols ? src[c] : E(0);
  }
}

// ---------------------------------------------------------------------------
// The block for a few tokens, where it is a walk over the weights: a warp
// takes a column of h (both its rows of w_in) or of y, four warps sharing a
// long row; each lane holds 16 bytes of the row at a time against the tokens'
// same columns in shared memory.  Rows are 16-byte aligned.
//
// Up to four tokens: every further one adds its arithmetic on all weights,
// while the product kernel takes the same time for one token as for eight.
// Whole forward from cold caches, us, walk / product kernel:
//   tokens            1             4             5             8
//   320 x 1280    6.1 / 12.3    9.0 / 12.7   11.6 / 12.7   13.3 / 12.6
//   640 x 2560    8.2 / 15.2   12.6 / 15.7   16.7 / 15.5   19.3 / 15.5
//   1280 x 5120  13.1 / 24.3   23.6 / 23.4   36.9 / 23.6   42.1 / 23.1

constexpr int kSkinnyTokens = 4;
constexpr int kSkinnyWarps = 8;

struct SkinnyParams {
  const void *x, *w, *bias;  // x [tokens, k], w [n or two runs of n, k]
  int64_t ld_x, ld_w, gate_row;
  int32_t tokens, n, k, hp;
  void* out;
  int64_t ld_out;
  int32_t act;
  DropArgs drop;
};

template <typename T, int TOKENS, bool GATED>
__global__ void __launch_bounds__(32 * kSkinnyWarps) skinny_kernel(const __grid_constant__ SkinnyParams p) {
  constexpr int kRows = GATED ? 2 : 1;
  constexpr int kShare = GATED ? 1 : 4;             // warps of a column
  constexpr int kChunk = 2048;                      // columns of x in shared memory at a time
  __shared__ __align__(16) T xs[TOKENS][kChunk];
  __shared__ float part[kSkinnyWarps][TOKENS];
  tc::dependency_wait();
  tc::let_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = blockIdx.x * (kSkinnyWarps / kShare) + warp / kShare;
  const bool live = n < p.n;
  float sum[kRows][TOKENS] = {};
  for (int k0 = 0; k0 < p.k; k0 += kChunk) {
    const int len = min(kChunk, p.k - k0);
    __syncthreads();
    for (int i = threadIdx.x; i < TOKENS * (kChunk / 8); i += 32 * kSkinnyWarps) {
      const int m = i / (kChunk / 8), c = i % (kChunk / 8) * 8;
      if (c >= len) continue;
      uint4 v = make_uint4(0, 0, 0, 0);
      const T* src = static_cast<const T*>(p.x) + m * p.ld_x + k0 + c;
      if (m < p.tokens && c + 8 <= len && GFB_IN_BOUNDS(within(m, p.tokens) && within(k0 + c, p.k, 8)))
        v = *reinterpret_cast<const uint4*>(src);
      *reinterpret_cast<uint4*>(&xs[m][c]) = v;
      if (m < p.tokens && c + 8 > len)
        for (int j = 0; c + j < len; ++j)
          if (GFB_IN_BOUNDS(within(k0 + c + j, p.k))) xs[m][c + j] = src[j];
    }
    __syncthreads();
    if (!live) continue;
    if (!GFB_IN_BOUNDS(within(n, p.n) && (kRows == 1 || p.gate_row == p.n))) continue;
    const T* w = static_cast<const T*>(p.w) + n * p.ld_w + k0;
    auto add = [&](const uint4 (&v)[kRows], int c) {
#pragma unroll
      for (int m = 0; m < TOKENS; ++m) {
        const uint4 xv = *reinterpret_cast<const uint4*>(&xs[m][c]);
        const uint32_t* xw = reinterpret_cast<const uint32_t*>(&xv);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const uint32_t* ww = reinterpret_cast<const uint32_t*>(&v[r]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 a = unpack2<T>(xw[j]), b = unpack2<T>(ww[j]);
            sum[r][m] = fmaf(a.x, b.x, fmaf(a.y, b.y, sum[r][m]));
          }
        }
      }
    };
    constexpr int kStep = 256 * kShare, kAhead = GATED ? 4 : 2;  // loads in flight
    static_assert(kAhead * kStep <= kChunk, "the pipelined loop has to fit the chunk, or no lane enters it");
    const int whole = len & ~7;
    int c = 8 * (lane + 32 * (warp % kShare));
    for (; c + (kAhead - 1) * kStep < whole; c += kAhead * kStep) {
      uint4 v[kAhead][kRows];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          v[i][r] = GFB_IN_BOUNDS(within(k0 + c + i * kStep, p.k, 8))
                        ? *reinterpret_cast<const uint4*>(w + r * p.gate_row * p.ld_w + c + i * kStep)
                        : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) add(v[i], c + i * kStep);
    }
    for (; c < len; c += kStep) {
      uint4 v[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const T* at = w + r * p.gate_row * p.ld_w + c;
        if (c < whole) {
          v[r] = GFB_IN_BOUNDS(within(k0 + c, p.k, 8)) ? *reinterpret_cast<const uint4*>(at) : make_uint4(0, 0, 0, 0);
        } else {  // the row's last few: what follows is not its own
          __align__(16) T tail[8];
          for (int j = 0; j < 8; ++j) tail[j] = c + j < len && GFB_IN_BOUNDS(within(k0 + c + j, p.k)) ? at[j] : T(0.0f);
          v[r] = *reinterpret_cast<const uint4*>(tail);
        }
      }
      add(v, c);
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r)
#pragma unroll
    for (int m = 0; m < TOKENS; ++m)
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum[r][m] += __shfl_xor_sync(0xFFFFFFFFu, sum[r][m], d);
  const T* bias = static_cast<const T*>(p.bias);
  if constexpr (GATED) {
    // lane m finishes token m; the padding columns of h are zeros
    float a = 0.0f, g = 0.0f;
#pragma unroll
    for (int m = 0; m < TOKENS; ++m)
      if (lane == m) a = sum[0][m], g = sum[1][m];
    if (live && lane < p.tokens) {
      if (bias) a += to_float(bias[n]), g += to_float(bias[p.n + n]);
      uint64_t value, slope;
      if (p.act == GF_ACT_GELU) activate<GF_ACT_GELU, false>(g, g, value, slope);
      else activate<GF_ACT_SILU, false>(g, g, value, slope);
      float h = a * tc::unpack_f2(value).x;
      if (p.drop.on) {
        const uint4 w = Philox(p.drop)((uint32_t)n >> 2, (uint32_t)lane);
        const uint32_t word = (n & 3) == 0 ? w.x : (n & 3) == 1 ? w.y : (n & 3) == 2 ? w.z : w.w;
        h = word >= p.drop.threshold ? h * p.drop.scale : 0.0f;
      }
      if (GFB_IN_BOUNDS(within(n, p.ld_out))) static_cast<T*>(p.out)[lane * p.ld_out + n] = from_float<T>(h);
    } else if (!live && n < p.hp && lane < p.tokens) {
      if (GFB_IN_BOUNDS(within(n, p.ld_out))) static_cast<T*>(p.out)[lane * p.ld_out + n] = T(0.0f);
    }
  } else {
    float y = 0.0f;
#pragma unroll
    for (int m = 0; m < TOKENS; ++m)
      if (lane == m) y = sum[0][m];
    if (lane < TOKENS) part[warp][lane] = y;
    __syncthreads();
    if (live && warp % kShare == 0 && lane < p.tokens) {
      y = bias ? to_float(bias[n]) : 0.0f;
#pragma unroll
      for (int i = 0; i < kShare; ++i) y += part[warp + i][lane];
      if (GFB_IN_BOUNDS(within(n, p.n))) static_cast<T*>(p.out)[lane * p.ld_out + n] = from_float<T>(y);
    }
  }
}

// ---------------------------------------------------------------------------
// dropout

struct DropoutParams {
  int64_t rows, groups;  // groups of V columns in a row
  int64_t cols;
  const void* x;
  int64_t x_rs, x_cs;
  const void* res;
  int64_t r_rs, r_cs;
  void* y;
  DropArgs drop;
};

// One thread takes V columns of a row at a time: 16 bytes of aligned rows, or
// (VEC false) four elements through any strides; two such groups per turn, so
// that the loads of both are on their way while the generator works.  ROWS:
// neighbouring threads take neighbouring rows, for inputs whose rows are the
// contiguous dimension.  I: the type that holds rows * groups.
template <typename T, bool VEC, bool ROWS, bool RES, typename I>
__global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutParams p) {
  constexpr int V = VEC ? 16 / sizeof(T) : 4, U = 2;
  tc::dependency_wait();
  tc::let_dependents();
  const Philox rng(p.drop);
  const I inner = (I)(ROWS ? p.rows : p.groups), outer = (I)(ROWS ? p.groups : p.rows);
  const I step = (I)gridDim.x * blockDim.x;
  const I step_o = step / inner, step_i = step - step_o * inner;
  I i = (I)blockIdx.x * blockDim.x + threadIdx.x;
  I o = i / inner;
  i -= o * inner;
  while (o < outer) {
    __align__(16) T in[U][V];
    __align__(16) T add[U][V];
    int64_t rows[U], cols[U];
    bool live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      live[u] = o < outer;
      const int64_t row = rows[u] = ROWS ? i : o, col = cols[u] = (int64_t)(ROWS ? o : i) * V;
      if (live[u] && GFB_IN_BOUNDS(within(row, p.rows) && within(col, p.cols, VEC ? V : 1))) {
        const T* x = static_cast<const T*>(p.x) + row * p.x_rs + col * p.x_cs;
        const T* res = static_cast<const T*>(p.res) + row * p.r_rs + col * p.r_cs;
        if constexpr (VEC) {
          *reinterpret_cast<uint4*>(in[u]) = *reinterpret_cast<const uint4*>(x);
          if constexpr (RES) *reinterpret_cast<uint4*>(add[u]) = *reinterpret_cast<const uint4*>(res);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (col + j < p.cols) {
              in[u][j] = x[j * p.x_cs];
              if constexpr (RES) add[u][j] = res[j * p.r_cs];
            }
        }
      }
      o += step_o;
      i += step_i;
      if (i >= inner) i -= inner, ++o;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!live[u]) continue;
      __align__(16) T out[V];
#pragma unroll
      for (int b = 0; b < V / 4; ++b) {
        const uint4 w = rng((uint32_t)(cols[u] / 4 + b), (uint64_t)rows[u]);
        const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v = word[j] >= p.drop.threshold ? to_float(in[u][4 * b + j]) * p.drop.scale : 0.0f;
          if constexpr (RES) v += to_float(add[u][4 * b + j]);
          out[4 * b + j] = from_float<T>(v);
        }
      }
      if (!GFB_IN_BOUNDS(within(rows[u], p.rows) && within(cols[u], p.cols, VEC ? V : 1))) continue;
      T* y = static_cast<T*>(p.y) + rows[u] * p.cols + cols[u];
      if constexpr (VEC) {
        *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(out);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (cols[u] + j < p.cols) y[j] = out[j];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// row quantisation: TPR threads per row.  VPL > 0: rows of 16-byte aligned
// pieces, VPL pieces of 8 values per thread held in registers between the
// maximum and the rounding; VPL = 0: any row, read twice (the second time from
// L1 or L2).
//
// Rounding to even by one fp32 addition: 1.5 * 2^23 + v has v's nearest whole
// number, as two's complement, in its low bits for |v| < 2^22.

constexpr float kTinyRow = 7.8886090522101181e-31f;  // 2^-100: below it 127 / max could overflow

__device__ __forceinline__ uint32_t round_to_int(float v, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.0f));
}

template <typename T, int TPR, int VPL>
__global__ void __launch_bounds__(256) quantize_rows_kernel(int64_t rows, int cols, const T* x, int64_t ld, int8_t* q,
                                                            int64_t ld_q, float* scale) {
  const int t = threadIdx.x % TPR;
  constexpr int64_t per_block = 256 / TPR;
  constexpr int kHeld = VPL > 0 ? VPL : 1;
  __shared__ uint32_t warp_max[8];
  tc::dependency_wait();
  tc::let_dependents();
  for (int64_t base = blockIdx.x * per_block; base < rows; base += gridDim.x * per_block) {
    const int64_t r = base + threadIdx.x / TPR;
    const bool live = r < rows;
    const T* row = x + r * ld;
    __align__(16) T held[kHeld][8];
    // magnitudes compare like their bits, with infinity and NaN above every finite value
    uint32_t top = 0;
    auto see = [&](float v) { top = max(top, __float_as_uint(v) & 0x7FFFFFFFu); };
    if (live) {
      if constexpr (VPL > 0) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
          const int c = 8 * (t + i * TPR);
#pragma unroll
          for (int k = 0; k < (int)sizeof(T) / 2; ++k)
            reinterpret_cast<uint4*>(held[i])[k] = c < cols && GFB_IN_BOUNDS(within(r, rows) && within(c, cols, 8))
                                                       ? reinterpret_cast<const uint4*>(row + c)[k]
                                                       : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) see(to_float(held[i][j]));
      } else {
        for (int c = t; c < cols; c += TPR)
          if (GFB_IN_BOUNDS(within(r, rows) && within(c, cols))) see(to_float(row[c]));
      }
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if constexpr (TPR > 32) {
      if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x / 32] = top;
      __syncthreads();
      top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, warp_max[i]);
      __syncthreads();
    }
    if (!live || !GFB_IN_BOUNDS(within(r, rows))) continue;
    const float most = __uint_as_float(top);
    float s = __fdiv_rn(most, 127.0f), inv = __fdiv_rn(127.0f, most);
    uint32_t mask = 0xFFFFFFFFu;
    if (most < kTinyRow) s = 0.0f, mask = 0;
    if (top >= 0x7F800000u) s = __uint_as_float(0x7FFFFFFFu), mask = 0;
    if (t == 0) scale[r] = s;
    int8_t* out = q + r * ld_q;
    if constexpr (VPL > 0) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int c = 8 * (t + i * TPR);
        uint32_t b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = round_to_int(to_float(held[i][j]), inv);
        auto join = [](uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
          return __byte_perm(__byte_perm(b0, b1, 0x0040), __byte_perm(b2, b3, 0x0040), 0x5410);
        };
        if (c < cols && GFB_IN_BOUNDS(within(c, ld_q, 8)))
          *reinterpret_cast<uint2*>(out + c) = make_uint2(join(b[0], b[1], b[2], b[3]) & mask, join(b[4], b[5], b[6], b[7]) & mask);
      }
      for (int64_t c = cols + t; c < ld_q; c += TPR) out[c] = 0;
    } else {
      for (int64_t c = t; c < ld_q; c += TPR)
        out[c] = c < cols ? (int8_t)(round_to_int(to_float(row[c]), inv) & mask) : (int8_t)0;
    }
  }
}

// ---------------------------------------------------------------------------
// host side

#define GFB_CUDA(call)                                                                            \
  do {                                                                                            \
    const cudaError_t e_ = (call);                                                                \
    if (e_ != cudaSuccess) return gf::fail(GF_ERR_CUDA, "%s: %s", #call, cudaGetErrorString(e_));     \
  } while (0)

// Launches with the dependent-launch attribute (see tc::dependency_wait).
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, int threads, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, P(args)...);
  return cudaGetLastError();
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

gf_status encode_fn(EncodeFn* out) {
  static std::atomic<void*> fn{nullptr};
  void* f = fn.load();
  if (!f) {
    cudaDriverEntryPointQueryResult found;
    GFB_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !f) return fail(GF_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    fn.store(f);
  }
  *out = reinterpret_cast<EncodeFn>(f);
  return GF_OK;
}

// A row-major operand: `rows` rows of `cols` elements, 16-byte aligned rows.
struct Operand {
  const void* ptr;
  int64_t rows, cols, ld;
};

inline bool aligned_rows(const void* ptr, int64_t rows, int64_t ld, int es) {
  return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0 && (rows == 1 || (ld * es) % 16 == 0);
}

gf_status make_map(CUtensorMap* map, const Operand& o, CUtensorMapDataType type, int es, int box_cols, int box_rows,
                   CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  EncodeFn encode;
  if (const gf_status s = encode_fn(&encode); s != GF_OK) return s;
  const int64_t ld = o.rows == 1 ? round_up<int64_t>(o.cols * es, 16) : o.ld * es;
  const cuuint64_t dims[2] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows}, strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, unit[2] = {1, 1};
  auto run = [&] {
    return encode(map, type, 2, const_cast<void*>(o.ptr), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = run();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {  // a thread that has made no runtime call yet (autograd's): give it the context
    int dev = 0;
    GFB_CUDA(cudaGetDevice(&dev));
    GFB_CUDA(cudaSetDevice(dev));
    r = run();
  }
  if (r != CUDA_SUCCESS)
    return fail(GF_ERR_CUDA, "cuTensorMapEncodeTiled(%lld x %lld, ld %lld): error %d", (long long)o.rows, (long long)o.cols,
                (long long)o.ld, (int)r);
  return GF_OK;
}

// Where the epilogue writes 64 bytes of 32 rows at a time.
gf_status make_out_map(CUtensorMap* map, const Operand& o, CUtensorMapDataType type, int es) {
  return make_map(map, o, type, es, 64 / es, 32, CU_TENSOR_MAP_SWIZZLE_64B);
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
      n <= 0) {
    cudaGetLastError();
    return 148;  // workspace queries work without a device
  }
  return n;
}

// Pairs or single CTAs, tile width, K ranges: whichever gives the least
// estimated time.  A tile takes the longest of its products (2 clocks a
// column and 64 k), its operands' way into the SM (70 bytes a clock) and its
// result's way to memory (about 11 bytes a clock for each SM when all write);
// the grid's time is that of the CTA with most tiles, the fill of its pipeline
// and one epilogue; K ranges add the partial products' way to memory and back.
struct Shape {
  bool pair;
  int bn, splits, kb_split, tiles_m, tiles_n;
  int rows_m() const { return tiles_m * kTileM * (pair ? 2 : 1); }
};
Shape search_shape(int64_t M, int64_t N, int64_t kb, int64_t kb2, int epi, bool may_split, int sms) {
  Shape best{};
  double best_cost = 0;
  const bool gated = epi == EPI_GATED || epi == EPI_GATED_BWD;
  // bytes a result element takes, over 11 bytes a clock, for 128 rows
  const double per_col = epi == EPI_GATED_BWD ? 48.0 : 24.0;
  for (int pair = 0; pair < 2; ++pair) {
    const int64_t tm = ceil_div(M, pair ? 2 * kTileM : kTileM), units = pair ? sms / 2 : sms;
    const int step = gated ? 64 : 32;
    for (int bn = step; bn <= kMaxN; bn += step) {
      const int cols = gated ? bn / 2 : bn;
      if (cols > 32 && cols - 32 >= N) break;  // wider than the result
      const int64_t tn = ceil_div(N, cols);
      const auto k_step = [&](int n) {  // clocks of 64 k: operands or products of n columns
        const double loads = (kTileM + (pair ? n / 2 : n)) * 128 / 70.0, products = 2.0 * n;
        return loads > products ? loads : products;
      };
      for (int64_t s = 1; s <= (may_split ? kb : 1) && s <= 64; s = s < 4 ? s + 1 : s + s / 4) {
        const int64_t per = ceil_div(kb, s);
        if (ceil_div(kb, per) != s) continue;
        const double waves = (double)ceil_div(tm * tn * s, units), epilogue = per_col * cols, main = per * k_step(bn);
        // the backward's dh overlaps the epilogue before it, value and gate do not
        const double under = epi == EPI_GATED_BWD ? kb2 * k_step(cols) : main;
        const double tile = (under > epilogue ? under : epilogue) + (epi == EPI_GATED_BWD ? main : 0.0);
        double cost = waves * (tile + 600.0) + 1500.0 + epilogue;
        if (s > 1) cost += 4000.0 + (double)(s + 1) * M * N * 4 / 3000.0;
        if (best.bn == 0 || cost < best_cost) {
          best_cost = cost;
          best = Shape{pair != 0, bn, (int)s, (int)per, (int)tm, (int)tn};
        }
      }
    }
  }
  return best;
}

// The search takes some microseconds: a thread remembers the last shapes it asked for.
Shape choose_shape(int64_t M, int64_t N, int64_t kb, int epi, bool may_split, int sms, int64_t kb2 = 0) {
  struct Entry {
    int64_t M, N, kb, kb2;
    int epi, may_split, sms;
    Shape shape;
  };
  thread_local Entry seen[64];  // zero: no size is
  const uint64_t hash = (uint64_t)M * 0x9E3779B97F4A7C15u ^ (uint64_t)N * 0xC2B2AE3D27D4EB4Fu ^ (uint64_t)kb * 0x165667B19E3779F9u ^
                        (uint64_t)(8 * kb2 + 2 * epi + may_split) * 0xD6E8FEB86659FD93u;
  Entry& e = seen[hash >> 58];
  if (e.M != M || e.N != N || e.kb != kb || e.kb2 != kb2 || e.epi != epi || e.may_split != may_split || e.sms != sms)
    e = Entry{M, N, kb, kb2, epi, may_split, sms, search_shape(M, N, kb, kb2, epi, may_split, sms)};
  return e.shape;
}

inline size_t partial_bytes(const Shape& s, int64_t N) {
  return s.splits > 1 ? (size_t)s.splits * s.rows_m() * round_up<int64_t>(N, 32) * 4 : 0;
}

template <int EPI, typename T, int ACT, bool DROP, bool PAIR>
gf_status launch_gemm(GemmParams p, int sms, cudaStream_t st) {
  using C = Config<EPI>;
  constexpr int smem_bytes = C::stage_room + C::side_bytes;
  static_assert(smem_bytes <= kSmemLimit && C::stage_room >= 3 * 49152, "shared memory of one SM");
  const auto kernel = gemm_kernel<EPI, T, ACT, DROP, PAIR>;
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is set
  int dev = 0;
  GFB_CUDA(cudaGetDevice(&dev));
  if (dev > 63 || !(ready.load() >> dev & 1)) {
    GFB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes));
    if (dev <= 63) ready.fetch_or(uint64_t(1) << dev);
  }
  p.stage_bytes = kABytes + 128 * round_up(PAIR ? p.bn / 2 : p.bn, 64);
  p.stages = C::stage_room / p.stage_bytes < kMaxStages ? C::stage_room / p.stage_bytes : kMaxStages;
  const int64_t items = (int64_t)p.tiles_m * p.tiles_n * p.splits, units = PAIR ? sms / 2 : sms;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(items < units ? items : units) * (PAIR ? 2 : 1));
  cfg.blockDim = dim3(C::threads);
  cfg.dynamicSmemBytes = smem_bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(GF_ERR_CUDA, "gemm_kernel: %s", cudaGetErrorString(e));
  }
  return GF_OK;
}
template <int EPI, typename T, int ACT, bool DROP>
gf_status launch_gemm(const GemmParams& p, const Shape& s, int sms, cudaStream_t st) {
  return s.pair ? launch_gemm<EPI, T, ACT, DROP, true>(p, sms, st) : launch_gemm<EPI, T, ACT, DROP, false>(p, sms, st);
}

inline int grid_for(int64_t work, int threads, int sms) {
  const int64_t b = ceil_div(work, threads);
  return (int)(b < 8 * (int64_t)sms ? (b > 0 ? b : 1) : 8 * (int64_t)sms);
}

// Fills the operand part of a product: A (m, k), B (n, k) as stored.
gf_status set_operands(GemmParams& p, const Shape& s, const Operand& a, bool a_mn, const Operand& b, bool b_mn, int es,
                       CUtensorMapDataType type, uint32_t acc, uint32_t fmt, bool gated) {
  const int line = 128 / es;
  p.tiles_m = s.tiles_m;
  p.tiles_n = s.tiles_n;
  p.splits = s.splits;
  p.kb_split = s.kb_split;
  p.rows_m = s.rows_m();
  p.bn = s.bn;
  p.cols = gated ? s.bn / 2 : s.bn;
  p.a_mn = a_mn;
  p.b_mn = b_mn;
  p.idesc = tc::instruction_desc(acc, fmt, a_mn, b_mn, s.bn, s.pair);
  const int b_cols = s.pair ? s.bn / 2 : s.bn;  // of one CTA
  p.tx_bytes = (kABytes + 128 * (b_mn ? round_up(b_cols, 64) : b_cols)) * (s.pair ? 2 : 1);
  gf_status r = a_mn ? make_map(&p.ma, a, type, es, 64, 64) : make_map(&p.ma, a, type, es, line, kTileM);
  if (r != GF_OK) return r;
  return b_mn ? make_map(&p.mb, b, type, es, 64, 64) : make_map(&p.mb, b, type, es, line, gated ? p.cols : b_cols);
}

// ---- the feed-forward block

struct Bump {  // workspace layout: offsets first (null base), pointers when it exists
  char* base;
  size_t used = 0;
  void* take(size_t bytes) {
    char* p = base ? base + used : nullptr;
    used += round_up<size_t>(bytes, 256);
    return p;
  }
};

struct FfPlan {
  int64_t M, D, F, O, Hp;
  bool skinny, copy_x, copy_w_in, copy_w_out, copy_dy;
  Shape in, out, dh, dx, dw_in, dw_out;
  int in_parts, in_run, out_parts, out_run;  // column sums
  void *x, *w_in, *w_out, *dy, *du, *partial, *in_sums, *out_sums;
  size_t bytes;
};

void column_runs(int64_t rows, int64_t cols, int sms, int* parts, int* run) {
  // about four CTAs of 32 columns for each SM, runs of at least 64 rows
  int64_t want = 4 * (int64_t)sms / ceil_div(cols, 32);
  if (want < 1) want = 1;
  int64_t r = ceil_div(rows, want);
  if (r < 64) r = 64;
  *run = (int)r;
  *parts = (int)ceil_div(rows, r);
}

FfPlan plan_ff(const gf_gated_ff& f, gf_pass pass, char* ws) {
  FfPlan p{};
  const int sms = sm_count();
  p.M = f.tokens, p.D = f.in_features, p.F = f.hidden, p.O = f.out_features;
  p.Hp = round_up<int64_t>(p.F, 64);
  const bool back = pass == GF_PASS_BACKWARD;
  p.skinny = !back && p.M <= kSkinnyTokens && aligned_rows(f.x, p.M, f.ld_x, 2) &&
             aligned_rows(f.w_in, 2 * p.F, f.ld_w_in, 2) && aligned_rows(f.w_out, p.O, f.ld_w_out, 2);
  if (p.skinny) {
    p.bytes = 256;
    return p;
  }
  const bool use_du = back && (f.dx || f.dw_in || f.db_in);
  const bool use_x = !back || use_du, use_w_in = use_x;
  const bool use_w_out = !back || use_du, use_dy = back && (use_du || f.dw_out);
  p.copy_x = use_x && !aligned_rows(f.x, p.M, f.ld_x, 2);
  p.copy_w_in = use_w_in && (p.Hp != p.F || !aligned_rows(f.w_in, 2 * p.F, f.ld_w_in, 2));
  p.copy_w_out = use_w_out && !aligned_rows(f.w_out, p.O, f.ld_w_out, 2);
  p.copy_dy = use_dy && !aligned_rows(f.dy, p.M, f.ld_dy, 2);
  Bump b{ws};
  if (p.copy_x) p.x = b.take(2 * p.M * round_up<int64_t>(p.D, 8));
  if (p.copy_w_in) p.w_in = b.take(2 * 2 * p.Hp * round_up<int64_t>(p.D, 8));
  if (p.copy_w_out) p.w_out = b.take(2 * p.O * round_up<int64_t>(p.F, 8));
  if (p.copy_dy) p.dy = b.take(2 * p.M * round_up<int64_t>(p.O, 8));
  size_t partial = 0;
  auto need = [&](const Shape& s, int64_t N) {
    const size_t n = partial_bytes(s, N);
    if (n > partial) partial = n;
  };
  if (!back) {
    p.in = choose_shape(p.M, p.Hp, ceil_div(p.D, 64), EPI_GATED, false, sms);
    p.out = choose_shape(p.M, p.O, ceil_div(p.F, 64), EPI_STORE, true, sms);
    need(p.out, p.O);
  } else {
    if (use_du) {
      p.du = b.take(2 * p.M * 2 * p.Hp);
      p.dh = choose_shape(p.M, p.Hp, ceil_div(p.D, 64), EPI_GATED_BWD, false, sms, ceil_div(p.O, 64));
    }
    if (f.dx) {
      p.dx = choose_shape(p.M, p.D, 2 * p.Hp / 64, EPI_STORE, true, sms);
      need(p.dx, p.D);
    }
    if (f.dw_in) {
      p.dw_in = choose_shape(2 * p.Hp, p.D, ceil_div(p.M, 64), EPI_STORE, true, sms);
      need(p.dw_in, p.D);
    }
    if (f.dw_out) {
      p.dw_out = choose_shape(p.O, p.F, ceil_div(p.M, 64), EPI_STORE, true, sms);
      need(p.dw_out, p.F);
    }
    if (f.db_in) {
      column_runs(p.M, 2 * p.Hp, sms, &p.in_parts, &p.in_run);
      p.in_sums = b.take((size_t)4 * p.in_parts * 2 * p.Hp);
    }
    if (f.db_out) {
      column_runs(p.M, p.O, sms, &p.out_parts, &p.out_run);
      p.out_sums = b.take((size_t)4 * p.out_parts * p.O);
    }
  }
  if (partial) p.partial = b.take(partial);
  p.bytes = b.used > 256 ? b.used : 256;
  return p;
}

// every pointer a multiple of its element's size (the kernels access whole elements)
template <typename... P>
gf_status check_elements(const char* who, int es, const P*... ptrs) {
  const uintptr_t all = (reinterpret_cast<uintptr_t>(ptrs) | ...);
  if (all % es) return fail(GF_ERR_INVALID_ARG, "%s: a pointer is not aligned to its %d-byte elements", who, es);
  return GF_OK;
}

gf_status check_ff(const char* who, const gf_gated_ff* f) {
  if (!f) return fail(GF_ERR_INVALID_ARG, "%s: the description must be non-null", who);
  if (f->tokens < 0 || f->in_features <= 0 || f->hidden <= 0 || f->out_features <= 0)
    return fail(GF_ERR_INVALID_ARG, "%s: sizes must be positive (tokens may be 0)", who);
  if (f->tokens > kMaxDim || f->in_features > kMaxDim || f->hidden > kMaxDim / 2 || f->out_features > kMaxDim)
    return fail(GF_ERR_UNSUPPORTED, "%s: a size is above 2^31 - 512 (2 * hidden counts)", who);
  if (f->dtype != GF_BF16 && f->dtype != GF_F16)
    return fail(GF_ERR_UNSUPPORTED, "%s: dtype must be GF_BF16 or GF_F16", who);
  if (f->activation != GF_ACT_GELU && f->activation != GF_ACT_SILU)
    return fail(GF_ERR_INVALID_ARG, "%s: unknown activation", who);
  if (const gf_status s = check_elements(who, 2, f->x, f->w_in, f->b_in, f->w_out, f->b_out, f->y, f->dy, f->dx, f->dw_in,
                                         f->db_in, f->dw_out, f->db_out);
      s != GF_OK)
    return s;
  if (f->ld_x < f->in_features || f->ld_w_in < f->in_features || f->ld_w_out < f->hidden)
    return fail(GF_ERR_INVALID_ARG, "%s: a leading dimension is smaller than its row", who);
  return check_rule(who, f->dropout);
}

gf_status check_workspace(const char* who, const void* ws, size_t have, size_t want) {
  if (!ws || (reinterpret_cast<uintptr_t>(ws) & 255u))
    return fail(GF_ERR_INVALID_ARG, "%s: workspace must be non-null and 256-byte aligned", who);
  if (have < want) return fail(GF_ERR_INVALID_ARG, "%s: workspace too small: %zu bytes given, %zu needed", who, have, want);
  return GF_OK;
}

void add_align(AlignJobs& jobs, const void* src, int64_t ld, int64_t rows, int64_t cols, void* dst, int64_t ld_dst,
               int64_t dst_rows, int64_t seg_pad, int64_t seg) {
  jobs.job[jobs.n++] = AlignJob{src, dst, ld, rows, dst_rows, (int)cols, (int)ld_dst, (int)seg_pad, (int)seg};
}
template <typename E>
gf_status run_align(const AlignJobs& jobs, int sms, cudaStream_t st) {
  if (jobs.n == 0) return GF_OK;
  int64_t rows = 0;
  for (int i = 0; i < jobs.n; ++i) rows = jobs.job[i].dst_rows > rows ? jobs.job[i].dst_rows : rows;
  const cudaError_t e = launch(align_kernel<E>, dim3(grid_for(rows, 8, sms), jobs.n), 256, st, jobs);
  if (e != cudaSuccess) return fail(GF_ERR_CUDA, "align_kernel: %s", cudaGetErrorString(e));
  return GF_OK;
}

#define GFB_TRY(call)                                 \
  do {                                                \
    const gf_status s_ = (call);                      \
    if (s_ != GF_OK) return s_;                       \
  } while (0)

// The operands of the block as the products see them: rows aligned, the two
// halves of w_in Hp rows apart.
struct FfOperands {
  Operand x, w_in, w_out, dy;
};
gf_status align_ff(const gf_gated_ff& f, const FfPlan& p, FfOperands* o, int sms, cudaStream_t st) {
  o->x = Operand{f.x, p.M, p.D, f.ld_x};
  o->w_in = Operand{f.w_in, 2 * p.Hp, p.D, f.ld_w_in};
  o->w_out = Operand{f.w_out, p.O, p.F, f.ld_w_out};
  o->dy = Operand{f.dy, p.M, p.O, f.ld_dy};
  const int64_t ld_d = round_up<int64_t>(p.D, 8), ld_f = round_up<int64_t>(p.F, 8), ld_o = round_up<int64_t>(p.O, 8);
  AlignJobs jobs{};
  if (p.copy_x) {
    add_align(jobs, f.x, f.ld_x, p.M, p.D, p.x, ld_d, p.M, 0, 0);
    o->x = Operand{p.x, p.M, p.D, ld_d};
  }
  if (p.copy_w_in) {
    add_align(jobs, f.w_in, f.ld_w_in, 2 * p.F, p.D, p.w_in, ld_d, 2 * p.Hp, p.Hp, p.F);
    o->w_in = Operand{p.w_in, 2 * p.Hp, p.D, ld_d};
  }
  if (p.copy_w_out) {
    add_align(jobs, f.w_out, f.ld_w_out, p.O, p.F, p.w_out, ld_f, p.O, 0, 0);
    o->w_out = Operand{p.w_out, p.O, p.F, ld_f};
  }
  if (p.copy_dy) {
    add_align(jobs, f.dy, f.ld_dy, p.M, p.O, p.dy, ld_o, p.M, 0, 0);
    o->dy = Operand{p.dy, p.M, p.O, ld_o};
  }
  return run_align<uint16_t>(jobs, sms, st);
}

template <typename T>
constexpr CUtensorMapDataType map_type() {
  return std::is_same_v<T, __nv_bfloat16> ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}
template <typename T>
constexpr uint32_t mma_format() {
  return std::is_same_v<T, __nv_bfloat16> ? tc::kFmtBf16 : tc::kFmtF16;
}

// out [M, N] = A B^T (+ bias), rows in one run or two
template <typename T>
gf_status product(const Shape& s, const Operand& a, bool a_mn, const Operand& b, bool b_mn, int64_t M, int64_t N, int64_t K,
                  void* out, int64_t ld_out, const void* bias, int64_t seg_pad, int64_t seg, void* partial, int sms,
                  cudaStream_t st) {
  GemmParams p{};
  GFB_TRY(set_operands(p, s, a, a_mn, b, b_mn, 2, map_type<T>(), tc::kAccF32, mma_format<T>(), false));
  p.M = (int)M;
  p.N = (int)N;
  p.kb_total = (int)ceil_div(K, 64);
  p.out = out;
  p.ld_out = ld_out;
  p.tma_out = aligned_rows(out, M, ld_out, 2) && !seg_pad;
  p.bias = bias;
  p.seg_pad = (int)seg_pad;
  p.seg = (int)seg;
  p.partial = static_cast<float*>(partial);
  p.ld_partial = round_up<int64_t>(N, 32);
  if (s.splits > 1)
    GFB_TRY(make_out_map(&p.mo, Operand{partial, (int64_t)s.splits * s.rows_m(), p.ld_partial, p.ld_partial},
                         CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4));
  else if (p.tma_out)
    GFB_TRY(make_out_map(&p.mo, Operand{out, M, N, ld_out}, map_type<T>(), 2));
  GFB_TRY((launch_gemm<EPI_STORE, T, 0, false>(p, s, sms, st)));
  if (s.splits > 1) {
    GFB_CUDA(launch(join_kernel<T>, dim3(grid_for(M * (p.ld_partial / 4), 256, sms)), 256, st, p));
  }
  return GF_OK;
}

template <int EPI, typename T>
gf_status gated(const GemmParams& p, const Shape& s, int act, int sms, cudaStream_t st) {
  if (act == GF_ACT_GELU)
    return p.drop.on ? launch_gemm<EPI, T, GF_ACT_GELU, true>(p, s, sms, st)
                     : launch_gemm<EPI, T, GF_ACT_GELU, false>(p, s, sms, st);
  return p.drop.on ? launch_gemm<EPI, T, GF_ACT_SILU, true>(p, s, sms, st)
                   : launch_gemm<EPI, T, GF_ACT_SILU, false>(p, s, sms, st);
}

template <typename T, bool GATED>
gf_status skinny(const SkinnyParams& p, cudaStream_t st) {
  // (gated: a warp per column of h, padding included; else four per column of y)
  const int cols = GATED ? p.hp : p.n, per = GATED ? kSkinnyWarps : kSkinnyWarps / 4;
  const int grid = (int)ceil_div(cols, per);
  const auto kernel = p.tokens == 1 ? skinny_kernel<T, 1, GATED> : skinny_kernel<T, kSkinnyTokens, GATED>;
  GFB_CUDA(launch(kernel, dim3(grid), 32 * kSkinnyWarps, st, p));
  return GF_OK;
}

template <typename T>
gf_status ff_skinny(const gf_gated_ff& f, const FfPlan& pl, cudaStream_t st) {
  SkinnyParams p{};
  p.x = f.x, p.ld_x = f.ld_x;
  p.w = f.w_in, p.ld_w = f.ld_w_in, p.gate_row = pl.F;
  p.bias = f.b_in;
  p.tokens = (int)pl.M, p.n = (int)pl.F, p.k = (int)pl.D, p.hp = (int)pl.Hp;
  p.out = f.h, p.ld_out = pl.Hp;
  p.act = f.activation;
  p.drop = drop_args(f.dropout);
  GFB_TRY((skinny<T, true>(p, st)));
  p.x = f.h, p.ld_x = pl.Hp;
  p.w = f.w_out, p.ld_w = f.ld_w_out;
  p.bias = f.b_out;
  p.n = (int)pl.O, p.k = (int)pl.F;
  p.out = f.y, p.ld_out = f.ld_y;
  return skinny<T, false>(p, st);
}

template <typename T>
gf_status ff_forward(const gf_gated_ff& f, const FfPlan& pl, cudaStream_t st) {
  if (pl.skinny) return ff_skinny<T>(f, pl, st);
  const int sms = sm_count();
  FfOperands o;
  GFB_TRY(align_ff(f, pl, &o, sms, st));
  GemmParams p{};
  GFB_TRY(set_operands(p, pl.in, o.x, false, o.w_in, false, 2, map_type<T>(), tc::kAccF32, mma_format<T>(), true));
  p.M = (int)pl.M;
  p.N = (int)pl.F;
  p.hp = (int)pl.Hp;
  p.gate_row = (int)pl.Hp;
  p.kb_total = (int)ceil_div(pl.D, 64);
  p.bias = f.b_in;
  p.drop = drop_args(f.dropout);
  GFB_TRY(make_out_map(&p.mo, Operand{f.h, pl.M, pl.Hp, pl.Hp}, map_type<T>(), 2));
  GFB_TRY((gated<EPI_GATED, T>(p, pl.in, f.activation, sms, st)));
  return product<T>(pl.out, Operand{f.h, pl.M, pl.Hp, pl.Hp}, false, o.w_out, false, pl.M, pl.O, pl.F, f.y, f.ld_y, f.b_out,
                    0, 0, pl.partial, sms, st);
}

template <typename T>
gf_status column_sums(const SumJobs& jobs, int n, cudaStream_t st) {
  int64_t cols = 0;
  int parts = 0;
  for (int i = 0; i < n; ++i) {
    cols = jobs.job[i].cols > cols ? jobs.job[i].cols : cols;
    parts = jobs.job[i].parts > parts ? jobs.job[i].parts : parts;
  }
  GFB_CUDA(launch(column_sums_kernel<T>, dim3((unsigned)ceil_div(cols, 32), parts, n), 256, st, jobs));
  GFB_CUDA(launch(column_join_kernel<T>, dim3((unsigned)ceil_div(cols, 256), 1, n), 256, st, jobs));
  return GF_OK;
}

template <typename T>
gf_status ff_backward(const gf_gated_ff& f, const FfPlan& pl, cudaStream_t st) {
  const int sms = sm_count();
  FfOperands o;
  GFB_TRY(align_ff(f, pl, &o, sms, st));
  const Operand du{pl.du, pl.M, 2 * pl.Hp, 2 * pl.Hp};
  if (pl.du) {
    GemmParams p{};
    GFB_TRY(set_operands(p, pl.dh, o.x, false, o.w_in, false, 2, map_type<T>(), tc::kAccF32, mma_format<T>(), true));
    p.M = (int)pl.M;
    p.N = (int)pl.F;
    p.hp = (int)pl.Hp;
    p.gate_row = (int)pl.Hp;
    p.kb_total = (int)ceil_div(pl.D, 64);
    p.bias = f.b_in;
    p.drop = drop_args(f.dropout);
    // dh: dy as stored, w_out with its columns along N
    const int half = pl.dh.pair ? p.cols / 2 : p.cols;
    p.kb2 = (int)ceil_div(pl.O, 64);
    p.idesc2 = tc::instruction_desc(tc::kAccF32, mma_format<T>(), false, true, p.cols, pl.dh.pair);
    p.tx_bytes2 = (kABytes + 128 * round_up(half, 64)) * (pl.dh.pair ? 2 : 1);
    GFB_TRY(make_map(&p.ma2, o.dy, map_type<T>(), 2, 64, kTileM));
    GFB_TRY(make_map(&p.mb2, o.w_out, map_type<T>(), 2, 64, 64));
    GFB_TRY(make_out_map(&p.mo, du, map_type<T>(), 2));
    GFB_TRY((gated<EPI_GATED_BWD, T>(p, pl.dh, f.activation, sms, st)));
  }
  if (f.dx)
    GFB_TRY(product<T>(pl.dx, du, false, o.w_in, true, pl.M, pl.D, 2 * pl.Hp, f.dx, pl.D, nullptr, 0, 0, pl.partial, sms, st));
  if (f.dw_in)
    GFB_TRY(product<T>(pl.dw_in, du, true, o.x, true, 2 * pl.Hp, pl.D, pl.M, f.dw_in, pl.D, nullptr,
                       pl.Hp == pl.F ? 0 : pl.Hp, pl.F, pl.partial, sms, st));
  if (f.dw_out)
    GFB_TRY(product<T>(pl.dw_out, o.dy, true, Operand{f.h, pl.M, pl.Hp, pl.Hp}, true, pl.O, pl.F, pl.M, f.dw_out, pl.F,
                       nullptr, 0, 0, pl.partial, sms, st));
  SumJobs sums{};
  int n = 0;
  if (f.db_in)
    sums.job[n++] = SumJob{pl.du, 2 * pl.Hp, (int)pl.M, (int)(2 * pl.Hp), pl.in_run, pl.in_parts,
                           pl.Hp == pl.F ? 0 : (int)pl.Hp, (int)pl.F, static_cast<float*>(pl.in_sums), f.db_in};
  if (f.db_out)
    sums.job[n++] = SumJob{f.dy, f.ld_dy, (int)pl.M, (int)pl.O, pl.out_run, pl.out_parts, 0, 0,
                           static_cast<float*>(pl.out_sums), f.db_out};
  return n ? column_sums<T>(sums, n, st) : GF_OK;
}

// ---- dropout and the 8-bit product

template <typename T, bool RES, typename I>
cudaError_t launch_dropout(const DropoutParams& p, bool vec, bool by_rows, int sms, cudaStream_t st) {
  const int grid = grid_for(ceil_div(p.rows * p.groups, 2), 256, sms);
  const auto kernel = vec       ? dropout_kernel<T, true, false, RES, I>
                      : by_rows ? dropout_kernel<T, false, true, RES, I>
                                : dropout_kernel<T, false, false, RES, I>;
  return launch(kernel, dim3(grid), 256, st, p);
}
template <typename T>
cudaError_t launch_dropout(DropoutParams& p, bool vec, bool by_rows, int sms, cudaStream_t st) {
  p.groups = ceil_div(p.cols, vec ? 16 / (int64_t)sizeof(T) : 4);
  // positions pass their end by up to two strides of the grid
  const bool narrow = p.rows * p.groups < (int64_t(1) << 31);
  if (p.res)
    return narrow ? launch_dropout<T, true, uint32_t>(p, vec, by_rows, sms, st)
                  : launch_dropout<T, true, uint64_t>(p, vec, by_rows, sms, st);
  return narrow ? launch_dropout<T, false, uint32_t>(p, vec, by_rows, sms, st)
                : launch_dropout<T, false, uint64_t>(p, vec, by_rows, sms, st);
}

template <typename T, int TPR, int VPL>
cudaError_t launch_quantize(int64_t rows, int64_t cols, const void* x, int64_t ld_x, int8_t* q, int64_t ld_q, float* scale, int sms,
                     cudaStream_t st) {
  return launch(quantize_rows_kernel<T, TPR, VPL>, dim3(grid_for(rows, 256 / TPR, sms)), 256, st, rows, (int)cols,
         static_cast<const T*>(x), ld_x, q, ld_q, scale);
}
template <typename T>
cudaError_t launch_quantize(int64_t rows, int64_t cols, const void* x, int64_t ld_x, int8_t* q, int64_t ld_q, float* scale, int sms,
                     cudaStream_t st) {
  const bool vec = aligned_rows(x, rows, ld_x, sizeof(T)) && cols % 8 == 0 && ld_q % 8 == 0 &&
                   (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
  // Aligned rows of up to 16384 values stay in registers.  A warp for a short
  // row, a CTA for a long one (a CTA holds at least 4096, so rows of 1280 leave
  // most of it idle), and a CTA too where every row can have its own at once.
  // us for bf16 rows from cold caches, warp / CTA:
  //   aligned  16384 x 1280  12.0 / 31.7   16384 x 2048  18.1 / 34.1   4736 x 2048  7.1 / 11.1
  //              592 x 2048   2.8 /  2.7     148 x 2048   2.1 /  1.4     64 x 1280  1.6 /  1.5
  //   others   16384 x 1001  27.2 / 35.1   16384 x 2047  47.0 / 43.7   4736 x 1537  15.1 / 15.2
  //             2368 x 333    3.7 /  4.5    1184 x 333    3.6 /  2.8     64 x 1001  5.4 /  2.5
  if (vec && cols <= 512) return launch_quantize<T, 32, 2>(rows, cols, x, ld_x, q, ld_q, scale, sms, st);
  if (vec && cols <= 1280) return launch_quantize<T, 32, 5>(rows, cols, x, ld_x, q, ld_q, scale, sms, st);
  if (vec && cols <= 2048 && rows > 4 * (int64_t)sms)
    return launch_quantize<T, 32, 8>(rows, cols, x, ld_x, q, ld_q, scale, sms, st);
  if (vec && cols <= 4096) return launch_quantize<T, 256, 2>(rows, cols, x, ld_x, q, ld_q, scale, sms, st);
  if (vec && cols <= 16384) return launch_quantize<T, 256, 8>(rows, cols, x, ld_x, q, ld_q, scale, sms, st);
  if (cols <= 1536 && rows > 8 * (int64_t)sms)
    return launch_quantize<T, 32, 0>(rows, cols, x, ld_x, q, ld_q, scale, sms, st);
  return launch_quantize<T, 256, 0>(rows, cols, x, ld_x, q, ld_q, scale, sms, st);
}

bool known_dtype(int d) { return d == GF_F32 || d == GF_BF16 || d == GF_F16; }
int dtype_size(int d) { return d == GF_F32 ? 4 : 2; }

struct Int8Plan {
  bool copy_a, copy_b;
  Shape shape;
  void *a, *b;
  size_t bytes;
};
gf_status check_int8(const char* who, const gf_int8_product* p, bool quantised) {
  if (!p) return fail(GF_ERR_INVALID_ARG, "%s: the description must be non-null", who);
  if (p->m < 0 || p->n <= 0 || p->k <= 0) return fail(GF_ERR_INVALID_ARG, "%s: sizes must be positive (m may be 0)", who);
  if (p->m > kMaxDim || p->n > kMaxDim) return fail(GF_ERR_UNSUPPORTED, "%s: a size is above 2^31 - 512", who);
  if (p->k > 131071) return fail(GF_ERR_UNSUPPORTED, "%s: k must be at most 131071 (the sums are 32-bit integers)", who);
  if (!known_dtype(p->dtype)) return fail(GF_ERR_UNSUPPORTED, "%s: dtype must be GF_F32, GF_BF16 or GF_F16", who);
  if (p->reserved != 0) return fail(GF_ERR_INVALID_ARG, "%s: reserved fields must be 0", who);
  if (const gf_status s = check_elements(who, dtype_size(p->dtype), p->bias, p->out); s != GF_OK) return s;
  if (const gf_status s = check_elements(who, 4, quantised ? p->a_scale : nullptr, p->b_scale); s != GF_OK) return s;
  if ((quantised && p->ld_a < p->k) || p->ld_b < p->k || p->ld_out < p->n)
    return fail(GF_ERR_INVALID_ARG, "%s: a leading dimension is smaller than its row", who);
  return GF_OK;
}
Int8Plan plan_int8(const gf_int8_product& p, char* ws, size_t used) {
  Int8Plan pl{};
  Bump b{ws, used};
  pl.copy_a = !aligned_rows(p.a, p.m, p.ld_a, 1);
  pl.copy_b = !aligned_rows(p.b, p.n, p.ld_b, 1);
  const int64_t ld = round_up<int64_t>(p.k, 16);
  if (pl.copy_a) pl.a = b.take(p.m * ld);
  if (pl.copy_b) pl.b = b.take(p.n * ld);
  pl.shape = choose_shape(p.m, p.n, ceil_div(p.k, 128), EPI_INT8, false, sm_count());
  pl.bytes = b.used > 256 ? b.used : 256;
  return pl;
}

// The quantised activations of gf_int8_linear, at the workspace's start.
struct Quantised {
  int64_t ld;
  int8_t* q;
  float* scale;
  size_t bytes;
};
Quantised place_quantised(const gf_int8_product& p, void* ws) {
  Quantised q{};
  Bump b{static_cast<char*>(ws)};
  q.ld = round_up<int64_t>(p.k, 16);
  q.q = static_cast<int8_t*>(b.take(p.m * q.ld));
  q.scale = static_cast<float*>(b.take(4 * p.m));
  q.bytes = b.used;
  return q;
}

gf_status int8_product(const gf_int8_product& d, const Int8Plan& pl, cudaStream_t st) {
  const int sms = sm_count(), es = dtype_size(d.dtype);
  Operand a{d.a, d.m, d.k, d.ld_a}, b{d.b, d.n, d.k, d.ld_b};
  const int64_t ld = round_up<int64_t>(d.k, 16);
  AlignJobs jobs{};
  if (pl.copy_a) {
    add_align(jobs, d.a, d.ld_a, d.m, d.k, pl.a, ld, d.m, 0, 0);
    a = Operand{pl.a, d.m, d.k, ld};
  }
  if (pl.copy_b) {
    add_align(jobs, d.b, d.ld_b, d.n, d.k, pl.b, ld, d.n, 0, 0);
    b = Operand{pl.b, d.n, d.k, ld};
  }
  GFB_TRY(run_align<uint8_t>(jobs, sms, st));
  GemmParams p{};
  GFB_TRY(set_operands(p, pl.shape, a, false, b, false, 1, CU_TENSOR_MAP_DATA_TYPE_UINT8, tc::kAccS32, tc::kFmtS8, false));
  p.M = (int)d.m;
  p.N = (int)d.n;
  p.kb_total = (int)ceil_div(d.k, 128);
  p.out = d.out;
  p.ld_out = d.ld_out;
  p.tma_out = aligned_rows(d.out, d.m, d.ld_out, es);
  if (p.tma_out)
    GFB_TRY(make_out_map(&p.mo, Operand{d.out, d.m, d.n, d.ld_out},
                         d.dtype == GF_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                         : d.dtype == GF_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                              : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         es));
  p.bias = d.bias;
  p.a_scale = d.a_scale;
  p.b_scale = d.b_scale;
  if (d.dtype == GF_F32) return launch_gemm<EPI_INT8, float, 0, false>(p, pl.shape, sms, st);
  if (d.dtype == GF_BF16) return launch_gemm<EPI_INT8, __nv_bfloat16, 0, false>(p, pl.shape, sms, st);
  return launch_gemm<EPI_INT8, __half, 0, false>(p, pl.shape, sms, st);
}

gf_status quantise(int64_t rows, int64_t cols, int32_t dtype, const void* x, int64_t ld_x, int8_t* q, int64_t ld_q,
                   float* scale, cudaStream_t st) {
  const int sms = sm_count();
  GFB_CUDA(dtype == GF_F32    ? launch_quantize<float>(rows, cols, x, ld_x, q, ld_q, scale, sms, st)
           : dtype == GF_BF16 ? launch_quantize<__nv_bfloat16>(rows, cols, x, ld_x, q, ld_q, scale, sms, st)
                              : launch_quantize<__half>(rows, cols, x, ld_x, q, ld_q, scale, sms, st));
  return GF_OK;
}

}  // namespace gfb

// ---------------------------------------------------------------------------
// C ABI

extern "C" {

size_t gf_gated_ff_workspace_bytes(const gf_gated_ff* ff, gf_pass pass) {
  if (gfb::check_ff("gf_gated_ff_workspace_bytes", ff) != GF_OK) return 0;
  return ff->tokens == 0 ? 256 : gfb::plan_ff(*ff, pass, nullptr).bytes;
}

gf_status gf_gated_ff_forward(const gf_gated_ff* ff, void* workspace, size_t workspace_bytes, gf_stream stream) {
  const char* who = "gf_gated_ff_forward";
  GFB_TRY(gfb::check_ff(who, ff));
  if (ff->ld_y < ff->out_features) return gf::fail(GF_ERR_INVALID_ARG, "%s: ld_y is smaller than its row", who);
  if (ff->tokens == 0) return GF_OK;
  if (!ff->x || !ff->w_in || !ff->w_out || !ff->h || !ff->y)
    return gf::fail(GF_ERR_INVALID_ARG, "%s: x, w_in, w_out, h and y must be non-null", who);
  if (reinterpret_cast<uintptr_t>(ff->h) & 15u) return gf::fail(GF_ERR_INVALID_ARG, "%s: h must be 16-byte aligned", who);
  const gfb::FfPlan pl = gfb::plan_ff(*ff, GF_PASS_FORWARD, static_cast<char*>(workspace));
  GFB_TRY(gfb::check_workspace(who, workspace, workspace_bytes, pl.bytes));
  gfb::Range r("gfblock.gated_ff_forward");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return ff->dtype == GF_BF16 ? gfb::ff_forward<__nv_bfloat16>(*ff, pl, st) : gfb::ff_forward<__half>(*ff, pl, st);
}

gf_status gf_gated_ff_backward(const gf_gated_ff* ff, void* workspace, size_t workspace_bytes, gf_stream stream) {
  const char* who = "gf_gated_ff_backward";
  GFB_TRY(gfb::check_ff(who, ff));
  if (ff->ld_dy < ff->out_features) return gf::fail(GF_ERR_INVALID_ARG, "%s: ld_dy is smaller than its row", who);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (ff->tokens == 0) {  // empty sums
    const size_t d = ff->in_features, f = ff->hidden, o = ff->out_features;
    if (ff->dw_in) GFB_CUDA(cudaMemsetAsync(ff->dw_in, 0, 2 * 2 * f * d, st));
    if (ff->db_in) GFB_CUDA(cudaMemsetAsync(ff->db_in, 0, 2 * 2 * f, st));
    if (ff->dw_out) GFB_CUDA(cudaMemsetAsync(ff->dw_out, 0, 2 * o * f, st));
    if (ff->db_out) GFB_CUDA(cudaMemsetAsync(ff->db_out, 0, 2 * o, st));
    return GF_OK;
  }
  if (!ff->dy) return gf::fail(GF_ERR_INVALID_ARG, "%s: dy must be non-null", who);
  if ((ff->dx || ff->dw_in || ff->db_in) && (!ff->x || !ff->w_in || !ff->w_out))
    return gf::fail(GF_ERR_INVALID_ARG, "%s: dx, dw_in and db_in need x, w_in and w_out", who);
  if (ff->dw_out && !ff->h) return gf::fail(GF_ERR_INVALID_ARG, "%s: dw_out needs h", who);
  if (reinterpret_cast<uintptr_t>(ff->h) & 15u) return gf::fail(GF_ERR_INVALID_ARG, "%s: h must be 16-byte aligned", who);
  const gfb::FfPlan pl = gfb::plan_ff(*ff, GF_PASS_BACKWARD, static_cast<char*>(workspace));
  GFB_TRY(gfb::check_workspace(who, workspace, workspace_bytes, pl.bytes));
  gfb::Range r("gfblock.gated_ff_backward");
  return ff->dtype == GF_BF16 ? gfb::ff_backward<__nv_bfloat16>(*ff, pl, st) : gfb::ff_backward<__half>(*ff, pl, st);
}

gf_status gf_dropout(int64_t rows, int64_t cols, int32_t dtype, const gf_dropout_rule* rule, const void* x,
                     int64_t x_row_stride, int64_t x_col_stride, const void* residual, int64_t r_row_stride,
                     int64_t r_col_stride, void* y, gf_stream stream) {
  const char* who = "gf_dropout";
  if (!rule) return gf::fail(GF_ERR_INVALID_ARG, "%s: the rule must be non-null", who);
  GFB_TRY(gfb::check_rule(who, *rule));
  if (rows < 0 || cols < 0) return gf::fail(GF_ERR_INVALID_ARG, "%s: sizes must not be negative", who);
  if (!gfb::known_dtype(dtype)) return gf::fail(GF_ERR_UNSUPPORTED, "%s: dtype must be GF_F32, GF_BF16 or GF_F16", who);
  if (rows == 0 || cols == 0) return GF_OK;
  if (cols > (int64_t(1) << 33) || rows > (int64_t(1) << 62) / cols)
    return gf::fail(GF_ERR_UNSUPPORTED, "%s: more than 2^33 columns or 2^62 elements", who);
  if (!x || !y) return gf::fail(GF_ERR_INVALID_ARG, "%s: x and y must be non-null", who);
  GFB_TRY(gfb::check_elements(who, gfb::dtype_size(dtype), x, residual, y));
  gfb::Range range("gfblock.dropout");
  const int es = gfb::dtype_size(dtype);
  gfb::DropoutParams p{};
  p.rows = rows, p.cols = cols;
  p.x = x, p.x_rs = x_row_stride, p.x_cs = x_col_stride;
  p.res = residual, p.r_rs = r_row_stride, p.r_cs = r_col_stride;
  p.y = y;
  p.drop = gfb::drop_args(*rule);
  // 16-byte accesses where every row of every operand starts on such a boundary
  const bool vec = cols % (16 / es) == 0 && x_col_stride == 1 && gfb::aligned_rows(x, rows, x_row_stride, es) &&
                   gfb::aligned_rows(y, rows, cols, es) &&
                   (!residual || (r_col_stride == 1 && gfb::aligned_rows(residual, rows, r_row_stride, es)));
  const bool by_rows = x_col_stride > x_row_stride && x_row_stride > 0;
  const int sms = gfb::sm_count();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  GFB_CUDA(dtype == GF_F32    ? gfb::launch_dropout<float>(p, vec, by_rows, sms, st)
           : dtype == GF_BF16 ? gfb::launch_dropout<__nv_bfloat16>(p, vec, by_rows, sms, st)
                              : gfb::launch_dropout<__half>(p, vec, by_rows, sms, st));
  return GF_OK;
}

gf_status gf_quantize_rows(int64_t rows, int64_t cols, int32_t dtype, const void* x, int64_t ld_x, int8_t* q, int64_t ld_q,
                           float* scale, gf_stream stream) {
  const char* who = "gf_quantize_rows";
  if (rows < 0 || cols <= 0) return gf::fail(GF_ERR_INVALID_ARG, "%s: sizes must be positive (rows may be 0)", who);
  if (cols > gfb::kMaxDim) return gf::fail(GF_ERR_UNSUPPORTED, "%s: cols is above 2^31 - 512", who);
  if (!gfb::known_dtype(dtype)) return gf::fail(GF_ERR_UNSUPPORTED, "%s: dtype must be GF_F32, GF_BF16 or GF_F16", who);
  if (ld_x < cols || ld_q < cols) return gf::fail(GF_ERR_INVALID_ARG, "%s: a leading dimension is smaller than its row", who);
  if (rows == 0) return GF_OK;
  if (!x || !q || !scale) return gf::fail(GF_ERR_INVALID_ARG, "%s: x, q and scale must be non-null", who);
  GFB_TRY(gfb::check_elements(who, gfb::dtype_size(dtype), x));
  GFB_TRY(gfb::check_elements(who, 4, scale));
  gfb::Range range("gfblock.quantize_rows");
  return gfb::quantise(rows, cols, dtype, x, ld_x, q, ld_q, scale, reinterpret_cast<cudaStream_t>(stream));
}

size_t gf_int8_product_workspace_bytes(const gf_int8_product* p) {
  if (gfb::check_int8("gf_int8_product_workspace_bytes", p, true) != GF_OK) return 0;
  return p->m == 0 ? 256 : gfb::plan_int8(*p, nullptr, 0).bytes;
}

gf_status gf_int8_matmul(const gf_int8_product* d, void* workspace, size_t workspace_bytes, gf_stream stream) {
  const char* who = "gf_int8_matmul";
  GFB_TRY(gfb::check_int8(who, d, true));
  if (d->m == 0) return GF_OK;
  if (!d->a || !d->b || !d->a_scale || !d->b_scale || !d->out)
    return gf::fail(GF_ERR_INVALID_ARG, "%s: a, b, a_scale, b_scale and out must be non-null", who);
  const gfb::Int8Plan pl = gfb::plan_int8(*d, static_cast<char*>(workspace), 0);
  GFB_TRY(gfb::check_workspace(who, workspace, workspace_bytes, pl.bytes));
  gfb::Range range("gfblock.int8_matmul");
  return gfb::int8_product(*d, pl, reinterpret_cast<cudaStream_t>(stream));
}

size_t gf_int8_linear_workspace_bytes(const gf_int8_product* p) {
  if (gfb::check_int8("gf_int8_linear_workspace_bytes", p, false) != GF_OK) return 0;
  if (p->m == 0) return 256;
  gf_int8_product d = *p;
  const gfb::Quantised q = gfb::place_quantised(d, nullptr);
  d.a = nullptr;  // aligned, as the workspace is
  d.ld_a = q.ld;
  return gfb::plan_int8(d, nullptr, q.bytes).bytes;
}

gf_status gf_int8_linear(const gf_int8_product* p, const void* x, int64_t ld_x, int32_t x_dtype, void* workspace,
                         size_t workspace_bytes, gf_stream stream) {
  const char* who = "gf_int8_linear";
  GFB_TRY(gfb::check_int8(who, p, false));
  if (!gfb::known_dtype(x_dtype)) return gf::fail(GF_ERR_UNSUPPORTED, "%s: x_dtype must be GF_F32, GF_BF16 or GF_F16", who);
  if (ld_x < p->k) return gf::fail(GF_ERR_INVALID_ARG, "%s: a leading dimension is smaller than its row", who);
  if (p->m == 0) return GF_OK;
  if (!x || !p->b || !p->b_scale || !p->out)
    return gf::fail(GF_ERR_INVALID_ARG, "%s: x, b, b_scale and out must be non-null", who);
  GFB_TRY(gfb::check_elements(who, gfb::dtype_size(x_dtype), x));
  gf_int8_product d = *p;
  const gfb::Quantised q = gfb::place_quantised(d, workspace);
  d.a = q.q;
  d.ld_a = q.ld;
  d.a_scale = q.scale;
  const gfb::Int8Plan pl = gfb::plan_int8(d, static_cast<char*>(workspace), q.bytes);
  GFB_TRY(gfb::check_workspace(who, workspace, workspace_bytes, pl.bytes));
  gfb::Range range("gfblock.int8_linear");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  GFB_TRY(gfb::quantise(d.m, d.k, x_dtype, x, ld_x, q.q, q.ld, q.scale, st));
  return gfb::int8_product(d, pl, st);
}

gf_status gf_block_status(gf_stream stream, int reset, uint32_t* flags_out) {
  if (!flags_out) return gf::fail(GF_ERR_INVALID_ARG, "gf_block_status: flags_out must be non-null");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const uint32_t zero = 0;
  uint32_t flags = 0;
  GFB_CUDA(cudaMemcpyFromSymbolAsync(&flags, gfb::g_status, sizeof(flags), 0, cudaMemcpyDeviceToHost, st));
  GFB_CUDA(cudaStreamSynchronize(st));
  if (reset) {
    GFB_CUDA(cudaMemcpyToSymbolAsync(gfb::g_status, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, st));
    GFB_CUDA(cudaStreamSynchronize(st));
  }
  *flags_out = flags;
  return GF_OK;
}

gf_status gf_block_status_async(uint32_t* flags_out, gf_stream stream) {
  const char* who = "gf_block_status_async";
  if (!flags_out) return gf::fail(GF_ERR_INVALID_ARG, "%s: flags_out must be non-null", who);
  GFB_TRY(gfb::check_elements(who, 4, flags_out));
  GFB_CUDA(cudaMemcpyFromSymbolAsync(flags_out, gfb::g_status, sizeof(uint32_t), 0, cudaMemcpyDeviceToDevice,
                                     reinterpret_cast<cudaStream_t>(stream)));
  return GF_OK;
}

}  // extern "C"
