// Products of microscaled matrices (formats: mx.cuh):  C = act(A B^T + bias),  A: M x K, B: N x K, both quantised along K.
//
// tcgen05.mma with block scales: kind::mxf8f6f4 for MXFP8 (32 of K an instruction), kind::mxf4 for MXFP4 (64), fp32 accumulators in
// TMEM.  A step of the main loop is 128 bytes of every row in either format (128 or 256 of K, four instructions); its
// codes arrive by TMA with a 128-byte swizzle, its scales as the 512-byte pieces in which they are kept, and the issuing thread copies
// those from shared memory into TMEM (tcgen05.cp) before the instructions that read them.  A set of scale columns
// is written again once the step that read it has ended.
//
// Two kernels.  Pairs: a cluster of two CTAs per 256 x 256 tile (cta_group::2), persistent, for products with tiles enough to fill
// the SMs, or two pairs per tile that share K.  Clusters: one tile of 128 columns of C (rows of B: the 128 rows of an instruction) by 16 to 128 rows of C per cluster of up to
// eight CTAs, each of which takes a part of K; the parts meet in distributed shared memory in the order of the CTAs.
#include "pair.cuh"
#include "mx.cuh"

#include <atomic>

#include <string.h>

using namespace gb;
using namespace gbmx;

namespace {

enum Act : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU_TANH = 2, ACT_GELU_ERF = 3 };
enum Out : int { OUT_BF16 = 0, OUT_F16 = 1, OUT_F32 = 2 };

struct MxArgs {
  int M, N, steps;         // steps of the main loop over all of K
  int num_m, num_n;        // tiles
  int splits, steps_per;   // slice s of a tile takes steps [s * steps_per, (s + 1) * steps_per)
  void* C;                 // rows ldc elements apart
  long long ldc;
  const void* bias;        // N values in C's type, or fp32; null: none
  int bias_f32, act, out;
  int vectors;             // rows of C on boundaries and of whole pieces of 32 or of 16 bytes: that; else 0
  int* status;
};

template <int FMT>
struct Fmt {
  static constexpr int PIECES = FMT == FP8 ? 1 : 2;          // scale pieces of a step: 128 columns each
  static constexpr uint32_t ELEM = FMT == FP8 ? 0u : 1u;     // E4M3 of kind::mxf8f6f4, E2M1 of kind::mxf4
  // instruction k of a step: piece, and byte of the four scales in a TMEM word
  static constexpr int piece(int k) { return FMT == FP8 ? 0 : k >> 1; }
  static constexpr uint32_t byte(int k) { return FMT == FP8 ? k : (k & 1) * 2; }
};

// Instruction descriptor of a block-scaled product: byte of B's scales at [4,6), formats at [7,10) and [10,13), N >> 3 at
// [17,23), scales in UE8M0 (bit 23), M >> 4 at [24,29), byte of A's scales at [29,31).  Both operands K-major.
__host__ __device__ constexpr uint32_t scaled_idesc(uint32_t elem, uint32_t M, uint32_t N, uint32_t byte) {
  return (byte << 4) | (elem << 7) | (elem << 10) | ((N >> 3) << 17) | (1u << 23) | ((M >> 4) << 24) | (byte << 29);
}

#define GB_MX_MMA(GROUP, KIND)                                                                            \
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"                                                \
               "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d), \
               "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory")
template <int FMT, int CTAS>
__device__ __forceinline__ void mma_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  if constexpr (FMT == FP8 && CTAS == 1) GB_MX_MMA("1", "mxf8f6f4.block_scale.scale_vec::1X");
  if constexpr (FMT == FP8 && CTAS == 2) GB_MX_MMA("2", "mxf8f6f4.block_scale.scale_vec::1X");
  if constexpr (FMT == FP4 && CTAS == 1) GB_MX_MMA("1", "mxf4.block_scale.scale_vec::2X");
  if constexpr (FMT == FP4 && CTAS == 2) GB_MX_MMA("2", "mxf4.block_scale.scale_vec::2X");
}
// A piece of 512 bytes (32 rows of 16) into four columns of TMEM, the same in each quarter of the lanes; in a pair, each CTA's own.
template <int CTAS>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem) {
  const uint64_t d = make_smem_desc_plain(smem, 16, 128);
  if (CTAS == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
  else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}

__device__ __forceinline__ float max_nan(float a, float b) {       // NaN stays NaN
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// GELU by tanh of two values, as v / (1 + exp(-2 u)) = v / 2 (1 + tanh u): without the cancellation of 1 + tanh u, in which an error of 2^-11
// (the hardware's tanh) is a fifth of the value at v = -3.  Both reciprocals are one of the product, so values stop at -7.4, where the
// result is -2e-17 (two exponentials of 2^59 still multiply); NaN of one does not reach the other.  One by one, two operations of the special
// function unit a value instead of one and a half, 16384 x 2304 x 768 bf16 in MXFP8 took 49.4 us, so 41.6 (the hardware's tanh 40.2; no activation 32.1).
__device__ __forceinline__ void gelu_tanh_two(float& x, float& y) {
  constexpr float c = -2.f * 0.7978845608f * 1.442695041f;
  const float lx = max_nan(x, -7.4f), ly = max_nan(y, -7.4f);
  const uint64_t v = pair_of(fmaxf(x, -7.4f), fmaxf(y, -7.4f));
  float a, b;
  parts_of(mul_pair(v, fma_pair(mul_pair(v, v), pair_of(0.044715f * c, 0.044715f * c), pair_of(c, c))), a, b);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
  parts_of(add_pair(pair_of(a, b), pair_of(1.f, 1.f)), a, b);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a * b));
  parts_of(mul_pair(pair_of(lx, ly), mul_pair(pair_of(r, r), pair_of(b, a))), x, y);
}
// GELU by the error function of two values: max(v, 0) - g(|v|) with g(a) = a / 2 erfc(a / sqrt 2) = a exp(-a^2 / 2) q(a), q = erfcx(a / sqrt 2) / 2
// as a polynomial in t = 1 / (1 + 0.3 a) (least largest relative error over [0, 13.2], 1.2e-7).  The form with 1 + erf loses the
// values of negative v, 1e-3 of them at -3.5 and all at -5.5.  1024 x 8192 x 2048 bf16 in MXFP8: 1 + erff 25.3 us, erfcf 44.6, so 20.7.
__device__ __forceinline__ void gelu_erf_two(float& x, float& y) {
  const auto both = [](float c) { return pair_of(c, c); };
  const uint64_t v = pair_of(fminf(fabsf(x), 13.2f), fminf(fabsf(y), 13.2f));
  float a, b, ea, eb, r;
  parts_of(fma_pair(v, both(0.3f), both(1.f)), a, b);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a * b));
  const uint64_t t = mul_pair(both(r), pair_of(b, a));
  parts_of(mul_pair(mul_pair(v, v), both(-0.5f * 1.442695041f)), ea, eb);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(ea));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(eb));
  uint64_t q = fma_pair(t, both(0.0360886380f), both(-0.158932477f));
  q = fma_pair(t, q, both(0.209343597f));
  q = fma_pair(t, q, both(-0.0564470105f));
  q = fma_pair(t, q, both(0.130030736f));
  q = fma_pair(t, q, both(0.0994656980f));
  q = fma_pair(t, q, both(0.1208262f));
  q = fma_pair(t, q, both(0.119624548f));
  parts_of(mul_pair(mul_pair(v, pair_of(ea, eb)), mul_pair(t, q)), a, b);
  x = max_nan(x, 0.f) - a;
  y = max_nan(y, 0.f) - b;
}
__device__ __forceinline__ void activate_two(float& x, float& y, int act) {
  switch (act) {
    case ACT_RELU:                         // (a block with a NaN or an infinity is NaN, and so are its products)
      x = max_nan(x, 0.f);
      y = max_nan(y, 0.f);
      break;
    case ACT_GELU_TANH: gelu_tanh_two(x, y); break;
    case ACT_GELU_ERF: gelu_erf_two(x, y); break;
  }
}
__device__ __forceinline__ float bias_at(const MxArgs& a, int col) {
  if (a.bias == nullptr || col >= a.N) return 0.f;
  if (a.bias_f32) return __ldg((const float*)a.bias + col);
  const uint16_t u = __ldg((const uint16_t*)a.bias + col);
  return a.out == OUT_BF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}
__device__ __forceinline__ uint32_t pack_out(const MxArgs& a, float x, float y) { return a.out == OUT_BF16 ? pack_bf16(x, y) : pack_f16(x, y); }
__device__ __forceinline__ void store_out(const MxArgs& a, long long at, float v) {
  if (a.out == OUT_F32) ((float*)a.C)[at] = v;
  else ((uint16_t*)a.C)[at] = (uint16_t)pack_out(a, v, 0.f);
}

// Tiles in groups of eight rows of tiles, so that those running together share operands in L2.
__device__ __forceinline__ void tile_at(int t, int num_m, int num_n, int& m, int& n) {
  const int per = 8 * num_n, g = t / per, first = g * 8, rows = min(8, num_m - first), r = t - g * per;
  m = first + r % rows;
  n = r / rows;
}

// ---------------------------------------------------------------------------------------------------------------------------
// Pairs: tiles of 256 x 256.  Each CTA stages its 128 rows of A with their scales and half of the tile's rows of B, and the scales of all of
// these (its half of the accumulator has all columns); CTA 0 issues.  Two accumulators of 256 columns and the scales do not fit into TMEM's
// 512, so the two overlap in columns 128 to 255: the epilogue drains those first, and then the next tile starts.  (Tiles of 192 columns,
// whose accumulators do not overlap, were no faster for a K of 768, 24 against 25 us at 16384 x 2304 in MXFP4, and slower for longer ones:
// 8192^3 437 against 358 us in MXFP8, bursts on one box; on others this one takes up to 387, and 440 at the power cap.)  Four sets of scale
// columns take turns.
// ---------------------------------------------------------------------------------------------------------------------------
template <int FMT>
struct PairCfg {
  static constexpr int STAGES = 6, EW = 8, THREADS = 96 + 32 * EW;
  static constexpr int A_BYTES = 128 * 128, B_BYTES = 128 * 128, TILE_BYTES = A_BYTES + B_BYTES;
  static constexpr int PIECE = 512, S_BYTES = 3 * Fmt<FMT>::PIECES * PIECE;      // A's row of pieces, B's two
  static constexpr int OFF_SCALES = STAGES * TILE_BYTES;
  static constexpr int OFF_OUT = OFF_SCALES + STAGES * S_BYTES;
  static constexpr int OUT_BUF = 1024;                       // of an epilogue warp
  static constexpr int OFF_BIAS = OFF_OUT + EW * OUT_BUF;    // two tiles' bias
  static constexpr int OFF_BARS = OFF_BIAS + 2 * 1024;
  static constexpr int BYTES = OFF_BARS + 256;
  static constexpr int ACC1 = 128, SCALES = 384, SETS = 4, SET = 12 * Fmt<FMT>::PIECES;      // TMEM columns
  static_assert(BYTES <= 232448 && OFF_OUT % 16 == 0, "shared memory");
  static_assert(SCALES + SETS * SET <= 512, "TMEM");
};

// 32 bytes: one store on a 32-byte boundary (wide), else two of which the second may be left out.
__device__ __forceinline__ void store32(uint32_t* to, bool wide, bool both, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, uint32_t f, uint32_t g, uint32_t h) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e), "r"(f), "r"(g), "r"(h) : "memory");
  } else {
    *reinterpret_cast<uint4*>(to) = make_uint4(a, b, c, d);
    if (both) *reinterpret_cast<uint4*>(to + 4) = make_uint4(e, f, g, h);
  }
}

// 32 x 32 results of a warp (a lane has a row) into C.  Rows on 32-byte boundaries: 32 bytes a lane and store, whole sectors straight from the
// registers (an SM stores 32 bytes a clock in any case; by way of shared memory and whole lines it took as long, 25.8 against 26.1 us at
// 16384 x 2304 x 768 in MXFP4, and that took the room of the sixth stage).  Other rows,
// a sector at a time, would write each sector many times: they go through `buf`, a column a lane (which takes 72 us for the 31 of
// vectors at 16384 x 2304 x 768 in MXFP8).
template <bool VECTORS>
__device__ __forceinline__ void store_chunk(const MxArgs& a, uint8_t* buf, int row0, int col0, const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  const long long first = row0;
  if constexpr (VECTORS) {
    if (row0 + lane >= a.M) return;
    const bool wide = a.vectors == 32;
    if (a.out == OUT_F32) {
      float* to = (float*)a.C + (first + lane) * a.ldc + col0;
#pragma unroll
      for (int j = 0; j < 32; j += 8)
        if (col0 + j < a.N) store32(reinterpret_cast<uint32_t*>(to + j), wide, col0 + j + 4 < a.N, __float_as_uint(v[j]), __float_as_uint(v[j + 1]), __float_as_uint(v[j + 2]),
                                    __float_as_uint(v[j + 3]), __float_as_uint(v[j + 4]), __float_as_uint(v[j + 5]), __float_as_uint(v[j + 6]), __float_as_uint(v[j + 7]));
    } else {
      uint16_t* to = (uint16_t*)a.C + (first + lane) * a.ldc + col0;
#pragma unroll
      for (int j = 0; j < 32; j += 16)
        if (col0 + j < a.N) store32(reinterpret_cast<uint32_t*>(to + j), wide, col0 + j + 8 < a.N, pack_out(a, v[j], v[j + 1]), pack_out(a, v[j + 2], v[j + 3]),
                                    pack_out(a, v[j + 4], v[j + 5]), pack_out(a, v[j + 6], v[j + 7]), pack_out(a, v[j + 8], v[j + 9]), pack_out(a, v[j + 10], v[j + 11]),
                                    pack_out(a, v[j + 12], v[j + 13]), pack_out(a, v[j + 14], v[j + 15]));
    }
    return;
  } else {
    const int rows = min(32, a.M - row0);
    if (a.out == OUT_F32) {                                    // eight rows at a time
      float* f = reinterpret_cast<float*>(buf);
#pragma unroll 1
      for (int h = 0; h < 4; h++) {
        __syncwarp();
        if (lane >> 3 == h) {
#pragma unroll
          for (int j = 0; j < 32; j++) f[(lane & 7) * 32 + (j ^ lane)] = v[j];
        }
        __syncwarp();
        if (col0 + lane < a.N)
          for (int r = 8 * h; r < min(rows, 8 * h + 8); r++) ((float*)a.C)[(first + r) * a.ldc + col0 + lane] = f[(r & 7) * 32 + (lane ^ r)];
      }
      return;
    }
    uint32_t* w = reinterpret_cast<uint32_t*>(buf);            // sixteen
#pragma unroll 1
    for (int h = 0; h < 2; h++) {
      __syncwarp();
      if (lane >> 4 == h) {
#pragma unroll
        for (int j = 0; j < 16; j++) w[(lane & 15) * 16 + (j ^ (lane & 15))] = pack_out(a, v[2 * j], v[2 * j + 1]);
      }
      __syncwarp();
      if (col0 + lane < a.N)
        for (int r = 16 * h; r < min(rows, 16 * h + 16); r++)
          ((uint16_t*)a.C)[(first + r) * a.ldc + col0 + lane] = (uint16_t)(w[(r & 15) * 16 + (lane >> 1 ^ (r & 15))] >> (16 * (lane & 1)));
    }
  }
}

__device__ __forceinline__ uint32_t address_in(uint32_t smem, uint32_t rank) {      // of the CTA `rank` of the cluster
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem), "r"(rank));
  return r;
}

// Bias, activation and 32 x 32 results of a warp into C; b: the columns' bias in shared memory.
template <bool VECTORS>
__device__ __forceinline__ void finish_chunk(const MxArgs& a, uint8_t* buf, int row0, int col0, const float* b, float (&v)[32]) {
  if (a.bias != nullptr) {
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 f = *reinterpret_cast<const float4*>(b + j);
      v[j] += f.x; v[j + 1] += f.y; v[j + 2] += f.z; v[j + 3] += f.w;
    }
  }
  if (a.act != ACT_NONE) {
#pragma unroll
    for (int j = 0; j < 32; j += 2) activate_two(v[j], v[j + 1], a.act);
  }
  store_chunk<VECTORS>(a, buf, row0, col0, v);
}

// SLICED: a tile per cluster of two pairs, each of which takes half of K; a pair finishes 128 of the columns, of which the other
// sends it its sums through distributed shared memory.  (2304 x 768 x 16384 in MXFP8: 43.8 us whole, 32.3 as two slices that a second kernel
// added, 28.6 so.  Four pairs were slower than clusters of smaller tiles wherever they fit: 256 x 2048 x 8192 15.7 against 14.6 us.)
template <int FMT, bool VECTORS, bool SLICED>
__global__ void __launch_bounds__(PairCfg<FMT>::THREADS, 1)
mx_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSA,
               const __grid_constant__ CUtensorMap tmSB, const MxArgs args) {
  using C = PairCfg<FMT>;
  using F = Fmt<FMT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) set_status(args.status, ST_BAD_INDEX, 1024);
    return;
  }
  uint64_t* full = (uint64_t*)(smem + C::OFF_BARS);          // [STAGES]  used in CTA 0
  uint64_t* empty = full + C::STAGES;                        // [STAGES]  per CTA
  uint64_t* ready = empty + C::STAGES;                       // [2]       per CTA: an accumulator is complete
  uint64_t* drained = ready + 2;                             //           used in CTA 0: the columns that the next tile needs are free
  uint64_t* bias_full = drained + 1;                         // [2]       per CTA
  uint64_t* bias_empty = bias_full + 2;                      // [2]       per CTA
  uint32_t* slot = (uint32_t*)(bias_empty + 2);
  volatile int* abort_flag = (volatile int*)(slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = warp & 3, half = (warp - 2) >> 2;      // (of the warps with the results)
  uint8_t* buf = smem + C::OFF_OUT + (warp - 2) * C::OUT_BUF;
  const uint32_t rank = cluster_ctarank(), cta = rank & 1;
  constexpr int S = SLICED ? 2 : 1;
  const int slice = SLICED ? (int)(rank >> 1) : 0, k0 = slice * args.steps_per, k1 = min(args.steps, k0 + args.steps_per);
  const int tiles = args.num_m * args.num_n, pair = blockIdx.x / (2 * S), pairs = gridDim.x / (2 * S);      // (SLICED: one tile for each cluster)
  const auto leaders = [&](uint32_t at) { return SLICED ? address_in(at, rank & ~1u) : at & ~kPeerBit; };   // an address in the pair's CTA 0, in its CTA 1
  const auto peers = [&](uint32_t at) { return SLICED ? address_in(at, rank | 1u) : at | kPeerBit; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&ready[i], 1);
      mbar_init(&bias_full[i], 1);
      mbar_init(&bias_empty[i], C::EW);
    }
    mbar_init(drained, 2 * C::EW);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSB);
  }
  if (warp == 1) {
    tmem_alloc_2sm(slot, 512);
    tmem_relinquish_2sm();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // the barriers of both CTAs are there before either touches the other's
  tc_fence_after();
  const uint32_t tmem = *slot;
  pdl_trigger();
  pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = pair; u < tiles && ok; u += pairs) {
        int mb, nb;
        tile_at(u, args.num_m, args.num_n, mb, nb);
        const int m0 = mb * 256 + (int)cta * 128, n0 = nb * 256 + (int)cta * 128;
        for (int k = k0; k < k1; k++) {
          ok = mbar_wait(&empty[stage], phase ^ 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 31);
          if (!ok) break;
          uint8_t* sa = smem + stage * C::TILE_BYTES;
          uint8_t* ss = smem + C::OFF_SCALES + stage * C::S_BYTES;
          const uint32_t fb = leaders(smem_u32(&full[stage]));        // what lands in either CTA counts on the leader's barrier
          if (cta == 0) mbar_expect_tx(&full[stage], 2 * (C::TILE_BYTES + C::S_BYTES));
          tma_load_3d_2sm(ss, &tmSA, fb, 0, k * F::PIECES, m0 >> 7);
          tma_load_3d_2sm(ss + F::PIECES * C::PIECE, &tmSB, fb, 0, k * F::PIECES, nb * 2);
          tma_load_3d_2sm(sa, &tmA, fb, k * 128, m0, 0);
          tma_load_3d_2sm(sa + C::A_BYTES, &tmB, fb, k * 128, n0, 0);
          if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) {   // a bounded time for the copies in flight
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) { }
      }
    }
  } else if (warp == 1) {
    if (cta == 0 && elect_one()) {
      int n = 0, local = 0;              // steps and tiles so far
      bool ok = true;
      for (int u = pair; u < tiles && ok; u += pairs, local++) {
        if (local > 0) {
          ok = mbar_wait(drained, (local - 1) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 32);
          if (!ok) break;
          tc_fence_after();
        }
        const uint32_t acc = tmem + (local & 1) * C::ACC1;
        for (int k = k0; k < k1; k++, n++) {
          const int stage = n % C::STAGES;
          ok = mbar_wait(&full[stage], (n / C::STAGES) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 33);
          // the step that read this set of scale columns has ended
          if (ok && n >= C::SETS) ok = mbar_wait(&empty[(n - C::SETS) % C::STAGES], ((n - C::SETS) / C::STAGES) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 34);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * C::TILE_BYTES), sb = sa + C::A_BYTES;
          const uint32_t ss = smem_u32(smem + C::OFF_SCALES + stage * C::S_BYTES);
          const uint32_t ta = tmem + C::SCALES + n % C::SETS * C::SET, tb = ta + 4 * F::PIECES;
#pragma unroll
          for (int p = 0; p < F::PIECES; p++) {
            copy_scales<2>(ta + 4 * p, ss + p * C::PIECE);
            copy_scales<2>(tb + 8 * p, ss + (F::PIECES + p) * C::PIECE);
            copy_scales<2>(tb + 8 * p + 4, ss + (2 * F::PIECES + p) * C::PIECE);
          }
#pragma unroll
          for (int i = 0; i < 4; i++)
            mma_scaled<FMT, 2>(acc, make_smem_desc_sw128(sa + i * 32, 16, 1024), make_smem_desc_sw128(sb + i * 32, 16, 1024),
                               scaled_idesc(F::ELEM, 256, 256, F::byte(i)), ta + 4 * F::piece(i), tb + 8 * F::piece(i), k > k0 || i != 0);
          const uint32_t eb = smem_u32(&empty[stage]);
          tc_commit_2sm(eb);
          tc_commit_2sm(peers(eb));
          if (k == k1 - 1) {
            const uint32_t rb = smem_u32(&ready[local & 1]);
            tc_commit_2sm(rb);
            tc_commit_2sm(peers(rb));
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 2 + C::EW) {
    // the bias of the tiles' columns, a tile or two ahead (fetched by the epilogue's warps before a tile's
    // results it kept them waiting: 16384 x 2304 x 768 in MXFP8 37 us, so 32.4; without a bias 30.5)
    if (args.bias != nullptr) {
      int local = 0;
      for (int u = pair; u < tiles; u += pairs, local++) {
        const int which = local & 1;
        int mb, nb;
        tile_at(u, args.num_m, args.num_n, mb, nb);
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = bias_at(args, nb * 256 + i * 32 + lane);
        if (!__all_sync(0xffffffffu, mbar_wait(&bias_empty[which], ((local >> 1) & 1) ^ 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 37))) break;
#pragma unroll
        for (int i = 0; i < 8; i++) reinterpret_cast<float*>(smem + C::OFF_BIAS)[which * 256 + i * 32 + lane] = f[i];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bias_full[which]);
      }
    }
  } else if (!SLICED) {
    int local = 0;
    for (int u = pair; u < tiles; u += pairs, local++) {
      const int which = local & 1;
      int mb, nb;
      tile_at(u, args.num_m, args.num_n, mb, nb);
      const int row0 = mb * 256 + (int)cta * 128 + q * 32;
      if (args.bias != nullptr && !mbar_wait(&bias_full[which], (local >> 1) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 36)) break;
      if (!mbar_wait(&ready[which], (local >> 1) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 35)) break;
      tc_fence_after();
      const uint32_t acc = tmem + which * C::ACC1 + ((uint32_t)(q * 32) << 16);
      // four chunks of 32 columns, two of them in flight; first the two that lie in the other accumulator's columns
      auto column = [&](int i) { return ((i < 2) == (which != 0) ? 0 : 128) + half * 64 + (i & 1) * 32; };
      uint32_t r[2][32];
      tmem_ld32(acc + column(0), r[0]);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        tmem_ld_wait();
        if (i + 1 < 4) tmem_ld32(acc + column(i + 1), r[(i + 1) & 1]);
        if (i == 0) {                      // the next tile may start
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(leaders(smem_u32(drained)));
        }
        const int col0 = nb * 256 + column(i);
        if (row0 >= args.M || col0 >= args.N) continue;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; j++) v[j] = __uint_as_float(r[i & 1][j]);
        finish_chunk<VECTORS>(args, buf, row0, col0, reinterpret_cast<const float*>(smem + C::OFF_BIAS) + which * 256 + column(i), v);
      }
      if (args.bias != nullptr) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&bias_empty[which]);
      }
    }
  }
  if constexpr (SLICED) {
    constexpr int W = 256 / S;             // columns that a pair finishes
    const bool works = warp >= 2 && warp < 2 + C::EW;
    __syncwarp();
    const bool ok = works && __all_sync(0xffffffffu, mbar_wait(&ready[0], 0, abort_flag, args.status, ST_GEMM_TIMEOUT, 38));
    tc_fence_after();
    __syncthreads();
    cluster_sync_all();                    // the products of every pair have been taken: their rings are free
    const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16);
    // sums lie in the ring as [columns / 4][row of 128][4]
    const auto at = [&](int c) { return (uint32_t)((c / 4 * 128 + q * 32 + lane) * 16); };
    if (ok) {
      const uint32_t to = address_in(smem_u32(smem), rank ^ 2);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int c = half * 64 + i * 32;
        uint32_t r[32];
        tmem_ld32(acc + (slice ^ 1) * W + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; j += 4)
          asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + at(c + j)), "r"(r[j]), "r"(r[j + 1]), "r"(r[j + 2]), "r"(r[j + 3]) : "memory");
      }
    }
    __syncwarp();
    cluster_sync_all();
    if (ok) {
      int mb, nb;
      tile_at(pair, args.num_m, args.num_n, mb, nb);
      const int row0 = mb * 256 + (int)cta * 128 + q * 32;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int c = half * 64 + i * 32;
        uint32_t r[32];
        tmem_ld32(acc + slice * W + c, r);
        tmem_ld_wait();
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; j += 4) {      // (the same sum in either order)
          const float4 f = *reinterpret_cast<const float4*>(smem + at(c + j));
          v[j] = __uint_as_float(r[j]) + f.x; v[j + 1] = __uint_as_float(r[j + 1]) + f.y;
          v[j + 2] = __uint_as_float(r[j + 2]) + f.z; v[j + 3] = __uint_as_float(r[j + 3]) + f.w;
        }
        const int col0 = nb * 256 + slice * W + c;
        if (row0 < args.M && col0 < args.N) finish_chunk<VECTORS>(args, buf, row0, col0, reinterpret_cast<const float*>(smem + C::OFF_BIAS) + slice * W + c, v);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // neither CTA leaves while the other may still use its memory or barriers
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_2sm(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Clusters.  The 128 rows of an instruction are rows of B (columns of C), so that a few rows of A cost no more of the tensor core
// than they need.  Where a tile's rows of A start within a scale piece, those of its 32, 64 or 96 first rows are turned to the front in
// shared memory.
// ---------------------------------------------------------------------------------------------------------------------------
template <int FMT, int BN>
struct ClusterCfg {
  // at most half of an SM's shared memory, so that the next kernel's CTAs set up beside this one's
  static constexpr int STAGES = BN <= 32 ? 5 : BN == 64 ? 4 : 3, THREADS = BN >= 32 ? 320 : 192;     // (more hands for the results)
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BN * 128, TILE_BYTES = A_BYTES + B_BYTES;
  static constexpr int PIECE = 512, S_BYTES = 2 * Fmt<FMT>::PIECES * PIECE;
  static constexpr int OFF_SCALES = STAGES * TILE_BYTES;
  static constexpr int OFF_BARS = OFF_SCALES + STAGES * S_BYTES;
  static constexpr int BYTES = OFF_BARS + 256;
  static constexpr int SET = 8 * Fmt<FMT>::PIECES, TMEM = BN <= 64 ? 128 : 256;      // columns: the accumulator, a set of scales for each stage
  static_assert(BYTES <= 115712 && BN * 512 <= OFF_SCALES, "shared memory (the partial tile reuses the ring)");
  static_assert(BN + STAGES * SET <= TMEM, "TMEM");
};

// Bytes that lie side by side (16-byte boundaries and sizes) into shared memory.
__device__ __forceinline__ void load_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Rows of x that the kernel quantises itself.
struct RowsArgs {
  const void* x;
  long long ld;
  int K, aligned;          // rows on 16-byte boundaries, K a multiple of eight
  Extent ext;
};

// Codes and scales of one step's columns of the rows of x, from a warp into a stage's shared memory, in the order of the swizzle.  (With a
// load in flight instead of four: 16 rows, 2048 -> 8192 in MXFP4, 10.7 against 8.6 us.)
template <int FMT, typename X>
__device__ __forceinline__ void stage_rows(const RowsArgs& x, int rows, int step, uint8_t* codes, uint8_t* scales) {
  constexpr int L = FMT == FP8 ? 8 : 16;                     // lanes of a row
  constexpr int AT_ONCE = 32 / L, U = 4;                     // rows; and so many loads in flight
  const int lane = threadIdx.x & 31, l = lane % L, k = (step * L + l) * 16;
  for (int r0 = 0; r0 < rows; r0 += U * AT_ONCE) {
    uint32_t w[U][4 * Elem<X>::SZ];
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int r = r0 + i * AT_ONCE + lane / L;
#pragma unroll
      for (int j = 0; j < 4 * Elem<X>::SZ; j++) w[i][j] = 0;
      if (r >= rows) continue;
      const X* row = reinterpret_cast<const X*>(x.x) + r * x.ld;
      if (x.aligned) load16<X, true>(row, k, x.K, false, x.ext, w[i]);
      else load16<X, false>(row, k, x.K, false, x.ext, w[i]);
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
      if (r0 + i * AT_ONCE >= rows) break;
      const int r = r0 + i * AT_ONCE + lane / L;
      float v[16];
      unpack16<X>(w[i], v);
      uint32_t c[4];
      const uint32_t word = quantize16<FMT>(v, largest16<X>(w[i]), 0xffu << (lane & 24), lane, c);
      if (r >= rows) continue;
      uint8_t* row = codes + r * 128;
      if (FMT == FP8) *reinterpret_cast<uint4*>(row + ((l ^ (r & 7)) << 4)) = make_uint4(c[0], c[1], c[2], c[3]);
      else *reinterpret_cast<uint2*>(row + ((l >> 1 ^ (r & 7)) << 4) + (l & 1) * 8) = make_uint2(c[0], c[1]);
      if ((lane & 7) == 0) *reinterpret_cast<uint32_t*>(scales + (l >> 3) * 512 + r * 16) = word;
    }
  }
}

// X: void, or the type of rows that come as they are (16 at most): the warps that wait for the results quantise them, each its steps, into the
// ring.  Every CTA does so for its part of K.  As two kernels | so, bf16, us: 768 -> 2304 in MXFP8 1 row 5.2 | 4.2, 8 5.6 | 4.6, 16 6.0 | 5.8;
// 2048 -> 8192 in MXFP4 1 row 6.0 | 5.0, 8 6.3 | 6.1, 16 6.7 | 8.6; of the host, 17 | 10.6 at any size, which is why the line is at 16.
template <int FMT, int BN, typename X>
__global__ void __launch_bounds__(ClusterCfg<FMT, BN>::THREADS, 2)
mx_cluster_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const uint8_t* __restrict__ sA, const uint8_t* __restrict__ sB,
                  const RowsArgs x, const MxArgs args) {
  // "A" of the instruction: the product's B (columns of C); its "B": the product's A (rows of C)
  constexpr bool ROWS = !std::is_same<X, void>::value;
  static_assert(!ROWS || BN == 16, "rows as they are: sixteen at most");
  using C = ClusterCfg<FMT, BN>;
  using F = Fmt<FMT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {      // the same in every CTA of the launch
    if (threadIdx.x == 0) set_status(args.status, ST_BAD_INDEX, 1024);
    return;
  }
  uint64_t* full = (uint64_t*)(smem + C::OFF_BARS);
  uint64_t* empty = full + C::STAGES;
  uint64_t* turned = empty + C::STAGES;        // the step's scales of rows of C start at its first row
  uint64_t* done = turned + C::STAGES;
  uint32_t* slot = (uint32_t*)(done + 1);
  volatile int* abort_flag = (volatile int*)(slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = args.splits, tile = blockIdx.x / S, rank = blockIdx.x - tile * S;
  const int c0 = (tile % args.num_n) * 128, r0 = (tile / args.num_n) * BN;       // columns and rows of C
  const int k0 = rank * args.steps_per, k1 = min(args.steps, k0 + args.steps_per);
  const int sub = r0 >> 5 & 3;                 // the tile's first 32 rows among the four of a scale piece
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; s++) { mbar_init(&full[s], ROWS ? 2 : 1); mbar_init(&empty[s], 1); mbar_init(&turned[s], 1); }
    mbar_init(done, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    if (!ROWS) tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(slot, C::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  pdl_trigger();
  pdl_wait();
  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      for (int k = k0, i = 0; k < k1; k++, i++) {
        const int stage = i % C::STAGES;
        ok = mbar_wait(&empty[stage], ((i / C::STAGES) & 1) ^ 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 41);
        if (!ok) break;
        uint8_t* sa = smem + stage * C::TILE_BYTES;
        uint8_t* ss = smem + C::OFF_SCALES + stage * C::S_BYTES;
        mbar_expect_tx(&full[stage], ROWS ? C::A_BYTES + C::S_BYTES / 2 : C::TILE_BYTES + C::S_BYTES);
        tma_load_3d(sa, &tmA, &full[stage], k * 128, c0, 0);
        load_bulk(ss, sA + ((long long)(c0 >> 7) * args.steps + k) * (F::PIECES * C::PIECE), F::PIECES * C::PIECE, &full[stage]);
        if (!ROWS) {
          tma_load_3d(sa + C::A_BYTES, &tmB, &full[stage], k * 128, r0, 0);
          load_bulk(ss + F::PIECES * C::PIECE, sB + ((long long)(r0 >> 7) * args.steps + k) * (F::PIECES * C::PIECE), F::PIECES * C::PIECE, &full[stage]);
        }
      }
      if (!ok) {   // a bounded time for the copies in flight
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) { }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      for (int k = k0, n = 0; k < k1; k++, n++) {
        const int stage = n % C::STAGES;
        if (!mbar_wait(&full[stage], (n / C::STAGES) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 42)) break;
        if (sub != 0 && !mbar_wait(&turned[stage], (n / C::STAGES) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 43)) break;
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + stage * C::TILE_BYTES), sb = sa + C::A_BYTES;
        const uint32_t ss = smem_u32(smem + C::OFF_SCALES + stage * C::S_BYTES);
        const uint32_t ta = tmem + BN + stage * C::SET, tb = ta + 4 * F::PIECES;
#pragma unroll
        for (int p = 0; p < 2 * F::PIECES; p++) copy_scales<1>(ta + 4 * p, ss + p * C::PIECE);
#pragma unroll
        for (int i = 0; i < 4; i++)
          mma_scaled<FMT, 1>(tmem, make_smem_desc_sw128(sa + i * 32, 16, 1024), make_smem_desc_sw128(sb + i * 32, 16, 1024),
                             scaled_idesc(F::ELEM, 128, BN, F::byte(i)), ta + 4 * F::piece(i), tb + 4 * F::piece(i), n > 0 || i != 0);
        tc_commit(&empty[stage]);
      }
      tc_commit(done);
    }
    __syncwarp();
  } else {
    if constexpr (ROWS) {
      for (int k = k0 + warp - 2, i = warp - 2; k < k1; k += 4, i += 4) {
        const int stage = i % C::STAGES;
        if (!__all_sync(0xffffffffu, mbar_wait(&empty[stage], ((i / C::STAGES) & 1) ^ 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 45))) break;
        stage_rows<FMT, X>(x, args.M, k, smem + stage * C::TILE_BYTES + C::A_BYTES, smem + C::OFF_SCALES + stage * C::S_BYTES + F::PIECES * C::PIECE);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[stage]);
      }
    }
    // (One warp, step by step: loads land in any order, and a warp that had not seen a stage's last phase end would take that for the next one's.)
    if (!ROWS && sub != 0 && warp == 2) {
      for (int i = 0; i < k1 - k0; i++) {
        const int stage = i % C::STAGES;
        if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], (i / C::STAGES) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 46))) break;
        uint4* s = reinterpret_cast<uint4*>(smem + C::OFF_SCALES + stage * C::S_BYTES + F::PIECES * C::PIECE);
#pragma unroll
        for (int p = 0; p < F::PIECES; p++) {
          const uint4 v = s[p * 32 + lane];
          s[p * 32 + lane] = sub == 1 ? make_uint4(v.y, v.z, v.w, v.x) : sub == 2 ? make_uint4(v.z, v.w, v.x, v.y) : make_uint4(v.w, v.x, v.y, v.z);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&turned[stage]);
      }
    }
    // the accumulator into the ring, transposed (every load has been consumed by then): rows of C of 128 fp32 columns
    const bool ok = mbar_wait(done, 0, abort_flag, args.status, ST_GEMM_TIMEOUT, 44);
    const int q = warp & 3, half = (warp - 2) >> 2;          // (of 320 threads: two warps for 32 lanes, 16 columns in turn)
    float* col = reinterpret_cast<float*>(smem) + q * 32 + lane;
    if (__all_sync(0xffffffffu, ok)) {
      tc_fence_after();
#pragma unroll
      for (int c = 16 * half; c < BN; c += 16 * ((C::THREADS - 64) / 128)) {
        if (c >= args.M - r0) break;                         // (rows of C that are not there)
        uint32_t r[16];
        if (k1 > k0) {
          tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + c, r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 16; j++) r[j] = 0u;
        }
#pragma unroll
        for (int j = 0; j < 16; j++) col[(c + j) * 128] = __uint_as_float(r[j]);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM);
  }
  if (S > 1) cluster_sync_all();
  // groups of four columns of a row, dealt to the CTAs of the cluster in turn: sum over the CTAs in order, epilogue, store.  A thread stays
  // in its columns; U groups are in flight.
  constexpr int U = BN >= 64 ? 4 : 2;
  const int groups = min(BN, args.M - r0) * 32, first = threadIdx.x * S + rank, stride = C::THREADS * S;
  const int c = c0 + (first & 31) * 4, size = args.out == OUT_F32 ? 4 : 2;
  static_assert(C::THREADS % 32 == 0, "a thread stays in its columns");
  const bool vector = c + 4 <= args.N && (((uintptr_t)args.C | (uintptr_t)(args.ldc * size)) & (4 * size - 1)) == 0;
  float bias[4];
#pragma unroll
  for (int j = 0; j < 4; j++) bias[j] = bias_at(args, c + j);
  for (int i0 = first; i0 < groups; i0 += U * stride) {
    float4 v[U];
#pragma unroll
    for (int k = 0; k < U; k++) {
      const int i = i0 + k * stride;
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i >= groups) continue;
      if (S == 1) {
        v[k] = *reinterpret_cast<const float4*>(smem + i * 16);
      } else {
        const uint32_t at = smem_u32(smem) + i * 16;
#pragma unroll 4
        for (int p = 0; p < S; p++) {
          uint32_t remote;
          float4 u;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(p));
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(u.x), "=f"(u.y), "=f"(u.z), "=f"(u.w) : "r"(remote) : "memory");
          v[k].x += u.x; v[k].y += u.y; v[k].z += u.z; v[k].w += u.w;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < U; k++) {
      const int i = i0 + k * stride;
      if (i >= groups || c >= args.N) break;
      float y[4] = {v[k].x + bias[0], v[k].y + bias[1], v[k].z + bias[2], v[k].w + bias[3]};
      activate_two(y[0], y[1], args.act);
      activate_two(y[2], y[3], args.act);
      const long long to = (long long)(r0 + (i >> 5)) * args.ldc + c;
      if (vector) {
        if (args.out == OUT_F32) *reinterpret_cast<float4*>((float*)args.C + to) = make_float4(y[0], y[1], y[2], y[3]);
        else *reinterpret_cast<uint2*>((uint16_t*)args.C + to) = make_uint2(pack_out(args, y[0], y[1]), pack_out(args, y[2], y[3]));
      } else {
        for (int j = 0; j < 4 && c + j < args.N; j++) store_out(args, to + j, y[j]);
      }
    }
  }
  if (S > 1) cluster_sync_all();   // nobody leaves while another may still read its shared memory
}

// ---------------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------------
struct Plan {
  int pair, bn, splits, steps, steps_per;
};

thread_local int g_kind = 0, g_rows = 0, g_splits = 0;       // gb_mx_tune

// Microseconds that a product takes in either kernel, by what was measured of them.  Pairs: a step takes 0.3 (an SM's 32 KB), 4 go by for the
// launch, the first loads and the last results, 1.5 for a tile's own; two slices exchange their sums, and 33 clusters of two pairs fit at a time.
// Clusters: a step takes 0.33 (the 1.6 us of a load over the 100 KB that a CTA has in flight) and more where CTAs share an SM, a launch 2.45, each
// of a tile's rows 0.026, the turning of scales 0.25; from two CTAs on the exchange, the longer the more CTAs share the way of its values;
// CTAs beyond those that fit at a time three quarters more.  What it chooses takes 1.2 % longer than the best (geometric mean over 116 sizes, 757 runs).  us, measured | so, MXFP8: 1 x 2048 x 8192 in clusters of 1, 2, 4, 8 20.6, 12.4, 7.9, 6.2 |
// 23.6, 13.9, 9.0, 7.0; 128 x 2304 x 768 in tiles of 32, 64, 128 rows 5.6, 6.1, 7.7 | 5.5, 6.3, 7.8, as pairs 7.0 | 7.3; 512 x 2048 x 8192: 64 rows in
// clusters of 2 18.4 | 19.4, 128 in 4 21.0 | 20.2, pairs whole 24.1 | 24.7, in two slices 17.0 | 17.4; 2304 x 768 x 16384 43.8 | 43.9, 28.6 | 28.1.
double pair_us(long long tiles, int steps, int splits) {
  const long long at_once = splits == 1 ? 74 : 33, waves = (tiles + at_once - 1) / at_once;
  return 4.0 + waves * ((steps + splits - 1) / splits * 0.3 + 1.5 + (splits > 1 ? 0.7 + 0.1 * (tiles < 33 ? tiles : 33) : 0.0));
}
double cluster_us(long long M, int bn, long long tiles, int steps, int splits) {
  const double ctas = (double)tiles * splits, rows = M < bn ? M : bn, load = ctas > 148 ? ctas / 148 - 1.0 : 0.0;      // (two CTAs on an SM)
  const double once = 2.45 + 0.026 * rows + 0.65 * load + (steps + splits - 1) / splits * 0.33 * (1.0 + 0.19 * load) + (M > bn && bn < 128 ? 0.25 : 0.0) +
                      (splits > 1 ? 0.56 + 0.16 * splits + 0.0033 * splits * rows * (ctas > 64 ? ctas / 64 : 1.0) : 0.0);
  return once * (ctas > 296 ? 1.0 + 0.75 * (ceil(ctas / 296) - 1.0) : 1.0);
}

struct Choice {
  int rows, splits;
  double us;
};
// Tiles of 16 rows for as many at most (scales of 32 rows stay together), else of 32, 64 or 128.
Choice best_clusters(long long M, long long N, int steps) {
  Choice c{0, 0, 1e300};
  for (int bn = M <= 16 ? 16 : 32; bn <= (M <= 16 ? 16 : 128); bn *= 2) {
    if (g_rows && M > 16 && bn != g_rows) continue;
    const long long tiles = ((M + bn - 1) / bn) * ((N + 127) / 128);
    for (int s = g_splits ? g_splits : 1; s <= 8; s *= 2) {
      if (g_splits ? s != g_splits : s > 1 && (s > steps || tiles * s > 296)) break;
      const double us = cluster_us(M, bn, tiles, steps, s);
      if (us < c.us) c = {bn, s, us};
    }
  }
  return c;
}
Choice best_pairs(long long M, long long N, int steps) {
  const long long tiles = ((M + 255) / 256) * ((N + 255) / 256);
  Choice c{256, 1, pair_us(tiles, steps, 1)};
  const double two = pair_us(tiles, steps, 2);
  if (steps > 1 && tiles < 0xffffff && (g_splits ? g_splits == 2 : two < c.us)) c = {256, 2, two};
  return c;
}

Plan plan_of(long long M, long long N, long long K, int fmt) {
  Plan p{};
  p.steps = (int)((K + (fmt == FP8 ? 127 : 255)) / (fmt == FP8 ? 128 : 256));
  const Choice pairs = best_pairs(M, N, p.steps), clusters = best_clusters(M, N, p.steps);
  p.pair = g_kind ? g_kind == 1 : pairs.us < clusters.us;
  p.bn = p.pair ? 256 : clusters.rows;
  p.splits = p.pair ? pairs.splits : clusters.splits;
  p.steps_per = (p.steps + p.splits - 1) / p.splits;
  return p;
}

// Opts a kernel into its shared memory once per device.
template <typename K>
int allow_shared(K kern, int bytes, std::atomic<uint32_t>& done) {
  int dev = 0;
  GB_CUDA_OK(cudaGetDevice(&dev));
  if (dev < 32 && (done.load() >> dev & 1u)) return gbh::E_OK;
  GB_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 32) done.fetch_or(1u << dev);
  return gbh::E_OK;
}

bool bad_operand(const void* p) { return p == nullptr || ((uintptr_t)p & 15) != 0; }

struct Maps {
  CUtensorMap a, b, sa, sb;
};

int map_codes(CUtensorMap* m, const void* p, long long rows, long long rb, int box_rows) {
  const uint64_t dims[3] = {(uint64_t)rb, (uint64_t)rows, 1}, strides[2] = {(uint64_t)rb, (uint64_t)(rb * rows)};
  const uint32_t box[3] = {128, (uint32_t)box_rows, 1};
  return gbh::encode_tmap(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
// Scale pieces as 128 words: `pieces` of a step, of `rows_of` rows of pieces.
int map_scales(CUtensorMap* m, const void* p, long long rows, int P, int pieces, int rows_of) {
  const uint64_t dims[3] = {128, (uint64_t)P, (uint64_t)((rows + 127) / 128)}, strides[2] = {512, (uint64_t)P * 512};
  const uint32_t box[3] = {128, (uint32_t)pieces, (uint32_t)rows_of};
  return gbh::encode_tmap(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <int FMT, bool VECTORS, bool SLICED>
int launch_pair(const Maps& tm, const MxArgs& args, cudaStream_t st) {
  using C = PairCfg<FMT>;
  static std::atomic<uint32_t> done{0};
  if (int rc = allow_shared(mx_pair_kernel<FMT, VECTORS, SLICED>, C::BYTES, done)) return rc;
  const long long tiles = (long long)args.num_m * args.num_n, clusters = SLICED || tiles < 74 ? tiles : 74;
  const unsigned size = SLICED ? 4 : 2;
  GB_CUDA_OK(gbh::launch(mx_pair_kernel<FMT, VECTORS, SLICED>, dim3((unsigned)clusters * size), dim3(C::THREADS), C::BYTES, st, size, tm.a, tm.b, tm.sa, tm.sb, args));
  return gbh::E_OK;
}
template <int FMT, int BN, typename X = void>
int launch_cluster(const Maps& tm, const void* sa, const void* sb, const MxArgs& args, cudaStream_t st, const RowsArgs& x = RowsArgs{}) {
  using C = ClusterCfg<FMT, BN>;
  static std::atomic<uint32_t> done{0};
  if (int rc = allow_shared(mx_cluster_kernel<FMT, BN, X>, C::BYTES, done)) return rc;
  GB_CUDA_OK(gbh::launch(mx_cluster_kernel<FMT, BN, X>, dim3(args.num_m * args.num_n * args.splits), dim3(C::THREADS), C::BYTES, st, args.splits, tm.a, tm.b,
                         (const uint8_t*)sa, (const uint8_t*)sb, x, args));
  return gbh::E_OK;
}

}  // namespace

// The kernel of products from this thread: kind 0 by size, 1 pairs, 2 clusters, 32, 64 or 128 clusters with tiles of so many rows (above 16 rows
// of C); splits 0 by size, else that many slices of K: up to two of pairs, eight of clusters.  (Of a single step of K a pair takes no half.)
GB_EXPORT int gb_mx_tune(int kind, int splits) {
  const int most = kind == 0 ? 0 : kind == 1 ? 2 : 8;
  if (((kind < 0 || kind > 2) && kind != 32 && kind != 64 && kind != 128) || splits < 0 || splits > most) {
    gbh::set_error("gb_mx_tune: kind %d, splits %d", kind, splits);
    return gbh::E_BAD_ARG;
  }
  g_kind = kind > 2 ? 2 : kind;
  g_rows = kind > 2 ? kind : 0;
  g_splits = splits;
  return gbh::E_OK;
}

static bool bad_extents(const char* what, long long M, long long N, long long K, int fmt) {
  if (M > 0 && N > 0 && K > 0 && M <= 0x7fffffffLL && N <= 0x7fffffffLL && K <= (1LL << 30) && (fmt == FP8 || fmt == FP4)) return false;
  gbh::set_error("%s: bad extents %lld x %lld x %lld, format %d", what, M, N, K, fmt);
  return true;
}

// How a product runs (for tests): 1 pairs, 2 clusters; rows of a tile; slices of K.
GB_EXPORT int gb_mx_plan(long long M, long long N, long long K, int fmt, long long* out3) {
  if (bad_extents("gb_mx_plan", M, N, K, fmt)) return gbh::E_BAD_ARG;
  const Plan p = plan_of(M, N, K, fmt);
  out3[0] = p.pair ? 1 : 2;
  out3[1] = p.bn;
  out3[2] = p.splits;
  return gbh::E_OK;
}

// C (M x N, rows ldc apart) = act(A B^T + bias).  out: DT_BF16, DT_F16 or DT_F32; bias in C's type or fp32 (bias_f32), or null.
GB_EXPORT int gb_mx_matmul(int fmt, const void* a, const void* sa, const void* b, const void* sb, void* c, long long ldc, const void* bias, int bias_f32, long long M,
                           long long N, long long K, int out, int act, void* stream) {
  if (bad_extents("gb_mx_matmul", M, N, K, fmt)) return gbh::E_BAD_ARG;
  if (out < 0 || out > 2 || act < 0 || act > 3 || ldc < N) {
    gbh::set_error("gb_mx_matmul: bad type %d, activation %d or row pitch %lld", out, act, ldc);
    return gbh::E_BAD_ARG;
  }
  if (bad_operand(a) || bad_operand(sa) || bad_operand(b) || bad_operand(sb) || c == nullptr) {
    gbh::set_error("gb_mx_matmul: codes and scales on 16-byte boundaries and a result are needed");
    return gbh::E_BAD_ARG;
  }
  const Plan p = plan_of(M, N, K, fmt);
  const int P = pieces((int)K, fmt), RB = row_bytes((int)K, fmt), per = fmt == FP8 ? 1 : 2;
  MxArgs args{};
  args.num_m = (int)((M + p.bn - 1) / p.bn);
  args.num_n = (int)(p.pair ? (N + 255) / 256 : (N + 127) / 128);
  if ((long long)args.num_m * args.num_n * p.splits * (p.pair ? 2 : 1) > 0x7fffffffLL) {
    gbh::set_error("gb_mx_matmul: %lld x %lld has too many tiles", M, N);
    return gbh::E_TOO_LARGE;
  }
  args.M = (int)M; args.N = (int)N; args.steps = p.steps;
  args.splits = p.splits; args.steps_per = p.steps_per;
  args.C = c; args.ldc = ldc; args.bias = bias; args.bias_f32 = bias_f32 || out == OUT_F32; args.act = act; args.out = out;
  args.status = gbh::status_ptr();
  cudaStream_t st = (cudaStream_t)stream;
  Maps tm;
  memset(&tm, 0, sizeof(tm));
  if (p.pair) {
    int rc = 0;
    const int size = out == OUT_F32 ? 4 : 2;
    const auto whole = [&](int bytes) { return (uintptr_t)c % bytes == 0 && ldc * size % bytes == 0 && N * size % bytes == 0; };
    args.vectors = whole(32) ? 32 : whole(16) ? 16 : 0;
    if (!rc) rc = map_codes(&tm.a, a, M, RB, 128);
    if (!rc) rc = map_codes(&tm.b, b, N, RB, 128);
    if (!rc) rc = map_scales(&tm.sa, sa, M, P, per, 1);
    if (!rc) rc = map_scales(&tm.sb, sb, N, P, per, 2);
    if (rc) return rc;
    if (p.splits > 1) {
      if (args.vectors) return fmt == FP8 ? launch_pair<FP8, true, true>(tm, args, st) : launch_pair<FP4, true, true>(tm, args, st);
      return fmt == FP8 ? launch_pair<FP8, false, true>(tm, args, st) : launch_pair<FP4, false, true>(tm, args, st);
    }
    if (args.vectors) return fmt == FP8 ? launch_pair<FP8, true, false>(tm, args, st) : launch_pair<FP4, true, false>(tm, args, st);
    return fmt == FP8 ? launch_pair<FP8, false, false>(tm, args, st) : launch_pair<FP4, false, false>(tm, args, st);
  }
  if (int rc = map_codes(&tm.a, b, N, RB, 128)) return rc;
  if (int rc = map_codes(&tm.b, a, M, RB, p.bn)) return rc;
  switch (p.bn) {
    case 16: return fmt == FP8 ? launch_cluster<FP8, 16>(tm, sb, sa, args, st) : launch_cluster<FP4, 16>(tm, sb, sa, args, st);
    case 32: return fmt == FP8 ? launch_cluster<FP8, 32>(tm, sb, sa, args, st) : launch_cluster<FP4, 32>(tm, sb, sa, args, st);
    case 64: return fmt == FP8 ? launch_cluster<FP8, 64>(tm, sb, sa, args, st) : launch_cluster<FP4, 64>(tm, sb, sa, args, st);
    default: return fmt == FP8 ? launch_cluster<FP8, 128>(tm, sb, sa, args, st) : launch_cluster<FP4, 128>(tm, sb, sa, args, st);
  }
}

// The same for up to 16 rows of x as they are (bf16, fp16 or fp32, K elements, ld apart), quantised within the product's kernel.
GB_EXPORT int gb_mx_matmul_rows(int dtype, int fmt, const void* x, long long ld, const void* b, const void* sb, void* c, long long ldc, const void* bias, int bias_f32,
                                long long M, long long N, long long K, int out, int act, void* stream) {
  if (bad_extents("gb_mx_matmul_rows", M, N, K, fmt)) return gbh::E_BAD_ARG;
  if (M > 16 || dtype < 0 || dtype > 2 || out < 0 || out > 2 || act < 0 || act > 3 || ldc < N || ld < 0) {
    gbh::set_error("gb_mx_matmul_rows: %lld rows (16 at most), types %d and %d, activation %d, row pitches %lld and %lld", M, dtype, out, act, ld, ldc);
    return gbh::E_BAD_ARG;
  }
  if (x == nullptr || bad_operand(b) || bad_operand(sb) || c == nullptr) {
    gbh::set_error("gb_mx_matmul_rows: rows, codes and scales on 16-byte boundaries and a result are needed");
    return gbh::E_BAD_ARG;
  }
  MxArgs args{};
  args.M = (int)M; args.N = (int)N;
  args.steps = (int)((K + (fmt == FP8 ? 127 : 255)) / (fmt == FP8 ? 128 : 256));
  args.num_m = 1;
  args.num_n = (int)((N + 127) / 128);
  args.splits = best_clusters(M, N, args.steps).splits;
  args.steps_per = (args.steps + args.splits - 1) / args.splits;
  args.C = c; args.ldc = ldc; args.bias = bias; args.bias_f32 = bias_f32 || out == OUT_F32; args.act = act; args.out = out;
  args.status = gbh::status_ptr();
  const int size = dtype == 2 ? 4 : 2;
  RowsArgs rows{x, ld, (int)K, ((uintptr_t)x & 15) == 0 && ld * size % 16 == 0 && K % 8 == 0, {reinterpret_cast<uintptr_t>(x), reinterpret_cast<uintptr_t>(x) + (uintptr_t)(((M - 1) * ld + K) * size)}};
  Maps tm;
  memset(&tm, 0, sizeof(tm));
  if (int rc = map_codes(&tm.a, b, N, row_bytes((int)K, fmt), 128)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == 0) return fmt == FP8 ? launch_cluster<FP8, 16, __nv_bfloat16>(tm, sb, nullptr, args, st, rows) : launch_cluster<FP4, 16, __nv_bfloat16>(tm, sb, nullptr, args, st, rows);
  if (dtype == 1) return fmt == FP8 ? launch_cluster<FP8, 16, __half>(tm, sb, nullptr, args, st, rows) : launch_cluster<FP4, 16, __half>(tm, sb, nullptr, args, st, rows);
  return fmt == FP8 ? launch_cluster<FP8, 16, float>(tm, sb, nullptr, args, st, rows) : launch_cluster<FP4, 16, float>(tm, sb, nullptr, args, st, rows);
}
