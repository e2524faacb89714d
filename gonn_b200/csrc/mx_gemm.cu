// Products of microscaled matrices (formats: mx.cuh):  C = act(A B^T + bias),  A: M x K, B: N x K, both quantised along K.
//
// tcgen05.mma with block scales: kind::mxf8f6f4 for MXFP8 (32 of K an instruction), kind::mxf4 for MXFP4 (64), fp32 accumulators in
// TMEM.  A step of the main loop is 128 bytes of every row in either format (128 or 256 of K, four instructions); its
// codes arrive by TMA with a 128-byte swizzle, its scales as the 512-byte pieces in which they are kept, and the issuing thread copies
// those from shared memory into TMEM (tcgen05.cp) before the instructions that read them.  Two sets of scale columns take
// turns; a set is written again once the step that read it has ended.
//
// Two kernels.  Pairs: a cluster of two CTAs per 256 x 256 tile (cta_group::2), persistent, for products with tiles enough to fill
// the SMs.  Clusters: one tile of 128 columns of C (rows of B: the 128 rows of an instruction) by 16 to 128 rows of C per cluster of up to
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
  int splits, steps_per;   // slice s takes steps [s * steps_per, (s + 1) * steps_per)
  void* C;                 // rows ldc elements apart
  long long ldc;
  const void* bias;        // N values in C's type, or fp32; null: none
  int bias_f32, act, out, tma_out;
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

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case ACT_RELU: return fmaxf(v, 0.f);
    case ACT_GELU_TANH: return gelu_tanh_f(v);
    case ACT_GELU_ERF: return gelu_erf_f(v);
    default: return v;
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
// Pairs.  Each CTA stages its 128 rows of A with their scales and 128 of the tile's 256 rows of B, and the scales of all 256 (its
// half of the accumulator has all columns); CTA 0 issues.  Two accumulators of 256 columns and the scales do not fit into TMEM's
// 512, so the two overlap in columns 192 to 255: the epilogue drains those first, and then the next tile starts.
// ---------------------------------------------------------------------------------------------------------------------------
template <int FMT>
struct PairCfg {
  static constexpr int STAGES = 5, EW = 8, THREADS = 64 + 32 * EW;
  static constexpr int A_BYTES = 128 * 128, B_BYTES = 128 * 128, TILE_BYTES = A_BYTES + B_BYTES;
  static constexpr int PIECE = 512, S_BYTES = 3 * Fmt<FMT>::PIECES * PIECE;      // A's row of pieces, B's two
  static constexpr int OFF_SCALES = STAGES * TILE_BYTES;
  static constexpr int OFF_OUT = OFF_SCALES + STAGES * S_BYTES;
  static constexpr int OUT_BUF = 4096;                       // of an epilogue warp: 32 x 32 values, two buffers of 16-bit ones
  static constexpr int OFF_BIAS = OFF_OUT + EW * OUT_BUF;
  static constexpr int OFF_BARS = OFF_BIAS + EW * 128;
  static constexpr int BYTES = OFF_BARS + 256;
  static constexpr int ACC1 = 192, SCALES = 448;             // TMEM columns
  static_assert(BYTES <= 232448 && OFF_OUT % 512 == 0, "shared memory");
  static_assert(SCALES + 32 + 12 * Fmt<FMT>::PIECES <= 512, "TMEM");
};

__device__ __forceinline__ void put_shared(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// 32 x 32 results of a warp (a lane has a row) into C: by way of `buf` and TMA, or, where C has no tensor map, row by row.
__device__ __forceinline__ void store_chunk(const MxArgs& a, const CUtensorMap* tmC, uint8_t* buf, int flip, int slice, int row0, int col0, const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  if (a.tma_out) {
    // 64-byte rows, swizzled in 16-byte pieces
    const uint32_t swz = (lane >> 1) & 3, row = smem_u32(buf) + lane * 64;
    if (a.out == OUT_F32) {
      if (lane == 0) tma_store_wait_read<0>();
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int j = 0; j < 4; j++)
          put_shared(row + h * 2048 + ((j ^ swz) << 4), make_uint4(__float_as_uint(v[h * 16 + j * 4]), __float_as_uint(v[h * 16 + j * 4 + 1]),
                                                                   __float_as_uint(v[h * 16 + j * 4 + 2]), __float_as_uint(v[h * 16 + j * 4 + 3])));
    } else {
      if (lane == 0) tma_store_wait_read<1>();               // the store before last has left this buffer
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; j++)
        put_shared(row + flip * 2048 + ((j ^ swz) << 4), make_uint4(pack_out(a, v[j * 8], v[j * 8 + 1]), pack_out(a, v[j * 8 + 2], v[j * 8 + 3]),
                                                                    pack_out(a, v[j * 8 + 4], v[j * 8 + 5]), pack_out(a, v[j * 8 + 6], v[j * 8 + 7])));
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (a.out == OUT_F32) {
        tma_store_3d(tmC, buf, col0, row0, slice);
        if (col0 + 16 < a.N) tma_store_3d(tmC, buf + 2048, col0 + 16, row0, slice);
      } else {
        tma_store_3d(tmC, buf + flip * 2048, col0, row0, slice);
      }
      tma_store_commit();
    }
    return;
  }
  float* f = reinterpret_cast<float*>(buf);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 32; j++) f[lane * 32 + (j ^ lane)] = v[j];
  __syncwarp();
  const int rows = min(32, a.M - row0);
  if (col0 + lane < a.N)
    for (int r = 0; r < rows; r++) store_out(a, (row0 + r) * a.ldc + col0 + lane, f[r * 32 + (lane ^ r)]);
}

template <int FMT>
__global__ void __launch_bounds__(PairCfg<FMT>::THREADS, 1)
mx_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSA,
               const __grid_constant__ CUtensorMap tmSB, const __grid_constant__ CUtensorMap tmC, const MxArgs args) {
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
  uint32_t* slot = (uint32_t*)(drained + 1);
  volatile int* abort_flag = (volatile int*)(slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = args.num_m * args.num_n, units = tiles * args.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&ready[0], 1);
    mbar_init(&ready[1], 1);
    mbar_init(drained, 2 * C::EW);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSB);
    if (args.tma_out) tma_prefetch_desc(&tmC);
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
      for (int u = pair; u < units && ok; u += pairs) {
        const int slice = u / tiles;
        int mb, nb;
        tile_at(u - slice * tiles, args.num_m, args.num_n, mb, nb);
        const int m0 = mb * 256 + (int)cta * 128, n0 = nb * 256 + (int)cta * 128;
        const int k1 = min(args.steps, (slice + 1) * args.steps_per);
        for (int k = slice * args.steps_per; k < k1; k++) {
          ok = mbar_wait(&empty[stage], phase ^ 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 31);
          if (!ok) break;
          uint8_t* sa = smem + stage * C::TILE_BYTES;
          uint8_t* ss = smem + C::OFF_SCALES + stage * C::S_BYTES;
          const uint32_t fb = smem_u32(&full[stage]) & ~kPeerBit;        // what lands in either CTA counts on the leader's barrier
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
      for (int u = pair; u < units && ok; u += pairs, local++) {
        if (local > 0) {
          ok = mbar_wait(drained, (local - 1) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 32);
          if (!ok) break;
          tc_fence_after();
        }
        const uint32_t acc = tmem + (local & 1) * C::ACC1;
        const int slice = u / tiles, k0 = slice * args.steps_per, k1 = min(args.steps, k0 + args.steps_per);
        for (int k = k0; k < k1; k++, n++) {
          const int stage = n % C::STAGES;
          ok = mbar_wait(&full[stage], (n / C::STAGES) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 33);
          // the step that read this set of scale columns has ended
          if (ok && n >= 2) ok = mbar_wait(&empty[(n - 2) % C::STAGES], ((n - 2) / C::STAGES) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 34);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * C::TILE_BYTES), sb = sa + C::A_BYTES;
          const uint32_t ss = smem_u32(smem + C::OFF_SCALES + stage * C::S_BYTES);
          const uint32_t ta = tmem + C::SCALES + (n & 1) * 32, tb = ta + 4 * F::PIECES;
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
          tc_commit_2sm(eb | kPeerBit);
          if (k == k1 - 1) {
            const uint32_t rb = smem_u32(&ready[local & 1]);
            tc_commit_2sm(rb);
            tc_commit_2sm(rb | kPeerBit);
          }
        }
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint8_t* buf = smem + C::OFF_OUT + (warp - 2) * C::OUT_BUF;
    float* sbias = reinterpret_cast<float*>(smem + C::OFF_BIAS) + (warp - 2) * 32;
    int local = 0, flip = 0;
    for (int u = pair; u < units; u += pairs, local++) {
      const int slice = u / tiles, which = local & 1;
      int mb, nb;
      tile_at(u - slice * tiles, args.num_m, args.num_n, mb, nb);
      const int row0 = mb * 256 + (int)cta * 128 + q * 32;
      // four chunks of 32 columns for a warp, the one that lies in the other accumulator's columns first
      int cols[4];
      float bl[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int c = i == 0 ? (which ? 0 : 6) + half : (which ? 2 : 0) + half * 3 + i - 1;
        cols[i] = c * 32;
        bl[i] = bias_at(args, nb * 256 + cols[i] + lane);
      }
      if (!mbar_wait(&ready[which], (local >> 1) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 35)) break;
      tc_fence_after();
      const uint32_t acc = tmem + which * C::ACC1 + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
      for (int i = 0; i < 4; i++) {
        uint32_t r[32];
        tmem_ld32(acc + cols[i], r);
        tmem_ld_wait();
        if (i == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(smem_u32(drained) & ~kPeerBit);
        }
        const int col0 = nb * 256 + cols[i];
        if (row0 >= args.M || col0 >= args.N) continue;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; j++) v[j] = __uint_as_float(r[j]);
        if (args.bias != nullptr) {
          __syncwarp();
          sbias[lane] = i == 0 ? bl[0] : i == 1 ? bl[1] : i == 2 ? bl[2] : bl[3];
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 b = *reinterpret_cast<const float4*>(sbias + j);
            v[j] += b.x; v[j + 1] += b.y; v[j + 2] += b.z; v[j + 3] += b.w;
          }
        }
        if (args.act != ACT_NONE) {
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = activate(v[j], args.act);
        }
        store_chunk(args, &tmC, buf, flip, slice, row0, col0, v);
        flip ^= 1;
      }
    }
    if (args.tma_out && lane == 0) tma_store_wait<0>();
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
// than they need.  A tile's rows of A start at a multiple of 128, as the scale pieces do.
// ---------------------------------------------------------------------------------------------------------------------------
template <int FMT, int BN>
struct ClusterCfg {
  static constexpr int STAGES = BN <= 32 ? 8 : 6, THREADS = 192;
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BN * 128, TILE_BYTES = A_BYTES + B_BYTES;
  static constexpr int PIECE = 512, S_BYTES = 2 * Fmt<FMT>::PIECES * PIECE;
  static constexpr int OFF_SCALES = STAGES * TILE_BYTES;
  static constexpr int OFF_BARS = OFF_SCALES + STAGES * S_BYTES;
  static constexpr int BYTES = OFF_BARS + 256;
  static constexpr int TMEM = BN <= 32 ? 64 : 2 * BN;        // the accumulator, then two sets of 8 x PIECES scale columns
  static_assert(BYTES <= 232448 && BN * 512 <= OFF_SCALES, "shared memory (the partial tile reuses the ring)");
  static_assert(BN + 16 + 8 * Fmt<FMT>::PIECES <= TMEM, "TMEM");
};

template <int FMT, int BN>
__global__ void __launch_bounds__(ClusterCfg<FMT, BN>::THREADS, 1)
mx_cluster_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSA,
                  const __grid_constant__ CUtensorMap tmSB, const MxArgs args) {
  // "A" of the instruction: args' B (columns of C); its "B": args' A (rows of C)
  using C = ClusterCfg<FMT, BN>;
  using F = Fmt<FMT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {      // the same in every CTA of the launch
    if (threadIdx.x == 0) set_status(args.status, ST_BAD_INDEX, 1024);
    return;
  }
  uint64_t* full = (uint64_t*)(smem + C::OFF_BARS);
  uint64_t* empty = full + C::STAGES;
  uint64_t* done = empty + C::STAGES;
  uint32_t* slot = (uint32_t*)(done + 1);
  volatile int* abort_flag = (volatile int*)(slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = args.splits, tile = blockIdx.x / S, rank = blockIdx.x - tile * S;
  const int c0 = (tile % args.num_n) * 128, r0 = (tile / args.num_n) * BN;       // columns and rows of C
  const int k0 = rank * args.steps_per, k1 = min(args.steps, k0 + args.steps_per);
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(done, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSB);
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
        mbar_expect_tx(&full[stage], C::TILE_BYTES + C::S_BYTES);
        tma_load_3d(sa, &tmA, &full[stage], k * 128, c0, 0);
        tma_load_3d(ss, &tmSA, &full[stage], 0, k * F::PIECES, c0 >> 7);
        tma_load_3d(sa + C::A_BYTES, &tmB, &full[stage], k * 128, r0, 0);
        tma_load_3d(ss + F::PIECES * C::PIECE, &tmSB, &full[stage], 0, k * F::PIECES, r0 >> 7);
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
        // the step that read this set of scale columns has ended
        if (n >= 2 && !mbar_wait(&empty[(n - 2) % C::STAGES], ((n - 2) / C::STAGES) & 1, abort_flag, args.status, ST_GEMM_TIMEOUT, 43)) break;
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + stage * C::TILE_BYTES), sb = sa + C::A_BYTES;
        const uint32_t ss = smem_u32(smem + C::OFF_SCALES + stage * C::S_BYTES);
        const uint32_t ta = tmem + BN + (n & 1) * (C::TMEM - BN) / 2, tb = ta + 4 * F::PIECES;
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
    // the accumulator into the ring, transposed (every load has been consumed by then): rows of C of 128 fp32 columns
    const bool ok = mbar_wait(done, 0, abort_flag, args.status, ST_GEMM_TIMEOUT, 44);
    const int q = warp & 3;
    float* col = reinterpret_cast<float*>(smem) + q * 32 + lane;
    if (__all_sync(0xffffffffu, ok)) {
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < BN; c += 16) {
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
  // groups of four columns of a row, dealt to the CTAs of the cluster in turn: sum over the CTAs in order, epilogue, store
  const int groups = min(BN, args.M - r0) * 32;
  for (int i = threadIdx.x * S + rank; i < groups; i += C::THREADS * S) {
    const int r = i >> 5, c = c0 + (i & 31) * 4;
    const uint32_t at = smem_u32(smem) + i * 16;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (S == 1) {
      const float4 u = *reinterpret_cast<const float4*>(smem + i * 16);
      v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    } else {
#pragma unroll 4
      for (int p = 0; p < S; p++) {
        uint32_t remote;
        float4 u;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(p));
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(u.x), "=f"(u.y), "=f"(u.z), "=f"(u.w) : "r"(remote) : "memory");
        v[0] += u.x; v[1] += u.y; v[2] += u.z; v[3] += u.w;
      }
    }
    if (c >= args.N) continue;
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = activate(v[j] + bias_at(args, c + j), args.act);
    const long long to = (r0 + r) * args.ldc + c;
    const int size = args.out == OUT_F32 ? 4 : 2;
    if (c + 4 <= args.N && (((uintptr_t)args.C + to * size) & (4 * size - 1)) == 0) {
      if (args.out == OUT_F32) *reinterpret_cast<float4*>((float*)args.C + to) = make_float4(v[0], v[1], v[2], v[3]);
      else *reinterpret_cast<uint2*>((uint16_t*)args.C + to) = make_uint2(pack_out(args, v[0], v[1]), pack_out(args, v[2], v[3]));
    } else {
      for (int j = 0; j < 4 && c + j < args.N; j++) store_out(args, to + j, v[j]);
    }
  }
  if (S > 1) cluster_sync_all();   // nobody leaves while another may still read its shared memory
}

// Slices of a product cut along K, summed in their order: C = act(sum + bias).
__global__ void __launch_bounds__(256) mx_finish_kernel(const float* __restrict__ part, const MxArgs a, int slices) {
  pdl_trigger();
  pdl_wait();
  const long long total = (long long)a.M * a.N, stride = (long long)gridDim.x * blockDim.x * 4;
  for (long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 4; i < total; i += stride) {      // (N is a multiple of 4)
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = 0; p < slices; p++) {
      const float4 u = __ldcs(reinterpret_cast<const float4*>(part + p * total + i));
      s.x += u.x; s.y += u.y; s.z += u.z; s.w += u.w;
    }
    const long long row = i / a.N;
    const int c = (int)(i - row * a.N);
    const float v[4] = {s.x, s.y, s.z, s.w};
    for (int j = 0; j < 4; j++) store_out(a, row * a.ldc + c + j, activate(v[j] + bias_at(a, c + j), a.act));
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------------
struct Plan {
  int pair, bn, splits, steps, steps_per;
  long long workspace;     // bytes: fp32 slices of a cut product of the pair kernel
};

Plan plan_of(long long M, long long N, long long K, int fmt) {
  Plan p{};
  p.steps = (int)((K + (fmt == FP8 ? 127 : 255)) / (fmt == FP8 ? 128 : 256));
  const long long tiles2 = ((M + 255) / 256) * ((N + 255) / 256);
  p.splits = 1;
  if (M > 128 && tiles2 >= 37) {
    p.pair = 1;
    p.steps_per = p.steps;
    return p;
  }
  p.bn = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  const long long tiles = ((M + p.bn - 1) / p.bn) * ((N + 127) / 128);
  while (p.splits < 8 && tiles * p.splits * 2 <= 148 + 18 && p.splits * 2 <= p.steps) p.splits *= 2;
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

struct Maps {
  CUtensorMap a, b, sa, sb, c;
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

template <int FMT>
int launch_pair(const Maps& tm, const MxArgs& args, cudaStream_t st) {
  using C = PairCfg<FMT>;
  static std::atomic<uint32_t> done{0};
  if (int rc = allow_shared(mx_pair_kernel<FMT>, C::BYTES, done)) return rc;
  const long long units = (long long)args.num_m * args.num_n * args.splits;
  const int pairs = units < 74 ? (int)units : 74;
  GB_CUDA_OK(gbh::launch(mx_pair_kernel<FMT>, dim3(2 * pairs), dim3(C::THREADS), C::BYTES, st, 2, tm.a, tm.b, tm.sa, tm.sb, tm.c, args));
  return gbh::E_OK;
}
template <int FMT, int BN>
int launch_cluster(const Maps& tm, const MxArgs& args, cudaStream_t st) {
  using C = ClusterCfg<FMT, BN>;
  static std::atomic<uint32_t> done{0};
  if (int rc = allow_shared(mx_cluster_kernel<FMT, BN>, C::BYTES, done)) return rc;
  GB_CUDA_OK(gbh::launch(mx_cluster_kernel<FMT, BN>, dim3(args.num_m * args.num_n * args.splits), dim3(C::THREADS), C::BYTES, st, args.splits, tm.a, tm.b, tm.sa, tm.sb, args));
  return gbh::E_OK;
}

}  // namespace

// How a product runs (for tests): 1 pairs, 2 clusters; rows of a cluster's tile; slices of K; workspace bytes.
GB_EXPORT int gb_mx_plan(long long M, long long N, long long K, int fmt, long long* out4) {
  if (M <= 0 || N <= 0 || K <= 0 || M > 0x7fffffffLL || N > 0x7fffffffLL || K > (1LL << 30) || (fmt != FP8 && fmt != FP4)) {
    gbh::set_error("gb_mx_plan: bad extents %lld x %lld x %lld, format %d", M, N, K, fmt);
    return gbh::E_BAD_ARG;
  }
  const Plan p = plan_of(M, N, K, fmt);
  out4[0] = p.pair ? 1 : 2;
  out4[1] = p.pair ? 256 : p.bn;
  out4[2] = p.splits;
  out4[3] = p.workspace;
  return gbh::E_OK;
}

// C (M x N, rows ldc apart) = act(A B^T + bias).  out: DT_BF16, DT_F16 or DT_F32; bias in C's type or fp32 (bias_f32), or null.
// workspace: as many bytes as gb_mx_plan says.
GB_EXPORT int gb_mx_matmul(int fmt, const void* a, const void* sa, const void* b, const void* sb, void* c, long long ldc, const void* bias, int bias_f32, long long M,
                           long long N, long long K, int out, int act, void* workspace, long long workspace_bytes, void* stream) {
  long long p4[4];
  if (int rc = gb_mx_plan(M, N, K, fmt, p4)) return rc;
  if (out < 0 || out > 2 || act < 0 || act > 3 || ldc < N) {
    gbh::set_error("gb_mx_matmul: bad type %d, activation %d or row pitch %lld", out, act, ldc);
    return gbh::E_BAD_ARG;
  }
  const Plan p = plan_of(M, N, K, fmt);
  if (p.workspace > 0 && (workspace == nullptr || workspace_bytes < p.workspace)) {
    gbh::set_error("gb_mx_matmul: workspace of %lld bytes, %lld are needed", workspace_bytes, p.workspace);
    return gbh::E_BAD_ARG;
  }
  const int P = pieces((int)K, fmt), RB = row_bytes((int)K, fmt), per = fmt == FP8 ? 1 : 2;
  MxArgs args{};
  args.M = (int)M; args.N = (int)N; args.steps = p.steps;
  args.splits = p.splits; args.steps_per = p.steps_per;
  args.C = c; args.ldc = ldc; args.bias = bias; args.bias_f32 = bias_f32 || out == OUT_F32; args.act = act; args.out = out;
  args.status = gbh::status_ptr();
  cudaStream_t st = (cudaStream_t)stream;
  Maps tm;
  memset(&tm, 0, sizeof(tm));
  int rc = 0;
  if (p.pair) {
    args.num_m = (int)((M + 255) / 256);
    args.num_n = (int)((N + 255) / 256);
    MxArgs run = args;
    if (p.splits > 1) {
      run.C = workspace; run.ldc = N; run.out = OUT_F32; run.bias = nullptr; run.act = ACT_NONE;
    }
    const int size = run.out == OUT_F32 ? 4 : 2;
    run.tma_out = ((uintptr_t)run.C & 15) == 0 && run.ldc * size % 16 == 0;
    if (run.tma_out) {
      const uint64_t dims[3] = {(uint64_t)N, (uint64_t)M, (uint64_t)p.splits}, strides[2] = {(uint64_t)(run.ldc * size), (uint64_t)(run.ldc * size * M)};
      const uint32_t box[3] = {(uint32_t)(64 / size), 32, 1};
      rc = gbh::encode_tmap(&tm.c, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, run.C, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
    }
    if (!rc) rc = map_codes(&tm.a, a, M, RB, 128);
    if (!rc) rc = map_codes(&tm.b, b, N, RB, 128);
    if (!rc) rc = map_scales(&tm.sa, sa, M, P, per, 1);
    if (!rc) rc = map_scales(&tm.sb, sb, N, P, per, 2);
    if (!rc) rc = fmt == FP8 ? launch_pair<FP8>(tm, run, st) : launch_pair<FP4>(tm, run, st);
    if (rc || p.splits == 1) return rc;
    const long long quads = M * N / 4;
    GB_CUDA_OK(gbh::launch(mx_finish_kernel, dim3((unsigned)(quads / 256 + 1 < 148 * 8 ? quads / 256 + 1 : 148 * 8)), dim3(256), 0, st, 1, (const float*)workspace, args, p.splits));
    return gbh::E_OK;
  }
  args.num_m = (int)((M + p.bn - 1) / p.bn);
  args.num_n = (int)((N + 127) / 128);
  if ((long long)args.num_m * args.num_n * p.splits > 0x7fffffffLL) {
    gbh::set_error("gb_mx_matmul: %lld x %lld has too many tiles", M, N);
    return gbh::E_TOO_LARGE;
  }
  rc = map_codes(&tm.a, b, N, RB, 128);
  if (!rc) rc = map_codes(&tm.b, a, M, RB, p.bn);
  if (!rc) rc = map_scales(&tm.sa, sb, N, P, per, 1);
  if (!rc) rc = map_scales(&tm.sb, sa, M, P, per, 1);
  if (rc) return rc;
  switch (p.bn) {
    case 16: return fmt == FP8 ? launch_cluster<FP8, 16>(tm, args, st) : launch_cluster<FP4, 16>(tm, args, st);
    case 32: return fmt == FP8 ? launch_cluster<FP8, 32>(tm, args, st) : launch_cluster<FP4, 32>(tm, args, st);
    case 64: return fmt == FP8 ? launch_cluster<FP8, 64>(tm, args, st) : launch_cluster<FP4, 64>(tm, args, st);
    default: return fmt == FP8 ? launch_cluster<FP8, 128>(tm, args, st) : launch_cluster<FP4, 128>(tm, args, st);
  }
}
