// Microscaled quantisation (formats: mx.cuh): rows of a tensor into codes and scales, back into values, and the residual's
// addition with the root-mean-square norm whose output is quantised where it is made.
//
// All are bound by memory, and by instructions if those are not few: a lane takes sixteen columns (32 bytes of a 16-bit type), two
// lanes a block, eight lanes the 128 columns whose scales are one word.  Magnitudes of 16-bit types compare in pairs, before anything is
// converted.
#include "mx.cuh"

#include <atomic>

using namespace gb;
using namespace gbmx;

namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------------------------------------------------------
// rows into codes and scales
// ---------------------------------------------------------------------------------------------------------------------------
struct QuantArgs {
  const void* x;
  uint8_t* data;
  uint8_t* scales;
  long long ld;            // elements from row to row of x
  int rows, K, pieces, row_bytes, wide;
  FastDiv by_units;
  Extent ext;
};

// A unit is L / 8 times 128 columns of a row.  L = 0: aligned rows, eight lanes, NU units of a lane in flight.  Others (Stage): 32 lanes, or
// eight of rows of up to 256.  Directly | by way of Stage, us: 50304 x 2048 bf16 to MXFP4 44.5 | 63.6 (and back 48.3 | 58.1); eight lanes | 32, 40 M
// bf16 values to MXFP8 in rows of 33 117 | 294, 201 48 | 53, 257 57 | 45, 1003 46 | 29.  (To MXFP4, whose scale pieces come in twos, rows of 33 220; of
// fp32, 136, 55, 53 and 35.)  What bounds the narrow ones is a load and a store into shared memory for each element.
template <typename T, int FMT, int L>
__global__ void __launch_bounds__(kThreads) mx_quantize_kernel(const QuantArgs a) {
  constexpr int NU = Elem<T>::SZ == 2 && L == 0 ? 2 : 1, LANES = L ? L : 8;
  __shared__ __align__(16) uint8_t shared[L ? kThreads / LANES * Stage<T, LANES>::BYTES : 16];
  pdl_trigger();
  pdl_wait();
  const Stage<T, LANES> stage(shared);
  const int lane = threadIdx.x & 31;
  const unsigned mask = 0xffu << (lane & 24);
  const uint32_t units = (uint32_t)a.rows * a.by_units.d, stride = gridDim.x * (kThreads / LANES);
  for (uint32_t u0 = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES; u0 < units; u0 += NU * stride) {
    uint32_t w[NU][4 * Elem<T>::SZ];
    uint32_t row[NU];
    int k[NU];
#pragma unroll
    for (int i = 0; i < NU; i++) {
      const uint32_t u = min(u0 + i * stride, units - 1);
      row[i] = a.by_units.div(u);
      const int first = (int)(u - row[i] * a.by_units.d) * (16 * LANES);
      k[i] = first + stage.lane * 16;
      const T* x = reinterpret_cast<const T*>(a.x) + row[i] * a.ld;
      if constexpr (L == 0) {
        load16<T, true>(x, k[i], a.K, a.wide, a.ext, w[i]);
      } else {
        typename Stage<T, LANES>::Bits raw[16];
        stage.fetch(x, first, a.K, stage.lane, raw);
        stage.turn(raw, w[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < NU; i++) {
      if (u0 + i * stride >= units) break;
      float v[16];
      unpack16<T>(w[i], v);
      uint32_t out[4];
      const uint32_t word = quantize16<FMT>(v, largest16<T>(w[i]), mask, lane, out);
      store_codes<FMT>(a.data + (long long)row[i] * a.row_bytes, k[i], a.row_bytes, out);
      if ((lane & 7) == 0 && k[i] >> 7 < a.pieces) *reinterpret_cast<uint32_t*>(a.scales + scale_word(row[i], k[i] >> 7, a.pieces)) = word;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// rows and columns into codes and scales (MXFP8), from one reading: the operands of a layer's gradients are quantised along the
// contraction of their product, which is the rows' dimension of one and the columns' of the other
// ---------------------------------------------------------------------------------------------------------------------------
struct BothArgs {
  const void* x;
  uint8_t* data;           // codes along the columns, rows x row_bytes
  uint8_t* scales;
  uint8_t* data_t;         // codes of the transpose along the rows, K x row_bytes_t
  uint8_t* scales_t;
  long long ld;
  int rows, K, pieces, row_bytes, pieces_t, row_bytes_t, wide;
  float* sums;             // column sums of each 128 rows (row pieces x K), or null
  Extent ext;
};

// A block takes 128 x 128 values, so that its scales are one piece of either result.  Rows are quantised as they arrive; the tile
// then stands in shared memory, a thread quantises two columns of 32 rows, and their codes leave by way of shared memory as
// 128-byte pieces of the transpose's rows.  Pieces of 16 bytes are exchanged within a lane's (swapped) so that no bank is met twice.
// As many CTAs as the registers allow load, compute and store in turn: 16384 x 2304 bf16 36.2 us with two of them on an SM and banks met
// twice to eight times, 35.0 so (floor 23.4), 16384 x 768 fp32 21.5 and 17.3 (11.7); rows at any address, 16384 x 2303 bf16 52, 16384 x 767 fp32 28.  Half of the issue slots are in use, 39 % of DRAM's rate.
template <typename T>
struct BothCfg {
  static constexpr int TILE = 128 * 128 * Elem<T>::SZ, PITCH = 128 + 16;
  static constexpr int BYTES = TILE + 128 * PITCH + 1024;
  static __device__ __forceinline__ int swapped(int l8) { return Elem<T>::SZ == 2 ? l8 >> 2 : l8 >> 1; }
};

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, Elem<T>::SZ == 4 ? 2 : ALIGNED ? 4 : 3) mx_quantize_both_kernel(const BothArgs a) {
  using C = BothCfg<T>;
  constexpr int W = 4 * Elem<T>::SZ;                     // words of sixteen elements
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* codes = smem + C::TILE;
  uint32_t* piece = reinterpret_cast<uint32_t*>(codes + 128 * C::PITCH);
  uint16_t* scales_t = reinterpret_cast<uint16_t*>(piece + 128);       // [4][64]: of 32 rows, two columns
  __shared__ float part[4][128];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, l8 = threadIdx.x & 7, h = threadIdx.x >> 3;
  const unsigned mask = 0xffu << (lane & 24);
  const int g = blockIdx.x % a.pieces, gt = blockIdx.x / a.pieces;       // pieces along the columns and the rows
  const int k = g * 128 + l8 * 16;
  uint32_t w[4][W];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const long long row = gt * 128LL + h + 32 * i;
#pragma unroll
    for (int j = 0; j < W; j++) w[i][j] = 0;
    if (row < a.rows) load16<T, ALIGNED>(reinterpret_cast<const T*>(a.x) + row * a.ld, k, a.K, a.wide, a.ext, w[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = h + 32 * i;
    const long long row = gt * 128LL + r;
#pragma unroll
    for (int j = 0; j < W / 4; j++)
      *reinterpret_cast<uint4*>(smem + r * 128 * Elem<T>::SZ + (l8 * (W / 4) + (j ^ C::swapped(l8))) * 16) = make_uint4(w[i][4 * j], w[i][4 * j + 1], w[i][4 * j + 2], w[i][4 * j + 3]);
    float v[16];
    unpack16<T>(w[i], v);
    uint32_t out[4];
    const uint32_t word = quantize16<FP8>(v, largest16<T>(w[i]), mask, lane, out);
    if (row < a.rows) store_codes<FP8>(a.data + row * a.row_bytes, k, a.row_bytes, out);
    if (l8 == 0) piece[h * 4 + i] = word;
  }
  __syncthreads();
  // columns 2 p and 2 p + 1, rows 32 b .. 32 b + 31
  const int p = threadIdx.x & 63, b = threadIdx.x >> 6;
  constexpr int PER = 8 / Elem<T>::SZ;                   // pairs of columns in 16 bytes
  const uint8_t* from = smem + b * 32 * 128 * Elem<T>::SZ + ((p / PER) ^ C::swapped(p >> 3)) * 16 + p % PER * 2 * Elem<T>::SZ;
  uint32_t m0 = 0, m1 = 0, u[32 * Elem<T>::SZ / 2];
  if constexpr (Elem<T>::SZ == 2) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) {
      u[i] = *reinterpret_cast<const uint32_t*>(from + i * 256);
      asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(u[i] & 0x7fff7fffu));
    }
    m0 = Elem<T>::bits(m & 0xffffu);
    m1 = Elem<T>::bits(m >> 16);
  } else {
#pragma unroll
    for (int i = 0; i < 32; i++) {
      const uint2 f = *reinterpret_cast<const uint2*>(from + i * 512);
      u[2 * i] = f.x; u[2 * i + 1] = f.y;
      m0 = max(m0, f.x & 0x7fffffffu);
      m1 = max(m1, f.y & 0x7fffffffu);
    }
  }
  const auto value = [&](int i) {                        // of both columns
    if constexpr (Elem<T>::SZ == 2) {
      const float2 f = Elem<T>::pair(u[i]);
      return pair_of(f.x, f.y);
    } else {
      return pair_of(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
    }
  };
  if (a.sums != nullptr) {
    uint64_t sum = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) sum = add_pair(sum, value(i));
    parts_of(sum, part[b][2 * p], part[b][2 * p + 1]);
  }
  const uint32_t c0 = scale_code(m0, FP8), c1 = scale_code(m1, FP8);
  const uint64_t inv = pair_of(scale_inverse(c0), scale_inverse(c1));
  scales_t[b * 64 + p] = (uint16_t)(c0 | c1 << 8);
#pragma unroll
  for (int half = 0; half < 2; half++) {                 // sixteen rows
    uint32_t q0[4], q1[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float x0[4], x1[4];
#pragma unroll
      for (int j = 0; j < 4; j++) parts_of(mul_pair(value(16 * half + 4 * i + j), inv), x0[j], x1[j]);
      q0[i] = e4m3x4(x0[0], x0[1], x0[2], x0[3]);
      q1[i] = e4m3x4(x1[0], x1[1], x1[2], x1[3]);
    }
    uint8_t* to = codes + 2 * p * C::PITCH + (b * 2 + (half ^ (p >> 2 & 1))) * 16;
    *reinterpret_cast<uint4*>(to) = make_uint4(q0[0], q0[1], q0[2], q0[3]);
    *reinterpret_cast<uint4*>(to + C::PITCH) = make_uint4(q1[0], q1[1], q1[2], q1[3]);
  }
  __syncthreads();
  if (a.sums != nullptr && threadIdx.x < 128 && g * 128 + threadIdx.x < a.K)
    a.sums[(long long)gt * a.K + g * 128 + threadIdx.x] = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
  if (threadIdx.x < 128) {
    reinterpret_cast<uint32_t*>(a.scales + ((long long)gt * a.pieces + g) * 512)[threadIdx.x] = piece[threadIdx.x];
  } else {
    const int t = threadIdx.x - 128;
    const uint8_t* s = reinterpret_cast<const uint8_t*>(scales_t) + (t >> 2) + 32 * (t & 3);
    reinterpret_cast<uint32_t*>(a.scales_t + ((long long)g * a.pieces_t + gt) * 512)[t] = s[0] | s[128] << 8 | s[256] << 16 | (uint32_t)s[384] << 24;
  }
  const int at = gt * 128 + l8 * 16;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int col = h + 32 * i;
    if (g * 128 + col < a.K && at < a.row_bytes_t)
      *reinterpret_cast<uint4*>(a.data_t + (g * 128LL + col) * a.row_bytes_t + at) = *reinterpret_cast<const uint4*>(codes + col * C::PITCH + (l8 ^ (col >> 3 & 1)) * 16);
  }
}

template <typename T>
__device__ __forceinline__ T to_type(float v);
template <> __device__ __forceinline__ float to_type<float>(float v) { return v; }
template <> __device__ __forceinline__ __half to_type<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 to_type<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Sums over the pieces of rows that mx_quantize_both_kernel left, in fp32 and in one order: 32 columns a block, eight strips of pieces.
template <typename T>
__global__ void __launch_bounds__(256) mx_column_sum_kernel(const float* __restrict__ sums, T* __restrict__ out, int pieces, int K) {
  __shared__ float part[8][32];
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), strip = threadIdx.x >> 5;
  float s = 0.f;
  if (c < K) {
#pragma unroll 8
    for (int i = strip; i < pieces; i += 8) s += __ldg(sums + (long long)i * K + c);
  }
  part[strip][threadIdx.x & 31] = s;
  __syncthreads();
  if (strip == 0 && c < K) {
#pragma unroll
    for (int i = 1; i < 8; i++) s += part[i][threadIdx.x];
    out[c] = to_type<T>(s);
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// codes and scales into values
// ---------------------------------------------------------------------------------------------------------------------------
struct DequantArgs {
  const uint8_t* data;
  const uint8_t* scales;
  void* y;                 // rows x K, contiguous
  int rows, K, pieces, row_bytes, wide;
  FastDiv by_units;
};

template <int FMT>
__device__ __forceinline__ void numbers16(const uint32_t (&c)[4], float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    uint32_t h;
    if (FMT == FP8) asm("{\n.reg .b16 t;\ncvt.u16.u32 t, %1;\ncvt.rn.f16x2.e4m3x2 %0, t;\n}" : "=r"(h) : "r"(c[i / 2] >> (16 * (i & 1))));
    else asm("{\n.reg .b8 t, u0, u1, u2;\nmov.b32 {t, u0, u1, u2}, %1;\ncvt.rn.f16x2.e2m1x2 %0, t;\n}" : "=r"(h) : "r"(c[i / 4] >> (8 * (i & 3))));
    const float2 f = unpack_f16(h);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// L: as in mx_quantize_kernel, for the rows of values.
template <typename T, int FMT, int L>
__global__ void __launch_bounds__(kThreads) mx_dequantize_kernel(const DequantArgs a) {
  constexpr int NU = L == 0 ? 2 : 1, LANES = L ? L : 8;
  __shared__ __align__(16) uint8_t shared[L ? kThreads / LANES * Stage<T, LANES>::BYTES : 16];
  pdl_trigger();
  pdl_wait();
  const Stage<T, LANES> stage(shared);
  const uint32_t units = (uint32_t)a.rows * a.by_units.d, stride = gridDim.x * (kThreads / LANES);
  for (uint32_t u0 = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES; u0 < units; u0 += NU * stride) {
    uint32_t c[NU][4], row[NU];
    int first[NU];
    uint8_t s[NU];
#pragma unroll
    for (int i = 0; i < NU; i++) {
      const uint32_t u = min(u0 + i * stride, units - 1);
      row[i] = a.by_units.div(u);
      first[i] = (int)(u - row[i] * a.by_units.d) * (16 * LANES);
      const int k = first[i] + stage.lane * 16, b = FMT == FP8 ? k : k / 2;
      const uint8_t* from = a.data + (long long)row[i] * a.row_bytes + b;
      c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0;
      s[i] = 0;
      if (b < a.row_bytes) {
        if (FMT == FP8) {
          const uint4 q = __ldg(reinterpret_cast<const uint4*>(from));
          c[i][0] = q.x; c[i][1] = q.y; c[i][2] = q.z; c[i][3] = q.w;
        } else {
          const uint2 q = __ldg(reinterpret_cast<const uint2*>(from));
          c[i][0] = q.x; c[i][1] = q.y;
        }
        s[i] = __ldg(a.scales + scale_word(row[i], k >> 7, a.pieces) + (k >> 5 & 3));
      }
    }
#pragma unroll
    for (int i = 0; i < NU; i++) {
      if (u0 + i * stride >= units) break;
      float v[16];
      numbers16<FMT>(c[i], v);
      const uint64_t scale = pair_of(scale_value(s[i]), scale_value(s[i]));
#pragma unroll
      for (int j = 0; j < 16; j += 2) parts_of(mul_pair(pair_of(v[j], v[j + 1]), scale), v[j], v[j + 1]);
      T* to = reinterpret_cast<T*>(a.y) + (long long)row[i] * a.K;
      if constexpr (L == 0) store16(to, first[i] + stage.lane * 16, a.K, a.wide, v);
      else stage.store(to, first[i], a.K, v);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// h = x + r; codes of h / sqrt(mean(h^2) + eps) * w
// ---------------------------------------------------------------------------------------------------------------------------
struct NormArgs {
  const void* x;
  const void* r;           // null: no residual, and h is not written
  const void* w;
  void* h;                 // rows x K, contiguous
  uint8_t* data;
  uint8_t* scales;
  long long ldx, ldr;
  int rows, K, pieces, row_bytes, w_f32, wide;
  double eps, inv_K;
  Extent ex, er, ew;
};

// fp64 of fp32, subnormal numbers too.
__device__ __forceinline__ double to_double(float v) {
  double d;
  asm("cvt.f64.f32 %0, %1;" : "=d"(d) : "f"(v));
  return d;
}
// 1 / sqrt(v) to a rounding of fp32: the approximation and a step of Newton's iteration in fp64.
__device__ __forceinline__ float inverse_root(double v) {
  float r0;
  asm("rsqrt.approx.f32 %0, %1;" : "=f"(r0) : "f"((float)v));
  return (float)fma(0.5 * (double)r0, fma(-v * (double)r0, (double)r0, 1.0), (double)r0);
}
// A row whose sum of squares s or mean square v = s / K + eps fp32 cannot be trusted with (all of its values but zeros are taken as next to a border).
__device__ __forceinline__ bool far_out(double s, double v) { return !(s > 1e-25 && s < 1e38 && v > 1e-36 && v < 1e36); }

// A value next to the border between two codes has to fall on the side where it belongs: by three roundings of fp32 one in a million falls on
// the other, a step of the code away.  Borders, and the powers of two at which a scale changes, have at most four leading bits of
// a fraction (E4M3; E2M1 two), so the last 19 (21) bits of a value in their neighbourhood are next to zero.  Eight roundings of 2^-24 each (the
// sum, in its square too, where it is not exact; half of the eight of a chain of squares; 1 / rms; its product) and the value's own move them by
// less than nine units of the last place, 4.25 times two for the largest fraction and half a unit.  A row with such a value (one value
// in 30 000 or 120 000; and infinities and NaN) gets its sum again, in fp64, and the blocks of such values are computed again in fp64, from
// what was added, and rounded to odd: the last bit stands for all that lies behind it, so that the rounding to a code afterwards is that of the
// value itself.
template <int FMT>
__device__ __forceinline__ uint32_t from_border(float y) {       // those bits and 8, above zeros
  constexpr uint32_t shift = FMT == FP8 ? 1u << 13 : 1u << 11;
  return __float_as_uint(y) * shift + 8u * shift;
}
template <int FMT> constexpr uint32_t kNear = 16u << (FMT == FP8 ? 13 : 11);

// (x + r) / rms * w * by, rounded to odd; what is above the largest number of fp32 becomes that (an odd one).
__device__ __forceinline__ float to_odd(float x, float r, float w, double rms, double by) {
  const double y = (to_double(x) + to_double(r)) / rms * to_double(w) * by;
  float z;
  asm("cvt.rz.f32.f64 %0, %1;" : "=f"(z) : "d"(y));
  return to_double(z) != y ? __uint_as_float(__float_as_uint(z) | 1u) : z;
}

// The sum over the G threads of a row: a half-warp, or whole warps (their sums in one order, the same for every thread).
template <int G>
__device__ __forceinline__ double row_sum(double s, double* red) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (G <= 32) return s;
  const int first = (int)threadIdx.x / G * (G / 32);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < G / 32; i++) s += red[first + i];
  return s;                              // (a barrier has to follow before the next: row_any's)
}
// Whether one of a warp's threads, or of a block's where a row takes more than a warp, says so.
template <int G>
__device__ __forceinline__ bool row_any(bool says) {
  if (G <= 32) return __any_sync(0xffffffffu, says);
  return __syncthreads_or(says);
}

// Sixteen columns of x + r, in pairs.
template <typename T>
__device__ __forceinline__ void sum16(const uint32_t (&wx)[4 * Elem<T>::SZ], const uint32_t (&wr)[4 * Elem<T>::SZ], uint64_t (&h)[8]) {
  float x[16], r[16];
  unpack16<T>(wx, x);
  unpack16<T>(wr, r);
#pragma unroll
  for (int j = 0; j < 8; j++) h[j] = add_pair(pair_of(x[2 * j], x[2 * j + 1]), pair_of(r[2 * j], r[2 * j + 1]));
}
// Their squares: two chains of eight in fp32, which an fp64 sum takes up.
__device__ __forceinline__ double squares(const uint64_t (&h)[8]) {
  uint64_t s = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) s = fma_pair(h[j], h[j], s);
  float a, b;
  parts_of(s, a, b);
  return (double)a + (double)b;
}

// The same in fp64, of x + r as it is before any rounding to fp32.
template <typename T>
__device__ __forceinline__ double squares_exact(const uint32_t (&wx)[4 * Elem<T>::SZ], const uint32_t (&wr)[4 * Elem<T>::SZ]) {
  float x[16], r[16];
  unpack16<T>(wx, x);
  unpack16<T>(wr, r);
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < 16; j++) {
    const double h = to_double(x[j]) + to_double(r[j]);
    s = fma(h, h, s);
  }
  return s;
}

template <typename T, bool ALIGNED, int L>
__device__ __forceinline__ void write_sum(const NormArgs& a, long long row, int k, const uint64_t (&h)[8], const Stage<T, L>& stage) {
  float v[16];
#pragma unroll
  for (int j = 0; j < 8; j++) parts_of(h[j], v[2 * j], v[2 * j + 1]);
  T* to = reinterpret_cast<T*>(a.h) + row * a.K;
  if constexpr (ALIGNED) store16(to, k, a.K, a.wide, v);
  else stage.store(to, k - stage.lane * 16, a.K, v);
}

// The weights of sixteen columns.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void weights16(const NormArgs& a, int k, float (&w)[16]) {
  if (sizeof(T) == 2 && a.w_f32) {
    uint32_t u[16];
    load16<float, false>(reinterpret_cast<const float*>(a.w), k, a.K, false, a.ew, u);
    unpack16<float>(u, w);
  } else {                               // (a row's weights stand still while rows come and go: vectors from L1)
    uint32_t u[4 * Elem<T>::SZ];
    load16<T, ALIGNED>(reinterpret_cast<const T*>(a.w), k, a.K, false, a.ew, u);
    unpack16<T>(u, w);
  }
}

// Codes of sixteen columns; whether one of the values may lie on the other side of a border.  far: the row's sum cannot be trusted.
template <typename T, int FMT, bool ALIGNED>
__device__ __forceinline__ bool write_norm(const NormArgs& a, long long row, int k, const uint64_t (&h)[8], float root, bool far) {
  float w[16], y[16];
  weights16<T, ALIGNED>(a, k, w);
  const uint64_t root2 = pair_of(root, root);
  // for the test, zeros become a number far from any border (sums of bf16 values are zero now and then) and others from 2^-101 on stay what they
  // are; lanes whose largest value is so small that the others count come again whole.  (What this does not see: a product with 1 / rms that is
  // subnormal, of a value 2^126 times below the row's, and comes back through a weight above 2^27.)
  const uint64_t tiny = pair_of(__uint_as_float(0x00955555u), __uint_as_float(0x00955555u));
  uint32_t near = ~0u;
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const uint64_t p = mul_pair(h[j], root2), w2 = pair_of(w[2 * j], w[2 * j + 1]);
    float a, b;
    parts_of(fma_pair(p, w2, tiny), a, b);
    near = min(near, min(from_border<FMT>(a), from_border<FMT>(b)));
    parts_of(mul_pair(p, w2), y[2 * j], y[2 * j + 1]);
    m = fmaxf(fmaxf(m, fabsf(y[2 * j])), fabsf(y[2 * j + 1]));
  }
  uint32_t out[4];
  const int lane = threadIdx.x & 31;     // (a flushed subnormal number has the same scale; infinities and NaN come again)
  const uint32_t word = quantize16<FMT>(y, __float_as_uint(m), 0xffu << (lane & 24), lane, out);
  store_codes<FMT>(a.data + row * a.row_bytes, k, a.row_bytes, out);
  if ((lane & 7) == 0) *reinterpret_cast<uint32_t*>(a.scales + scale_word(row, k >> 7, a.pieces)) = word;
  if (far || m < 0x1p-80f) {             // (a block's borders go down to 2^-19 of its largest value)
    uint64_t some = 0;                   // zeros are what they are, unless the root makes NaN of them
#pragma unroll
    for (int j = 0; j < 8; j++) some |= (h[j] | pair_of(y[2 * j], y[2 * j + 1])) & 0x7fffffff7fffffffull;
    return some != 0;
  }
  return near <= kNear<FMT>;
}
template <typename T> __device__ __forceinline__ float element(const T* from, long long i) {
  return Elem<T>::one(__ldg(reinterpret_cast<const typename Stage<T, 32>::Bits*>(from) + i));
}
// Codes and scale of the block from column k on, in fp64, a column a lane (a lane that computes its sixteen one after the other takes 3 us for
// them: 600 x 2048 bf16 5.5 | 8.5).  A block that holds more than fp32 does is taken 2^16 times smaller (a norm's values are below 2^15
// times the weight).
template <typename T, int FMT>
__device__ __forceinline__ void write_block_exact(const NormArgs& a, long long row, int k, double rms) {
  const int lane = threadIdx.x & 31, c = k + lane;
  float x = 0.f, r = 0.f, w = 0.f;
  if (c < a.K) {
    x = element(reinterpret_cast<const T*>(a.x), row * a.ldx + c);
    if (a.r != nullptr) r = element(reinterpret_cast<const T*>(a.r), row * a.ldr + c);
    w = a.w_f32 ? __ldg(reinterpret_cast<const float*>(a.w) + c) : element(reinterpret_cast<const T*>(a.w), c);
  }
  float y;
  uint32_t amax = 0, up = 0;
  for (double by = 1.0;; by = 0x1p-16, up = 16) {
    y = c < a.K ? to_odd(x, r, w, rms, by) : 0.f;        // (zeros behind the end of a row of NaN too)
    amax = __reduce_max_sync(0xffffffffu, __float_as_uint(y) & 0x7fffffffu);
    if (up != 0 || amax != 0x7f7fffffu) break;
  }
  const uint32_t code = up == 0 ? scale_code(amax, FMT) : min(scale_code(amax, FMT) + up, 254u);
  const float q = mul_exact(y, scale_inverse(code - up)), next = __shfl_down_sync(0xffffffffu, q, 1);
  uint8_t* to = a.data + row * a.row_bytes;
  if (FMT == FP8) {
    if (c < a.row_bytes) to[c] = (uint8_t)e4m3x4(q, 0.f, 0.f, 0.f);
  } else {
    const float v[8] = {q, next, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c / 2 < a.row_bytes && (lane & 1) == 0) to[c / 2] = (uint8_t)e2m1x8(v);
  }
  if (lane == 0) a.scales[scale_word(row, k >> 7, a.pieces) + (k >> 5 & 3)] = (uint8_t)code;
}

// G threads of a block take a row (sixteen, or whole warps), VPT vectors of sixteen columns each, which stay in registers between the two
// passes.  VPT = 0: rows of any length, read a second time for their codes.  BLOCKS: on an SM.  What counts is how many warps there are to
// hide each other's latency: with 14 of 124 registers on an SM, three vectors each, 16384 x 2048 bf16 took 51 us, with 24 of 80 44; rows that
// bulk copies brought to 16 warps ahead of time 69.  Rows at any address spill from 64 registers: 5003 x 2001 bf16 28.2 us, with 80 26.9.
constexpr int norm_threads(int G) { return G >= 256 ? G : 256 / G * G; }
constexpr int norm_blocks(int size, int vpt, int G, bool aligned) {
  return (vpt == 1 ? (size == 4 || !aligned ? 768 : 1024) : vpt == 2 ? (size == 4 ? 512 : 768) : 512) / norm_threads(G);
}

template <typename T, int FMT, int G, int VPT, bool ALIGNED>
__global__ void __launch_bounds__(norm_threads(G), norm_blocks(sizeof(T), VPT, G, ALIGNED)) mx_norm_kernel(const NormArgs a) {
  constexpr int THREADS = norm_threads(G), W = 4 * Elem<T>::SZ, L = G < 32 ? G : 32, per = THREADS / G;
  __shared__ double red[32];
  __shared__ __align__(16) uint8_t shared[ALIGNED ? 16 : THREADS / L * Stage<T, L>::BYTES];
  pdl_trigger();
  pdl_wait();
  const Stage<T, L> stage(shared);
  const int t = threadIdx.x % G;
  const int vecs = a.pieces * 8;                         // whole pieces: eight lanes work together
  const bool sum = a.r != nullptr;
  for (long long first = (long long)blockIdx.x * per; first < a.rows; first += (long long)gridDim.x * per) {
    const long long row = first + threadIdx.x / G;
    const bool live = row < a.rows;
    const int K = live ? a.K : 0, KR = sum ? K : 0;
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    const T* r = reinterpret_cast<const T*>(a.r) + row * a.ldr;
    // vector i of x and r (a row's threads take each step together, for the way through shared memory)
    auto take = [&](int i, uint32_t (&wx)[W], uint32_t (&wr)[W]) {
      if constexpr (ALIGNED) {
#pragma unroll
        for (int j = 0; j < W; j++) wx[j] = wr[j] = 0;
        if (live) {
          load16<T, true>(x, i * 16, a.K, a.wide, a.ex, wx);
          if (sum) load16<T, true>(r, i * 16, a.K, a.wide, a.er, wr);
        }
      } else {
        typename Stage<T, L>::Bits bx[16], br[16];
        stage.fetch(x, (i - stage.lane) * 16, K, stage.lane, bx);
        stage.fetch(r, (i - stage.lane) * 16, KR, stage.lane, br);
        stage.turn(bx, wx);
        stage.turn(br, wr);
      }
    };
    double s = 0.0, v;
    float root;
    uint32_t near = 0;                                   // which of the thread's vectors have to come again (the last bit: from the 32nd on)
    if constexpr (VPT > 0) {
      uint64_t h[VPT][8];
      if constexpr (ALIGNED) {
        uint32_t wx[VPT][W], wr[VPT][W];
#pragma unroll
        for (int i = 0; i < VPT; i++) take(t + i * G, wx[i], wr[i]);
#pragma unroll
        for (int i = 0; i < VPT; i++) {
          sum16<T>(wx[i], wr[i], h[i]);                  // (zeros without a residual)
          s += squares(h[i]);
        }
      } else {
        typename Stage<T, L>::Bits bx[VPT][16], br[VPT][16];
#pragma unroll
        for (int i = 0; i < VPT; i++) {
          const int k = (t - stage.lane + i * G) * 16;
          stage.fetch(x, k, K, stage.lane, bx[i]);
          stage.fetch(r, k, KR, stage.lane, br[i]);
        }
#pragma unroll
        for (int i = 0; i < VPT; i++) {
          uint32_t wx[W], wr[W];
          stage.turn(bx[i], wx);
          stage.turn(br[i], wr);
          sum16<T>(wx, wr, h[i]);
          s += squares(h[i]);
        }
      }
      if (sum && live) {
#pragma unroll
        for (int i = 0; i < VPT; i++) write_sum<T, ALIGNED, L>(a, row, (t + i * G) * 16, h[i], stage);
      }
      s = row_sum<G>(s, red);
      v = fma(s, a.inv_K, a.eps);
      root = inverse_root(v);
#pragma unroll
      for (int i = 0; i < VPT; i++)
        if (live && t + i * G < vecs && write_norm<T, FMT, ALIGNED>(a, row, (t + i * G) * 16, h[i], root, far_out(s, v))) near |= 1u << i;
    } else {
      for (int i = t; i - t < vecs; i += G) {
        uint32_t wx[W], wr[W];
        uint64_t h[8];
        take(i, wx, wr);
        sum16<T>(wx, wr, h);
        if (sum) write_sum<T, ALIGNED, L>(a, row, i * 16, h, stage);
        s += squares(h);
      }
      s = row_sum<G>(s, red);
      v = fma(s, a.inv_K, a.eps);
      root = inverse_root(v);
      for (int i = t, n = 0; i - t < vecs; i += G, n++) {
        uint32_t wx[W], wr[W];
        uint64_t h[8];
        take(i, wx, wr);
        sum16<T>(wx, wr, h);
        if (i < vecs && write_norm<T, FMT, ALIGNED>(a, row, i * 16, h, root, far_out(s, v))) near |= 1u << min(n, 31);
      }
    }
    if (row_any<G>(near != 0)) {
      double exact = 0.0;
      if constexpr (ALIGNED) {
        for (int i = t; i < vecs; i += G) {
          uint32_t wx[W], wr[W];
          take(i, wx, wr);
          exact += squares_exact<T>(wx, wr);
        }
      } else {
        const auto from = [&](const T* p, int k, int K) { return k < K ? element(p, k) : 0.f; };
#pragma unroll 1
        for (int k = t; k < K; k += 8 * G) {             // (a sum has any order; eight columns of a thread in flight)
          float ex[8], er[8];
#pragma unroll
          for (int j = 0; j < 8; j++) ex[j] = from(x, k + j * G, K), er[j] = from(r, k + j * G, KR);
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const double h = to_double(ex[j]) + to_double(er[j]);
            exact = fma(h, h, exact);
          }
        }
      }
      const double rms = sqrt(row_sum<G>(exact, red) / a.K + a.eps);
      __syncwarp();                                      // the blocks' first codes, of any lane of the warp, are there
      const int lane = threadIdx.x & 31;
      const int steps = VPT > 0 ? VPT : (vecs + G - 1) / G;
#pragma unroll 1
      for (int n = 0; n < steps; n++) {
        const unsigned those = __ballot_sync(0xffffffffu, t + n * G < vecs && (near >> min(n, 31) & 1));
        for (unsigned pairs = (those | those >> 1) & 0x55555555u; pairs != 0; pairs &= pairs - 1) {
          const int from = __ffs(pairs) - 1;             // the first lane of a block: its row, its columns
          const double its = G < 32 ? __shfl_sync(0xffffffffu, rms, from) : rms;
          write_block_exact<T, FMT>(a, first + (threadIdx.x - lane + from) / G, ((threadIdx.x - lane + from) % G + n * G) * 16, its);
        }
      }
      if (G > 32) __syncthreads();
    }
  }
}

Extent extent_of(const void* p, long long rows, long long ld, long long K, int size) {
  Extent e;
  e.begin = reinterpret_cast<uintptr_t>(p);
  e.end = e.begin + (uintptr_t)(((rows - 1) * ld + K) * size);
  return e;
}

bool bad_shape(const char* what, const void* x, long long rows, long long K, long long ld, int fmt, const void* data, const void* scales) {
  if (rows <= 0 || K <= 0 || rows > 0x7fffffffLL || K > (1LL << 30) || ld < 0 || (fmt != FP8 && fmt != FP4)) {
    gbh::set_error("%s: bad extents %lld x %lld, row pitch %lld, format %d", what, rows, K, ld, fmt);
    return true;
  }
  if (x == nullptr || data == nullptr || scales == nullptr || ((uintptr_t)data & 15) || ((uintptr_t)scales & 15)) {
    gbh::set_error("%s: a tensor, and codes and scales on 16-byte boundaries are needed", what);
    return true;
  }
  return false;
}

// Rows per launch: units are counted in 31 bits.
long long rows_at_once(long long rows, int P) {
  const long long most = (0x7fffffffLL / P) / 128 * 128;
  return rows < most ? rows : most;
}

unsigned grid_of(long long units, int per_block, int blocks_per_sm) {
  const long long g = (units + per_block - 1) / per_block, most = 148LL * blocks_per_sm;
  return (unsigned)(g < 1 ? 1 : g < most ? g : most);
}

// Rows on 16-byte boundaries, whole vectors of eight; and of sixteen, on 32-byte boundaries.
bool aligned_rows(const void* p, long long ld, long long K, int size) { return ((uintptr_t)p & 15) == 0 && ld * size % 16 == 0 && K % 8 == 0; }
bool wide_rows(const void* p, long long ld, long long K, int size) { return ((uintptr_t)p & 31) == 0 && ld * size % 32 == 0 && K % 16 == 0; }

// How a row of `vecs` vectors is dealt out: one to a thread, the shortest way, or two, which holds more in flight, for what does not stay in
// L2.  One | two, bf16, us: 600 x 2048 4.0 | 5.2, 2400 x 2048 8.1 | 9.4, 8192 x 768 10.6 | 11.5, 2400 x 4096 13.6 | 13.7, 16384 x 768 21.5 | 19.1,
// 16384 x 2048 44 | 43.5, 8192 x 8192 91 | 82; fp32, 8192 x 2048 42 | 42, 4096 x 8192 95 | 78 (before rows with a value next to a border took
// their sum again, which costs 5 to 10 % of either).  Now, with inputs in turn beyond L2: 16384 x 768 21.4, 16384 x 2048 50, 8192 x 8192 94, fp32
// 16384 x 768 33.7, 8192 x 8192 167; rows at any address, 16384 x 1003 42.9, fp32 53.
template <typename T, int FMT, bool ALIGNED>
cudaError_t norm_launch(const NormArgs& a, cudaStream_t st) {
  const int vecs = a.pieces * 8;
  auto go = [&](auto kern, int G) {
    const int threads = norm_threads(G), per = threads / G;
    const long long ctas = ((long long)a.rows + per - 1) / per, most = 148LL * 8;
    return gbh::launch(kern, dim3((unsigned)(ctas < most ? ctas : most)), dim3(threads), 0, st, 1, a);
  };
  if (vecs <= 16) return go(mx_norm_kernel<T, FMT, 16, 1, ALIGNED>, 16);
  if constexpr (ALIGNED) {
    if ((long long)a.rows * a.K > 9 << 20) {
      if (vecs > 32 && vecs <= 64) return go(mx_norm_kernel<T, FMT, 32, 2, true>, 32);
      if (vecs > 64 && vecs <= 128) return go(mx_norm_kernel<T, FMT, 64, 2, true>, 64);
      if (vecs > 128 && vecs <= 192) return go(mx_norm_kernel<T, FMT, 96, 2, true>, 96);
      if (vecs > 192 && vecs <= 256) return go(mx_norm_kernel<T, FMT, 128, 2, true>, 128);
      if (vecs > 256 && vecs <= 512) return go(mx_norm_kernel<T, FMT, 256, 2, true>, 256);
    }
    if (vecs > 512 && vecs <= 1024) return go(mx_norm_kernel<T, FMT, 512, 2, true>, 512);
  }
  if (vecs <= 32) return go(mx_norm_kernel<T, FMT, 32, 1, ALIGNED>, 32);
  if (vecs <= 64) return go(mx_norm_kernel<T, FMT, 64, 1, ALIGNED>, 64);
  if (vecs <= 128) return go(mx_norm_kernel<T, FMT, 128, 1, ALIGNED>, 128);
  if (vecs <= 256) return go(mx_norm_kernel<T, FMT, 256, 1, ALIGNED>, 256);
  if (vecs <= 512) return go(mx_norm_kernel<T, FMT, 512, 1, ALIGNED>, 512);
  return go(mx_norm_kernel<T, FMT, 512, 0, ALIGNED>, 512);
}

}  // namespace

enum { DT_BF16 = 0, DT_F16 = 1, DT_F32 = 2 };

// CALL with the type T and the format FMT.
#define GB_MX_PICK(TYPE, fmt, CALL)                       \
  {                                                       \
    using T = TYPE;                                       \
    if (fmt == FP8) { constexpr int FMT = FP8; CALL; }    \
    else { constexpr int FMT = FP4; CALL; }               \
  }
#define GB_MX_DISPATCH(dtype, fmt, CALL)                       \
  if (dtype == DT_BF16) GB_MX_PICK(__nv_bfloat16, fmt, CALL)   \
  else if (dtype == DT_F16) GB_MX_PICK(__half, fmt, CALL)      \
  else GB_MX_PICK(float, fmt, CALL)

// Codes and scales of x (rows x K, rows `ld` elements apart).  The scales of rows up to the next multiple of 128 are left as they were.
GB_EXPORT int gb_mx_quantize(int dtype, int fmt, const void* x, long long ld, void* data, void* scales, long long rows, long long K, void* stream) {
  if (bad_shape("gb_mx_quantize", x, rows, K, ld, fmt, data, scales)) return gbh::E_BAD_ARG;
  if (dtype != DT_BF16 && dtype != DT_F16 && dtype != DT_F32) {
    gbh::set_error("gb_mx_quantize: unsupported dtype %d", dtype);
    return gbh::E_BAD_ARG;
  }
  const int P = pieces((int)K, fmt), RB = row_bytes((int)K, fmt), size = dtype == DT_F32 ? 4 : 2;
  const int lanes = aligned_rows(x, ld, K, size) ? 0 : K <= 256 ? 8 : 32;
  for (long long r0 = 0, n; r0 < rows; r0 += n) {
    n = rows_at_once(rows - r0, P);
    QuantArgs a{(const uint8_t*)x + r0 * ld * size, (uint8_t*)data + r0 * RB, (uint8_t*)scales + r0 / 128 * P * 512, ld, (int)n, (int)K, P, RB,
                wide_rows(x, ld, K, size), FastDiv((uint32_t)(lanes == 32 ? (P + 3) / 4 : P)), extent_of(x, rows, ld, K, size)};
    cudaError_t e = cudaSuccess;
    auto go = [&](auto kern) { e = gbh::launch(kern, dim3(grid_of(n * a.by_units.d, kThreads / (lanes ? lanes : 8), 8)), dim3(kThreads), 0, (cudaStream_t)stream, 1, a); };
    GB_MX_DISPATCH(dtype, fmt, lanes == 0 ? go(mx_quantize_kernel<T, FMT, 0>) : lanes == 8 ? go(mx_quantize_kernel<T, FMT, 8>) : go(mx_quantize_kernel<T, FMT, 32>))
    GB_CUDA_OK(e);
  }
  return gbh::E_OK;
}

// Codes and scales (MXFP8) of x (rows x K, rows `ld` elements apart) along its columns, and of its transpose along the rows.  sums: null, or
// fp32 scratch of (rows / 128, rounded up) x K, for the column sums of x in column_sums (of type sum_dtype).
GB_EXPORT int gb_mx_quantize_both(int dtype, const void* x, long long ld, void* data, void* scales, void* data_t, void* scales_t, float* sums, void* column_sums,
                                  int sum_dtype, long long rows, long long K, void* stream) {
  if (bad_shape("gb_mx_quantize_both", x, rows, K, ld, FP8, data, scales) || bad_shape("gb_mx_quantize_both", x, K, rows, ld, FP8, data_t, scales_t)) return gbh::E_BAD_ARG;
  const int P = pieces((int)K, FP8), PT = pieces((int)rows, FP8);
  const long long blocks = (long long)P * PT;
  if (blocks > 0x7fffffffLL) {
    gbh::set_error("gb_mx_quantize_both: %lld x %lld is too large", rows, K);
    return gbh::E_TOO_LARGE;
  }
  if (sums != nullptr && (column_sums == nullptr || sum_dtype < DT_BF16 || sum_dtype > DT_F32)) {
    gbh::set_error("gb_mx_quantize_both: column sums of type %d", sum_dtype);
    return gbh::E_BAD_ARG;
  }
  const int size = dtype == DT_F32 ? 4 : 2;
  const BothArgs a{x, (uint8_t*)data, (uint8_t*)scales, (uint8_t*)data_t, (uint8_t*)scales_t, ld, (int)rows, (int)K, P, row_bytes((int)K, FP8), PT,
                   row_bytes((int)rows, FP8), wide_rows(x, ld, K, size), sums, extent_of(x, rows, ld, K, size)};
  cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto kern, int bytes, std::atomic<uint32_t>& done) -> int {
    int dev = 0;
    GB_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 32 || !(done.load() >> dev & 1u)) {       // more shared memory than 48 KB: once per device
      GB_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
      if (dev < 32) done.fetch_or(1u << dev);
    }
    GB_CUDA_OK(gbh::launch(kern, dim3((unsigned)blocks), dim3(kThreads), bytes, st, 1, a));
    return gbh::E_OK;
  };
  static std::atomic<uint32_t> done[6];
  const bool aligned = aligned_rows(x, ld, K, size);
  int rc;
  switch (dtype) {
    case DT_BF16: rc = aligned ? go(mx_quantize_both_kernel<__nv_bfloat16, true>, BothCfg<__nv_bfloat16>::BYTES, done[0])
                               : go(mx_quantize_both_kernel<__nv_bfloat16, false>, BothCfg<__nv_bfloat16>::BYTES, done[1]); break;
    case DT_F16: rc = aligned ? go(mx_quantize_both_kernel<__half, true>, BothCfg<__half>::BYTES, done[2])
                              : go(mx_quantize_both_kernel<__half, false>, BothCfg<__half>::BYTES, done[3]); break;
    case DT_F32: rc = aligned ? go(mx_quantize_both_kernel<float, true>, BothCfg<float>::BYTES, done[4])
                              : go(mx_quantize_both_kernel<float, false>, BothCfg<float>::BYTES, done[5]); break;
    default: gbh::set_error("gb_mx_quantize_both: unsupported dtype %d", dtype); return gbh::E_BAD_ARG;
  }
  if (rc || sums == nullptr) return rc;
  const dim3 grid((unsigned)((K + 31) / 32));
  if (sum_dtype == DT_BF16) GB_CUDA_OK(gbh::launch(mx_column_sum_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, 1, (const float*)sums, (__nv_bfloat16*)column_sums, PT, (int)K));
  else if (sum_dtype == DT_F16) GB_CUDA_OK(gbh::launch(mx_column_sum_kernel<__half>, grid, dim3(256), 0, st, 1, (const float*)sums, (__half*)column_sums, PT, (int)K));
  else GB_CUDA_OK(gbh::launch(mx_column_sum_kernel<float>, grid, dim3(256), 0, st, 1, (const float*)sums, (float*)column_sums, PT, (int)K));
  return gbh::E_OK;
}

// The values (rows x K, contiguous) that codes and scales stand for.
GB_EXPORT int gb_mx_dequantize(int dtype, int fmt, const void* data, const void* scales, void* y, long long rows, long long K, void* stream) {
  if (bad_shape("gb_mx_dequantize", y, rows, K, K, fmt, data, scales)) return gbh::E_BAD_ARG;
  if (dtype != DT_BF16 && dtype != DT_F16 && dtype != DT_F32) {
    gbh::set_error("gb_mx_dequantize: unsupported dtype %d", dtype);
    return gbh::E_BAD_ARG;
  }
  const int P = pieces((int)K, fmt), RB = row_bytes((int)K, fmt), size = dtype == DT_F32 ? 4 : 2;
  const int lanes = aligned_rows(y, K, K, size) ? 0 : K <= 256 ? 8 : 32;
  for (long long r0 = 0, n; r0 < rows; r0 += n) {
    n = rows_at_once(rows - r0, P);
    DequantArgs a{(const uint8_t*)data + r0 * RB, (const uint8_t*)scales + r0 / 128 * P * 512, (uint8_t*)y + r0 * K * size, (int)n, (int)K, P, RB, wide_rows(y, K, K, size),
                  FastDiv((uint32_t)(lanes == 32 ? (P + 3) / 4 : P))};
    cudaError_t e = cudaSuccess;
    auto go = [&](auto kern) { e = gbh::launch(kern, dim3(grid_of(n * a.by_units.d, kThreads / (lanes ? lanes : 8), 8)), dim3(kThreads), 0, (cudaStream_t)stream, 1, a); };
    GB_MX_DISPATCH(dtype, fmt, lanes == 0 ? go(mx_dequantize_kernel<T, FMT, 0>) : lanes == 8 ? go(mx_dequantize_kernel<T, FMT, 8>) : go(mx_dequantize_kernel<T, FMT, 32>))
    GB_CUDA_OK(e);
  }
  return gbh::E_OK;
}

// h = x + r (r null: h is x, and is not written), codes and scales of (x + r) / sqrt(mean((x + r)^2) + eps) * w.  x, r: rows ldx / ldr
// elements apart; w in x's type, or fp32 (w_f32); h contiguous.
GB_EXPORT int gb_mx_add_rms_norm(int dtype, int fmt, const void* x, long long ldx, const void* r, long long ldr, const void* w, int w_f32, void* h, void* data,
                                 void* scales, long long rows, long long K, double eps, void* stream) {
  if (bad_shape("gb_mx_add_rms_norm", x, rows, K, ldx < ldr ? ldx : ldr, fmt, data, scales)) return gbh::E_BAD_ARG;
  if (dtype != DT_BF16 && dtype != DT_F16 && dtype != DT_F32) {
    gbh::set_error("gb_mx_add_rms_norm: unsupported dtype %d", dtype);
    return gbh::E_BAD_ARG;
  }
  if (w == nullptr || (r != nullptr && h == nullptr)) {
    gbh::set_error("gb_mx_add_rms_norm: a weight, and with a residual room for the sum are needed");
    return gbh::E_BAD_ARG;
  }
  const int size = dtype == DT_F32 ? 4 : 2;
  const bool aligned = aligned_rows(x, ldx, K, size) && aligned_rows(w, K, K, 2) && (r == nullptr || (aligned_rows(r, ldr, K, size) && aligned_rows(h, K, K, size)));
  const bool wide = wide_rows(x, ldx, K, size) && (r == nullptr || (wide_rows(r, ldr, K, size) && wide_rows(h, K, K, size)));
  const NormArgs a{x, r, w, h, (uint8_t*)data, (uint8_t*)scales, ldx, ldr, (int)rows, (int)K, pieces((int)K, fmt), row_bytes((int)K, fmt), w_f32, wide, eps, 1.0 / (double)K,
                   extent_of(x, rows, ldx, K, size), extent_of(r, rows, ldr, K, size), extent_of(w, 1, K, K, w_f32 ? 4 : size)};
  cudaError_t e = cudaSuccess;
  GB_MX_DISPATCH(dtype, fmt, (e = aligned ? norm_launch<T, FMT, true>(a, (cudaStream_t)stream) : norm_launch<T, FMT, false>(a, (cudaStream_t)stream)))
  GB_CUDA_OK(e);
  return gbh::E_OK;
}
