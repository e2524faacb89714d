// Microscaled quantisation (formats: mx.cuh): rows of a tensor into codes and scales, back into values, and the residual's
// addition with the root-mean-square norm whose output is quantised where it is made.
//
// All three are bound by memory.  Sixteen lanes hold 128 columns, eight each: 16-byte loads of 16-bit types, a block's largest
// magnitude by two shuffles over its four lanes, its scales as one word by two more, codes of 8 or 4 bytes a lane in whole lines.
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
  int rows, K, pieces, row_bytes;
  FastDiv by_pieces;
  Extent ext;
};

// A unit is 128 columns of a row, taken by sixteen lanes; NU units of a lane are in flight.
template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) mx_quantize_kernel(const QuantArgs a) {
  constexpr int NU = 2;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, l16 = threadIdx.x & 15;
  const unsigned mask = 0xffffu << (lane & 16);
  const uint32_t units = (uint32_t)a.rows * (uint32_t)a.pieces, stride = gridDim.x * (kThreads / 16);
  for (uint32_t u0 = blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4); u0 < units; u0 += NU * stride) {
    uint32_t w[NU][2 * Elem<T>::SZ];
    uint32_t row[NU];
    int g[NU];
#pragma unroll
    for (int i = 0; i < NU; i++) {
      const uint32_t u = u0 + i * stride;
      row[i] = a.by_pieces.div(u < units ? u : u0);
      g[i] = (int)((u < units ? u : u0) - row[i] * a.by_pieces.d);
      load8(reinterpret_cast<const T*>(a.x) + row[i] * a.ld, g[i] * 128 + l16 * 8, a.K, a.ext, w[i]);
    }
#pragma unroll
    for (int i = 0; i < NU; i++) {
      if (u0 + i * stride >= units) break;
      float v[8];
      Elem<T>::unpack(w[i], v);
      uint32_t out[2];
      const uint32_t word = quantize8(v, FMT, mask, lane, out);
      const int b = (g[i] * 128 + l16 * 8) / (FMT == FP8 ? 1 : 2);
      if (b < a.row_bytes) {
        uint8_t* to = a.data + (long long)row[i] * a.row_bytes + b;
        if (FMT == FP8) *reinterpret_cast<uint2*>(to) = make_uint2(out[0], out[1]);
        else *reinterpret_cast<uint32_t*>(to) = out[0];
      }
      if (l16 == 0) *reinterpret_cast<uint32_t*>(a.scales + scale_word(row[i], g[i], a.pieces)) = word;
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
  int rows, K, pieces, row_bytes, pieces_t, row_bytes_t;
  Extent ext;
};

// A block takes 128 x 128 values, so that its scales are one piece of either result.  Rows are quantised as they arrive; the tile
// then stands in shared memory, a thread quantises two columns of 32 rows, and their codes leave by way of shared memory as
// 128-byte pieces of the transpose's rows.
template <typename T>
struct BothCfg {
  static constexpr int TILE = 128 * 128 * Elem<T>::SZ, PITCH = 128 + 16;
  static constexpr int BYTES = TILE + 128 * PITCH + 1024;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) mx_quantize_both_kernel(const BothArgs a) {
  using C = BothCfg<T>;
  constexpr int W = 2 * Elem<T>::SZ;                     // words of eight elements
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* codes = smem + C::TILE;
  uint32_t* piece = reinterpret_cast<uint32_t*>(codes + 128 * C::PITCH);
  uint8_t* piece_t = reinterpret_cast<uint8_t*>(piece + 128);
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, l16 = threadIdx.x & 15, h = threadIdx.x >> 4;
  const int g = blockIdx.x % a.pieces, gt = blockIdx.x / a.pieces;       // pieces along the columns and the rows
  const int k = g * 128 + l16 * 8;
#pragma unroll 4
  for (int i = 0; i < 8; i++) {
    const int r = h + 16 * i;
    const long long row = gt * 128LL + r;
    uint32_t w[W];
#pragma unroll
    for (int j = 0; j < W; j++) w[j] = 0;
    if (row < a.rows) load8(reinterpret_cast<const T*>(a.x) + row * a.ld, k, a.K, a.ext, w);
#pragma unroll
    for (int j = 0; j < W; j += 4) *reinterpret_cast<uint4*>(smem + (r * 128 + l16 * 8) * Elem<T>::SZ + j * 4) = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
    float v[8];
    Elem<T>::unpack(w, v);
    uint32_t out[2];
    const uint32_t word = quantize8(v, FP8, 0xffffu << (lane & 16), lane, out);
    if (row < a.rows && k < a.row_bytes) *reinterpret_cast<uint2*>(a.data + row * a.row_bytes + k) = make_uint2(out[0], out[1]);
    if (l16 == 0) piece[(r & 31) * 4 + (r >> 5)] = word;
  }
  __syncthreads();
  // columns 2 p and 2 p + 1, rows 32 b .. 32 b + 31
  const int p = threadIdx.x & 63, b = threadIdx.x >> 6;
  float x0[32], x1[32];
  uint32_t m0 = 0, m1 = 0;
#pragma unroll
  for (int i = 0; i < 32; i++) {
    const uint8_t* at = smem + ((b * 32 + i) * 128 + p * 2) * Elem<T>::SZ;
    if constexpr (Elem<T>::SZ == 4) {
      const float2 f = *reinterpret_cast<const float2*>(at);
      x0[i] = f.x; x1[i] = f.y;
    } else if constexpr (sizeof(T) == 2) {
      const uint32_t u = *reinterpret_cast<const uint32_t*>(at);
      const float2 f = Elem<T>::pair(u);
      x0[i] = f.x; x1[i] = f.y;
    }
    m0 = max(m0, __float_as_uint(x0[i]) & 0x7fffffffu);
    m1 = max(m1, __float_as_uint(x1[i]) & 0x7fffffffu);
  }
  const uint32_t c0 = scale_code(m0, FP8), c1 = scale_code(m1, FP8);
  const float i0 = scale_inverse(c0), i1 = scale_inverse(c1);
#pragma unroll
  for (int c = 0; c < 2; c++) {
    const float (&x)[32] = c == 0 ? x0 : x1;
    const float inv = c == 0 ? i0 : i1;
    uint32_t q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = e4m3x4(mul_exact(x[4 * i], inv), mul_exact(x[4 * i + 1], inv), mul_exact(x[4 * i + 2], inv), mul_exact(x[4 * i + 3], inv));
    const int col = 2 * p + c;
    uint4* to = reinterpret_cast<uint4*>(codes + col * C::PITCH + b * 32);
    to[0] = make_uint4(q[0], q[1], q[2], q[3]);
    to[1] = make_uint4(q[4], q[5], q[6], q[7]);
    piece_t[(col & 31) * 16 + (col >> 5) * 4 + b] = (uint8_t)(c == 0 ? c0 : c1);
  }
  __syncthreads();
  if (threadIdx.x < 128) reinterpret_cast<uint32_t*>(a.scales + ((long long)gt * a.pieces + g) * 512)[threadIdx.x] = piece[threadIdx.x];
  else reinterpret_cast<uint32_t*>(a.scales_t + ((long long)g * a.pieces_t + gt) * 512)[threadIdx.x - 128] = reinterpret_cast<const uint32_t*>(piece_t)[threadIdx.x - 128];
  const int at = gt * 128 + (threadIdx.x & 7) * 16;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int col = (threadIdx.x >> 3) + 32 * i;
    if (g * 128 + col < a.K && at < a.row_bytes_t)
      *reinterpret_cast<uint4*>(a.data_t + (g * 128LL + col) * a.row_bytes_t + at) = *reinterpret_cast<const uint4*>(codes + col * C::PITCH + (threadIdx.x & 7) * 16);
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// codes and scales into values
// ---------------------------------------------------------------------------------------------------------------------------
struct DequantArgs {
  const uint8_t* data;
  const uint8_t* scales;
  void* y;                 // rows x K, contiguous
  int rows, K, pieces, row_bytes;
  FastDiv by_pieces;
};

template <typename T>
__device__ __forceinline__ T to_type(float v);
template <> __device__ __forceinline__ float to_type<float>(float v) { return v; }
template <> __device__ __forceinline__ __half to_type<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 to_type<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) mx_dequantize_kernel(const DequantArgs a) {
  pdl_trigger();
  pdl_wait();
  const int l16 = threadIdx.x & 15;
  const uint32_t units = (uint32_t)a.rows * (uint32_t)a.pieces, stride = gridDim.x * (kThreads / 16);
  for (uint32_t u = blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4); u < units; u += stride) {
    const uint32_t row = a.by_pieces.div(u);
    const int g = (int)(u - row * a.by_pieces.d), k = g * 128 + l16 * 8;
    if (k >= a.K) continue;
    const uint8_t* from = a.data + (long long)row * a.row_bytes + k / (FMT == FP8 ? 1 : 2);
    const float s = scale_value(__ldg(a.scales + scale_word(row, g, a.pieces) + (l16 >> 2)));
    float v[8];
    if (FMT == FP8) {
      const uint2 c = __ldg(reinterpret_cast<const uint2*>(from));
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t two = ((i < 2 ? c.x : c.y) >> (16 * (i & 1))) & 0xffffu;
        uint32_t h;
        asm("{\n.reg .b16 t;\ncvt.u16.u32 t, %1;\ncvt.rn.f16x2.e4m3x2 %0, t;\n}" : "=r"(h) : "r"(two));
        const float2 f = unpack_f16(h);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    } else {
      const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(from));
#pragma unroll
      for (int i = 0; i < 4; i++) {
        uint32_t h;
        asm("{\n.reg .b8 t, u0, u1, u2;\nmov.b32 {t, u0, u1, u2}, %1;\ncvt.rn.f16x2.e2m1x2 %0, t;\n}" : "=r"(h) : "r"(c >> (8 * i)));
        const float2 f = unpack_f16(h);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = mul_exact(v[i], s);
    T* to = reinterpret_cast<T*>(a.y) + (long long)row * a.K + k;
    if (k + 8 <= a.K && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        *reinterpret_cast<uint4*>(to) = make_uint4(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]), Elem<T>::pack(v[4], v[5]), Elem<T>::pack(v[6], v[7]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (k + i < a.K) to[i] = to_type<T>(v[i]);
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
  int rows, K, pieces, row_bytes, w_f32, fmt;
  float eps;
  Extent ex, er, ew;
};

// The sum of a row in fp32; its inverse root in fp64 and rounded once (approximations of a last bit would move a row's values
// over the borders between codes more often than the roundings of the two products do).
__device__ __forceinline__ float inverse_root(float sum, int K, float eps) { return (float)(1.0 / sqrt((double)sum / K + (double)eps)); }

template <typename T>
__device__ __forceinline__ void weights8(const NormArgs& a, int k, float* f) {
  if (a.w_f32) {
    uint32_t u[8];
    load8(reinterpret_cast<const float*>(a.w), k, a.K, a.ew, u);
    Elem<float>::unpack(u, f);
  } else {
    uint32_t u[2 * Elem<T>::SZ];
    load8(reinterpret_cast<const T*>(a.w), k, a.K, a.ew, u);
    Elem<T>::unpack(u, f);
  }
}

// x + r of eight columns, in fp32 and unrounded for the norm, rounded into h.
template <typename T>
__device__ __forceinline__ void sum8(const NormArgs& a, long long row, int k, bool write, float* v) {
  uint32_t u[2 * Elem<T>::SZ];
  load8(reinterpret_cast<const T*>(a.x) + row * a.ldx, k, a.K, a.ex, u);
  Elem<T>::unpack(u, v);
  if (a.r == nullptr) return;
  float f[8];
  load8(reinterpret_cast<const T*>(a.r) + row * a.ldr, k, a.K, a.er, u);
  Elem<T>::unpack(u, f);
#pragma unroll
  for (int i = 0; i < 8; i++) asm("add.rn.f32 %0, %1, %2;" : "=f"(v[i]) : "f"(v[i]), "f"(f[i]));     // (keeps subnormal sums)
  if (!write || k >= a.K) return;
  T* to = reinterpret_cast<T*>(a.h) + row * a.K + k;
  if (k + 8 <= a.K && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(to) = make_uint4(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]), Elem<T>::pack(v[4], v[5]), Elem<T>::pack(v[6], v[7]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (k + i < a.K) to[i] = to_type<T>(v[i]);
  }
}

template <typename T>
__device__ __forceinline__ void norm8(const NormArgs& a, long long row, int k, float* v, float rstd) {
  float w[8];
  weights8<T>(a, k, w);
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = mul_exact(mul_exact(v[i], rstd), w[i]);
  uint32_t out[2];
  const int lane = threadIdx.x & 31;
  const uint32_t word = quantize8(v, a.fmt, 0xffffu << (lane & 16), lane, out);
  const int b = k / (a.fmt == FP8 ? 1 : 2);
  if (b < a.row_bytes) {
    uint8_t* to = a.data + row * a.row_bytes + b;
    if (a.fmt == FP8) *reinterpret_cast<uint2*>(to) = make_uint2(out[0], out[1]);
    else *reinterpret_cast<uint32_t*>(to) = out[0];
  }
  if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(a.scales + scale_word(row, k >> 7, a.pieces)) = word;
}

template <int G>
__device__ __forceinline__ float row_sum(float s, float* red) {
  s = warp_sum(s);
  if (G == 32) return s;
  // the row's warps: their sums in one order, the same for every thread
  const int warp = threadIdx.x >> 5, first = (threadIdx.x / G) * (G / 32);
  if ((threadIdx.x & 31) == 0) red[warp] = s;
  __syncthreads();
  s = 0.f;
#pragma unroll
  for (int i = 0; i < G / 32; i++) s += red[first + i];
  __syncthreads();
  return s;
}

// G threads of a block take a row, VPT vectors of eight columns each, which stay in registers between the two passes.  VPT = 0: rows
// of any length, read a second time for their codes.
template <typename T, int G, int VPT>
__global__ void __launch_bounds__(G > kThreads ? G : kThreads) mx_norm_kernel(const NormArgs a) {
  __shared__ float red[32];
  pdl_trigger();
  pdl_wait();
  const int t = threadIdx.x % G;
  const int vecs = a.pieces * 16;                        // whole pieces: sixteen lanes work together
  const int per = blockDim.x / G;
  for (long long first = (long long)blockIdx.x * per; first < a.rows; first += (long long)gridDim.x * per) {
    const long long row = first + threadIdx.x / G;
    const bool live = row < a.rows;
    float s = 0.f;
    if constexpr (VPT > 0) {
      float v[VPT][8];
#pragma unroll
      for (int i = 0; i < VPT; i++)
        if (live && t + i * G < vecs) {
          sum8<T>(a, row, (t + i * G) * 8, true, v[i]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) v[i][j] = 0.f;
        }
#pragma unroll
      for (int i = 0; i < VPT; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) s = fmaf(v[i][j], v[i][j], s);
      const float rstd = inverse_root(row_sum<G>(s, red), a.K, a.eps);
#pragma unroll
      for (int i = 0; i < VPT; i++)
        if (live && t + i * G < vecs) norm8<T>(a, row, (t + i * G) * 8, v[i], rstd);
    } else {
      if (live)
        for (int i = t; i < vecs; i += G) {
          float v[8];
          sum8<T>(a, row, i * 8, true, v);
#pragma unroll
          for (int j = 0; j < 8; j++) s = fmaf(v[j], v[j], s);
        }
      const float rstd = inverse_root(row_sum<G>(s, red), a.K, a.eps);
      if (live)
        for (int i = t; i < vecs; i += G) {
          float v[8];
          sum8<T>(a, row, i * 8, false, v);
          norm8<T>(a, row, i * 8, v, rstd);
        }
    }
  }
}

Extent extent_of(const void* p, long long rows, long long ld, long long K, int size) {
  Extent e;
  e.begin = reinterpret_cast<uintptr_t>(p);
  e.end = e.begin + (uintptr_t)(((rows - 1) * ld + K) * size);
  return e;
}

bool bad_shape(const char* what, long long rows, long long K, long long ld, int fmt, const void* data, const void* scales) {
  if (rows <= 0 || K <= 0 || rows > 0x7fffffffLL || K > (1LL << 30) || ld < 0 || (fmt != FP8 && fmt != FP4)) {
    gbh::set_error("%s: bad extents %lld x %lld, row pitch %lld, format %d", what, rows, K, ld, fmt);
    return true;
  }
  if (((uintptr_t)data & 15) || ((uintptr_t)scales & 15)) {
    gbh::set_error("%s: codes and scales must be 16-byte aligned", what);
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

template <typename T>
int norm_launch(const NormArgs& a, cudaStream_t st) {
  const int vecs = a.pieces * 16;
  auto go = [&](auto kern, int G, int threads) {
    const int per = threads / G;
    const long long blocks = ((long long)a.rows + per - 1) / per, most = 148LL * (2048 / threads);
    return gbh::launch(kern, dim3((unsigned)(blocks < most ? blocks : most)), dim3(threads), 0, st, 1, a);
  };
  // few rows: a row's loads over as many threads as it has vectors
  const bool few = a.rows <= 2 * 148;
  cudaError_t e;
  if (vecs <= 32) e = go(mx_norm_kernel<T, 32, 1>, 32, kThreads);
  else if (vecs <= 64 && !few) e = go(mx_norm_kernel<T, 32, 2>, 32, kThreads);
  else if (vecs <= 128 && !few) e = go(mx_norm_kernel<T, 32, 4>, 32, kThreads);
  else if (vecs <= 256) e = go(mx_norm_kernel<T, 256, 1>, 256, 256);
  else if (vecs <= 512) e = go(mx_norm_kernel<T, 256, 2>, 256, 256);
  else if (vecs <= 1024) e = go(mx_norm_kernel<T, 256, 4>, 256, 256);
  else if (vecs <= 4096) e = go(mx_norm_kernel<T, 1024, 4>, 1024, 1024);
  else e = go(mx_norm_kernel<T, 1024, 0>, 1024, 1024);
  GB_CUDA_OK(e);
  return gbh::E_OK;
}

}  // namespace

enum { DT_BF16 = 0, DT_F16 = 1, DT_F32 = 2 };

// Bytes of a row of codes and of the scales of a matrix (fmt 0: MXFP8, 1: MXFP4).
GB_EXPORT long long gb_mx_row_bytes(long long K, int fmt) { return K <= 0 || K > (1LL << 30) ? 0 : row_bytes((int)K, fmt); }
GB_EXPORT long long gb_mx_scale_bytes(long long rows, long long K, int fmt) {
  return K <= 0 || K > (1LL << 30) ? 0 : (rows + 127) / 128 * pieces((int)K, fmt) * 512;
}

// Codes and scales of x (rows x K, rows `ld` elements apart).  The scales of rows up to the next multiple of 128 are left as they were.
GB_EXPORT int gb_mx_quantize(int dtype, int fmt, const void* x, long long ld, void* data, void* scales, long long rows, long long K, void* stream) {
  if (bad_shape("gb_mx_quantize", rows, K, ld, fmt, data, scales)) return gbh::E_BAD_ARG;
  if (dtype != DT_BF16 && dtype != DT_F16 && dtype != DT_F32) {
    gbh::set_error("gb_mx_quantize: unsupported dtype %d", dtype);
    return gbh::E_BAD_ARG;
  }
  const int P = pieces((int)K, fmt), RB = row_bytes((int)K, fmt), size = dtype == DT_F32 ? 4 : 2;
  for (long long r0 = 0, n; r0 < rows; r0 += n) {
    n = rows_at_once(rows - r0, P);
    QuantArgs a{(const uint8_t*)x + r0 * ld * size, (uint8_t*)data + r0 * RB, (uint8_t*)scales + r0 / 128 * P * 512, ld, (int)n, (int)K, P, RB, FastDiv((uint32_t)P),
                extent_of(x, rows, ld, K, size)};
    auto go = [&](auto kern) { return gbh::launch(kern, dim3(grid_of(n * P, kThreads / 16, 8)), dim3(kThreads), 0, (cudaStream_t)stream, 1, a); };
    if (dtype == DT_BF16) GB_CUDA_OK(fmt == FP8 ? go(mx_quantize_kernel<__nv_bfloat16, FP8>) : go(mx_quantize_kernel<__nv_bfloat16, FP4>));
    else if (dtype == DT_F16) GB_CUDA_OK(fmt == FP8 ? go(mx_quantize_kernel<__half, FP8>) : go(mx_quantize_kernel<__half, FP4>));
    else GB_CUDA_OK(fmt == FP8 ? go(mx_quantize_kernel<float, FP8>) : go(mx_quantize_kernel<float, FP4>));
  }
  return gbh::E_OK;
}

// Codes and scales (MXFP8) of x (rows x K, rows `ld` elements apart) along its columns, and of its transpose along the rows.
GB_EXPORT int gb_mx_quantize_both(int dtype, const void* x, long long ld, void* data, void* scales, void* data_t, void* scales_t, long long rows, long long K, void* stream) {
  if (bad_shape("gb_mx_quantize_both", rows, K, ld, FP8, data, scales) || bad_shape("gb_mx_quantize_both", K, rows, ld, FP8, data_t, scales_t)) return gbh::E_BAD_ARG;
  const int P = pieces((int)K, FP8), PT = pieces((int)rows, FP8);
  const long long blocks = (long long)P * PT;
  if (blocks > 0x7fffffffLL) {
    gbh::set_error("gb_mx_quantize_both: %lld x %lld is too large", rows, K);
    return gbh::E_TOO_LARGE;
  }
  auto go = [&](auto kern, int bytes, int size, std::atomic<uint32_t>& done) -> int {
    int dev = 0;
    GB_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 32 || !(done.load() >> dev & 1u)) {       // more shared memory than 48 KB: once per device
      GB_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
      if (dev < 32) done.fetch_or(1u << dev);
    }
    BothArgs a{x, (uint8_t*)data, (uint8_t*)scales, (uint8_t*)data_t, (uint8_t*)scales_t, ld, (int)rows, (int)K, P, row_bytes((int)K, FP8), PT, row_bytes((int)rows, FP8),
               extent_of(x, rows, ld, K, size)};
    GB_CUDA_OK(gbh::launch(kern, dim3((unsigned)blocks), dim3(kThreads), bytes, (cudaStream_t)stream, 1, a));
    return gbh::E_OK;
  };
  static std::atomic<uint32_t> done[3];
  switch (dtype) {
    case DT_BF16: return go(mx_quantize_both_kernel<__nv_bfloat16>, BothCfg<__nv_bfloat16>::BYTES, 2, done[0]);
    case DT_F16: return go(mx_quantize_both_kernel<__half>, BothCfg<__half>::BYTES, 2, done[1]);
    case DT_F32: return go(mx_quantize_both_kernel<float>, BothCfg<float>::BYTES, 4, done[2]);
    default: gbh::set_error("gb_mx_quantize_both: unsupported dtype %d", dtype); return gbh::E_BAD_ARG;
  }
}

// The values (rows x K, contiguous) that codes and scales stand for.
GB_EXPORT int gb_mx_dequantize(int dtype, int fmt, const void* data, const void* scales, void* y, long long rows, long long K, void* stream) {
  if (bad_shape("gb_mx_dequantize", rows, K, K, fmt, data, scales)) return gbh::E_BAD_ARG;
  if (dtype != DT_BF16 && dtype != DT_F16 && dtype != DT_F32) {
    gbh::set_error("gb_mx_dequantize: unsupported dtype %d", dtype);
    return gbh::E_BAD_ARG;
  }
  const int P = pieces((int)K, fmt), RB = row_bytes((int)K, fmt), size = dtype == DT_F32 ? 4 : 2;
  for (long long r0 = 0, n; r0 < rows; r0 += n) {
    n = rows_at_once(rows - r0, P);
    DequantArgs a{(const uint8_t*)data + r0 * RB, (const uint8_t*)scales + r0 / 128 * P * 512, (uint8_t*)y + r0 * K * size, (int)n, (int)K, P, RB, FastDiv((uint32_t)P)};
    auto go = [&](auto kern) { return gbh::launch(kern, dim3(grid_of(n * P, kThreads / 16, 8)), dim3(kThreads), 0, (cudaStream_t)stream, 1, a); };
    if (dtype == DT_BF16) GB_CUDA_OK(fmt == FP8 ? go(mx_dequantize_kernel<__nv_bfloat16, FP8>) : go(mx_dequantize_kernel<__nv_bfloat16, FP4>));
    else if (dtype == DT_F16) GB_CUDA_OK(fmt == FP8 ? go(mx_dequantize_kernel<__half, FP8>) : go(mx_dequantize_kernel<__half, FP4>));
    else GB_CUDA_OK(fmt == FP8 ? go(mx_dequantize_kernel<float, FP8>) : go(mx_dequantize_kernel<float, FP4>));
  }
  return gbh::E_OK;
}

// h = x + r (r null: h is x, and is not written), codes and scales of h / sqrt(mean(h^2) + eps) * w.  x, r: rows ldx / ldr
// elements apart; w in x's type, or fp32 (w_f32); h contiguous.
GB_EXPORT int gb_mx_add_rms_norm(int dtype, int fmt, const void* x, long long ldx, const void* r, long long ldr, const void* w, int w_f32, void* h, void* data,
                                 void* scales, long long rows, long long K, float eps, void* stream) {
  if (bad_shape("gb_mx_add_rms_norm", rows, K, ldx < ldr ? ldx : ldr, fmt, data, scales)) return gbh::E_BAD_ARG;
  if (dtype != DT_BF16 && dtype != DT_F16 && dtype != DT_F32) {
    gbh::set_error("gb_mx_add_rms_norm: unsupported dtype %d", dtype);
    return gbh::E_BAD_ARG;
  }
  const int size = dtype == DT_F32 ? 4 : 2;
  NormArgs a{x, r, w, h, (uint8_t*)data, (uint8_t*)scales, ldx, ldr, (int)rows, (int)K, pieces((int)K, fmt), row_bytes((int)K, fmt), w_f32 || dtype == DT_F32, fmt, eps,
             extent_of(x, rows, ldx, K, size), extent_of(r, rows, ldr, K, size), extent_of(w, 1, K, K, w_f32 ? 4 : size)};
  if (dtype == DT_BF16) return norm_launch<__nv_bfloat16>(a, (cudaStream_t)stream);
  if (dtype == DT_F16) return norm_launch<__half>(a, (cudaStream_t)stream);
  return norm_launch<float>(a, (cudaStream_t)stream);
}
