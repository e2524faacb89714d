// Microscaled formats (OCP Microscaling 1.0): blocks of 32 values that share a power of two.
//
// A block's scale is 2^e with e = clamp(floor(log2(largest magnitude)) - E, -127, 127), held as e + 127 in a byte (E8M0); its
// values are v / 2^e rounded to nearest even, saturating: MXFP8 has E4M3 codes (E = 8, largest 448), MXFP4 E2M1 codes
// (E = 2, largest 6), two to a byte, the first in the lower half.  A block of zeros has e = -127.  A block that holds an
// infinity or a NaN has scale code 255, which makes every value of it NaN, here and in the tensor core.
//
// Codes: row-major, each row padded with zeros to whole blocks (32 or 16 bytes).  Scales: as the tensor core's copies into TMEM
// take them, in pieces of 512 bytes for 128 rows and four blocks (of 128 columns of the matrix), the pieces of a row
// of pieces behind one another; row r of a piece lies at byte 16 (r % 32) + 4 (r / 32).  A row of pieces covers whole 128-byte
// steps of the codes, so MXFP4 has an even number of pieces; the scales behind the last block are zeros.
#pragma once
#include "common.cuh"

#include <type_traits>

namespace gbmx {

enum Format : int { FP8 = 0, FP4 = 1 };

__host__ __device__ constexpr int pieces(int K, int fmt) { return fmt == FP8 ? (K + 127) / 128 : 2 * ((K + 255) / 256); }
__host__ __device__ constexpr int row_bytes(int K, int fmt) { return (K + 31) / 32 * (fmt == FP8 ? 32 : 16); }

// Where the four scales of columns 128 g .. 128 g + 127 of a row lie; P: pieces of a row of pieces.
__device__ __forceinline__ long long scale_word(long long row, int g, int P) {
  return ((row >> 7) * P + g) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// Products with powers of two must keep subnormal operands and results, which -ftz=true (part of --use_fast_math) would not.
__device__ __forceinline__ float mul_exact(float a, float b) {
  float d;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Two numbers at a time.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void parts_of(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// The scale code of a block whose largest magnitude has these bits (as fp32), and 1 / scale.  (Magnitudes compare as whole numbers:
// an infinity or a NaN is above all others, subnormal numbers are not lost.)
__device__ __forceinline__ uint32_t scale_code(uint32_t amax, int fmt) {
  const int c = (int)(amax >> 23) - (fmt == FP8 ? 8 : 2);
  return amax >= 0x7f800000u ? 255u : (uint32_t)max(c, 0);
}
__device__ __forceinline__ float scale_inverse(uint32_t code) { return code == 255u ? 0.f : __uint_as_float((254u - code) << 23); }
__device__ __forceinline__ float scale_value(uint32_t code) {
  return __uint_as_float(code == 255u ? 0x7fffffffu : code == 0u ? 0x00400000u : code << 23);      // (2^-127 is subnormal)
}

// Eight scaled values as codes: E4M3 in 8 bytes, E2M1 in 4.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n.reg .b16 lo, hi;\ncvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\ncvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\nmov.b32 %0, {lo, hi};\n}"
      : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
  uint32_t r;
  asm("{\n.reg .b8 b0, b1, b2, b3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      "mov.b32 %0, {b0, b1, b2, b3};\n}"
      : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// n / d for n below 2^31 by a multiplication (Granlund and Montgomery's division by invariant integers).
struct FastDiv {
  uint32_t d, m, s;
  __host__ explicit FastDiv(uint32_t div) : d(div), m(0), s(0) {
    while ((1ull << s) < d) s++;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

template <typename T> struct Elem;
template <> struct Elem<__nv_bfloat16> {     // (not by way of fp32 arithmetic, which would lose subnormal numbers)
  static constexpr int SZ = 2;
  static __device__ __forceinline__ void unpack(const uint32_t* w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; i++) { const float2 p = pair(w[i]); f[2 * i] = p.x; f[2 * i + 1] = p.y; }
  }
  static __device__ __forceinline__ float2 pair(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return gb::pack_bf16(a, b); }
  static __device__ __forceinline__ uint32_t bits(uint32_t h) { return h << 16; }
  static __device__ __forceinline__ float one(uint32_t h) { return __uint_as_float(bits(h)); }
};
template <> struct Elem<__half> {
  static constexpr int SZ = 2;
  static __device__ __forceinline__ void unpack(const uint32_t* w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; i++) { const float2 p = pair(w[i]); f[2 * i] = p.x; f[2 * i + 1] = p.y; }
  }
  static __device__ __forceinline__ float2 pair(uint32_t w) { return gb::unpack_f16(w); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return gb::pack_f16(a, b); }
  static __device__ __forceinline__ uint32_t bits(uint32_t h) { return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h))); }
  static __device__ __forceinline__ float one(uint32_t h) { return __uint_as_float(bits(h)); }
};
template <> struct Elem<float> {
  static constexpr int SZ = 4;
  static __device__ __forceinline__ void unpack(const uint32_t* w, float* f) {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ float one(uint32_t w) { return __uint_as_float(w); }
};

// Extent of a matrix in memory: vectors are read as long as they lie within it.
struct Extent {
  uintptr_t begin, end;
};

// Elements k .. k + 7 of a row of K (zeros behind its end) as raw words: W = 4 for 16-bit types, 8 for fp32.
// A row that does not start on a 16-byte boundary is read as the vectors around it, shifted.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int k, int K, const Extent& ext, uint32_t (&w)[2 * Elem<T>::SZ]) {
  constexpr int W = 2 * Elem<T>::SZ;                     // words of eight elements
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + k);
  const uint32_t o = at & 15;
  if (k + 8 <= K && o == 0) {
    const uint4* p = reinterpret_cast<const uint4*>(at);
#pragma unroll
    for (int i = 0; i < W / 4; i++) { const uint4 u = __ldg(p + i); w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w; }
    return;
  }
  const uintptr_t first = at & ~(uintptr_t)15;
  if (k + 8 <= K && first >= ext.begin && first + 4 * W + 16 <= ext.end) {
    uint32_t v[W + 5];
    const uint4* p = reinterpret_cast<const uint4*>(first);
#pragma unroll
    for (int i = 0; i < W / 4 + 1; i++) { const uint4 u = __ldg(p + i); v[4 * i] = u.x; v[4 * i + 1] = u.y; v[4 * i + 2] = u.z; v[4 * i + 3] = u.w; }
    v[W + 4] = 0;
    if (o & 8) {
#pragma unroll
      for (int i = 0; i < W + 2; i++) v[i] = v[i + 2];
    }
    if (o & 4) {
#pragma unroll
      for (int i = 0; i < W + 1; i++) v[i] = v[i + 1];
    }
#pragma unroll
    for (int i = 0; i < W; i++) w[i] = Elem<T>::SZ == 4 ? v[i] : __funnelshift_r(v[i], v[i + 1], (o & 2) * 8);
    return;
  }
#pragma unroll
  for (int i = 0; i < W; i++) w[i] = 0;
  if (Elem<T>::SZ == 4) {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (k + i < K) w[i % W] = __ldg(reinterpret_cast<const uint32_t*>(row) + k + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (k + i < K) w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(row) + k + i) << (16 * (i & 1));
  }
}

// Sixteen elements from k on as raw words.  Rows on 16-byte boundaries with K a multiple of eight (ALIGNED) are read in vectors, of
// 32 bytes where every row starts on such a boundary and K is a multiple of sixteen (wide).
template <typename T, bool ALIGNED>
__device__ __forceinline__ void load16(const T* row, int k, int K, bool wide, const Extent& ext, uint32_t (&w)[4 * Elem<T>::SZ]) {
  constexpr int W = 4 * Elem<T>::SZ;
  if constexpr (!ALIGNED) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      uint32_t u[W / 2];
      load8(row, k + 8 * h, K, ext, u);
#pragma unroll
      for (int i = 0; i < W / 2; i++) w[h * (W / 2) + i] = u[i];
    }
  } else if (wide) {
#pragma unroll
    for (int i = 0; i < W; i++) w[i] = 0;
    if (k < K) {
#pragma unroll
      for (int i = 0; i < W; i += 8)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]), "=r"(w[i + 6]), "=r"(w[i + 7])
                     : "l"(reinterpret_cast<const uint32_t*>(row + k) + i));
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (k + (i < W / 2 ? 0 : 8) < K) u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(row + k) + i);
      w[i] = u.x; w[i + 1] = u.y; w[i + 2] = u.z; w[i + 3] = u.w;
    }
  }
}
template <typename T>
__device__ __forceinline__ void unpack16(const uint32_t (&w)[4 * Elem<T>::SZ], float (&v)[16]) {
  Elem<T>::unpack(w, v);
  Elem<T>::unpack(w + 2 * Elem<T>::SZ, v + 8);
}

// Sixteen values to consecutive elements on a 16-byte boundary (wide: 32), of which those from K on are left out (whole vectors of eight).  A
// store of 32 bytes fills a sector, two of 16 write it twice: 50304 x 2048 bf16 into MXFP4 and back 115 us with two, 97 with one.
__device__ __forceinline__ void store8(void* to, bool wide, const uint32_t* w) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(to)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(to)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
template <typename T>
__device__ __forceinline__ void store16(T* row, int k, int K, bool wide, const float (&v)[16]) {
  if (k >= K) return;
  uint32_t w[4 * Elem<T>::SZ];
#pragma unroll
  for (int i = 0; i < 4 * Elem<T>::SZ; i++) {
    if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
    else w[i] = Elem<T>::pack(v[2 * i], v[2 * i + 1]);
  }
  uint32_t* to = reinterpret_cast<uint32_t*>(row + k);
  if constexpr (sizeof(T) == 4) {
    store8(to, wide, w);
    if (k + 8 < K) store8(to + 8, wide, w + 8);
  } else if (k + 8 < K) {
    store8(to, wide, w);
  } else {
    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// Rows at any address, by way of shared memory: L lanes side by side hold 16 L consecutive columns, which come and go a column a lane and
// step, so that loads and stores are of neighbours whatever they start on, and stand in shared memory as sixteen a lane, 16 bytes
// between them (no bank is met twice).
template <typename T, int L>
struct Stage {
  static constexpr int PITCH = 16 * sizeof(T) + 16, BYTES = L * PITCH;     // of a group of L lanes
  using Bits = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
  uint8_t* buf;
  int lane;
  unsigned mask;
  // for a block's shared memory of THREADS / L groups
  __device__ __forceinline__ explicit Stage(uint8_t* shared)
      : buf(shared + threadIdx.x / L * BYTES), lane(threadIdx.x % L), mask(L == 32 ? 0xffffffffu : ((1u << L) - 1u) << (threadIdx.x & 31 & ~(L - 1))) {}
  __device__ __forceinline__ uint8_t* at(int j) const { return buf + ((j * L + lane) >> 4) * PITCH + ((j * L + lane) & 15) * sizeof(T); }
  // columns first + j L + lane of the group's row
  static __device__ __forceinline__ void fetch(const T* row, int first, int K, int lane, Bits (&raw)[16]) {
#pragma unroll
    for (int j = 0; j < 16; j++) raw[j] = first + j * L + lane < K ? __ldg(reinterpret_cast<const Bits*>(row) + first + j * L + lane) : (Bits)0;
  }
  // into sixteen columns a lane, as load16 has them
  __device__ __forceinline__ void turn(const Bits (&raw)[16], uint32_t (&w)[4 * Elem<T>::SZ]) const {
    __syncwarp(mask);
#pragma unroll
    for (int j = 0; j < 16; j++) *reinterpret_cast<Bits*>(at(j)) = raw[j];
    __syncwarp(mask);
#pragma unroll
    for (int i = 0; i < 4 * Elem<T>::SZ; i += 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(buf + lane * PITCH + i * 4);
      w[i] = u.x; w[i + 1] = u.y; w[i + 2] = u.z; w[i + 3] = u.w;
    }
  }
  // sixteen values a lane to the row's columns from `first` on
  __device__ __forceinline__ void store(T* row, int first, int K, const float (&v)[16]) const {
    __syncwarp(mask);
#pragma unroll
    for (int i = 0; i < 4 * Elem<T>::SZ; i += 4) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(v[i + k]);
        else w[k] = Elem<T>::pack(v[2 * (i + k)], v[2 * (i + k) + 1]);
      }
      *reinterpret_cast<uint4*>(buf + lane * PITCH + i * 4) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncwarp(mask);
#pragma unroll
    for (int j = 0; j < 16; j++)
      if (first + j * L + lane < K) reinterpret_cast<Bits*>(row)[first + j * L + lane] = *reinterpret_cast<const Bits*>(at(j));
  }
};

// Bits of the largest magnitude of sixteen elements.  16-bit magnitudes compare in pairs, as whole numbers.
template <typename T>
__device__ __forceinline__ uint32_t largest16(const uint32_t (&w)[4 * Elem<T>::SZ]) {
  if constexpr (Elem<T>::SZ == 2) {
    uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 8; i++) asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
    return Elem<T>::bits(max(m >> 16, m & 0xffffu));
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) m = max(m, w[i] & 0x7fffffffu);
    return m;
  }
}
// The same of sixteen numbers (NaN if there is one; keeps subnormal numbers).
__device__ __forceinline__ uint32_t largest16(const float (&v)[16]) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < 15; i += 2) asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(v[i])), "f"(fabsf(v[i + 1])));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v[15])));
  return __float_as_uint(m);
}

// Sixteen values of a lane, two lanes to a block, eight (all of them here) to 128 columns; amax: bits of the largest magnitude of the
// lane's.  Codes of the lane in `out` (two words for FP4), the scales of the four blocks as a word in every lane.
template <int FMT>
__device__ __forceinline__ uint32_t quantize16(const float (&v)[16], uint32_t amax, unsigned mask, int lane, uint32_t (&out)[4]) {
  amax = max(amax, __shfl_xor_sync(mask, amax, 1));
  const uint32_t code = scale_code(amax, FMT);
  const uint64_t inv = pair_of(scale_inverse(code), scale_inverse(code));
  float q[16];
#pragma unroll
  for (int i = 0; i < 16; i += 2) parts_of(mul_pair(pair_of(v[i], v[i + 1]), inv), q[i], q[i + 1]);
  if (FMT == FP8) {
#pragma unroll
    for (int i = 0; i < 4; i++) out[i] = e4m3x4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
  } else {
    out[0] = e2m1x8(q);
    out[1] = e2m1x8(q + 8);
  }
  uint32_t word = code << (8 * ((lane >> 1) & 3));
  word |= __shfl_xor_sync(mask, word, 2);
  word |= __shfl_xor_sync(mask, word, 4);
  return word;
}
// Codes of columns k .. k + 15 of a row.
template <int FMT>
__device__ __forceinline__ void store_codes(uint8_t* row, int k, int row_bytes, const uint32_t (&c)[4]) {
  const int b = FMT == FP8 ? k : k / 2;
  if (b >= row_bytes) return;
  if (FMT == FP8) *reinterpret_cast<uint4*>(row + b) = make_uint4(c[0], c[1], c[2], c[3]);
  else *reinterpret_cast<uint2*>(row + b) = make_uint2(c[0], c[1]);
}

}  // namespace gbmx
