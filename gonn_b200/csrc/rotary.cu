// Rotary positions, and the same on the way into a paged cache of keys and values.
//
// A pair (a, b) of a head at position p becomes (a cos - b sin, a sin + b cos) * amplitude with the angle p w_i; pairs are
// (i, i + dim / 2) or (2 i, 2 i + 1), columns from dim on are copied.  The gradient is the same kernel with the opposite angle.
//
// Angles.  p w in fp32 is off by p 2^-24: by 0.008 at position 131 072, twice a bf16's last bit.  So a frequency is held as the fraction
// w / 2 pi of a turn in 64 bits of fixed point, and p times it, modulo 2^64, is the fraction of a turn that is left: an integer
// product whose overflow is the reduction, off by p 2^-65 turns.  Its upper 32 bits become a float in half turns (off by 2^-25) for
// sincospif.  No table: sine and cosine of a token are taken once per CTA, in shared memory, and serve all of its heads.
//
// What bounds it: memory, every element read and written once.  A CTA takes a few tokens with all of their heads, a thread two
// vectors of 16 bytes (narrower ones where a size or an address is odd): the two halves of its pairs.
#include "common.cuh"

using namespace gb;

namespace {

constexpr int kThreads = 256;
constexpr int kAngles = 1024;         // sines and cosines that a CTA holds
constexpr int kMaxTokens = 16;

struct Part {                         // a tensor (batch, tokens, heads, width) and where its rows go
  const void* src;
  void* dst;                          // (batch, tokens, heads, width), contiguous; a cache for keys and values
  long long sb, st, sh;               // strides of src in elements
  long long dp, dh, dr;               // strides of a cache: page, head, row
  int heads;
};

struct RotaryArgs {
  Part q, k, v;
  int batch, tokens, width, dim;      // dim: columns that are turned, even
  int half, vec;                      // dim / 2; elements of a vector
  const unsigned long long* turns;    // [half] fractions of a turn a position, times 2^64
  float amplitude;
  int back;                           // turn the other way
  // rotary alone: positions of the tokens
  const void* positions;              // null: 0, 1, ..
  int positions64;
  long long pb, pt;                   // strides, 0 where all share one
  // append
  const int* table;
  long long table_stride;
  int columns, pages, page;
  const int* lengths;
  const int* counts;                  // null: all tokens count
  int* status;
  int per_cta;                        // tokens of a CTA
  int early;
};

template <int BYTES> struct VecOf;
template <> struct VecOf<16> { using type = uint4; };
template <> struct VecOf<8> { using type = uint2; };
template <> struct VecOf<4> { using type = uint32_t; };
template <> struct VecOf<2> { using type = uint16_t; };

template <typename T, int V>
struct Pack {
  T e[V];
  __device__ __forceinline__ void load(const T* p) { *reinterpret_cast<typename VecOf<V * sizeof(T)>::type*>(e) = __ldg(reinterpret_cast<const typename VecOf<V * sizeof(T)>::type*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<typename VecOf<V * sizeof(T)>::type*>(p) = *reinterpret_cast<const typename VecOf<V * sizeof(T)>::type*>(e); }
};

__device__ __forceinline__ float2 angle_of(unsigned long long turns, long long position, float amplitude, bool back) {
  const unsigned long long phase = turns * (unsigned long long)position;
  float s, c;
  sincospif((float)(int)(phase >> 32) * 4.656612873077393e-10f, &s, &c);       // 2^-31: half turns in [-1, 1)
  return make_float2(c * amplitude, (back ? -s : s) * amplitude);
}

// Two vectors of pairs turned: halves of a head apart, or one behind the other with each pair side by side.
template <typename T, int V, bool INTER>
__device__ __forceinline__ void turn(Pack<T, V>& u, Pack<T, V>& w, const float2* cs) {
#pragma unroll
  for (int j = 0; j < V; j++) {
    float2 t = cs[j];
    if constexpr (!INTER) {
      const float a = (float)u.e[j], b = (float)w.e[j];
      u.e[j] = (T)(a * t.x - b * t.y);
      w.e[j] = (T)(a * t.y + b * t.x);
    } else if constexpr (V == 1) {
      const float a = (float)u.e[0], b = (float)w.e[0];
      u.e[0] = (T)(a * t.x - b * t.y);
      w.e[0] = (T)(a * t.y + b * t.x);
    } else {
      Pack<T, V>& x = j < V / 2 ? u : w;
      const int i = 2 * (j % (V / 2));
      const float a = (float)x.e[i], b = (float)x.e[i + 1];
      x.e[i] = (T)(a * t.x - b * t.y);
      x.e[i + 1] = (T)(a * t.y + b * t.x);
    }
  }
}

template <typename T, int V, bool INTER, bool APPEND>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a) {
  __shared__ __align__(16) float2 s_cs[kAngles];
  __shared__ long long s_row[2][kMaxTokens];     // where a token's row starts in either cache, -1: nowhere
  __shared__ int s_live[kMaxTokens];
  if (a.early) pdl_trigger();
  pdl_wait();
  const int n_all = a.batch * a.tokens, n0 = blockIdx.x * a.per_cta, n = min(a.per_cta, n_all - n0);
  auto position_of = [&](int token, bool& live) -> long long {
    const int b = token / a.tokens, t = token - b * a.tokens;
    live = true;
    if constexpr (APPEND) {
      live = a.counts == nullptr || t < a.counts[b];
      return (long long)a.lengths[b] + t;
    }
    if (a.positions == nullptr) return t;
    const long long i = b * a.pb + t * a.pt;
    return a.positions64 ? reinterpret_cast<const long long*>(a.positions)[i] : reinterpret_cast<const int*>(a.positions)[i];
  };
  // A head is half / V turned items of two vectors, then items of up to two vectors of the rest.
  const int turned = a.half / V, rest = a.width - a.dim, items = turned + (rest + 2 * V - 1) / (2 * V);
  const int flat = (a.width + 2 * V - 1) / (2 * V);       // items of a head of values
  const int per_token = APPEND ? (a.q.heads + a.k.heads) * items + a.v.heads * flat : a.q.heads * items;
  struct Item {
    int k, which, h, at, second, cs;      // token of the CTA; queries, keys, values; first columns of the two vectors; first angle, -1: copied
    Pack<T, V> u, w;
  };
  auto fetch = [&](int i, Item& x) {
    x.k = i / per_token;
    int j = i - x.k * per_token;
    const int token = n0 + x.k, b = token / a.tokens, t = token - b * a.tokens;
    const Part* part = &a.q;
    x.which = 0;
    int width_items = items, first = turned;
    if constexpr (APPEND) {
      if (j >= a.q.heads * items) {
        j -= a.q.heads * items;
        part = &a.k;
        x.which = 1;
        if (j >= a.k.heads * items) {
          j -= a.k.heads * items;
          part = &a.v;
          x.which = 2;
          width_items = flat;
          first = 0;
        }
      }
    }
    x.h = j / width_items;
    const int item = j - x.h * width_items;
    if (item < first) {
      x.at = INTER ? item * 2 * V : item * V;
      x.second = INTER ? x.at + V : x.at + a.half;
      x.cs = item * V;
    } else {
      x.at = (x.which == 2 ? 0 : a.dim) + (item - first) * 2 * V;
      x.second = x.at + V;
      x.cs = -1;
    }
    const T* src = (const T*)part->src + b * part->sb + t * part->st + x.h * part->sh;
    x.u.load(src + x.at);
    if (x.second < a.width) x.w.load(src + x.second);
  };
  // The first item is on its way while the angles are computed, and each one while the one before it is turned.
  const int total = n * per_token;
  Item x;
  if ((int)threadIdx.x < total) fetch(threadIdx.x, x);
  for (int i = threadIdx.x; i < n * a.half; i += kThreads) {
    const int k = i / a.half;
    bool live;
    s_cs[i] = angle_of(a.turns[i - k * a.half], position_of(n0 + k, live), a.amplitude, a.back);
  }
  if constexpr (APPEND) {
    if (threadIdx.x < n) {
      bool live;
      const long long p = position_of(n0 + threadIdx.x, live);
      long long rk = -1, rv = -1;
      if (live) {
        const int b = (n0 + threadIdx.x) / a.tokens;
        int page = -1;
        if (p >= 0 && p < (long long)a.columns * a.page) page = a.table[b * a.table_stride + p / a.page];
        if (page < 0 || page >= a.pages) {
          set_status(a.status, ST_BAD_INDEX, b);
        } else {
          const long long r = p % a.page;
          rk = page * a.k.dp + r * a.k.dr;
          rv = page * a.v.dp + r * a.v.dr;
        }
      }
      s_row[0][threadIdx.x] = rk;
      s_row[1][threadIdx.x] = rv;
      s_live[threadIdx.x] = live;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < total; i += kThreads) {
    Item y;
    if (i + kThreads < total) fetch(i + kThreads, y);
    T* dst = nullptr;
    if (!APPEND || x.which == 0) {
      dst = (T*)a.q.dst + ((long long)(n0 + x.k) * a.q.heads + x.h) * a.width;
    } else {
      const Part& part = x.which == 1 ? a.k : a.v;
      const long long row = s_row[x.which - 1][x.k];
      if (row >= 0) dst = (T*)part.dst + row + x.h * part.dh;
    }
    if (dst) {
      if (x.cs >= 0) turn<T, V, INTER>(x.u, x.w, s_cs + x.k * a.half + x.cs);
      if (APPEND && x.which == 0 && !s_live[x.k]) {
#pragma unroll
        for (int e = 0; e < V; e++) x.u.e[e] = x.w.e[e] = (T)0.f;
      }
      x.u.store(dst + x.at);
      if (x.second < a.width) x.w.store(dst + x.second);
    }
    x = y;
  }
}

template <typename T, int V, bool APPEND>
int launch_rotary(RotaryArgs& a, int inter, cudaStream_t s) {
  const int n = a.batch * a.tokens;
  // Tokens of a CTA: as many as keep every thread busy with four items, as their angles fit, and as leave two CTAs for every SM.
  const long long items = (long long)(a.q.heads + (APPEND ? 2 * a.k.heads : 0)) * ((a.width + 2 * V - 1) / (2 * V));
  long long per = (4 * kThreads + items - 1) / items;
  per = per < kMaxTokens ? per : kMaxTokens;
  if (per * a.half > kAngles) per = kAngles / a.half;
  const long long spread = (n + 2 * 148 - 1) / (2 * 148);
  per = per < spread ? per : spread;
  if (per < 1) per = 1;
  a.per_cta = (int)per;
  const unsigned ctas = (unsigned)((n + per - 1) / per);
  a.early = starts_early(per * items * 4 * V * sizeof(T), ctas);
  if (inter) GB_CUDA_OK(gbh::launch_if(a.early, rotary_kernel<T, V, true, APPEND>, dim3(ctas), dim3(kThreads), 0, s, a));
  else GB_CUDA_OK(gbh::launch_if(a.early, rotary_kernel<T, V, false, APPEND>, dim3(ctas), dim3(kThreads), 0, s, a));
  return gbh::E_OK;
}

template <bool APPEND>
int dispatch(int dtype, RotaryArgs& a, int inter, cudaStream_t s) {
  if (dtype == 2) {
    switch (a.vec) {
      case 4: return launch_rotary<float, 4, APPEND>(a, inter, s);
      case 2: return launch_rotary<float, 2, APPEND>(a, inter, s);
      default: return launch_rotary<float, 1, APPEND>(a, inter, s);
    }
  }
  if (dtype == 0) {
    switch (a.vec) {
      case 8: return launch_rotary<__nv_bfloat16, 8, APPEND>(a, inter, s);
      case 4: return launch_rotary<__nv_bfloat16, 4, APPEND>(a, inter, s);
      case 2: return launch_rotary<__nv_bfloat16, 2, APPEND>(a, inter, s);
      default: return launch_rotary<__nv_bfloat16, 1, APPEND>(a, inter, s);
    }
  }
  switch (a.vec) {
    case 8: return launch_rotary<__half, 8, APPEND>(a, inter, s);
    case 4: return launch_rotary<__half, 4, APPEND>(a, inter, s);
    case 2: return launch_rotary<__half, 2, APPEND>(a, inter, s);
    default: return launch_rotary<__half, 1, APPEND>(a, inter, s);
  }
}

// The widest vector (elements) that divides every size, stride and address.
int vector_of(int size, const RotaryArgs& a, int extra) {
  int v = 16 / size;
  auto fits = [&](const Part& p, bool cache) {
    if (!p.src) return true;
    const uintptr_t at = (uintptr_t)p.src | (uintptr_t)p.dst;
    long long s = p.sb | p.st | p.sh;
    if (cache) s |= p.dp | p.dh | p.dr;
    return at % (v * size) == 0 && s % v == 0;
  };
  while (v > 1 && !(a.half % v == 0 && a.width % v == 0 && fits(a.q, false) && fits(a.k, extra) && fits(a.v, extra))) v >>= 1;
  return v;
}

int checked(const char* what, int dtype, const RotaryArgs& a) {
  if (dtype < 0 || dtype > 2) {
    gbh::set_error("%s: bad dtype %d", what, dtype);
    return gbh::E_BAD_ARG;
  }
  if (a.batch < 0 || a.tokens < 0 || a.width < 1 || a.dim < 0 || a.dim > a.width || a.dim % 2 || a.half > kAngles || a.q.heads < 0 ||
      a.k.heads < 0 || (a.half && !a.turns)) {
    gbh::set_error("%s: bad sizes (batch %d, tokens %d, width %d, dim %d)", what, a.batch, a.tokens, a.width, a.dim);
    return gbh::E_BAD_ARG;
  }
  const long long n = (long long)a.batch * a.tokens, wide = (long long)(a.q.heads + 2LL * a.k.heads) * a.width;
  if (n >= 0x7fffffffLL || wide * kMaxTokens >= 0x7fffffffLL) {
    gbh::set_error("%s: %lld tokens of %lld columns are too many for one call", what, n, wide);
    return gbh::E_TOO_LARGE;
  }
  return gbh::E_OK;
}

}  // namespace

// y = x turned: x (batch, tokens, heads, width) with strides (elements), y contiguous.  positions: int32 or int64 with strides (0 where
// shared), or null for 0, 1, ...
GB_EXPORT int gb_rotary(int dtype, const void* x, long long sb, long long st, long long sh, void* y, int batch, int tokens, int heads, int width,
                        int dim, int interleaved, const void* turns, double amplitude, int back, const void* positions, int positions64,
                        long long pb, long long pt, void* stream) {
  RotaryArgs a = {};
  a.q = {x, y, sb, st, sh, 0, 0, 0, heads};
  a.batch = batch; a.tokens = tokens; a.width = width; a.dim = dim; a.half = dim / 2;
  a.turns = (const unsigned long long*)turns;
  a.amplitude = (float)amplitude;
  a.back = back;
  a.positions = positions; a.positions64 = positions64; a.pb = pb; a.pt = pt;
  const int rc = checked("gb_rotary", dtype, a);
  if (rc != gbh::E_OK) return rc;
  if (batch == 0 || tokens == 0 || heads == 0) return gbh::E_OK;
  if (!x || !y) {
    gbh::set_error("gb_rotary: null pointer");
    return gbh::E_BAD_ARG;
  }
  a.vec = vector_of(dtype == 2 ? 4 : 2, a, 0);
  return dispatch<false>(dtype, a, interleaved, (cudaStream_t)stream);
}

// k and v (batch, tokens, heads, width) into the pages of their sequences, k turned (dim 0: as it is); q, where there is one, turned
// into q_out.  Strides in elements: of q, k, v (batch, token, head), of both caches (page, head, row: strides[0..5]).
GB_EXPORT int gb_cache_append(int dtype, const void* q, long long q_sb, long long q_st, long long q_sh, void* q_out, const void* k, long long k_sb,
                              long long k_st, long long k_sh, const void* v, long long v_sb, long long v_st, long long v_sh, void* k_cache,
                              void* v_cache, const long long* strides, int batch, int tokens, int q_heads, int heads, int width, int dim, int interleaved,
                              const void* turns, double amplitude, const void* table, long long table_stride, int columns, int pages, int page,
                              const void* lengths, const void* counts, void* stream) {
  RotaryArgs a = {};
  const long long zero[6] = {0, 0, 0, 0, 0, 0}, *s = strides ? strides : zero;
  a.q = {q, q_out, q_sb, q_st, q_sh, 0, 0, 0, q ? q_heads : 0};
  a.k = {k, k_cache, k_sb, k_st, k_sh, s[0], s[1], s[2], heads};
  a.v = {v, v_cache, v_sb, v_st, v_sh, s[3], s[4], s[5], heads};
  a.batch = batch; a.tokens = tokens; a.width = width; a.dim = dim; a.half = dim / 2;
  a.turns = (const unsigned long long*)turns;
  a.amplitude = (float)amplitude;
  a.table = (const int*)table; a.table_stride = table_stride; a.columns = columns; a.pages = pages; a.page = page;
  a.lengths = (const int*)lengths;
  a.counts = (const int*)counts;
  const int rc = checked("gb_cache_append", dtype, a);
  if (rc != gbh::E_OK) return rc;
  if (batch == 0 || tokens == 0) return gbh::E_OK;
  if (!k || !v || !k_cache || !v_cache || !strides || !table || !lengths || (q && !q_out) || page < 1 || columns < 1 || pages < 1 || heads < 1) {
    gbh::set_error("gb_cache_append: null pointer or empty cache");
    return gbh::E_BAD_ARG;
  }
  a.status = gbh::status_ptr();
  a.vec = vector_of(dtype == 2 ? 4 : 2, a, 1);
  return dispatch<true>(dtype, a, interleaved, (cudaStream_t)stream);
}
