// Rotary positions, and the same on the way into a paged cache of keys and values.
//
// A pair (a, b) of a head at position p becomes (a cos - b sin, a sin + b cos) * amplitude with the angle p w_i; pairs are
// (i, i + dim / 2) or (2 i, 2 i + 1), columns from dim on are copied.  The gradient is the same kernel with the opposite angle.
//
// Angles.  p w in fp32 is off by p 2^-24: by 0.008 at position 131 072, twice a bf16's last bit.  So a frequency is held as the fraction
// w / 2 pi of a turn in 64 bits of fixed point, and p times it, modulo 2^64, is the fraction of a turn that is left: an integer
// product whose overflow is the reduction.  The fraction is a quotient in fp64, off by 2^-55 for w up to 1: p times it by p 2^-55 turns, as the
// product p w itself in fp64 is, which is less than what comes next up to position 2^27.  For fp32 rows the upper two bits are the
// quarter and the next 32 a float of up to an eighth of a turn either way, off by pi 2^-27 (2.4e-8; with the upper 32 bits as a float of half a turn
// 9.4e-8), for sincospif; for 16-bit rows the upper 32 bits become that float of half a turn, off by 9.4e-8.
//
// What bounds it: memory, every element read and written once.  A thread takes an item, two vectors of 16 bytes (narrower ones where a size or an
// address is odd) with the two halves of its pairs, of several heads of one token: their loads and the position's are on their way at once, and sines and
// cosines serve all of these heads.  No table, no shared memory, no barrier.  16 x 1024 tokens of 24 heads of 64 in bf16: 17.4 us, 0.88 of copy bandwidth
// (a CTA that computed the angles of a few tokens in shared memory for all of their heads: 21 to 25); four prompts of 2048 tokens with 16 heads of
// 128 appended and their queries turned: 38.4 us, 0.80.
#include "common.cuh"

using namespace gb;

namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 4;              // whose loads a thread has on their way (two: 40 to 42 us for the prompts above)

struct Part {                         // a tensor (batch, tokens, heads, width) and where its rows go
  const void* src;
  void* dst;                          // (batch, tokens, heads, width), src itself perhaps; a cache for keys and values
  long long sb, st, sh;               // strides of src in elements
  long long dp, dh, dr;               // strides of dst: batch, head, token; of a cache: page, head, row
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
  int groups;                         // threads that share a token's heads of an item
};

template <int BYTES> struct VecOf;
template <> struct VecOf<16> { using type = uint4; };
template <> struct VecOf<8> { using type = uint2; };
template <> struct VecOf<4> { using type = uint32_t; };
template <> struct VecOf<2> { using type = uint16_t; };

template <typename T, int V>
struct Pack {
  T e[V];
  // CONST: nothing writes there meanwhile.  Four prompts appended: 38.4 us so, 48.1 with loads that might see a store.
  template <bool CONST>
  __device__ __forceinline__ void load(const T* p) {
    using U = typename VecOf<V * sizeof(T)>::type;
    *reinterpret_cast<U*>(e) = CONST ? __ldg(reinterpret_cast<const U*>(p)) : *reinterpret_cast<const U*>(p);
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<typename VecOf<V * sizeof(T)>::type*>(p) = *reinterpret_cast<const typename VecOf<V * sizeof(T)>::type*>(e); }
};

// Cosine and sine of a position's angle.  For fp32 rows sincospif; for 16-bit rows the hardware's functions, off by 2^-21 at most within half a turn,
// where the rows themselves are off by 2^-12 or 2^-9 (the prompts above: 40.9 us with sincospif).
template <typename T>
__device__ __forceinline__ float2 angle_of(unsigned long long turns, long long position, float amplitude, bool back) {
  const unsigned long long phase = turns * (unsigned long long)position;
  float s, c;
  if constexpr (sizeof(T) == 4) {
    const unsigned quarter = (unsigned)((phase + (1ull << 61)) >> 62);
    sincospif((float)(int)(phase >> 30) * 1.1641532182693481e-10f, &s, &c);    // 2^-33: half turns from the nearest quarter, in [-1/4, 1/4)
    if (quarter & 1) {
      const float t = s;
      s = c;
      c = -t;
    }
    if (quarter & 2) {
      s = -s;
      c = -c;
    }
  } else {
    const float x = (float)(int)(phase >> 32) * 4.656612873077393e-10f;        // 2^-31: half turns in [-1, 1)
    s = __sinf(x * 3.14159265358979f);
    c = __cosf(x * 3.14159265358979f);
  }
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

// A head of any part is `items` items of two vectors: half / V turned ones, then the rest (of values: all of it) as it lies.
template <typename T, int V, bool INTER, bool APPEND, bool IN_PLACE>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a) {
  pdl_trigger();                      // (two heads a thread and more, or 1 184 CTAs at most: starts_early() holds for any size)
  const int items = (a.width + 2 * V - 1) / (2 * V), heads = APPEND ? a.q.heads + 2 * a.k.heads : a.q.heads;
  const unsigned i = blockIdx.x * kThreads + threadIdx.x, per_token = (unsigned)a.groups * items, token = i / per_token;
  const unsigned in_token = i - token * per_token, group = in_token / items;
  const int item = in_token - group * items, b = token / a.tokens, t = token - b * a.tokens;
  pdl_wait();
  if (b >= a.batch) return;
  const bool turns = item < a.half / V;
  const int flat = item * 2 * V, first = turns && !INTER ? item * V : flat, second = turns && !INTER ? first + a.half : first + V;
  struct Pair {
    Pack<T, V> u, w;
    int which, h;                         // queries, keys, values; the head
  };
  // (values chosen one by one: a pointer to a part of the arguments would have them copied to local memory)
  auto of = [&](int which, auto q, auto k, auto v) { return !APPEND || which == 0 ? q : which == 1 ? k : v; };
  auto fetch = [&](Pair& x, int h) {
    x.which = 0;
    if (APPEND && h >= a.q.heads) {
      x.which = 1;
      h -= a.q.heads;
      if (h >= a.k.heads) {
        x.which = 2;
        h -= a.k.heads;
      }
    }
    x.h = h;
    const bool value = APPEND && x.which == 2;
    const T* src = (const T*)of(x.which, a.q.src, a.k.src, a.v.src) + b * of(x.which, a.q.sb, a.k.sb, a.v.sb) +
                   t * of(x.which, a.q.st, a.k.st, a.v.st) + h * of(x.which, a.q.sh, a.k.sh, a.v.sh);
    const int at = value ? flat : first, to = value ? flat + V : second;
    x.u.template load<!IN_PLACE>(src + at);
    if (to < a.width) x.w.template load<!IN_PLACE>(src + to);
  };
  // kHeads heads at a time, the first ones on their way before anything else is known.
  Pair x[kHeads];
  int h = group;
#pragma unroll
  for (int k = 0; k < kHeads; k++)
    if (h + k * a.groups < heads) fetch(x[k], h + k * a.groups);
  long long position = t;
  if constexpr (APPEND) {
    position = (long long)a.lengths[b] + t;
  } else if (a.positions != nullptr) {
    const long long at = b * a.pb + t * a.pt;
    position = a.positions64 ? reinterpret_cast<const long long*>(a.positions)[at] : reinterpret_cast<const int*>(a.positions)[at];
  }
  bool live = true;
  int page = -1, in_page = 0;
  if constexpr (APPEND) {
    live = a.counts == nullptr || t < a.counts[b];
    if (live) {
      if (position >= 0 && position < (long long)a.columns * a.page) {
        const unsigned column = (unsigned)position / (unsigned)a.page;
        in_page = (int)((unsigned)position - column * (unsigned)a.page);
        page = a.table[b * a.table_stride + column];
      }
      if (page < 0 || page >= a.pages) {
        if (in_token == 0) set_status(a.status, ST_BAD_INDEX, b);
        page = -1;
      }
    }
  }
  float2 cs[V];
  if (turns) {
#pragma unroll
    for (int k = 0; k < V; k++) cs[k] = angle_of<T>(a.turns[item * V + k], position, a.amplitude, a.back);
  }
  for (; h < heads; h += kHeads * a.groups) {
#pragma unroll
    for (int k = 0; k < kHeads; k++) {
      if (h + k * a.groups >= heads) break;
      const bool value = APPEND && x[k].which == 2;
      if (turns && !value) turn<T, V, INTER>(x[k].u, x[k].w, cs);
      T* dst;
      if (!APPEND || x[k].which == 0) {
        dst = (T*)a.q.dst + b * a.q.dp + t * a.q.dr + x[k].h * a.q.dh;
        if (APPEND && !live) {
#pragma unroll
          for (int e = 0; e < V; e++) x[k].u.e[e] = x[k].w.e[e] = (T)0.f;
        }
      } else {
        if (page < 0) continue;
        dst = value ? (T*)a.v.dst + page * a.v.dp + x[k].h * a.v.dh + in_page * a.v.dr
                    : (T*)a.k.dst + page * a.k.dp + x[k].h * a.k.dh + in_page * a.k.dr;
      }
      const int at = value ? flat : first, to = value ? flat + V : second;
      x[k].u.store(dst + at);
      if (to < a.width) x[k].w.store(dst + to);
    }
#pragma unroll
    for (int k = 0; k < kHeads; k++)
      if (h + (k + kHeads) * a.groups < heads) fetch(x[k], h + (k + kHeads) * a.groups);
  }
}

template <typename T, int V, bool APPEND>
int launch_rotary(RotaryArgs& a, int inter, cudaStream_t s) {
  const unsigned long long tokens = (unsigned long long)a.batch * a.tokens;
  const int heads = a.q.heads + (APPEND ? 2 * a.k.heads : 0), items = (a.width + 2 * V - 1) / (2 * V);
  // Heads of a thread: four where that leaves the SMs full twice over, two where it does so once, else one.  The tokens above with one, two, four and six
  // heads to a thread: 31, 22, 18.2 and 18.5 us, the prompts 72, 49, 38.6 and 41.
  int per = 4;
  while (per > 1 && tokens * items * ((heads + per - 1) / per) < (per > 2 ? 2ull : 1ull) * 148 * 1024) per >>= 1;
  a.groups = (heads + per - 1) / per;
  const unsigned long long threads = tokens * items * a.groups;
  if (threads >= 0xffff0000ull) {
    gbh::set_error("rotary: %llu tokens of %d heads are too many for one call", tokens, heads);
    return gbh::E_TOO_LARGE;
  }
  const unsigned ctas = (unsigned)((threads + kThreads - 1) / kThreads);
  const auto go = [&](auto kernel) { return gbh::launch(kernel, dim3(ctas), dim3(kThreads), 0, s, 1, a); };
  if constexpr (!APPEND) {
    if (a.q.src == a.q.dst) {
      GB_CUDA_OK(inter ? go(rotary_kernel<T, V, true, false, true>) : go(rotary_kernel<T, V, false, false, true>));
      return gbh::E_OK;
    }
  }
  GB_CUDA_OK(inter ? go(rotary_kernel<T, V, true, APPEND, false>) : go(rotary_kernel<T, V, false, APPEND, false>));
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

// The widest vector (elements) that divides every size, stride and address.  An odd half leaves one element: 16 x 1024 tokens of 24 heads of 52 bf16 with 52
// columns turned 17.8 us, with 50 or 26 30.6.
int vector_of(int size, const RotaryArgs& a) {
  int v = 16 / size;
  auto fits = [&](const Part& p) {
    if (!p.src) return true;
    const uintptr_t at = (uintptr_t)p.src | (uintptr_t)p.dst;
    const long long s = p.sb | p.st | p.sh | p.dp | p.dh | p.dr;
    return at % (v * size) == 0 && s % v == 0;
  };
  while (v > 1 && !(a.half % v == 0 && a.width % v == 0 && fits(a.q) && fits(a.k) && fits(a.v))) v >>= 1;
  return v;
}

// Sizes that are kept in 32 bits from here on.
bool sizes_fit(const char* what, const long long* sizes, int first, int last) {
  for (int i = first; i <= last; i++)
    if (sizes[i] < 0 || sizes[i] > 0x7fffffffLL) {
      gbh::set_error("%s: size %d is %lld, beyond 31 bits", what, i, sizes[i]);
      return false;
    }
  return true;
}

int checked(const char* what, int dtype, const RotaryArgs& a) {
  if (dtype < 0 || dtype > 2) {
    gbh::set_error("%s: bad dtype %d", what, dtype);
    return gbh::E_BAD_ARG;
  }
  if (a.batch < 0 || a.tokens < 0 || a.width < 1 || a.dim < 0 || a.dim > a.width || a.dim % 2 || a.q.heads < 0 ||
      a.k.heads < 0 || (a.half && !a.turns)) {
    gbh::set_error("%s: bad sizes (batch %d, tokens %d, width %d, dim %d)", what, a.batch, a.tokens, a.width, a.dim);
    return gbh::E_BAD_ARG;
  }
  if ((long long)a.batch * a.tokens >= 0x7fffffffLL || (long long)a.columns * a.page >= 0x7fffffffLL) {
    gbh::set_error("%s: %d x %d tokens or a table of %d pages of %d positions are too many for one call", what, a.batch, a.tokens, a.columns, a.page);
    return gbh::E_TOO_LARGE;
  }
  return gbh::E_OK;
}

}  // namespace

// Sizes and strides (in elements) come as one array of 64-bit words: a call of many arguments costs its caller more than the launch.

// y = x turned, both (batch, tokens, heads, width); y may be x.  sizes: [0..2] strides of x (batch, token, head), [3..5] of y, [6..9] batch, tokens,
// heads, width, [10] columns that are turned, [11] pairs side by side, [12] turn back, [13] positions are int64, [14..15] their strides (batch, token; 0
// where shared).  positions: null for 0, 1, ...
GB_EXPORT int gb_rotary(int dtype, const void* x, void* y, const long long* sizes, const void* turns, const void* positions, double amplitude,
                        void* stream) {
  if (!sizes) {
    gbh::set_error("gb_rotary: null pointer");
    return gbh::E_BAD_ARG;
  }
  const long long* z = sizes;
  if (!sizes_fit("gb_rotary", z, 6, 10)) return gbh::E_TOO_LARGE;
  RotaryArgs a = {};
  a.q = {x, y, z[0], z[1], z[2], z[3], z[5], z[4], (int)z[8]};
  a.batch = (int)z[6]; a.tokens = (int)z[7]; a.width = (int)z[9]; a.dim = (int)z[10]; a.half = a.dim / 2;
  a.turns = (const unsigned long long*)turns;
  a.amplitude = (float)amplitude;
  a.back = (int)z[12];
  a.positions = positions; a.positions64 = (int)z[13]; a.pb = z[14]; a.pt = z[15];
  const int rc = checked("gb_rotary", dtype, a);
  if (rc != gbh::E_OK) return rc;
  if (a.batch == 0 || a.tokens == 0 || a.q.heads == 0) return gbh::E_OK;
  if (!x || !y) {
    gbh::set_error("gb_rotary: null pointer");
    return gbh::E_BAD_ARG;
  }
  a.vec = vector_of(dtype == 2 ? 4 : 2, a);
  return dispatch<false>(dtype, a, (int)z[11], (cudaStream_t)stream);
}

// k and v (batch, tokens, heads, width) into the pages of their sequences, k turned (dim 0: as it is); q, where there is one, turned
// into q_out (contiguous).  sizes: [0..8] strides of q, k, v (batch, token, head), [9..14] of both caches (page, head, row), [15..19] batch, tokens, heads of
// queries and of keys, width, [20] columns that are turned, [21] pairs side by side, [22] the table's stride, [23] its columns, [24] pages, [25] positions
// of a page.
GB_EXPORT int gb_cache_append(int dtype, const void* q, void* q_out, const void* k, const void* v, void* k_cache, void* v_cache, const long long* sizes,
                              const void* turns, double amplitude, const void* table, const void* lengths, const void* counts, void* stream) {
  if (!sizes) {
    gbh::set_error("gb_cache_append: null pointer");
    return gbh::E_BAD_ARG;
  }
  const long long* z = sizes;
  if (!sizes_fit("gb_cache_append", z, 15, 20) || !sizes_fit("gb_cache_append", z, 23, 25)) return gbh::E_TOO_LARGE;
  RotaryArgs a = {};
  a.batch = (int)z[15]; a.tokens = (int)z[16]; a.width = (int)z[19]; a.dim = (int)z[20]; a.half = a.dim / 2;
  const int q_heads = q ? (int)z[17] : 0, heads = (int)z[18];
  a.q = {q, q_out, z[0], z[1], z[2], (long long)a.tokens * q_heads * a.width, a.width, (long long)q_heads * a.width, q_heads};
  a.k = {k, k_cache, z[3], z[4], z[5], z[9], z[10], z[11], heads};
  a.v = {v, v_cache, z[6], z[7], z[8], z[12], z[13], z[14], heads};
  a.turns = (const unsigned long long*)turns;
  a.amplitude = (float)amplitude;
  a.table = (const int*)table; a.table_stride = z[22]; a.columns = (int)z[23]; a.pages = (int)z[24]; a.page = (int)z[25];
  a.lengths = (const int*)lengths;
  a.counts = (const int*)counts;
  const int rc = checked("gb_cache_append", dtype, a);
  if (rc != gbh::E_OK) return rc;
  if (a.batch == 0 || a.tokens == 0) return gbh::E_OK;
  if (!k || !v || !k_cache || !v_cache || !table || !lengths || (q && !q_out) || a.page < 1 || a.columns < 1 || a.pages < 1 || heads < 1) {
    gbh::set_error("gb_cache_append: null pointer or empty cache");
    return gbh::E_BAD_ARG;
  }
  a.status = gbh::status_ptr();
  a.vec = vector_of(dtype == 2 ? 4 : 2, a);
  return dispatch<true>(dtype, a, (int)z[21], (cudaStream_t)stream);
}
