// Attention of new tokens over a paged cache of keys and values, and of a batch whose first pages are shared.
//
// Token t < counts[b] of sequence b sits at position lengths[b] + t and sees the positions up to its own:
// o = sum_j p_j v_j / sum_j p_j with p_j = exp(scale q . k_j - m).  One pass over the keys with the running maximum m and sum l of
// each row, in fp32; H / Hkv query heads share a key head and are rows of one tile.  The weights p are at most 1 and are rounded to the
// inputs' type for the second product (2^-9 of each in bf16, as in csrc/flash_attn.cu; in the kernel for many rows they are at most 2^8, which changes
// nothing of that); their sum is taken before.
//
// What bounds it: every key and value is read once for a few rows of queries, so memory does (64 sequences of up to 32 768 positions, 32 / 8 heads
// of 128 bf16: 722 us, 7.0 TB/s).  The work is a list of tiles of 32 KB of keys and values:
// sequence by sequence, key head by key head.  Its length is known on the device alone (lengths[]), so every CTA adds the
// lengths up itself and takes an equal share of the list, across sequences and heads: no plan, no host, no idle SM with ragged
// lengths.  A (sequence, head) whose tiles fall to several CTAs leaves partial rows (m, l, o) behind, which a second kernel joins in
// the list's order; no atomics.
//
// Where few (sequence, head) pairs have short tables, a cluster of up to eight CTAs takes each of them, and their sums meet in distributed shared
// memory instead: no second kernel (one token behind 2 047 positions of 16 heads, in a graph: 8.5 us, 10.5 with it).  There a long sequence keeps its
// cluster alone, see plan().
//
// A shared prefix is one more entry at the head of the list whose rows are the queries of all sequences: its keys are read once for
// every 16, 32 or 64 rows.  The sequences' own entries then start behind it, and all rows are joined by the second kernel.  A sequence that ends within
// the prefix takes no part in it, so that no row meets a value that its own sequence does not have: all its keys are its own entry's.
//
// A CTA: four warps that multiply (mma.sync for 16-bit types, FMA for fp32) and four that copy through a ring of stages: by TMA, a box of
// as many rows as divide both a page and a tile, where these are at least eight (a multiple of the swizzle's period); else with cp.async,
// 16 bytes a lane, a page looked up for every key (64 sequences of up to 8 192 positions: pages of 64 222 us, of 8 225, of 4 250; with one
// copying warp 228, 368, 396).  What stands behind a sequence's last key in its last page may be anything, NaN
// too: those scores are masked, and those rows of V become zeros in shared memory.
#include "common.cuh"
#include "pair.cuh"

#include <string.h>

#include <atomic>

using namespace gb;

namespace {

constexpr int kThreads = 256;
constexpr int kConsumers = 4, kCopiers = 4;      // warps
constexpr int kPeers = 8;                        // most CTAs of a cluster

struct CacheArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;                               // (B, T, H, D), contiguous
  long long q_sb, q_st, q_sh;
  long long k_sp, k_sh, k_sr, v_sp, v_sh, v_sr;
  const int* table;
  long long table_stride;
  int columns, pages, page, room;          // room: columns page
  const int* lengths;
  const int* counts;
  int B, T, H, Hkv, G, D;
  int prefix;                              // shared positions (whole pages)
  float scale_log2;
  int own_tiles, prefix_tiles;             // row tiles of a sequence, of the prefix
  int ctas;
  float* part;                             // [slots][rows of a tile][D] unscaled sums
  float2* stat;                            // [slots][rows of a tile] (m, l)
  int box;                                 // rows of a TMA box
  int peers;                               // CTAs of a cluster, 0: the list is dealt out
  int shared;                              // a prefix is joined to the sequences' own keys
  int wide_prefix, wide_own;               // which of them the kernel for many rows takes
  int wide_tiles, splits, wide_group;      // its row tiles, of a sequence or of the prefix; runs of keys; runs whose tiles go together
  int slot_rows;                           // rows of the other kernel's tiles
  int2* owner;                             // [(prefix tiles + B own_tiles) Hkv] first slot and last CTA, first -1: no keys
  int* status;
};

template <typename T> struct Elem;
template <> struct Elem<__nv_bfloat16> {
  static constexpr bool kMma = true;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16(a, b); }
};
template <> struct Elem<__half> {
  static constexpr bool kMma = true;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_f16(a, b); }
};
template <> struct Elem<float> { static constexpr bool kMma = false; };

// Rows of a tile: 16 RG in 16 bits, 4, 16 or 8 (RG = 0, 1, 2) in fp32.  Row groups of 16 rows times key groups of a quarter, a half or all of the keys are the four
// warps of the 16-bit kernel; in fp32 a warp takes a quarter of the keys and all rows.  Two CTAs to an SM: while one waits, joins or stores, the other multiplies.
template <typename T, int HD_, int RG_, bool TMA>
struct Cfg {
  static constexpr int HD = HD_, RG = RG_;
  static constexpr bool kMma = Elem<T>::kMma;
  static constexpr int ROWS = kMma ? 16 * RG : RG == 0 ? 4 : RG == 1 ? 16 : 8;
  static constexpr int TILE = kMma ? (HD == 64 ? 128 : 64) : HD == 64 ? 64 : 32;      // 16 KB of keys
  static constexpr int KG = kMma ? 4 / (RG ? RG : 1) : 4;
  static constexpr int SUB = TILE * HD * (int)sizeof(T);          // one K or V tile
  static constexpr int STAGES = 2;
  static constexpr int SEGS = ROWS * HD * (int)sizeof(T) <= 4096 ? 3 : 2;           // segments (queries, rows) on their way
  static constexpr int Q_BYTES = ROWS * HD * (int)sizeof(T);
  static constexpr int CHUNKS = HD * (int)sizeof(T) / 16;         // 16-byte chunks of a row
  static constexpr int COLS = HD * (int)sizeof(T) / 128;          // columns of 128 bytes
  static constexpr int PAD = HD + 8;                              // floats of a row of sums: eight rows' columns in different banks
  static constexpr int RJ = ROWS < 8 ? ROWS : 8;                  // rows whose four sums are joined at a time
  static constexpr int JOIN = (KG == 4 ? 4 * RJ : KG == 2 ? ROWS : 0) * (PAD * 4 + 8);      // of two key groups one hands its sums to the other
  static constexpr int WEIGHTS = kMma ? 0 : TILE * ROWS * 4;      // fp32: the weights of a tile
  static constexpr int PEERS = KG == 4 ? kPeers * ROWS * 8 : 0;   // statistics of a cluster's CTAs; their sums lie in the second buffer for queries
  static_assert(KG < 4 || (SEGS - 1) * Q_BYTES >= ROWS * HD * 4, "sums of a cluster");
  static constexpr int SMEM = 2 * STAGES * SUB + SEGS * Q_BYTES + JOIN + WEIGHTS + PEERS + 1024 + SEGS * (ROWS * 12 + 32) + ROWS * 8 + 256 + (TMA ? 0 : 2 * TILE * 8);
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs to an SM");
};

// ---------------------------------------------------------------------------------------------------------------------------
// the list of tiles
// ---------------------------------------------------------------------------------------------------------------------------
struct Entry {                // rows of queries over a range of keys, for every key head
  int b;                      // -1: all sequences, over the prefix
  int row0;                   // first row
  int begin, end;             // keys
  int tiles;                  // of one key head
  bool cut;                   // keys behind the end of its table were asked for
};

// L2: past the SM's own cache, for a kernel that may start before the one in front of it has ended and waits for it at its end alone.
template <bool L2>
__device__ __forceinline__ int read(const int* p) { return L2 ? __ldcg(p) : *p; }

template <bool L2 = false>
__device__ __forceinline__ int count_of(const CacheArgs& a, int b) {
  const int c = a.counts ? read<L2>(a.counts + b) : a.T;
  return c < 0 ? 0 : c < a.T ? c : a.T;
}

template <int ROWS, int TILE>
__device__ __forceinline__ Entry entry_of(const CacheArgs& a, int e) {
  Entry x;
  x.cut = false;
  if (e < a.prefix_tiles) {
    x.b = -1;
    x.row0 = e * ROWS;
    x.begin = 0;
    x.end = a.prefix;
  } else {
    e -= a.prefix_tiles;
    long long end, whole;                                              // of these rows, of the sequence
    if (a.own_tiles == 1) {
      x.b = e;
      x.row0 = 0;
      const int c = count_of(a, e);
      end = whole = c > 0 ? (long long)a.lengths[e] + c : 0;
    } else {
      x.b = e / a.own_tiles;
      x.row0 = (e - x.b * a.own_tiles) * ROWS;
      const int c = count_of(a, x.b), last = min(a.T * a.G, x.row0 + ROWS) - 1;
      const int seen = min(c, last / a.G + 1);                       // tokens of these rows that count, and those before them
      end = x.row0 / a.G < c ? (long long)a.lengths[x.b] + seen : 0;
      whole = (long long)a.lengths[x.b] + c;
    }
    x.begin = whole < a.prefix ? 0 : a.prefix;                       // (one that ends within the prefix takes no part in it)
    x.cut = end > a.room;
    x.end = (int)(x.cut ? (long long)a.room : end > 0 ? end : 0);
  }
  x.tiles = x.end > x.begin ? (x.end - x.begin + TILE - 1) / TILE : 0;
  return x;
}

// The list cut into equal shares: `per` tiles for every CTA and one more for the first `rem`.
struct Shares {
  unsigned per, rem;
  __device__ __forceinline__ unsigned first(unsigned cta) const { return cta * per + min(cta, rem); }
  __device__ __forceinline__ unsigned cta_of(unsigned tile) const {
    const unsigned longer = rem * (per + 1);
    return tile < longer ? tile / (per + 1) : rem + (tile - longer) / per;
  }
};

// A CTA's place in the list, held by the warps that copy.
template <int ROWS, int TILE>
struct Cursor {
  Shares shares;
  Entry x;
  int e, h, entries, tile;
  unsigned left, segment0;           // tiles to go; the list's number of the segment's first tile

  // Adds up the tiles of all entries, an entry or a run of them a lane, and finds this CTA's share.  (Totals stay below 2^31.)
  __device__ __forceinline__ void start(const CacheArgs& a, int lane) {
    entries = a.prefix_tiles + a.B * a.own_tiles;
    const int per = (entries + 31) / 32, lo = min(entries, lane * per), hi = min(entries, lo + per);
    unsigned mine = 0;
    Entry first_entry;
#pragma unroll 4
    for (int k = lo; k < hi; k++) {
      const Entry y = entry_of<ROWS, TILE>(a, k);
      if (k == lo) first_entry = y;
      mine += y.tiles;
      if (blockIdx.x == 0 && threadIdx.x < 32 * (kConsumers + 1)) {
        if (y.cut) set_status(a.status, ST_BAD_INDEX, y.b);
        if (y.tiles == 0)
          for (int i = 0; i < a.Hkv; i++) a.owner[k * a.Hkv + i] = make_int2(-1, -1);
      }
    }
    mine *= a.Hkv;
    unsigned sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += up;
    }
    const unsigned total = __shfl_sync(0xffffffffu, sum, 31), before = sum - mine;
    const unsigned ctas = min((unsigned)a.ctas, total);              // so that none between two others has nothing
    left = 0;
    if (blockIdx.x >= ctas) return;
    shares.per = total / ctas;
    shares.rem = total - shares.per * ctas;
    const unsigned first = shares.first(blockIdx.x);
    left = shares.per + (blockIdx.x < shares.rem);
    const unsigned owner = __ffs(__ballot_sync(0xffffffffu, first >= before && first < sum)) - 1;
    unsigned at = before;
    if (lane == owner) {
      x = first_entry;
      for (e = lo;; ) {
        const unsigned n = (unsigned)x.tiles * a.Hkv;
        if (first < at + n) break;
        at += n;
        x = entry_of<ROWS, TILE>(a, ++e);
      }
      h = (first - at) / x.tiles;
      at += h * x.tiles;
    }
    e = __shfl_sync(0xffffffffu, e, owner);
    h = __shfl_sync(0xffffffffu, h, owner);
    segment0 = __shfl_sync(0xffffffffu, at, owner);
    x.b = __shfl_sync(0xffffffffu, x.b, owner);
    x.row0 = __shfl_sync(0xffffffffu, x.row0, owner);
    x.begin = __shfl_sync(0xffffffffu, x.begin, owner);
    x.end = __shfl_sync(0xffffffffu, x.end, owner);
    x.tiles = __shfl_sync(0xffffffffu, x.tiles, owner);
    tile = first - segment0;
  }
  // The share of a CTA whose cluster has one entry and key head for itself.
  __device__ __forceinline__ void start_cluster(const CacheArgs& a, int peers, int rank) {
    const int seg = blockIdx.x / peers;
    e = seg / a.Hkv;
    h = seg - e * a.Hkv;
    x = entry_of<ROWS, TILE>(a, e);
    if (x.cut && rank == 0 && threadIdx.x == 32 * kConsumers) set_status(a.status, ST_BAD_INDEX, x.b);
    tile = x.tiles * rank / peers;
    left = x.tiles * (rank + 1) / peers - tile;
  }
  __device__ __forceinline__ void next_segment(const CacheArgs& a) {
    segment0 += x.tiles;
    tile = 0;
    if (++h < a.Hkv) return;
    h = 0;
    do {
      if (++e >= entries) return;
      x = entry_of<ROWS, TILE>(a, e);
    } while (x.tiles == 0);
  }
};

// ---------------------------------------------------------------------------------------------------------------------------
// matrix instructions
// ---------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && __is_same(T, __nv_bfloat16))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ unsigned long long pair(uint32_t lo, uint32_t hi) { return (unsigned long long)hi << 32 | lo; }
__device__ __forceinline__ unsigned long long pairf(float lo, float hi) { return pair(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float lo_of(unsigned long long v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_of(unsigned long long v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ unsigned long long fmul2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ unsigned long long ffma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long fadd2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Byte of a 16-byte chunk in a tile: rows lie in columns of 128 bytes, and a chunk's place in its row is exchanged by the row's last three
// bits, so that eight rows' chunks lie in eight different banks (the 128-byte swizzle of TMA).
template <int TILE>
__device__ __forceinline__ uint32_t chunk_at(int row, int chunk) {
  return (uint32_t)((chunk >> 3) * (TILE * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// Zeros in place of the rows from..to of V.  By a warp.
template <int TILE, int CHUNKS>
__device__ __forceinline__ void clear_rows(uint8_t* tile, int from, int to, int lane) {
  for (int i = from * CHUNKS + lane; i < to * CHUNKS; i += 32)
    *reinterpret_cast<uint4*>(tile + chunk_at<TILE>(i / CHUNKS, i % CHUNKS)) = make_uint4(0u, 0u, 0u, 0u);
  fence_proxy_async_smem();                // before a copy overwrites them
  __syncwarp();
}

// After a wait that has given up: a copy on its way has to land before its CTA's memory is another's.  Bounded, too.
__device__ __forceinline__ void let_land(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 < 10000000ull) {
  }
}

// A row of a tile: its query, and how many keys it sees.
struct Row {
  int b, t, g;
  bool there;            // a row of the entry
  bool counts;           // of a token that counts
  int sees;
};

template <bool L2 = false>
__device__ __forceinline__ Row row_of(const CacheArgs& a, const Entry& x, int r) {
  Row w;
  int i = x.row0 + r;
  const int per = a.T * a.G;
  w.there = i < (x.b < 0 ? a.B * per : per);
  if (!w.there) i = 0;
  w.b = x.b;
  if (x.b < 0) {
    w.b = i / per;
    i -= w.b * per;
  }
  w.t = i / a.G;
  w.g = i - w.t * a.G;
  const int c = count_of<L2>(a, w.b);
  const long long length = read<L2>(a.lengths + w.b);
  // Of the prefix, rows of sequences that have all of it: behind another one's end a row of V may be anything, and NaN times a weight of 0 is NaN.
  w.counts = w.there && w.t < c && (x.b >= 0 || length + c >= a.prefix);
  const long long sees = w.counts ? length + w.t + 1 : 0;
  w.sees = (int)(sees < 0x7fffffffLL ? sees : 0x7fffffffLL);
  return w;
}

__device__ __forceinline__ uint32_t peer_address(uint32_t smem, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_peer(uint32_t at, float x, float y) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(x), "f"(y) : "memory");
}
template <int N>
__device__ __forceinline__ void load_floats(float* v, const float* from) {
  if constexpr (N == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(from);
  else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(from);
}
template <int N>
__device__ __forceinline__ void store_floats(float* to, const float* v) {
  if constexpr (N == 4) *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(v);
  else *reinterpret_cast<float2*>(to) = *reinterpret_cast<const float2*>(v);
}

// What the copying warps hand to the others with a segment (the tiles of one entry and key head that fall to this CTA).
struct Segment {
  int tiles, key0, end;      // 0 tiles: no more segments; the first tile's first key; the entry's end of keys
  int rows;                  // rows that there are
  int direct;                // rows go to the output, else to partial rows
};

template <typename T, int HD, int RG, bool TMA, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, 2)
cache_attn_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const CacheArgs a) {
  using C = Cfg<T, HD, RG, TMA>;
  constexpr int ROWS = C::ROWS, TILE = C::TILE, STAGES = C::STAGES, SUB = C::SUB, SEGS = C::SEGS, KG = C::KG;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* s_k = smem;
  uint8_t* s_v = s_k + STAGES * SUB;
  uint8_t* s_q = s_v + STAGES * SUB;
  float* s_join = reinterpret_cast<float*>(s_q + SEGS * C::Q_BYTES);
  long long* s_dst = reinterpret_cast<long long*>((uint8_t*)s_join + C::JOIN + C::WEIGHTS + C::PEERS);       // [SEGS][ROWS] where a row goes
  long long* s_from = s_dst + SEGS * ROWS;                                           // [ROWS] where a row's query is, for the copying warp
  long long* s_off = s_from + ROWS;                                                  // where the keys and values of a tile start (cp.async)
  int* s_sees = reinterpret_cast<int*>(s_off + (TMA ? 0 : 2 * TILE));                          // [SEGS][ROWS] keys that a row sees, 0: it does not count
  Segment* s_seg = reinterpret_cast<Segment*>(s_sees + SEGS * ROWS);
  uint64_t* full = reinterpret_cast<uint64_t*>(((uintptr_t)(s_seg + SEGS) + 7) & ~(uintptr_t)7);
  uint64_t* empty = full + STAGES;
  uint64_t* seg_full = empty + STAGES;
  uint64_t* seg_empty = seg_full + SEGS;
  uint64_t* joined = seg_empty + SEGS;                                               // sums written, sums read
  volatile int* abort_flag = (volatile int*)(joined + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; i++) {
      mbar_init(&full[i], TMA ? kCopiers : 32 * kCopiers);
      mbar_init(&empty[i], kConsumers);
    }
    for (int i = 0; i < SEGS; i++) {
      mbar_init(&seg_full[i], 33 * kCopiers);    // every lane's copies, and a warp's first one's arrival behind all other stores
      mbar_init(&seg_empty[i], kConsumers);
    }
    mbar_init(&joined[0], kConsumers);
    mbar_init(&joined[1], kConsumers);
    *abort_flag = 0;
    mbar_fence_init();
  }
  // Sums and statistics of the cluster's CTAs, for the columns that this one joins.
  const int peers = CLUSTER ? a.peers : 1, rank = CLUSTER ? (int)cluster_ctarank() : 0, slice = HD / peers;
  float* x_sum = reinterpret_cast<float*>(s_q + C::Q_BYTES);                         // [peers][ROWS][slice]
  float2* x_stat = reinterpret_cast<float2*>((uint8_t*)s_join + C::JOIN + C::WEIGHTS);      // [peers][ROWS]
  if constexpr (CLUSTER) {
    for (int i = threadIdx.x; i < kPeers * ROWS; i += kThreads) x_stat[i] = make_float2(-INFINITY, 0.f);
    cluster_sync_all();                          // all of them are there before one writes to another
  } else {
    __syncthreads();
  }
  pdl_wait();
  pdl_trigger();

  // Registers: 128 a thread at launch, of which the copying warps hand 64 to those that multiply.
  auto copies = [&]() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    const int me = warp - kConsumers;
    Cursor<ROWS, TILE> at;
    if constexpr (CLUSTER) at.start_cluster(a, peers, rank);
    else at.start(a, lane);
    constexpr int MINE = TILE / kCopiers;                            // keys of this warp for cp.async
    constexpr int PER = 32 / C::CHUNKS;                              // rows of one instruction of the warp
    const int sub = lane / C::CHUNKS, chunk = lane % C::CHUNKS;
    const bool inside = chunk * 16 < a.D * (int)sizeof(T);
    // A TMA copy is a box of rows by 128 bytes of keys or of values; they are dealt out to the warps and to their lanes, which take turns at
    // 60 ns a copy.
    const int units = TMA ? TILE / a.box * C::COLS * 2 : 0, unit = lane * kCopiers + me;
    const int box = unit / (2 * C::COLS), col = unit / 2 % C::COLS;  // (columns behind the head's last one: zeros)
    const int bytes = units > me ? (units - me + kCopiers - 1) / kCopiers * a.box * 128 : 0;
    const int unit_to = col * (TILE * 128) + box * a.box * 128;
    // Pages of the next tile, asked for while this one is copied and looked at when its turn comes: of a box a lane, or of a key a lane.
    // -1: behind the last key.
    int page, in_page;
    auto look_up = [&]() {
      const int key = at.x.begin + at.tile * TILE + (TMA ? box * a.box : me * MINE + lane);
      page = -1;
      in_page = 0;
      if ((TMA ? unit < units : lane < MINE) && key < at.x.end) {
        const unsigned p = (unsigned)key / (unsigned)a.page;
        in_page = (int)((unsigned)key - p * (unsigned)a.page);
        const int got = a.table[(key < a.prefix ? 0 : at.x.b) * a.table_stride + p];
        page = got == -1 ? -2 : got;
      }
    };
    int st = 0, sg = 0;
    uint32_t ph = 0, sph = 0;
    // Copies the tile whose pages have been looked up, and asks for the next one's if there is one in the segment.
    auto copy_tile = [&](bool more) {
      if (page < -1 || page >= a.pages) {
        set_status(a.status, ST_BAD_INDEX, at.x.b);
        page = -1;
      }
      if constexpr (TMA) {
        const int pg = page < 0 ? a.pages : page, row = in_page;                     // behind the last page: zeros
        at.tile++;
        if (more) look_up();
        if (!mbar_wait(&empty[st], ph ^ 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 20)) return false;
        if (lane == 0) {
          if (bytes) mbar_expect_tx(&full[st], bytes);
          else mbar_arrive(&full[st]);
        }
        __syncwarp();
        if (unit < units) {
          const bool v = unit & 1;
          tma_load_4d((v ? s_v : s_k) + st * SUB + unit_to, v ? &tm_v : &tm_k, &full[st], col * (128 / (int)sizeof(T)), row, at.h, pg);
        }
        __syncwarp();
      } else {
        long long* off = s_off + me * 2 * MINE;
        if (lane < MINE) {
          off[lane] = page < 0 ? -1 : page * a.k_sp + at.h * a.k_sh + in_page * a.k_sr;
          off[MINE + lane] = page < 0 ? -1 : page * a.v_sp + at.h * a.v_sh + in_page * a.v_sr;
        }
        __syncwarp();
        at.tile++;
        if (more) look_up();
        if (!mbar_wait(&empty[st], ph ^ 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 20)) return false;
        uint8_t* dk = s_k + st * SUB;
        uint8_t* dv = s_v + st * SUB;
#pragma unroll 4
        for (int r = 0; r < MINE; r += PER) {
          const long long ko = off[r + sub], vo = off[MINE + r + sub];
          const int size = ko >= 0 && inside ? 16 : 0;
          const uint32_t to = chunk_at<TILE>(me * MINE + r + sub, chunk);
          cp_async16(dk + to, (const T*)a.k + (size ? ko + chunk * (16 / (int)sizeof(T)) : 0), size);
          cp_async16(dv + to, (const T*)a.v + (size ? vo + chunk * (16 / (int)sizeof(T)) : 0), size);
        }
        __syncwarp();
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[st])) : "memory");
      }
      if (++st == STAGES) { st = 0; ph ^= 1; }
      return true;
    };
    bool first_segment = true;
    const int per = a.T * a.G;
    while (CLUSTER || at.left) {
      // While the pages of the first tile are looked up, the segment is described: where its rows go; its queries are copied behind that tile.
      const int n = (int)min(at.left, (unsigned)(at.x.tiles - at.tile)), tile0 = at.tile;
      if (n > 0) look_up();
      if (!mbar_wait(&seg_empty[sg], sph ^ 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 23)) break;
      const bool whole = n == at.x.tiles, direct = whole && !a.shared;
      const int slot = 2 * blockIdx.x + (first_segment ? 0 : 1);
      const int rows = min(ROWS, (at.x.b < 0 ? a.B * per : per) - at.x.row0);
      if (lane == 0 && me == 0) {
        s_seg[sg] = Segment{n, at.x.begin + tile0 * TILE, at.x.end, rows, direct};
        if (!CLUSTER && tile0 == 0) a.owner[at.e * a.Hkv + at.h] = make_int2(slot, (int)at.shares.cta_of(at.segment0 + at.x.tiles - 1));
      }
      // Whole segments of a batch with a shared prefix leave partial rows too: in the output's order, those of the prefix behind the sequences'.
      // The warps take a quarter of the rows each.
      constexpr int RW = ROWS / kCopiers;
      static_assert(RW >= 1, "rows of a warp");
      if (lane < RW) {
        const int r = me * RW + lane;
        const Row w = row_of(a, at.x, r);
        const long long row = ((long long)w.b * a.T + w.t) * a.H + at.h * a.G + w.g;
        s_sees[sg * ROWS + r] = w.counts ? max(w.sees, 0) : 0;
        s_dst[sg * ROWS + r] = CLUSTER || direct ? row : !whole ? (long long)slot * ROWS + r
                                                      : 2LL * a.ctas * ROWS + (at.x.b < 0 ? (long long)a.B * a.T * a.H : 0) + row;
        s_from[r] = w.counts ? w.b * a.q_sb + w.t * a.q_st + (long long)(at.h * a.G + w.g) * a.q_sh : -1;
      }
      __syncwarp();
      if (n > 0 && !copy_tile(n > 1)) break;
      uint8_t* dq = s_q + sg * C::Q_BYTES;
#pragma unroll 4
      for (int r0 = me * RW; r0 < min(rows, me * RW + RW); r0 += PER) {      // (rows behind the last one: anything, nothing comes of them)
        if (RW < PER && sub >= RW) break;
        const long long from = s_from[r0 + sub];
        const int bytes = from >= 0 && inside ? 16 : 0;
        // (fp32: rows as they are, which all lanes read alike, at offsets that the compiler knows)
        cp_async16(dq + (C::kMma ? chunk_at<ROWS>(r0 + sub, chunk) : (uint32_t)((r0 + sub) * C::CHUNKS + chunk) * 16), (const T*)a.q + (bytes ? from + chunk * (16 / (int)sizeof(T)) : 0), bytes);
      }
      __syncwarp();
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&seg_full[sg])) : "memory");
      if (lane == 0) mbar_arrive(&seg_full[sg]);
      if (++sg == SEGS) { sg = 0; sph ^= 1; }
      first_segment = false;
      at.left -= n;
      bool ok = true;
      for (int i = 1; i < n && ok; i++) ok = copy_tile(i + 1 < n);
      if (!ok || CLUSTER) break;
      if (at.left) at.next_segment(a);
    }
    if (!CLUSTER && at.left == 0 && mbar_wait(&seg_empty[sg], sph ^ 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 23)) {
      if (lane == 0 && me == 0) s_seg[sg] = Segment{0, 0, 0, 0, 0};  // no more
      __syncwarp();
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&seg_full[sg])) : "memory");
      if (lane == 0) mbar_arrive(&seg_full[sg]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (TMA && *abort_flag)
      for (int i = 0; i < STAGES; i++) let_land(&full[i], i < st ? ph : ph ^ 1);
  };

  auto products = [&]() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    int st = 0, sg = 0;
    uint32_t ph = 0, sph = 0, jph = 0;
    const int rg = warp / KG, kg = warp % KG;
    float2* s_stat = reinterpret_cast<float2*>(s_join + (KG == 4 ? 4 * C::RJ : KG == 2 ? ROWS : 0) * C::PAD);
    // Four key groups' sums of the rows from..from + RJ - 1 meet in shared memory; a warp joins every fourth row.
    auto join_rows = [&](const Segment& seg, int from) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&joined[0]);
      if (!mbar_wait(&joined[0], jph, abort_flag, a.status, ST_ATTN_TIMEOUT, 26)) return false;
      jph ^= 1;
      constexpr int CPL = HD / 32;                                     // columns of a lane
      const int col = lane * CPL;
#pragma unroll
      for (int i = 0; i < C::RJ / 4; i++) {
        const int r = i * 4 + warp;
        if (r >= seg.rows - from) break;
        float w[4], top = -INFINITY, l = 0.f, sum[CPL];
#pragma unroll
        for (int k = 0; k < 4; k++) top = fmaxf(top, s_stat[k * C::RJ + r].x);
#pragma unroll
        for (int c = 0; c < CPL; c++) sum[c] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float2 y = s_stat[k * C::RJ + r];
          w[k] = y.x == -INFINITY ? (y.y == 0.f ? 0.f : 1.f) : exp2f(y.x - top);     // (scores of NaN leave no maximum, but a sum)
          l += y.y * w[k];
          float v[CPL];
          load_floats<CPL>(v, s_join + (k * C::RJ + r) * C::PAD + col);
#pragma unroll
          for (int c = 0; c < CPL; c++) sum[c] += v[c] * w[k];
        }
        if constexpr (CLUSTER) {
          const int to = col / slice, at = col - to * slice;
          const uint32_t p = peer_address(smem_u32(x_sum + (rank * ROWS + from + r) * slice + at), to);
#pragma unroll
          for (int c = 0; c < CPL; c += 2) st_peer(p + 4 * c, sum[c], sum[c + 1]);
          if (at == 0) st_peer(peer_address(smem_u32(x_stat + rank * ROWS + from + r), to), top, l);
        } else {
          const long long row = s_dst[sg * ROWS + from + r];
          const bool sees = s_sees[sg * ROWS + from + r], counts = sees && l != 0.f;
          if (col < a.D) {
            if (!seg.direct) {
              store_floats<CPL>(a.part + row * a.D + col, sum);
            } else {
              const float f = counts ? __frcp_rn(l) : 0.f;
#pragma unroll
              for (int c = 0; c < CPL; c++) sum[c] = counts ? sum[c] * f : 0.f;
              if constexpr (C::kMma) {
#pragma unroll
                for (int c = 0; c < CPL; c += 2) *reinterpret_cast<uint32_t*>((T*)a.out + row * a.D + col + c) = Elem<T>::pack(sum[c], sum[c + 1]);
              } else {
                store_floats<CPL>((float*)a.out + row * a.D + col, sum);
              }
            }
          }
          if (!seg.direct && lane == 0) a.stat[row] = sees ? make_float2(top, l) : make_float2(-INFINITY, 0.f);      // (no key is seen: nothing to join)
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&joined[1]);
      return true;
    };
    for (;;) {
      if (!mbar_wait(&seg_full[sg], sph, abort_flag, a.status, ST_ATTN_TIMEOUT, 24)) return;
      const Segment seg = s_seg[sg];
      if (seg.tiles == 0) return;                  // no more; of a cluster, none for this CTA
      const int* sees_of = s_sees + sg * ROWS;
      const long long* dst_of = s_dst + sg * ROWS;

      if constexpr (C::kMma) {
        constexpr int NK = TILE / KG;                                  // keys of this warp
        const int r0 = rg * 16 + (lane >> 2), r1 = r0 + 8;
        // rows of nothing are masked nowhere: what they add up to is not used
        int sees0 = sees_of[r0], sees1 = sees_of[r1];
        const bool idle = !__any_sync(0xffffffffu, sees0 | sees1);
        sees0 = sees0 ? sees0 : 0x7fffffff;
        sees1 = sees1 ? sees1 : 0x7fffffff;
        uint32_t qf[HD / 16][4];
        {
          const uint32_t qa = smem_u32(s_q + sg * C::Q_BYTES);
#pragma unroll
          for (int x = 0; x < HD / 16; x++) ldm4(qf[x], qa + chunk_at<ROWS>(rg * 16 + (lane & 15), x * 2 + (lane >> 4)));
        }
        float o[HD / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 8; j++)
#pragma unroll
          for (int i = 0; i < 4; i++) o[j][i] = 0.f;

        for (int i = 0; i < seg.tiles; i++) {
          if (!mbar_wait(&full[st], ph, abort_flag, a.status, ST_ATTN_TIMEOUT, 21)) return;
          const int key0 = seg.key0 + i * TILE + kg * NK;
          if (!idle && key0 < seg.end) {
            const uint32_t ka = smem_u32(s_k + st * SUB), va = smem_u32(s_v + st * SUB);
            float s[NK / 8][4], odd[2][4];
#pragma unroll
            for (int j = 0; j < NK / 8; j++)
#pragma unroll
              for (int c = 0; c < 4; c++) s[j][c] = 0.f;
            // A warp with few keys has few chains of dependent products: two of half the length for each.
            constexpr bool kHalves = NK == 16;
#pragma unroll
            for (int c = 0; c < 8; c++) odd[c / 4][c % 4] = 0.f;
#pragma unroll
            for (int j = 0; j < NK / 16; j++) {                        // 16 keys: two n8 tiles
              const int row = kg * NK + j * 16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
              for (int x = 0; x < HD / 16; x++) {
                uint32_t b[4];
                ldm4(b, ka + chunk_at<TILE>(row, x * 2 + ((lane >> 3) & 1)));
                mma16<T>(kHalves && x % 2 ? odd[0] : s[2 * j], qf[x], b[0], b[1]);
                mma16<T>(kHalves && x % 2 ? odd[1] : s[2 * j + 1], qf[x], b[2], b[3]);
              }
            }
            if (kHalves) {
#pragma unroll
              for (int c = 0; c < 8; c++) s[c / 4][c % 4] += odd[c / 4][c % 4];
            }
            const int low = min(min(sees0, sees1), seg.end);           // (zeros stand in for keys behind the last one)
            if (__any_sync(0xffffffffu, low - key0 < NK)) {
#pragma unroll
              for (int j = 0; j < NK / 8; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                  const int key = key0 + j * 8 + (lane & 3) * 2 + (c & 1);
                  if (key >= min((c & 2) ? sees1 : sees0, seg.end)) s[j][c] = -INFINITY;
                }
            }
            if (TMA && seg.end - key0 < NK) clear_rows<TILE, C::CHUNKS>(s_v + st * SUB, kg * NK + seg.end - key0, kg * NK + NK, lane);
            float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
            for (int j = 0; j < NK / 8; j++) {
              x0 = fmaxf(x0, fmaxf(s[j][0], s[j][1]));
              x1 = fmaxf(x1, fmaxf(s[j][2], s[j][3]));
            }
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) {
              x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
              x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
            }
            const float n0 = fmaxf(m0, x0 * a.scale_log2), n1 = fmaxf(m1, x1 * a.scale_log2);
            if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
              const float f0 = m0 == -INFINITY ? 0.f : exp2f(m0 - n0), f1 = m1 == -INFINITY ? 0.f : exp2f(m1 - n1);
              m0 = n0;
              m1 = n1;
              l0 *= f0;
              l1 *= f1;
#pragma unroll
              for (int j = 0; j < HD / 8; j++) {
                o[j][0] *= f0;
                o[j][1] *= f0;
                o[j][2] *= f1;
                o[j][3] *= f1;
              }
            }
            const float z0 = m0 == -INFINITY ? 0.f : m0, z1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
            for (int j = 0; j < NK / 8; j++) {
              s[j][0] = exp2f(fmaf(s[j][0], a.scale_log2, -z0));
              s[j][1] = exp2f(fmaf(s[j][1], a.scale_log2, -z0));
              s[j][2] = exp2f(fmaf(s[j][2], a.scale_log2, -z1));
              s[j][3] = exp2f(fmaf(s[j][3], a.scale_log2, -z1));
              l0 += s[j][0] + s[j][1];
              l1 += s[j][2] + s[j][3];
            }
#pragma unroll
            for (int j = 0; j < NK / 16; j++) {
              const uint32_t p[4] = {Elem<T>::pack(s[2 * j][0], s[2 * j][1]), Elem<T>::pack(s[2 * j][2], s[2 * j][3]),
                                     Elem<T>::pack(s[2 * j + 1][0], s[2 * j + 1][1]), Elem<T>::pack(s[2 * j + 1][2], s[2 * j + 1][3])};
              const int row = kg * NK + j * 16 + (lane & 15);
#pragma unroll
              for (int x = 0; x < HD / 16; x++) {                      // 16 columns
                uint32_t b[4];
                ldm4t(b, va + chunk_at<TILE>(row, x * 2 + (lane >> 4)));
                mma16<T>(o[2 * x], p, b[0], b[1]);
                mma16<T>(o[2 * x + 1], p, b[2], b[3]);
              }
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[st]);
          if (++st == STAGES) { st = 0; ph ^= 1; }
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
          l0 += __shfl_xor_sync(0xffffffffu, l0, d);
          l1 += __shfl_xor_sync(0xffffffffu, l1, d);
        }
        if constexpr (KG > 1) {
          auto hand_over = [&](int half, int to_row) {
            const int r = half ? r1 : r0;
            if (r < seg.rows) {
              float* to = s_join + to_row * C::PAD + (lane & 3) * 2;
#pragma unroll
              for (int j = 0; j < HD / 8; j++) *reinterpret_cast<float2*>(to + j * 8) = make_float2(o[j][2 * half], o[j][2 * half + 1]);
              if ((lane & 3) == 0) s_stat[to_row] = half ? make_float2(m1, l1) : make_float2(m0, l0);
            }
          };
          if constexpr (RG == 1) {
            static_assert(C::RJ == 8, "a half of a warp's rows");
#pragma unroll
            for (int half = 0; half < 2; half++) {
              if (half && seg.rows <= 8) break;
              if (!mbar_wait(&joined[1], jph ^ 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 25)) return;      // (the last rows have been read)
              hand_over(half, kg * 8 + (lane >> 2));
              if (!join_rows(seg, half * 8)) return;
            }
          } else {
            // of two key groups one hands its sums to the other
            if (!mbar_wait(&joined[1], jph ^ 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 25)) return;
            if (kg == 1) {
              hand_over(0, r0);
              hand_over(1, r1);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&joined[0]);
            if (!mbar_wait(&joined[0], jph, abort_flag, a.status, ST_ATTN_TIMEOUT, 26)) return;
            jph ^= 1;
#pragma unroll
            for (int half = 0; half < 2; half++) {
              const int r = half ? r1 : r0;
              float& m = half ? m1 : m0;
              float& l = half ? l1 : l0;
              if (kg == 0 && r < seg.rows) {
                const float2 y = s_stat[r];
                const float top = fmaxf(m, y.x);
                const float f = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2f(m - top), w = y.x == -INFINITY ? (y.y == 0.f ? 0.f : 1.f) : exp2f(y.x - top);
                m = top;
                l = l * f + y.y * w;
                const float* from = s_join + r * C::PAD + (lane & 3) * 2;
#pragma unroll
                for (int j = 0; j < HD / 8; j++) {
                  const float2 v = *reinterpret_cast<const float2*>(from + j * 8);
                  o[j][2 * half] = o[j][2 * half] * f + v.x * w;
                  o[j][2 * half + 1] = o[j][2 * half + 1] * f + v.y * w;
                }
              }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&joined[1]);
          }
        }
        if (RG > 1 && kg == 0) {
#pragma unroll
          for (int half = 0; half < 2; half++) {
            const float m = half ? m1 : m0, l = half ? l1 : l0;
            const int r = half ? r1 : r0;
            if (r < seg.rows) {
              const long long row = dst_of[r];
              if (seg.direct) {
                const float f = sees_of[r] && l != 0.f ? __frcp_rn(l) : 0.f;
                T* to = (T*)a.out + row * a.D + (lane & 3) * 2;
#pragma unroll
                for (int j = 0; j < HD / 8; j++)
                  if (j * 8 < a.D)
                    *reinterpret_cast<uint32_t*>(to + j * 8) = f == 0.f ? 0u : Elem<T>::pack(o[j][2 * half] * f, o[j][2 * half + 1] * f);
              } else {
                float* to = a.part + row * a.D + (lane & 3) * 2;
#pragma unroll
                for (int j = 0; j < HD / 8; j++)
                  if (j * 8 < a.D) *reinterpret_cast<float2*>(to + j * 8) = make_float2(o[j][2 * half], o[j][2 * half + 1]);
                if ((lane & 3) == 0) a.stat[row] = sees_of[r] ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
              }
            }
          }
        }
      } else {
        // fp32: a warp's quarter of the keys of a tile for all rows.  Scores: LPK lanes share a key, every LPK-th chunk of its columns each; products with
        // the values: a lane is HD / 32 columns.
        constexpr int KW = TILE / 4, LPK = 32 / KW, CPL = HD / 32;
        const uint8_t* q = s_q + sg * C::Q_BYTES;
        float* s_p = reinterpret_cast<float*>((uint8_t*)s_join + C::JOIN) + warp * (KW * ROWS);      // [KW][ROWS] of this warp
        const int mykey = lane / LPK, slice = lane % LPK;
        float o[ROWS][CPL], m[ROWS], l[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
          m[r] = -INFINITY;
          l[r] = 0.f;
#pragma unroll
          for (int c = 0; c < CPL; c++) o[r][c] = 0.f;
        }
        for (int i = 0; i < seg.tiles; i++) {
          if (!mbar_wait(&full[st], ph, abort_flag, a.status, ST_ATTN_TIMEOUT, 22)) return;
          const int key0 = seg.key0 + i * TILE + warp * KW, there = min(KW, seg.end - key0);
          if (there > 0) {
            const uint8_t* kt = s_k + st * SUB;
            const uint8_t* vt = s_v + st * SUB;
            const int key = key0 + mykey;
            float s[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; r++) s[r] = 0.f;
            const uint8_t* mine = q + slice * 16;
#pragma unroll 4
            for (int c = 0; c < HD / 4 / LPK; c++) {
              const float4 kk = *reinterpret_cast<const float4*>(kt + chunk_at<TILE>(warp * KW + mykey, c * LPK + slice));
#pragma unroll
              for (int r = 0; r < ROWS; r++) {
                const float4 qq = *reinterpret_cast<const float4*>(mine + (r * (HD / 4) + c * LPK) * 16);
                s[r] = fmaf(qq.x, kk.x, s[r]);
                s[r] = fmaf(qq.y, kk.y, s[r]);
                s[r] = fmaf(qq.z, kk.z, s[r]);
                s[r] = fmaf(qq.w, kk.w, s[r]);
              }
            }
            // (step by step over all rows, whose exchanges between lanes do not wait for one another: row by row they took 2 us of a tile's 6)
#pragma unroll
            for (int d = 1; d < LPK; d <<= 1)
#pragma unroll
              for (int r = 0; r < ROWS; r++) s[r] += __shfl_xor_sync(0xffffffffu, s[r], d);
            float top[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
              const int sees = s_sees[sg * ROWS + r];
              s[r] = key < min(sees ? sees : 0x7fffffff, seg.end) ? s[r] : -INFINITY;
              top[r] = s[r];
            }
#pragma unroll
            for (int d = LPK; d < 32; d <<= 1)
#pragma unroll
              for (int r = 0; r < ROWS; r++) top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], d));
            bool moved = false;
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
              top[r] = fmaxf(m[r], top[r] * a.scale_log2);
              moved |= top[r] > m[r];
            }
            if (moved) {                                               // (the same for all lanes)
#pragma unroll
              for (int r = 0; r < ROWS; r++) {
                const float f = m[r] == -INFINITY ? 0.f : exp2f(m[r] - top[r]);
                m[r] = top[r];
                l[r] *= f;
#pragma unroll
                for (int c = 0; c < CPL; c++) o[r][c] *= f;
              }
            }
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
              // (scaled and subtracted in one rounding)
              s[r] = exp2f(fmaf(s[r], a.scale_log2, m[r] == -INFINITY ? 0.f : -m[r]));
              l[r] += slice == 0 ? s[r] : 0.f;                         // this lane's keys; summed over lanes at the end
            }
            if (slice == 0) {
#pragma unroll
              for (int r = 0; r < ROWS; r += 4) *reinterpret_cast<float4*>(s_p + mykey * ROWS + r) = make_float4(s[r], s[r + 1], s[r + 2], s[r + 3]);
            }
            __syncwarp();
#pragma unroll 4
            for (int j = 0; j < there; j++) {                          // (rows of V behind the last key are not read)
              float v[CPL];
              const uint8_t* vr = vt + chunk_at<TILE>(warp * KW + j, lane * CPL / 4);
              if constexpr (CPL == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(vr);
              else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(vr + (lane & 1) * 8);
#pragma unroll
              for (int r = 0; r < ROWS; r += 4) {
                const float4 p = *reinterpret_cast<const float4*>(s_p + j * ROWS + r);
#pragma unroll
                for (int c = 0; c < CPL; c++) {
                  o[r][c] = fmaf(p.x, v[c], o[r][c]);
                  o[r + 1][c] = fmaf(p.y, v[c], o[r + 1][c]);
                  o[r + 2][c] = fmaf(p.z, v[c], o[r + 2][c]);
                  o[r + 3][c] = fmaf(p.w, v[c], o[r + 3][c]);
                }
              }
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[st]);
          if (++st == STAGES) { st = 0; ph ^= 1; }
        }
#pragma unroll
        for (int from = 0; from < ROWS; from += C::RJ) {
          if (from >= seg.rows) break;
          if (!mbar_wait(&joined[1], jph ^ 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 25)) return;      // (the last rows have been read)
#pragma unroll
          for (int r = 0; r < C::RJ; r++) {
            const float sum = warp_sum(l[from + r]);
            float* to = s_join + (warp * C::RJ + r) * C::PAD + lane * CPL;
#pragma unroll
            for (int c = 0; c < CPL; c++) to[c] = o[from + r][c];
            if (lane == 0) s_stat[warp * C::RJ + r] = make_float2(m[from + r], sum);
          }
          if (!join_rows(seg, from)) return;
        }
      }
      if constexpr (CLUSTER) return;
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[sg]);
      if (++sg == SEGS) { sg = 0; sph ^= 1; }
    }
  };

  if (warp >= kConsumers) copies();
  else products();
  if constexpr (CLUSTER) {
    __syncwarp();
    cluster_sync_all();                          // (every wait before it ends, and none reads or writes another's memory behind it)
    if (warp < kConsumers && !*abort_flag) {
      const int rows = s_seg[0].rows;
      for (int i = threadIdx.x; i < rows * slice; i += 32 * kConsumers) {
        const int r = i / slice, col = i - r * slice;
        float top = -INFINITY, l = 0.f, sum = 0.f;
        for (int p = 0; p < peers; p++) top = fmaxf(top, x_stat[p * ROWS + r].x);
        for (int p = 0; p < peers; p++) {
          const float2 y = x_stat[p * ROWS + r];
          if (y.x == -INFINITY && y.y == 0.f) continue;                              // (of a CTA without keys)
          const float w = y.x == -INFINITY ? 1.f : exp2f(y.x - top);
          l += y.y * w;
          sum += x_sum[(p * ROWS + r) * slice + col] * w;
        }
        const int to = rank * slice + col;
        if (to < a.D) ((T*)a.out)[s_dst[r] * a.D + to] = (T)(s_sees[r] && l != 0.f ? sum * __frcp_rn(l) : 0.f);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// many rows of 16 bits: tcgen05
// ---------------------------------------------------------------------------------------------------------------------------
// More than 64 rows share their keys: a batch over its shared prefix, or several tokens of a sequence.  Then the products count and not the keys'
// bytes, and a CTA takes 128 rows over a run of keys: scores and sums in TMEM, Q in shared memory, K and V by TMA in sub-tiles of 64
// keys, weights written over their scores as the second product's operand; two score buffers, so that the next scores are computed while
// a softmax warp (a row a thread) works.  The sum is rescaled only when the maximum has moved by more than 2^8.  Where the row tiles are too few
// for the SMs, the keys are cut into `splits` runs, which leave partial rows.  Four prompts of 2048 tokens behind 2048 others, 16 heads of 128 bf16:
// 187 us, 987 TFLOP/s of the pairs that are seen; a softmax warp's chain bounds it (tensor pipe 51 % busy, exponentials 52 %).
constexpr int kWideRows = 128, kWideKeys = 64, kWideThreads = 256, kWideCopiers = 3;

template <int HD>
struct Wide {
  static constexpr int CH = HD / 64, Q_BYTES = CH * kWideRows * 128, SUB = CH * kWideKeys * 128;
  static constexpr int STAGES = HD == 64 ? 3 : 2;
  static constexpr int SMEM = Q_BYTES + 2 * STAGES * SUB + 1024 + 256 + 2 * kWideKeys * 8;
  static constexpr int COLS = 256, COL_O = 128;
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs to an SM");
};

template <typename T, int HD, bool TMA, bool PREFIX>
__global__ void __launch_bounds__(kWideThreads, 2)
cache_wide_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const CacheArgs a) {
  using C = Wide<HD>;
  constexpr int STAGES = C::STAGES, SUB = C::SUB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = smem;
  uint8_t* s_k = s_q + C::Q_BYTES;
  uint8_t* s_v = s_k + STAGES * SUB;
  uint64_t* q_full = (uint64_t*)(s_v + STAGES * SUB);
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + STAGES;
  uint64_t* v_full = k_empty + STAGES;
  uint64_t* v_empty = v_full + STAGES;
  uint64_t* s_full = v_empty + STAGES;
  uint64_t* p_full = s_full + 2;
  uint64_t* pv_done = p_full + 2;
  long long* s_off = (long long*)(pv_done + 2);                      // where the keys and values of a sub-tile start (cp.async)
  uint32_t* tmem_slot = (uint32_t*)(s_off + 2 * kWideKeys);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 4);
    for (int i = 0; i < STAGES; i++) {
      mbar_init(&k_full[i], kWideCopiers);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], kWideCopiers);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kWideCopiers) {
    tmem_alloc(tmem_slot, C::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Beside the kernel for few rows, which was launched first and has waited for all that came before: this one waits for that one's end alone, and at
  // its own, so that what follows it follows both.  What it reads it reads from L2.
  if (!PREFIX) pdl_wait();
  pdl_trigger();

  // Row tiles of a sequence run from its last one, which sees the most keys, to its first: over the heads of a group, so that the kernel ends on
  // the shortest ones.  (sequence, head, run of keys) by groups, in a group by row tiles.
  const unsigned runs = (unsigned)a.splits * a.Hkv * (PREFIX ? 1 : a.B), per_group = (unsigned)a.wide_group * a.wide_tiles;
  const unsigned group = blockIdx.x / per_group, in_group = blockIdx.x - group * per_group, size = min((unsigned)a.wide_group, runs - group * a.wide_group);
  const int rank = in_group / size;
  unsigned idx = group * a.wide_group + in_group - rank * size;
  const int split = idx % a.splits;
  idx /= a.splits;
  const int h = idx % a.Hkv;
  Entry x;
  x.b = PREFIX ? -1 : (int)(idx / a.Hkv);
  x.row0 = (PREFIX ? rank : a.wide_tiles - 1 - rank) * kWideRows;
  x.begin = 0;
  if (PREFIX) {
    x.end = a.prefix;
  } else {
    const int c = count_of(a, x.b), last = min(a.T * a.G, x.row0 + kWideRows) - 1;
    const long long end = x.row0 / a.G < c ? (long long)a.lengths[x.b] + min(c, last / a.G + 1) : 0;
    x.end = (int)max(0LL, min(end, (long long)a.room));
    if (end > a.room && threadIdx.x == 0 && split == 0) set_status(a.status, ST_BAD_INDEX, x.b);
  }
  x.tiles = (x.end + kWideKeys - 1) / kWideKeys;
  const int first = (int)((long long)x.tiles * split / a.splits), n_kv = (int)((long long)x.tiles * (split + 1) / a.splits) - first;

  if (warp < kWideCopiers) {
    int st = 0;
    uint32_t ph = 0;
    // the page of a key, for sub-tile j; -1: behind the last key
    int page = -1, in_page = 0;
    auto look_up = [&](int key, bool mine) {
      page = -1;
      in_page = 0;
      if (mine && key < x.end) {
        const unsigned p = (unsigned)key / (unsigned)a.page;
        in_page = (int)((unsigned)key - p * (unsigned)a.page);
        const int* entry = a.table + (key < a.prefix ? 0 : x.b) * a.table_stride + p;
        page = read<PREFIX>(entry);
        page = page == -1 ? -2 : page;
      }
    };
    auto check = [&]() {
      if (page < -1 || page >= a.pages) {
        set_status(a.status, ST_BAD_INDEX, x.b);
        page = -1;
      }
    };
    if constexpr (TMA) {
      // boxes of rows by 64 columns, dealt out to the warps and their lanes
      const int units = kWideKeys / a.box * C::CH, unit = lane * kWideCopiers + warp, box = unit / C::CH, col = unit % C::CH;
      const bool mine = unit < units;
      const int bytes = units > warp ? (units - warp + kWideCopiers - 1) / kWideCopiers * a.box * 128 : 0;
      const int to = col * (kWideKeys * 128) + box * a.box * 128;
      auto copy = [&](uint8_t* tile, const CUtensorMap* map, uint64_t* bar, int pg, int row) {
        if (lane == 0) {
          if (bytes) mbar_expect_tx(bar, bytes);
          else mbar_arrive(bar);
        }
        __syncwarp();
        if (mine) tma_load_4d(tile + to, map, bar, col * 64, row, h, pg);
        __syncwarp();
      };
      if (n_kv > 0) look_up(first * kWideKeys + box * a.box, mine);
      int half = 0;                              // 1: keys of a stage have been asked for, its values not
      for (int j = 0; j < n_kv; j++) {
        check();
        const int pg = page < 0 ? a.pages : page, row = in_page;     // behind the last page: zeros
        if (j + 1 < n_kv) look_up((first + j + 1) * kWideKeys + box * a.box, mine);
        if (!mbar_wait(&k_empty[st], ph ^ 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 30)) break;
        copy(s_k + st * SUB, &tm_k, &k_full[st], pg, row);
        half = 1;
        if (!mbar_wait(&v_empty[st], ph ^ 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 31)) break;
        copy(s_v + st * SUB, &tm_v, &v_full[st], pg, row);
        half = 0;
        if (++st == STAGES) { st = 0; ph ^= 1; }
      }
      if (*abort_flag)
        for (int i = 0; i < STAGES; i++) {
          // (keys of stage st whose values' place was waited for in vain have been asked for)
          let_land(&k_full[i], i < st + half ? ph : ph ^ 1);
          let_land(&v_full[i], i < st ? ph : ph ^ 1);
        }
    } else {
      // Key by key with cp.async, which the tensor core sees after a fence of the thread that copied: a sub-tile is handed on when the next copy is
      // on its way.
      constexpr int CHUNKS = HD / 8, PER = 32 / CHUNKS, MOST = (kWideKeys + kWideCopiers - 1) / kWideCopiers;
      const int row0 = warp * MOST, rows = min(MOST, kWideKeys - row0), sub = lane / CHUNKS, chunk = lane % CHUNKS;
      const bool inside = chunk * 8 < a.D;
      long long* off = s_off + 2 * row0;
      uint64_t* waiting = nullptr;
      auto hand_on = [&](uint64_t* next) {
        if (next) asm volatile("cp.async.commit_group;\ncp.async.wait_group 1;" ::: "memory");
        else asm volatile("cp.async.wait_all;" ::: "memory");
        if (waiting) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(waiting);
        }
        waiting = next;
      };
      auto copy = [&](uint8_t* tile, const T* from, const long long* at) {
#pragma unroll 4
        for (int r = 0; r < rows; r += PER) {
          const long long o = r + sub < rows ? at[r + sub] : -1;
          const int size = o >= 0 && inside ? 16 : 0;
          if (r + sub < rows) cp_async16(tile + chunk_at<kWideKeys>(row0 + r + sub, chunk), from + (size ? o + chunk * 8 : 0), size);
        }
      };
      if (n_kv > 0) look_up(first * kWideKeys + row0 + lane, lane < rows);
      bool ok = true;
      for (int j = 0; j < n_kv; j++) {
        check();
        __syncwarp();
        if (lane < rows) {
          off[lane] = page < 0 ? -1 : page * a.k_sp + h * a.k_sh + in_page * a.k_sr;
          off[rows + lane] = page < 0 ? -1 : page * a.v_sp + h * a.v_sh + in_page * a.v_sr;
        }
        __syncwarp();
        if (j + 1 < n_kv) look_up((first + j + 1) * kWideKeys + row0 + lane, lane < rows);
        ok = mbar_wait(&k_empty[st], ph ^ 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 30);
        if (!ok) break;
        copy(s_k + st * SUB, (const T*)a.k, off);
        hand_on(&k_full[st]);
        ok = mbar_wait(&v_empty[st], ph ^ 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 31);
        if (!ok) break;
        copy(s_v + st * SUB, (const T*)a.v, off + rows);
        hand_on(&v_full[st]);
        if (++st == STAGES) { st = 0; ph ^= 1; }
      }
      hand_on(nullptr);
    }
    __syncwarp();
  } else if (warp == kWideCopiers) {
    if (elect_one()) {
      const uint32_t fmt = __is_same(T, __nv_bfloat16) ? 1u : 0u;
      const uint32_t idesc_s = make_idesc(1u, fmt, false, false, kWideRows, kWideKeys);
      const uint32_t idesc_o = make_idesc(1u, fmt, false, true, kWideRows, HD);
      const uint32_t qa = smem_u32(s_q);
      bool ok = n_kv > 0 && mbar_wait(q_full, 0, abort_flag, a.status, ST_ATTN_TIMEOUT, 32);
      int st_s = 0, st = 0;
      uint32_t ph_s = 0, ph = 0;
      auto issue_s = [&](int j) {
        if (!mbar_wait(&k_full[st_s], ph_s, abort_flag, a.status, ST_ATTN_TIMEOUT, 33)) return false;
        tc_fence_after();
        const uint32_t ka = smem_u32(s_k + st_s * SUB);
#pragma unroll
        for (int k = 0; k < HD / 16; k++)
          tc_mma_f16(tmem + (j & 1) * kWideKeys, make_smem_desc_sw128(qa + (k / 4) * (kWideRows * 128) + (k % 4) * 32, 16, 1024),
                     make_smem_desc_sw128(ka + (k / 4) * (kWideKeys * 128) + (k % 4) * 32, 16, 1024), idesc_s, k != 0);
        tc_commit(&k_empty[st_s]);
        tc_commit(&s_full[j & 1]);
        if (++st_s == STAGES) { st_s = 0; ph_s ^= 1; }
        return true;
      };
      if (ok) ok = issue_s(0);
      for (int j = 0; j < n_kv && ok; j++) {
        if (j + 1 < n_kv) ok = issue_s(j + 1);
        ok = ok && mbar_wait(&p_full[j & 1], (j >> 1) & 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 34);
        ok = ok && mbar_wait(&v_full[st], ph, abort_flag, a.status, ST_ATTN_TIMEOUT, 35);
        if (!ok) break;
        tc_fence_after();
        const uint32_t va = smem_u32(s_v + st * SUB), p_tmem = tmem + (j & 1) * kWideKeys;
#pragma unroll
        for (int k = 0; k < kWideKeys / 16; k++)
          tc_mma_f16_ts(tmem + C::COL_O, p_tmem + (k >> 1) * 32 + (k & 1) * 8, make_smem_desc_sw128(va + k * 16 * 128, kWideKeys * 128, 1024), idesc_o,
                        (j | k) != 0);
        tc_commit(&v_empty[st]);
        tc_commit(&pv_done[j & 1]);
        if (++st == STAGES) { st = 0; ph ^= 1; }
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    const Row w = row_of<PREFIX>(a, x, r);
    bool ok = true;
    if (n_kv > 0) {
      // this row of Q, zeros where there is none
      const uint4* q = reinterpret_cast<const uint4*>((const T*)a.q + w.b * a.q_sb + w.t * a.q_st + (long long)(h * a.G + w.g) * a.q_sh);
#pragma unroll
      for (int c = 0; c < HD / 8; c++)
        *reinterpret_cast<uint4*>(s_q + chunk_at<kWideRows>(r, c)) = w.counts && c * 8 < a.D ? (PREFIX ? __ldcg(q + c) : __ldg(q + c)) : make_uint4(0u, 0u, 0u, 0u);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    // keys that this row, all rows and any row of the warp see; a row of nothing is masked nowhere
    const int sees = w.counts ? min(w.sees, x.end) : x.end;
    const int sees_all = __reduce_min_sync(0xffffffffu, sees), sees_any = __reduce_max_sync(0xffffffffu, w.counts ? sees : 0);
    float m = -INFINITY;
    unsigned long long l2 = 0ull;
    const unsigned long long sl2 = pairf(a.scale_log2, a.scale_log2);
    uint32_t s[2][32];
    for (int j = 0; j < n_kv; j++) {
      ok = mbar_wait(&s_full[j & 1], (j >> 1) & 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 36);
      if (!ok) break;
      tc_fence_after();
      const uint32_t at = lane_addr + (j & 1) * kWideKeys;
      const int kv0 = (first + j) * kWideKeys;
      if (kv0 + kWideKeys > x.end) {
        // the last keys of all: zeros behind them in V, whose copy has to be there first
        ok = mbar_wait(&v_full[j % STAGES], (j / STAGES) & 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 37);
        if (!ok) break;
        const int from = x.end - kv0, each = (kWideKeys - from + 3) / 4;
        clear_rows<kWideKeys, HD / 8>(s_v + j % STAGES * SUB, min(kWideKeys, from + quarter * each), min(kWideKeys, from + (quarter + 1) * each), lane);
      }
      if (kv0 >= sees_any) {                      // none of this warp's rows sees any of them
        uint32_t zero[16];
#pragma unroll
        for (int i = 0; i < 16; i++) zero[i] = 0u;
        tmem_st16(at, zero);
        tmem_st16(at + 32, zero);
      } else {
        tmem_ld32(at, s[0]);
        tmem_ld32(at + 32, s[1]);
        tmem_ld_wait();
        if (kv0 + kWideKeys > sees_all) {
#pragma unroll
          for (int c = 0; c < 64; c++)
            if (kv0 + c >= sees) s[c / 32][c % 32] = 0xff800000u;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 64; c++) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(s[c / 32][c % 32]));
        const float next = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2);
        const bool need = m == -INFINITY ? next > m : next - m > 8.f;
        if (__any_sync(0xffffffffu, need)) {
          float f = 1.f;
          if (need) {
            f = m == -INFINITY ? 0.f : exp2f(m - next);
            m = next;
            l2 = fmul2(l2, pairf(f, f));
          }
          if (j > 0) {
            ok = mbar_wait(&pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 38);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < HD / 16; c++) {
              uint32_t ro[16];
              tmem_ld16(lane_addr + C::COL_O + c * 16, ro);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; i++) ro[i] = __float_as_uint(__uint_as_float(ro[i]) * f);
              tmem_st16(lane_addr + C::COL_O + c * 16, ro);
            }
            tmem_st_wait();
          }
        }
        const float z = m == -INFINITY ? 0.f : m;
        const unsigned long long nz = pairf(-z, -z);
#pragma unroll
        for (int g = 1; g >= 0; g--) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const unsigned long long y = ffma2(pair(s[g][2 * i], s[g][2 * i + 1]), sl2, nz);
            const float p0 = exp2f(lo_of(y)), p1 = exp2f(hi_of(y));
            l2 = fadd2(l2, pairf(p0, p1));
            pk[i] = Elem<T>::pack(p0, p1);
          }
          tmem_st16(at + g * 32, pk);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[j & 1]);
    }
    if (ok && n_kv > 0) ok = mbar_wait(&pv_done[(n_kv - 1) & 1], ((n_kv - 1) >> 1) & 1, abort_flag, a.status, ST_ATTN_TIMEOUT, 39);
    if (ok) {
      tc_fence_after();
      const float l = lo_of(l2) + hi_of(l2);
      const bool direct = !PREFIX && a.splits == 1;
      const float f = direct ? (w.counts && l != 0.f ? __frcp_rn(l) : 0.f) : 1.f;
      const long long all = (long long)a.B * a.T * a.H;
      const long long here = w.there ? ((long long)w.b * a.T + w.t) * a.H + h * a.G + w.g : -1;
      const long long row = here < 0 || direct ? here : (PREFIX ? 2LL * a.ctas * a.slot_rows + all : 0) + split * all + here;
      if (row >= 0 && !direct) a.stat[row] = w.counts ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
      // through this warp's part of Q's tile (all products have read it), so that a row leaves in whole lines: 32 rows of 64 fp32 or HD 16-bit values
      uint8_t* buf = s_q + quarter * (32 * 128) * C::CH;
      constexpr int PIECE = HD == 128 ? 64 : 32;                     // fp32 columns at a time
#pragma unroll
      for (int half = 0; half < HD / PIECE; half++) {
        const bool last_half = half == HD / PIECE - 1;
#pragma unroll
        for (int c = 0; c < PIECE / 16; c++) {
          uint32_t ro[16];
          if (n_kv > 0) {
            tmem_ld16(lane_addr + C::COL_O + half * PIECE + c * 16, ro);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 16; i++) ro[i] = 0u;
          }
          if (direct) {
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = f == 0.f ? 0u : Elem<T>::pack(__uint_as_float(ro[2 * i]) * f, __uint_as_float(ro[2 * i + 1]) * f);
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const int chunk = half * (PIECE / 8) + c * 2 + i;
              *reinterpret_cast<uint4*>(buf + (lane * (HD / 8) + (chunk ^ (lane & 7))) * 16) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
              *reinterpret_cast<uint4*>(buf + (lane * (PIECE / 4) + ((c * 4 + i) ^ (lane & 7))) * 16) = make_uint4(ro[4 * i], ro[4 * i + 1], ro[4 * i + 2], ro[4 * i + 3]);
          }
        }
        if (direct && !last_half) continue;
        __syncwarp();
        const int chunks = direct ? HD / 8 : PIECE / 4, per = direct ? 8 : 4, from = direct ? 0 : half * PIECE;
        const int size = direct ? (int)sizeof(T) : 4;
        uint8_t* base = direct ? (uint8_t*)a.out : (uint8_t*)a.part;
        for (int i = lane; i < 32 * chunks; i += 32) {
          const int rr = i / chunks, chunk = i % chunks;
          const long long to = __shfl_sync(0xffffffffu, row, rr);
          if (to >= 0 && from + chunk * per < a.D)
            *reinterpret_cast<uint4*>(base + (to * a.D + from + chunk * per) * size) = *reinterpret_cast<const uint4*>(buf + (rr * chunks + (chunk ^ (rr & 7))) * 16);
        }
        __syncwarp();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWideCopiers) {
    tc_fence_after();
    tmem_dealloc(tmem, C::COLS);
  }
  if (PREFIX) pdl_wait();
}

// Joins the partial rows of a query row: those of the prefix and those of its own sequence.  WPR warps a row, a lane four columns.  First the
// statistics, a part a lane, so that they are one wait and not one for each part; then the sums with their weights, eight parts on their
// way at a time.  With eight warps to a row, every eighth part is a warp's, and they meet in shared memory: where rows are few and parts many,
// which a warp alone would wait for by eights.  Rows that the first kernel has written are left alone; rows that see nothing become zeros.
template <typename T, int ROWS, int WPR>
__global__ void __launch_bounds__(256) cache_join_kernel(const CacheArgs a) {
  __shared__ float s_o[WPR > 1 ? 8 : 1][128];
  __shared__ float2 s_st[8];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WPR;
  const unsigned rows = (unsigned)a.B * a.T * a.H, i = blockIdx.x * (8 / WPR) + warp / WPR;
  if (i >= rows) return;                         // (with eight warps to a row: none)
  const unsigned bt = i / a.H;
  const int head = i - bt * a.H, h = head / a.G, g = head - h * a.G, b = bt / a.T, t = bt - b * a.T;
  T* out = (T*)a.out + (long long)i * a.D;
  // parts: row `first`, then rest + k step, 0 < k < n
  struct Parts { long long first, rest, step; int n; };
  Parts pre = {0, 0, 0, 0}, own = {0, 0, 0, 0};
  const long long whole = 2LL * a.ctas * ROWS;
  auto find = [&](Parts& p, const int2 c, int r, long long at) {
    if (c.x < 0) return true;                     // no keys
    const int cta = c.x >> 1;
    if (cta == c.y) {                             // one CTA had all of it
      p = {at, at, 0, 1};
      return a.shared != 0;
    }
    // The first part may be that CTA's second one (slot 2 cta + 1); the others are the first ones of theirs.
    p = {(long long)c.x * ROWS + r, 2LL * cta * ROWS + r, 2 * ROWS, c.y - cta + 1};
    return true;
  };
  const int per = a.T * a.G, r = t * a.G + g;
  const int all = b * per + r, e_pre = all / ROWS, e_own = a.prefix_tiles + b * a.own_tiles + r / ROWS;
  // (asked for at once, before it is known whether they matter)
  const int2 c_pre = a.prefix_tiles ? a.owner[e_pre * a.Hkv + h] : make_int2(0, 0), c_own = a.wide_own ? make_int2(0, 0) : a.owner[e_own * a.Hkv + h];
  if (t < count_of(a, b)) {
    if (a.wide_prefix) pre = {whole + rows + i, whole + rows + i, rows, a.splits};
    else if (a.prefix_tiles) find(pre, c_pre, all % ROWS, whole + rows + i);
    if (a.wide_own) own = {i, i, rows, a.splits};
    else if (!find(own, c_own, r % ROWS, whole + i)) return;
  }
  const int n = pre.n + own.n;
  float top = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < n; k0 += 32 * WPR) {
    const int k = k0 + lane * WPR + sub;
    long long row = 0;
    float2 st = make_float2(-INFINITY, 0.f);
    if (k < n) {
      row = k < pre.n ? (k == 0 ? pre.first : pre.rest + k * pre.step) : (k == pre.n ? own.first : own.rest + (k - pre.n) * own.step);
      st = a.stat[row];
    }
    const int m = min(32, (n - k0 - sub + WPR - 1) / WPR);
    float4 v[8];
    auto fetch = [&](int j0) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const long long at = __shfl_sync(0xffffffffu, row, (j0 + j) & 31) * a.D + 4 * lane;
        v[j] = j0 + j < m && 4 * lane < a.D ? __ldg(reinterpret_cast<const float4*>(a.part + at)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    };
    fetch(0);                                    // beside the statistics
    const bool none = st.x == -INFINITY && st.y == 0.f;                                     // no key of this part is seen: nothing of it counts
    const float next = fmaxf(top, warp_max(st.x)), f = top == -INFINITY ? 0.f : exp2f(top - next);
    const float w = none ? -1.f : st.x == -INFINITY ? 1.f : exp2f(st.x - next);             // (scores of NaN leave no maximum, but a sum)
    top = next;
    sum = sum * f + warp_sum(none ? 0.f : st.y * w);
#pragma unroll
    for (int c = 0; c < 4; c++) o[c] *= f;
    for (int j0 = 0; j0 < m; j0 += 8) {
      if (j0) fetch(j0);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float wj = __shfl_sync(0xffffffffu, w, (j0 + j) & 31);
        if (j0 + j < m && wj >= 0.f) {
          o[0] += v[j].x * wj;
          o[1] += v[j].y * wj;
          o[2] += v[j].z * wj;
          o[3] += v[j].w * wj;
        }
      }
    }
  }
  if constexpr (WPR > 1) {
    *reinterpret_cast<float4*>(&s_o[sub][4 * lane]) = make_float4(o[0], o[1], o[2], o[3]);
    if (lane == 0) s_st[sub] = make_float2(top, sum);
    __syncthreads();
    if (sub) return;
    top = -INFINITY;
    sum = 0.f;
#pragma unroll
    for (int c = 0; c < 4; c++) o[c] = 0.f;
    for (int k = 0; k < WPR; k++) top = fmaxf(top, s_st[k].x);
    for (int k = 0; k < WPR; k++) {
      const float2 st = s_st[k];
      const float w = st.x == -INFINITY ? (st.y == 0.f ? 0.f : 1.f) : exp2f(st.x - top);
      sum += st.y * w;
#pragma unroll
      for (int c = 0; c < 4; c++) o[c] += s_o[k][4 * lane + c] * w;
    }
  }
  const float f = sum != 0.f ? __frcp_rn(sum) : 0.f;
  if (4 * lane < a.D) {
#pragma unroll
    for (int c = 0; c < 4; c++) o[c] = f == 0.f ? 0.f : o[c] * f;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out + 4 * lane) = make_float4(o[0], o[1], o[2], o[3]);
    else *reinterpret_cast<uint2*>(out + 4 * lane) = make_uint2(Elem<T>::pack(o[0], o[1]), Elem<T>::pack(o[2], o[3]));
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------------
constexpr int kCtas = 2 * 148;
constexpr long long kMost = 0x7fffffffLL - 256;  // positions of a table, and rows of queries: a tile that starts within them ends within 32 bits
constexpr long long kFewRows = 148 * 8;          // rows that are joined by eight warps each: those CTAs all fit at a time

struct Sizes {
  int rows;                      // of a tile of the kernel for few rows
  int own_tiles, prefix_tiles;
  int wide_prefix, wide_own, wide_tiles, splits, peers;
  long long entries, part, stat, owner, total;      // bytes of the workspace's parts
};

// Which kernel takes what, and the workspace.
bool plan(Sizes& z, int dtype, long long B, long long T, long long H, long long Hkv, long long D, int prefix, long long room) {
  if (B * T * H > kMost || room > kMost) return false;
  const long long own = T * (H / Hkv), all = B * own;
  z = Sizes{};
  // Many rows of a sequence: its keys with the prefix among them, which is then read and multiplied for each sequence.  Many rows of the batch alone: its
  // prefix.  (64 sequences behind 16 384 shared positions, 16 heads to each of four keys of 128 bf16, in a graph: of four tokens, who share, 164 us; of five,
  // 80 rows to a key head, who do not, 236, and 333 if every sequence has pages of its own.)
  // us, few rows' kernel | this one, bf16, eight key heads of 128, 32, 48, 64, 96 rows to a key head: 8 sequences of 8 192 positions 63 | 60, 68 | 61, 70 | 62,
  // 117 | 64; of 1 024 to 8 192 41 | 52, 50 | 54, 53 | 57; 64 such ones 211 | 241, 249 | 256, 263 | 254.  Heads of 64 37 | 39, 43 | 43, 45 | 44, 72 | 46.  A shared
  // prefix of 16 384 (and 200 of its own for each sequence) 31 | 39, 37 | 40, 38 | 43, 51 | 46; 256 rows 91 | 57.
  const bool wide = dtype != 2;
  z.wide_own = wide && own > 64;
  const bool shared = prefix > 0 && !z.wide_own;
  z.wide_prefix = shared && wide && all > 64;
  if (z.wide_own || z.wide_prefix) {
    z.wide_tiles = (int)(((z.wide_own ? own : all) + kWideRows - 1) / kWideRows);
    const long long items = z.wide_tiles * Hkv * (z.wide_own ? B : 1);
    // Runs of keys, as many as one round of CTAs (two to an SM) holds, 16 at most and of 256 keys at least in a prefix.
    z.splits = items >= kCtas ? 1 : (int)(kCtas / items);
    if (z.splits > 16) z.splits = 16;
    if (z.wide_prefix && z.splits > prefix / 256) z.splits = prefix / 256 < 1 ? 1 : prefix / 256;
  }
  const long long most = shared && !z.wide_prefix ? all : own;
  z.rows = dtype == 2 ? (most <= 4 ? 4 : most <= 8 ? 8 : 16) : most <= 16 ? 16 : most <= 32 ? 32 : 64;
  const long long ot = z.wide_own ? 0 : (own + z.rows - 1) / z.rows, pt = shared && !z.wide_prefix ? (all + z.rows - 1) / z.rows : 0;
  z.entries = pt + B * ot;
  if (z.entries * Hkv >= 0x7fffffffLL) return false;
  z.own_tiles = (int)ot;
  z.prefix_tiles = (int)pt;
  // A cluster for each (sequence, row tile, key head): as many CTAs, up to eight, as leave all of them on the SMs at a time.  It saves the second
  // kernel, but the longest sequence's CTAs (a full table: `each` tiles at 0.75 us) may be at work when the others have ended, while
  // the list, of half that length on average, takes 2.5 ns for each 32 KB tile on all SMs.  us in a graph, list | clusters, 16 heads of 128 bf16, equal
  // lengths: one sequence of 1 000 positions 9.2 | 7.0, 2 047 10.5 | 8.5, 4 000 13.2 | 11.8; four of 2 000 15.8 | 12.3, 8 000 47.5 | 42.6; sixteen of 500
  // 16.1 | 12.0, 2 000 48.8 | 43.1.
  // The rule was fitted to equal lengths of up to 256 CTAs.  Near 296 it lets go of its limit on `each`, and ragged lengths lose there.  Eight key
  // heads, table of 32 768 positions: 37 sequences (one CTA each) of 8 000 174 | 172, one of 32 000 beside 36 of 500 44 | 397; nine (four CTAs each) of 8 000 53 | 73,
  // one of 32 000 beside eight of 500 36 | 101.
  if (!shared && !z.wide_own && z.rows <= 16 && z.entries * Hkv <= kCtas) {
    const long long tile = 16384 / ((D <= 64 ? 64 : 128) * (dtype == 2 ? 4 : 2)), tiles = (room + tile - 1) / tile;
    z.peers = kPeers;
    while (z.peers > 1 && z.entries * Hkv * z.peers > kCtas) z.peers >>= 1;
    const long long each = (tiles + z.peers - 1) / z.peers, ctas = z.entries * Hkv * z.peers;
    if (each * (300 - ctas) > 2400) z.peers = 0;
    if (z.peers) return true;                                        // without a workspace
  }
  const long long rows = z.wide_own ? (z.splits > 1 ? z.splits * B * T * H : 0)
                                    : 2LL * kCtas * z.rows + (shared ? B * T * H * (1 + (z.wide_prefix ? z.splits : 1)) : 0);
  auto up = [](long long n) { return (n + 255) / 256 * 256; };
  z.part = up(rows * D * 4);
  z.stat = up(rows * 8);
  z.owner = up(z.entries * Hkv * 8);
  z.total = z.part + z.stat + z.owner;
  return true;
}

template <typename K>
int allow_shared(K kernel, int bytes, std::atomic<uint32_t>& done) {
  int dev = 0;
  GB_CUDA_OK(cudaGetDevice(&dev));
  if (dev < 32 && (done.load() >> dev & 1u)) return gbh::E_OK;
  GB_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 32) done.fetch_or(1u << dev);
  return gbh::E_OK;
}

template <typename T, int HD, bool TMA>
int launch_wide(const CUtensorMap& tk, const CUtensorMap& tv, const CacheArgs& a, cudaStream_t s) {
  using C = Wide<HD>;
  static std::atomic<uint32_t> done[2];
  const auto kernel = a.wide_prefix ? cache_wide_kernel<T, HD, TMA, true> : cache_wide_kernel<T, HD, TMA, false>;
  const int rc = allow_shared(kernel, C::SMEM, done[a.wide_prefix ? 1 : 0]);
  if (rc) return rc;
  const long long ctas = (long long)a.wide_tiles * a.splits * a.Hkv * (a.wide_prefix ? 1 : a.B);
  GB_CUDA_OK(gbh::launch(kernel, dim3((unsigned)ctas), dim3(kWideThreads), C::SMEM, s, 1, tk, tv, a));
  return gbh::E_OK;
}

template <typename T, int ROWS>
int launch_join(const CacheArgs& a, cudaStream_t s) {
  const long long rows = (long long)a.B * a.T * a.H;
  // about as many parts as the CTAs are times the segments: above eight, which a warp fetches at a time
  const bool many_parts = a.wide_own || a.wide_prefix ? a.splits > 8 : kCtas > 8LL * a.Hkv * (a.prefix_tiles + (long long)a.B * a.own_tiles);
  if (rows <= kFewRows && many_parts) GB_CUDA_OK(gbh::launch(cache_join_kernel<T, ROWS, 8>, dim3((unsigned)rows), dim3(256), 0, s, 1, a));
  else GB_CUDA_OK(gbh::launch(cache_join_kernel<T, ROWS, 1>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, s, 1, a));
  return gbh::E_OK;
}

template <typename T, int HD, int RG, bool TMA, bool CLUSTER>
int launch_kernel(const CUtensorMap& tk, const CUtensorMap& tv, CacheArgs& a, cudaStream_t s) {
  using C = Cfg<T, HD, RG, TMA>;
  const auto kernel = cache_attn_kernel<T, HD, RG, TMA, CLUSTER>;
  static std::atomic<uint32_t> done{0};
  const int rc = allow_shared(kernel, C::SMEM, done);
  if (rc) return rc;
  if constexpr (CLUSTER) {
    GB_CUDA_OK(gbh::launch(kernel, dim3((unsigned)(a.peers * a.B * a.own_tiles * a.Hkv)), dim3(kThreads), C::SMEM, s, a.peers, tk, tv, a));
    return gbh::E_OK;
  } else {
    GB_CUDA_OK(gbh::launch(kernel, dim3(a.ctas), dim3(kThreads), C::SMEM, s, 1, tk, tv, a));
    if constexpr (C::kMma) {
      if (a.wide_prefix) {
        const int rc = a.box ? (a.D <= 64 ? launch_wide<T, 64, true>(tk, tv, a, s) : launch_wide<T, 128, true>(tk, tv, a, s))
                             : (a.D <= 64 ? launch_wide<T, 64, false>(tk, tv, a, s) : launch_wide<T, 128, false>(tk, tv, a, s));
        if (rc) return rc;
      }
    }
    return launch_join<T, C::ROWS>(a, s);
  }
}

template <typename T, int HD, int RG, bool TMA>
int launch_attn(const CUtensorMap& tk, const CUtensorMap& tv, CacheArgs& a, cudaStream_t s) {
  if constexpr (Cfg<T, HD, RG, TMA>::KG == 4) {
    if (a.peers) return launch_kernel<T, HD, RG, TMA, true>(tk, tv, a, s);
  }
  return launch_kernel<T, HD, RG, TMA, false>(tk, tv, a, s);
}

// (columns, rows of a page, heads, pages) in boxes of 128 bytes by `rows` rows
int cache_map(CUtensorMap* m, int dtype, const void* base, int D, int page, int heads, int pages, const long long* strides, int rows) {
  const int size = dtype == 2 ? 4 : 2;
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)page, (uint64_t)heads, (uint64_t)pages};
  const uint64_t st[3] = {(uint64_t)strides[2] * size, (uint64_t)strides[1] * size, (uint64_t)strides[0] * size};
  const uint32_t box[4] = {128u / size, (uint32_t)rows, 1u, 1u};
  const CUtensorMapDataType type = dtype == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  return gbh::encode_tmap(m, type, 4, base, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Rows of a TMA box, 0 where there can be none: a power of two that divides a page and a tile; strides that a tensor map holds.
int box_of(int page, int dtype, int D, const long long* strides) {
  const int size = dtype == 2 ? 4 : 2;
  int rows = dtype == 2 && D > 64 ? 32 : 64;
  while (rows > 1 && page % rows) rows >>= 1;
  for (int i = 0; i < 6; i++)
    if (strides[i] <= 0 || strides[i] * size >= (1LL << 40)) return 0;
  return rows >= 8 ? rows : 0;
}

template <typename T, bool TMA>
int launch_type(const CUtensorMap& k, const CUtensorMap& v, CacheArgs& a, int rows, cudaStream_t s) {
  if constexpr (Elem<T>::kMma) {
    if (a.D <= 64)
      return rows == 16 ? launch_attn<T, 64, 1, TMA>(k, v, a, s) : rows == 32 ? launch_attn<T, 64, 2, TMA>(k, v, a, s) : launch_attn<T, 64, 4, TMA>(k, v, a, s);
    return rows == 16 ? launch_attn<T, 128, 1, TMA>(k, v, a, s) : rows == 32 ? launch_attn<T, 128, 2, TMA>(k, v, a, s) : launch_attn<T, 128, 4, TMA>(k, v, a, s);
  } else {
    if (rows == 4) return a.D <= 64 ? launch_attn<T, 64, 0, TMA>(k, v, a, s) : launch_attn<T, 128, 0, TMA>(k, v, a, s);
    if (rows == 8) return a.D <= 64 ? launch_attn<T, 64, 2, TMA>(k, v, a, s) : launch_attn<T, 128, 2, TMA>(k, v, a, s);
    return a.D <= 64 ? launch_attn<T, 64, 1, TMA>(k, v, a, s) : launch_attn<T, 128, 1, TMA>(k, v, a, s);
  }
}

template <typename T>
int launch_any(const CUtensorMap& k, const CUtensorMap& v, CacheArgs& a, int rows, cudaStream_t s) {
  if constexpr (Elem<T>::kMma) {
    if (a.wide_own) {
      const int rc = a.box ? (a.D <= 64 ? launch_wide<T, 64, true>(k, v, a, s) : launch_wide<T, 128, true>(k, v, a, s))
                           : (a.D <= 64 ? launch_wide<T, 64, false>(k, v, a, s) : launch_wide<T, 128, false>(k, v, a, s));
      if (rc) return rc;
      return a.splits > 1 ? launch_join<T, 64>(a, s) : gbh::E_OK;
    }
  }
  return a.box ? launch_type<T, true>(k, v, a, rows, s) : launch_type<T, false>(k, v, a, rows, s);
}

}  // namespace

// Bytes of the workspace of gb_cache_attn (0: none), or a negative error.  room: positions that a row of the table holds.
GB_EXPORT long long gb_cache_attn_bytes(int dtype, long long B, long long T, long long H, long long Hkv, long long D, int prefix,
                                        long long room) {
  Sizes z;
  if (dtype < 0 || dtype > 2 || B < 0 || T < 1 || H < 1 || Hkv < 1 || H % Hkv || D < 1 || D > 128 ||
      !plan(z, dtype, B, T, H, Hkv, D, prefix, room)) {
    gbh::set_error("gb_cache_attn: too many rows or positions, or bad sizes (%lld sequences, %lld tokens, %lld and %lld heads of %lld)", B, T, H, Hkv, D);
    return gbh::E_TOO_LARGE;
  }
  return z.total;
}

// Kernels that gb_cache_attn launches.
GB_EXPORT int gb_cache_attn_kernels(int dtype, long long B, long long T, long long H, long long Hkv, long long D, int prefix, long long room) {
  Sizes z;
  if (B < 1 || T < 1 || H < 1 || Hkv < 1 || !plan(z, dtype, B, T, H, Hkv, D, prefix, room)) return 0;
  return z.peers ? 1 : z.wide_own ? 1 + (z.splits > 1) : 2 + z.wide_prefix;
}

// out (B, T, H, D) = attention of q over the pages of its sequences.  sizes (64-bit words; strides in elements, rows aligned to 16 bytes): [0..2]
// strides of q (batch, token, head), [3..8] of both caches (page, head, row), [9..13] B, T, H, Hkv, D, [14] the table's stride, [15] its columns, [16] pages,
// [17] positions of a page, [18] positions, a multiple of the page, that all sequences have in the pages of the first one's.  The workspace belongs to this
// call until its kernels have run.
GB_EXPORT int gb_cache_attn(int dtype, const void* q, const void* k, const void* v, void* out, const long long* sizes, const void* table,
                            const void* lengths, const void* counts, double scale, void* ws, long long ws_bytes, void* stream) {
  if (!sizes) {
    gbh::set_error("gb_cache_attn: null pointer");
    return gbh::E_BAD_ARG;
  }
  for (int i = 9; i <= 18; i++)                  // kept in 32 bits, but for the table's stride
    if (i != 14 && (sizes[i] < 0 || sizes[i] > 0x7fffffffLL)) {
      gbh::set_error("gb_cache_attn: size %d is %lld, beyond 31 bits", i, sizes[i]);
      return gbh::E_TOO_LARGE;
    }
  const long long q_sb = sizes[0], q_st = sizes[1], q_sh = sizes[2], *strides = sizes + 3, table_stride = sizes[14];
  const int B = (int)sizes[9], T = (int)sizes[10], H = (int)sizes[11], Hkv = (int)sizes[12], D = (int)sizes[13], columns = (int)sizes[15];
  const int pages = (int)sizes[16], page = (int)sizes[17], prefix = (int)sizes[18];
  const int size = dtype == 2 ? 4 : 2;
  if (dtype < 0 || dtype > 2 || B < 0 || T < 0 || H < 1 || Hkv < 1 || H % Hkv || D < 1 || D > 128 || D * size % 16) {
    gbh::set_error("gb_cache_attn: bad type or sizes (type %d, %d sequences, %d tokens, %d and %d heads of %d)", dtype, B, T, H, Hkv, D);
    return gbh::E_BAD_ARG;
  }
  if (B == 0 || T == 0) return gbh::E_OK;
  if (!q || !k || !v || !out || !table || !lengths || page < 1 || columns < 1 || pages < 1) {
    gbh::set_error("gb_cache_attn: null pointer or empty cache");
    return gbh::E_BAD_ARG;
  }
  if ((long long)columns * page > kMost || prefix < 0 || prefix > (long long)columns * page || prefix % page || !(scale >= 1e-37 && scale <= 1e38)) {          // (a scale that fp32 holds: 0 times a masked score is NaN)
    gbh::set_error("gb_cache_attn: a table of %d pages of %d positions, %d of them shared, scale %g", columns, page, prefix, scale);
    return gbh::E_BAD_ARG;
  }
  long long cache = 0;
  for (int i = 0; i < 6; i++) cache |= strides[i];
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)ws) & 15 || cache * size % 16 || (uintptr_t)q & 15 || (q_sb | q_st | q_sh) * size % 16 ||
      (uintptr_t)out & 15) {
    gbh::set_error("gb_cache_attn: misaligned tensor");
    return gbh::E_BAD_ARG;
  }
  CacheArgs a = {};
  a.box = box_of(page, dtype, D, strides);
  Sizes z;
  if (!plan(z, dtype, B, T, H, Hkv, D, prefix, (long long)columns * page) || ws_bytes < z.total || (z.total && !ws)) {
    gbh::set_error("gb_cache_attn: workspace of %lld bytes is too small, or too many rows", ws_bytes);
    return gbh::E_TOO_LARGE;
  }
  // (the list of tiles is numbered in 32 bits)
  const long long tiles = ((long long)columns * page + 31) / 32 * Hkv * (z.entries > 0 ? z.entries : 1);
  if (tiles >= 0x7fffffffLL || (long long)z.wide_tiles * z.splits * Hkv * B >= 0x7fffffffLL) {
    gbh::set_error("gb_cache_attn: too many rows");
    return gbh::E_TOO_LARGE;
  }
  a.q = q; a.k = k; a.v = v; a.out = out;
  a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.k_sp = strides[0]; a.k_sh = strides[1]; a.k_sr = strides[2];
  a.v_sp = strides[3]; a.v_sh = strides[4]; a.v_sr = strides[5];
  a.table = (const int*)table; a.table_stride = table_stride;
  a.columns = columns; a.pages = pages; a.page = page; a.room = columns * page;
  a.lengths = (const int*)lengths; a.counts = (const int*)counts;
  a.B = B; a.T = T; a.H = H; a.Hkv = Hkv; a.G = H / Hkv; a.D = D;
  a.prefix = prefix;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.own_tiles = z.own_tiles; a.prefix_tiles = z.prefix_tiles;
  a.shared = prefix > 0 && !z.wide_own;
  a.wide_prefix = z.wide_prefix; a.wide_own = z.wide_own; a.wide_tiles = z.wide_tiles; a.splits = z.splits;
  a.slot_rows = z.rows;
  // Groups of one size, about a round of CTAs each, whose keys and values stay in L2 (of 126 MB) while their tiles run.  Four prompts of 2048
  // tokens behind 2048 others, 64 heads of 16 row tiles: in groups of 16 191 us, 19 212, 32 201, all 212, one by one 211.
  if (z.wide_own || z.wide_prefix) {
    const long long runs = (long long)z.splits * Hkv * (z.wide_own ? B : 1), groups = (runs * z.wide_tiles + kCtas - 1) / kCtas;
    const long long run = (long long)a.room * D * 4 / z.splits, fit = run > 0 ? (64LL << 20) / run : runs, size = (runs + groups - 1) / groups;
    a.wide_group = (int)(size < fit ? size : fit > 1 ? fit : 1);
  }
  a.peers = z.peers;
  a.ctas = kCtas;
  a.part = (float*)ws;
  a.stat = (float2*)((uint8_t*)ws + z.part);
  a.owner = (int2*)((uint8_t*)ws + z.part + z.stat);
  a.status = gbh::status_ptr();
  cudaStream_t s = (cudaStream_t)stream;
  CUtensorMap tk, tv;
  memset(&tk, 0, sizeof(tk));
  memset(&tv, 0, sizeof(tv));
  if (a.box) {
    int rc;
    if ((rc = cache_map(&tk, dtype, k, D, page, Hkv, pages, strides, a.box))) return rc;
    if ((rc = cache_map(&tv, dtype, v, D, page, Hkv, pages, strides + 3, a.box))) return rc;
  }
  if (dtype == 0) return launch_any<__nv_bfloat16>(tk, tv, a, z.rows, s);
  if (dtype == 1) return launch_any<__half>(tk, tv, a, z.rows, s);
  return launch_any<float>(tk, tv, a, z.rows, s);
}
