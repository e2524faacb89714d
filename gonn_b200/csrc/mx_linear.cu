// Layers on microscaled products in one call each: rows quantised and multiplied with quantised weights; a training layer's forward
// and backward.  (A layer's host time is that of its calls: as three to seven of them a small training layer took 260 us.)
#include "mx.cuh"

using namespace gbmx;

GB_EXPORT int gb_mx_quantize(int dtype, int fmt, const void* x, long long ld, void* data, void* scales, long long rows, long long K, void* stream);
GB_EXPORT int gb_mx_quantize_both(int dtype, const void* x, long long ld, void* data, void* scales, void* data_t, void* scales_t, float* sums, void* column_sums,
                                  int sum_dtype, long long rows, long long K, void* stream);
GB_EXPORT int gb_mx_matmul(int fmt, const void* a, const void* sa, const void* b, const void* sb, void* c, long long ldc, const void* bias, int bias_f32, long long M,
                           long long N, long long K, int out, int act, void* stream);
GB_EXPORT int gb_mx_matmul_rows(int dtype, int fmt, const void* x, long long ld, const void* b, const void* sb, void* c, long long ldc, const void* bias, int bias_f32,
                                long long M, long long N, long long K, int out, int act, void* stream);

namespace {

constexpr int kFew = 16;         // rows that the product's kernel quantises itself

long long up256(long long n) { return (n + 255) & ~255LL; }
bool fits(long long rows, long long K) { return rows > 0 && K > 0 && rows <= 0x7fffffffLL && K <= (1LL << 30); }
long long code_bytes(long long rows, long long K, int fmt) { return up256(rows * row_bytes((int)K, fmt)); }
long long packed_bytes(long long rows, long long K, int fmt) { return code_bytes(rows, K, fmt) + up256((rows + 127) / 128 * pieces((int)K, fmt) * 512); }

// Pieces of a buffer, each on a 256-byte boundary.
struct Packed {
  uint8_t *codes, *scales;
};
struct Carver {
  uint8_t* at;
  Packed packed(long long rows, long long K, int fmt) {
    Packed p{at, at + code_bytes(rows, K, fmt)};
    at += packed_bytes(rows, K, fmt);
    return p;
  }
  uint8_t* bytes(long long n) {
    uint8_t* p = at;
    at += up256(n);
    return p;
  }
};

// Bytes of a training layer's buffers: what it keeps from forward to backward, and the scratch of either.
long long kept_bytes(long long M, long long N, long long K, int need_x, int need_w) { return (need_w ? packed_bytes(K, M, FP8) : 0) + (need_x ? packed_bytes(K, N, FP8) : 0); }
long long forward_bytes(long long M, long long N, long long K) { return packed_bytes(M, K, FP8) + packed_bytes(N, K, FP8); }
long long backward_bytes(long long M, long long N, long long K) {
  return packed_bytes(M, N, FP8) + packed_bytes(N, M, FP8) + up256((M + 127) / 128 * N * 4);
}

// need: bytes of scratch, 0 where the extents are bad.
bool bad(const char* what, long long M, long long N, long long K, const void* scratch, long long have, long long need) {
  if (need <= 0) {
    gbh::set_error("%s: bad extents %lld x %lld x %lld", what, M, N, K);
    return true;
  }
  if (scratch == nullptr || ((uintptr_t)scratch & 255) || have < need) {
    gbh::set_error("%s: scratch of %lld bytes on a 256-byte boundary, %lld are needed", what, have, need);
    return true;
  }
  return false;
}

}  // namespace

// Scratch bytes of gb_mx_linear, 0 for none (16 rows at most) and for bad extents.
GB_EXPORT long long gb_mx_linear_bytes(long long M, long long N, long long K, int fmt) {
  return M > kFew && fits(M, K) && fits(N, K) ? packed_bytes(M, K, fmt) : 0;
}

// y (M x N, of x's type or `out`) = act(Q(x) W^T + bias): x M x K, rows `ld` apart; W quantised (N, K).
GB_EXPORT int gb_mx_linear(int dtype, int fmt, const void* x, long long ld, const void* w, const void* sw, void* y, const void* bias, int bias_f32, long long M, long long N,
                           long long K, int out, int act, void* scratch, long long scratch_bytes, void* stream) {
  if (M <= kFew) return gb_mx_matmul_rows(dtype, fmt, x, ld, w, sw, y, N, bias, bias_f32, M, N, K, out, act, stream);
  if (bad("gb_mx_linear", M, N, K, scratch, scratch_bytes, gb_mx_linear_bytes(M, N, K, fmt))) return gbh::E_BAD_ARG;
  Carver c{(uint8_t*)scratch};
  const Packed q = c.packed(M, K, fmt);
  if (int rc = gb_mx_quantize(dtype, fmt, x, ld, q.codes, q.scales, M, K, stream)) return rc;
  return gb_mx_matmul(fmt, q.codes, q.scales, w, sw, y, N, bias, bias_f32, M, N, K, out, act, stream);
}

// Bytes of a training layer: which 0: kept from forward to backward, 1: forward's scratch, 2: backward's.  0 for bad extents.
GB_EXPORT long long gb_mx_train_bytes(long long M, long long N, long long K, int need_x, int need_w, int which) {
  if (!fits(M, K) || !fits(N, K) || !fits(M, N) || !fits(N, M) || !fits(K, M)) return 0;
  return which == 0 ? kept_bytes(M, N, K, need_x, need_w) : which == 1 ? forward_bytes(M, N, K) : backward_bytes(M, N, K);
}

// y (M x N, x's type) = Q(x) Q(W)^T + bias in MXFP8.  need_x, need_w: whose gradients will be asked for; kept: the codes that those read.
GB_EXPORT int gb_mx_train_forward(int dtype, int wdtype, const void* x, long long ldx, const void* w, long long ldw, void* y, const void* bias, int bias_f32, long long M,
                                  long long N, long long K, int need_x, int need_w, void* kept, long long kept_size, void* scratch, long long scratch_size, void* stream) {
  if (bad("gb_mx_train_forward", M, N, K, scratch, scratch_size, gb_mx_train_bytes(M, N, K, need_x, need_w, 1))) return gbh::E_BAD_ARG;
  if ((need_x || need_w) && bad("gb_mx_train_forward", M, N, K, kept, kept_size, kept_bytes(M, N, K, need_x, need_w))) return gbh::E_BAD_ARG;
  Carver c{(uint8_t*)scratch}, k{(uint8_t*)kept};
  const Packed xq = c.packed(M, K, FP8), wq = c.packed(N, K, FP8);
  int rc;
  if (need_w) {
    const Packed t = k.packed(K, M, FP8);
    rc = gb_mx_quantize_both(dtype, x, ldx, xq.codes, xq.scales, t.codes, t.scales, nullptr, nullptr, 0, M, K, stream);
  } else {
    rc = gb_mx_quantize(dtype, FP8, x, ldx, xq.codes, xq.scales, M, K, stream);
  }
  if (rc) return rc;
  if (need_x) {
    const Packed t = k.packed(K, N, FP8);
    rc = gb_mx_quantize_both(wdtype, w, ldw, wq.codes, wq.scales, t.codes, t.scales, nullptr, nullptr, 0, N, K, stream);
  } else {
    rc = gb_mx_quantize(wdtype, FP8, w, ldw, wq.codes, wq.scales, N, K, stream);
  }
  if (rc) return rc;
  return gb_mx_matmul(FP8, xq.codes, xq.scales, wq.codes, wq.scales, y, N, bias, bias_f32, M, N, K, dtype, 0, stream);
}

// dx (M x K, of type dtype_x) = Q(dy) Q(W^T)^T, dw (N x K, dtype_w) = Q(dy^T) Q(x^T)^T, db (N, dtype_b) = column sums of dy; null: not
// asked for (db only with dw).  kept: what gb_mx_train_forward left.
GB_EXPORT int gb_mx_train_backward(int dtype, const void* dy, long long ld, const void* kept, void* dx, int dtype_x, void* dw, int dtype_w, void* db, int dtype_b, long long M,
                                   long long N, long long K, void* scratch, long long scratch_size, void* stream) {
  if (bad("gb_mx_train_backward", M, N, K, scratch, scratch_size, gb_mx_train_bytes(M, N, K, 1, 1, 2))) return gbh::E_BAD_ARG;
  if (db != nullptr && dw == nullptr) {
    gbh::set_error("gb_mx_train_backward: db comes with dw only");
    return gbh::E_BAD_ARG;
  }
  if (kept == nullptr || ((uintptr_t)kept & 255)) {
    gbh::set_error("gb_mx_train_backward: what the forward pass kept, on a 256-byte boundary, is needed");
    return gbh::E_BAD_ARG;
  }
  Carver c{(uint8_t*)scratch}, k{(uint8_t*)const_cast<void*>(kept)};
  const Packed g = c.packed(M, N, FP8), gt = c.packed(N, M, FP8);
  float* sums = (float*)c.bytes((M + 127) / 128 * N * 4);
  int rc = 0;
  if (dw != nullptr) rc = gb_mx_quantize_both(dtype, dy, ld, g.codes, g.scales, gt.codes, gt.scales, db != nullptr ? sums : nullptr, db, dtype_b, M, N, stream);
  else if (dx != nullptr) rc = gb_mx_quantize(dtype, FP8, dy, ld, g.codes, g.scales, M, N, stream);
  if (rc) return rc;
  Packed xt{};
  if (dw != nullptr) xt = k.packed(K, M, FP8);
  if (dx != nullptr) {
    const Packed wt = k.packed(K, N, FP8);
    if ((rc = gb_mx_matmul(FP8, g.codes, g.scales, wt.codes, wt.scales, dx, K, nullptr, 0, M, K, N, dtype_x, 0, stream))) return rc;
  }
  if (dw != nullptr) rc = gb_mx_matmul(FP8, gt.codes, gt.scales, xt.codes, xt.scales, dw, K, nullptr, 0, N, K, M, dtype_w, 0, stream);
  return rc;
}
