// extern "C" entry points of the 4-bit key/value cache (declared in include/dscq.h):
// argument checks, then asynchronous launches on the caller's stream.

#include <algorithm>

#include "../../include/dscq.h"
#include "kv4.h"

namespace dscq {

int kv_append(const KvAppend& a, int D, bool is_bf16, bool rotate, hipStream_t stream);
int kv_read(const KvRead& a, int D, bool is_bf16, bool rotate, hipStream_t stream);
int kv_attention(const KvAttend& a, int D, bool is_bf16, void* ws, hipStream_t stream);
int64_t kv_attention_workspace_bytes(int D, int B, int Hq, int H, int max_q, int64_t max_length,
                                     int64_t window);

namespace {

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_cache(const void* cache, int64_t pages, int64_t page_size, int64_t heads, int64_t D) {
  if (D != 64 && D != 128)
    return fail("kv cache: head_dim must be 64 or 128 (got %lld)", (long long)D);
  if (page_size < kKvTile || page_size % kKvTile || page_size > 4096)
    return fail("kv cache: page size must be a multiple of 16 up to 4096 (got %lld)",
                (long long)page_size);
  if (!(pages > 0 && pages <= 0x7FFFFFFFLL && heads > 0 && heads <= 1024))
    return fail("kv cache: invalid dimensions");
  if (!cache || !aligned(cache, 16)) return fail("kv cache: needs a 16-byte aligned buffer");
  return DSCQ_OK;
}

int check_dtype(int dtype) {
  if (dtype != DSCQ_F16 && dtype != DSCQ_BF16)
    return fail("kv cache: only FP16 and BF16 rows are supported");
  return DSCQ_OK;
}

// A window that no sequence reaches the end of is none.
int64_t window_of(int64_t window) { return window > kKvMaxLength ? 0 : window; }

// Rows (query, head) of a sequence: twice as many threads, and a workgroup's more a key/value
// head, make less than 2^32.
constexpr int64_t kMaxRows = (int64_t{1} << 31) - (int64_t{1} << 20);

// Tokens of one call, in as many launches as they take.
constexpr int64_t kMaxTokens = int64_t{1} << 30;

int check_attention(int64_t B, int64_t Hq, int64_t heads, int64_t D, int64_t max_q,
                    int64_t max_length, int64_t window) {
  if (D != 64 && D != 128)
    return fail("kv cache: head_dim must be 64 or 128 (got %lld)", (long long)D);
  if (!(heads > 0 && heads <= 1024 && Hq > 0 && Hq <= 4096 && Hq % heads == 0))
    return fail("kv attention: query heads must be a multiple of the cache's heads");
  if (!(B >= 0 && B <= 65535 && max_q >= 0 && max_q * Hq <= 0x7FFFFFFFLL && max_length >= 0 &&
        window >= 0))
    return fail("kv attention: invalid dimensions");
  return DSCQ_OK;
}

}  // namespace
}  // namespace dscq

using namespace dscq;

extern "C" {

int dscq_kv_append(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                   int64_t k_token_stride, int64_t k_head_stride, const void* v,
                   int64_t v_token_stride, int64_t v_head_stride, int dtype, int64_t T, int64_t Hq,
                   int64_t H, int64_t D, const int64_t* positions, const float* cos,
                   const float* sin, int64_t table_rows, int64_t rotary, int interleaved,
                   int rotate, const int64_t* slots, uint8_t* cache, int64_t pages,
                   int64_t page_size, void* q_out, void* stream) {
  DisarmOnExit disarm;
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check_cache(cache, pages, page_size, H, D)) return rc;
  if (!(T >= 0 && T <= kMaxTokens && Hq >= 0 && Hq <= 4096))
    return fail("kv append: invalid dimensions");
  if (T == 0) return DSCQ_OK;
  if (!k || !v || !slots || (q && (!q_out || Hq == 0))) return fail("kv append: null buffer");
  if (!cos != !sin || (cos && (!positions || table_rows <= 0)))
    return fail("kv append: cos, sin and positions go together");
  if (cos && !(rotary >= 16 && rotary <= D && rotary % 16 == 0))
    return fail("kv append: the turned part of a head must be a multiple of 16 up to head_dim "
                "(got %lld)", (long long)rotary);
  KvAppend a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.k_ts = k_token_stride;
  a.k_hs = k_head_stride;
  a.v_ts = v_token_stride;
  a.v_hs = v_head_stride;
  a.T = T;
  a.Hq = q ? (int32_t)Hq : 0;
  a.cos = cos;
  a.sin = sin;
  a.table_rows = table_rows;
  a.rotary = (int32_t)rotary;
  a.interleaved = interleaved != 0;
  a.positions = positions;
  a.slots = slots;
  a.q_out = q_out;
  a.cache = {cache, pages, (int32_t)page_size, (int32_t)H};
  return kv_append(a, (int)D, dtype == DSCQ_BF16, rotate != 0, static_cast<hipStream_t>(stream));
}

int dscq_kv_read(const uint8_t* cache, int64_t pages, int64_t page_size, int64_t H, int64_t D,
                 const int64_t* slots, int64_t T, int rotate, int dtype, void* k, void* v,
                 void* stream) {
  DisarmOnExit disarm;
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check_cache(cache, pages, page_size, H, D)) return rc;
  if (!(T >= 0 && T <= kMaxTokens)) return fail("kv read: invalid dimensions");
  if (T == 0) return DSCQ_OK;
  if (!slots || !k || !v) return fail("kv read: null buffer");
  KvRead a;
  a.cache = {const_cast<uint8_t*>(cache), pages, (int32_t)page_size, (int32_t)H};
  a.slots = slots;
  a.T = T;
  a.k = k;
  a.v = v;
  return kv_read(a, (int)D, dtype == DSCQ_BF16, rotate != 0, static_cast<hipStream_t>(stream));
}

int64_t dscq_kv_attention_workspace_bytes(int64_t B, int64_t Hq, int64_t H, int64_t D,
                                          int64_t max_q, int64_t max_length, int64_t window) {
  if (int rc = check_attention(B, Hq, H, D, max_q, max_length, window)) return rc;
  if (B == 0 || max_q == 0) return 0;
  return kv_attention_workspace_bytes((int)D, (int)B, (int)Hq, (int)H, (int)max_q, max_length,
                                      window_of(window));
}

int dscq_kv_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype,
                      int64_t T, int64_t Hq, const uint8_t* cache, int64_t pages,
                      int64_t page_size, int64_t H, int64_t D, const int32_t* tables,
                      int64_t width, const int32_t* lengths, const int32_t* starts, int64_t B,
                      int64_t max_q, int64_t max_length, float scale, int64_t window, void* out,
                      float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  DisarmOnExit disarm;
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check_cache(cache, pages, page_size, H, D)) return rc;
  if (int rc = check_attention(B, Hq, H, D, max_q, max_length, window)) return rc;
  if (!(T >= 0 && T <= kMaxTokens && width >= 0 && width <= kKvMaxLength / page_size &&
        std::min(max_q, T) * Hq <= kMaxRows))
    return fail("kv attention: invalid dimensions");
  if (!(scale > 0.0f && scale < 3.0e38f)) return fail("kv attention: scale must be positive");
  if (T == 0) return DSCQ_OK;
  const bool none = B == 0 || max_q == 0;
  if (!out || (!none && (!q || !lengths || (width && !tables))))
    return fail("kv attention: null buffer");
  if (!none && !starts && max_q != 1)
    return fail("kv attention: without starts every sequence has one query");
  if (!none && !starts && T != B)
    return fail("kv attention: without starts there are B queries");
  const int64_t need = none ? 0
                            : kv_attention_workspace_bytes((int)D, (int)B, (int)Hq, (int)H,
                                                           (int)max_q, max_length,
                                                           window_of(window));
  if (need && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
    return fail("kv attention: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  KvAttend a;
  a.q = q;
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.T = T;
  a.cache = {const_cast<uint8_t*>(cache), pages, (int32_t)page_size, (int32_t)H};
  a.Hq = (int32_t)Hq;
  a.tables = tables;
  a.width = width;
  a.lengths = lengths;
  a.starts = starts;
  a.B = (int32_t)B;
  a.max_q = (int32_t)max_q;
  a.max_length = max_length;
  a.scale = scale;
  a.window = window_of(window);
  a.out = out;
  a.lse = lse;
  return kv_attention(a, (int)D, dtype == DSCQ_BF16, workspace, static_cast<hipStream_t>(stream));
}

}  // extern "C"
