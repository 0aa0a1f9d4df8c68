// Attention of many rows over the 4-bit key/value cache: prompts and their chunks.
//
// The mathematics of kv4_attend.hip.  With hundreds of rows a key/value head the products
// bound the time, and next to them the softmax (an exponential and four other operations a
// score) and the unpacking, so the codes are unpacked once for a workgroup: its four or
// eight waves take 64 or 128 tokens in turn, a 16-token tile each, and leave keys and values
// in LDS (twice, so that the next tokens are written while these are used), values as fp16 and
// keys in the queries' type, which holds their whole numbers exactly and is then the queries'
// own: every wave multiplies all of them with 32 rows of its own, which it holds in registers
// as they are, but for a power of two.
// 32 x 32 x 16 products: S^T (32 tokens x 32 rows) leaves lane (c, h) = (lane % 32, lane / 32)
// the scores of row c and tokens 8 a + 4 h + i, which as they lie are the operand of
// O^T += V^T P^T over the token order 16 s + 4 h + 0..3, 16 s + 8 + 4 h + 0..3; V^T is stored
// in that order.
//
// A value's scale f' goes into the exponent: with t = s log2 e + log2 f' the weight times the
// scale is 2^(t - reference) at once, and the softmax sum adds it times 1 / f'.  The products
// start from (log2 f') / (f scale log2 e), so one multiply-add makes t of them.  The reference
// follows the row's largest t, which may pass it by eight binary places before it moves.
//
// Measured: 4096 queries after 12288 tokens, 64 query and 8 key/value heads of 128, bf16:
// 1.97 ms (980 TFLOP/s of 4 D operations a visible pair; a large library product of the
// type reaches 1190).  The matrix pipes are busy 43% of the cycles, a third of that beside
// vector instructions (2.1 GHz under this load).  Without its exponentials the kernel would
// take 3% less, without reading values from LDS 2%, without unpacking 4%, with an eighth of
// either product 20%.  2048 queries of 32 heads, fp16: 72 us (480 TFLOP/s): 256 workgroups,
// the longest of them 64 steps of 1.2 us one after another.  64 rows a wave (half the LDS
// reads a product) do not fit its registers: 6.1 ms.  Instructions interleaved by hand, wave
// priorities round the products and other orders of the workgroups made no difference.
//
// LDS.  A key row is a token's D 16-bit numbers, a value row an element's of all tokens; both
// are 16 bytes longer than that, and value rows move on by 16 more after every eight, so
// that the eight lanes that read or write 16 bytes together (and the sixteen that write 8)
// meet all banks, and a lane's places differ by constants.

#include <algorithm>

#include "kv4_attend.h"

namespace dscq {

namespace {

// A workgroup of NW waves takes 32 NW rows, 16 NW tokens at a time.
template <int D, int NW>
struct Layout {
  static constexpr int kTokens = 16 * NW, kSteps = kTokens / 32;
  static constexpr int kKeyRow = 2 * D + 16, kValueRow = 2 * kTokens + 16;  // bytes
  // A buffer (there are two): keys, values, and for each token three fp32 numbers: the
  // factor of its scores, what they start from, and one over its value's scale; then a word
  // a tile, not 0 where one of its values is not finite.
  static constexpr int kKeys = kTokens * kKeyRow;
  static constexpr int kFactors = kKeys + D * kValueRow + D * 2;
  static constexpr int kStarts = kFactors + 4 * kTokens, kInverses = kStarts + 4 * kTokens;
  static constexpr int kBad = kInverses + 4 * kTokens;
  static constexpr int kAll = kBad + 4 * NW;

  static __host__ __device__ constexpr int value_row(int d) {
    return d * kValueRow + (d >> 3) * 16;
  }
};

// Eight numbers as a product with rows of type T takes them; whole numbers of fp16 so.
template <typename T>
struct Operand {
  typedef h8 V;
  static constexpr float kRows = 1.0f;  // what rows are multiplied by
  static __device__ __forceinline__ V rows(const Raw<T>& x) { return __builtin_bit_cast(V, x.w); }
  static __device__ __forceinline__ V of(const h2 e[4]) { return join8(e[0], e[1], e[2], e[3]); }
  static __device__ __forceinline__ f16 mfma(V a, V b, f16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Operand<bf16> {
  typedef __bf16 V __attribute__((ext_vector_type(8)));
  // Products of the largest queries with D whole numbers stay within fp32 (2^127 2^-16 2^11).
  static constexpr float kRows = 0x1p-16f;
  static __device__ __forceinline__ V rows(const Raw<bf16>& x) {
    float y[8];
    to_f32(x, y);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_pair<bf16>(y[2 * i] * kRows, y[2 * i + 1] * kRows);
    return __builtin_bit_cast(V, make_uint4(w[0], w[1], w[2], w[3]));
  }
  static __device__ __forceinline__ V of(const h2 e[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // the upper halves of two fp32 numbers
      w[i] = __builtin_amdgcn_perm(__float_as_uint((float)e[i][1]), __float_as_uint((float)e[i][0]),
                                   0x07060302u);
    return __builtin_bit_cast(V, make_uint4(w[0], w[1], w[2], w[3]));
  }
  static __device__ __forceinline__ f16 mfma(V a, V b, f16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// Words below fp32's smallest normal number are a scale of 0, as a cache holds where nothing
// was stored: their rows are zeros.  Factors of scores below kLeastFactor are none, so that
// logarithms of scales over them stay finite.
constexpr uint32_t kLeastWord = 0x00800000u;
constexpr float kLeastFactor = 0x1p-118f;

// One wave's tile of the next tokens, between memory and LDS: the keys while the first half
// of a step computes, the values during the second, so that one of them is in registers.
template <int D, typename T, int NW>
struct Stage {
  using L = Layout<D, NW>;
  using V = typename Operand<T>::V;
  Words<D> codes;
  uint32_t kw, vw;  // the words of token lane % 16
  uint4 vq;         // the values' words of the quad
  const uint8_t *tile_codes, *tile_words;
  int token;     // the tile's first
  bool there;

  // Lane: key lane % 16, quarter lane / 16; values: chunk and quad such that sixteen lanes
  // that write together hold eight chunks and both halves of a 16-byte place.
  static __device__ __forceinline__ int chunk(int lane) {
    return (lane & 7) | ((lane >> 1) & 8);
  }
  static __device__ __forceinline__ int quad(int lane) {
    return ((lane >> 2) & 2) | (lane >> 5);
  }

  __device__ __forceinline__ void load_keys(const KvAttend& a, const uint8_t* head,
                                            int64_t page_bytes, Place p, int tile, int lane) {
    there = p.page >= 0 && p.page < a.cache.pages;
    token = tile * kKvTile;
    const int P = a.cache.P;
    const uint8_t* block = head + (there ? p.page * page_bytes : 0);
    tile_codes = block + p.at * (8 * D);
    tile_words = block + P * D + p.at * (4 * kKvTile);
    codes = load_words<D>(tile_codes + lane * (D / 8));
    kw = *reinterpret_cast<const uint32_t*>(tile_words + (lane & 15) * 4);
    vw = *reinterpret_cast<const uint32_t*>(tile_words + P * 4 + (lane & 15) * 4);
  }
  __device__ __forceinline__ void load_values(int P, int lane) {
    codes = load_words<D>(tile_codes + P * (D / 2) + (quad(lane) * 16 + chunk(lane)) * (D / 8));
    vq = *reinterpret_cast<const uint4*>(tile_words + P * 4 + quad(lane) * 16);
  }

  __device__ __forceinline__ void store_keys(uint8_t* lds, int wave, int lane, float to2,
                                             int begin, int end, const Masks& masks) const {
    const int g = lane >> 4, t = wave * kKvTile + (lane & 15);
    // A key whose scores are 0 whatever its codes: zeros, with a factor that has a reciprocal.
    const bool none = fabsf(__uint_as_float(kw) * to2) < kLeastFactor;
    const uint32_t zero = none ? 0u : kw;
    const ZeroPair z = zero_pair(zero, zero, masks);
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
      h2 e[4];
      unpack_word(none ? 0u : codes.w[w], z, masks, e);
      *reinterpret_cast<V*>(lds + t * L::kKeyRow + g * (D / 2) + w * 16) = Operand<T>::of(e);
    }
    const int j = token + (lane & 15);
    const bool in = there && j >= begin && j < end;
    const float y = vw < kLeastWord ? 1.0f : __uint_as_float(vw);
    const bool bad = in && !(y > 0.0f);
    const uint64_t any = __builtin_amdgcn_ballot_w64(bad);
    if (lane == 0) *(reinterpret_cast<uint32_t*>(lds + L::kBad) + wave) = any != 0;
    if (g == 0) {
      // The three numbers of a token.  A page that is not there: infinite scores, so that it
      // is noticed; a token outside the workgroup's: zeros (whoever looks there masks it);
      // one whose value is zeros: as of scale 1; is not finite: that, with the sign to tell.
      const float f = none ? 1.0f : __uint_as_float(kw) * to2;
      const float start = __builtin_amdgcn_logf(y) * __builtin_amdgcn_rcpf(f);
      float* out = reinterpret_cast<float*>(lds + L::kFactors) + t;
      out[0] = !there ? INFINITY : in ? f : 0.0f;
      out[L::kTokens] = !there ? INFINITY : in && !bad ? start : 0.0f;
      out[2 * L::kTokens] = bad ? -1.0f : in ? __builtin_amdgcn_rcpf(y) : 0.0f;
    }
  }
  __device__ __forceinline__ void store_values(uint8_t* lds, int wave, int lane,
                                               const Masks& masks) const {
    const int c = chunk(lane), q = quad(lane);
    const int to = L::kKeys + L::value_row(c * (D / 16)) + wave * 32 + (q & 1) * 16 + (q >> 1) * 8;
    uint4 words = vq;
    Words<D> from = codes;
    const uint32_t least = min(min(vq.x, vq.y), min(vq.z, vq.w));
    if (__builtin_amdgcn_ballot_w64(least < kLeastWord)) {
      // Values of scale 0: zeros, whatever their codes (two tokens a word of codes).
      const uint32_t keep[2] = {(vq.x < kLeastWord ? 0u : 0xFFFFu) |
                                    (vq.y < kLeastWord ? 0u : 0xFFFF0000u),
                                (vq.z < kLeastWord ? 0u : 0xFFFFu) |
                                    (vq.w < kLeastWord ? 0u : 0xFFFF0000u)};
      words = make_uint4(vq.x & keep[0], vq.y & (keep[0] >> 16), vq.z & keep[1],
                         vq.w & (keep[1] >> 16));
#pragma unroll
      for (int m = 0; m < D / 32; ++m) from.w[m] &= keep[m / (D / 64)];
    }
    const ZeroPair z[2] = {zero_pair(words.x, words.y, masks), zero_pair(words.z, words.w, masks)};
#pragma unroll
    for (int m = 0; m < D / 64; ++m) {
      h2 e[2][4];
      unpack_word(from.w[m], z[0], masks, e[0]);
      unpack_word(from.w[D / 64 + m], z[1], masks, e[1]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<h4*>(lds + to + (4 * m + j) * L::kValueRow) =
            (h4){e[0][j][0], e[0][j][1], e[1][j][0], e[1][j][1]};
      }
    }
  }
};

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// The running state of a wave's 32 rows.
template <int D, typename T, int NW>
struct Wave {
  using L = Layout<D, NW>;
  using V = typename Operand<T>::V;
  V q[D / 16];
  f16 o[D / 32];
  float off = 0.0f, limit = -INFINITY, l = 0.0f;  // less the reference; what moves it; the sum
  int lo, hi, all_lo, all_hi;                     // the row's tokens; those of all rows
  int key_at, value_at, word_at;                  // the lane's places in LDS

  __device__ __forceinline__ void clear(int lane) {
    const int c = lane & 31, h = lane >> 5;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) o[d] = (f16)(0.0f);
    key_at = c * L::kKeyRow + 16 * h;
    value_at = L::kKeys + L::value_row(c) + 16 * h;
    word_at = L::kFactors + 16 * h;
  }

  // q . (c - z) + start of 32 tokens.
  __device__ __forceinline__ f16 scores(const uint8_t* lds, int sub) const {
    f16 t;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const f4 x = *reinterpret_cast<const f4*>(lds + word_at + 4 * L::kTokens +
                                                (32 * sub + 8 * n) * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) t[4 * n + i] = x[i];
    }
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const V k = *reinterpret_cast<const V*>(lds + key_at + sub * 32 * L::kKeyRow + ks * 32);
      t = Operand<T>::mfma(k, q[ks], t);
      // Not all keys in registers at once.
      if (ks == D / 32 - 1) asm volatile("" ::: "memory");
    }
    return t;
  }

  // Values of the buffer's tokens, from j0 on, that are not finite: the rows that see one are
  // NaN from here on (the weights and their sum are not, so that log sums are the scores').
  __device__ __forceinline__ void look(const uint8_t* lds, int j0) {
    const float* r = reinterpret_cast<const float*>(lds + L::kInverses);
    bool bad = false;
#pragma unroll 1
    for (int n = 0; n < L::kTokens; ++n) bad |= (r[n] < 0.0f) & (j0 + n >= lo) & (j0 + n < hi);
#pragma unroll
    for (int d = 0; d < D / 32; ++d) o[d] *= bad ? __uint_as_float(kKvNan) : 1.0f;
  }

  // The tokens j0 .. j0 + 31, the sub-th of the buffer, with their products t; NEXT: then t
  // are the following ones, whose products run beside this softmax.
  template <bool NEXT>
  __device__ __forceinline__ void step(const uint8_t* lds, int sub, int j0, f16& t) {
    const uint8_t* const words = lds + word_at + 32 * sub * 4;
    f16 s;
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const f4 f = *reinterpret_cast<const f4*>(words + 8 * n * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[4 * n + i] = __builtin_fmaf(t[4 * n + i], f[i], off);
        top = fmaxf(top, s[4 * n + i]);
      }
    }
    if (__builtin_amdgcn_ballot_w64(top > limit) != 0 || j0 < all_lo || j0 + 32 > all_hi) {
      const int j = j0 + ((word_at - L::kFactors) >> 2);
      top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float f = *reinterpret_cast<const float*>(words + 8 * (i >> 2) * 4);
        const int at = j + 8 * (i >> 2) + (i & 3);
        const bool seen = (f != INFINITY) & (at >= lo) & (at < hi);
        s[i] = seen ? s[i] : -INFINITY;
        top = fmaxf(top, s[i]);
      }
      top = fmaxf(top, other_half(top));
      const bool up = top > limit;
      const float delta = up ? kReference - top : 0.0f;
      const float keep = limit == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(delta);
      limit = up ? kReference + 8.0f : limit;
      off += delta;
      l *= keep;
      if (__builtin_amdgcn_ballot_w64(up)) {
#pragma unroll
        for (int d = 0; d < D / 32; ++d) o[d] *= keep;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] += delta;
      }
    }
    if (NEXT) t = scores(lds, sub + 1);
    h8 p[2];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const f4 r = *reinterpret_cast<const f4*>(words + (2 * L::kTokens + 8 * n) * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(s[4 * n + i]);
        l = __builtin_fmaf(e, fabsf(r[i]), l);
        p[n >> 1][4 * (n & 1) + i] = (_Float16)e;
      }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int d = 0; d < D / 32; ++d) {
        const h8 v = *reinterpret_cast<const h8*>(lds + value_at + L::value_row(32 * d) +
                                                  (2 * sub + n) * 32);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[n], o[d], 0, 0, 0);
      }
  }
};

// Grid: (row groups * H, B, chunks of the tokens); a workgroup takes 32 NW rows.
template <int D, typename T, int NW>
__global__ __launch_bounds__(64 * NW, 2) void kv_attend_prompt_kernel(KvAttend a, Part part,
                                                                      int groups, int least) {
  using L = Layout<D, NW>;
  __shared__ alignas(16) uint8_t lds[2 * L::kAll];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int b = blockIdx.y, H = a.cache.H;
  // The last rows see the most tokens: longest first.
  const int head = blockIdx.x % H, group = groups - 1 - blockIdx.x / H, chunks = gridDim.z;
  const int G = a.Hq / H;
  const Sequence s = sequence_of(a, b);
  clear_outside(a, s, D, 64 * NW);
  if (s.past && group == 0 && blockIdx.z == 0)
    clear_rows(a, D, s.first + s.n + head, s.first + s.n + s.past, H, 64 * NW);
  const int count = s.n * G, g0 = group * (32 * NW);
  if (g0 >= count) return;

  // The workgroup's tokens, and this chunk's steps among them.
  const int g1 = min(g0 + 32 * NW, count) - 1;
  const int begin = row_begin(a, s, g0 / G), end = row_end(s, g1 / G);
  const int first = begin / L::kTokens, last = (end + L::kTokens - 1) / L::kTokens;
  const int each = max((last - first + chunks - 1) / chunks, least);
  const int from = first + blockIdx.z * each, to = min(from + each, last);
  if (blockIdx.z > 0 && from >= last) return;

  // The wave's rows: tokens that some see, and that all see.
  Wave<D, T, NW> w;
  w.clear(lane);
  const int r0 = g0 + wave * 32, row = r0 + c, i = min(row, count - 1) / G;
  const int i0 = min(r0, count - 1) / G, i1 = (min(r0 + 32, count) - 1) / G;
  const int wave_lo = row_begin(a, s, i0), wave_hi = r0 < count ? row_end(s, i1) : 0;
  w.all_lo = row_begin(a, s, i1);
  w.all_hi = row_end(s, i0);
  w.lo = row_begin(a, s, i);
  w.hi = row_end(s, i);

  const T* qrow = static_cast<const T*>(a.q) + (s.first + i) * a.q_ts +
                  (head * G + min(row, count - 1) - i * G) * a.q_hs;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
    w.q[ks] = Operand<T>::rows(load_raw_at<T>(qrow, 16 * ks + 8 * h));
  const float to2 = a.scale * kLog2e / Operand<T>::kRows;

  const uint8_t* const block = a.cache.data + head * kv_block_bytes<D>(a.cache.P);
  const int64_t page_bytes = H * kv_block_bytes<D>(a.cache.P);
  const Places places = places_of(a, b, end);
  const Masks masks;
  Stage<D, T, NW> stage;
  if (from < to) {
    stage.load_keys(a, block, page_bytes, place_of(places, NW * from + wave), NW * from + wave,
                    lane);
    stage.store_keys(lds, wave, lane, to2, begin, end, masks);
    stage.load_values(a.cache.P, lane);
    stage.store_values(lds, wave, lane, masks);
  }
  Place place = place_of(places, NW * (from + 1) + wave);  // of the next tile, a step ahead
  __syncthreads();
  for (int at = from; at < to; ++at) {
    const int j0 = at * L::kTokens;
    uint8_t* const now = lds + ((at - from) & 1) * L::kAll;
    uint8_t* const next = lds + ((at - from + 1) & 1) * L::kAll;
    const bool more = at + 1 < to, work = j0 < wave_hi && j0 + L::kTokens > wave_lo;
    if (more) stage.load_keys(a, block, page_bytes, place, NW * (at + 1) + wave, lane);
    place = place_of(places, NW * (at + 2) + wave);
    f16 t;
    uint32_t bad = 0;  // of tile lane % NW
    if (work) {
      bad = *reinterpret_cast<const uint32_t*>(now + L::kBad + 4 * (lane & (NW - 1)));
      t = w.scores(now, 0);
#pragma unroll
      for (int sub = 0; sub < L::kSteps / 2; ++sub)
        w.template step<true>(now, sub, j0 + 32 * sub, t);
    }
    if (more) {
      stage.store_keys(next, wave, lane, to2, begin, end, masks);
      stage.load_values(a.cache.P, lane);
    }
    if (work) {
#pragma unroll
      for (int sub = L::kSteps / 2; sub < L::kSteps - 1; ++sub)
        w.template step<true>(now, sub, j0 + 32 * sub, t);
      w.template step<false>(now, L::kSteps - 1, j0 + L::kTokens - 32, t);
      if (__builtin_amdgcn_ballot_w64(bad != 0)) w.look(now, j0);
    }
    if (more) stage.store_values(next, wave, lane, masks);
    __syncthreads();
  }

  const int hq = head * G + row - i * G;
  const float sum = w.l + other_half(w.l);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const float log = sum == 0.0f ? -INFINITY : __builtin_amdgcn_logf(sum) - w.off;
  if (row >= count) return;
  if (last - first > each) {  // the row has parts
    const int64_t to_row = (((int64_t)b * a.max_q + i) * a.Hq + hq) * chunks + blockIdx.z;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        f4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = w.o[d][4 * n + e] * inv;
        *reinterpret_cast<f4*>(part.out + to_row * D + 32 * d + 8 * n + 4 * h) = y;
      }
    if (h == 0) part.log[to_row] = log;
  } else {
    const int64_t to_row = (s.first + i) * a.Hq + hq;
    uint16_t* out = static_cast<uint16_t*>(a.out) + to_row * D;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        u32x2_a2 y;
        y[0] = pack_pair<T>(w.o[d][4 * n] * inv, w.o[d][4 * n + 1] * inv);
        y[1] = pack_pair<T>(w.o[d][4 * n + 2] * inv, w.o[d][4 * n + 3] * inv);
        *reinterpret_cast<u32x2_a2*>(out + 32 * d + 8 * n + 4 * h) = y;
      }
    if (a.lse && h == 0) a.lse[to_row] = log * kLn2;
  }
}

template <int D, typename T>
int prompt_typed(const KvAttend& a, const Part& part, int waves, int chunks, int least,
                 hipStream_t stream) {
  // max_q may be far above what there is, and a grid of 2^32 threads wraps.
  const int64_t rows = std::min<int64_t>(a.max_q, a.T) * (a.Hq / a.cache.H), per = 32 * waves;
  const int groups = (int)((rows + per - 1) / per);
  const dim3 grid((uint32_t)(groups * a.cache.H), a.B, chunks);
  if (waves == 8)
    launch(kv_attend_prompt_kernel<D, T, 8>, grid, dim3(512), stream, a, part, groups, least);
  else
    launch(kv_attend_prompt_kernel<D, T, 4>, grid, dim3(256), stream, a, part, groups, least);
  return launch_status("kv_attention");
}

}  // namespace

// Rows in workgroups of 32 for each of 4 or 8 waves, their tokens in up to `chunks` parts
// of at least `least` steps (16 tokens for each wave); rows of several parts are joined by
// the caller.
int kv_attend_prompt(const KvAttend& a, int D, bool is_bf16, const Part& part, int waves,
                     int chunks, int least, hipStream_t stream) {
  if (D == 128)
    return is_bf16 ? prompt_typed<128, bf16>(a, part, waves, chunks, least, stream)
                   : prompt_typed<128, __half>(a, part, waves, chunks, least, stream);
  return is_bf16 ? prompt_typed<64, bf16>(a, part, waves, chunks, least, stream)
                 : prompt_typed<64, __half>(a, part, waves, chunks, least, stream);
}

}  // namespace dscq
