// Attention over the 4-bit key/value cache (layout: kv4.h).
//
// For query i of a sequence of L cached tokens, the last n of them the queries' own, at
// place p = L - n + i, over the tokens j <= p (and j > p - window):
//   s_j = scale q . k_j,  m = max s_j,  o = sum e^(s_j - m) v_j / sum e^(s_j - m),
//   lse = m + log sum e^(s_j - m);  no visible token: o = 0, lse = -inf.
//
// Rows.  The G = Hq / H query heads of a key/value head read the same tokens, so a row is
// (query, head of the group), r = i G + g, and sixteen rows fill a matrix instruction.
//
// Products.  A key is k = (c - z) f with whole numbers c, z in [0, 15] and the row's scale f:
// q . k = f (q . (c - z)), and c - z is exact in fp16, so keys and values enter the products
// as what they are.  q enters as fp16; a bf16 q is first multiplied by the power of two that
// takes its largest element to [2^14, 2^15) (eight bits of each element, so exact but for
// elements 2^38 times smaller than the row's largest).  Both products are made transposed,
//   S^T = K q^T  (16 tokens x 16 rows),  O^T += V^T P^T  (16 elements x 16 rows),
// because then a lane holds scores of one row only -- lane (c, g) = (lane % 16, lane / 16)
// those of row c and tokens 4 g .. 4 g + 3 of a tile -- so maximum, sum and rescaling are
// a lane's own, and the scores are the next product's operand as they lie: its 32-token
// index may run in any order, and runs 4 g + i, 16 + 4 g + i over the two tiles of a step.
//
// Weights.  p'_j = 2^((s_j - m) log2 e + x) f'_j for the value's scale f', rounded to fp16 (the
// one rounding here that is not fp32's: 2^-11 of a weight, the size of an fp16 output's own),
// and the sum is that of 2^((s_j - m) log2 e + x) in fp32.  The exponent x keeps the largest
// f' 2^x in [2^6, 2^7), and m lags the true maximum by up to 8 binary places, so weights are at
// most 2^15: within fp16, and its small numbers end 2^39 below.  While neither has to move
// (a vote of the wave) a step rescales nothing.

#include <algorithm>

#include "kv4.h"
#include "mma_int4.h"
#include "rowquant.h"

namespace dscq {

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kWaves = 4;
constexpr int kStep = 2 * kKvTile;  // tokens of a step

// A value every lane holds alike, read through the scalar cache.
__device__ __forceinline__ int32_t uniform_load(const int32_t* p) {
  typedef const __attribute__((address_space(4))) int32_t* Ptr;
  return *(Ptr)(reinterpret_cast<uintptr_t>(p));
}

// Sequence b's queries (rows first .. first + n - 1 of q) and length.
struct Sequence {
  int64_t first;
  int n, L;
};
__device__ __forceinline__ Sequence sequence_of(const KvAttend& a, int b) {
  int64_t s0 = b, s1 = b + 1;
  if (a.starts) {
    s0 = max(uniform_load(a.starts + b), 0);
    s1 = uniform_load(a.starts + b + 1);
  }
  s0 = min(s0, a.T);
  s1 = min(max(s1, s0), a.T);
  const int64_t L = min((int64_t)max(uniform_load(a.lengths + b), 0), a.width * a.cache.P);
  return {s0, (int)min(s1 - s0, (int64_t)a.max_q), (int)L};
}

// One past the last token that query i sees, and the first.
__device__ __forceinline__ int row_end(const Sequence& s, int i) { return max(s.L - s.n + i + 1, 0); }
__device__ __forceinline__ int row_begin(const KvAttend& a, const Sequence& s, int i) {
  const int64_t b = (int64_t)(s.L - s.n + i + 1) - a.window;
  return a.window && b > 0 ? (int)b : 0;
}

template <int D>
struct Words {  // a lane's D/8 bytes of a tile
  uint32_t w[D / 32];
};
template <int D>
__device__ __forceinline__ Words<D> load_words(const uint8_t* p) {
  Words<D> r;
  if constexpr (D == 128) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    r.w[0] = x.x; r.w[1] = x.y; r.w[2] = x.z; r.w[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    r.w[0] = x.x; r.w[1] = x.y;
  }
  return r;
}

// What a lane reads of a 16-token tile.
template <int D>
struct Tile {
  Words<D> k, v;
  uint32_t kz;   // the word of key lane % 16, whose zero-point its operand needs
  uint4 kf, vf;  // the words of tokens 4 g .. 4 g + 3
  bool there;    // uniform: the tile's page is one of the cache
};

template <int D>
struct Pages {
  const uint8_t* head;  // the head's block of page 0
  const int32_t* table;
  int64_t page_bytes, pages;
  int P, per, end;      // tokens and tiles of a page; one past the last token
  uint32_t inverse;     // ceil(2^32 / per)
};

template <int D>
__device__ __forceinline__ int page_index(const Pages<D>& g, int tile) {
  return g.per == 1 ? tile : (int)__umulhi((uint32_t)tile, g.inverse);
}
// The table's entry for a tile, -1 past the end.
template <int D>
__device__ __forceinline__ int page_of(const Pages<D>& g, int tile) {
  return tile * kKvTile < g.end ? uniform_load(g.table + page_index(g, tile)) : -1;
}

template <int D>
__device__ __forceinline__ Tile<D> load_tile(const Pages<D>& g, int tile, int page, int lane) {
  Tile<D> t;
  t.there = page >= 0 && page < g.pages;
  const int at = t.there ? (tile - page_index(g, tile) * g.per) * kKvTile : 0;
  const uint8_t* block = g.head + (int64_t)(t.there ? page : 0) * g.page_bytes;
  t.k = load_words<D>(block + at * (D / 2) + lane * (D / 8));
  t.v = load_words<D>(block + (g.P + at) * (D / 2) + lane * (D / 8));
  const uint8_t* words = block + g.P * D + at * 4;
  t.kz = *reinterpret_cast<const uint32_t*>(words + (lane & 15) * 4);
  t.kf = *reinterpret_cast<const uint4*>(words + (lane >> 4) * 16);
  t.vf = *reinterpret_cast<const uint4*>(words + g.P * 4 + (lane >> 4) * 16);
  return t;
}

// Two nibbles 16 bits apart as fp16 numbers less their zero-points.  0x6400 | c is the
// fp16 number 1024 + c; with the nibble four bits up, 1024 + 16 c, a sixteenth of which is
// 64 + c.  Both subtractions are exact.
struct ZeroPair {
  h2 low, high;  // -(1024 + z), -(64 + z)
};
__device__ __forceinline__ ZeroPair zero_pair(uint32_t word0, uint32_t word1) {
  // Bytes 0 of the two words, 16 bits apart (the bytes between are masked off).
  const uint32_t z = __builtin_amdgcn_perm(word1, word0, 0x0C040C00u);
  ZeroPair r;
  r.low = __builtin_bit_cast(h2, (z & 0x000F000Fu) | 0xE400E400u);
  r.high = __builtin_bit_cast(h2, ((z << 4) & 0x00F000F0u) | 0xD400D400u);
  return r;
}
__device__ __forceinline__ void unpack_word(uint32_t w, const ZeroPair& z, h2 out[4]) {
  const h2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = w >> (8 * i);
    out[2 * i] = __builtin_bit_cast(h2, (x & 0x000F000Fu) | 0x64006400u) + z.low;
    out[2 * i + 1] = __builtin_elementwise_fma(
        __builtin_bit_cast(h2, (x & 0x00F000F0u) | 0x64006400u), sixteenth, z.high);
  }
}
__device__ __forceinline__ h8 join8(h2 a, h2 b, h2 c, h2 d) {
  return (h8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float xor16(float v) { return __shfl_xor(v, 16); }
__device__ __forceinline__ float xor32(float v) { return __shfl_xor(v, 32); }
// Over the four lanes that hold a row.
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, xor16(v));
  return fmaxf(v, xor32(v));
}
__device__ __forceinline__ float row_sum(float v) {
  v += xor16(v);
  return v + xor32(v);
}

// A lane's quarter of one row of q: elements g D/4 .. + D/4 - 1, as fp16 times 2^k; k.
template <int D, typename T>
__device__ __forceinline__ int load_q(const T* row, bool in, int g, h8 q[D / 32]) {
  float x[D / 32][8];
  float top = 0.0f;
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    to_f32(load_raw_at<T>(row, (uint32_t)(in ? g * (D / 4) + 8 * w : 0)), x[w]);
    mask_f32<T>(in, x[w]);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[w][e]));
  }
  int k = 0;
  if constexpr (std::is_same<T, bf16>::value) {
    top = row_max(top);
    if (top > 0.0f && top < INFINITY) k = 15 - __builtin_amdgcn_frexp_expf(top);
  }
#pragma unroll
  for (int w = 0; w < D / 32; ++w)
#pragma unroll
    for (int e = 0; e < 8; ++e) q[w][e] = (_Float16)__builtin_amdgcn_ldexpf(x[w][e], k);
  return k;
}

// The running state of RT tiles of sixteen rows in one wave; lane (c, g) holds row c's
// statistics (l: of its own tokens) and its elements g D/4 .. + D/4 - 1 of the output.
template <int D, int RT>
struct Rows {
  h8 q[RT][D / 32];
  f4 o[RT][D / 16];  // o[r][t][i]: element (4 g + i) D/16 + t
  float to2[RT];     // scores to binary places: scale log2 e 2^-k
  float m[RT], off[RT], limit[RT], l[RT];  // maximum; x - m to2; what moves the maximum
  int begin[RT], end[RT];                  // the row's tokens
  float x, value_limit;                    // the values' exponent, the scale that moves it

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
      for (int t = 0; t < D / 16; ++t) o[r][t] = (f4){0, 0, 0, 0};
      m[r] = limit[r] = -INFINITY;
      off[r] = l[r] = 0.0f;
    }
    x = value_limit = 0.0f;
  }

  // The 32 tokens from j0 in tiles a and b; `whole`: every row sees them all.
  __device__ __forceinline__ void step(const Tile<D>& a, const Tile<D>& b, int j0, int lane,
                                       bool whole) {
    const int g4 = (lane >> 4) * 4;
    h8 kk[2][D / 32];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Tile<D>& t = h ? b : a;
      const ZeroPair z = zero_pair(t.kz, t.kz);
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        h2 e[4];
        unpack_word(t.k.w[w], z, e);
        kk[h][w] = join8(e[0], e[1], e[2], e[3]);
      }
    }
    float vf[8] = {__uint_as_float(a.vf.x), __uint_as_float(a.vf.y), __uint_as_float(a.vf.z),
                   __uint_as_float(a.vf.w), __uint_as_float(b.vf.x), __uint_as_float(b.vf.y),
                   __uint_as_float(b.vf.z), __uint_as_float(b.vf.w)};
    const float kf[8] = {__uint_as_float(a.kf.x), __uint_as_float(a.kf.y), __uint_as_float(a.kf.z),
                         __uint_as_float(a.kf.w), __uint_as_float(b.kf.x), __uint_as_float(b.kf.y),
                         __uint_as_float(b.kf.z), __uint_as_float(b.kf.w)};
    float s[RT][8];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      f4 c0 = {0, 0, 0, 0}, c1 = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        c0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk[0][w], q[r][w], c0, 0, 0, 0);
        c1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk[1][w], q[r][w], c1, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[r][i] = c0[i] * kf[i];
        s[r][4 + i] = c1[i] * kf[4 + i];
      }
    }
    if (!whole) {
      // Tokens a row does not see, and pages that are not there: score -inf, and a scale
      // of 0, for what lies there may be anything.
      bool none[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) none[i] = true;
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = j0 + (i < 4 ? g4 + i : 12 + g4 + i);
          const bool seen = (i < 4 ? a.there : b.there) && j >= begin[r] && j < end[r];
          s[r][i] = seen ? s[r][i] : -INFINITY;
          none[i] = none[i] && !seen;
        }
#pragma unroll
      for (int i = 0; i < 8; ++i) vf[i] = none[i] ? 0.0f : vf[i];
    }
    float top[RT];
    bool move = false;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      top[r] = fmaxf(fmaxf(fmaxf(s[r][0], s[r][1]), fmaxf(s[r][2], s[r][3])),
                     fmaxf(fmaxf(s[r][4], s[r][5]), fmaxf(s[r][6], s[r][7])));
      move = move || top[r] > limit[r];
    }
    float most = fmaxf(fmaxf(fmaxf(vf[0], vf[1]), fmaxf(vf[2], vf[3])),
                       fmaxf(fmaxf(vf[4], vf[5]), fmaxf(vf[6], vf[7])));
    move = move || most > value_limit;
    if (__builtin_amdgcn_ballot_w64(move)) {
      float shift = 0.0f;
      // Masked rows can differ in what they see, so the largest scale is the wave's.
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
      if (most > value_limit) {
        const float to = (float)(7 - __builtin_amdgcn_frexp_expf(most));
        shift = to - x;
        x = to;
        value_limit = __builtin_amdgcn_ldexpf(1.0f, 7 - (int)to);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float was = m[r] * to2[r];
        m[r] = fmaxf(m[r], row_max(top[r]));
        const float base = m[r] == -INFINITY ? 0.0f : m[r] * to2[r];
        off[r] = x - base;
        limit[r] = m[r] + 8.0f / to2[r];
        const float keep = m[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(was - base + shift);
        l[r] *= keep;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) o[r][t] *= keep;
      }
    }
    h8 p[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][i], to2[r], off[r]));
        l[r] += e[i];
        e[i] *= vf[i];
      }
      if (!whole) {
        // A token that this row does not see may be NaN to another row of the lane.
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = s[r][i] == -INFINITY ? 0.0f : e[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) p[r][i] = (_Float16)e[i];
    }
    const ZeroPair z[4] = {zero_pair(a.vf.x, a.vf.y), zero_pair(a.vf.z, a.vf.w),
                           zero_pair(b.vf.x, b.vf.y), zero_pair(b.vf.z, b.vf.w)};
#pragma unroll
    for (int w = 0; w < D / 64; ++w) {
      h2 e[4][4];
      unpack_word(a.v.w[w], z[0], e[0]);
      unpack_word(a.v.w[D / 64 + w], z[1], e[1]);
      unpack_word(b.v.w[w], z[2], e[2]);
      unpack_word(b.v.w[D / 64 + w], z[3], e[3]);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const h8 v = join8(e[0][t], e[1][t], e[2][t], e[3][t]);
#pragma unroll
        for (int r = 0; r < RT; ++r)
          o[r][4 * w + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[r], o[r][4 * w + t], 0, 0, 0);
      }
    }
  }

  // The steps first, first + stride, ... below `last` (tokens / 32).
  __device__ __forceinline__ void run(const Pages<D>& g, int first, int last, int stride, int lane) {
    if (first >= last) return;
    int lo = 0, hi = 0x7FFFFFFF;  // every row sees the tokens lo .. hi - 1
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      lo = max(lo, begin[r]);
      hi = min(hi, end[r]);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      lo = max(lo, __shfl_xor(lo, d));
      hi = min(hi, __shfl_xor(hi, d));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    Tile<D> a = load_tile<D>(g, 2 * first, page_of(g, 2 * first), lane);
    Tile<D> b = load_tile<D>(g, 2 * first + 1, page_of(g, 2 * first + 1), lane);
    int pa = page_of(g, 2 * (first + stride)), pb = page_of(g, 2 * (first + stride) + 1);
    for (int st = first; st < last; st += stride) {
      const int next = st + stride;
      const Tile<D> na = load_tile<D>(g, 2 * next, pa, lane);
      const Tile<D> nb = load_tile<D>(g, 2 * next + 1, pb, lane);
      pa = page_of(g, 2 * (next + stride));
      pb = page_of(g, 2 * (next + stride) + 1);
      step(a, b, st * kStep, lane,
           st * kStep >= lo && st * kStep + kStep <= hi && a.there && b.there);
      a = na;
      b = nb;
    }
  }
};

// The launch's plan; `chunks` > 1: the tokens are split over that many workgroups and the
// parts joined by a second kernel.
struct Plan {
  int rt, chunks;
  bool rows;  // the waves of a workgroup take different rows, not different tokens
};

struct Part {  // a row's result over some of its tokens
  float* out;  // [rows][chunks][D], rows = (b max_q + i) Hq + head
  float* log;  // [rows][chunks]: log2 of the softmax sum
};

template <int D>
__device__ __forceinline__ Pages<D> pages_of(const KvAttend& a, int b, int h, int end) {
  Pages<D> g;
  g.P = a.cache.P;
  g.per = g.P / kKvTile;
  g.inverse = (uint32_t)((0x100000000ull + g.per - 1) / g.per);
  g.page_bytes = a.cache.H * kv_block_bytes<D>(g.P);
  g.head = a.cache.data + h * kv_block_bytes<D>(g.P);
  g.pages = a.cache.pages;
  g.table = a.tables + b * a.width;
  g.end = end;
  return g;
}

template <int D, typename T, int RT>
__device__ __forceinline__ void begin_rows(Rows<D, RT>& rows, const KvAttend& a, const Sequence& s,
                                           int h, int G, int r0, int lane) {
  rows.clear();
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = r0 + 16 * r + (lane & 15), i = row / G;
    const bool in = i < s.n;
    const T* p = static_cast<const T*>(a.q) + (s.first + (in ? i : 0)) * a.q_ts +
                 (h * G + (in ? row - i * G : 0)) * a.q_hs;
    const int k = load_q<D, T>(p, in, lane >> 4, rows.q[r]);
    rows.to2[r] = __builtin_amdgcn_ldexpf(a.scale * kLog2e, -k);
    // A row past the last one sees what the last one does.
    rows.begin[r] = row_begin(a, s, min(i, s.n - 1));
    rows.end[r] = row_end(s, min(i, s.n - 1));
  }
}

// log2 of a row's softmax sum.
template <int D, int RT>
__device__ __forceinline__ float log_sum(const Rows<D, RT>& rows, int r, float l) {
  return rows.m[r] == -INFINITY && l == 0.0f
             ? -INFINITY
             : __builtin_amdgcn_logf(l) + rows.m[r] * rows.to2[r] - rows.x;
}

// Grid: (chunks, H * row tiles, B); the four waves of a workgroup take every fourth step of
// its tokens and join their results through LDS.
template <int D, typename T, int RT>
__global__ __launch_bounds__(64 * kWaves) void kv_attend_split_kernel(KvAttend a, Part part,
                                                                      int row_tiles) {
  constexpr int kRow = D + 4;
  __shared__ float out[kWaves][16][kRow];
  __shared__ float logs[kWaves][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.z, h = blockIdx.y / row_tiles, tile = blockIdx.y - h * row_tiles;
  const int G = a.Hq / a.cache.H, r0 = tile * 16 * RT, chunks = gridDim.x;
  const Sequence s = sequence_of(a, b);
  const int count = s.n * G;
  if (r0 >= count) return;
  const int i0 = r0 / G, i1 = min(r0 + 16 * RT, count) - 1;
  const int first = row_begin(a, s, i0) / kStep;
  const int last = (row_end(s, i1 / G) + kStep - 1) / kStep;
  const int each = max((last - first + chunks - 1) / chunks, 1);
  const int from = first + blockIdx.x * each, to = min(from + each, last);
  if (blockIdx.x > 0 && from >= last) return;
  Rows<D, RT> rows;
  begin_rows<D, T, RT>(rows, a, s, h, G, r0, lane);
  const Pages<D> pages = pages_of<D>(a, b, h, row_end(s, i1 / G));
  rows.run(pages, from + wave, to, kWaves, lane);
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    if (r) __syncthreads();
    const float l = row_sum(rows.l[r]);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < D / 16; ++t)
        out[wave][c][(4 * g + i) * (D / 16) + t] = rows.o[r][t][i] * inv;
    if (g == 0) logs[wave][c] = log_sum(rows, r, l);
    __syncthreads();
    const int row = threadIdx.x >> 4, d = (threadIdx.x & 15) * (D / 16);
    const int R = r0 + 16 * r + row;
    if (R < count) {
      float top = logs[0][row];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = fmaxf(top, logs[w][row]);
      const float base = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, y[D / 16] = {};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float p = __builtin_amdgcn_exp2f(logs[w][row] - base);
        sum += p;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) y[e] = __builtin_fmaf(p, out[w][row][d + e], y[e]);
      }
      const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
      const float log = sum == 0.0f ? -INFINITY : base + __builtin_amdgcn_logf(sum);
      const int i = R / G, hq = h * G + R - i * G;
      if (chunks > 1) {
        const int64_t at = (((int64_t)b * a.max_q + i) * a.Hq + hq) * chunks + blockIdx.x;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) part.out[at * D + d + e] = y[e] * scale;
        if (d == 0) part.log[at] = log;
      } else {
        const int64_t at = (s.first + i) * a.Hq + hq;
        uint16_t* o = static_cast<uint16_t*>(a.out) + at * D + d;
#pragma unroll
        for (int e = 0; e < D / 16; ++e)
          o[e] = __builtin_bit_cast(uint16_t, to_out<T>(y[e] * scale));
        if (a.lse && d == 0) a.lse[at] = log * kLn2;
      }
    }
  }
}

// Grid: (max_q Hq, B), a wave a row: its parts weighted by their sums.
template <int D, typename T>
__global__ __launch_bounds__(64) void kv_attend_join_kernel(KvAttend a, Part part, int chunks,
                                                            int rt) {
  const int lane = threadIdx.x, b = blockIdx.y, i = blockIdx.x / a.Hq, hq = blockIdx.x - i * a.Hq;
  const Sequence s = sequence_of(a, b);
  if (i >= s.n) return;
  // How many parts the row's workgroup made: as kv_attend_split_kernel.
  const int G = a.Hq / a.cache.H, count = s.n * G;
  const int r0 = (i * G + hq % G) / (16 * rt) * (16 * rt);
  const int first = row_begin(a, s, r0 / G) / kStep;
  const int last = (row_end(s, (min(r0 + 16 * rt, count) - 1) / G) + kStep - 1) / kStep;
  const int each = max((last - first + chunks - 1) / chunks, 1);
  const int used = max((last - first + each - 1) / each, 1);
  const int64_t at = (((int64_t)b * a.max_q + i) * a.Hq + hq) * chunks;
  float top = -INFINITY;
  for (int c = lane; c < used; c += 64) top = fmaxf(top, part.log[at + c]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, y[D / 64] = {};
  for (int c = 0; c < used; ++c) {
    const float p = __builtin_amdgcn_exp2f(part.log[at + c] - base);
    sum += p;
#pragma unroll
    for (int e = 0; e < D / 64; ++e)
      y[e] = __builtin_fmaf(p, part.out[(at + c) * D + lane * (D / 64) + e], y[e]);
  }
  const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
  const int64_t to = (s.first + i) * a.Hq + hq;
  uint16_t* o = static_cast<uint16_t*>(a.out) + to * D + lane * (D / 64);
#pragma unroll
  for (int e = 0; e < D / 64; ++e) o[e] = __builtin_bit_cast(uint16_t, to_out<T>(y[e] * scale));
  if (a.lse && lane == 0)
    a.lse[to] = sum == 0.0f ? -INFINITY : (base + __builtin_amdgcn_logf(sum)) * kLn2;
}

// Grid: (H * row tiles / 4, B): a wave takes 64 rows over all their tokens.
template <int D, typename T, int RT>
__global__ __launch_bounds__(64 * kWaves) void kv_attend_rows_kernel(KvAttend a, int row_tiles) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y, groups = (row_tiles + kWaves - 1) / kWaves;
  const int h = blockIdx.x % a.cache.H;
  const int tile = (groups - 1 - blockIdx.x / a.cache.H) * kWaves + wave;
  const int G = a.Hq / a.cache.H, r0 = tile * 16 * RT;
  const Sequence s = sequence_of(a, b);
  const int count = s.n * G;
  if (r0 >= count) return;
  const int i0 = r0 / G, i1 = (min(r0 + 16 * RT, count) - 1) / G;
  Rows<D, RT> rows;
  begin_rows<D, T, RT>(rows, a, s, h, G, r0, lane);
  const int end = row_end(s, i1);
  const Pages<D> pages = pages_of<D>(a, b, h, end);
  rows.run(pages, row_begin(a, s, i0) / kStep, (end + kStep - 1) / kStep, 1, lane);
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = r0 + 16 * r + c, i = row / G;
    const float l = row_sum(rows.l[r]);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (row < count) {
      const int64_t at = (s.first + i) * a.Hq + h * G + row - i * G;
      uint16_t* o = static_cast<uint16_t*>(a.out) + at * D + g * (D / 4);
#pragma unroll
      for (int e = 0; e < D / 4; e += 8) {
        u32x4_a2 w;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int d = e + 2 * x;
          w[x] = pack_pair<T>(rows.o[r][d % (D / 16)][d / (D / 16)] * inv,
                              rows.o[r][(d + 1) % (D / 16)][d / (D / 16)] * inv);
        }
        *reinterpret_cast<u32x4_a2*>(o + e) = w;
      }
      if (a.lse && g == 0) a.lse[at] = log_sum(rows, r, l) * kLn2;
    }
  }
}

Plan plan_of(int B, int Hq, int H, int max_q, int64_t max_length, int64_t window) {
  const int64_t rows = (int64_t)max_q * (Hq / H);
  Plan p = {4, 1, rows > 64};
  if (p.rows) return p;
  p.rt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  int64_t length = window ? std::min(max_length, window + max_q - 1) : max_length;
  const int64_t most = (length + kWaves * kStep - 1) / (kWaves * kStep);
  const int64_t want = (3 * (int64_t)cu_count() + B * H - 1) / (B * H);
  p.chunks = (int)std::max<int64_t>(1, std::min(most, want));
  return p;
}

template <int D, typename T, int RT>
int attend_split(const KvAttend& a, const Plan& p, void* ws, hipStream_t stream) {
  const int rows = a.max_q * (a.Hq / a.cache.H), tiles = (rows + 16 * RT - 1) / (16 * RT);
  Part part = {nullptr, nullptr};
  if (p.chunks > 1) {
    part.out = static_cast<float*>(ws);
    part.log = part.out + (int64_t)a.B * a.max_q * a.Hq * p.chunks * D;
  }
  const KernelEvents ev = take_kernel_events();
  arm_kernel_events({ev.start, p.chunks > 1 ? nullptr : ev.stop});
  launch(kv_attend_split_kernel<D, T, RT>, dim3(p.chunks, a.cache.H * tiles, a.B),
         dim3(64 * kWaves), stream, a, part, tiles);
  if (p.chunks > 1) {
    arm_kernel_events({nullptr, ev.stop});
    launch(kv_attend_join_kernel<D, T>, dim3(a.max_q * a.Hq, a.B), dim3(64), stream, a, part,
           p.chunks, RT);
  }
  return launch_status("kv_attention");
}

template <int D, typename T>
int attend(const KvAttend& a, void* ws, hipStream_t stream) {
  const Plan p = plan_of(a.B, a.Hq, a.cache.H, a.max_q, a.max_length, a.window);
  if (p.rows) {
    const int64_t rows = (int64_t)a.max_q * (a.Hq / a.cache.H), tiles = (rows + 63) / 64;
    launch(kv_attend_rows_kernel<D, T, 4>,
           dim3((uint32_t)((tiles + kWaves - 1) / kWaves * a.cache.H), a.B), dim3(64 * kWaves),
           stream, a, (int)tiles);
    return launch_status("kv_attention");
  }
  if (p.rt == 1) return attend_split<D, T, 1>(a, p, ws, stream);
  if (p.rt == 2) return attend_split<D, T, 2>(a, p, ws, stream);
  return attend_split<D, T, 4>(a, p, ws, stream);
}

}  // namespace

int64_t kv_attention_workspace_bytes(int D, int B, int Hq, int H, int max_q, int64_t max_length,
                                     int64_t window) {
  const Plan p = plan_of(B, Hq, H, max_q, max_length, window);
  return p.chunks > 1 ? (int64_t)B * max_q * Hq * p.chunks * (D + 1) * 4 : 0;
}

int kv_attention(const KvAttend& a, int D, bool is_bf16, void* ws, hipStream_t stream) {
  if (D == 128)
    return is_bf16 ? attend<128, bf16>(a, ws, stream) : attend<128, __half>(a, ws, stream);
  return is_bf16 ? attend<64, bf16>(a, ws, stream) : attend<64, __half>(a, ws, stream);
}

}  // namespace dscq
