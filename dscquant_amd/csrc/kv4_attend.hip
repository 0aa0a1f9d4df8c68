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

#include "kv4_attend.h"

namespace dscq {

int kv_attend_prompt(const KvAttend& a, int D, bool is_bf16, const Part& part, int waves,
                     int chunks, int least, hipStream_t stream);

namespace {

constexpr int kWaves = 4;
constexpr int kStep = 2 * kKvTile;  // tokens of a step

// What a lane reads of a 16-token tile.
template <int D>
struct Tile {
  Words<D> k, v;
  uint32_t kz;   // the word of key lane % 16, whose zero-point its operand needs
  uint4 kf, vf;  // the words of tokens 4 g .. 4 g + 3
  bool there;    // uniform: the tile's page is one of the cache
};

// A tile's address is a uniform one (its page's block and place) and a lane's offset that
// never changes, the two addends of a global load.
template <int D>
struct Pages {
  Places places;
  const uint8_t* head;  // the head's block of page 0
  int64_t page_bytes, pages;
  uint32_t k_at, v_at, kz_at, kf_at, vf_at;  // the lane's
};

template <int D>
__device__ __forceinline__ Tile<D> load_tile(const Pages<D>& g, Place p) {
  Tile<D> t;
  t.there = p.page >= 0 && p.page < g.pages;
  const uint8_t* block = g.head + (t.there ? p.page * g.page_bytes : 0);
  const uint8_t* codes = block + p.at * (8 * D);
  const uint8_t* words = block + p.at * (4 * kKvTile);
  t.k = load_words<D>(codes + g.k_at);
  t.v = load_words<D>(codes + g.v_at);
  t.kz = *reinterpret_cast<const uint32_t*>(words + g.kz_at);
  t.kf = *reinterpret_cast<const uint4*>(words + g.kf_at);
  t.vf = *reinterpret_cast<const uint4*>(words + g.vf_at);
  return t;
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
    const Masks masks;
    h8 kk[2][D / 32];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Tile<D>& t = h ? b : a;
      const ZeroPair z = zero_pair(t.kz, t.kz, masks);
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        h2 e[4];
        unpack_word(t.k.w[w], z, masks, e);
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
    const ZeroPair z[4] = {zero_pair(a.vf.x, a.vf.y, masks), zero_pair(a.vf.z, a.vf.w, masks),
                           zero_pair(b.vf.x, b.vf.y, masks), zero_pair(b.vf.z, b.vf.w, masks)};
#pragma unroll
    for (int w = 0; w < D / 64; ++w) {
      h2 e[4][4];
      unpack_word(a.v.w[w], z[0], masks, e[0]);
      unpack_word(a.v.w[D / 64 + w], z[1], masks, e[1]);
      unpack_word(b.v.w[w], z[2], masks, e[2]);
      unpack_word(b.v.w[D / 64 + w], z[3], masks, e[3]);
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
    Tile<D> a = load_tile<D>(g, place_of(g.places, 2 * first));
    Tile<D> b = load_tile<D>(g, place_of(g.places, 2 * first + 1));
    Place pa = place_of(g.places, 2 * (first + stride)), pb = place_of(g.places, 2 * (first + stride) + 1);
    for (int st = first; st < last; st += stride) {
      const int next = st + stride;
      const Tile<D> na = load_tile<D>(g, pa);
      const Tile<D> nb = load_tile<D>(g, pb);
      pa = place_of(g.places, 2 * (next + stride));
      pb = place_of(g.places, 2 * (next + stride) + 1);
      step(a, b, st * kStep, lane,
           st * kStep >= lo && st * kStep + kStep <= hi && a.there && b.there);
      a = na;
      b = nb;
    }
  }
};

// The launch's plan.  Rows go in groups of `rows`, their tokens in up to `chunks` parts of
// whole steps of `step` tokens, at least `least` of them each; groups of more than one part
// are joined by a second kernel (launched where chunks > 1).
struct Plan {
  int rows, step, chunks, least;
  bool prompt;  // kv4_prompt.hip
};

// The steps of a group's tokens and of each part, and how many parts it has.
struct Parts {
  int first, last, each, used;
};
__device__ __forceinline__ Parts parts_of(const KvAttend& a, const Sequence& s, const Plan& p, int G,
                                          int r0) {
  const int r1 = min(r0 + p.rows, s.n * G) - 1;
  Parts x;
  x.first = row_begin(a, s, r0 / G) / p.step;
  x.last = (row_end(s, r1 / G) + p.step - 1) / p.step;
  x.each = max((x.last - x.first + p.chunks - 1) / p.chunks, p.least);
  x.used = max((x.last - x.first + x.each - 1) / x.each, 1);
  return x;
}

template <int D>
__device__ __forceinline__ Pages<D> pages_of(const KvAttend& a, int b, int h, int end, int lane) {
  Pages<D> g;
  const int P = a.cache.P;
  g.places = places_of(a, b, end);
  g.page_bytes = a.cache.H * kv_block_bytes<D>(P);
  g.head = a.cache.data + h * kv_block_bytes<D>(P);
  g.pages = a.cache.pages;
  g.k_at = lane * (D / 8);
  g.v_at = P * (D / 2) + lane * (D / 8);
  g.kz_at = P * D + (lane & 15) * 4;
  g.kf_at = P * D + (lane >> 4) * 16;
  g.vf_at = P * (D + 4) + (lane >> 4) * 16;
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

// Grid: (chunks, H, B), up to 16 RT rows; the four waves of a workgroup take every fourth
// step of its tokens and join their results through LDS.
template <int D, typename T, int RT>
__global__ __launch_bounds__(64 * kWaves, RT == 1 ? 3 : 1) void kv_attend_split_kernel(
    KvAttend a, Part part, Plan plan) {
  constexpr int kRow = D + 4;
  __shared__ float out[kWaves][16][kRow];
  __shared__ float logs[kWaves][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.z, h = blockIdx.y;
  const int G = a.Hq / a.cache.H;
  const Sequence s = sequence_of(a, b);
  const int count = s.n * G;
  if (count == 0) return;
  const Parts parts = parts_of(a, s, plan, G, 0);
  if ((int)blockIdx.x >= parts.used) return;
  const int from = parts.first + blockIdx.x * parts.each;
  const int to = min(from + parts.each, parts.last);
  Rows<D, RT> rows;
  begin_rows<D, T, RT>(rows, a, s, h, G, 0, lane);
  const Pages<D> pages = pages_of<D>(a, b, h, row_end(s, s.n - 1), lane);
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
    const int R = 16 * r + row;
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
      if (parts.used > 1) {
        const int64_t at = (((int64_t)b * a.max_q + i) * a.Hq + hq) * plan.chunks + blockIdx.x;
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

// Grid: (max_q Hq, B): a row's parts weighted by their sums.  The four waves of a workgroup
// take every fourth part, eight at a time so that their loads are in flight together.
template <int D, typename T>
__global__ __launch_bounds__(64 * kWaves) void kv_attend_join_kernel(
    KvAttend a, Part part, Plan plan, int per) {
  __shared__ float out[kWaves][D], sums[kWaves];
  const int lane = threadIdx.x & 63;
  // This wave's share of its row: every `per`-th part.
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y;
  const int row = blockIdx.x * (kWaves / per) + wave / per, i = row / a.Hq, hq = row - i * a.Hq;
  wave %= per;
  const Sequence s = sequence_of(a, b);
  const int G = a.Hq / a.cache.H, chunks = plan.chunks;
  int used = 0;
  if (i < s.n) used = parts_of(a, s, plan, G, (i * G + hq % G) / plan.rows * plan.rows).used;
  const bool in = used > 1;  // a row of one part is done
  if (per == kWaves && !in) return;
  const int64_t at = (((int64_t)b * a.max_q + i) * a.Hq + hq) * chunks;
  float top = -INFINITY;
  for (int c = lane; c < used; c += 64) top = fmaxf(top, part.log[at + c]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float base = top == -INFINITY ? 0.0f : top;
  constexpr int kE = D / 64, kMany = 8;
  float sum = 0.0f, y[kE] = {};
  for (int c = wave; in && c < used; c += kMany * per) {
    float log[kMany], x[kMany][kE];
#pragma unroll
    for (int m = 0; m < kMany; ++m) {
      const int64_t from = at + min(c + m * per, used - 1);
      log[m] = part.log[from];
#pragma unroll
      for (int e = 0; e < kE; ++e) x[m][e] = part.out[from * D + lane * kE + e];
    }
#pragma unroll
    for (int m = 0; m < kMany; ++m) {
      const float p = c + m * per < used ? __builtin_amdgcn_exp2f(log[m] - base) : 0.0f;
      sum += p;
#pragma unroll
      for (int e = 0; e < kE; ++e) y[e] = p == 0.0f ? y[e] : __builtin_fmaf(p, x[m][e], y[e]);
    }
  }
  if (per > 1) {
    const int w = threadIdx.x >> 6;
#pragma unroll
    for (int e = 0; e < kE; ++e) out[w][lane * kE + e] = y[e];
    if (lane == 0) sums[w] = sum;
    __syncthreads();
    if (wave) return;
    for (int o = 1; o < per; ++o) {
      sum += sums[w + o];
#pragma unroll
      for (int e = 0; e < kE; ++e) y[e] += out[w + o][lane * kE + e];
    }
  }
  if (!in) return;
  const int64_t to = (s.first + i) * a.Hq + hq;
  uint16_t* o = static_cast<uint16_t*>(a.out) + to * D + lane * kE;
#pragma unroll
  for (int e = 0; e < kE; ++e)
    o[e] = __builtin_bit_cast(uint16_t, to_out<T>(sum == 0.0f ? 0.0f : y[e] / sum));
  if (a.lse && lane == 0)
    a.lse[to] = sum == 0.0f ? -INFINITY : (base + __builtin_amdgcn_logf(sum)) * kLn2;
}

Plan plan_of(int B, int Hq, int H, int max_q, int64_t max_length, int64_t window) {
  const int64_t rows = (int64_t)max_q * (Hq / H), cus = cu_count();
  const int64_t length =
      std::min<int64_t>(window ? std::min(max_length, window + max_q - 1) : max_length, kKvMaxLength);
  Plan p = {};
  int64_t groups = 1, slots;
  if (rows > 64) {
    // 256 rows a workgroup, one of which a CU holds, or 128 (two).
    p.prompt = true;
    p.rows = rows > 128 ? 256 : 128;
    p.step = p.rows / 2;
    p.least = 2;
    groups = (rows + p.rows - 1) / p.rows;
    slots = cus * (256 / p.rows);
  } else {
    // As many workgroups as the device holds at once: each has the same tokens to read, so
    // a second round would only add its start and end (131072 tokens of 8 heads: 36 us in
    // one round, 41 in two, 49 in four).
    p.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    p.step = kStep;
    p.least = kWaves;
    slots = cus * (p.rows == 16 ? 3 : 1);
  }
  const int64_t steps = (length + p.step - 1) / p.step + 1, wgs = groups * B * H;
  const int64_t want = p.prompt ? slots / wgs : (slots + wgs - 1) / wgs;
  p.chunks = (int)std::max<int64_t>(1, std::min((steps + p.least - 1) / p.least, want));
  p.least = (int)std::max<int64_t>(p.least, (steps + p.chunks - 1) / p.chunks);
  return p;
}

template <int D, typename T>
int attend(const KvAttend& a, void* ws, hipStream_t stream) {
  const Plan p = plan_of(a.B, a.Hq, a.cache.H, a.max_q, a.max_length, a.window);
  Part part = {nullptr, nullptr};
  if (p.chunks > 1) {
    part.out = static_cast<float*>(ws);
    part.log = part.out + (int64_t)a.B * a.max_q * a.Hq * p.chunks * D;
  }
  // Timing events, if armed, span both kernels.
  const KernelEvents ev = take_kernel_events();
  arm_kernel_events({ev.start, p.chunks > 1 ? nullptr : ev.stop});
  const dim3 grid(p.chunks, a.cache.H, a.B), block(64 * kWaves);
  int rc = 0;
  if (p.prompt)
    rc = kv_attend_prompt(a, D, std::is_same<T, bf16>::value, part, p.rows / 32, p.chunks, p.least,
                          stream);
  else if (p.rows == 16)
    launch(kv_attend_split_kernel<D, T, 1>, grid, block, stream, a, part, p);
  else if (p.rows == 32)
    launch(kv_attend_split_kernel<D, T, 2>, grid, block, stream, a, part, p);
  else
    launch(kv_attend_split_kernel<D, T, 4>, grid, block, stream, a, part, p);
  if (rc) return rc;
  if (p.chunks > 1) {
    // A row's parts by one wave, or, where there are many, by four.
    const int per = p.chunks <= 16 ? 1 : kWaves, rows = kWaves / per;
    arm_kernel_events({nullptr, ev.stop});
    launch(kv_attend_join_kernel<D, T>, dim3((a.max_q * a.Hq + rows - 1) / rows, a.B), block, stream,
           a, part, p, per);
  }
  return launch_status("kv_attention");
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
