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
// as what they are.  q enters as fp16; a bf16 row is first multiplied by the power of two that
// takes its largest element to [2^14, 2^15) (eight bits of each element, so exact but for
// elements 2^31 times smaller than the row's largest).  Both products are made transposed,
//   S^T = K q^T  (16 tokens x 16 rows),  O^T += V^T P^T  (16 elements x 16 rows),
// because then a lane holds scores of one row only -- lane (c, g) = (lane % 16, lane / 16)
// those of row c and tokens 4 g .. 4 g + 3 of a tile -- so maximum, sum and rescaling are
// a lane's own, and the scores are the next product's operand as they lie: its 32-token
// index may run in any order, and runs 4 g + i, 16 + 4 g + i over the two tiles of a step.
//
// Weights.  p'_j = 2^((s_j - m) log2 e + x) f'_j for the value's scale f', rounded to fp16 (the
// one rounding here that is not fp32's: 2^-11 of a weight, the size of an fp16 output's own),
// and the sum is that of 2^((s_j - m) log2 e + x) in fp32.  The row's reference x - m follows
// its largest weight times scale, which it puts at 2^7 and which may pass that by 8 binary
// places before the reference moves: within fp16, whose small numbers end 2^31 below.  A value
// without weight moves nothing, however large.  A step whose largest score and largest scale
// together stay below the limit (a vote of the wave) rescales nothing.
//
// This file: up to sixteen rows a key/value head (single tokens, a few drafted ones), bound by
// the cache's bytes, D + 8 a token and head.  A step of a wave is 32 tokens, 4352 bytes at
// D = 128, for 240 vector instructions (160 of them unpack) and 16 matrix ones, which two
// waves on a SIMD issue in 1.1 us together.  Measured (D = 128): 131072 tokens of 8 heads
// (143 MB) 31.8 us and 5.2 for the join, 4.5 TB/s (a large copy here: 5.2); 64 sequences of 1
// to 4096 tokens (143 MB) 45.4 and 5.6; 777 tokens of 32 heads 9.6, where start and end are 5.
// More rows: kv4_prompt.hip.
//
// Measured and not kept: codes as fp16 subnormals, which the matrix cores take as they are
// (160 instructions a step, 3% faster), because products of subnormals keep 17 bits or so; the
// loop's body three times with two steps on their way (first fetches of instructions cost
// more: 48 us for the 64 sequences); 32 and 64 rows a wave (13 us before the first step).

#include <algorithm>

#include "kv4_attend.h"

namespace dscq {

int kv_attend_prompt(const KvAttend& a, int D, bool is_bf16, const Part& part, int waves,
                     int chunks, int least, hipStream_t stream);

namespace {

constexpr int kWaves = 4;
constexpr int kStep = 2 * kKvTile;  // tokens of a step
// What a scale below it counts as where the reference is chosen: values of zeros have weights
// too, whose sum stays within fp32 this way.  (The rule's least scale is 2^-27.)
constexpr float kLeastScale = 0x1p-32f;

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

// The running state of sixteen rows in one wave; lane (c, g) holds row c's statistics (l: of
// its own tokens) and its elements g D/4 .. + D/4 - 1 of the output.
template <int D>
struct Rows {
  h8 q[D / 32];
  f4 o[D / 16];                                   // o[t][i]: element (4 g + i) D/16 + t
  float off = 0.0f, limit = -INFINITY, l = 0.0f;  // the reference; what moves it; the sum
  float to2;                                      // scores to binary places: scale log2 e 2^-k
  int begin, end, all_begin, all_end;             // the row's tokens; those that every row sees

  // The rows of a sequence and key/value head h: their q, and what they see.
  template <typename T>
  __device__ __forceinline__ void load(const KvAttend& a, const Sequence& s, int h, int G,
                                       int lane) {
    // A row past the last one is the last one over again; it is not stored.
    const int g = lane >> 4, row = min(lane & 15, s.n * G - 1), i = row / G;
    const T* p = static_cast<const T*>(a.q) + (s.first + i) * a.q_ts +
                 (h * G + row - i * G) * a.q_hs;
    Raw<T> raw[D / 32];
#pragma unroll
    for (int w = 0; w < D / 32; ++w) raw[w] = load_raw_at<T>(p, g * (D / 4) + 8 * w);
#pragma unroll
    for (int t = 0; t < D / 16; ++t) o[t] = (f4){0, 0, 0, 0};
    begin = row_begin(a, s, i);
    end = row_end(s, i);
    all_begin = row_begin(a, s, s.n - 1);
    all_end = row_end(s, 0);
    int k = 0;
    if constexpr (std::is_same<T, bf16>::value) {
      float top = 0.0f, y[8];
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        to_f32(raw[w], y);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(y[e]));
      }
      top = row_max(top);
      if (top > 0.0f && top < INFINITY) k = 15 - __builtin_amdgcn_frexp_expf(top);
    }
    to2 = __builtin_amdgcn_ldexpf(a.scale * kLog2e, -k);
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
      float y[8];
      to_f32(raw[w], y);
#pragma unroll
      for (int e = 0; e < 8; ++e) q[w][e] = (_Float16)__builtin_amdgcn_ldexpf(y[e], k);
    }
  }

  // The 32 tokens from j0 in tiles a and b.
  __device__ __forceinline__ void step(const Tile<D>& a, const Tile<D>& b, int j0, int lane,
                                       const Masks& masks) {
    float vf[8] = {__uint_as_float(a.vf.x), __uint_as_float(a.vf.y), __uint_as_float(a.vf.z),
                   __uint_as_float(a.vf.w), __uint_as_float(b.vf.x), __uint_as_float(b.vf.y),
                   __uint_as_float(b.vf.z), __uint_as_float(b.vf.w)};
    const float kf[8] = {__uint_as_float(a.kf.x), __uint_as_float(a.kf.y), __uint_as_float(a.kf.z),
                         __uint_as_float(a.kf.w), __uint_as_float(b.kf.x), __uint_as_float(b.kf.y),
                         __uint_as_float(b.kf.z), __uint_as_float(b.kf.w)};
    float s[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Tile<D>& t = h ? b : a;
      const ZeroPair z = zero_pair(t.kz, t.kz, masks);
      f4 c = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        h2 e[4];
        unpack_word(t.k.w[w], z, masks, e);
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(join8(e[0], e[1], e[2], e[3]), q[w], c, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * h + i] = __builtin_fmaf(c[i], kf[4 * h + i] * to2, off);
      // One tile's numbers in registers at a time.
      __builtin_amdgcn_sched_barrier(0);
    }
    const bool whole = j0 >= all_begin && j0 + kStep <= all_end && a.there && b.there;
    if (!whole) {
      // Tokens a row does not see, and pages that are not there: score -inf, and a scale
      // of 0, for what lies there may be anything.
      const int g4 = (lane >> 4) * 4;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = j0 + (i < 4 ? g4 + i : 12 + g4 + i);
        const bool seen = (i < 4 ? a.there : b.there) & (j >= begin) & (j < end);
        s[i] = seen ? s[i] : -INFINITY;
        vf[i] = seen ? vf[i] : 0.0f;
      }
    }
    const float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])),
                            fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    float most = kLeastScale;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, vf[i]);
    if (__builtin_amdgcn_ballot_w64(top + __builtin_amdgcn_logf(most) > limit)) {
      float high = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        high = fmaxf(high, s[i] + __builtin_amdgcn_logf(fmaxf(vf[i], kLeastScale)));
      high = row_max(high);
      const bool up = high > limit;
      const float delta = up ? kReference - high : 0.0f;
      const float keep = limit == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(delta);
      limit = up ? kReference + 8.0f : limit;
      off += delta;
      l *= keep;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) o[t] *= keep;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += delta;
    }
    h8 p;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = __builtin_amdgcn_exp2f(s[i]);
      l += e;
      p[i] = (_Float16)(e * vf[i]);
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
      for (int t = 0; t < 4; ++t)
        o[4 * w + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            join8(e[0][t], e[1][t], e[2][t], e[3][t]), p, o[4 * w + t], 0, 0, 0);
    }
  }

  // The steps first, first + stride, ... below `last` (tokens / 32).  While one step is
  // computed the next one's codes are on their way, and the one's after it pages.  The body
  // stands once and the codes move from register to register: a second copy of it would cost
  // a short run more, in instructions fetched for the first time, than the moves do.
  __device__ __forceinline__ void run(const Pages<D>& g, int first, int last, int stride,
                                      int lane) {
    if (first >= last) return;
    Tile<D> a = load_tile<D>(g, place_of(g.places, 2 * first));
    Tile<D> b = load_tile<D>(g, place_of(g.places, 2 * first + 1));
    Place pa = place_of(g.places, 2 * (first + stride));
    Place pb = place_of(g.places, 2 * (first + stride) + 1);
    const Masks masks;
#pragma unroll 1
    for (int at = first; at < last; at += stride) {
      const Tile<D> na = load_tile<D>(g, pa), nb = load_tile<D>(g, pb);
      pa = place_of(g.places, 2 * (at + 2 * stride));
      pb = place_of(g.places, 2 * (at + 2 * stride) + 1);
      step(a, b, at * kStep, lane, masks);
      a = na;
      b = nb;
    }
  }
};

// The launch's plan.
//   kWhole   a workgroup takes all tokens of its rows: grid (1, H, B), one kernel;
//   kParts   a sequence's tokens in up to `chunks` parts of at least `least` steps (step
//            tokens each): grid (chunks, H, B); a second kernel joins the parts;
//   kShares  each of `wgs` workgroups a head takes the same share of the batch's steps
//            (in order, at least `least`), whichever sequences that is, joined likewise;
//   kPrompt  kv4_prompt.hip: groups of `rows` rows, their tokens in parts as in kParts,
//            joined where chunks > 1.
enum Form { kWhole, kParts, kShares, kPrompt };
struct Plan {
  Form form;
  int rows, waves, step, wgs, chunks, least;
};

// The 32-token steps of a sequence's rows: one at least if there are any (empty rows are
// written too).
struct Steps {
  int first, count;
};
__device__ __forceinline__ Steps steps_of(const KvAttend& a, const Sequence& s) {
  if (s.n <= 0) return {0, 0};
  const int first = row_begin(a, s, 0) / kStep;
  return {first, max((row_end(s, s.n - 1) + kStep - 1) / kStep - first, 1)};
}

// Where a sequence's parts are, written by kv_attend_split_kernel for the join: the first
// one's slot, and how many (1: the rows are done).
struct Where {
  int slot, used;
};
struct Shares {
  Part part;     // [slots][H][rows][D]
  Where* where;  // [B]
};

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

template <int D, int NW>
struct Joint {  // LDS in which the waves of a workgroup join their results
  float out[NW][16][D + 4];
  float log[NW][16];
};

// Steps from .. to - 1 of sequence b for head h, joined over the waves: the rows' result, or
// (slot >= 0) their part, the slot-th of `chunks` of each row or in a slot of its own.
template <int D, typename T, int NW>
__device__ __forceinline__ void attend_steps(const KvAttend& a, const Shares& shares,
                                             Joint<D, NW>& joint, const Sequence& s, int b,
                                             int h, int from, int to, int64_t slot,
                                             int chunks = 0) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.Hq / a.cache.H, count = s.n * G;
  Rows<D> rows;
  const Pages<D> pages = pages_of<D>(a, b, h, row_end(s, s.n - 1), lane);
  rows.template load<T>(a, s, h, G, lane);
  rows.run(pages, from + wave, to, NW, lane);
  const int c = lane & 15, g = lane >> 4;
  const float l = row_sum(rows.l), inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < D / 16; t += 4)
      *reinterpret_cast<f4*>(&joint.out[wave][c][(4 * g + i) * (D / 16) + t]) =
          (f4){rows.o[t][i] * inv, rows.o[t + 1][i] * inv, rows.o[t + 2][i] * inv,
               rows.o[t + 3][i] * inv};
  if (g == 0) joint.log[wave][c] = l == 0.0f ? -INFINITY : __builtin_amdgcn_logf(l) - rows.off;
  __syncthreads();
  // Sixteen lanes a row, D/16 elements each.
  const int row = threadIdx.x >> 4;
  if (row < count) {
    const int d = (threadIdx.x & 15) * (D / 16);
    float top = joint.log[0][row];
#pragma unroll
    for (int w = 1; w < NW; ++w) top = fmaxf(top, joint.log[w][row]);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, y[D / 16] = {};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float p = __builtin_amdgcn_exp2f(joint.log[w][row] - base);
      sum += p;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) y[e] = __builtin_fmaf(p, joint.out[w][row][d + e], y[e]);
    }
    const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
    const float log = sum == 0.0f ? -INFINITY : base + __builtin_amdgcn_logf(sum);
    if (slot >= 0) {
      const int i = row / G, hq = h * G + row - i * G;
      const int64_t at = chunks ? (((int64_t)b * a.max_q + i) * a.Hq + hq) * chunks + slot
                                : (slot * a.cache.H + h) * ((int64_t)a.max_q * G) + row;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) shares.part.out[at * D + d + e] = y[e] * scale;
      if (d == 0) shares.part.log[at] = log;
    } else {
      const int i = row / G;
      const int64_t at = (s.first + i) * a.Hq + h * G + row - i * G;
      uint16_t* o = static_cast<uint16_t*>(a.out) + at * D + d;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) o[e] = __builtin_bit_cast(uint16_t, to_out<T>(y[e] * scale));
      if (a.lse && d == 0) a.lse[at] = log * kLn2;
    }
  }
}

// Up to sixteen rows a key/value head, the waves of a workgroup on every NW-th step; two
// waves share a SIMD.
template <int D, typename T, int NW, Form FORM>
__global__ __launch_bounds__(64 * NW, 2) void kv_attend_split_kernel(
    KvAttend a, Shares shares, Plan plan) {
  __shared__ alignas(16) Joint<D, NW> joint;
  if constexpr (FORM != kShares) {
    const int b = blockIdx.z, h = blockIdx.y;
    const Sequence s = sequence_of(a, b);
    clear_outside(a, s, D, 64 * NW);
    if (s.n <= 0) return;
    if (s.past && blockIdx.x == 0)
      clear_rows(a, D, s.first + s.n + h, s.first + s.n + s.past, a.cache.H, 64 * NW);
    const Steps steps = steps_of(a, s);
    int from = steps.first, to = from + steps.count;
    int64_t slot = -1;
    if constexpr (FORM == kParts) {
      const int each = max((steps.count + plan.chunks - 1) / plan.chunks, plan.least);
      from += blockIdx.x * each;
      if (from >= to) return;
      slot = steps.count > each ? (int64_t)blockIdx.x : -1;
      to = min(from + each, to);
    }
    attend_steps<D, T, NW>(a, shares, joint, s, b, h, from, to, slot,
                           FORM == kParts ? plan.chunks : 0);
    return;
  }
  clear_outside(a, sequence_of(a, 0), D, 64 * NW);
  // Where in the batch's steps this workgroup's share begins: the steps of all sequences,
  // summed by the threads, a run of sequences each.
  __shared__ int64_t wave_sums[NW];
  __shared__ int64_t found_start;
  __shared__ int found;
  const int h = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int run = (a.B + 64 * NW - 1) / (64 * NW), b0 = min(t * run, a.B), b1 = min(b0 + run, a.B);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += steps_of(a, sequence_of(a, b)).count;
  int64_t before = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t x = __shfl_up(before, d);
    before += lane >= d ? x : 0;
  }
  if (lane == 63) wave_sums[wave] = before;
  before -= mine;
  __syncthreads();
  int64_t all = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    before += w < wave ? wave_sums[w] : 0;
    all += wave_sums[w];
  }
  const int64_t share = max((all + gridDim.x - 1) / (int64_t)gridDim.x, (int64_t)plan.least);
  const int64_t from = blockIdx.x * share, to = min(from + share, all);
  if (from >= all) return;
  if (before <= from && from < before + mine) {
    int b = b0;
    for (;; ++b) {
      const int n = steps_of(a, sequence_of(a, b)).count;
      if (from < before + n) break;
      before += n;
    }
    found = b;
    found_start = before;
  }
  __syncthreads();
  int b = __builtin_amdgcn_readfirstlane(found);
  int64_t start = found_start;
  for (int64_t at = from; at < to; ++b) {
    const Sequence s = sequence_of(a, b);
    const Steps steps = steps_of(a, s);
    if (steps.count == 0) continue;
    const int64_t end = start + steps.count;
    const int64_t part0 = start / share, used = (end - 1) / share - part0 + 1;
    if (at == start) {
      if (h == 0 && t == 0) shares.where[b] = {(int)part0 + b, (int)used};
      if (s.past)
        clear_rows(a, D, s.first + s.n + h, s.first + s.n + s.past, a.cache.H, 64 * NW);
    }
    const int s0 = __builtin_amdgcn_readfirstlane((int)(at - start));
    const int s1 = __builtin_amdgcn_readfirstlane((int)(min(to, end) - start));
    attend_steps<D, T, NW>(a, shares, joint, s, b, h, steps.first + s0, steps.first + s1,
                               used > 1 ? (int64_t)blockIdx.x + b : -1);
    at = start = end;
    __syncthreads();
  }
}

// A row's parts, weighted by their sums.  Grid: (max_q Hq, B) rows, one a wave, or (`per` = 4)
// a workgroup, whose waves take every fourth part; eight at a time, so that their loads are
// in flight together.  A part that is NaN makes its row NaN, whatever its weight.
template <int D, typename T>
__global__ __launch_bounds__(64 * kWaves) void kv_attend_join_kernel(KvAttend a, Shares shares,
                                                                     Plan plan, int per) {
  __shared__ float out[kWaves][D], sums[kWaves];
  const int lane = threadIdx.x & 63, b = blockIdx.y;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x * (kWaves / per) + wave / per, i = row / a.Hq, hq = row - i * a.Hq;
  wave %= per;
  const Sequence s = sequence_of(a, b);
  const int H = a.cache.H, G = a.Hq / H, h = hq / G;
  int used = 0;
  int64_t at = 0, stride = 1;
  if (i < s.n && plan.form == kShares) {
    const int slot = uniform_load(&shares.where[b].slot);
    used = uniform_load(&shares.where[b].used);
    stride = H * (int64_t)a.max_q * G;
    at = slot * stride + h * ((int64_t)a.max_q * G) + i * G + hq - h * G;
  } else if (i < s.n) {
    // As the kernels of parts.
    const int r0 = (i * G + hq - h * G) / plan.rows * plan.rows;
    const int r1 = min(r0 + plan.rows, s.n * G) - 1;
    const int first = row_begin(a, s, r0 / G) / plan.step;
    const int last = (row_end(s, r1 / G) + plan.step - 1) / plan.step;
    const int each = max((last - first + plan.chunks - 1) / plan.chunks, plan.least);
    used = (max(last - first, 1) + each - 1) / each;
    at = (((int64_t)b * a.max_q + i) * a.Hq + hq) * plan.chunks;
  }
  const bool in = used > 1;  // a row of one part is done
  if (per == kWaves && !in) return;
  const Part& part = shares.part;
  float top = -INFINITY;
  for (int c = lane; in && c < used; c += 64) top = fmaxf(top, part.log[at + c * stride]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float base = top == -INFINITY ? 0.0f : top;
  constexpr int kE = D / 64, kMany = 8;
  float sum = 0.0f, y[kE] = {};
  for (int c = wave; in && c < used; c += kMany * per) {
    float log[kMany], x[kMany][kE];
#pragma unroll
    for (int m = 0; m < kMany; ++m) {
      const int64_t from = at + min(c + m * per, used - 1) * stride;
      log[m] = part.log[from];
#pragma unroll
      for (int e = 0; e < kE; ++e) x[m][e] = part.out[from * D + lane * kE + e];
    }
#pragma unroll
    for (int m = 0; m < kMany; ++m) {
      const float p = c + m * per < used ? __builtin_amdgcn_exp2f(log[m] - base) : 0.0f;
      sum += p;
#pragma unroll
      for (int e = 0; e < kE; ++e) y[e] = __builtin_fmaf(p, x[m][e], y[e]);
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

// No sequences, or no queries of them: every row is one that nothing is computed for.
__global__ __launch_bounds__(64 * kWaves) void kv_attend_none_kernel(KvAttend a, int D) {
  clear_rows(a, D, blockIdx.x, a.T, gridDim.x, 64 * kWaves);
}

Plan plan_of(int B, int Hq, int H, int max_q, int64_t max_length, int64_t window) {
  const int64_t rows = (int64_t)max_q * (Hq / H), cus = cu_count();
  const int64_t length =
      std::min<int64_t>(window ? std::min(max_length, window + max_q - 1) : max_length,
                        kKvMaxLength);
  Plan p = {};
  p.chunks = 1;
  if (rows > 16) {
    // 256 rows a workgroup, one of which a CU holds, or 128 (two); few of them: their
    // tokens in parts.
    p.form = kPrompt;
    p.rows = rows > 128 ? 256 : 128;
    p.waves = p.rows / 32;
    p.step = p.rows / 2;
    const int64_t steps = (length + p.step - 1) / p.step + 1;
    const int64_t wgs = (rows + p.rows - 1) / p.rows * B * H, slots = cus * (256 / p.rows);
    p.chunks = (int)std::max<int64_t>(1, std::min((steps + 1) / 2, slots / wgs));
    p.least = (int)std::max<int64_t>(2, (steps + p.chunks - 1) / p.chunks);
    return p;
  }
  p.rows = 16;
  p.step = kStep;
  // Up to 1024 tokens by the eight waves of one workgroup: four steps a wave cost less than
  // the second kernel (8 sequences of 1000 tokens, 64/8 heads: 10.2 us, 13.3 in parts; one of
  // 777, 32/32 heads: 8.7 and 9.9).
  p.form = length <= 1024 ? kWhole : kParts;
  p.waves = p.form == kWhole ? 8 : kWaves;
  if (p.form == kWhole) return p;
  // As many workgroups as the device holds at once: a second round would only add its start
  // and end (131072 tokens of 8 heads: 36 us in one round, 41 in two, 49 in four).  With
  // four of them a sequence or more, parts are a sequence's own; with fewer, a ragged batch
  // would leave most of the device waiting for its longest (64 sequences of 1 to 4096
  // tokens: 57 us in two parts each, 46 in equal shares), but a share that spans two
  // sequences begins and ends twice (17 sequences of 2000 in shares: 21.6 us; 16 in parts:
  // 16.1).
  p.wgs = (int)std::max<int64_t>(1, 2 * cus / H);
  p.least = kWaves;
  if (B > p.wgs / 4) {
    p.form = kShares;
  } else {
    const int64_t steps = (length + kStep - 1) / kStep + 1;
    p.chunks = (int)std::min<int64_t>(p.wgs / B, (steps + p.least - 1) / p.least);
    p.least = (int)std::max<int64_t>(p.least, (steps + p.chunks - 1) / p.chunks);
  }
  return p;
}

// Bytes of the parts, before what says where they are.
int64_t part_bytes(const Plan& p, int D, int B, int Hq, int max_q) {
  const int64_t rows = (int64_t)max_q * Hq;
  if (p.form == kShares) return (p.wgs + B) * rows * (D + 1) * 4;
  return p.chunks > 1 ? B * rows * p.chunks * (D + 1) * 4 : 0;
}

template <int D, typename T>
int attend(const KvAttend& a, void* ws, hipStream_t stream) {
  const Plan p = plan_of(a.B, a.Hq, a.cache.H, a.max_q, a.max_length, a.window);
  const bool joins = p.form == kShares || p.chunks > 1;
  Shares shares = {};
  if (joins) {
    const int64_t bytes = part_bytes(p, D, a.B, a.Hq, a.max_q);
    shares.part.out = static_cast<float*>(ws);
    shares.part.log = shares.part.out + bytes / 4 / (D + 1) * D;
    shares.where = reinterpret_cast<Where*>(static_cast<uint8_t*>(ws) + (bytes + 15) / 16 * 16);
  }
  // Timing events, if armed, span both kernels.
  const KernelEvents ev = take_kernel_events();
  arm_kernel_events({ev.start, joins ? nullptr : ev.stop});
  const dim3 grid = p.form == kShares ? dim3(p.wgs, a.cache.H, 1) : dim3(p.chunks, a.cache.H, a.B);
  const dim3 block(64 * p.waves);
  int rc = 0;
  if (p.form == kPrompt)
    rc = kv_attend_prompt(a, D, std::is_same<T, bf16>::value, shares.part, p.waves, p.chunks,
                          p.least, stream);
  else if (p.form == kWhole)
    launch(kv_attend_split_kernel<D, T, 8, kWhole>, grid, block, stream, a, shares, p);
  else if (p.form == kParts)
    launch(kv_attend_split_kernel<D, T, kWaves, kParts>, grid, block, stream, a, shares, p);
  else
    launch(kv_attend_split_kernel<D, T, kWaves, kShares>, grid, block, stream, a, shares, p);
  if (rc) return rc;
  if (joins) {
    // One wave a row where there are rows enough, else four.
    const int per = (int64_t)a.max_q * a.Hq * a.B >= 4 * cu_count() ? 1 : kWaves;
    const int rows = kWaves / per;
    arm_kernel_events({nullptr, ev.stop});
    launch(kv_attend_join_kernel<D, T>, dim3((a.max_q * a.Hq + rows - 1) / rows, a.B),
           dim3(64 * kWaves), stream, a, shares, p, per);
  }
  return launch_status("kv_attention");
}

}  // namespace

int64_t kv_attention_workspace_bytes(int D, int B, int Hq, int H, int max_q, int64_t max_length,
                                     int64_t window) {
  const Plan p = plan_of(B, Hq, H, max_q, max_length, window);
  const int64_t bytes = part_bytes(p, D, B, Hq, max_q);
  return p.form == kShares ? (bytes + 15) / 16 * 16 + B * (int64_t)sizeof(Where) : bytes;
}

int kv_attention(const KvAttend& a, int D, bool is_bf16, void* ws, hipStream_t stream) {
  if (a.B == 0 || a.max_q == 0) {
    launch(kv_attend_none_kernel, dim3((uint32_t)std::min<int64_t>(a.T, 8 * cu_count())),
           dim3(64 * kWaves), stream, a, D);
    return launch_status("kv_attention");
  }
  if (D == 128)
    return is_bf16 ? attend<128, bf16>(a, ws, stream) : attend<128, __half>(a, ws, stream);
  return is_bf16 ? attend<64, bf16>(a, ws, stream) : attend<64, __half>(a, ws, stream);
}

}  // namespace dscq
