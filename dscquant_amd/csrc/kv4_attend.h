// Device code that the kernels of attention over the 4-bit key/value cache share: which
// tokens a row sees, where they are, and codes as matrix operands.
#pragma once

#include "kv4.h"
#include "mma_int4.h"
#include "rowquant.h"

namespace dscq {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The binary place that a row's largest weight times scale is given, and may pass by eight.
constexpr float kReference = 7.0f;

// A value every lane holds alike, read through the scalar cache.
__device__ __forceinline__ int32_t uniform_load(const int32_t* p) {
  typedef const __attribute__((address_space(4))) int32_t* Ptr;
  return *(Ptr)(reinterpret_cast<uintptr_t>(p));
}

// Sequence b's queries (rows first .. first + n - 1 of q) and the first one's place among its
// tokens, less than 0 where it has more queries than tokens.  max_q cuts n off, not the places.
struct Sequence {
  int64_t first;
  int n, place;
  int64_t past;     // queries past max_q
  int64_t lo, hi;  // the rows of all sequences (loaded here so that one wait is enough)
};
__device__ __forceinline__ Sequence sequence_of(const KvAttend& a, int b) {
  int64_t s0 = b, s1 = b + 1, lo = 0, hi = a.T;
  if (a.starts) {
    lo = min(max(uniform_load(a.starts), 0), a.T);
    hi = max(uniform_load(a.starts + a.B), 0);
    s0 = max(uniform_load(a.starts + b), 0);
    s1 = uniform_load(a.starts + b + 1);
  }
  const int64_t L = min((int64_t)max(uniform_load(a.lengths + b), 0), a.width * a.cache.P);
  const int place = (int)(L - max(s1 - s0, 0));
  s0 = min(s0, a.T);
  s1 = min(max(s1, s0), a.T);
  const int n = (int)min(s1 - s0, (int64_t)a.max_q);
  return {s0, n, place, s1 - s0 - n, lo, hi};
}

// One past the last token that query i sees, and the first.
__device__ __forceinline__ int row_end(const Sequence& s, int i) {
  return max(s.place + i + 1, 0);
}
__device__ __forceinline__ int row_begin(const KvAttend& a, const Sequence& s, int i) {
  const int64_t b = (int64_t)(s.place + i + 1) - a.window;
  return a.window && b > 0 ? (int)b : 0;
}

// Rows that nothing is computed for, of no sequence or past max_q: results 0, log sums -inf.
// Every step-th of the rows from r0 to r1 - 1, by the threads of a workgroup.
__device__ __forceinline__ void clear_rows(const KvAttend& a, int D, int64_t r0, int64_t r1,
                                           int64_t step, int threads) {
  const int row = a.Hq * D;
#pragma unroll 1
  for (int64_t r = r0; r < r1; r += step) {
    uint16_t* out = static_cast<uint16_t*>(a.out) + r * row;
    for (int e = threadIdx.x * 8; e < row; e += threads * 8)
      *reinterpret_cast<u32x4_a2*>(out + e) = (u32x4_a2){0, 0, 0, 0};
    for (int h = threadIdx.x; a.lse && h < a.Hq; h += threads) a.lse[r * a.Hq + h] = -INFINITY;
  }
}
// The rows before the first sequence's and after the last one's, dealt out to all workgroups.
__device__ __forceinline__ void clear_outside(const KvAttend& a, const Sequence& s, int D,
                                              int threads) {
  if (s.lo == 0 && s.hi >= a.T) return;
  const int64_t all = (int64_t)gridDim.x * gridDim.y * gridDim.z;
  const int64_t mine = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
  clear_rows(a, D, mine, s.lo, all, threads);
  clear_rows(a, D, s.hi + mine, a.T, all, threads);
}

struct Part {  // rows' results over some of their tokens
  float* out;  // [rows][chunks][D], rows = (b max_q + i) Hq + head
  float* log;  // [rows][chunks]: log2 of the softmax sum
};

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

// Where a sequence's tiles are.
struct Places {
  const int32_t* table;
  int per, end;      // tiles of a page; one past the last token
  uint32_t inverse;  // ceil(2^32 / per)
};
__device__ __forceinline__ Places places_of(const KvAttend& a, int b, int end) {
  const int per = a.cache.P / kKvTile;
  return {a.tables + b * a.width, per, end, (uint32_t)((0x100000000ull + per - 1) / per)};
}
struct Place {
  int page, at;  // the table's entry, -1 past the end; the tile's place in its page
};
__device__ __forceinline__ Place place_of(const Places& g, int tile) {
  const int i = g.per == 1 ? tile : (int)__umulhi((uint32_t)tile, g.inverse);
  return {tile * kKvTile < g.end ? uniform_load(g.table + i) : -1, tile - i * g.per};
}

// Two nibbles 16 bits apart as fp16 numbers less their zero-points.  0x6400 | c is the
// fp16 number 1024 + c; with the nibble four bits up, 1024 + 16 c, a sixteenth of which is
// 64 + c.  Both subtractions are exact.
struct ZeroPair {
  h2 low, high;  // -(1024 + z), -(64 + z)
};
// (x & mask) | bits in one instruction: with both as literals the compiler needs two (an
// instruction takes one), so it is not shown their values.
struct Masks {
  uint32_t low = 0x000F000Fu, high = 0x00F000F0u, magic = 0x64006400u;
  uint32_t zero_low = 0xE400E400u, zero_high = 0xD400D400u;
  __device__ __forceinline__ Masks() {
    asm("" : "+s"(low), "+s"(high), "+v"(magic), "+v"(zero_low), "+v"(zero_high));
  }
};
__device__ __forceinline__ ZeroPair zero_pair(uint32_t word0, uint32_t word1, const Masks& m) {
  // Bytes 0 of the two words, 16 bits apart.
  const uint32_t z = __builtin_amdgcn_perm(word1, word0, 0x0C040C00u);
  ZeroPair r;
  r.low = __builtin_bit_cast(h2, (z & m.low) | m.zero_low);
  r.high = __builtin_bit_cast(h2, ((z << 4) & m.high) | m.zero_high);
  return r;
}
__device__ __forceinline__ void unpack_word(uint32_t w, const ZeroPair& z, const Masks& m,
                                            h2 out[4]) {
  const h2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = w >> (8 * i);
    out[2 * i] = __builtin_bit_cast(h2, (x & m.low) | m.magic) + z.low;
    out[2 * i + 1] = __builtin_elementwise_fma(__builtin_bit_cast(h2, (x & m.high) | m.magic),
                                               sixteenth, z.high);
  }
}
__device__ __forceinline__ h8 join8(h2 a, h2 b, h2 c, h2 d) {
  return (h8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace dscq
