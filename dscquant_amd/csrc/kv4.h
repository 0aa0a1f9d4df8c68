// The 4-bit paged key/value cache: its layout and the arguments of its kernels.
//
// The cache is u8 [pages, H, P, D + 8]: pages of P tokens (P % 16 == 0), H key/value
// heads of D = 64 or 128 elements.  The P (D + 8) bytes of one (page, head) are a block,
// so a page moves as one piece:
//
//   keys    [P/16][4][16][D/32] words: token 16 a + r, elements g D/4 + 8 w .. + 7 are
//           word [a][g][r][w]; element e of the eight is nibble 0 4 1 5 2 6 3 7 [e]
//   values  [P/4][16][2][D/64] words: token 4 a + 2 b + h, element c D/16 + 4 m + j is
//           nibble 4 h + j of word [a][c][b][m]
//   words   [P] of the keys, [P] of the values: the row's scale and zero-point
//
// Both orders are those in which a 16 x 16 x 32 matrix instruction's lanes take their
// operand, so the 64 lanes of a wave read sixteen tokens as one contiguous piece, and
// two nibbles 16 bits apart become one register of two fp16 numbers.
//
// A row's word is its scale as an fp32 number whose last four bits are its zero-point
// (kv_row_word); code c stands for (c - zero) * scale.
#pragma once

#include "common.h"

namespace dscq {

constexpr int kKvTile = 16;      // tokens of a key tile; pages are whole tiles
constexpr int64_t kKvMaxLength = int64_t{1} << 28;  // tokens of a sequence
constexpr uint32_t kKvNan = 0x7FC00000u;  // the word of a row that is not finite

struct KvCache {
  uint8_t* data;
  int64_t pages;
  int32_t P, H;  // tokens of a page, key/value heads
};

// Bytes of one (page, head) block.
template <int D>
__host__ __device__ __forceinline__ int64_t kv_block_bytes(int P) {
  return (int64_t)P * (D + 8);
}
// Byte offsets inside a block: the D/8 bytes of token t's quarter g; the D/8 bytes of
// chunk c (D/16 elements) of the four tokens that t is among; the two words.
template <int D>
__host__ __device__ __forceinline__ int kv_key_at(int t, int g) {
  return ((t >> 4) * 64 + g * 16 + (t & 15)) * (D / 8);
}
template <int D>
__host__ __device__ __forceinline__ int kv_value_at(int P, int t, int c) {
  return P * (D / 2) + ((t >> 2) * 16 + c) * (D / 8);
}
template <int D>
__host__ __device__ __forceinline__ int kv_word_at(int P, int t, bool value) {
  return P * D + ((value ? P : 0) + t) * 4;
}

struct KvAppend {
  const void *q, *k, *v;  // rows [T, heads, D] at the strides below; q may be null
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // token and head strides, elements
  int64_t T;
  int32_t Hq;
  const float *cos, *sin;  // [table_rows, rotary / 2]; null: no turn
  int64_t table_rows;
  int32_t rotary, interleaved;
  const int64_t *positions, *slots;
  void* q_out;  // [T, Hq, D]
  KvCache cache;
};

struct KvRead {
  KvCache cache;
  const int64_t* slots;
  int64_t T;
  void *k, *v;  // [T, H, D]
};

struct KvAttend {
  const void* q;  // rows [T, Hq, D] at the strides below
  int64_t q_ts, q_hs, T;
  KvCache cache;
  int32_t Hq;
  const int32_t* tables;  // [B, width] pages of each sequence
  int64_t width;
  const int32_t* lengths;  // [B] cached tokens, the new ones among them
  const int32_t* starts;   // [B + 1] each sequence's first query; null: query b is sequence b's
  int32_t B, max_q;
  int64_t max_length;
  float scale;
  int64_t window;  // 0: none
  void* out;       // [T, Hq, D]
  float* lse;      // [T, Hq] or null
};

}  // namespace dscq
