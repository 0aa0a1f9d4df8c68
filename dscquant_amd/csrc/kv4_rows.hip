// Rows into and out of the 4-bit key/value cache (layout: kv4.h).
//
// Both kernels are one pass over their rows and bound by memory: an appended token
// reads 2 D (Hq + 2 H) bytes and writes 2 D Hq + H (D + 8), a token read back moves
// H (D + 8) in and 4 D H out, for some ten operations an element.  D/8 lanes hold a row,
// eight elements each, so a lane's load and store are 16 bytes and its elements are one
// word of a key row and one chunk of a value row; a wave takes 64 / (D/8) tokens of one
// head and a workgroup sixteen or more consecutive ones, whose pieces of the cache lie
// side by side when their slots do.
//
// Measured: 8192 tokens of 64 query and 8 key/value heads of 128 (bf16, turned and rotated)
// appended in 115 us (315 MB, 2.7 TB/s: a workgroup's heads come one after another, each
// waiting for its row), one token of 32 heads in 4.0; 16384 tokens of 8 heads read back in
// 16.8 us (85 MB, 5.1 TB/s, the rate of a large copy).

#include <algorithm>

#include "kv4.h"
#include "mma_int4.h"
#include "rowquant.h"

namespace dscq {

namespace {

constexpr int kHalfMirror = 0x141;  // DPP row_half_mirror: lane i reads lane i ^ 7
constexpr int kQuadXor3 = 0x1B;

// The partner lane's value, for lane distances 1, 2, 4 and 8 inside a row of 16 lanes.
template <int H>
__device__ __forceinline__ float lane_xor(float v) {
  if constexpr (H == 1) return dpp_f32<kDppQuadXor1>(v);
  if constexpr (H == 2) return dpp_f32<kDppQuadXor2>(v);
  if constexpr (H == 4) return dpp_f32<kQuadXor3>(dpp_f32<kHalfMirror>(v));
  if constexpr (H == 8) return dpp_f32<kDppRowRor8>(v);
}

template <int D>
__device__ __forceinline__ float row_min(float v) {
  v = fminf(v, lane_xor<1>(v));
  v = fminf(v, lane_xor<2>(v));
  v = fminf(v, lane_xor<4>(v));
  return D == 128 ? fminf(v, lane_xor<8>(v)) : v;
}

template <int H>
__device__ __forceinline__ void fwht_lanes(float x[8], int lane) {
  const float s = (lane & H) ? -1.0f : 1.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf(s, x[i], lane_xor<H>(x[i]));
}

// x <- H_D x over the D/8 lanes of a row (index bits in ascending order).
template <int D>
__device__ __forceinline__ void fwht_row(float x[8], int lane) {
  fwht_chunk(x);
  fwht_lanes<1>(x, lane);
  fwht_lanes<2>(x, lane);
  fwht_lanes<4>(x, lane);
  if constexpr (D == 128) fwht_lanes<8>(x, lane);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float x[8]) {
  u32x4_a2 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_pair<T>(x[2 * i], x[2 * i + 1]);
  *reinterpret_cast<u32x4_a2*>(p) = w;
}

// Elements e0 .. e0 + 7 of a row turned by position.  In halves element i < R/2 pairs
// with i + R/2 (read beside it: the row is in the cache of the CU), else 2 i with 2 i + 1.
template <typename T>
__device__ __forceinline__ void turn(const T* row, int e0, const float* cos, const float* sin,
                                     int R, bool interleaved, float x[8]) {
  if (e0 >= R) return;
  const int half = R >> 1;
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = cos[(e0 >> 1) + i], s = sin[(e0 >> 1) + i];
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = a * c - b * s;
      x[2 * i + 1] = b * c + a * s;
    }
  } else {
    const bool low = e0 < half;
    float y[8];
    to_f32(load_raw_at<T>(row, (uint32_t)(low ? e0 + half : e0 - half)), y);
    const int at = low ? e0 : e0 - half;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = cos[at + i], s = sin[at + i];
      const float own = x[i] * c, other = y[i] * s;
      x[i] = low ? own - other : own + other;
    }
  }
}

// The row's word and the codes of this lane's eight elements (as whole floats).
// The scale is rounded up so that its last four bits can hold the zero-point; with them
// it is at most 31 last places above (hi - lo) / 15, and the codes are made with it as
// it is, so nothing is lost by the place the zero-point takes.  A row that holds an
// infinity or a NaN, or whose range overflows, gets the NaN word: what attends to it is
// NaN, as with the row itself.
template <int D>
__device__ __forceinline__ uint32_t kv_row_word(const float x[8], float q[8]) {
  float lo = fminf(x[0], 0.0f), hi = fmaxf(x[0], 0.0f);
  float big = 0.0f;  // NaN where x[i] * 0 is
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    big = __builtin_fmaf(x[i], 0.0f, big);
  }
  lo = row_min<D>(lo);
  hi = -row_min<D>(-hi);
  big += lane_xor<1>(big);
  big += lane_xor<2>(big);
  big += lane_xor<4>(big);
  if constexpr (D == 128) big += lane_xor<8>(big);
  const float base = fmaxf((hi - lo) / 15.0f, 1e-8f);
  const uint32_t bits = (__float_as_uint(base) + 15u) & ~15u;
  const float zero =
      __builtin_amdgcn_fmed3f(__builtin_rintf(-lo / __uint_as_float(bits)), 0.0f, 15.0f);
  const uint32_t word = bits | (uint32_t)zero;
  const float scale = __uint_as_float(word);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    q[i] = __builtin_amdgcn_fmed3f(__builtin_rintf(x[i] / scale + zero), 0.0f, 15.0f);
  return big == 0.0f && bits < 0x7F800000u ? word : kKvNan;
}

// One row into its place: the lane's word of a key row, or its D/64 two-byte pieces of
// the value quad's words.
template <int D>
__device__ __forceinline__ void store_codes(uint8_t* block, int P, int t, bool value, int lane,
                                            uint32_t word, const float q[8]) {
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = (uint32_t)q[i];
  if (value) {
    // lane `lane` holds elements 8 lane ..: chunk lane (D = 128) or lanes' halves of two
    // chunks of four (D = 64).
    const uint32_t w0 = c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12;
    const uint32_t w1 = c[4] | c[5] << 4 | c[6] << 8 | c[7] << 12;
    const int b = (t >> 1) & 1, h = t & 1;
    uint16_t *p0, *p1;
    if constexpr (D == 128) {
      p0 = reinterpret_cast<uint16_t*>(block + kv_value_at<D>(P, t, lane) + b * 8 + h * 2);
      p1 = p0 + 2;
    } else {
      p0 = reinterpret_cast<uint16_t*>(block + kv_value_at<D>(P, t, 2 * lane) + b * 4 + h * 2);
      p1 = p0 + 4;
    }
    *p0 = (uint16_t)w0;
    *p1 = (uint16_t)w1;
  } else {
    const uint32_t w = c[0] | c[2] << 4 | c[4] << 8 | c[6] << 12 | c[1] << 16 | c[3] << 20 |
                       c[5] << 24 | c[7] << 28;
    constexpr int kLanes = D / 32;  // of a quarter row
    *reinterpret_cast<uint32_t*>(block + kv_key_at<D>(t, lane / kLanes) + lane % kLanes * 4) = w;
  }
  if (lane == 0) *reinterpret_cast<uint32_t*>(block + kv_word_at<D>(P, t, value)) = word;
}

constexpr int kRowThreads = 256;

// Grid: (tokens / (256 / (D/8)), groups of `per` heads); the heads of a group are a range
// of q heads, then key heads, then value heads.
template <int D, typename T, bool ROT>
__global__ __launch_bounds__(kRowThreads) void kv_append_kernel(KvAppend a, int per) {
  constexpr int kLanes = D / 8;
  const int lane = threadIdx.x % kLanes;
  const int64_t token = (int64_t)blockIdx.x * (kRowThreads / kLanes) + threadIdx.x / kLanes;
  if (token >= a.T) return;
  const int H = a.cache.H, first = a.q ? 0 : a.Hq;
  const int h0 = first + blockIdx.y * per, h1 = min(h0 + per, a.Hq + 2 * H);
  const int64_t slot = a.slots[token];
  int64_t pos = 0;
  bool known = true;
  if (a.cos) {
    pos = a.positions[token];
    known = pos >= 0 && pos < a.table_rows;
    pos = known ? pos : 0;
  }
  const int64_t page = slot / a.cache.P;
  const int t = (int)(slot - page * a.cache.P);
  const bool kept = known && slot >= 0 && page < a.cache.pages;
  const float* cos = a.cos ? a.cos + pos * (a.rotary >> 1) : nullptr;
  const float* sin = a.cos ? a.sin + pos * (a.rotary >> 1) : nullptr;
  for (int h = h0; h < h1; ++h) {
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + H;
    const int at = is_q ? h : is_v ? h - a.Hq - H : h - a.Hq;
    const T* row = is_q ? static_cast<const T*>(a.q) + token * a.q_ts + at * a.q_hs
                   : is_v ? static_cast<const T*>(a.v) + token * a.v_ts + at * a.v_hs
                          : static_cast<const T*>(a.k) + token * a.k_ts + at * a.k_hs;
    float x[8];
    to_f32(load_raw_at<T>(row, 8 * lane), x);
    if (!is_v) {
      if (cos) turn<T>(row, 8 * lane, cos, sin, a.rotary, a.interleaved, x);
      if constexpr (ROT) fwht_row<D>(x, lane);
    }
    if (is_q) {
      if constexpr (ROT) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= 1.0f / D;
      }
      if (!known) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(kKvNan);
      }
      store8<T>(static_cast<T*>(a.q_out) + (token * a.Hq + at) * D + 8 * lane, x);
    } else {
      float q[8];
      const uint32_t word = kv_row_word<D>(x, q);
      if (kept)
        store_codes<D>(a.cache.data + (page * H + at) * kv_block_bytes<D>(a.cache.P), a.cache.P, t,
                       is_v, lane, word, q);
    }
  }
}

// Grid as above, the heads of a group key/value heads; a slot outside the cache gives zeros.
template <int D, typename T, bool ROT>
__global__ __launch_bounds__(kRowThreads) void kv_read_kernel(KvRead a, int per) {
  constexpr int kLanes = D / 8;
  const int lane = threadIdx.x % kLanes;
  const int64_t token = (int64_t)blockIdx.x * (kRowThreads / kLanes) + threadIdx.x / kLanes;
  if (token >= a.T) return;
  const int H = a.cache.H, P = a.cache.P;
  const int h0 = blockIdx.y * per, h1 = min(h0 + per, H);
  const int64_t slot = a.slots[token];
  const int64_t page = slot / P;
  const int t = (int)(slot - page * P);
  const bool kept = slot >= 0 && page < a.cache.pages;
  for (int h = h0; h < h1; ++h) {
    float k[8] = {}, v[8] = {};
    if (kept) {
      const uint8_t* block = a.cache.data + (page * H + h) * kv_block_bytes<D>(P);
      constexpr int kQ = D / 32;
      const uint32_t kw =
          *reinterpret_cast<const uint32_t*>(block + kv_key_at<D>(t, lane / kQ) + lane % kQ * 4);
      const uint32_t ks = *reinterpret_cast<const uint32_t*>(block + kv_word_at<D>(P, t, false));
      const uint32_t vs = *reinterpret_cast<const uint32_t*>(block + kv_word_at<D>(P, t, true));
      const int b = (t >> 1) & 1, odd = t & 1;
      uint32_t v0, v1;
      if constexpr (D == 128) {
        const uint8_t* p = block + kv_value_at<D>(P, t, lane) + b * 8 + odd * 2;
        v0 = *reinterpret_cast<const uint16_t*>(p);
        v1 = *reinterpret_cast<const uint16_t*>(p + 4);
      } else {
        const uint8_t* p = block + kv_value_at<D>(P, t, 2 * lane) + b * 4 + odd * 2;
        v0 = *reinterpret_cast<const uint16_t*>(p);
        v1 = *reinterpret_cast<const uint16_t*>(p + 8);
      }
      const float kz = (float)(ks & 15u), kf = __uint_as_float(ks);
      const float vz = (float)(vs & 15u), vf = __uint_as_float(vs);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int n = (i & 1) * 4 + (i >> 1);
        k[i] = ((float)((kw >> (4 * n)) & 15u) - kz) * kf;
        v[i] = ((float)(((i < 4 ? v0 : v1) >> (4 * (i & 3))) & 15u) - vz) * vf;
      }
    }
    if constexpr (ROT) {
      fwht_row<D>(k, lane);
#pragma unroll
      for (int i = 0; i < 8; ++i) k[i] *= 1.0f / D;
    }
    const int64_t at = (token * H + h) * D + 8 * lane;
    store8<T>(static_cast<T*>(a.k) + at, k);
    store8<T>(static_cast<T*>(a.v) + at, v);
  }
}

// Heads a workgroup takes one after another: all of them once there are workgroups
// enough without splitting the heads, so that a token's angles and slot are read once.
int heads_per_group(int64_t tiles, int heads) {
  const int64_t want = 8 * (int64_t)cu_count();
  const int64_t groups = tiles >= want ? 1 : (want + tiles - 1) / tiles;
  return (int)((heads + groups - 1) / groups);
}

// Tokens of a launch: a grid that holds 2^32 threads or more (2^28 tokens of D = 128) is not
// refused but wraps, so more tokens than this take several launches.
constexpr int64_t kLaunchTokens = int64_t{1} << 27;

// `launch(first, n)` for ranges of T tokens; timing events, if armed, span all of them.
template <typename F>
int in_launches(int64_t T, F launch) {
  if (T <= kLaunchTokens) return launch(0, T);
  const KernelEvents ev = take_kernel_events();
  for (int64_t t = 0; t < T; t += kLaunchTokens) {
    const int64_t n = std::min(kLaunchTokens, T - t);
    arm_kernel_events({t == 0 ? ev.start : nullptr, t + n == T ? ev.stop : nullptr});
    if (int rc = launch(t, n)) return rc;
  }
  return 0;
}

template <int D, typename T>
int append_rows(const KvAppend& a, bool rotate, hipStream_t stream) {
  const int64_t tiles = (a.T + kRowThreads / (D / 8) - 1) / (kRowThreads / (D / 8));
  const int heads = (a.q ? a.Hq : 0) + 2 * a.cache.H;
  const int per = heads_per_group(tiles, heads);
  const dim3 grid((uint32_t)tiles, (uint32_t)((heads + per - 1) / per));
  if (rotate)
    launch(kv_append_kernel<D, T, true>, grid, dim3(kRowThreads), stream, a, per);
  else
    launch(kv_append_kernel<D, T, false>, grid, dim3(kRowThreads), stream, a, per);
  return launch_status("kv_append");
}

template <int D, typename T>
int read_rows(const KvRead& a, bool rotate, hipStream_t stream) {
  const int64_t tiles = (a.T + kRowThreads / (D / 8) - 1) / (kRowThreads / (D / 8));
  const int per = heads_per_group(tiles, a.cache.H);
  const dim3 grid((uint32_t)tiles, (uint32_t)((a.cache.H + per - 1) / per));
  if (rotate)
    launch(kv_read_kernel<D, T, true>, grid, dim3(kRowThreads), stream, a, per);
  else
    launch(kv_read_kernel<D, T, false>, grid, dim3(kRowThreads), stream, a, per);
  return launch_status("kv_read");
}

}  // namespace

int kv_append(const KvAppend& a, int D, bool is_bf16, bool rotate, hipStream_t stream) {
  return in_launches(a.T, [&](int64_t first, int64_t n) {
    KvAppend p = a;  // rows of 16-bit elements
    p.T = n;
    if (a.q) p.q = static_cast<const uint16_t*>(a.q) + first * a.q_ts;
    p.k = static_cast<const uint16_t*>(a.k) + first * a.k_ts;
    p.v = static_cast<const uint16_t*>(a.v) + first * a.v_ts;
    if (a.cos) p.positions = a.positions + first;
    p.slots = a.slots + first;
    if (a.q) p.q_out = static_cast<uint16_t*>(a.q_out) + first * a.Hq * D;
    if (D == 128)
      return is_bf16 ? append_rows<128, bf16>(p, rotate, stream)
                     : append_rows<128, __half>(p, rotate, stream);
    return is_bf16 ? append_rows<64, bf16>(p, rotate, stream)
                   : append_rows<64, __half>(p, rotate, stream);
  });
}

int kv_read(const KvRead& a, int D, bool is_bf16, bool rotate, hipStream_t stream) {
  return in_launches(a.T, [&](int64_t first, int64_t n) {
    KvRead p = a;  // rows of 16-bit elements
    p.T = n;
    p.slots = a.slots + first;
    p.k = static_cast<uint16_t*>(a.k) + first * a.cache.H * D;
    p.v = static_cast<uint16_t*>(a.v) + first * a.cache.H * D;
    if (D == 128)
      return is_bf16 ? read_rows<128, bf16>(p, rotate, stream)
                     : read_rows<128, __half>(p, rotate, stream);
    return is_bf16 ? read_rows<64, bf16>(p, rotate, stream)
                   : read_rows<64, __half>(p, rotate, stream);
  });
}

}  // namespace dscq
