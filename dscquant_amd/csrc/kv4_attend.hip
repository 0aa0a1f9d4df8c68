// Attention over the 4-bit key/value cache (layout: kv4.h).
//
// For query i of a sequence of L cached tokens, the last n of them the queries' own, at
// place p = L - n + i, over the tokens j <= p (and j > p - window):
//   s_j = scale q . k_j,  m = max s_j,  o = sum e^(s_j - m) v_j / sum e^(s_j - m),
//   lse = m + log sum e^(s_j - m);  no visible token: o = 0, lse = -inf.
// One wave per query row: 64 tokens a step, a token's score per lane, the sums kept with
// the running maximum.

#include "kv4.h"
#include "mma_int4.h"
#include "rowquant.h"

namespace dscq {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <int D, typename T>
__global__ __launch_bounds__(64) void kv_attend_plain_kernel(KvAttend a) {
  __shared__ float q[D], p[64];
  const int lane = threadIdx.x, b = blockIdx.z, hq = blockIdx.y;
  const int64_t s0 = a.starts ? min(max((int64_t)a.starts[b], (int64_t)0), a.T) : min((int64_t)b, a.T);
  const int64_t s1 =
      a.starts ? min(max((int64_t)a.starts[b + 1], s0), a.T) : min((int64_t)b + 1, a.T);
  const int n = (int)min(s1 - s0, (int64_t)a.max_q), i = blockIdx.x;
  if (i >= n) return;
  const int P = a.cache.P, H = a.cache.H, h = hq / (a.Hq / H);
  const int64_t L = min(max((int64_t)a.lengths[b], (int64_t)0), a.width * P);
  const T* row = static_cast<const T*>(a.q) + (s0 + i) * a.q_ts + hq * a.q_hs;
  for (int d = lane; d < D; d += 64) q[d] = elem_f32(row[d]);
  __syncthreads();
  const int64_t end = L - n + i + 1;  // one past the last visible token
  const int64_t begin = a.window ? max(end - a.window, (int64_t)0) : 0;
  float m = -INFINITY, l = 0.0f, o[D / 64] = {};
  for (int64_t j0 = begin & ~(int64_t)63; j0 < end; j0 += 64) {
    const int64_t j = j0 + lane;
    const bool seen = j >= begin && j < end;
    const int64_t page = seen ? a.tables[b * a.width + j / P] : -1;
    const bool there = page >= 0 && page < a.cache.pages;
    const uint8_t* block = a.cache.data + ((there ? page : 0) * H + h) * kv_block_bytes<D>(P);
    const int t = (int)(j % P);
    float s = -INFINITY;
    if (there) {
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(block + kv_word_at<D>(P, t, false));
      float acc = 0.0f;
      for (int w = 0; w < D / 8; ++w) {
        const uint32_t c = *reinterpret_cast<const uint32_t*>(
            block + kv_key_at<D>(t, w / (D / 32)) + w % (D / 32) * 4);
        for (int e = 0; e < 8; ++e)
          acc = __builtin_fmaf(
              q[8 * w + e], (float)((c >> (4 * ((e & 1) * 4 + (e >> 1)))) & 15) - (float)(kw & 15),
              acc);
      }
      s = acc * __uint_as_float(kw) * a.scale;
    }
    float top = s;
    for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    top = fmaxf(top, m);
    const float base = top == -INFINITY ? 0.0f : top;
    const float e = __builtin_amdgcn_exp2f((s - base) * kLog2e);
    const float keep = __builtin_amdgcn_exp2f((m - base) * kLog2e);
    float sum = e;
    for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
    l = l * keep + sum;
    m = top;
    p[lane] = e;
    __syncthreads();
    for (int r = 0; r < D / 64; ++r) o[r] *= keep;
    for (int x = 0; x < 64 && j0 + x < end; ++x) {
      const int64_t jj = j0 + x;
      if (jj < begin) continue;
      const int64_t pg = a.tables[b * a.width + jj / P];
      if (pg < 0 || pg >= a.cache.pages) continue;
      const uint8_t* bl = a.cache.data + (pg * H + h) * kv_block_bytes<D>(P);
      const int tt = (int)(jj % P);
      const uint32_t vw = *reinterpret_cast<const uint32_t*>(bl + kv_word_at<D>(P, tt, true));
      for (int r = 0; r < D / 64; ++r) {
        const int d = lane + 64 * r, c = d / (D / 16), k = d % (D / 16);
        const uint8_t byte = bl[kv_value_at<D>(P, tt, c) + ((tt >> 1) & 1) * (D / 16) + k / 4 * 4 +
                                (tt & 1) * 2 + k % 4 / 2];
        const float code = (float)((byte >> (4 * (k & 1))) & 15) - (float)(vw & 15);
        o[r] = __builtin_fmaf(p[x], code * __uint_as_float(vw), o[r]);
      }
    }
    __syncthreads();
  }
  T* out = static_cast<T*>(a.out) + ((s0 + i) * a.Hq + hq) * D;
  for (int r = 0; r < D / 64; ++r) {
    const float y = l > 0.0f || l != l ? o[r] / l : 0.0f;
    out[lane + 64 * r] = __builtin_bit_cast(T, to_out<T>(y));
  }
  if (a.lse && lane == 0) a.lse[(s0 + i) * a.Hq + hq] = m + __builtin_amdgcn_logf(l) * kLn2;
}

template <int D>
int attend(const KvAttend& a, bool is_bf16, hipStream_t stream) {
  const dim3 grid(a.max_q, a.Hq, a.B);
  if (is_bf16)
    launch(kv_attend_plain_kernel<D, bf16>, grid, dim3(64), stream, a);
  else
    launch(kv_attend_plain_kernel<D, __half>, grid, dim3(64), stream, a);
  return launch_status("kv_attention");
}

}  // namespace

int64_t kv_attention_workspace_bytes(int D, int B, int Hq, int H, int max_q, int64_t max_length,
                                     int64_t window) {
  return 0;
}

int kv_attention(const KvAttend& a, int D, bool is_bf16, void* ws, hipStream_t stream) {
  return D == 128 ? attend<128>(a, is_bf16, stream) : attend<64>(a, is_bf16, stream);
}

}  // namespace dscq
