// Attention of drafted tokens over a paged cache and their own ancestors.
//
// Request b has len_b cached tokens, positions 0 .. len_b - 1, in the pages of its table row, and drafted tokens
// cu_b .. cu_b+1 - 1 whose keys and values are not in the cache. Token t of request b at position p_t sees
//   cached key at position n         iff n > p_t - window (every n when window = 0)
//   drafted key j of its own request iff bit j of its mask is set (without a mask: j <= t) and p_j > p_t - window
// and its output is sum_n softmax_n(scale q.k_n) v_n over what it sees, its log-sum-exp log sum_n exp(scale q.k_n).
// A token that sees nothing has output 0 and log-sum-exp -inf. What is not seen is never part of a result, whatever
// its bits are: NaN or infinities beyond a request's length, in another branch or outside the window change nothing.
#pragma once
#include "draft_rows.cuh"

namespace hsg {

struct DraftAttnArgs {
  const void* q;             // [tokens][hq][dim] by strides (elements)
  const void *k, *v;         // [tokens][hkv][dim] by strides
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  PageCache cache;
  const int32_t* table;      // [rows][width], rows table_stride apart
  int64_t table_stride;
  const int32_t* lens;       // [rows]
  const int32_t* cu;         // [rows + 1]
  const int32_t* positions;  // [tokens], or NULL: len + index (read only with a window)
  const uint32_t* mask;      // [tokens][words], or NULL: the chain
  int rows, width, tokens, words, max_tree, hq, hkv, window;
  float scale;
  void* out;                 // [tokens][hq][dim]
  float* lse;                // [tokens][hq]
  int* err;
};

constexpr int DA_THREADS = 128;

// The plainest form: one warp a (drafted token, query head), key after key with a running maximum and sum.
template <int D, typename T>
__global__ void __launch_bounds__(DA_THREADS) draft_attn_simple_kernel(const DraftAttnArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t job = (int64_t)blockIdx.x * (DA_THREADS / 32) + (threadIdx.x >> 5);
  if (job >= (int64_t)a.tokens * a.hq) return;
  const int t = (int)(job / a.hq), h = (int)(job % a.hq), g = h / (a.hq / a.hkv);
  int lo = 0, hi = a.rows;  // the last request that starts at or before t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= t) lo = mid; else hi = mid;
  }
  const int b = lo, t0 = a.cu[b];
  int t1 = a.cu[b + 1];
  if (t0 < 0 || t1 < t0 || t1 > a.tokens || t1 - t0 > a.max_tree) {
    set_error(a.err, ERR_BAD_LEN);
    t1 = t0;  // nothing of this request is read
  }
  constexpr int E = D / 32;
  float q[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = t < t1 ? (float)((const T*)a.q)[t * a.q_ts + h * a.q_hs + e * 32 + lane] : 0.f;
    acc[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  auto key = [&](const T* kp, const T* vp) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += q[e] * (float)kp[e * 32 + lane];
    s = warp_sum(s) * a.scale;
    const float top = fmaxf(m, s);
    const float w = s == -INFINITY ? 0.f : expf(s - top), keep = m == -INFINITY ? 0.f : expf(m - top);
    m = top;
    l = l * keep + w;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * keep + (s == -INFINITY ? 0.f : w * (float)vp[e * 32 + lane]);
  };
  int len = a.lens[b];
  if (len < 0 || len > (int64_t)a.width * a.cache.page) {
    set_error(a.err, ERR_BAD_LEN);
    len = 0;
  }
  if (t < t1 && t >= t0) {
    const int64_t qp = a.window && a.positions ? a.positions[t] : (int64_t)len + t - t0;
    const int64_t low = a.window ? qp - a.window : -1;  // seen: positions above it
    for (int64_t n = low < 0 ? 0 : low + 1; n < len; ++n) {
      const int page = a.table[b * a.table_stride + n / a.cache.page];
      if (page < 0 || page >= a.cache.pages) {
        set_error(a.err, ERR_BAD_PAGE);
        continue;
      }
      const int64_t at = page * a.cache.page_stride + n % a.cache.page * a.cache.token_stride + g * a.cache.head_stride;
      key((const T*)a.cache.k + at, (const T*)a.cache.v + at);
    }
    for (int j = 0; j < t1 - t0; ++j) {
      if (a.mask ? (j >= 32 * a.words || !(a.mask[(int64_t)t * a.words + (j >> 5)] >> (j & 31) & 1)) : j > t - t0) continue;
      if (a.window && (a.positions ? a.positions[t0 + j] : (int64_t)len + j) <= low) continue;
      key((const T*)a.k + (t0 + j) * a.k_ts + g * a.k_hs, (const T*)a.v + (t0 + j) * a.v_ts + g * a.v_hs);
    }
  }
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) ((T*)a.out)[job * D + e * 32 + lane] = (T)(acc[e] * inv);
  if (lane == 0 && a.lse) a.lse[job] = l > 0.f || l != l ? m + logf(l) : -INFINITY;
}

}  // namespace hsg
