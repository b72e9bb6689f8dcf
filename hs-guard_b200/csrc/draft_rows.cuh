// Rows of queries, keys and values in draft scoring: per-head RMSNorm and position rotation (draft_norm_kernel) and the
// copy of accepted rows into the pages of a cache (draft_store_kernel). The engine's attn_prep_kernel is the same
// mathematics bound to one projection layout, start + t positions and the ring; these take any head counts, strides,
// types and positions.
#pragma once
#include "common.cuh"

namespace hsg {

// A paged cache: K and V elements (page, token, head, d) at page * page_stride + token * token_stride +
// head * head_stride + d (in elements, 64-bit), the same strides for both.
struct PageCache {
  void* k;
  void* v;
  int64_t page_stride, token_stride, head_stride;
  int pages, page;
};

// Eight consecutive elements as fp32, and back (rounded to nearest even).
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __half* p, float (&x)[8]) {
  const uint4 r = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack_half2(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 r = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __half*) { return pack_half2(a, b); }
__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2(x[0], x[1], p), pack2(x[2], x[3], p), pack2(x[4], x[5], p),
                                            pack2(x[6], x[7], p));
}

struct DraftNormArgs {
  const void *q, *k, *v;     // [tokens][heads][dim] by strides (elements)
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  const float *qw, *kw;      // [dim] norm weights
  const float* inv_freq;     // [rot / 2]
  const int32_t* positions;  // [tokens]
  int tokens, hq, hkv, rot;
  float eps;
  void* q_out;               // [tokens][hq][dim]
  void *k_out, *v_out;       // [tokens][hkv][dim], unless slots is given
  const int32_t* slots;      // [tokens] cache slots for k and v; < 0: not kept
  PageCache cache;
  int* err;
};

// sin and cos of position * frequency. The product in fp32 is off by up to 2^-24 of the angle (4e-3 at position 65,536,
// more than an fp16 result's own rounding) and positions above 2^24 are not fp32 numbers, so the product and its
// remainder by whole turns are taken in fp64: two roundings of 2^-53 of at most 2^31, below 1e-6. What is left is at
// most half a turn, which sincosf takes without its slow path for large arguments.
__device__ __forceinline__ void rotation(int position, float freq, float& s, float& c) {
  constexpr double kTurn = 6.283185307179586476925;
  const double angle = (double)position * (double)freq;
  sincosf((float)fma(-kTurn, rint(angle * (1.0 / kTurn)), angle), &s, &c);
}

constexpr int DN_THREADS = 256;

// One thread block a token. dim / 8 lanes share a head, eight consecutive elements each, so a warp works on 256 / dim
// heads at once; the rotation's partner (d and d + rot / 2) is rot / 16 lanes away.
template <int D, typename TI, typename TO>
__global__ void __launch_bounds__(DN_THREADS) draft_norm_kernel(const DraftNormArgs a) {
  __shared__ float s_cos[D / 2], s_sin[D / 2];
  constexpr int LPH = D / 8;
  const int64_t t = blockIdx.x;
  const int half = a.rot / 2;
  for (int i = threadIdx.x; i < half; i += DN_THREADS) rotation(a.positions[t], a.inv_freq[i], s_sin[i], s_cos[i]);
  __syncthreads();
  const int heads = a.hq + 2 * a.hkv, j = threadIdx.x % LPH;
  // every thread of a warp takes part in the shuffles: the loop's trip count is the warp's
  for (int base = 0; base < heads; base += DN_THREADS / LPH) {
    const int h = base + threadIdx.x / LPH;
    const bool live = h < heads;
    const bool is_q = h < a.hq, is_k = !is_q && h < a.hq + a.hkv;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) {
      const TI* src = is_q ? (const TI*)a.q + t * a.q_ts + h * a.q_hs
                           : is_k ? (const TI*)a.k + t * a.k_ts + (h - a.hq) * a.k_hs
                                  : (const TI*)a.v + t * a.v_ts + (h - a.hq - a.hkv) * a.v_hs;
      load8(src + j * 8, x);
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (is_q || is_k) {
      const float r = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
      const float* w = (is_q ? a.qw : a.kw) + j * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
    }
    const int d = j * 8, lane = threadIdx.x & 31;
    const bool first = d < half, turned = d < a.rot && (is_q || is_k);
    const int partner = d < a.rot ? (first ? lane + half / 8 : lane - half / 8) : lane;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], partner);
    if (turned) {
      const int f = first ? d : d - half;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = first ? x[i] * s_cos[f + i] - y[i] * s_sin[f + i] : x[i] * s_cos[f + i] + y[i] * s_sin[f + i];
    }
    if (!live) continue;
    if (is_q) {
      store8((TO*)a.q_out + (t * a.hq + h) * D + d, x);
      continue;
    }
    const int g = is_k ? h - a.hq : h - a.hq - a.hkv;
    if (!a.slots) {
      store8((TO*)(is_k ? a.k_out : a.v_out) + (t * a.hkv + g) * D + d, x);
      continue;
    }
    const int slot = a.slots[t], page = slot / a.cache.page;
    if (slot < 0) continue;
    if (page >= a.cache.pages) {
      if (j == 0) set_error(a.err, ERR_BAD_SLOT);
      continue;
    }
    store8((TO*)(is_k ? a.cache.k : a.cache.v) + page * a.cache.page_stride +
               (slot - page * a.cache.page) * a.cache.token_stride + g * a.cache.head_stride + d, x);
  }
}

struct DraftStoreArgs {
  const void *k, *v;      // [rows][heads][dim] 16-bit elements, by strides
  int64_t k_ts, k_hs, v_ts, v_hs;
  const int32_t* source;  // [count] row of k and v for each entry, or NULL: row i
  const int32_t* slots;   // [count]; < 0: not kept
  int count, rows, heads, dim;
  PageCache cache;
  int* err;
};

constexpr int DS_THREADS = 256;

// One thread block an entry: its K and V rows in 16-byte pieces.
__global__ void __launch_bounds__(DS_THREADS) draft_store_kernel(const DraftStoreArgs a) {
  const int i = blockIdx.x;
  const int slot = a.slots[i], page = slot / a.cache.page;
  const int src = a.source ? a.source[i] : i;
  if (slot < 0) return;
  if (page >= a.cache.pages || src < 0 || src >= a.rows) {
    if (threadIdx.x == 0) set_error(a.err, ERR_BAD_SLOT);
    return;
  }
  const int64_t to = page * a.cache.page_stride + (slot - page * a.cache.page) * a.cache.token_stride;
  const int per = a.dim / 8, n = a.heads * per;
  for (int c = threadIdx.x; c < 2 * n; c += DS_THREADS) {
    const bool is_v = c >= n;
    const int h = (is_v ? c - n : c) / per, d = (c % per) * 8;
    const uint16_t* from = (const uint16_t*)(is_v ? a.v : a.k) + (int64_t)src * (is_v ? a.v_ts : a.k_ts) +
                           h * (is_v ? a.v_hs : a.k_hs) + d;
    *reinterpret_cast<uint4*>((uint16_t*)(is_v ? a.cache.v : a.cache.k) + to + h * a.cache.head_stride + d) =
        *reinterpret_cast<const uint4*>(from);
  }
}

}  // namespace hsg
