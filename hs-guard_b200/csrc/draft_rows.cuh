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

constexpr int DN_THREADS = 128;
constexpr int DN_LIVE = 4;  // tokens a lane has under way

// dim / 8 lanes share a head, eight consecutive elements each, so a warp works on 256 / dim heads at once; the
// rotation's partner (d and d + rot / 2) is rot / 16 lanes away. A block takes `per` tokens: their angles once into
// shared memory, then units of (a warp's heads, DN_LIVE tokens) spread over its warps, so that what depends on the head
// (kind, addresses, weights) is found once for DN_LIVE tokens. Measured at 22,528 tokens of 12 fp32 heads of 256 (415 MB):
// 74 us, 5.6 TB/s, bound by HBM; units of one head and token, whose index is divided by the head count at every step,
// took 110 us (instructions), blocks of 256 threads 81 us at 8 tokens and 86 us at 16 (a last wave partly empty).
template <int D, typename TI, typename TO>
__global__ void __launch_bounds__(DN_THREADS) draft_norm_kernel(const __grid_constant__ DraftNormArgs a, int per) {
  extern __shared__ __align__(16) float2 s_turn[];  // [per][rot / 2] (cos, sin), read two at a time
  constexpr int LPH = D / 8, HPW = 32 / LPH, WARPS = DN_THREADS / 32;
  const int t0 = blockIdx.x * per, tokens = min(per, a.tokens - t0), half = a.rot / 2;
  const int heads = a.hq + 2 * a.hkv, groups = (heads + HPW - 1) / HPW;
  const int units = groups * ((tokens + DN_LIVE - 1) / DN_LIVE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = lane % LPH * 8;
  const bool first = d < half, in_rot = d < a.rot;
  const int partner = in_rot ? (first ? lane + half / 8 : lane - half / 8) : lane, f = first ? d : d - half;
  bool turned = false;  // the angles are there
  for (int unit = warp; unit < units || !turned; unit += WARPS) {
    const int chunk = unit / groups, h = (unit - chunk * groups) * HPW + lane / LPH, c0 = chunk * DN_LIVE;
    const int live = unit < units && h < heads ? min(DN_LIVE, tokens - c0) : 0;
    const bool is_q = h < a.hq, is_k = !is_q && h < a.hq + a.hkv;
    const int g = is_q ? h : is_k ? h - a.hq : h - a.hq - a.hkv;  // index among its kind
    const int64_t ts = is_q ? a.q_ts : is_k ? a.k_ts : a.v_ts;
    const TI* src = (const TI*)(is_q ? a.q : is_k ? a.k : a.v) + (t0 + c0) * ts + g * (is_q ? a.q_hs : is_k ? a.k_hs : a.v_hs) + d;
    float x[DN_LIVE][8];
#pragma unroll
    for (int u = 0; u < DN_LIVE; ++u) {
      if (u < live) {
        load8(src + u * ts, x[u]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[u][i] = 0.f;
      }
    }
    float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    if (live && (is_q || is_k)) load8((is_q ? a.qw : a.kw) + d, w);
    if (!turned) {  // while the first heads are on their way
      for (int i = threadIdx.x; i < tokens * half; i += DN_THREADS) {
        const int t = i / half;
        rotation(a.positions[t0 + t], a.inv_freq[i - t * half], s_turn[i].y, s_turn[i].x);
      }
      __syncthreads();
      turned = true;
    }
#pragma unroll
    for (int u = 0; u < DN_LIVE; ++u) {
      if (__any_sync(0xffffffffu, u < live && (is_q || is_k))) {  // every lane of the warp takes part in the shuffles
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x[u][i] * x[u][i];
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = is_q || is_k ? rsqrtf(ss * (1.0f / D) + a.eps) : 1.f;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[u][i] = x[u][i] * r * w[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[u][i], partner);
        if (in_rot && u < live && (is_q || is_k)) {
          const float4* cs = reinterpret_cast<const float4*>(s_turn + (c0 + u) * half + f);
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const float4 v = cs[i / 2];
            x[u][i] = fmaf(first ? -y[i] : y[i], v.y, x[u][i] * v.x);
            x[u][i + 1] = fmaf(first ? -y[i + 1] : y[i + 1], v.w, x[u][i + 1] * v.z);
          }
        }
      }
      if (u >= live) continue;
      const int64_t tok = t0 + c0 + u;
      if (is_q) {
        store8((TO*)a.q_out + (tok * a.hq + g) * D + d, x[u]);
      } else if (!a.slots) {
        store8((TO*)(is_k ? a.k_out : a.v_out) + (tok * a.hkv + g) * D + d, x[u]);
      } else {
        const int slot = a.slots[tok], page = slot / a.cache.page;
        if (slot < 0) continue;
        if (page >= a.cache.pages) {
          if (d == 0) set_error(a.err, ERR_BAD_SLOT);
          continue;
        }
        store8((TO*)(is_k ? a.cache.k : a.cache.v) + page * a.cache.page_stride +
                   (slot - page * a.cache.page) * a.cache.token_stride + g * a.cache.head_stride + d, x[u]);
      }
    }
  }
}

struct DraftStoreArgs {
  const void *k, *v;      // [rows][heads][dim] 16-bit elements, by strides
  int64_t k_ts, k_hs, v_ts, v_hs;
  const int32_t* source;  // [count] row of k and v for each entry, or NULL: row i
  const int32_t* slots;   // [count]; < 0: not kept
  int count, rows, heads;
  PageCache cache;
  int* err;
};

constexpr int DS_THREADS = 256;
constexpr int DS_LIVE = 8;  // 16-byte pieces a lane has under way

// One warp an entry: its K and V rows in 16-byte pieces, DS_LIVE requested by a lane before the first is written. Bound
// by HBM: 30,000 entries of 2 x 2 KB (246 MB in and out) take 42 us, 5.9 TB/s; one block an entry took 59 us.
template <int D>
__global__ void __launch_bounds__(DS_THREADS) draft_store_kernel(const __grid_constant__ DraftStoreArgs a) {
  constexpr int PER = D / 8;  // pieces a head
  const int i = blockIdx.x * (DS_THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= a.count) return;
  const int slot = a.slots[i], page = slot / a.cache.page;
  const int src = a.source ? a.source[i] : i;
  if (slot < 0) return;
  if (page >= a.cache.pages || src < 0 || src >= a.rows) {
    if (lane == 0) set_error(a.err, ERR_BAD_SLOT);
    return;
  }
  const int64_t to = page * a.cache.page_stride + (slot - page * a.cache.page) * a.cache.token_stride;
  const uint16_t *k = (const uint16_t*)a.k + src * a.k_ts, *v = (const uint16_t*)a.v + src * a.v_ts;
  const int n = a.heads * PER;
  for (int base = lane; base < 2 * n; base += 32 * DS_LIVE) {
    uint4 x[DS_LIVE];
#pragma unroll
    for (int u = 0; u < DS_LIVE; ++u) {
      const int c = base + 32 * u, p = c < n ? c : c - n, h = p / PER, d = p % PER * 8;
      if (c < 2 * n) x[u] = *reinterpret_cast<const uint4*>(c < n ? k + h * a.k_hs + d : v + h * a.v_hs + d);
    }
#pragma unroll
    for (int u = 0; u < DS_LIVE; ++u) {
      const int c = base + 32 * u, p = c < n ? c : c - n, h = p / PER, d = p % PER * 8;
      if (c < 2 * n)
        *reinterpret_cast<uint4*>((uint16_t*)(c < n ? a.cache.k : a.cache.v) + to + h * a.cache.head_stride + d) = x[u];
    }
  }
}

}  // namespace hsg
