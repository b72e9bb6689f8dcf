// Rows of a cache in 8 bits: rotation of queries and keys and the write of keys and values into e4m3 pages
// (append8_kernel).
//
// A block of consecutive tokens of a page and a key head share one scale in K and one in V: the cache stands for
// code * scale. Scales are powers of two. e4m3 has 4 bits of precision over 2^15 of range, so a power of two costs no
// precision against the exact largest / 448, and a block whose scale has to rise when a larger token joins it keeps its
// codes' bits (only what falls below the normal range is rounded again).
//
// The scale that a token asks for must not depend on how its rotation was rounded, or two builds of this kernel would
// differ by a factor of two where the largest value lies at a border. So it is made from |a| + |b| of each rotated pair, an
// upper bound of what any angle makes of it, rounded once and times |rope_scale| rounded once: the same bits everywhere, at
// the cost of at most half a binade of range.
#pragma once
#include <cuda_fp8.h>

#include "draft_rows.cuh"
#include "draft_tables.cuh"  // FastDiv

namespace hsg {

// Pages of e4m3 codes: (page, token, head, d) at page * page_stride + token * token_stride + head * head_stride + d (bytes),
// and scales [pages][page / block][heads].
struct Cache8 {
  uint8_t *k, *v;
  float *ks, *vs;
  int64_t page_stride, token_stride, head_stride;
  int pages, page, block, blocks;  // blocks of a page
  FastDiv page_div, block_div;
};

struct Append8Args {
  const void *q, *k, *v;     // q [count][hq][dim]; k, v [rows][hkv][dim], by strides (elements)
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  const int32_t* source;     // [count] row of k and v, or NULL: i
  const int32_t* slots;      // [count]; < 0: not kept
  const int32_t* positions;  // [count], with a rotation
  const float* inv_freq;     // [rot / 2]
  int count, rows, hq, hkv, rot, pairs;  // pairs: 1: dims (2 i, 2 i + 1) turn together, 0: (i, i + rot / 2)
  float rope_scale;
  void* q_out;               // [count][hq][dim]
  Cache8 cache;
  int* err;
};

constexpr int A8R_THREADS = 256;
constexpr int A8R_CHUNK = 16;     // tokens whose angles lie in shared memory at once
constexpr float F8_MAX = 448.f;
constexpr int SCALE_MIN_EXP = -100, SCALE_MAX_EXP = 120;

// The smallest power of two that brings `bound` to at most 448 = 1.75 * 2^8, from its bits.
__device__ __forceinline__ float scale8_of(float bound) {
  const int bits = __float_as_int(bound);
  int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  e = min(max(e, SCALE_MIN_EXP), SCALE_MAX_EXP);
  return __int_as_float((e + 127) << 23);
}

// Two values as e4m3 codes (round to nearest even); what is not finite becomes NaN.
__device__ __forceinline__ uint32_t f8_pair(float a, float b) {
  a = fabsf(a) < INFINITY ? a : __int_as_float(0x7fffffff);
  b = fabsf(b) < INFINITY ? b : __int_as_float(0x7fffffff);
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 f8_values(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return __half22float2(__half2(h));
}

// One run of entries at a time: ones whose slots ascend within one block, with entries that are not kept between them at most (each
// of which is a run by itself). A block that takes `per` entries does the runs that begin there. Units of a warp are heads:
//   1  keys and values: the run's bound, the block's scale (from the run alone if it holds the block's first token, else at
//      least what it was), rows that were there rounded to a risen scale;
//   2  angles of up to 16 tokens into shared memory, then rows of q, k and v: rotated, scaled, written.
// Rows are read twice, the second time mostly from L1 or L2. dim / 8 lanes share a row, eight elements each.
template <int D, typename T>
__global__ void __launch_bounds__(A8R_THREADS) append8_kernel(const __grid_constant__ Append8Args a, int per) {
  extern __shared__ __align__(16) float2 s_angles[];  // [chunk][rot / 2] (cos, sin) times rope_scale
  constexpr int LPR = D / 8, RPW = 32 / LPR, WARPS = A8R_THREADS / 32;
  float* s_scale = reinterpret_cast<float*>(s_angles + A8R_CHUNK * (a.rot / 2));  // [2 hkv] inverse scales of the run
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = lane % LPR * 8, sub = lane / LPR, half = a.rot / 2;
  const bool in_rot = d < a.rot, first_half = d < half;
  const int partner = in_rot && !a.pairs ? (first_half ? lane + half / 8 : lane - half / 8) : lane;
  const float factor = fabsf(a.rope_scale);
  const Cache8& c = a.cache;
  auto row_of = [&](int i) {  // of k and v; -1: not kept, -2: not there
    if (a.slots[i] < 0) return -1;
    const int r = a.source ? a.source[i] : i;
    return r >= 0 && r < a.rows ? r : -2;
  };
  const int end = min(a.count, (int)(blockIdx.x + 1) * per);
  for (int i0 = blockIdx.x * per; i0 < end; ++i0) {
    const int slot0 = a.slots[i0], blk = slot0 >= 0 ? slot0 / c.block : -1;
    // the kept entry before this one
    int before = -1;
    if (slot0 >= 0) {
      for (int j = i0 - 1 - lane;; j -= 32) {
        const int s = j >= 0 ? a.slots[j] : -1;
        const unsigned kept = __ballot_sync(0xffffffffu, s >= 0);
        if (kept) before = __shfl_sync(0xffffffffu, s, __ffs(kept) - 1);
        if (kept || j + lane - 31 <= 0) break;
      }
    }
    const bool same = before >= 0 && before / c.block == blk;
    if (same && slot0 > before) continue;  // inside a run that began earlier
    // the run's end: its slots ascend, so it holds at most a block of entries that are kept
    int n = 1;
    for (int j0 = i0 + 1, last = slot0; slot0 >= 0 && j0 < a.count && last % c.block != c.block - 1; j0 += 32) {
      const int j = j0 + lane, s = j < a.count ? a.slots[j] : -1;
      const unsigned kept = __ballot_sync(0xffffffffu, s >= 0), below = kept & ((1u << lane) - 1u);
      const int prev = __shfl_sync(0xffffffffu, s, below ? 31 - __clz(below) : 0);
      const bool fits = s < 0 || (s / c.block == blk && s > (below ? prev : last));
      const unsigned stop = __ballot_sync(0xffffffffu, j >= a.count || !fits);
      const unsigned in = kept & (stop ? (stop & -stop) - 1u : ~0u);
      const int top = in ? 31 - __clz(in) : 0, newest = __shfl_sync(0xffffffffu, s, top);
      if (in) {
        n = j0 + top + 1 - i0;
        last = newest;
      }
      if (stop) break;
    }
    const int per_page = c.page / c.block, page = blk >= 0 ? blk / per_page : 0;
    bool keep = slot0 >= 0;
    if (keep && (same || page >= c.pages)) {  // a slot that does not ascend, or no page
      keep = false;
      if (threadIdx.x == 0) set_error(a.err, ERR_BAD_SLOT);
    }
    const int inner = keep ? blk - page * per_page : 0, first = keep ? slot0 - blk * c.block : 0;  // block and row
    const int64_t base = (int64_t)page * c.page_stride + (int64_t)inner * c.block * c.token_stride;
    if (keep) {
      for (int u = warp; u < 2 * a.hkv; u += WARPS) {
        const bool is_k = u < a.hkv;
        const int h = is_k ? u : u - a.hkv;
        const T* src = (const T*)(is_k ? a.k : a.v) + h * (is_k ? a.k_hs : a.v_hs) + d;
        const int64_t ts = is_k ? a.k_ts : a.v_ts;
        float* where = (is_k ? c.ks : c.vs) + ((int64_t)page * per_page + inner) * a.hkv + h;
        const float old = first ? *where : 0.f;
        float bound = 0.f;
#pragma unroll 2
        for (int t = sub; t < n + sub; t += RPW) {  // every lane of a row's lanes takes part in the shuffles
          const int r = t < n ? row_of(i0 + t) : -1;
          float x[8];
          if (r >= 0) {
            load8(src + r * ts, x);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.f;
          }
          if (is_k && half) {
            float y[8];
            if (a.pairs) {
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = x[e ^ 1];
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = __shfl_sync(0xffffffffu, x[e], partner);
            }
            if (in_rot) {
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = (fabsf(x[e]) + fabsf(y[e])) * factor;
            }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) bound = fmaxf(bound, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.f);
        }
        bound = warp_max(bound);
        float scale = scale8_of(bound);
        if (first) scale = fmaxf(scale, old);
        if (first && scale > old) {  // rows that are there, to the new scale
          const float ratio = old / scale;
          uint8_t* rows = (is_k ? c.k : c.v) + base + h * c.head_stride;
          for (int e = lane; e < first * (D / 16); e += 32) {
            uint4* at = reinterpret_cast<uint4*>(rows + e / (D / 16) * c.token_stride + e % (D / 16) * 16);
            uint4 w = *at;
            uint32_t* x = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float2 lo = f8_values(x[q] & 0xffffu), hi = f8_values(x[q] >> 16);
              x[q] = f8_pair(lo.x * ratio, lo.y * ratio) | f8_pair(hi.x * ratio, hi.y * ratio) << 16;
            }
            *at = w;
          }
        }
        if (lane == 0) {
          *where = scale;
          s_scale[u] = 1.0f / scale;
        }
      }
    }
    for (int t0 = 0; t0 < n; t0 += A8R_CHUNK) {
      const int tokens = min(A8R_CHUNK, n - t0);
      __syncthreads();
      for (int e = threadIdx.x; e < tokens * half; e += A8R_THREADS) {
        const int t = e / half;
        float s, co;
        rotation(a.positions[i0 + t0 + t], a.inv_freq[e - t * half], s, co);
        s_angles[e] = make_float2(co * a.rope_scale, s * a.rope_scale);
      }
      __syncthreads();
      for (int u = warp; u < a.hq + (keep ? 2 * a.hkv : 0); u += WARPS) {
        const bool is_q = u < a.hq, is_k = !is_q && u < a.hq + a.hkv;
        const int h = is_q ? u : is_k ? u - a.hq : u - a.hq - a.hkv;
        const T* src = (const T*)(is_q ? a.q : is_k ? a.k : a.v) + h * (is_q ? a.q_hs : is_k ? a.k_hs : a.v_hs) + d;
        const int64_t ts = is_q ? a.q_ts : is_k ? a.k_ts : a.v_ts;
        const float inv = is_q ? 1.f : s_scale[u - a.hq];
#pragma unroll 2
        for (int t = sub; t < tokens + sub; t += RPW) {
          const int i = i0 + t0 + t, r = t >= tokens ? -1 : !is_q ? row_of(i) : a.slots[i] >= 0 || n == 1 ? i : -1;
          float x[8];
          if (r >= 0) {
            load8(src + r * ts, x);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.f;
          }
          if ((is_q || is_k) && half) {
            if (a.pairs) {
              if (in_rot && r >= 0) {
                const float4* cs = reinterpret_cast<const float4*>(s_angles + t * half + d / 2);
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                  const float4 w = cs[e / 4];
                  const float p = x[e], q = x[e + 1], p2 = x[e + 2], q2 = x[e + 3];
                  x[e] = fmaf(-q, w.y, p * w.x);
                  x[e + 1] = fmaf(p, w.y, q * w.x);
                  x[e + 2] = fmaf(-q2, w.w, p2 * w.z);
                  x[e + 3] = fmaf(p2, w.w, q2 * w.z);
                }
              }
            } else {
              float y[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = __shfl_sync(0xffffffffu, x[e], partner);
              if (in_rot && r >= 0) {
                const float4* cs = reinterpret_cast<const float4*>(s_angles + t * half + (first_half ? d : d - half));
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                  const float4 w = cs[e / 2];
                  x[e] = fmaf(first_half ? -y[e] : y[e], w.y, x[e] * w.x);
                  x[e + 1] = fmaf(first_half ? -y[e + 1] : y[e + 1], w.w, x[e + 1] * w.z);
                }
              }
            }
          }
          if (r < 0) {
            if (r == -2 && d == 0) set_error(a.err, ERR_BAD_SLOT);
            continue;
          }
          if (is_q) {
            store8((T*)a.q_out + ((int64_t)i * a.hq + h) * D + d, x);
          } else {
            const int at = a.slots[i] - blk * c.block;
            uint2 w;
            w.x = f8_pair(x[0] * inv, x[1] * inv) | f8_pair(x[2] * inv, x[3] * inv) << 16;
            w.y = f8_pair(x[4] * inv, x[5] * inv) | f8_pair(x[6] * inv, x[7] * inv) << 16;
            *reinterpret_cast<uint2*>((is_k ? c.k : c.v) + base + at * c.token_stride + h * c.head_stride + d) = w;
          }
        }
      }
    }
    __syncthreads();  // shared memory is free for the next run
  }
}

}  // namespace hsg
