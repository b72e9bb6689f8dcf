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
//
// Measured on B200: 37,500 tokens of 20 prompts, 32 / 8 heads of 128: 845 MB in 193 to 202 us, 4.3 TB/s (queries alone 5.1: of keys
// and values the instructions count, 90 a row of 128 for both passes); 1,320 tokens of 352 requests: 18 us, a run's chain of waits
// (slots, rows, old scales, rows again) in the blocks that find room at once; one token: 5.3 us. The same 352 requests' entries in a
// list of 8,192: 78 us, of 37,500: 79 (with queries 98 and 131), since a thread block takes 32 entries of a long list and their runs one
// after the other.
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
constexpr int A8R_LIVE = 4;       // 16-byte pieces a lane has under way
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
// Eight values times `by`; infinities may be among them if `checked`.
__device__ __forceinline__ uint2 f8_eight(const float (&x)[8], float by, bool checked) {
  if (checked)
    return make_uint2(f8_pair(x[0] * by, x[1] * by) | f8_pair(x[2] * by, x[3] * by) << 16,
                      f8_pair(x[4] * by, x[5] * by) | f8_pair(x[6] * by, x[7] * by) << 16);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i] * by, x[2 * i + 1] * by), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}
__device__ __forceinline__ float2 f8_values(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return __half22float2(__half2(h));
}

// Eight 16-bit numbers as fp32.
template <typename T> __device__ __forceinline__ void unpack8(const uint4& r, float (&x)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value) {
      const float2 f = unpack_half2(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// How a lane turns the eight elements from d on of a row that dim / 8 lanes share: the other element of a pair is among its own
// eight (pairs) or rot / 16 lanes away. A lane keeps the angles of its row while it goes through the row's heads: read from shared
// memory for every head they took 64 bytes for 16 of data, at a fourth of the banks' rate (37,500 tokens of 40 heads 326 and
// 264 us, before the other steps).
//
// A frequency is the 64-bit fraction of a turn that one position adds, made once a block in fp64 (2^-53 of itself); a position
// times it, modulo 2^64, is where the position stands within the turn, whatever its size. The 32 upper bits of that go to fp32
// and sincospif: the angle is off by less than 2e-7.
struct A8Turn {
  int half, d, partner;
  bool in_rot, first_half, pairs;
  float2 cs[8];  // (cos, sin) times rope_scale of the lane's elements; pairs: the first four, of its pairs
  __device__ __forceinline__ A8Turn(const Append8Args& a, int lane, int dim)
      : half(a.rot / 2), d(lane % (dim / 8) * 8), in_rot(d < a.rot), first_half(d < half), pairs(a.pairs) {
    partner = in_rot && !pairs ? (first_half ? lane + half / 8 : lane - half / 8) : lane;
  }
  __device__ __forceinline__ void at(const Append8Args& a, int position, const uint64_t* steps) {
    if (!in_rot) return;
    const uint64_t* mine = steps + (pairs ? d / 2 : first_half ? d : d - half);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= 4 && pairs) break;
      const int within = (int)((uint64_t)((int64_t)position * (int64_t)mine[e]) >> 32);
      float s, c;
      sincospif((float)within * 4.6566128730773926e-10f, &s, &c);  // half turns: 2^-31
      cs[e] = make_float2(c * a.rope_scale, (first_half || pairs ? s : -s) * a.rope_scale);
    }
  }
  // every lane of the warp calls both
  __device__ __forceinline__ uint4 others(const uint4& raw) const {
    if (pairs) return raw;
    return make_uint4(__shfl_sync(0xffffffffu, raw.x, partner), __shfl_sync(0xffffffffu, raw.y, partner),
                      __shfl_sync(0xffffffffu, raw.z, partner), __shfl_sync(0xffffffffu, raw.w, partner));
  }
  template <typename T> __device__ __forceinline__ void apply(const uint4& raw, bool turn, float (&x)[8]) const {
    unpack8<T>(raw, x);
    if (!turn || !half) return;
    if (pairs) {
      if (!in_rot) return;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float p = x[e], q = x[e + 1];
        x[e] = fmaf(-q, cs[e / 2].y, p * cs[e / 2].x);
        x[e + 1] = fmaf(p, cs[e / 2].y, q * cs[e / 2].x);
      }
      return;
    }
    float y[8];
    unpack8<T>(others(raw), y);
    if (!in_rot) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(-y[e], cs[e].y, x[e] * cs[e].x);
  }
  // what the eight elements ask of the scale but for |rope_scale|: pairs that turn count with the sum of their magnitudes, at most
  // fp32's largest number. Without NaN; infinite if one is or such a sum is, unless `finite` leaves infinite elements out
  template <typename T, bool finite> __device__ __forceinline__ float bound(const uint4& raw, bool turns) const {
    float x[8], y[8], most = 0.f;
    unpack8<T>(raw, x);
    if (turns && half) unpack8<T>(others(raw), y);
    const bool both = turns && in_rot;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = fabsf(x[e]), q = both ? fabsf(y[pairs ? e ^ 1 : e]) : 0.f, z = p + q;
      most = fmaxf(most, !finite ? z : p < INFINITY && q < INFINITY ? fminf(z, 0x1.fffffep127f) : 0.f);
    }
    return most;
  }
};

__device__ __forceinline__ void append8_steps(const Append8Args& a, uint64_t* steps) {
  for (int e = threadIdx.x; e < a.rot / 2; e += A8R_THREADS) {
    const double turns = (double)a.inv_freq[e] * 0.15915494309189533577;
    steps[e] = (uint64_t)__double2ll_rn((turns - rint(turns)) * 9223372036854775808.0) << 1;
  }
}

// Queries: `tokens` entries from the first-th on. A warp takes as many tokens as it has rows of lanes; `split` warps share those
// tokens' heads, of which A8R_LIVE are under way at a time.
template <int D, typename T>
__device__ __forceinline__ void append8_queries(const Append8Args& a, int first, int tokens, int split, const uint64_t* steps) {
  constexpr int LPR = D / 8, RPW = 32 / LPR;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = warp / split * RPW + lane / LPR, i = first + t;
  A8Turn turn(a, lane, D);
  if (__all_sync(0xffffffffu, t >= tokens)) return;
  const bool mine = t < tokens;
  const T* src = (const T*)a.q + i * a.q_ts + turn.d;
  uint4 raw[A8R_LIVE];
  auto load = [&](int h0) {
#pragma unroll
    for (int u = 0; u < A8R_LIVE; ++u) {
      raw[u] = make_uint4(0u, 0u, 0u, 0u);
      if (mine && h0 + u * split < a.hq) raw[u] = *reinterpret_cast<const uint4*>(src + (h0 + u * split) * a.q_hs);
    }
  };
  load(warp % split);
  if (mine && a.rot) turn.at(a, a.positions[i], steps);  // while the first heads are on their way
  T* dst = (T*)a.q_out + (int64_t)i * a.hq * D + turn.d;
  for (int h0 = warp % split; h0 < a.hq; h0 += A8R_LIVE * split) {
#pragma unroll
    for (int u = 0; u < A8R_LIVE; ++u) {
      const int h = h0 + u * split, next = h + A8R_LIVE * split;
      float x[8];
      turn.apply<T>(raw[u], true, x);
      if (mine && next < a.hq) raw[u] = *reinterpret_cast<const uint4*>(src + next * a.q_hs);
      if (mine && h < a.hq) store8(dst + h * D, x);
    }
  }
}

// Keys and values, one run of entries at a time: ones whose slots ascend within one block, with entries that are not kept between
// them at most. (In a list that has others between, a block's entries are several runs, one after the other.) Warps take tokens and
// share their heads of K and V like those of queries:
//   1  the heads' bounds, joined in shared memory;
//   2  the block's scales (from the run alone if it holds the block's first token, else at least what they were), rows that were
//      there rounded to a risen scale;
//   3  rows, read again (mostly from L2), turned, scaled and written.
// Returns whether there is such a page; then (odd, last) are in s_odd, for all threads after a barrier.
template <int D, typename T>
__device__ __forceinline__ bool append8_run(const Append8Args& a, int i0, int n, int slot0, const uint64_t* steps, uint32_t* s_units, int odd,
                                            int last, int* s_odd) {
  constexpr int LPR = D / 8, RPW = 32 / LPR, WARPS = A8R_THREADS / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LPR;
  A8Turn turn(a, lane, D);
  const float factor = fabsf(a.rope_scale);
  const Cache8& c = a.cache;
  const int blk = c.block_div.div(slot0), page = blk / c.blocks, inner = blk - page * c.blocks, first = slot0 - blk * c.block;
  if (page >= c.pages) {
    if (threadIdx.x == 0) set_error(a.err, ERR_BAD_SLOT);
    return false;
  }
  const int64_t base = (int64_t)page * c.page_stride + (int64_t)inner * c.block * c.token_stride;
  const int units = 2 * a.hkv, groups = (n + RPW - 1) / RPW;
  const int split = groups >= WARPS ? 1 : WARPS / groups, teams = WARPS / split, team = warp / split, u_first = warp % split;
  for (int u = threadIdx.x; u < 2 * units; u += A8R_THREADS) s_units[u] = 0u;
  __syncthreads();
  if (threadIdx.x < 2) s_odd[threadIdx.x] = threadIdx.x ? last : odd;  // what is read after this run does not take a register through it
  int row = -1, at = 0;  // of K and V, and within the block; -1: not kept or not there
  auto token = [&](int g) {
    const int t = g * RPW + sub, i = i0 + t;
    row = -1;
    if (t < n) {
      const int slot = a.slots[i];
      if (slot >= 0) {
        at = slot - blk * c.block;
        row = a.source ? a.source[i] : i;
        if (row < 0 || row >= a.rows) {
          set_error(a.err, ERR_BAD_SLOT);
          row = -1;
        }
      }
    }
  };
  uint4 raw[A8R_LIVE];
  auto load = [&](int v, int u0) {  // the v-th of the units from u0 on
    const int u = u0 + v * split, h = u < a.hkv ? u : u - a.hkv;
    raw[v] = make_uint4(0u, 0u, 0u, 0u);
    if (row >= 0 && u < units)
      raw[v] = *reinterpret_cast<const uint4*>(u < a.hkv ? (const T*)a.k + row * a.k_ts + h * a.k_hs + turn.d
                                                         : (const T*)a.v + row * a.v_ts + h * a.v_hs + turn.d);
  };
  auto bound_of = [&](int u, float most, bool wild) {  // (times |rope_scale| where the pair turns: rounding keeps the order)
    const float z = u < a.hkv && turn.in_rot ? most * factor : most;
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(z < INFINITY ? z : 0x1.fffffep127f));
    if (lane == 0) {
      atomicMax(&s_units[u], bits);
      if (wild) s_units[units + u] = 1u;
    }
  };
  // bounds: of a few groups of tokens several heads are under way, else several groups of one head
  const bool few = groups <= 2 * teams;
  for (int g = team; few && g < groups && team < teams; g += teams) {
    token(g);
#pragma unroll
    for (int v = 0; v < A8R_LIVE; ++v) load(v, u_first);
    for (int u0 = u_first; u0 < units; u0 += A8R_LIVE * split) {
#pragma unroll
      for (int v = 0; v < A8R_LIVE; ++v) {
        const int u = u0 + v * split;
        if (u >= units) break;
        float most = turn.bound<T, false>(raw[v], u < a.hkv);
        const bool wild = __any_sync(0xffffffffu, most == INFINITY);
        if (wild) most = turn.bound<T, true>(raw[v], u < a.hkv);
        load(v, u0 + A8R_LIVE * split);
        bound_of(u, most, wild);
      }
    }
  }
  for (int g0 = team; !few && g0 < groups && team < teams; g0 += A8R_LIVE * teams) {
    int rows[A8R_LIVE];
#pragma unroll
    for (int v = 0; v < A8R_LIVE; ++v) {
      token(g0 + v * teams);
      rows[v] = row;
    }
    auto fetch = [&](int u, uint4 (&x)[A8R_LIVE]) {
      const int h = u < a.hkv ? u : u - a.hkv;
      const T* src = (u < a.hkv ? (const T*)a.k + h * a.k_hs : (const T*)a.v + h * a.v_hs) + turn.d;
#pragma unroll
      for (int v = 0; v < A8R_LIVE; ++v) {
        x[v] = make_uint4(0u, 0u, 0u, 0u);
        if (rows[v] >= 0 && u < units) x[v] = *reinterpret_cast<const uint4*>(src + rows[v] * (u < a.hkv ? a.k_ts : a.v_ts));
      }
    };
    uint4 ahead[A8R_LIVE];
    fetch(u_first, ahead);
    for (int u = u_first; u < units; u += split) {
#pragma unroll
      for (int v = 0; v < A8R_LIVE; ++v) raw[v] = ahead[v];
      fetch(u + split, ahead);
      float most = 0.f;
#pragma unroll
      for (int v = 0; v < A8R_LIVE; ++v) most = fmaxf(most, turn.bound<T, false>(raw[v], u < a.hkv));
      const bool wild = __any_sync(0xffffffffu, most == INFINITY);
      if (wild) {
        most = 0.f;
#pragma unroll 1
        for (int v = 0; v < A8R_LIVE; ++v) most = fmaxf(most, turn.bound<T, true>(v == 0 ? raw[0] : v == 1 ? raw[1] : v == 2 ? raw[2] : raw[3], u < a.hkv));
      }
      bound_of(u, most, wild);
    }
  }
  __syncthreads();
  for (int u = warp; u < units; u += WARPS) {
    const bool is_k = u < a.hkv;
    const int h = is_k ? u : u - a.hkv;
    float* where = (is_k ? c.ks : c.vs) + ((int64_t)page * c.blocks + inner) * a.hkv + h;
    float scale = scale8_of(__uint_as_float(s_units[u]));
    if (first) {
      const float old = *where;
      scale = fmaxf(scale, old);
      if (scale > old) {  // rows that are there, to the new scale
        const float ratio = old / scale;
        uint8_t* rows = (is_k ? c.k : c.v) + base + h * c.head_stride;
        for (int e = lane; e < first * (D / 16); e += 32) {
          uint4* to = reinterpret_cast<uint4*>(rows + e / (D / 16) * c.token_stride + e % (D / 16) * 16);
          uint4 w = *to;
          uint32_t* x = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float2 lo = f8_values(x[q] & 0xffffu), hi = f8_values(x[q] >> 16);
            x[q] = f8_pair(lo.x * ratio, lo.y * ratio) | f8_pair(hi.x * ratio, hi.y * ratio) << 16;
          }
          *to = w;
        }
      }
    }
    __syncwarp();  // every lane has read the bound and the old scale
    if (lane == 0) {
      *where = scale;
      s_units[u] = __float_as_uint(1.0f / scale);
    }
  }
  __syncthreads();
  if (team < teams) {
    for (int g = team; g < groups; g += teams) {
      token(g);
#pragma unroll
      for (int v = 0; v < A8R_LIVE; ++v) load(v, u_first);
      if (row >= 0 && a.rot) turn.at(a, a.positions[i0 + g * RPW + sub], steps);
      for (int u0 = u_first; u0 < units; u0 += A8R_LIVE * split) {
#pragma unroll
        for (int v = 0; v < A8R_LIVE; ++v) {
          const int u = u0 + v * split, h = u < a.hkv ? u : u - a.hkv;
          if (u >= units) break;
          float x[8];
          turn.apply<T>(raw[v], u < a.hkv, x);
          load(v, u0 + A8R_LIVE * split);
          if (row >= 0)
            *reinterpret_cast<uint2*>((u < a.hkv ? c.k : c.v) + base + at * c.token_stride + h * c.head_stride + turn.d) =
                f8_eight(x, __uint_as_float(s_units[u]), s_units[units + u]);
        }
      }
    }
  }
  return true;
}

// The first entry that is kept from j on (Dir 1; count: none) or from j back (Dir -1; below 0: none). Lists are padded to what a
// captured call has room for. With walks of 32 entries a step, a load's latency each, and made by blocks of padding too, ten tokens in a
// list of 2^17 entries took 3,800 us; 53 with these, 11 unpadded. Called by the whole block.
constexpr int A8R_WALK = 16;  // entries of a thread under way
template <int Dir>
__device__ __noinline__ int append8_kept(const Append8Args& a, int j, int* s_warps) {
  const int none = Dir > 0 ? a.count : -1;
  while (Dir > 0 ? j < a.count : j >= 0) {
    int slots[A8R_WALK], found = Dir > 0 ? INT_MAX : INT_MIN;
#pragma unroll
    for (int u = 0; u < A8R_WALK; ++u) {
      const int at = j + Dir * (u * A8R_THREADS + (int)threadIdx.x);
      slots[u] = (Dir > 0 ? at < a.count : at >= 0) ? a.slots[at] : -1;
    }
#pragma unroll
    for (int u = A8R_WALK - 1; u >= 0; --u)
      if (slots[u] >= 0) found = j + Dir * (u * A8R_THREADS + (int)threadIdx.x);
    found = Dir > 0 ? __reduce_min_sync(0xffffffffu, found) : __reduce_max_sync(0xffffffffu, found);
    __syncthreads();  // the last ones have been read
    if ((threadIdx.x & 31) == 0) s_warps[threadIdx.x >> 5] = found;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < A8R_THREADS / 32; ++w) found = Dir > 0 ? min(found, s_warps[w]) : max(found, s_warps[w]);
    if (found != (Dir > 0 ? INT_MAX : INT_MIN)) return found;
    j += Dir * A8R_WALK * A8R_THREADS;
  }
  return none;
}

// From entry j on, the next of last's block whose slot is above `last`, before any of another block; -1: none. Called by the whole block.
__device__ __noinline__ int append8_above(const Append8Args& a, int j, int last, int* s_warps) {
  const int lane = threadIdx.x & 31, blk = a.cache.block_div.div(last);
  for (; j < a.count; j = append8_kept<1>(a, j + 32, s_warps)) {
    const int s = j + lane < a.count ? a.slots[j + lane] : -1;
    const bool other = s < blk * a.cache.block || s - blk * a.cache.block >= a.cache.block;
    const unsigned hit = __ballot_sync(0xffffffffu, s >= 0 && (other || s > last));
    if (hit) return __shfl_sync(0xffffffffu, (int)other, __ffs(hit) - 1) ? -1 : j + __ffs(hit) - 1;
  }
  return -1;
}

// Blocks 0 .. kv_blocks - 1 take `per` entries each, of which they write the runs that begin there; the others queries, whose heads
// `split` warps share. (Queries first, or both spread among each other, took 1.2 times as long.)
template <int D, typename T>
__global__ void __launch_bounds__(A8R_THREADS, 3) append8_kernel(const __grid_constant__ Append8Args a, int kv_blocks, int per, int split) {
  __shared__ uint64_t s_steps[128];      // [rot / 2]
  __shared__ int s_odd[2], s_warps[A8R_THREADS / 32];
  extern __shared__ uint32_t s_units[];  // [2 hkv] bounds, then inverse scales; [2 hkv] whether infinities are among the rows
  pdl_wait();
  pdl_trigger();
  const int kv = min((int)blockIdx.x, kv_blocks);
  if ((int)blockIdx.x >= kv_blocks) {
    append8_steps(a, s_steps);
    __syncthreads();
    const int per_q = A8R_THREADS / 32 / split * (256 / D), first = (blockIdx.x - kv) * per_q;
    append8_queries<D, T>(a, first, min(per_q, a.count - first), split, s_steps);
    return;
  }
  const Cache8& c = a.cache;
  const int lane = threadIdx.x & 31, begin = kv * per;
  // lane l has entry begin + l, and of the entries before them the l-th
  const int slot = lane < per && begin + lane < a.count ? a.slots[begin + lane] : -1;
  const int ahead = begin - 1 - lane >= 0 ? a.slots[begin - 1 - lane] : -1;
  const unsigned own = __ballot_sync(0xffffffffu, slot >= 0);
  if (!own) return;  // padding, say: what is before it does not matter
  // the kept entry before each
  int before = -1;
  {
    const unsigned kept = __ballot_sync(0xffffffffu, ahead >= 0);
    if (kept) {
      before = __shfl_sync(0xffffffffu, ahead, __ffs(kept) - 1);
    } else if (begin > 32) {
      const int at = append8_kept<-1>(a, begin - 33, s_warps);
      if (at >= 0) before = a.slots[at];
    }
    const unsigned below = own & ((1u << lane) - 1u);
    const int prev = __shfl_sync(0xffffffffu, slot, below ? 31 - __clz(below) : 0);
    if (below) before = prev;
  }
  const bool joined = slot >= 0 && before >= 0 && c.block_div.div(slot) == c.block_div.div(before);
  if (joined && slot <= before && threadIdx.x < 32) set_error(a.err, ERR_BAD_SLOT);
  // a block's entries are its first one's
  unsigned leaders = __ballot_sync(0xffffffffu, slot >= 0 && !joined);
  if (!leaders) return;
  append8_steps(a, s_steps);
  for (; leaders; leaders &= leaders - 1) {
    const int l = __ffs(leaders) - 1;
    int i = begin + l, slot0 = __shfl_sync(0xffffffffu, slot, l);
    do {
      const int blk = c.block_div.div(slot0);
      auto in_block = [&](int s) { return s >= blk * c.block && s - blk * c.block < c.block; };
      // the run's end: its slots ascend, so it holds at most a block of entries that are kept
      int n = 1, last = slot0, odd = -1;  // odd: where an entry of the block comes next that does not ascend
      int next = i + 1 + lane < a.count ? a.slots[i + 1 + lane] : -1;
      for (int j0 = i + 1; j0 < a.count && last - blk * c.block != c.block - 1;) {
        const int s = next;
        const unsigned kept = __ballot_sync(0xffffffffu, s >= 0), below = kept & ((1u << lane) - 1u);
        const int prev = __shfl_sync(0xffffffffu, s, below ? 31 - __clz(below) : 0);
        const unsigned stop = __ballot_sync(0xffffffffu, s >= 0 && !(in_block(s) && s > (below ? prev : last)));
        const unsigned in = kept & (stop ? (stop & -stop) - 1u : ~0u);
        const int top = in ? 31 - __clz(in) : 0, newest = __shfl_sync(0xffffffffu, s, top);
        if (in) {
          n = j0 + top + 1 - i;
          last = newest;
        }
        if (stop) {
          if (in_block(__shfl_sync(0xffffffffu, s, __ffs(stop) - 1))) odd = j0 + __ffs(stop) - 1;
          break;
        }
        j0 = kept ? j0 + 32 : append8_kept<1>(a, j0 + 32, s_warps);
        next = j0 + lane < a.count ? a.slots[j0 + lane] : -1;
      }
      if (!append8_run<D, T>(a, i, n, slot0, s_steps, s_units, odd, last, s_odd)) break;
      __syncthreads();  // shared memory is free for the next run, and what this one wrote is there
      i = s_odd[0];
      if (i >= 0) {
        i = append8_above(a, i, s_odd[1], s_warps);
        if (i >= 0) slot0 = a.slots[i];
      }
    } while (i >= 0);
  }
}

}  // namespace hsg
