// Attention of a request's newest tokens over its pages of a cache in 8 bits (e4m3 codes, a scale for each block of tokens and
// key head).
//
// Request b has len_b tokens in its pages, the last n_b = cu_b+1 - cu_b of which are the queries' own. Token t of them, at
// position p_t (len_b - n_b + t unless positions are given), sees
//   token j < len_b - n_b       iff j > p_t - window or j < sinks (every j without a window)
//   token len_b - n_b + u       iff bit u of its mask is set (without a mask: u <= t), and likewise for position p_u
// and its output is sum_j softmax_j(scale ks_j q.k_j) vs_j v_j over what it sees, its log-sum-exp that of the same scores.
// A token that sees nothing has output 0 and log-sum-exp -inf. What is not seen is never part of a result, whatever its codes
// and scales are.
#pragma once
#include "cache8_rows.cuh"
#include "draft_attn.cuh"  // pack2, ex2_approx

namespace hsg {

struct Attn8Args {
  const void* q;             // [tokens][hq][dim] by strides (elements)
  int64_t q_ts, q_hs;
  Cache8 cache;
  const int32_t* table;      // [rows][width], rows table_stride apart
  int64_t table_stride;
  const int32_t* lens;       // [rows]
  const int32_t* cu;         // [rows + 1]
  const int32_t* positions;  // [tokens] or NULL (read only with a window)
  const uint32_t* mask;      // [tokens][words] or NULL: the chain
  int rows, width, tokens, words, max_new, hq, hkv, window, sinks;
  float scale;
  void* out;                 // [tokens][hq][dim]
  float* lse;                // [tokens][hq] or NULL
  int* err;
};

// This kernel is for few rows a key head, where reading the cache is all that counts; products are warp-level (16 rows by 8
// keys by 16 dims), since the 128 rows of a tcgen05 product would be padding. A request's rows of a key head, row r = (token
// r / G, query head r % G), in blocks of 16, and the 128-key tiles that such a block can see are an item; all items are one
// line that is cut into equal pieces, one a thread block, as the 16-bit attention does. Warp w of a block takes keys
// 16 w .. 16 w + 15 of each tile of its piece: it copies them into its own ring of stages (cp.async, 16 bytes a lane; keys
// outside what the item can see are filled with zeros and not read), and keeps its own running maximum, sums and
// accumulators, so warps meet only at an item's end.
//
// Codes become fp16 exactly in registers. Queries are fp16 as well: an fp16 q as it is, a bf16 q times a power of two for
// each row that brings its largest element to 2^14 (what then falls below fp16's range is under 2^-38 of it). A V scale would
// multiply the weight; it enters the weight's exponent instead, w_j = 2^(s_j + log2 vs_j - m) with m the running maximum of
// that sum, so that weights use fp16's range however the scales differ, and the row sum takes w_j / vs_j. Weights are rounded to
// fp16 (2^-11, the largest between 2^11 and 2^15, as in the 16-bit attention); sums, maxima and accumulators are fp32.
//
// The order of dims within a product is free as long as both factors agree: a lane reads 16 consecutive bytes of a key, which
// are its elements of four steps of 16 dims, and for P V consecutive dims of two keys, interleaved bytewise.
constexpr int A8_THREADS = 256;
constexpr int A8_WARPS = 8;
constexpr int A8_ROWS = 16;
constexpr int A8_TILE = 128;        // keys: 16 a warp
constexpr int A8_PIECES = 148;      // one thread block an SM
constexpr int A8_COST = 2;          // what an item costs besides its tiles, in tiles
constexpr int A8_RING = 24576;      // bytes of a warp's ring
constexpr float A8_LIFT = 11.f, A8_SLACK = 4.f;

__host__ __device__ constexpr int a8_stage(int dim) { return 2 * 16 * dim; }
__host__ __device__ constexpr int a8_stages(int dim) { return A8_RING / a8_stage(dim); }
// rings, scales, query fragments, accumulators, maxima and sums
__host__ __device__ constexpr int a8_smem(int dim) {
  return A8_WARPS * (A8_RING + a8_stages(dim) * 16) + A8_ROWS * dim * 2 + A8_ROWS * dim * 4 + 4096;
}
__host__ __device__ constexpr size_t a8_partial_floats(int dim, int rows = A8_ROWS) { return (size_t)rows * (dim + 2); }
struct A8Split {  // an item that begins in a piece and ends in a later one
  int b, h, block, last;
  int first_slot;
  int pad[3];
};
__host__ __device__ constexpr size_t a8_workspace_bytes(int dim, int rows) {
  return A8_PIECES * sizeof(A8Split) + 2 * A8_PIECES * a8_partial_floats(dim, rows) * sizeof(float);
}

// A request, its rows in blocks of ROWS; n = 0 if its lengths are out of range.
struct A8Req {
  int len, t0, n, blocks;
};
template <int ROWS>
__device__ __forceinline__ A8Req a8_request(const Attn8Args& a, int G, int b, bool report) {
  A8Req r;
  r.len = a.lens[b];
  r.t0 = a.cu[b];
  const int t1 = a.cu[b + 1];
  r.n = t1 - r.t0;
  if (r.len < 0 || r.len > (int64_t)a.width * a.cache.page || r.t0 < 0 || t1 < r.t0 || t1 > a.tokens || r.n > a.max_new ||
      r.n > r.len) {
    if (report) set_error(a.err, ERR_BAD_LEN);
    r.n = 0;
  }
  r.blocks = (int)(((int64_t)r.n * G + ROWS - 1) / ROWS);
  return r;
}

// What a block of rows can see, in tiles of TILE keys: tokens [0, ahead) and [lo, hi), in tiles [0, lead) and [first, first + n - lead).
struct A8Span {
  int ahead, lo, hi, lead, first, n;
};
template <int ROWS, int TILE>
__device__ __forceinline__ A8Span a8_span(const Attn8Args& a, const A8Req& r, int G, int block) {
  A8Span s;
  const int old = r.len - r.n;
  const int t_lo = block * ROWS / G, t_hi = min(r.n - 1, (block * ROWS + ROWS - 1) / G);
  s.hi = a.mask ? r.len : old + t_hi + 1;
  s.lo = s.ahead = 0;
  if (a.window) {
    s.lo = max(0, old + (a.mask || a.positions ? 0 : t_lo) - a.window + 1);
    s.ahead = min(a.sinks, s.lo);
  }
  s.lead = (s.ahead + TILE - 1) / TILE;
  s.first = max(s.lead, s.lo / TILE);
  s.n = s.lead + max(0, (s.hi - 1) / TILE + 1 - s.first);  // a length may be close to 2^31
  return s;
}

// A place on the line of tiles: item (request, key head, block of rows) and tile.
struct A8At {
  int b, h, block, i;
};
template <int ROWS, int TILE>
struct A8Walk {
  A8At at;
  A8Req r;
  A8Span s;
  __device__ __forceinline__ void start(const Attn8Args& a, int G, const A8At& from) {
    at = from;
    r = a8_request<ROWS>(a, G, at.b, false);
    s = a8_span<ROWS, TILE>(a, r, G, at.block);
  }
  __device__ __forceinline__ void next_item(const Attn8Args& a, int G) {
    at.i = 0;
    if (++at.block >= r.blocks) {
      at.block = 0;
      if (++at.h >= a.hkv) {
        at.h = 0;
        do {
          if (++at.b >= a.rows) {
            r.n = 0;
            s.n = 0;
            return;
          }
          r = a8_request<ROWS>(a, G, at.b, false);
        } while (r.n == 0);
      }
    }
    s = a8_span<ROWS, TILE>(a, r, G, at.block);
  }
  __device__ __forceinline__ int base(int tile) const { return (tile < s.lead ? tile : s.first + tile - s.lead) * TILE; }
};

// Where a thread block's piece of the line begins: item and tile (`from`), where that item begins on the line (`begin`), where the
// piece ends (w1) and how long pieces are (step). An item is its tiles and `cost` more; a piece holds at least one tile. Every
// thread of the block calls it, with room for THREADS / 32 + 3 numbers; false: nothing is left for this piece.
template <int ROWS, int TILE, int THREADS>
__device__ __forceinline__ bool a8_piece(const Attn8Args& a, int G, int cost, int piece, int64_t* room, A8At& from, int64_t& begin,
                                         int64_t& w1, int64_t& step) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = (a.rows + THREADS - 1) / THREADS, rb0 = min(a.rows, tid * per), rb1 = min(a.rows, rb0 + per);
  auto units_of = [&](const A8Req& r) {  // of one key head
    int64_t u = 0;
    for (int k = 0; k < r.blocks; ++k) u += a8_span<ROWS, TILE>(a, r, G, k).n + cost;
    return u;
  };
  int64_t mine = 0;
  for (int b = rb0; b < rb1; ++b) mine += units_of(a8_request<ROWS>(a, G, b, piece == 0)) * a.hkv;
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  if (lane == 31) room[warp] = upto;
  __syncthreads();
  int64_t before = upto - mine, units = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += room[w];
    units += room[w];
  }
  step = max((int64_t)(cost + 1), (units + A8_PIECES - 1) / A8_PIECES);
  const int64_t w0 = min(units, piece * step);
  w1 = min(units, w0 + step);
  if (w0 >= w1) return false;
  int64_t* found = room + THREADS / 32;
  A8At* at_found = reinterpret_cast<A8At*>(found + 1);
  if (w0 >= before && w0 < before + mine) {
    int64_t at = before;
    for (int b = rb0; b < rb1; ++b) {
      const A8Req r = a8_request<ROWS>(a, G, b, false);
      const int64_t one = units_of(r), all = one * a.hkv;
      if (w0 >= at && w0 < at + all) {
        const int h = (int)((w0 - at) / one);
        int64_t u = at + h * one;
        for (int k = 0; k < r.blocks; ++k) {
          const int n = a8_span<ROWS, TILE>(a, r, G, k).n + cost;
          if (w0 < u + n) {
            *at_found = A8At{b, h, k, (int)max((int64_t)0, w0 - u - cost)};
            *found = u;
            break;
          }
          u += n;
        }
        break;
      }
      at += all;
    }
  }
  __syncthreads();
  from = *at_found;
  begin = *found;
  return true;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Byte offset of 16-byte piece ch of key k of a warp's 16 keys, so that neither way of reading meets a bank twice: K by
// (key n, piece c) for eight n and four c, V by (keys 2 c, dims of piece x) for four c and two or four x at a time.
template <int D> __device__ __forceinline__ uint32_t a8_k_at(int k, int ch) {
  return k * D + ((D == 64 ? ch : ch ^ ((k & 1) << 2)) << 4);
}
template <int D> __device__ __forceinline__ uint32_t a8_v_at(int k, int ch) {
  if constexpr (D == 64) return (k >> 1) * 128 + ((((k & 1) << 2 | ch) ^ ((k >> 1 & 3) << 1)) << 4);
  else if constexpr (D == 128) return k * 128 + ((ch ^ (k & 6)) << 4);
  else return k * 256 + ((ch ^ ((k >> 1 & 1) | (k & 4))) << 4);
}

// Four codes as fp16, two pairs.
__device__ __forceinline__ uint32_t f8_half2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What brings a row whose largest element is `most` to [2^14, 2^15), and back. A row of zeros, or of values below 2^-100, stays.
__device__ __forceinline__ void a8_row_scale(float most, float& up, float& back) {
  const int e = (__float_as_int(most) >> 23) - 127, by = e < -100 ? 0 : min(14 - e, 100);
  up = __int_as_float((by + 127) << 23);
  back = __int_as_float((127 - by) << 23);
}

template <typename T> __device__ __forceinline__ void mma16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  mma_f16_16816(d, a.x, a.y, a.z, a.w, b0, b1);
}

// Whether row token t (index among the request's new ones, at position p) sees token j.
__device__ __forceinline__ bool a8_sees(const Attn8Args& a, const A8Req& r, int t, int p, int j) {
  if (j >= r.len || t >= r.n) return false;
  const int u = j - (r.len - r.n);
  int at = j;
  if (u >= 0) {
    if (a.mask) {
      if (u >= 32 * a.words || !(a.mask[(int64_t)(r.t0 + t) * a.words + (u >> 5)] >> (u & 31) & 1)) return false;
    } else if (u > t) {
      return false;
    }
    if (a.window && a.positions) at = a.positions[r.t0 + u];
  }
  return !a.window || at > p - a.window || at < a.sinks;
}

template <int D, typename T>
__global__ void __launch_bounds__(A8_THREADS, 1)
attn8_kernel(const __grid_constant__ Attn8Args a, A8Split* splits, float* partials) {
  constexpr int STAGE = a8_stage(D), ST = a8_stages(D), STEPS = D / 16, NT = D / 8;
  extern __shared__ __align__(128) uint8_t a8_smem_raw[];
  uint8_t* rings = a8_smem_raw;                                        // [warps][ST][K 16 x D, V 16 x D]
  float* ring_scales = reinterpret_cast<float*>(rings + A8_WARPS * A8_RING);  // [warps][ST][ks 2, vs 2]
  uint4* s_q = reinterpret_cast<uint4*>(ring_scales + A8_WARPS * ST * 4);     // [steps][32 lanes] fragments of 16 rows
  float* s_o = reinterpret_cast<float*>(s_q + STEPS * 32);              // [16][D]
  float* s_m = s_o + A8_ROWS * D;                                       // [warps][16]
  float* s_l = s_m + A8_WARPS * A8_ROWS;                                // [warps][16]
  float* s_rowscale = s_l + A8_WARPS * A8_ROWS;                         // [16]
  int64_t* s_scan = reinterpret_cast<int64_t*>(s_rowscale + 16);        // a8_piece's

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, piece = blockIdx.x;
  const int G = a.hq / a.hkv, quad = lane & 3, x8 = lane >> 2;
  pdl_wait();
  if (tid == 0) splits[piece].last = -1;

  int64_t begin, w1, step;
  A8At from;
  if (!a8_piece<A8_ROWS, A8_TILE, A8_THREADS>(a, G, A8_COST, piece, s_scan, from, begin, w1, step)) return;  // nobody waits for this block

  // What of an item lies in this piece, from where the item begins on the line: tiles [i0, i1).
  auto part_end = [&](int64_t unit, int n) { return (int)min((int64_t)n, max((int64_t)0, w1 - unit - A8_COST)); };

  // ---- the copying side of a warp: a walk of its own, ahead by ST stages ----
  A8Walk<A8_ROWS, A8_TILE> put;
  put.start(a, G, from);
  int64_t put_unit = begin;
  int put_i = put.at.i, put_i1 = part_end(put_unit, put.s.n);
  bool put_more = true;
  uint8_t* ring = rings + warp * A8_RING;
  float* scales = ring_scales + warp * ST * 4;
  const uint32_t ring_u = smem_u32(ring), scales_u = smem_u32(scales);
  int put_slot = 0;
  int put_base = 0, put_page = -1;  // of the tile to be copied next: this warp's first key; lanes 0 and 1: its groups' pages
  bool put_asked = false;           // (if the item can see one of the group's keys)
  auto settle = [&]() {  // to the next tile that exists, and ask for its pages
    while (put_more && put_i >= put_i1) {
      put_unit += put.s.n + A8_COST;
      if (put_unit + A8_COST >= w1) {  // no tile of the next item lies in this piece
        put_more = false;
        break;
      }
      put.next_item(a, G);
      put_i = 0;
      put_i1 = part_end(put_unit, put.s.n);
    }
    if (!put_more) return;
    put_base = put.base(put_i) + warp * 16;
    put_page = -1;
    const int j = put_base + (lane & 1) * 8;
    put_asked = lane < 2 && j < put.s.hi && (j > put.s.lo - 8 || j < put.s.ahead);
    if (put_asked) put_page = a.table[put.at.b * a.table_stride + a.cache.page_div.div(j)];
  };
  settle();
  auto copy = [&]() {
    if (put_more) {
      const Cache8& c = a.cache;
      int off[2];
      const uint8_t *kb[2], *vb[2];
      bool good[2];
      int pages[2];
      if (put_asked && (put_page < 0 || put_page >= c.pages)) set_error(a.err, ERR_BAD_PAGE);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int page = __shfl_sync(0xffffffffu, put_page, g);
        const int j = put_base + 8 * g;
        pages[g] = page;
        good[g] = page >= 0 && page < c.pages;
        off[g] = j - (int)c.page_div.div(j) * c.page;
        const int64_t at = good[g] ? (int64_t)page * c.page_stride + off[g] * c.token_stride + put.at.h * c.head_stride : 0;
        kb[g] = c.k + at;
        vb[g] = c.v + at;
      }
      const uint32_t dst = ring_u + put_slot * STAGE;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int e = lane + 32 * i, k = e / (D / 16), ch = e % (D / 16), g = k >> 3, j = put_base + k;
        const bool there = good[g] && j < put.s.hi && (j >= put.s.lo || j < put.s.ahead);
        const int64_t o = (k & 7) * c.token_stride + ch * 16;
        cp_async16(dst + a8_k_at<D>(k, ch), there ? kb[g] + o : c.k, there);
        cp_async16(dst + 16 * D + a8_v_at<D>(k, ch), there ? vb[g] + o : c.v, there);
      }
      if (lane < 4) {
        const int g = lane & 1;
        const int page = g ? pages[1] : pages[0], from_row = g ? off[1] : off[0];
        const bool there = g ? good[1] : good[0];
        const float* from = lane < 2 ? c.ks : c.vs;
        const int64_t at = there ? ((int64_t)page * c.blocks + c.block_div.div(from_row)) * a.hkv + put.at.h : 0;
        cp_async4(scales_u + (put_slot * 4 + lane) * 4, from + at, there);
      }
      if (++put_slot == ST) put_slot = 0;
      ++put_i;
      settle();
    }
    cp_async_commit();
  };
#pragma unroll 1
  for (int s = 0; s < ST; ++s) copy();

  // ---- items ----
  A8Walk<A8_ROWS, A8_TILE> get;
  get.start(a, G, from);
  int64_t unit = begin;
  int slot = 0;
  const float to_log2 = a.scale * 1.4426950408889634f;
  for (int item = 0;; ++item) {
    const int i0 = get.at.i, i1 = part_end(unit, get.s.n);
    const A8Req r = get.r;
    const A8Span sp = get.s;
    const int row0 = get.at.block * A8_ROWS;
    // queries as fragments: step s of a lane takes dims 16 (quad + 4 (s / 4)) + 4 (s % 4) + 0 .. 3 of rows x8 and x8 + 8
    {
      const int row = tid >> 4, sub = tid & 15;  // 16 threads a row, D / 16 dims each
      const int at = row0 + row, t = at / G, g = at - t * G;
      constexpr int N = D / 16;
      float v[N];
      const bool there = t < r.n;
      const T* src = (const T*)a.q + (int64_t)(r.t0 + t) * a.q_ts + (int64_t)(get.at.h * G + g) * a.q_hs + sub * N;
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = there ? (float)src[e] : 0.f;
      float back = 1.f;
      if constexpr (!std::is_same<T, __half>::value) {
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) most = fmaxf(most, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.f);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        float up;
        a8_row_scale(most, up, back);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= up;
      }
      if (sub == 0) s_rowscale[row] = back * to_log2;
      // dims d, d + 1 (d even) are half a register of lane (row % 8) * 4 + c of step s: d = 16 (c + 4 i) + 4 q + 2 hi, s = 4 i + q
      uint32_t* frag = reinterpret_cast<uint32_t*>(s_q);
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const int d = sub * N + e, ch = d >> 4, cq = ch & 3, st = (ch >> 2) * 4 + ((d >> 2) & 3), up = d >> 1 & 1;
        frag[(st * 32 + (row & 7) * 4 + cq) * 4 + up * 2 + (row >> 3)] = pack_half2(v[e], v[e + 1]);
      }
    }
    __syncthreads();
    const int ta = (row0 + x8) / G, tb = (row0 + x8 + 8) / G;
    const float scale_a = s_rowscale[x8], scale_b = s_rowscale[x8 + 8];
    const int old = r.len - r.n;
    int pa = 0, pb = 0;
    if (a.window) {
      pa = ta < r.n ? (a.positions ? a.positions[r.t0 + ta] : old + ta) : 0;
      pb = tb < r.n ? (a.positions ? a.positions[r.t0 + tb] : old + tb) : 0;
    }
    // keys below `sure` and above `low` are seen by every row
    const int sure = a.mask ? old : old + row0 / G + 1;
    int low = -1;
    if (a.window) {
      low = max(ta < r.n ? pa - a.window : -1, tb < r.n ? pb - a.window : -1);
      low = __reduce_max_sync(0xffffffffu, low);
    }
    float o[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
    float ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f;
    for (int i = i0; i < i1; ++i) {
      cp_async_wait<ST - 1>();
      __syncwarp();
      const int base = get.base(i) + warp * 16;
      const bool any = base < sp.hi && (base > sp.lo - 16 || base < sp.ahead);
      if (any) {
        float s[2][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][e] = s[1][e] = 0.f;
#pragma unroll
        for (int i4 = 0; i4 < D / 64; ++i4) {
          uint4 kw[2];
#pragma unroll
          for (int n = 0; n < 2; ++n)
            kw[n] = *reinterpret_cast<const uint4*>(ring + slot * STAGE + a8_k_at<D>(n * 8 + x8, quad + 4 * i4));
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint4 f = s_q[(i4 * 4 + q) * 32 + lane];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const uint32_t w = q == 0 ? kw[n].x : q == 1 ? kw[n].y : q == 2 ? kw[n].z : kw[n].w;
              mma16<T>(s[n], f, f8_half2(w & 0xffffu), f8_half2(w >> 16));
            }
          }
        }
        const float4 sc = *reinterpret_cast<const float4*>(scales + slot * 4);  // ks 0, 1, vs 0, 1
        const float ks[2] = {sc.x, sc.y};
        // a V scale of 0 or beyond what append_8bit writes is taken as the nearest that it would write; NaN stays
        const float vs[2] = {sc.z != sc.z ? sc.z : fminf(fmaxf(sc.z, 0x1p-100f), 0x1p120f),
                             sc.w != sc.w ? sc.w : fminf(fmaxf(sc.w, 0x1p-100f), 0x1p120f)};
        const bool special = base > sure - 16 || (a.window && base <= low);
        uint32_t seen = 0xff;
        if (special) {
          seen = 0;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (a8_sees(a, r, e < 2 ? ta : tb, e < 2 ? pa : pb, base + n * 8 + 2 * quad + (e & 1))) seen |= 1u << (4 * n + e);
        }
        float top_a = -INFINITY, top_b = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float lv = __log2f(vs[n]), fa = scale_a * ks[n], fb = scale_b * ks[n];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[n][e] = fmaf(s[n][e], e < 2 ? fa : fb, lv);
            if (special && !(seen >> (4 * n + e) & 1)) s[n][e] = -INFINITY;
          }
          top_a = fmaxf(top_a, fmaxf(s[n][0], s[n][1]));
          top_b = fmaxf(top_b, fmaxf(s[n][2], s[n][3]));
        }
        // the maximum is raised only when a score exceeds it by 2^A8_SLACK
        if (__any_sync(0xffffffffu, top_a > ma + A8_SLACK || top_b > mb + A8_SLACK)) {
#pragma unroll
          for (int d = 1; d < 4; d <<= 1) {
            top_a = fmaxf(top_a, __shfl_xor_sync(0xffffffffu, top_a, d));
            top_b = fmaxf(top_b, __shfl_xor_sync(0xffffffffu, top_b, d));
          }
          float by_a = 1.f, by_b = 1.f;
          if (top_a > ma + A8_SLACK) {
            by_a = ma == -INFINITY ? 0.f : ex2_approx(ma - top_a);
            ma = top_a;
          }
          if (top_b > mb + A8_SLACK) {
            by_b = mb == -INFINITY ? 0.f : ex2_approx(mb - top_b);
            mb = top_b;
          }
          la *= by_a;
          lb *= by_b;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            o[j][0] *= by_a;
            o[j][1] *= by_a;
            o[j][2] *= by_b;
            o[j][3] *= by_b;
          }
        }
        const float off_a = ma == -INFINITY ? 0.f : A8_LIFT - ma, off_b = mb == -INFINITY ? 0.f : A8_LIFT - mb;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float rv = 1.0f / vs[n];
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = ex2_approx(s[n][e] + (e < 2 ? off_a : off_b));
          // a block that a row sees nothing of must not count by its scale either
          const float wa = s[n][0] + s[n][1], wb = s[n][2] + s[n][3];
          la += !special || (seen >> (4 * n) & 3) ? wa * rv : 0.f;
          lb += !special || (seen >> (4 * n + 2) & 3) ? wb * rv : 0.f;
        }
        const uint4 p = make_uint4(pack_half2(s[0][0], s[0][1]), pack_half2(s[0][2], s[0][3]), pack_half2(s[1][0], s[1][1]),
                                   pack_half2(s[1][2], s[1][3]));
        // O += P V: dims x8 * D / 8 + j of keys 2 quad, 2 quad + 1 and those 8 further on
        constexpr int BYTES = D / 8;  // of a key that a lane reads
        constexpr int WORDS = BYTES / 4;
        uint32_t vw[4][WORDS];
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) {
          const int k = 2 * quad + (k4 & 1) + (k4 >> 1) * 8;
          if constexpr (D == 64) {
            const uint2 y = *reinterpret_cast<const uint2*>(ring + slot * STAGE + 16 * D + a8_v_at<D>(k, x8 >> 1) + (x8 & 1) * 8);
            vw[k4][0] = y.x;
            vw[k4][1] = y.y;
          } else {
#pragma unroll
            for (int e = 0; e < D / 128; ++e) {
              const uint4 y = *reinterpret_cast<const uint4*>(ring + slot * STAGE + 16 * D + a8_v_at<D>(k, x8 * (D / 128) + e));
              vw[k4][4 * e] = y.x;
              vw[k4][4 * e + 1] = y.y;
              vw[k4][4 * e + 2] = y.z;
              vw[k4][4 * e + 3] = y.w;
            }
          }
        }
        bool nan = false;
        if (special) {  // a NaN of V is for the rows that see its key
          uint32_t bad = 0;
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4)
#pragma unroll
            for (int w = 0; w < WORDS; ++w) bad |= ((vw[k4][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
          nan = __any_sync(0xffffffffu, bad != 0);
        }
        if (nan) {
          uint4 see;  // 1 where a row sees a key
          uint32_t* f = reinterpret_cast<uint32_t*>(&see);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = (seen >> (2 * e) & 1 ? 0x3c00u : 0u) | (seen >> (2 * e + 1) & 1 ? 0x3c000000u : 0u);
#pragma unroll
          for (int w = 0; w < WORDS; ++w) {
            uint32_t ind[4];  // 1.0 where a code is NaN, which becomes 0
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4) {
              const uint32_t hit = (((vw[k4][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
              ind[k4] = hit * 0x38u;
              vw[k4][w] &= ~(hit * 0xffu);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t sel = e < 2 ? 0x5140u : 0x7362u;
              const uint32_t b0 = __byte_perm(ind[0], ind[1], sel), b1 = __byte_perm(ind[2], ind[3], sel);
              float hits[4] = {0.f, 0.f, 0.f, 0.f};
              mma16<T>(hits, see, f8_half2(e & 1 ? b0 >> 16 : b0 & 0xffffu), f8_half2(e & 1 ? b1 >> 16 : b1 & 0xffffu));
#pragma unroll
              for (int z = 0; z < 4; ++z)
                if (hits[z] > 0.f) o[4 * w + e][z] = __int_as_float(0x7fffffff);
            }
          }
        }
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
#pragma unroll
          for (int pr = 0; pr < 2; ++pr) {
            const uint32_t sel = pr == 0 ? 0x5140u : 0x7362u;
            const uint32_t b0 = __byte_perm(vw[0][w], vw[1][w], sel), b1 = __byte_perm(vw[2][w], vw[3][w], sel);
            mma16<T>(o[4 * w + 2 * pr], p, f8_half2(b0 & 0xffffu), f8_half2(b1 & 0xffffu));
            mma16<T>(o[4 * w + 2 * pr + 1], p, f8_half2(b0 >> 16), f8_half2(b1 >> 16));
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      copy();
      if (++slot == ST) slot = 0;
    }
    // ---- the item's warps meet ----
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      la += __shfl_xor_sync(0xffffffffu, la, d);
      lb += __shfl_xor_sync(0xffffffffu, lb, d);
    }
    if (quad == 0) {
      s_m[warp * 16 + x8] = ma;
      s_m[warp * 16 + x8 + 8] = mb;
      s_l[warp * 16 + x8] = la;
      s_l[warp * 16 + x8 + 8] = lb;
    }
    __syncthreads();
    float top_a = -INFINITY, top_b = -INFINITY;
#pragma unroll
    for (int w = 0; w < A8_WARPS; ++w) {
      top_a = fmaxf(top_a, s_m[w * 16 + x8]);
      top_b = fmaxf(top_b, s_m[w * 16 + x8 + 8]);
    }
    const float by_a = ma == -INFINITY ? 0.f : ex2_approx(ma - top_a), by_b = mb == -INFINITY ? 0.f : ex2_approx(mb - top_b);
    const bool none_a = ma == -INFINITY && la == 0.f, none_b = mb == -INFINITY && lb == 0.f;  // saw nothing: O may be 0 times junk
    for (int w = 0; w < A8_WARPS; ++w) {
      if (warp == w) {
        // dims 2 quad D / 8 + j and the next D / 8 of row x8 and of row x8 + 8
        float* to = s_o + x8 * D + 2 * quad * (D / 8);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float* at = to + (e >> 1) * 8 * D + (e & 1) * (D / 8);
          const float by = e < 2 ? by_a : by_b;
          const bool none = e < 2 ? none_a : none_b;
#pragma unroll
          for (int j = 0; j < NT; j += 4) {
            float4 y = w ? *reinterpret_cast<float4*>(at + j) : make_float4(0.f, 0.f, 0.f, 0.f);
            if (!none) {
              y.x += o[j][e] * by;
              y.y += o[j + 1][e] * by;
              y.z += o[j + 2][e] * by;
              y.w += o[j + 3][e] * by;
            }
            *reinterpret_cast<float4*>(at + j) = y;
          }
        }
      }
      __syncthreads();
    }
    {
      const int row = tid >> 4, sub = tid & 15, at = row0 + row, t = at / G, g = at - t * G;
      constexpr int N = D / 16;
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < A8_WARPS; ++w) m = fmaxf(m, s_m[w * 16 + row]);
#pragma unroll
      for (int w = 0; w < A8_WARPS; ++w) {
        const float mw = s_m[w * 16 + row], lw = s_l[w * 16 + row];
        l += mw == -INFINITY ? lw : lw * ex2_approx(mw - m);
      }
      const bool whole = i0 == 0 && i1 == sp.n;
      float* part = partials + (size_t)(2 * piece + (item > 0 ? 1 : 0)) * a8_partial_floats(D);
      if (t < r.n) {
        if (whole) {
          const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
          const int64_t orow = (int64_t)(r.t0 + t) * a.hq + get.at.h * G + g;
          T* dst = (T*)a.out + orow * D + sub * N;
#pragma unroll
          for (int e = 0; e < N; e += 2)
            *reinterpret_cast<uint32_t*>(dst + e) = pack2(s_o[row * D + sub * N + e] * inv, s_o[row * D + sub * N + e + 1] * inv, dst);
          if (sub == 0 && a.lse) a.lse[orow] = l > 0.f || l != l ? (m - A8_LIFT + log2f(l)) * 0.6931471805599453f : -INFINITY;
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) part[row * D + sub * N + e] = s_o[row * D + sub * N + e];
          if (sub == 0) *reinterpret_cast<float2*>(part + A8_ROWS * D + 2 * row) = make_float2(m, l);
        }
      }
      if (tid == 0 && i0 == 0 && i1 < sp.n)
        splits[piece] = A8Split{get.at.b, get.at.h, get.at.block, (int)((unit + A8_COST + sp.n - 1) / step),
                                2 * piece + (item > 0 ? 1 : 0), {0, 0, 0}};
    }
    unit += sp.n + A8_COST;
    if (unit + A8_COST >= w1) break;
    get.next_item(a, G);
    __syncthreads();  // queries, maxima and sums are free
  }
  cp_async_wait<0>();
}

// Tokens from .. to - 1 as if they saw nothing, by `count` threads of which this is number `me`.
template <int D, typename T>
__device__ __noinline__ void a8_blank(const Attn8Args& a, int64_t from, int64_t to, int64_t me, int64_t count) {
  constexpr int PER = D / 8;
  for (int64_t i = from * a.hq * PER + me; i < to * a.hq * PER; i += count) reinterpret_cast<uint4*>(a.out)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (a.lse)
    for (int64_t i = from * a.hq + me; i < to * a.hq; i += count) a.lse[i] = -INFINITY;
}

// Joins the parts of an item that was cut, in piece order, a warp a row: block (c, y) takes the item that begins in piece c,
// rows 8 y .. 8 y + 7. And writes the tokens that no item has: those of no request, by all blocks, and those of requests whose
// lengths are out of range.
constexpr int A8J_THREADS = 256;
template <int D, int ROWS, typename T>
__global__ void __launch_bounds__(A8J_THREADS) attn8_join_kernel(const __grid_constant__ Attn8Args a, const A8Split* splits,
                                                                const float* partials) {
  pdl_wait();
  const int c = blockIdx.x, lane = threadIdx.x & 31, G = a.hq / a.hkv;
  const A8Split s = splits[c];
  const int lead = a.cu[0], trail = a.cu[a.rows];
  if (lead > 0 || trail < a.tokens) {
    const int64_t me = ((int64_t)blockIdx.y * A8_PIECES + c) * A8J_THREADS + threadIdx.x,
                  all = (int64_t)gridDim.y * A8_PIECES * A8J_THREADS;
    a8_blank<D, T>(a, 0, min(lead, a.tokens), me, all);
    a8_blank<D, T>(a, max(trail, 0), a.tokens, me, all);
  }
  if (blockIdx.y == 0) {
    for (int b0 = c + A8_PIECES * (threadIdx.x & ~31); b0 < a.rows; b0 += A8_PIECES * A8J_THREADS) {
      const int b = b0 + A8_PIECES * lane;
      const bool out = b < a.rows && a.cu[b + 1] > a.cu[b] && a8_request<ROWS>(a, G, b, false).n == 0;
      for (unsigned rest = __ballot_sync(0xffffffffu, out); rest; rest &= rest - 1) {
        const int r = b0 + A8_PIECES * (__ffs(rest) - 1);
        a8_blank<D, T>(a, max(a.cu[r], 0), min(a.cu[r + 1], a.tokens), lane, 32);
      }
    }
  }
  if (s.last < 0) return;
  const int row = blockIdx.y * (A8J_THREADS / 32) + (threadIdx.x >> 5), at = s.block * ROWS + row, tok = at / G, t0 = a.cu[s.b];
  if (tok >= a.cu[s.b + 1] - t0) return;
  const size_t size = a8_partial_floats(D, ROWS);
  auto part = [&](int p) { return partials + (p == c ? (size_t)s.first_slot : 2 * (size_t)p) * size; };
  float m = -INFINITY;
  for (int p = c + lane; p <= s.last; p += 32) m = fmaxf(m, part(p)[ROWS * D + 2 * row]);
  m = warp_max(m);
  float l = 0.f, o[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) o[e] = 0.f;
  for (int p = c; p <= s.last; ++p) {
    const float* x = part(p);
    const float2 ml = *reinterpret_cast<const float2*>(x + ROWS * D + 2 * row);
    if (ml.x == -INFINITY && ml.y == 0.f) continue;  // saw nothing
    const float w = ml.x == -INFINITY ? 1.f : ex2_approx(ml.x - m);  // -inf with a sum: NaN, which stays
    l += ml.y * w;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) o[e] += w * x[row * D + e * 32 + lane];
  }
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
  const int64_t orow = (int64_t)(t0 + tok) * a.hq + s.h * G + at - tok * G;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) ((T*)a.out)[orow * D + e * 32 + lane] = (T)(o[e] * inv);
  if (lane == 0 && a.lse) a.lse[orow] = l > 0.f || l != l ? (m - A8_LIFT + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace hsg
