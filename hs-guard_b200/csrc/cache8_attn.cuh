// Attention of a request's newest tokens over its pages of a cache in 8 bits (e4m3 codes, a scale for each block of tokens and
// key head).
//
// Request b has len_b tokens in its pages, the last n_b = cu_b+1 - cu_b of which are the queries' own. Token t of them, at
// position p_t (len_b - n_b + t unless positions are given), sees
//   token j < len_b - n_b       iff j > p_t - window or j < sinks (every j without a window)
//   token len_b - n_b + u       iff bit u of its mask is set (without a mask: u <= t), and likewise for position p_u
// and its output is sum_j softmax_j(scale ks_j q.k_j) vs_j v_j over what it sees, its log-sum-exp that of the same scores.
// A token that sees nothing has output 0 and log-sum-exp -inf. What is not seen is never part of a result, whatever its codes
// and scales are. Tokens of a page that the cache does not have (which is recorded) are not seen.
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

// This kernel is for few rows a key head, where reading the cache is all that counts; products are warp-level, since the 128 rows
// of a tcgen05 product would be padding, and have keys or dims as their 16 rows (S^T = K Q^T, O^T = V^T P^T) and 8 queries as
// their columns, so that 8 rows or fewer waste nothing (with queries as the 16 rows it took twice the products, accumulators and
// exponentials: 352 conversations 63 us). A request's rows of a key head, row r = (token
// r / G, query head r % G), in blocks of 8 or 16, and the slices of 32 keys (16 at head dim 256) that such a block can see are an item; all items are one
// line that is cut into equal pieces, one a warp, eight warps an SM (16 for 8 rows of 64 dims), whatever the requests' lengths. Warps do not meet: each has
// its ring of slices, which it fills itself ahead of its use (TMA, one box, or as many as a page's size takes), its own running maximum, sums and accumulators. An item that lies in one piece is written out; of one that is cut, each
// piece leaves its sums in the workspace, and attn8_join_kernel joins them in piece order, so results do not depend on timing.
//
// Codes become fp16 exactly in registers. Queries are fp16 as well: an fp16 q as it is, a bf16 q times a power of two for
// each row that brings its largest element to 2^14 (what then falls below fp16's range is under 2^-38 of it). A V scale would
// multiply the weight; it enters the weight's exponent instead, w_j = 2^(s_j + log2 vs_j - m) with m the running maximum of
// that sum, so that weights use fp16's range however the scales differ, and the row sum takes w_j / vs_j. Weights are rounded to
// fp16 (2^-11, the largest between 2^11 and 2^15, as in the 16-bit attention); sums, maxima and accumulators are fp32.
//
// Measured on B200: 352 requests of one or two tokens, 512-token window and 4 first tokens, 8 / 2 heads of 256: 186 MB in 57 us,
// 3.3 TB/s: 6 us until the first slice is there, HBM at 4 to 5 TB/s, then the last pieces (they end up to 14% after the mean) and 5
// for the join. 4 requests of up to 50,001 tokens, 3 tokens, 32 / 8 heads of 128: 228 MB in 87 to 94 us (with queries as the products'
// 16 rows these 12 rows a key head took 74), 64 requests of up to 2,100 tokens, 16 / 16 heads of 64, pages of 8: 195 MB in 60 us.
// Instructions of few warps bound those (1.3 a clock and SM, waits for results of the ones before): codes to fp16, and at pages of 8 the
// copies, of which each costs a warp about 30. One token: 14 us of latencies.
//
// The order of dims and keys within a product is free as long as both factors agree: a lane reads 16 consecutive bytes of a key,
// which are its elements of four steps of 16 dims, and for P V consecutive dims of two keys, interleaved bytewise. Which keys
// (a8_key) and which dims (a8_piece_of) a lane takes is chosen so that reading the swizzled slices meets no bank twice at head dims
// 128 and 256 (twice at 64, for V).
// Warps of a thread block, each with its own ring. The accumulators of 8 rows of 64 dims leave room for 16 warps of 128 registers: the
// 64 requests above take 59 us, with 8 warps 80. The others need up to 255 registers: with 12 warps of 168, up to 2 KB a thread would
// go to local memory.
__host__ __device__ constexpr int a8_warps(int dim, int nr) { return dim == 64 && nr == 1 ? 16 : 8; }
constexpr int A8_BLOCKS = 148;      // one thread block an SM
constexpr int A8_COST = 2;          // what an item costs besides its slices, in slices
constexpr float A8_LIFT = 11.f, A8_SLACK = 4.f;
constexpr int A8_LOST = -(1 << 30);  // below every key: each slice is looked at key by key

__host__ __device__ constexpr int a8_slice(int dim) { return dim == 256 ? 16 : 32; }  // keys
__host__ __device__ constexpr int a8_stage(int dim) { return 2 * a8_slice(dim) * dim; }
__host__ __device__ constexpr int a8_stages(int dim, int nr) { return dim == 64 ? (nr == 1 ? 3 : 6) : dim == 128 ? 3 : 2; }
// a warp's ring, scales and barriers; where the pieces begin
__host__ __device__ constexpr int a8_smem(int dim, int nr) {
  return 1024 + a8_warps(dim, nr) * a8_stages(dim, nr) * (a8_stage(dim) + 40) + 2048;
}
__host__ __device__ constexpr size_t a8_partial_floats(int dim, int rows) { return (size_t)rows * (dim + 2); }
struct A8Split {  // an item that begins in a piece and ends in a later one
  int b, h, block, last;
  int first_slot;
  int pad[3];
};
// `subs` pieces a thread block, of blocks of `rows` rows
__host__ __device__ constexpr size_t a8_workspace_bytes(int dim, int subs, int rows) {
  return A8_BLOCKS * subs * (sizeof(A8Split) + 2 * a8_partial_floats(dim, rows) * sizeof(float));
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

// Of a block that begins with new token t: tokens below this are seen by all its rows, but for a window. A window that goes by given
// positions may leave any of the new ones out, also ones whose places are behind its end.
__device__ __forceinline__ int a8_sure(const Attn8Args& a, int old, int t) {
  return a.mask || (a.window && a.positions) ? old : old + t + 1;
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

// Quotient of numbers that are not negative; mostly both are short.
__device__ __forceinline__ int64_t a8_div(int64_t x, int64_t y) {
  return ((x | y) >> 32) == 0 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y;
}

// A piece of the line: where it begins (item and tile), where that item begins on the line, and where the piece ends. An item is
// its tiles and `cost` more; a piece holds at least one tile, or nothing (b < 0).
struct A8Lot {
  A8At from;
  int64_t begin, end;
};
// The pieces of a thread block, SUBS of them: piece s * A8_BLOCKS + block. Every thread of the block calls it, with room for
// THREADS / 32 numbers. Returns how long pieces are.
template <int ROWS, int TILE, int THREADS, int SUBS>
__device__ __forceinline__ int64_t a8_lots(const Attn8Args& a, int G, int cost, int block, int64_t* room, A8Lot* lots) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = (a.rows + THREADS - 1) / THREADS, rb0 = min(a.rows, tid * per), rb1 = min(a.rows, rb0 + per);
  auto units_of = [&](const A8Req& r) {  // of one key head
    int64_t u = 0;
    for (int k = 0; k < r.blocks; ++k) u += a8_span<ROWS, TILE>(a, r, G, k).n + cost;
    return u;
  };
  int64_t mine = 0;
  for (int b = rb0; b < rb1; ++b) mine += units_of(a8_request<ROWS>(a, G, b, block == 0)) * a.hkv;
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  if (lane == 31) room[warp] = upto;
  if (tid < SUBS) lots[tid].from.b = -1;
  __syncthreads();
  int64_t before = upto - mine, units = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += room[w];
    units += room[w];
  }
  const int64_t step = max((int64_t)(cost + 1), a8_div(units + SUBS * A8_BLOCKS - 1, SUBS * A8_BLOCKS));
  // the first piece of this block that begins at or after this thread's first unit
  int64_t s0 = before > block * step ? a8_div(a8_div(before + step - 1, step) - block + A8_BLOCKS - 1, A8_BLOCKS) : 0;
  if (mine > 0 && s0 < SUBS && (s0 * A8_BLOCKS + block) * step < before + mine) {
    int64_t at = before;
    for (int b = rb0; b < rb1; ++b) {
      const A8Req r = a8_request<ROWS>(a, G, b, false);
      const int64_t one = units_of(r), all = one * a.hkv;
      for (; s0 < SUBS; ++s0) {
        const int64_t w0 = (s0 * A8_BLOCKS + block) * step;
        if (w0 >= at + all) break;
        const int h = (int)a8_div(w0 - at, one);
        int64_t u = at + h * one;
        for (int k = 0; k < r.blocks; ++k) {
          const int n = a8_span<ROWS, TILE>(a, r, G, k).n + cost;
          if (w0 < u + n) {
            lots[s0] = A8Lot{A8At{b, h, k, (int)max((int64_t)0, w0 - u - cost)}, u, min(units, w0 + step)};
            break;
          }
          u += n;
        }
      }
      at += all;
    }
  }
  __syncthreads();
  return step;
}

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Of the 8 keys of a product, the one that stands in column n; of a key's 16-byte pieces, the one that lane group x takes for P V
// (of each 128 bytes; at head dim 64 the x-th 8 bytes). Swizzled places differ in the bits that pairs of lanes would share.
template <int D> __device__ __forceinline__ int a8_key(int n) { return D == 64 ? n : (n & 1) << 2 | n >> 1; }
__device__ __forceinline__ int a8_piece_of(int x) { return (x & 1) << 2 | x >> 1; }
// Byte offset of 16-byte piece ch of key k in a slice, as TMA writes it: blocks of 128 bytes a key (64 at head dim 64)
template <int D> __device__ __forceinline__ uint32_t a8_at(int k, int ch) {
  if constexpr (D == 64) return sw64_off(k, ch);
  else return (ch >> 3) * (a8_slice(D) * 128) + (k >> 3) * 1024 + sw128_off(k & 7, ch & 7);
}

// V scales are taken within [2^-80, 2^120]. The row sums of weights over them, up to 2^15 each, so stay below 2^128 over 2^31 keys (with
// 2^-100, which blocks of zeros have, the sum over 150,000 keys did not); what codes of smaller scales stand for is below 4e-22 either way.
__device__ __forceinline__ float a8_v_scale(float scale) { return fminf(fmaxf(scale, 0x1p-80f), 0x1p120f); }

// Four codes as fp16: the lower two and the upper two.
__device__ __forceinline__ void f8_halves(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(four));
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What brings a row whose largest element is `most` to [2^14, 2^15), and back. A row of zeros, or of values below 2^-100, stays.
__device__ __forceinline__ void a8_row_scale(float most, float& up, float& back) {
  const int e = (__float_as_int(most) >> 23) - 127, by = e < -100 ? 0 : min(14 - e, 100);
  up = __int_as_float((by + 127) << 23);
  back = __int_as_float((127 - by) << 23);
}

// An 8 x 8 matrix of 16-bit numbers, a row of two numbers a lane, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void mma16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
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

template <int D, int NR, typename T>
__global__ void __launch_bounds__(32 * a8_warps(D, NR), 1)
attn8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Attn8Args a,
             int box, A8Split* splits, float* partials) {
  constexpr int KEYS = a8_slice(D), GROUPS = KEYS / 8, STAGE = a8_stage(D), ST = a8_stages(D, NR), WARPS = a8_warps(D, NR), STEPS = D / 16,
                NT = D / 16, BLOCKS = D == 256 ? 2 : 1, ROWS = 8 * NR;
  extern __shared__ __align__(1024) uint8_t a8_smem_raw[];
  uint8_t* rings = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(a8_smem_raw) + 1023) & ~uintptr_t(1023));  // [warps][ST][K, V]
  float* ring_scales = reinterpret_cast<float*>(rings + WARPS * ST * STAGE);            // [warps][ST][ks, vs]
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring_scales + WARPS * ST * 8);           // [warps][ST] a slice has landed
  A8Lot* lots = reinterpret_cast<A8Lot*>(bars + WARPS * ST);                            // [warps]
  int64_t* scan = reinterpret_cast<int64_t*>(lots + WARPS);
  // [warps][ST] groups of a slice whose page the cache does not have: their place holds what was there before
  uint32_t* lost = reinterpret_cast<uint32_t*>(scan + WARPS) + (threadIdx.x >> 5) * ST;

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int piece = warp * A8_BLOCKS + blockIdx.x, G = a.hq / a.hkv, quad = lane & 3, x8 = lane >> 2;
  if (tid < WARPS * ST) {
    mbar_init(bars + tid, 1);
    fence_barrier_init();
  }
  if (lane < ST) lost[lane] = 0;
  if (tid == 0) {
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  pdl_wait();
  // the join's blocks may come: at once where most of the device is idle, else when this warp's last slice is on its way (352
  // conversations take 61 and 64 us, one 21.5 and 15.5)
  if (gridDim.x < A8_BLOCKS) pdl_trigger();
  if (lane == 0) splits[piece].last = -1;
  const int64_t step = a8_lots<ROWS, KEYS, 32 * WARPS, WARPS>(a, G, A8_COST, blockIdx.x, scan, lots);
  const A8Lot lot = lots[warp];
  if (lot.from.b < 0) return;
  // of an item that begins at `unit` on the line, slices up to this lie in the piece
  auto part_end = [&](int64_t unit, int n) { return (int)min((int64_t)n, max((int64_t)0, lot.end - unit - A8_COST)); };

  // ---- the copying side: a walk of its own, ahead by the ring's stages ----
  A8Walk<ROWS, KEYS> put;
  put.start(a, G, lot.from);
  int64_t put_unit = lot.begin;
  int put_i = put.at.i, put_i1 = part_end(put_unit, put.s.n);
  bool put_more = true, asked = false;
  int sure = 0;  // keys below this, and above `low`, are seen by every row of the item; A8_LOST once a page was not there
  uint8_t* ring = rings + warp * ST * STAGE;
  float* scales = ring_scales + warp * ST * 8;
  uint64_t* full = bars + warp * ST;
  int put_slot = 0, put_base = 0, page = 0, within = 0;  // of the slice to be copied next; lane i < GROUPS: of keys 8 i .. 8 i + 7
  auto settle = [&]() {  // to the next slice that exists, and ask for its pages
    while (put_i >= put_i1) {
      put_unit += put.s.n + A8_COST;
      if (put_unit + A8_COST >= lot.end) {  // no slice of the next item lies in this piece
        put_more = false;
        return;
      }
      put.next_item(a, G);
      put_i = 0;
      put_i1 = part_end(put_unit, put.s.n);
    }
    put_base = put.base(put_i);
    const int j = put_base + lane * 8;
    asked = lane < GROUPS && j < put.s.hi && (j > put.s.lo - 8 || j < put.s.ahead);
    if (asked) {
      const int p = a.cache.page_div.div(j);
      within = j - p * a.cache.page;
      page = a.table[put.at.b * a.table_stride + p];
    }
  };
  settle();
  int issued = 0;
  auto copy = [&]() {
    if (put_more) {
      const Cache8& c = a.cache;
      const bool good = asked && page >= 0 && page < c.pages;
      if (__any_sync(0xffffffffu, asked && !good) || sure == A8_LOST) {
        const unsigned gone = __ballot_sync(0xffffffffu, asked && !good);
        if (lane == 0) lost[put_slot] = gone;
        if (asked && !good) set_error(a.err, ERR_BAD_PAGE);
        sure = A8_LOST;
      }
      // lane i brings the i-th box of K and of V if it has a group that is asked for (a box is of one page), and knows where from
      // by that group's lane
      const unsigned groups = __ballot_sync(0xffffffffu, good);
      const int per = box >> 3, g0 = lane * per;  // groups a box; this lane's box's first
      const unsigned mine = g0 < GROUPS ? groups >> g0 & ((1u << per) - 1u) : 0u;
      const int from = mine ? g0 + __ffs(mine) - 1 : 0;
      const int box_page = __shfl_sync(0xffffffffu, page, from), box_row = __shfl_sync(0xffffffffu, within, from) - 8 * (from - g0);
      const unsigned boxes = __ballot_sync(0xffffffffu, mine != 0);
      if (lane == 0) mbar_arrive_expect_tx(&full[put_slot], __popc(boxes) * box * 2 * D);
      __syncwarp();
      if (mine) {
        uint8_t* dst = ring + put_slot * STAGE + lane * box * (D == 64 ? 64 : 128);
        const int cols = D == 256 && box < KEYS ? 2 : 1;  // a box of fewer keys would pack its blocks of 128 bytes closer
#pragma unroll 1
        for (int e = 0; e < cols; ++e) {
          tma_load_5d(dst + e * (KEYS * 128), &tm_k, 0, box_row, e, put.at.h, box_page, &full[put_slot]);
          tma_load_5d(dst + KEYS * D + e * (KEYS * 128), &tm_v, 0, box_row, e, put.at.h, box_page, &full[put_slot]);
        }
      }
      // the groups' scales: K's by lanes 0 .. GROUPS - 1, V's by lanes 4 ..
      const int g = lane & 3, pg = __shfl_sync(0xffffffffu, page, g), in = __shfl_sync(0xffffffffu, within, g);
      if (lane < 8 && g < GROUPS) {
        const bool there = groups >> g & 1;
        const int64_t at = there ? ((int64_t)pg * c.blocks + c.block_div.div(in)) * a.hkv + put.at.h : 0;
        cp_async4(smem_u32(scales + put_slot * 8 + lane), (lane < 4 ? c.ks : c.vs) + at, there);
      }
      ++issued;
      if (++put_slot == ST) put_slot = 0;
      ++put_i;
      settle();
    }
    cp_async_commit();
  };
#pragma unroll 1
  for (int s = 0; s < ST; ++s) copy();

  // ---- items ----
  A8Walk<ROWS, KEYS> get;
  get.start(a, G, lot.from);
  int64_t unit = lot.begin;
  int slot = 0, taken = 0;
  uint32_t phase = 0;
  bool ok = true;
  const float to_log2 = a.scale * 1.4426950408889634f;
  for (int item = 0;; ++item) {
    const int i0 = get.at.i, i1 = part_end(unit, get.s.n);
    const A8Req r = get.r;
    const A8Span sp = get.s;
    const int row0 = get.at.block * ROWS, old = r.len - r.n;
    // queries as columns: step s takes dims 16 (quad + 4 (s / 4)) + 4 (s % 4) + 0 .. 3 of row x8 of each 8
    uint2 qf[STEPS][NR];
    // what a lane's scores belong to: rows 2 quad and 2 quad + 1 of each 8
    float scale[NR][2];
    int tok[NR][2], pos[NR][2];
    int low = -1;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      const int at = row0 + 8 * nr + x8, t = at / G;
      const T* src = (const T*)a.q + (int64_t)(r.t0 + t) * a.q_ts + (int64_t)(get.at.h * G + at - t * G) * a.q_hs + quad * 16;
      uint32_t w[D / 64][8];
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
        if (t < r.n) {
          lo = reinterpret_cast<const uint4*>(src + 64 * i)[0];
          hi = reinterpret_cast<const uint4*>(src + 64 * i)[1];
        }
        w[i][0] = lo.x; w[i][1] = lo.y; w[i][2] = lo.z; w[i][3] = lo.w;
        w[i][4] = hi.x; w[i][5] = hi.y; w[i][6] = hi.z; w[i][7] = hi.w;
      }
      float back = 1.f;
      if constexpr (!std::is_same<T, __half>::value) {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float x = fabsf(__uint_as_float(w[i][k] << 16)), y = fabsf(__uint_as_float(w[i][k] & 0xffff0000u));
            most = fmaxf(most, fmaxf(x < INFINITY ? x : 0.f, y < INFINITY ? y : 0.f));
          }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
        float up;
        a8_row_scale(most, up, back);
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
          for (int k = 0; k < 8; ++k)
            w[i][k] = pack_half2(__uint_as_float(w[i][k] << 16) * up, __uint_as_float(w[i][k] & 0xffff0000u) * up);
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) qf[s][nr] = make_uint2(w[s / 4][2 * (s % 4)], w[s / 4][2 * (s % 4) + 1]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        scale[nr][e] = to_log2 * __shfl_sync(0xffffffffu, back, (2 * quad + e) * 4);
        tok[nr][e] = (row0 + 8 * nr + 2 * quad + e) / G;
        pos[nr][e] = 0;
        if (a.window && tok[nr][e] < r.n) {
          pos[nr][e] = a.positions ? a.positions[r.t0 + tok[nr][e]] : old + tok[nr][e];
          low = max(low, pos[nr][e] - a.window);
        }
      }
    }
    if (sure != A8_LOST) sure = a8_sure(a, old, row0 / G);
    if (a.window) low = __reduce_max_sync(0xffffffffu, low);
    float o[NT][NR][4], m[NR][2], l[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][nr][e] = 0.f;
      m[nr][0] = m[nr][1] = -INFINITY;
      l[nr][0] = l[nr][1] = 0.f;
    }
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
      cp_async_wait<ST - 1>();
      ok = da_wait(&full[slot], phase, a.err, ERR_TIMEOUT_TMA);
      if (!__all_sync(0xffffffffu, ok)) break;
      __syncwarp();  // the scales that four lanes have waited for
      ++taken;
      const int base = get.base(i);
      const uint8_t* kb = ring + slot * STAGE;
      const uint8_t* vb = kb + KEYS * D;
      // S^T: element e of a lane is key a8_key(x8) (+ 8 from e = 2 on) of 16, row 2 quad + e % 2
      float s[KEYS / 16][NR][4];
#pragma unroll
      for (int kh = 0; kh < KEYS / 16; ++kh)
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[kh][nr][e] = 0.f;
#pragma unroll
      for (int i4 = 0; i4 < D / 64; ++i4) {
#pragma unroll
        for (int kh = 0; kh < KEYS / 16; ++kh) {
          const uint4 k0 = *reinterpret_cast<const uint4*>(kb + a8_at<D>(16 * kh + a8_key<D>(x8), quad + 4 * i4));
          const uint4 k1 = *reinterpret_cast<const uint4*>(kb + a8_at<D>(16 * kh + 8 + a8_key<D>(x8), quad + 4 * i4));
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4 f;
            f8_halves(w0[q], f.x, f.z);
            f8_halves(w1[q], f.y, f.w);
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) mma16(s[kh][nr], f, qf[i4 * 4 + q][nr].x, qf[i4 * 4 + q][nr].y);
          }
        }
      }
      float vs[GROUPS];
#pragma unroll
      for (int n = 0; n < GROUPS; ++n) {
        vs[n] = a8_v_scale(scales[slot * 8 + 4 + n]);
        const float ks = scales[slot * 8 + n], lv = __log2f(vs[n]);
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int e = 0; e < 2; ++e) s[n / 2][nr][2 * (n & 1) + e] = fmaf(s[n / 2][nr][2 * (n & 1) + e], scale[nr][e] * ks, lv);
      }
      const bool special = base > sure - KEYS || (a.window && base <= low);
      uint32_t seen = ~0u;  // bit 8 of a half, 4 of 8 rows, element
      if (special) {
        const unsigned gone = lost[slot];
        seen = 0;
#pragma unroll
        for (int kh = 0; kh < KEYS / 16; ++kh)
#pragma unroll
          for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = gone >> (2 * kh + (e >> 1)) & 1 ? INT_MAX : base + 16 * kh + 8 * (e >> 1) + a8_key<D>(x8);
              const bool see = a8_sees(a, r, tok[nr][e & 1], pos[nr][e & 1], j);
              seen |= see ? 1u << (8 * kh + 4 * nr + e) : 0u;
              s[kh][nr][e] = see ? s[kh][nr][e] : -INFINITY;
            }
      }
      float top[NR][2];
      bool raise = false;
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[nr][e] = fmaxf(s[0][nr][e], s[0][nr][e + 2]);
          if constexpr (KEYS == 32) top[nr][e] = fmaxf(top[nr][e], fmaxf(s[1][nr][e], s[1][nr][e + 2]));
          raise |= top[nr][e] > m[nr][e] + A8_SLACK;
        }
      // the maximum is raised only when a score exceeds it by 2^A8_SLACK
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
          float by[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top[nr][e] = fmaxf(top[nr][e], __shfl_xor_sync(0xffffffffu, top[nr][e], d));
            by[e] = 1.f;
            if (top[nr][e] > m[nr][e] + A8_SLACK) {
              by[e] = m[nr][e] == -INFINITY ? 1.f : ex2_approx(m[nr][e] - top[nr][e]);  // from -inf: sums are 0, or NaN
              m[nr][e] = top[nr][e];
            }
            l[nr][e] *= by[e];
          }
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][nr][e] *= by[e & 1];
        }
      }
      // weights, and as P^T: keys as rows become keys as columns
      uint2 p[KEYS / 16][NR];
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) {
        const float off[2] = {m[nr][0] == -INFINITY ? 0.f : A8_LIFT - m[nr][0], m[nr][1] == -INFINITY ? 0.f : A8_LIFT - m[nr][1]};
#pragma unroll
        for (int n = 0; n < GROUPS; ++n) {
          float* x = &s[n / 2][nr][2 * (n & 1)];
          const float rv = rcp_approx(vs[n]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            x[e] = ex2_approx(x[e] + off[e]);
            l[nr][e] = fmaf(x[e], rv, l[nr][e]);
          }
          (n & 1 ? p[n / 2][nr].y : p[n / 2][nr].x) = transposed(pack_half2(x[0], x[1]));
        }
      }
      // O^T += V^T P^T: of the keys in columns 2 quad and 2 quad + 1 of both halves, the dims of piece a8_piece_of(x8) of each 128
      constexpr int WORDS = D == 64 ? 2 : 4;
#pragma unroll
      for (int part = 0; part < KEYS / 16 * BLOCKS; ++part) {
        const int blk = part % BLOCKS, kh = part / BLOCKS;  // of 128 dims, of 16 keys
        uint32_t vw[4][WORDS];
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) {
          const int k = a8_key<D>(2 * quad + (k4 & 1)) + (k4 >> 1) * 8 + 16 * kh;
          if constexpr (D == 64) {
            const uint2 y = *reinterpret_cast<const uint2*>(vb + a8_at<D>(k, x8 >> 1) + (x8 & 1) * 8);
            vw[k4][0] = y.x;
            vw[k4][1] = y.y;
          } else {
            const uint4 y = *reinterpret_cast<const uint4*>(vb + a8_at<D>(k, a8_piece_of(x8) + 8 * blk));
            vw[k4][0] = y.x;
            vw[k4][1] = y.y;
            vw[k4][2] = y.z;
            vw[k4][3] = y.w;
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
          uint2 see[NR];  // 1 where a row sees a key
#pragma unroll
          for (int nr = 0; nr < NR; ++nr) {
            const uint32_t bits = seen >> (8 * kh + 4 * nr);
            see[nr].x = transposed((bits & 1 ? 0x3c00u : 0u) | (bits & 2 ? 0x3c000000u : 0u));
            see[nr].y = transposed((bits & 4 ? 0x3c00u : 0u) | (bits & 8 ? 0x3c000000u : 0u));
          }
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
            for (int pr = 0; pr < 2; ++pr) {
              const uint32_t sel = pr == 0 ? 0x5140u : 0x7362u;
              uint4 f;
              f8_halves(__byte_perm(ind[0], ind[1], sel), f.x, f.y);
              f8_halves(__byte_perm(ind[2], ind[3], sel), f.z, f.w);
#pragma unroll
              for (int nr = 0; nr < NR; ++nr) {
                float hits[4] = {0.f, 0.f, 0.f, 0.f};
                mma16(hits, f, see[nr].x, see[nr].y);
#pragma unroll
                for (int z = 0; z < 4; ++z)
                  if (hits[z] > 0.f) o[8 * blk + 2 * w + pr][nr][z] = __int_as_float(0x7fffffff);
              }
            }
          }
        }
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
#pragma unroll
          for (int pr = 0; pr < 2; ++pr) {
            const uint32_t sel = pr == 0 ? 0x5140u : 0x7362u;
            uint4 f;
            f8_halves(__byte_perm(vw[0][w], vw[1][w], sel), f.x, f.y);
            f8_halves(__byte_perm(vw[2][w], vw[3][w], sel), f.z, f.w);
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) mma16(o[8 * blk + 2 * w + pr][nr], f, p[kh][nr].x, p[kh][nr].y);
          }
        }
      }
      __syncwarp();  // every lane has read the slice
      copy();
      if (++slot == ST) {
        slot = 0;
        phase ^= 1u;
      }
    }
    if (!__all_sync(0xffffffffu, ok)) break;
    if (!put_more) pdl_trigger();
    // ---- the item, or this piece's part of it ----
    const bool whole = i0 == 0 && i1 == sp.n;
    const int part_slot = 2 * piece + (item > 0 ? 1 : 0);
    float* part = partials + (size_t)part_slot * a8_partial_floats(D, ROWS);
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[nr][e];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const int row = 8 * nr + 2 * quad + e, t = tok[nr][e];
        if (t >= r.n) continue;
        const int64_t orow = (int64_t)(r.t0 + t) * a.hq + get.at.h * G + row0 + row - t * G;
        const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
#pragma unroll
        for (int blk = 0; blk < BLOCKS; ++blk) {  // 8 or 16 dims of each 128
          constexpr int RUN = D == 64 ? 8 : 16;
          const int d0 = D == 64 ? 8 * x8 : 128 * blk + 16 * a8_piece_of(x8);
#pragma unroll
          for (int j = 0; j < RUN; j += 8) {
            float y[8];
#pragma unroll
            for (int z = 0; z < 8; ++z) y[z] = o[8 * blk + j / 2 + z / 2][nr][2 * (z & 1) + e];
            if (whole) {
#pragma unroll
              for (int z = 0; z < 8; ++z) y[z] *= inv;
              store8((T*)a.out + orow * D + d0 + j, y);
            } else {
              float4* to = reinterpret_cast<float4*>(part + row * D + d0 + j);
              to[0] = make_float4(y[0], y[1], y[2], y[3]);
              to[1] = make_float4(y[4], y[5], y[6], y[7]);
            }
          }
        }
        if (x8 == 0) {
          if (!whole) *reinterpret_cast<float2*>(part + ROWS * D + 2 * row) = make_float2(m[nr][e], sum);
          else if (a.lse) a.lse[orow] = sum > 0.f || sum != sum ? (m[nr][e] - A8_LIFT + log2f(sum)) * 0.6931471805599453f : -INFINITY;
        }
      }
    if (lane == 0 && i0 == 0 && i1 < sp.n)
      splits[piece] = A8Split{get.at.b, get.at.h, get.at.block, (int)a8_div(unit + A8_COST + sp.n - 1, step), part_slot, {0, 0, 0}};
    unit += sp.n + A8_COST;
    if (unit + A8_COST >= lot.end) break;
    get.next_item(a, G);
  }
  cp_async_wait<0>();
  // after a wait that gave up: what is still on its way lands before the memory goes
  for (int s = taken; s < issued && !ok; ++s) da_wait(&full[s % ST], (s / ST) & 1, nullptr, 0);
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
  const int c = blockIdx.x, lane = threadIdx.x & 31, G = a.hq / a.hkv, pieces = gridDim.x;
  const A8Split s = splits[c];
  const int lead = a.cu[0], trail = a.cu[a.rows];
  if (lead > 0 || trail < a.tokens) {
    const int64_t me = ((int64_t)blockIdx.y * pieces + c) * A8J_THREADS + threadIdx.x,
                  all = (int64_t)gridDim.y * pieces * A8J_THREADS;
    a8_blank<D, T>(a, 0, min(lead, a.tokens), me, all);
    a8_blank<D, T>(a, max(trail, 0), a.tokens, me, all);
  }
  if (blockIdx.y == 0) {
    for (int b0 = c + pieces * (threadIdx.x & ~31); b0 < a.rows; b0 += pieces * A8J_THREADS) {
      const int b = b0 + pieces * lane;
      const bool out = b < a.rows && a.cu[b + 1] > a.cu[b] && a8_request<ROWS>(a, G, b, false).n == 0;
      for (unsigned rest = __ballot_sync(0xffffffffu, out); rest; rest &= rest - 1) {
        const int r = b0 + pieces * (__ffs(rest) - 1);
        a8_blank<D, T>(a, max(a.cu[r], 0), min(a.cu[r + 1], a.tokens), lane, 32);
      }
    }
  }
  if (s.last < 0) return;
  const int row = blockIdx.y * (A8J_THREADS / 32) + (threadIdx.x >> 5), at = s.block * ROWS + row, tok = at / G, t0 = a.cu[s.b];
  if (tok >= a.cu[s.b + 1] - t0) return;
  const size_t size = a8_partial_floats(D, ROWS);
  auto part = [&](int p) { return partials + (p == c ? (size_t)s.first_slot : 2 * (size_t)p) * size; };
  auto sums = [&](int p) {
    return p <= s.last ? *reinterpret_cast<const float2*>(part(p) + ROWS * D + 2 * row) : make_float2(-INFINITY, 0.f);
  };
  const float2 first = sums(c + lane);
  float m = first.x;
  for (int p = c + 32 + lane; p <= s.last; p += 32) m = fmaxf(m, sums(p).x);
  m = warp_max(m);
  float l = 0.f, o[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) o[e] = 0.f;
  for (int p0 = c; p0 <= s.last; p0 += 32) {
    // lane i: what the i-th of these parts counts (-inf with a sum is NaN, which stays)
    const float2 ml = p0 == c ? first : sums(p0 + lane);
    const float by = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : ex2_approx(ml.x - m);
    l += warp_sum(by * ml.y);
    const int n = min(32, s.last + 1 - p0);
    for (int k0 = 0; k0 < n; k0 += 8) {  // parts beyond the last: the last again, for nothing
      float x[8][D / 32];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float* from = part(min(p0 + k0 + k, s.last)) + row * D + lane;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) x[k][e] = from[e * 32];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = __shfl_sync(0xffffffffu, by, k0 + k);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) o[e] = k0 + k < n ? fmaf(w, x[k][e], o[e]) : o[e];
      }
    }
  }
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
  const int64_t orow = (int64_t)(t0 + tok) * a.hq + s.h * G + at - tok * G;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) ((T*)a.out)[orow * D + e * 32 + lane] = (T)(o[e] * inv);
  if (lane == 0 && a.lse) a.lse[orow] = l > 0.f || l != l ? (m - A8_LIFT + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace hsg
