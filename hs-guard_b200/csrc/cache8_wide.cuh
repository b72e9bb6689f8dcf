// Attention over a cache in 8 bits for many rows a key head (drafted trees, chunks of prompts), on tcgen05. What is computed is
// said in cache8_attn.cuh.
//
// The rows of a request and key head, in blocks of 128, and the tiles of KT keys (128, or 64 at head dim 256) that such a block
// can see are an item; all items are one line, cut into equal pieces, one a thread block. Per tile S = Q K^T (TMEM), softmax with
// a running maximum in registers (a row a thread), P in fp16 over S in TMEM, O += P V (A = P from TMEM, B = V, N-major).
//
// S takes K's codes as they are (kind::f8f6f4): a query is scaled by a power of two for each row, which brings its largest element to
// (224, 448], and written as a sum of e4m3 numbers, each the rounding of what the ones before left: two for bf16 (8 bits), three for
// fp16 (11). e4m3's last step there is 2^-9: a bf16 element is exact from 2^-2 on (2^-10.8 to 2^-9.8 of the row's largest), an fp16
// element from 2 on (2^-7.8 to 2^-6.8 of it), and smaller ones are off by at most 2^-10, which is up to 2^-17.8 of the largest: a score
// by that times scale sum |k| beside a query with an outlier. P V is a product of fp16 (weights rounded once; e4m3 weights would have to
// be two or three numbers each): V's codes become fp16 on the way, which is exact. K converted as well (1,316 us for 2,000-token chunks)
// kept four warps longer than the softmax takes. Keys
// that the item cannot see have V written as zeros. A NaN of V in a tile that not every row sees alike is written as zero as well,
// and put back for the rows that see it at the end. Scales, and log2 and reciprocal of V's, of each 8 keys go to the softmax through
// a ring of their own: a weight is 2^(s ks + log2 vs - m), m the running maximum of that exponent, and adds itself over vs to the
// row's sum.
//
// Warps (four to a scheduler's slot of the register file, 128 registers a thread):
//   0      codes of K (TMA, lane i the i-th box of one page) and scales; 3: codes of V into a staging ring, and the queries and
//          what the item is as an item begins (attn8_split_kernel has made the sums beforehand: made here, by a warp an item ahead,
//          they took as long as ten tiles)
//   1      S, up to NS tiles ahead of P V;  2: P V
//   4-7    softmax of even tiles, 8-11 of odd ones, one handing the rows' maxima on to the other before its exponentials;
//          whichever has an item's last tile writes the result
//   12-15  V from the staging ring to fp16
// Codes lie as [dim / 128][keys][128 B] (64 bytes a key at head dim 64), V as [8 keys][dim / 64][8][128 B], both swizzled.
//
// Measured on B200: 40 requests of up to 6,000 tokens, trees of 64, 32 / 4 heads of 128, bf16: 258 to 279 us (the products 82 at the
// measured bf16 rate, the cache 27); chunks of 2,000 tokens over up to 8,000, 32 / 8 heads of 128: 635 to 698 (products 225). A tile
// takes 2,650 clocks where one follows the other, of which the softmax of one group takes 4,000 for its every second one (maximum
// 950, hand-over and rescaling 600, weights 2,450: three clocks an instruction), the products 1,024, the conversion of V 1,100.
//
// A wait tells a barrier's phase from its neighbours only. S, P and P V of tile g use barrier g % NS, maxima that of their group
// (as in the attention over 16-bit pages, where the argument is written out). Scales of tile g lie in place g % 8, with a
// barrier each: they are written after K of tile g was asked for, which waited for S of tile g - 3, which waited for P V of tile
// g - 3 - NS > g - 8 at the earliest, by when the softmax of tile g - 8 was through. So are V's reports (v_seen). Reports of NaN
// have four places: V of an item of one tile waited for P V of an item at most three before it, which waited for that one's
// predecessor to be written out.
#pragma once
#include "cache8_attn.cuh"

namespace hsg {

constexpr int W8_THREADS = 512;
constexpr int W8_ROWS = 128;
constexpr int W8_COST = 3;         // what an item costs besides its tiles, in tiles
constexpr int W8_PLACES = 8;       // of scales
constexpr int W8_K_BUFS = 3, W8_STAGED = 2;

__host__ __device__ constexpr int w8_tile(int dim) { return dim == 256 ? 64 : 128; }
__host__ __device__ constexpr int w8_scores(int dim) { return dim == 256 ? 4 : 3; }
// `parts`: e4m3 numbers of a query's element
__host__ __device__ constexpr int w8_q_bufs(int dim, int parts) { return dim == 64 || (dim == 128 && parts == 2) ? 2 : 1; }
__host__ __device__ constexpr int w8_v_bufs(int dim, int parts) { return dim == 256 && parts == 3 ? 1 : 2; }
__host__ __device__ constexpr int w8_smem(int dim, int parts) {
  return 1024 + w8_q_bufs(dim, parts) * parts * W8_ROWS * dim + (W8_K_BUFS + W8_STAGED + 2 * w8_v_bufs(dim, parts)) * w8_tile(dim) * dim + 9216;
}

// A bounded wait whose slow checks (the clock, another block's error) come every 1,024th poll: a load from global memory between
// polls delays the wait's end by its latency.
__device__ __noinline__ bool w8_wait_on(uint64_t* bar, uint32_t parity, int* err, int code) {
  const uint64_t t0 = global_ns();
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 1023) == 0) {
      if (err) {
        const int e = *reinterpret_cast<volatile int*>(err);
        if (e == ERR_TIMEOUT_TMA || e == ERR_TIMEOUT_MMA) return false;
      }
      if (global_ns() - t0 > WAIT_LIMIT_NS) {
        set_error(err, code);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool w8_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  return mbar_try_wait(bar, parity) || w8_wait_on(bar, parity, err, code);
}

struct W8Item {
  A8Req r;
  A8Span s;
  int b, h, block, i0, i1, sure, lows, last, end;  // end: the piece's last item
};
struct W8Tile {  // of codes, for those who convert V
  int base, lo, hi, ahead;
  uint32_t what, groups;  // bit 0: first of its item here, 1: last, 2: the piece's last, 3: keys that not all rows see, 4: keys that
  int item;               // none sees; groups of 8 keys that were brought
};

// D[tmem] (+)= A[smem] B[smem]^T of e4m3 numbers.
__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Queries as sums of PARTS e4m3 numbers, [part][key head][token, head of the group][dim], and what a row was divided by,
// [key head][token, head of the group]. dim / 8 lanes a row.
template <int D, typename T>
__global__ void __launch_bounds__(256) attn8_split_kernel(const T* q, int64_t q_ts, int64_t q_hs, int tokens, int hq, int G, uint8_t* parts, float* scales) {
  constexpr int PARTS = std::is_same<T, __half>::value ? 3 : 2, LPR = D / 8, RPW = 32 / LPR;
  const int lane = threadIdx.x & 31, ch = lane % LPR;
  const int64_t rows = (int64_t)tokens * hq, at = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * RPW + lane / LPR;
  pdl_wait();
  pdl_trigger();
  // rows in the order of the tokens' memory
  const int t = (int)(min(at, rows - 1) / hq), h = (int)(min(at, rows - 1) - (int64_t)t * hq);
  float v[8], most = 0.f;
  unpack8<T>(*reinterpret_cast<const uint4*>(q + t * q_ts + h * q_hs + ch * 8), v);
#pragma unroll
  for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.f);
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (at >= rows) return;
  const float down = scale8_of(most), up = 1.0f / down;  // to (224, 448]
  const int64_t row = (int64_t)(h / G) * tokens * G + (int64_t)t * G + h % G;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= up;
#pragma unroll
  for (int part = 0; part < PARTS; ++part) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = f8_pair(v[2 * e], v[2 * e + 1]);
      const float2 y = f8_values(w[e]);  // what it leaves
      v[2 * e] -= y.x;
      v[2 * e + 1] -= y.y;
    }
    *reinterpret_cast<uint2*>(parts + (part * rows + row) * D + ch * 8) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
  }
  if (ch == 0) scales[row] = down;
}

// Which of tokens j0 .. j0 + 31 the new token t, at position p, of a request sees.
__device__ __noinline__ uint32_t w8_seen(const Attn8Args& a, const A8Req& r, int t, int p, int j0) {
  auto below = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; };
  const int old = r.len - r.n;
  uint32_t bits = below((a.mask ? r.len : min(r.len, old + t + 1)) - j0);
  const bool fresh = j0 > old - 32;  // new tokens among them
  const uint32_t cached = fresh ? below(old - j0) : ~0u;
  if (a.mask && fresh) {
    const int u0 = j0 - old, w = u0 >> 5;  // floor
    const uint32_t* words = a.mask + (int64_t)(r.t0 + t) * a.words;
    const uint32_t lo = w >= 0 && w < a.words ? words[w] : 0u, hi = w + 1 >= 0 && w + 1 < a.words ? words[w + 1] : 0u;
    bits &= cached | __funnelshift_r(lo, hi, u0 & 31);
  }
  if (a.window) {
    const uint32_t in = ~below(p - a.window + 1 - j0) | below(a.sinks - j0);
    if (!fresh || !a.positions) {
      bits &= in;
    } else {
      bits &= in | ~cached;
      if (p - a.window >= old) {  // a window so short that it ends among the new tokens
        for (uint32_t rest = bits & ~cached; rest; rest &= rest - 1) {
          const int j = j0 + __ffs(rest) - 1, at = a.positions[r.t0 + j - old];
          if (at <= p - a.window && at >= a.sinks) bits &= ~(rest & -rest);
        }
      }
    }
  }
  return bits;
}

// NaN for the dims in which a V row that token t sees, of the tiles that not every row sees alike, is NaN: it was 0 in the product.
template <int KT, int D, typename Y>
__device__ __noinline__ void w8_restore(const Attn8Args& a, const W8Item& it, int t, int p, Y* row) {
  for (int i = it.i0; i < it.i1; ++i) {
    const int base = (i < it.s.lead ? i : it.s.first + i - it.s.lead) * KT;
    if (base <= it.sure - KT && !a.window) continue;
    for (int j = base; j < base + KT && j < it.s.hi; ++j) {
      if (j < it.s.lo && j >= it.s.ahead) continue;
      if (!(w8_seen(a, it.r, t, p, j) & 1)) continue;
      const int pg = a.table[it.b * a.table_stride + j / a.cache.page];
      if (pg < 0 || pg >= a.cache.pages) continue;
      const uint8_t* v = a.cache.v + pg * a.cache.page_stride + j % a.cache.page * a.cache.token_stride + it.h * a.cache.head_stride;
#pragma unroll 1
      for (int d = 0; d < D; ++d)
        if ((v[d] & 0x7f) == 0x7f) row[d] = (Y)__int_as_float(0x7fffffff);
    }
  }
}

template <int D, typename T>
__global__ void __launch_bounds__(W8_THREADS, 1)
attn8_wide_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const __grid_constant__ Attn8Args a, int box, const float* q_scales, A8Split* splits, float* partials) {
  constexpr int PARTS = std::is_same<T, __half>::value ? 3 : 2;
  constexpr int KT = w8_tile(D), NC = D / 64, ROW = D == 64 ? 64 : 128, NS = w8_scores(D);
  constexpr int QB = w8_q_bufs(D, PARTS), NB = W8_K_BUFS, NBV = w8_v_bufs(D, PARTS), NST = W8_STAGED;
  constexpr int CODES = KT * D, V_BUF = KT * D * 2, Q_PART = W8_ROWS * D, Q_BUF = PARTS * Q_PART, GROUPS = KT / 8;
  constexpr uint32_t O_COL = NS * KT;
  static_assert(O_COL + D <= 512, "S buffers and O fill TMEM");
  static_assert(NB + NS < W8_PLACES, "scales outlive their tile's softmax");
  extern __shared__ __align__(1024) uint8_t w8_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(w8_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* qs = smem;                            // [QB][PARTS][COLS][128 rows][ROW]
  uint8_t* ks = qs + QB * Q_BUF;                 // [NB][COLS][KT][ROW]
  uint8_t* staged = ks + NB * CODES;             // [NST], likewise
  uint8_t* vs = staged + NST * CODES;            // [NBV][KT / 8][NC][8][128 B]
  float4* group_scales = reinterpret_cast<float4*>(vs + NBV * V_BUF);  // [8][16] K scale, log2 and reciprocal of V's
  float* row_scale = reinterpret_cast<float*>(group_scales + W8_PLACES * 16);  // [2][128] of even / odd items
  float2* ml_rows = reinterpret_cast<float2*>(row_scale + 256);     // [2][128] (m, l) of the group without the last tile
  float* m_rows = reinterpret_cast<float*>(ml_rows + 256);          // [2][128] maxima after even / odd tiles
  W8Item* items = reinterpret_cast<W8Item*>(m_rows + 256);          // [2]
  uint64_t* bars = reinterpret_cast<uint64_t*>((reinterpret_cast<uintptr_t>(items + 2) + 7) & ~uintptr_t(7));
  uint64_t* k_full = bars;                       // [3] K of a tile has landed
  uint64_t* k_empty = k_full + 3;                // [3] the products that read it are done
  uint64_t* st_full = k_empty + 3;               // [2] V's codes have landed
  uint64_t* st_empty = st_full + 2;              // [2] they have been converted
  uint64_t* v_full = st_empty + 2;               // [2] V of a tile is written
  uint64_t* v_empty = v_full + 2;                // [2]
  uint64_t* q_full = v_empty + 2;                // [2]
  uint64_t* q_empty = q_full + 2;                // [2]
  uint64_t* s_full = q_empty + 2;                // [NS] S of a tile is there
  uint64_t* p_full = s_full + 4;                 // [NS] P of a tile is written, O rescaled
  uint64_t* pv_done = p_full + 4;                // [NS] O includes the tile
  uint64_t* sc_full = pv_done + 4;               // [8] a tile's scales are there
  uint64_t* v_seen = sc_full + W8_PLACES;        // [8] V of a tile is written, and its NaN reported
  uint64_t* all_done = v_seen + W8_PLACES;       // [2] of warps 1 and 2, when a role has given up
  uint64_t* m_full = all_done + 2;               // [2][4] a softmax warp's maxima
  uint64_t* item_full = m_full + 8;              // [2] what an item is, and its rows' scales
  uint64_t* item_empty = item_full + 2;          // [2]
  uint64_t* ml_full = item_empty + 2;            // [2] the group without an item's last tile is through with it
  uint64_t* o_free = ml_full + 2;                // O has been read
  constexpr int N_BARS = 6 + 4 + 4 + 4 + 12 + 16 + 2 + 8 + 6 + 1;
  int64_t* scan = reinterpret_cast<int64_t*>(bars + N_BARS);        // [16] a8_lots'
  A8Lot* lot_here = reinterpret_cast<A8Lot*>(scan + 16);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(lot_here + 1);
  int* poison = reinterpret_cast<int*>(tmem_slot + 2);              // [4] of item & 3: item + 1 if a NaN of V was zeroed
  uint32_t* k_info = reinterpret_cast<uint32_t*>(poison + 4);       // [NB], [NBV] W8Tile's bits 0 to 2
  uint32_t* v_info = k_info + 3;
  W8Tile* tiles = reinterpret_cast<W8Tile*>(v_info + 3);            // [NST]

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, piece = blockIdx.x;
  const int G = a.hq / a.hkv;
  if (tid < N_BARS) {
    uint64_t* bar = bars + tid;
    const bool four = (bar >= st_empty && bar < v_empty) || (bar >= p_full && bar < pv_done) || (bar >= v_seen && bar < all_done) ||
                      (bar >= ml_full && bar < ml_full + 2) || bar == o_free;
    mbar_init(bar, four ? 4 : bar >= item_empty && bar < ml_full ? 8 : 1);
    fence_barrier_init();
  }
  if (tid == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (tid < 4) poison[tid] = 0;
  pdl_wait();
  if (tid == 0) splits[piece].last = -1;
  const int64_t step = a8_lots<W8_ROWS, KT, W8_THREADS, 1>(a, G, W8_COST, piece, scan, lot_here);
  const A8At from = lot_here->from;
  const int64_t begin = lot_here->begin, w1 = lot_here->end;
  if (from.b < 0) return;  // the whole block
  if (warp == 3) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  bool ok = true;  // no wait of this thread has given up
  int issued = 0, q_issued = 0;  // warps 0 and 3: tiles of K or V asked for; warp 3: queries
  // of an item that begins at `unit` on the line, tiles up to this lie in the piece
  auto part_end = [&](int64_t unit, int n) { return (int)min((int64_t)n, max((int64_t)0, w1 - unit - W8_COST)); };

  if (warp >= 12) {
    // ---- V: each thread the same 16 bytes of every few keys ----
    constexpr int PIECES = D / 16, STRIDE = 4 * (32 / PIECES), N = KT / STRIDE;  // pieces a key; keys of all warps at once
    static_assert(STRIDE % 8 == 0, "a thread's keys have one place among eight");
    const int wc = warp - 12, rest = lane >> 3, flip = lane & 4 ? 5 : 0;
    // eight lanes take four pieces of two keys whose numbers differ in bits 0 and 2: neither read nor written do they meet a bank twice
    const int ch = (lane & 3) + (D == 64 ? 0 : D == 128 ? 4 * (rest & 1) : 4 * rest);
    const int in8 = (D == 64 ? rest : D == 128 ? 2 * (wc & 1) + (rest >> 1) : wc) ^ flip;
    const int key0 = 8 * (D == 64 ? wc : D == 128 ? wc >> 1 : 0) + in8;
    const uint32_t from_at = D == 64 ? sw64_off(key0, ch) : (ch >> 3) * (KT * 128) + (key0 >> 3) * 1024 + sw128_off(key0 & 7, ch & 7);
    const uint32_t at0 = da_offset<NC>(key0, 2 * ch), at1 = da_offset<NC>(key0, 2 * ch + 1);
    DaRing st_ring, ring;
#pragma unroll 1
    for (int g = 0;; ++g) {
      ok = __all_sync(0xffffffffu, w8_wait(&st_full[st_ring.at], st_ring.phase, a.err, ERR_TIMEOUT_TMA));
      if (ok && g >= NBV) ok = __all_sync(0xffffffffu, w8_wait(&v_empty[ring.at], ring.phase ^ 1u, a.err, ERR_TIMEOUT_MMA));
      if (!ok) break;
      const W8Tile tile = tiles[st_ring.at];
      const uint8_t* x = staged + st_ring.at * CODES + from_at;
      uint8_t* to = vs + ring.at * V_BUF;
      uint32_t bad = 0;
      const bool careful = tile.what & 24u;
#pragma unroll 4
      for (int n = 0; n < N; ++n) {
        uint4 v = *reinterpret_cast<const uint4*>(x + n * STRIDE * ROW);
        if (careful) {
          const int k = key0 + n * STRIDE, j = tile.base + k;
          if (!(tile.groups >> (k >> 3) & 1) || j >= tile.hi || (j < tile.lo && j >= tile.ahead)) v = make_uint4(0u, 0u, 0u, 0u);
          uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t hit = tile.what & 8u ? (((w[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7 : 0u;
            bad |= hit;
            w[e] &= ~(hit * 0xffu);
          }
        }
        uint32_t y[8];
        f8_halves(v.x, y[0], y[1]);
        f8_halves(v.y, y[2], y[3]);
        f8_halves(v.z, y[4], y[5]);
        f8_halves(v.w, y[6], y[7]);
        *reinterpret_cast<uint4*>(to + at0 + n * (STRIDE / 8 * NC * 1024)) = make_uint4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<uint4*>(to + at1 + n * (STRIDE / 8 * NC * 1024)) = make_uint4(y[4], y[5], y[6], y[7]);
      }
      if (bad) poison[tile.item & 3] = tile.item + 1;
      if (wc == 0 && lane == 0) v_info[ring.at] = tile.what;
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&st_empty[st_ring.at]);
        mbar_arrive(&v_full[ring.at]);
        mbar_arrive(&v_seen[g % W8_PLACES]);
      }
      st_ring.next(NST);
      ring.next(NBV);
      if (tile.what & 4u) break;
    }
  } else if (warp == 0 || warp == 3) {
    // ---- codes of K and scales (warp 0), codes of V, queries and items (warp 3) ----
    const bool is_v = warp == 3;
    const CUtensorMap* map = is_v ? &tm_v : &tm_k;
    uint64_t *full = is_v ? st_full : k_full, *empty = is_v ? st_empty : k_empty;
    uint8_t* bufs = is_v ? staged : ks;
    const int n_bufs = is_v ? NST : NB;
    const Cache8& c = a.cache;
    A8Walk<W8_ROWS, KT> walk;
    walk.start(a, G, from);
    int64_t unit = begin;
    int i = walk.at.i, i1 = part_end(unit, walk.s.n), item = 0;
    // A tile: what it holds; lane l: the page of keys 8 l .. 8 l + 7, asked for two tiles before its codes are, and their scales
    struct Tile {
      W8Tile t;
      int h, page, within;
      bool asked, lost;  // lost: the cache has no such page
      float ksc, vsc;
    };
    // warp 3: what an item is, and its rows' scales (lane l: rows l, l + 32 ...), as its first tile is taken
    W8Item next_item{}, cur_item{};
    float next_scale[4], cur_scale[4] = {0.f, 0.f, 0.f, 0.f};
    auto describe = [&]() {
      const int old = walk.r.len - walk.r.n, row0 = walk.at.block * W8_ROWS;
      int lows = -1;
      if (a.window) {
        const int t1 = min(walk.r.n, (row0 + W8_ROWS - 1) / G + 1);
        for (int t = row0 / G + lane; t < t1; t += 32)
          lows = max(lows, (a.positions ? a.positions[walk.r.t0 + t] : old + t) - a.window);
        lows = __reduce_max_sync(0xffffffffu, lows);
      }
      next_item = W8Item{walk.r, walk.s, walk.at.b, walk.at.h, walk.at.block, i, i1, a8_sure(a, old, row0 / G), lows,
                         (int)a8_div(unit + W8_COST + walk.s.n - 1, step), unit + walk.s.n + 2 * W8_COST >= w1};
      const int64_t first = (int64_t)walk.at.h * a.tokens * G + (int64_t)walk.r.t0 * G + row0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        next_scale[e] = row0 + lane + 32 * e < walk.r.n * G ? q_scales[first + lane + 32 * e] : 1.f;
    };
    auto take = [&](bool begins) {  // the walk's tile, and the walk to the next one
      const int old = walk.r.len - walk.r.n, sure = a8_sure(a, old, walk.at.block * W8_ROWS / G), base = walk.base(i);
      Tile x{{base, walk.s.lo, walk.s.hi, walk.s.ahead, begins || i == 0 ? 1u : 0u, 0u, item}, walk.at.h, 0, 0, false, false, 0.f, 1.f};
      if (is_v && (x.t.what & 1u)) describe();
      if (base > sure - KT || a.window) x.t.what |= 8u;
      if (base < x.t.lo || base > x.t.hi - KT) x.t.what |= 16u;
      const int j = base + 8 * lane;
      x.asked = lane < GROUPS && j < x.t.hi && (j > x.t.lo - 8 || j < x.t.ahead);
      if (x.asked) {
        const int p = c.page_div.div(j);
        x.within = j - p * c.page;
        x.page = a.table[walk.at.b * a.table_stride + p];
      }
      if (++i >= i1) {
        x.t.what |= 2u;
        unit += walk.s.n + W8_COST;
        ++item;
        if (unit + W8_COST >= w1) {
          x.t.what |= 4u;
        } else {
          walk.next_item(a, G);
          i = 0;
          i1 = part_end(unit, walk.s.n);
        }
      }
      return x;
    };
    auto resolve = [&](Tile& x) {  // its page has come: which groups can be brought, and their scales
      const bool good = x.asked && x.page >= 0 && x.page < c.pages;
      x.lost = x.asked && !good;
      if (x.lost) set_error(a.err, ERR_BAD_PAGE);
      x.t.what |= __any_sync(0xffffffffu, x.lost) ? 16u : 0u;
      x.t.groups = __ballot_sync(0xffffffffu, good);
      if (good && !is_v) {
        const int64_t at = ((int64_t)x.page * c.blocks + c.block_div.div(x.within)) * a.hkv + x.h;
        x.ksc = c.ks[at];
        x.vsc = c.vs[at];
      }
    };
    // lane i brings the i-th box if it has a group that can be brought, and knows where from by that group's lane
    const int per = box >> 3, g0 = lane * per;
    auto bring = [&](uint8_t* to, const Tile& x, uint64_t* bar) {
      const unsigned mine = g0 < GROUPS ? x.t.groups >> g0 & (per == 32 ? ~0u : (1u << per) - 1u) : 0u;
      const int src = mine ? g0 + __ffs(mine) - 1 : 0;
      const int page = __shfl_sync(0xffffffffu, x.page, src), row = __shfl_sync(0xffffffffu, x.within, src) - 8 * (src - g0);
      const unsigned boxes = __ballot_sync(0xffffffffu, mine != 0);
      if (lane == 0) mbar_arrive_expect_tx(bar, __popc(boxes) * box * D);
      __syncwarp();
      if (mine) {
        const int cols = D == 256 && box < KT ? 2 : 1;  // a box of fewer keys would pack its blocks of 128 bytes closer
#pragma unroll 1
        for (int e = 0; e < cols; ++e) tma_load_5d(to + lane * box * ROW + e * (KT * 128), map, 0, row, e, x.h, page, bar);
      }
    };
    Tile cur = take(true), next = cur;
    resolve(cur);
    cur_item = next_item;
#pragma unroll
    for (int e = 0; e < 4; ++e) cur_scale[e] = next_scale[e];
    if (!(cur.t.what & 4u)) next = take(false);
    DaRing ring, q_ring;
    int items_done = 0;
#pragma unroll 1
    for (int g = 0;; ++g) {
      if (is_v && (cur.t.what & 1u)) {
        if (items_done >= 2)
          ok = __all_sync(0xffffffffu, w8_wait(&item_empty[items_done & 1], ((items_done >> 1) - 1) & 1, a.err, ERR_TIMEOUT_MMA));
        if (ok && items_done >= QB) ok = __all_sync(0xffffffffu, w8_wait(&q_empty[q_ring.at], q_ring.phase ^ 1u, a.err, ERR_TIMEOUT_MMA));
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&q_full[q_ring.at], Q_BUF);
          items[items_done & 1] = cur_item;
        }
        __syncwarp();
        if (lane < PARTS)
          tma_load_4d(qs + q_ring.at * Q_BUF + lane * Q_PART, &tm_q, 0, cur_item.h * a.tokens * G + cur_item.r.t0 * G + cur_item.block * W8_ROWS, 0,
                      lane, &q_full[q_ring.at]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          row_scale[(items_done & 1) * W8_ROWS + lane + 32 * e] = cur_scale[e] * a.scale * 1.4426950408889634f;
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_full[items_done & 1]);
        ++items_done;
        ++q_issued;
        q_ring.next(QB);
      }
      if (g >= n_bufs) ok = __all_sync(0xffffffffu, w8_wait(&empty[ring.at], ring.phase ^ 1u, a.err, ERR_TIMEOUT_MMA));
      if (!ok) break;
      if (lane == 0) {
        if (is_v) tiles[ring.at] = cur.t;
        else k_info[ring.at] = cur.t.what;
      }
      if (!is_v && __any_sync(0xffffffffu, cur.lost)) {
        // keys of no page: codes of 0 in place of what was there before, and a scale of V that leaves their weights at 0
        if (cur.lost)
#pragma unroll 1
          for (int e = 0; e < 8 * D / 16; ++e)
            *reinterpret_cast<uint4*>(bufs + ring.at * CODES + (e / (ROW / 2)) * (KT * 128) + lane * (8 * ROW) + e % (ROW / 2) * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async();
        __syncwarp();
      }
      bring(bufs + ring.at * CODES, cur, &full[ring.at]);
      ++issued;
      if (!is_v) {
        const float v = a8_v_scale(cur.vsc);
        if (lane < GROUPS) group_scales[(g % W8_PLACES) * 16 + lane] = make_float4(cur.ksc, cur.lost ? -INFINITY : __log2f(v), rcp_approx(v), 0.f);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sc_full[g % W8_PLACES]);
      }
      ring.next(n_bufs);
      if (cur.t.what & 4u) break;
      cur = next;
      resolve(cur);
      if (is_v && (cur.t.what & 1u)) {
        cur_item = next_item;
#pragma unroll
        for (int e = 0; e < 4; ++e) cur_scale[e] = next_scale[e];
      }
      if (!(cur.t.what & 4u)) next = take(false);
    }
    if (!is_v && lane == 0) pdl_trigger();
  } else if (warp == 1) {
    // ---- S ----
    const uint32_t idesc = (1u << 4) | ((uint32_t)(KT >> 3) << 17) | ((uint32_t)(W8_ROWS >> 4) << 24);  // e4m3 by e4m3, fp32
    DaRing ring, q_ring, s_ring;
    for (int g = 0;; ++g) {
      ok = __all_sync(0xffffffffu, w8_wait(&k_full[ring.at], ring.phase, a.err, ERR_TIMEOUT_TMA));
      if (!ok) break;
      const uint32_t what = __shfl_sync(0xffffffffu, k_info[ring.at], 0);
      if (what & 1) ok = __all_sync(0xffffffffu, w8_wait(&q_full[q_ring.at], q_ring.phase, a.err, ERR_TIMEOUT_TMA));
      if (ok && g >= NS) ok = __all_sync(0xffffffffu, w8_wait(&pv_done[s_ring.at], s_ring.phase ^ 1u, a.err, ERR_TIMEOUT_MMA));
      if (!ok) break;
      tc_fence_after();
      const uint32_t qa = smem_u32(qs + q_ring.at * Q_BUF), ka = smem_u32(ks + ring.at * CODES);
      const uint64_t qd = D == 64 ? sw64_desc(qa) : sw128_desc(qa), kd = D == 64 ? sw64_desc(ka) : sw128_desc(ka);
      const uint32_t d = tmem + (uint32_t)(s_ring.at * KT);
      if (elect_one()) {
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
#pragma unroll
          for (int kk = 0; kk < D / 32; ++kk)
            mma_f8(d, qd + (uint64_t)((part * Q_PART + (kk >> 2) * (W8_ROWS * 128) + (kk & 3) * 32) >> 4),
                   kd + (uint64_t)(((kk >> 2) * (KT * 128) + (kk & 3) * 32) >> 4), idesc, (part > 0 || kk > 0) ? 1u : 0u);
        mma_commit(&s_full[s_ring.at]);
        mma_commit(&k_empty[ring.at]);
        if (what & 2) mma_commit(&q_empty[q_ring.at]);
      }
      __syncwarp();
      ring.next(NB);
      if (what & 2) q_ring.next(QB);
      s_ring.next(NS);
      if (what & 4) break;
    }
  } else if (warp == 2) {
    // ---- P V ----
    const uint32_t idesc = DaType<__half>::idesc(D) | DA_B_N_MAJOR;
    DaRing ring, p_ring;
    int item = 0;
    for (;;) {
      ok = __all_sync(0xffffffffu, w8_wait(&v_full[ring.at], ring.phase, a.err, ERR_TIMEOUT_TMA));
      if (!ok) break;
      const uint32_t what = __shfl_sync(0xffffffffu, v_info[ring.at], 0);
      if (what & 1) {
        if (item > 0) ok = __all_sync(0xffffffffu, w8_wait(o_free, (item - 1) & 1, a.err, ERR_TIMEOUT_MMA));
        ++item;
      }
      if (ok) ok = __all_sync(0xffffffffu, w8_wait(&p_full[p_ring.at], p_ring.phase, a.err, ERR_TIMEOUT_MMA));
      if (!ok) break;
      tc_fence_after();
      const uint64_t vd = da_v_desc<NC>(smem_u32(vs + ring.at * V_BUF));
      const uint32_t p = tmem + (uint32_t)(p_ring.at * KT);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < KT / 16; ++kk)
          mma_tmem_a(tmem + O_COL, p + kk * 8, vd + (uint64_t)((kk * 2 * NC * 1024) >> 4), idesc, (!(what & 1) || kk > 0) ? 1u : 0u);
        mma_commit(&pv_done[p_ring.at]);
        mma_commit(&v_empty[ring.at]);
      }
      __syncwarp();
      ring.next(NBV);
      p_ring.next(NS);
      if (what & 4) break;
    }
  } else {
    // ---- softmax: thread = row = TMEM lane; group 0 (warps 4-7) takes even tiles, group 1 (warps 8-11) odd ones ----
    const int group = warp >= 8, row = tid & 127, quarter = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    DaRing ring;  // of tile g's S and P
    int reached = 0;
    int g0 = 0;  // the item's first tile
    for (int item = 0;; ++item) {
      if (ok) ok = w8_wait(&item_full[item & 1], (item >> 1) & 1, a.err, ERR_TIMEOUT_TMA);
      if (!__all_sync(0xffffffffu, ok)) {  // without the item there is nothing to go by
        ok = false;
        break;
      }
      const W8Item& it = items[item & 1];
      const int i0 = it.i0, i1 = it.i1;
      const int at = it.block * W8_ROWS + row, tok = at / G;
      const bool valid = tok < it.r.n;
      const bool live = __any_sync(0xffffffffu, valid);
      const bool end = it.end;
      const float rs = row_scale[(item & 1) * W8_ROWS + row];
      const int p = !valid || !a.window ? 0 : a.positions ? a.positions[it.r.t0 + tok] : it.r.len - it.r.n + tok;
      float m = -INFINITY, l = 0.f;  // maximum of the last tile that this group took part in, sum of its own weights
      for (int i = i0 + ((g0 ^ group) & 1); i < i1; i += 2) {
        const int g = g0 + i - i0;
        for (; reached < g; ++reached) ring.next(NS);
        const uint32_t s_col = lanes + (uint32_t)(ring.at * KT);  // S, later P
        const int base = (i < it.s.lead ? i : it.s.first + i - it.s.lead) * KT;
        const bool special = base > it.sure - KT || (a.window && base <= it.lows);
        const float4* sc = group_scales + (g % W8_PLACES) * 16;
        if (ok) ok = w8_wait(&sc_full[g % W8_PLACES], (g / W8_PLACES) & 1, a.err, ERR_TIMEOUT_TMA);
        if (ok) ok = w8_wait(&s_full[ring.at], ring.phase, a.err, ERR_TIMEOUT_MMA);
        tc_fence_after();
        __syncwarp();
        float top = -INFINITY;
        if (live) {
          // S is read twice, for the maximum and for the weights, 32 columns at a time
#pragma unroll 1
          for (int c = 0; c < KT / 32; ++c) {
            uint32_t x[32];
            tmem_ld32_async(s_col + 32 * c, x);
            tmem_ld_wait();
            da_pin(x);
            if (special) {  // -inf where the row does not see the key, for the second reading as well
              const uint32_t bits = valid ? w8_seen(a, it.r, tok, p, base + 32 * c) : 0u;
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = bits >> j & 1 ? x[j] : 0xff800000u;
              tmem_st32_async(s_col + 32 * c, x);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // 8 keys of one scale
              float t = __uint_as_float(x[8 * e]);
#pragma unroll
              for (int j = 1; j < 8; ++j) t = fmaxf(t, __uint_as_float(x[8 * e + j]));
              const float4 s = sc[4 * c + e];
              top = fmaxf(top, fmaf(t, fmaxf(rs * s.x, 0x1p-126f), s.y));  // (-inf times 0 would not be -inf)
            }
          }
          if (special) tmem_st_wait();
        }
        // the maximum so far, from the other group; it is raised only when a tile exceeds it by 2^A8_SLACK
        if (ok && g > 0) ok = w8_wait(&m_full[4 * (group ^ 1) + quarter], ((g - 1) >> 1) & 1, a.err, ERR_TIMEOUT_MMA);
        const float seen = i > i0 ? m_rows[128 * (group ^ 1) + row] : -INFINITY;
        const bool raise = valid && (top > seen + A8_SLACK || (seen == -INFINITY && top > -INFINITY));
        const float now = raise ? top : seen;
        m_rows[128 * group + row] = now;
        __syncwarp();
        if (lane == 0) mbar_arrive(&m_full[4 * group + quarter]);
        if (live) {
          if (now != m) {  // m = -inf: l is 0, or NaN
            l *= m == -INFINITY ? 1.f : ex2_approx(m - now);
            m = now;
          }
          if (i > i0 && __any_sync(0xffffffffu, raise)) {
            if (ok) ok = w8_wait(&pv_done[(g - 1) % NS], ((g - 1) / NS) & 1, a.err, ERR_TIMEOUT_MMA);
            tc_fence_after();
            __syncwarp();
            const float alpha = !raise || seen == -INFINITY ? 1.f : ex2_approx(seen - now);  // from -inf: O is 0, or NaN
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              float o[32];
              tmem_ld32(lanes + O_COL + c, o);
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] *= alpha;
              tmem_st32(lanes + O_COL + c, o);
            }
          }
          const float less = m == -INFINITY ? 0.f : A8_LIFT - m;
          __syncwarp();
#pragma unroll 1
          for (int c = 0; c < KT / 32; ++c) {
            uint32_t x[32], pk[16];
            tmem_ld32_async(s_col + 32 * c, x);
            float4 s[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = sc[4 * c + e];
            tmem_ld_wait();
            da_pin(x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float by = fmaxf(rs * s[e].x, 0x1p-126f);
              const float2 mul = make_float2(by, by), off = make_float2(s[e].y + less, s[e].y + less);
              float2 sum = make_float2(0.f, 0.f);
#pragma unroll
              for (int j = 8 * e; j < 8 * e + 8; j += 2) {
                float2 y = fma2(make_float2(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), mul, off);
                y = make_float2(ex2_approx(y.x), ex2_approx(y.y));
                sum = add2(sum, y);
                pk[j >> 1] = pack_half2(y.x, y.y);
              }
              l = fmaf(sum.x + sum.y, s[e].z, l);
            }
            tmem_st16_async(s_col + 16 * c, pk);  // over scores that have been read
          }
          tmem_st_wait();
        }
        if ((special || a.window) && ok) ok = w8_wait(&v_seen[g % W8_PLACES], (g / W8_PLACES) & 1, a.err, ERR_TIMEOUT_TMA);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[ring.at]);
      }
      // ---- epilogue of the item, or of this piece's part of it: by the group that has its last tile, while the other
      // goes on to the next item ----
      const int last = g0 + i1 - i0 - 1;  // its last tile
      g0 += i1 - i0;
      if ((last & 1) != group) {
        ml_rows[128 * (item & 1) + row] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&ml_full[item & 1]);
          mbar_arrive(&item_empty[item & 1]);
        }
        if (end) break;
        continue;
      }
      if (ok) ok = w8_wait(&ml_full[item & 1], (item >> 1) & 1, a.err, ERR_TIMEOUT_MMA);
      {
        const float2 theirs = ml_rows[128 * (item & 1) + row];  // their maximum is no larger than m, the last tile's
        l += theirs.y * (theirs.x == m || theirs.x == -INFINITY ? 1.f : ex2_approx(theirs.x - m));
      }
      if (ok) ok = w8_wait(&pv_done[last % NS], (last / NS) & 1, a.err, ERR_TIMEOUT_MMA);
      tc_fence_after();
      const bool mend = *(volatile int*)&poison[item & 3] == item + 1;
      const bool whole = i0 == 0 && i1 == it.s.n;
      const int slot = 2 * piece + (item > 0 ? 1 : 0), h = it.h;
      float* part = partials + slot * a8_partial_floats(D, W8_ROWS);
      const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
      const int64_t orow = (int64_t)(it.r.t0 + tok) * a.hq + h * G + at - tok * G;
      if (live) {
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float o[32];
          __syncwarp();
          tmem_ld32(lanes + O_COL + c, o);
          if (!valid) continue;
          if (whole) {
            T* dst = (T*)a.out + orow * D + c;
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              const float y[8] = {o[j] * inv, o[j + 1] * inv, o[j + 2] * inv, o[j + 3] * inv,
                                  o[j + 4] * inv, o[j + 5] * inv, o[j + 6] * inv, o[j + 7] * inv};
              store8(dst + j, y);
            }
          } else {
            float* dst = part + row * D + c;
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              *reinterpret_cast<float4*>(dst + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      if (mend && valid) {
        if (whole) w8_restore<KT, D, T>(a, it, tok, p, (T*)a.out + orow * D);
        else w8_restore<KT, D, float>(a, it, tok, p, part + row * D);
      }
      if (valid) {
        if (!whole)
          *reinterpret_cast<float2*>(part + W8_ROWS * D + 2 * row) = make_float2(m, l);
        else if (a.lse)
          a.lse[orow] = l > 0.f || l != l ? (m - A8_LIFT + log2f(l)) * 0.6931471805599453f : -INFINITY;
      }
      if (row == 0 && i0 == 0 && i1 < it.s.n) splits[piece] = A8Split{it.b, h, it.block, it.last, slot, {0, 0, 0}};
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[item & 1]);
      if (end) break;
    }
  }
  // ---- teardown: if every role went through, every copy and product has been waited for; else those in flight end first ----
  __syncwarp();
  tc_fence_before();
  if (!__syncthreads_and(ok)) {
    if (warp == 0 || warp == 3) {
      const int n_bufs = warp == 3 ? NST : NB;
      for (int g = max(0, issued - n_bufs); g < issued; ++g) w8_wait(&(warp == 3 ? st_full : k_full)[g % n_bufs], (g / n_bufs) & 1, nullptr, 0);
      for (int e = max(0, q_issued - QB); e < q_issued; ++e) w8_wait(&q_full[e % QB], (e / QB) & 1, nullptr, 0);
    } else if (warp == 1 || warp == 2) {
      if (elect_one()) mma_commit(&all_done[warp - 1]);
      __syncwarp();
      w8_wait(&all_done[warp - 1], 0, nullptr, 0);
    }
    tc_fence_before();
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace hsg
