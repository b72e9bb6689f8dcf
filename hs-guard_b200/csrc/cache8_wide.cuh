// Attention over a cache in 8 bits for many rows a key head (drafted trees, chunks of prompts), on tcgen05. What is computed is
// said in cache8_attn.cuh.
//
// The rows of a request and key head, in blocks of 128, and the tiles of KT keys (128, or 64 at head dim 256) that such a block
// can see are an item; all items are one line, cut into equal pieces, one a thread block. Per tile S = Q K^T (TMEM), softmax with
// a running maximum in registers (a row a thread), P in fp16 over S in TMEM, O += P V (A = P from TMEM, B = V, N-major).
//
// Codes become fp16 on the way into shared memory, which is exact. (e4m3
// products could take the codes as they are, but a bf16 query is two e4m3 numbers and an fp16 query or weight three: as much or
// more product time, and the softmax would have to split its weights.) Keys that the item cannot see are written as zeros and not
// read. A NaN of V in a tile that not every row sees alike is written as zero as well, and put back for the rows that see it at
// the end. Scales, and log2 and reciprocal of V's, of each 8 keys go to the softmax through a ring of their own: a weight is
// 2^(s ks + log2 vs - m), m the running maximum of that exponent, and adds itself over vs to the row's sum.
//
// Warps (four to a scheduler's slot of the register file, 128 registers a thread):
//   0, 3   queries, as fp16 (bf16: times a power of two for each row), an item ahead; 3 also says what the item is
//   1      S, up to NS tiles ahead of P V;  2: P V
//   4-7    softmax of even tiles, 8-11 of odd ones, one handing the rows' maxima on to the other before its exponentials;
//          whichever has an item's last tile writes the result
//   12-15  K and V tiles: four warps copy codes three tiles of K or V ahead and convert them
// A K or V tile lies in shared memory as [8 keys][dim / 64][8][128 B], 128-byte swizzle.
//
// A wait tells a barrier's phase from its neighbours only. S, P and P V of tile g use barrier g % NS, maxima that of their group
// (as in the attention over 16-bit pages, where the argument is written out). Scales of tile g lie in place g % 8, with a
// barrier each: they are written when K of tile g is, which waited for S of tile g - 2 or g - 3, which waited for P V of tile
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
constexpr int W8_COPY = 128;       // threads that bring K and V

__host__ __device__ constexpr int w8_tile(int dim) { return dim == 256 ? 64 : 128; }
__host__ __device__ constexpr int w8_scores(int dim) { return dim == 256 ? 4 : 3; }
__host__ __device__ constexpr int w8_q_bufs(int dim) { return dim == 64 ? 2 : 1; }
__host__ __device__ constexpr int w8_k_bufs(int dim) { return dim == 64 ? 3 : 2; }
__host__ __device__ constexpr int w8_v_bufs(int dim) { return dim == 64 ? 3 : dim == 128 ? 2 : 1; }
__host__ __device__ constexpr int w8_buffer(int dim) { return w8_tile(dim) * dim * 2; }
__host__ __device__ constexpr int w8_smem(int dim) {
  return 1024 + w8_q_bufs(dim) * W8_ROWS * dim * 2 + (w8_k_bufs(dim) + w8_v_bufs(dim)) * w8_buffer(dim) +
         3 * w8_tile(dim) * dim + 9216;
}

struct W8Item {
  A8Req r;
  A8Span s;
  int b, h, block, i0, i1, sure, lows, last, end;  // end: the piece's last item
};

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
attn8_wide_kernel(const __grid_constant__ Attn8Args a, A8Split* splits, float* partials) {
  constexpr int KT = w8_tile(D), NC = D / 64, BUF = w8_buffer(D), NS = w8_scores(D), QB = w8_q_bufs(D), NB = w8_k_bufs(D), NBV = w8_v_bufs(D);
  constexpr int Q_BUF = W8_ROWS * D * 2, Q_BOX = W8_ROWS * 128, GROUPS = KT / 8;
  constexpr uint32_t O_COL = NS * KT;
  static_assert(O_COL + D <= 512, "S buffers and O fill TMEM");
  static_assert(NB + NS < W8_PLACES, "scales outlive their tile's softmax");
  extern __shared__ __align__(1024) uint8_t w8_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(w8_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* qs = smem;                            // [QB][NC][128 rows][128 B], SW128
  uint8_t* ks = qs + QB * Q_BUF;                 // [NB][KT / 8][NC][8][128 B], SW128
  uint8_t* vs = ks + NB * BUF;                   // [NBV], likewise
  uint8_t* codes = vs + NBV * BUF;               // [3][pieces a thread][128 threads][16 B]
  float4* group_scales = reinterpret_cast<float4*>(codes + 3 * KT * D);  // [8][GROUPS] K scale, log2 and reciprocal of V's
  float* row_scale = reinterpret_cast<float*>(group_scales + W8_PLACES * 16);  // [2][128] of even / odd items
  float2* ml_rows = reinterpret_cast<float2*>(row_scale + 256);     // [2][128] (m, l) of the group without the last tile
  float* m_rows = reinterpret_cast<float*>(ml_rows + 256);          // [2][128] maxima after even / odd tiles
  W8Item* items = reinterpret_cast<W8Item*>(m_rows + 256);          // [2]
  uint64_t* bars = reinterpret_cast<uint64_t*>((reinterpret_cast<uintptr_t>(items + 2) + 7) & ~uintptr_t(7));
  uint64_t* k_full = bars;                       // [3] a tile is written
  uint64_t* k_empty = k_full + 3;                // [3] the products that read it are done
  uint64_t* v_full = k_empty + 3;
  uint64_t* v_empty = v_full + 3;
  uint64_t* q_full = v_empty + 3;                // [2]
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
  constexpr int N_BARS = 12 + 4 + 12 + 16 + 2 + 8 + 6 + 1;
  int64_t* scan = reinterpret_cast<int64_t*>(bars + N_BARS);        // [16] a8_lots'
  A8Lot* lot_here = reinterpret_cast<A8Lot*>(scan + 16);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(lot_here + 1);
  int* poison = reinterpret_cast<int*>(tmem_slot + 2);              // [4] of item & 3: item + 1 if a NaN of V was zeroed
  uint32_t* k_info = reinterpret_cast<uint32_t*>(poison + 4);       // [NB], [NB] bit 0: first of its item here, 1: last, 2: the piece's last
  uint32_t* v_info = k_info + 3;
  uint32_t* tile_info = v_info + 3;                                 // [4 warps][4] likewise, and bit 3: keys that not all rows see, 4-19: item
  float* raw_scales = reinterpret_cast<float*>(tile_info + 16);     // [4][K 16, V 16]

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, piece = blockIdx.x;
  const int G = a.hq / a.hkv;
  if (tid < N_BARS) {
    uint64_t* bar = bars + tid;
    const bool four = (bar >= k_full && bar < k_empty) || (bar >= v_full && bar < v_empty) || (bar >= p_full && bar < pv_done) ||
                      (bar >= v_seen && bar < all_done) || (bar >= ml_full && bar < ml_full + 2) || bar == o_free;
    const bool two = (bar >= q_full && bar < q_empty) || (bar >= item_full && bar < item_empty);
    mbar_init(bar, four ? 4 : two ? 2 : bar >= item_empty && bar < ml_full ? 8 : 1);
    fence_barrier_init();
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
  // of an item that begins at `unit` on the line, tiles up to this lie in the piece
  auto part_end = [&](int64_t unit, int n) { return (int)min((int64_t)n, max((int64_t)0, w1 - unit - W8_COST)); };

  if (warp >= 12) {
    // ---- K and V in turn. A thread copies 16-byte pieces of codes into places of its own (cp.async), three tiles of K or V
    // ahead, and converts what it copied itself, so that only the products wait for other threads' work. ----
    constexpr int PIECES = D / 16, AT_ONCE = 32 / PIECES, STRIDE = 4 * AT_ONCE, N = KT / STRIDE;  // keys a warp, all; pieces a thread
    static_assert(STRIDE % 8 == 0, "a thread's keys have one place among eight");
    const int me = tid - 384, wc = warp - 12;
    // eight lanes take four pieces of two keys: written, they meet no bank twice
    const int ch = (lane & 3) + 4 * ((lane >> 3) % (PIECES / 4));
    const int key0 = wc * AT_ONCE + ((lane >> 2) & 1) + 2 * ((lane >> 3) / (PIECES / 4));
    const uint32_t at0 = da_offset<NC>(key0, 2 * ch), at1 = da_offset<NC>(key0, 2 * ch + 1);
    const Cache8& c = a.cache;
    const int64_t own = (key0 & 7) * c.token_stride + ch * 16;
    uint8_t* my_codes = codes + me * 16;
    A8Walk<W8_ROWS, KT> walk;
    walk.start(a, G, from);
    int64_t unit = begin;
    int i = walk.at.i, i1 = part_end(unit, walk.s.n), item = 0;
    // the walk's tile: lane l has the page of keys 8 l .. 8 l + 7, which is asked for a tile before it is needed
    bool more = true, asked = false;
    int page = 0, within = 0;
    auto ask = [&]() {
      const int j = walk.base(i) + 8 * lane;
      asked = lane < GROUPS && j < walk.s.hi && (j > walk.s.lo - 8 || j < walk.s.ahead);
      if (asked) {
        const int p = c.page_div.div(j);
        within = j - p * c.page;
        page = a.table[walk.at.b * a.table_stride + p];
      }
    };
    ask();
    int64_t start = -1;  // where those keys begin in the pages; < 0: nowhere
    int base = 0, hi = 0, lo = 0, ahead = 0;  // of the tile that is being copied
    auto copy = [&](int b) {  // b even: K of the walk's tile, odd: V, and on to the next
      if (more) {
        if (!(b & 1)) {
          const bool good = asked && page >= 0 && page < c.pages;
          if (asked && !good) set_error(a.err, ERR_BAD_PAGE);
          start = good ? (int64_t)page * c.page_stride + within * c.token_stride + walk.at.h * c.head_stride : -1;
          base = walk.base(i);
          hi = walk.s.hi;
          lo = walk.s.lo;
          ahead = walk.s.ahead;
          if (wc == 0 && lane < GROUPS) {
            const int64_t at = good ? ((int64_t)page * c.blocks + c.block_div.div(within)) * a.hkv + walk.at.h : 0;
            const uint32_t to = smem_u32(raw_scales + (b / 2 % 4) * 32 + lane);
            cp_async4(to, c.ks + at, good);
            cp_async4(to + 64, c.vs + at, good);
          }
          const int old = walk.r.len - walk.r.n, sure = a.mask ? old : old + walk.at.block * W8_ROWS / G + 1;
          uint32_t what = (b == 0 || i == 0 ? 1u : 0u) | (base > sure - KT || a.window ? 8u : 0u) | (uint32_t)(item & 0xffff) << 4;
          if (++i >= i1) {
            what |= 2u;
            unit += walk.s.n + W8_COST;
            ++item;
            if (unit + W8_COST >= w1) {
              what |= 4u;
            } else {
              walk.next_item(a, G);
              i = 0;
              i1 = part_end(unit, walk.s.n);
            }
          }
          if (lane == 0) tile_info[wc * 4 + b / 2 % 4] = what;
          if (!(what & 4u)) ask();
          else i = -1;
        } else if (i < 0) {
          more = false;
        }
        const uint8_t* from_codes = (b & 1 ? c.v : c.k) + own;
        const uint32_t to = smem_u32(my_codes + (b % 3) * (KT * D));
        const bool whole = base >= lo && base <= hi - KT;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int k = key0 + n * STRIDE, j = base + k;
          const int64_t at = __shfl_sync(0xffffffffu, start, k >> 3);
          const bool there = at >= 0 && (whole || (j < hi && (j >= lo || j < ahead)));
          cp_async16(to + n * (W8_COPY * 16), there ? from_codes + at : c.k, there);
        }
      }
      cp_async_commit();
    };
#pragma unroll 1
    for (int b = 0; b < 3; ++b) copy(b);
#pragma unroll 1
    for (int b = 0;; ++b) {
      const bool is_v = b & 1;
      const int g = b >> 1;
      cp_async_wait<2>();
      __syncwarp();
      const uint32_t what = tile_info[wc * 4 + g % 4];
      const int nb = is_v ? NBV : NB, slot = g % nb;
      if (g >= nb)
        ok = __all_sync(0xffffffffu, da_wait(&(is_v ? v_empty : k_empty)[slot], (g / nb - 1) & 1, a.err, ERR_TIMEOUT_MMA));
      if (!ok) break;
      uint8_t* to = (is_v ? vs : ks) + slot * BUF;
      const uint8_t* x = my_codes + (b % 3) * (KT * D);
      uint32_t bad = 0;
      const bool mend = is_v && (what & 8u);
#pragma unroll 4
      for (int n = 0; n < N; ++n) {
        const uint4 v = *reinterpret_cast<const uint4*>(x + n * (W8_COPY * 16));
        uint32_t w[4] = {v.x, v.y, v.z, v.w}, y[8];
        if (mend) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t hit = (((w[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
            bad |= hit;
            w[e] &= ~(hit * 0xffu);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f8_halves(w[e], y[2 * e], y[2 * e + 1]);
        }
        *reinterpret_cast<uint4*>(to + at0 + n * (STRIDE / 8 * NC * 1024)) = make_uint4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<uint4*>(to + at1 + n * (STRIDE / 8 * NC * 1024)) = make_uint4(y[4], y[5], y[6], y[7]);
      }
      const int it = (int)(what >> 4 & 0xffff);
      if (bad) poison[it & 3] = it + 1;
      if (me == 0) (is_v ? v_info : k_info)[slot] = what;
      if (!is_v && wc == 0 && lane < GROUPS) {
        // scales of 0 or beyond what append_8bit writes are taken as the nearest that it would write
        const float* raw = raw_scales + (g % 4) * 32 + lane;
        const float v = fminf(fmaxf(raw[16], 0x1p-100f), 0x1p120f);
        group_scales[(g % W8_PLACES) * 16 + lane] = make_float4(raw[0], __log2f(v), 1.0f / v, 0.f);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&(is_v ? v_full : k_full)[slot]);
        if (is_v) mbar_arrive(&v_seen[g % W8_PLACES]);
        else if (wc == 0) mbar_arrive(&sc_full[g % W8_PLACES]);
      }
      if (is_v && (what & 4u)) break;
      copy(b + 3);
    }
    cp_async_wait<0>();
  } else if (warp == 0 || warp == 3) {
    // ---- queries: LPR lanes a row, 16 bytes each; and what each item is ----
    constexpr int LPR = D / 8, RPW = 32 / LPR, N = W8_ROWS / 2 / RPW, LIVE = 16;
    A8Walk<W8_ROWS, KT> walk;
    walk.start(a, G, from);
    int64_t unit = begin;
    const int ch = lane % LPR, sub = lane / LPR;
    DaRing ring;
    for (int item = 0;; ++item) {
      const int i0 = walk.at.i, i1 = part_end(unit, walk.s.n), row0 = walk.at.block * W8_ROWS;
      const bool end = unit + walk.s.n + 2 * W8_COST >= w1;
      uint8_t* q = qs + ring.at * Q_BUF;
#pragma unroll 1
      for (int n0 = 0; n0 < N; n0 += LIVE) {
        uint4 x[LIVE];
#pragma unroll
        for (int n = 0; n < LIVE; ++n) {
          const int row = (warp ? W8_ROWS / 2 : 0) + (n0 + n) * RPW + sub, at = row0 + row, t = at / G;
          x[n] = make_uint4(0u, 0u, 0u, 0u);
          if (t < walk.r.n)
            x[n] = *reinterpret_cast<const uint4*>((const T*)a.q + (int64_t)(walk.r.t0 + t) * a.q_ts +
                                                   (int64_t)(walk.at.h * G + at - t * G) * a.q_hs + ch * 8);
        }
        if (n0 == 0) {  // the first rows are on their way
          if (item >= 2) ok = __all_sync(0xffffffffu, da_wait(&item_empty[item & 1], ((item >> 1) - 1) & 1, a.err, ERR_TIMEOUT_MMA));
          if (ok && item >= QB) ok = __all_sync(0xffffffffu, da_wait(&q_empty[ring.at], ring.phase ^ 1u, a.err, ERR_TIMEOUT_MMA));
          if (!ok) break;
        }
#pragma unroll
        for (int n = 0; n < LIVE; ++n) {
          const int row = (warp ? W8_ROWS / 2 : 0) + (n0 + n) * RPW + sub;
          float back = 1.f;
          if constexpr (!std::is_same<T, __half>::value) {
            float v[8], most = 0.f;
            const uint32_t w[4] = {x[n].x, x[n].y, x[n].z, x[n].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[2 * e] = __uint_as_float(w[e] << 16);
              v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.f);
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            float up;
            a8_row_scale(most, up, back);
            x[n] = make_uint4(pack_half2(v[0] * up, v[1] * up), pack_half2(v[2] * up, v[3] * up),
                              pack_half2(v[4] * up, v[5] * up), pack_half2(v[6] * up, v[7] * up));
          }
          *reinterpret_cast<uint4*>(q + (ch >> 3) * Q_BOX + (row >> 3) * 1024 + sw128_off(row & 7, ch & 7)) = x[n];
          if (ch == 0) row_scale[(item & 1) * W8_ROWS + row] = back * a.scale * 1.4426950408889634f;
        }
      }
      if (!ok) break;
      if (warp == 3) {
        const int old = walk.r.len - walk.r.n;
        int lows = -1;
        if (a.window) {
          const int t1 = min(walk.r.n, (row0 + W8_ROWS - 1) / G + 1);
          for (int t = row0 / G + lane; t < t1; t += 32)
            lows = max(lows, (a.positions ? a.positions[walk.r.t0 + t] : old + t) - a.window);
          lows = __reduce_max_sync(0xffffffffu, lows);
        }
        if (lane == 0)
          items[item & 1] = W8Item{walk.r, walk.s, walk.at.b, walk.at.h, walk.at.block, i0, i1,
                                   a.mask ? old : old + row0 / G + 1, lows, (int)((unit + W8_COST + walk.s.n - 1) / step), end};
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&q_full[ring.at]);
        mbar_arrive(&item_full[item & 1]);
      }
      ring.next(QB);
      unit += walk.s.n + W8_COST;
      if (end) break;
      walk.next_item(a, G);
    }
    if (warp == 0 && lane == 0) pdl_trigger();
  } else if (warp == 1) {
    // ---- S ----
    const uint32_t idesc = DaType<__half>::idesc(KT);
    DaRing ring, q_ring, s_ring;
    for (int g = 0;; ++g) {
      ok = __all_sync(0xffffffffu, da_wait(&k_full[ring.at], ring.phase, a.err, ERR_TIMEOUT_TMA));
      if (!ok) break;
      const uint32_t what = __shfl_sync(0xffffffffu, k_info[ring.at], 0);
      if (what & 1) ok = __all_sync(0xffffffffu, da_wait(&q_full[q_ring.at], q_ring.phase, a.err, ERR_TIMEOUT_TMA));
      if (ok && g >= NS) ok = __all_sync(0xffffffffu, da_wait(&pv_done[s_ring.at], s_ring.phase ^ 1u, a.err, ERR_TIMEOUT_MMA));
      if (!ok) break;
      tc_fence_after();
      const uint64_t qd = sw128_desc(smem_u32(qs + q_ring.at * Q_BUF)), kd = da_k_desc<NC>(smem_u32(ks + ring.at * BUF));
      const uint32_t d = tmem + (uint32_t)(s_ring.at * KT);
      if (elect_one()) {
#pragma unroll
        for (int cc = 0; cc < NC; ++cc)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_bf16(d, qd + (uint64_t)((cc * Q_BOX + kk * 32) >> 4), kd + (uint64_t)((cc * 1024 + kk * 32) >> 4), idesc,
                     (cc > 0 || kk > 0) ? 1u : 0u);
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
      ok = __all_sync(0xffffffffu, da_wait(&v_full[ring.at], ring.phase, a.err, ERR_TIMEOUT_TMA));
      if (!ok) break;
      const uint32_t what = __shfl_sync(0xffffffffu, v_info[ring.at], 0);
      if (what & 1) {
        if (item > 0) ok = __all_sync(0xffffffffu, da_wait(o_free, (item - 1) & 1, a.err, ERR_TIMEOUT_MMA));
        ++item;
      }
      if (ok) ok = __all_sync(0xffffffffu, da_wait(&p_full[p_ring.at], p_ring.phase, a.err, ERR_TIMEOUT_MMA));
      if (!ok) break;
      tc_fence_after();
      const uint64_t vd = da_v_desc<NC>(smem_u32(vs + ring.at * BUF));
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
      if (ok) ok = da_wait(&item_full[item & 1], (item >> 1) & 1, a.err, ERR_TIMEOUT_TMA);
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
        if (ok) ok = da_wait(&sc_full[g % W8_PLACES], (g / W8_PLACES) & 1, a.err, ERR_TIMEOUT_TMA);
        if (ok) ok = da_wait(&s_full[ring.at], ring.phase, a.err, ERR_TIMEOUT_MMA);
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
        if (ok && g > 0) ok = da_wait(&m_full[4 * (group ^ 1) + quarter], ((g - 1) >> 1) & 1, a.err, ERR_TIMEOUT_MMA);
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
            if (ok) ok = da_wait(&pv_done[(g - 1) % NS], ((g - 1) / NS) & 1, a.err, ERR_TIMEOUT_MMA);
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
        if ((special || a.window) && ok) ok = da_wait(&v_seen[g % W8_PLACES], (g / W8_PLACES) & 1, a.err, ERR_TIMEOUT_TMA);
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
      if (ok) ok = da_wait(&ml_full[item & 1], (item >> 1) & 1, a.err, ERR_TIMEOUT_MMA);
      {
        const float2 theirs = ml_rows[128 * (item & 1) + row];  // their maximum is no larger than m, the last tile's
        l += theirs.y * (theirs.x == m || theirs.x == -INFINITY ? 1.f : ex2_approx(theirs.x - m));
      }
      if (ok) ok = da_wait(&pv_done[last % NS], (last / NS) & 1, a.err, ERR_TIMEOUT_MMA);
      tc_fence_after();
      const bool mend = *(volatile int*)&poison[item & 3] == (item & 0xffff) + 1;
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
  // ---- teardown: if every role went through, every product has been waited for; else those in flight end first ----
  __syncwarp();
  tc_fence_before();
  if (!__syncthreads_and(ok)) {
    if (warp == 1 || warp == 2) {
      if (elect_one()) mma_commit(&all_done[warp - 1]);
      __syncwarp();
      da_wait(&all_done[warp - 1], 0, nullptr, 0);
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
