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
#include "ring_prefill_tc.cuh"  // ex2_approx

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

// One kernel for every shape, on tcgen05. The drafted tokens of a request that share a key head are the rows of a matrix
// product, row r = (token r / G, query head r % G of the group of G); 128 rows and all of a request's keys in tiles of
// KT (128, or 64 at head dim 256) are an item (request, key head, block of 128 rows). All items' tiles, in order, are one
// line that is cut into equal pieces, one a thread block, whatever the requests' lengths, so a long cache is split over
// many SMs and short ones share one; the lengths are read on the device. An item that lies in one piece is written
// out; of one that is cut, each piece leaves its unnormalised sums, row maxima and row sums in the workspace and
// draft_join_kernel joins them in piece order, so results do not depend on timing.
//
// Per tile: S = Q K^T (tcgen05, TMEM), softmax with a running maximum in registers (a row a thread), P in the type of V
// written over S in TMEM, O += P V (A = P from TMEM, B = V as it lies in shared memory, N-major). Warp 0 brings K and
// V tiles by TMA, page by page, 128-byte swizzle, through one ring of buffers in the order in which the products use
// them; warp 1 issues the products, S of the next tile before P V of this one; warps 2-3 gather Q; warps 4-7 do the
// softmax and the epilogue. Tiles of the next item are under way during an item's epilogue.
//
// S, P and P V of a tile each have two barriers, for even and odd tiles: a wait tells a phase from its neighbours only,
// and whoever waits for tile g of one of them knows tile g - 2 to be done and g + 2 to be impossible before it goes on
// (S of tile g + 2 is issued after P of tile g has been waited for, and its commit covers every product before it).
//
// The weights are rounded to V's type for the second product (relative 2^-11 or 2^-8 each, as the result itself is);
// scores, maxima, sums and O are fp32, and the row sum adds the weights before they are rounded.
constexpr int DA_THREADS = 256;
constexpr int DA_ROWS = 128;
constexpr int DA_MIN_TILES = 2;       // a piece is at least this long
constexpr int DA_SMEM_LIMIT = 227 * 1024;
constexpr uint32_t DA_TMEM_COLS = 512;  // S (later P) of even and odd tiles, then O

__host__ __device__ constexpr int da_tile(int dim) { return dim == 256 ? 64 : 128; }
__host__ __device__ constexpr int da_buffer_bytes(int dim) { return da_tile(dim) * dim * 2; }

struct DaPlan {  // launch shape, chosen by the host
  int q_rows;    // rows a Q buffer holds: a multiple of 8 up to 128
  int q_bufs;
  int kv_bufs;
  int box;       // tokens of one TMA box of the cache: the largest power of two that divides the page, at most KT
  int pieces;    // thread blocks
};
__host__ __device__ inline int da_smem_bytes(const DaPlan& p, int dim) {
  return p.q_bufs * p.q_rows * dim * 2 + p.kv_bufs * da_buffer_bytes(dim) + 1024 + 512;
}

// Workspace: per piece two partial results (its first and its last item) of 128 rows, O [128][dim], then (m, l) [128],
// and the item that begins in it and ends in a later piece.
struct DaSplit {
  int b, h, block, last;  // last: the piece it ends in; -1: none
  int first_slot;         // partial result of the piece it begins in
  int pad[3];
};
__host__ __device__ inline size_t da_partial_floats(int dim) { return (size_t)DA_ROWS * (dim + 2); }
__host__ __device__ inline size_t da_workspace_bytes(int dim, int pieces) {
  return pieces * sizeof(DaSplit) + 2 * pieces * da_partial_floats(dim) * sizeof(float);
}

// What a request asks for: its drafted tokens, first visible tile and tile counts; n = 0 if it drafts nothing or its
// lengths are out of range.
struct DaReq {
  int len, t0, fresh, lo, first, cached, n, blocks;
};
template <int KT>
__device__ __forceinline__ DaReq da_request(const DraftAttnArgs& a, int b, bool report) {
  DaReq r;
  r.len = a.lens[b];
  r.t0 = a.cu[b];
  const int t1 = a.cu[b + 1];
  r.fresh = t1 - r.t0;
  if (r.len < 0 || r.len > (int64_t)a.width * a.cache.page || r.t0 < 0 || t1 < r.t0 || t1 > a.tokens ||
      r.fresh > a.max_tree) {
    if (report) set_error(a.err, ERR_BAD_LEN);
    r.fresh = 0;
  }
  r.lo = a.window ? max(0, r.len - a.window + 1) : 0;
  r.first = r.lo / KT;
  r.cached = r.lo < r.len ? (r.len + KT - 1) / KT - r.first : 0;
  r.n = r.fresh ? r.cached + (r.fresh + KT - 1) / KT : 0;
  r.blocks = (r.fresh * (a.hq / a.hkv) + DA_ROWS - 1) / DA_ROWS;
  return r;
}

// A place on the line of tiles.
template <int KT>
struct DaWalk {
  const DraftAttnArgs* a;
  DaReq r;
  int b, h, block, i;
  __device__ __forceinline__ void start(const DraftAttnArgs& args, int b0, int64_t within) {
    a = &args;
    b = b0;
    r = da_request<KT>(args, b, false);
    const int64_t item = within / r.n;
    i = (int)(within - item * r.n);
    h = (int)(item / r.blocks);
    block = (int)(item - (int64_t)h * r.blocks);
  }
  __device__ __forceinline__ void skip(int tiles) {  // at most to the item's end
    i += tiles;
    if (i < r.n) return;
    i = 0;
    if (++block < r.blocks) return;
    block = 0;
    if (++h < a->hkv) return;
    h = 0;
    do {
      if (++b >= a->rows) return;
      r = da_request<KT>(*a, b, false);
    } while (r.n == 0);
  }
};

// fp16 / bf16: instruction descriptors with B K-major (S) and N-major (P V), packing, and the bits of a non-finite value
template <typename T> struct DaType;
template <> struct DaType<__half> {
  static __host__ __device__ constexpr uint32_t idesc(int n) { return idesc_f16(DA_ROWS, n); }
  static constexpr uint32_t kExp = 0x7c00u;
};
template <> struct DaType<__nv_bfloat16> {
  static __host__ __device__ constexpr uint32_t idesc(int n) { return idesc_bf16(DA_ROWS, n); }
  static constexpr uint32_t kExp = 0x7f80u;
};
constexpr uint32_t DA_B_N_MAJOR = 1u << 16;

// Shared-memory descriptor of an N-major operand in 128-byte swizzle: blocks of 64 n-elements (128 bytes) `block_bytes`
// apart (leading byte offset), in each 8 k-rows are 1024 bytes (stride byte offset).
__device__ __forceinline__ uint64_t sw128_n_major_desc(uint32_t saddr, uint32_t block_bytes) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)(block_bytes >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// D[tmem] (+)= A[tmem] B[smem], kind::f16: A's 16-bit elements two a column, one lane a row.
__device__ __forceinline__ void mma_tmem_a(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(smem_dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

// 32 packed 32-bit values a thread into TMEM columns taddr .. taddr + 31 of its lane; completes with tmem_st_wait.
__device__ __forceinline__ void tmem_st32_async(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

struct DaBox {  // one lane's TMA box of a K or V tile
  int kind;     // 0: none, 1: cache, 2: drafted
  int row, page, head;
};

template <int D, typename T>
__global__ void __launch_bounds__(DA_THREADS, 1)
draft_attn_kernel(const __grid_constant__ CUtensorMap tm_ck, const __grid_constant__ CUtensorMap tm_cv,
                  const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const __grid_constant__ DraftAttnArgs a, const DaPlan plan, DaSplit* splits, float* partials) {
  constexpr int KT = da_tile(D), NC = D / 64, BUF = da_buffer_bytes(D);
  constexpr uint32_t O_COL = 2 * KT;
  extern __shared__ __align__(1024) uint8_t da_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(da_smem_raw) + 1023) & ~uintptr_t(1023));
  const int q_buf = plan.q_rows * D * 2, q_box = plan.q_rows * 128;
  uint8_t* qs = smem;                            // [q_bufs][NC][q_rows][128 B], SW128
  uint8_t* kvs = qs + plan.q_bufs * q_buf;       // [kv_bufs][NC][KT][128 B], SW128
  uint64_t* bars = reinterpret_cast<uint64_t*>(kvs + plan.kv_bufs * BUF);
  uint64_t* full = bars;                         // [kv_bufs <= 12] a tile has landed
  uint64_t* empty = full + 12;                   // [kv_bufs] the products that read it are done
  uint64_t* q_full = empty + 12;                 // [2]
  uint64_t* q_empty = q_full + 2;                // [2]
  uint64_t* s_full = q_empty + 2;                // [2] S of even / odd tiles
  uint64_t* p_full = s_full + 2;                 // [2] P of a tile is written, O rescaled, V mended
  uint64_t* pv_done = p_full + 2;                // [2] O includes the tile
  uint64_t* all_done = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(all_done + 1);
  int* poison = reinterpret_cast<int*>(tmem_slot + 1);  // [2] of even / odd items: item + 1 if it met a non-finite V
  int* low_max = poison + 2;                     // [4] a softmax warp's largest row bound
  int64_t* s_scan = reinterpret_cast<int64_t*>(((uintptr_t)(low_max + 4) + 7) & ~uintptr_t(7));  // [8] warp sums, then
  int* s_start = reinterpret_cast<int*>(s_scan + 8);  // the piece's first request

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, piece = blockIdx.x;
  const int G = a.hq / a.hkv;
  if (tid == 0) {
    for (int i = 0; i < plan.kv_bufs; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 64);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(all_done, 1);
    fence_barrier_init();
    prefetch_tmap(&tm_ck);
    prefetch_tmap(&tm_cv);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    poison[0] = poison[1] = 0;
    *s_start = -1;
  }
  if (warp == 1) tmem_alloc(tmem_slot, DA_TMEM_COLS);
  pdl_trigger();

  // ---- this piece of the line: requests' tile counts summed over the block ----
  const int per = (a.rows + DA_THREADS - 1) / DA_THREADS, rb0 = min(a.rows, tid * per), rb1 = min(a.rows, rb0 + per);
  auto tiles_of = [&](int b, bool report) -> int64_t {
    const DaReq r = da_request<KT>(a, b, report);
    return (int64_t)r.n * r.blocks * a.hkv;
  };
  int64_t mine = 0;
  for (int b = rb0; b < rb1; ++b) mine += tiles_of(b, piece == 0);
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) s_scan[warp] = upto;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int64_t total = 0, before = upto - mine;
  for (int w = 0; w < DA_THREADS / 32; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  const int64_t even = (total + plan.pieces - 1) / plan.pieces, step = even < DA_MIN_TILES ? DA_MIN_TILES : even;
  const int64_t w0 = piece * step < total ? piece * step : total, w1 = w0 + step < total ? w0 + step : total;
  const int n_tiles = (int)(w1 - w0);
  if (n_tiles > 0 && w0 >= before && w0 < before + mine) {
    int64_t at = before;
    for (int b = rb0; b < rb1; ++b) {
      const int64_t n = tiles_of(b, false);
      if (w0 < at + n) {
        s_start[0] = b;
        *reinterpret_cast<int64_t*>(s_start + 2) = w0 - at;
        break;
      }
      at += n;
    }
  }
  if (tid == 0) splits[piece].last = -1;
  __syncthreads();
  const uint32_t tmem = *tmem_slot;
  int issued = 0;  // warp 0: tiles requested
  if (n_tiles > 0) {
    DaWalk<KT> walk;
    walk.start(a, s_start[0], *reinterpret_cast<const int64_t*>(s_start + 2));
    // K of tile g is the ring's entry 0 (g = 0) or 2 g - 1, V of tile g entry 2 g + 2, or 2 g + 1 for the last
    auto v_entry = [&](int g) { return g + 1 < n_tiles ? 2 * g + 2 : 2 * g + 1; };
    if (warp == 0) {
      // ---- K and V tiles: every lane one box ----
      const int rb = lane / NC, cb = lane % NC;
      auto box_of = [&](const DaWalk<KT>& w) {
        DaBox x{0, 0, 0, w.h};
        if (w.i < w.r.cached) {
          const int pos = (w.r.first + w.i) * KT + rb * plan.box;
          if (rb < KT / plan.box && pos < w.r.len && pos + plan.box > w.r.lo) {
            const int p = pos / a.cache.page;
            x.kind = 1;
            x.row = pos - p * a.cache.page;
            x.page = a.table[w.b * a.table_stride + p];
          }
        } else {
          const int j = (w.i - w.r.cached) * KT + rb * 8;
          if (rb < KT / 8 && j < w.r.fresh) {
            x.kind = 2;
            x.row = w.r.t0 + j;
          }
        }
        return x;
      };
      bool ok = true;
      auto bring = [&](const DaBox& x, bool v) {
        const int s = issued % plan.kv_bufs, turn = issued / plan.kv_bufs;
        if (turn > 0) ok = mbar_wait(&empty[s], (turn - 1) & 1, a.err, ERR_TIMEOUT_MMA);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        const bool in_cache = x.kind == 1 && x.page >= 0 && x.page < a.cache.pages;
        if (x.kind == 1 && !in_cache) set_error(a.err, ERR_BAD_PAGE);
        const unsigned c = __ballot_sync(0xffffffffu, in_cache), d = __ballot_sync(0xffffffffu, x.kind == 2);
        if (lane == 0) mbar_arrive_expect_tx(&full[s], __popc(c) * plan.box * 128 + __popc(d) * 8 * 128);
        __syncwarp();
        uint8_t* dst = kvs + s * BUF + cb * KT * 128 + rb * (x.kind == 1 ? plan.box : 8) * 128;
        if (in_cache) tma_load_4d(dst, v ? &tm_cv : &tm_ck, cb * 64, x.row, x.head, x.page, &full[s]);
        if (x.kind == 2) tma_load_3d(dst, v ? &tm_v : &tm_k, cb * 64, x.row, x.head, &full[s]);
        ++issued;
      };
      DaBox cur = box_of(walk), next = cur, later = cur;
      if (n_tiles > 1) {
        walk.skip(1);
        next = box_of(walk);
      }
      bring(cur, false);
      for (int g = 0; g < n_tiles && ok; ++g) {
        if (g + 2 < n_tiles) {  // the table entries of the tile after the next, ahead of the waits
          walk.skip(1);
          later = box_of(walk);
        }
        if (g + 1 < n_tiles) bring(next, false);
        if (ok) bring(cur, true);
        cur = next;
        next = later;
      }
    } else if (warp == 1) {
      // ---- products ----
      if (lane == 0) {
        bool ok = true;
        const uint32_t idesc_s = DaType<T>::idesc(KT), idesc_o = DaType<T>::idesc(D) | DA_B_N_MAJOR;
        int entry = 0, item = -1;
        bool begins = true;
        auto score = [&](int g) {  // S of tile g (the walk's place), then the walk moves on
          if (begins) {
            ++item;
            ok = mbar_wait(&q_full[item % plan.q_bufs], (item / plan.q_bufs) & 1, a.err, ERR_TIMEOUT_MMA);
          }
          if (ok) ok = mbar_wait(&full[entry % plan.kv_bufs], (entry / plan.kv_bufs) & 1, a.err, ERR_TIMEOUT_TMA);
          if (!ok) return;
          tc_fence_after();
          const uint32_t qb = smem_u32(qs + (item % plan.q_bufs) * q_buf), kb = smem_u32(kvs + (entry % plan.kv_bufs) * BUF);
          const uint32_t d = tmem + (uint32_t)((g & 1) * KT);
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_bf16(d, sw128_desc(qb + c * q_box + kk * 32), sw128_desc(kb + c * KT * 128 + kk * 32), idesc_s,
                       (c > 0 || kk > 0) ? 1u : 0u);
          mma_commit(&s_full[g & 1]);
          mma_commit(&empty[entry % plan.kv_bufs]);
          const bool ends = walk.i + 1 == walk.r.n || g + 1 == n_tiles;
          if (ends) mma_commit(&q_empty[item % plan.q_bufs]);
          begins = ends;
          if (g + 1 < n_tiles) walk.skip(1);
          ++entry;
        };
        bool first = true;  // of its item (or of this piece's part of it)
        score(0);
        for (int g = 0; g < n_tiles && ok; ++g) {
          const bool ends = begins;  // the tile that was scored last is the last of its item: tile g
          if (g + 1 < n_tiles) score(g + 1);
          if (ok) ok = mbar_wait(&p_full[g & 1], (g >> 1) & 1, a.err, ERR_TIMEOUT_MMA);
          if (ok) ok = mbar_wait(&full[entry % plan.kv_bufs], (entry / plan.kv_bufs) & 1, a.err, ERR_TIMEOUT_TMA);
          if (!ok) break;
          tc_fence_after();
          const uint32_t vb = smem_u32(kvs + (entry % plan.kv_bufs) * BUF), p = tmem + (uint32_t)((g & 1) * KT);
#pragma unroll
          for (int kk = 0; kk < KT / 16; ++kk)
            mma_tmem_a(tmem + O_COL, p + kk * 8, sw128_n_major_desc(vb + kk * 2048, KT * 128), idesc_o,
                       (!first || kk > 0) ? 1u : 0u);
          mma_commit(&pv_done[g & 1]);
          mma_commit(&empty[entry % plan.kv_bufs]);
          ++entry;
          first = ends;
        }
      }
    } else if (warp < 4) {
      // ---- Q rows of every item into its buffer ----
      bool ok = true;
      int left = n_tiles;
      for (int item = 0; left > 0; ++item) {
        const int s = item % plan.q_bufs, turn = item / plan.q_bufs;
        if (ok && turn > 0) ok = mbar_wait(&q_empty[s], (turn - 1) & 1, a.err, ERR_TIMEOUT_MMA);
        const int rows = min(DA_ROWS, walk.r.fresh * G - walk.block * DA_ROWS);
        for (int c = tid - 64; c < rows * (D / 8); c += 64) {
          const int r = c / (D / 8), ch = c % (D / 8), all = walk.block * DA_ROWS + r;
          const T* src = (const T*)a.q + (int64_t)(walk.r.t0 + all / G) * a.q_ts + (int64_t)(walk.h * G + all % G) * a.q_hs;
          *reinterpret_cast<uint4*>(qs + s * q_buf + (ch >> 3) * q_box + sw128_off(r, ch & 7)) =
              *reinterpret_cast<const uint4*>(src + ch * 8);
        }
        fence_proxy_async();
        mbar_arrive(&q_full[s]);
        const int tiles = min(left, walk.r.n - walk.i);
        left -= tiles;
        walk.skip(tiles);
      }
    } else {
      // ---- softmax: thread = row = TMEM lane ----
      bool ok = true;
      const int row = tid - 128;
      const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
      const float sl2 = a.scale * 1.4426950408889634f;  // scores in log2 units
      int g = 0;
      for (int item = 0; g < n_tiles; ++item) {
        const DaReq r = walk.r;
        const int all = walk.block * DA_ROWS + row, tok = all / G;
        const bool valid = tok < r.fresh;
        const bool live = (walk.block * DA_ROWS + (row & ~31)) / G < r.fresh;  // some row of this warp is
        const int i0 = walk.i, i1 = min(r.n, i0 + n_tiles - g);
        // keys of this row are those at positions above `low`
        int low = r.lo - 1, lows = -1;
        if (a.window) {
          if (valid) low = max(low, (a.positions ? a.positions[r.t0 + tok] : r.len + tok) - a.window);
          int x = valid ? low : -1;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) x = max(x, __shfl_xor_sync(0xffffffffu, x, o));
          named_sync_id<2, 128>();  // the last item's readers are done
          if (lane == 0) low_max[warp & 3] = x;
          named_sync_id<2, 128>();
          lows = max(max(low_max[0], low_max[1]), max(low_max[2], low_max[3]));
        }
        float m = -INFINITY, l = 0.f;
        for (int i = i0; i < i1; ++i, ++g) {
          const bool tree = i >= r.cached;
          const int base = tree ? (i - r.cached) * KT : (r.first + i) * KT;  // first key: drafted index or position
          const int end = min(KT, (tree ? r.fresh : r.len) - base);          // keys that exist
          const int begin = tree ? 0 : max(0, r.lo - base);
          const bool some = tree || (a.window && base <= lows);              // not every row sees the same keys
          if (ok) ok = mbar_wait(&s_full[g & 1], (g >> 1) & 1, a.err, ERR_TIMEOUT_MMA);
          tc_fence_after();
          __syncwarp();
          if (live) {
            float sc[KT];
#pragma unroll
            for (int c = 0; c < KT; c += 32) tmem_ld32(lanes + (uint32_t)((g & 1) * KT + c), *reinterpret_cast<float(*)[32]>(sc + c));
            if (some || begin > 0 || end < KT) {
              uint32_t vis[KT / 32];
#pragma unroll
              for (int w = 0; w < KT / 32; ++w) {
                const int from = tree ? 0 : max(0, low + 1 - base), z = min(32, max(0, end - 32 * w));
                const int f = min(32, max(0, from - 32 * w));
                uint32_t bits = (z == 32 ? ~0u : (1u << z) - 1u) & (f == 32 ? 0u : ~0u << f);
                if (tree && valid) {
                  const int word = (base >> 5) + w;
                  if (a.mask)
                    bits &= word < a.words ? a.mask[(int64_t)(r.t0 + tok) * a.words + word] : 0u;
                  else
                    bits &= tok >= base + 32 * w + 31 ? ~0u : tok < base + 32 * w ? 0u : (2u << (tok - base - 32 * w)) - 1u;
                  if (a.window) {
                    for (uint32_t rest = bits; rest; rest &= rest - 1) {
                      const int j = base + 32 * w + __ffs(rest) - 1;
                      if ((a.positions ? a.positions[r.t0 + j] : r.len + j) <= low) bits &= ~(rest & -rest);
                    }
                  }
                }
                vis[w] = bits;
              }
#pragma unroll
              for (int j = 0; j < KT; ++j) sc[j] = vis[j >> 5] >> (j & 31) & 1 ? sc[j] : -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < KT; ++j) top = fmaxf(top, sc[j]);
            top *= sl2;
            // the maximum is raised only when a tile exceeds it by 2^8: weights stay below that, which fp16 holds
            const bool raise = valid && (top > m + 8.f || (m == -INFINITY && top > -INFINITY));
            const float alpha = raise && m > -INFINITY ? ex2_approx(m - top) : raise ? 0.f : 1.f;
            if (raise) {
              m = top;
              l *= alpha;
            }
            if (i > i0 && __any_sync(0xffffffffu, raise)) {
              if (ok) ok = mbar_wait(&pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, a.err, ERR_TIMEOUT_MMA);
              tc_fence_after();
              __syncwarp();
#pragma unroll 1
              for (int c = 0; c < D; c += 32) {
                float o[32];
                tmem_ld32(lanes + O_COL + c, o);
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] *= alpha;
                tmem_st32(lanes + O_COL + c, o);
              }
            }
            const float base_m = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int c = 0; c < KT; c += 64) {
              uint32_t pk[32];
#pragma unroll
              for (int j = 0; j < 64; j += 2) {
                const float p0 = ex2_approx(fmaf(sc[c + j], sl2, -base_m)), p1 = ex2_approx(fmaf(sc[c + j + 1], sl2, -base_m));
                l += p0 + p1;
                pk[j >> 1] = pack2(p0, p1, (const T*)nullptr);
              }
              __syncwarp();
              tmem_st32_async(lanes + (uint32_t)((g & 1) * KT + c / 2), pk);
            }
            tmem_st_wait();
          }
          if (some || begin > 0 || end < KT) {
            // V rows that nobody sees become 0 (0 times whatever lay there must not count); where rows differ in what
            // they see, so do V's infinities and NaN, which the epilogue puts back for the rows that see them
            const int e = v_entry(g);
            if (ok) ok = mbar_wait(&full[e % plan.kv_bufs], (e / plan.kv_bufs) & 1, a.err, ERR_TIMEOUT_TMA);
            uint8_t* vb = kvs + (e % plan.kv_bufs) * BUF;
            for (int c = row; c < KT * (D / 8); c += 128) {
              const int k = c / (D / 8), ch = c % (D / 8);
              uint4* at = reinterpret_cast<uint4*>(vb + (ch >> 3) * KT * 128 + sw128_off(k, ch & 7));
              if (k < begin || k >= end) {
                *at = make_uint4(0u, 0u, 0u, 0u);
              } else if (some) {
                uint4 v = *at;
                uint32_t* w = reinterpret_cast<uint32_t*>(&v);
                bool bad = false;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  constexpr uint32_t E = DaType<T>::kExp;
                  const bool lo_bad = (w[q] & E) == E, hi_bad = (w[q] >> 16 & E) == E;
                  bad |= lo_bad | hi_bad;
                  w[q] &= (lo_bad ? 0u : 0xffffu) | (hi_bad ? 0u : 0xffff0000u);
                }
                if (bad) {
                  *at = v;
                  poison[item & 1] = item + 1;
                }
              }
            }
            fence_proxy_async();
          }
          tc_fence_before();
          mbar_arrive(&p_full[g & 1]);
        }
        // ---- epilogue of the item, or of this piece's part of it ----
        if (ok) ok = mbar_wait(&pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, a.err, ERR_TIMEOUT_MMA);
        tc_fence_after();
        named_sync_id<2, 128>();  // every warp's poison is written (the next item's goes to the other word)
        const bool mend = poison[item & 1] == item + 1;
        const bool whole = i0 == 0 && i1 == r.n;
        const int slot = 2 * piece + (item > 0 ? 1 : 0);
        float* part = partials + slot * da_partial_floats(D);
        const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
        const int64_t orow = (int64_t)(r.t0 + tok) * a.hq + walk.h * G + all % G;
        if (live) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            float o[32];
            __syncwarp();
            tmem_ld32(lanes + O_COL + c, o);
            if (!valid) continue;
            if (mend) {  // rare, and slow: key after key
              for (int i = i0; i < i1; ++i) {
                const bool tree = i >= r.cached;
                const int base = tree ? (i - r.cached) * KT : (r.first + i) * KT;
                if (!tree && !(a.window && base <= lows)) continue;
                for (int j = base; j < base + KT && j < (tree ? r.fresh : r.len); ++j) {
                  const T* v;
                  if (tree) {
                    if (a.mask ? (j >= 32 * a.words || !(a.mask[(int64_t)(r.t0 + tok) * a.words + (j >> 5)] >> (j & 31) & 1)) : j > tok) continue;
                    if (a.window && (a.positions ? a.positions[r.t0 + j] : r.len + j) <= low) continue;
                    v = (const T*)a.v + (int64_t)(r.t0 + j) * a.v_ts + (int64_t)walk.h * a.v_hs;
                  } else {
                    if (j <= low) continue;
                    const int pg = a.table[walk.b * a.table_stride + j / a.cache.page];
                    if (pg < 0 || pg >= a.cache.pages) continue;
                    v = (const T*)a.cache.v + pg * a.cache.page_stride + j % a.cache.page * a.cache.token_stride +
                        walk.h * a.cache.head_stride;
                  }
#pragma unroll
                  for (int x = 0; x < 32; ++x) {
                    const float f = (float)v[c + x];
                    if (!(fabsf(f) < INFINITY)) o[x] += f;
                  }
                }
              }
            }
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
          if (valid) {
            if (!whole)
              *reinterpret_cast<float2*>(part + DA_ROWS * D + 2 * row) = make_float2(m, l);
            else if (a.lse)
              a.lse[orow] = l > 0.f || l != l ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
          }
        }
        if (row == 0 && i0 == 0 && i1 < r.n) {
          const int64_t start = w0 + g - (i1 - i0);
          splits[piece] = DaSplit{walk.b, walk.h, walk.block, (int)((start + r.n - 1) / step), slot, {0, 0, 0}};
        }
        tc_fence_before();
        walk.skip(i1 - i0);
      }
    }
  }
  // ---- teardown: roles are done or have given up; products and copies in flight end before the memory goes ----
  __syncwarp();
  if (warp == 0) {
    for (int e = max(0, issued - plan.kv_bufs); e < issued; ++e)
      mbar_wait(&full[e % plan.kv_bufs], (e / plan.kv_bufs) & 1, nullptr, 0);
  }
  if (tid == 32) {
    mma_commit(all_done);
    mbar_wait(all_done, 0, a.err, ERR_TIMEOUT_MMA);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, DA_TMEM_COLS);
  }
}

constexpr int DJ_THREADS = 256;

// Joins the parts of an item that was cut: one warp a row, parts in piece order. Block (c, y): the item that begins in
// piece c, rows 8 y .. 8 y + 7.
template <int D, typename T>
__global__ void __launch_bounds__(DJ_THREADS) draft_join_kernel(const __grid_constant__ DraftAttnArgs a,
                                                                const DaSplit* splits, const float* partials) {
  pdl_wait();
  const int c = blockIdx.x, lane = threadIdx.x & 31;
  const DaSplit s = splits[c];
  if (s.last < 0) return;
  const int row = blockIdx.y * (DJ_THREADS / 32) + (threadIdx.x >> 5), G = a.hq / a.hkv;
  const int all = s.block * DA_ROWS + row, tok = all / G, t0 = a.cu[s.b];
  if (tok >= a.cu[s.b + 1] - t0) return;
  const size_t size = da_partial_floats(D);
  auto part = [&](int p) { return partials + (p == c ? (size_t)s.first_slot : 2 * (size_t)p) * size; };
  float m = -INFINITY;
  for (int p = c + lane; p <= s.last; p += 32) {
    const float x = part(p)[DA_ROWS * D + 2 * row];
    m = fmaxf(m, x);
  }
  m = warp_max(m);
  float l = 0.f, o[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) o[e] = 0.f;
  for (int p = c; p <= s.last; ++p) {
    const float* x = part(p);
    const float2 ml = *reinterpret_cast<const float2*>(x + DA_ROWS * D + 2 * row);
    const float w = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - m);
    if (ml.x == -INFINITY && ml.y == 0.f) continue;  // saw nothing
    l += ml.y * w;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) o[e] += w * x[row * D + e * 32 + lane];
  }
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
  const int64_t orow = (int64_t)(t0 + tok) * a.hq + s.h * G + all % G;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) ((T*)a.out)[orow * D + e * 32 + lane] = (T)(o[e] * inv);
  if (lane == 0 && a.lse) a.lse[orow] = l > 0.f || l != l ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace hsg
