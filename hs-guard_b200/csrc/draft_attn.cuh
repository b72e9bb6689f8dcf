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
// product, row r = (token r / G, query head r % G of the group of G); as many whole tokens as fit 128 rows and all of a
// request's keys in tiles of KT (128, or 64 at head dim 256) are an item (request, key head, block of tokens). All items' tiles, in order, are one
// line that is cut into equal pieces, one a thread block, whatever the requests' lengths, so a long cache is split over
// many SMs and short ones share one; the lengths are read on the device. An item that lies in one piece is written
// out; of one that is cut, each piece leaves its unnormalised sums, row maxima and row sums in the workspace and
// draft_join_kernel joins them in piece order, so results do not depend on timing.
//
// Per tile: S = Q K^T (tcgen05, TMEM), softmax with a running maximum in registers (a row a thread), P in the type of V
// written over S in TMEM, O += P V (A = P from TMEM, B = V as it lies in shared memory, N-major). Warps 0 and 3 bring K
// and V tiles by TMA, eight tokens of one page a box, through one ring of buffers in the order in which the products use
// them; warp 1 issues the products, S of the next tile before P V of this one; warp 2 brings Q; warps 4-7 do the
// softmax and the epilogue. A K or V tile lies in shared memory as [8 keys][dim / 64][8][128 B], 128-byte swizzle: boxes
// of any page size then sit at one stride, which is all that a product's descriptor can say. Warp 1 runs as a whole warp
// with one elected lane at each group of products, so that their descriptors stay in uniform registers: issued from a
// branch on the lane, each took about 150 cycles. Copies are the other way round: 32 lanes with a box each take 64 to 95
// cycles a box (1 to 4 KB), one elected lane in a loop over boxes 135 to 240, and one warp alone falls short of HBM. Tiles of the next item are under way during an item's epilogue.
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
  int block;     // drafted tokens of an item: at most 128 rows
  int q_rows;    // rows a Q buffer holds: block * G rounded up to a multiple of 8
  int q_bufs;
  int kv_bufs;
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
__device__ __forceinline__ DaReq da_request(const DraftAttnArgs& a, int block, int b, bool report) {
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
  r.blocks = (r.fresh + block - 1) / block;
  return r;
}

// A place on the line of tiles.
template <int KT>
struct DaWalk {
  const DraftAttnArgs* a;
  DaReq r;
  int size;  // tokens of a block
  int b, h, block, i;
  __device__ __forceinline__ void start(const DraftAttnArgs& args, int block_size, int b0, int64_t within) {
    a = &args;
    size = block_size;
    b = b0;
    r = da_request<KT>(args, size, b, false);
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
      r = da_request<KT>(*a, size, b, false);
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

// Shared-memory descriptors of a tile that lies as [8 keys][NC][8][128 B] in 128-byte swizzle: as a K-major operand (S:
// rows are keys, stride byte offset from 8 keys to the next 8) and as an N-major one (P V: leading byte offset from 64
// dims to the next 64, stride byte offset from 8 keys to the next 8).
template <int NC> __device__ __forceinline__ uint64_t da_k_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(NC * 1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
template <int NC> __device__ __forceinline__ uint64_t da_v_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)(1024 >> 4) << 16 | (uint64_t)(NC * 1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Byte offset of 16-byte piece ch of key k in such a tile.
template <int NC> __device__ __forceinline__ uint32_t da_offset(int k, int ch) {
  return (uint32_t)(((k >> 3) * NC + (ch >> 3)) * 1024) + sw128_off(k & 7, ch & 7);
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

// true in one lane of a converged warp, always the same one
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(smem_dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(void* smem_dst, const CUtensorMap* map, int x, int y, int z, int w, int u,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
      "[%7];" ::"r"(smem_u32(smem_dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(u), "r"(smem_u32(bar))
      : "memory");
}

// TMEM columns taddr .. taddr + 31 of a thread's lane, complete after tmem_ld_wait; da_pin keeps what uses them behind it.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void da_pin(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]),
                 "+r"(r[i + 6]), "+r"(r[i + 7]));
}
// 32 packed 32-bit values a thread into TMEM columns taddr .. taddr + 31 of its lane; complete after tmem_st_wait.
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

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Position in a ring of buffers and the parity of its use.
struct DaRing {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int size) {
    if (++at == size) {
      at = 0;
      phase ^= 1u;
    }
  }
};

// What a lane fetches of a K or V tile: eight keys.
struct DaFetch {
  int row, page;  // token within the page and page id, or drafted token
  int drafted, head;
  bool mine;      // some of them exist
};

template <int D, typename T>
__global__ void __launch_bounds__(DA_THREADS, 1)
draft_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_ck,
                  const __grid_constant__ CUtensorMap tm_cv, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ DraftAttnArgs a, const DaPlan plan,
                  DaSplit* splits, float* partials) {
  constexpr int KT = da_tile(D), NC = D / 64, BUF = da_buffer_bytes(D);
  constexpr uint32_t O_COL = 2 * KT;
  extern __shared__ __align__(1024) uint8_t da_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(da_smem_raw) + 1023) & ~uintptr_t(1023));
  const int q_buf = plan.q_rows * D * 2, q_box = plan.q_rows * 128;
  uint8_t* qs = smem;                            // [q_bufs][NC][q_rows][128 B], SW128
  uint8_t* kvs = qs + plan.q_bufs * q_buf;       // [kv_bufs][KT / 8][NC][8][128 B], SW128
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

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, piece = blockIdx.x;
  const int G = a.hq / a.hkv;
  if (tid == 0) {
    for (int i = 0; i < plan.kv_bufs; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(all_done, 1);
    fence_barrier_init();
    prefetch_tmap(&tm_q);
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
    const DaReq r = da_request<KT>(a, plan.block, b, report);
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
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  bool ok = true;  // no wait of this thread has given up
  int issued = 0;  // warps 0 and 3: ring entries up to their last one; warp 2: Q tiles
  if (n_tiles > 0) {
    DaWalk<KT> walk;
    walk.start(a, plan.block, s_start[0], *reinterpret_cast<const int64_t*>(s_start + 2));
    // K and V of tile g are the ring's entries 2 g - 1 (0 for g = 0) and 2 g + 2 (2 g + 1 for the last)
    if (warp == 0 || warp == 3) {
      // ---- K tiles (warp 0) and V tiles (warp 3): lane i brings keys 8 i .. 8 i + 7 ----
      const bool is_v = warp == 3;
      const CUtensorMap *cache = is_v ? &tm_cv : &tm_ck, *drafted = is_v ? &tm_v : &tm_k;
      auto fetch_of = [&](const DaWalk<KT>& w) {
        DaFetch x{0, -1, 0, w.h, false};
        if (w.i < w.r.cached) {
          const int base = (w.r.first + w.i) * KT, pos = base + lane * 8;
          x.mine = lane < KT / 8 && pos < w.r.len && pos + 8 > w.r.lo;
          if (x.mine) {
            const int p = pos / a.cache.page;
            x.row = pos - p * a.cache.page;
            x.page = a.table[w.b * a.table_stride + p];
          }
        } else {
          const int j = (w.i - w.r.cached) * KT + lane * 8;
          x.mine = lane < KT / 8 && j < w.r.fresh;
          x.row = w.r.t0 + j;
          x.drafted = 1;
        }
        return x;
      };
      DaRing ring;
      if (is_v) ring.next(plan.kv_bufs);
      DaFetch cur = fetch_of(walk), next = cur;
      for (int g = 0; g < n_tiles && ok; ++g) {
        if (g + 1 < n_tiles) {  // the next tile's table entries, ahead of the wait
          walk.skip(1);
          next = fetch_of(walk);
        }
        if (is_v && g + 1 < n_tiles) ring.next(plan.kv_bufs);
        const int e = is_v ? (g + 1 < n_tiles ? 2 * g + 2 : 2 * g + 1) : g ? 2 * g - 1 : 0;
        if (e >= plan.kv_bufs) ok = __all_sync(0xffffffffu, mbar_wait(&empty[ring.at], ring.phase ^ 1u, a.err, ERR_TIMEOUT_MMA));
        if (!ok) break;
        const bool good = cur.drafted || (cur.page >= 0 && cur.page < a.cache.pages);
        if (cur.mine && !good) set_error(a.err, ERR_BAD_PAGE);
        const bool bring = cur.mine && good;
        const unsigned boxes = __ballot_sync(0xffffffffu, bring);
        uint8_t* dst = kvs + ring.at * BUF + lane * NC * 1024;
        if (lane == 0) mbar_arrive_expect_tx(&full[ring.at], __popc(boxes) * (NC * 1024));
        __syncwarp();
        if (bring) {
          if (cur.drafted) tma_load_4d(dst, drafted, 0, cur.row, 0, cur.head, &full[ring.at]);
          else tma_load_5d(dst, cache, 0, cur.row, 0, cur.head, cur.page, &full[ring.at]);
        }
        issued = e + 1;
        ring.next(plan.kv_bufs);
        if (!is_v && g > 0) ring.next(plan.kv_bufs);
        cur = next;
      }
    } else if (warp == 1) {
      // ---- products ----
      const uint32_t idesc_s = DaType<T>::idesc(KT), idesc_o = DaType<T>::idesc(D) | DA_B_N_MAJOR;
      DaRing ring, q_ring;
      bool begins = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, a.err, code));
      };
      auto score = [&](int g) {  // S of tile g (the walk's place), then the walk moves on
        if (begins) wait(&q_full[q_ring.at], q_ring.phase, ERR_TIMEOUT_TMA);
        wait(&full[ring.at], ring.phase, ERR_TIMEOUT_TMA);
        if (!ok) return;
        tc_fence_after();
        const bool ends = __shfl_sync(0xffffffffu, (int)(walk.i + 1 == walk.r.n), 0) || g + 1 == n_tiles;
        const uint64_t qd = sw128_desc(smem_u32(qs + q_ring.at * q_buf)), kd = da_k_desc<NC>(smem_u32(kvs + ring.at * BUF));
        const uint32_t d = tmem + (uint32_t)((g & 1) * KT);
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_bf16(d, qd + (uint64_t)((c * q_box + kk * 32) >> 4), kd + (uint64_t)((c * 1024 + kk * 32) >> 4), idesc_s,
                       (c > 0 || kk > 0) ? 1u : 0u);
          mma_commit(&s_full[g & 1]);
          mma_commit(&empty[ring.at]);
          if (ends) mma_commit(&q_empty[q_ring.at]);
        }
        __syncwarp();
        if (ends) q_ring.next(plan.q_bufs);
        begins = ends;
        if (g + 1 < n_tiles) walk.skip(1);
        ring.next(plan.kv_bufs);
      };
      bool first = true;  // of its item (or of this piece's part of it)
      score(0);
      for (int g = 0; g < n_tiles && ok; ++g) {
        const bool ends = begins;  // the tile that was scored last, tile g, is the last of its item
        if (g + 1 < n_tiles) score(g + 1);
        wait(&p_full[g & 1], (g >> 1) & 1, ERR_TIMEOUT_MMA);
        wait(&full[ring.at], ring.phase, ERR_TIMEOUT_TMA);
        if (!ok) break;
        tc_fence_after();
        const uint64_t vd = da_v_desc<NC>(smem_u32(kvs + ring.at * BUF));
        const uint32_t p = tmem + (uint32_t)((g & 1) * KT);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < KT / 16; ++kk)
            mma_tmem_a(tmem + O_COL, p + kk * 8, vd + (uint64_t)((kk * 2 * NC * 1024) >> 4), idesc_o,
                       (!first || kk > 0) ? 1u : 0u);
          mma_commit(&pv_done[g & 1]);
          mma_commit(&empty[ring.at]);
        }
        __syncwarp();
        ring.next(plan.kv_bufs);
        first = ends;
      }
    } else if (warp == 2) {
      // ---- Q of every item: block tokens x G heads, one box for each 64 dims ----
      DaRing ring;
      int left = n_tiles;
      for (int item = 0; left > 0 && ok; ++item) {
        if (item >= plan.q_bufs) ok = __all_sync(0xffffffffu, mbar_wait(&q_empty[ring.at], ring.phase ^ 1u, a.err, ERR_TIMEOUT_MMA));
        if (!ok) break;
        const int token = __shfl_sync(0xffffffffu, walk.r.t0 + walk.block * plan.block, 0);
        const int head = __shfl_sync(0xffffffffu, walk.h * G, 0);
        if (elect_one()) {
          mbar_arrive_expect_tx(&q_full[ring.at], plan.block * G * D * 2);
#pragma unroll
          for (int c = 0; c < NC; ++c)
            tma_load_3d(qs + ring.at * q_buf + c * q_box, &tm_q, c * 64, head, token, &q_full[ring.at]);
        }
        __syncwarp();
        ++issued;
        ring.next(plan.q_bufs);
        const int tiles = min(left, walk.r.n - walk.i);
        left -= tiles;
        walk.skip(tiles);
      }
    } else if (warp >= 4) {
      // ---- softmax: thread = row = TMEM lane ----
      const int row = tid - 128;
      const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
      const float sl2 = a.scale * 1.4426950408889634f;  // scores in log2 units
      int g = 0;
      for (int item = 0; g < n_tiles; ++item) {
        const DaReq r = walk.r;
        const int tok = walk.block * plan.block + row / G;
        const bool valid = row < plan.block * G && tok < r.fresh;
        const bool live = __any_sync(0xffffffffu, valid);
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
          const bool special = some || begin > 0 || end < KT;
          if (ok) ok = mbar_wait(&s_full[g & 1], (g >> 1) & 1, a.err, ERR_TIMEOUT_MMA);
          tc_fence_after();
          __syncwarp();
          if (live) {
            uint32_t sc[KT];
#pragma unroll
            for (int c = 0; c < KT; c += 32) tmem_ld32_async(lanes + (uint32_t)((g & 1) * KT + c), sc + c);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < KT; c += 32) da_pin(sc + c);
            auto at = [&](int j) { return __uint_as_float(sc[j]); };
            if (special) {
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
#pragma unroll
                for (int j = 0; j < 32; ++j) sc[32 * w + j] = bits >> j & 1 ? sc[32 * w + j] : 0xff800000u;  // -inf
              }
            }
            float tops[4] = {at(0), at(1), at(2), at(3)};
#pragma unroll
            for (int j = 4; j + 4 < KT; j += 8)
#pragma unroll
              for (int q = 0; q < 4; ++q) tops[q] = fmaxf(fmaxf(tops[q], at(j + q)), at(j + 4 + q));
#pragma unroll
            for (int q = 0; q < 4; ++q) tops[q] = fmaxf(tops[q], at(KT - 4 + q));
            const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * sl2;
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
            const float2 mul = make_float2(sl2, sl2), off = m == -INFINITY ? make_float2(0.f, 0.f) : make_float2(-m, -m);
            float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            __syncwarp();
#pragma unroll
            for (int c = 0; c < KT; c += 64) {
              uint32_t pk[32];
#pragma unroll
              for (int j = 0; j < 64; j += 2) {
                float2 x = fma2(make_float2(at(c + j), at(c + j + 1)), mul, off);
                x = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                sums[j >> 1 & 1] = add2(sums[j >> 1 & 1], x);
                pk[j >> 1] = pack2(x.x, x.y, (const T*)nullptr);
              }
              tmem_st32_async(lanes + (uint32_t)((g & 1) * KT + c / 2), pk);
            }
            sums[0] = add2(sums[0], sums[1]);
            l += sums[0].x + sums[0].y;
            tmem_st_wait();
          }
          if (special) {
            // V rows that nobody sees become 0 (0 times whatever lay there must not count); where rows differ in what
            // they see, so do V's infinities and NaN, which the epilogue puts back for the rows that see them
            const int e = g + 1 < n_tiles ? 2 * g + 2 : 2 * g + 1;
            if (ok) ok = mbar_wait(&full[e % plan.kv_bufs], (e / plan.kv_bufs) & 1, a.err, ERR_TIMEOUT_TMA);
            uint8_t* vb = kvs + (e % plan.kv_bufs) * BUF;
            for (int c = row; c < KT * (D / 8); c += 128) {
              const int k = c / (D / 8), ch = c % (D / 8);
              uint4* at = reinterpret_cast<uint4*>(vb + da_offset<NC>(k, ch));
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
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[g & 1]);
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
        const int64_t orow = (int64_t)(r.t0 + tok) * a.hq + walk.h * G + row % G;
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
  // ---- teardown. If every role went through, every copy and product has been waited for. If one gave up, those still
  // in flight end before the memory goes. ----
  __syncwarp();
  tc_fence_before();
  if (!__syncthreads_and(ok)) {
    if (warp == 0 || warp == 3) {
      for (int e = max(0, issued - plan.kv_bufs); e < issued; ++e) {
        const bool v_entry = (e > 0 && e % 2 == 0) || e == 2 * n_tiles - 1;
        if (v_entry == (warp == 3)) mbar_wait(&full[e % plan.kv_bufs], (e / plan.kv_bufs) & 1, nullptr, 0);
      }
    } else if (warp == 2) {
      for (int e = max(0, issued - plan.q_bufs); e < issued; ++e)
        mbar_wait(&q_full[e % plan.q_bufs], (e / plan.q_bufs) & 1, nullptr, 0);
    } else if (warp == 1) {
      if (elect_one()) mma_commit(all_done);
      __syncwarp();
      mbar_wait(all_done, 0, nullptr, 0);
    }
    tc_fence_before();
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, DA_TMEM_COLS);
  }
}

constexpr int DJ_THREADS = 256;

// Joins the parts of an item that was cut: one warp a row, parts in piece order. Block (c, y): the item that begins in
// piece c, rows 8 y .. 8 y + 7.
template <int D, typename T>
__global__ void __launch_bounds__(DJ_THREADS) draft_join_kernel(const __grid_constant__ DraftAttnArgs a, int block,
                                                                const DaSplit* splits, const float* partials) {
  pdl_wait();
  const int c = blockIdx.x, lane = threadIdx.x & 31;
  const DaSplit s = splits[c];
  if (s.last < 0) return;
  const int row = blockIdx.y * (DJ_THREADS / 32) + (threadIdx.x >> 5), G = a.hq / a.hkv;
  const int tok = s.block * block + row / G, t0 = a.cu[s.b];
  if (row >= block * G || tok >= a.cu[s.b + 1] - t0) return;
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
  const int64_t orow = (int64_t)(t0 + tok) * a.hq + s.h * G + row % G;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) ((T*)a.out)[orow * D + e * 32 + lane] = (T)(o[e] * inv);
  if (lane == 0 && a.lse) a.lse[orow] = l > 0.f || l != l ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace hsg
