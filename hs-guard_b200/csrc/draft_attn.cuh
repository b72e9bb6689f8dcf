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
// request's keys in tiles of KT (128, or 64 at head dim 256) are an item (request, key head, block of tokens). All items,
// in order, are one line, an item up to DA_ITEM_COST units (its set-up and epilogue) and then a unit a tile long, that is cut
// into equal pieces, one a thread block, whatever the requests' lengths, so a long cache is split over many SMs and short
// ones share one; a few long items are cut into fewer (what a part costs their join is said at the cut). The lengths are
// read on the device. (Without the units for items, pieces with many short ones ran up to half as long again as the mean.)
// An item that lies in one piece is written out; of one that is cut, each piece leaves its unnormalised sums, row maxima
// and row sums in the workspace and draft_join_kernel joins them in piece order, so results do not depend on timing.
//
// Per tile: S = Q K^T (tcgen05, TMEM), softmax with a running maximum in registers (a row a thread), P in the type of V
// written over S in TMEM, O += P V (A = P from TMEM, B = V as it lies in shared memory, N-major). Warps:
//   0   K tiles, and Q of each item; 3: V tiles: TMA, tokens of one page a box, each through a ring of buffers, with a word
//       for each tile that says what the product has to know
//   1   S, up to NS tiles ahead of P V;  2: P V
//   4-7 the softmax of even tiles, 8-11 that of odd ones, one handing the rows' maxima on to the other before its
//       exponentials; whichever has an item's last tile writes the result, while the other goes on to the next item.
//       Warp 3 tells them what an item is, its tokens' positions and first mask words, an item ahead.
// A K or V tile lies in shared memory as [8 keys][dim / 64][8][128 B], 128-byte swizzle: boxes of any page size then sit at
// one stride, which is all that a product's descriptor can say.
//
// What was measured on the way (cycles a tile of 128 rows and 128 keys at head dim 128):
//  - products issued from a branch on the lane took about 150 each, since their descriptors are then not uniform; a whole
//    warp that elects a lane for a tile's products issues them at the tensor cores' rate (64 a 128 x 128 x 16 step; issue
//    blocks at that rate).
//  - one warp for S and P V was the bottleneck: 1,600 of products and 1,400 of waits and bookkeeping between them in one
//    line. Hence two warps, and words written by the copying warps instead of a walk over requests.
//  - copies are the other way round: 32 lanes with a box each take 64 to 136 cycles a box (1 to 8 KB, 8 to 64 rows of 128
//    bytes), one elected lane in a loop over boxes 135 to 240. Boxes of 8 tokens at head dim 128 (2 KB) bound a tile of K
//    and V at 2,400 cycles, short of HBM: hence boxes of several 8-token groups where page size and strides allow one map to
//    describe them (plan_draft_attn).
//  - two buffers of S put softmax, P V and S of a group's next tile in one line; NS = 3 or 4 take S out of it.
//  - three of eight pairs of exponentials by a polynomial on the FMA units made a tile's softmax slower (1,303 to 1,531): one
//    or two warps a scheduler wait for latency, not for the special-function unit.
//  - an L2 policy that keeps a share of the keys for a request's next block of rows changed neither time nor HBM bytes.
//
// Measured on B200, means of three sets of inputs in short loops (in sustained ones the clock falls: 2 to 16% longer, by size
// and GPU): four requests of up to 50,001 cached tokens, 13 drafts, 32 / 8 heads of 128: 534 MB in 99 us, 5.4 TB/s, bound by
// HBM. 352 requests, 512-token window, up to 9 drafts, 8 / 2 heads of 256: 384 MB in 85 us, 4.5 TB/s: ten tiles an item, so
// items' set-up and epilogues and masked tiles count. 40 requests of up to 6,000 tokens, 64 drafts, 32 / 4 heads of 128: 210 us;
// four blocks of rows read a head's keys, and of 362 MB that one set has, 1.06 GB come from HBM and 2.3 GB through L2. One
// token: 11 us of latencies and 3 for the join. 352 requests of up to 100 cached tokens, one draft, 8 / 8 heads of 64 or 128:
// 113 and 117 us for 51 and 101 MB: 2,816 items of two tiles, one after the other in each thread block.
//
// The weights are rounded to V's type for the second product (tcgen05 takes both factors of one 16-bit type; a second
// product with what the rounding left would double that product): relative 2^-11 or 2^-8 each, as the result itself is. For
// fp16 that needs its whole range: weights are 2^(s - m + 11) with m at most 2^4 short of the maximum, so that the largest
// lies between 2^11 and 2^15 and one of 2^-25 of it, 17 nats below, is still a normal number; what is smaller yet is rounded
// to multiples of 2^-35 of the largest. The factor 2^11 is in O and in the row sums alike. bf16 has fp32's range and takes
// none. Scores, maxima, sums and O are fp32, and the row sum adds the weights before they are rounded.
//
// A wait tells a barrier's phase from its neighbours only. S, P and P V of tile g use barrier g % NS: S of tile g waits for
// P V of tile g - NS, which waited for P of that tile, which its softmax wrote after it had read S; so whoever waits there
// for tile g knows tile g - NS to be done and g + NS to be impossible before it goes on. The rows' maxima of tile g use the
// barrier of its group: who waits for it has waited for g - 2 and is itself needed for g + 2. The rings of K, V and Q have
// one warp that fills them and one that empties them, both in order.
constexpr int DA_THREADS = 384;
constexpr int DA_ROWS = 128;
constexpr int DA_PIECES = 148;        // one thread block an SM
constexpr int DA_ITEM_COST = 3;       // what an item costs besides its tiles, in tiles, where pieces are long
constexpr int DA_SMEM_LIMIT = 227 * 1024;
constexpr int DA_MAX_BUFS = 6;
constexpr int DA_BARS = 4 * DA_MAX_BUFS + 37;
constexpr int DA_BOX_BYTES = 8192;     // of a TMA box of the cache, at most
constexpr uint32_t DA_TMEM_COLS = 512;  // da_scores buffers of S (later P), then O

__host__ __device__ constexpr int da_tile(int dim) { return dim == 256 ? 64 : 128; }
__host__ __device__ constexpr int da_scores(int dim) { return dim == 256 ? 4 : 3; }
// barriers, items, row maxima and sums, and for each token of two items its position and first mask words
__host__ __device__ constexpr int da_extra(int dim, int block) { return 4608 + 8 * block * (1 + da_tile(dim) / 32); }
__host__ __device__ constexpr int da_buffer_bytes(int dim) { return da_tile(dim) * dim * 2; }

struct DaPlan {  // launch shape, chosen by the host
  int block;     // drafted tokens of an item: at most 128 rows
  int q_rows;    // rows a Q buffer holds: block * G rounded up to a multiple of 8
  int q_bufs;
  int k_bufs, v_bufs;  // at most DA_MAX_BUFS each
  int fold;      // how the cache's maps tell heads apart: 0 by a dimension of their own (boxes of 8 tokens), 1 by the dimension
                 // of 64-dim blocks, 2 by the dimension of 8-token groups (boxes of `groups` of them)
  int groups;    // 8-token groups of a box
  int head_step; // fold 1 or 2: what a head adds to its coordinate
};
__host__ __device__ inline int da_smem_bytes(const DaPlan& p, int dim) {
  return p.q_bufs * p.q_rows * dim * 2 + (p.k_bufs + p.v_bufs) * da_buffer_bytes(dim) + 1024 + da_extra(dim, p.block);
}

// Whose mask words, of an item's block of tokens, a row reads: its own token's, or the last one's if it has none (it then
// counts for nothing, but reads like the others of its warp).
__host__ __device__ constexpr int da_row_token(int row, int group, int block) {
  return row / group < block ? row / group : block - 1;
}
constexpr bool da_row_tokens_fit() {
  for (int group = 1; group <= DA_ROWS; ++group)
    for (int row = 0; row < DA_ROWS; ++row)
      if (da_row_token(row, group, DA_ROWS / group) >= DA_ROWS / group || da_row_token(row, group, 1) > 0) return false;
  return true;
}
static_assert(da_row_tokens_fit(), "rows read mask words of their block's tokens only");

// Workspace: per piece two partial results (its first and its last item) of 128 rows, O [128][dim], then (m, l) [128],
// and the item that begins in it and ends in a later piece.
struct DaSplit {
  int b, h, block, last;  // last: the piece it ends in; -1: none
  int first_slot;         // partial result of the piece it begins in
  int pad[3];
};
__host__ __device__ inline size_t da_partial_floats(int dim) { return (size_t)DA_ROWS * (dim + 2); }
__host__ __device__ inline size_t da_workspace_bytes(int dim) {
  return DA_PIECES * sizeof(DaSplit) + 2 * DA_PIECES * da_partial_floats(dim) * sizeof(float);
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
  r.cached = r.lo < r.len ? (r.len - 1) / KT + 1 - r.first : 0;  // a length may be close to 2^31
  r.n = r.fresh ? r.cached + (r.fresh + KT - 1) / KT : 0;
  r.blocks = (r.fresh + block - 1) / block;
  return r;
}

// Where a piece begins.
struct DaStart {
  int b, h, block, i;  // request, head, block of tokens, tile
  int64_t unit;        // where that item begins
};

// A place on the line of tiles.
template <int KT>
struct DaWalk {
  const DraftAttnArgs* a;
  DaReq r;
  int size;      // tokens of a block
  int b, h, block, i;
  int cost;      // units of an item before its tiles
  int64_t unit;  // where the item begins
  __device__ __forceinline__ void start(const DraftAttnArgs& args, int block_size, int item_cost, const DaStart& at) {
    a = &args;
    size = block_size;
    cost = item_cost;
    b = at.b;
    h = at.h;
    block = at.block;
    i = at.i;
    unit = at.unit;
    r = da_request<KT>(args, size, b, false);
  }
  __device__ __forceinline__ void skip(int tiles) {  // at most to the item's end
    i += tiles;
    if (i < r.n) return;
    i = 0;
    unit += r.n + cost;
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

// fp16 / bf16: instruction descriptors with B K-major (S) and N-major (P V), the bits of a non-finite value, and of the
// softmax weights 2^(s - m + kLift): m rises when a score exceeds it by more than kSlack. A larger kSlack rescales O less often,
// kSlack + kLift is what the type holds above 1.
template <typename T> struct DaType;
template <> struct DaType<__half> {
  static __host__ __device__ constexpr uint32_t idesc(int n) { return idesc_f16(DA_ROWS, n); }
  static constexpr uint32_t kExp = 0x7c00u;
  static constexpr float kSlack = 4.f, kLift = 11.f;
};
template <> struct DaType<__nv_bfloat16> {
  static __host__ __device__ constexpr uint32_t idesc(int n) { return idesc_bf16(DA_ROWS, n); }
  static constexpr uint32_t kExp = 0x7f80u;
  static constexpr float kSlack = 8.f, kLift = 0.f;
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
// 32 32-bit values a thread into TMEM columns taddr .. taddr + 31 of its lane; complete after tmem_st_wait.
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
// 16 packed 32-bit values a thread into TMEM columns taddr .. taddr + 15 of its lane; complete after tmem_st_wait.
__device__ __forceinline__ void tmem_st16_async(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
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

// mbar_wait with its loop out of line: the kernel waits in two dozen places.
__device__ __noinline__ bool da_wait_on(uint64_t* bar, uint32_t parity, int* err, int code) {
  return mbar_wait(bar, parity, err, code);
}
__device__ __forceinline__ bool da_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  return mbar_try_wait(bar, parity) || da_wait_on(bar, parity, err, code);
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

// An item, or a piece's part of it, as warp 3 describes it to the softmax.
struct DaItem {
  int b, h, block, t0, fresh, len, lo, first, cached, n;  // as in DaReq and DaWalk
  int i0, i1;  // this piece's tiles
  int lows;    // with a window: the largest of its tokens' positions - window; else -1
  int last;    // the piece in which it ends
  int pad[2];
};

// What a lane fetches of a K or V tile: one box.
struct DaFetch {
  int row, page;  // token within the page and page id, or drafted token
  int drafted, head, block, t0;
  uint32_t info;
  bool mine;      // some of them exist
};

// The kernel's program is kept small: what is rare, or common to several places, is out of line.

// Which of keys w .. w + 31 of a tile the drafted token `tok` of a request sees. The tile begins at key `base` (a cached
// position or a drafted index) and has `end` keys; cached keys are seen from position low + 1 on. word: the mask's word
// for these keys if it is at hand.
__device__ __noinline__ uint32_t da_seen(const DraftAttnArgs& a, bool tree, int t0, int fresh, int len, int base, int w, int end,
                                         int low, int tok, const uint32_t* word) {
  const int from = tree ? 0 : max(0, low + 1 - base), z = min(32, max(0, end - w)), f = min(32, max(0, from - w));
  uint32_t bits = (z == 32 ? ~0u : (1u << z) - 1u) & (f == 32 ? 0u : ~0u << f);
  if (!tree || tok >= fresh) return bits;
  if (a.mask) {
    const int at = (base + w) >> 5;
    bits &= word ? *word : at < a.words ? a.mask[(int64_t)(t0 + tok) * a.words + at] : 0u;
  } else {
    bits &= tok >= base + w + 31 ? ~0u : tok < base + w ? 0u : (2u << (tok - base - w)) - 1u;
  }
  if (a.window && low >= len) {  // a window so short that it ends among the drafted tokens
    for (uint32_t rest = bits; rest; rest &= rest - 1) {
      const int j = base + w + __ffs(rest) - 1;
      if ((a.positions ? a.positions[t0 + j] : len + j) <= low) bits &= ~(rest & -rest);
    }
  }
  return bits;
}

// Adds the non-finite elements of the V rows that token `tok` of `it` sees, among those that not every row sees, to its
// written result: they were 0 in the product. Rare, and slow: key after key. Y: the type of `row`.
template <int KT, int D, typename T, typename Y>
__device__ __noinline__ void da_restore(const DraftAttnArgs& a, const DaItem& it, int tok, int low, Y* row) {
  for (int i = it.i0; i < it.i1; ++i) {
    const bool tree = i >= it.cached;
    const int base = tree ? (i - it.cached) * KT : (it.first + i) * KT;
    for (int j = base; j < min(base + KT, tree ? it.fresh : min(it.len, it.lows + 1)); ++j) {
      const T* v;
      if (tree) {
        if (!(da_seen(a, true, it.t0, it.fresh, it.len, base, (j - base) & ~31, it.fresh - base, low, tok, nullptr) >> (j & 31) & 1))
          continue;
        v = (const T*)a.v + (int64_t)(it.t0 + j) * a.v_ts + (int64_t)it.h * a.v_hs;
      } else {
        if (j <= low) continue;
        const int pg = a.table[it.b * a.table_stride + j / a.cache.page];
        if (pg < 0 || pg >= a.cache.pages) continue;
        v = (const T*)a.cache.v + pg * a.cache.page_stride + j % a.cache.page * a.cache.token_stride + it.h * a.cache.head_stride;
      }
#pragma unroll 1
      for (int d = 0; d < D; ++d) {
        const float x = (float)v[d];
        if (!(fabsf(x) < INFINITY)) row[d] = (Y)((float)row[d] + x);
      }
    }
  }
}

template <int D, typename T>
__global__ void __launch_bounds__(DA_THREADS, 1)
draft_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_ck,
                  const __grid_constant__ CUtensorMap tm_cv, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ DraftAttnArgs a, const DaPlan plan,
                  DaSplit* splits, float* partials) {
  constexpr int KT = da_tile(D), NC = D / 64, BUF = da_buffer_bytes(D), NS = da_scores(D);
  constexpr float LIFT = DaType<T>::kLift;
  constexpr uint32_t O_COL = NS * KT;
  static_assert(O_COL + D <= DA_TMEM_COLS, "S buffers and O fill TMEM");
  extern __shared__ __align__(1024) uint8_t da_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(da_smem_raw) + 1023) & ~uintptr_t(1023));
  const int q_buf = plan.q_rows * D * 2, q_box = plan.q_rows * 128;
  uint8_t* qs = smem;                            // [q_bufs][NC][q_rows][128 B], SW128
  uint8_t* ks = qs + plan.q_bufs * q_buf;        // [k_bufs][KT / 8][NC][8][128 B], SW128
  uint8_t* vs = ks + plan.k_bufs * BUF;          // [v_bufs], likewise
  uint64_t* bars = reinterpret_cast<uint64_t*>(vs + plan.v_bufs * BUF);
  uint64_t* k_full = bars;                       // [k_bufs] a tile has landed
  uint64_t* k_empty = k_full + DA_MAX_BUFS;      // [k_bufs] the products that read it are done
  uint64_t* v_full = k_empty + DA_MAX_BUFS;
  uint64_t* v_empty = v_full + DA_MAX_BUFS;
  uint64_t* q_full = v_empty + DA_MAX_BUFS;      // [2]
  uint64_t* q_empty = q_full + 2;                // [2]
  uint64_t* s_full = q_empty + 2;                // [NS] S of a tile is there
  uint64_t* p_full = s_full + 4;                 // [NS] P of a tile is written, O rescaled, V mended
  uint64_t* pv_done = p_full + 4;                // [NS] O includes the tile
  uint64_t* v_there = pv_done + 4;               // [NS] V of the tile has landed
  uint64_t* all_done = v_there + 4;              // [2] of warps 1 and 2, when a role has given up
  uint64_t* m_full = all_done + 2;               // [2][4] a softmax warp's maxima
  uint64_t* item_full = m_full + 8;              // [2] what an item is, for the softmax
  uint64_t* item_empty = item_full + 2;          // [2]
  uint64_t* ml_full = item_empty + 2;            // [2] the group without an item's last tile is through with it
  uint64_t* o_free = ml_full + 2;                // O has been read
  static_assert(DA_BARS == 4 * DA_MAX_BUFS + 4 + 4 * 4 + 2 + 8 + 2 + 2 + 2 + 1, "every barrier is initialised");
  int64_t* s_scan = reinterpret_cast<int64_t*>(bars + DA_BARS);  // [12][2] warp sums of items and tiles
  int64_t* s_tiles = s_scan + 24;                // [2] tiles before the piece and up to its end
  DaStart* s_start = reinterpret_cast<DaStart*>(s_tiles + 2);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_start + 1);
  int* poison = reinterpret_cast<int*>(tmem_slot + 2);       // [2] of even / odd items: item + 1 if it met a non-finite V
  uint32_t* k_info = reinterpret_cast<uint32_t*>(poison + 2);  // [k_bufs], [v_bufs] of the tile in a buffer, see below
  uint32_t* v_info = k_info + DA_MAX_BUFS;
  DaItem* items = reinterpret_cast<DaItem*>(v_info + DA_MAX_BUFS);  // [2]
  float2* ml_rows = reinterpret_cast<float2*>(items + 2);    // [2][128] (m, l) of that group
  float* m_rows = reinterpret_cast<float*>(ml_rows + 256);   // [2][128] maxima after even / odd tiles
  int* row_pos = reinterpret_cast<int*>(m_rows + 256);       // [2][block] an item's tokens: positions, with a window
  uint32_t* row_words = reinterpret_cast<uint32_t*>(row_pos + 2 * plan.block);  // [2][block][KT / 32] first mask words

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, piece = blockIdx.x;
  const int G = a.hq / a.hkv;
  if (tid >= 32 && tid < 32 + DA_BARS) {  // one barrier a thread
    const int i = tid - 32;
    uint64_t* bar = bars + i;
    mbar_init(bar, bar >= p_full && bar < pv_done ? 4 : bar >= m_full ? (bar < item_full ? 1 : bar < item_empty ? 1 : bar < ml_full ? 8 : 4) : 1);
    fence_barrier_init();
  }
  if (tid == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_ck);
    prefetch_tmap(&tm_cv);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    poison[0] = poison[1] = 0;
  }
  pdl_wait();  // nothing above reads or writes what an earlier kernel may use
  if (tid == 0) splits[piece].last = -1;
  // not before the wait: a block that held tensor memory there could keep it from the kernel that it waits for
  if (warp == 3) tmem_alloc(tmem_slot, DA_TMEM_COLS);

  // requests' items and tiles
  const int per = (a.rows + DA_THREADS - 1) / DA_THREADS, rb0 = min(a.rows, tid * per), rb1 = min(a.rows, rb0 + per);
  struct Span {
    int64_t items, tiles;
  };
  auto span_of = [&](int b, bool report) {
    const DaReq r = da_request<KT>(a, plan.block, b, report);
    const int64_t items = r.n ? (int64_t)r.blocks * a.hkv : 0;
    return Span{items, items * r.n};
  };
  Span mine{0, 0};
  for (int b = rb0; b < rb1; ++b) {
    const Span x = span_of(b, piece == 0);
    mine.items += x.items;
    mine.tiles += x.tiles;
  }
  // ---- this piece of the line ----
  Span upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, upto.items, o), y = __shfl_up_sync(0xffffffffu, upto.tiles, o);
    if (lane >= o) {
      upto.items += x;
      upto.tiles += y;
    }
  }
  if (lane == 31) {
    s_scan[2 * warp] = upto.items;
    s_scan[2 * warp + 1] = upto.tiles;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  Span total{0, 0}, before{upto.items - mine.items, upto.tiles - mine.tiles};
  for (int w = 0; w < DA_THREADS / 32; ++w) {
    if (w < warp) {
      before.items += s_scan[2 * w];
      before.tiles += s_scan[2 * w + 1];
    }
    total.items += s_scan[2 * w];
    total.tiles += s_scan[2 * w + 1];
  }
  // An item counts DA_ITEM_COST tiles more than it has, but not where a piece has hardly more tiles than that. Without and
  // with it, at about 4, 8, 12 and 24 tiles a piece: head dim 256, window 512, 21.7 and 19.8 us, 29.2 and 27.2, 35.0 and
  // 31.8, 49.9 and 47.4; head dim 128, caches of 200, 26.1 and 22.9, 32.7 and 29.5, 43.8 and 38.2, 76.2 and 67.5; of 5,000,
  // 22.8 and 19.3, 28.1 and 23.3, 33.0 and 26.4, 45.8 and 42.5; head dim 64, caches of 600, 20.7 and 18.9, 31.9 and 27.0,
  // 39.6 and 33.5, 64.5 and 55.2.
  const int64_t mean = (total.tiles + DA_PIECES - 1) / DA_PIECES;
  const int cost = mean > DA_ITEM_COST ? DA_ITEM_COST : 0;
  // An item of n tiles cut into pieces of s costs about 2 us for each of a piece's tiles and 0.37 us for each of the n / s
  // parts that its join reads: s + 1 tiles a piece pay from n = 5 s (s + 1) on. That bounds the pieces from below where
  // items are few and long. One request, one key head of 16 rows, head dim 128, without this and with it: 9,000 keys 31.6
  // and 20.8 us, 17,000 keys 48.9 and 24.0, 40,000 keys 52.7 and 31.7; four key heads: 4,400 keys 20.9 and 17.5, 1,000 keys
  // (one tile a piece either way) 15.7 and 15.6; head dim 64, four key heads, 2,500 keys 16.2 and 15.4; head dim 256, two key
  // heads, 2,200 keys 28.1 and 21.3. A fixed two tiles a piece: two tiles an item 13.9 to 15.5. The mean over all items
  // decides, so a long one among many short ones is cut like those.
  const float item_tiles = (float)total.tiles / (float)max((int64_t)1, total.items);
  const int64_t least = max(1, (int)(sqrtf(0.2f * item_tiles + 0.25f) + 0.5f));
  const int64_t units = total.tiles + cost * total.items, step = max(least, (units + DA_PIECES - 1) / DA_PIECES);
  const int64_t w0 = min(units, piece * step), w1 = min(units, w0 + step);
  // whose requests hold the piece's first unit, or the one past its last, says how many tiles lie before it
  const int64_t first = before.tiles + cost * before.items, past = first + mine.tiles + cost * mine.items;
  const bool has0 = w0 >= first && w0 < past, has1 = w1 >= first && w1 < past;
  if (has0 || has1) {
    Span at = before;
    for (int b = rb0; b < rb1; ++b) {
      const DaReq r = da_request<KT>(a, plan.block, b, false);
      const int64_t items = r.n ? (int64_t)r.blocks * a.hkv : 0, at_unit = at.tiles + cost * at.items;
      const int64_t end = at_unit + items * (r.n + cost);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t w = e ? w1 : w0;
        if (!(e ? has1 : has0) || w < at_unit || w >= end) continue;
        const int64_t within = w - at_unit;
        const int len = r.n + cost;
        const int64_t item = within <= INT32_MAX ? (int64_t)((uint32_t)within / (uint32_t)len) : within / len;
        const int i = max(0, (int)(within - item * len) - cost);
        s_tiles[e] = at.tiles + item * r.n + i;
        if (e == 0) {
          const int h = (int)((uint32_t)item / (uint32_t)r.blocks);  // items of a request: heads x blocks
          *s_start = DaStart{b, h, (int)item - h * r.blocks, i, at_unit + item * len};
        }
      }
      at.items += items;
      at.tiles += items * r.n;
    }
  }
  if (tid == 0 && w0 >= units) s_tiles[0] = s_tiles[1] = total.tiles;  // past the line's end
  if (tid == 0 && w0 < units && w1 >= units) s_tiles[1] = total.tiles;
  __syncthreads();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const int n_tiles = (int)(s_tiles[1] - s_tiles[0]);
  bool ok = true;  // no wait of this thread has given up
  int issued = 0, q_issued = 0;  // warps 0 and 3: K and V tiles requested; warp 0: Q tiles
  if (n_tiles > 0) {
    DaWalk<KT> walk;
    walk.start(a, plan.block, cost, *s_start);
    // info: of a K tile bit 0: first of its item in this piece, bit 1: last; of a V tile bit 0 as well, then the steps of
    // 16 keys that hold keys: bits 4-7 the first, bits 8-11 one past the last
    if (warp == 0 || warp == 3) {
      // ---- K tiles and Q (warp 0), V tiles (warp 3): lane i brings the i-th box ----
      const int box = 8 * plan.groups;  // cached tokens of one
      const bool is_v = warp == 3;
      const CUtensorMap *cache = is_v ? &tm_cv : &tm_ck, *drafted = is_v ? &tm_v : &tm_k;
      uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
      uint32_t* info = is_v ? v_info : k_info;
      uint8_t* bufs = is_v ? vs : ks;
      const int n_bufs = is_v ? plan.v_bufs : plan.k_bufs;
      auto fetch_of = [&](const DaWalk<KT>& w, bool begins, bool ends) {
        DaFetch x{0, -1, 0, w.h, w.block, w.r.t0, 0u, false};
        int begin = 0, end;
        if (w.i < w.r.cached) {
          const int base = (w.r.first + w.i) * KT, pos = base + lane * box;
          begin = max(0, w.r.lo - base);
          end = min(KT, w.r.len - base);
          x.mine = lane * box < end && lane * box + box > begin;
          if (x.mine) {
            const int p = pos / a.cache.page;
            x.row = pos - p * a.cache.page;
            x.page = a.table[w.b * a.table_stride + p];
          }
        } else {
          const int j = (w.i - w.r.cached) * KT;
          end = min(KT, w.r.fresh - j);
          x.mine = lane * 8 < end;
          x.row = w.r.t0 + j + lane * 8;
          x.drafted = 1;
        }
        x.info = (begins ? 1u : 0u) | (ends ? 2u : 0u) | (uint32_t)(begin >> 4) << 4 | (uint32_t)((end + 15) >> 4) << 8;
        return x;
      };
      DaRing ring, q_ring;
      auto fetch = [&](int g) { return fetch_of(walk, g == 0 || walk.i == 0, g + 1 == n_tiles || walk.i + 1 == walk.r.n); };
      auto item_of = [&](int g) {
        const DaReq& r = walk.r;
        return DaItem{walk.b, walk.h, walk.block, r.t0, r.fresh, r.len, r.lo, r.first, r.cached, r.n, walk.i,
                      min(r.n, walk.i + n_tiles - g), -1, (int)((walk.unit + cost + r.n - 1) / step), {0, 0}};
      };
      DaFetch cur{}, next{};
      DaItem cur_item{}, next_item{};
      int item = 0;  // warp 3: items described
      for (int g = -1; g < n_tiles && ok; ++g) {
        if (g + 1 < n_tiles) {  // the next tile's table entries, ahead of the wait
          if (g >= 0) walk.skip(1);
          next = fetch(g + 1);
          if (is_v && (next.info & 1)) next_item = item_of(g + 1);
        }
        if (g < 0) {
          cur = next;
          cur_item = next_item;
          continue;
        }
        if (is_v && (cur.info & 1)) {  // the item, for the softmax
          if (item >= 2)
            ok = __all_sync(0xffffffffu, da_wait(&item_empty[item & 1], ((item >> 1) - 1) & 1, a.err, ERR_TIMEOUT_MMA));
          if (!ok) break;
          const int size = plan.block, tokens = min(size, cur_item.fresh - cur_item.block * size);
          const int t = cur_item.t0 + cur_item.block * size;
          int lows = -1;
          for (int k = lane; k < tokens; k += 32) {
            if (a.window) {
              const int pos = a.positions ? a.positions[t + k] : cur_item.len + cur_item.block * size + k;
              row_pos[(item & 1) * size + k] = pos;
              lows = max(lows, pos - a.window);
            }
            if (a.mask)
              for (int w = 0; w < KT / 32; ++w)
                row_words[((item & 1) * size + k) * (KT / 32) + w] = w < a.words ? a.mask[(int64_t)(t + k) * a.words + w] : 0u;
          }
          lows = __reduce_max_sync(0xffffffffu, lows);
          if (lane == 0) {
            cur_item.lows = max(lows, a.window ? cur_item.lo - 1 : -1);
            items[item & 1] = cur_item;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&item_full[item & 1]);
          ++item;
        }
        if (!is_v && (cur.info & 1)) {  // Q: block tokens x G heads, one box for each 64 dims
          if (q_issued >= plan.q_bufs)
            ok = __all_sync(0xffffffffu, da_wait(&q_empty[q_ring.at], q_ring.phase ^ 1u, a.err, ERR_TIMEOUT_MMA));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&q_full[q_ring.at], plan.block * G * D * 2);
          __syncwarp();
          if (lane < NC)
            tma_load_3d(qs + q_ring.at * q_buf + lane * q_box, &tm_q, lane * 64, cur.head * G, cur.t0 + cur.block * plan.block,
                        &q_full[q_ring.at]);
          ++q_issued;
          q_ring.next(plan.q_bufs);
        }
        if (g >= n_bufs) ok = __all_sync(0xffffffffu, da_wait(&empty[ring.at], ring.phase ^ 1u, a.err, ERR_TIMEOUT_MMA));
        if (!ok) break;
        const bool good = cur.drafted || (cur.page >= 0 && cur.page < a.cache.pages);
        if (cur.mine && !good) set_error(a.err, ERR_BAD_PAGE);
        const bool bring = cur.mine && good;
        const unsigned boxes = __ballot_sync(0xffffffffu, bring);
        const int box_groups = cur.drafted ? 1 : plan.groups;
        if (lane == 0) {
          info[ring.at] = cur.info;
          mbar_arrive_expect_tx(&full[ring.at], __popc(boxes) * box_groups * (NC * 1024));
        }
        __syncwarp();
        if (bring) {
          uint8_t* dst = bufs + ring.at * BUF + lane * box_groups * NC * 1024;
          if (cur.drafted) tma_load_4d(dst, drafted, 0, cur.row, 0, cur.head, &full[ring.at]);
          else if (plan.fold == 0) tma_load_5d(dst, cache, 0, cur.row, 0, cur.head, cur.page, &full[ring.at]);
          else if (plan.fold == 1) tma_load_5d(dst, cache, 0, 0, cur.head * plan.head_step, cur.row >> 3, cur.page, &full[ring.at]);
          else tma_load_5d(dst, cache, 0, 0, 0, cur.head * plan.head_step + (cur.row >> 3), cur.page, &full[ring.at]);
        }
        issued = g + 1;
        ring.next(n_bufs);
        cur = next;
        cur_item = next_item;
      }
      if (lane == 0 && !is_v) pdl_trigger();  // (at the kernel's begin it costs a microsecond)
    } else if (warp == 1) {
      // ---- S ----
      const uint32_t idesc = DaType<T>::idesc(KT);
      DaRing ring, q_ring, s_ring;
      for (int g = 0; g < n_tiles && ok; ++g) {
        ok = __all_sync(0xffffffffu, da_wait(&k_full[ring.at], ring.phase, a.err, ERR_TIMEOUT_TMA));
        const uint32_t what = k_info[ring.at];
        if (ok && (what & 1)) ok = __all_sync(0xffffffffu, da_wait(&q_full[q_ring.at], q_ring.phase, a.err, ERR_TIMEOUT_TMA));
        if (ok && g >= NS) ok = __all_sync(0xffffffffu, da_wait(&pv_done[s_ring.at], s_ring.phase ^ 1u, a.err, ERR_TIMEOUT_MMA));
        if (!ok) break;
        tc_fence_after();
        const uint64_t qd = sw128_desc(smem_u32(qs + q_ring.at * q_buf)), kd = da_k_desc<NC>(smem_u32(ks + ring.at * BUF));
        const uint32_t d = tmem + (uint32_t)(s_ring.at * KT);
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_bf16(d, qd + (uint64_t)((c * q_box + kk * 32) >> 4), kd + (uint64_t)((c * 1024 + kk * 32) >> 4), idesc,
                       (c > 0 || kk > 0) ? 1u : 0u);
          mma_commit(&s_full[s_ring.at]);
          mma_commit(&k_empty[ring.at]);
          if (what & 2) mma_commit(&q_empty[q_ring.at]);
        }
        __syncwarp();
        ring.next(plan.k_bufs);
        if (what & 2) q_ring.next(plan.q_bufs);
        s_ring.next(NS);
      }
    } else if (warp == 2) {
      // ---- P V ----
      const uint32_t idesc = DaType<T>::idesc(D) | DA_B_N_MAJOR;
      DaRing ring, p_ring;
      int item = 0;
      for (int g = 0; g < n_tiles && ok; ++g) {
        ok = __all_sync(0xffffffffu, da_wait(&v_full[ring.at], ring.phase, a.err, ERR_TIMEOUT_TMA));
        const uint32_t what = v_info[ring.at];
        if (ok && lane == 0) mbar_arrive(&v_there[p_ring.at]);
        __syncwarp();
        if (what & 1) {
          if (ok && item > 0) ok = __all_sync(0xffffffffu, da_wait(o_free, (item - 1) & 1, a.err, ERR_TIMEOUT_MMA));
          ++item;
        }
        if (ok) ok = __all_sync(0xffffffffu, da_wait(&p_full[p_ring.at], p_ring.phase, a.err, ERR_TIMEOUT_MMA));
        if (!ok) break;
        tc_fence_after();
        const uint64_t vd = da_v_desc<NC>(smem_u32(vs + ring.at * BUF));
        const uint32_t p = tmem + (uint32_t)(p_ring.at * KT);
        // steps of 16 keys that exist: the others' V is whatever lay in the buffer
        const int k0 = what >> 4 & 15, k1 = what >> 8 & 15;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < KT / 16; ++kk)
            if (kk >= k0 && kk < k1)
              mma_tmem_a(tmem + O_COL, p + kk * 8, vd + (uint64_t)((kk * 2 * NC * 1024) >> 4), idesc,
                         (!(what & 1) || kk > k0) ? 1u : 0u);
          mma_commit(&pv_done[p_ring.at]);
          mma_commit(&v_empty[ring.at]);
        }
        __syncwarp();
        ring.next(plan.v_bufs);
        p_ring.next(NS);
      }
    } else if (warp >= 4) {
      // ---- softmax: thread = row = TMEM lane; group 0 (warps 4-7) takes even tiles, group 1 (warps 8-11) odd ones ----
      const int group = warp >= 8, row = tid & 127, quarter = warp & 3;
      const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
      const float sl2 = a.scale * 1.4426950408889634f;        // scores in log2 units
      const int row_tok = row / G;                            // token within the block
      DaRing ring;  // of tile g's S and P
      int reached = 0;
      int g0 = 0;  // the item's first tile
      for (int item = 0; g0 < n_tiles; ++item) {
        if (ok) ok = da_wait(&item_full[item & 1], (item >> 1) & 1, a.err, ERR_TIMEOUT_TMA);
        if (!__all_sync(0xffffffffu, ok)) {  // without the item there is nothing to go by
          ok = false;
          break;
        }
        const DaItem& it = items[item & 1];
        const int i0 = it.i0, i1 = it.i1, cached = it.cached, len = it.len, fresh = it.fresh, t0 = it.t0;
        const int tok = it.block * plan.block + row_tok;
        const bool valid = row < plan.block * G && tok < fresh;
        const bool live = __any_sync(0xffffffffu, valid);
        // keys of this row are those at positions above `low`; no row's bound is above it.lows
        int low = it.lo - 1;
        if (a.window && valid) low = max(low, row_pos[(item & 1) * plan.block + row_tok] - a.window);
        const uint32_t* first_words = row_words + ((item & 1) * plan.block + da_row_token(row, G, plan.block)) * (KT / 32);
        float m = -INFINITY, l = 0.f;  // maximum of the last tile that this group took part in, sum of its own weights
        for (int i = i0 + ((g0 ^ group) & 1); i < i1; i += 2) {
          const int g = g0 + i - i0;
          for (; reached < g; ++reached) ring.next(NS);
          const uint32_t s_col = lanes + (uint32_t)(ring.at * KT);  // S, later P
          const bool tree = i >= cached;
          const int base = tree ? (i - cached) * KT : (it.first + i) * KT;  // first key: drafted index or position
          const int end = min(KT, (tree ? fresh : len) - base);             // keys that exist
          const int begin = tree ? 0 : max(0, it.lo - base);
          // keys up to here are seen by some rows and not by others
          const int mixed = tree ? end : a.window ? min(end, it.lows + 1 - base) : 0;
          const bool special = mixed > 0 || begin > 0 || end < KT;
          if (ok) ok = da_wait(&s_full[ring.at], ring.phase, a.err, ERR_TIMEOUT_MMA);
          tc_fence_after();
          __syncwarp();
          float top = -INFINITY;
          if (live) {
            // S is read twice, for the maximum and for the weights, 32 columns at a time in loops that are not unrolled:
            // unrolled over a tile, with a copy for masked ones, a tile of 128 keys took 1.3 times as long (twelve warps in
            // seven places of a large program)
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
            for (int c = 0; c < KT / 32; ++c) {
              uint32_t x[32];
              tmem_ld32_async(s_col + 32 * c, x);
              tmem_ld_wait();
              da_pin(x);
              if (special) {  // -inf where the row does not see the key, for the second reading as well
                const uint32_t bits = da_seen(a, tree, t0, fresh, len, base, 32 * c, end, low, tok, base == 0 ? &first_words[c] : nullptr);
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] = bits >> j & 1 ? x[j] : 0xff800000u;
                tmem_st32_async(s_col + 32 * c, x);
              }
#pragma unroll
              for (int j = 0; j < 32; j += 8)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  tops[q] = fmaxf(fmaxf(tops[q], __uint_as_float(x[j + q])), __uint_as_float(x[j + 4 + q]));
            }
            if (special) tmem_st_wait();
            top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * sl2;
          }
          // the maximum so far, from the other group; it is raised only when a tile exceeds it by 2^kSlack
          if (ok && g > 0) ok = da_wait(&m_full[4 * (group ^ 1) + quarter], ((g - 1) >> 1) & 1, a.err, ERR_TIMEOUT_MMA);
          const float seen = i > i0 ? m_rows[128 * (group ^ 1) + row] : -INFINITY;
          const bool raise = valid && (top > seen + DaType<T>::kSlack || (seen == -INFINITY && top > -INFINITY));
          const float now = raise ? top : seen;
          m_rows[128 * group + row] = now;
          __syncwarp();
          if (lane == 0) mbar_arrive(&m_full[4 * group + quarter]);
          if (live) {
            if (now != m) {  // m = -inf: l is 0
              l *= m == -INFINITY ? 0.f : ex2_approx(m - now);
              m = now;
            }
            if (i > i0 && __any_sync(0xffffffffu, raise)) {
              if (ok) ok = da_wait(&pv_done[(g - 1) % NS], ((g - 1) / NS) & 1, a.err, ERR_TIMEOUT_MMA);
              tc_fence_after();
              __syncwarp();
              const float alpha = !raise ? 1.f : seen == -INFINITY ? 0.f : ex2_approx(seen - now);
#pragma unroll 1
              for (int c = 0; c < D; c += 32) {
                float o[32];
                tmem_ld32(lanes + O_COL + c, o);
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] *= alpha;
                tmem_st32(lanes + O_COL + c, o);
              }
            }
            const float2 mul = make_float2(sl2, sl2), off = m == -INFINITY ? make_float2(0.f, 0.f) : make_float2(LIFT - m, LIFT - m);
            float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            __syncwarp();
#pragma unroll 1
            for (int c = 0; c < KT / 32; ++c) {
              uint32_t x[32], pk[16];
              tmem_ld32_async(s_col + 32 * c, x);
              tmem_ld_wait();
              da_pin(x);
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                float2 y = fma2(make_float2(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), mul, off);
                y = make_float2(ex2_approx(y.x), ex2_approx(y.y));
                sums[j >> 1 & 1] = add2(sums[j >> 1 & 1], y);
                pk[j >> 1] = pack2(y.x, y.y, (const T*)nullptr);
              }
              tmem_st16_async(s_col + 16 * c, pk);  // over scores that have been read
            }
            sums[0] = add2(sums[0], sums[1]);
            l += sums[0].x + sums[0].y;
            tmem_st_wait();
          }
          if (special) {
            // V rows that nobody sees become 0 (0 times whatever lay there must not count), as far as the product
            // reaches: whole steps of 16 keys. Where rows differ in what they see, V's infinities and NaN become 0,
            // and the epilogue puts them back for the rows that see them.
            if (ok) ok = da_wait(&v_there[ring.at], ring.phase, a.err, ERR_TIMEOUT_TMA);
            uint8_t* vb = vs + (g % plan.v_bufs) * BUF;
            const int head_rows = begin & 15, z0 = begin - head_rows, tail_rows = -end & 15;
            for (int c = row; c < (head_rows + tail_rows) * (D / 8); c += 128) {
              const int k = c / (D / 8);
              *reinterpret_cast<uint4*>(vb + da_offset<NC>(k < head_rows ? z0 + k : end + k - head_rows, c % (D / 8))) =
                  make_uint4(0u, 0u, 0u, 0u);
            }
            for (int c = begin * (D / 8) + row; c < mixed * (D / 8); c += 128) {
              uint4* at = reinterpret_cast<uint4*>(vb + da_offset<NC>(c / (D / 8), c % (D / 8)));
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
            fence_proxy_async();
          }
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
          continue;
        }
        if (ok) ok = da_wait(&ml_full[item & 1], (item >> 1) & 1, a.err, ERR_TIMEOUT_MMA);
        {
          const float2 theirs = ml_rows[128 * (item & 1) + row];  // their maximum is no larger than m, the last tile's
          const float w = theirs.x == m ? 1.f : theirs.x == -INFINITY ? 0.f : ex2_approx(theirs.x - m);
          l += theirs.y * w;
        }
        if (ok) ok = da_wait(&pv_done[last % NS], (last / NS) & 1, a.err, ERR_TIMEOUT_MMA);
        tc_fence_after();
        const bool mend = poison[item & 1] == item + 1;  // every tile's P has been waited for, so its scan is done
        const bool whole = i0 == 0 && i1 == it.n;
        const int slot = 2 * piece + (item > 0 ? 1 : 0), h = it.h;
        float* part = partials + slot * da_partial_floats(D);
        const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
        const int64_t orow = (int64_t)(t0 + tok) * a.hq + h * G + row % G;
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
          if (whole) da_restore<KT, D, T, T>(a, it, tok, low, (T*)a.out + orow * D);
          else da_restore<KT, D, T, float>(a, it, tok, low, part + row * D);
        }
        if (valid) {
          if (!whole)
            *reinterpret_cast<float2*>(part + DA_ROWS * D + 2 * row) = make_float2(m, l);
          else if (a.lse)
            a.lse[orow] = l > 0.f || l != l ? (m - LIFT + log2f(l)) * 0.6931471805599453f : -INFINITY;
        }
        if (row == 0 && i0 == 0 && i1 < it.n) splits[piece] = DaSplit{it.b, h, it.block, it.last, slot, {0, 0, 0}};
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[item & 1]);
      }
    }
  }
  // ---- teardown. If every role went through, every copy and product has been waited for. If one gave up, those still
  // in flight end before the memory goes. ----
  __syncwarp();
  tc_fence_before();
  if (!__syncthreads_and(ok)) {
    if (warp == 0 || warp == 3) {
      const int n_bufs = warp == 3 ? plan.v_bufs : plan.k_bufs;
      for (int g = max(0, issued - n_bufs); g < issued; ++g)
        da_wait(&(warp == 3 ? v_full : k_full)[g % n_bufs], (g / n_bufs) & 1, nullptr, 0);
      for (int e = max(0, q_issued - plan.q_bufs); e < q_issued; ++e)
        da_wait(&q_full[e % plan.q_bufs], (e / plan.q_bufs) & 1, nullptr, 0);
    } else if (warp < 3) {
      if (elect_one()) mma_commit(&all_done[warp - 1]);
      __syncwarp();
      da_wait(&all_done[warp - 1], 0, nullptr, 0);
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

// Tokens from .. to - 1 as if they saw nothing, by `count` threads of which this is number `me`.
template <int D, typename T>
__device__ __noinline__ void da_blank(const DraftAttnArgs& a, int64_t from, int64_t to, int64_t me, int64_t count) {
  constexpr int PER = D / 8;
  for (int64_t i = from * a.hq * PER + me; i < to * a.hq * PER; i += count) reinterpret_cast<uint4*>(a.out)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (a.lse)
    for (int64_t i = from * a.hq + me; i < to * a.hq; i += count) a.lse[i] = -INFINITY;
}

// Joins the parts of an item that was cut: one warp a row, parts in piece order. Block (c, y): the item that begins in
// piece c, rows 8 y .. 8 y + 7. And writes the tokens that no item has: those before cu_0 and from cu_rows on, by all blocks,
// and those of requests whose lengths are out of range, by the blocks (request mod pieces, 0).
template <int D, typename T>
__global__ void __launch_bounds__(DJ_THREADS) draft_join_kernel(const __grid_constant__ DraftAttnArgs a, int block,
                                                                const DaSplit* splits, const float* partials) {
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();  // the next call's set-up
  const int c = blockIdx.x, lane = threadIdx.x & 31;
  const DaSplit s = splits[c];
  const int lead = a.cu[0], trail = a.cu[a.rows];
  if (lead > 0 || trail < a.tokens) {
    const int64_t me = ((int64_t)blockIdx.y * DA_PIECES + c) * DJ_THREADS + threadIdx.x, all = (int64_t)gridDim.y * DA_PIECES * DJ_THREADS;
    da_blank<D, T>(a, 0, min(lead, a.tokens), me, all);
    da_blank<D, T>(a, max(trail, 0), a.tokens, me, all);
  }
  if (blockIdx.y == 0) {
    for (int b0 = c + DA_PIECES * (threadIdx.x & ~31); b0 < a.rows; b0 += DA_PIECES * DJ_THREADS) {
      const int b = b0 + DA_PIECES * lane;
      const bool out = b < a.rows && a.cu[b + 1] > a.cu[b] && da_request<da_tile(D)>(a, block, b, false).n == 0;
      for (unsigned rest = __ballot_sync(0xffffffffu, out); rest; rest &= rest - 1) {
        const int r = b0 + DA_PIECES * (__ffs(rest) - 1);
        da_blank<D, T>(a, max(a.cu[r], 0), min(a.cu[r + 1], a.tokens), lane, 32);
      }
    }
  }
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
  if (lane == 0 && a.lse) a.lse[orow] = l > 0.f || l != l ? (m - DaType<T>::kLift + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace hsg
