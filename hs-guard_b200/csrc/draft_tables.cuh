// Integer bookkeeping of draft scoring: block tables and slot maps of a paged key/value cache (draft_tables_kernel)
// and the positions and ancestor masks of drafted trees (draft_tree_kernel). No counterpart in the reference, whose
// rings have one fixed place for every position and whose ticks are chains.
//
// Pages. Request b holds len_b tokens in ceil(len_b / page) pages, listed in order in its row of the table. Free pages
// wait in a ring: counters = (head, tail), both only ever growing, entries head .. tail - 1 (modulo the ring's size)
// are free. A request that grows takes entries from the head in request order, one that shrinks puts its last pages
// back at the tail. Takes read entries below the tail at entry and returns write from that tail on, as far as the ring has
// places that hold no free page at entry (a ring with an entry for every page always has); returns beyond them are not
// made. So a call neither reads what it writes nor needs an order between thread blocks, and running it again on the same
// inputs gives the same result. A page id that is negative, or whose slots are beyond 32 bits, is none: it moves on as -1, so
// that no other page is handed out in its place, its tokens have slot -1, and the error word says so.
//
// Every block sums over all requests by itself (two block scans: cheaper than a second launch or a wait between blocks)
// and then takes its share of the pages and tokens, found by bisection in the prefix sums. Bound by launch and latency up
// to some 100,000 tokens, by the 12 bytes written a token beyond: 5.9 us for 352 requests that accept or withdraw a few
// tokens, 13.1 us for 870,000 tokens of 1,000 prompts (10 MB, 0.8 TB/s). Blocks of 1,024 threads took 10.6 us for the first: their warps
// issue the same few scalar steps four times as often.
#pragma once
#include "common.cuh"

namespace hsg {

constexpr int DT_THREADS = 256;
constexpr int DT_MAX_ROWS = 4096;

// Division of 0 <= n < 2^31 by d: n * m >> (31 + s) with m = floor(2^(31 + s) / d) + 1, 2^(s - 1) < d <= 2^s.
struct FastDiv {
  uint32_t d, m;
  int s;
  __host__ static FastDiv of(int d) {
    FastDiv f{(uint32_t)d, 0, 0};
    while ((1ll << f.s) < d) ++f.s;
    f.m = (uint32_t)((1ull << (31 + f.s)) / (uint64_t)d + 1);
    return f;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)((uint64_t)n * m >> (31 + s)); }
};

struct DraftTablesArgs {
  const int32_t* lens;       // [rows]
  const int32_t* delta;      // [rows] tokens to append (> 0) or take back (< 0)
  int32_t* table;            // [rows][width], rows table_stride apart
  int64_t table_stride;
  int32_t* ring;             // [ring_size] page ids
  const int64_t* counters;   // head, tail
  int rows, width, ring_size;
  FastDiv page;
  uint32_t page_ids;         // ids below this have slots below 2^31
  int32_t* lens_out;         // [rows]
  int64_t* counters_out;
  int32_t* cu;               // [rows + 1] appended tokens before each request
  int32_t* slots;            // [capacity] page id * page + offset; -1 past the last token, like the next two
  int32_t* token_rows;       // [capacity] request
  int32_t* positions;        // [capacity]
  int capacity;
  int* err;
};

// Sums that stay at 2^32 - 1 when they would pass it: counts of pages and tokens are compared with less than 2^31.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;
  return s < a ? 0xffffffffu : s;
}

// Exclusive prefix sums of two values at once over the block's threads; the totals go to tot.
__device__ __forceinline__ uint2 block_scan2(uint2 v, uint2* warp_sums, uint2& tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint2 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, s.x, o), y = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) s = make_uint2(add_sat(s.x, x), add_sat(s.y, y));
  }
  __syncthreads();  // an earlier scan's readers of warp_sums are done
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  const uint32_t px = __shfl_up_sync(0xffffffffu, s.x, 1), py = __shfl_up_sync(0xffffffffu, s.y, 1);
  uint2 before = lane ? make_uint2(px, py) : make_uint2(0, 0);
  tot = make_uint2(0, 0);
#pragma unroll
  for (int w = 0; w < DT_THREADS / 32; ++w) {
    const uint2 t = warp_sums[w];
    if (w < warp) before = make_uint2(add_sat(before.x, t.x), add_sat(before.y, t.y));
    tot = make_uint2(add_sat(tot.x, t.x), add_sat(tot.y, t.y));
  }
  return before;
}

// The last entry of the ascending first[0 .. n) that is at most i; first[0] <= i.
__device__ __forceinline__ int last_at_most(const uint32_t* first, int n, uint32_t i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

constexpr int DT_ROW_BYTES = 20;  // of shared memory a request

__global__ void __launch_bounds__(DT_THREADS) draft_tables_kernel(const __grid_constant__ DraftTablesArgs a) {
  extern __shared__ uint32_t dt_smem[];
  __shared__ uint2 warp_sums[DT_THREADS / 32];
  __shared__ int s_ring[4];       // head and tail modulo the ring's size, free pages, places without one
  __shared__ uint32_t s_given;    // pages given back, where not all can be
  uint32_t* s_cu = dt_smem;       // [rows] tokens before the request
  uint32_t* s_take = s_cu + a.rows;  // [rows] pages taken before it
  uint32_t* s_give = s_take + a.rows;  // [rows] pages given back before it
  int* s_len = reinterpret_cast<int*>(s_give + a.rows);  // [rows] its length
  int* s_to = s_len + a.rows;     // [rows] and what that becomes
  const int tid = threadIdx.x;
  const bool writes = blockIdx.x == 0;
  const int most = a.width * (int)a.page.d;  // tokens a table row can hold (checked to be below 2^31)
  auto pages = [&](int n) { return n <= 0 ? 0 : (int)a.page.div((uint32_t)(n - 1)) + 1; };
  auto ring_at = [&](int from, uint32_t i) {
    const uint32_t x = (uint32_t)from + i;
    return (int)(x < (uint32_t)a.ring_size ? x : x % (uint32_t)a.ring_size);
  };
  for (int b = tid; b < a.rows; b += DT_THREADS) {
    const int len = a.lens[b];
    const int64_t want = (int64_t)len + a.delta[b];
    const bool good = len >= 0 && len <= most;
    if (!good && writes) set_error(a.err, ERR_BAD_LEN);
    s_len[b] = len;
    s_to[b] = !good || want > most ? len : want < 0 ? 0 : (int)want;
  }
  if (tid == DT_THREADS - 1) {
    const int64_t head = a.counters[0], tail = a.counters[1];
    const bool sane = head >= 0 && tail >= head && tail - head <= a.ring_size;
    if (!sane && writes) set_error(a.err, ERR_BAD_LEN);
    s_ring[0] = sane ? (int)(head % a.ring_size) : 0;
    s_ring[1] = sane ? (int)(tail % a.ring_size) : 0;
    s_ring[2] = sane ? (int)(tail - head) : 0;
    s_ring[3] = sane ? a.ring_size - (int)(tail - head) : 0;
    s_given = 0;
  }
  __syncthreads();
  const int head_at = s_ring[0], tail_at = s_ring[1];
  const uint32_t avail = (uint32_t)s_ring[2], room = (uint32_t)s_ring[3];
  const int per = (a.rows + DT_THREADS - 1) / DT_THREADS, b0 = min(a.rows, tid * per), b1 = min(a.rows, b0 + per);
  uint2 sum = make_uint2(0, 0), tot;  // pages wanted, pages given back
  for (int b = b0; b < b1; ++b) {
    const int d = pages(s_to[b]) - pages(s_len[b]);
    sum = make_uint2(add_sat(sum.x, max(d, 0)), add_sat(sum.y, max(-d, 0)));
  }
  const uint2 at = block_scan2(sum, warp_sums, tot);
  // a place may hold a page that this call takes, so a return into it would have to come after the take
  const uint32_t returned = tot.y;
  if (returned > room && writes && tid == 0) set_error(a.err, ERR_BAD_LEN);
  uint2 grown = make_uint2(0, 0);  // tokens, pages
  uint32_t need = at.x, back = at.y;
  for (int b = b0; b < b1; ++b) {
    const int len = s_len[b], d = pages(s_to[b]) - pages(len);
    need = add_sat(need, max(d, 0));
    back = add_sat(back, max(-d, 0));
    if ((d > 0 && need > avail) || (d < 0 && back > room)) s_to[b] = len;  // not served
    else if (d < 0 && returned > room) atomicMax(&s_given, back);
    if (s_to[b] > len) grown = make_uint2(add_sat(grown.x, s_to[b] - len), add_sat(grown.y, d));
  }
  const uint2 put = block_scan2(grown, warp_sums, tot);
  const uint32_t given = returned > room ? s_given : returned;
  const uint32_t total = min(tot.x, (uint32_t)a.capacity), taken = tot.y;
  uint32_t tokens = put.x, take = put.y, give = at.y;
  for (int b = b0; b < b1; ++b) {
    const int len = s_len[b], to = s_to[b], d = pages(to) - pages(len);
    s_cu[b] = tokens;
    s_take[b] = take;
    s_give[b] = give;
    if (writes) {
      a.lens_out[b] = to;
      a.cu[b] = (int)min(tokens, 0x7fffffffu);
    }
    if (to > len) {
      tokens = add_sat(tokens, to - len);
      take = add_sat(take, d);
    }
    give = add_sat(give, max(-d, 0));
  }
  if (writes && tid == 0) {
    a.cu[a.rows] = (int)min(tot.x, 0x7fffffffu);
    a.counters_out[0] = a.counters[0] + taken;
    a.counters_out[1] = a.counters[1] + given;
    if (tot.x > (uint32_t)a.capacity) set_error(a.err, ERR_BAD_LEN);
  }
  __syncthreads();
  bool bad = false;  // this thread has met an id that is none (recorded at the end: a branch here would wait for each load)
  auto id_of = [&](int id) {
    const bool is = (uint32_t)id < a.page_ids;
    bad |= !is;
    return is ? id : -1;
  };
  // warps of all blocks in turn, so that a few entries spread over the SMs
  const uint32_t me = ((tid >> 5) * gridDim.x + blockIdx.x) * 32 + (tid & 31), all = gridDim.x * DT_THREADS;
  for (uint32_t i = me; i < taken; i += all) {
    const int b = last_at_most(s_take, a.rows, i);
    a.table[b * a.table_stride + pages(s_len[b]) + (i - s_take[b])] = id_of(a.ring[ring_at(head_at, i)]);
  }
  for (uint32_t i = me; i < given; i += all) {
    const int b = last_at_most(s_give, a.rows, i);
    a.ring[ring_at(tail_at, i)] = id_of(a.table[b * a.table_stride + pages(s_to[b]) + (i - s_give[b])]);
  }
  // the page's first slot, or -1 if its id is none. A token in a page of this call's finds its page in the ring, whether or
  // not another block has already written it to the table
  auto page_of = [&](int b, int no, int held) {
    const int id = id_of(no < held ? a.table[b * a.table_stride + no] : a.ring[ring_at(head_at, s_take[b] + (no - held))]);
    return id < 0 ? -1 : id * (int)a.page.d;
  };
  auto slot_in = [&](int first, int offset) { return (first + offset) | first >> 31; };
  const bool wide = ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.token_rows) |
                      reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0;
  if (!wide || (uint32_t)a.capacity <= 4 * all) {  // few: a token a thread, for the shortest chain of loads
    for (uint32_t i = me; i < (uint32_t)a.capacity; i += all) {
      int slot = -1, row = -1, pos = -1;
      if (i < total) {
        row = last_at_most(s_cu, a.rows, i);
        pos = s_len[row] + (int)(i - s_cu[row]);
        const int no = (int)a.page.div((uint32_t)pos);
        slot = slot_in(page_of(row, no, pages(s_len[row])), pos - no * (int)a.page.d);
      }
      a.slots[i] = slot;
      a.token_rows[i] = row;
      a.positions[i] = pos;
    }
    if (bad) set_error(a.err, ERR_BAD_PAGE);
    return;
  }
  const uint32_t quads = ((uint32_t)a.capacity + 3) / 4;  // many: four at a time
  for (uint32_t q = me; q < quads; q += all) {
    int slot[4], row[4], pos[4];
    int b = -1, held = 0, first = 0, page_no = -1;  // first: slot of page page_no of request b
    uint32_t next = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t i = 4 * q + k;
      slot[k] = row[k] = pos[k] = -1;
      if (i >= total) continue;
      if (i >= next) {
        b = last_at_most(s_cu, a.rows, i);
        next = b + 1 < a.rows ? s_cu[b + 1] : total;
        held = pages(s_len[b]);
        page_no = -1;
      }
      const int p = s_len[b] + (int)(i - s_cu[b]), no = (int)a.page.div((uint32_t)p);
      if (no != page_no) {
        page_no = no;
        first = page_of(b, no, held);
      }
      slot[k] = slot_in(first, p - no * (int)a.page.d);
      row[k] = b;
      pos[k] = p;
    }
    if (4 * q + 4 <= (uint32_t)a.capacity) {
      reinterpret_cast<int4*>(a.slots)[q] = make_int4(slot[0], slot[1], slot[2], slot[3]);
      reinterpret_cast<int4*>(a.token_rows)[q] = make_int4(row[0], row[1], row[2], row[3]);
      reinterpret_cast<int4*>(a.positions)[q] = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (4 * q + k >= (uint32_t)a.capacity) break;
        a.slots[4 * q + k] = slot[k];
        a.token_rows[4 * q + k] = row[k];
        a.positions[4 * q + k] = pos[k];
      }
    }
  }
  if (bad) set_error(a.err, ERR_BAD_PAGE);
}

struct DraftTreeArgs {
  const int32_t* parents;  // [tokens] index within the request, -1 for a child of the last cached token
  const int32_t* cu;       // [rows + 1]
  const int32_t* lens;     // [rows] cached tokens
  int rows, tokens, words;
  int32_t* positions;      // [tokens]
  uint32_t* mask;          // [tokens][words]: bit j of node i set iff j is i or one of its ancestors
  int* err;
};

constexpr int DTREE_THREADS = 128;

// Nodes from .. to - 1, as far as they exist, as those of no request. Rare, so out of line.
__device__ __noinline__ void dtree_blank(const DraftTreeArgs& a, int64_t from, int64_t to) {
  for (int64_t t = max(from, (int64_t)0) + threadIdx.x; t < min(to, (int64_t)a.tokens); t += DTREE_THREADS) {
    a.positions[t] = -1;
    for (int w = 0; w < a.words; ++w) a.mask[t * a.words + w] = 0;
  }
}

// One thread block a request, one thread a node: the node's chain of parents, which ends because every link goes to
// an earlier node. The indexes along it fall, so a mask word is complete once the chain has passed below it. Nodes of no
// request (before cu_0 and from cu_rows on, by the first and the last block) and of a request that is refused have position -1 and no bits.
__global__ void __launch_bounds__(DTREE_THREADS) draft_tree_kernel(const __grid_constant__ DraftTreeArgs a) {
  const int b = blockIdx.x;
  const int64_t t0 = a.cu[b], t1 = a.cu[b + 1];
  const bool refused = t0 < 0 || t1 < t0 || t1 > a.tokens || t1 - t0 > 32 * a.words;
  if (b == 0 && t0 > 0) dtree_blank(a, 0, t0);
  if (b == a.rows - 1 && t1 < a.tokens) dtree_blank(a, t1, a.tokens);
  if (refused) {
    if (threadIdx.x == 0) set_error(a.err, ERR_BAD_LEN);
    dtree_blank(a, t0, t1);
    return;
  }
  for (int i = threadIdx.x; i < t1 - t0; i += DTREE_THREADS) {
    uint32_t* out = a.mask + (t0 + i) * a.words;
    int word = a.words - 1, depth = -1;
    uint32_t bits = 0;
    for (int j = i; j >= 0; ++depth) {
      for (; word > (j >> 5); --word) {
        out[word] = bits;
        bits = 0;
      }
      bits |= 1u << (j & 31);
      const int p = a.parents[t0 + j];
      if (p < -1 || p >= j) {
        set_error(a.err, ERR_BAD_PARENT);
        ++depth;
        break;
      }
      j = p;
    }
    for (; word >= 0; --word) {
      out[word] = bits;
      bits = 0;
    }
    a.positions[t0 + i] = a.lens[b] + depth;
  }
}

}  // namespace hsg
