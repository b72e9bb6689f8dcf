// Integer bookkeeping of draft scoring: block tables and slot maps of a paged key/value cache (draft_tables_kernel)
// and the positions and ancestor masks of drafted trees (draft_tree_kernel). No counterpart in the reference, whose
// rings have one fixed place for every position and whose ticks are chains.
//
// Pages. Request b holds len_b tokens in ceil(len_b / page) pages, listed in order in its row of the table. Free pages
// wait in a ring: counters = (head, tail), both only ever growing, entries head .. tail - 1 (modulo the ring's size)
// are free. A request that grows takes entries from the head in request order, one that shrinks puts its last pages
// back at the tail. Takes read entries below the tail at entry and returns write from that tail on, so a call neither
// reads what it writes nor needs an order between thread blocks, and running it again on the same inputs gives the
// same result.
#pragma once
#include "common.cuh"

namespace hsg {

constexpr int DT_THREADS = 1024;
constexpr int DT_MAX_ROWS = 4096;

struct DraftTablesArgs {
  const int32_t* lens;       // [rows]
  const int32_t* delta;      // [rows] tokens to append (> 0) or take back (< 0)
  int32_t* table;            // [rows][width], rows table_stride apart
  int64_t table_stride;
  int32_t* ring;             // [ring_size] page ids
  const int64_t* counters;   // head, tail
  int rows, width, ring_size, page;
  int32_t* lens_out;         // [rows]
  int64_t* counters_out;
  int32_t* cu;               // [rows + 1] appended tokens before each request
  int32_t* slots;            // [capacity] page id * page + offset; -1 past the last token, like the next two
  int32_t* token_rows;       // [capacity] request
  int32_t* positions;        // [capacity]
  int capacity;
  int* err;
};

// Exclusive prefix sums over the block's threads of two values at once; the totals go to tot.
__device__ __forceinline__ longlong2 block_scan2(longlong2 v, longlong2* warp_tot, longlong2& tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  longlong2 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, s.x, o), y = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) { s.x += x; s.y += y; }
  }
  __syncthreads();  // an earlier scan's readers of warp_tot are done
  if (lane == 31) warp_tot[warp] = s;
  __syncthreads();
  longlong2 before = make_longlong2(0, 0);
  tot = make_longlong2(0, 0);
  for (int w = 0; w < DT_THREADS / 32; ++w) {
    const longlong2 t = warp_tot[w];
    if (w < warp) { before.x += t.x; before.y += t.y; }
    tot.x += t.x;
    tot.y += t.y;
  }
  return make_longlong2(before.x + s.x - v.x, before.y + s.y - v.y);
}

// One thread block: every request's pages, then every token's slot.
__global__ void __launch_bounds__(DT_THREADS) draft_tables_kernel(const DraftTablesArgs a) {
  __shared__ longlong2 warp_tot[DT_THREADS / 32];
  __shared__ int s_cu[DT_MAX_ROWS + 1];
  const int tid = threadIdx.x;
  const int64_t head = a.counters[0], tail = a.counters[1];
  const int per = (a.rows + DT_THREADS - 1) / DT_THREADS, b0 = min(a.rows, tid * per), b1 = min(a.rows, b0 + per);
  auto target = [&](int b) -> int64_t {
    const int64_t len = a.lens[b], to = len + a.delta[b];
    if (len < 0 || len > (int64_t)a.width * a.page) {
      set_error(a.err, ERR_BAD_LEN);
      return len;
    }
    return to < 0 ? 0 : to > (int64_t)a.width * a.page ? len : to;
  };
  auto pages = [&](int64_t n) { return n <= 0 ? 0 : (n + a.page - 1) / a.page; };
  longlong2 sum = make_longlong2(0, 0), tot;
  for (int b = b0; b < b1; ++b) {
    const int64_t d = pages(target(b)) - pages(a.lens[b]);
    sum.x += d > 0 ? d : 0;
    sum.y += d < 0 ? -d : 0;
  }
  longlong2 at = block_scan2(sum, warp_tot, tot);
  const int64_t back_total = tot.y;
  longlong2 grown = make_longlong2(0, 0);
  {
    int64_t need = at.x;
    for (int b = b0; b < b1; ++b) {
      const int64_t to = target(b), d = pages(to) - pages(a.lens[b]);
      need += d > 0 ? d : 0;
      const bool served = d <= 0 || need <= tail - head;
      if (served && to > a.lens[b]) grown.x += to - a.lens[b];
      if (served && d > 0) grown.y += d;
    }
  }
  longlong2 tok = block_scan2(grown, warp_tot, tot);
  {
    int64_t need = at.x, back = at.y, t = tok.x;
    for (int b = b0; b < b1; ++b) {
      const int64_t len = a.lens[b], to = target(b), p0 = pages(len), p1 = pages(to);
      const int64_t first = need;
      need += p1 > p0 ? p1 - p0 : 0;
      const bool served = p1 <= p0 || need <= tail - head;
      int32_t* row = a.table + b * a.table_stride;
      if (served)
        for (int64_t p = p0; p < p1; ++p) row[p] = a.ring[(head + first + p - p0) % a.ring_size];
      for (int64_t p = p1; p < p0; ++p) a.ring[(tail + back++) % a.ring_size] = row[p];
      a.lens_out[b] = (int32_t)(served ? to : len);
      s_cu[b] = (int)(t > a.capacity ? a.capacity : t);
      a.cu[b] = (int32_t)t;
      if (served && to > len) t += to - len;
    }
  }
  if (tid == 0) {
    a.cu[a.rows] = (int32_t)tot.x;
    a.counters_out[0] = head + tot.y;
    a.counters_out[1] = tail + back_total;
    if (tot.x > a.capacity) set_error(a.err, ERR_BAD_LEN);
  }
  __threadfence_block();
  __syncthreads();
  const int total = (int)(tot.x > a.capacity ? a.capacity : tot.x);
  for (int i = tid; i < a.capacity; i += DT_THREADS) {
    int slot = -1, r = -1, pos = -1;
    if (i < total) {
      int lo = 0, hi = a.rows;  // the last request that starts at or before i
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= i) lo = mid; else hi = mid;
      }
      r = lo;
      pos = a.lens[r] + i - s_cu[r];
      slot = a.table[r * a.table_stride + pos / a.page] * a.page + pos % a.page;
    }
    a.slots[i] = slot;
    a.token_rows[i] = r;
    a.positions[i] = pos;
  }
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

// One thread block a request, one thread a node: the node's chain of parents, which ends because every link goes to
// an earlier node. The indexes along it fall, so a mask word is complete once the chain has passed below it.
__global__ void __launch_bounds__(DTREE_THREADS) draft_tree_kernel(const DraftTreeArgs a) {
  const int b = blockIdx.x;
  int64_t t0 = a.cu[b], t1 = a.cu[b + 1];
  if (t0 < 0 || t1 < t0 || t1 > a.tokens || t1 - t0 > 32 * a.words) {
    if (threadIdx.x == 0) set_error(a.err, ERR_BAD_LEN);
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
