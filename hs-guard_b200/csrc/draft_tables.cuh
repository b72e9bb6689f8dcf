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
//
// Every block sums over all requests by itself (two block scans, a few microseconds at most: cheaper than a second
// launch or a wait between blocks) and then takes its share of the pages and tokens, found by bisection in the prefix
// sums. Bound by launch and scan latency up to some 100,000 tokens, by the 12 bytes written a token beyond.
#pragma once
#include "common.cuh"

namespace hsg {

constexpr int DT_THREADS = 1024;
constexpr int DT_MAX_ROWS = 4096;
constexpr int DT_PER = DT_MAX_ROWS / DT_THREADS;  // requests a thread

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
  int32_t* lens_out;         // [rows]
  int64_t* counters_out;
  int32_t* cu;               // [rows + 1] appended tokens before each request
  int32_t* slots;            // [capacity] page id * page + offset; -1 past the last token, like the next two
  int32_t* token_rows;       // [capacity] request
  int32_t* positions;        // [capacity]
  int capacity;
  int* err;
};

// Exclusive prefix sums of two values at once over the block's threads; the totals go to tot.
__device__ __forceinline__ longlong2 block_scan2(longlong2 v, longlong2* warp_sums, longlong2& tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto scan = [&](longlong2 s) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, s.x, o), y = __shfl_up_sync(0xffffffffu, s.y, o);
      if (lane >= o) { s.x += x; s.y += y; }
    }
    return s;
  };
  const longlong2 s = scan(v);
  __syncthreads();  // an earlier scan's readers of warp_sums are done
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) warp_sums[lane] = scan(warp_sums[lane]);
  __syncthreads();
  tot = warp_sums[DT_THREADS / 32 - 1];
  const longlong2 before = warp ? warp_sums[warp - 1] : make_longlong2(0, 0);
  return make_longlong2(before.x + s.x - v.x, before.y + s.y - v.y);
}

// The last entry of the ascending first[0 .. n) that is at most i; first[0] <= i.
__device__ __forceinline__ int last_at_most(const int* first, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(DT_THREADS) draft_tables_kernel(const __grid_constant__ DraftTablesArgs a) {
  extern __shared__ int dt_smem[];
  __shared__ longlong2 warp_sums[DT_THREADS / 32];
  int* s_cu = dt_smem;            // [rows] tokens before the request, at most capacity
  int* s_take = s_cu + a.rows;    // [rows] pages taken before it
  int* s_give = s_take + a.rows;  // [rows] pages given back before it
  const int tid = threadIdx.x;
  const bool writes = blockIdx.x == 0;
  const int64_t head = a.counters[0], tail = a.counters[1];
  const bool sane = head >= 0 && tail >= head && tail - head <= a.ring_size;
  if (!sane && writes && tid == 0) set_error(a.err, ERR_BAD_LEN);
  const int64_t avail = sane ? tail - head : 0;
  const int head_at = sane ? (int)(head % a.ring_size) : 0, tail_at = sane ? (int)(tail % a.ring_size) : 0;
  const int most = a.width * (int)a.page.d;  // tokens a table row can hold (checked to be below 2^31)
  auto pages = [&](int n) { return n <= 0 ? 0 : (int)a.page.div((uint32_t)(n - 1)) + 1; };
  auto ring_at = [&](int from, int i) {
    const uint32_t x = (uint32_t)from + (uint32_t)i;
    return (int)(x < (uint32_t)a.ring_size ? x : x % (uint32_t)a.ring_size);
  };
  const int per = (a.rows + DT_THREADS - 1) / DT_THREADS, b0 = tid * per;
  int len[DT_PER], to[DT_PER];
  longlong2 sum = make_longlong2(0, 0), tot;
#pragma unroll
  for (int k = 0; k < DT_PER; ++k) {
    len[k] = to[k] = 0;
    if (k >= per || b0 + k >= a.rows) continue;
    len[k] = to[k] = a.lens[b0 + k];
    if (len[k] < 0 || len[k] > most) {
      if (writes) set_error(a.err, ERR_BAD_LEN);
      continue;
    }
    const int64_t want = (int64_t)len[k] + a.delta[b0 + k];
    if (want <= most) to[k] = want < 0 ? 0 : (int)want;
    const int d = pages(to[k]) - pages(len[k]);
    sum.x += max(d, 0);
    sum.y += max(-d, 0);
  }
  const longlong2 at = block_scan2(sum, warp_sums, tot);
  // more pages than the ring has cannot come back: lengths that say so are wrong
  const bool returns = tot.y <= a.ring_size;
  if (!returns && writes && tid == 0) set_error(a.err, ERR_BAD_LEN);
  const int given = returns ? (int)tot.y : 0;
  longlong2 grown = make_longlong2(0, 0);  // tokens, pages
  int64_t need = at.x;
#pragma unroll
  for (int k = 0; k < DT_PER; ++k) {
    const int d = pages(to[k]) - pages(len[k]);
    need += max(d, 0);
    if (d > 0 && need > avail) to[k] = len[k];  // not served
    grown.x += max(to[k] - len[k], 0);
    if (to[k] > len[k]) grown.y += d;
  }
  const longlong2 put = block_scan2(grown, warp_sums, tot);
  const int total = (int)(tot.x < a.capacity ? tot.x : a.capacity), taken = (int)tot.y;
  {
    int64_t tokens = put.x;
    int take = (int)put.y, give = (int)at.y;
#pragma unroll
    for (int k = 0; k < DT_PER; ++k) {
      const int b = b0 + k;
      if (k >= per || b >= a.rows) continue;
      const int d = pages(to[k]) - pages(len[k]);
      s_cu[b] = (int)(tokens < a.capacity ? tokens : a.capacity);
      s_take[b] = take;
      s_give[b] = give;
      if (writes) {
        a.lens_out[b] = to[k];
        a.cu[b] = (int)(tokens < INT32_MAX ? tokens : INT32_MAX);
      }
      tokens += max(to[k] - len[k], 0);
      take += max(d, 0);
      give += max(-d, 0);
    }
  }
  if (writes && tid == 0) {
    a.cu[a.rows] = (int)(tot.x < INT32_MAX ? tot.x : INT32_MAX);
    a.counters_out[0] = head + taken;
    a.counters_out[1] = tail + given;
    if (tot.x > a.capacity) set_error(a.err, ERR_BAD_LEN);
  }
  __syncthreads();
  const int me = blockIdx.x * DT_THREADS + tid, all = gridDim.x * DT_THREADS;
  for (int i = me; i < taken; i += all) {
    const int b = last_at_most(s_take, a.rows, i);
    a.table[b * a.table_stride + pages(a.lens[b]) + i - s_take[b]] = a.ring[ring_at(head_at, i)];
  }
  for (int i = me; i < given; i += all) {
    // the last pages of a request that keeps its first pages(to): to is lens_out's value, found again
    const int b = last_at_most(s_give, a.rows, i);
    const int64_t want = (int64_t)a.lens[b] + a.delta[b];
    a.ring[ring_at(tail_at, i)] = a.table[b * a.table_stride + pages(want < 0 ? 0 : (int)want) + i - s_give[b]];
  }
  // four tokens at a time; a token in a page of this call's finds its page in the ring, whether or not another block
  // has already written it to the table
  const bool wide = ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.token_rows) |
                      reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0;
  const int quads = a.capacity / 4 + (a.capacity % 4 != 0);
  for (int q = me; q < quads; q += all) {
    int slot[4], row[4], pos[4];
    int b = -1, next = 0, n = 0, held = 0, page_id = 0, page_no = -1;  // page_id: of page page_no of request b
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = 4 * q + k;
      slot[k] = row[k] = pos[k] = -1;
      if (i >= total) continue;
      if (i >= next || b < 0) {
        b = last_at_most(s_cu, a.rows, i);
        next = b + 1 < a.rows ? s_cu[b + 1] : total;
        n = a.lens[b];
        held = pages(n);
        page_no = -1;
      }
      const int p = n + i - s_cu[b], no = (int)a.page.div((uint32_t)p);
      if (no != page_no) {
        page_no = no;
        page_id = no < held ? a.table[b * a.table_stride + no] : a.ring[ring_at(head_at, s_take[b] + no - held)];
      }
      slot[k] = page_id * (int)a.page.d + p - no * (int)a.page.d;
      row[k] = b;
      pos[k] = p;
    }
    if (wide && 4 * q + 4 <= a.capacity) {
      reinterpret_cast<int4*>(a.slots)[q] = make_int4(slot[0], slot[1], slot[2], slot[3]);
      reinterpret_cast<int4*>(a.token_rows)[q] = make_int4(row[0], row[1], row[2], row[3]);
      reinterpret_cast<int4*>(a.positions)[q] = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (4 * q + k >= a.capacity) break;
        a.slots[4 * q + k] = slot[k];
        a.token_rows[4 * q + k] = row[k];
        a.positions[4 * q + k] = pos[k];
      }
    }
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
