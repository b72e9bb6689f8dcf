// Log-probabilities of given tokens, entropy and the most likely alternatives, from rows of logits (logprobs_kernel).
//
// With z_i = x_i / T and m the row's largest x: S = sum e^(z_i - m / T), U = sum e^(z_i - m / T) (z_i - m / T), then
//   log-sum-exp = m / T + ln S,  entropy = ln S - U / S,  log p_i = (x_i - m) / T - ln S.
// One pass over the row keeps (m, S, U) a thread, S and U rescaled when a thread's m rises. Differences to m are taken before
// they are scaled, so that rows of the type's lowest value are rows like others, and are kept above -200 (in powers of two):
// e^-inf is 0 and 0 times that difference 0, while NaN stays NaN.
//
// Alternatives: a thread also remembers the largest value that it met. A value tau that at least `top` threads' largest reach
// (a bisection over its bits, threads counted by a block-wide vote) is no larger than the top-th value of the block's share,
// so every alternative is at least tau and lies with a thread whose largest is: only what those few threads read is read
// again, by all threads, and what reaches tau becomes a candidate (about as many as are asked for), ranked by counting.
// Equal values rank by token, the lowest first. If too many values reach tau, the alternatives
// are taken one by one instead: the block's largest, after which its owner's warp looks for that thread's next. That happens in long
// runs of equal or ascending values, and where fewer threads than alternatives meet anything but -inf (a grammar that leaves a
// few tokens or a run of them): 30 allowed tokens and 20 alternatives take one row of 248,320 fp32 43 us, 352 rows of bf16 351, 2,500
// rows of 50,001 fp16 415.
//
// A row is shared by a cluster of up to 8 blocks, whose parts meet in the first one's shared memory.
//
// Bound by HBM and, for 16-bit logits, by exponentials (16 a clock and SM) and instructions nearly alike: 352 rows of 248,320 bf16 in 46 us,
// 3.8 TB/s; 2,500 rows of 50,001 fp16 in 71 us, 3.5 TB/s, of which the alternatives take 16 and the turn from row to row most of
// the rest; one row of 248,320 fp32 in 10.7 us, a chain of latencies.
#pragma once
#include "draft_rows.cuh"
#include "draft_attn.cuh"  // ex2_approx, add2, fma2

namespace hsg {

struct LogprobsArgs {
  const void* x;           // [rows][vocab], rows `stride` elements apart, on any element
  int64_t stride;
  const int32_t* given;    // [rows][n_given]; < 0: none
  int rows, vocab, n_given, top;
  float inv_t;             // 1 / temperature
  float* logprobs;         // [rows][n_given]
  float* entropy;          // [rows]
  float* lse;              // [rows]
  float* top_logprobs;     // [rows][top]
  int32_t* top_ids;        // [rows][top]
  int* err;
};

constexpr int LP_MAX_TOP = 64;
constexpr int LP_CLUSTER = 8;
constexpr int LP_CAND = 512;      // candidates that are ranked by counting
constexpr int LP_MORE = 12;       // threads beyond `top` whose values are read again, as far as the bisection can tell
constexpr int LP_LIVE = 4;        // 16-byte pieces a thread has under way

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Order of values as unsigned numbers; NaN is above everything.
__device__ __forceinline__ uint32_t lp_order(float x) {
  const uint32_t b = __float_as_uint(x);
  return x != x ? ~0u : b ^ ((b >> 31) ? ~0u : 0x80000000u);
}
// A value and its token as one number: larger values first, of equal ones the lower token. Never 0.
__device__ __forceinline__ uint64_t lp_key(float x, int i) {
  // -0 and 0 are equal
  return (uint64_t)lp_order(x == 0.f ? 0.f : x) << 32 | (uint32_t)~(uint32_t)i;
}
__device__ __forceinline__ float lp_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : ~0u));
}
__device__ __forceinline__ int lp_token(uint64_t key) { return (int)~(uint32_t)key; }

template <typename T, int N> __device__ __forceinline__ void lp_unpack(const uint4& r, float (&x)[N]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      x[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = unpack_half2(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <typename T, int N> __device__ __forceinline__ void lp_load(const T* p, float (&x)[N]) {
  lp_unpack<T>(__ldg(reinterpret_cast<const uint4*>(p)), x);
}
// The largest of them; NaN do not count beside numbers.
template <typename T> __device__ __forceinline__ float lp_max(const uint4 (&r)[LP_LIVE]) {
  uint32_t w[4 * LP_LIVE];
#pragma unroll
  for (int u = 0; u < LP_LIVE; ++u) {
    w[4 * u] = r[u].x;
    w[4 * u + 1] = r[u].y;
    w[4 * u + 2] = r[u].z;
    w[4 * u + 3] = r[u].w;
  }
  if constexpr (sizeof(T) == 4) {
    float t = __uint_as_float(w[0]);
#pragma unroll
    for (int i = 1; i < 4 * LP_LIVE; ++i) t = fmaxf(t, __uint_as_float(w[i]));
    return t;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 t = *reinterpret_cast<const T2*>(&w[0]);
#pragma unroll
    for (int i = 1; i < 4 * LP_LIVE; ++i) t = __hmax2(t, *reinterpret_cast<const T2*>(&w[i]));
    return fmaxf((float)t.x, (float)t.y);
  }
}

// (m, S, U) of a thread, in x's units and powers of two.
struct LpSum {
  float m = -INFINITY, s = 0.f, u = 0.f;
  // to a larger maximum
  __device__ __forceinline__ void raise(float to, float c) {
    const float d = m == -INFINITY ? 0.f : max_nan((m - to) * c, -200.f), f = ex2_approx(d);
    u = f * fmaf(d, s, u);
    s *= f;
    m = to;
  }
  // four or eight at a time, two in an instruction
  template <int N> __device__ __forceinline__ void add_all(const float (&x)[N], float off, float c) {
    float2 s2 = make_float2(s, 0.f), u2 = make_float2(u, 0.f);
    const float2 less = make_float2(-off, -off), by = make_float2(c, c), zero = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      float2 d = fma2(add2(make_float2(x[i], x[i + 1]), less), by, zero);
      d = make_float2(max_nan(d.x, -200.f), max_nan(d.y, -200.f));
      const float2 e = make_float2(ex2_approx(d.x), ex2_approx(d.y));
      s2 = add2(s2, e);
      u2 = fma2(e, d, u2);
    }
    s = s2.x + s2.y;
    u = u2.x + u2.y;
  }
  __device__ __forceinline__ void add(float x, float off, float c) {
    const float d = max_nan((x - off) * c, -200.f), e = ex2_approx(d);
    s += e;
    u = fmaf(e, d, u);
  }
  __device__ __forceinline__ void join(float m2, float s2, float u2, float c) {
    if (m2 > m) {
      raise(m2, c);
      s += s2;
      u += u2;
    } else if (m2 == -INFINITY) {  // nothing, or NaN
      s += s2;
      u += u2;
    } else {
      LpSum o;
      o.m = m2;
      o.s = s2;
      o.u = u2;
      o.raise(m, c);
      s += o.s;
      u += o.u;
    }
  }
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint64_t cluster_load64(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ float cluster_load32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) logprobs_kernel(const __grid_constant__ LogprobsArgs a) {
  constexpr int V = 16 / sizeof(T), WARPS = THREADS / 32;  // elements of a 16-byte piece
  __shared__ uint64_t s_top[LP_MAX_TOP];           // the block's alternatives, best first; 0: none
  __shared__ uint64_t s_cand[LP_CAND];
  __shared__ uint64_t s_all[LP_CLUSTER * LP_MAX_TOP];
  __shared__ float s_sum[3];                       // the block's (m, S, U)
  __shared__ float s_warp[3][WARPS];
  __shared__ uint32_t s_best[WARPS];
  __shared__ uint64_t s_key[WARPS];
  __shared__ int s_owner[THREADS];
  __shared__ int s_n[2];                           // candidates, owners
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank(), size = (int)cluster_size(), row = blockIdx.x / size;
  const T* x = (const T*)a.x + row * a.stride;
  const float c = a.inv_t * 1.4426950408889634f;
  // the row as single elements up to a 16-byte boundary, pieces, and single elements again
  const int head = min(a.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
  const int pieces = (a.vocab - head) / V, tail = a.vocab - head - pieces * V;
  const int share = (pieces + size - 1) / size, p0 = min(pieces, rank * share), p1 = min(pieces, p0 + share);
  const T* body = x + head;
  // one more element for some threads: of the head with the first block, of the tail with the last
  const int extra = rank == 0 && tid < head ? tid : rank == size - 1 && tid >= 32 && tid < 32 + tail ? a.vocab - tail + tid - 32 : -1;

  pdl_wait();
  pdl_trigger();
  // the first given token and its logit, by the block that writes it, ahead of the row
  int given = -1;
  float given_x = 0.f;
  if (rank == 0 && tid < a.n_given) {
    given = a.given[(int64_t)row * a.n_given + tid];
    if (given >= 0 && given < a.vocab) given_x = (float)x[given];
  }
  LpSum sum;  // its m is the largest value that the thread meets
  if (extra >= 0) {
    const float v = (float)x[extra];
    sum.m = v == v ? v : -INFINITY;
    sum.add(v, sum.m == -INFINITY ? 0.f : sum.m, c);
  }
  uint4 ahead[LP_LIVE];
  auto fetch = [&](int p) {  // beyond the end: the type's -inf
#pragma unroll
    for (int u = 0; u < LP_LIVE; ++u) {
      constexpr uint32_t none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
      ahead[u] = make_uint4(none, none, none, none);
      if (p + u * THREADS < p1) ahead[u] = __ldg(reinterpret_cast<const uint4*>(body + (int64_t)(p + u * THREADS) * V));
    }
  };
  fetch(p0 + tid);
  for (int p = p0 + tid; p < p1; p += THREADS * LP_LIVE) {
    uint4 raw[LP_LIVE];
#pragma unroll
    for (int u = 0; u < LP_LIVE; ++u) raw[u] = ahead[u];
    fetch(p + THREADS * LP_LIVE);
    // the maximum rises once for all of them: piece by piece some thread of a warp had a new one nearly every time
    const float t = lp_max<T>(raw);
    if (t > sum.m) sum.raise(t, c);
    const float off = sum.m == -INFINITY ? 0.f : sum.m;
#pragma unroll
    for (int u = 0; u < LP_LIVE; ++u) {
      float v[V];
      lp_unpack<T>(raw[u], v);
      sum.add_all(v, off, c);
    }
  }
  // (0 if the thread had nothing)
  const uint32_t mine = p0 + tid < p1 || extra >= 0 ? max(1u, lp_order(sum.m == 0.f ? 0.f : sum.m)) : 0u;
  const uint32_t warp_best = __reduce_max_sync(0xffffffffu, mine);
  // ---- the block's sums ----
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, sum.m, o), s2 = __shfl_xor_sync(0xffffffffu, sum.s, o),
                u2 = __shfl_xor_sync(0xffffffffu, sum.u, o);
    sum.join(m2, s2, u2, c);
  }
  if (lane == 0) {
    s_warp[0][warp] = sum.m;
    s_warp[1][warp] = sum.s;
    s_warp[2][warp] = sum.u;
    s_best[warp] = warp_best;
  }
  if (tid < LP_MAX_TOP) s_top[tid] = 0;
  if (tid < 2) s_n[tid] = 0;
  __syncthreads();
  if (warp == 0) {
    LpSum all;
    if (lane < WARPS) {
      all.m = s_warp[0][lane];
      all.s = s_warp[1][lane];
      all.u = s_warp[2][lane];
    }
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1)
      all.join(__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o),
               __shfl_xor_sync(0xffffffffu, all.u, o), c);
    if (lane == 0) {
      s_sum[0] = all.m;
      s_sum[1] = all.s;
      s_sum[2] = all.u;
    }
  }
  // ---- the block's alternatives ----
  if (a.top) {
    // at least `top` threads reach lo (or all that have anything), fewer reach hi; values of an eighth of the largest or more first
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) hi = max(hi, s_best[w]);
    const uint32_t near = hi > 1u << 24 ? hi - (1u << 24) : 0u;
    hi = hi == ~0u ? hi : hi + 1;
    int reach = __syncthreads_count(mine >= near);
    if (reach >= a.top) lo = near;
    else reach = THREADS, hi = near;
    while (hi - lo > 1 && reach > a.top + LP_MORE) {
      const uint32_t mid = lo + (hi - lo) / 2;
      const int n = __syncthreads_count(mine >= mid);
      if (n >= a.top) {
        lo = mid;
        reach = n;
      } else {
        hi = mid;
      }
    }
    const uint32_t tau = max(1u, lo);
    if (mine >= tau) s_owner[atomicAdd(&s_n[1], 1)] = tid;
    __syncthreads();
    auto consider = [&](float v, int i) {
      if (lp_order(v == 0.f ? 0.f : v) >= tau) {
        const int at = atomicAdd(&s_n[0], 1);
        if (at < LP_CAND) s_cand[at] = lp_key(v, i);
      }
    };
    if (extra >= 0) consider((float)x[extra], extra);
    const int each = (p1 - p0 + THREADS - 1) / THREADS, again = s_n[1] * each;  // pieces of a thread, to be read again
    for (int j = tid; j < again; j += THREADS) {
      const int o = j / each, p = p0 + s_owner[o] + (j - o * each) * THREADS;
      if (p >= p1) continue;
      float v[V];
      lp_load(body + (int64_t)p * V, v);
#pragma unroll
      for (int e = 0; e < V; ++e) consider(v[e], head + p * V + e);
    }
    __syncthreads();
    const int n = s_n[0];
    if (n <= LP_CAND) {
      for (int i = tid; i < n; i += THREADS) {  // as many as twice the threads
        const uint64_t key = s_cand[i];
        int ahead = 0;
        for (int j = 0; j < n; ++j) ahead += s_cand[j] > key;
        if (ahead < a.top) s_top[ahead] = key;
      }
    } else {
      // one by one: `next` is this thread's best that has not been taken
      uint64_t next = 0;
      if (extra >= 0) next = lp_key((float)x[extra], extra);
      for (int p = p0 + tid; p < p1; p += THREADS) {
        float v[V];
        lp_load(body + (int64_t)p * V, v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint64_t key = lp_key(v[e], head + p * V + e);
          if (key > next) next = key;
        }
      }
      for (int k = 0; k < a.top; ++k) {
        uint64_t most = next;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t y = __shfl_xor_sync(0xffffffffu, most, o);
          most = y > most ? y : most;
        }
        if (lane == 0) s_key[warp] = most;
        __syncthreads();
        uint64_t taken = 0;
        for (int w = 0; w < WARPS; ++w) taken = s_key[w] > taken ? s_key[w] : taken;
        if (taken == 0) break;
        if (tid == 0) s_top[k] = taken;
        const unsigned owns = __ballot_sync(0xffffffffu, next == taken);
        if (owns) {  // this warp looks for that thread's next one
          const int l = __ffs(owns) - 1, t = warp * 32 + l, ex = __shfl_sync(0xffffffffu, extra, l);
          uint64_t found = 0;
          if (lane == 0 && ex >= 0) {
            const uint64_t key = lp_key((float)x[ex], ex);
            if (key < taken) found = key;
          }
          for (int p = p0 + t + lane * THREADS; p < p1; p += 32 * THREADS) {
            float v[V];
            lp_load(body + (int64_t)p * V, v);
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const uint64_t key = lp_key(v[e], head + p * V + e);
              if (key < taken && key > found) found = key;
            }
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            const uint64_t y = __shfl_xor_sync(0xffffffffu, found, o);
            found = y > found ? y : found;
          }
          if (lane == l) next = found;
        }
        __syncthreads();
      }
    }
  }
  // ---- the row's, by the first block ----
  if (size > 1) {
    cluster_sync();
    if (rank == 0) {
      if (warp == 0) {
        LpSum all;
        if (lane < size) {
          all.m = cluster_load32(cluster_addr(&s_sum[0], lane));
          all.s = cluster_load32(cluster_addr(&s_sum[1], lane));
          all.u = cluster_load32(cluster_addr(&s_sum[2], lane));
        }
        for (int o = LP_CLUSTER / 2; o > 0; o >>= 1)
          all.join(__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o),
                   __shfl_xor_sync(0xffffffffu, all.u, o), c);
        __syncwarp();
        if (lane == 0) {
          s_warp[0][0] = all.m;
          s_warp[1][0] = all.s;
          s_warp[2][0] = all.u;
        }
      }
      for (int j = tid; j < size * a.top; j += THREADS) {
        const int r = j / a.top;
        s_all[j] = cluster_load64(cluster_addr(&s_top[j - r * a.top], r));
      }
    }
    cluster_sync();  // the others' shared memory has been read
    if (rank) return;
    if (tid < 3) s_sum[tid] = s_warp[tid][0];
    if (tid < a.top) s_top[tid] = 0;
    __syncthreads();
    for (int j = tid; j < size * a.top; j += THREADS) {
      const uint64_t key = s_all[j];
      if (!key) continue;
      const int r = j / a.top;
      int ahead = j - r * a.top;
      for (int o = 0; o < size; ++o) {
        if (o == r) continue;
        int from = 0, to = a.top;  // how many of that block's are larger
        while (from < to) {
          const int mid = (from + to) / 2;
          if (s_all[o * a.top + mid] > key) from = mid + 1;
          else to = mid;
        }
        ahead += from;
      }
      if (ahead < a.top) s_top[ahead] = key;
    }
  }
  __syncthreads();
  const float m = s_sum[0], s = s_sum[1], u = s_sum[2];
  const bool good = s > 0.f && s < INFINITY && fabsf(m) < INFINITY;  // else: no probability anywhere, an infinite one, or NaN
  constexpr float kLn2 = 0.6931471805599453f;
  const float nan = __int_as_float(0x7fffffff), log_s = kLn2 * log2f(s);
  if (tid == 0) {
    a.lse[row] = good ? fmaf(m, a.inv_t, log_s) : s == 0.f ? -INFINITY : nan;
    a.entropy[row] = good ? log_s - kLn2 * (u / s) : nan;
  }
  for (int j = tid; j < a.n_given; j += THREADS) {
    const int i = j == tid ? given : a.given[(int64_t)row * a.n_given + j];
    float y = 0.f;
    if (i >= a.vocab) {
      set_error(a.err, ERR_BAD_TOKEN);
      y = nan;
    } else if (i >= 0) {
      y = good ? fmaf((j == tid ? given_x : (float)x[i]) - m, a.inv_t, -log_s) : nan;
    }
    a.logprobs[(int64_t)row * a.n_given + j] = y;
  }
  for (int j = tid; j < a.top; j += THREADS) {
    const uint64_t key = s_top[j];
    a.top_logprobs[(int64_t)row * a.top + j] = good ? fmaf(lp_value(key) - m, a.inv_t, -log_s) : nan;
    a.top_ids[(int64_t)row * a.top + j] = good ? lp_token(key) : -1;
  }
}

}  // namespace hsg
