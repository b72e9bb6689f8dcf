// C entry points of the 8-bit cache and of token log-probabilities (hsg_append8, hsg_attention8, hsg_token_logprobs): argument
// checks and launches. Part of the one translation unit of the library.
#pragma once
#include "cache8_wide.cuh"
#include "draft_api.cuh"
#include "logprobs.cuh"

namespace {

int check_cache8(const hsg_cache8& c, int heads, int dim) {
  if (!c.k || !c.v || !c.k_scale || !c.v_scale) return fail(HSG_ERR_INVALID, "the cache's k, v or scales are NULL");
  if (c.pages < 1 || c.page_size < 8 || c.page_size % 8)
    return fail(HSG_ERR_INVALID, "a cache has at least one page of a multiple of 8 tokens, got %d of %d", c.pages, c.page_size);
  if (c.block < 8 || c.block % 8 || c.page_size % c.block)
    return fail(HSG_ERR_INVALID, "blocks must be a multiple of 8 tokens that divides a page's %d, got %d", c.page_size, c.block);
  if ((int64_t)c.pages * c.page_size > INT32_MAX)
    return fail(HSG_ERR_INVALID, "%d pages of %d tokens are beyond 32-bit slots", c.pages, c.page_size);
  if (!aligned16(c.k) || !aligned16(c.v) || c.page_stride % 16 || c.token_stride % 16 || c.head_stride % 16 ||
      c.page_stride < 0 || c.token_stride < 0 || c.head_stride < 0)
    return fail(HSG_ERR_INVALID, "cache rows must lie on 16-byte boundaries, at strides that are not negative");
  if ((reinterpret_cast<uintptr_t>(c.k_scale) | reinterpret_cast<uintptr_t>(c.v_scale)) & 3)
    return fail(HSG_ERR_INVALID, "scales must lie on 4-byte boundaries");
  if (c.pages > 1 && c.page_stride == 0) return fail(HSG_ERR_INVALID, "the cache's pages must differ");
  if (c.token_stride < dim || (heads > 1 && c.head_stride < dim))
    return fail(HSG_ERR_INVALID, "cache rows of %d bytes overlap (token stride %lld, head stride %lld)", dim,
                (long long)c.token_stride, (long long)c.head_stride);
  return HSG_OK;
}

Cache8 cache8(const hsg_cache8& c) {
  return Cache8{static_cast<uint8_t*>(c.k), static_cast<uint8_t*>(c.v), c.k_scale, c.v_scale, c.page_stride, c.token_stride,
                c.head_stride, c.pages, c.page_size, c.block, c.page_size / c.block, FastDiv::of(c.page_size), FastDiv::of(c.block)};
}

static_assert(A8_BLOCKS == SM_COUNT, "one piece an SM");
// Rows of a key head, on average over the requests, up to which warp-level products are taken. Narrow and wide, us: head dim 128, 40
// requests of 6,000 tokens, 8 query heads a key head: 16 rows 60 and 77, 24 rows 79 and 78, 48 rows 115 and 82; 5 requests of
// 50,000: 12 rows 87 and 92, 24 rows 138 and 93; head dim 256, 352 requests, window 512: 12 rows 104 and 145, 24 rows 151 and
// 148, 48 rows 252 and 162; head dim 64, 64 requests of 2,100: 12 rows 104 and 160, 24 rows 175 and 162.
// One kernel takes the whole call. A chunk of 2,000 tokens (179 us by itself) beside 256 requests of one token over 3,000 (324): 702, all
// wide; beside 1,000 (1,216): 1,959, all narrow. Callers do better with a call for each kind.
constexpr int A8_WIDE_ROWS = 20;

template <int D, typename T>
int launch_append8(const Append8Args& p, cudaStream_t st) {
  // entries a thread block: one where that leaves few blocks idle, else up to a block's, of which most continue a run
  const int per = p.count <= 16 * SM_COUNT ? 1 : std::min(32, p.cache.block), kv_blocks = (p.count + per - 1) / per;
  // warps that share a token's query heads: as few as leave four blocks an SM
  constexpr int WARPS = A8R_THREADS / 32, RPW = 256 / D;
  int split = 1;
  while (split < WARPS && (int64_t)(p.count + WARPS / split * RPW - 1) / (WARPS / split * RPW) < 4 * SM_COUNT) split *= 2;
  const int per_q = WARPS / split * RPW, q_blocks = p.hq ? (p.count + per_q - 1) / per_q : 0;
  const int smem = 4 * p.hkv * (int)sizeof(uint32_t);
  if (smem > 40 * 1024) return fail(HSG_ERR_INVALID, "too many key heads (%d)", p.hkv);
  CU(launch_k(append8_kernel<D, T>, dim3((unsigned)(kv_blocks + q_blocks)), dim3(A8R_THREADS), smem, st, true, p, kv_blocks, per, split));
  return HSG_OK;
}
template <typename T>
int launch_append8_dim(const Append8Args& p, int dim, cudaStream_t st) {
  return dim == 64 ? launch_append8<64, T>(p, st) : dim == 128 ? launch_append8<128, T>(p, st) : launch_append8<256, T>(p, st);
}

// Tensor map of a cache's codes: `keys` tokens of one page and head a box, blocks of 128 bytes a token (64 at head dim 64), all
// `cols` of them.
int make_codes_map(CUtensorMap* map, const uint8_t* base, const Cache8& c, int dim, int heads, int keys, int cols) {
  if (get_encoder() != HSG_OK) return HSG_ERR_CUDA;
  const int wide = std::min(dim, 128);
  const cuuint64_t dims[5] = {(cuuint64_t)wide, (cuuint64_t)c.page, (cuuint64_t)(dim / wide), (cuuint64_t)heads, (cuuint64_t)c.pages};
  // a stride whose dimension has one element is never used, but the encoder wants a valid one
  const cuuint64_t strides[4] = {(cuuint64_t)c.token_stride, 128, (cuuint64_t)(heads > 1 ? c.head_stride : 128),
                                 (cuuint64_t)(c.pages > 1 ? c.page_stride : 128)};
  const cuuint32_t box[5] = {(cuuint32_t)wide, (cuuint32_t)keys, (cuuint32_t)cols, 1, 1}, one[5] = {1, 1, 1, 1, 1};
  CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<uint8_t*>(base), dims, strides, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                        // (256 bytes at a time brought 337 MB for 195 where a row has 64 and the heads of a token lie together)
                        dim == 64 ? CU_TENSOR_MAP_L2_PROMOTION_NONE : CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(HSG_ERR_CUDA, "cuTensorMapEncodeTiled (codes) failed (%d)", (int)r);
  return HSG_OK;
}

// Workspace: partial results of either kernel, then what the wide one makes of the queries
size_t attn8_fixed_bytes(int dim) {
  const size_t one = a8_workspace_bytes(dim, a8_warps(dim, 1), 8), two = a8_workspace_bytes(dim, a8_warps(dim, 2), 16);
  return (std::max(std::max(one, two), a8_workspace_bytes(dim, 1, W8_ROWS)) + 127) / 128 * 128;
}

template <int D, int NR, typename T>
int launch_attn8_narrow(const Attn8Args& p, A8Split* splits, cudaStream_t st) {
  constexpr int PIECES = A8_BLOCKS * a8_warps(D, NR);
  float* partials = reinterpret_cast<float*>(splits + PIECES);
  int box = a8_slice(D);  // tokens of a TMA box: all of one page
  while (p.cache.page % box) box /= 2;
  const int cols = D == 256 && box == a8_slice(D) ? 2 : 1;
  CUtensorMap k, v;
  int rc;
  if ((rc = make_codes_map(&k, p.cache.k, p.cache, D, p.hkv, box, cols)) != HSG_OK ||
      (rc = make_codes_map(&v, p.cache.v, p.cache, D, p.hkv, box, cols)) != HSG_OK)
    return rc;
  CU(cudaFuncSetAttribute(attn8_kernel<D, NR, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, a8_smem(D, NR)));
  // as many thread blocks as can have a piece: items, and the slices that one can see at most
  const int64_t group = p.hq / p.hkv, reach = std::min<int64_t>((int64_t)p.width * p.cache.page, p.window ? (int64_t)p.window + p.sinks + p.max_new : INT64_MAX);
  const int64_t items = std::min<int64_t>(p.tokens * group, (p.tokens * group) / (8 * NR) + p.rows) * p.hkv;
  const int64_t pieces = std::max<int64_t>(1, std::min<int64_t>(PIECES, items * (reach / a8_slice(D) + 4 + A8_COST) / (A8_COST + 1) + 1));
  CU(launch_k(attn8_kernel<D, NR, T>, dim3((unsigned)std::min<int64_t>(A8_BLOCKS, pieces)), dim3(32 * a8_warps(D, NR)), a8_smem(D, NR), st, true, k, v, p, box,
              splits, partials));
  const int64_t most = std::min<int64_t>(8 * NR, p.max_new * group);  // rows of an item
  CU(launch_k(attn8_join_kernel<D, 8 * NR, T>, dim3((unsigned)pieces, (unsigned)((most + A8J_THREADS / 32 - 1) / (A8J_THREADS / 32))),
              dim3(A8J_THREADS), 0, st, true, p, (const A8Split*)splits, (const float*)partials));
  return HSG_OK;
}
template <int D, typename T>
int launch_attn8(const Attn8Args& p, void* workspace, cudaStream_t st) {
  A8Split* splits = static_cast<A8Split*>(workspace);
  // rows of a key head, as far as the host can tell: no request has more than max_new tokens, all have `tokens` together
  const int64_t rows = std::min<int64_t>(p.max_new, ((int64_t)p.tokens + p.rows - 1) / p.rows) * (p.hq / p.hkv);
  if (rows > A8_WIDE_ROWS) {
    float* partials = reinterpret_cast<float*>(splits + A8_BLOCKS);
    int box = w8_tile(D);  // tokens of a TMA box: all of one page
    while (p.cache.page % box) box /= 2;
    const int cols = D == 256 && box == w8_tile(D) ? 2 : 1, smem = w8_smem(D, std::is_same<T, __half>::value ? 3 : 2);
    CUtensorMap k, v;
    int rc;
    if ((rc = make_codes_map(&k, p.cache.k, p.cache, D, p.hkv, box, cols)) != HSG_OK ||
        (rc = make_codes_map(&v, p.cache.v, p.cache, D, p.hkv, box, cols)) != HSG_OK)
      return rc;
    // queries as sums of e4m3 numbers, behind the partial results
    constexpr int PARTS = std::is_same<T, __half>::value ? 3 : 2;
    const int64_t q_rows = (int64_t)p.tokens * p.hq;
    uint8_t* parts = static_cast<uint8_t*>(workspace) + attn8_fixed_bytes(D);
    float* q_scales = reinterpret_cast<float*>(parts + 3 * q_rows * D);
    CUtensorMap q;
    {
      const int wide = std::min(D, 128);
      const cuuint64_t dims[4] = {(cuuint64_t)wide, (cuuint64_t)q_rows, (cuuint64_t)(D / wide), PARTS};
      const cuuint64_t strides[3] = {(cuuint64_t)D, 128, (cuuint64_t)q_rows * D};
      const cuuint32_t boxes[4] = {(cuuint32_t)wide, W8_ROWS, (cuuint32_t)(D / wide), 1}, one[4] = {1, 1, 1, 1};
      CUresult r = g_encode(&q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, parts, dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
      if (r != CUDA_SUCCESS) return fail(HSG_ERR_CUDA, "cuTensorMapEncodeTiled (queries) failed (%d)", (int)r);
    }
    constexpr int ROWS_A_BLOCK = 8 * 256 / D;
    CU(launch_k(attn8_split_kernel<D, T>, dim3((unsigned)((q_rows + ROWS_A_BLOCK - 1) / ROWS_A_BLOCK)), dim3(256), 0, st, true, (const T*)p.q, p.q_ts,
                p.q_hs, p.tokens, p.hq, p.hq / p.hkv, parts, q_scales));
    CU(cudaFuncSetAttribute(attn8_wide_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    CU(launch_k(attn8_wide_kernel<D, T>, dim3(A8_BLOCKS), dim3(W8_THREADS), smem, st, true, q, k, v, p, box, (const float*)q_scales, splits, partials));
    CU(launch_k(attn8_join_kernel<D, W8_ROWS, T>, dim3(A8_BLOCKS, W8_ROWS / (A8J_THREADS / 32)), dim3(A8J_THREADS), 0, st, true, p,
                (const A8Split*)splits, (const float*)partials));
    return HSG_OK;
  }
  // blocks of 8 rows where none has more
  return (int64_t)p.max_new * (p.hq / p.hkv) <= 8 ? launch_attn8_narrow<D, 1, T>(p, splits, st) : launch_attn8_narrow<D, 2, T>(p, splits, st);
}
template <typename T>
int launch_attn8_dim(const Attn8Args& p, int dim, void* ws, cudaStream_t st) {
  return dim == 64 ? launch_attn8<64, T>(p, ws, st) : dim == 128 ? launch_attn8<128, T>(p, ws, st) : launch_attn8<256, T>(p, ws, st);
}

template <typename T, int THREADS>
int launch_logprobs_of(const LogprobsArgs& p, int size, cudaStream_t st) {
  CU(launch_cluster(logprobs_kernel<T, THREADS>, dim3((unsigned)(p.rows * size)), dim3(THREADS), size, 0, st, true, p));
  return HSG_OK;
}
template <typename T>
int launch_logprobs(const LogprobsArgs& p, cudaStream_t st) {
  // Rows that fill the device with four blocks an SM have 256 threads each, so that one row's selection overlaps others' reading;
  // fewer have 512, and as many blocks a row as two an SM leave room for, up to eight. 2,500 rows of 50,001 fp16: 71 us with 256
  // threads, 91 with 512; 352 of 248,320 bf16: 63 and 46 (51 with two blocks a row); one of 248,320 fp32: 12.1 with eight blocks of
  // 256, 10.7 of 512, 11.9 of 1,024 (sixteen of those: 13.7).
  if (p.rows >= 4 * SM_COUNT) return launch_logprobs_of<T, 256>(p, 1, st);
  int size = 1;
  while (size < LP_CLUSTER && (int64_t)p.rows * size * 2 <= 2 * SM_COUNT) size *= 2;
  return launch_logprobs_of<T, 512>(p, size, st);
}

}  // namespace

extern "C" int hsg_append8(const hsg_append8_args* a) {
  DRAFT_ARGS(a);
  if (a->count < 0 || a->rows < 0 || a->hkv < 1 || a->hq < 0)
    return fail(HSG_ERR_INVALID, "bad shape (count %d, rows %d, heads %d / %d)", a->count, a->rows, a->hq, a->hkv);
  if (a->count > INT32_MAX - 2 * A8R_WALK * A8R_THREADS) return fail(HSG_ERR_INVALID, "too many entries (%d)", a->count);
  if (!head_dim_ok(a->dim)) return fail(HSG_ERR_INVALID, "head_dim must be 64, 128 or 256, got %d", a->dim);
  if (a->rot < 0 || a->rot > a->dim || a->rot % 16)
    return fail(HSG_ERR_INVALID, "the rotated dims must be a multiple of 16 up to head_dim, got %d", a->rot);
  if (a->dtype != HSG_DT_F16 && a->dtype != HSG_DT_BF16) return fail(HSG_ERR_INVALID, "q, k and v must be fp16 or bf16");
  if (!(fabsf(a->rope_scale) < INFINITY)) return fail(HSG_ERR_INVALID, "rope_scale must be finite");
  if (a->count == 0) return HSG_OK;
  if (!a->slots || (a->rows && (!a->k || !a->v)) || (a->hq && (!a->q || !a->q_out)) || (a->rot && (!a->positions || !a->inv_freq)))
    return fail(HSG_ERR_INVALID, "NULL argument");
  if (a->hq && a->source) return fail(HSG_ERR_INVALID, "q goes with entries in order: source must be NULL");
  if (!aligned16(a->k) || !aligned16(a->v) || !rows16(a->k_token_stride, a->k_head_stride, 2) ||
      !rows16(a->v_token_stride, a->v_head_stride, 2) ||
      (a->hq && (!aligned16(a->q) || !aligned16(a->q_out) || !rows16(a->q_token_stride, a->q_head_stride, 2))))
    return fail(HSG_ERR_INVALID, "q, k and v rows must lie on 16-byte boundaries");
  int rc;
  if ((rc = check_cache8(a->cache, a->hkv, a->dim)) != HSG_OK) return rc;
  Append8Args p{a->q, a->k, a->v, a->q_token_stride, a->q_head_stride, a->k_token_stride, a->k_head_stride, a->v_token_stride,
                a->v_head_stride, a->source, a->slots, a->positions, a->inv_freq, a->count, a->rows, a->hq, a->hkv, a->rot,
                a->interleaved != 0, a->rope_scale, a->q_out, cache8(a->cache), a->err};
  cudaStream_t st = (cudaStream_t)a->stream;
  return a->dtype == HSG_DT_F16 ? launch_append8_dim<__half>(p, a->dim, st) : launch_append8_dim<__nv_bfloat16>(p, a->dim, st);
}

extern "C" size_t hsg_attention8_workspace(int head_dim, int tokens, int hq) {
  return head_dim_ok(head_dim) && tokens >= 0 && hq > 0 ? attn8_fixed_bytes(head_dim) + (size_t)tokens * hq * (3 * head_dim + 4) : 0;
}

extern "C" int hsg_attention8(const hsg_attention8_args* a) {
  DRAFT_ARGS(a);
  if (a->rows < 0 || a->tokens < 0 || a->hq < 1 || a->hkv < 1 || a->hq % a->hkv)
    return fail(HSG_ERR_INVALID, "bad shape (rows %d, tokens %d, heads %d / %d)", a->rows, a->tokens, a->hq, a->hkv);
  if (a->hq / a->hkv > DA_ROWS)
    return fail(HSG_ERR_INVALID, "at most %d query heads a key head, got %d", DA_ROWS, a->hq / a->hkv);
  if (!head_dim_ok(a->dim)) return fail(HSG_ERR_INVALID, "head_dim must be 64, 128 or 256, got %d", a->dim);
  if (a->dtype != HSG_DT_F16 && a->dtype != HSG_DT_BF16) return fail(HSG_ERR_INVALID, "dtype must be fp16 or bf16");
  if (a->max_new < 1 || a->max_new > HSG_MAX_NEW)
    return fail(HSG_ERR_INVALID, "max_new must be in [1, %d], got %d", HSG_MAX_NEW, a->max_new);
  if (a->mask && (int64_t)a->words * 32 < a->max_new)
    return fail(HSG_ERR_INVALID, "%d mask words hold fewer than max_new = %d bits", a->words, a->max_new);
  if (!(a->scale > 0.f) || !(a->scale < INFINITY)) return fail(HSG_ERR_INVALID, "scale must be positive");
  if (a->window < 0 || a->sinks < 0) return fail(HSG_ERR_INVALID, "window and sinks must not be negative, got %d and %d", a->window, a->sinks);
  if (a->rows == 0 || a->tokens == 0) return HSG_OK;
  if (!a->q || !a->table || !a->lens || !a->cu || !a->out) return fail(HSG_ERR_INVALID, "NULL argument");
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < (int64_t)hsg_attention8_workspace(a->dim, a->tokens, a->hq))
    return fail(HSG_ERR_INVALID, "the workspace must have %zu bytes on a 16-byte boundary",
                hsg_attention8_workspace(a->dim, a->tokens, a->hq));
  if (a->width < 1 || a->table_stride < a->width)
    return fail(HSG_ERR_INVALID, "bad table shape (width %d, stride %lld)", a->width, (long long)a->table_stride);
  int rc;
  if ((rc = check_cache8(a->cache, a->hkv, a->dim)) != HSG_OK) return rc;
  if ((int64_t)a->width * a->cache.page_size > INT32_MAX)
    return fail(HSG_ERR_INVALID, "%d pages of %d tokens are beyond 32-bit positions", a->width, a->cache.page_size);
  if (!aligned16(a->q) || !aligned16(a->out) || !rows16(a->q_token_stride, a->q_head_stride, 2))
    return fail(HSG_ERR_INVALID, "q rows must lie on 16-byte boundaries");
  if ((int64_t)a->tokens * a->hq > INT32_MAX || (int64_t)a->max_new * (a->hq / a->hkv) > INT32_MAX / 2) return fail(HSG_ERR_INVALID, "too many rows a key head");
  Attn8Args p{a->q, a->q_token_stride, a->q_head_stride, cache8(a->cache), a->table, a->table_stride, a->lens, a->cu,
              a->positions, a->mask, a->rows, a->width, a->tokens, a->words, a->max_new, a->hq, a->hkv, a->window, a->sinks,
              a->scale, a->out, a->lse, a->err};
  cudaStream_t st = (cudaStream_t)a->stream;
  return a->dtype == HSG_DT_F16 ? launch_attn8_dim<__half>(p, a->dim, a->workspace, st)
                                : launch_attn8_dim<__nv_bfloat16>(p, a->dim, a->workspace, st);
}

extern "C" int hsg_token_logprobs(const hsg_logprobs_args* a) {
  DRAFT_ARGS(a);
  if (a->rows < 0 || a->vocab < 1 || a->n_given < 0)
    return fail(HSG_ERR_INVALID, "bad shape (rows %d, vocabulary %d, given %d)", a->rows, a->vocab, a->n_given);
  if (a->dtype < HSG_DT_F32 || a->dtype > HSG_DT_BF16) return fail(HSG_ERR_INVALID, "logits must be fp32, fp16 or bf16");
  if (a->top < 0 || a->top > HSG_MAX_TOP || a->top > a->vocab)
    return fail(HSG_ERR_INVALID, "top must be in [0, %d] and at most the vocabulary, got %d", HSG_MAX_TOP, a->top);
  if (!(a->temperature >= 1e-4f) || !(a->temperature <= 1e4f))
    return fail(HSG_ERR_INVALID, "temperature must be in [1e-4, 1e4], got %g", a->temperature);
  if (a->rows == 0) return HSG_OK;
  if (!a->logits || !a->entropy || !a->lse || (a->n_given && (!a->given || !a->logprobs)) || (a->top && (!a->top_logprobs || !a->top_ids)))
    return fail(HSG_ERR_INVALID, "NULL argument");
  if (a->rows > 1 && a->row_stride < 0) return fail(HSG_ERR_INVALID, "rows of logits must not descend");
  if (reinterpret_cast<uintptr_t>(a->logits) % (a->dtype == HSG_DT_F32 ? 4 : 2))
    return fail(HSG_ERR_INVALID, "logits must lie on an element's boundary");
  if (a->rows > INT32_MAX / LP_CLUSTER) return fail(HSG_ERR_INVALID, "too many rows (%d)", a->rows);
  LogprobsArgs p{a->logits, a->row_stride, a->given, a->rows, a->vocab, a->n_given, a->top, 1.0f / a->temperature, a->logprobs,
                 a->entropy, a->lse, a->top_logprobs, a->top_ids, a->err};
  cudaStream_t st = (cudaStream_t)a->stream;
  return a->dtype == HSG_DT_F32 ? launch_logprobs<float>(p, st)
                                : a->dtype == HSG_DT_F16 ? launch_logprobs<__half>(p, st) : launch_logprobs<__nv_bfloat16>(p, st);
}
