// C entry points of draft scoring (hsg_advance_tables, hsg_plan_tree, hsg_norm_rope, hsg_tree_attention,
// hsg_store_rows): argument checks and launches. Part of the one translation unit of the library.
#pragma once
#include "draft_attn.cuh"
#include "draft_rows.cuh"
#include "draft_tables.cuh"

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// `bytes`-wide elements: strides that keep every row on a 16-byte boundary
bool rows16(int64_t a, int64_t b, int bytes) { return (a * bytes) % 16 == 0 && (b * bytes) % 16 == 0; }
bool head_dim_ok(int d) { return d == 64 || d == 128 || d == 256; }

int check_cache(const hsg_page_cache& c, int heads, int dim) {
  if (!c.k || !c.v) return fail(HSG_ERR_INVALID, "the cache's k or v is NULL");
  if (c.pages < 1 || c.page_size < 8 || c.page_size % 8)
    return fail(HSG_ERR_INVALID, "a cache has at least one page of a multiple of 8 tokens, got %d of %d", c.pages,
                c.page_size);
  if ((int64_t)c.pages * c.page_size > INT32_MAX)
    return fail(HSG_ERR_INVALID, "%d pages of %d tokens are beyond 32-bit slots", c.pages, c.page_size);
  if (!aligned16(c.k) || !aligned16(c.v) || c.page_stride % 8 || c.token_stride % 8 || c.head_stride % 8 ||
      c.page_stride < 0 || c.token_stride < 0 || c.head_stride < 0)
    return fail(HSG_ERR_INVALID, "cache rows must lie on 16-byte boundaries, at strides that are not negative");
  if (c.pages > 1 && c.page_stride == 0) return fail(HSG_ERR_INVALID, "the cache's pages must differ");
  if ((c.page_size > 1 && c.token_stride < dim) || (heads > 1 && c.head_stride < dim))
    return fail(HSG_ERR_INVALID, "cache rows of %d elements overlap (token stride %lld, head stride %lld)", dim,
                (long long)c.token_stride, (long long)c.head_stride);
  return HSG_OK;
}

PageCache page_cache(const hsg_page_cache& c) {
  return PageCache{c.k, c.v, c.page_stride, c.token_stride, c.head_stride, c.pages, c.page_size};
}

static_assert(DA_PIECES == SM_COUNT, "one piece an SM");
static_assert(DT_MAX_ROWS == HSG_MAX_TABLE_ROWS, "the header states the kernel's limit");

#define DRAFT_ARGS(a)                                                                                  \
  do {                                                                                                 \
    if (!(a)) return fail(HSG_ERR_INVALID, "args is NULL");                                            \
    if ((a)->size != (int64_t)sizeof(*(a)))                                                            \
      return fail(HSG_ERR_INVALID, "args has %lld bytes, this library expects %lld", (long long)(a)->size, \
                  (long long)sizeof(*(a)));                                                            \
  } while (0)

template <int D, typename TI, typename TO>
int launch_norm(const DraftNormArgs& n, cudaStream_t st) {
  // tokens a block: one unit of every head, as long as that leaves four blocks an SM
  const int per = std::max(1, std::min(DN_LIVE, n.tokens / (4 * SM_COUNT)));
  draft_norm_kernel<D, TI, TO><<<(n.tokens + per - 1) / per, DN_THREADS, per * (n.rot / 2) * sizeof(float2), st>>>(n, per);
  CU(cudaGetLastError());
  return HSG_OK;
}
template <int D, typename TI>
int launch_norm_out(const DraftNormArgs& n, int out, cudaStream_t st) {
  return out == HSG_DT_F16 ? launch_norm<D, TI, __half>(n, st) : launch_norm<D, TI, __nv_bfloat16>(n, st);
}
template <int D>
int launch_norm_in(const DraftNormArgs& n, int in, int out, cudaStream_t st) {
  if (in == HSG_DT_F32) return launch_norm_out<D, float>(n, out, st);
  return in == HSG_DT_F16 ? launch_norm_out<D, __half>(n, out, st) : launch_norm_out<D, __nv_bfloat16>(n, out, st);
}

// Tensor map of 16-bit rows of `dim` elements, read 64 dims at a time in 128-byte swizzle: dimension 0 is 64 dims, the
// others as given (element strides). A stride whose dimension has one element is never used, but the encoder wants a
// valid one.
int make_rows_map(CUtensorMap* map, const void* base, CUtensorMapDataType type, int rank, const int64_t* sizes,
                  const int64_t* strides, const int* boxes) {
  if (get_encoder() != HSG_OK) return HSG_ERR_CUDA;
  cuuint64_t dims[5], bytes[4];
  cuuint32_t box[5], one[5];
  for (int i = 0; i < rank; ++i) {
    dims[i] = (cuuint64_t)sizes[i];
    box[i] = (cuuint32_t)boxes[i];
    one[i] = 1;
    if (i) bytes[i - 1] = (cuuint64_t)(sizes[i] > 1 ? strides[i] : 64) * 2;
  }
  CUresult r = g_encode(map, type, rank, const_cast<void*>(base), dims, bytes, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(HSG_ERR_CUDA, "cuTensorMapEncodeTiled (%d-d rows) failed (%d)", rank, (int)r);
  return HSG_OK;
}

// As many whole drafted tokens as fit 128 rows; Q double-buffered up to 64 KB, the rest of shared memory for K and V.
// Boxes of the cache: 8 tokens with page, head, 64-dim block, token and dim as the five dimensions that a map may have.
// Several 8-token groups at a constant stride need a dimension of their own, which the heads give up where they continue
// another: the 64-dim blocks, if a token's heads are contiguous (fold 1), or the groups, if a head's rows begin a whole
// number of groups after the last head's (fold 2). Then a box takes up to 8 KB, as far as the page size divides.
DaPlan plan_draft_attn(int max_tree, int group, int dim, int heads, const PageCache& c) {
  DaPlan p;
  const int64_t eight = 8 * c.token_stride;
  p.groups = 1;
  while (p.groups * 2 * 16 * dim <= DA_BOX_BYTES && 16 * p.groups <= da_tile(dim) && c.page % (16 * p.groups) == 0) p.groups *= 2;
  p.fold = p.groups == 1 ? 0 : heads == 1 || c.head_stride == dim ? 1 : c.head_stride % eight == 0 ? 2 : 0;
  if (p.fold == 0) p.groups = 1;
  p.head_step = p.fold == 1 ? dim / 64 : p.fold == 2 ? (int)(c.head_stride / eight) : 0;
  p.block = std::min(max_tree, DA_ROWS / group);
  p.q_rows = (p.block * group + 7) / 8 * 8;
  const int q = p.q_rows * dim * 2;
  p.q_bufs = q <= 32768 ? 2 : 1;
  const int bufs = std::min(2 * DA_MAX_BUFS, (DA_SMEM_LIMIT - 1024 - da_extra(dim, p.block) - p.q_bufs * q) / da_buffer_bytes(dim));
  p.k_bufs = bufs / 2;
  p.v_bufs = bufs - p.k_bufs;
  return p;
}

template <int D, typename T>
int launch_draft_attn(const DraftAttnArgs& d, void* workspace, cudaStream_t st) {
  constexpr CUtensorMapDataType type =
      std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  constexpr int NC = D / 64;
  const int group = d.hq / d.hkv;
  const PageCache& c = d.cache;
  const DaPlan p = plan_draft_attn(d.max_tree, group, D, d.hkv, c);
  CUtensorMap q, ck, cv, k, v;
  int rc;
  {
    const int64_t sizes[3] = {D, d.hq, d.tokens}, strides[3] = {1, d.q_hs, d.q_ts};
    const int boxes[3] = {64, group, p.block};
    if ((rc = make_rows_map(&q, d.q, type, 3, sizes, strides, boxes)) != HSG_OK) return rc;
  }
  {
    const int64_t own[5] = {64, c.page, NC, d.hkv, c.pages}, own_strides[5] = {1, c.token_stride, 64, c.head_stride, c.page_stride};
    const int64_t folded[5] = {64, 8, p.fold == 1 ? NC * d.hkv : NC,
                               c.page / 8 + (p.fold == 2 ? (int64_t)(d.hkv - 1) * p.head_step : 0), c.pages};
    const int64_t folded_strides[5] = {1, c.token_stride, 64, 8 * c.token_stride, c.page_stride};
    const int64_t *sizes = p.fold ? folded : own, *strides = p.fold ? folded_strides : own_strides;
    const int boxes[5] = {64, 8, NC, p.fold ? p.groups : 1, 1};
    if ((rc = make_rows_map(&ck, c.k, type, 5, sizes, strides, boxes)) != HSG_OK ||
        (rc = make_rows_map(&cv, c.v, type, 5, sizes, strides, boxes)) != HSG_OK)
      return rc;
  }
  {
    const int64_t sizes[4] = {64, d.tokens, NC, d.hkv};
    const int64_t ks[4] = {1, d.k_ts, 64, d.k_hs}, vs[4] = {1, d.v_ts, 64, d.v_hs};
    const int boxes[4] = {64, 8, NC, 1};
    if ((rc = make_rows_map(&k, d.k, type, 4, sizes, ks, boxes)) != HSG_OK ||
        (rc = make_rows_map(&v, d.v, type, 4, sizes, vs, boxes)) != HSG_OK)
      return rc;
  }
  DaSplit* splits = static_cast<DaSplit*>(workspace);
  float* partials = reinterpret_cast<float*>(splits + DA_PIECES);
  CU(cudaFuncSetAttribute(draft_attn_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, DA_SMEM_LIMIT));
  CU(launch_k(draft_attn_kernel<D, T>, dim3(DA_PIECES), dim3(DA_THREADS), da_smem_bytes(p, D), st, true, q, ck, cv, k, v, d,
              p, splits, partials));
  const int rows = p.q_rows;
  CU(launch_k(draft_join_kernel<D, T>, dim3(DA_PIECES, (rows + DJ_THREADS / 32 - 1) / (DJ_THREADS / 32)),
              dim3(DJ_THREADS), 0, st, true, d, p.block, (const DaSplit*)splits, (const float*)partials));
  return HSG_OK;
}
template <typename T>
int launch_draft_attn_dim(const DraftAttnArgs& d, int dim, void* ws, cudaStream_t st) {
  return dim == 64 ? launch_draft_attn<64, T>(d, ws, st)
                   : dim == 128 ? launch_draft_attn<128, T>(d, ws, st) : launch_draft_attn<256, T>(d, ws, st);
}

}  // namespace

extern "C" int hsg_advance_tables(const hsg_tables_args* a) {
  DRAFT_ARGS(a);
  if (a->rows < 0 || a->rows > DT_MAX_ROWS)
    return fail(HSG_ERR_INVALID, "rows must be in [0, %d], got %d", DT_MAX_ROWS, a->rows);
  if (a->width < 1 || a->ring_size < 1 || a->page_size < 1 || a->capacity < 0 || a->table_stride < a->width)
    return fail(HSG_ERR_INVALID, "bad table shape (width %d, stride %lld, ring %d, page %d, capacity %d)", a->width,
                (long long)a->table_stride, a->ring_size, a->page_size, a->capacity);
  if ((int64_t)a->width * a->page_size > INT32_MAX || (int64_t)a->ring_size * a->page_size > INT32_MAX)
    return fail(HSG_ERR_INVALID, "%d pages of %d tokens are beyond 32-bit positions or slots",
                std::max(a->width, a->ring_size), a->page_size);
  if (!a->ring || !a->counters || !a->counters_out || !a->cu ||
      (a->rows && (!a->lens || !a->delta || !a->table || !a->lens_out)) ||
      (a->capacity && (!a->slots || !a->token_rows || !a->positions)))
    return fail(HSG_ERR_INVALID, "NULL argument");
  if ((a->rows && a->lens_out == a->lens) || a->counters_out == a->counters)
    return fail(HSG_ERR_INVALID, "lens_out and counters_out must not be the inputs");
  DraftTablesArgs t{a->lens, a->delta, a->table, a->table_stride, a->ring, a->counters, a->rows, a->width,
                    a->ring_size, FastDiv::of(a->page_size), (uint32_t)((1ll << 31) / a->page_size), a->lens_out,
                    a->counters_out, a->cu, a->slots, a->token_rows, a->positions, a->capacity, a->err};
  const int smem = a->rows * DT_ROW_BYTES;
  if (smem > 47 * 1024)
    CU(cudaFuncSetAttribute(draft_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DT_MAX_ROWS * DT_ROW_BYTES));
  // a block for 1,024 listed tokens or 2,048 table entries, any of which may change hands, at most two an SM
  const int64_t share = std::max<int64_t>(a->capacity / (4 * DT_THREADS), (int64_t)a->rows * a->width / (8 * DT_THREADS));
  const int blocks = (int)std::max<int64_t>(1, std::min<int64_t>(2 * SM_COUNT, share));
  draft_tables_kernel<<<blocks, DT_THREADS, smem, (cudaStream_t)a->stream>>>(t);
  CU(cudaGetLastError());
  return HSG_OK;
}

extern "C" int hsg_plan_tree(const hsg_tree_args* a) {
  DRAFT_ARGS(a);
  if (a->rows < 0 || a->tokens < 0 || a->words < 1 || a->words > HSG_MAX_TREE / 32)
    return fail(HSG_ERR_INVALID, "bad tree shape (rows %d, tokens %d, words %d)", a->rows, a->tokens, a->words);
  if (a->rows == 0 || a->tokens == 0) return HSG_OK;
  if (!a->parents || !a->cu || !a->lens || !a->positions || !a->mask) return fail(HSG_ERR_INVALID, "NULL argument");
  DraftTreeArgs t{a->parents, a->cu, a->lens, a->rows, a->tokens, a->words, a->positions, a->mask, a->err};
  draft_tree_kernel<<<a->rows, DTREE_THREADS, 0, (cudaStream_t)a->stream>>>(t);
  CU(cudaGetLastError());
  return HSG_OK;
}

extern "C" int hsg_norm_rope(const hsg_norm_rope_args* a) {
  DRAFT_ARGS(a);
  if (a->tokens < 0 || a->hq < 1 || a->hkv < 1) return fail(HSG_ERR_INVALID, "bad shape (tokens %d, heads %d / %d)",
                                                            a->tokens, a->hq, a->hkv);
  if (!head_dim_ok(a->dim)) return fail(HSG_ERR_INVALID, "head_dim must be 64, 128 or 256, got %d", a->dim);
  if (a->rot < 16 || a->rot > a->dim || a->rot % 16)
    return fail(HSG_ERR_INVALID, "the rotated dims must be a multiple of 16 up to head_dim, got %d", a->rot);
  if (a->in_dtype < HSG_DT_F32 || a->in_dtype > HSG_DT_BF16 || (a->out_dtype != HSG_DT_F16 && a->out_dtype != HSG_DT_BF16))
    return fail(HSG_ERR_INVALID, "inputs are fp32, fp16 or bf16, outputs fp16 or bf16");
  if (a->tokens == 0) return HSG_OK;
  if (!a->q || !a->k || !a->v || !a->q_weight || !a->k_weight || !a->inv_freq || !a->positions || !a->q_out)
    return fail(HSG_ERR_INVALID, "NULL argument");
  if (!a->slots && (!a->k_out || !a->v_out)) return fail(HSG_ERR_INVALID, "k_out and v_out, or slots, are needed");
  const int bytes = a->in_dtype == HSG_DT_F32 ? 4 : 2;
  if (!aligned16(a->q_weight) || !aligned16(a->k_weight))
    return fail(HSG_ERR_INVALID, "q_weight and k_weight must lie on 16-byte boundaries");
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->q_out) ||
      !rows16(a->q_token_stride, a->q_head_stride, bytes) || !rows16(a->k_token_stride, a->k_head_stride, bytes) ||
      !rows16(a->v_token_stride, a->v_head_stride, bytes) || (!a->slots && (!aligned16(a->k_out) || !aligned16(a->v_out))))
    return fail(HSG_ERR_INVALID, "q, k and v rows must lie on 16-byte boundaries");
  int rc;
  DraftNormArgs n{a->q, a->k, a->v, a->q_token_stride, a->q_head_stride, a->k_token_stride, a->k_head_stride,
                  a->v_token_stride, a->v_head_stride, a->q_weight, a->k_weight, a->inv_freq, a->positions, a->tokens,
                  a->hq, a->hkv, a->rot, a->eps, a->q_out, a->k_out, a->v_out, a->slots, PageCache{}, a->err};
  if (a->slots) {
    if ((rc = check_cache(a->cache, a->hkv, a->dim)) != HSG_OK) return rc;
    n.cache = page_cache(a->cache);
  }
  cudaStream_t st = (cudaStream_t)a->stream;
  if (a->dim == 64) return launch_norm_in<64>(n, a->in_dtype, a->out_dtype, st);
  if (a->dim == 128) return launch_norm_in<128>(n, a->in_dtype, a->out_dtype, st);
  return launch_norm_in<256>(n, a->in_dtype, a->out_dtype, st);
}

extern "C" size_t hsg_tree_attention_workspace(int head_dim) {
  return head_dim_ok(head_dim) ? da_workspace_bytes(head_dim) : 0;
}

extern "C" int hsg_tree_attention(const hsg_tree_attention_args* a) {
  DRAFT_ARGS(a);
  if (a->rows < 0 || a->tokens < 0 || a->hq < 1 || a->hkv < 1 || a->hq % a->hkv)
    return fail(HSG_ERR_INVALID, "bad shape (rows %d, tokens %d, heads %d / %d)", a->rows, a->tokens, a->hq, a->hkv);
  if (a->hq / a->hkv > DA_ROWS)
    return fail(HSG_ERR_INVALID, "at most %d query heads a key head, got %d", DA_ROWS, a->hq / a->hkv);
  if (!head_dim_ok(a->dim)) return fail(HSG_ERR_INVALID, "head_dim must be 64, 128 or 256, got %d", a->dim);
  if (a->dtype != HSG_DT_F16 && a->dtype != HSG_DT_BF16) return fail(HSG_ERR_INVALID, "dtype must be fp16 or bf16");
  if (a->max_tree < 1 || a->max_tree > HSG_MAX_TREE)
    return fail(HSG_ERR_INVALID, "max_tree must be in [1, %d], got %d", HSG_MAX_TREE, a->max_tree);
  if (a->mask && (int64_t)a->words * 32 < a->max_tree)
    return fail(HSG_ERR_INVALID, "%d mask words hold fewer than max_tree = %d bits", a->words, a->max_tree);
  if (!(a->scale > 0.f) || !(a->scale < INFINITY)) return fail(HSG_ERR_INVALID, "scale must be positive");
  if (a->window < 0) return fail(HSG_ERR_INVALID, "window must not be negative, got %d", a->window);
  if (a->rows == 0 || a->tokens == 0) return HSG_OK;
  if (!a->q || !a->k || !a->v || !a->table || !a->lens || !a->cu || !a->out) return fail(HSG_ERR_INVALID, "NULL argument");
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < (int64_t)hsg_tree_attention_workspace(a->dim))
    return fail(HSG_ERR_INVALID, "the workspace must have %zu bytes on a 16-byte boundary",
                hsg_tree_attention_workspace(a->dim));
  if (a->width < 1 || a->table_stride < a->width)
    return fail(HSG_ERR_INVALID, "bad table shape (width %d, stride %lld)", a->width, (long long)a->table_stride);
  int rc;
  if ((rc = check_cache(a->cache, a->hkv, a->dim)) != HSG_OK) return rc;
  if ((int64_t)a->width * a->cache.page_size > INT32_MAX)
    return fail(HSG_ERR_INVALID, "%d pages of %d tokens are beyond 32-bit positions", a->width, a->cache.page_size);
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out) ||
      !rows16(a->q_token_stride, a->q_head_stride, 2) || !rows16(a->k_token_stride, a->k_head_stride, 2) ||
      !rows16(a->v_token_stride, a->v_head_stride, 2))
    return fail(HSG_ERR_INVALID, "q, k and v rows must lie on 16-byte boundaries");
  // tiles are read through tensor maps, which know no stride of 0 (a broadcast dimension)
  if ((a->tokens > 1 && (a->q_token_stride <= 0 || a->k_token_stride <= 0 || a->v_token_stride <= 0)) ||
      (a->hq > 1 && a->q_head_stride <= 0) || (a->hkv > 1 && (a->k_head_stride <= 0 || a->v_head_stride <= 0)))
    return fail(HSG_ERR_INVALID, "q, k and v must have positive strides: a broadcast dimension has to be written out");
  DraftAttnArgs d{a->q, a->k, a->v, a->q_token_stride, a->q_head_stride, a->k_token_stride, a->k_head_stride,
                  a->v_token_stride, a->v_head_stride, page_cache(a->cache), a->table, a->table_stride, a->lens, a->cu,
                  a->positions, a->mask, a->rows, a->width, a->tokens, a->words, a->max_tree, a->hq, a->hkv, a->window,
                  a->scale, a->out, a->lse, a->err};
  cudaStream_t st = (cudaStream_t)a->stream;
  return a->dtype == HSG_DT_F16 ? launch_draft_attn_dim<__half>(d, a->dim, a->workspace, st)
                                : launch_draft_attn_dim<__nv_bfloat16>(d, a->dim, a->workspace, st);
}

extern "C" int hsg_store_rows(const hsg_store_args* a) {
  DRAFT_ARGS(a);
  if (a->count < 0 || a->rows < 0 || a->heads < 1) return fail(HSG_ERR_INVALID, "bad shape (count %d, rows %d, heads %d)",
                                                               a->count, a->rows, a->heads);
  if (!head_dim_ok(a->dim)) return fail(HSG_ERR_INVALID, "head_dim must be 64, 128 or 256, got %d", a->dim);
  if (a->count == 0) return HSG_OK;
  if (!a->k || !a->v || !a->slots) return fail(HSG_ERR_INVALID, "NULL argument");
  if (!aligned16(a->k) || !aligned16(a->v) || !rows16(a->k_token_stride, a->k_head_stride, 2) ||
      !rows16(a->v_token_stride, a->v_head_stride, 2))
    return fail(HSG_ERR_INVALID, "k and v rows must lie on 16-byte boundaries");
  int rc;
  if ((rc = check_cache(a->cache, a->heads, a->dim)) != HSG_OK) return rc;
  DraftStoreArgs s{a->k, a->v, a->k_token_stride, a->k_head_stride, a->v_token_stride, a->v_head_stride, a->source,
                   a->slots, a->count, a->rows, a->heads, page_cache(a->cache), a->err};
  const int blocks = (a->count + DS_THREADS / 32 - 1) / (DS_THREADS / 32);
  cudaStream_t st = (cudaStream_t)a->stream;
  if (a->dim == 64) draft_store_kernel<64><<<blocks, DS_THREADS, 0, st>>>(s);
  else if (a->dim == 128) draft_store_kernel<128><<<blocks, DS_THREADS, 0, st>>>(s);
  else draft_store_kernel<256><<<blocks, DS_THREADS, 0, st>>>(s);
  CU(cudaGetLastError());
  return HSG_OK;
}

extern "C" const char* hsg_device_error_text(int code) { return code ? device_error_text(code) : "no error"; }
