"""Draft scoring: trees of drafted tokens attended over a paged cache before any of them is accepted.

A host model that drafts several continuations of a conversation has all of them scored in one pass. Per tick and
attention layer (requests b, drafted tokens in request order, ``cu`` [rows + 1] their offsets):

    positions, mask = plan_tree(parents, cu, lens, max_tree)             # once a tick
    q, k, v = norm_rope(q, k, v, qw, kw, inv_freq, positions, eps, torch.float16)
    out, lse = tree_attention(q, k, v, k_cache, v_cache, table, lens, cu, scale, max_tree, mask, positions, window)

and once a branch is accepted:

    t = advance_tables(lens, delta, table, ring, counters, page_size, capacity)    # once a tick
    store_rows(k, v, k_cache, v_cache, t.slots, source)                            # every layer

``DraftCache`` holds the pages, tables and counters of several layers and calls the last two. Every function queues
work on torch's current stream of its tensors' device and waits for nothing; outputs are new tensors unless they are
said to change in place. Arguments of a wrong shape, type, device or alignment raise ``ValueError`` before anything
is queued. Values on the device are checked by the kernels, which skip an index outside its range and record the
reason in ``err`` (an int32 tensor of one element, 0 at first; see ``raise_device_error``).

The C entry points are hsg_plan_tree, hsg_norm_rope, hsg_tree_attention, hsg_advance_tables and hsg_store_rows of
include/hsg.h. The reference has no counterpart: its ticks are chains and its caches 512-token rings.
"""
from __future__ import annotations

from collections import namedtuple
from struct import Struct

import torch

from . import _lib
from ._lib import check

MAX_TREE = 1024        # drafted tokens of one request
MAX_TABLE_ROWS = 4096  # requests of one advance_tables call
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

# The argument structs of include/hsg.h (native alignment; "0q" pads the end as the C compiler does). Packed in one
# call: a ctypes.Structure with as many fields takes several times as long to fill.
_CACHE = "PPqqqii"
_TABLES = Struct("@qPPPqPPPPPPPPPPiiiii0q")
_TREE = Struct("@qPPPPPPPiii0q")
_NORM = Struct("@qPPPqqqqqqPPPPPPPP" + _CACHE + "PPiiiiiiif0q")
_ATTENTION = Struct("@qPPPqqqqqq" + _CACHE + "PqPPPPPPPqPPiiiiiiiiiif0q")
_STORE = Struct("@qPPqqqqPP" + _CACHE + "PPiiii0q")

Tables = namedtuple("Tables", "lens counters cu slots rows positions")


def _tensor(name, t, ndim, dtype, device):
    """``t`` is a CUDA tensor of these dimensions and this type on ``device``, its last dimension contiguous."""
    if not isinstance(t, torch.Tensor) or t.dim() != ndim or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be a {ndim}-d {dtype} tensor on {device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    return t


def _vector(name, t, dtype, device, size=None):
    _tensor(name, t, 1, dtype, device)
    if size is not None and t.shape[0] != size:
        raise ValueError(f"{name} must have {size} elements, got {t.shape[0]}")
    return t.data_ptr()


def _err(err, device):
    return 0 if err is None else _vector("err", err, torch.int32, device, 1)


def _device(t, name):
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.device


def _call(fn, device, pack, *values):
    """Pack the argument struct (its size first) and call ``fn`` with the tensors' device current."""
    args = pack.pack(pack.size, *values)
    if torch.cuda.current_device() == device.index:
        check(fn(args))
    else:
        with torch.cuda.device(device):
            check(fn(args))


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _cache(k, v, heads, dim, dtype, device):
    """The hsg_page_cache fields of k and v [pages, page_size, heads, dim], which have the same strides."""
    _tensor("k_cache", k, 4, dtype, device)
    _tensor("v_cache", v, 4, dtype, device)
    shape, stride = k.shape, k.stride()
    if v.shape != shape or v.stride() != stride or shape[2] != heads or shape[3] != dim:
        raise ValueError(f"k_cache and v_cache must be alike, [pages, page_size, {heads}, {dim}]")
    return k.data_ptr(), v.data_ptr(), stride[0], stride[1], stride[2], shape[0], shape[1]


def _heads(q, k, v):
    """(tokens, hq, hkv, dim) of q [tokens, hq, dim], k and v [tokens, hkv, dim]."""
    tokens, hq, dim = q.shape
    if k.shape != v.shape or k.shape[0] != tokens or k.shape[2] != dim:
        raise ValueError("k and v must be alike, [tokens, kv heads, dim] with q's tokens and dim")
    return tokens, hq, k.shape[1], dim


def raise_device_error(err):
    """Wait for ``err``'s device work and raise HsgError if a kernel recorded a problem there; clears the word."""
    code = int(err.item())
    if code:
        err.zero_()
        raise _lib.HsgError(_lib.HSG_ERR_DEVICE, "device error %d: %s" %
                            (code, _lib.lib().hsg_device_error_text(code).decode()))


def advance_tables(lens, delta, table, ring, counters, page_size, capacity, err=None):
    """Append (delta > 0) or take back (delta < 0) tokens: pages from and to the ring of free pages, slots, positions.

    lens, delta [rows] int32; table [rows, width] int32 (page ids of each request in order) and ring [n] int32 (free
    pages are entries counters[0] .. counters[1] - 1, modulo n) change in place; counters [2] int64. Returns
    ``Tables(lens, counters, cu, slots, rows, positions)``: the new lengths and counters, and for the appended tokens in
    request order their offsets cu [rows + 1] and, each [capacity] with -1 past the last token, cache slot
    (page id * page_size + offset), request and position. An append that the free pages or the table's width cannot
    hold is not made: its length stays as it was. The inputs lens and counters are kept, so the same call again gives
    the same result."""
    device = _device(lens, "lens")
    rows, i32 = lens.shape[0] if lens.dim() else 0, torch.int32
    if rows > MAX_TABLE_ROWS:
        raise ValueError(f"at most {MAX_TABLE_ROWS} requests a call, got {rows}")
    _tensor("table", table, 2, i32, device)
    if table.shape[0] != rows:
        raise ValueError(f"table must have {rows} rows, got {table.shape[0]}")
    if not isinstance(capacity, int) or capacity < 0:
        raise ValueError("capacity must be a non-negative integer")
    room = (capacity + 3) // 4 * 4  # the three lists each begin on a 16-byte boundary
    out = torch.empty(2 * rows + 1 + 3 + 3 * room, dtype=i32, device=device)
    new_counters = torch.empty(2, dtype=torch.int64, device=device)
    lists = (2 * rows + 1 + 3) // 4 * 4
    base = out.data_ptr()
    at = base + 4 * lists
    _call(_lib.lib().hsg_advance_tables, device, _TABLES, _vector("lens", lens, i32, device),
          _vector("delta", delta, i32, device, rows), table.data_ptr(), table.stride(0) if rows > 1 else table.shape[1],
          _vector("ring", ring, i32, device), _vector("counters", counters, torch.int64, device, 2), base,
          new_counters.data_ptr(), base + 4 * rows, at, at + 4 * room, at + 8 * room, _err(err, device),
          _stream(device), rows, table.shape[1], ring.shape[0], page_size, capacity)
    return Tables(out[:rows], new_counters, out[rows:2 * rows + 1], out[lists:lists + capacity],
                  out[lists + room:lists + room + capacity], out[lists + 2 * room:lists + 2 * room + capacity])


def plan_tree(parents, cu, lens, max_tree, err=None):
    """Positions [tokens] int32 and ancestor masks [tokens, words] int32 of drafted trees of at most max_tree tokens.

    parents [tokens] int32: each token's parent as an index within its request (an earlier token) or -1; cu [rows + 1]
    and lens [rows] int32. A token's position is its request's length plus its depth; bit j of its mask is set iff j is
    the token itself or one of its ancestors."""
    device = _device(parents, "parents")
    i32 = torch.int32
    if not isinstance(max_tree, int) or not 1 <= max_tree <= MAX_TREE:
        raise ValueError(f"max_tree must be in [1, {MAX_TREE}]")
    p = _vector("parents", parents, i32, device)
    n = _vector("lens", lens, i32, device)
    rows, tokens, words = lens.shape[0], parents.shape[0], (max_tree + 31) // 32
    c = _vector("cu", cu, i32, device, rows + 1)
    positions = torch.empty(tokens, dtype=i32, device=device)
    mask = torch.empty(tokens, words, dtype=i32, device=device)
    _call(_lib.lib().hsg_plan_tree, device, _TREE, p, c, n, positions.data_ptr(), mask.data_ptr(), _err(err, device),
          _stream(device), rows, tokens, words)
    return positions, mask


def _norm_rope(q, k, v, q_weight, k_weight, inv_freq, positions, eps, dtype, k_cache, v_cache, slots, err):
    device, dtypes = _device(q, "q"), _DTYPES
    if q.dtype not in dtypes:
        raise ValueError("q, k and v must be fp32, fp16 or bf16")
    for name, t in (("q", q), ("k", k), ("v", v)):
        _tensor(name, t, 3, q.dtype, device)
    tokens, hq, hkv, dim = _heads(q, k, v)
    f32 = torch.float32
    out = torch.empty(tokens, hq, dim, dtype=dtype, device=device)
    if slots is None:
        kv = torch.empty(2, tokens, hkv, dim, dtype=dtype, device=device)
        k_out, v_out = kv.unbind(0)
        kp, vp, sp, cache = k_out.data_ptr(), v_out.data_ptr(), 0, (0, 0, 0, 0, 0, 0, 0)
    else:
        k_out = v_out = None
        kp, vp, sp = 0, 0, _vector("slots", slots, torch.int32, device, tokens)
        cache = _cache(k_cache, v_cache, hkv, dim, dtype, device)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    _call(_lib.lib().hsg_norm_rope, device, _NORM, q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1],
          vs[0], vs[1], _vector("q_weight", q_weight, f32, device, dim), _vector("k_weight", k_weight, f32, device, dim),
          _vector("inv_freq", inv_freq, f32, device), _vector("positions", positions, torch.int32, device, tokens),
          out.data_ptr(), kp, vp, sp, *cache, _err(err, device), _stream(device), tokens, hq, hkv, dim,
          2 * inv_freq.shape[0], dtypes[q.dtype], dtypes[dtype], eps)
    return out, k_out, v_out


def norm_rope(q, k, v, q_weight, k_weight, inv_freq, positions, eps, dtype, err=None):
    """Per-head RMSNorm of q and k, then rotation of their first 2 * len(inv_freq) dims; v is only converted.

    q [tokens, hq, dim], k and v [tokens, hkv, dim] (fp32, fp16 or bf16; any token and head strides that keep rows on
    16-byte boundaries, such as slices of one projection); q_weight, k_weight [dim] fp32; inv_freq [rot / 2] fp32;
    positions [tokens] int32; dim 64, 128 or 256, rot a multiple of 16. Dims d and d + rot / 2 turn by
    positions * inv_freq[d]. Returns contiguous (q, k, v) in ``dtype`` (fp16 or bf16)."""
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("dtype must be torch.float16 or torch.bfloat16")
    return _norm_rope(q, k, v, q_weight, k_weight, inv_freq, positions, eps, dtype, None, None, None, err)


def norm_rope_store(q, k, v, q_weight, k_weight, inv_freq, positions, eps, k_cache, v_cache, slots, err=None):
    """``norm_rope`` for tokens that are committed at once: k and v go to cache slots [tokens] int32 (a negative slot:
    nowhere) of k_cache, v_cache [pages, page_size, hkv, dim], in the cache's type. Returns q."""
    if not isinstance(k_cache, torch.Tensor) or k_cache.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("the cache must be fp16 or bf16")
    if slots is None:
        raise ValueError("slots must be given")
    return _norm_rope(q, k, v, q_weight, k_weight, inv_freq, positions, eps, k_cache.dtype, k_cache, v_cache, slots,
                      err)[0]


_WORKSPACE = {}


def attention_workspace(dim):
    """Bytes of workspace a ``tree_attention`` call of this head dim uses."""
    if dim not in _WORKSPACE:
        _WORKSPACE[dim] = int(_lib.lib().hsg_tree_attention_workspace(dim))
    return _WORKSPACE[dim]


def tree_attention(q, k, v, k_cache, v_cache, table, lens, cu, scale, max_tree, mask=None, positions=None, window=0,
                   workspace=None, err=None):
    """Attention of drafted tokens over their request's cached tokens and their own ancestors.

    q [tokens, hq, dim], k and v [tokens, hkv, dim] (fp16 or bf16, hq a multiple of hkv, dim 64, 128 or 256; any
    strides that keep rows on 16-byte boundaries); k_cache and v_cache [pages, page_size, hkv, dim] views of the same
    type, alike in strides; table [rows, width], lens [rows], cu [rows + 1] int32. mask [tokens, words] int32 as
    ``plan_tree`` makes it (any bits may be set or not; None: a chain). With window > 0 only keys at positions above
    the query's own minus window are seen; positions [tokens] int32 (None: length + index) are read only then.
    Returns out [tokens, hq, dim] in q's type and the log-sum-exp [tokens, hq] fp32; a token that sees nothing gets 0
    and -inf. ``workspace`` (a uint8 tensor of ``attention_workspace(dim)`` bytes, for one call at a time) is allocated
    when it is not given."""
    device, i32 = _device(q, "q"), torch.int32
    dtype = q.dtype
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise ValueError("q, k, v and the cache must be fp16 or bf16")
    _tensor("q", q, 3, dtype, device)
    _tensor("k", k, 3, dtype, device)
    _tensor("v", v, 3, dtype, device)
    tokens, hq, hkv, dim = _heads(q, k, v)
    cache = _cache(k_cache, v_cache, hkv, dim, dtype, device)
    _tensor("table", table, 2, i32, device)
    rows, width = table.shape
    n = _vector("lens", lens, i32, device, rows)
    c = _vector("cu", cu, i32, device, rows + 1)
    words, m, p = 0, 0, 0
    if mask is not None:
        _tensor("mask", mask, 2, i32, device)
        words = mask.shape[1]
        if mask.shape[0] != tokens or not mask.is_contiguous():
            raise ValueError(f"mask must be contiguous, [{tokens}, words]")
        m = mask.data_ptr()
    if positions is not None:
        p = _vector("positions", positions, i32, device, tokens)
    if not isinstance(max_tree, int) or not 1 <= max_tree <= MAX_TREE:
        raise ValueError(f"max_tree must be in [1, {MAX_TREE}]")
    need = attention_workspace(dim)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    else:
        _tensor("workspace", workspace, 1, torch.uint8, device)
    out = torch.empty(tokens, hq, dim, dtype=dtype, device=device)
    lse = torch.empty(tokens, hq, dtype=torch.float32, device=device)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    _call(_lib.lib().hsg_tree_attention, device, _ATTENTION, q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1],
          ks[0], ks[1], vs[0], vs[1], *cache, table.data_ptr(), table.stride(0) if rows > 1 else width, n, c, p, m,
          out.data_ptr(), lse.data_ptr(), workspace.data_ptr(), workspace.numel(), _err(err, device), _stream(device),
          rows, width, tokens, words, max_tree, hq, hkv, dim, window, _DTYPES[dtype], scale)
    return out, lse


def store_rows(k, v, k_cache, v_cache, slots, source=None, err=None):
    """Copy rows of k and v [rows, hkv, dim] into cache slots, in place: row source[i] (None: i) to slots[i], both
    [count] int32; a negative slot is skipped. The slots must differ. fp16 or bf16, as the cache."""
    device, i32 = _device(k, "k"), torch.int32
    if k.dtype is not torch.float16 and k.dtype is not torch.bfloat16:
        raise ValueError("k, v and the cache must be fp16 or bf16")
    _tensor("k", k, 3, k.dtype, device)
    _tensor("v", v, 3, k.dtype, device)
    if k.shape != v.shape:
        raise ValueError("k and v must be alike, [rows, kv heads, dim]")
    rows, heads, dim = k.shape
    cache = _cache(k_cache, v_cache, heads, dim, k.dtype, device)
    s = _vector("slots", slots, i32, device)
    count = slots.shape[0]
    if source is None and count > rows:
        raise ValueError(f"{count} slots for {rows} rows")
    src = 0 if source is None else _vector("source", source, i32, device, count)
    ks, vs = k.stride(), v.stride()
    _call(_lib.lib().hsg_store_rows, device, _STORE, k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1], src, s,
          *cache, _err(err, device), _stream(device), count, rows, heads, dim)


class DraftCache:
    """Pages of keys and values for several layers that share one table, and the tables themselves.

    ``k[layer]``, ``v[layer]`` [pages, page_size, kv_heads, dim]; ``table`` [rows, width], ``lens`` [rows], free-page
    ``ring`` [pages] and ``counters`` as ``advance_tables`` takes them: ``advance`` moves them on. Rows are the callers'
    requests; a finished one gives its pages back with a delta of minus its length."""

    def __init__(self, layers, rows, pages, page_size, max_len, kv_heads, dim, dtype=torch.float16, device=None):
        if min(layers, rows, pages, max_len, kv_heads) < 1 or rows > MAX_TABLE_ROWS:
            raise ValueError("layers, rows, pages, max_len and kv_heads must be positive, rows at most %d" %
                             MAX_TABLE_ROWS)
        if page_size < 8 or page_size % 8 or dim not in (64, 128, 256):
            raise ValueError("page_size must be a multiple of 8, dim 64, 128 or 256")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("the cache must be fp16 or bf16")
        device = torch.device("cuda", torch.cuda.current_device() if device is None else device)
        pool = torch.zeros(2, layers, pages, page_size, kv_heads, dim, dtype=dtype, device=device)
        self.k, self.v, self.page_size = pool[0], pool[1], page_size
        self.table = torch.full((rows, (max_len + page_size - 1) // page_size), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.ring = torch.arange(pages, dtype=torch.int32, device=device)
        self.counters = torch.tensor([0, pages], dtype=torch.int64, device=device)
        self.err = torch.zeros(1, dtype=torch.int32, device=device)
        self.workspace = torch.empty(attention_workspace(dim), dtype=torch.uint8, device=device)

    def advance(self, delta, capacity):
        """``advance_tables`` by delta [rows]; the cache's lengths and counters become the new ones."""
        t = advance_tables(self.lens, delta, self.table, self.ring, self.counters, self.page_size, capacity, self.err)
        self.lens, self.counters = t.lens, t.counters
        return t

    def store(self, layer, k, v, slots, source=None):
        """``store_rows`` into a layer's pages."""
        store_rows(k, v, self.k[layer], self.v[layer], slots, source, self.err)

    def attend(self, layer, q, k, v, cu, scale, max_tree, mask=None, positions=None, window=0):
        """``tree_attention`` over a layer's pages: (out, lse)."""
        return tree_attention(q, k, v, self.k[layer], self.v[layer], self.table, self.lens, cu, scale, max_tree, mask,
                              positions, window, self.workspace, self.err)

    def raise_device_error(self):
        """Wait for the device and raise HsgError if a kernel met an index outside its range."""
        raise_device_error(self.err)
