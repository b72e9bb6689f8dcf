"""Draft scoring: trees of drafted tokens attended over a paged cache before any of them is accepted.

A host model that drafts several continuations of a conversation has all of them scored in one pass. Per tick and
attention layer (requests b, drafted tokens in request order, ``cu`` [rows + 1] their offsets):

    positions, mask = plan_tree(parents, cu, lens, max_tree)             # once a tick
    q, k, v = norm_rope(q, k, v, qw, kw, inv_freq, positions, eps, torch.float16)
    out, lse = tree_attention(q, k, v, k_cache, v_cache, table, lens, cu, scale, max_tree, mask, positions, window)

and once a branch is accepted:

    t = advance_tables(lens, delta, table, ring, counters, page_size, capacity)    # once a tick
    store_rows(k, v, k_cache, v_cache, t.slots, source)                            # every layer

``DraftCache`` holds the pages, tables and counters of several layers and calls the last two; ``ring_cache`` shows a live
engine's 512-token rings as such a cache. All of this is one softmax layer's part: the layer's projections come from the
host's model, and what its attention gives goes back there. Every function queues work on torch's current stream of its
tensors' device and waits for nothing; outputs are new tensors unless they are said to change in place. Arguments of a
wrong shape, type, device or alignment raise ``ValueError`` before anything is queued, and so do tensors that require
gradients outside ``torch.no_grad()``: there are no backward passes. Values on the device are checked by the kernels, which
skip an index outside its range and record the reason in ``err`` (an int32 tensor of one element, 0 at first; see
``raise_device_error``); without ``err`` nothing says that one was met.

The same over a cache in 8 bits, half the memory and half the reading: keys and values as e4m3 codes with a scale for each block
of tokens and key head. There the newest tokens (one, a chunk of a prompt, a drafted tree) are appended first and then attended
where they lie; what is not accepted is taken back with ``advance_tables``:

    t = advance_tables(...)
    q = append_8bit(k, v, k_cache, v_cache, k_scale, v_scale, t.slots, positions=t.positions, inv_freq=inv_freq, q=q)   # rotates
    out, lse = attention_8bit(q, k_cache, v_cache, k_scale, v_scale, table, t.lens, t.cu, scale, max_new, window=512, sinks=4)

``DraftCache8`` holds such pages. ``token_logprobs`` says from a host's logits how likely the drafted tokens were, how sure the
model is and which tokens it likes best.

Arguments are checked and outputs allocated by the extension module _hsg_torch (csrc/hsg_torch.cpp), which calls
hsg_plan_tree, hsg_norm_rope, hsg_tree_attention, hsg_advance_tables, hsg_store_rows, hsg_append8, hsg_attention8 and
hsg_token_logprobs of include/hsg.h. The reference has no counterpart: its ticks are chains and its caches 512-token rings.
"""
from __future__ import annotations

from collections import namedtuple

import torch

from . import _lib
from .build import tensors

MAX_TREE = 1024        # drafted tokens of one request
MAX_TABLE_ROWS = 4096  # requests of one advance_tables call
MAX_NEW = 1 << 20      # newest tokens of one request in attention_8bit
MAX_TOP = 64           # alternatives of token_logprobs

Tables = namedtuple("Tables", "lens counters cu slots rows positions")
Logprobs = namedtuple("Logprobs", "logprobs entropy lse top top_ids")


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
    hold is not made: its length stays as it was. So is a return that the ring has no room for beside the pages free at
    entry, which is recorded in ``err`` as well: a ring should have an entry for every page. The inputs lens and counters are kept, so the same call again gives
    the same result."""
    return Tables(*tensors().advance_tables(lens, delta, table, ring, counters, page_size, capacity, err))


def plan_tree(parents, cu, lens, max_tree, err=None):
    """Positions [tokens] int32 and ancestor masks [tokens, words] int32 of drafted trees; words hold max_tree bits.

    parents [tokens] int32: each token's parent as an index within its request (an earlier token) or -1; cu [rows + 1]
    and lens [rows] int32. A token's position is its request's length plus its depth; bit j of its mask is set iff j is
    the token itself or one of its ancestors. Tokens outside cu[0] .. cu[rows] - 1, and those of a request whose offsets are
    out of range or which has more tokens than its masks have bits (recorded in ``err``), have position -1 and no bits."""
    return tensors().plan_tree(parents, cu, lens, max_tree, err)


def norm_rope(q, k, v, q_weight, k_weight, inv_freq, positions, eps, dtype, err=None):
    """Per-head RMSNorm of q and k, then rotation of their first 2 * len(inv_freq) dims; v is only converted.

    q [tokens, hq, dim], k and v [tokens, hkv, dim] (fp32, fp16 or bf16; any token and head strides that keep rows on
    16-byte boundaries, such as slices of one projection); q_weight, k_weight [dim] fp32; inv_freq [rot / 2] fp32;
    positions [tokens] int32; dim 64, 128 or 256, rot a multiple of 16. Dims d and d + rot / 2 turn by
    positions * inv_freq[d]. Returns contiguous (q, k, v) in ``dtype`` (fp16 or bf16)."""
    return tensors().norm_rope(q, k, v, q_weight, k_weight, inv_freq, positions, eps, dtype, err)


def norm_rope_store(q, k, v, q_weight, k_weight, inv_freq, positions, eps, k_cache, v_cache, slots, err=None):
    """``norm_rope`` for tokens that are committed at once: k and v go to cache slots [tokens] int32 (a negative slot:
    nowhere) of k_cache, v_cache [pages, page_size, hkv, dim], in the cache's type. Returns q."""
    return tensors().norm_rope_store(q, k, v, q_weight, k_weight, inv_freq, positions, eps, k_cache, v_cache, slots, err)


def attention_workspace(dim):
    """Bytes of workspace a ``tree_attention`` call of this head dim uses."""
    return int(_lib.lib().hsg_tree_attention_workspace(dim))


def tree_attention(q, k, v, k_cache, v_cache, table, lens, cu, scale, max_tree, mask=None, positions=None, window=0,
                   workspace=None, err=None):
    """Attention of drafted tokens over their request's cached tokens and their own ancestors.

    q [tokens, hq, dim], k and v [tokens, hkv, dim] (fp16 or bf16, hq a multiple of hkv, dim 64, 128 or 256; any
    strides that keep rows on 16-byte boundaries); k_cache and v_cache [pages, page_size, hkv, dim] views of the same
    type, alike in strides; table [rows, width], lens [rows], cu [rows + 1] int32. mask [tokens, words] int32 as
    ``plan_tree`` makes it (any bits may be set or not; None: a chain). With window > 0 only keys at positions above
    the query's own minus window are seen; positions [tokens] int32 (None: length + index) are read only then.
    Returns out [tokens, hq, dim] in q's type and the log-sum-exp [tokens, hq] fp32; a token that sees nothing gets 0
    and -inf, as do tokens outside cu[0] .. cu[rows] - 1 and those of a request whose lengths are out of range (which
    ``err`` records). ``workspace`` (a uint8 tensor of ``attention_workspace(dim)`` bytes, for one call at a time) is allocated
    when it is not given."""
    return tensors().tree_attention(q, k, v, k_cache, v_cache, table, lens, cu, scale, max_tree, mask, positions, window,
                                    workspace, err)


def store_rows(k, v, k_cache, v_cache, slots, source=None, err=None):
    """Copy rows of k and v [rows, hkv, dim] into cache slots, in place: row source[i] (None: i) to slots[i], both
    [count] int32; a negative slot is skipped. The slots must differ. fp16 or bf16, as the cache."""
    tensors().store_rows(k, v, k_cache, v_cache, slots, source, err)


def append_8bit(k, v, k_cache, v_cache, k_scale, v_scale, slots, source=None, positions=None, inv_freq=None, interleaved=False,
                rope_scale=1.0, q=None, err=None):
    """Write rows of k and v [rows, hkv, dim] (fp16 or bf16) into slots [count] int32 of an 8-bit cache, in place: row source[i]
    (None: i) to slots[i]; a negative slot is skipped.

    k_cache, v_cache [pages, page_size, hkv, dim] float8_e4m3fn views, alike in strides, rows on 16-byte boundaries; k_scale, v_scale
    [pages, page_size // block, hkv] fp32, contiguous, block a multiple of 8. With inv_freq [rot / 2] fp32 and positions [count]
    int32, the first rot dims of k (a multiple of 16) turn by positions * inv_freq and are multiplied by rope_scale, as rotations stretched for long
    contexts want it: dims (j, j + rot / 2), or (2 j, 2 j + 1) if ``interleaved``. Then q [count, hq, dim] may be given too: its turned
    rows are returned, those of skipped slots among them.

    Entries of one block must stand together (but for skipped ones), in ascending slots (as ``advance_tables`` lists them). A block's scale becomes the
    power of two that its largest appended element asks for (a pair that turns counts with the sum of its magnitudes, so that
    rounding decides nothing); unless its first token is among the entries it does not fall, and when it rises the tokens that
    were there are rounded again. Elements that are not finite become NaN. Slots that do not stand above all of their block's
    before them or lie beyond the pages, and sources outside the rows, are skipped and recorded in ``err``."""
    return tensors().append_8bit(k, v, k_cache, v_cache, k_scale, v_scale, slots, source, positions, inv_freq, interleaved,
                                 rope_scale, q, err)


def attention_8bit_workspace(dim, tokens, heads):
    """Bytes of workspace that an ``attention_8bit`` call of this head dim and up to so many query tokens and heads uses."""
    return int(_lib.lib().hsg_attention8_workspace(dim, tokens, heads))


def attention_8bit(q, k_cache, v_cache, k_scale, v_scale, table, lens, cu, scale, max_new, mask=None, positions=None, window=0,
                   sinks=0, workspace=None, err=None):
    """Attention of each request's newest tokens over its pages of an 8-bit cache.

    q [tokens, hq, dim] (fp16 or bf16, hq a multiple of hkv, at most 128 query heads a key head, dim 64, 128 or 256; any strides
    that keep rows on 16-byte boundaries); cache and scales as in ``append_8bit`` (any positive scales; of v_scale what is below
    2^-80 or above 2^120 is taken as those); table [rows, width], lens [rows], cu [rows + 1] int32. Request b has lens[b] tokens in its pages, the last cu[b + 1] - cu[b] (at most max_new) being
    those of q. They see all tokens before them, and among themselves the earlier ones and their own, or the ones whose bits
    mask [tokens, words] int32 has set (as ``plan_tree`` makes it). With window > 0 only tokens at positions above the query's own
    minus window, or below ``sinks``, are seen; positions [tokens] int32 of q's tokens (at least as many as there are
    tokens before q's; None: their places in the cache) are read only then. Returns out [tokens, hq, dim] in q's type and the log-sum-exp [tokens, hq] fp32; a token that sees nothing gets
    0 and -inf, as do tokens outside cu[0] .. cu[rows] - 1 and those of a request whose lengths are out of range (which ``err``
    records). Tokens of a page outside the cache (recorded as well) are not seen. One kernel is taken for all requests, by their mean number
    of new tokens: chunks of prompts and single tokens are faster in a call each. ``workspace`` (a uint8 tensor of
    ``attention_8bit_workspace(dim, tokens, hq)`` bytes, for one call at a time) is allocated when it is not given."""
    return tensors().attention_8bit(q, k_cache, v_cache, k_scale, v_scale, table, lens, cu, scale, max_new, mask, positions, window,
                                    sinks, workspace, err)


def token_logprobs(logits, given=None, top=0, temperature=1.0, err=None):
    """Log-probabilities of given tokens under softmax(logits / temperature), its entropy and its most likely tokens.

    logits [rows, vocab] fp32, fp16 or bf16, rows at any stride; given [rows] or [rows, n] int32, -1: none; top at most MAX_TOP.
    Returns ``Logprobs(logprobs, entropy, lse, top, top_ids)``: logprobs in given's shape (0 for none; NaN, and recorded in
    ``err``, for a token beyond the vocabulary), entropy and log-sum-exp of logits / temperature [rows], and [rows, top] the
    log-probabilities and ids (int32) of the most likely tokens, of equally likely ones the lowest first. Logits of -inf have no
    probability; a row of nothing else, or with NaN or +inf, has NaN everywhere (but lse -inf for the former) and ids -1."""
    return Logprobs(*tensors().token_logprobs(logits, given, top, temperature, err))


def ring_cache(engine, layer, slots):
    """A live engine's rings of softmax layer ``layer`` (0 .. 5) as the paged cache of ``tree_attention``: (k_cache, v_cache,
    table, lens) for requests ``slots``, to be used with window <= 512 and positions from the slots' lengths on.

    Nothing is copied: the rings [slots + 1, kv heads, 513, dim] are seen as pages of 64 columns that may begin at any
    row, and logical page j of a slot is columns 64 (j mod 8) on. The engine writes its rings on its own stream, and its
    calls return when they have ended: drafted tokens may be attended between its ticks. ``ring_done`` after the last call
    that reads the rings makes the next tick wait for it."""
    cfg, pools = engine.cfg, engine.pools()
    ring_k, ring_v = pools["ring_k"], pools["ring_v"]
    if not 0 <= layer < ring_k.shape[0]:
        raise ValueError(f"layer must be in [0, {ring_k.shape[0]})")
    slots = [int(x) for x in slots]
    if not slots or min(slots) < 0 or max(slots) >= engine.max_slots:
        raise ValueError(f"slots must be in [0, {engine.max_slots})")
    page, cols, heads, dim = 64, cfg.window + 1, cfg.kv_heads, cfg.attn_head_dim
    rows = ring_k[layer].numel() // dim - (heads - 1) * cols - (page - 1)
    if rows * page > 2 ** 31 - 1:
        raise ValueError("the engine's rings are beyond 32-bit page slots: use fewer slots")
    views = [r[layer].as_strided((rows, page, heads, dim), (dim, dim, cols * dim, 1)) for r in (ring_k, ring_v)]
    device = engine.device
    lens = torch.as_tensor(engine.length[slots], dtype=torch.int32, device=device)
    width = max(1, -(-int(engine.length[slots].max()) // page))
    logical = torch.arange(width, device=device) % (cfg.window // page) * page
    table = torch.as_tensor(slots, device=device)[:, None] * (heads * cols) + logical
    return views[0], views[1], table.to(torch.int32), lens


def ring_done(engine):
    """Order the engine's next tick, reset or restore behind what torch's current stream holds by now (calls over its
    ``ring_cache``). Nothing waits on the host; calls on other streams need a call of their own."""
    stream = engine._lib.hsg_stream(engine.handle)
    torch.cuda.ExternalStream(stream, engine.device).wait_stream(torch.cuda.current_stream(engine.device))


class DraftCache:
    """Pages of keys and values for several layers that share one table, and the tables themselves.

    ``k[layer]``, ``v[layer]`` [pages, page_size, kv_heads, dim]; ``table`` [rows, width], ``lens`` [rows], free-page
    ``ring`` [pages] and ``counters`` as ``advance_tables`` takes them: ``advance`` moves them on. Rows are the callers'
    requests; a finished one gives its pages back with a delta of minus its length. Calls that change the cache (advance,
    store) and calls that read it are ordered by their stream; on several streams that order is the caller's."""

    _dtypes = (torch.float16, torch.bfloat16)

    def __init__(self, layers, rows, pages, page_size, max_len, kv_heads, dim, dtype=torch.float16, device=None):
        if min(layers, rows, pages, max_len, kv_heads) < 1 or rows > MAX_TABLE_ROWS:
            raise ValueError("layers, rows, pages, max_len and kv_heads must be positive, rows at most %d" %
                             MAX_TABLE_ROWS)
        if page_size < 8 or page_size % 8 or dim not in (64, 128, 256):
            raise ValueError("page_size must be a multiple of 8, dim 64, 128 or 256")
        if dtype not in self._dtypes:
            raise ValueError("the cache must be %s" % " or ".join(str(d)[6:] for d in self._dtypes))
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError("the cache lives on a CUDA device, got %s" % device)
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        pool = torch.zeros(2, layers, pages, page_size, kv_heads, dim, dtype=dtype, device=device)
        self.k, self.v, self.page_size = pool[0], pool[1], page_size
        self.table = torch.full((rows, (max_len + page_size - 1) // page_size), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.ring = torch.arange(pages, dtype=torch.int32, device=device)
        self.counters = torch.tensor([0, pages], dtype=torch.int64, device=device)
        self.err = torch.zeros(1, dtype=torch.int32, device=device)

    def advance(self, delta, capacity):
        """``advance_tables`` by delta [rows]; the cache's lengths and counters become the new ones."""
        t = advance_tables(self.lens, delta, self.table, self.ring, self.counters, self.page_size, capacity, self.err)
        self.lens, self.counters = t.lens, t.counters
        return t

    def store(self, layer, k, v, slots, source=None):
        """``store_rows`` into a layer's pages."""
        store_rows(k, v, self.k[layer], self.v[layer], slots, source, self.err)

    def attend(self, layer, q, k, v, cu, scale, max_tree, mask=None, positions=None, window=0):
        """``tree_attention`` over a layer's pages: (out, lse). Each call has a workspace of its own, so calls on several
        streams may overlap."""
        return tree_attention(q, k, v, self.k[layer], self.v[layer], self.table, self.lens, cu, scale, max_tree, mask,
                              positions, window, None, self.err)

    def raise_device_error(self):
        """Wait for the device and raise HsgError if a kernel met an index outside its range."""
        raise_device_error(self.err)


class DraftCache8(DraftCache):
    """``DraftCache`` in 8 bits: ``k[layer]``, ``v[layer]`` are e4m3 codes and ``k_scale[layer]``, ``v_scale[layer]`` [pages,
    page_size // block, kv_heads] their scales. New tokens are stored before they are attended: ``advance`` makes room (and takes
    back what was not accepted), ``store`` appends, ``attend`` lets the newest tokens of each request see its pages."""

    _dtypes = (torch.float8_e4m3fn,)

    def __init__(self, layers, rows, pages, page_size, max_len, kv_heads, dim, block=None, device=None):
        block = page_size if block is None else block
        if block < 8 or block % 8 or page_size % block:
            raise ValueError("block must be a multiple of 8 that divides page_size")
        super().__init__(layers, rows, pages, page_size, max_len, kv_heads, dim, torch.float8_e4m3fn, device)
        scales = torch.ones(2, layers, pages, page_size // block, kv_heads, dtype=torch.float32, device=self.k.device)
        self.k_scale, self.v_scale = scales[0], scales[1]

    def store(self, layer, k, v, slots, source=None, positions=None, inv_freq=None, interleaved=False, rope_scale=1.0, q=None):
        """``append_8bit`` into a layer's pages; returns the turned q, if it was given."""
        return append_8bit(k, v, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], slots, source, positions,
                           inv_freq, interleaved, rope_scale, q, self.err)

    def attend(self, layer, q, cu, scale, max_new, mask=None, positions=None, window=0, sinks=0):
        """``attention_8bit`` of each request's newest tokens over a layer's pages: (out, lse)."""
        return attention_8bit(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], self.table, self.lens, cu,
                              scale, max_new, mask, positions, window, sinks, None, self.err)
