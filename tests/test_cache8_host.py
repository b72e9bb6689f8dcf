"""The 8-bit cache and token log-probabilities on the host: argument checks of the C entry points and of the Python layer, no GPU."""
import struct

import pytest
import torch

from hs_guard_b200 import _lib, drafts

# the argument structs of include/hsg.h as a host without a C compiler packs them ("0q" pads the end as C does)
CACHE = "PPPPqqqiiii"
APPEND = struct.Struct("@qPPPqqqqqqPPPPP" + CACHE + "PPiiiiiiiif0q")
ATTENTION = struct.Struct("@qPqq" + CACHE + "PqPPPPPPPqPPiiiiiiiiiiif0q")
LOGPROBS = struct.Struct("@qPqPPPPPPPPiiiiif0q")


@pytest.fixture(scope="module")
def L():
    from hs_guard_b200.build import build
    build()
    return _lib.lib()


PACKS = [("hsg_append8", APPEND), ("hsg_attention8", ATTENTION), ("hsg_token_logprobs", LOGPROBS)]


@pytest.mark.parametrize("name,pack", PACKS, ids=[n for n, _ in PACKS])
def test_argument_structs_have_the_librarys_size(L, name, pack):
    fn = getattr(L, name)
    zeros = [0] * (len(pack.unpack(bytes(pack.size))) - 1)
    assert fn(pack.pack(pack.size, *zeros)) != 0
    assert "expects" not in L.hsg_last_error().decode()
    assert fn(pack.pack(pack.size - 8, *zeros)) == _lib.HSG_ERR_INVALID
    assert "expects %d" % pack.size in L.hsg_last_error().decode()
    assert fn(None) == _lib.HSG_ERR_INVALID


CACHE_FIELDS = "ck cv ks vs ps ts hs pages page block reserved"
CACHE_OK = dict(ck=16, cv=16, ks=16, vs=16, ps=4096, ts=256, hs=128, pages=4, page=16, block=8)
BAD_CACHE = [dict(ck=0), dict(cv=0), dict(ks=0), dict(vs=0), dict(ck=8), dict(cv=20), dict(ks=2), dict(ps=8), dict(ts=250), dict(hs=-128),
             dict(ts=64), dict(hs=64), dict(ps=0), dict(pages=0), dict(page=12), dict(page=4), dict(block=0), dict(block=4), dict(block=12),
             dict(block=24), dict(pages=1 << 28, page=16)]


def _call(L, name, pack, fields, ok, kw):
    a = dict.fromkeys(fields.split(), 0)
    a.update(ok)
    a.update(kw)
    return getattr(L, name)(pack.pack(pack.size, *(a[f] for f in fields.split())))


def _append(L, **kw):
    fields = ("q k v qt qh kt kh vt vh source slots positions inv qo " + CACHE_FIELDS + " err stream count rows hq hkv dim rot pairs dtype "
              "factor")
    ok = dict(q=16, k=16, v=16, qt=1024, qh=128, kt=256, kh=128, vt=256, vh=128, slots=16, positions=16, inv=16, qo=16, count=3, rows=3,
              hq=8, hkv=2, dim=128, rot=64, dtype=1, factor=1.0, **CACHE_OK)
    return _call(L, "hsg_append8", APPEND, fields, ok, kw)


@pytest.mark.parametrize("bad", BAD_CACHE + [
    dict(k=0), dict(v=0), dict(slots=0), dict(q=0), dict(qo=0), dict(positions=0), dict(inv=0), dict(k=8), dict(v=24), dict(q=4), dict(qo=8),
    dict(qt=1025), dict(kh=4), dict(source=16), dict(count=-1), dict(rows=-1), dict(hq=-1), dict(hkv=0), dict(dim=96), dict(rot=8),
    dict(rot=144), dict(rot=-16), dict(dtype=0), dict(dtype=3), dict(factor=float("inf")), dict(factor=float("nan"))])
def test_append_refuses(L, bad):
    assert _append(L, **bad) == _lib.HSG_ERR_INVALID
    assert L.hsg_last_error()


def _attention(L, **kw):
    fields = ("q qt qh " + CACHE_FIELDS + " table tstride lens cu positions mask out lse ws wsb err stream rows width tokens words max_new "
              "hq hkv dim window sinks dtype scale")
    ok = dict(q=16, qt=1024, qh=128, table=16, tstride=2, lens=16, cu=16, mask=16, out=16, lse=16, ws=16, wsb=1 << 40, rows=1, width=2,
              tokens=3, words=1, max_new=3, hq=8, hkv=2, dim=128, dtype=1, scale=1.0, **CACHE_OK)
    return _call(L, "hsg_attention8", ATTENTION, fields, ok, kw)


@pytest.mark.parametrize("bad", BAD_CACHE + [
    dict(q=0), dict(table=0), dict(lens=0), dict(cu=0), dict(out=0), dict(q=8), dict(out=4), dict(qt=1025), dict(qh=4), dict(rows=-1),
    dict(tokens=-1), dict(hq=0), dict(hkv=0), dict(hkv=3), dict(hq=258), dict(dim=96), dict(dtype=0), dict(dtype=3), dict(max_new=0),
    dict(max_new=33), dict(max_new=(1 << 20) + 1, mask=0), dict(window=-1), dict(sinks=-1), dict(width=0), dict(tstride=1),
    dict(width=1 << 28, tstride=1 << 28), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(ws=0),
    dict(ws=8), dict(wsb=1000)])
def test_attention_refuses(L, bad):
    assert _attention(L, **bad) == _lib.HSG_ERR_INVALID
    assert L.hsg_last_error()


def _logprobs(L, **kw):
    fields = "logits stride given lp ent lse top ids err stream rows vocab n_given n_top dtype t"
    ok = dict(logits=16, stride=100, given=16, lp=16, ent=16, lse=16, top=16, ids=16, rows=2, vocab=100, n_given=1, n_top=5, dtype=2, t=1.0)
    return _call(L, "hsg_token_logprobs", LOGPROBS, fields, ok, kw)


@pytest.mark.parametrize("bad", [
    dict(logits=0), dict(given=0), dict(lp=0), dict(ent=0), dict(lse=0), dict(top=0), dict(ids=0), dict(rows=-1), dict(vocab=0),
    dict(n_given=-1), dict(n_top=-1), dict(n_top=65), dict(vocab=4), dict(dtype=-1), dict(dtype=3), dict(t=0.0), dict(t=-1.0),
    dict(t=float("nan")), dict(t=1e5), dict(stride=-1), dict(logits=17), dict(logits=18, dtype=0), dict(rows=1 << 30)])
def test_logprobs_refuses(L, bad):
    assert _logprobs(L, **bad) == _lib.HSG_ERR_INVALID
    assert L.hsg_last_error()


def test_a_call_without_work_does_nothing(L):
    assert _append(L, count=0) == _lib.HSG_OK
    assert _attention(L, tokens=0) == _lib.HSG_OK
    assert _attention(L, rows=0) == _lib.HSG_OK
    assert _logprobs(L, rows=0) == _lib.HSG_OK


def test_workspace(L):
    assert drafts.attention_8bit_workspace(96, 1, 8) == 0
    small, large = drafts.attention_8bit_workspace(64, 1, 8), drafts.attention_8bit_workspace(256, 1, 8)
    assert 0 < small <= large < drafts.attention_8bit_workspace(256, 2, 8) == drafts.attention_8bit_workspace(256, 1, 16)


def test_host_tensors_are_refused():
    x, i = torch.zeros(2, 2, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        drafts.append_8bit(x, x, x, x, x, x, i)
    with pytest.raises(ValueError, match="CUDA"):
        drafts.attention_8bit(x, x, x, x, x, i, i, i, 1.0, 4)
    with pytest.raises(ValueError, match="CUDA"):
        drafts.token_logprobs(x, i)
    with pytest.raises(ValueError, match="block"):
        drafts.DraftCache8(1, 1, 4, 16, 64, 2, 64, block=24)
    with pytest.raises(ValueError, match="device"):
        drafts.DraftCache8(1, 1, 4, 16, 64, 2, 64, device="cpu")
