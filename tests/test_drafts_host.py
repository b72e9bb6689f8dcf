"""Draft scoring on the host: argument checks of the C entry points and of the Python layer, no GPU."""
import struct

import pytest
import torch

from hs_guard_b200 import _lib, drafts

# the argument structs of include/hsg.h as a host without a C compiler packs them ("0q" pads the end as C does)
CACHE = "PPqqqii"
TABLES = struct.Struct("@qPPPqPPPPPPPPPPiiiii0q")
TREE = struct.Struct("@qPPPPPPPiii0q")
NORM = struct.Struct("@qPPPqqqqqqPPPPPPPP" + CACHE + "PPiiiiiiif0q")
ATTENTION = struct.Struct("@qPPPqqqqqq" + CACHE + "PqPPPPPPPqPPiiiiiiiiiif0q")
STORE = struct.Struct("@qPPqqqqPP" + CACHE + "PPiiii0q")


@pytest.fixture(scope="module")
def L():
    from hs_guard_b200.build import build
    build()
    return _lib.lib()


PACKS = [("hsg_advance_tables", TABLES), ("hsg_plan_tree", TREE), ("hsg_norm_rope", NORM),
         ("hsg_tree_attention", ATTENTION), ("hsg_store_rows", STORE)]


@pytest.mark.parametrize("name,pack", PACKS, ids=[n for n, _ in PACKS])
def test_argument_structs_have_the_librarys_size(L, name, pack):
    fn = getattr(L, name)
    zeros = [0] * (len(pack.unpack(bytes(pack.size))) - 1)
    assert fn(pack.pack(pack.size, *zeros)) != 0
    assert "expects" not in L.hsg_last_error().decode()
    assert fn(pack.pack(pack.size - 8, *zeros)) == _lib.HSG_ERR_INVALID
    assert "expects %d" % pack.size in L.hsg_last_error().decode()
    assert fn(None) == _lib.HSG_ERR_INVALID


def _attention(**kw):
    fields = ("q k v qt qh kt kh vt vh ck cv ps ts hs pages page table tstride lens cu positions mask out lse ws wsb err "
              "stream rows width tokens words max_tree hq hkv dim window dtype scale").split()
    a = dict.fromkeys(fields, 0)
    a.update(q=16, k=16, v=16, qt=1024, qh=128, kt=256, kh=128, vt=256, vh=128, ck=16, cv=16, ps=4096, ts=256, hs=128, pages=4,
             page=16, table=16, tstride=2, lens=16, cu=16, mask=16, out=16, lse=16, ws=16, wsb=1 << 40, rows=1, width=2, tokens=3,
             words=1, max_tree=3, hq=8, hkv=2, dim=128, dtype=1, scale=1.0)
    a.update(kw)
    return ATTENTION.pack(ATTENTION.size, *(a[f] for f in fields))


@pytest.mark.parametrize("bad", [
    dict(q=0), dict(k=0), dict(v=0), dict(table=0), dict(lens=0), dict(cu=0), dict(out=0), dict(ck=0), dict(q=8), dict(v=24),
    dict(cv=20), dict(qt=1025), dict(kh=4), dict(ts=250), dict(hs=-128), dict(ts=64), dict(pages=0), dict(page=0), dict(page=12),
    dict(page=4), dict(pages=1 << 30, page=16), dict(rows=-1), dict(tokens=-1), dict(hq=0), dict(hkv=0), dict(hkv=3), dict(dim=96),
    dict(dtype=0), dict(dtype=3), dict(max_tree=0), dict(max_tree=1025), dict(max_tree=33), dict(window=-1), dict(width=0),
    dict(tstride=1), dict(width=1 << 28, tstride=1 << 28), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
    dict(scale=float("nan")), dict(hq=258), dict(qt=0), dict(qh=0), dict(kt=0),
    dict(vh=0), dict(vt=-8), dict(ps=0), dict(ws=0), dict(ws=8), dict(wsb=1000)])
def test_tree_attention_refuses(L, bad):
    assert L.hsg_tree_attention(_attention(**bad)) == _lib.HSG_ERR_INVALID
    assert L.hsg_last_error()


def test_a_call_without_work_does_nothing(L):
    assert L.hsg_tree_attention(_attention(tokens=0)) == _lib.HSG_OK
    assert L.hsg_tree_attention(_attention(rows=0)) == _lib.HSG_OK
    assert L.hsg_plan_tree(TREE.pack(TREE.size, *[0] * 7, 4, 0, 1)) == _lib.HSG_OK


def test_advance_tables_refuses_aliased_outputs(L):
    def call(lens_out=48, counters_out=64, lens=16, counters=32, rows=1, ring=4, page=16, capacity=0):
        return L.hsg_advance_tables(TABLES.pack(
            TABLES.size, lens, 16, 16, 2, 16, counters, lens_out, counters_out, 16, 16, 16, 16, 0, 0, rows, 2, ring,
            page, capacity))
    assert call(lens_out=16) == _lib.HSG_ERR_INVALID
    assert call(counters_out=32) == _lib.HSG_ERR_INVALID
    assert call(rows=4097) == _lib.HSG_ERR_INVALID
    assert call(ring=1 << 30, page=16) == _lib.HSG_ERR_INVALID
    assert call(capacity=-1) == _lib.HSG_ERR_INVALID


def test_host_tensors_are_refused():
    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        drafts.plan_tree(i, i, i, 4)
    with pytest.raises(ValueError, match="CUDA"):
        drafts.advance_tables(i, i, i, i, i, 16, 4)
    with pytest.raises(ValueError, match="CUDA"):
        drafts.norm_rope(x, x, x, i, i, i, i, 1e-6, torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        drafts.tree_attention(x, x, x, x, x, i, i, i, 1.0, 4)
    with pytest.raises(ValueError, match="CUDA"):
        drafts.store_rows(x, x, x, x, i)


def test_device_error_texts(L):
    assert L.hsg_device_error_text(0) == b"no error"
    assert b"page" in L.hsg_device_error_text(6) and b"parent" in L.hsg_device_error_text(7)
