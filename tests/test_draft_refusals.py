"""Host-side refusals of the draft operators (no GPU): sizes, types and pointers
that the C entry points must answer with cudaErrorInvalidValue before any CUDA
call, and the Python helpers' own errors."""

import ctypes

import numpy as np
import pytest

from helpers import pkg

INVALID, OK = 1, 0
F32, F16, BF16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    pkg("_build").build()
    return pkg("_lib").load()


def aligned(n=4096):
    raw = ctypes.create_string_buffer(n + 16)
    return raw, (ctypes.addressof(raw) + 15) & ~15


TREE = dict(dtype=F32, rows=4, max_drafts=4, vk=F32, batch=2, hq=8, hkv=2, d=128, page=16, group=128, max_pages=4,
            num_pages=8, window=0, sinks=0)


def tree(lib, p, null=(), **kw):
    a = {**TREE, **kw}
    ptr = {k: (None if k in null else p) for k in ("q", "k", "v", "mask", "offs", "kp", "vp", "sz", "bt", "sl", "out", "ws")}
    ptr.update({k: kw[k] for k in ptr if k in kw})
    return lib.int4kv_paged_tree_decode(
        ptr["q"], ptr["k"], ptr["v"], a["dtype"], ptr["mask"], ptr["offs"], a["rows"], a["max_drafts"], ptr["kp"],
        ptr["vp"], a["vk"], ptr["sz"], ptr["bt"], ptr["sl"], a["batch"], a["hq"], a["hkv"], a["d"], a["page"],
        a["group"], a["max_pages"], a["num_pages"], a["window"], a["sinks"], ptr["out"], ptr["ws"], 0, None, None)


@pytest.mark.parametrize("bad", [
    dict(batch=0), dict(batch=65536), dict(hq=0), dict(hkv=0), dict(hq=7), dict(hq=1, hkv=2), dict(d=96), dict(d=512),
    dict(page=32), dict(group=0), dict(group=24), dict(max_pages=0), dict(num_pages=0), dict(max_pages=1 << 27),
    dict(max_drafts=-1), dict(max_drafts=65), dict(rows=-1), dict(window=-1), dict(sinks=-1), dict(dtype=3),
    dict(vk=-1), dict(dtype=F16), dict(dtype=BF16, vk=F16), dict(hq=1 << 20, hkv=1 << 20),
    dict(batch=65535, hq=64, hkv=64, max_drafts=64, max_pages=1 << 20),
], ids=str)
def test_tree_decode_refuses(lib, bad):
    keep, p = aligned()
    assert tree(lib, p, **bad) == INVALID


@pytest.mark.parametrize("null", ["q", "k", "v", "mask", "offs", "kp", "vp", "sz", "bt", "sl", "out", "ws"])
def test_tree_decode_refuses_null(lib, null):
    keep, p = aligned()
    assert tree(lib, p, null=(null,)) == INVALID


@pytest.mark.parametrize("name", ["q", "k", "v", "kp", "vp", "sz", "out", "ws"])
def test_tree_decode_refuses_misaligned(lib, name):
    keep, p = aligned()
    assert tree(lib, p, **{name: p + 8}) == INVALID


def test_nothing_to_do_is_no_error(lib):
    keep, p = aligned()
    assert tree(lib, p, rows=0) == OK
    assert tree(lib, p, max_drafts=0) == OK


WINDOW = dict(dtype=F32, vk=F32, batch=2, hq=8, hkv=2, d=128, page=16, group=128, max_pages=4, num_pages=8, window=8,
              sinks=0)


@pytest.mark.parametrize("bad", [
    dict(batch=0), dict(hq=7), dict(d=32), dict(page=8), dict(group=8), dict(max_pages=0), dict(num_pages=-1),
    dict(window=0), dict(window=-3), dict(sinks=-1), dict(dtype=9), dict(dtype=F16, vk=F32), dict(q=None), dict(out=None),
    dict(ws=None), dict(sl=None),
], ids=str)
def test_window_decode_refuses(lib, bad):
    keep, p = aligned()
    a = {**WINDOW, **bad}
    ptr = {k: bad.get(k, p) for k in ("q", "kp", "vp", "sz", "bt", "sl", "out", "ws")}
    assert lib.int4kv_paged_window_decode(
        ptr["q"], a["dtype"], ptr["kp"], ptr["vp"], a["vk"], ptr["sz"], ptr["bt"], ptr["sl"], a["batch"], a["hq"],
        a["hkv"], a["d"], a["page"], a["group"], a["max_pages"], a["num_pages"], a["window"], a["sinks"], ptr["out"],
        ptr["ws"], 0, None, None) == INVALID


@pytest.mark.parametrize("bad", [dict(batch=0), dict(d=60), dict(hq=3), dict(max_drafts=65), dict(out=None)], ids=str)
def test_workspace_size_refuses(lib, bad):
    n = ctypes.c_size_t()
    a = {**TREE, **bad}
    out = None if "out" in bad else ctypes.byref(n)
    assert lib.int4kv_paged_attention_workspace_size(a["batch"], a["hq"], a["hkv"], a["d"], a["max_drafts"], out) == INVALID


EXTEND = dict(kd=F32, src=4, nrows=4, slots=2, batch=2, max_rows=4, heads=2, d=64, group=64, page=16, max_pages=4,
              num_pages=8, vk=F32)


def extend(lib, p, **kw):
    a = {**EXTEND, **kw}
    ptr = {k: kw.get(k, p) for k in ("k", "v", "offs", "start", "slot", "stage", "bt", "kp", "vp", "sz")}
    return lib.int4kv_cache_extend(
        ptr["k"], ptr["v"], a["kd"], a["src"], ptr["offs"], ptr["start"], None, a["nrows"], ptr["slot"], ptr["stage"],
        a["slots"], a["batch"], a["max_rows"], a["heads"], a["d"], a["group"], a["page"], ptr["bt"], a["max_pages"],
        a["num_pages"], ptr["kp"], ptr["vp"], a["vk"], ptr["sz"], None, None)


@pytest.mark.parametrize("bad", [
    dict(batch=0), dict(batch=65536), dict(max_rows=-1), dict(heads=0), dict(d=0), dict(d=66), dict(slots=0),
    dict(src=-1), dict(nrows=-1), dict(page=0), dict(group=0), dict(group=40), dict(group=256), dict(kd=3), dict(vk=4),
    dict(max_pages=0), dict(num_pages=0), dict(max_pages=1 << 28), dict(heads=1 << 24, d=128), dict(k=None),
    dict(offs=None), dict(start=None), dict(slot=None), dict(stage=None), dict(bt=None), dict(kp=None), dict(sz=None),
    dict(vp=None), dict(max_rows=1 << 23),
], ids=str)
def test_extend_refuses(lib, bad):
    keep, p = aligned()
    assert extend(lib, p, **bad) == INVALID


def test_extend_refuses_misaligned(lib):
    keep, p = aligned()
    for name in ("k", "v", "kp", "vp", "stage"):
        assert extend(lib, p, **{name: p + 8}) == INVALID
    assert extend(lib, p, max_rows=0) == OK


READ = dict(vk=F32, batch=2, rows=4, max_rows=4, heads=2, d=64, group=64, page=16, max_pages=4, num_pages=8, out=F32)


def read(lib, p, **kw):
    a = {**READ, **kw}
    ptr = {k: kw.get(k, p) for k in ("kp", "vp", "sz", "bt", "start", "offs", "ko", "vo")}
    return lib.int4kv_cache_read(
        ptr["kp"], ptr["vp"], a["vk"], ptr["sz"], ptr["bt"], ptr["start"], ptr["offs"], a["batch"], a["rows"],
        a["max_rows"], a["heads"], a["d"], a["group"], a["page"], a["max_pages"], a["num_pages"], a["out"], ptr["ko"],
        ptr["vo"], None, None)


@pytest.mark.parametrize("bad", [
    dict(batch=0), dict(batch=65536), dict(rows=-1), dict(max_rows=-1), dict(heads=0), dict(d=0), dict(d=6), dict(group=0),
    dict(group=24), dict(page=0), dict(max_pages=0), dict(num_pages=0), dict(out=5), dict(vk=7), dict(kp=None),
    dict(sz=None), dict(bt=None), dict(start=None), dict(offs=None), dict(ko=None), dict(vo=None),
], ids=str)
def test_read_refuses(lib, bad):
    keep, p = aligned()
    assert read(lib, p, **bad) == INVALID


@pytest.mark.parametrize("name", ["kp", "vp", "sz", "ko", "vo"])
def test_read_refuses_misaligned(lib, name):
    keep, p = aligned()
    assert read(lib, p, **{name: p + 4}) == INVALID


def test_tree_mask_words():
    torch = pytest.importorskip("torch")
    P = pkg("paged")
    words = P.tree_mask([[-1, 0, 0, 1, -1], [], [-1]], device="cpu")
    assert words.dtype == torch.int64
    assert words.tolist() == [1, 3, 5, 11, 16, 1]
    # draft 63 is the word's top bit
    chain = P.tree_mask([list(range(-1, 63))], device="cpu")
    assert np.array(chain.tolist(), np.int64).view(np.uint64)[-1] == np.uint64(2 ** 64 - 1)
    for bad in ([[0]], [[-1, 1]], [[-2]], [[-1] * 65]):
        with pytest.raises(ValueError):
            P.tree_mask(bad, device="cpu")


def test_the_gpu_is_required():
    torch = pytest.importorskip("torch")
    C = pkg("_C")
    k = torch.zeros((2, 2, 16, 32), dtype=torch.uint8)
    with pytest.raises(RuntimeError):
        C.cache_read(k, None, torch.zeros((2, 2, 2, 64)), torch.zeros((1, 2), dtype=torch.int32),
                     torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 1, 1)
