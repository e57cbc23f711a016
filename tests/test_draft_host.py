"""Host side of the draft operators without a GPU: what ``PagedKVCache`` hands to
the binding (replaced by a recorder), on CPU tensors, and limits of the C entry points."""

import contextlib
import ctypes

import pytest

from helpers import pkg
from test_draft_refusals import (BF16 as K_BF16, F16 as K_F16, INVALID, OK, aligned, extend,  # noqa: F401
                                 lib, read, tree)  # (lib: a fixture)

torch = pytest.importorskip("torch")
C = pkg("_C")
L = pkg("_lib")
P = pkg("paged")

F32, F16, BF16, F64 = torch.float32, torch.float16, torch.bfloat16, torch.float64


@pytest.fixture
def calls(monkeypatch):
    """The binding's draft entry points, recorded as (name, positional, keyword) in order."""
    seen = []

    def record(name, result=None):
        def call(*args, **kw):
            seen.append((name, args, kw))
            return result(*args, **kw) if result else None
        monkeypatch.setattr(C, name, call)

    record("cache_extend")
    record("cache_read", lambda *a, **kw: (None, None))
    record("paged_window_decode", lambda q, *a, **kw: q)
    record("paged_tree_decode", lambda q, *a, **kw: kw["out"] if kw.get("out") is not None else torch.full_like(q, 7.0))
    return seen


def cache(values=F32, pages=8, group=32):
    return P.PagedKVCache(pages, 2, 8, group_tokens=group, device="cpu", value_dtype=values, max_open_sequences=2)


def rows(n, dtype, seed=0):
    return (torch.randn((n, 2, 8), generator=torch.Generator().manual_seed(seed)) * 3).to(dtype)


@pytest.mark.parametrize("kd,vd", [(BF16, F32), (F16, F32), (F16, BF16), (BF16, F16), (F32, BF16), (BF16, F64), (F32, F64)])
def test_extend_narrows_neither_keys_nor_values(calls, kd, vd):
    """Keys and values of different types reach the kernel in one that holds both."""
    k, v = rows(3, kd), rows(3, vd, 1)
    v[0, 0, 0] = 1e5 if vd != F16 else 6e4  # beyond float16
    cache().extend([4], [3], k, v)
    (_, args, _), = calls
    assert args[0].dtype == args[1].dtype
    assert torch.equal(args[0].float(), k.float()) and torch.equal(args[1].float(), v.float())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_extend_passes_equal_types_on(calls, dtype):
    k, v = rows(3, dtype), rows(3, dtype, 1)
    cache().extend([4], [3], k, v)
    (_, args, _), = calls
    assert args[0].dtype == args[1].dtype == dtype


def test_tables_end_before_positions_do(lib):  # noqa: F811
    """The longest table leaves the kernels' positions room below 2^31."""
    keep, p = aligned()
    longest = (2 ** 31 - 1025) // 16
    for call in (extend, read):
        assert call(lib, p, max_pages=longest + 1) == INVALID
        assert call(lib, p, max_pages=2 ** 31 - 1024, page=1, group=64) == INVALID
        assert call(lib, p, max_pages=longest, max_rows=0) == OK


@pytest.fixture
def bound(monkeypatch):
    """(window, sinks) as the C entry points receive them from the binding, with CPU tensors let through."""
    got = []

    class Lib:
        def int4kv_paged_tree_decode(self, *a):
            got.append((ctypes.c_int(a[22]).value, ctypes.c_int(a[23]).value))
            return 0

        def int4kv_paged_window_decode(self, *a):
            got.append((ctypes.c_int(a[16]).value, ctypes.c_int(a[17]).value))
            return 0

    monkeypatch.setattr(L, "load", lambda: Lib())
    monkeypatch.setattr(C, "_check_input", lambda t, name: None)
    monkeypatch.setattr(C, "_check_pools", lambda k, v, sz: (k.shape[0], k.shape[1], 16, k.shape[3] * 2))
    monkeypatch.setattr(C, "_check_table", lambda bt, b: bt.shape[1])
    monkeypatch.setattr(C, "_guard", lambda i: contextlib.nullcontext())
    monkeypatch.setattr(C, "_attention_need", lambda *a: 16)
    monkeypatch.setattr(C, "_stream", lambda t: 0)
    return got


MOST = 2 ** 31 - 1


@pytest.mark.parametrize("window,sinks,want", [
    (5, 3, (5, 3)), (MOST, MOST, (MOST, MOST)), (2 ** 31, 0, (MOST, 0)), (2 ** 32 + 7, 2 ** 32 + 1, (MOST, MOST)),
    (10 ** 12, 2 ** 40, (MOST, MOST)), (2 ** 63 - 1, 2 ** 63 - 1, (MOST, MOST))])
def test_window_and_sinks_past_32_bits_reach_over_everything(bound, window, sinks, want):
    q = torch.zeros((1, 2, 64))
    k_pool = torch.zeros((2, 2, 16, 32), dtype=torch.uint8)
    v_pool, sz = torch.zeros((2, 2, 16, 64)), torch.zeros((2, 2, 2, 64))
    bt, sl, offs = (torch.zeros(s, dtype=torch.int32) for s in ((1, 2), (1,), (2,)))
    C.paged_window_decode(q, k_pool, v_pool, sz, bt, sl, window, sinks)
    C.paged_tree_decode(q, q, q, torch.zeros(1, dtype=torch.int64), offs, k_pool, v_pool, sz, bt, sl, 1, window=window,
                        sinks=sinks)
    assert bound == [want, want]


@pytest.mark.parametrize("group", [2 ** 31, 2 ** 32 + 16])
def test_groups_past_32_bits_are_refused(bound, group):
    q = torch.zeros((1, 2, 64))
    pools = torch.zeros((2, 2, 16, 32), dtype=torch.uint8), torch.zeros((2, 2, 16, 64)), torch.zeros((2, 2, 2, 64))
    bt, sl = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="group_tokens"):
        C.paged_window_decode(q, *pools, bt, sl, 5, group_tokens=group)
    assert not bound


def state(c):
    return (dict(c.lens), {s: list(p) for s, p in c.pages.items()}, list(c._free), dict(c._stage_slot),
            list(c._stage_free))


REFUSED = {
    "keys of float64": dict(keys=rows(4, F64)), "both of float64": dict(keys=rows(4, F64), values=rows(4, F64)),
    "integer keys": dict(keys=rows(4, F32).int()), "fewer values": dict(values=rows(4, F32)[:3]),
    "row past the keys": dict(rows=torch.tensor([0, 1, 4])),
    "negative row": dict(rows=torch.tensor([0, -1, 2], dtype=torch.int32)),
    "fractional rows": dict(rows=torch.tensor([0.0, 1.0, 2.0])), "rows of two axes": dict(rows=torch.tensor([[0], [1], [2]])),
    "too few rows": dict(rows=torch.tensor([0, 1])), "row past 32 bits": dict(rows=torch.tensor([0, 1, 2 ** 32 + 2])),
    "twice the same": dict(ids=[7, 7]), "negative count": dict(counts=[1, -1]), "too many": dict(counts=[4, 4]),
    "a count too few": dict(counts=[1]),
}


@pytest.mark.parametrize("what", REFUSED)
def test_a_refused_extend_leaves_the_cache_as_it_was(calls, what):
    c = cache()
    c.extend([7], [20], rows(20, F32), rows(20, F32))
    before = state(c)
    a = dict(ids=[7, 9], counts=[1, 2], keys=rows(4, F32), values=rows(4, F32, 1), rows=None)
    a.update(REFUSED[what])
    with pytest.raises(ValueError):
        c.extend(a["ids"], a["counts"], a["keys"], a["values"], rows=a["rows"])
    assert state(c) == before and len(calls) == 1


def test_rows_of_any_integer_type_name_the_new_tokens(calls):
    for dtype in (torch.int32, torch.int64, torch.int16, torch.uint8):
        # (entries past the counts' sum name no token: any value)
        cache().extend([1, 2], [2, 1], rows(4, F32), rows(4, F32), rows=torch.tensor([3, 0, 3, 77], dtype=dtype))
        passed = calls[-1][2]["rows"]
        assert passed.dtype == torch.int32 and passed[:3].tolist() == [3, 0, 3]


def test_draft_calls_share_the_cache_s_status_word(calls):
    c = cache()
    c.extend([1], [3], rows(3, F32), rows(3, F32))
    q = torch.zeros((1, 2, 8))
    c.window_decode(q, [1], 4)
    c.tree_decode(q, q, q, [1], [1], torch.ones(1, dtype=torch.int64))
    c.read(1)
    assert [name for name, _, _ in calls] == ["cache_extend", "paged_window_decode", "paged_tree_decode", "cache_read"]
    assert all(kw["status"] is c.status for _, _, kw in calls)
    c.check()
    for bits, words in ((1, "page"), (2, "length"), (4, "wait"), (3, "page")):
        c.status.fill_(bits)
        with pytest.raises(RuntimeError, match=words):
            c.check()
        c.check()  # told once


def test_tree_rows_that_no_sequence_has_are_zeros(calls):
    c = cache()
    c.extend([1, 2], [3, 1], rows(4, F32), rows(4, F32))
    q = torch.ones((7, 2, 8))
    out = c.tree_decode(q, q, q, [1, 2], [2, 3], torch.ones(7, dtype=torch.int64))
    assert (out[:5] == 7).all() and (out[5:] == 0).all()


def test_no_batch_is_refused_that_the_kernels_can_count(lib):  # noqa: F811
    """Units of work are counted in 31 bits, in tiles and chunks of the kernel that runs: a large
    serving batch (64 drafts, 8 query heads a kv head, tables of 131072 tokens) is none too many.
    (Without a GPU what passes the checks ends at the device; with one, at the empty workspace.)"""
    if torch.cuda.is_available():
        pytest.skip("the answer without a GPU is asked for")
    keep, p = aligned()
    big = dict(d=128, max_drafts=64, rows=64, max_pages=8192, num_pages=1 << 20)
    for kw in (dict(batch=512, hq=64, hkv=8), dict(batch=4096, hq=64, hkv=8), dict(batch=1024, hq=32, hkv=32),
               dict(batch=65535, hq=8, hkv=1)):
        for dtype in (K_F16, K_BF16):
            assert tree(lib, p, **{**big, **kw}, dtype=dtype, vk=dtype) != INVALID
    # behind a window only its tiles count
    assert tree(lib, p, **{**big, "max_pages": 1 << 26}, batch=4096, hq=64, hkv=8, dtype=K_BF16, vk=K_BF16, window=4096,
                sinks=64) != INVALID
    # what is past 31 bits stays refused, in either kernel
    assert tree(lib, p, **{**big, "max_pages": 1 << 26}, batch=4096, hq=64, hkv=8, dtype=K_BF16, vk=K_BF16) == INVALID
    assert tree(lib, p, **{**big, "max_pages": 1 << 20}, batch=4096, hq=64, hkv=8) == INVALID


def test_an_empty_read_is_no_error(lib):  # noqa: F811
    """Outputs of no rows have no address."""
    keep, p = aligned()
    assert read(lib, p, rows=0, ko=None, vo=None) == OK
    assert read(lib, p, max_rows=0, ko=None, vo=None) == OK
    assert read(lib, p, rows=0, vp=None, ko=None, vo=None) == OK
    assert read(lib, p, vo=None) == INVALID and read(lib, p, vp=None) == INVALID


def misaligned(t):
    flat = torch.empty(t.numel() + 1, dtype=t.dtype)[1:].view(t.shape)
    assert flat.copy_(t).data_ptr() % 16
    return flat


def test_tensors_that_start_anywhere_are_taken(calls):
    """The kernels load 16 bytes at a time: what does not start on such a boundary is copied."""
    c = cache()
    c.extend([1], [3], misaligned(rows(3, BF16)), misaligned(rows(3, BF16, 1)))
    q = misaligned(rows(1, F32))
    c.tree_decode(q, q, q, [1], [1], torch.ones(1, dtype=torch.int64))
    c.window_decode(q, [1], 5)
    for (_, args, _), n in zip(calls, (2, 3, 1)):
        assert all(t.data_ptr() % 16 == 0 and t.is_contiguous() for t in args[:n])
    assert torch.equal(calls[0][1][0], rows(3, BF16)) and torch.equal(calls[0][1][1], rows(3, BF16, 1))
