"""Host side of the draft operators without a GPU: what ``PagedKVCache`` hands to
the binding (replaced by a recorder), on CPU tensors, and limits of the C entry points."""

import pytest

from helpers import pkg
from test_draft_refusals import INVALID, OK, aligned, extend, lib, read  # noqa: F401 (lib: a fixture)

torch = pytest.importorskip("torch")
C = pkg("_C")
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
