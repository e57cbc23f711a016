"""The draft operators in corners of what they allow: mixed types, weights that sum to one,
logits of any size, the end of the longest tables."""

import pytest

from helpers import pkg
from test_gpu_draft_steps import Step
from test_gpu_drafts import BF16, F16, F32, logical

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
C = pkg("_C")
P = pkg("paged")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("values", [F32, F16, BF16])
@pytest.mark.parametrize("kd,vd", [(BF16, F32), (F16, F32), (F16, BF16), (BF16, F16), (F32, BF16), (F32, F16)])
def test_extend_of_mixed_types_equals_bulk_write(kd, vd, values):
    """Keys and values of different types: each is stored as a bulk write of it stores it, bit for bit."""
    heads, d, group, start, new = 2, 64, 32, [0, 5, 40], [3, 30, 1]
    g = torch.Generator(device="cuda").manual_seed(2)
    keys = [(torch.randn((a + b, heads, d), generator=g, device="cuda") * 3 + 1).to(kd) for a, b in zip(start, new)]
    vals = [(torch.randn((a + b, heads, d), generator=g, device="cuda") * 2).to(vd) for a, b in zip(start, new)]
    if vd != F16 and values != F16:
        vals[0][1, 0, 3] = 1e5  # beyond float16
    caches = [P.PagedKVCache(40, heads, d, group_tokens=group, device="cuda", seed=s, value_dtype=values) for s in (1, 2)]
    ids = [0, 1, 2]
    caches[0].write_sequences(ids, keys, vals)
    caches[1].write_sequences(ids, [k[:n] for k, n in zip(keys, start)], [v[:n] for v, n in zip(vals, start)])
    caches[1].extend(ids, new, torch.cat([k[n:] for k, n in zip(keys, start)]),
                     torch.cat([v[n:] for v, n in zip(vals, start)]))
    for s in ids:
        for x, y in zip(logical(caches[1], s), logical(caches[0], s)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hkv,d,drafts", [(8, 4, 128, 8), (8, 2, 128, 8), (16, 2, 64, 8), (32, 2, 128, 8), (8, 4, 256, 13)])
def test_weights_sum_to_one(hq, hkv, d, drafts, dtype):
    """Where every value is 1 every output is: the sum takes the weights as the product does,
    rounded. (Exact: float32 sums are off by 2^-24 times the count of tokens at most, below
    2^-12 here, and 1 is the nearest 16-bit value to all that is closer than that.)"""
    s = Step([1000, 130, 0, 2000], [drafts] * 4, hq, hkv, d, 128, dtype, dtype, seed=d)
    s.v.fill_(1)
    s.pools[1].fill_(1)
    s.q *= 12  # few tokens carry most of the weight
    assert (s.run() == 1).all()
    out = C.paged_window_decode(s.q[:4].contiguous(), *s.pools[:5], window=300, sinks=5, group_tokens=128)
    assert (out[[0, 1, 3]] == 1).all()


@pytest.mark.parametrize("dtype,size", [(BF16, 1e3), (BF16, 30.0), (F16, 1e4), (F16, 200.0), (F32, 1e16)])
def test_logits_of_any_size(dtype, size):
    """Logits from 10^5 to 10^34 (bfloat16: up to 2^29), above and below zero: a row's only token has
    weight 1, the lower of two none, and two equal ones a half each."""
    s = Step([0, 0, 0, 0, 40], [1, 3, 2, 300 // 6, 2], 8, 2, 128, 64, dtype, dtype)
    words = s.words.copy()
    words[:6] = [1, 1, 2, 4, 3, 3]
    s.q.fill_(size)
    s.q[:, 1::2].neg_()
    s.k.fill_(-size)
    s.k[5] = -2 * size
    s.k[6:] = -2 * size
    s.k[20] = -size
    s.k[31] = -size
    words[6:56] = (1 << 50) - 1
    out = s.run(words=words)
    v = s.v.double().repeat_interleave(4, dim=1)
    for row in range(4):
        assert torch.equal(out[row], v[row].to(dtype))
    low = torch.tensor([False, True] * 4, device="cuda")[:, None]  # heads of negative queries: positive logits
    # q > 0: the higher logit is that of draft 4, of the key nearer to zero; q < 0: draft 5's
    for row in (4, 5):
        assert torch.equal(out[row], torch.where(low, v[5], v[4]).to(dtype))
    half = ((v[20] + v[31]) / 2).expand(50, 8, 128)
    tol = torch.finfo(dtype).eps / 2 * half.abs() + 2.0 ** -22 * (v[20].abs() + v[31].abs())
    assert ((out[6:56].double() - half).abs() <= tol)[:, 0::2].all()
    # a cache of keys from -20 to -5 times 2^e, one of them seen
    k_pool, v_pool, sz, bt, sl, _ = s.pools
    scale = {1e16: 2.0 ** 60, 1e3: 2.0 ** 6, 30.0: 2.0 ** 4, 1e4: 2.0 ** 60, 200.0: 2.0 ** 5}[size]
    sz[:, :, 0], sz[:, :, 1] = scale, 20
    q = torch.full((5, 8, 128), size, device="cuda").to(dtype)
    out = C.paged_window_decode(q, *s.pools[:5], window=1, group_tokens=64)
    assert torch.equal(out[4].view(2, 4, 128), v_pool[bt[4, 39 // 16], :, 39 % 16][:, None].expand(2, 4, 128))


@pytest.mark.parametrize("bound", [40, 4000])  # the rows there are, and a bound that reaches past 2^31
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_end_of_the_longest_table(dtype, bound):
    """The last 40 tokens of the longest table there may be: as the same tokens of a short one."""
    heads, d, group, n = 2, 64, 128, 40
    pages = (2 ** 31 - 1025) // 16
    first = pages * 16 // group * group  # the last group, of 112 tokens
    start = pages * 16 - n
    k, v = (torch.randn((n, heads, d), device="cuda").to(dtype) for _ in range(2))
    stage = torch.randn((1, group, heads * d), device="cuda")
    longest = torch.full((1, pages), -1, dtype=torch.int32, device="cuda")
    short = i32([[3, 1, 0, 5, 2, 6, 4]])
    longest[:, first // 16:] = short
    got = []
    for table, at in ((longest, start), (short, start - first)):
        pools = [torch.zeros((8, heads, 16, d // 2), dtype=torch.uint8, device="cuda"),
                 torch.zeros((8, heads, 16, d), dtype=dtype, device="cuda"), torch.zeros((8, heads, 2, d), device="cuda")]
        staged, status = stage.clone(), i32([0])
        C.cache_extend(k, v, i32([0, n]), i32([at]), i32([0]), staged, table, *pools, bound, group, status=status)
        out = C.cache_read(*pools, table, i32([at]), i32([0, n]), n, bound, group, dtype=dtype, status=status)
        assert status.item() == 0
        got.append((*pools, staged, *out))
    assert all(torch.equal(x, y) for x, y in zip(*got))
    assert torch.equal(got[0][5], v)


def test_the_cache_reports_what_its_calls_met():
    """A row index on the device that names no row, a page outside the pool: found by ``check``."""
    k = torch.randn((4, 2, 64), device="cuda")
    cache = P.PagedKVCache(8, 2, 64, group_tokens=32, device="cuda")
    cache.extend([1], [3], k, k, rows=i32([0, 3, 1]))
    q = torch.randn((1, 4, 64), device="cuda")
    cache.window_decode(q, [1], 2)
    cache.read(1)
    cache.check()
    cache.extend([1], [2], k, k, rows=i32([4, 0]))
    with pytest.raises(RuntimeError, match="length"):
        cache.check()
    cache.extend([1], [1], k, k, rows=torch.tensor([2 ** 32 + 1], device="cuda"))
    with pytest.raises(RuntimeError, match="length"):
        cache.check()
    cache.check()
    cache.pages[1][0] = 8
    for call in (lambda: cache.window_decode(q, [1], 2), lambda: cache.read(1), lambda: cache.extend([1], [1], k, k),
                 lambda: cache.tree_decode(q, k[:1], k[:1], [1], [1], P.tree_mask([[-1]]))):
        call()
        with pytest.raises(RuntimeError, match="page"):
            cache.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_padded_drafts_come_back_as_zeros(dtype):
    """More query rows than the counts add up to (a batch of fixed size)."""
    cache = P.PagedKVCache(16, 2, 64, group_tokens=32, device="cuda", value_dtype=dtype)
    k = torch.randn((40, 2, 64), device="cuda").to(dtype)
    cache.extend([1, 2], [20, 3], k, k)
    q = torch.randn((12, 4, 64), device="cuda").to(dtype)
    mask = torch.cat([P.tree_mask([[-1, 0, 1], [-1, -1]]), torch.zeros(7, dtype=torch.int64, device="cuda")])
    want = cache.tree_decode(q[:5], k[:5], k[:5], [1, 2], [3, 2], mask[:5])
    for _ in range(3):
        torch.full_like(q, 9.0)  # (memory that the allocator may hand out next)
        out = cache.tree_decode(q, k[:12], k[:12], [1, 2], [3, 2], mask)
        assert torch.equal(out[:5], want) and (out[5:] == 0).all()
    assert (cache.tree_decode(q, k[:12], k[:12], [1, 2], [0, 0], mask) == 0).all()


@pytest.mark.parametrize("bound", [64, 63])  # values by blocks of their own, and with the keys
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_malformed_rows_and_pages_leave_the_rest(dtype, bound):
    """Groups of 64 tokens: a row index that names no row writes zeros, a page outside the pool is
    not written, and everything else is as it is without them."""
    heads, d, group, n = 2, 64, 64, 40
    k, v = (torch.randn((2 * n, heads, d), device="cuda").to(dtype) for _ in range(2))
    rows = torch.arange(2 * n, dtype=torch.int32, device="cuda").flip(0).contiguous()
    table = i32([[5, 0, 3, 1], [2, 7, 4, 6]])

    def go(rows, table):
        pools = [torch.zeros((8, heads, 16, d // 2), dtype=torch.uint8, device="cuda"),
                 torch.full((8, heads, 16, d), 5.0, dtype=dtype, device="cuda"),
                 torch.full((8, heads, 2, d), 5.0, device="cuda")]
        stage, status = torch.zeros((2, group, heads * d), device="cuda"), i32([0])
        C.cache_extend(k, v, i32([0, n, 2 * n]), i32([0, 0]), i32([1, 0]), stage, table, *pools, bound, group, rows=rows,
                       status=status)
        return status.item(), *pools, stage

    ok = go(rows, table)
    assert ok[0] == 0
    assert torch.equal(ok[2][table[1, :2].long()].transpose(1, 2).reshape(-1, heads, d), v.flip(0)[n:n + 32])
    bad = rows.clone()
    bad[3], bad[n + 17] = -1, 2 * n
    got = go(bad, table)
    assert got[0] == 2
    assert (got[2][5, :, 3] == 0).all() and (got[2][7, :, 1] == 0).all()
    same = torch.ones_like(ok[2], dtype=torch.bool)
    same[5, :, 3] = same[7, :, 1] = False
    assert torch.equal(got[2][same], ok[2][same])
    broken = table.clone()
    broken[0, 1] = 8
    got = go(rows, broken)
    assert got[0] == 1 and (got[2][0] == 5).all()
    rest = [p for p in range(8) if p != 0]
    for x, y in zip(got[1:4], ok[1:4]):
        assert torch.equal(x[rest], y[rest])
    assert torch.equal(got[4], ok[4])


@pytest.mark.parametrize("values", [F32, BF16, None])
def test_an_empty_range_reads_as_no_rows(values):
    cache = P.PagedKVCache(8, 2, 64, group_tokens=32, device="cuda", values=values is not None,
                           value_dtype=values or F32)
    k = torch.randn((20, 2, 64), device="cuda")
    cache.extend([1, 2], [20, 0], k, k if values is not None else None)
    for seq, start, stop in ((1, 0, 0), (1, 20, 20), (1, 7, 7), (2, 0, None)):
        got_k, got_v = cache.read(seq, start, stop, dtype=BF16)
        assert got_k.shape == (0, 2, 64) and got_k.dtype == BF16
        assert got_v is None if values is None else got_v.shape == (0, 2, 64)
    cache.check()


@pytest.mark.parametrize("dtype,values", [(F32, F32), (F32, F16), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("lens,counts", [([3000, 20, 0], [9, 3, 1]), ([17], [2]), ([100] * 40, [5] * 40), ([0, 0], [1, 0])])
def test_a_workspace_may_hold_anything(dtype, values, lens, counts):
    """Leftovers of other calls, notes of streams among them: the results are the same bits."""
    s = Step(lens, counts, 8, 2, 128, 64, dtype, values, seed=7)
    other = Step([2500, 2500], [60, 64], 8, 2, 128, 64, dtype, values, seed=8)
    need = C.paged_attention_workspace_bytes(max(len(lens), 2), 8, 2, 128, 64)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    want = s.run(workspace=ws, max_drafts=64)
    for leave in (lambda: ws.fill_(255), lambda: ws.fill_(1), lambda: ws.view(torch.int32)[:need // 4].random_(0, 200),
                  lambda: ws.random_(0, 256), lambda: other.run(workspace=ws)):
        leave()
        assert torch.equal(s.run(workspace=ws, max_drafts=64), want)
