"""Tree attention, windowed decode, multi-token extend and read-back on the GPU.

Attention is compared with a float64 evaluation of the definition, row by row.
Tolerances, relative to the largest output (values are N(0, 1), outputs at most
that of the values):

* float32: a logit is a sum of head_dim float32 products of size <= |q| |k|;
  its rounding error is below head_dim * 2^-24 * sum |q_c k_c|, here < 128 *
  6e-8 * 20; an error e of the logits moves the outputs by at most 2 e max|v|.
  Measured errors are near 1e-6; the bound used is 1e-4 * max|v| / 4 = 1e-4.
* 16 bits: keys (or their products' operands) rounded to 11 bits (float16
  operands), weights and outputs to the type: per logit 2^-11 * sum |q_c k_c|
  (below 2^-11 * 8 at these inputs), per weight and output eps / 2 each.
"""

import numpy as np
import pytest

import oracle
from helpers import pkg

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
C = pkg("_C")
P = pkg("paged")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make_cache(lens, heads, d, group, values, seed=0, spare=4):
    """Pools of random codes with N(0, 1) values and keys of moderate size; block table."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [(n + 15) // 16 for n in lens]
    pool = sum(need) + spare
    order = np.random.default_rng(seed).permutation(pool)
    bt = np.zeros((len(lens), max(1, max(need))), np.int32)
    at = 0
    for i, k in enumerate(need):
        bt[i, :k] = order[at:at + k]
        at += k
    k_pool = torch.randint(0, 256, (pool, heads, 16, d // 2), generator=g, device="cuda",
                           dtype=torch.uint8)
    scale = torch.rand((pool, heads, d), generator=g, device="cuda") * 0.3 + 0.05
    zp = torch.randn((pool, heads, d), generator=g, device="cuda") * 3 + 7.5
    sz = torch.stack([scale, zp], 2).contiguous()
    v = torch.randn((pool, heads, 16, d), generator=g, device="cuda").to(values)
    return (k_pool, v, sz, torch.from_numpy(bt).cuda(),
            torch.tensor(lens, dtype=torch.int32, device="cuda"), g)


def tokens64(pools, b, lo, hi, group):
    k_pool, v_pool, sz, bt = pools[:4]
    pos = torch.arange(lo, hi, device="cuda")
    row = bt[b].long()
    page, slot = row[pos // 16], pos % 16
    kb = k_pool[page, :, slot]
    codes = torch.stack([kb & 15, kb >> 4], -1).flatten(-2).double()
    s = sz[row[pos // group * (group // 16)]].double()
    return (codes - s[:, :, 1]) * s[:, :, 0], v_pool[page, :, slot].double()


def random_trees(counts, seed, chains=0.5):
    rng = np.random.default_rng(seed)
    words = []
    for n in counts:
        rows = []
        for i in range(n):
            parent = i - 1 if rng.random() < chains else int(rng.integers(-1, i)) if i else -1
            rows.append((rows[parent] if parent >= 0 else 0) | (1 << i))
        words += rows
    return np.array(words, np.uint64).view(np.int64)


def tree64(q, kd, vd, words, offs, pools, group, window, sinks):
    """Float64 rows of the tree attention."""
    lens = pools[4].tolist()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    hkv, d = kd.shape[1], kd.shape[2]
    for b, n in enumerate(lens):
        o, t = int(offs[b]), int(offs[b + 1] - offs[b])
        kc, vc = tokens64(pools, b, 0, n, group)
        mine = [int(w) % (1 << 64) & ((1 << t) - 1) for w in words[o:o + t]]
        depth = [bin(w & ~(1 << j)).count("1") for j, w in enumerate(mine)]
        for i in range(t):
            p = n + depth[i]
            pos = torch.arange(n, device="cuda")
            sees = torch.ones_like(pos, dtype=torch.bool)
            keep = [j for j in range(t) if mine[i] >> j & 1]
            if window:
                sees = (pos > p - window) | (pos < sinks)
                keep = [j for j in keep if n + depth[j] > p - window or n + depth[j] < sinks]
            k = torch.cat([kc[sees], kd[o:o + t][keep].double()])
            v = torch.cat([vc[sees], vd[o:o + t][keep].double()])
            if k.shape[0]:
                x = torch.einsum("hgd,jhd->hgj", q[o + i].double().view(hkv, -1, d), k)
                out[o + i] = torch.einsum("hgj,jhd->hgd", torch.softmax(x, -1), v).reshape(-1, d)
    return out


def close(out, want, dtype):
    tol = {F32: 1e-4, F16: 2.0 ** -11 * 24, BF16: 2.0 ** -8 * 6}[dtype]
    err = (out.double() - want).abs().max().item()
    assert torch.isfinite(out).all()
    assert err <= tol * max(1.0, want.abs().max().item()), err


TREES = [
    # lens, counts, q heads, kv heads, head_dim, group, dtype, values, window, sinks
    ([37], [1], 4, 4, 64, 128, F32, F32, 0, 0),
    ([0, 1, 15, 16, 17], [1, 2, 3, 4, 5], 4, 2, 128, 128, F32, F32, 0, 0),
    ([300, 0, 129, 1], [7, 5, 0, 64], 8, 2, 128, 128, F32, BF16, 0, 0),
    ([513, 2000], [33, 9], 14, 2, 64, 64, F32, F16, 0, 0),
    ([260, 700], [5, 12], 6, 2, 256, 128, F32, F32, 0, 0),
    ([900, 63, 5], [8, 64, 6], 8, 4, 128, 128, F32, F32, 100, 4),
    ([900, 63, 5], [8, 64, 6], 4, 4, 64, 32, F32, F32, 3, 0),
    ([1500, 1024], [6, 20], 4, 1, 128, 16, F32, F32, 511, 40),
    ([37], [1], 4, 4, 64, 128, BF16, BF16, 0, 0),
    ([0, 1, 15, 16, 17, 128, 129], [1, 2, 3, 4, 5, 6, 7], 8, 2, 128, 128, BF16, BF16, 0, 0),
    ([300, 0, 129, 1], [7, 5, 0, 64], 8, 2, 128, 128, BF16, BF16, 0, 0),
    ([513, 2000, 4096], [33, 9, 64], 14, 2, 64, 64, F16, F16, 0, 0),
    ([260, 700], [5, 12], 6, 2, 256, 128, BF16, BF16, 0, 0),
    ([900, 63, 5], [8, 64, 6], 8, 4, 128, 128, F16, F16, 100, 4),
    ([900, 63, 5], [8, 64, 6], 4, 4, 64, 32, BF16, BF16, 3, 0),
    ([1500, 1024], [6, 20], 4, 1, 128, 16, BF16, BF16, 511, 40),
    ([3000, 10], [60, 3], 32, 4, 128, 128, BF16, BF16, 0, 0),
    ([700, 33], [40, 64], 16, 2, 256, 32, F16, F16, 300, 17),
]


@pytest.mark.parametrize("case", TREES, ids=lambda c: f"{c[2]}-{c[3]}x{c[4]}-{str(c[6])[6:]}-{str(c[7])[6:]}-w{c[8]}-L{max(c[0])}")
def test_tree_decode_matches_float64(case):
    lens, counts, hq, hkv, d, group, dtype, values, window, sinks = case
    pools = make_cache(lens, hkv, d, group, values, seed=len(lens) + d)
    g = pools[-1]
    rows = sum(counts)
    q = (torch.randn((rows, hq, d), generator=g, device="cuda") / d ** 0.5).to(dtype)
    kd = torch.randn((rows, hkv, d), generator=g, device="cuda").to(dtype)
    vd = torch.randn((rows, hkv, d), generator=g, device="cuda").to(dtype)
    words = random_trees(counts, 3)
    offs = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = C.paged_tree_decode(q, kd, vd, torch.from_numpy(words).cuda(), torch.from_numpy(offs).cuda(),
                              *pools[:5], max_drafts=max(counts), group_tokens=group,
                              window=window or None, sinks=sinks, status=status)
    assert status.item() == 0
    close(out, tree64(q, kd, vd, words, offs, pools, group, window, sinks), dtype)


WINDOWS = [
    # lens, q heads, kv heads, head_dim, group, dtype, values, window, sinks
    ([1, 0, 16, 100], 4, 4, 64, 128, F32, F32, 16, 4),
    ([1000, 4096, 17], 8, 2, 128, 128, F32, BF16, 256, 0),
    ([1000, 4096, 17], 8, 8, 128, 128, F32, F32, 1, 0),
    ([3000, 555], 8, 1, 256, 64, F32, F16, 1000, 100),
    ([1, 0, 16, 100], 4, 4, 64, 128, F16, F16, 16, 4),
    ([1000, 4096, 17], 8, 2, 128, 128, BF16, BF16, 256, 0),
    ([1000, 4096, 17], 28, 4, 128, 128, BF16, BF16, 1, 3),
    ([3000, 555], 8, 1, 256, 64, BF16, BF16, 1000, 100),
    ([5000, 200, 5000], 32, 8, 128, 128, BF16, BF16, 100000, 9),
]


@pytest.mark.parametrize("case", WINDOWS, ids=lambda c: f"{c[1]}-{c[2]}x{c[3]}-{str(c[5])[6:]}-{str(c[6])[6:]}-w{c[7]}")
def test_window_decode_matches_float64(case):
    lens, hq, hkv, d, group, dtype, values, window, sinks = case
    pools = make_cache(lens, hkv, d, group, values, seed=d + hq)
    q = (torch.randn((len(lens), hq, d), generator=pools[-1], device="cuda") / d ** 0.5).to(dtype)
    out = C.paged_window_decode(q, *pools[:5], window=window, sinks=sinks, group_tokens=group)
    want = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        k, v = tokens64(pools, b, 0, n, group)
        pos = torch.arange(n, device="cuda")
        sees = (pos >= n - window) | (pos < sinks)
        if sees.any():
            x = torch.einsum("hgd,jhd->hgj", q[b].double().view(hkv, -1, d), k[sees])
            want[b] = torch.einsum("hgj,jhd->hgd", torch.softmax(x, -1), v[sees]).reshape(-1, d)
    close(out, want, dtype)
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all()


def test_window_beyond_the_cache_equals_the_plain_decode():
    pools = make_cache([700, 2048], 4, 128, 128, F32)
    q = torch.randn((2, 8, 128), generator=pools[-1], device="cuda") / 11
    a = C.paged_window_decode(q, *pools[:5], window=4096)
    b = C.paged_decode(q, *pools[:5])
    assert (a - b).abs().max().item() < 1e-5


def bulk(cache_args, keys, vals, group, values):
    cache = P.PagedKVCache(*cache_args, group_tokens=group, device="cuda", seed=5, value_dtype=values)
    cache.write_sequences(list(range(len(keys))), keys, vals)
    return cache


def logical(cache, s):
    n, group = cache.lens[s], cache.group_tokens
    pages = cache.pages[s]
    if n == 0:
        return None
    k = torch.cat([cache.k_pool[p] for p in pages], 1)[:, :n]
    v = torch.cat([cache.v_pool[p] for p in pages], 1)[:, :n]
    gp = group // 16
    sz = torch.stack([cache.sz_pool[pages[i * gp]] for i in range((n + group - 1) // group)])
    return k, v, sz


@pytest.mark.parametrize("dtype,values", [(F32, F32), (F32, F16), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("group", [128, 32, 16])
def test_extend_equals_bulk_write(group, dtype, values):
    heads, d = 3, 64
    rng = np.random.default_rng(group)
    start = [0, 5, group, group - 1, 3 * group + 7, 40, 0]
    new = [1, 3, 1, 2, 5 * group, 0, 2 * group]
    g = torch.Generator(device="cuda").manual_seed(1)
    keys = [(torch.randn((a + b, heads, d), generator=g, device="cuda") * 3 + 1).to(dtype).float()
            for a, b in zip(start, new)]
    vals = [torch.randn((a + b, heads, d), generator=g, device="cuda").to(dtype).float()
            for a, b in zip(start, new)]
    want = bulk((400, heads, d), keys, vals, group, values)
    cache = P.PagedKVCache(400, heads, d, group_tokens=group, device="cuda", seed=2, value_dtype=values)
    ids = list(range(len(start)))
    cache.write_sequences(ids, [k[:n] for k, n in zip(keys, start)], [v[:n] for v, n in zip(vals, start)])
    # the new rows come out of a larger set, in the order of `rows`
    total = sum(new)
    perm = rng.permutation(2 * total)[:total].astype(np.int32)
    src_k = torch.full((2 * total, heads, d), 7.0, device="cuda", dtype=dtype)
    src_v = torch.full((2 * total, heads, d), 7.0, device="cuda", dtype=dtype)
    src_k[torch.from_numpy(perm).long().cuda()] = torch.cat([k[n:] for k, n in zip(keys, start)]).to(dtype)
    src_v[torch.from_numpy(perm).long().cuda()] = torch.cat([v[n:] for v, n in zip(vals, start)]).to(dtype)
    cache.extend(ids, new, src_k, src_v, rows=torch.from_numpy(perm).cuda())
    for s in ids:
        assert cache.lens[s] == start[s] + new[s]
        if cache.lens[s]:
            for x, y in zip(logical(cache, s), logical(want, s)):
                assert torch.equal(x, y)
    # the staged rows are those of the open groups: appends go on from there
    one_k = torch.randn((len(ids), heads, d), generator=g, device="cuda")
    one_v = torch.randn((len(ids), heads, d), generator=g, device="cuda")
    cache.append(ids, one_k, one_v)
    want.append(ids, one_k, one_v)
    for s in ids:
        for x, y in zip(logical(cache, s), logical(want, s)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("d,group", [(64, 128), (128, 32), (256, 128), (12, 16), (96, 64)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("values", [F32, F16, BF16])
def test_read_back(d, group, dtype, values):
    lens = [0, 1, 16, 33, 300]
    pools = make_cache(lens, 3, d, group, values, seed=d)
    start, count = [0, 0, 3, 17, 100], [0, 1, 13, 16, 199]
    offs = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    total = int(offs[-1]) + 2  # two rows that no sequence covers
    k_out = torch.full((total, 3, d), 5.0, dtype=dtype, device="cuda")
    v_out = torch.full((total, 3, d), 5.0, dtype=dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    C.cache_read(*pools[:4], torch.tensor(start, dtype=torch.int32, device="cuda"),
                 torch.from_numpy(offs).cuda(), num_rows=total, max_rows_per_seq=199,
                 group_tokens=group, dtype=dtype, k_out=k_out, v_out=v_out, status=status)
    assert status.item() == 0
    assert (k_out[-2:] == 5).all() and (v_out[-2:] == 5).all()
    for b in range(len(lens)):
        if count[b]:
            k, v = tokens64(pools, b, start[b], start[b] + count[b], group)
            mine = slice(offs[b], offs[b + 1])
            # two float32 roundings (the product zp s, then the sum) and the output's
            row = pools[3][b].long()
            pos = torch.arange(start[b], start[b] + count[b], device="cuda")
            sz = pools[2][row[pos // group * (group // 16)]].double()
            slack = 2.0 ** -23 * (sz[:, :, 0] * (sz[:, :, 1].abs() + 15))
            half = torch.finfo(dtype).eps / 2
            assert ((k_out[mine].double() - k).abs() <= half * 1.001 * k.abs() + slack + 2.0 ** -24).all()
            assert torch.equal(v_out[mine], v.to(values).to(dtype))
