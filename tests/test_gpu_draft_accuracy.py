"""Draft attention against float64, each row measured by the roundings that it may have
(draft_error.py): a lost tile or record of a long stream, whose outputs are small, shows.
"""

import numpy as np
import pytest

import draft_error
from helpers import pkg
from test_gpu_draft_steps import Step
from test_gpu_drafts import BF16, F16, F32, make_cache, tokens64

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
C = pkg("_C")
P = pkg("paged")


def steps_of(pools, b, n, group):
    """The quantisation step of each cached key, [n, H, D]."""
    pos = torch.arange(n, device="cuda")
    return pools[2][pools[3][b].long()[pos // group * (group // 16)]][:, :, 0].double()


def worst(out, q, pools, group, sequences, dtype, window=0, sinks=0):
    """Largest excess over the rows of all sequences: (first row, cached tokens, drafted keys, values
    and words, or None for a window's one row each)."""
    top = 0.0
    for b, (row0, n, drafts) in enumerate(sequences):
        kc, vc = tokens64(pools, b, 0, n, group)
        st = steps_of(pools, b, n, group)
        pos = torch.arange(n, device="cuda")
        if drafts is None:
            t, at = 1, torch.tensor([n - 1], device="cuda")
            k, v, tree = kc, vc, torch.zeros((1, 0), dtype=torch.bool, device="cuda")
            where = pos
        else:
            kd, vd, words = drafts
            t = len(words)
            bits = [[int(w) % (1 << 64) >> u & 1 for u in range(t)] for w in words]
            tree = torch.tensor(bits, dtype=torch.bool, device="cuda").view(t, t)
            depth = torch.tensor([sum(r) - r[i] for i, r in enumerate(bits)], device="cuda", dtype=torch.long)
            at, where = n + depth, torch.cat([pos, n + depth])
            k, v = torch.cat([kc, kd.double()]), torch.cat([vc, vd.double()])
            st = torch.cat([st, torch.zeros_like(kd, dtype=torch.float64)])
        seen = torch.cat([torch.ones((t, n), dtype=torch.bool, device="cuda"), tree], 1)
        if window:
            seen &= (where[None] > at[:, None] - window) | (where[None] < sinks)
        if not t or not k.shape[0]:
            continue
        h = k.shape[1]
        want, rms = draft_error.expected(q[row0:row0 + t].double().view(t, h, -1, k.shape[2]), k, v, st,
                                         torch.arange(k.shape[0], device="cuda") < n, seen, dtype)
        top = max(top, draft_error.excess(out[row0:row0 + t].view(want.shape), want, rms))
    return top


def tree_worst(s, out, dtype, window=0, sinks=0):
    seqs = []
    for b, n in enumerate(s.lens):
        lo, hi = int(s.offs[b]), int(s.offs[b + 1])
        seqs.append((lo, n, (s.k[lo:hi], s.v[lo:hi], s.words[lo:hi])))
    return worst(out, s.q, s.pools, s.group, seqs, dtype, window, sinks)


RNG = np.random.default_rng(4)
RAGGED = [int(x) for x in RNG.integers(0, 6000, 20)]
COUNTS = [int(x) for x in RNG.integers(0, 33, 20)]

SHAPES = [
    # lens, counts, q heads, kv heads, head_dim, group
    (RAGGED, COUNTS, 32, 8, 128, 128),
    ([6000, 5000, 20, 0, 3001], [9, 64, 64, 3, 1], 8, 8, 128, 128),
    ([4001, 257, 1000, 2500], [33, 33, 20, 5], 28, 4, 64, 64),
    ([3000, 129, 511], [30, 7, 16], 16, 2, 256, 32),
    ([8192] * 3, [16] * 3, 16, 4, 128, 128),
    ([5999], [1], 4, 4, 128, 128),
    ([333] * 60, [4] * 60, 8, 2, 128, 16),
    ([7000, 100], [64, 64], 32, 4, 128, 128),
]


@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 20)])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{len(s[0])}x{max(s[0])}-{s[2]}-{s[3]}x{s[4]}")
@pytest.mark.parametrize("dtype,values", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16)])
def test_tree_rows(dtype, values, shape, window, sinks):
    lens, counts, hq, hkv, d, group = shape
    s = Step(lens, counts, hq, hkv, d, group, dtype, values, seed=d + len(lens))
    out = s.run(window=window or None, sinks=sinks)
    assert tree_worst(s, out, dtype, window, sinks) < 1
    s.q *= 3  # few tokens carry the weight
    assert tree_worst(s, s.run(window=window or None, sinks=sinks), dtype, window, sinks) < 1


@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 4), (2000, 70), (100000, 0)])
@pytest.mark.parametrize("hq,hkv,d,group", [(32, 8, 128, 128), (8, 8, 64, 64), (16, 1, 256, 32)])
@pytest.mark.parametrize("dtype,values", [(F32, F32), (F32, F16), (BF16, BF16), (F16, F16)])
def test_window_rows(dtype, values, hq, hkv, d, group, window, sinks):
    lens = [5000, 1, 17, 2048, 128, 4097, 999, 0]
    pools = make_cache(lens, hkv, d, group, values, seed=d)
    q = (torch.randn((len(lens), hq, d), generator=pools[-1], device="cuda") / d ** 0.5).to(dtype)
    out = C.paged_window_decode(q, *pools[:5], window=window, sinks=sinks, group_tokens=group)
    assert worst(out, q, pools, group, [(b, n, None) for b, n in enumerate(lens)], dtype, window, sinks) < 1


@pytest.mark.parametrize("values", [F32, F16, BF16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 6)])
def test_a_server_s_verified_rows(values, window, sinks):
    """Draft, verify, accept through PagedKVCache: the rows of ``tree_decode`` with the block table,
    offsets and masks that the cache makes, at every step."""
    heads, hq, d, group = 2, 8, 128, 32
    g = torch.Generator(device="cuda").manual_seed(3)
    rng = np.random.default_rng(9)
    cache = P.PagedKVCache(200, heads, d, group_tokens=group, device="cuda", seed=1, value_dtype=values)
    ids, lens = [7, 3, 11, 5], [130, 0, 61, 700]
    data = [[(torch.randn((n, heads, d), generator=g, device="cuda")).to(values).float() for n in lens] for _ in range(2)]
    cache.write_sequences(ids, *data)
    for step in range(4):
        counts = [int(rng.integers(0, 20)) for _ in ids]
        parents = [[int(rng.integers(-1, i)) if i else -1 for i in range(n)] for n in counts]
        rows = sum(counts) + 3  # padded
        q = (torch.randn((rows, hq, d), generator=g, device="cuda") / d ** 0.5).to(values)
        k, v = (torch.randn((rows, heads, d), generator=g, device="cuda").to(values) for _ in range(2))
        words = P.tree_mask(parents)
        mask = torch.cat([words, words.new_zeros(3)])
        out = cache.tree_decode(q, k, v, ids, counts, mask, window=window, sinks=sinks)
        pools = (cache.k_pool, cache.v_pool, cache.sz_pool, cache.block_table(ids)[0])
        offs = np.concatenate([[0], np.cumsum(counts)]).astype(int)
        seqs = [(offs[b], cache.lens[s], (k[offs[b]:offs[b + 1]], v[offs[b]:offs[b + 1]], words[offs[b]:offs[b + 1]].tolist()))
                for b, s in enumerate(ids)]
        assert worst(out, q, pools, group, seqs, values, window or 0, sinks) < 1
        assert (out[sum(counts):] == 0).all()
        # the path to one draft of each tree is accepted
        picked, lengths = [], []
        for b, par in enumerate(parents):
            path, t = [], int(rng.integers(0, len(par))) if par else -1
            while t >= 0:
                path.insert(0, int(offs[b]) + t)
                t = par[t]
            picked += path
            lengths.append(len(path))
        cache.extend(ids, lengths, k, v, rows=torch.tensor(picked, dtype=torch.int32))
        cache.check()
