"""The draft operators as a server uses them, and where they can go wrong: rows
that see nothing, what stands in hidden places, malformed metadata, offsets past
32 bits, many sequences, magnitudes beyond float16, captured graphs, side
streams, and whole speculative steps.

Comparisons with float64 and their tolerances are those of test_gpu_drafts.py
(derived there); everything else is exact.
"""

import numpy as np
import pytest

from helpers import pkg
from test_gpu_drafts import (BF16, F16, F32, close, logical, make_cache, random_trees, tokens64, tree64)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
C = pkg("_C")
P = pkg("paged")

BAD_PAGE, BAD_LENGTH = 1, 2
NAN, INF = float("nan"), float("inf")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Step:
    """A batch of drafted trees over a cache of random codes."""

    def __init__(self, lens, counts, hq, hkv, d, group, dtype, values, seed=0, extra=0, chains=0.5):
        self.pools = make_cache(lens, hkv, d, group, values, seed=seed)
        self.group, self.dtype, self.lens, self.counts = group, dtype, lens, counts
        g = self.pools[-1]
        rows = sum(counts) + extra
        self.q = (torch.randn((rows, hq, d), generator=g, device="cuda") / d ** 0.5).to(dtype)
        self.k = torch.randn((rows, hkv, d), generator=g, device="cuda").to(dtype)
        self.v = torch.randn((rows, hkv, d), generator=g, device="cuda").to(dtype)
        words = np.zeros(rows, np.int64)
        words[:sum(counts)] = random_trees(counts, seed, chains)
        self.words = words
        self.offs = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)

    def run(self, **kw):
        a = dict(max_drafts=max(self.counts), group_tokens=self.group)
        a.update(kw)
        words = a.pop("words", self.words)
        offs = a.pop("offs", torch.from_numpy(self.offs).cuda())
        pools = a.pop("pools", self.pools[:4])
        sl = a.pop("seq_lens", self.pools[4])
        return C.paged_tree_decode(self.q, self.k, self.v, torch.from_numpy(words).cuda(), offs, *pools, sl, **a)

    def want(self, window=0, sinks=0, words=None):
        return tree64(self.q, self.k, self.v, self.words if words is None else words, self.offs, self.pools,
                      self.group, window, sinks)


KINDS = [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16)]


@pytest.mark.parametrize("dtype,values", KINDS)
def test_rows_that_see_nothing(dtype, values):
    s = Step([0, 70, 0], [5, 4, 64], 8, 2, 128, 128, dtype, values)
    words = s.words.copy()
    words[[0, 3]] = 0            # nothing at all: an empty cache and no draft
    words[5] = 0                 # the cache alone
    words[9] = 0
    words[10] = 1 << 62          # one late draft alone
    out = s.run(words=words)
    close(out, s.want(words=words), dtype)
    assert (out[[0, 3, 9]] == 0).all()
    # a window that shuts even the draft itself out of nothing: position p sees p
    lens0 = C.paged_window_decode(s.q[:3].contiguous(), *s.pools[:4], i32([0, 70, 0]), window=1, group_tokens=128)
    assert (lens0[[0, 2]] == 0).all() and torch.isfinite(lens0).all() and (lens0[1] != 0).any()


@pytest.mark.parametrize("dtype,values", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_hidden_places_do_not_matter(dtype, values, d):
    lens, counts = [37, 300, 0, 129], [6, 17, 3, 20]
    s = Step(lens, counts, 4, 2, d, 64, dtype, values, extra=30)
    hide = {0: 4, 1: 9, 3: 19}   # (sequence, draft) nobody sees, not even itself
    words = s.words.copy()
    for b, t in hide.items():
        o = s.offs[b]
        words[o:o + counts[b]] &= ~(1 << t)
    clean = s.run(words=words)
    close(clean[:sum(counts)], s.want(words=words)[:sum(counts)], dtype)
    for bad in (NAN, INF, torch.finfo(dtype).min):
        for b, t in hide.items():
            s.k[s.offs[b] + t] = bad if bad != INF else NAN
            s.v[s.offs[b] + t] = bad
        s.k[sum(counts):] = bad      # rows past the last sequence
        s.v[sum(counts):] = bad
        k_pool, v_pool, sz, bt, sl, _ = s.pools
        v2 = v_pool.clone()
        for b, n in enumerate(lens):
            if n % 16:
                v2[bt[b, n // 16].long(), :, n % 16:] = bad
        used = {int(p) for b, n in enumerate(lens) for p in bt[b, :(n + 15) // 16]}
        for p in range(k_pool.shape[0]):
            if p not in used:
                v2[p] = bad
                sz[p] = NAN
        out = s.run(words=words, pools=(k_pool, v2, sz, bt))
        assert torch.equal(out[:sum(counts)], clean[:sum(counts)]), bad


@pytest.mark.parametrize("dtype,values", KINDS)
def test_infinite_and_nan_drafts_reach_only_their_rows(dtype, values):
    """A drafted value that is not finite belongs to the rows that see its draft."""
    s = Step([200, 5], [40, 9], 8, 2, 128, 128, dtype, values)
    clean = s.run()
    for t, bad in ((7, NAN), (21, INF), (40, -INF)):
        s.v[t, 1, 5] = bad
    out = s.run()
    for row in range(49):
        o = 0 if row < 40 else 40
        seen = [u for u in (7, 21, 40) if o <= u < o + (40 if o == 0 else 9) and int(s.words[row]) >> (u - o) & 1]
        if not seen:
            assert torch.equal(out[row], clean[row])
            continue
        hit = out[row, 4:8, 5]      # the q heads of kv head 1
        want = {7: NAN, 21: INF, 40: -INF}
        expect = sum(want[u] for u in seen)
        assert torch.equal(torch.isnan(hit), torch.full_like(hit, expect != expect, dtype=torch.bool))
        if expect == expect:
            assert (hit == expect).all()
        rest = torch.ones(out.shape[1:], dtype=torch.bool, device="cuda")
        rest[4:8, 5] = False
        assert torch.equal(out[row][rest], clean[row][rest])


@pytest.mark.parametrize("dtype,values", [(F32, F32), (BF16, BF16), (F16, F16)])
def test_window_hides_what_it_must(dtype, values):
    lens = [1000, 77, 16, 333]
    pools = make_cache(lens, 2, 128, 32, values, seed=5)
    q = (torch.randn((4, 8, 128), generator=pools[-1], device="cuda") / 11.3).to(dtype)
    clean = C.paged_window_decode(q, *pools[:5], window=100, sinks=20, group_tokens=32)
    k_pool, v_pool, sz, bt, sl, _ = pools
    for b, n in enumerate(lens):
        for t in range(n):
            if t >= 20 and t <= n - 1 - 100:
                v_pool[bt[b, t // 16].long(), :, t % 16] = NAN
        for first in range(0, n, 32):  # whole groups of scales nobody sees
            if first >= 32 and first + 32 <= n - 100:
                sz[bt[b, first // 16].long()] = NAN
    assert torch.equal(C.paged_window_decode(q, *pools[:5], window=100, sinks=20, group_tokens=32), clean)


@pytest.mark.parametrize("dtype,values", KINDS)
def test_rows_past_the_last_sequence_stay(dtype, values):
    s = Step([20, 0, 300], [3, 0, 9], 4, 2, 64, 128, dtype, values, extra=5)
    out = torch.full_like(s.q, 7.0)
    status = i32([0])
    s.run(out=out, status=status)
    assert (out[12:] == 7).all() and status.item() == 0
    close(out[:12], s.want()[:12], dtype)


@pytest.mark.parametrize("dtype,values", KINDS)
def test_bad_pages_and_lengths_are_reported(dtype, values):
    s = Step([200, 64, 90], [3, 5, 2], 4, 2, 128, 64, dtype, values)
    clean = s.run()
    k_pool, v_pool, sz, bt, sl, _ = s.pools
    status = i32([0])
    bad = bt.clone()
    bad[0, 2], bad[0, 9] = -1, k_pool.shape[0]
    out = s.run(pools=(k_pool, v_pool, sz, bad), status=status)
    assert status.item() == BAD_PAGE
    assert torch.equal(out[3:], clean[3:]) and torch.isfinite(out).all()
    # the same tokens, as if they were not there: the float64 form without pages 2 and 9
    keep = torch.cat([torch.arange(0, 32), torch.arange(48, 144), torch.arange(160, 200)]).cuda()
    kc, vc = tokens64((k_pool, v_pool, sz, bt), 0, 0, 200, 64)
    # (a page that is bad where its group's scales live hides its whole group: neither does here)
    for i in range(3):
        seen = [j for j in range(3) if int(s.words[i]) >> j & 1]
        k = torch.cat([kc[keep], s.k[:3][seen].double()])
        v = torch.cat([vc[keep], s.v[:3][seen].double()])
        x = torch.einsum("hgd,jhd->hgj", s.q[i].double().view(2, -1, 128), k)
        want = torch.einsum("hgj,jhd->hgd", torch.softmax(x, -1), v).reshape(-1, 128)
        close(out[i], want, dtype)
    # lengths: negative counts as empty, too long as the whole table
    status.zero_()
    out = s.run(seq_lens=i32([200, -5, 90]), status=status)
    assert status.item() == BAD_LENGTH
    assert torch.equal(out[:3], clean[:3]) and torch.equal(out[8:], clean[8:])
    status.zero_()
    s.run(seq_lens=i32([200, 64, 1 << 30]), status=status)
    assert status.item() & BAD_LENGTH
    # offsets: past the rows, decreasing, more drafts than promised
    for offs, spoilt in (([0, 3, 8, 11], 2), ([0, 3, 2, 10], 1), ([-1, 3, 8, 10], 0)):
        status.zero_()
        mark = torch.full_like(s.q, 7.0)
        s.run(offs=i32(offs), out=mark, status=status)
        assert status.item() & BAD_LENGTH
        if spoilt:
            assert torch.equal(mark[:3], clean[:3])
    status.zero_()
    mark = torch.full_like(s.q, 7.0)
    s.run(max_drafts=4, out=mark, status=status)
    assert status.item() == BAD_LENGTH
    assert (mark[3:8] == 7).all()
    close(mark[:3], s.want()[:3], dtype)
    status.zero_()
    one = C.paged_window_decode(s.q[:3].contiguous(), k_pool, v_pool, sz, bad, sl, window=1000, group_tokens=64, status=status)
    assert status.item() == BAD_PAGE and torch.isfinite(one).all()


@pytest.mark.parametrize("dtype,values", [(F32, F32), (BF16, BF16), (F16, F16)])
def test_many_sequences(dtype, values):
    """More sequences than a warp has lanes, most of them short, some taking no part."""
    rng = np.random.default_rng(11)
    n = 150
    lens = [int(x) for x in rng.choice([0, 1, 15, 16, 17, 100, 127, 128, 129, 400], n)]
    counts = [int(x) for x in rng.choice([0, 0, 1, 2, 3, 8], n)]
    s = Step(lens, counts, 4, 2, 64, 16, dtype, values, seed=3)
    close(s.run(), s.want(), dtype)
    out = C.paged_window_decode((torch.randn((n, 4, 64), generator=s.pools[-1], device="cuda") / 8).to(dtype),
                                *s.pools[:5], window=40, sinks=3, group_tokens=16)
    assert torch.isfinite(out).all()
    empty = torch.tensor([x == 0 for x in lens], device="cuda")
    assert (out[empty] == 0).all()


@pytest.mark.parametrize("hq,hkv,d,dtype", [(32, 8, 128, BF16), (32, 8, 128, F32), (32, 8, 64, F16), (16, 4, 256, BF16),
                                            (16, 4, 256, F32), (16, 16, 128, F16)])
@pytest.mark.parametrize("tokens,drafts", [(20, 31), (148, 31), (148, 4), (256, 9), (257, 16), (390, 32), (0, 12)])
def test_many_short_streams(hq, hkv, d, dtype, tokens, drafts):
    """Several streams a CTA, each of a few tiles: one's queries, values and sums replace another's."""
    s = Step([tokens] * 40, [drafts] * 40, hq, hkv, d, 128, dtype, dtype, seed=tokens)
    first = s.run()
    close(first, s.want(), dtype)
    for _ in range(3):
        assert torch.equal(s.run(), first)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(32, 8, 128, BF16), (8, 8, 64, F16), (16, 4, 256, BF16), (8, 2, 128, F32)])
def test_logits_that_rise_late(hq, hkv, d, dtype):
    """The largest logits in a stream's last tile: every sum and output before it shrinks."""
    s = Step([300] * 30 + [100, 129], [20] * 32, hq, hkv, d, 128, dtype, dtype, seed=2)
    s.k *= 8
    first = s.run()
    close(first, s.want(), dtype)
    for _ in range(3):
        assert torch.equal(s.run(), first)


@pytest.mark.parametrize("batch,tokens", [(1, 300), (40, 300), (6, 2500)])
@pytest.mark.parametrize("hq,hkv,d,drafts", [(32, 4, 128, 40), (28, 4, 64, 33), (16, 2, 256, 30)])
def test_rows_in_chunks(batch, tokens, hq, hkv, d, drafts):
    """More rows a kv head than a chunk holds, with little and with much to do a CTA."""
    s = Step([tokens] * batch, [drafts] * batch, hq, hkv, d, 64, BF16, BF16, seed=batch)
    close(s.run(), s.want(), BF16)
    close(s.run(window=200, sinks=10), s.want(200, 10), BF16)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_ragged_batch(dtype):
    rng = np.random.default_rng(0)
    s = Step([int(x) for x in rng.integers(0, 6000, 24)], [int(x) for x in rng.integers(0, 33, 24)], 32, 8, 128, 128,
             dtype, dtype, seed=6)
    close(s.run(), s.want(), dtype)
    q = s.q[:24].contiguous()
    out = C.paged_window_decode(q, *s.pools[:5], window=2000, sinks=20, group_tokens=128)
    for b, n in enumerate(s.lens):
        k, v = tokens64(s.pools, b, 0, n, 128)
        pos = torch.arange(n, device="cuda")
        sees = (pos > n - 1 - 2000) | (pos < 20)
        x = torch.einsum("hgd,jhd->hgj", q[b].double().view(8, 4, 128), k[sees])
        want = torch.einsum("hgj,jhd->hgd", torch.softmax(x, -1), v[sees]).reshape(-1, 128)
        close(out[b], want, dtype)


@pytest.mark.parametrize("group", [16, 48, 256, 4096])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_sizes(group, dtype):
    s = Step([1000, 47, 300], [4, 5, 6], 8, 4, 128, group, dtype, dtype, seed=group)
    close(s.run(), s.want(), dtype)
    close(s.run(window=77, sinks=50), s.want(77, 50), dtype)


@pytest.mark.parametrize("what", ["queries", "cached", "drafted", "mixed", "rows", "in range"])
def test_magnitudes_beyond_float16(what):
    """bfloat16 reaches further than the float16 the tensor cores multiply: powers of two come in."""
    s = Step([300, 50], [20, 6], 8, 2, 128, 64, BF16, BF16, seed=8)
    big = 2.0 ** 20
    k_pool, v_pool, sz, bt, sl, _ = s.pools
    if what == "queries":
        s.q *= big
        s.k /= big
        sz[:, :, 0] /= big
    elif what == "cached":
        s.q /= big
        sz[:, :, 0] *= big
    elif what == "drafted":
        s.q /= big
        s.k *= big
    elif what == "rows":  # rows of very different size side by side, some zero
        s.q[::2] /= 2.0 ** 30
        s.q[1::4] *= 4
        s.q[3] = 0
        sz[:, :, 0] *= 2
    elif what == "in range":  # large keys of small queries, none of them scaled
        s.q /= 2.0 ** 6
        s.k *= 2.0 ** 6
        sz[:, :, 0] *= 2.0 ** 6
    else:  # every second group and every third draft
        s.q /= big
        sz[::2, :, 0] *= big
        s.k[::3] *= big
    out = s.run()
    close(out, s.want(), BF16)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements, the sequence's pages at its far end."""
    pages, heads, d = 270000, 8, 128
    assert pages * heads * 16 * d > 2 ** 32
    g = torch.Generator(device="cuda").manual_seed(0)
    lens, used = [100, 33], 10
    small = make_cache(lens, heads, d, 64, BF16, seed=1, spare=used - 10)
    k_pool = torch.empty((pages, heads, 16, d // 2), dtype=torch.uint8, device="cuda")
    v_pool = torch.empty((pages, heads, 16, d), dtype=BF16, device="cuda")
    sz = torch.empty((pages, heads, 2, d), device="cuda")
    shift = pages - small[0].shape[0]
    k_pool[shift:], v_pool[shift:], sz[shift:] = small[0], small[1], small[2]
    bt = small[3] + shift
    rows = 7
    q = (torch.randn((rows, 16, d), generator=g, device="cuda") / 11.3).to(BF16)
    k = torch.randn((rows, heads, d), generator=g, device="cuda").to(BF16)
    v = torch.randn((rows, heads, d), generator=g, device="cuda").to(BF16)
    words = torch.from_numpy(random_trees([4, 3], 2)).cuda()
    offs = i32([0, 4, 7])
    for cast in (BF16, F32):
        a = C.paged_tree_decode(q.to(cast), k.to(cast), v.to(cast), words, offs, k_pool, v_pool, sz, bt, small[4], 4, 64)
        b = C.paged_tree_decode(q.to(cast), k.to(cast), v.to(cast), words, offs, *small[:5], 4, 64)
        assert torch.equal(a, b)
        a = C.paged_window_decode(q[:2].to(cast), k_pool, v_pool, sz, bt, small[4], 50, 2, 64)
        b = C.paged_window_decode(q[:2].to(cast), *small[:5], 50, 2, 64)
        assert torch.equal(a, b)
    ka, va = C.cache_read(k_pool, v_pool, sz, bt, i32([0, 0]), i32([0, 100, 133]), 133, 100, 64)
    kb, vb = C.cache_read(*small[:4], i32([0, 0]), i32([0, 100, 133]), 133, 100, 64)
    assert torch.equal(ka, kb) and torch.equal(va, vb)
    stage = torch.zeros((2, 64, heads * d), device="cuda")
    for kp, vp, zp, table in ((k_pool, v_pool, sz, bt), small[:4]):
        stage.zero_()
        C.cache_extend(k, v, offs, i32([64, 0]), i32([0, 1]), stage, table, kp, vp, zp, 4, 64)
    ka, va = C.cache_read(k_pool, v_pool, sz, bt, i32([64, 0]), offs, 7, 4, 64)
    kb, vb = C.cache_read(*small[:4], i32([64, 0]), offs, 7, 4, 64)
    assert torch.equal(ka, kb) and torch.equal(va, vb)
    assert torch.equal(va.to(BF16), v)


@pytest.mark.parametrize("dtype,values", [(F32, F32), (BF16, BF16)])
def test_equal_calls_give_equal_bits(dtype, values):
    s = Step([3000, 1, 777], [16, 5, 33], 32, 8, 128, 128, dtype, values)
    first = s.run()
    for _ in range(3):
        assert torch.equal(s.run(), first)


@pytest.mark.parametrize("dtype,values", [(F32, F32), (BF16, BF16)])
def test_side_streams_with_their_own_workspaces(dtype, values):
    """Two calls at once on two streams, and inputs made on the stream that uses them."""
    a = Step([2000, 30], [16, 5], 16, 4, 128, 128, dtype, values, seed=1)
    b = Step([900, 1500], [7, 31], 16, 4, 128, 128, dtype, values, seed=2)
    want = [a.run(), b.run()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [None, None]
    for _ in range(4):
        for i, (s, st) in enumerate(zip((a, b), streams)):
            with torch.cuda.stream(st):
                outs[i] = s.run()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs, want))


@pytest.mark.parametrize("dtype,values", [(F32, F32), (BF16, BF16)])
def test_captured_step_follows_its_inputs(dtype, values):
    """Two graphs (tree + extend + read, window) replayed after their inputs changed in place."""
    lens, counts = [500, 40, 129], [6, 3, 12]
    s = Step(lens, counts, 8, 2, 128, 64, dtype, values, seed=4)
    k_pool, v_pool, sz, bt, sl, g = s.pools
    words, offs = torch.from_numpy(s.words).cuda(), torch.from_numpy(s.offs).cuda()
    need = C.paged_attention_workspace_bytes(3, 8, 2, 128, 12)
    ws = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
    out, win = torch.zeros_like(s.q), torch.zeros_like(s.q[:3])
    qw = s.q[:3].clone()

    def tree():
        C.paged_tree_decode(s.q, s.k, s.v, words, offs, k_pool, v_pool, sz, bt, sl, 12, 64, out=out, workspace=ws[0])

    def window():
        C.paged_window_decode(qw, k_pool, v_pool, sz, bt, sl, 100, 4, 64, out=win, workspace=ws[1])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tree(), window()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for f in (tree, window):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            f()
        graphs.append(graph)
    for turn in range(3):
        s.q.copy_((torch.randn(s.q.shape, generator=g, device="cuda") / 11.3).to(dtype))
        qw.copy_(s.q[:3])
        sl.copy_(i32([500 - 130 * turn, 40, turn]))
        out.fill_(9), win.fill_(9)
        for graph in graphs[::-1] if turn % 2 else graphs:
            graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), win.clone()
        tree(), window()
        assert torch.equal(out, got[0]) and torch.equal(win, got[1])
        close(out, s.want(), dtype)


@pytest.mark.parametrize("values", [F32, F16, BF16])
@pytest.mark.parametrize("group", [16, 128])
def test_speculative_steps_equal_a_bulk_cache(values, group):
    """Draft, verify, accept, again: the cache and the attention of a server's loop against a cache
    that is written in bulk, the verified rows against the plain decode after the path is accepted."""
    heads, hq, d = 2, 8, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    rng = np.random.default_rng(9)
    cache = P.PagedKVCache(200, heads, d, group_tokens=group, device="cuda", seed=1, value_dtype=values)
    ids, lens = [7, 3, 11], [130, 0, 61]
    keys = [torch.randn((n, heads, d), generator=g, device="cuda").to(values).float() for n in lens]
    vals = [torch.randn((n, heads, d), generator=g, device="cuda").to(values).float() for n in lens]
    cache.write_sequences(ids, keys, vals)
    for step in range(4):
        counts = [int(rng.integers(1, 20)) for _ in ids]
        parents = [[-1] + [int(rng.integers(-1, i)) for i in range(1, n)] for n in counts]
        rows = sum(counts)
        q = (torch.randn((rows, hq, d), generator=g, device="cuda") / d ** 0.5).to(values)
        k = torch.randn((rows, heads, d), generator=g, device="cuda").to(values)
        v = torch.randn((rows, heads, d), generator=g, device="cuda").to(values)
        out = cache.tree_decode(q, k, v, ids, counts, P.tree_mask(parents))
        # accept the path to one draft of each tree (of the second sequence, nothing)
        picked, path_len, leaf = [], [], []
        at = 0
        for i, (n, par) in enumerate(zip(counts, parents)):
            path, t = [], int(rng.integers(0, n))
            while t >= 0 and i != 1:
                path.insert(0, t)
                t = par[t]
            leaf.append(at + path[-1] if path else -1)
            picked += [at + t for t in path]
            path_len.append(len(path))
            keys[i] = torch.cat([keys[i], k[[at + t for t in path]].float()])
            vals[i] = torch.cat([vals[i], v[[at + t for t in path]].float()])
            at += n
        cache.extend(ids, path_len, k, v, rows=i32(picked))
        bulk = P.PagedKVCache(200, heads, d, group_tokens=group, device="cuda", seed=4, value_dtype=values)
        bulk.write_sequences(ids, keys, vals)
        for s in ids:
            assert cache.lens[s] == bulk.lens[s]
            if cache.lens[s]:
                for x, y in zip(logical(cache, s), logical(bulk, s)):
                    assert torch.equal(x, y)
                for x, y in zip(cache.read(s, dtype=values), bulk.read(s, dtype=values)):
                    assert torch.equal(x, y)
        # windows over the extended cache and over the bulk one
        one = (torch.randn((3, hq, d), generator=g, device="cuda") / d ** 0.5).to(values)
        assert torch.equal(cache.window_decode(one, ids, 50, 4), bulk.window_decode(one, ids, 50, 4))
        # a window wider than the cache is the plain decode
        plain = cache.decode(one.float(), ids)
        close(cache.window_decode(one, ids, 10000), plain.double(), values)
        # the accepted leaf's verified output: its own and its ancestors' keys were exact there and
        # are INT4 now, so only a tree without drafted keys of weight equals it; checked by shape here
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_same_row_taken_twice(dtype):
    """An input row may be the source of several tokens, of one sequence and of two."""
    heads, d = 2, 64
    k = torch.randn((3, heads, d), device="cuda").to(dtype)
    a = P.PagedKVCache(20, heads, d, group_tokens=32, device="cuda", value_dtype=F32)
    b = P.PagedKVCache(20, heads, d, group_tokens=32, device="cuda", value_dtype=F32)
    rows = [2, 2, 0, 1, 2]
    a.extend([0, 1], [3, 2], k, k, rows=i32(rows))
    b.extend([0, 1], [3, 2], k[rows], k[rows])
    for s in (0, 1):
        assert all(torch.equal(x, y) for x, y in zip(a.read(s), b.read(s)))


@pytest.mark.parametrize("bound", [3, 300])  # values written with the keys, and by blocks of their own
def test_extend_reports_malformed_metadata(bound):
    heads, d, group = 2, 64, 32
    k = torch.randn((6, heads, d), device="cuda")
    base = dict(offs=[0, 3, 6], start=[0, 0], slots=[0, 1], rows=None, table=[[0, 1], [2, 3]], max_rows=bound)

    def go(**kw):
        a = {**base, **kw}
        kp = torch.zeros((4, heads, 16, d // 2), dtype=torch.uint8, device="cuda")
        vp = torch.full((4, heads, 16, d), 5.0, device="cuda")
        sz = torch.full((4, heads, 2, d), 5.0, device="cuda")
        stage = torch.full((2, group, heads * d), 5.0, device="cuda")
        status = i32([0])
        C.cache_extend(k, k, i32(a["offs"]), i32(a["start"]), i32(a["slots"]), stage, i32(a["table"]), kp, vp, sz,
                       a["max_rows"], group, rows=i32(a["rows"]) if a["rows"] else None, status=status)
        return status.item(), kp, vp, sz, stage

    ok = go()
    assert ok[0] == 0
    # the second sequence is malformed: it is left alone, the first is written as ever
    for kw in (dict(offs=[0, 3, 2]), dict(offs=[0, 3, 7]), dict(start=[0, -1]), dict(start=[0, 30]), dict(slots=[0, 2]),
               dict(slots=[0, -1]), dict(start=[0, 2 ** 31 - 2])):
        st, kp, vp, sz, stage = go(**kw)
        assert st == BAD_LENGTH, kw
        assert torch.equal(vp[:2], ok[2][:2]) and (vp[2:] == 5).all() and (stage[1] == 5).all(), kw
        assert torch.equal(kp[:2], ok[1][:2]) and (kp[2:] == 0).all() and (sz[2:] == 5).all(), kw
    st, kp, vp, sz, stage = go(max_rows=2)
    assert st == BAD_LENGTH and (vp == 5).all()
    # rows outside the input write zeros
    st, kp, vp, sz, stage = go(rows=[0, 6, 2, -1, 4, 5])
    assert st == BAD_LENGTH
    assert (vp[0, :, 1] == 0).all() and (vp[2, :, 0] == 0).all() and torch.equal(vp[0, :, 2], k[2])
    # pages outside the pool are not written
    for page in (-1, 4):
        st, kp, vp, sz, stage = go(table=[[0, 1], [page, 3]])
        assert st == BAD_PAGE
        assert torch.equal(vp[:2], ok[2][:2]) and (vp[2:] == 5).all() and (sz[2:] == 5).all()


def test_read_reports_malformed_metadata():
    pools = make_cache([40, 40], 2, 64, 32, F32, seed=1)
    base = dict(start=[0, 0], offs=[0, 20, 40], table=pools[3], max_rows=20)

    def go(**kw):
        a = {**base, **kw}
        ko = torch.full((40, 2, 64), 7.0, device="cuda")
        vo, status = ko.clone(), i32([0])
        C.cache_read(*pools[:3], a["table"], i32(a["start"]), i32(a["offs"]), 40, a["max_rows"], 32, k_out=ko, v_out=vo,
                     status=status)
        return status.item(), ko, vo

    ok = go()
    assert ok[0] == 0
    for kw in (dict(offs=[0, 20, 41]), dict(offs=[0, 20, 10]), dict(start=[0, -1]), dict(start=[0, 2 ** 31 - 5]),
               dict(start=[0, 30])):
        st, ko, vo = go(**kw)
        assert st == BAD_LENGTH, kw
        assert torch.equal(ko[:20], ok[1][:20]) and (ko[20:] == 7).all() and (vo[20:] == 7).all(), kw
    bad = pools[3].clone()
    bad[1, 1] = 1 << 20
    st, ko, vo = go(table=bad)
    assert st == BAD_PAGE
    assert torch.equal(ko[:36], ok[1][:36]) and (ko[36:] == 0).all() and (vo[36:] == 0).all()


def test_binding_refusals():
    s = Step([20], [3], 4, 2, 64, 32, F32, F32)
    k_pool, v_pool, sz, bt, sl, _ = s.pools
    words, offs = torch.from_numpy(s.words).cuda(), i32([0, 3])

    def tree(**kw):
        a = dict(q=s.q, k=s.k, v=s.v, w=words, o=offs, kp=k_pool, vp=v_pool, sz=sz, bt=bt, sl=sl, n=3, g=32)
        rest = {x: kw.pop(x) for x in list(kw) if x not in a}
        a.update(kw)
        return C.paged_tree_decode(a["q"], a["k"], a["v"], a["w"], a["o"], a["kp"], a["vp"], a["sz"], a["bt"], a["sl"],
                                   a["n"], a["g"], **rest)

    tree()
    wide = torch.zeros(3 * 4 * 64 + 1, device="cuda")
    for kw in (dict(q=s.q.double()), dict(q=s.q.half()), dict(q=s.q[:, :3].contiguous()), dict(q=s.q.transpose(0, 1)),
               dict(q=s.q.cpu()), dict(q=wide[1:].view(3, 4, 64)), dict(k=s.k[:2]), dict(k=s.k.half()), dict(v=s.v[:, :1]),
               dict(w=words.int()), dict(w=words[:2]), dict(o=i32([0, 3, 3])), dict(o=offs.long()), dict(vp=None),
               dict(vp=v_pool[:1]), dict(sz=sz.half()), dict(bt=bt[:0]), dict(bt=bt.long()), dict(n=65), dict(n=-1),
               dict(g=24), dict(g=0), dict(window=0), dict(window=-2), dict(sinks=-1), dict(out=s.q), dict(out=s.q.half()),
               dict(out=torch.zeros((3, 4, 128), device="cuda")[:, :, ::2]),
               dict(workspace=torch.zeros(16, dtype=torch.uint8, device="cuda")), dict(status=torch.zeros(1))):
        with pytest.raises(RuntimeError):
            tree(**kw)
    with pytest.raises(RuntimeError):
        C.paged_window_decode(s.q[:1], k_pool, v_pool, sz, bt, sl, window=None)
    with pytest.raises(RuntimeError):
        C.paged_window_decode(s.q, k_pool, v_pool, sz, bt, sl, window=5)
    cache = P.PagedKVCache(8, 2, 64, group_tokens=32, device="cuda")
    cache.extend([1], [3], s.k, s.v)
    for bad in (lambda: cache.extend([1, 1], [1, 1], s.k, s.v), lambda: cache.extend([1], [1, 2], s.k, s.v),
                lambda: cache.extend([1], [-1], s.k, s.v), lambda: cache.extend([1], [4], s.k, s.v),
                lambda: cache.extend([1], [1], s.k[:, :1], s.v), lambda: cache.extend([1], [1], s.k, s.v[:1]),
                lambda: cache.read(1, 2, 9), lambda: cache.read(1, 3, 2),
                lambda: cache.tree_decode(s.q, s.k, s.v, [1], [4], words)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(MemoryError):
        big = torch.zeros((200, 2, 64), device="cuda")
        cache.extend([2], [200], big, big)
    assert cache.lens == {1: 3} or cache.lens == {1: 3, 2: 0}
