"""Cases that measure the cache operators of speculative and sliding-window serving.

Four operators over the paged INT4 key cache: attention for a tree of drafted
tokens (``tree``), single-token attention over a sliding window with sinks
(``window``), quantising several tokens per sequence as they are written
(``extend``, followed by reading the touched groups back), and reading a token
range back (``read``). ``run`` computes a case in plain tensor operations, or
through the package's entry points where ``own`` is set; ``exact`` evaluates the
same definition in 64 bits.
"""

import importlib
import math
import random

import numpy as np
import torch

own = False

PAGE = 16
PACKAGE = "int4-kv-cache-quantization-cuda-triton-pallas_b200"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------

def _tree(name, batch, q_heads, kv_heads, dim, ctx, drafts, ragged=False, dtype="bf16",
          values="bf16", window=0, sinks=0, group=128):
    return {"name": name, "op": "tree", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "ctx": ctx, "drafts": drafts, "ragged": ragged, "dtype": dtype,
            "values": values, "window": window, "sinks": sinks, "group": group}


def _window(name, batch, q_heads, kv_heads, dim, ctx, window, sinks, ragged=False, dtype="bf16",
            values="bf16", group=128):
    return {"name": name, "op": "window", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "ctx": ctx, "window": window, "sinks": sinks, "ragged": ragged,
            "dtype": dtype, "values": values, "group": group}


def _extend(name, batch, kv_heads, dim, ctx, new, ragged=False, picked=False, dtype="f32",
            values="f32", group=128):
    return {"name": name, "op": "extend", "batch": batch, "kv_heads": kv_heads, "dim": dim,
            "ctx": ctx, "new": new, "ragged": ragged, "picked": picked, "dtype": dtype,
            "values": values, "group": group}


def _read(name, batch, kv_heads, dim, ctx, count, ragged=False, dtype="bf16", values="bf16",
          group=128):
    return {"name": name, "op": "read", "batch": batch, "kv_heads": kv_heads, "dim": dim,
            "ctx": ctx, "count": count, "ragged": ragged, "dtype": dtype, "values": values,
            "group": group}


def listed():
    return [
        # one interactive user, a short conversation and eight drafted tokens: latency
        _tree("tree 1x777 8 drafts", 1, 32, 8, 128, 777, 8),
        # a usual serving batch with trees of different sizes (one sequence new, one without drafts)
        _tree("tree 8x2048 16 drafts", 8, 32, 8, 128, 2048, 16, ragged=True),
        # a full batch of long conversations and wide trees: the largest matrix work
        _tree("tree 32x8192 32 drafts", 32, 32, 8, 128, 8192, 32),
        # float32 multi-head models of the decode benchmark's shape, verified four drafts at a time
        _tree("tree f32 8x2048 4 drafts", 8, 32, 32, 128, 2048, 4, dtype="f32", values="f32"),
        # a sliding-window layer of a small-head model, odd lengths and short groups
        _tree("tree f16 window 5x4001 33", 5, 28, 4, 64, 4001, 33, ragged=True, dtype="f16",
              values="f16", window=1024, sinks=4, group=64),
        # one user's next token on a sliding-window layer: latency
        _window("window 1x4096", 1, 32, 8, 128, 4096, 1024, 4),
        # a batch of long conversations of a grouped-query model
        _window("window 64x8192", 64, 32, 8, 128, 8192, 4096, 64, ragged=True),
        # float32 multi-head model of the decode benchmark's shape behind a window
        _window("window f32 32x4096", 32, 32, 32, 128, 4096, 2000, 4, dtype="f32", values="f32"),
        # the accepted paths of a batch's trees, picked out of the drafted rows
        _extend("extend 64x8 accepted", 64, 8, 128, 2048, 8, ragged=True, picked=True, dtype="bf16",
                values="bf16"),
        # the next chunk of long prompts
        _extend("extend 8x1000 chunk", 8, 32, 128, 1111, 1000),
        # one conversation taken out of the cache
        _read("read 1x517", 1, 8, 128, 777, 517),
        # whole prompts for a dense prefill over a cached prefix
        _read("read 8x4096 f32", 8, 32, 128, 4096, 4096, dtype="f32", values="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST = {}  # bytes and operations of the largest listed case of each operator


def draw(rng):
    """One more case of the listed ranges, no larger than the largest listed one of its operator."""
    if not _MOST:
        for c in listed():
            w, m = work(c), _MOST.setdefault(c["op"], {"bytes": 0, "flops": 0})
            m.update({k: max(m[k], w[k]) for k in m})
    while True:
        op = rng.choice(["tree", "tree", "window", "window", "extend", "read"])
        kv = rng.choice([1, 2, 4, 8, 8, 16, 32])
        per = rng.choice([1, 2, 3, 4, 4, 7, 8])
        dim = rng.choice([64, 128, 128, 128, 256])
        group = rng.choice([128, 128, 128, 64, 32])
        dtype, values = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"),
                                    ("f32", "f32"), ("f32", "bf16"), ("f32", "f16")])
        batch, ctx = _log(rng, 1, 64), _log(rng, 16, 16384)
        ragged = rng.random() < 0.6
        if op == "tree":
            win = rng.choice([0, 0, 0, _log(rng, 128, 4096)])
            c = _tree("", batch, kv * per, kv, dim, ctx, rng.randint(1, 64), ragged, dtype, values,
                      win, rng.randint(0, 100) if win else 0, group)
        elif op == "window":
            c = _window("", batch, kv * per, kv, dim, ctx, _log(rng, 16, 8192), rng.randint(0, 100),
                        ragged, dtype, values, group)
        elif op == "extend":
            c = _extend("", batch, kv, dim, ctx, _log(rng, 1, 2048), ragged, rng.random() < 0.5, dtype,
                        values, group)
        else:
            c = _read("", batch, kv, dim, ctx, rng.randint(1, ctx), ragged, dtype, values, group)
        del c["name"]
        w = work(c)
        if w["bytes"] > 1e5 and all(w[k] <= _MOST[op][k] for k in w):
            return c


def _sizes(case):
    """Cached tokens of each sequence, and its drafted / new / read tokens (fixed by the case)."""
    rng = random.Random("%(batch)d %(ctx)d %(dim)d %(kv_heads)d" % case)
    batch, ctx, op = case["batch"], case["ctx"], case["op"]
    most = {"tree": "drafts", "extend": "new", "read": "count"}.get(op)
    most = case[most] if most else 1
    lens, counts = [ctx] * batch, [most] * batch
    if case["ragged"]:
        lens = [ctx] + [rng.randint(max(1, ctx // 4), ctx) for _ in range(batch - 1)]
        counts = [most] + [rng.randint(1, most) for _ in range(batch - 1)]
        if batch >= 4:
            lens[batch // 2] = 0  # a new sequence
            if op != "window":
                counts[batch // 3] = 0  # a sequence that takes no part
    if op == "read":
        counts = [min(c, n) for c, n in zip(counts, lens)]
    return lens, counts


def _visible(case, n):
    """(visible cached tokens, 128-token groups touched) of one query behind n cached tokens."""
    win = case.get("window", 0)
    if not win:
        return n, -(-n // case["group"])
    lo = max(0, n - win)
    head = min(case["sinks"], lo)
    return n - lo + head, -(-n // case["group"]) - lo // case["group"] + -(-head // case["group"])


def work(case):
    """Bytes that have to be read and written once, and the products' operations."""
    lens, counts = _sizes(case)
    d, h, vb = case["dim"], case["kv_heads"], BYTES[case["values"]]
    eb = BYTES[case["dtype"]]
    nbytes = flops = 0
    for n, t in zip(lens, counts):
        if case["op"] in ("tree", "window"):
            if not t:
                continue
            vis, groups = _visible(case, n)
            hq = case["q_heads"]
            nbytes += h * (vis * (d // 2 + vb * d) + 8 * d * groups) + 4 * -(-vis // PAGE)
            nbytes += 2 * eb * t * hq * d
            flops += 4 * d * hq * t * vis
            if case["op"] == "tree":
                nbytes += 2 * eb * t * h * d + 8 * t
        elif case["op"] == "extend":
            if not t:
                continue
            c, old = h * d, n % case["group"]
            span, groups = old + t, -(-(old + t) // case["group"])
            opened = (n + t) % case["group"]
            nbytes += c * (t * 2 * eb + old * 4 + span // 2 + 8 * groups + t * vb)  # the write
            nbytes += 4 * c * min(opened, t)  # staged keys of the open group
            nbytes += c * (span // 2 + 8 * groups + span * vb + span * 8)  # the values read back
            flops += 10 * c * span
        else:
            c = h * d
            nbytes += c * (t // 2 + 8 * -(-t // case["group"]) + t * vb + t * 2 * eb)
            flops += 2 * c * t
    return {"bytes": nbytes, "flops": flops}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def prepare(case, seed):
    lens, counts = _sizes(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed)
    b, h, d, group = case["batch"], case["kv_heads"], case["dim"], case["group"]
    dtype, values = TYPES[case["dtype"]], TYPES[case["values"]]
    full = [n + (t if case["op"] == "extend" else 0) for n, t in zip(lens, counts)]
    need = [-(-n // PAGE) for n in full]
    pool = sum(need) + 3
    order = list(range(pool))
    host.shuffle(order)
    table = np.zeros((b, max(1, max(need))), np.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    # post-rotary keys: every channel has its own spread and offset
    spread = torch.rand((h, d), generator=g, device="cuda") * 2.5 + 0.5
    offset = normal(h, d) * 2.0
    codes = (normal(pool, h, PAGE, d) * 2.6 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    k_pool = codes[..., 0::2] | (codes[..., 1::2] << 4)
    del codes
    scale = spread * (0.34 + 0.08 * torch.rand((pool, h, d), generator=g, device="cuda"))
    sz_pool = torch.stack([scale, 7.5 - offset / scale], dim=2)
    s = {"case": case, "lens": lens, "counts": counts, "group": group, "dtype": dtype,
         "k_pool": k_pool.contiguous(), "sz_pool": sz_pool.contiguous(),
         "v_pool": normal(pool, h, PAGE, d).to(values),
         "block_table": torch.from_numpy(table).cuda(),
         "seq_lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    offs = _offsets(counts)
    s["offsets"] = torch.from_numpy(offs).cuda()
    total = int(offs[-1])
    if case["op"] in ("tree", "window"):
        # the queries carry the softmax scale
        s["q"] = (normal(total if case["op"] == "tree" else b, case["q_heads"], d) / math.sqrt(d)).to(dtype)
    if case["op"] == "tree":
        s["k"] = (normal(total, h, d) * spread + offset).to(dtype)
        s["v"] = normal(total, h, d).to(dtype)
        words = []
        for t in counts:
            rows = []
            for i in range(t):
                parent = i - 1 if host.random() < 0.5 else host.randint(-1, i - 1)
                word = (rows[parent] if parent >= 0 else 0) | (1 << i)
                rows.append(word)
            words += rows
        s["tree"] = torch.from_numpy(np.array(words, np.uint64).view(np.int64)).cuda()
    if case["op"] == "extend":
        source = total * 2 if case["picked"] else total
        s["k"] = (normal(source, h, d) * spread + offset).to(dtype)
        s["v"] = normal(source, h, d).to(dtype)
        s["rows"] = None
        if case["picked"]:
            s["rows"] = torch.tensor(sorted(host.sample(range(source), total)), dtype=torch.int32,
                                     device="cuda")
        s["stage"] = normal(b + 2, group, h * d) * spread.reshape(-1) + offset.reshape(-1)
        slots = list(range(b + 2))
        host.shuffle(slots)
        s["slots"] = torch.tensor(slots[:b], dtype=torch.int32, device="cuda")
        # what is read back: each touched sequence from its first touched group on
        first = [n // group * group for n in lens]
        spans = [n + t - f if t else 0 for n, t, f in zip(lens, counts, first)]
        s["read_start"] = torch.tensor(first, dtype=torch.int32, device="cuda")
        s["read_offsets"] = torch.from_numpy(_offsets(spans)).cuda()
        s["spans"] = spans
    if case["op"] == "read":
        start = [host.randint(0, n - t) for n, t in zip(lens, counts)]
        s["read_start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
        s["read_offsets"] = s["offsets"]
        s["spans"] = counts
    return s


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------

def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2).float()


def _pages(s, index):
    """Keys and values [B, H, pages * 16, D] of logical pages index [B, pages], in 32 bits."""
    table = s["block_table"].long()
    last = table.shape[1] - 1
    phys = table.gather(1, index.clamp(0, last))
    per = s["group"] // PAGE
    sz = s["sz_pool"][table.gather(1, (index // per * per).clamp(0, last))]
    scale, zero = sz[:, :, :, 0, None], sz[:, :, :, 1, None]
    k = _unpack(s["k_pool"][phys]) * scale - zero * scale
    v = s["v_pool"][phys].float()
    return tuple(x.transpose(1, 2).flatten(2, 3) for x in (k, v))


def _softmax_sum(logits, seen, v):
    logits = logits.masked_fill(~seen, -math.inf)
    top = logits.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (logits - top).exp()
    return (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-10)


def _popcount(x, bits):
    return ((x[:, None] >> torch.arange(bits, device=x.device)) & 1).sum(1)


def _plain_tree(s):
    case = s["case"]
    b, h, d, most = case["batch"], case["kv_heads"], case["dim"], case["drafts"]
    per, dev = case["q_heads"] // h, s["q"].device
    offs = s["offsets"].long()
    count = offs[1:] - offs[:-1]
    t = torch.arange(most, device=dev)
    real = t < count[:, None]                                     # [B, T]
    row = (offs[:-1, None] + t).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[row].view(b, most, h, per, d).permute(0, 2, 1, 3, 4).reshape(b, h, most * per, d)
    kd, vd = (s[x].float()[row].transpose(1, 2) * real[:, None, :, None] for x in ("k", "v"))
    npages = s["block_table"].shape[1]
    kc, vc = _pages(s, torch.arange(npages, device=dev).expand(b, -1))
    n = s["seq_lens"].long()[:, None, None]
    bits = (s["tree"][row][:, :, None] >> t) & 1                  # [B, T, T]
    above = (bits * (t[:, None] != t)).sum(-1)                    # ancestors of each draft
    pos = torch.arange(npages * PAGE, device=dev)
    in_cache = (pos < n).expand(b, most, -1)
    in_tree = (bits == 1) & real[:, None, :]
    if case["window"]:
        edge = n + above[:, :, None] - case["window"]             # positions up to here are out
        in_cache = in_cache & ((pos > edge) | (pos < case["sinks"]))
        at = n + above[:, None, :]
        in_tree = in_tree & ((at > edge) | (at < case["sinks"]))
    seen = torch.cat([in_cache, in_tree], -1).repeat_interleave(per, 1)[:, None]
    logits = torch.cat([q @ kc.transpose(2, 3), q @ kd.transpose(2, 3)], -1)
    vc = vc * (pos < n)[:, :, :, None]
    out = _softmax_sum(logits, seen, torch.cat([vc, vd], 2))
    out = out.view(b, h, most, per, d).permute(0, 2, 1, 3, 4).reshape(b * most, h * per, d)
    which = torch.repeat_interleave(torch.arange(b, device=dev), count, output_size=s["q"].shape[0])
    flat = torch.arange(s["q"].shape[0], device=dev) - offs[which] + which * most
    return out[flat].to(s["dtype"])


def _plain_window(s):
    case = s["case"]
    b, h, d = case["batch"], case["kv_heads"], case["dim"]
    per, dev = case["q_heads"] // h, s["q"].device
    n = s["seq_lens"].long()[:, None]
    lo = (n - case["window"]).clamp(min=0)
    heads = torch.arange(-(-case["sinks"] // PAGE), device=dev).expand(b, -1)
    tails = lo // PAGE + torch.arange(-(-case["window"] // PAGE) + 1, device=dev)
    index = torch.cat([heads, tails], 1)
    pos = index[:, :, None] * PAGE + torch.arange(PAGE, device=dev)
    head = torch.arange(index.shape[1], device=dev)[:, None] < heads.shape[1]
    seen = torch.where(head, pos < torch.minimum(lo, lo.new_tensor(case["sinks"]))[:, :, None],
                       (pos >= lo[:, :, None]) & (pos < n[:, :, None])).flatten(1)
    k, v = _pages(s, index)
    q = s["q"].float().view(b, h, per, d)
    out = _softmax_sum(q @ k.transpose(2, 3), seen[:, None, None], v * seen[:, None, :, None])
    return out.reshape(b, h * per, d).to(s["dtype"])


def _places(s, start, spans):
    """(sequence, position) of each token of the ranges start[b] + [0, spans[b]), flat."""
    dev = start.device
    spans_t = torch.tensor(spans, device=dev)
    first = torch.cumsum(spans_t, 0) - spans_t
    seq = torch.repeat_interleave(torch.arange(len(spans), device=dev), spans_t, output_size=sum(spans))
    return seq, torch.arange(sum(spans), device=dev) - first[seq] + start.long()[seq]


def _plain_read(s, start, spans, dtype):
    seq, pos = _places(s, start, spans)
    table, group = s["block_table"].long(), s["group"]
    phys, slot = table[seq, pos // PAGE], pos % PAGE
    sz = s["sz_pool"][table[seq, pos // group * (group // PAGE)]]
    scale, zero = sz[:, :, 0], sz[:, :, 1]
    k = _unpack(s["k_pool"][phys, :, slot]) * scale - zero * scale
    return k.to(dtype), s["v_pool"][phys, :, slot].to(dtype)


def _plain_extend(s):
    case, group = s["case"], s["group"]
    h, d = case["kv_heads"], case["dim"]
    start, dev = s["seq_lens"].long(), s["k"].device
    seq, pos = _places(s, s["read_start"], s["spans"])
    new = pos >= start[seq]
    src = (s["offsets"].long()[seq] + pos - start[seq]).clamp(0, sum(s["counts"]) - 1)
    if s["rows"] is not None:
        src = s["rows"].long()[src]
    slot = s["slots"].long()[seq]
    x = torch.where(new[:, None], s["k"].float().flatten(1)[src], s["stage"][slot, pos % group])
    # groups in the order of the touched tokens
    edge = torch.ones_like(pos)
    edge[1:] = ((pos[1:] // group != pos[:-1] // group) | (seq[1:] != seq[:-1])).long()
    gid = edge.cumsum(0) - 1
    groups = sum(-(-n // group) for n in s["spans"])
    lo = x.new_full((groups, h * d), math.inf).index_reduce_(0, gid, x, "amin")
    hi = x.new_full((groups, h * d), -math.inf).index_reduce_(0, gid, x, "amax")
    scale = (hi - lo).clamp(min=1e-8) / torch.full_like(lo, 15.0)
    zero = -lo / scale
    codes = ((x - lo[gid]) / scale[gid]).round().clamp(0, 15).to(torch.uint8).view(-1, h, d)
    table = s["block_table"].long()
    phys, at = table[seq, pos // PAGE], pos % PAGE
    s["k_pool"][phys, :, at] = codes[..., 0::2] | (codes[..., 1::2] << 4)
    home = table[seq, pos // group * (group // PAGE)]
    s["sz_pool"][home] = torch.stack([scale[gid], zero[gid]], 1).view(-1, 2, h, d).transpose(1, 2)
    # old tokens keep their values; rows of the open group are staged
    v = torch.where(new[:, None, None], s["v"].float()[src].to(s["v_pool"].dtype),
                    s["v_pool"][phys, :, at])
    s["v_pool"][phys, :, at] = v
    end = start + (s["offsets"][1:] - s["offsets"][:-1]).long()
    staged = new & (pos >= (end // group * group)[seq])
    spare = torch.full_like(slot, s["stage"].shape[0])  # rows that are not staged go to no slot
    wide = torch.cat([s["stage"], s["stage"][:1]])
    wide[torch.where(staged, slot, spare), pos % group] = x
    s["stage"].copy_(wide[:-1])


def _extended(s, k, v):
    return {"k": k, "v": v, "scale_zp": s["sz_pool"], "values": s["v_pool"], "stage": s["stage"]}


def run(state):
    s, op = state, state["case"]["op"]
    case = s["case"]
    if not own:
        if op == "tree":
            return _plain_tree(s)
        if op == "window":
            return _plain_window(s)
        if op == "extend":
            _plain_extend(s)
            return _extended(s, *_plain_read(s, s["read_start"], s["spans"], torch.float32))
        return dict(zip("kv", _plain_read(s, s["read_start"], s["spans"], s["dtype"])))
    C = importlib.import_module(PACKAGE + "._C")
    pools = (s["k_pool"], s["v_pool"], s["sz_pool"])
    if op in ("tree", "window") and "workspace" not in s:  # kept, as a serving loop keeps it
        need = C.paged_attention_workspace_bytes(case["batch"], case["q_heads"], case["kv_heads"],
                                                 case["dim"], case.get("drafts", 1), s["q"].device)
        s["workspace"] = torch.empty((need,), dtype=torch.uint8, device=s["q"].device)
    if op == "tree":
        return C.paged_tree_decode(s["q"], s["k"], s["v"], s["tree"], s["offsets"], *pools,
                                   s["block_table"], s["seq_lens"], max_drafts=case["drafts"],
                                   group_tokens=s["group"], window=case["window"] or None,
                                   sinks=case["sinks"], workspace=s["workspace"])
    if op == "window":
        return C.paged_window_decode(s["q"], *pools, s["block_table"], s["seq_lens"],
                                     window=case["window"], sinks=case["sinks"],
                                     group_tokens=s["group"], workspace=s["workspace"])
    if op == "extend":
        C.cache_extend(s["k"], s["v"], s["offsets"], s["seq_lens"], s["slots"], s["stage"],
                       s["block_table"], *pools, max_rows_per_seq=case["new"],
                       group_tokens=s["group"], rows=s["rows"])
        most = case["new"] + s["group"] - 1
        return _extended(s, *C.cache_read(*pools, s["block_table"], s["read_start"],
                                          s["read_offsets"], num_rows=sum(s["spans"]),
                                          max_rows_per_seq=most, group_tokens=s["group"]))
    return dict(zip("kv", C.cache_read(*pools, s["block_table"], s["read_start"], s["read_offsets"],
                                       num_rows=sum(s["spans"]), max_rows_per_seq=case["count"],
                                       group_tokens=s["group"], dtype=s["dtype"])))


# --------------------------------------------------------------------------
# 64-bit evaluation, one sequence at a time
# --------------------------------------------------------------------------

def _exact_tokens(s, b, lo, hi):
    """Keys and values [tokens, H, D] of sequence b's tokens lo .. hi-1 in float64."""
    if hi <= lo:
        shape = (0, s["k_pool"].shape[1], s["v_pool"].shape[3])
        return torch.zeros(shape, dtype=torch.float64, device="cuda"), \
            torch.zeros(shape, dtype=torch.float64, device="cuda")
    where = torch.arange(lo, hi, device="cuda")
    row = s["block_table"][b].long()
    page, slot = row[torch.div(where, 16, rounding_mode="floor")], where.remainder(16)
    home = row[torch.div(where, s["group"], rounding_mode="floor") * (s["group"] // 16)]
    byte = s["k_pool"][page, :, slot].int()
    code = torch.zeros(byte.shape[:2] + (byte.shape[2] * 2,), dtype=torch.float64, device="cuda")
    code[..., 0::2] = (byte % 16).double()
    code[..., 1::2] = (byte // 16).double()
    sz = s["sz_pool"][home].double()
    return (code - sz[:, :, 1]) * sz[:, :, 0], s["v_pool"][page, :, slot].double()


def _exact_attention(s, b, rows, drafts):
    """Rows of sequence b (a slice of the queries), drafts = (k, v, visible words) or None."""
    case = s["case"]
    n, win, sinks = s["lens"][b], case["window"], case["sinks"]
    per = case["q_heads"] // case["kv_heads"]
    q = s["q"][rows].double()
    k, v = _exact_tokens(s, b, 0, n)
    where = torch.arange(n, device="cuda")
    out = torch.zeros_like(q)
    for i in range(q.shape[0]):
        if drafts is None:
            at, keep, depth = n - 1, None, None
        else:
            words = drafts[2]
            depth = [bin(w & ~(1 << j)).count("1") for j, w in enumerate(words)]
            at = n + depth[i]
            keep = [j for j in range(len(words)) if words[i] >> j & 1 and
                    (not win or n + depth[j] > at - win or n + depth[j] < sinks)]
        mine = torch.ones_like(where, dtype=torch.bool) if not win else (where > at - win) | (where < sinks)
        kk, vv = k[mine], v[mine]
        if drafts is not None:
            kk, vv = torch.cat([kk, drafts[0][keep]]), torch.cat([vv, drafts[1][keep]])
        if kk.shape[0]:
            x = torch.einsum("hgd,jhd->hgj", q[i].view(-1, per, case["dim"]), kk)
            out[i] = torch.einsum("hgj,jhd->hgd", torch.softmax(x, -1), vv).reshape(q[i].shape)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    lens, counts, op = s["lens"], s["counts"], case["op"]
    offs = [0]
    for c in counts:
        offs.append(offs[-1] + c)
    if op in ("tree", "window"):
        # the row-by-row evaluation reads every key once a row: too long for the largest trees
        reads = sum(n * (c if op == "tree" else 1) for n, c in zip(lens, counts))
        if reads * case["q_heads"] * case["dim"] > 6e10:
            return None
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            if op == "window":
                out[b:b + 1] = _exact_attention(s, b, slice(b, b + 1), None)
                continue
            mine = slice(offs[b], offs[b + 1])
            words = [w % (1 << 64) & ((1 << counts[b]) - 1) for w in s["tree"][mine].tolist()]
            out[mine] = _exact_attention(s, b, mine, (s["k"][mine].double(), s["v"][mine].double(), words))
        return out
    if op == "read":
        got = [_exact_tokens(s, b, lo, lo + c) for b, (lo, c) in enumerate(zip(s["read_start"].tolist(), counts))]
        return {"k": torch.cat([k for k, _ in got]), "v": torch.cat([v for _, v in got])}
    # extend: the codes are defined by IEEE float32 steps, what they stand for is taken in 64 bits
    keys, vals, group = [], [], s["group"]
    width = case["kv_heads"] * case["dim"]
    for b in range(case["batch"]):
        if not counts[b]:
            continue
        take = torch.arange(offs[b], offs[b + 1], device="cuda")
        if s["rows"] is not None:
            take = s["rows"].long()[take]
        old = lens[b] % group
        x = torch.cat([s["stage"][int(s["slots"][b]), :old], s["k"][take].float().reshape(-1, width)])
        _, before = _exact_tokens(s, b, lens[b] - old, lens[b])
        vals.append(torch.cat([before, s["v"][take].float().to(s["v_pool"].dtype).double()]))
        for lo in range(0, x.shape[0], group):
            part = x[lo:lo + group].cpu().numpy()
            small, big = part.min(0), part.max(0)
            scale = np.maximum(big - small, np.float32(1e-8)) / np.float32(15)
            code = np.clip(np.rint((part - small) / scale), 0, 15).astype(np.float64)
            zero = (-small / scale).astype(np.float64)
            value = (code - zero) * scale.astype(np.float64)
            keys.append(torch.from_numpy(value).cuda().view(-1, case["kv_heads"], case["dim"]))
    return {"k": torch.cat(keys), "v": torch.cat(vals), "scale_zp": None, "values": None, "stage": None}
