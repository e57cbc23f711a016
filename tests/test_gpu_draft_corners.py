"""The draft operators in corners of what they allow: keys and values of different types."""


import numpy as np
import pytest

from helpers import pkg
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
