"""GPU: a page number outside the cache reaches the queries that see a key of that page, which get NaN, and no others, also not those
of the same block of rows.  Tolerances as in test_gpu_paged_attention.py."""
import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao
from tests.test_gpu_paged_attention import MIXED, Batch, numbers

pytestmark = pytest.mark.gpu

# blocks of 16, 128 and 256 rows, whole and in parts, last rows in parts
FORMS = {"few": dict(lengths=[(100, 8), (50, 4), (40, 8)], dim=64), "few codes": dict(lengths=[(100, 8), (50, 4), (40, 8)], dim=128, fp8=True),
         "many": dict(lengths=[(150, 60), (90, 90), (200, 150)], dim=128), "many codes": dict(lengths=[(150, 60), (90, 90)], dim=64, fp8=True),
         "wide": dict(lengths=[(150, 60), (90, 90)], dim=256), "parts": dict(lengths=[(900, 4), (300, 2)], dim=128, kv_heads=1),
         "many parts": dict(lengths=[(6000, 4)], dim=64, kv_heads=1), "parts of many": dict(lengths=[(900, 40)], dim=80, kv_heads=1),
         "last rows": dict(lengths=MIXED, heads=64, kv_heads=64, dim=64), "blocks of 256": dict(lengths=[(300, 300)] * 16, heads=32, kv_heads=8, dim=128)}


@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("kind", ["causal", "window", "tree", "tree of 300", "all"])
@pytest.mark.parametrize("page", [16, 7])
def test_only_those_who_see_it(name, kind, page):
    form = FORMS[name]
    window = 40 if kind == "window" else 0
    b = Batch(41, page=page, tree_words={"tree": 2, "tree of 300": 5}.get(kind, 0), **form)
    more = dict(window=window) if window else dict(causal=False) if kind == "all" else {}
    want, limit = b.limits(**more)
    hit = np.zeros(len(b.q), dtype=bool)
    for i, (n, queries) in enumerate(b.lengths):
        if i % 2 or queries == 0:
            continue   # (some sequences stay as they are)
        first = int(b.starts[i])
        sight = ao.visible(n, queries, kind != "all", window, None if b.tree is None else b.tree[first:first + queries].numpy())
        # a page in the middle of the queries' own keys, and the last one
        for at, number in (((n - queries // 2 - 1) // page, -1), ((n - 1) // page, len(b.k))):
            keys = slice(at * page, min((at + 1) * page, n))
            b.table[i, at] = number
            hit[first:first + queries] |= sight[:, keys].any(axis=1)
    got = numbers(b.call(**more))
    assert hit.any() != (name == "blocks of 256" and kind == "tree")   # (there both pages are of drafts past the 128 bits, which nobody sees)
    assert np.isnan(got[hit]).all()
    assert (np.abs(got - want)[~hit] <= limit[~hit]).all(), np.argwhere(~(np.abs(got - want) <= limit))[:5]
    if kind == "causal" and name in ("many", "wide", "blocks of 256"):
        assert not hit[int(b.starts[0])]   # the sequence's first query sees neither
    assert torch.equal(b.call(**more).isnan(), torch.from_numpy(np.isnan(got)).to("cuda:0"))
