"""GPU: attention over a paged cache where scores are infinite.  By the definition a key of score -infinity counts nothing beside
others, but a query all of whose keys have that score has no softmax: NaN, not the zeros of a query that sees no key.  A score of
+infinity is NaN too.  Tolerances as in test_gpu_paged_attention.py."""
import numpy as np
import pytest
import torch

from tests.test_gpu_paged_attention import HALF_STEP, MIXED, Batch, numbers

pytestmark = pytest.mark.gpu
INF = float("inf")

# few rows and many, whole and in parts that one wavefront or eight join, last rows in parts, queries that see nothing
FORMS = {"few": dict(lengths=[(100, 2), (1, 1), (40, 3), (3, 5)], dim=64), "few codes": dict(lengths=[(100, 2), (1, 1), (40, 3), (3, 5)], dim=128, fp8=True),
         "many": dict(lengths=[(150, 60), (90, 90), (20, 33)], dim=128), "many codes": dict(lengths=[(150, 60), (90, 90), (20, 33)], dim=64, fp8=True),
         "wide": dict(lengths=[(150, 60), (90, 90), (20, 33)], dim=256), "parts": dict(lengths=[(900, 3), (2, 4)], dim=128, kv_heads=1),
         "many parts": dict(lengths=[(6000, 1)], dim=64, kv_heads=1), "parts of many": dict(lengths=[(900, 40), (30, 33)], dim=80, kv_heads=1),
         "last rows": dict(lengths=MIXED, heads=64, kv_heads=64, dim=64)}


def limit_of(b, want, size, most, softcap=0.0):
    """As Batch.limits, with the largest score sum given."""
    h, u = HALF_STEP[b.dtype], 2.0 ** -24
    e = (b.dim + 8) * u * most + 2.0 ** -22 + softcap * 2.0 ** -20
    return size * (h + 2 * e[:, :, None] + max(n for n, _ in b.lengths) * u) + np.abs(want) * h + 2.0 ** -24


def check(got, want, limit):
    got = numbers(got)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), (np.argwhere(np.isnan(got) != nan)[:5], np.isnan(got).sum(), nan.sum())
    assert (np.abs(got - want)[~nan] <= limit[~nan]).all()
    return nan


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("name", FORMS)
def test_queries_whose_scores_are_all_minus_infinity(name, tree):
    b = Batch(31, tree_words=2 if tree else 0, **FORMS[name])
    most = b.want()[2]
    if b.k_scale is None:
        b.k[..., 5] = 1.0
    else:
        b.k.view(torch.uint8)[..., 5] = 0x38
    most = np.maximum(most, b.want()[2])
    b.q[::3, :, 5] = -INF
    want, size, _ = b.want()
    nan = check(b.call(), want, limit_of(b, want, size, most))
    assert nan.any()   # (and zeros where nothing is seen, an infinity in the query or not, are the oracle's)


@pytest.mark.parametrize("name", ["few", "many", "many codes", "parts"])
def test_capped_infinities_are_finite(name):
    """cap * tanh(-infinity) = -cap for every key: their mean."""
    b = Batch(32, **FORMS[name])
    if b.k_scale is None:
        b.k[..., 5] = 1.0
    else:
        b.k.view(torch.uint8)[..., 5] = 0x38
    most = b.want(softcap=20.0)[2]
    b.q[::3, :, 5] = -INF
    want, size, _ = b.want(softcap=20.0)
    most[::3] = 20.0
    assert not check(b.call(softcap=20.0), want, limit_of(b, want, size, most, 20.0)).any()


@pytest.mark.parametrize("name", [n for n in FORMS if "codes" not in n])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_what_an_infinite_key_gives_to_those_who_see_it(name, sign):
    """-infinity: the same as without that key, NaN where it is the only one; +infinity: NaN.  Others see none of it."""
    b = Batch(33, **FORMS[name])
    b.q[..., 5] = b.q[..., 5].abs() + 0.5
    at = []
    for i, (n, queries) in enumerate(b.lengths):
        for key in {0, n - 1, max(n - queries, 0)} if n else ():
            at.append((int(b.table[i, key // 16]), key % 16))
    for page, slot in at:
        b.k[page, slot, 0, 5] = 0.0
    most = b.want()[2]
    for page, slot in at:
        b.k[page, slot, 0, 5] = sign * INF
    want, size, _ = b.want()
    nan = check(b.call(), want, limit_of(b, want, size, most))
    assert nan.any() == (sign > 0 or any(n > 0 and (n == 1 or queries >= n) for n, queries in b.lengths))
