"""GPU: batches that would take more scratch memory than the bound get fewer parts, or none, and are as right.  Tolerances as in
test_gpu_paged_attention.py."""
import numpy as np
import pytest
import torch

from tests.test_gpu_paged_attention import Batch, numbers, parts_of_tails

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,longer,parts", [(128, 0, 2), (128, 700, 3), (256, 0, 0), (256, 700, 0)])   # (4 parts, or 2 of so few keys, without a bound)
def test_last_rows_of_many_sequences(dim, longer, parts):
    lengths = [(70 + 7 * (i % 40) + (longer if i % 100 == 39 else 0), 1 + i * 5 % 18) for i in range(512)]
    b = Batch(91, lengths, heads=32, kv_heads=8, dim=dim, behind=2)
    assert parts_of_tails(b, 8) == pytest.approx(parts)
    got = b.call()
    assert (got[-2:] == 0).all() and torch.equal(got, b.call())
    for i in (0, 1, 7, 39, 255, 300, 511):   # some, each as a batch of its own
        n, queries = lengths[i]
        one = Batch(91, [(n, queries)], heads=32, kv_heads=8, dim=dim)
        first = int(b.starts[i])
        one.q, one.k, one.v = b.q[first:first + queries], b.k[b.table[i, :-(-n // 16)].long()], b.v[b.table[i, :-(-n // 16)].long()]
        one.table = torch.arange(len(one.k), dtype=torch.int32)[None]
        one.check(got[first:first + queries])
    assert np.isfinite(numbers(got)).all()
