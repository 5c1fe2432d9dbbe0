"""GPU: parts of the keys follow the lengths on the device, whatever the host says, with more sequences than a wavefront looks at in
one go.  Tolerances as in test_gpu_paged_attention.py."""
import pytest
import torch

from tests.test_gpu_paged_attention import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs", [62, 64, 100, 150, 255])
@pytest.mark.parametrize("queries", [1, 9])
def test_the_same_parts_for_any_longest_length(seqs, queries):
    """Where the host takes as many parts at most for two longest lengths that it is told, the parts are the same, and so are the bits."""
    from sonar_amd import _lib
    lengths = [(700 + 13 * (i * 29 % 97), queries) for i in range(seqs)]
    b = Batch(61, lengths, heads=4, kv_heads=1, dim=128)
    b.check(b.call())
    alike = {}
    for longest in (max(n for n, _ in lengths), 4096, 6000, 40000, 1 << 20):
        size = _lib.load_attention().sonar_paged_attention_scratch_bytes(len(b.q), seqs, 4, 1, 128, 1, longest, 0)
        alike.setdefault(size, []).append(b.call(longest))
    assert max(map(len, alike.values())) > 1 and 0 not in alike
    for got in alike.values():
        assert all(torch.equal(g, got[0]) for g in got)
    want = b.call(1 << 17)
    b.table = torch.nn.functional.pad(b.table, (0, (1 << 17) // 16 - b.table.shape[1]), value=-1)
    assert torch.equal(b.call(), want)   # a table that wide says the same


@pytest.mark.parametrize("seqs,keys", [(32, 2000), (64, 2000), (70, 700), (32, 4096), (70, 4096)])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_wide_table_gives_the_parts_of_the_lengths(seqs, keys, dim):
    """What the host would choose if it were told the longest length is chosen on the device where it was not: the same bits.  (Where
    it would split no rows but the last ones, the device splits none.)"""
    from sonar_amd import _lib
    lengths = [(keys - 7 * (i % 50), 33) for i in range(seqs)]
    b = Batch(62, lengths, heads=16, kv_heads=4, dim=dim)
    size = _lib.load_attention().sonar_paged_attention_scratch_bytes(len(b.q), seqs, 16, 4, dim, 1, keys, 0)
    parts = size / (len(b.q) * 16 * (4 * dim + 8))
    want = b.call(keys)
    b.table = torch.nn.functional.pad(b.table, (0, (1 << 17) // 16 - b.table.shape[1]), value=-1)
    got = b.call()
    if keys == 4096:
        assert parts in (2, 3, 5)
    if parts == int(parts):
        assert torch.equal(got, want)
    if keys <= 2000:
        b.check(got)
