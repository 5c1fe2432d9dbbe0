"""CPU: the scratch memory of the attention over a paged cache has a bound that no size passes: 256 MiB."""
import random

import pytest

MOST = 256 << 20


def scratch(tokens, seqs, heads, kv_heads, dim, fp8, longest, window=0):
    from sonar_amd import _lib
    lib = _lib.load_attention()
    return lib.sonar_paged_attention_scratch_bytes(tokens, seqs, heads, kv_heads, dim, _lib.CACHE_FP8 if fp8 else 1, longest, window)


@pytest.mark.parametrize("tokens,seqs,heads,kv_heads,dim,fp8,longest", [
    (9000, 1024, 32, 8, 256, False, 100000), (9000, 1024, 32, 8, 128, False, 100000),   # last rows in parts: 1032 and 520 MiB once
    (2112, 64, 32, 8, 128, False, 131072),                                              # parts of many rows: 536 MiB
    (4096, 4096, 128, 8, 128, True, 131072), (60000, 60000, 64, 8, 256, True, 2 ** 30)])  # parts of few rows: 1040 MiB and more
def test_large_batches(tokens, seqs, heads, kv_heads, dim, fp8, longest):
    assert scratch(tokens, seqs, heads, kv_heads, dim, fp8, longest) <= MOST


def test_any_batch():
    rng = random.Random(81)
    for _ in range(20000):
        kv_heads = 2 ** rng.randrange(8)
        heads = kv_heads * rng.randint(1, 16)
        seqs = int(2 ** rng.uniform(0, 18))
        tokens = min(int(seqs * 2 ** rng.uniform(0, 14)), ((1 << 31) - 1) // heads)
        case = (tokens, seqs, heads, kv_heads, 16 * rng.randint(1, 16), rng.random() < 0.5, int(2 ** rng.uniform(0, 31)) - 1,
                rng.choice([0, 0, int(2 ** rng.uniform(0, 20))]))
        assert scratch(*case) <= MOST, case


def test_what_takes_less_keeps_its_parts():
    """Batches below the bound take what their parts need (a row of a part: its numbers, a maximum and a sum)."""
    assert scratch(1, 1, 32, 8, 128, False, 8000) > 0
    assert scratch(64, 64, 8, 1, 128, False, 4096) == 8 * 64 * 8 * (128 * 4 + 8)
    assert scratch(1056, 32, 32, 8, 128, False, 4096) == 3 * 1056 * 32 * (128 * 4 + 8)
    assert scratch(16001, 17, 32, 8, 128, False, 100000) == 15 * 17 * 8 * 32 * (128 * 4 + 8)
