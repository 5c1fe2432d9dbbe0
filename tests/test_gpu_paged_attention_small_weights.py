"""GPU: many weights far below the largest one, whose key has a value of zero, so that the result is theirs alone.  float16 holds less
of such weights than bfloat16.

Tolerances: those of test_gpu_paged_attention.py, and for float16 what it does not hold.  The largest weight is rounded as a number
between 2^7 and 2^15, so that the others are off by half a step, or, where they are subnormal, by 2^-25, which is 2^-32 of the
largest: keys * 2^-32 of the largest |v|."""
import numpy as np
import pytest
import torch

from tests.test_gpu_paged_attention import HALF_STEP, Batch, numbers
from tests.test_gpu_paged_attention_places import double_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("below", [12.0, 18.3, 24.4, 26.3])
@pytest.mark.parametrize("lengths,heads,dim,fp8", [
    ([(300, 1)], 4, 64, False), ([(300, 2)], 4, 128, True), ([(20000, 1)], 4, 64, False), ([(20000, 2)], 4, 128, True), ([(3000, 1)] * 40, 8, 64, False), ([(20000, 30)], 4, 128, False),
    ([(5000, 30), (5000, 40)], 16, 256, False), ([(5000, 150)] * 3, 32, 128, False), ([(5000, 40)] * 2, 8, 128, True)])
def test_far_below_the_largest(dtype, below, lengths, heads, dim, fp8):
    b = Batch(51, lengths, heads=heads, kv_heads=2, dim=dim, dtype=dtype, fp8=fp8)
    rng = torch.Generator().manual_seed(52)
    # scores: q = (4, small numbers), k = (0, small numbers), of the large key (its distance / 4, 0)
    b.q = (torch.randn(b.q.shape, generator=rng) * 0.25).to(b.q.dtype)
    b.q[..., 0] = 4.0
    k = torch.randn(b.k.shape, generator=rng) * 0.25
    v = torch.rand(b.v.shape, generator=rng) * 4 + 4
    k[..., 0] = 0.0
    for i in range(len(lengths)):
        page = int(b.table[i, 50 // 16])
        k[page, 50 % 16], v[page, 50 % 16] = 0.0, 0.0
        k[page, 50 % 16, :, 0] = below * np.log(2) / 4 * dim ** 0.5
    b.k, b.v = k.to(b.k.dtype), v.to(b.v.dtype)
    if fp8:
        b.k_scale, b.v_scale = torch.ones(1), torch.ones(1)
    got = b.call()
    table = b.table.to("cuda:0")
    want, size, most = double_attention(b.q.to("cuda:0"), b.k.to("cuda:0").float(), b.v.to("cuda:0").float(), lengths, table, 16)
    h, u, keys = HALF_STEP[dtype], 2.0 ** -24, max(n for n, _ in lengths)
    e = (dim + 8) * u * most + 2.0 ** -22
    limit = size * (h + 2 * e + keys * u) + want.abs() * h + 2.0 ** -24 + (keys * 2.0 ** -32 * 8 if dtype == "fp16" else 0)
    off = (got.double() - want).abs()
    assert (off <= limit).all(), float((off / limit).max())
    assert float((limit / want.abs()).max()) < 0.2 and numbers(got).min() > 0
