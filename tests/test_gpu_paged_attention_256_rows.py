"""GPU: the forms of 256 rows with codes, caps and slopes against the definition in 64 bits, each number by its own tolerance (those of
test_gpu_paged_attention.py)."""
import pytest
import torch

from tests.test_gpu_paged_attention import DEV, HALF_STEP, Batch

pytestmark = pytest.mark.gpu


def double_attention(b, cap, slopes):
    """Causal attention of one sequence in 64 bits, a head at a time: (out, mean of |v|, largest score sum)."""
    (n, queries), = b.lengths
    q = b.q.to(DEV).double()
    slots = b.table[0].long().to(DEV)
    k, v = (c.to(DEV).double()[slots].reshape(-1, *c.shape[2:])[:n] * (1.0 if s is None else s.to(DEV).double()) for c, s in ((b.k, b.k_scale), (b.v, b.v_scale)))
    at, keys = torch.arange(n - queries, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
    out, size, most = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(3))
    for h in range(q.shape[1]):
        g = h // (q.shape[1] // k.shape[1])
        x, kt = q[:, h].contiguous(), k[:, g].t().contiguous()
        s = (x @ kt) * b.dim ** -0.5
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            s = s - slopes[h].double() * (at - keys)
        p = torch.softmax(s.masked_fill(keys > at, -float("inf")), dim=1)
        out[:, h], size[:, h] = p @ v[:, g], p @ v[:, g].abs()
        most[:, h] = ((x.abs() @ kt.abs()) * b.dim ** -0.5).masked_fill(keys > at, 0).amax(1, keepdim=True)
    return out, size, most


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("score", ["plain", "capped", "sloped"])
@pytest.mark.parametrize("length,queries", [(4200, 4100), (4096, 4096)])
def test_codes_and_scores(dtype, fp8, score, length, queries):
    b = Batch(71, [(length, queries)], heads=32, kv_heads=4, dim=128, fp8=fp8, dtype=dtype)
    cap = 20.0 if score == "capped" else 0.0
    slopes = torch.linspace(0.001, 0.5, 32, device=DEV) if score == "sloped" else None
    got = b.call(softcap=cap, alibi_slopes=slopes)
    want, size, most = double_attention(b, cap, slopes)
    h, u = HALF_STEP[dtype], 2.0 ** -24
    # (a slope's share of a score, at most half the distance, is formed with 3 roundings)
    e = (128 + 8) * u * most + 2.0 ** -22 + cap * 2.0 ** -20 + (3 * u * 0.5 * length if slopes is not None else 0.0)
    limit = size * (h + 2 * e + length * u) + want.abs() * h + 2.0 ** -24
    assert ((got.double() - want).abs() <= limit).all()
