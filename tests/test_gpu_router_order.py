"""GPU: the router ranks a choice, score + bias, by all the bits of its double: choices below float32's range, choices that
differ in the last bits of the sum, and exact zeros (the score of a logit of -inf) among them.

A kernel's score is within a few 2^-53 of itself (of a score e^-d: d + 4 of them), as is the oracle's.  So wherever two choices
of a row differ at all, the inputs keep them apart by more: by a factor of e^0.1 and above where scores are tiny (equal logits
are equal choices), by 3 units in the last place of the sums and above where a bias is added to scores near 1."""
import numpy as np
import pytest
import torch

from oracle import layer_oracle as lo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
RTOL = 40 * 2.0 ** -24   # (derived in test_gpu_router.py)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# few tokens: a wavefront each, with 1, 4 and 16 experts a lane (8 lanes up to 8 experts); from 4096 on 8 to 32 lanes a token
EXPERTS = [8, 32, 60, 64, 100, 128, 256, 500, 1024]
TOKENS = [6, 4099]


def check(x, bias, topk, scoring, renormalize, groups=1, kept=1):
    from sonar_amd import ops
    w, ids = ops.topk_routing(x.to(DEV), topk, scoring, renormalize, bias.to(DEV), groups, kept)
    rows = sorted({*range(3), *range(x.shape[0] // 2, x.shape[0], max(1, x.shape[0] // 40)), x.shape[0] - 2, x.shape[0] - 1})
    want_w, want_ids = lo.topk_routing(x[rows].double().numpy(), topk, scoring, renormalize, bias.double().numpy(), groups, kept)
    assert np.array_equal(ids.cpu().numpy()[rows], want_ids)
    np.testing.assert_allclose(w.cpu().double().numpy()[rows], want_w, rtol=RTOL, atol=1e-40)


def shuffled(seed, tokens, values):
    """`values` in another order in each row."""
    gen = torch.Generator().manual_seed(seed)
    return values[torch.rand((tokens, values.numel()), generator=gen).argsort(1)]


@pytest.mark.parametrize("experts", EXPERTS)
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_scores_below_float32(experts, tokens, scoring, dtype):
    """An even bias of zero, as a new correction bias is, and logits from -110 to -310 (110 to 310 below a row's largest):
    their scores are 1e-48 to 1e-135.  Every third expert is masked with -inf and has the score 0, below all of them."""
    x = shuffled(experts, tokens, torch.linspace(-310, -110, experts)).to(DTYPES[dtype])
    x[:, ::3] = -float("inf")
    x[1, : experts // 2] = -float("inf")
    if scoring == "softmax":
        x[:, experts - 1] = 0.0
    bias = torch.zeros(experts)
    for topk in (1, min(8, experts), min(experts, 40)):
        check(x, bias, topk, scoring, True)
        check(x, bias, topk, scoring, False)
    if experts % 4 == 0:
        check(x, bias, min(8, experts // 2), scoring, True, 4, 2)


@pytest.mark.parametrize("experts", EXPERTS)
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("start,bias", [(17.5, 63 + 5 * 2.0 ** -18), (17.5, -101.0), (21.0, 0.0953)])
def test_sums_that_differ_in_their_last_bits(experts, tokens, start, bias):
    """Neighbouring float32 logits (2^-19 apart) and one bias for all.  Near 17.5 the sigmoids are e^-17.5 2^-19 = 4.8e-14 apart,
    3.3 units of a sum near 64 or -100 (2^-46); near 21 e^-21 2^-19 = 1.4e-15, 6 units of a sum near 1.1 (2^-52)."""
    values = torch.from_numpy((start + np.arange(experts) * 2.0 ** -19).astype(np.float32))
    s = 1 / (1 + np.exp(-values.double().numpy())) + np.float64(np.float32(bias))
    assert (np.diff(s) >= 2.9 * np.spacing(np.abs(s[1:]))).all()
    x = shuffled(experts + 1, tokens, values)
    for topk in (1, min(8, experts), min(experts, 40)):
        check(x, torch.full((experts,), bias), topk, "sigmoid", topk > 1)
