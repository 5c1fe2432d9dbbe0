"""GPU: the router against the 64-bit oracle.  The experts are equal number by number.  Weights, with u = 2^-24: a softmax
term e^d (d the distance to the largest logit, off by |d| u) is off by at most (2 |d| + 3) u where it is taken in float32, so
the sum of the terms by the mean of that over them (|d| is ln 1024 at most in the mean: 17 u) and 21 u of its additions; the
result's rounding adds one: 40 u with the chosen term itself, the quotients and the factor taken in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import layer_oracle as lo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
RTOL = 40 * 2.0 ** -24
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def make(seed, tokens, experts, dtype="fp32", bias=False, spread=1.5):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn((tokens, experts), generator=gen) * spread).to(DTYPES[dtype])
    return x, 0.1 * torch.randn(experts, generator=gen) if bias else None


def check(x, topk, scoring, renormalize, bias, groups=1, kept=1, factor=1.0, given=None):
    from sonar_amd import ops
    w, ids = ops.topk_routing(x.to(DEV) if given is None else given, topk, scoring, renormalize, None if bias is None else bias.to(DEV),
                              groups, kept, factor)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32 and w.shape == ids.shape == (x.shape[0], topk)
    want_w, want_ids = lo.topk_routing(x.double().numpy(), topk, scoring, renormalize, None if bias is None else bias.double().numpy(),
                                       groups, kept, factor)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    np.testing.assert_allclose(w.cpu().double().numpy(), want_w, rtol=RTOL, atol=1e-40)


EXPERTS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 60, 63, 64, 65, 96, 100, 127, 128, 129, 160, 200, 255, 256, 257, 384, 500, 512, 513,
           768, 1000, 1023, 1024]


@pytest.mark.parametrize("experts", EXPERTS)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_experts(experts, scoring, biased):
    for i, (topk, dtype) in enumerate([(1, "fp32"), (2, "bf16"), (6, "fp16"), (8, "fp32")]):
        x, bias = make(experts + i, 5, experts, dtype, biased)
        check(x, min(topk, experts), scoring, i % 2 == 0, bias, factor=1.0 if i < 2 else 2.5)


@pytest.mark.parametrize("tokens", [1, 2, 3, 7, 8, 9, 15, 16, 17, 63, 64, 65, 100, 257, 1001])
@pytest.mark.parametrize("experts", [8, 32, 64, 256])
def test_tokens(tokens, experts):
    x, bias = make(tokens, tokens, experts, "fp32", tokens % 2 == 0)
    check(x, 2 if experts == 8 else 8, "softmax" if tokens % 3 else "sigmoid", True, bias)


@pytest.mark.parametrize("experts,topk", [(64, 64), (16, 16), (1024, 64), (100, 33), (9, 9), (33, 32), (256, 17)])
@pytest.mark.parametrize("biased", [False, True])
def test_many_choices(experts, topk, biased):
    x, bias = make(experts, 6, experts, "bf16", biased)
    check(x, topk, "softmax", False, bias)
    check(x, topk, "sigmoid", True, bias)


@pytest.mark.parametrize("experts,groups,kept,topk", [(256, 8, 4, 8), (160, 8, 3, 6), (64, 64, 7, 7), (64, 8, 8, 8), (512, 16, 1, 10),
                                                      (12, 4, 2, 6), (30, 3, 2, 20), (1024, 64, 64, 64), (1024, 2, 1, 8), (8, 8, 1, 1),
                                                      (1000, 8, 3, 12), (4, 2, 1, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_groups(experts, groups, kept, topk, scoring, biased):
    for dtype in ("fp32", "bf16"):
        x, bias = make(experts + groups, 9, experts, dtype, biased)
        check(x, topk, scoring, True, bias, groups, kept, 2.5)


@pytest.mark.parametrize("experts,groups,kept", [(8, 1, 1), (60, 1, 1), (64, 8, 3), (256, 8, 4), (300, 3, 2), (1024, 4, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_ties(experts, groups, kept, scoring, biased):
    """Equal logits (and an even bias) go to the lowest number, equal groups likewise."""
    x = torch.round(make(3, 40, experts)[0])
    x[0] = 0
    bias = torch.full((experts,), 0.25) if biased else None
    topk = min(8, kept * (experts // groups))
    check(x, topk, scoring, True, bias, groups, kept)
    check(x.to(torch.bfloat16), topk, scoring, False, bias, groups, kept)


@pytest.mark.parametrize("experts,groups,kept,topk", [(8, 1, 1, 2), (32, 1, 1, 32), (100, 1, 1, 8), (256, 8, 4, 8), (64, 4, 1, 16), (1000, 1, 1, 8)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_masks_and_numbers_that_are_none(experts, groups, kept, topk, scoring, biased, dtype):
    """Experts masked with -inf or the type's lowest number, rows that a mask leaves empty, NaN, infinities, and logits so
    far down that float32 has no number for their sigmoid."""
    x, bias = make(experts + topk, 16, experts, dtype, biased)
    low = torch.finfo(DTYPES[dtype]).min
    x[0] = -float("inf")
    x[1] = low
    x[2, ::2] = -float("inf")
    x[3, 1::2] = low
    x[4] = float("nan")
    x[5, experts // 2] = float("nan")
    x[6, :] = -float("inf")
    x[6, experts - 1] = 0.5
    x[7, 0] = x[7, experts - 1] = float("inf")
    x[8] = x[8] * 0.01 - 200
    x[9] = x[9] * 0.01 + 50
    x[10] = x[10] * 20
    x[11, : experts // 2] = -float("inf")
    x[12] = -float("inf")
    x[12, : max(1, experts // groups // 2)] = torch.linspace(-1, 1, max(1, experts // groups // 2)).to(x.dtype)
    for renormalize in (False, True):
        check(x, topk, scoring, renormalize, bias, groups, kept)


@pytest.mark.parametrize("experts,groups,kept,topk", [(6, 1, 1, 2), (8, 4, 2, 3), (9, 1, 1, 9), (32, 1, 1, 4), (32, 8, 3, 5), (30, 3, 2, 20), (33, 1, 1, 6),
                                                      (64, 16, 5, 20), (64, 1, 1, 64), (100, 1, 1, 33), (128, 8, 4, 8), (128, 1, 1, 40),
                                                      (160, 8, 3, 6), (250, 1, 1, 8), (256, 8, 4, 8), (256, 1, 1, 64), (256, 32, 3, 8)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_many_tokens(experts, groups, kept, topk, scoring, biased, dtype):
    """From 4096 tokens several share a wavefront.  Rows with ties, masks, NaN and infinities among them; the last ones
    share theirs with nobody.  Some rows of each kind are compared."""
    from sonar_amd import ops
    tokens = 4099
    x, bias = make(experts + topk, tokens, experts, dtype, biased)
    low = torch.finfo(DTYPES[dtype]).min
    x[1::10] = torch.round(x[1::10].float()).to(x.dtype)
    x[2::10, ::2] = -float("inf")
    x[3::10] = -float("inf")
    x[4::10, 1::3] = low
    x[5::10, experts // 2] = float("nan")
    x[6::10, 0] = x[6::10, experts - 1] = float("inf")
    x[7::10] = x[7::10] * 0.01 - 200
    if biased:
        bias[experts // 2] = bias[0]   # (equal choices at equal logits)
    for renormalize in (True, False):
        w, ids = ops.topk_routing(x.to(DEV), topk, scoring, renormalize, None if bias is None else bias.to(DEV), groups, kept, 1.5)
        rows = sorted({*range(0, tokens, 97), *range(tokens - 12, tokens)})
        want_w, want_ids = lo.topk_routing(x[rows].double().numpy(), topk, scoring, renormalize,
                                           None if bias is None else bias.double().numpy(), groups, kept, 1.5)
        assert np.array_equal(ids.cpu().numpy()[rows], want_ids)
        np.testing.assert_allclose(w.cpu().double().numpy()[rows], want_w, rtol=RTOL, atol=1e-40)


def test_more_tokens_than_a_launch_takes():
    """2^25 tokens of 8 experts are a launch; the next one's results lie behind the first one's."""
    from sonar_amd import ops
    tokens = (1 << 25) + 1000
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((tokens, 8), generator=gen, device=DEV, dtype=torch.bfloat16)
    got = ops.topk_routing(x, 2, renormalize=True)
    for start in (0, (1 << 25) - 500, tokens - 900):
        want = ops.topk_routing(x[start:start + 900], 2, renormalize=True)
        assert all(torch.equal(a[start:start + 900], b) for a, b in zip(got, want))
    check(x[-64:].cpu(), 2, "softmax", True, None)


@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 4), (5, 2)])
def test_offsets_past_32_bits(groups, kept):
    from sonar_amd import ops
    tokens, experts = 8400000, 260 if groups == 5 else 256
    x = torch.empty((tokens, experts), device=DEV, dtype=torch.bfloat16).normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    bias = torch.linspace(-0.1, 0.1, experts, device=DEV)
    args = 8, "sigmoid", True, bias, groups, kept, 2.5
    got = ops.topk_routing(x, *args)
    for start in (0, tokens // 2, tokens - 5000):
        want = ops.topk_routing(x[start:start + 5000], *args)
        assert all(torch.equal(a[start:start + 5000], b) for a, b in zip(got, want))


def test_a_bias_that_masks():
    """Experts that the bias switches off, and choices that differ in the last bits of the sum."""
    x, _ = make(8, 12, 64)
    bias = torch.zeros(64)
    bias[::3] = -float("inf")
    bias[1] = float("nan")
    check(x, 6, "sigmoid", True, bias)
    check(x, 6, "softmax", True, bias)
    check(x, 6, "sigmoid", True, bias, 8, 4)
    x[:, 1:] = x[:, :1] + torch.arange(63) * 2.0 ** -22
    check(x, 8, "sigmoid", True, torch.full((64,), 100.0))
    check(x, 8, "sigmoid", True, -torch.sigmoid(x[0].double()).float())


def test_views():
    from sonar_amd import ops
    x, bias = make(4, 20, 48, "bf16", True)
    wide = torch.zeros((20, 100), dtype=torch.bfloat16, device=DEV)
    wide[:, 3:51] = x.to(DEV)
    check(x, 4, "softmax", True, bias, given=wide[:, 3:51])
    check(x, 4, "softmax", True, bias, given=x.to(DEV).t().contiguous().t())
    check(x[:1].expand(7, 48), 4, "softmax", True, bias, given=x.to(DEV)[:1].expand(7, 48))
    check(x[::3], 4, "softmax", True, bias, given=x.to(DEV)[::3])
    w, ids = ops.topk_routing(x.to(DEV)[:0], 4)
    assert w.shape == ids.shape == (0, 4)
    single = torch.randn((9, 1), device=DEV)
    check(single.cpu(), 1, "sigmoid", False, None, given=single)


def test_refusals():
    from sonar_amd import ops
    x = torch.zeros((4, 64), device=DEV)
    f = ops.topk_routing
    for call, message in (
            (lambda: f(x, 0), "topk"), (lambda: f(x, 65), "topk"), (lambda: f(x, -1), "topk"), (lambda: f(x, 4, "tanh"), "scoring_func"),
            (lambda: f(x[0], 4), "tokens, experts"), (lambda: f(x.double(), 4), "float32"), (lambda: f(x, 4, bias=torch.zeros(63, device=DEV)), "bias"),
            (lambda: f(x, 4, bias=torch.zeros(64, device=DEV).half()), "bias"), (lambda: f(x, 4, bias=torch.zeros(64)), "bias"),
            (lambda: f(x, 4, num_expert_group=7), "groups"), (lambda: f(x, 4, num_expert_group=8, topk_group=9), "kept_groups"),
            (lambda: f(x, 9, num_expert_group=8, topk_group=1), "topk"), (lambda: f(torch.zeros((4, 1025), device=DEV), 4), "experts"),
            (lambda: f(x[:, :0], 1), "experts")):
        with pytest.raises(RuntimeError, match=message):
            call()


def test_the_host_functions():
    from sonar_amd.fused_moe import fused_topk, grouped_topk
    x, bias = make(6, 10, 64, "bf16", True)
    h = torch.empty((10, 8), device=DEV)
    for args, want in ((fused_topk(h, x.to(DEV), 4, True), lo.topk_routing(x.double().numpy(), 4, "softmax", True)),
                       (fused_topk(h, x.to(DEV), 4, False, "sigmoid", bias.to(DEV)),
                        lo.topk_routing(x.double().numpy(), 4, "sigmoid", False, bias.double().numpy())),
                       (grouped_topk(h, x.to(DEV), 6, True, 8, 3, "sigmoid", 2.5, bias.to(DEV)),
                        lo.topk_routing(x.double().numpy(), 6, "sigmoid", True, bias.double().numpy(), 8, 3, 2.5))):
        assert np.array_equal(args[1].cpu().numpy(), want[1])
        np.testing.assert_allclose(args[0].cpu().double().numpy(), want[0], rtol=RTOL)


def test_streams_and_graph():
    from sonar_amd import ops
    x, bias = make(2, 100, 256, "fp32", True)
    dx, db = x.to(DEV), bias.to(DEV)
    def call():
        return ops.topk_routing(dx, 8, "sigmoid", True, db, 8, 4, 2.5)
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for seed in range(3):
        dx.copy_(make(seed, 100, 256)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, call()))
