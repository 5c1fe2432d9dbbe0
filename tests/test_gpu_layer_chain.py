"""GPU: the operators around the GEMMs one after the other, as a decoder layer calls them: the residual's sum, its norm and
codes, the int8 projection and the W4A8 one that read them, the router on the norm's 16-bit copy, and the experts."""
import numpy as np
import pytest
import torch

from oracle import layer_oracle as lo
from oracle import marlin_oracle as mo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HIDDEN, QKV, INTER, EXPERTS, TOPK, GROUP = 512, 768, 256, 16, 4, 128
EPS = 1e-5


class Layer:
    def __init__(self, seed=1):
        from sonar_amd import marlin_utils as mu
        from sonar_amd import ops
        gen = torch.Generator(device=DEV).manual_seed(seed)
        f16 = torch.float16
        self.norm_weight = (1 + 0.2 * torch.randn(HIDDEN, device=DEV, generator=gen)).to(f16)
        self.qkv = torch.randint(-127, 128, (QKV, HIDDEN), device=DEV, generator=gen, dtype=torch.int8)
        self.qkv_scales = torch.rand(QKV, device=DEV, generator=gen) * 1e-3 + 1e-4
        self.gate = torch.randn((EXPERTS, HIDDEN), device=DEV, generator=gen).to(f16) * 0.1
        self.bias = torch.randn(EXPERTS, device=DEV, generator=gen) * 0.05
        def experts(k, n):
            q = torch.randint(-2 ** 31, 2 ** 31 - 1, (EXPERTS, k // 16, 2 * n), dtype=torch.int32, device=DEV, generator=gen)
            return q, (torch.rand((EXPERTS, k // GROUP, n), device=DEV, generator=gen) * 3e-3 + 1e-3).to(f16)
        self.w1, self.s1 = experts(HIDDEN, 2 * INTER)
        self.w2, self.s2 = experts(INTER, HIDDEN)
        # a W4A8 projection of the same codes
        self.made = mo.make_layer(7, HIDDEN, 256, GROUP, "fp16")
        empty = torch.empty(0, dtype=torch.int32, device=DEV)
        self.w4 = ops.gptq_marlin_repack(torch.from_numpy(mo.gptq_pack(self.made["q"])).to(DEV), empty, HIDDEN, 256, 4, True)
        self.ints, self.factor = mo.marlin_act_int8_process_scales(self.made["scales"])
        self.w4_scales = torch.from_numpy(mo.marlin_permute_scales_a8(self.ints, HIDDEN, 256, GROUP).copy()).to(DEV).view(f16)
        self.workspace, self.empty = mu.marlin_make_workspace_new(torch.device(DEV), 4), empty

    def experts(self, y, weights, ids):
        from sonar_amd import fused_moe
        from sonar_amd.scalar_type import scalar_types
        return fused_moe.fused_marlin_moe(y, self.w1, self.w2, None, None, self.s1, self.s2, weights, ids, scalar_types.uint4b8.id)

    def __call__(self, x, residual):
        from sonar_amd import fused_moe, ops
        from sonar_amd.scalar_type import scalar_types
        q, s, z, y = ops.rms_norm_per_token_quant(x, self.norm_weight, EPS, torch.int8, residual, True)
        qkv = ops.scaled_mm_int8(q, self.qkv.t(), s, self.qkv_scales, torch.float16)
        w4a8 = ops.marlin_gemm(q, None, self.w4, None, self.w4_scales, s * float(self.factor), None, self.empty, self.empty, self.empty,
                               self.workspace, scalar_types.uint4b8, q.shape[0], 256, HIDDEN, True, False, True, False)
        logits = torch.nn.functional.linear(y, self.gate)
        weights, ids = fused_moe.grouped_topk(y, logits, TOPK, True, 4, 2, "sigmoid", 2.5, self.bias)
        return q, s, z, y, qkv, w4a8, logits, weights, ids, self.experts(y, weights, ids)


@pytest.fixture(scope="module")
def layer():
    return Layer()


def inputs(seed, tokens):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn((tokens, HIDDEN), generator=gen).half(), (2 * torch.randn((tokens, HIDDEN), generator=gen)).half()


@pytest.mark.parametrize("tokens", [1, 5, 64, 300])
def test_layer(layer, tokens):
    x, residual = inputs(tokens, tokens)
    q, s, z, y, qkv, w4a8, logits, weights, ids, out = layer(x.to(DEV), residual.to(DEV))
    f64 = lambda t: t.cpu().double().numpy()  # noqa: E731
    want_z, want_y = lo.rms_norm(f64(x), f64(layer.norm_weight), EPS, f64(residual), "fp16")
    assert np.array_equal(f64(z), want_z)
    assert (np.abs(f64(y) - want_y) <= np.abs(want_y) * (2.0 ** -11 + 2.0 ** -22) + 2.0 ** -25).all()
    # the codes times their scales: half a code off, so the projection by the sum of the weights' sizes
    want = lo.scaled_mm_int8(q.cpu().numpy(), layer.qkv.cpu().numpy(), f64(s), f64(layer.qkv_scales))
    assert (np.abs(f64(qkv) - want) <= np.abs(want) * (2.0 ** -11 + 2.0 ** -21) + 2.0 ** -25).all()
    dense = want_y @ (f64(layer.qkv) * f64(layer.qkv_scales)[:, None]).T
    most = (0.5 + 2 ** -12) * f64(s) * (np.abs(f64(layer.qkv)).sum(1) * f64(layer.qkv_scales))[None]
    assert (np.abs(f64(qkv) - dense) <= most + np.abs(dense) * 2.0 ** -10).all()
    a_s = (s.cpu().numpy() * np.float32(layer.factor)).astype(np.float32)
    assert np.array_equal(w4a8.float().cpu().numpy(), mo.gemm_w4a8_int8(q.cpu().numpy(), a_s, layer.made["q"], GROUP, layer.ints, "fp16"))
    want_w, want_ids = lo.topk_routing(f64(logits), TOPK, "sigmoid", True, f64(layer.bias), 4, 2, 2.5)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    np.testing.assert_allclose(f64(weights), want_w, rtol=40 * 2.0 ** -24)
    # the experts with the oracle's routing: weights within 40 * 2^-24, so at most the sum's terms round the other way
    again = layer.experts(y, torch.from_numpy(want_w).float().to(DEV), torch.from_numpy(want_ids).to(torch.int32).to(DEV))
    error = (out.double() - again.double()).norm() / again.double().norm()
    assert torch.isfinite(out).all() and error < 2.0 ** -10, error


def test_layer_in_a_graph(layer):
    for tokens in (3, 200):
        x, residual = (t.to(DEV) for t in inputs(0, tokens))
        layer(x, residual)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = layer(x, residual)
        for seed in range(1, 4):
            for t, new in zip((x, residual), inputs(seed, tokens)):
                t.copy_(new)
            graph.replay()
            torch.cuda.synchronize()
            want = layer(x, residual)
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(held, want)):
                assert torch.equal(a, b), i


def test_two_graphs_that_share_a_pool():
    """Replayed in turn, with eager calls between them, each gives what eager calls give."""
    from sonar_amd import ops
    xs, graphs, held = [], [], []
    pool = torch.cuda.graph_pool_handle()
    b = torch.randint(-127, 128, (512, 14336), device=DEV, dtype=torch.int8)
    sb = torch.rand(512, device=DEV)
    w = torch.ones(14336, device=DEV, dtype=torch.bfloat16)
    def call(x):
        q, s, _, y = ops.rms_norm_per_token_quant(x, w, 1e-5, with_norm=True)
        return ops.scaled_mm_int8(q, b.t(), s, sb, torch.bfloat16), *ops.topk_routing(y[:, :256], 8, "sigmoid", True, sb[:256], 8, 4)
    for m in (40, 200):   # (both split K)
        xs.append(torch.randn((m, 14336), device=DEV, dtype=torch.bfloat16))
        call(xs[-1])
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            out = call(xs[-1])
            held.append([t.clone() for t in out])
    for turn in range(4):
        for x, graph, mine in zip(xs, graphs, held):
            x.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(mine, call(x))), turn


def test_opcheck():
    """Schema, fake results, no autograd formula, dynamic shapes: what the ops declare is what they do."""
    from sonar_amd import ops  # noqa: F401
    utils = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")
    x, residual = (t.to(DEV) for t in inputs(0, 6))
    w = torch.ones(HIDDEN, device=DEV, dtype=torch.float16)
    s = torch.ops.sonar_amd
    for res in (None, residual):
        for norm in (False, True):
            torch.library.opcheck(s.rms_norm_per_token_quant, (x, w, res, EPS, torch.int8, norm), test_utils=utils)
    a = torch.randint(-127, 128, (6, HIDDEN), device=DEV, dtype=torch.int8)
    b = torch.randint(-127, 128, (48, HIDDEN), device=DEV, dtype=torch.int8)
    scales = torch.rand(6, device=DEV), torch.rand(48, device=DEV)
    for bias in (None, torch.zeros(48, device=DEV, dtype=torch.bfloat16)):
        torch.library.opcheck(s.scaled_mm_int8, (a, b.t(), *scales, torch.bfloat16, bias), test_utils=utils)
    for bias in (None, torch.zeros(HIDDEN, device=DEV)):
        torch.library.opcheck(s.topk_routing, (x, 4, "sigmoid", True, bias, 8, 2, 1.0), test_utils=utils)
