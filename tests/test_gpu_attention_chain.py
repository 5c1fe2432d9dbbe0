"""GPU: the attention half of a decoder layer as a server runs it, operator after operator: the norm with 8-bit codes, the int8 qkv
projection, norms and rotation of the heads with the append to the cache, attention over the pages, codes of its output and the int8
output projection; prompts, single tokens, drafted trees, and the single-token step in a graph."""
import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao
from oracle import layer_oracle as lo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HIDDEN, HEADS, KV, DIM, PAGE, PAGES = 512, 8, 2, 64, 16, 40
EPS, BF16 = 1e-5, torch.bfloat16


def numbers(t):
    return t.detach().float().cpu().double().numpy()


class Layer:
    def __init__(self, fp8, seed=1):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        randn = lambda *shape: torch.randn(shape, device=DEV, generator=gen)  # noqa: E731
        self.norm = (1 + 0.2 * randn(HIDDEN)).to(BF16)
        self.q_norm, self.k_norm = (1 + 0.2 * randn(DIM)).to(BF16), (1 + 0.2 * randn(DIM)).to(BF16)
        self.qkv = torch.randint(-127, 128, ((HEADS + 2 * KV) * DIM, HIDDEN), device=DEV, generator=gen, dtype=torch.int8)
        self.o = torch.randint(-127, 128, (HIDDEN, HEADS * DIM), device=DEV, generator=gen, dtype=torch.int8)
        self.qkv_scales, self.o_scales = torch.rand(len(self.qkv), device=DEV, generator=gen) * 1e-3 + 1e-4, torch.rand(HIDDEN, device=DEV, generator=gen) * 1e-3
        from sonar_amd.rotary import rotary_cos_sin
        self.table = rotary_cos_sin(DIM, 512, scaling={"rope_type": "linear", "factor": 2.0}, device=DEV)
        cache = torch.float8_e4m3fn if fp8 else BF16
        both = randn(PAGES, 2, PAGE, KV, DIM).to(cache)   # what was there before: other sequences' numbers
        self.k, self.v = both[:, 0], both[:, 1]
        self.scales = [torch.full((1,), s, device=DEV) if fp8 else None for s in (0.02, 0.01)]
        self.pages = torch.randperm(PAGES, device=DEV, generator=gen).to(torch.int32)[:PAGES // 2 * 2].view(2, -1)   # two sequences

    def slots(self, seq, positions):
        return self.pages[seq].long()[positions // PAGE] * PAGE + positions % PAGE

    def __call__(self, x, positions, slots, lens, starts, tree=None, longest=None):
        from sonar_amd import ops
        codes, scales, _, _ = ops.rms_norm_per_token_quant(x, self.norm, EPS)
        qkv = ops.scaled_mm_int8(codes, self.qkv.t(), scales, self.qkv_scales, BF16)
        q, k, v = (t.unflatten(1, (-1, DIM)) for t in qkv.split([HEADS * DIM, KV * DIM, KV * DIM], dim=1))
        q_out = ops.qk_norm_rope_append(q, k, v, self.k, self.v, slots, positions, self.table, self.q_norm, self.k_norm, EPS,
                                        k_scale=self.scales[0], v_scale=self.scales[1])
        out = ops.paged_attention(q_out, self.k, self.v, self.pages, lens, starts, tree_mask=tree, k_scale=self.scales[0],
                                  v_scale=self.scales[1], max_seq_len=longest)
        codes, scales = ops.per_token_quant_int8(out.flatten(1))
        return qkv, q_out, out, ops.scaled_mm_int8(codes, self.o.t(), scales, self.o_scales, BF16), codes, scales

    def check(self, got, positions, slots, lens, starts, tree=None):
        """Each operator's result from what the one before it left."""
        qkv, q_out, out, y, codes, scales = got
        q, k, v = (numbers(t.unflatten(1, (-1, DIM))) for t in qkv.split([HEADS * DIM, KV * DIM, KV * DIM], dim=1))
        at, table = positions.cpu().numpy(), numbers(self.table)
        half, u = 2.0 ** -8, 2.0 ** -24
        want = ao.qk_norm_rope(q, at, table, numbers(self.q_norm), EPS)
        assert (np.abs(numbers(q_out) - want) <= np.abs(want) * half + 60 * u * np.abs(want).max()).all()
        rows = slots.cpu().numpy()
        written = [numbers(c.reshape(-1, KV, DIM) if c.is_contiguous() else c.contiguous().view(torch.uint8).view(c.dtype).view(-1, KV, DIM))[rows]
                   for c in (self.k, self.v)]
        for x, w, s in ((ao.qk_norm_rope(k, at, table, numbers(self.k_norm), EPS), written[0], self.scales[0]), (v, written[1], self.scales[1])):
            if s is None:
                assert (np.abs(w - x) <= np.abs(x) * half + 60 * u * np.abs(x).max()).all()
            else:   # an e4m3 code of x / scale: 2^-4 of it, 2^-10 among the smallest
                x = np.clip(x / float(s), -448, 448)
                assert (np.abs(w - x) <= np.abs(x) * (2.0 ** -4 + 2 * u) + 2.0 ** -10 + 60 * u * np.abs(x).max()).all()
        k, v = (numbers(c.contiguous().float()) * (1.0 if s is None else float(s)) for c, s in ((self.k, self.scales[0]), (self.v, self.scales[1])))
        want, size, most = ao.paged_attention(numbers(q_out), k, v, self.pages.cpu().numpy(), lens.cpu().numpy(), starts.cpu().numpy(),
                                              DIM ** -0.5, tree=None if tree is None else tree.cpu().numpy())
        e = (DIM + 8) * u * most[:, :, None] + 2.0 ** -22
        assert (np.abs(numbers(out) - want) <= size * (half + 2 * e + 400 * u) + np.abs(want) * half + u).all()
        want = lo.scaled_mm_int8(codes.cpu().numpy(), self.o.cpu().numpy(), numbers(scales), numbers(self.o_scales))
        assert (np.abs(numbers(y) - want) <= np.abs(want) * (half + 2.0 ** -21) + 2.0 ** -25).all()


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def hidden(seed, tokens):
    return torch.randn((tokens, HIDDEN), generator=torch.Generator().manual_seed(seed)).to(BF16).to(DEV)


@pytest.mark.parametrize("fp8", [False, True])
def test_prompts_then_tokens_then_drafts(fp8):
    layer = Layer(fp8)
    lengths = [37, 150]
    at = torch.cat([torch.arange(n, device=DEV) for n in lengths])
    slots = torch.cat([layer.slots(i, torch.arange(n, device=DEV)) for i, n in enumerate(lengths)])
    args = at, slots, ints(*lengths), ints(0, 37, 187)
    layer.check(layer(hidden(1, 187), *args), *args)
    for step in range(3):   # a token each
        at = torch.tensor([n + step for n in lengths], device=DEV)
        slots = torch.cat([layer.slots(i, at[i:i + 1]) for i in range(2)])
        args = at, slots, ints(*(int(p) + 1 for p in at)), ints(0, 1, 2)
        layer.check(layer(hidden(10 + step, 2), *args), *args)
    # six drafts behind each: 0 - 1 - 2, 0 - 3, 4 - 5; a draft's position is its depth
    seen, depth = [0b1, 0b11, 0b111, 0b1001, 0b10000, 0b110000], [0, 1, 2, 1, 0, 1]
    tree = torch.tensor(seen * 2, device=DEV)[:, None]
    at = torch.tensor([n + 3 + d for n in lengths for d in depth], device=DEV)
    slots = torch.cat([layer.slots(i, torch.arange(n + 3, n + 9, device=DEV)) for i, n in enumerate(lengths)])
    args = at, slots, ints(*(n + 9 for n in lengths)), ints(0, 6, 12), tree
    drafted = layer(hidden(20, 12), *args)
    layer.check(drafted, *args)
    # the accepted branch 0 - 3 as two ordinary tokens gives what the tree gave (other sums: within both tolerances)
    x = hidden(20, 12)
    for j, row in enumerate((0, 3)):
        at = torch.tensor([n + 3 + j for n in lengths], device=DEV)
        slots = torch.cat([layer.slots(i, at[i:i + 1]) for i in range(2)])
        got = layer(x[[row, 6 + row]], at, slots, ints(*(int(p) + 1 for p in at)), ints(0, 1, 2))
        assert (got[2].double() - drafted[2][[row, 6 + row]].double()).abs().max() <= 2.0 ** -6 * drafted[2].abs().max()


@pytest.mark.parametrize("fp8", [False, True])
def test_the_single_token_step_in_a_graph(fp8):
    layer, other = Layer(fp8), Layer(fp8)
    at = torch.arange(100, device=DEV).repeat(2)
    slots = torch.cat([layer.slots(i, torch.arange(100, device=DEV)) for i in range(2)])
    for l in (layer, other):
        l(hidden(2, 200), at, slots, ints(100, 100), ints(0, 100, 200))
    x, at, slots, lens, starts = hidden(3, 2), torch.tensor([100, 100], device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV), ints(101, 101), ints(0, 1, 2)
    slots.fill_(-1)   # (the capture appends nothing)
    layer(x, at, slots, lens, starts, longest=150)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer(x, at, slots, lens, starts, longest=150)
    for step in range(5):
        x.copy_(hidden(30 + step, 2))
        at.fill_(100 + step)
        slots.copy_(torch.cat([layer.slots(i, at[i:i + 1]) for i in range(2)]))
        lens.fill_(101 + step)
        graph.replay()
        torch.cuda.synchronize()
        want = other(x, at, slots, lens, starts, longest=150)
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(held, want)):
            assert torch.equal(a, b), (step, i)
        raw = lambda c: c.contiguous().view(torch.uint8)  # noqa: E731
        assert torch.equal(raw(layer.k), raw(other.k)) and torch.equal(raw(layer.v), raw(other.v))
