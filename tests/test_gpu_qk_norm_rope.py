"""GPU: norms, rotation and the append to a paged cache against the 64-bit oracle.

Tolerances, with u = 2^-24 and h half a step of the result's type: a norm's sum of head_dim squares is off by at most head_dim u of
itself, its root by half of that, the root, the quotient and the two products by 5 u more (the root and quotient to a last bit): n =
(head_dim / 2 + 6) u of the number.  A rotated number is a cos - b sin: off by n (|a cos| + |b sin|), and two roundings of the sum and
one product, 3 u of the same.  Then h of itself, or half of the smallest step among the smallest.  A code of an 8-bit cache is
the nearest to a number that is off by that and 2 u (the reciprocal and its product): 2^-4 of it, or 2^-10 among the smallest."""
import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
HALF_STEP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}
SMALLEST = {"fp16": 2.0 ** -25, "bf16": 2.0 ** -134, "fp32": 2.0 ** -150}
U = 2.0 ** -24
EPS = 1e-5
FP8 = torch.float8_e4m3fn


def numbers(t):
    return t.detach().cpu().double().numpy()


def make(seed, tokens, heads, kv_heads, dim, rotary, dtype, weights=True, positions=64, rising=False):
    gen = torch.Generator().manual_seed(seed)
    qkv = (torch.randn((tokens, (heads + 2 * kv_heads) * dim), generator=gen) * 2).to(DTYPES[dtype])
    parts = qkv.to(DEV).split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1)   # views, as a projection leaves them
    q, k, v = (t.unflatten(1, (-1, dim)) for t in parts)
    table = torch.randn((positions, rotary), generator=gen) if rotary else None
    at = torch.arange(tokens) % positions if rising else torch.randint(0, positions, (tokens,), generator=gen)
    w = [(1 + 0.3 * torch.randn(dim, generator=gen)).to(DTYPES[dtype]) if weights else None for _ in range(2)]
    return q, k, v, table, at, w


def limits(x, at, table, weight, half, dim):
    """(exact, what fp32 may be off) of heads x."""
    want = ao.qk_norm_rope(x, at, table, weight, EPS, half)
    plain = np.abs(ao.qk_norm_rope(x, None, None, weight, EPS))
    if table is not None:   # |a cos| + |b sin| and |b cos| + |a sin|, by a turn whose minus is a plus
        size = ao.qk_norm_rope(plain, at, np.abs(table), None, EPS, half)
        rotary = table.shape[1]
        rows = np.abs(table[np.clip(at, 0, len(table) - 1)])[:, None]
        first = np.arange(rotary // 2) if half else np.arange(0, rotary, 2)
        second = first + (rotary // 2 if half else 1)
        size[..., first] = plain[..., first] * rows[..., :rotary // 2] + plain[..., second] * rows[..., rotary // 2:]
    else:
        size = plain
    return want, size * ((dim / 2 + 6) * U * (weight is not None) + 3 * U * (table is not None))


def check(got, want, off, dtype):
    limit = off + np.abs(want) * HALF_STEP[dtype] + SMALLEST[dtype]
    bad = ~((np.abs(numbers(got) - want) <= limit) | (np.isnan(want) & np.isnan(numbers(got))))
    assert got.dtype == DTYPES[dtype] and not bad.any(), np.argwhere(bad)[:5]


def opt(t):
    return None if t is None else numbers(t)


def dev(t):
    return None if t is None else t.to(DEV)


WIDTHS = [(2, 2), (6, 4), (16, 16), (20, 0), (32, 8), (64, 64), (64, 16), (80, 20), (80, 80), (96, 32), (96, 24), (100, 50), (101, 50),
          (112, 112), (128, 128), (128, 64), (128, 2), (192, 192), (256, 256), (256, 0), (256, 10), (512, 512), (520, 516), (1024, 1024),
          (1000, 998)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("dim,rotary", WIDTHS)
def test_widths(dtype, half, dim, rotary):
    from sonar_amd import ops
    for weights in (True, False):
        q, k, _, table, at, w = make(dim + rotary, 7, 5, 3, dim, rotary, dtype, weights)
        got = ops.qk_norm_rope(q, k, dev(at) if rotary else None, dev(table), dev(w[0]), dev(w[1]), EPS, half)
        for x, y, weight in ((q, got[0], w[0]), (k, got[1], w[1])):
            want, off = limits(numbers(x), at.numpy(), opt(table), opt(weight), half, dim)
            assert y.shape == x.shape and y.is_contiguous()
            check(y, want, off, dtype)


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 32, 8), (3, 2, 1), (130, 14, 2), (65, 40, 40), (2000, 3, 1), (33, 128, 8)])
@pytest.mark.parametrize("dim", [64, 128])
def test_counts(tokens, heads, kv_heads, dim):
    from sonar_amd import ops
    q, k, _, table, at, w = make(tokens, tokens, heads, kv_heads, dim, dim, "bf16", positions=4096)
    got = ops.qk_norm_rope(q, k, dev(at).int(), dev(table), dev(w[0]), None, EPS)   # int32 positions, a norm of the queries only
    for x, y, weight in ((q, got[0], w[0]), (k, got[1], None)):
        want, off = limits(numbers(x), at.numpy(), opt(table), opt(weight), True, dim)
        check(y, want, off, "bf16")


@pytest.mark.parametrize("layout", ["transposed heads", "odd token stride", "odd address", "strided numbers", "one token, odd stride"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strides(layout, dtype):
    from sonar_amd import ops
    q, k, _, table, at, w = make(1, 9, 4, 2, 64, 32, dtype)

    def lay(x):
        if layout == "transposed heads":
            return x.transpose(0, 1).contiguous().transpose(0, 1)
        if layout == "odd token stride":
            return torch.nn.functional.pad(x.flatten(1), (0, 3))[:, :-3].unflatten(1, (-1, 64))
        if layout == "odd address":
            return torch.nn.functional.pad(x.flatten(), (1, 0))[1:].view(x.shape)
        if layout == "strided numbers":
            return x.repeat_interleave(2, dim=2)[..., ::2]
        return x
    if layout == "one token, odd stride":
        q, k, at = q[:1].as_strided((1, 4, 64), (777, 64, 1)), k[:1], at[:1]
    got = ops.qk_norm_rope(lay(q), lay(k), dev(at), dev(table), dev(w[0]), dev(w[1]), EPS)
    want = ops.qk_norm_rope(q.contiguous(), k.contiguous(), dev(at), dev(table), dev(w[0]), dev(w[1]), EPS)
    # (the sum of a norm is taken in another order where no vector fits)
    for a, b in zip(got, want):
        assert a.is_contiguous()
        np.testing.assert_allclose(numbers(a), numbers(b), rtol=2 * HALF_STEP[dtype] + 64 * U, atol=64 * U * 8)


def make_caches(seed, pages, page, kv_heads, dim, cache, layout="slots first"):
    gen = torch.Generator().manual_seed(seed)
    shape = (pages, kv_heads, page, dim) if layout == "heads first" else (pages, page, kv_heads, dim)
    if layout == "side by side":   # keys and values of a page behind each other
        both = torch.randn((pages, 2, page, kv_heads, dim), generator=gen).to(cache).to(DEV)
        return both[:, 0], both[:, 1]
    caches = [torch.randn(shape, generator=gen).to(cache).to(DEV) for _ in range(2)]
    return [c.transpose(1, 2) for c in caches] if layout == "heads first" else caches


@pytest.mark.parametrize("dtype,fp8", [("bf16", False), ("fp16", False), ("bf16", True), ("fp16", True), ("fp32", False)])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (80, 20), (96, 32), (100, 50), (101, 50), (128, 128), (256, 128)])
@pytest.mark.parametrize("layout", ["slots first", "heads first", "side by side"])
def test_append(dtype, fp8, dim, rotary, layout):
    from sonar_amd import ops
    tokens, heads, kv_heads, page, pages = 23, 6, 3, 5, 9
    for norm, half, scales in ((True, True, 1), (False, False, kv_heads)):
        q, k, v, table, at, w = make(dim, tokens, heads, kv_heads, dim, rotary, dtype, norm)
        keys, values = make_caches(2, pages, page, kv_heads, dim, FP8 if fp8 else DTYPES[dtype], layout)
        gen = torch.Generator().manual_seed(3)
        slots = torch.randperm(pages * page, generator=gen)[:tokens]
        slots[3], slots[5], slots[6] = -1, pages * page, -(2 ** 40)   # nowhere
        k_scale, v_scale = (torch.rand(scales, generator=gen) * 0.05 + 0.01 if fp8 else None for _ in range(2))
        before = numbers(keys.float()), numbers(values.float())
        got = ops.qk_norm_rope_append(q, k, v, keys, values, dev(slots), dev(at), dev(table), dev(w[0]), dev(w[1]), EPS, half,
                                      dev(k_scale), dev(v_scale))
        want, off = limits(numbers(q), at.numpy(), opt(table), opt(w[0]), half, dim)
        check(got, want, off, dtype)
        want_k, off_k = limits(numbers(k), at.numpy(), opt(table), opt(w[1]), half, dim)
        for cache, old, rows, off, scale in ((keys, before[0], want_k, off_k, k_scale), (values, before[1], numbers(v), 0 * off_k, v_scale)):
            limit = off + np.abs(rows) * HALF_STEP[dtype] + SMALLEST[dtype]
            if fp8:
                by = numbers(scale)[:, None] if scales > 1 else numbers(scale)
                rows, off = np.clip(rows / by, -448, 448), off / by
                limit = off + np.abs(rows) * (2.0 ** -4 + 2 * U) + 2.0 ** -10
            here = numbers(cache.float())
            written = ao.append(np.zeros(old.shape), np.ones_like(rows), slots.numpy()) != 0
            assert np.array_equal(here[~written], old[~written])   # everything else is as it was
            exact, limit = ao.append(old, rows, slots.numpy()), ao.append(np.zeros(old.shape), limit, slots.numpy())
            assert (np.abs(here - exact) <= limit).all()


def test_append_is_the_rotation_and_a_copy():
    from sonar_amd import ops
    q, k, v, table, at, w = make(4, 50, 8, 2, 128, 128, "bf16")
    keys, values = make_caches(5, 8, 16, 2, 128, torch.bfloat16)
    slots = torch.randperm(128)[:50].to(DEV)
    got = ops.qk_norm_rope_append(q, k, v, keys, values, slots.int(), dev(at), dev(table), dev(w[0]), dev(w[1]), EPS)
    want_q, want_k = ops.qk_norm_rope(q, k, dev(at), dev(table), dev(w[0]), dev(w[1]), EPS)
    assert torch.equal(got, want_q) and torch.equal(keys.reshape(128, 2, 128)[slots], want_k)
    assert torch.equal(values.reshape(128, 2, 128)[slots], v)
    # without norm and table: the plain append
    again = ops.qk_norm_rope_append(q, k, v, keys, values, slots)
    assert torch.equal(again, q) and torch.equal(keys.reshape(128, 2, 128)[slots], k)


def test_positions_outside_the_table_and_special_numbers():
    from sonar_amd import ops
    for dim, rotary in ((64, 32), (101, 50)):
        q, k, _, table, at, w = make(6, 6, 4, 2, dim, rotary, "bf16")
        at = torch.tensor([0, 63, 64, -1, 2 ** 40, 5])
        got = ops.qk_norm_rope(q, k, dev(at), dev(table), dev(w[0]), dev(w[1]), EPS)
        for x, y, weight in ((q, got[0], w[0]), (k, got[1], w[1])):
            want, off = limits(numbers(x), at.numpy(), opt(table), opt(weight), True, dim)
            assert np.isnan(want[2:5, :, :rotary]).all() and not np.isnan(want[2:5, :, rotary:]).any()
            off = np.where(np.isnan(off), 0, off)
            check(y, want, off, "bf16")
        # a head's NaN stays in the head; zeros stay zeros; values copy every number that there is
        q = q.clone()
        q[0, 1, 3], q[1] = float("nan"), 0
        y = ops.qk_norm_rope(q, k, dev(torch.zeros(6, dtype=torch.int64)), dev(table), dev(w[0]), dev(w[1]), EPS)[0]
        assert y[0, 1].isnan().all() and not y[0, 0].isnan().any() and not y[0, 2:].isnan().any() and (y[1] == 0).all()
    keys, values = make_caches(5, 2, 4, 2, 64, torch.float16)
    v = torch.tensor([float("inf"), float("-inf"), float("nan"), 0.0, -0.0, 6e-8, 65504.0, 1.0], device=DEV).half().repeat(2, 2, 8)
    slots = torch.tensor([7, 2], device=DEV)
    ops.qk_norm_rope_append(v, v, v, keys, values, slots)
    for c in (keys, values):
        assert torch.equal(c.view(8, 2, 64)[slots].view(torch.int16), v.view(torch.int16))
    keys, values = (c.to(FP8) for c in (keys, values))
    one = torch.ones(1, device=DEV)
    ops.qk_norm_rope_append(v, v, v, keys, values, slots, k_scale=one, v_scale=one)
    got = values.view(8, 2, 64)[slots].float()[0, 0, :8].tolist()
    assert got[:2] == [448, -448] and got[2] != got[2] and got[3:] == [0, 0, 0, 448, 1]


def test_no_tokens_and_no_pages():
    from sonar_amd import ops
    q, k, v, table, at, w = make(4, 3, 8, 2, 64, 64, "fp16")
    got = ops.qk_norm_rope(q[:0], k[:0], dev(at[:0]), dev(table))
    assert got[0].shape == (0, 8, 64) and got[1].shape == (0, 2, 64)
    got = ops.qk_norm_rope(q, k, dev(at), dev(table[:0]))   # no position is in the table
    assert got[0].isnan().all() and got[1].isnan().all()
    keys, values = make_caches(5, 0, 16, 2, 64, torch.float16)
    got = ops.qk_norm_rope_append(q, k, v, keys, values, torch.arange(3, device=DEV), dev(at), dev(table))
    assert torch.equal(got, ops.qk_norm_rope(q, k, dev(at), dev(table))[0])


def test_a_cache_past_32_bits():
    """Slots whose numbers lie more than 2^32 elements behind the cache's start; pages of 2^31 slots in all."""
    from sonar_amd import ops
    q, k, v, table, at, w = make(4, 3, 2, 1, 64, 64, "bf16")
    pages = (1 << 32) // (16 * 64) + 9
    keys = torch.zeros((pages, 16, 1, 64), device=DEV, dtype=FP8)
    values = torch.zeros((pages, 16, 1, 64), device=DEV, dtype=FP8)
    last = pages * 16 - 1
    slots = torch.tensor([last, 5, last - 100], device=DEV)
    one = torch.ones(1, device=DEV)
    ops.qk_norm_rope_append(q, k, v, keys, values, slots, k_scale=one, v_scale=one)
    want = v.float().to(FP8)
    got = values.view(-1, 1, 64).view(torch.uint8)
    assert torch.equal(got[slots].view(FP8).float(), want.float()) and int((got != 0).sum()) <= 3 * 64
    del keys, values, got
    torch.cuda.empty_cache()


def test_more_heads_than_a_launch_has_threads_for():
    """Every head a wavefront, in more wavefronts than 2^32 threads have: odd heads, number by number."""
    from sonar_amd import ops
    tokens, gen = 36_000_000, torch.Generator(device=DEV).manual_seed(3)
    q, k = (torch.randn((tokens, 1, 3), device=DEV, generator=gen, dtype=torch.float16) for _ in range(2))
    got_q, got_k = ops.qk_norm_rope(q, k)
    assert torch.equal(got_q, q) and torch.equal(got_k, k)


def test_one_cache_for_keys_and_values_is_refused():
    from sonar_amd import ops
    x, cache = torch.zeros((2, 2, 64), device=DEV), torch.zeros((4, 16, 2, 64), device=DEV)
    with pytest.raises(RuntimeError, match="(?i)overlap|memory"):
        ops.qk_norm_rope_append(x, x, x, cache, cache, torch.zeros(2, dtype=torch.int64, device=DEV))
