"""GPU: the product of 8-bit integers against the 64-bit oracle.

The sum is exact.  With u = 2^-24: the sum as a float32 u, the product of the scales u, their product u, the addition of the
bias u of the result, and the result's own rounding half a step: |off| <= 3.01u |product| + (u + half a step) |result| (1 + 2^-8),
and 2^-25 where float16 has no smaller number."""
import numpy as np
import pytest
import torch

from oracle import layer_oracle as lo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def make(seed, m, k, n, dtype, bias, low=-128, high=128):
    rng = np.random.default_rng(seed)
    a = rng.integers(low, high, (m, k), dtype=np.int64).astype(np.int8)
    b = rng.integers(low, high, (n, k), dtype=np.int64).astype(np.int8)
    sa = (rng.random((m, 1)) * 0.02 + 0.001).astype(np.float32)
    sb = (rng.random(n) * 1e-3 + 1e-4).astype(np.float32)
    add = torch.from_numpy(rng.standard_normal(n)).to(DTYPES[dtype]) if bias else None
    return a, b, sa, sb, add


def dev(x):
    return None if x is None else (torch.from_numpy(x) if isinstance(x, np.ndarray) else x).to(DEV)


def check(c, a, b, sa, sb, add, dtype):
    product = lo.scaled_mm_int8(a, b, sa, sb)
    want = product if add is None else product + add.double().numpy()
    got = c.cpu().double().numpy()
    tol = 3.01 * U * np.abs(product) + (U + HALF_STEP[dtype]) * np.abs(want) * (1 + 2 ** -8) + (2 ** -25 if dtype == "fp16" else 0)
    off = np.abs(got - want)
    assert got.shape == want.shape and (off <= tol).all(), (off - tol).max()


def run(m, k, n, dtype="bf16", bias=False, seed=0, **kw):
    from sonar_amd import ops
    a, b, sa, sb, add = make(seed + m + 3 * k + 7 * n, m, k, n, dtype, bias, **kw)
    c = ops.scaled_mm_int8(dev(a), dev(b).t(), dev(sa), dev(sb), DTYPES[dtype], dev(add))
    check(c, a, b, sa, sb, add, dtype)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 300, 520])
@pytest.mark.parametrize("k,n", [(256, 256), (1040, 272), (512, 1000)])
def test_rows(m, k, n):
    run(m, k, n, "bf16" if m % 2 else "fp16", bias=m % 3 == 0)


@pytest.mark.parametrize("k", [1, 2, 15, 16, 17, 31, 32, 48, 64, 100, 112, 127, 128, 129, 144, 256, 272, 1003, 4096, 4112, 14336])
@pytest.mark.parametrize("m", [1, 16, 40, 130])
def test_depths(k, m):
    run(m, k, 192, "fp16" if k % 2 else "bf16", bias=k % 3 == 0)


@pytest.mark.parametrize("n", [1, 2, 3, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1537])
@pytest.mark.parametrize("m", [1, 20, 70, 260])
@pytest.mark.parametrize("k", [272, 203])
def test_columns(n, m, k):
    run(m, k, n, "fp16" if n % 2 else "bf16", bias=n % 2 == 0)


@pytest.mark.parametrize("m,k,n", [(1, 4096, 4096), (16, 4096, 6144), (64, 2880, 5760), (200, 4096, 6144), (333, 2880, 5760),
                                   (700, 14336, 512), (1500, 1024, 4096), (2050, 4096, 1030), (77, 1003, 1537), (200, 1003, 1537)])
def test_larger(m, k, n):
    run(m, k, n, bias=True)


FORMS = {0: 1 << 20, 1: 16, 2: 16, 3: 1 << 20, 4: 1 << 20, 5: 1 << 20, 6: 1 << 20, 7: 1 << 20, 8: 1 << 20}   # and the rows each takes


@pytest.fixture
def force():
    from sonar_amd import _lib
    lib = _lib.load_layer()
    yield lambda form, splits=1: _lib.check_layer(lib.sonar_debug_int8_form(form, splits))
    lib.sonar_debug_int8_form(-1, 1)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_every_form(form, dtype, force):
    """Each kernel form at sizes around its tile, K shorter than its ring, K that ends inside a round, and at each of
    them with and without aligned rows."""
    force(form)
    for m in (1, 16, 32, 63, 65, 129, 257, 300):
        if m > FORMS[form]:
            continue
        for k in (16, 64, 112, 128, 256, 272, 400, 1024, 1040, 2944, 203):
            for n in (40, 264):
                run(m, k, n, dtype, bias=(m + k) % 2 == 0, seed=form)


@pytest.mark.parametrize("form", [4, 5, 6, 7, 8])
@pytest.mark.parametrize("splits", [2, 3, 5, 8])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_split_sums(form, splits, dtype, force):
    """K in parts that its rounds do not divide into evenly."""
    force(form, splits)
    for m, k, n in ((70, 512 * splits, 136), (33, 512 * splits + 16, 300), (130, 4400, 72), (40, 600 * splits + 3, 130)):
        run(m, k, n, dtype, bias=True)


def test_a_form_with_too_few_rows_is_refused(force):
    force(2)
    with pytest.raises(RuntimeError, match="rows"):
        run(17, 64, 64)


def test_extremes_of_the_sum():
    """Every product 128 * 128, over the deepest K: 2^31 - 2^14 is the largest sum that 32 bits hold; and its opposite."""
    from sonar_amd import ops
    for m in (3, 33, 130):
        for k in (131071, 131056):
            a = np.full((m, k), -128, dtype=np.int8)
            b = np.full((40, k), -128, dtype=np.int8)
            b[1::2] = 127
            sa, sb = np.full((m, 1), 2.0 ** -10, dtype=np.float32), np.full(40, 2.0 ** -10, dtype=np.float32)
            c = ops.scaled_mm_int8(dev(a), dev(b).t(), dev(sa), dev(sb), torch.bfloat16)
            check(c, a, b, sa, sb, None, "bf16")


@pytest.mark.parametrize("m", [1, 16, 77, 300])
@pytest.mark.parametrize("lda,ldb,shift", [(300, 300, 0), (257, 300, 0), (272, 259, 0), (256, 256, 1), (256, 256, 4), (272, 288, 16), (264, 264, 8)])
def test_strides_and_alignment(m, lda, ldb, shift):
    """Rows that lie apart and start anywhere; what lies between them is not read into the sums."""
    from sonar_amd import ops
    k, n = 256, 130
    a, b, sa, sb, add = make(m + lda + ldb, m, k, n, "bf16", True)
    def spread(x, pitch):
        store = torch.full((x.shape[0] * pitch + shift,), 77, dtype=torch.int8, device=DEV)
        view = store[shift:].view(-1, pitch)[:, :k]
        view.copy_(dev(x))
        return view
    c = ops.scaled_mm_int8(spread(a, lda), spread(b, ldb).t(), dev(sa), dev(sb), torch.bfloat16, dev(add))
    check(c, a, b, sa, sb, add, "bf16")


def test_one_scale_and_shapes():
    from sonar_amd import ops
    a, b, sa, sb, add = make(5, 12, 64, 48, "fp16", True)
    da, db = dev(a), dev(b).t()
    one_a, one_b = torch.tensor([0.25], device=DEV), torch.tensor(0.5, device=DEV)
    c = ops.scaled_mm_int8(da, db, one_a, one_b, torch.float16, dev(add))
    check(c, a, b, np.full((12, 1), 0.25, np.float32), np.full(48, 0.5, np.float32), add, "fp16")
    want = ops.scaled_mm_int8(da, db, dev(sa), dev(sb), torch.float16, dev(add))
    got = ops.scaled_mm_int8(da.view(3, 4, 64), db, dev(sa).view(3, 4, 1), dev(sb).view(1, 48), torch.float16, dev(add))
    assert got.shape == (3, 4, 48) and torch.equal(got.view(12, 48), want)
    strided = torch.stack([dev(sa).view(-1), dev(sa).view(-1)], 1)[:, 0]
    assert torch.equal(ops.scaled_mm_int8(da, db, strided, dev(sb), torch.float16, dev(add)), want)
    assert torch.equal(ops.scaled_mm_int8(da.t().contiguous().t(), db, dev(sa), dev(sb), torch.float16, dev(add)), want)
    row = ops.scaled_mm_int8(da[0], db, dev(sa)[0], dev(sb), torch.float16, dev(add))
    assert row.shape == (48,) and torch.equal(row, want[0])
    same = ops.scaled_mm_int8(da[:1].expand(5, 64), db, dev(sa)[:1], dev(sb), torch.float16, dev(add))
    assert torch.equal(same, want[:1].expand(5, 48))


def test_empty():
    from sonar_amd import ops
    i8 = dict(dtype=torch.int8, device=DEV)
    one = torch.ones(1, device=DEV)
    assert ops.scaled_mm_int8(torch.zeros((0, 64), **i8), torch.zeros((48, 64), **i8).t(), one, one, torch.bfloat16).shape == (0, 48)
    assert ops.scaled_mm_int8(torch.zeros((5, 64), **i8), torch.zeros((0, 64), **i8).t(), one, one, torch.bfloat16).shape == (5, 0)
    bias = torch.randn(48, device=DEV).to(torch.bfloat16)
    c = ops.scaled_mm_int8(torch.zeros((5, 0), **i8), torch.zeros((48, 0), **i8).t(), one, one, torch.bfloat16, bias)
    assert torch.equal(c, bias.expand(5, 48))


@pytest.mark.parametrize("m,k,n", [(1, 4096, 600000), (40, 4096, 600000), (300, 4096, 600000), (300, 64, 8400000), (70, 63, 33000000), (300, 63, 8400000)])
def test_offsets_past_32_bits(m, k, n):
    """Weights of more than 2^31 bytes, results of more than 2^31 numbers: the first and last channels are those of a call of their own."""
    from sonar_amd import ops
    gen = torch.Generator(device=DEV).manual_seed(m + k)
    a = torch.randint(-127, 128, (m, k), device=DEV, generator=gen, dtype=torch.int8)
    b = torch.randint(-127, 128, (n, k), device=DEV, generator=gen, dtype=torch.int8)
    sa, sb = torch.rand(m, device=DEV, generator=gen), torch.rand(n, device=DEV, generator=gen)
    got = ops.scaled_mm_int8(a, b.t(), sa, sb, torch.bfloat16)
    for start in (0, n // 2 - 100, n - 700):
        want = ops.scaled_mm_int8(a, b[start:start + 700].t(), sa, sb[start:start + 700], torch.bfloat16)
        assert torch.equal(got[:, start:start + 700], want)


def test_scales_that_are_no_numbers():
    """A NaN or infinite scale reaches its own row or column and no other."""
    from sonar_amd import ops
    for m in (8, 200):
        a, b, sa, sb, _ = make(m, m, 128, 144, "bf16", False, low=1, high=100)
        sa[3], sb[7] = np.nan, np.inf
        c = ops.scaled_mm_int8(dev(a), dev(b).t(), dev(sa), dev(sb), torch.bfloat16)
        assert torch.isnan(c[3]).all() and torch.isinf(c[[i for i in range(m) if i != 3], 7]).all()
        c[3], c[:, 7] = 0, 0
        assert torch.isfinite(c).all()


def test_results_beyond_the_type():
    from sonar_amd import ops
    a, b = np.full((2, 256), 127, np.int8), np.full((16, 256), 127, np.int8)
    c = ops.scaled_mm_int8(dev(a), dev(b).t(), torch.ones(1, device=DEV), torch.ones(1, device=DEV), torch.float16)
    assert torch.isinf(c).all()


def test_refusals():
    from sonar_amd import ops
    i8 = dict(dtype=torch.int8, device=DEV)
    a, b, one = torch.zeros((4, 64), **i8), torch.zeros((48, 64), **i8), torch.ones(1, device=DEV)
    f, bf = ops.scaled_mm_int8, torch.bfloat16
    for call, message in (
            (lambda: f(a, b, one, one, bf), "Shape mismatch"), (lambda: f(a, torch.zeros((64, 48), **i8), one, one, bf), "column by column"),
            (lambda: f(a.half(), b.t(), one, one, bf), "int8"), (lambda: f(a, b.t(), one, one, torch.float32), "out_dtype"),
            (lambda: f(a, b.t(), one.expand(3).contiguous(), one, bf), "a_scales"), (lambda: f(a, b.t(), one, one.half(), bf), "b_scales"),
            (lambda: f(a, b.t(), one, one, bf, torch.zeros(48, device=DEV)), "bias"),
            (lambda: f(a, b.t(), one, one, bf, torch.zeros(47, device=DEV, dtype=bf)), "bias"),
            (lambda: f(a, b.t().cpu(), one, one, bf), "device"), (lambda: f(a, b[:1].expand(48, 64).t(), one, one, bf), "column by column"),
            (lambda: f(torch.zeros((1, 131072), **i8), torch.zeros((1, 131072), **i8).t(), one, one, bf), "131072")):
        with pytest.raises(RuntimeError, match=message):
            call()


def test_smaller_scratch_gives_the_same_bits():
    """The C ABI takes any scratch, also none: the sums are integers, so nothing changes but the time."""
    from sonar_amd import _lib
    from tests import gpu_util as gu
    lib = _lib.load_layer()
    for m, k, n in ((1, 4096, 512), (40, 14336, 256), (200, 4096, 1024), (520, 8192, 512), (40, 1003, 300), (100, 14335, 200)):
        a, b, sa, sb, _ = make(m, m, k, n, "bf16", False)
        da, db, dsa, dsb = dev(a), dev(b), dev(sa), dev(sb)
        full = lib.sonar_scaled_mm_int8_scratch_bytes(m, n, k, int(k % 16 == 0))
        results = []
        for size in {0, full // 2 // 16 * 16, full}:
            scratch = torch.full((size + 64,), 99, dtype=torch.uint8, device=DEV)
            c = torch.full((m + 1, n), 3.0, dtype=torch.bfloat16, device=DEV)
            _lib.check_layer(lib.sonar_scaled_mm_int8(
                gu.ptr(da), k, gu.ptr(db), k, gu.ptr(c), gu.ptr(dsa), m, gu.ptr(dsb), n, None, gu.ptr(scratch) if size else None,
                size, _lib.DTYPE_BF16, m, n, k, gu.stream()))
            torch.cuda.synchronize()
            assert (scratch[size:] == 99).all() and (c[m] == 3).all()
            results.append(c[:m])
        assert all(torch.equal(r, results[0]) for r in results)
        check(results[0], a, b, sa, sb, None, "bf16")


def test_streams_and_graphs():
    """Two streams at once, and a graph that is replayed with other inputs, against eager calls."""
    from sonar_amd import ops
    for m in (4, 200):
        a, b, sa, sb, add = make(m, m, 4096, 768, "bf16", True)
        da, db, dsa, dsb, dadd = dev(a), dev(b), dev(sa), dev(sb), dev(add)
        def call():
            return ops.scaled_mm_int8(da, db.t(), dsa, dsb, torch.bfloat16, dadd)
        want = call()
        check(want, a, b, sa, sb, add, "bf16")
        sides = [torch.cuda.Stream(), torch.cuda.Stream()]
        got = []
        for side in sides:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got += [call() for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = call()
        for seed in range(4):
            da.copy_(dev(make(seed, m, 4096, 768, "bf16", False)[0]))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, call())
