"""GPU: the norm with 8-bit codes against the 64-bit oracle.

Tolerances, with u = 2^-24 (half a step of float32): y = z * r * weight has three roundings (r, and two products), so it is
within 3u of the exact y; a maximum is as close, the scale rounds once more (int8: 4u; fp8: 4u).  An int8 code comes from
y * (127 / max): 3u + 3u + u + u of at most 127, and half is added in float32 (2^-18), so that it lies within
0.5 + 127 * 8u + 2^-18 < 0.5 + 2^-13 of the exact y over the exact scale.  An fp8 code is the number nearest to a value that
is within 8u: 2^-4 of it, or 2^-10 among the smallest."""
import numpy as np
import pytest
import torch

from oracle import layer_oracle as lo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
HALF_STEP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}
SMALLEST = {"fp16": 2.0 ** -25, "bf16": 0.0, "fp32": 0.0}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
EPS = 1e-5


def numbers(t):
    return t.detach().cpu().double().numpy()


def make(seed, rows, cols, dtype, residual=True):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=gen).to(DTYPES[dtype])
    w = (1 + 0.3 * torch.randn(cols, generator=gen)).to(DTYPES[dtype])
    res = (torch.randn((rows, cols), generator=gen) * 3).to(DTYPES[dtype]) if residual else None
    return x, w, res


def check(got, x, w, res, dtype, code, norm):
    q, scales, z, y = got
    assert q.dtype == CODES[code] and q.shape == x.shape and scales.dtype == torch.float32
    assert scales.shape == x.shape[:-1] + (1,) and (z is None) == (res is None) and (y is None) == (not norm)
    want_z, want_y = lo.rms_norm(numbers(x), numbers(w), EPS, None if res is None else numbers(res), dtype)
    if res is not None:
        assert np.array_equal(numbers(z), want_z)
    want_s = lo.scales_of(want_y, code)
    np.testing.assert_allclose(numbers(scales), want_s, rtol=4.01 * U, atol=0)
    t = want_y / want_s
    if code == "int8":
        assert np.abs(q.cpu().numpy() - t).max() <= 0.5 + 2 ** -13
    else:
        off = np.abs(numbers(q.float()) - t)
        assert (off <= np.maximum(np.abs(t) * 2 ** -4, 2 ** -10) + 448 * 8 * U).all()
    if norm:
        assert (np.abs(numbers(y) - want_y) <= np.abs(want_y) * (HALF_STEP[dtype] + 3.01 * U) + SMALLEST[dtype]).all()


def to_dev(*tensors):
    return [None if t is None else t.to(DEV) for t in tensors]


# lengths of one and around every width that the kernel takes at once; 4096 and 2880 as in a decoder; past the registers
COLS = [1, 2, 7, 8, 63, 64, 65, 255, 256, 264, 504, 512, 513, 1000, 1024, 2040, 2048, 2056, 2880, 4096, 4104, 8192, 16384, 16392, 20001]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_every_length(cols, dtype):
    from sonar_amd import ops
    for i, (code, residual, norm) in enumerate([("int8", True, False), ("fp8", True, True), ("int8", False, True), ("fp8", False, False)]):
        for rows in (1, 5):
            x, w, res = make(cols + i, rows, cols, dtype, residual)
            dx, dw, dres = to_dev(x, w, res)
            check(ops.rms_norm_per_token_quant(dx, dw, EPS, CODES[code], dres, norm), x, w, res, dtype, code, norm)
            assert torch.equal(dx.cpu(), x) and (res is None or torch.equal(dres.cpu(), res))


@pytest.mark.parametrize("rows", [2, 3, 4, 17, 255, 1000, 5000])
@pytest.mark.parametrize("cols", [64, 128, 520, 768])
def test_many_rows(rows, cols):
    from sonar_amd import ops
    x, w, res = make(rows + cols, rows, cols, "bf16")
    dx, dw, dres = to_dev(x, w, res)
    check(ops.rms_norm_per_token_quant(dx, dw, EPS, torch.int8, dres, True), x, w, res, "bf16", "int8", True)


@pytest.mark.parametrize("rows,cols", [(131081, 64), (131081, 520), (32773, 1032), (32773, 2056), (32773, 4104), (517, 8200), (1030, 20000), (5000, 77)])
@pytest.mark.parametrize("residual", [False, True])
def test_more_rows_than_workgroups(rows, cols, residual):
    """Workgroups that go on to further rows: bit for bit what the rows give in pieces that the grid holds."""
    from sonar_amd import ops
    gen = torch.Generator(device=DEV).manual_seed(cols)
    x = torch.randn((rows, cols), generator=gen, device=DEV, dtype=torch.bfloat16)
    w = torch.randn(cols, generator=gen, device=DEV, dtype=torch.bfloat16)
    res = torch.randn((rows, cols), generator=gen, device=DEV, dtype=torch.bfloat16) if residual else None
    got = ops.rms_norm_per_token_quant(x, w, EPS, torch.int8, res, True)
    some = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device=DEV)
    check([None if t is None else t[some] for t in got], x[some].cpu(), w.cpu(), res[some].cpu() if residual else None, "bf16", "int8", True)
    step = rows // 5 if cols > 77 else 500
    if cols > 8192:
        step = 200
    for i in range(0, rows, step):
        want = ops.rms_norm_per_token_quant(x[i:i + step], w, EPS, torch.int8, res[i:i + step] if residual else None, True)
        for a, b in zip(got, want):
            assert a is None and b is None or torch.equal(a[i:i + step], b)


@pytest.mark.parametrize("rows,cols", [(600000, 4096), (2150000, 1003)])
def test_offsets_past_32_bits(rows, cols):
    from sonar_amd import ops
    x = torch.empty((rows, cols), device=DEV, dtype=torch.float16).normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    w = torch.ones(cols, device=DEV, dtype=torch.float16)
    got = ops.rms_norm_per_token_quant(x, w, EPS, torch.int8, x, True)
    for start in (0, rows // 2, rows - 50):
        want = ops.rms_norm_per_token_quant(x[start:start + 50], w, EPS, torch.int8, x[start:start + 50], True)
        for a, b in zip(got, want):
            assert torch.equal(a[start:start + 50], b)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("cols,pitch,shift", [(512, 520, 0), (512, 513, 0), (512, 512, 1), (500, 512, 4), (4096, 4100, 0), (24, 64, 8)])
def test_strides_and_alignment(dtype, cols, pitch, shift):
    """Rows that lie apart, and rows that no vector is aligned to: the results of the same numbers packed."""
    from sonar_amd import ops
    x, w, res = make(cols + pitch, 6, cols, dtype)
    def spread(t):
        store = torch.full((6 * pitch + shift + 8,), 7.0, dtype=t.dtype, device=DEV)
        view = store[shift:shift + 6 * pitch].view(6, pitch)[:, :cols]
        view.copy_(t)
        return view
    dw = torch.empty(cols + 1, dtype=w.dtype, device=DEV)[1:]
    dw.copy_(w)
    got = ops.rms_norm_per_token_quant(spread(x), dw, EPS, torch.int8, spread(res), True)
    want = ops.rms_norm_per_token_quant(*to_dev(x, w), EPS, torch.int8, res.to(DEV), True)
    check(got, x, w, res, dtype, "int8", True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_other_views():
    from sonar_amd import ops
    x, w, res = make(3, 6, 96, "bf16")
    dx, dw, dres = to_dev(x, w, res)
    want = ops.rms_norm_per_token_quant(dx, dw, EPS, torch.int8, dres)
    got = ops.rms_norm_per_token_quant(dx.view(2, 3, 96), dw, EPS, torch.int8, dres.view(2, 3, 96))
    assert got[0].shape == (2, 3, 96) and got[1].shape == (2, 3, 1)
    turned = ops.rms_norm_per_token_quant(dx.t().contiguous().t(), dw, EPS, torch.int8, dres.t().contiguous().t())
    for a, b, c in zip(want[:3], got[:3], turned[:3]):
        assert torch.equal(a.view(6, -1), b.view(6, -1)) and torch.equal(a, c)
    one = ops.rms_norm_per_token_quant(dx[:1].expand(4, 96), dw, EPS, torch.int8, dres[:1].expand(4, 96))
    assert torch.equal(one[0], want[0][:1].expand(4, 96))
    vector = ops.rms_norm_per_token_quant(dx[0], dw, EPS, torch.int8, dres[0])
    assert vector[0].shape == (96,) and vector[1].shape == (1,) and torch.equal(vector[0], want[0][0])
    none = ops.rms_norm_per_token_quant(dx[:0], dw, EPS, torch.int8, dres[:0], True)
    assert [tuple(t.shape) for t in none] == [(0, 96), (0, 1), (0, 96), (0, 96)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("cols", [64, 512, 4096, 4099])
@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_zeros_extremes_and_numbers_that_are_none(dtype, cols, code):
    """Rows of zeros stay zeros; rows of numbers whose squares no float32 holds do not overflow on the way (the mean square
    is taken in 64 bits); an infinity or a NaN marks its row's scale, and no other row."""
    from sonar_amd import ops
    t = DTYPES[dtype]
    x, w, _ = make(9, 7, cols, dtype, False)
    x[0] = 0
    x[1] = torch.finfo(t).max if dtype == "fp16" else 2.0 ** 120
    x[2] = 0
    x[2, cols // 3] = -torch.finfo(t).max
    x[3, cols - 1] = float("inf")
    x[4, 0] = float("nan")
    x[5] = torch.finfo(t).smallest_normal
    dx, dw = to_dev(x, w)
    q, scales, _, y = ops.rms_norm_per_token_quant(dx, dw, EPS, CODES[code], None, dtype != "fp16")
    assert torch.isnan(scales[[3, 4]]).all() and torch.isfinite(scales[[0, 1, 2, 5, 6]]).all()
    fine = [0, 1, 2, 5, 6]
    check((q[fine], scales[fine], None, None if y is None else y[fine]), x[fine], w, None, dtype, code, y is not None)
    assert q[0].float().abs().max() == 0


def test_the_64_bit_mean():
    """Numbers whose squares' mean would lose its last digits in 32 bits: one large, many small."""
    from sonar_amd import ops
    cols = 8192
    x = torch.full((2, cols), 0.0625, dtype=torch.float32)
    x[0, 0] = 4096.0
    w = torch.ones(cols)
    got = ops.rms_norm_per_token_quant(*to_dev(x, w), EPS, torch.int8, None, True)
    check(got, x, w, None, "fp32", "int8", True)


@pytest.mark.parametrize("cols", [96, 4096, 4097, 16392])
def test_in_place_through_the_c_abi(cols):
    """residual_out over the residual, or over x: the row's own numbers, nothing behind them."""
    from sonar_amd import _lib
    from tests import gpu_util as gu
    lib = _lib.load_layer()
    for over in ("residual", "x"):
        x, w, res = make(cols, 5, cols, "bf16")
        store = torch.full((3, 7, cols), 5.0, dtype=torch.bfloat16, device=DEV)
        store[0, :5], store[1, :5] = x.to(DEV), res.to(DEV)
        q = torch.zeros((7, cols), dtype=torch.int8, device=DEV)
        scales = torch.zeros(7, device=DEV)
        dw = w.to(DEV)
        out = store[1] if over == "residual" else store[0]
        _lib.check_layer(lib.sonar_rms_norm_per_token_quant(
            gu.ptr(store[0]), cols, gu.ptr(store[1]), cols, gu.ptr(dw), gu.ptr(out), None, gu.ptr(q), _lib.ADTYPE_INT8,
            gu.ptr(scales), _lib.DTYPE_BF16, 5, cols, EPS, gu.stream()))
        check((q[:5], scales[:5].view(5, 1), out[:5], None), x, w, res, "bf16", "int8", False)
        assert (store[:, 5:] == 5).all() and (q[5:] == 0).all() and (scales[5:] == 0).all()


def test_refusals():
    from sonar_amd import ops
    x, w, res = to_dev(*make(1, 4, 64, "bf16"))
    f = ops.rms_norm_per_token_quant
    for call, message in (
            (lambda: f(x, w[:32], EPS), "weight"), (lambda: f(x, w.float(), EPS), "weight"), (lambda: f(x, w.cpu(), EPS), "weight"),
            (lambda: f(x, w, EPS, torch.int32), "quant_dtype"), (lambda: f(x, w, EPS, torch.int8, res[:3]), "residual"),
            (lambda: f(x, w, EPS, torch.int8, res.half()), "residual"), (lambda: f(x, w, 0.0), "epsilon"),
            (lambda: f(x.to(torch.float64), w, EPS), "float32"), (lambda: f(x[:, :0], w[:0], EPS), "last dimension")):
        with pytest.raises(RuntimeError, match=message):
            call()


def test_streams_and_graph():
    from sonar_amd import ops
    x, w, res = to_dev(*make(2, 33, 2880, "bf16"))
    want = ops.rms_norm_per_token_quant(x, w, EPS, torch.int8, res, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rms_norm_per_token_quant(x, w, EPS, torch.int8, res, True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.rms_norm_per_token_quant(x, w, EPS, torch.int8, res, True)
    for seed in range(3):
        x.copy_(make(seed, 33, 2880, "bf16")[0])
        graph.replay()
        torch.cuda.synchronize()
        want = ops.rms_norm_per_token_quant(x, w, EPS, torch.int8, res, True)
        assert all(torch.equal(a, b) for a, b in zip(held, want))
