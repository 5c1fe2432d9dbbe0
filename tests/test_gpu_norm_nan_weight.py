"""GPU: numbers of the norm's weight that are none.  y = z * r * weight: a NaN in the weight makes one in every row (also
where z is 0), an infinity makes an infinity in every row where z is not 0, else a NaN.  A row's scale goes by its largest
magnitude, so that it says so: NaN, or infinite."""
import numpy as np
import pytest
import torch

from oracle import layer_oracle as lo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
EPS = 1e-5


def make(rows, cols, dtype, residual):
    gen = torch.Generator().manual_seed(rows + cols)
    x = torch.randn((rows, cols), generator=gen).to(DTYPES[dtype])
    w = (1 + 0.3 * torch.randn(cols, generator=gen)).to(DTYPES[dtype])
    return x, w, torch.randn((rows, cols), generator=gen).to(DTYPES[dtype]) if residual else None


# every width of a row's threads, and columns that no vector fits
SHAPES = [(3, 1), (3, 8), (5, 64), (5, 512), (3, 1000), (600, 1024), (3, 2048), (3, 4096), (3, 4100), (3, 4099), (3, 8192), (3, 16384), (3, 20000)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_a_nan_in_the_weight(rows, cols, dtype, code):
    from sonar_amd import ops
    for at in {0, cols // 2, cols - 1}:
        x, w, res = make(rows, cols, dtype, at == 0)
        x[1, at] = 0
        w[at] = float("nan")
        q, scales, z, y = ops.rms_norm_per_token_quant(x.to(DEV), w.to(DEV), EPS, CODES[code], None if res is None else res.to(DEV), True)
        assert torch.isnan(scales).all()
        # codes that stand for no number, as a row whose z holds a NaN has them: 0, or the type's NaN
        assert (q == 0).all() if code == "int8" else torch.isnan(q.float()).all()
        _, want = lo.rms_norm(x.double().numpy(), w.double().numpy(), EPS, None if res is None else res.double().numpy(), dtype)
        got = y.cpu().double().numpy()
        assert np.isnan(got[:, at]).all() and np.array_equal(np.isnan(got), np.isnan(want))


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_an_infinity_in_the_weight(rows, cols, dtype, code):
    from sonar_amd import ops
    x, w, _ = make(rows, cols, dtype, False)
    at = cols // 2
    x[:, at] = 1
    x[1, at] = 0
    w[at] = -float("inf")
    q, scales, _, y = ops.rms_norm_per_token_quant(x.to(DEV), w.to(DEV), EPS, CODES[code], None, True)
    others = [r for r in range(rows) if r != 1]
    assert torch.isnan(scales[1]).all() and (scales[others] == float("inf")).all()
    assert torch.isnan(y[1, at]) and (y[others, at] == -float("inf")).all()
    # y times 1 / infinity: 0, and of the infinity itself no number
    codes = q.float().cpu()[others]
    assert (np.delete(codes.numpy(), at, 1) == 0).all()
    assert (codes[:, at] == 0).all() if code == "int8" else torch.isnan(codes[:, at]).all()


@pytest.mark.parametrize("cols", [64, 4096, 4099, 20000])
@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_codes_of_rows_that_hold_no_number(cols, code):
    """An infinity or a NaN in z: the scale NaN and no code that stands for a number; rows beside it keep theirs."""
    from sonar_amd import ops
    x, w, _ = make(6, cols, "bf16", False)
    want = ops.rms_norm_per_token_quant(x.to(DEV), w.to(DEV), EPS, CODES[code])
    x[1, 0] = float("nan")
    x[4, cols - 1] = float("inf")
    q, scales, _, _ = ops.rms_norm_per_token_quant(x.to(DEV), w.to(DEV), EPS, CODES[code])
    assert torch.isnan(scales[[1, 4]]).all()
    assert (q[[1, 4]] == 0).all() if code == "int8" else torch.isnan(q.float()[[1, 4]]).all()
    others = [0, 2, 3, 5]
    assert torch.equal(q.view(torch.int8)[others], want[0].view(torch.int8)[others]) and torch.equal(scales[others], want[1][others])
