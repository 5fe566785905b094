"""Layer norm gradients of rows whose mean times rstd is no fp32 number."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(3, 1), (5, 8), (70, 37), (9, 200), (33, 1001), (7, 1504), (4, 5001)])
def test_constant_rows_of_large_values(gpu, rows, cols, dtype):
    """Every value is its row's mean: xhat is zero, whatever a place behind the row's end would deviate by."""
    import torch
    t = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    x = torch.full((rows, cols), 2.0 ** 100, device="cuda").to(t)
    x[1] = 3.0
    mean = x[:, 0].float().contiguous()
    rstd = torch.full((rows,), 2.0 ** 30, device="cuda")
    dy = torch.randn((rows, cols), device="cuda").to(t)
    dx, dw, db = torch.empty_like(x), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    gpu.primitives.layer_norm_grad(dy, x, mean, rstd, dx, None, dw, db)
    d = dy.double()
    want = (d - d.mean(1, keepdim=True)) * 2.0 ** 30
    # cols additions for the mean, its product, one difference, the result's rounding.
    unit = 2.0 ** -24 if dtype == "f32" else 2.0 ** -8
    bound = 2.0 ** 30 * (cols + 2) * 2.0 ** -24 * d.abs().mean(1, keepdim=True) + (unit + 2.0 ** -23) * (want.abs() + 2.0 ** 30 * 2.0 ** -20)
    assert ((dx.double() - want).abs() <= bound).all()
    assert not dw.any() and ((db.double() - d.sum(0)).abs() <= (rows + 1) * 2.0 ** -24 * d.abs().sum(0)).all()
