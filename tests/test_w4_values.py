"""Products with 4-bit weights, number by number: infinities and NaN to the outputs that the formula sends them to, and errors within what the
kernels' own roundings make, without the room that tests/test_w4_ops.py leaves for weights in bf16."""
import pytest
import torch

from pie_b200 import ops

from test_w4_ops import FORMS, expert_case, product_case

IDS = lambda f: f"{f[0]}{'z' if f[1] else ''}-{str(f[2])[6:]}-{f[3]}"


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("m", [2, 8, 12, 24, 40, 300])
def test_infinities_and_nan_go_where_the_formula_sends_them(m, form):
    x, w, _, _, _ = product_case(m, 128, 384, form)
    x[0, 5], x[1, 380] = float("inf"), float("nan")
    want = x.double() @ w.dequant(torch.float64).T
    assert torch.isinf(want[0]).any() and torch.isnan(want[1]).all() and torch.isfinite(want[2:]).all()
    y = ops.gemm_w4(x, w).double()
    sure = torch.isinf(want)
    assert torch.equal(y[sure], want[sure]) and not torch.isfinite(y[0]).any() and torch.isnan(y[1]).all() and torch.isfinite(y[2:]).all()
    ops.check_kernel_status()


def differences(rows, k, gen):
    """Rows with 2^e at one place and -2^e at another: their products are differences of two weights."""
    x = torch.zeros(rows, k)
    at = torch.stack([torch.randperm(k, generator=gen)[:2] for _ in range(rows)])
    size = torch.exp2(torch.randint(-20, 21, (rows,), generator=gen).float())
    x[torch.arange(rows), at[:, 0]], x[torch.arange(rows), at[:, 1]] = size, -size
    return x.bfloat16().cuda()


def assert_differences(y, x, w64, rounded):
    """Few rows: codes and scales are exact, and so is everything for one scale in bf16 times q - 8 (4 + 8 bits, of which the kernel's fp16
    holds 11: |q - 8| is 8 or has three), and for e2m1 times a power of two. Others (`rounded`) are rounded once to fp16, by 2^-11 of the
    weight at most. The sum is of two products: some roundings of 2^-22 of the larger. The output is rounded to bf16 (2^-8). A weight rounded
    to bf16 would be off by up to 2^-8 of it, which is more than all of this for most differences of neighbouring codes."""
    want, size = x.double() @ w64.T, x.double().abs() @ w64.abs().T
    room = size * ((2.0 ** -11 if rounded else 0.0) + 2.0 ** -20)
    off = (y.double() - want).abs() - (room + 2.0 ** -8 * (want.abs() + room))
    assert off.max().item() <= 0, off.max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("m", [1, 5, 8, 13, 16, 30, 40, 100, 128, 300])
def test_differences_of_weights(m, form):
    for n, k in ((384, 640), (136, 4096)):
        _, w, _, _, _ = product_case(m, n, k, form)
        x = differences(m, k, torch.Generator().manual_seed(m))
        w64 = w.dequant(torch.float64)
        exact = (form[0] == "int4" and not form[1] and form[2] == torch.bfloat16) or form[0] == "fp4"
        assert_differences(ops.gemm_w4(x, w), x, w64, not exact and m > w._gpu.rows)
    ops.check_kernel_status()


@pytest.mark.gpu
@pytest.mark.parametrize("form", [FORMS[0], FORMS[2], FORMS[5]], ids=IDS)
def test_differences_of_weights_of_experts(form):
    counts, n, k = [1, 0, 9, 40, 130], 136, 640
    a, w, buf, mt, _, _, _ = expert_case(counts, n, k, form, ops.EPI_STORE)
    a.copy_(differences(a.shape[0], k, torch.Generator().manual_seed(5)))
    exact = form[0] == "fp4" or not form[1]
    for rows in (1, 1 << 40):
        out = torch.zeros(mt * 128, n, device="cuda").bfloat16()
        ops.grouped_gemm(a, w, buf.tile_expert, out, mt, ops.EPI_STORE, buf.tile_list, rows)
        row = 0
        for e, c in enumerate(counts):
            if c:
                assert_differences(out[row:row + c], a[row:row + c], w.dequant(torch.float64)[e], not exact and rows > 1)
            row += -(-c // 128) * 128
    ops.check_kernel_status()
