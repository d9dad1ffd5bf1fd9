"""Gates of 8-bit rows far from zero, and gates that are no number, against the formula in 64 bits.

Tolerance.  The exponent, of up to 89, is made with up to eight roundings of 2^-24 of its size, which the exponential turns into
8 * 89 * 2^-24 = 2^-14.5 of its result; its own error, the reciprocal's and the products' are below 2^-20.  So a value is off by at
most 2^-14 of itself, and of its row's largest, which the scale is made of; a code lies within half of the formula's quotient,
plus 127 times both."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SLACK = 2.0 ** -14
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def gates(g, u, act):
    """(codes, scales) of the kernel for g and u [rows, width]."""
    from xeno_rt_b200.csrc import ops
    codes = ops.int8_rows(*g.shape, DEV)
    scales = torch.full((g.shape[0],), 7.0, device=DEV)
    ops.swiglu_int8(codes, scales, torch.cat([g, u], dim=1), act)
    return codes, scales


def formula(g, u, act):
    g, u = g.double(), u.double()
    if not isinstance(act, str):
        g, u = g.clamp(max=act.limit), u.clamp(-act.limit, act.limit)
        return g * torch.sigmoid(act.alpha * g) * (u + 1)
    z = g if act == "silu" else 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)
    return g * torch.sigmoid(z) * u  # (1 + tanh(z)) / 2 is sigmoid(2 z), which 64 bits hold where tanh is near -1


def check(codes, scales, y):
    want = torch.clamp(y.abs().amax(dim=1) / 127, min=2.0 ** -126)
    assert bool(((scales.double() - want).abs() <= want * (SLACK + 2.0 ** -22)).all())
    assert float((codes.double() - y / want[:, None]).abs().max()) <= 0.5 + 127 * (2 * SLACK + 2.0 ** -21)


# gates whose exponent is near that of the smallest sigmoid (of 2^-128, at -88.7; the tanh form's at -10.04)
FAR = {"silu": [-80.0, -87.0, -87.5, -88.0, -88.5], "gelu_tanh": [-9.5, -9.9375, -9.96875, -10.0, -10.03125]}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("rows,width", [(5, 7), (5, 96), (5, 5000), (5, 40000), (600, 4096), (600, 4099)])
def test_gates_alone_in_their_row_far_below_zero(rows, width, act, dtype):
    """Rows all of whose gates are so small that only a large other half keeps them: the largest of them is the scale."""
    at = torch.tensor(FAR[act], device=DEV)
    g = at[torch.arange(rows, device=DEV) % 5][:, None].expand(rows, width).to(DT[dtype]).contiguous()
    u = (100 * (1 + torch.rand(rows, width, generator=torch.Generator().manual_seed(1)))).to(DEV).to(DT[dtype])
    u[:, ::3] *= -1
    codes, scales = gates(g, u, act)
    y = formula(g, u, act)
    assert float((y.abs().amax(dim=1) / 127).min()) > 2.0 ** -126 and bool((codes.abs().amax(dim=1) == 127).all())
    check(codes, scales, y)


@pytest.mark.parametrize("width", [7, 96, 5000])
def test_limited_gates_far_below_zero(width):
    from xeno_rt_b200.csrc import ops
    act = ops.Gate("gated_sigmoid", 200.0, 1.5)
    g = torch.tensor([-50.0, -58.0, -58.5, -59.0], device=DEV)[:, None].expand(4, width).contiguous()
    u = torch.linspace(100, 199, width, device=DEV).expand(4, width).contiguous()
    codes, scales = gates(g, u, act)
    check(codes, scales, formula(g, u, act))


def test_gates_beyond_the_last_one_are_zero():
    g = torch.full((2, 64), -120.0, device=DEV)
    codes, scales = gates(g, torch.ones_like(g), "silu")
    assert not bool(codes.any()) and bool((scales == 2.0 ** -126).all())


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,width", [(8, 7), (8, 96), (8, 5000), (8, 40000), (600, 4096), (600, 4099)])
def test_limited_gates_that_are_no_number_break_their_row(rows, width, dtype, biased):
    """A NaN on either side, and a gate of minus infinity (times sigmoid's 0); infinities that a limit cuts off do not."""
    from xeno_rt_b200.csrc import ops
    act = ops.Gate("gated_sigmoid", 2.0, 1.7, torch.zeros(2 * width, device=DEV) if biased else None)
    gen = torch.Generator().manual_seed(2)
    g, u = (torch.randn(rows, width, generator=gen).to(DEV).to(DT[dtype]) for _ in range(2))
    nan, inf = float("nan"), float("inf")
    g[0, 0], g[1, width - 1], u[2, width // 2], u[3, width - 1], g[4, 3] = nan, nan, nan, nan, -inf
    g[5, 2], u[6, 1], u[7, width - 1] = inf, inf, -inf
    codes, scales = gates(g, u, act)
    assert bool(torch.isnan(scales[:5]).all()) and not bool(codes[:5].any())
    check(codes[5:], scales[5:], formula(g[5:], u[5:], act))
