"""The 8-bit operators against their formulas in 64 bits: rows, gates and norms as integers with a scale a row, and the
product of such rows with 8-bit weights.

Tolerances, derived.  A value y that a kernel computes in 32-bit from inputs of 32 bits or fewer differs from the formula's by
at most ``slack`` of the row's largest value: a plain row 0, a norm 2^-19 (a 32-bit sum of squares of up to 40,000 terms
in partial sums of at most 40 numbers and two trees, then five roundings of 2^-24), a gate 2^-15 (the exponent x, |x| <= 40, is made
with up to eight roundings of 2^-24 of its size, so the exponential is off by 8 |x| units of 2^-24 and 4 of its own, the fast
division by 4, two products by 2; the largest value itself may be off by that too).  A scale is the
largest value over 127, so it is off by the same and one rounding.  A code is the nearest whole number to y / scale, so it lies
within 0.5 of the formula's quotient, plus 127 times the slack of value and scale."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}
TINY = 2.0 ** -126
WIDTHS = [1, 7, 16, 100, 1032, 4096, 5003, 8200, 14336, 16388, 25600, 32769, 40000]


def ops():
    from xeno_rt_b200.csrc import ops as o
    return o


def normal(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV).to(dtype)


def room(rows, width):
    """(codes with poisoned bytes behind every row, scales, the whole buffer)."""
    codes = ops().int8_rows(rows, width, DEV)
    whole = codes.as_strided((rows, codes.stride(0)), (codes.stride(0), 1))
    whole.fill_(77)
    return codes, torch.full((rows,), 7.0, device=DEV), whole


def check_codes(codes, scales, whole, y, slack):
    """codes and scales of the rows y (float64)."""
    width = y.shape[1]
    want = torch.clamp(y.abs().amax(dim=1) / 127, min=TINY)
    # one more rounding, and one step of the numbers below 2^-126 that y may be rounded to
    assert bool(((scales.double() - want).abs() <= want * (slack + 2.0 ** -22)).all())
    off = (codes.double() - y / want[:, None]).abs()
    assert float(off.max()) <= 0.5 + 127 * (2 * slack + 2.0 ** -21)
    assert int(codes.abs().max()) <= 127
    assert bool((whole[:, width:] == 77).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("width", WIDTHS)
def test_rows(width, dtype):
    x = normal(5, width, dtype=DT[dtype])
    x[3] = 0
    codes, scales, whole = room(5, width)
    ops().quantize_rows(codes, scales, x)
    check_codes(codes, scales, whole, x.double(), 0.0)
    assert float(scales[3]) == TINY and not bool(codes[3].any())


def test_ties_go_to_even_and_the_largest_is_127():
    x = torch.tensor([[127.0, -127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, 125.5]], device=DEV)
    codes, scales, _ = room(1, 10)
    ops().quantize_rows(codes, scales, x)
    assert float(scales[0]) == 1.0
    assert codes[0].tolist() == [127, -127, 0, 2, 2, 0, -2, -2, 126, 126]


@pytest.mark.parametrize("rows,width", [(3, 100), (5, 4096), (600, 4096), (500, 8191), (3, 40000)])
def test_rows_are_divided_as_32_bit_numbers_are(rows, width):
    """Of 16-bit values, whose quotients often lie in the middle: the codes of x / scale, rounded, then to even."""
    x = (normal(rows, width, seed=80) * 8).round().to(torch.bfloat16)  # few values, many ties
    codes, scales, _ = room(rows, width)
    ops().quantize_rows(codes, scales, x)
    x = x.float().cpu().numpy()  # (numpy divides; torch multiplies by the inverse of a number)
    scale = np.maximum(np.abs(x).max(axis=1) / np.float32(127), np.float32(TINY))
    assert scale.dtype == np.float32 and np.array_equal(scales.cpu().numpy(), scale)
    assert np.array_equal(codes.cpu().numpy(), np.rint(x / scale[:, None]))


@pytest.mark.parametrize("rows", [1, 3, 700])
@pytest.mark.parametrize("width", [33, 512])
def test_rows_whose_addresses_allow_only_single_values(rows, width):
    buffer = normal(rows * width + 1)
    x = buffer[1:].view(rows, width)  # 4 bytes beyond a 16-byte boundary
    codes, scales, whole = room(rows, width)
    ops().quantize_rows(codes, scales, x)
    check_codes(codes, scales, whole, x.double(), 0.0)


# more rows than blocks: rows that come through a ring, at every 16-byte phase, with rows that begin and end anywhere
MANY = [(700, 4100), (450, 8204), (150, 25604), (3000, 33), (1500, 1600), (1300, 3001), (700, 4096), (1203, 4099), (333, 8190), (150, 14337), (400, 16384), (450, 25600),
        (449, 25001), (301, 26000), (300, 30000), (152, 33000)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,width", MANY)
def test_many_rows(rows, width, dtype):
    x = normal(rows, width, seed=70, dtype=DT[dtype])
    x[rows // 2] = 0
    x[1, width - 1] = float("nan")
    codes, scales, whole = room(rows, width)
    ops().quantize_rows(codes, scales, x)
    assert bool(torch.isnan(scales[1])) and not bool(codes[1].any())
    keep = torch.arange(rows, device=DEV) != 1
    check_codes(codes[keep], scales[keep], whole, x[keep].double(), 0.0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("rows,width", [(1203, 1999), (900, 2052), (700, 4096), (620, 4100), (333, 7005), (301, 14336), (160, 12800), (155, 12801), (151, 20004)])
def test_many_gates(rows, width, act, dtype):
    gate_up = (normal(rows, 2 * width, seed=71) * 3).to(DT[dtype])
    codes, scales, whole = room(rows, width)
    ops().swiglu_int8(codes, scales, gate_up, act)
    check_codes(codes, scales, whole, gate_formula(gate_up, act), 2.0 ** -15)


@pytest.mark.parametrize("add", [None, "float32", "bfloat16"])
@pytest.mark.parametrize("rows,width", [(1203, 1999), (9000, 1028), (5000, 2052), (6000, 2048), (4000, 4096), (3700, 4100), (613, 4099), (333, 8190), (1400, 13000),
                                        (170, 20001)])
def test_many_norms(rows, width, add):
    x = normal(rows, width, seed=72)
    w = 1 + 0.1 * normal(width, seed=73)
    more = None if add is None else normal(rows, width, seed=74).to(DT[add])
    s = x if add is None else x + more.float()
    want = s.double() / torch.sqrt((s.double() ** 2).mean(dim=1, keepdim=True) + 3e-6) * w.double()
    codes, scales, whole = room(rows, width)
    ops().rmsnorm_int8(codes, scales, x, w, 3e-6, add=more)
    check_codes(codes, scales, whole, want, 2.0 ** -19)
    assert torch.equal(x, s)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,width", [(500, 4099), (700, 4102), (301, 7001), (160, 20003)])
def test_many_rows_into_codes_that_lie_anywhere(rows, width, dtype):
    """Codes without gaps between rows, from any byte on: what lies before and behind them stays."""
    for shift in (0, 1, 2):
        buffer = torch.full((rows * width + 8,), 99, dtype=torch.int8, device=DEV)
        codes, scales = buffer[shift:shift + rows * width].view(rows, width), torch.empty(rows, device=DEV)
        beside, beside_scales, whole = room(rows, width)
        x = normal(rows, width, seed=75, dtype=DT[dtype])
        ops().quantize_rows(codes, scales, x)
        ops().quantize_rows(beside, beside_scales, x)
        check_codes(beside, beside_scales, whole, x.double(), 0.0)
        assert torch.equal(codes, beside) and torch.equal(scales, beside_scales)
        gate_up = normal(rows, 2 * width, seed=76).to(DT[dtype])
        ops().swiglu_int8(codes, scales, gate_up)
        ops().swiglu_int8(beside, beside_scales, gate_up)
        check_codes(beside, beside_scales, whole, gate_formula(gate_up, "silu"), 2.0 ** -15)
        assert torch.equal(codes, beside) and torch.equal(scales, beside_scales)
        assert bool((buffer[:shift] == 99).all()) and bool((buffer[shift + rows * width:] == 99).all())


@pytest.mark.parametrize("add", [None, "float32", "bfloat16"])
@pytest.mark.parametrize("rows,width", [(2000, 5124), (1800, 5122), (1200, 8192), (1300, 10244), (1301, 12300)])
def test_many_long_norms(rows, width, add):
    """Long enough for a ring of rows, in pieces of eight, four and one."""
    test_many_norms(rows, width, add)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("width", [7, 96, 5000])
def test_gates_at_the_ends(width, act, dtype):
    """Gates whose square or exponential is no 32-bit number: the unit is then g u or 0.  And gates that are no number."""
    gate_up = torch.ones(6, 2 * width, device=DEV)
    gate_up[0, :width], gate_up[0, width:] = 2.0 ** 100, 2.0 ** -99
    gate_up[0, 1] = 2.0 ** 99
    gate_up[1, :width] = -2.0 ** 100
    gate_up[1, 2], gate_up[1, width + 2] = 2.0 ** 100, 2.0 ** -100
    gate_up[2, :width] = -200
    gate_up[3, 3], gate_up[4, 3], gate_up[5, width + 3] = float("inf"), float("nan"), float("inf")
    codes, scales, whole = room(6, width)
    ops().swiglu_int8(codes, scales, gate_up.to(DT[dtype]), act)
    assert codes[0].tolist() == [127] + [64] + [127] * (width - 2)  # 63.5 goes to the even one
    assert abs(scales[0].item() * 127 / 2 - 1) < 2.0 ** -20
    assert codes[1].tolist() == [0, 0, 127] + [0] * (width - 3)
    assert not bool(codes[2].any()) and scales[2].item() == 2.0 ** -126
    assert not bool(codes[3:].any()) and bool(torch.isnan(scales[3:]).all())


def gate_formula(gate_up, act):
    g, u = gate_up.double().chunk(2, dim=1)
    if act == "silu":
        return g * torch.sigmoid(g) * u
    if act == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3))) * u
    bias = act.bias.double().chunk(2) if act.bias is not None else (0, 0)
    g, u = g + bias[0], u + bias[1]
    if act.act == "silu":
        return g * torch.sigmoid(g) * u
    g, u = g.clamp(max=act.limit), u.clamp(-act.limit, act.limit)
    return g * torch.sigmoid(act.alpha * g) * (u + 1)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("width", WIDTHS)
def test_gate(width, act, dtype):
    gate_up = (normal(4, 2 * width, seed=1) * 3).to(DT[dtype])
    codes, scales, whole = room(4, width)
    ops().swiglu_int8(codes, scales, gate_up, act)
    check_codes(codes, scales, whole, gate_formula(gate_up, act), 2.0 ** -15)


@pytest.mark.parametrize("width", [5, 96, 1000])
@pytest.mark.parametrize("kind", ["limited", "limited and biased", "biased"])
def test_gate_options(width, kind):
    bias = normal(2 * width, seed=2) if "biased" in kind else None
    gate = ops().Gate("gated_sigmoid", 2.0, 1.7, bias) if "limited" in kind else ops().Gate("silu", bias=bias)
    gate_up = normal(6, 2 * width, seed=3) * 2
    codes, scales, whole = room(6, width)
    ops().swiglu_int8(codes, scales, gate_up, gate)
    check_codes(codes, scales, whole, gate_formula(gate_up, gate), 2.0 ** -15)


@pytest.mark.parametrize("width", [4096, 4100, 4099, 17001])
@pytest.mark.parametrize("kind", ["limited", "limited and biased", "biased"])
def test_gate_options_of_many_rows(width, kind):
    bias = normal(2 * width, seed=2) if "biased" in kind else None
    gate = ops().Gate("gated_sigmoid", 2.0, 1.7, bias) if "limited" in kind else ops().Gate("silu", bias=bias)
    gate_up = (normal(500, 2 * width, seed=3) * 2).bfloat16()
    codes, scales, whole = room(500, width)
    ops().swiglu_int8(codes, scales, gate_up, gate)
    check_codes(codes, scales, whole, gate_formula(gate_up, gate), 2.0 ** -15)


@pytest.mark.parametrize("add", [None, "float32", "bfloat16"])
@pytest.mark.parametrize("w_dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("width", WIDTHS)
def test_norm(width, w_dtype, add):
    x = normal(5, width, seed=4) * 3
    x[:, ::17] *= 6
    w = (1 + 0.1 * normal(width, seed=5)).to(DT[w_dtype])
    more = None if add is None else normal(5, width, seed=6).to(DT[add])
    s = x.double() if add is None else (x + more.float()).double()
    want = s / torch.sqrt((s * s).mean(dim=1, keepdim=True) + 3e-6) * w.double()
    codes, scales, whole = room(5, width)
    before = x.clone()
    out = None if add is None else torch.full_like(x, 9.0)
    ops().rmsnorm_int8(codes, scales, x, w, 3e-6, add=more, out=out)
    assert torch.equal(x, before)
    check_codes(codes, scales, whole, want, 2.0 ** -19)
    if add is not None:
        assert torch.equal(out, x + more.float())
        again, scales2, _ = room(5, width)
        ops().rmsnorm_int8(again, scales2, x, w, 3e-6, add=more)  # into x itself
        assert torch.equal(x, out) and torch.equal(again, codes) and torch.equal(scales2, scales)


@pytest.mark.parametrize("width", [64, 100, 9000, 33000])
def test_rows_of_zeros_tiny_huge_and_broken_values(width):
    x = normal(8, width, seed=7)
    x[1] = 0
    x[2] *= 1e-42  # numbers below 2^-126
    x[3] *= 1e37
    x[4, width // 2] = float("nan")
    x[5, 3] = float("inf")
    x[6, width - 1] = -float("inf")
    codes, scales, whole = room(8, width)
    ops().quantize_rows(codes, scales, x)
    good = [0, 1, 2, 3, 7]
    check_codes(codes[good], scales[good], whole, x[good].double(), 0.0)
    assert bool(torch.isnan(scales[4:7]).all()) and not bool(codes[4:7].any())
    # the norm: zeros stay zeros (of any eps), and what is added may be what breaks a row
    w = torch.ones(width, device=DEV)
    add = torch.zeros_like(x)
    add[0, 1] = float("nan")
    x[3] = 1.0
    ops().rmsnorm_int8(codes, scales, x, w, 1e-6, add=add)
    assert bool(torch.isnan(scales[[0, 4, 5, 6]]).all()) and not bool(codes[[0, 1, 4, 5, 6]].any())
    assert float(scales[1]) == TINY and bool((codes[3] == 127).all())
    check_codes(codes[7:], scales[7:], whole, (x[7:].double() / torch.sqrt((x[7:].double() ** 2).mean() + 1e-6)), 2.0 ** -19)


def coded(rows, width, seed):
    codes = ops().int8_rows(rows, width, DEV)
    whole = codes.as_strided((rows, codes.stride(0)), (codes.stride(0), 1))
    whole.fill_(99)  # what lies between the rows is not read
    codes.copy_(torch.randint(-128, 128, (rows, width), generator=torch.Generator().manual_seed(seed)).to(DEV))
    scales = torch.rand(rows, generator=torch.Generator().manual_seed(seed + 1)).to(DEV) * 0.02 + 0.001
    return codes, scales


def product(codes, scales, w, w_scales, bias=None):
    """(the formula, the size of what is rounded on the way) in 64 bits; the sums are whole numbers below 2^53."""
    total = (codes.double() @ w.double().t()) * scales.double()[:, None] * w_scales.double()
    size = total.abs()
    return (total, size) if bias is None else (total + bias.double(), size + bias.double().abs())


def check_product(out, want, size):
    """32-bit: the sum's rounding, two products, at most two additions: five halves of 2^-23; bfloat16: half of 2^-7 more."""
    allowed = size * 5 * 2.0 ** -24
    if out.dtype == torch.bfloat16:
        allowed = allowed + (want.abs() + allowed) * 2.0 ** -8
    assert bool(((out.double() - want).abs() <= allowed + 1e-40).all())


SHAPES = [(1, 1, 1), (1, 6144, 4096), (2, 128, 128), (3, 5, 17), (7, 130, 1000), (8, 4096, 14336), (15, 515, 640), (16, 512, 2048),
          (17, 260, 4100), (33, 1000, 272), (64, 2048, 4096), (65, 300, 129), (100, 777, 5003), (127, 129, 4096), (128, 640, 512),
          (129, 256, 256), (200, 2048, 1024), (256, 512, 16), (257, 1030, 333), (333, 5003, 1999), (600, 1300, 2048), (1500, 4100, 700)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k, biased, dtype):
    codes, scales = coded(m, k, 10)
    w, w_scales = coded(n, k, 20)
    bias = normal(n, seed=8) if biased else None
    out = torch.full((m, n), 5.0, dtype=DT[dtype], device=DEV)
    ops().gemm_int8(out, codes, scales, w, w_scales, bias=bias)
    check_product(out, *product(codes, scales, w, w_scales, bias))


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_added_into_strided_rows(m, n, k, biased):
    codes, scales = coded(m, k, 11)
    w, w_scales = coded(n, k, 21)
    bias = normal(n, seed=9) if biased else None
    whole = normal(m + 1, n + 3, seed=10)
    before = whole.clone()
    ops().gemm_int8(whole[:m, 1:n + 1], codes, scales, w, w_scales, accumulate=True, bias=bias)
    want, size = product(codes, scales, w, w_scales, bias)
    old = before[:m, 1:n + 1].double()
    check_product(whole[:m, 1:n + 1], want + old, size + old.abs())
    whole[:m, 1:n + 1] = before[:m, 1:n + 1]
    assert torch.equal(whole, before)  # nothing beside the rows was written


@pytest.mark.parametrize("rows", [1, 8, 40, 128, 200])
def test_the_longest_sums_do_not_overflow(rows):
    k = ops().INT8_MAX_INPUTS
    codes, w = ops().int8_rows(rows, k, DEV), ops().int8_rows(130, k, DEV)
    codes.fill_(-128)
    w.fill_(-128)
    w[1] = 127
    ones = torch.ones(max(rows, 130), device=DEV)
    out = torch.empty(rows, 130, device=DEV)
    ops().gemm_int8(out, codes, ones[:rows], w, ones[:130])
    assert bool((out[:, 0] == float(np.float32(128 * 128 * k))).all()) and bool((out[:, 1] == float(np.float32(-128 * 127 * k))).all())


def test_product_of_a_broken_row_is_nan_and_of_zeros_is_the_bias():
    x = normal(20, 96, seed=11)
    x[2, 5] = float("nan")
    x[3] = 0
    codes, scales, _ = room(20, 96)
    ops().quantize_rows(codes, scales, x)
    w, w_scales = coded(72, 96, 22)
    bias = normal(72, seed=12)
    out = torch.empty(20, 72, device=DEV)
    ops().gemm_int8(out, codes, scales, w, w_scales, bias=bias)
    assert bool(torch.isnan(out[2]).all()) and torch.equal(out[3], bias)
    assert bool(torch.isfinite(out[[i for i in range(20) if i != 2]]).all())


def test_a_row_does_not_depend_on_the_rows_beside_it():
    codes, scales = coded(300, 2000, 12)
    w, w_scales = coded(700, 2000, 23)
    out = torch.empty(300, 700, device=DEV)
    ops().gemm_int8(out, codes, scales, w, w_scales)
    for begin, m in ((0, 1), (5, 9), (17, 64), (100, 128), (3, 200)):
        part = torch.empty(m, 700, device=DEV)
        ops().gemm_int8(part, codes[begin:begin + m], scales[begin:begin + m], w, w_scales)
        assert torch.equal(part, out[begin:begin + m])


def feed_forward(x, add, norm_w, w1, s1, w2, s2):
    """norm(x + add) -> product -> gate -> product into the stream: what a layer's second half does."""
    n, width = x.shape
    inner = w1.shape[0] // 2
    o = ops()
    stream = torch.empty_like(x)
    h, h_scales = o.int8_rows(n, width, DEV), torch.empty(n, device=DEV)
    o.rmsnorm_int8(h, h_scales, x, norm_w, 1e-5, add=add, out=stream)
    both = torch.empty(n, 2 * inner, dtype=torch.bfloat16, device=DEV)
    o.gemm_int8(both, h, h_scales, w1, s1)
    a, a_scales = o.int8_rows(n, inner, DEV), torch.empty(n, device=DEV)
    o.swiglu_int8(a, a_scales, both)
    o.gemm_int8(stream, a, a_scales, w2, s2, accumulate=True)
    return h, h_scales, both, a, a_scales, stream


def layer(n, width, inner, seed=30):
    x, add = normal(n, width, seed=seed), normal(n, width, seed=seed + 1)
    norm_w = 1 + 0.1 * normal(width, seed=seed + 2)
    w1, w2 = o_rows(normal(2 * inner, width, seed=seed + 3) * 0.05), o_rows(normal(width, inner, seed=seed + 4) * 0.05)
    return [x, add, norm_w, *w1, *w2]


def o_rows(w):
    codes, scales = ops().int8_rows(*w.shape, DEV), torch.empty(w.shape[0], device=DEV)
    ops().quantize_rows(codes, scales, w)
    return codes, scales


@pytest.mark.parametrize("n", [1, 9, 70, 300])
def test_a_feed_forward_of_them(n):
    args = layer(n, 200, 328)
    x, add, norm_w, w1, s1, w2, s2 = args
    h, h_scales, both, a, a_scales, stream = feed_forward(*args)
    s = (x + add).double()
    y = s / torch.sqrt((s * s).mean(dim=1, keepdim=True) + 1e-5) * norm_w.double()
    whole = torch.full((n, 208), 77, dtype=torch.int8, device=DEV)
    check_codes(h, h_scales, whole, y, 2.0 ** -19)
    check_product(both, *product(h, h_scales, w1, s1))
    whole = torch.full((n, 336), 77, dtype=torch.int8, device=DEV)
    check_codes(a, a_scales, whole, gate_formula(both, "silu"), 2.0 ** -15)
    want, size = product(a, a_scales, w2, s2)
    check_product(stream, want + s, size + s.abs())
    # against the unrounded feed-forward: three roundings to 8 bits, each at most half a step of 1/127 of its row's largest
    # value (rows of normal numbers: largest about 3 to 4 rms, so about 1 percent of a row's rms each, and weights likewise)
    g, u = (y @ (w1.double() * s1.double()[:, None]).t()).chunk(2, dim=1)
    whole_precision = (g * torch.sigmoid(g) * u) @ (w2.double() * s2.double()[:, None]).t()
    delta = stream.double() - s
    assert float((delta - whole_precision).norm() / whole_precision.norm()) < 0.05


@pytest.mark.parametrize("n", [1, 40, 300])
def test_captured_replayed_and_on_another_stream(n):
    args = layer(n, 256, 384)
    first = feed_forward(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = feed_forward(*args)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(first, other):
        assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = feed_forward(*args)
    for seed in (50, 60):
        new = layer(n, 256, 384, seed=seed)
        for old, value in zip(args, new):
            old.copy_(value)
        graph.replay()
        for p, q in zip(held, feed_forward(*new)):
            assert torch.equal(p, q)


def test_two_products_at_once():
    """Calls on two streams share nothing: neither's result depends on the other's."""
    cases = [(coded(8, 4096, 40 + i), coded(2048, 4096, 50 + i)) for i in range(2)]
    alone = []
    for (c, s), (w, ws) in cases:
        out = torch.empty(8, 2048, device=DEV)
        ops().gemm_int8(out, c, s, w, ws)
        alone.append(out)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[torch.empty(8, 2048, device=DEV) for _ in range(20)] for _ in cases]
    torch.cuda.synchronize()
    for turn in range(20):
        for ((c, s), (w, ws)), stream, out in zip(cases, streams, outs):
            with torch.cuda.stream(stream):
                ops().gemm_int8(out[turn], c, s, w, ws)
    torch.cuda.synchronize()
    for want, got in zip(alone, outs):
        for out in got:
            assert torch.equal(out, want)


def test_weights_that_the_call_before_wrote():
    """A norm and a product whose weights were made right before them, without ``constant_weight``."""
    o = ops()
    x = normal(4, 4096, seed=90)
    w = [normal(4096, 4096, seed=91 + i) for i in range(4)]
    ones = torch.ones(4096, device=DEV)
    want = [o_rows(one) for one in w]
    held, held_scales = o.int8_rows(4096, 4096, DEV), torch.empty(4096, device=DEV)
    h, h_scales = o.int8_rows(4, 4096, DEV), torch.empty(4, device=DEV)
    o.rmsnorm_int8(h, h_scales, x, ones, 1e-5)
    outs = [torch.empty(4, 4096, device=DEV) for _ in w]
    torch.cuda.synchronize()
    for one, out in zip(w, outs):
        o.quantize_rows(held, held_scales, one)
        o.gemm_int8(out, h, h_scales, held, held_scales)
    for (codes, scales), out in zip(want, outs):
        check_product(out, *product(h, h_scales, codes, scales))


def test_empty_calls():
    o = ops()
    w, w_scales = coded(40, 32, 60)
    none, scales = o.int8_rows(0, 32, DEV), torch.empty(0, device=DEV)
    o.quantize_rows(none, scales, torch.empty(0, 32, device=DEV))
    o.swiglu_int8(none, scales, torch.empty(0, 64, device=DEV))
    o.rmsnorm_int8(none, scales, torch.empty(0, 32, device=DEV), torch.ones(32, device=DEV), 1e-5)
    o.gemm_int8(torch.empty(0, 40, device=DEV), none, scales, w, w_scales)


def test_refusals_on_the_device():
    from xeno_rt_b200.core import KernelError
    o = ops()
    x = normal(4, 32)
    codes, scales, _ = room(4, 32)
    w, w_scales = coded(40, 32, 61)
    out = torch.empty(4, 40, device=DEV)
    bad = [
        lambda: o.quantize_rows(codes, scales.cpu(), x),
        lambda: o.quantize_rows(codes.cpu(), scales, x),
        lambda: o.quantize_rows(codes, scales, x.half()),
        lambda: o.quantize_rows(codes, scales, x.t().contiguous().t()),
        lambda: o.swiglu_int8(codes, scales, x),
        lambda: o.swiglu_int8(codes, scales, normal(4, 64), "relu"),
        lambda: o.swiglu_int8(codes, scales, normal(4, 64), o.Gate("silu", bias=normal(32))),
        lambda: o.rmsnorm_int8(codes, scales, x.bfloat16(), torch.ones(32, device=DEV), 1e-5),
        lambda: o.rmsnorm_int8(codes, scales, x, torch.ones(32, device=DEV), 1e-5, add=normal(1, 32).expand(4, 32)),
        lambda: o.rmsnorm_int8(codes, scales, x, torch.ones(32, device=DEV), 1e-5, add=normal(4, 32).half()),
        lambda: o.gemm_int8(out.half(), codes, scales, w, w_scales),
        lambda: o.gemm_int8(out, codes, scales, w.cpu(), w_scales),
        lambda: o.gemm_int8(out.bfloat16(), codes, scales, w, w_scales, accumulate=True),
    ]
    for call in bad:
        with pytest.raises(KernelError):
            call()
    torch.cuda.synchronize()
