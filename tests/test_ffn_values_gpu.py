"""Values of the feed-forward operators near the ends of their types' ranges, against their definitions in 64 bits."""
import pytest
import torch

import cfk_b200 as cfk
from ffn_helpers import ACTS, TINY, activation64, check, half

pytestmark = pytest.mark.gpu

# The kernels hold an activation or a slope in fp32.  Its relative error is that of the argument of the exponential times the argument,
# which reaches 2 * 126 log 2 = 175 where r = 2^-126.  Half units in the last place (2^-24) in the argument: SiLU 2 (constant, product),
# GELU's density 3 and erfc 2 with arguments to 90, the tanh form 7 (two constants, four operations of the polynomial, product):
# 175 * 7 * 2^-24 = 7.3e-5, and a few units in the last place beside that.  Absolute error 2^-145: half the smallest subnormal, 2^-150, of
# what is multiplied by at most 14 (GELU's erfc), and of the value itself.
FAR_REL, FAR_ABS = 8e-5, 2.0 ** -145


def far_gates():
    g = torch.cat([torch.linspace(-160, -80, 321), torch.linspace(-20, -3, 69), torch.linspace(80, 100, 10)])
    return g.bfloat16()                                  # 400: the channels of a call


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("large", [1e3, 1e37])
@pytest.mark.parametrize("m", [3, 300])
def test_small_activations_beside_a_large_factor(lib, cuda, act, large, m):
    """SiLU and the tanh form of GELU fall like e^x, GELU like e^(-x^2 / 2): with a factor of 1e37 behind them such values are normal
    numbers of bf16 down to gates of about -170 and -18, far beyond where e^x, or its inverse, is one of fp32."""
    gates = far_gates().cuda()
    n, k = gates.numel(), 8
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = x[:, 1] = 1
    wg, wu = (torch.zeros(n, k, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    wg[:, 0], wu[:, 1] = gates, large                    # gate and up are these numbers exactly
    h = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    lib.ffn_gated(x, wg, wu, h, dtype=cfk.BF16, out_dtype=cfk.BF16, activation=act, m=m, n=n, k=k)
    lib.check_device()
    z, u = gates.double(), wu[:, 1].double()
    value, slope = activation64(act, z)
    want = torch.where((value * u).abs() < 3e38, value * u, value.clamp(max=1) * 1e30).expand(m, n)
    got = torch.where((value * u).abs() < 3e38, h.double(), value.clamp(max=1) * 1e30)       # what passes the type's range is not compared
    check(got, want, (FAR_REL + half(cfk.BF16)) * want.abs() + FAR_ABS * u + TINY[cfk.BF16])

    gate, up = gates.expand(m, n).contiguous(), wu[:, 1].expand(m, n).contiguous()
    for d0, u0 in ((1.0, large), (large, 1.0)):
        dh, up = torch.full_like(gate, d0), torch.full_like(gate, u0)
        dgate, dup = torch.zeros_like(gate), torch.zeros_like(gate)
        lib.ffn_gated_backward(dh, x, wg, wu, gate, up, dgate, dup, dtype=cfk.BF16, activation=act, m=m, n=n, k=k)
        lib.check_device()
        d, u = dh.double(), up.double()
        check(dgate, d * u * slope, (FAR_REL + half(cfk.BF16)) * (d * u * slope).abs() + FAR_ABS * d * u + TINY[cfk.BF16])
        fits = (d * value).abs() < 3e38
        want, got = torch.where(fits, d * value, 0.0), torch.where(fits, dup.double(), 0.0)
        check(got, want, (FAR_REL + half(cfk.BF16)) * want.abs() + FAR_ABS * d + TINY[cfk.BF16])


# ---- scales ------------------------------------------------------------------------------------------------------------------------
def far_scales(g, count, lo, hi):
    """Scales over the range of fp32, of either sign."""
    e = torch.rand(count, generator=g, device="cuda") * (hi - lo) + lo
    sign = torch.where(torch.rand(count, generator=g, device="cuda") < 0.2, -1.0, 1.0)
    return torch.exp2(e) * sign


@pytest.mark.parametrize("m", [1, 7, 40, 300])
@pytest.mark.parametrize("bias", [False, True])
def test_scales_over_the_whole_range_of_fp32(lib, cuda, m, bias):
    """Row scales from 2^-140 to 2^120 beside column scales of the inverse size and others: whatever the row's scale does to a sum on the
    way, a result that fp32 holds has its value, and one beyond it is infinite.  A sum, its product with a scale and the result round
    to 32 bits, or to the smallest subnormal."""
    n, k = 264, 400
    g = torch.Generator(device="cuda").manual_seed(m)
    a = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    b = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    a[:, ::3], b[:, ::3] = 127, 127                      # sums of both sizes, up to 2^22
    sa, sb = far_scales(g, m, -140, 120), far_scales(g, n, -140, 120)
    sa[0], sb[:32] = 2.0 ** 120, far_scales(g, 32, -140, -110)
    bs = torch.exp2(torch.rand(n, generator=g, device="cuda") * 100 - 50) if bias else None
    c = torch.zeros(m, n, device="cuda")
    lib.gemm_i8(a, b, c, m=m, n=n, k=k, out_dtype=cfk.FP32, a_scale=sa, b_scale=sb, bias=bs)
    lib.check_device()
    y0 = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()[None, :]
    y = y0 + bs.double() if bias else y0
    fits = y0.abs() < 3.4e38
    assert int((fits & (y0.abs() > 1e25)).sum()) > 0 and bool(c[~fits & (y0.abs() > 3.5e38)].isinf().all())
    bound = 4 * 2.0 ** -24 * (y0.abs() + y.abs()) + 2 * TINY[cfk.FP32]
    check(c[fits].double(), y[fits], bound[fits])


@pytest.mark.parametrize("m", [2, 40, 300])
def test_a_row_of_the_largest_values_through_the_8_bit_block(lib, cuda, m):
    """Tokens up to 3e38 quantise to scales of 2^121; with weights of 1e-36 gate and up are ordinary numbers."""
    n, k = 200, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.rand(m, k, generator=g, device="cuda") * 2 - 1).bfloat16()
    x[::2] *= 2.0 ** 127
    xq, xs = torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda")
    lib.quantize_rows(x, xq, xs, src_dtype=cfk.BF16, rows=m, cols=k)
    w = [torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8) for _ in range(2)]
    ws = torch.full((n,), 2.0 ** -127, device="cuda")    # a subnormal number
    h, gate, up = (torch.zeros(m, n, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    lib.ffn_gated(xq, w[0], w[1], h, dtype=cfk.INT8, out_dtype=cfk.BF16, activation=cfk.ACT_RELU, m=m, n=n, k=k, gate=gate, up=up,
                  x_scale=xs, gate_scale=ws, up_scale=ws)
    lib.check_device()
    z, u = ((xq.double() @ t.double().T) * xs.double()[:, None] * ws.double() for t in w)
    assert float(z.abs().max()) > 10
    half_bf16, e = half(cfk.BF16), 4 * 2.0 ** -24
    check(gate, z, (half_bf16 + e) * z.abs() + TINY[cfk.BF16])
    check(up, u, (half_bf16 + e) * u.abs() + TINY[cfk.BF16])
    want = z.clamp(min=0) * u
    check(h, want, (half_bf16 + 3 * e) * want.abs() + TINY[cfk.BF16])
