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
