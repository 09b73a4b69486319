"""Paths of the feed-forward kernels that only calls of some size take, chosen by what the plan of a call says, and compared whole."""
import math

import pytest
import torch

import cfk_b200 as cfk
from ffn_helpers import ACTS, TINY, TORCH, activation64, check, half, quantized, randn

pytestmark = pytest.mark.gpu

PAIRS = 74                                # CTA pairs of a launch


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def matrix(rows, cols, dtype, align=16):
    """Rows at multiples of `align` elements, NaN behind their end."""
    full = torch.full((rows, (cols + align - 1) // align * align), float("nan") if dtype.is_floating_point else 99, dtype=dtype, device="cuda")
    return full[:, :cols]


def held(x, dtype, align=16):
    y = matrix(x.shape[0], x.shape[1], dtype, align)
    y.copy_(x)
    return y


class Backward:
    """Inputs of a backward call and its results' buffers."""

    def __init__(self, dtype, m, n, k, seed, align=16):
        g, dt = gen(seed), TORCH[dtype]
        self.dtype, self.m, self.n, self.k = dtype, m, n, k
        self.x = held(randn(g, m, k), dt, align)
        self.wg, self.wu = (held(randn(g, n, k) / math.sqrt(k), dt, align) for _ in range(2))
        self.gate, self.up, self.dh = (held(randn(g, m, n), dt, align) for _ in range(3))

    def plan(self, dx=True, dw=True):
        return cfk.load().ffn_plan(cfk.FfnGatedBackwardArgs(self.dtype, 0, self.m, self.n, self.k, *range(0x1000, 0x9000, 0x1000),
                                                            0x9000 if dx else None, *((0xa000, 0xb000) if dw else (None, None)),
                                                            *[1 << 20] * 7))

    def run(self, lib, act, dx=True, dw=True):
        m, n, k, dt = self.m, self.n, self.k, TORCH[self.dtype]
        like = lambda t: matrix(t.shape[0], t.shape[1], dt, t.stride(0))      # noqa: E731
        dgate, dup, gx, gwg, gwu = like(self.gate), like(self.up), like(self.x), like(self.wg), like(self.wu)
        lib.ffn_gated_backward(self.dh, self.x, self.wg, self.wu, self.gate, self.up, dgate, dup, dx=gx if dx else None,
                               dw_gate=gwg if dw else None, dw_up=gwu if dw else None, dtype=self.dtype, activation=act, m=m, n=n, k=k,
                               dh_stride=self.dh.stride(0), x_stride=self.x.stride(0), w_stride=self.wg.stride(0),
                               pre_stride=self.gate.stride(0), dpre_stride=dgate.stride(0), dx_stride=gx.stride(0) if dx else 0,
                               dw_stride=gwg.stride(0) if dw else 0)
        lib.check_device()
        return dgate, dup, gx if dx else None, gwg if dw else None, gwu if dw else None

    def check(self, act, dgate, dup, gx, gwg, gwu):
        """Every element against 64 bits (bounds: ffn_helpers.py; the products read the rounded dgate and dup)."""
        d, u, z = self.dh.double(), self.up.double(), self.gate.double()
        value, slope = activation64(act, z)
        check(dgate, d * u * slope, 3e-5 * (d * u).abs() + half(self.dtype) * (d * u * slope).abs() + TINY[self.dtype])
        check(dup, d * value, 3e-5 * (d * value).abs() + half(self.dtype) * (d * value).abs() + TINY[self.dtype])
        dg, du, xd, gd, ud = (t.double() for t in (dgate, dup, self.x, self.wg, self.wu))

        def product(got, want, magnitude, length):
            e = length * 2.0 ** -23 * magnitude
            check(got, want, e + half(self.dtype) * (want.abs() + e) + TINY[self.dtype])

        if gx is not None:
            product(gx, dg @ gd + du @ ud, dg.abs() @ gd.abs() + du.abs() @ ud.abs(), 2 * self.n)
        if gwg is not None:
            product(gwg, dg.T @ xd, dg.abs().T @ xd.abs(), self.m)
            product(gwu, du.T @ xd, du.abs().T @ xd.abs(), self.m)


@pytest.mark.parametrize("m,n,k", [(2000, 512, 1027), (1400, 1030, 715), (1100, 264, 1500)])
@pytest.mark.parametrize("dtype", [cfk.FP16, cfk.BF16])
@pytest.mark.parametrize("align", [8, 16])
def test_whole_and_partial_gradients_of_either_alignment(lib, cuda, dtype, m, n, k, align):
    """Rows at multiples of 16 and of 32 bytes (which are stored in other pieces), behind widths that no piece divides; the distance of
    rows of a gradient that is left out is 0 and says nothing about the others."""
    b = Backward(dtype, m, n, k, m + k, align)
    assert b.plan()[0] == b.plan(dw=False)[0] == 0
    for parts in (dict(), dict(dw=False), dict(dx=False)):
        b.check(0, *b.run(lib, 0, **parts))
