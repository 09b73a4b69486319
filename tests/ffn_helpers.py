"""Definitions of the feed-forward operators in 64 bits, matrices with guarded padding, and the error bounds of the tests.

Bounds.  A rounding to a type is off by at most eps / 2 of the value (half the smallest subnormal below the normal range).  A sum of K
products in the tensor core is off by at most K * 2^-23 of the sum of the products' magnitudes: products of 16-bit values
are exact in 32 bits, and each of the K additions cuts at most one unit in the last place of a partial sum, which is no larger than that sum of magnitudes.
"""
import math

import torch

import cfk_b200 as cfk

TORCH = {cfk.FP16: torch.float16, cfk.BF16: torch.bfloat16, cfk.FP32: torch.float32, cfk.INT8: torch.int8}
ACTS = [cfk.ACT_SILU, cfk.ACT_GELU, cfk.ACT_GELU_TANH, cfk.ACT_RELU]
TINY = {cfk.FP16: 2.0 ** -25, cfk.BF16: 2.0 ** -134, cfk.FP32: 2.0 ** -150}      # half the smallest subnormal

# Values and derivatives of the activations as the kernels compute them (special-function exponential, fast division): relative
# error of the logistic function 1.5 ulp of ex2 and 2 of the division plus |x| log2(e) 2^-24 from the rounded argument, below 1e-5 for
# |x| < 80; the polynomial in front of it rounds three times.  Derivatives are bounded by 1.13 and are sums of terms below 1.2.
ACT_REL = 1e-5


def half(code):
    return torch.finfo(TORCH[code]).eps / 2


def activation64(act, z):
    """(value, derivative) in 64 bits."""
    if act == cfk.ACT_SILU:
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    if act == cfk.ACT_GELU:
        cdf = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == cfk.ACT_GELU_TANH:
        c = math.sqrt(2 / math.pi)
        a2 = 2 * c * (z + 0.044715 * z ** 3)
        s = torch.sigmoid(a2)
        return z * s, s + z * s * torch.sigmoid(-a2) * 2 * c * (1 + 3 * 0.044715 * z * z)
    return torch.clamp(z, min=0), (z > 0).to(z.dtype)


class Padded:
    """A matrix within a larger buffer whose other elements hold a guard value: NaN (or 99 in 8-bit integers) in an operand shows a
    read behind a row's end, a changed guard a write."""

    def __init__(self, rows, cols, dtype, pad=0, values=None, extra_rows=2):
        align = 16 // torch.empty(0, dtype=dtype).element_size()
        self.stride = (cols + align - 1) // align * align + pad * align
        self.guard = 99 if dtype == torch.int8 else float("nan")
        self.full = torch.full((rows + extra_rows, self.stride), self.guard, dtype=dtype, device="cuda")
        self.view = self.full[:rows, :cols]
        if values is not None:
            self.view.copy_(values)

    def data_ptr(self):
        return self.full.data_ptr()

    def check_guards(self):
        rest = torch.ones_like(self.full, dtype=torch.bool)
        rest[:self.view.shape[0], :self.view.shape[1]] = False
        outside = self.full[rest]
        assert bool((outside == 99).all() if self.full.dtype == torch.int8 else outside.isnan().all()), "written behind a row"


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def quantized(g, rows, cols):
    """(int8 values, fp32 scales) of N(0, 1) rows."""
    x = randn(g, rows, cols)
    scale = (x.abs().amax(1) / 127).clamp(min=1e-6)
    return torch.round(x / scale[:, None]).to(torch.int8), scale


def check(got, want, bound):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[0].tolist(), float((got.double() - want).abs().max()))
