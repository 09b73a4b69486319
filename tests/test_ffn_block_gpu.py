"""A 16-bit feed-forward block of any number of tokens and any width with its projection back.  cfk_gemm takes packed rows and multiples of
8: h, its gradient and the weight have rows and columns of zeros up to one, which the calls leave as they are."""
import math

import pytest
import torch

import cfk_b200 as cfk
from ffn_helpers import TORCH, randn

pytestmark = pytest.mark.gpu


def up8(x):
    return (x + 7) // 8 * 8


def padded(x, dtype):
    y = torch.zeros(up8(x.shape[0]), up8(x.shape[1]), dtype=dtype, device="cuda")
    y[:x.shape[0], :x.shape[1]] = x
    return y


@pytest.mark.parametrize("dtype", [cfk.FP16, cfk.BF16])
@pytest.mark.parametrize("m,n,k", [(1, 1000, 136), (1, 2731, 1027), (5, 333, 70), (129, 515, 264), (777, 2731, 1027)])
def test_forward_and_gradients_of_the_block_with_its_projection_back(lib, cuda, dtype, m, n, k):
    g, dt, act = torch.Generator(device="cuda").manual_seed(m + n), TORCH[dtype], cfk.ACT_SILU
    M, N, K = up8(m), up8(n), up8(k)
    x, dy = padded(randn(g, m, k), dt), padded(randn(g, m, k), dt)
    wg, wu = (padded(randn(g, n, k) / math.sqrt(k), dt) for _ in range(2))
    wd = padded(randn(g, k, n) / math.sqrt(n), dt)
    h, dh, gate, up = (torch.zeros(M, N, dtype=dt, device="cuda") for _ in range(4))
    y, dwd = torch.zeros(M, K, dtype=dt, device="cuda"), torch.zeros(K, N, dtype=dt, device="cuda")
    dx, dwg, dwu = torch.zeros_like(x), torch.zeros_like(wg), torch.zeros_like(wu)

    lib.ffn_gated(x, wg, wu, h, dtype=dtype, out_dtype=dtype, activation=act, m=m, n=n, k=k, gate=gate, up=up, x_stride=K, w_stride=K,
                  h_stride=N, pre_stride=N)
    lib.gemm(h, wd, y, dtype=dtype, m=M, n=K, k=N, c_row_major=True)
    # gradients: of h, with the weight transposed; of the weight, with both factors transposed (their rows are the reduction)
    wd_t, h_t, dy_t = (t.T.contiguous() for t in (wd, h, dy))
    lib.gemm(dy, wd_t, dh, dtype=dtype, m=M, n=N, k=K, c_row_major=True)
    lib.gemm(dy_t, h_t, dwd, dtype=dtype, m=K, n=N, k=M, c_row_major=True)
    lib.ffn_gated_backward(dh, x, wg, wu, gate, up, gate, up, dx=dx, dw_gate=dwg, dw_up=dwu, dtype=dtype, activation=act, m=m, n=n, k=k,
                           x_stride=K, dh_stride=N, w_stride=K, pre_stride=N, dpre_stride=N, dx_stride=K, dw_stride=K)
    lib.check_device()

    p = [t.double().requires_grad_() for t in (x[:m, :k], wg[:n, :k], wu[:n, :k], wd[:k, :n])]
    z, u = p[0] @ p[1].T, p[0] @ p[2].T
    hd = torch.nn.functional.silu(z) * u
    yd = hd @ p[3].T
    yd.backward(dy[:m, :k].double())
    # roundings to the type on the way, each at most half a step of its element: h, y (2); gate, up, dh, dgate, dup and the result (6,
    # where a slope or a value doubles the one of gate at most); h, dwd (2).  As relative 2-norms they add at most linearly.
    step = torch.finfo(dt).eps / 2
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())      # noqa: E731
    assert rel(y[:m, :k], yd.detach()) <= 2.1 * step and rel(dwd[:k, :n], p[3].grad) <= 2.1 * step
    for got, want in ((dx[:m, :k], p[0].grad), (dwg[:n, :k], p[1].grad), (dwu[:n, :k], p[2].grad)):
        assert rel(got, want) <= 7 * step
    for t, rows, cols in ((h, m, n), (gate, m, n), (up, m, n), (dx, m, k), (dwg, n, k), (dwu, n, k), (dh, m, n), (y, m, k), (dwd, k, n)):
        assert bool((t[rows:] == 0).all()) and bool((t[:, cols:] == 0).all())
