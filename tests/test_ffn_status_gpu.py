"""The feed-forward calls behind a wait that gave up: nothing is lost, and the call can be repeated."""
import math

import pytest
import torch

import cfk_b200 as cfk
from ffn_helpers import randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [cfk.FP16, cfk.BF16])
@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (3, 131, 70), (24, 1000, 264), (700, 520, 136)])
def test_a_skipped_backward_in_place_keeps_what_it_would_overwrite(lib, cuda, dtype, m, n, k):
    """dgate on gate and dup on up: with the status word set the call must leave both as they were, so that the same call gives the
    gradients once the word has been read."""
    dt = torch.float16 if dtype == cfk.FP16 else torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(m + n)

    def matrix(rows, cols, scale=1.0):                   # rows at multiples of 16 bytes, guarded behind their end
        full = torch.full((rows, (cols + 7) // 8 * 8), float("nan"), dtype=dt, device="cuda")
        full[:, :cols] = randn(g, rows, cols) * scale
        return full

    dh, gate, up, x = matrix(m, n), matrix(m, n), matrix(m, n), matrix(m, k)
    wg, wu = matrix(n, k, 1 / math.sqrt(k)), matrix(n, k, 1 / math.sqrt(k))
    strides = dict(dh_stride=dh.shape[1], x_stride=x.shape[1], w_stride=x.shape[1], pre_stride=gate.shape[1], dpre_stride=gate.shape[1],
                   dx_stride=x.shape[1], dw_stride=x.shape[1])

    def call(gate, up, dgate, dup, outs):
        lib.ffn_gated_backward(dh, x, wg, wu, gate, up, dgate, dup, dx=outs[0], dw_gate=outs[1], dw_up=outs[2], dtype=dtype,
                               activation=cfk.ACT_SILU, m=m, n=n, k=k, **strides)

    bits = lambda t: t.view(torch.int16).clone()         # noqa: E731  the guards are NaN
    fresh = lambda: [torch.full_like(t, -3) for t in (x, wg, wu)]      # noqa: E731
    want, want_pre = fresh(), [gate.clone(), up.clone()]
    call(gate, up, want_pre[0], want_pre[1], want)
    lib.check_device()

    saved, outs = [bits(gate), bits(up)], fresh()
    assert lib.selftest_wait_gives_up(20) == 0
    call(gate, up, gate, up, outs)
    assert lib.device_status() == (6, 901)
    assert torch.equal(bits(gate), saved[0]) and torch.equal(bits(up), saved[1])
    assert all(bool((o == -3).all()) for o in outs)

    call(gate, up, gate, up, outs)
    lib.check_device()
    assert torch.equal(bits(gate), bits(want_pre[0])) and torch.equal(bits(up), bits(want_pre[1]))
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
