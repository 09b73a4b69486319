"""Reductions that take longer than the two seconds that other waits of the kernels have."""
import pytest
import torch

import cfk_b200 as cfk
from ffn_helpers import TINY, activation64, check, half, randn

pytestmark = pytest.mark.gpu


def test_weight_gradients_of_900_million_tokens(lib, cuda):
    """One tile per weight with 14 million k-blocks.  All but 600 tokens have a gradient of zero, so those give the result."""
    m, n, k, dt = 900_000_000, 8, 8, torch.float16
    torch.cuda.empty_cache()
    g = torch.Generator(device="cuda").manual_seed(1)
    dh, gate, up, x = (torch.zeros(m, c, dtype=dt, device="cuda") for c in (n, n, n, k))        # 14.4 GB each
    at = torch.cat([torch.arange(100, device="cuda"), m - 1 - torch.arange(100, device="cuda"),
                    torch.randint(100, m - 100, (400,), generator=g, device="cuda").unique()])
    rows = {}
    for name, t in (("dh", dh), ("gate", gate), ("up", up), ("x", x)):
        rows[name] = randn(g, len(at), 8).to(dt)
        t[at] = rows[name]
    wg, wu = (torch.zeros(n, k, dtype=dt, device="cuda") for _ in range(2))
    dwg, dwu = (torch.full((n, k), float("nan"), dtype=dt, device="cuda") for _ in range(2))
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    lib.ffn_gated_backward(dh, x, wg, wu, gate, up, gate, up, dw_gate=dwg, dw_up=dwu, dtype=cfk.FP16, activation=cfk.ACT_SILU, m=m, n=n,
                           k=k, stream=torch.cuda.current_stream().cuda_stream)
    end.record()
    lib.check_device()
    print(f"{start.elapsed_time(end) / 1e3:.2f} s")
    # the products read the rounded dgate and dup, which are where gate and up were; additions of zeros are exact
    dg, du, xs = gate[at].double(), up[at].double(), rows["x"].double()
    value, slope = activation64(cfk.ACT_SILU, rows["gate"].double())
    check(du, rows["dh"].double() * value, (half(cfk.FP16) + 1e-5) * (rows["dh"].double() * value).abs() + TINY[cfk.FP16])
    del dh, gate, up, x
    torch.cuda.empty_cache()
    for got, d in ((dwg, dg), (dwu, du)):
        want = d.T @ xs
        e = len(at) * 2.0 ** -23 * (d.abs().T @ xs.abs())
        check(got, want, e + half(cfk.FP16) * (want.abs() + e) + TINY[cfk.FP16])
