"""The feed-forward operators against their definitions in 64 bits (bounds: ffn_helpers.py)."""
import math
import random

import pytest
import torch

import cfk_b200 as cfk
from ffn_helpers import ACT_REL, ACTS, TINY, TORCH, Padded, activation64, check, half, quantized, randn

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- quantisation ----------------------------------------------------------------------------------------------------------------
def quantize_definition(x):
    """The definition, in the 32-bit operations that it names.  (Divided by a tensor: by a number torch multiplies with its inverse.)"""
    x = x.float()
    amax = x.abs().amax(1)
    scale = amax / torch.full_like(amax, 127.0)
    scale = torch.where(torch.isfinite(x).all(1), scale, torch.full_like(scale, float("nan")))
    q = torch.clamp(torch.round(x / scale[:, None]), -127, 127)
    return torch.where((scale > 0)[:, None], q, torch.zeros_like(q)).to(torch.int8), scale


@pytest.mark.parametrize("dtype", [cfk.FP16, cfk.BF16, cfk.FP32])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (3, 7, 1), (9, 16, 0), (1, 1024, 0), (130, 1023, 1), (5, 1025, 0), (33, 4096, 2),
                                           (2, 16384, 0), (3, 16391, 1), (2, 40001, 0)])
def test_quantize_is_its_definition_bit_for_bit(lib, cuda, dtype, rows, cols, pad):
    g = gen(rows * cols + dtype)
    x = randn(g, rows, cols) * torch.exp(randn(g, rows, 1) * 4).clamp(max=1e3)
    x = Padded(rows, cols, TORCH[dtype], pad, x)
    q, scale = Padded(rows, cols, torch.int8, pad), Padded(1, rows, torch.float32)
    lib.quantize_rows(x, q, scale, src_dtype=dtype, rows=rows, cols=cols, src_stride=x.stride, dst_stride=q.stride)
    lib.check_device()
    want_q, want_scale = quantize_definition(x.view)
    assert torch.equal(scale.view[0], want_scale) and torch.equal(q.view, want_q)
    q.check_guards(), scale.check_guards(), x.check_guards()


def test_quantize_ties_zero_rows_underflow_and_what_is_not_finite(lib, cuda):
    """Every half of the grid (scale 1: values k + 1/2 go to the even neighbour), zero rows of either sign, rows whose scale is a
    subnormal number or underflows to 0, and rows with an infinity or a NaN anywhere."""
    cols = 512
    rows = [torch.arange(cols) * 0.5 - 127.0, torch.zeros(cols), -torch.zeros(cols)]
    rows[0] = rows[0].clamp(-127, 127)
    rows += [torch.linspace(-1, 1, cols) * s for s in (1e-38, 3e-40, 190 * 2.0 ** -149, 60 * 2.0 ** -149, 3e38)]
    for bad in (float("inf"), float("-inf"), float("nan")):
        for at in (0, 300, cols - 1):
            r = torch.linspace(-2, 2, cols)
            r[at] = bad
            rows.append(r)
    x = torch.stack(rows).cuda()
    q = torch.full((len(rows), cols), 77, dtype=torch.int8, device="cuda")
    scale = torch.full((len(rows),), -1.0, device="cuda")
    lib.quantize_rows(x, q, scale, src_dtype=cfk.FP32, rows=len(rows), cols=cols)
    lib.check_device()
    want_q, want_scale = quantize_definition(x)
    assert torch.equal(scale.isnan(), want_scale.isnan())
    assert torch.equal(scale[~scale.isnan()], want_scale[~want_scale.isnan()]) and torch.equal(q, want_q)
    assert bool(scale[-9:].isnan().all()) and bool((q[-9:] == 0).all()) and scale[1] == 0


def test_quantize_next_to_the_middle_between_two_integers(lib, cuda):
    """Values two units in the last place or less from (k + 1/2) scale, for scales over the range of fp32: where a quotient that is
    not rounded correctly would go to the wrong side."""
    rows, cols = 512, 2048
    g = gen(8)
    amax = torch.exp2(torch.rand(rows, 1, generator=g, device="cuda") * 240 - 120)
    middle = (torch.randint(-126, 126, (rows, cols), generator=g, device="cuda") + 0.5) * (amax / torch.full_like(amax, 127.0))
    nudge = torch.randint(-2, 3, (rows, cols), generator=g, device="cuda", dtype=torch.int32)
    x = (middle.view(torch.int32) + nudge).view(torch.float32)
    x[:, :1] = amax
    q, scale = torch.zeros(rows, cols, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    lib.quantize_rows(x, q, scale, src_dtype=cfk.FP32, rows=rows, cols=cols)
    lib.check_device()
    want_q, want_scale = quantize_definition(x)
    assert torch.equal(scale, want_scale) and torch.equal(q, want_q)


# ---- 8-bit product -----------------------------------------------------------------------------------------------------------------
def run_gemm_i8(lib, m, n, k, out, bias, pad=0, seed=0, stream=None):
    g = gen(seed)
    (a, sa), (b, sb) = quantized(g, m, k), quantized(g, n, k)
    a, b = Padded(m, k, torch.int8, pad, a), Padded(n, k, torch.int8, pad, b)
    bs = randn(g, n) if bias else None
    c = Padded(m, n, TORCH[out], pad)
    lib.gemm_i8(a, b, c, m=m, n=n, k=k, out_dtype=out, a_scale=sa, b_scale=sb, bias=bs, a_stride=a.stride, b_stride=b.stride,
                c_stride=c.stride, stream=stream)
    lib.check_device()
    # the sum is exact; its conversion, two products and the addition of the bias round to 32 bits, then the result to its type
    y0 = (a.view.double() @ b.view.double().T) * sa.double()[:, None] * sb.double()[None, :]
    y = y0 + bs.double() if bias else y0
    check(c.view, y, 4 * 2.0 ** -24 * (y0.abs() + y.abs()) + half(out) * y.abs() + TINY[out])
    a.check_guards(), b.check_guards(), c.check_guards()


@pytest.mark.parametrize("m,n,k,pad", [
    (1, 1, 1, 0), (1, 8, 16, 0), (2, 130, 100, 1), (1, 4096, 512, 0), (7, 1000, 128, 0), (16, 256, 1040, 0), (17, 129, 127, 0),
    (33, 640, 2048, 0), (64, 257, 300, 2), (65, 96, 129, 0), (128, 128, 128, 0), (129, 1301, 2061, 0), (255, 255, 255, 1),
    (256, 256, 256, 0), (300, 2000, 640, 0), (777, 1301, 2061, 0), (2100, 3000, 200, 0), (5000, 40, 96, 0)])
@pytest.mark.parametrize("out", [cfk.FP16, cfk.BF16, cfk.FP32])
def test_gemm_i8_matches(lib, cuda, m, n, k, pad, out):
    run_gemm_i8(lib, m, n, k, out, bias=(m + n + out) % 2 == 0, pad=pad, seed=m + n + k)


@pytest.mark.parametrize("m", [1, 40, 600])
def test_gemm_i8_sums_are_exact_at_their_largest(lib, cuda, m):
    """All operands -128 at the largest reduction: 131071 * 2^14 is just below 2^31; with alternating signs the sum is small."""
    k, n = 131071, 48
    a = Padded(m, k, torch.int8, 0, torch.full((m, k), -128))
    b = Padded(n, k, torch.int8, 0, torch.full((n, k), -128))
    b.view[1::2, ::2] = 127
    c = Padded(m, n, torch.float32)
    ones = torch.ones(max(m, n), device="cuda")
    lib.gemm_i8(a, b, c, m=m, n=n, k=k, out_dtype=cfk.FP32, a_scale=ones, b_scale=ones, a_stride=a.stride, b_stride=b.stride,
                c_stride=c.stride)
    lib.check_device()
    want = (a.view.double() @ b.view.double().T).float()        # one rounding of the exact sum
    assert torch.equal(c.view, want)
    c.check_guards()


@pytest.mark.parametrize("m", [3, 300])
def test_scales_that_are_not_finite_or_zero_reach_their_row_or_column_only(lib, cuda, m):
    n, k = 200, 96
    g = gen(5)
    (a, sa), (b, sb) = quantized(g, m, k), quantized(g, n, k)
    sa[1], sb[7], sb[150] = float("nan"), float("inf"), 0.0
    sa[2] = 0.0
    c = torch.zeros(m, n, device="cuda")
    lib.gemm_i8(a, b, c, m=m, n=n, k=k, out_dtype=cfk.FP32, a_scale=sa, b_scale=sb)
    lib.check_device()
    want = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()[None, :]
    assert torch.equal(c.isnan(), want.isnan()) and torch.equal(c.isinf(), want.isinf())
    ok = want.isfinite()
    check(c[ok], want[ok], 4 * 2.0 ** -24 * want[ok].abs())


# ---- gated block -------------------------------------------------------------------------------------------------------------------
def gated_bound(act, g, u, eg, eu, out):
    """Bound of h = act(g) u for errors eg, eu of g, u (|act'| <= 1.13)."""
    value = activation64(act, g)[0]
    h = (value * u).abs()
    return (1.13 * eg) * (u.abs() + eu) + eu * value.abs() + ACT_REL * h + half(out) * (h + 1.13 * eg * u.abs() + eu * value.abs()) + \
        TINY[out] + 1e-30


def run_gated(lib, dtype, out, act, m, n, k, keep, pad=0, seed=0, scale=1.0):
    g = gen(seed)
    kw = {}
    if dtype == cfk.INT8:
        (x, sx), (wg, sg), (wu, su) = quantized(g, m, k), quantized(g, n, k), quantized(g, n, k)
        sg, su = sg / math.sqrt(k), su / math.sqrt(k)
        kw = dict(x_scale=sx, gate_scale=sg, up_scale=su)
    else:
        x, wg, wu = randn(g, m, k) * scale, randn(g, n, k) / math.sqrt(k), randn(g, n, k) / math.sqrt(k)
    x, wg, wu = (Padded(t.shape[0], k, TORCH[dtype], pad, t) for t in (x, wg, wu))
    h = Padded(m, n, TORCH[out], pad)
    gate, up = (Padded(m, n, TORCH[out], pad), Padded(m, n, TORCH[out], pad)) if keep else (None, None)
    lib.ffn_gated(x, wg, wu, h, dtype=dtype, out_dtype=out, activation=act, m=m, n=n, k=k, gate=gate, up=up, x_stride=x.stride,
                  w_stride=wg.stride, h_stride=h.stride, pre_stride=gate.stride if keep else 0, **kw)
    lib.check_device()
    xd, gd, ud = x.view.double(), wg.view.double(), wu.view.double()
    zg, zu = xd @ gd.T, xd @ ud.T
    if dtype == cfk.INT8:
        zg, zu = zg * sx.double()[:, None] * sg.double(), zu * sx.double()[:, None] * su.double()
        eg, eu = 4 * 2.0 ** -24 * zg.abs(), 4 * 2.0 ** -24 * zu.abs()
    else:
        eg, eu = (k * 2.0 ** -23) * (xd.abs() @ gd.abs().T), (k * 2.0 ** -23) * (xd.abs() @ ud.abs().T)
    check(h.view, activation64(act, zg)[0] * zu, gated_bound(act, zg, zu, eg, eu, out))
    if keep:
        check(gate.view, zg, eg + half(out) * (zg.abs() + eg) + TINY[out])
        check(up.view, zu, eu + half(out) * (zu.abs() + eu) + TINY[out])
    for t in (x, wg, wu, h) + ((gate, up) if keep else ()):
        t.check_guards()


GATED_SIZES = [(1, 1, 1, 0), (1, 8, 8, 0), (1, 4096, 512, 0), (2, 131, 70, 1), (9, 300, 1000, 0), (16, 128, 64, 0), (17, 257, 65, 2),
               (33, 640, 200, 0), (64, 120, 129, 0), (65, 1000, 256, 0), (128, 128, 128, 0), (129, 64, 511, 1), (256, 512, 320, 0),
               (300, 700, 96, 0), (777, 1301, 515, 0), (3000, 1500, 72, 0)]


@pytest.mark.parametrize("m,n,k,pad", GATED_SIZES)
@pytest.mark.parametrize("dtype,out", [(cfk.FP16, cfk.FP16), (cfk.BF16, cfk.BF16), (cfk.INT8, cfk.FP16), (cfk.INT8, cfk.BF16)])
def test_ffn_gated_matches(lib, cuda, m, n, k, pad, dtype, out):
    i = m + n + k + dtype
    run_gated(lib, dtype, out, ACTS[i % 4], m, n, k, keep=i % 3 != 0, pad=pad, seed=i)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [5, 300])
@pytest.mark.parametrize("keep", [False, True])
def test_ffn_gated_activations(lib, cuda, act, m, keep):
    for dtype, out in ((cfk.FP16, cfk.FP16), (cfk.BF16, cfk.BF16), (cfk.INT8, cfk.BF16)):
        run_gated(lib, dtype, out, act, m, 200, 144, keep=keep, seed=act, scale=4.0)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [4, 260])
def test_ffn_gated_far_pre_activations(lib, cuda, act, m):
    """Gates from -60000 to 60000 with up = 1: the activations' ends are finite, -0 or the gate itself, in fp16."""
    n, k = 136, 8
    x = torch.zeros(m, k, dtype=torch.float16, device="cuda")
    x[:, 0], x[:, 1] = 1.0, 1.0
    gates = torch.linspace(-60000, 60000, n)
    gates[:40] = torch.linspace(-120, -2, 40)
    wg, wu = torch.zeros(n, k).half(), torch.zeros(n, k).half()
    wg[:, 0], wu[:, 1] = gates.half(), 1.0
    wg, wu = wg.cuda(), wu.cuda()
    h = torch.zeros(m, n, dtype=torch.float16, device="cuda")
    lib.ffn_gated(x, wg, wu, h, dtype=cfk.FP16, out_dtype=cfk.FP16, activation=act, m=m, n=n, k=k)
    lib.check_device()
    want = activation64(act, wg[:, 0].double())[0].expand(m, n)
    check(h, want, (ACT_REL + half(cfk.FP16)) * want.abs() + TINY[cfk.FP16] + 1e-30)


@pytest.mark.parametrize("m", [3, 300])
def test_a_bad_token_or_channel_stays_in_its_row_or_column(lib, cuda, m):
    n, k = 152, 80
    g = gen(9)
    x, wg, wu = randn(g, m, k).half(), (randn(g, n, k) / 9).half(), (randn(g, n, k) / 9).half()
    h0, h1 = torch.zeros(m, n, dtype=torch.float16, device="cuda"), torch.zeros(m, n, dtype=torch.float16, device="cuda")
    kw = dict(dtype=cfk.FP16, out_dtype=cfk.FP16, activation=cfk.ACT_SILU, m=m, n=n, k=k)
    lib.ffn_gated(x, wg, wu, h0, **kw)
    x[1, 5], wu[20, 3], wg[70, 0] = float("nan"), float("inf"), float("nan")
    lib.ffn_gated(x, wg, wu, h1, **kw)
    lib.check_device()
    hit = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    hit[1], hit[:, 20], hit[:, 70] = True, True, True
    assert torch.equal(h1[~hit], h0[~hit]) and not bool(h1[hit].isfinite().any())


# ---- backward ------------------------------------------------------------------------------------------------------------------------
def run_backward(lib, dtype, act, m, n, k, pad=0, seed=0, in_place=False, dx=True, dw=True):
    g = gen(seed)
    dt = TORCH[dtype]
    x = Padded(m, k, dt, pad, randn(g, m, k))
    wg, wu = (Padded(n, k, dt, pad, randn(g, n, k) / math.sqrt(k)) for _ in range(2))
    gate, up = (Padded(m, n, dt, pad, randn(g, m, n) * 2) for _ in range(2))
    dh = Padded(m, n, dt, pad, randn(g, m, n))
    z, u, d = gate.view.double(), up.view.double(), dh.view.double()
    dgate, dup = (gate, up) if in_place else (Padded(m, n, dt, pad), Padded(m, n, dt, pad))
    gx = Padded(m, k, dt, pad) if dx else None
    gwg, gwu = (Padded(n, k, dt, pad), Padded(n, k, dt, pad)) if dw else (None, None)
    lib.ffn_gated_backward(dh, x, wg, wu, gate, up, dgate, dup, dx=gx, dw_gate=gwg, dw_up=gwu, dtype=dtype, activation=act, m=m, n=n,
                           k=k, x_stride=x.stride, w_stride=wg.stride, pre_stride=gate.stride, dh_stride=dh.stride,
                           dpre_stride=dgate.stride, dx_stride=gx.stride if dx else 0, dw_stride=gwg.stride if dw else 0)
    lib.check_device()
    value, slope = activation64(act, z)
    check(dgate.view, d * u * slope, 3 * ACT_REL * (d * u).abs() + half(dtype) * (d * u * slope).abs() + TINY[dtype] + 1e-30)
    check(dup.view, d * value, 3 * ACT_REL * (d * value).abs() + half(dtype) * (d * value).abs() + TINY[dtype] + 1e-30)
    # the products read the rounded dgate and dup
    dg, du, xd, gd, ud = dgate.view.double(), dup.view.double(), x.view.double(), wg.view.double(), wu.view.double()

    def product(got, want, magnitude, length):
        e = length * 2.0 ** -23 * magnitude
        check(got.view, want, e + half(dtype) * (want.abs() + e) + TINY[dtype])
        got.check_guards()

    if dx:
        product(gx, dg @ gd + du @ ud, dg.abs() @ gd.abs() + du.abs() @ ud.abs(), 2 * n)
    if dw:
        product(gwg, dg.T @ xd, dg.abs().T @ xd.abs(), m)
        product(gwu, du.T @ xd, du.abs().T @ xd.abs(), m)
    for t in (x, wg, wu, gate, up, dh, dgate, dup):
        t.check_guards()
    return gx, gwg, gwu


BACKWARD_SIZES = [(1, 1, 1, 0), (1, 8, 8, 0), (1, 500, 300, 0), (3, 131, 70, 1), (16, 1000, 129, 0), (17, 64, 257, 2), (64, 130, 520, 0),
                  (65, 300, 64, 0), (128, 128, 128, 0), (129, 257, 255, 1), (300, 700, 96, 0), (777, 515, 1301, 0), (1500, 72, 1000, 0)]


@pytest.mark.parametrize("m,n,k,pad", BACKWARD_SIZES)
@pytest.mark.parametrize("dtype", [cfk.FP16, cfk.BF16])
def test_backward_matches(lib, cuda, m, n, k, pad, dtype):
    i = m + n + k + dtype
    run_backward(lib, dtype, ACTS[i % 4], m, n, k, pad=pad, seed=i)


@pytest.mark.parametrize("act", ACTS)
def test_backward_activations_in_place_and_in_parts(lib, cuda, act):
    for dtype in (cfk.FP16, cfk.BF16):
        whole = run_backward(lib, dtype, act, 150, 200, 136, seed=act)
        same = run_backward(lib, dtype, act, 150, 200, 136, seed=act, in_place=True)
        only_dx = run_backward(lib, dtype, act, 150, 200, 136, seed=act, dw=False)
        only_dw = run_backward(lib, dtype, act, 150, 200, 136, seed=act, dx=False)
        for i in range(3):
            assert torch.equal(whole[i].view, same[i].view)
        assert torch.equal(whole[0].view, only_dx[0].view) and torch.equal(whole[1].view, only_dw[1].view)
        run_backward(lib, dtype, act, 20, 72, 40, seed=act, dx=False, dw=False)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [6, 300])
def test_backward_agrees_with_differences(lib, cuda, act, m):
    """Directional derivatives of L = sum(dh * h) by central differences in 64 bits against the products of the kernel's gradients
    with the directions.  Their error: dgate and dup are rounded to fp16 (eps / 2 each, ACT_REL), the sums and the results
    round as in run_backward; the difference quotient's own is below 1e-6 of the magnitudes at a step of 1e-4."""
    n, k, dtype = 120, 72, cfk.FP16
    g = gen(20 + act)
    x = randn(g, m, k).half()
    wg, wu = (randn(g, n, k) / math.sqrt(k)).half(), (randn(g, n, k) / math.sqrt(k)).half()
    dh = randn(g, m, n).half()
    h, gate, up, dgate, dup = (torch.zeros(m, n, dtype=torch.float16, device="cuda") for _ in range(5))
    dx, dwg, dwu = torch.zeros_like(x), torch.zeros_like(wg), torch.zeros_like(wu)
    lib.ffn_gated(x, wg, wu, h, dtype=dtype, out_dtype=dtype, activation=act, m=m, n=n, k=k, gate=gate, up=up)
    lib.ffn_gated_backward(dh, x, wg, wu, gate, up, dgate, dup, dx=dx, dw_gate=dwg, dw_up=dwu, dtype=dtype, activation=act, m=m,
                           n=n, k=k)
    lib.check_device()
    at = [t.double() for t in (x, wg, wu)]
    d = dh.double()

    def loss(p):
        return (d * activation64(act, p[0] @ p[1].T)[0] * (p[0] @ p[2].T)).sum()

    z, u = at[0] @ at[1].T, at[0] @ at[2].T
    value, slope = activation64(act, z)
    # gate and up reach the backward pass rounded: dgate and dup move by their derivatives (|act''| <= 1.2, |act'| <= 1.13) times eps/2
    r = half(dtype) + 1e-6
    near = (z.abs() < 2 * r * (1 + z.abs())).double() if act == cfk.ACT_RELU else 0.0      # relu's step: the slope may flip
    eg = d.abs() * (u.abs() * (1.2 * r * z.abs() + near) + 1.13 * r * u.abs()) + (r + 3 * ACT_REL) * (d * u).abs() * (slope.abs() + 1)
    eu = d.abs() * 1.13 * r * z.abs() + (r + 3 * ACT_REL) * (d * value).abs()
    tol = [eg @ at[1].abs() + eu @ at[2].abs(), eg.T @ at[0].abs(), eu.T @ at[0].abs()]
    step = 1e-4 if act != cfk.ACT_RELU else 1e-6
    for i, grad in enumerate((dx, dwg, dwu)):
        for seed in range(3):
            v = torch.randn(at[i].shape, generator=gen(seed), device="cuda").double()
            plus, minus = list(at), list(at)
            plus[i], minus[i] = at[i] + step * v, at[i] - step * v
            want = (loss(plus) - loss(minus)) / (2 * step)
            bound = ((tol[i] + (r + 2 * m * 2.0 ** -23) * grad.double().abs() + TINY[dtype]) * v.abs()).sum()
            assert abs(float((grad.double() * v).sum() - want)) <= float(bound) + 1e-6 * float((d * u).abs().sum()), (i, seed)
            assert float(bound) < 0.2 * float((grad.double().abs() * v.abs()).sum())      # the bound can tell a wrong gradient


@pytest.mark.parametrize("act", ACTS)
def test_backward_far_pre_activations_are_finite(lib, cuda, act):
    """Gates out to the largest bf16: the derivative is 0 or 1 there and nothing becomes NaN."""
    n = 64
    gate = torch.cat([torch.logspace(0, 38.5, n // 2), -torch.logspace(0, 38.5, n // 2)]).bfloat16().cuda()[None]
    up, dh = torch.full_like(gate, 2.0), torch.full_like(gate, 1.0)
    x, wg, wu = (torch.zeros(r, 8, dtype=torch.bfloat16, device="cuda") for r in (1, n, n))
    dgate, dup = torch.zeros_like(gate), torch.zeros_like(gate)
    lib.ffn_gated_backward(dh, x, wg, wu, gate, up, dgate, dup, dtype=cfk.BF16, activation=act, m=1, n=n, k=8)
    lib.check_device()
    value, slope = activation64(act, gate.double().clamp(-1e4, 1e4))
    value = torch.where(gate.double().abs() > 1e4, gate.double().clamp(min=0), value)
    check(dgate, 2 * slope, (2 * half(cfk.BF16) + 1e-4) * slope.abs() + 1e-4 * ACT_REL + 6 * ACT_REL)
    check(dup, value, (half(cfk.BF16) + 3 * ACT_REL) * value.abs() + 1e-30)


# ---- every cut -----------------------------------------------------------------------------------------------------------------------
def smallest_of_every_plan(lib, args_of, seed, fewest):
    """One shape, the smallest found, for every plan that random shapes get: kernel, tile width, parts of the reduction."""
    rng = random.Random(seed)
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))      # noqa: E731
    best = {}
    for _ in range(6000):
        shape = log(1, 3000), log(8, 3000), log(8, 3000)
        plan = lib.ffn_plan(args_of(*shape))
        cost = shape[0] * shape[1] * shape[2]
        if plan not in best or cost < best[plan][0]:
            best[plan] = (cost, shape)
    assert len(best) >= fewest and {p[0] for p in best} == {0, 1} and {p[1] for p in best if not p[0]} == {64, 96, 128}
    return [shape for _, shape in best.values()]


def packed_args(cls, *head):
    """Arguments for a plan: valid made-up addresses and strides."""
    at = [0x1000 * (i + 1) for i in range(11)]
    if cls is cfk.GemmI8Args:
        return lambda m, n, k: cls(cfk.FP16, m, n, k, *at[:5], None, *[1 << 20] * 3)
    if cls is cfk.FfnGatedArgs:
        scales = at[4:7] if head[0] == cfk.INT8 else [None] * 3
        return lambda m, n, k: cls(head[0], cfk.FP16, 0, m, n, k, *at[:4], None, None, *scales, *[1 << 20] * 4)
    return lambda m, n, k: cls(cfk.FP16, 0, m, n, k, *at, *[1 << 20] * 7)


def test_every_cut_of_the_8_bit_product(lib, cuda):
    for i, (m, n, k) in enumerate(smallest_of_every_plan(lib, packed_args(cfk.GemmI8Args), 1, 8)):
        run_gemm_i8(lib, m, n, k, [cfk.FP16, cfk.BF16, cfk.FP32][i % 3], bias=i % 2 == 0, seed=i)


@pytest.mark.parametrize("dtype", [cfk.FP16, cfk.INT8])
def test_every_cut_of_the_gated_block(lib, cuda, dtype):
    for i, (m, n, k) in enumerate(smallest_of_every_plan(lib, packed_args(cfk.FfnGatedArgs, dtype), 2, 7)):
        run_gated(lib, dtype, cfk.FP16, ACTS[i % 4], m, n, k, keep=i % 2 == 0, seed=i)


def test_every_cut_of_the_backward_pass(lib, cuda):
    for i, (m, n, k) in enumerate(smallest_of_every_plan(lib, packed_args(cfk.FfnGatedBackwardArgs), 3, 20)):
        run_backward(lib, cfk.FP16 if i % 2 else cfk.BF16, ACTS[i % 4], m, n, k, seed=i)


@pytest.mark.parametrize("seed", range(4))
def test_random_calls(lib, cuda, seed):
    """Sizes over the whole range, on a logarithm, with types, padding, options and gradients left out at random."""
    rng = random.Random(100 + seed)
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))      # noqa: E731
    for i in range(25):
        m, n, k, pad = log(1, 2500), log(1, 3000), log(1, 3000), rng.choice([0, 0, 1, 3])
        if rng.random() < 0.5:
            n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
        out, act = rng.choice([cfk.FP16, cfk.BF16]), rng.choice(ACTS)
        kind = rng.randrange(4)
        if kind == 0:
            run_gemm_i8(lib, m, n, k, rng.choice([cfk.FP16, cfk.BF16, cfk.FP32]), bias=rng.random() < 0.5, pad=pad, seed=i)
        elif kind == 1:
            run_gated(lib, out, out, act, m, n, k, keep=rng.random() < 0.5, pad=pad, seed=i)
        elif kind == 2:
            run_gated(lib, cfk.INT8, out, act, m, n, k, keep=rng.random() < 0.5, pad=pad, seed=i)
        else:
            parts = rng.choice([(True, True), (True, True), (True, False), (False, True)])
            run_backward(lib, out, act, m, n, k, pad=pad, seed=i, in_place=rng.random() < 0.5, dx=parts[0], dw=parts[1])


# ---- together ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("m", [1, 19, 300])
def test_an_8_bit_block_end_to_end(lib, cuda, m):
    """Tokens quantised, the gated block, its result quantised, the projection back: every step equals its definition applied to the
    step before it, and the whole is near the block of the unquantised tokens."""
    n, k = 520, 264
    g = gen(m)
    x = randn(g, m, k).bfloat16()
    (wg, sg), (wu, su), (wd, sd) = quantized(g, n, k), quantized(g, n, k), quantized(g, k, n)
    sg, su, sd = sg / math.sqrt(k), su / math.sqrt(k), sd / math.sqrt(n)
    xq, hq = Padded(m, k, torch.int8), Padded(m, n, torch.int8)
    sx, sh = torch.zeros(m, device="cuda"), torch.zeros(m, device="cuda")
    wd = Padded(k, n, torch.int8, 0, wd)
    wg, wu = Padded(n, k, torch.int8, 0, wg), Padded(n, k, torch.int8, 0, wu)
    h = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    lib.quantize_rows(x, xq, sx, src_dtype=cfk.BF16, rows=m, cols=k, dst_stride=xq.stride)
    lib.ffn_gated(xq, wg, wu, h, dtype=cfk.INT8, out_dtype=cfk.BF16, activation=cfk.ACT_SILU, m=m, n=n, k=k, x_scale=sx,
                  gate_scale=sg, up_scale=su, x_stride=xq.stride, w_stride=wg.stride)
    lib.quantize_rows(h, hq, sh, src_dtype=cfk.BF16, rows=m, cols=n, dst_stride=hq.stride)
    lib.gemm_i8(hq, wd, y, m=m, n=k, k=n, out_dtype=cfk.BF16, a_scale=sh, b_scale=sd, a_stride=hq.stride, b_stride=wd.stride)
    lib.check_device()
    q, s = quantize_definition(x)
    assert torch.equal(xq.view, q) and torch.equal(sx, s)
    z = (q.double() @ wg.view.double().T) * s.double()[:, None] * sg.double()
    u = (q.double() @ wu.view.double().T) * s.double()[:, None] * su.double()
    hd = activation64(cfk.ACT_SILU, z)[0] * u
    check(h, hd, gated_bound(cfk.ACT_SILU, z, u, 2.0 ** -22 * z.abs(), 2.0 ** -22 * u.abs(), cfk.BF16))
    q2, s2 = quantize_definition(h)
    assert torch.equal(hq.view, q2) and torch.equal(sh, s2)
    want = (q2.double() @ wd.view.double().T) * s2.double()[:, None] * sd.double()
    check(y, want, (half(cfk.BF16) + 2.0 ** -22) * want.abs() + 1e-30)
    # tokens in full precision: a quantised value is off by half a step, about amax / 254 = 1.5 % of the spread, in x and in h
    zx, ux = (x.double() @ (w.view.double() * s_.double()[:, None]).T for w, s_ in ((wg, sg), (wu, su)))
    full = (activation64(cfk.ACT_SILU, zx)[0] * ux) @ (wd.view.double() * sd.double()[:, None]).T
    assert float((y.double() - full).norm() / full.norm()) < 0.05


@pytest.mark.parametrize("m", [2, 300])
def test_a_training_step_of_the_whole_block(lib, cuda, m):
    """Forward (pre-activations kept), projection back with cfk_gemm, its gradient, backward: against the same in 64 bits."""
    n, k, dt = 320, 128, torch.bfloat16
    g = gen(40 + m)
    x = randn(g, m, k).to(dt)
    wg, wu = (randn(g, n, k) / math.sqrt(k)).to(dt), (randn(g, n, k) / math.sqrt(k)).to(dt)
    wd = (randn(g, k, n) / math.sqrt(n)).to(dt)
    rows = (m + 7) // 8 * 8                              # cfk_gemm takes multiples of 8 rows; the rest are zeros
    dy = torch.zeros(rows, k, dtype=dt, device="cuda")
    dy[:m] = randn(g, m, k).to(dt)
    h, dh = torch.zeros(rows, n, dtype=dt, device="cuda"), torch.zeros(rows, n, dtype=dt, device="cuda")
    gate, up = torch.zeros(m, n, dtype=dt, device="cuda"), torch.zeros(m, n, dtype=dt, device="cuda")
    y = torch.zeros(rows, k, dtype=dt, device="cuda")
    dx, dwg, dwu = torch.zeros_like(x), torch.zeros_like(wg), torch.zeros_like(wu)
    lib.ffn_gated(x, wg, wu, h, dtype=cfk.BF16, out_dtype=cfk.BF16, activation=cfk.ACT_GELU_TANH, m=m, n=n, k=k, gate=gate, up=up)
    lib.gemm(h, wd, y, dtype=cfk.BF16, m=rows, n=k, k=n, c_row_major=True)
    wdt = wd.T.contiguous()
    lib.gemm(dy, wdt, dh, dtype=cfk.BF16, m=rows, n=n, k=k, c_row_major=True)
    lib.ffn_gated_backward(dh, x, wg, wu, gate, up, gate, up, dx=dx, dw_gate=dwg, dw_up=dwu, dtype=cfk.BF16,
                           activation=cfk.ACT_GELU_TANH, m=m, n=n, k=k)
    lib.check_device()
    p = [t.double().requires_grad_() for t in (x, wg, wu)]
    z, u = p[0] @ p[1].T, p[0] @ p[2].T
    hd = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))) * u
    yd = hd @ wd.double().T
    yd.backward(dy[:m].double())
    # bf16 roundings of independent elements: h, y; gate, up, dh, dgate, dup and the result: sqrt(6) * 2^-8 / sqrt(3) at most, 2-norm
    rel = lambda a, b: float((a.detach().double() - b.detach()).norm() / b.detach().norm())      # noqa: E731
    assert rel(y[:m], yd) < 2 * 2.0 ** -8
    for got, want in ((dx, p[0].grad), (dwg, p[1].grad), (dwu, p[2].grad)):
        assert rel(got, want) < 3 * 2.0 ** -8
    assert bool((h[m:] == 0).all())


# ---- streams, graphs, repeated and simultaneous calls ----------------------------------------------------------------------------------
def block_calls(lib, m, n, k, seed):
    """Inputs, outputs and a function that enqueues every operator on a stream."""
    g = gen(seed)
    x = randn(g, m, k).half()
    wg, wu = (randn(g, n, k) / 8).half(), (randn(g, n, k) / 8).half()
    wq, sw = quantized(g, n, k)
    xq, sx = torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda")
    outs = [torch.zeros(m, n, dtype=torch.float16, device="cuda") for _ in range(6)]
    h, gate, up, dgate, dup, hq = outs
    c = torch.zeros(m, n, device="cuda")
    dx, dwg, dwu = torch.zeros_like(x), torch.zeros_like(wg), torch.zeros_like(wu)
    outs += [xq, sx, c, dx, dwg, dwu]

    def calls(stream):
        lib.quantize_rows(x, xq, sx, src_dtype=cfk.FP16, rows=m, cols=k, stream=stream)
        lib.gemm_i8(xq, wq, c, m=m, n=n, k=k, out_dtype=cfk.FP32, a_scale=sx, b_scale=sw, stream=stream)
        lib.ffn_gated(xq, wq, wq, hq, dtype=cfk.INT8, out_dtype=cfk.FP16, activation=0, m=m, n=n, k=k, x_scale=sx, gate_scale=sw,
                      up_scale=sw, stream=stream)
        lib.ffn_gated(x, wg, wu, h, dtype=cfk.FP16, out_dtype=cfk.FP16, activation=0, m=m, n=n, k=k, gate=gate, up=up, stream=stream)
        lib.ffn_gated_backward(h, x, wg, wu, gate, up, dgate, dup, dx=dx, dw_gate=dwg, dw_up=dwu, dtype=cfk.FP16, activation=0, m=m,
                               n=n, k=k, stream=stream)
    return outs, calls


@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (24, 1024, 256), (300, 512, 128)])
def test_a_graph_replays_what_the_calls_give(lib, cuda, m, n, k):
    outs, calls = block_calls(lib, m, n, k, 1)
    calls(torch.cuda.current_stream().cuda_stream)
    lib.check_device()
    want = [o.clone() for o in outs]
    for o in outs:
        o.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(torch.cuda.current_stream().cuda_stream)
    assert all(bool((o == 0).all()) for o in outs)
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        lib.check_device()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_calls_on_several_streams_at_once(lib, cuda):
    sets = [block_calls(lib, m, n, k, i) for i, (m, n, k) in enumerate([(1, 2048, 1024), (40, 1024, 512), (700, 512, 256), (8, 4096, 256)])]
    for outs, calls in sets:
        calls(None)
    lib.check_device()
    want = [[o.clone() for o in outs] for outs, _ in sets]
    for outs, _ in sets:
        for o in outs:
            o.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(8):
        for (outs, calls), s in zip(sets, streams):
            calls(s.cuda_stream)
    lib.check_device()
    for (outs, _), w in zip(sets, want):
        assert all(torch.equal(o, x) for o, x in zip(outs, w))


@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (5, 256, 256), (260, 256, 128)])
def test_a_call_reads_what_the_launch_before_it_wrote(lib, cuda, m, n, k):
    """New tokens every round, enqueued without a wait: fill -> quantise -> product and gated block, each launch set up while the ones
    before still run.  Every round must give what it gives alone."""
    rounds = 60
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    xq, sx = torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda")
    (wq, sw), wg, wu = quantized(gen(0), n, k), (randn(gen(1), n, k) / 9).bfloat16(), (randn(gen(2), n, k) / 9).bfloat16()

    def one(seed, y, h, stream):
        lib.fill(x, cfk.BF16, m * k, seed, scale=1.0 + seed % 7, stream=stream)
        lib.quantize_rows(x, xq, sx, src_dtype=cfk.BF16, rows=m, cols=k, stream=stream)
        lib.gemm_i8(xq, wq, y, m=m, n=n, k=k, out_dtype=cfk.FP32, a_scale=sx, b_scale=sw, stream=stream)
        lib.ffn_gated(x, wg, wu, h, dtype=cfk.BF16, out_dtype=cfk.BF16, activation=cfk.ACT_SILU, m=m, n=n, k=k, stream=stream)

    shape = (rounds, m, n)
    y0, y1 = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    h0, h1 = torch.zeros(shape, dtype=torch.bfloat16, device="cuda"), torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
    for i in range(rounds):
        one(i, y0[i], h0[i], None)
        lib.check_device()
    stream = torch.cuda.Stream()
    for i in range(rounds):
        one(i, y1[i], h1[i], stream.cuda_stream)
    lib.check_device()
    assert torch.equal(y0, y1) and torch.equal(h0, h1)
    assert len({float(v) for v in y0.abs().amax((1, 2))}) > rounds // 2       # the rounds differ


def test_offsets_beyond_32_bits(lib, cuda):
    """Results of more than 2^31 elements: the last rows and columns are where they belong."""
    m, n, k = 66000, 33000, 16
    g = gen(3)
    (a, sa), (b, sb) = quantized(g, m, k), quantized(g, n, k)
    c = torch.zeros(m, n, dtype=torch.float16, device="cuda")
    lib.gemm_i8(a, b, c, m=m, n=n, k=k, out_dtype=cfk.FP16, a_scale=sa, b_scale=sb)
    lib.check_device()
    for rows in (slice(0, 3), slice(33000, 33004), slice(m - 5, m)):
        want = (a[rows].double() @ b.double().T) * sa[rows].double()[:, None] * sb.double()
        check(c[rows], want, (half(cfk.FP16) + 2.0 ** -22) * want.abs() + TINY[cfk.FP16])
    del c
    # few tokens whose rows lie far apart
    m, n, k = 5, 200, 64
    far = torch.zeros(5 * (1 << 29), dtype=torch.int8, device="cuda")
    a = far.view(5, 1 << 29)[:, :k]
    x, sx = quantized(g, m, k)
    a.copy_(x)
    b, sb = quantized(g, n, k)
    c = torch.zeros(m, n, device="cuda")
    lib.gemm_i8(a, b, c, m=m, n=n, k=k, out_dtype=cfk.FP32, a_scale=sx, b_scale=sb, a_stride=1 << 29)
    lib.check_device()
    want = (x.double() @ b.double().T) * sx.double()[:, None] * sb.double()
    check(c, want, 2.0 ** -22 * want.abs())


@pytest.mark.parametrize("m", [5, 300])
def test_rows_that_lie_far_apart(lib, cuda, m):
    """Forward with pre-activations and backward, in place, on matrices whose last rows begin behind 2^31 elements."""
    n, k, dt = 72, 40, torch.float16
    stride = ((1 << 31) // m + 4096) // 16 * 16
    far = lambda: torch.empty(m * stride, dtype=dt, device="cuda").view(m, stride)[:, :n]      # noqa: E731
    g = gen(m)
    x, dh, h, gate, up = far(), far(), far(), far(), far()
    x = x[:, :k]
    x.copy_(randn(g, m, k)), dh.copy_(randn(g, m, n))
    dx = far()[:, :k]
    wg, wu = (randn(g, n, k) / 6).to(dt), (randn(g, n, k) / 6).to(dt)
    dwg, dwu = torch.zeros_like(wg), torch.zeros_like(wu)
    kw = dict(dtype=cfk.FP16, activation=cfk.ACT_SILU, m=m, n=n, k=k, x_stride=stride, pre_stride=stride)
    lib.ffn_gated(x, wg, wu, h, out_dtype=cfk.FP16, gate=gate, up=up, h_stride=stride, **kw)
    lib.check_device()
    z, u = x.double() @ wg.double().T, x.double() @ wu.double().T
    e = k * 2.0 ** -23 * (x.double().abs() @ wg.double().abs().T), k * 2.0 ** -23 * (x.double().abs() @ wu.double().abs().T)
    check(h, activation64(cfk.ACT_SILU, z)[0] * u, gated_bound(cfk.ACT_SILU, z, u, *e, cfk.FP16))
    gate0, up0 = gate.double(), up.double()
    lib.ffn_gated_backward(dh, x, wg, wu, gate, up, gate, up, dx=dx, dw_gate=dwg, dw_up=dwu, dh_stride=stride, dpre_stride=stride,
                           dx_stride=stride, **kw)
    lib.check_device()
    value, slope = activation64(cfk.ACT_SILU, gate0)
    d = dh.double()
    check(gate, d * up0 * slope, 3 * ACT_REL * (d * up0).abs() + half(cfk.FP16) * (d * up0 * slope).abs() + TINY[cfk.FP16])
    dg, du, w = gate.double(), up.double(), (wg.double(), wu.double())
    want = dg @ w[0] + du @ w[1]
    b = 2 * n * 2.0 ** -23 * (dg.abs() @ w[0].abs() + du.abs() @ w[1].abs())
    check(dx, want, b + half(cfk.FP16) * (want.abs() + b) + TINY[cfk.FP16])
    want = du.T @ x.double()
    b = m * 2.0 ** -23 * (du.abs().T @ x.double().abs())
    check(dwu, want, b + half(cfk.FP16) * (want.abs() + b) + TINY[cfk.FP16])


@pytest.mark.parametrize("m,n,k", [(1, 256, 4096), (2, 256, 64), (2048, 2048, 256)])
def test_products_skip_together_behind_a_wait_that_ran_out(lib, cuda, m, n, k):
    """With the status word set the products write nothing; once it has been read the same calls run.  One token: clusters that
    share a reduction; two: single CTAs; many: CTA pairs."""
    outs, calls = block_calls(lib, m, n, k, 4)
    xq, sx, c, dx, dwg, dwu = outs[6:]
    calls(None)
    lib.check_device()
    want = [o.clone() for o in outs]
    plan = lib.ffn_plan(cfk.FfnGatedArgs(cfk.FP16, cfk.FP16, 0, m, n, k, 16, 16, 16, 16, None, None, None, None, None, 0, 0, 0, 0))
    assert (plan[0], plan[2] > 1) == {1: (1, True), 2: (1, False), 2048: (0, False)}[m]
    products = [outs[0], outs[1], outs[2], outs[5], c, dx, dwg, dwu]
    for o in products:
        o.fill_(-3)
    assert lib.selftest_wait_gives_up(20) == 0
    calls(None)
    rc, code = lib.device_status()
    assert rc == 6 and code == 901
    assert all(bool((o == -3).all()) for o in products)
    calls(None)
    lib.check_device()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
