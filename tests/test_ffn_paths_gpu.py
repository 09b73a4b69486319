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


# ---- several tiles per pair, rings that turn, two lists ----------------------------------------------------------------------------
def up_to(a, b):
    return -(-a // b)


def product_args(m, n, k):
    return cfk.GemmI8Args(cfk.FP32, m, n, k, 0x1000, 0x2000, 0x3000, 0x4000, 0x5000, None, *[1 << 20] * 3)


def gated_args(dtype, m, n, k):
    scales = (0x5000, 0x6000, 0x7000) if dtype == cfk.INT8 else (None,) * 3
    return cfk.FfnGatedArgs(dtype, cfk.BF16 if dtype == cfk.INT8 else dtype, 0, m, n, k, 0x1000, 0x2000, 0x3000, 0x4000, None, None, *scales,
                            *[1 << 20] * 4)


def check_product(lib, m, n, k, out, bias, seed):
    g = gen(seed)
    (a, sa), (b, sb) = quantized(g, m, k), quantized(g, n, k)
    a, b = held(a, torch.int8), held(b, torch.int8)
    bs = randn(g, n) if bias else None
    c = matrix(m, n, TORCH[out])
    lib.gemm_i8(a, b, c, m=m, n=n, k=k, out_dtype=out, a_scale=sa, b_scale=sb, bias=bs, a_stride=a.stride(0), b_stride=b.stride(0),
                c_stride=c.stride(0))
    lib.check_device()
    y0 = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()
    y = y0 + bs.double() if bias else y0
    check(c, y, 4 * 2.0 ** -24 * (y0.abs() + y.abs()) + half(out) * y.abs() + TINY[out])


def check_gated(lib, dtype, out, act, m, n, k, seed, keep=True):
    """The kept pre-activations and h, every element (bounds as in test_ffn_gpu.py: |act'| <= 1.13, 1e-5 for the activation)."""
    g, kw, dt = gen(seed), {}, TORCH[out]
    if dtype == cfk.INT8:
        (x, sx), (wg, sg), (wu, su) = quantized(g, m, k), quantized(g, n, k), quantized(g, n, k)
        sg, su = sg / math.sqrt(k), su / math.sqrt(k)
        kw = dict(x_scale=sx, gate_scale=sg, up_scale=su)
    else:
        x, wg, wu = randn(g, m, k), randn(g, n, k) / math.sqrt(k), randn(g, n, k) / math.sqrt(k)
    x, wg, wu = (held(t, TORCH[dtype]) for t in (x, wg, wu))
    h, gate, up = matrix(m, n, dt), matrix(m, n, dt) if keep else None, matrix(m, n, dt) if keep else None
    lib.ffn_gated(x, wg, wu, h, dtype=dtype, out_dtype=out, activation=act, m=m, n=n, k=k, gate=gate, up=up, x_stride=x.stride(0),
                  w_stride=wg.stride(0), h_stride=h.stride(0), pre_stride=gate.stride(0) if keep else 0, **kw)
    lib.check_device()
    xd, gd, ud = x.double(), wg.double(), wu.double()
    z, u = xd @ gd.T, xd @ ud.T
    if dtype == cfk.INT8:
        z, u = z * sx.double()[:, None] * sg.double(), u * sx.double()[:, None] * su.double()
        ez, eu = 4 * 2.0 ** -24 * z.abs(), 4 * 2.0 ** -24 * u.abs()
    else:
        ez, eu = (k * 2.0 ** -23 * (xd.abs() @ w.abs().T) for w in (gd, ud))
    value = activation64(act, z)[0]
    e = 1.13 * ez * (u.abs() + eu) + eu * value.abs() + 1e-5 * (value * u).abs()
    check(h, value * u, e + half(out) * ((value * u).abs() + e) + TINY[out] + 1e-30)
    if keep:
        check(gate, z, ez + half(out) * (z.abs() + ez) + TINY[out])
        check(up, u, eu + half(out) * (u.abs() + eu) + TINY[out])


# (m, n, k), tile width: more than 8 k-blocks (the ring turns) and a pair with a third tile (both accumulators are used again)
@pytest.mark.parametrize("m,n,k,width,tiles", [(266, 14261, 663, 128, 4), (3877, 1713, 609, 96, 4), (7525, 419, 998, 64, 3)])
@pytest.mark.parametrize("dtype", [cfk.FP16, cfk.BF16])
def test_gated_16_bits_with_several_tiles_per_pair(lib, cuda, dtype, m, n, k, width, tiles):
    assert lib.ffn_plan(gated_args(dtype, m, n, k))[:2] == (0, width)
    assert up_to(up_to(m, 256) * up_to(n, width), PAIRS) == tiles and up_to(k, 64) >= 9
    for act in (ACTS[0], ACTS[2]):
        check_gated(lib, dtype, dtype, act, m, n, k, seed=m, keep=act == ACTS[0])


@pytest.mark.parametrize("m,n,k,width,tiles", [(263, 14505, 1042, 128, 4), (1795, 3465, 1072, 96, 4), (7601, 401, 2025, 64, 3)])
def test_gated_8_bits_with_several_tiles_per_pair(lib, cuda, m, n, k, width, tiles):
    assert lib.ffn_plan(gated_args(cfk.INT8, m, n, k))[:2] == (0, width)
    assert up_to(up_to(m, 256) * up_to(n, width), PAIRS) == tiles and up_to(k, 128) >= 9
    for out, act in ((cfk.BF16, ACTS[0]), (cfk.FP16, ACTS[1])):
        check_gated(lib, cfk.INT8, out, act, m, n, k, seed=m, keep=out == cfk.FP16)


@pytest.mark.parametrize("m,n,k,width,tiles", [(842, 14266, 1026, 128, 4), (1612, 7974, 1085, 96, 4), (7783, 781, 2100, 64, 3)])
@pytest.mark.parametrize("out", [cfk.BF16, cfk.FP32])
def test_8_bit_products_with_several_tiles_per_pair(lib, cuda, out, m, n, k, width, tiles):
    assert lib.ffn_plan(product_args(m, n, k))[:2] == (0, width)
    assert up_to(up_to(m, 256) * up_to(n, 2 * width), PAIRS) == tiles and up_to(k, 128) >= 9
    check_product(lib, m, n, k, out, out == cfk.FP32, seed=m)


@pytest.mark.parametrize("m,n,k,swapped,unequal,most", [
    (541, 546, 5398, False, False, False), (1285, 647, 5589, False, False, True), (549, 525, 4750, False, True, False),
    (1065, 525, 5486, False, True, True), (1923, 264, 4200, True, False, False), (1388, 518, 5466, True, False, True),
    (1617, 277, 3865, True, True, False), (1282, 559, 4957, True, True, True), (4000, 2100, 3000, False, None, True)])
@pytest.mark.parametrize("dtype", [cfk.FP16, cfk.BF16])
def test_backward_whose_pairs_have_tiles_of_both_lists(lib, cuda, dtype, m, n, k, swapped, unequal, most):
    """dx and the weights' gradients in one launch, the list of longer tiles first.  Pairs with one tile more of the first list take a
    share of the second: the tiles that the other pairs could do in the time of that tile do not take up the whole second list (a
    tile of the first list takes at most twice as long per k-block)."""
    b = Backward(dtype, m, n, k, m)
    few, width, _, dw = b.plan()
    assert few == 0
    tiles = [up_to(m, 256) * up_to(k, 2 * width), 2 * up_to(n, 256) * up_to(k, 2 * dw)]
    blocks = [2 * up_to(n, 64), up_to(m, 64)]
    assert swapped == (blocks[1] > blocks[0]) and unequal in (None, width != dw)
    if swapped:
        tiles.reverse(), blocks.reverse()
    pairs = min(PAIRS, sum(tiles))
    more = tiles[0] % pairs
    assert most == (tiles[0] >= pairs) and more > 0 and tiles[1] >= pairs + 2 * max(1, blocks[0] / blocks[1]) * (pairs - more)
    act = ACTS[(m + dtype) % 4]
    b.check(act, *b.run(lib, act))


# CTAs of clusters of so many parts that are resident with one CTA per SM; bytes of half and of all of an SM's shared memory for a ring
ONE_PER_SM = {1: 148, 2: 74, 3: 45, 4: 33, 6: 22, 8: 15}
HALF_RING, FULL_RING = 113 * 1024 - 1280, 226 * 1024 - 1280


def few_cut(plan, weights, m, n, k, block):
    """(two CTAs per SM, waves beyond the resident, parts, turns of the ring) of a call in the kernel for few tokens."""
    few, width, parts = plan
    assert few
    stage = weights * 16384 + width * 128
    tiles = up_to(n, 128) * up_to(m, width)
    two = HALF_RING // stage >= 3 and tiles > ONE_PER_SM[parts]
    stages = min(12, (HALF_RING if two else FULL_RING) // stage)
    return two, tiles > (2 if two else 1) * ONE_PER_SM[parts], parts, up_to(k, block) // parts // stages


@pytest.mark.parametrize("m,n,k,two,waves,parts", [
    (1, 1042, 800, False, False, 1), (1, 3078, 3347, False, False, 4), (33, 39571, 721, False, True, 1), (41, 2025, 1529, True, False, 3),
    (1, 19127, 393, True, False, 1), (1, 39340, 417, True, True, 1), (9, 25600, 2000, True, False, 1)])
@pytest.mark.parametrize("dtype", [cfk.FP16, cfk.BF16])
def test_few_tokens_gated_16_bits_turn_their_ring(lib, cuda, dtype, m, n, k, two, waves, parts):
    *cut, turns = few_cut(lib.ffn_plan(gated_args(dtype, m, n, k)), 2, m, n, k, 64)
    assert tuple(cut) == (two, waves, parts) and turns >= 2
    check_gated(lib, dtype, dtype, ACTS[m % 4], m, n, k, seed=n)


@pytest.mark.parametrize("m,n,k,two,waves,parts", [
    (31, 2975, 3384, False, False, 2), (1, 1060, 1598, False, False, 1), (37, 38421, 1309, False, True, 1), (47, 2041, 3049, True, False, 3),
    (1, 19845, 780, True, False, 1), (1, 39099, 819, True, True, 1), (9, 25600, 2000, True, False, 1)])
def test_few_tokens_gated_8_bits_turn_their_ring(lib, cuda, m, n, k, two, waves, parts):
    *cut, turns = few_cut(lib.ffn_plan(gated_args(cfk.INT8, m, n, k)), 2, m, n, k, 128)
    assert tuple(cut) == (two, waves, parts) and turns >= 2
    check_gated(lib, cfk.INT8, cfk.BF16 if m % 2 else cfk.FP16, ACTS[m % 4], m, n, k, seed=n)


@pytest.mark.parametrize("m,n,k,two,waves,parts", [
    (1, 5394, 3082, False, False, 1), (1, 19270, 1542, True, False, 1), (1, 38514, 1646, True, True, 1), (40, 25600, 4000, True, False, 1)])
def test_few_tokens_8_bit_products_turn_their_ring(lib, cuda, m, n, k, two, waves, parts):
    *cut, turns = few_cut(lib.ffn_plan(product_args(m, n, k)), 1, m, n, k, 128)
    assert tuple(cut) == (two, waves, parts) and turns >= 2
    check_product(lib, m, n, k, [cfk.FP16, cfk.BF16, cfk.FP32][n % 3], bool(n % 2), seed=n)


@pytest.mark.parametrize("m", [5, 300])
def test_both_weight_gradients_of_rows_that_lie_far_apart(lib, cuda, m):
    """Matrices whose last rows begin behind 2^31 elements, in place; dw_gate and dw_up packed."""
    n, k, dt = 72, 40, torch.float16
    stride = ((1 << 31) // m + 4096) // 16 * 16
    g = gen(m)

    def far(cols, x=None):
        t = torch.empty(m * stride, dtype=dt, device="cuda").view(m, stride)[:, :cols]
        return t if x is None else t.copy_(x)

    dh, x, gate, up = far(n, randn(g, m, n)), far(k, randn(g, m, k)), far(n, randn(g, m, n)), far(n, randn(g, m, n))
    d, z, u, xd = dh.double(), gate.double(), up.double(), x.double()
    wg, wu = (randn(g, n, k) / 6).to(dt), (randn(g, n, k) / 6).to(dt)
    dwg, dwu = torch.zeros_like(wg), torch.zeros_like(wu)
    lib.ffn_gated_backward(dh, x, wg, wu, gate, up, gate, up, dw_gate=dwg, dw_up=dwu, dtype=cfk.FP16, activation=cfk.ACT_GELU, m=m, n=n, k=k,
                           x_stride=stride, dh_stride=stride, pre_stride=stride, dpre_stride=stride)
    lib.check_device()
    value, slope = activation64(cfk.ACT_GELU, z)
    check(gate, d * u * slope, 3e-5 * (d * u).abs() + half(cfk.FP16) * (d * u * slope).abs() + TINY[cfk.FP16])
    check(up, d * value, 3e-5 * (d * value).abs() + half(cfk.FP16) * (d * value).abs() + TINY[cfk.FP16])
    for got, t in ((dwg, gate.double()), (dwu, up.double())):
        e = m * 2.0 ** -23 * (t.abs().T @ xd.abs())
        check(got, t.T @ xd, e + half(cfk.FP16) * ((t.T @ xd).abs() + e) + TINY[cfk.FP16])
