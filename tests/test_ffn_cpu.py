"""Arguments that the feed-forward operators refuse, before they touch a device, and the layout of their structs."""
import ctypes as C
import random

import pytest

import cfk_b200 as cfk


def test_struct_layouts(lib):
    assert C.sizeof(cfk.GemmI8Args) == 4 * 4 + 6 * 8 + 3 * 8
    assert C.sizeof(cfk.FfnGatedArgs) == 6 * 4 + 9 * 8 + 4 * 8
    assert C.sizeof(cfk.FfnGatedBackwardArgs) == 5 * 4 + 4 + 11 * 8 + 7 * 8


def refused(call, *args, **kw):
    with pytest.raises(cfk.CfkError) as e:
        call(*args, **kw)
    return e.value.code


@pytest.mark.parametrize("over,code", [
    (dict(src=0), 1), (dict(dst=0), 1), (dict(scale=0), 1), (dict(scale=0x3002), 1), (dict(rows=0), 1), (dict(cols=0), 1),
    (dict(src_dtype=cfk.INT8), 1), (dict(src_dtype=cfk.E4M3), 1), (dict(src=0x1008), 1), (dict(dst=0x2008), 1),
    (dict(cols=72, src_stride=64, dst_stride=80), 1), (dict(cols=72), 1),        # a packed row of 72 bytes
    (dict(cols=20, src_stride=20, dst_stride=32), 1), (dict(cols=20, src_stride=24, dst_stride=24), 1),
    (dict(rows=-5), 1), (dict(src_stride=-64), 1),
])
def test_quantize_refuses(lib, over, code):
    kw = dict(src=0x1000, dst=0x2000, scale=0x3000, src_dtype=cfk.BF16, rows=4, cols=64, src_stride=0, dst_stride=0)
    kw.update(over)
    assert refused(lib.quantize_rows, kw.pop("src") or None, kw.pop("dst") or None, kw.pop("scale") or None, **kw) == code


@pytest.mark.parametrize("over,code", [
    (dict(a=None), 1), (dict(b=None), 1), (dict(c=None), 1), (dict(a_scale=None), 1), (dict(b_scale=None), 1),
    (dict(a_scale=0x4002), 1), (dict(bias=0x6001), 1), (dict(m=0), 1), (dict(n=-1), 1), (dict(k=0), 1),
    (dict(out_dtype=cfk.E4M3), 1), (dict(out_dtype=cfk.INT8), 1), (dict(a=0x1004), 1), (dict(c=0x3008), 1),
    (dict(k=72), 1), (dict(n=100), 1), (dict(n=100, c_stride=100), 1), (dict(a_stride=32), 1), (dict(b_stride=72), 1),
    (dict(k=131072), 2), (dict(c_stride=1 << 31), 1), (dict(m=0x7fffff01), 2),
    (dict(m=0x7fffff00, n=0x7fffff00, c_stride=0x7fffffc0), 2),
])
def test_gemm_i8_refuses(lib, over, code):
    kw = dict(a=0x1000, b=0x2000, c=0x3000, a_scale=0x4000, b_scale=0x5000, m=4, n=64, k=64, out_dtype=cfk.FP16)
    kw.update(over)
    assert refused(lib.gemm_i8, kw.pop("a"), kw.pop("b"), kw.pop("c"), **kw) == code
    assert lib.lib.cfk_gemm_i8(None, None) == 1


@pytest.mark.parametrize("over,code", [
    (dict(x=None), 1), (dict(w_up=None), 1), (dict(h=None), 1), (dict(m=0), 1), (dict(k=-4), 1),
    (dict(dtype=cfk.FP32, out_dtype=cfk.FP32), 1), (dict(dtype=cfk.E4M3), 1), (dict(out_dtype=cfk.FP16), 1),
    (dict(out_dtype=cfk.FP32), 1), (dict(activation=4), 1), (dict(activation=-1), 1), (dict(gate=0x5000), 1), (dict(up=0x5000), 1),
    (dict(x_scale=0x6000), 1), (dict(dtype=cfk.INT8), 1), (dict(dtype=cfk.INT8, x_scale=0x6000, gate_scale=0x7000), 1),
    (dict(x=0x1002), 1), (dict(w_gate=0x2008), 1), (dict(k=60), 1), (dict(x_stride=60, k=60), 1), (dict(n=60), 1),
    (dict(gate=0x5000, up=0x6008), 1), (dict(gate=0x5000, up=0x5000), 1), (dict(gate=0x4000, up=0x5000), 1), (dict(gate=0x5000, up=0x6000, pre_stride=32), 1), (dict(h_stride=56), 1),
    (dict(dtype=cfk.INT8, x_scale=0x6000, gate_scale=0x7000, up_scale=0x8000, k=131072), 2), (dict(m=0x7fffff01), 2),
])
def test_ffn_gated_refuses(lib, over, code):
    kw = dict(x=0x1000, w_gate=0x2000, w_up=0x3000, h=0x4000, dtype=cfk.BF16, out_dtype=cfk.BF16, activation=0, m=4, n=64, k=64)
    kw.update(over)
    assert refused(lib.ffn_gated, kw.pop("x"), kw.pop("w_gate"), kw.pop("w_up"), kw.pop("h"), **kw) == code
    assert lib.lib.cfk_ffn_gated(None, None) == 1


@pytest.mark.parametrize("over,code", [
    (dict(dh=None), 1), (dict(x=None), 1), (dict(w_gate=None), 1), (dict(gate=None), 1), (dict(dgate=None), 1), (dict(dup=None), 1),
    (dict(dw_gate=0xa000), 1), (dict(dw_up=0xa000), 1), (dict(dtype=cfk.INT8), 1), (dict(dtype=cfk.FP32), 1), (dict(activation=9), 1),
    (dict(m=0), 1), (dict(dh=0x1008), 1), (dict(dx=0x9004), 1), (dict(dw_gate=0xa000, dw_up=0xb002), 1),
    (dict(dgate=0x8000), 1),                              # one buffer for both gradients
    (dict(dgate=0x6000), 1), (dict(dup=0x5000), 1),       # crossed: dgate on up, dup on gate
    (dict(dgate=0x1000), 1), (dict(dup=0x1000), 1),       # on dh
    (dict(dgate=0x5000, dpre_stride=128), 1),             # in place, other stride
    (dict(n=60), 1), (dict(dx=0x9000, dx_stride=32), 1), (dict(w_stride=68), 1),
    (dict(m=1 << 30, n=256), 2), (dict(m=0x7fffffff), 2),
])
def test_ffn_gated_backward_refuses(lib, over, code):
    kw = dict(dh=0x1000, x=0x2000, w_gate=0x3000, w_up=0x4000, gate=0x5000, up=0x6000, dgate=0x7000, dup=0x8000, dtype=cfk.BF16,
              activation=0, m=4, n=64, k=64)
    kw.update(over)
    order = ["dh", "x", "w_gate", "w_up", "gate", "up", "dgate", "dup"]
    assert refused(lib.ffn_gated_backward, *[kw.pop(o) for o in order], **kw) == code
    assert lib.lib.cfk_ffn_gated_backward(None, None) == 1


P = list(range(0x1000, 0x10000, 0x1000))
TOKENS = [16, 32, 48, 64, 96, 128, 192, 256]


def product(m, n, k, out=cfk.BF16):
    return cfk.GemmI8Args(out, m, n, k, P[0], P[1], P[2], P[3], P[4], None, 1 << 20, 1 << 20, 1 << 20)


def gated(m, n, k, dtype=cfk.BF16):
    scales = (P[4], P[5], P[6]) if dtype == cfk.INT8 else (None, None, None)
    return cfk.FfnGatedArgs(dtype, cfk.BF16, 0, m, n, k, P[0], P[1], P[2], P[3], None, None, *scales, *[1 << 20] * 4)


def backward(m, n, k, dx=True, dw=True):
    return cfk.FfnGatedBackwardArgs(cfk.BF16, 0, m, n, k, *P[:8], P[8] if dx else None, *((P[9], P[10]) if dw else (None, None)),
                                    *[1 << 20] * 7)


def test_plans_can_be_run_and_cover_both_kernels(lib):
    """Over sizes and types: tile widths and cluster sizes that the kernels have; few tokens go to the kernel for them, large products to
    the CTA pairs; the plan does not depend on the output's type, addresses or strides."""
    rng = random.Random(5)
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))      # noqa: E731
    seen = set()
    for _ in range(3000):
        m, n, k = log(1, 20000), log(1, 20000), log(1, 20000)
        for args, widest in ((product(m, n, k), 256), (gated(m, n, k), 128), (gated(m, n, k, cfk.INT8), 128)):
            few, width, parts = plan = lib.ffn_plan(args)
            seen.add((widest, few))
            if few:
                assert width in TOKENS and width <= widest and (width == 16 or TOKENS[TOKENS.index(width) - 1] < m)
                assert parts in (1, 2, 3, 4, 6, 8)
            else:
                assert width in (64, 96, 128) and parts == 1
            if m <= 4 and n >= 128:
                assert few
            if m * n >= 256 * 256 * 74 * 4 and m >= 2048 and k >= 512:
                assert not few
        assert lib.ffn_plan(product(m, n, k, cfk.FP32)) == lib.ffn_plan(product(m, n, k))
        few, width, parts, dw = lib.ffn_plan(backward(m, n, k))
        assert (width in TOKENS and parts in (1, 2, 3, 4, 6, 8)) if few else (width in (64, 96, 128) and parts == 1)
        assert dw in (64, 96, 128)
        assert lib.ffn_plan(backward(m, n, k, dx=False))[:3] == (0, 0, 1) and lib.ffn_plan(backward(m, n, k, dw=False))[3] == 0
    assert seen == {(256, 0), (256, 1), (128, 0), (128, 1)}


def test_plans_refuse_what_the_calls_refuse(lib):
    for args in (product(0, 8, 8), gated(1, 0, 8), backward(1, 8, 0)):
        with pytest.raises(cfk.CfkError) as e:
            lib.ffn_plan(args)
        assert e.value.code == 1
    for name in ("cfk_gemm_i8_plan", "cfk_ffn_gated_plan", "cfk_ffn_gated_backward_plan"):
        assert getattr(lib.lib, name)(None, None) == 1
    assert lib.lib.cfk_gemm_i8_plan(C.byref(product(8, 8, 8)), None) == 1


def test_int8_is_no_type_of_the_other_entry_points(lib):
    assert lib.lib.cfk_fill(0x1000, cfk.INT8, 10, 1, 0, 0, 1.0, 0.0, None) == 1
    assert lib.lib.cfk_convert(0x1000, cfk.INT8, 0x2000, cfk.FP32, 10, 1.0, None) == 1
    g = cfk.GemmArgs(cfk.INT8, 128, 128, 128, 1, 0x1000, 0x2000, 0x3000, 1.0, 0.0, 1, 1, None)
    assert lib.gemm_raw(g) == 2
