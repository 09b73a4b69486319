"""Results of the feed-forward calls that share memory with each other or with what is read: refused before a device is touched.  A call
that is not refused gets as far as the device, which is none here (status 5) or, with one, is a GPU test."""
import pytest

import cfk_b200 as cfk

M, N, K = 4, 64, 64                       # 16-bit matrices of 4 x 64: 512 bytes
SIZE = 0x200
SCALES = dict(x_scale=0x20000, gate_scale=0x21000, up_scale=0x22000)


def no_device():
    import torch
    return not torch.cuda.is_available()


pytestmark = pytest.mark.skipif(not no_device(), reason="made-up addresses: only where nothing can be launched")


def status(call, *args, **kw):
    with pytest.raises(cfk.CfkError) as e:
        call(*args, **kw)
    return e.value.code


def gated(lib, **over):
    kw = dict(x=0x10000, w_gate=0x11000, w_up=0x13000, h=0x15000, gate=None, up=None, dtype=cfk.BF16, out_dtype=cfk.BF16, activation=0,
              m=M, n=N, k=K)
    kw.update(over)
    return status(lib.ffn_gated, kw.pop("x"), kw.pop("w_gate"), kw.pop("w_up"), kw.pop("h"), **kw)


def backward(lib, **over):
    kw = dict(dh=0x10000, x=0x11000, w_gate=0x12000, w_up=0x14000, gate=0x16000, up=0x17000, dgate=0x18000, dup=0x19000, dx=0x1a000,
              dw_gate=0x1b000, dw_up=0x1d000, dtype=cfk.BF16, activation=0, m=M, n=N, k=K)
    kw.update(over)
    return status(lib.ffn_gated_backward, *[kw.pop(o) for o in ("dh", "x", "w_gate", "w_up", "gate", "up", "dgate", "dup")], **kw)


def gemm_i8(lib, **over):
    kw = dict(a=0x10000, b=0x11000, c=0x13000, a_scale=0x15000, b_scale=0x16000, bias=0x17000, m=M, n=N, k=K, out_dtype=cfk.FP32)
    kw.update(over)
    return status(lib.gemm_i8, kw.pop("a"), kw.pop("b"), kw.pop("c"), **kw)


def quantize(lib, **over):
    kw = dict(src=0x10000, dst=0x11000, scale=0x12000, src_dtype=cfk.BF16, rows=M, cols=K)
    kw.update(over)
    return status(lib.quantize_rows, kw.pop("src"), kw.pop("dst"), kw.pop("scale"), **kw)


def test_matrices_apart_are_accepted(lib):
    assert gated(lib) == gated(lib, gate=0x16000, up=0x17000) == gated(lib, dtype=cfk.INT8, **SCALES) == 5
    assert backward(lib) == backward(lib, dgate=0x16000, dup=0x17000) == backward(lib, dx=None) == backward(lib, dw_gate=None, dw_up=None) == 5
    assert gemm_i8(lib) == gemm_i8(lib, bias=None) == 5
    # inputs may be shared, and end to end is not shared
    assert gated(lib, w_up=0x11000) == gated(lib, h=0x10000 + SIZE) == backward(lib, w_up=0x12000, up=0x16000, dh=0x16000) == 5
    assert backward(lib, dx=0x11000 + SIZE) == backward(lib, dw_up=0x1b000 + N * K * 2) == 5


def test_halves_of_one_matrix_are_accepted(lib):
    """gate and up, and their gradients, as the two halves of a row of 2 n; outputs beside inputs in one row."""
    assert gated(lib, gate=0x16000, up=0x16000 + 2 * N, pre_stride=2 * N) == 5
    assert backward(lib, gate=0x16000, up=0x16000 + 2 * N, pre_stride=2 * N, dgate=0x18000, dup=0x18000 + 2 * N, dpre_stride=2 * N) == 5
    assert backward(lib, gate=0x16000, up=0x16000 + 2 * N, pre_stride=2 * N, dgate=0x16000, dup=0x16000 + 2 * N, dpre_stride=2 * N) == 5
    assert gated(lib, x=0x30000, x_stride=2 * K, h=0x30000 + 2 * K, h_stride=2 * K) == 5
    # the same with the results a row further down, and the last row of one before the first of the other
    assert gated(lib, x=0x30000, x_stride=2 * K, h=0x30000 + 6 * K, h_stride=2 * K) == 5
    assert gated(lib, x=0x30000, x_stride=2 * K, h=0x30000 + 3 * 4 * K + 2 * K, h_stride=2 * K) == 5


@pytest.mark.parametrize("over", [
    dict(h=0x10000), dict(h=0x11000), dict(h=0x13000), dict(h=0x10000 + SIZE - 16), dict(h=0x10000 - SIZE + 16),
    dict(gate=0x10000, up=0x17000), dict(gate=0x16000, up=0x11000), dict(gate=0x16000, up=0x16000 + SIZE - 16),
    dict(gate=0x16000, up=0x15000 + 16), dict(gate=0x16000, up=0x16000 + 2 * N - 16, pre_stride=2 * N),
    dict(x=0x30000, x_stride=2 * K, h=0x30000 + 2 * K + 16, h_stride=2 * K),               # the end of h's rows is in x's next rows
    dict(x=0x30000, x_stride=2 * K, h=0x30000 + 2 * K), dict(x=0x30000 + 16, h=0x30000, h_stride=2 * K),
    dict(dtype=cfk.INT8, **dict(SCALES, x_scale=0x15000)), dict(dtype=cfk.INT8, **dict(SCALES, gate_scale=0x15100)),
    dict(dtype=cfk.INT8, **dict(SCALES, up_scale=0x15000 - 16)),
])
def test_gated_refuses(lib, over):
    assert gated(lib, **over) == 1


@pytest.mark.parametrize("over", [
    dict(dw_up=0x1b000), dict(dx=0x18000), dict(dx=0x11000), dict(dgate=0x11000), dict(dw_gate=0x12000), dict(dw_up=0x14000), dict(dx=0x10000),
    dict(dx=0x16000), dict(dx=0x17010), dict(dup=0x11010), dict(dgate=0x12000), dict(dup=0x14000), dict(dw_gate=0x1a000), dict(dw_gate=0x18000),
    dict(dgate=0x16010), dict(dup=0x17000 + SIZE - 16), dict(dgate=0x18000, dup=0x18000 + SIZE - 16), dict(dw_up=0x1b000 + N * K * 2 - 16),
    dict(dgate=0x16000, dx=0x16000), dict(dgate=0x16000, dup=0x17000, dw_gate=0x17000),
    dict(gate=0x16000, up=0x16000 + 2 * N, pre_stride=2 * N, dgate=0x16000, dup=0x16000 + 2 * N - 16, dpre_stride=2 * N),
])
def test_backward_refuses(lib, over):
    assert backward(lib, **over) == 1


@pytest.mark.parametrize("over", [dict(c=0x10000), dict(c=0x11010), dict(c=0x15000), dict(b_scale=0x13010), dict(bias=0x13000 + 4 * M * N - 4)])
def test_gemm_i8_refuses(lib, over):
    assert gemm_i8(lib, **over) == 1


@pytest.mark.parametrize("over", [dict(dst=0x10000), dict(dst=0x10100), dict(scale=0x10000 + 2 * M * K - 4), dict(scale=0x11000), dict(src=0x10f00)])
def test_quantize_refuses(lib, over):
    assert quantize(lib, **over) == 1


def test_what_is_shared_agrees_with_a_list_of_bytes(lib):
    """Small matrices of many offsets and strides against the set of their bytes: a call is refused if and only if h and x share one,
    where the rows of both are the same distance apart or one of them has no gaps."""
    for x_stride in (16, 24, 40):
        for h_stride in (8, 16, 24, 40):
            if x_stride != h_stride and (x_stride, h_stride) not in ((16, 8), (24, 8), (40, 8)):
                continue
            for offset in range(-160, 400, 16):
                rows, base = 3, 0x40000
                x = {base + r * 2 * x_stride + b for r in range(rows) for b in range(32)}
                h = {base + offset + r * 2 * h_stride + b for r in range(rows) for b in range(16)}
                got = gated(lib, x=base, h=base + offset, m=rows, n=8, k=16, x_stride=x_stride, h_stride=h_stride, w_stride=16)
                certain = x_stride == h_stride or offset >= 0
                if certain or not x & h:
                    assert got == (1 if x & h else 5), (x_stride, h_stride, offset)
