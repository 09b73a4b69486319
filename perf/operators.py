"""The feed-forward operators that are measured: 8-bit integer products with a scale for each token and channel (with the
quantisation of the tokens that feeds them), and the gated feed-forward block, forward in 16 and 8 bits and backward.

`run` computes them in their plain form, or, with `own` set, through the library's Python binding.  Sizes are generic; `n` is the
width of the block or the output channels, `k` the width of the model or the reduction, `m` the tokens of the call.  Rows whose
length is not a multiple of 16 elements are padded to one, as the library asks for rows that start at 16-byte boundaries.
"""
import math
import os
import sys

import torch

own = False

TORCH = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4, "int8": 1}
ACTS = ["silu", "gelu", "gelu_tanh", "relu"]


def _linear(name, prec, m, n, k, bias=False):
    """Tokens in 16 bits through a layer with 8-bit weights: their quantisation and the product."""
    c = {"op": "linear", "prec": prec, "m": m, "n": n, "k": k, "bias": bias}
    return dict(c, name=name) if name else c


def _product(name, out, m, n, k, bias=False):
    """The product alone, of tokens that are held in 8 bits already (shared by several layers)."""
    c = {"op": "product", "prec": out, "m": m, "n": n, "k": k, "bias": bias}
    return dict(c, name=name) if name else c


def _gated(name, prec, m, n, k, act="silu", keep=False, out=None):
    """The gated block; prec int8 with output in `out`; `keep`: the pre-activations are written for a backward pass."""
    c = {"op": "gated", "prec": prec, "out": out or prec, "m": m, "n": n, "k": k, "act": act, "keep": keep}
    return dict(c, name=name) if name else c


def _backward(name, prec, m, n, k, act="silu"):
    c = {"op": "backward", "prec": prec, "m": m, "n": n, "k": k, "act": act}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token through a projection: latency, and the weights read once
        _linear("linear one token", "bf16", 1, 4096, 4096),
        # a step of a running batch through the projection back from the wide side
        _linear("linear batch step", "bf16", 48, 4096, 11264, bias=True),
        # a long prompt, or several at once
        _linear("linear prompt", "bf16", 8192, 8192, 8192),
        # lengths that no tile divides, result in 32 bits for what follows in them
        _product("product ragged", "fp32", 777, 1301, 2061, bias=True),
        # one new token through the block
        _gated("gated one token", "bf16", 1, 11264, 4096),
        # a step of a running batch with 8-bit weights
        _gated("gated i8 batch step", "int8", 16, 11264, 4096, out="bf16"),
        # a prompt with 8-bit weights
        _gated("gated i8 prompt", "int8", 2048, 11264, 4096, out="bf16"),
        # a long prompt in 16 bits
        _gated("gated prompt", "bf16", 4096, 11264, 4096),
        # a training step of uneven sizes, pre-activations kept
        _gated("gated train ragged", "fp16", 1000, 2731, 1027, act="gelu_tanh", keep=True),
        # gradients of a full training batch
        _backward("backward train", "bf16", 8192, 11264, 4096),
        # gradients at uneven sizes
        _backward("backward ragged", "fp16", 777, 2731, 1027, act="gelu"),
        # gradients of a short batch: the weights' traffic counts as much as the products
        _backward("backward short", "bf16", 64, 5632, 2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Mostly a multiple of 16 or 128, as widths are; now and then any length."""
    v = _log(rng, lo, hi)
    step = rng.choice([1, 16, 128, 128])
    return max(lo, v // step * step)


def draw(rng):
    op = rng.choice(["linear", "linear", "product", "gated", "gated", "gated i8", "backward", "backward"])
    m = _log(rng, 1, 64) if rng.random() < 0.35 else _log(rng, 1, 8192)
    n, k = _size(rng, 128, 11264), _size(rng, 128, 8192)
    limit = {"linear": 1.0e12, "product": 1.0e12, "gated": 3.5e11, "gated i8": 3.5e11, "backward": 2.8e12}[op]
    per = {"linear": 2.0, "product": 2.0, "gated": 4.0, "gated i8": 4.0, "backward": 8.0}[op]
    while per * m * n * k > limit:
        m = max(1, m // 2)
    prec = rng.choice(["bf16", "bf16", "fp16"])
    bias = rng.random() < 0.3
    if op == "linear":
        return _linear(None, prec, m, n, k, bias)
    if op == "product":
        return _product(None, rng.choice(["bf16", "fp16", "fp32"]), m, n, k, bias)
    act = rng.choice(["silu", "silu"] + ACTS[1:])
    if op == "gated":
        return _gated(None, prec, m, n, k, act, keep=rng.random() < 0.5)
    if op == "gated i8":
        return _gated(None, "int8", m, n, k, act, out=prec)
    return _backward(None, prec, m, n, k, act)


def _rows(rows, cols, dtype):
    """A matrix whose rows start at multiples of 16 elements; its padding holds zeros."""
    return torch.zeros(rows, (cols + 15) // 16 * 16, dtype=dtype, device="cuda")[:, :cols]


def _held(x, dtype):
    y = _rows(x.shape[0], x.shape[1], dtype)
    y.copy_(x)
    return y


def _tokens(g, m, k):
    """Activations: N(0, 1), with some channels an order of magnitude larger, as behind a norm with learned weights."""
    x = torch.randn(m, k, generator=g, device="cuda")
    loud = torch.rand(k, generator=g, device="cuda") < 0.005
    return x * torch.where(loud, 12.0, 1.0)


def _weights8(g, n, k):
    """8-bit weights of N(0, 1 / k), a scale for each output channel."""
    w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
    scale = w.abs().amax(1) / 127.0
    return _held(torch.round(w / scale[:, None]), torch.int8), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    m, n, k, op = case["m"], case["n"], case["k"], case["op"]
    st = dict(case)
    if op in ("linear", "product"):
        x = _tokens(g, m, k)
        st["w"], st["w_scale"] = _weights8(g, n, k)
        st["b"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        if op == "linear":
            st["x"] = _held(x, TORCH[case["prec"]])
            st["q"] = _rows(m, k, torch.int8)
            st["x_scale"] = torch.zeros(m, device="cuda")
        else:
            st["x_scale"] = x.abs().amax(1) / 127.0
            st["q"] = _held(torch.round(x / st["x_scale"][:, None]), torch.int8)
        st["y"] = _rows(m, n, TORCH[case["prec"]])
    elif op == "gated":
        x = _tokens(g, m, k)
        dt = TORCH[case["out"]]
        if case["prec"] == "int8":
            st["x_scale"] = x.abs().amax(1) / 127.0
            st["x"] = _held(torch.round(x / st["x_scale"][:, None]), torch.int8)
            st["wg"], st["wg_scale"] = _weights8(g, n, k)
            st["wu"], st["wu_scale"] = _weights8(g, n, k)
        else:
            st["x"] = _held(x, dt)
            st["wg"] = _held(torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k), dt)
            st["wu"] = _held(torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k), dt)
        st["h"] = _rows(m, n, dt)
        if case["keep"]:
            st["gate"], st["up"] = _rows(m, n, dt), _rows(m, n, dt)
    else:
        dt = TORCH[case["prec"]]
        st["x"] = _held(_tokens(g, m, k), dt)
        st["wg"] = _held(torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k), dt)
        st["wu"] = _held(torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k), dt)
        # the pre-activations of such tokens, and a gradient of the scale that a mean over the batch gives
        st["gate"] = _held(torch.randn(m, n, generator=g, device="cuda") * 1.3, dt)
        st["up"] = _held(torch.randn(m, n, generator=g, device="cuda") * 1.3, dt)
        st["dh"] = _held(torch.randn(m, n, generator=g, device="cuda") * 0.02, dt)
        st["dgate"], st["dup"] = _rows(m, n, dt), _rows(m, n, dt)
        st["dx"] = _rows(m, k, dt)
        st["dwg"], st["dwu"] = _rows(n, k, dt), _rows(n, k, dt)
    return st


def _act(name, g):
    if name == "silu":
        return g / (1.0 + torch.exp(-g))
    if name == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))
    return torch.clamp(g, min=0.0)


def _act_slope(name, g):
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s * (1.0 + g * (1.0 - s))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g * g * g))
        return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)
    return (g > 0).to(g.dtype)


def _run_plain(st):
    op = st["op"]
    if op in ("linear", "product"):
        if op == "linear":
            x = st["x"].float()
            x_scale = x.abs().amax(1) / 127.0
            q = torch.clamp(torch.round(x / x_scale[:, None]), -127.0, 127.0)
        else:
            x_scale, q = st["x_scale"], st["q"].float()
        # sums of products of 8-bit integers: exact in 32 bits for sums of these sizes (below 2^24)
        y = (q @ st["w"].float().T) * x_scale[:, None] * st["w_scale"][None, :]
        if st["b"] is not None:
            y = y + st["b"]
        y = y.to(TORCH[st["prec"]])
        return (y, x_scale) if op == "linear" else y
    if op == "gated":
        x, wg, wu = st["x"].float(), st["wg"].float(), st["wu"].float()
        gate, up = x @ wg.T, x @ wu.T
        if st["prec"] == "int8":
            gate = gate * st["x_scale"][:, None] * st["wg_scale"][None, :]
            up = up * st["x_scale"][:, None] * st["wu_scale"][None, :]
        dt = TORCH[st["out"]]
        h = (_act(st["act"], gate) * up).to(dt)
        return (h, gate.to(dt), up.to(dt)) if st["keep"] else h
    x, wg, wu, gate, up, dh = (st[t].float() for t in ("x", "wg", "wu", "gate", "up", "dh"))
    dgate = dh * up * _act_slope(st["act"], gate)
    dup = dh * _act(st["act"], gate)
    dt = TORCH[st["prec"]]
    return tuple(t.to(dt) for t in (dgate @ wg + dup @ wu, dgate.T @ x, dup.T @ x, dgate, dup))


def _library():
    pkg = os.path.join(os.getcwd(), "cutlass-kernels_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import cfk_b200
    return cfk_b200, cfk_b200.load()


def _run_own(st):
    cfk, lib = _library()
    op, m, n, k = st["op"], st["m"], st["n"], st["k"]
    code = {"fp16": cfk.FP16, "bf16": cfk.BF16, "fp32": cfk.FP32, "int8": cfk.INT8}
    stream = torch.cuda.current_stream().cuda_stream
    if op in ("linear", "product"):
        q, y = st["q"], st["y"]
        if op == "linear":
            lib.quantize_rows(st["x"], q, st["x_scale"], src_dtype=code[st["prec"]], rows=m, cols=k,
                              src_stride=st["x"].stride(0), dst_stride=q.stride(0), stream=stream)
        lib.gemm_i8(q, st["w"], y, m=m, n=n, k=k, out_dtype=code[st["prec"]], a_scale=st["x_scale"], b_scale=st["w_scale"],
                    bias=st["b"], a_stride=q.stride(0), b_stride=st["w"].stride(0), c_stride=y.stride(0), stream=stream)
        return (y, st["x_scale"]) if op == "linear" else y
    act = {"silu": cfk.ACT_SILU, "gelu": cfk.ACT_GELU, "gelu_tanh": cfk.ACT_GELU_TANH, "relu": cfk.ACT_RELU}[st["act"]]
    x, wg, wu = st["x"], st["wg"], st["wu"]
    if op == "gated":
        gate, up = st.get("gate"), st.get("up")
        lib.ffn_gated(x, wg, wu, st["h"], dtype=code[st["prec"]], out_dtype=code[st["out"]], activation=act, m=m, n=n, k=k,
                      gate=gate, up=up, x_scale=st.get("x_scale"), gate_scale=st.get("wg_scale"), up_scale=st.get("wu_scale"),
                      x_stride=x.stride(0), w_stride=wg.stride(0), h_stride=st["h"].stride(0),
                      pre_stride=gate.stride(0) if st["keep"] else 0, stream=stream)
        return (st["h"], gate, up) if st["keep"] else st["h"]
    lib.ffn_gated_backward(st["dh"], x, wg, wu, st["gate"], st["up"], st["dgate"], st["dup"], dx=st["dx"], dw_gate=st["dwg"],
                           dw_up=st["dwu"], dtype=code[st["prec"]], activation=act, m=m, n=n, k=k, x_stride=x.stride(0),
                           w_stride=wg.stride(0), pre_stride=st["gate"].stride(0), dh_stride=st["dh"].stride(0),
                           dpre_stride=st["dgate"].stride(0), dx_stride=st["dx"].stride(0), dw_stride=st["dwg"].stride(0),
                           stream=stream)
    return st["dx"], st["dwg"], st["dwu"], st["dgate"], st["dup"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    m, n, k, e = case["m"], case["n"], case["k"], SIZE[case["prec"]]
    if case["op"] == "linear":
        return {"bytes": e * m * k + n * k + e * m * n + 8 * m + 4 * n * (2 if case["bias"] else 1), "flops": 2.0 * m * n * k}
    if case["op"] == "product":
        return {"bytes": m * k + n * k + e * m * n + 4 * m + 4 * n * (2 if case["bias"] else 1), "flops": 2.0 * m * n * k}
    if case["op"] == "gated":
        scales = 4 * (m + 2 * n) if case["prec"] == "int8" else 0
        return {"bytes": e * (m * k + 2 * n * k) + SIZE[case["out"]] * m * n * (3 if case["keep"] else 1) + scales,
                "flops": 4.0 * m * n * k}
    return {"bytes": e * (2 * m * k + 4 * n * k + 5 * m * n), "flops": 8.0 * m * n * k}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------
def _activation64(name, z):
    """(value, derivative) of the activation at z, in 64 bits."""
    if name == "relu":
        pos = z > 0
        return torch.where(pos, z, torch.zeros_like(z)), pos.double()
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * torch.sigmoid(-z)
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / 2.0 ** 0.5)
        return z * cdf, cdf + z * torch.exp(-z * z / 2.0) / (2.0 * math.pi) ** 0.5
    # 0.5 (1 + tanh(a)) is the logistic function of 2 a
    a2 = 2.0 * (2.0 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)
    p = torch.sigmoid(a2)
    slope = 2.0 * (2.0 / math.pi) ** 0.5 * (1.0 + 0.134145 * z ** 2)
    return z * p, p + z * p * torch.sigmoid(-a2) * slope


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("linear", "product"):
        if op == "linear":
            x = st["x"].double()
            scale64 = x.abs().max(dim=1).values / 127.0
            scale = scale64.float().double()          # the scale is held in 32 bits, and the integers are relative to it
            whole = torch.round(x / scale.unsqueeze(1)).clamp(-127, 127)
        else:
            scale64 = scale = st["x_scale"].double()
            whole = st["q"].double()
        y = torch.matmul(whole, st["w"].double().t())
        y = y * torch.outer(scale, st["w_scale"].double())
        if case["bias"]:
            y += st["b"].double().unsqueeze(0)
        return (y, scale64) if op == "linear" else y
    if op == "gated":
        x, wg, wu = st["x"].double(), st["wg"].double(), st["wu"].double()
        if case["prec"] == "int8":
            x = x * st["x_scale"].double().unsqueeze(1)
            wg = wg * st["wg_scale"].double().unsqueeze(1)
            wu = wu * st["wu_scale"].double().unsqueeze(1)
        z, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
        h = _activation64(case["act"], z)[0] * u
        return (h, z, u) if case["keep"] else h
    z, u, d = st["gate"].double(), st["up"].double(), st["dh"].double()
    value, slope = _activation64(case["act"], z)
    dz, du = d * u * slope, d * value
    x = st["x"].double()
    dx = torch.matmul(dz, st["wg"].double()) + torch.matmul(du, st["wu"].double())
    return dx, torch.matmul(dz.t(), x), torch.matmul(du.t(), x), dz, du
