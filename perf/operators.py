"""The operators of the microscaled 4-bit (MXFP4) path and of the gated feed-forward block, as cases.

    quant   a tensor into MXFP4 (32 values share a power-of-two scale), and back to the values it stands for
    gemm    the product of two MXFP4 operands
    gated   act(A Wg^T) * (A Wu^T) on MXFP4 operands
    ffn     a whole MXFP4 feed-forward block: quantise, gated projections, down projection
    dense   act(X Wg^T) * (X Wu^T) in bf16 or fp16, with G and U kept where a backward pass follows
    grad    that block's backward pass: gradients of X, Wg and Wu

With `own` the calls go to pantheon_b200; without, they are elementary torch operations in 32 bits.
"""
import math

import torch

own = False

_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # a decode step's activations, 4 rows of an 8192-wide model: latency
        {"name": "quant_decode", "op": "quant", "m": 4, "k": 8192, "pad": 0, "dtype": "bf16"},
        # a slice of a wider fp32 buffer, with a width that is no multiple of the block
        {"name": "quant_ragged", "op": "quant", "m": 3001, "k": 4099, "pad": 13, "dtype": "f32"},
        # a whole weight matrix
        {"name": "quant_weights", "op": "quant", "m": 28672, "k": 8192, "pad": 0, "dtype": "bf16"},
        # the decode projection of one token
        {"name": "gemm_token", "op": "gemm", "m": 1, "n": 28672, "k": 8192, "out": "bf16"},
        # a short prompt with ragged sizes
        {"name": "gemm_ragged", "op": "gemm", "m": 333, "n": 1001, "k": 4128, "out": "bf16"},
        # a prefill projection
        {"name": "gemm_prompt", "op": "gemm", "m": 4096, "n": 8192, "k": 8192, "out": "bf16"},
        # the gated projections of a batch of 16 sequences, one token each
        {"name": "gated_decode", "op": "gated", "m": 16, "n": 14336, "k": 4096, "act": "silu"},
        # the whole block on a prompt
        {"name": "ffn_prompt", "op": "ffn", "m": 2048, "n": 28672, "k": 8192, "act": "silu"},
        # a training step's forward pass, its intermediates kept
        {"name": "dense_train", "op": "dense", "m": 4096, "n": 8192, "k": 4096, "act": "silu", "dtype": "bf16", "keep": True},
        # inference with ragged sizes
        {"name": "dense_ragged", "op": "dense", "m": 777, "n": 2728, "k": 1032, "act": "gelu", "dtype": "f16", "keep": False},
        # the same training step's backward pass, and a ragged one
        {"name": "grad_train", "op": "grad", "m": 4096, "n": 8192, "k": 4096, "act": "silu", "dtype": "bf16"},
        {"name": "grad_ragged", "op": "grad", "m": 515, "n": 1368, "k": 520, "act": "gelu", "dtype": "f16"},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step`, spread over the logarithm of the range."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return min(hi, max(lo, int(v) // step * step)) if step > 1 else min(hi, max(lo, int(v)))


def draw(rng):
    op = rng.choice(["quant", "gemm", "gated", "ffn", "dense", "grad"])
    if op == "quant":
        m, k = _log(rng, 1, 28672), _log(rng, 32, 8192)
        return {"op": op, "m": m, "k": k, "pad": rng.choice([0, 0, 1, 8, 37]), "dtype": rng.choice(["bf16", "f16", "f32"])}
    act = rng.choice(["silu", "gelu"])
    if op == "gemm":
        return {"op": op, "m": _log(rng, 1, 4096), "n": _log(rng, 16, 28672), "k": _log(rng, 32, 8192, 32), "out": rng.choice(["bf16", "bf16", "f32"])}
    if op == "gated":
        return {"op": op, "m": _log(rng, 1, 2048), "n": _log(rng, 16, 28672), "k": _log(rng, 32, 8192, 32), "act": act}
    if op == "ffn":
        return {"op": op, "m": _log(rng, 1, 2048), "n": _log(rng, 64, 28672, 32), "k": _log(rng, 64, 8192, 32), "act": act}
    c = {"op": op, "m": _log(rng, 1, 4096), "n": _log(rng, 64, 8192, 8), "k": _log(rng, 64, 4096, 8), "act": act, "dtype": rng.choice(["bf16", "f16"])}
    return {**c, "keep": rng.random() < 0.5} if op == "dense" else c


# ---------------------------------------------------------------- inputs

def _up(a, b):
    return -(-a // b) * b


def _power(byte):
    """fp32 2^(byte - 127), from its bits."""
    b = byte.to(torch.int32)
    return torch.where(b > 0, b << 23, torch.full_like(b, 1 << 22)).view(torch.float32)


def _scale_and_codes(x):
    """fp32 [M, K], K % 32 == 0 -> (scale byte [M, K/32], code [M, K]) of the MX conversion."""
    b = x.reshape(x.shape[0], -1, 32)
    amax = b.abs().amax(-1)
    e = ((amax.view(torch.int32) >> 23) - 129).clamp(min=-127)            # floor(log2 amax) - 2
    a = b.abs() * _power(127 - e)[..., None]
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
            + 8 * torch.signbit(b).to(torch.uint8))
    return (e + 127).to(torch.uint8), code.reshape(x.shape)


def _pack(x):
    """fp32 [M, K] -> (codes [M, K/2], scale atoms)."""
    e, code = _scale_and_codes(x)
    rows, blocks = e.shape
    t = torch.zeros((_up(rows, 128), _up(blocks, 4)), dtype=torch.uint8, device=x.device)
    t[:rows, :blocks] = e
    atoms = t.view(t.shape[0] // 128, 4, 32, t.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), atoms


def _activations(g, m, k):
    """Unit normal with a few wide columns and some rows of small values, as a norm's output has."""
    x = torch.randn((m, k), device="cuda", generator=g)
    x *= 1 + 7 * (torch.rand((1, k), device="cuda", generator=g) < 0.01)
    x *= torch.where(torch.rand((m, 1), device="cuda", generator=g) < 0.05, 1e-3, 1.0)
    return x


def _weight(g, n, k, scale=1.0):
    return torch.randn((n, k), device="cuda", generator=g).mul_(scale / math.sqrt(k))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, m, k = case["op"], case["m"], case["k"]
    s = {"case": case}
    if op == "quant":
        x = _activations(g, m, k + case["pad"]).to(_TYPES[case["dtype"]])
        s["x"] = x[:, :k]
        return s
    n = case["n"]
    if op == "gemm":
        s["a"] = _pack(_activations(g, m, k))
        s["b"] = _pack(_weight(g, n, k))
    elif op == "gated":
        s["a"] = _pack(_activations(g, m, k))
        s["g"], s["u"] = _pack(_weight(g, n, k)), _pack(_weight(g, n, k))
    elif op == "ffn":
        s["x"] = _activations(g, m, k).to(torch.bfloat16)
        s["g"], s["u"], s["d"] = _pack(_weight(g, n, k)), _pack(_weight(g, n, k)), _pack(_weight(g, k, n))
    else:
        t = _TYPES[case["dtype"]]
        s["x"] = _activations(g, m, k).to(t)
        s["wg"], s["wu"] = _weight(g, n, k).to(t), _weight(g, n, k).to(t)
        if op == "grad":
            # what the forward pass left: unit normal projections, and the gradient that arrives
            s["g"] = torch.randn((m, n), device="cuda", generator=g).to(t)
            s["u"] = torch.randn((m, n), device="cuda", generator=g).to(t)
            s["dh"] = torch.randn((m, n), device="cuda", generator=g).mul_(0.1).to(t)
    return s


# ---------------------------------------------------------------- the plain form

def _values(operand):
    """(codes, atoms) -> fp32 [rows, K]."""
    codes, atoms = operand
    rows, k = codes.shape[0], 2 * codes.shape[1]
    rb, kc = -(-rows // 128), -(-k // 128)
    e = atoms.view(rb, kc, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rb * 128, kc * 4)[:rows, : k // 32]
    scale = _power(e)
    table = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), device=codes.device)
    q = table[torch.stack((codes & 15, codes >> 4), dim=-1).to(torch.int32)].view(rows, k // 32, 32)
    return (q * scale[..., None]).view(rows, k)


def _act(g, act):
    if act == "silu":
        return g / (1 + torch.exp(-g))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))


def _slope(g, act):
    if act == "silu":
        p = 1 / (1 + torch.exp(-g))
        return p * (1 + g * (1 - p))
    t = torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g))
    return 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)


def _round_trip(x):
    """fp32 [M, K], K % 32 == 0 -> the values that its MXFP4 form stands for."""
    e, code = _scale_and_codes(x)
    table = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), device=x.device)
    q = table[code.to(torch.int32)].view(x.shape[0], -1, 32)
    return (q * _power(e)[..., None]).view(x.shape)


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "quant":
        x = s["x"].float()
        return _round_trip(torch.nn.functional.pad(x, (0, -x.shape[1] % 32))).to(torch.bfloat16)
    if op == "gemm":
        return (_values(s["a"]) @ _values(s["b"]).T).to(_TYPES[c["out"]])
    if op == "gated":
        a = _values(s["a"])
        return (_act(a @ _values(s["g"]).T, c["act"]) * (a @ _values(s["u"]).T)).to(torch.bfloat16)
    if op == "ffn":
        a = _round_trip(s["x"].float())
        h = _act(a @ _values(s["g"]).T, c["act"]) * (a @ _values(s["u"]).T)
        return (_round_trip(h) @ _values(s["d"]).T).to(torch.bfloat16)
    t = _TYPES[c["dtype"]]
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    if op == "dense":
        g, u = x @ wg.T, x @ wu.T
        h = (_act(g, c["act"]) * u).to(t)
        return (h, g.to(t), u.to(t)) if c["keep"] else h
    g, u, dh = s["g"].float(), s["u"].float(), s["dh"].float()
    dg, du = dh * u * _slope(g, c["act"]), dh * _act(g, c["act"])
    return (dg @ wg + du @ wu).to(t), (dg.T @ x).to(t), (du.T @ x).to(t)


# ---------------------------------------------------------------- the framework's calls

def _own(s):
    import pantheon_b200 as pb
    c = s["case"]
    op = c["op"]
    if op == "quant":
        return pb.dequant_mxfp4(*pb.quant_mxfp4(s["x"]))
    if op == "gemm":
        return pb.gemm_mxfp4(*s["a"], *s["b"], out_type=pb.QG_OUT_BF16 if c["out"] == "bf16" else pb.QG_OUT_F32)
    act = pb.QG_ACT_SILU if c["act"] == "silu" else pb.QG_ACT_GELU_TANH
    if op == "gated":
        return pb.gemm_gated_mxfp4(*s["a"], *s["g"], *s["u"], act=act)
    if op == "ffn":
        h = pb.gemm_gated_mxfp4(*pb.quant_mxfp4(s["x"]), *s["g"], *s["u"], act=act, out_type=pb.QG_OUT_MXFP4)
        return pb.gemm_mxfp4(*h, *s["d"])
    if op == "dense":
        call = pb.gemm_gated_bf16 if c["dtype"] == "bf16" else pb.gemm_gated_f16
        return call(s["x"], s["wg"], s["wu"], act=act, keep=c["keep"])
    call = pb.gemm_gated_bf16_backward if c["dtype"] == "bf16" else pb.gemm_gated_f16_backward
    return call(s["dh"], s["x"], s["wg"], s["wu"], s["g"], s["u"], act=act)


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    op, m, k = case["op"], case["m"], case["k"]
    if op == "quant":
        kp = _up(k, 32)
        # the tensor read, its values written; the codes and scales between the two calls are the caller's too
        return {"bytes": m * (k * _BYTES[case["dtype"]] + kp * 2) + m * kp * (0.5 + 1 / 32), "flops": 0}
    n = case["n"]
    four = 0.5 + 1 / 32
    if op == "gemm":
        return {"bytes": (m + n) * k * four + m * n * _BYTES[case["out"]], "flops": 2 * m * n * k}
    if op == "gated":
        return {"bytes": (m + 2 * n) * k * four + 2 * m * n, "flops": 4 * m * n * k}
    if op == "ffn":
        return {"bytes": 2 * m * k + 3 * n * k * four + 2 * m * k, "flops": 6 * m * n * k}
    if op == "dense":
        return {"bytes": 2 * (m * k + 2 * n * k + (3 if case["keep"] else 1) * m * n), "flops": 4 * m * n * k}
    return {"bytes": 2 * (2 * m * k + 4 * n * k + 3 * m * n), "flops": 8 * m * n * k}


# ---------------------------------------------------------------- the definition, in 64 bits

def _two64(e):
    """2^e in 64 bits, from its bits: pow() rounds."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _decode64(operand):
    """Value (r, k) of an MXFP4 operand straight from the layout's formulas."""
    codes, atoms = operand
    rows, k = codes.shape[0], 2 * codes.shape[1]
    r = torch.arange(rows, device=codes.device)[:, None]
    j = torch.arange(k // 32, device=codes.device)[None, :]
    at = ((r // 128) * (-(-k // 128)) + j // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + j % 4
    scale = _two64(atoms[at].long() - 127)
    out = torch.empty((rows, k), dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        c = (codes >> (4 * half)) & 15
        exp, man = (c >> 1) & 3, (c & 1).double()
        mag = torch.where(exp == 0, 0.5 * man, (1 + 0.5 * man) * _two64(exp.long() - 1))
        out[:, half::2] = torch.where(c >= 8, -mag, mag)
    return (out.view(rows, -1, 32) * scale[..., None]).view(rows, k)


def _grid64(x):
    """The nearest MXFP4 values of [M, K] (K % 32 == 0), ties to even."""
    b = x.view(x.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    unit = _two64(torch.where(top == 0, -127, (torch.frexp(top).exponent - 3).clamp(min=-127)))
    a = b.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.sign(b) * (torch.round(a / step) * step).clamp(max=6.0) * unit).view(x.shape)


def _gate64(g, u, act):
    if act == "silu":
        return g * torch.sigmoid(g) * u
    return g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)) * u


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        x = s["x"].double()
        return _grid64(torch.nn.functional.pad(x, (0, -x.shape[1] % 32)))
    if op == "gemm":
        return torch.matmul(_decode64(s["a"]), _decode64(s["b"]).t())
    if op == "gated":
        a = _decode64(s["a"])
        return _gate64(torch.matmul(a, _decode64(s["g"]).t()), torch.matmul(a, _decode64(s["u"]).t()), case["act"])
    if op == "ffn":
        a = _grid64(s["x"].double())
        h = _gate64(torch.matmul(a, _decode64(s["g"]).t()), torch.matmul(a, _decode64(s["u"]).t()), case["act"])
        return torch.matmul(_grid64(h), _decode64(s["d"]).t())
    x, wg, wu = s["x"].double(), s["wg"].double(), s["wu"].double()
    if op == "dense":
        g, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
        h = _gate64(g, u, case["act"])
        return (h, g, u) if case["keep"] else h
    g, u, dh = s["g"].double(), s["u"].double(), s["dh"].double()
    if case["act"] == "silu":
        p = torch.sigmoid(g)
        slope = p + g * p * (1 - p)
    else:
        r = 2 * math.sqrt(2 / math.pi)                      # 0.5 (1 + tanh(z)) = sigmoid(2 z)
        p = torch.sigmoid(r * (g + 0.044715 * g ** 3))
        slope = p + g * p * (1 - p) * r * (1 + 3 * 0.044715 * g ** 2)
    dg, du = dh * u * slope, dh * g * p
    return torch.matmul(dg, wg) + torch.matmul(du, wu), torch.matmul(dg.t(), x), torch.matmul(du.t(), x)
