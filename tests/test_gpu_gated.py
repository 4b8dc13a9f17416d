"""The gated projections in bf16 and fp16, and their backward pass, against a plain 64-bit statement.

Tolerances: fp32 sums and the activation as in mxfp4_reference; half a step of the type for each
rounding (2^-8 of a bf16 value, 2^-11 of an fp16 value, at least half of its smallest step).  The
backward pass rounds dG and dU once before the products, so their half step enters them by the
operand's magnitude.
"""
import numpy as np
import pytest
import torch

import pantheon_b200 as pb
from tests import mxfp4_reference as R

pytestmark = pytest.mark.gpu

ACTS = [pb.QG_ACT_SILU, pb.QG_ACT_GELU_TANH]
TYPES = {"bf16": (torch.bfloat16, 2.0 ** -8, 2.0 ** -134, pb.gemm_gated_bf16, pb.gemm_gated_bf16_backward),
         "f16": (torch.float16, 2.0 ** -11, 2.0 ** -25, pb.gemm_gated_f16, pb.gemm_gated_f16_backward)}
SHAPES = [(1, 8, 8), (1, 64, 200), (2, 136, 64), (17, 128, 72), (127, 264, 136), (128, 256, 64), (257, 392, 264),
          (300, 1000, 520), (520, 128, 1032)]


def _np(t):
    return t.detach().cpu().double().numpy()


def _half_step(v, kind):
    _, rel, least, _, _ = TYPES[kind]
    return np.maximum(rel * np.abs(v), least)


def _inputs(shape, kind, dev, seed=0):
    M, N, K = shape
    g = torch.Generator().manual_seed(seed + M + 3 * N + 7 * K)
    t = TYPES[kind][0]
    x = torch.randn((M, K), generator=g).to(t)
    wg, wu = (torch.randn((N, K), generator=g).mul_(2 / K ** 0.5).to(t) for _ in range(2))
    return x.to(dev), wg.to(dev), wu.to(dev)


def _check_forward(x, wg, wu, act, kind, h, g=None, u=None):
    x, wg, wu = _np(x), _np(wg), _np(wu)
    gate, up = x @ wg.T, x @ wu.T
    eg, eu = R.sum_bound(x, wg), R.sum_bound(x, wu)
    ref = R.activation(gate, act) * up
    e = R.gated_bound(gate, up, eg, eu, act)
    assert (np.abs(_np(h) - ref) <= e + _half_step(np.abs(ref) + e, kind)).all()
    if g is not None:
        assert (np.abs(_np(g) - gate) <= eg + _half_step(np.abs(gate) + eg, kind)).all()
        assert (np.abs(_np(u) - up) <= eu + _half_step(np.abs(up) + eu, kind)).all()


def _check_backward(dh, x, wg, wu, g, u, act, kind, got):
    dh, x, wg, wu, g, u = (_np(t) for t in (dh, x, wg, wu, g, u))
    dg, du = dh * u * R.slope(g, act), dh * R.activation(g, act)
    y = np.abs(R.act_arg(g, act))
    dy = 1.0 if act == 0 else 1.6 + 0.2141 * np.minimum(g * g, 900)
    # p, p (1 - p), their products: units by |y| as in the forward pass; 1 - p is off by one unit of 1
    units = (20 + 10 * y) * 2.0 ** -23
    edg = np.abs(dh * u) * units * (1 + np.abs(g) * dy) + _half_step(dg, kind) * (1 + 2.0 ** -8)
    edu = np.abs(du) * units + 2e-38 * np.abs(dh * g) + _half_step(du, kind) * (1 + 2.0 ** -8)
    refs = (dg @ wg + du @ wu, dg.T @ x, du.T @ x)
    es = (edg @ np.abs(wg) + edu @ np.abs(wu) + 2 * R.sum_bound(np.abs(dg) + edg, wg.T) + 2 * R.sum_bound(np.abs(du) + edu, wu.T),
          edg.T @ np.abs(x) + R.sum_bound(np.abs(dg).T + edg.T, x.T), edu.T @ np.abs(x) + R.sum_bound(np.abs(du).T + edu.T, x.T))
    for have, ref, e in zip(got, refs, es):
        if have is not None:
            assert (np.abs(_np(have) - ref) <= e + _half_step(np.abs(ref) + e, kind)).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_matches_the_definition(cuda_device, shape, act, kind):
    x, wg, wu = _inputs(shape, kind, cuda_device)
    f = TYPES[kind][3]
    h = f(x, wg, wu, act=act)
    kept = f(x, wg, wu, act=act, keep=True)
    assert torch.equal(h, kept[0])
    _check_forward(x, wg, wu, act, kind, *kept)
    assert pb.device_status(0) == 0


# the kernel for few rows: each of its tiles, whole and with K in two to eight parts, one row tile and
# several; and two pairs of CTAs to a tile, whose shapes lie beside those
FEW = [(1, 8, 4104), (1, 9608, 264), (16, 1000, 520), (17, 136, 1032), (32, 72, 2056), (33, 72, 520), (64, 5000, 264),
       (65, 264, 1032), (129, 136, 4104), (300, 1000, 2056), (300, 1608, 2120), (513, 1032, 2056)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", FEW, ids=lambda s: "x".join(map(str, s)))
def test_forward_of_few_rows(cuda_device, shape, kind):
    x, wg, wu = _inputs(shape, kind, cuda_device)
    act = ACTS[shape[0] % 2]
    f = TYPES[kind][3]
    h, g, u = f(x, wg, wu, act=act, keep=True)
    _check_forward(x, wg, wu, act, kind, h, g, u)
    assert torch.equal(f(x, wg, wu, act=act), h)
    assert pb.device_status(0) == 0


# the same for dX, in one and two terms of dG and dU, with N inside a block of 64 and K inside a tile
FEW_DX = [(1, 8, 8), (1, 4104, 136), (7, 9608, 264), (16, 520, 1000), (20, 1032, 136), (40, 3000, 72), (64, 264, 9608),
          (65, 1032, 264), (100, 2056, 1000), (129, 4104, 136), (130, 264, 72), (1300, 520, 264), (2050, 520, 520),
          (32, 4104, 72), (40, 1032, 136), (66, 520, 136), (300, 4104, 264),
          (200, 1288, 3104), (100, 600, 5000), (270, 800, 1800)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", FEW_DX, ids=lambda s: "x".join(map(str, s)))
def test_backward_of_few_rows(cuda_device, shape, kind):
    x, wg, wu = _inputs(shape, kind, cuda_device)
    forward, backward = TYPES[kind][3:]
    act = ACTS[shape[0] % 2]
    _, g, u = forward(x, wg, wu, act=act, keep=True)
    dh = torch.randn(g.shape, device=cuda_device, generator=torch.Generator(cuda_device).manual_seed(6)).to(g.dtype)
    got = backward(dh, x, wg, wu, g, u, act=act)
    _check_backward(dh, x, wg, wu, g, u, act, kind, got)
    assert torch.equal(backward(dh, x, wg, wu, g, u, act=act, need_dw=False)[0], got[0])
    assert all(torch.equal(a, b) for a, b in zip(backward(dh, x, wg, wu, g, u, act=act, need_dx=False)[1:], got[1:]))
    assert pb.device_status(0) == 0


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_backward_matches_the_formula(cuda_device, shape, act, kind):
    x, wg, wu = _inputs(shape, kind, cuda_device)
    forward, backward = TYPES[kind][3:]
    _, g, u = forward(x, wg, wu, act=act, keep=True)
    dh = torch.randn(g.shape, device=cuda_device, generator=torch.Generator(cuda_device).manual_seed(5)).to(g.dtype)
    got = backward(dh, x, wg, wu, g, u, act=act)
    _check_backward(dh, x, wg, wu, g, u, act, kind, got)
    only_x = backward(dh, x, wg, wu, g, u, act=act, need_dw=False)
    only_w = backward(dh, x, wg, wu, g, u, act=act, need_dx=False)
    assert torch.equal(only_x[0], got[0]) and only_x[1] is None and only_x[2] is None
    assert only_w[0] is None and torch.equal(only_w[1], got[1]) and torch.equal(only_w[2], got[2])
    assert pb.device_status(0) == 0


# several tiles per CTA pair (forward 96 tiles; backward 165 tiles of two lengths), dX split alone
# beside whole dWg and dWu, gradients in two terms and in one, all three split with tiles
# of dWg and dWu the longer ones, dX split in two or four with whole dWg and dWu in one launch, and
# dWg and dWu split beside a whole dX or before it
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", [(700, 4000, 136), (1100, 1032, 2600), (100, 5000, 256), (256, 512, 776),
                                   (257, 512, 776), (2000, 64, 256), (1500, 136, 72), (515, 1368, 520),
                                   (200, 1368, 520), (4096, 512, 264), (2600, 1032, 776), (20000, 256, 512),
                                   (100, 12000, 512)],
                         ids=lambda s: "x".join(map(str, s)))
def test_larger_shapes(cuda_device, shape, kind):
    x, wg, wu = _inputs(shape, kind, cuda_device)
    forward, backward = TYPES[kind][3:]
    act = ACTS[shape[0] % 2]
    h, g, u = forward(x, wg, wu, act=act, keep=True)
    _check_forward(x, wg, wu, act, kind, h, g, u)
    dh = torch.randn(g.shape, device=cuda_device, generator=torch.Generator(cuda_device).manual_seed(6)).to(g.dtype)
    got = backward(dh, x, wg, wu, g, u, act=act)
    _check_backward(dh, x, wg, wu, g, u, act, kind, got)
    assert torch.equal(backward(dh, x, wg, wu, g, u, act=act, need_dw=False)[0], got[0])
    assert torch.equal(backward(dh, x, wg, wu, g, u, act=act, need_dx=False)[2], got[2])
    assert pb.device_status(0) == 0


@pytest.mark.parametrize("kind", list(TYPES))
def test_few_values_carry_no_intermediate_rounding(cuda_device, kind):
    """Up to 65536 values dG and dU go as value and remainder: what is left of their rounding is a
    half step of the remainder, so the results are within their own rounding and the fp32 bounds."""
    M, N, K = 48, 264, 136
    x, wg, wu = _inputs((M, N, K), kind, cuda_device)
    forward, backward, step = TYPES[kind][3], TYPES[kind][4], TYPES[kind][1]
    _, g, u = forward(x, wg, wu, keep=True)
    dh = torch.randn(g.shape, device=cuda_device, generator=torch.Generator(cuda_device).manual_seed(7)).to(g.dtype)
    dx, dwg, dwu = (_np(t) for t in backward(dh, x, wg, wu, g, u))
    dh, x, wg, wu, g, u = (_np(t) for t in (dh, x, wg, wu, g, u))
    dg, du = dh * u * R.slope(g, 0), dh * R.activation(g, 0)
    # fp32 gradients: 40 units with |g| of a few (checked below); remainder: step^2, or fp16's least half step
    assert np.abs(g).max() < 16
    rel, least = 200 * 2.0 ** -23 + step * step, TYPES[kind][2]
    edg, edu = rel * (np.abs(dh * u) + np.abs(dg)) + least, rel * (np.abs(dh) * (1 + np.abs(g)) + np.abs(du)) + least
    for have, ref, e in ((dx, dg @ wg + du @ wu, edg @ np.abs(wg) + edu @ np.abs(wu) + 4 * R.sum_bound(np.abs(dg), wg.T) + 4 * R.sum_bound(np.abs(du), wu.T)),
                         (dwg, dg.T @ x, edg.T @ np.abs(x) + 2 * R.sum_bound(dg.T, x.T)),
                         (dwu, du.T @ x, edu.T @ np.abs(x) + 2 * R.sum_bound(du.T, x.T))):
        assert (np.abs(have - ref) <= e + _half_step(np.abs(ref) + e, kind)).all()


@pytest.mark.parametrize("act", ACTS)
def test_backward_against_differences(cuda_device, act):
    """Central differences of the 64-bit forward pass.  X and the weights are small multiples of 1/2,
    so G and U are exact in bf16 and the two sides differentiate at the same point."""
    M, N, K = 5, 16, 16
    rng = np.random.default_rng(3)
    x = rng.integers(-1, 2, (M, K)).astype(float)
    wg, wu = (rng.integers(-2, 3, (N, K)) / 2.0 for _ in range(2))
    dh = rng.integers(-4, 5, (M, N)) / 4.0
    d = lambda a: torch.from_numpy(a).to(torch.bfloat16).to(cuda_device)
    _, g, u = pb.gemm_gated_bf16(d(x), d(wg), d(wu), act=act, keep=True)
    np.testing.assert_array_equal(_np(g), x @ wg.T)
    got = pb.gemm_gated_bf16_backward(d(dh), d(x), d(wg), d(wu), g, u, act=act)

    def loss():
        return (dh * R.activation(x @ wg.T, act) * (x @ wu.T)).sum()

    step = 1e-5
    dg, du = np.abs(dh * (x @ wu.T) * R.slope(x @ wg.T, act)), np.abs(dh * R.activation(x @ wg.T, act))
    # half a step of dG and dU through the products, then of the result; the fp32 part and the
    # differences' own error (step^2 and 1e-16 / step of a loss of a few hundred) stay below 1e-5
    terms = (dg @ np.abs(wg) + du @ np.abs(wu), dg.T @ np.abs(x), du.T @ np.abs(x))
    for have, var, term in zip(got, (x, wg, wu), terms):
        have = _np(have)
        for i in np.ndindex(var.shape):
            keep = var[i]
            var[i] = keep + step
            hi = loss()
            var[i] = keep - step
            lo = loss()
            var[i] = keep
            assert abs(have[i] - (hi - lo) / (2 * step)) <= 2.0 ** -8 * (1.01 * term[i] + abs(have[i])) + 1e-5


@pytest.mark.parametrize("kind", list(TYPES))
def test_large_arguments(cuda_device, kind):
    """Far from zero the activations are 0 and g, their slopes 0 and 1: no NaN from 0 * infinity."""
    t, _, _, forward, backward = TYPES[kind]
    big = 3e4 if kind == "f16" else 1e30
    vals = torch.tensor([0.0, -0.0, 20.0, -20.0, 90.0, -90.0, 1e4, -1e4, big, -big], dtype=torch.float64)
    x = torch.zeros((len(vals), 8), dtype=t, device=cuda_device)
    x[:, 0], x[:, 1] = vals.to(t).to(cuda_device), 1.0
    wg, wu = (torch.zeros((8, 8), dtype=t, device=cuda_device) for _ in range(2))
    wg[:, 0], wu[:, 1] = 1.0, 1.0
    for act in ACTS:
        h, g, u = forward(x, wg, wu, act=act, keep=True)
        gate = _np(x[:, :1]).repeat(8, 1)
        with np.errstate(over="ignore"):
            ref, slope = R.activation(gate, act), R.slope(np.clip(gate, -100, 100), act)
        tol = _half_step(ref, kind) * 1.01 + 2e-38 * (1 + np.abs(gate)) + 40 * 2.0 ** -23 * np.abs(ref) * (1 + np.minimum(np.abs(gate), 100))
        assert np.isfinite(_np(h)).all() and (np.abs(_np(h) - ref) <= tol).all()
        dh = torch.ones_like(h)
        dx, dwg, dwu = backward(dh, x, wg, wu, g, u, act=act)
        for v in (dx, dwg, dwu):
            assert not v.isnan().any()       # act(big) * big in dWu passes both types' range: infinity is its value
        # column 0 of dX sums the 8 equal gate gradients: 8 * slope
        assert (np.abs(_np(dx)[:, 0] - 8 * slope[:, 0]) <= 8 * 2 * 1.01 * (TYPES[kind][1] * np.abs(slope[:, 0]) + 1e-5)).all()


def test_offsets_past_32_bits(cuda_device):
    """2.8e9 values of G, U and dH: the last rows of H and dX, and dWg and dWu whose sums have few rows of
    values other than zero, the last ones."""
    M, N, K = 70000, 40000, 64
    g = torch.Generator().manual_seed(11)
    x = torch.zeros((M, K), dtype=torch.bfloat16, device=cuda_device)
    x[-40:] = torch.randn((40, K), generator=g).to(torch.bfloat16).to(cuda_device)
    wg, wu = ((torch.randn((N, K), generator=g) / 4).to(torch.bfloat16).to(cuda_device) for _ in range(2))
    h, gate, up = pb.gemm_gated_bf16(x, wg, wu, keep=True)
    _check_forward(x[-40:], wg, wu, 0, "bf16", h[-40:], gate[-40:], up[-40:])
    assert (h[:-40] == 0).all()
    dh = torch.zeros_like(h)
    dh[-40:] = torch.randn((40, N), generator=g).to(torch.bfloat16).to(cuda_device)
    dx, dwg, dwu = pb.gemm_gated_bf16_backward(dh, x, wg, wu, gate, up)
    assert (dx[:-40] == 0).all()
    _check_backward(dh[-40:], x[-40:], wg, wu, gate[-40:], up[-40:], 0, "bf16", (dx[-40:], dwg, dwu))


@pytest.mark.parametrize("shape", [(260, 264, 136), (20, 1032, 136)], ids=lambda s: "x".join(map(str, s)))
def test_captured_and_replayed_beside_an_eager_call(cuda_device, shape):
    x, wg, wu = _inputs(shape, "bf16", cuda_device)
    _, g, u = pb.gemm_gated_bf16(x, wg, wu, keep=True)
    dh = torch.randn_like(g)
    ws = torch.empty((pb.gemm_gated_backward_workspace_bytes(*shape[:2]),), dtype=torch.uint8, device=cuda_device)

    def step():
        h, g, u = pb.gemm_gated_bf16(x, wg, wu, keep=True)
        return (h, *pb.gemm_gated_bf16_backward(dh, x, wg, wu, g, u, workspace=ws))

    eager = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, eager))
    x.mul_(-0.5)
    dh.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    again = step()
    assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_a_training_step_and_its_decode(cuda_device):
    """One step of a block with a dense down projection moves the loss the way its gradient says, and
    the trained weights run in MXFP4 on one token."""
    M, N, K = 264, 512, 256
    x, wg, wu = _inputs((M, N, K), "bf16", cuda_device)
    h, g, u = pb.gemm_gated_bf16(x, wg, wu, keep=True)
    dh = (h.float() / h.numel()).to(torch.bfloat16)           # gradient of sum(h^2) / (2 n)
    dx, dwg, dwu = pb.gemm_gated_bf16_backward(dh, x, wg, wu, g, u)
    assert dx.shape == x.shape and dwg.shape == wg.shape and dwu.shape == wu.shape
    _check_backward(dh, x, wg, wu, g, u, pb.QG_ACT_SILU, "bf16", (dx, dwg, dwu))
    q = [pb.quant_mxfp4(t) for t in (x[:1], wg, wu)]
    one = pb.gemm_gated_mxfp4(*q[0], *q[1], *q[2])
    val = [_np(pb.dequant_mxfp4(*t, pb.QG_OUT_F32)) for t in q]
    gate, up = val[0] @ val[1].T, val[0] @ val[2].T
    e = R.gated_bound(gate, up, R.sum_bound(val[0], val[1]), R.sum_bound(val[0], val[2]), 0)
    ref = R.activation(gate, 0) * up
    assert (np.abs(_np(one) - ref) <= e + 2.0 ** -8 * (np.abs(ref) + e)).all()


def test_python_refusals(cuda_device):
    x, wg, wu = _inputs((16, 32, 24), "bf16", cuda_device)
    h, g, u = pb.gemm_gated_bf16(x, wg, wu, keep=True)
    with pytest.raises(ValueError):
        pb.gemm_gated_bf16(x, wg, wu[:-8])
    with pytest.raises(ValueError):
        pb.gemm_gated_bf16(x.half(), wg, wu)
    with pytest.raises(ValueError):
        pb.gemm_gated_f16(x, wg, wu)
    with pytest.raises(ValueError):
        pb.gemm_gated_bf16(x[:, :16], wg, wu)
    with pytest.raises(ValueError):
        pb.gemm_gated_bf16(x.t().contiguous().t(), wg, wu)
    with pytest.raises(ValueError):
        pb.gemm_gated_bf16(x, wg, wu.cpu())
    with pytest.raises(pb.QGError):
        pb.gemm_gated_bf16(x, wg, wu, act=7)
    with pytest.raises(pb.QGError):
        pb.gemm_gated_bf16(x[:, :20].contiguous(), wg[:, :20].contiguous(), wu[:, :20].contiguous())   # K = 20
    with pytest.raises(ValueError):
        pb.gemm_gated_bf16_backward(h, x, wg, wu, g, u[:8])
    with pytest.raises(ValueError):
        pb.gemm_gated_bf16_backward(h.float(), x, wg, wu, g, u)
    with pytest.raises(pb.QGError):
        pb.gemm_gated_bf16_backward(h, x, wg, wu, g, u, workspace=torch.empty((64,), dtype=torch.uint8, device=cuda_device))
    with pytest.raises(pb.QGError):
        pb.gemm_gated_bf16_backward(h, x, wg, wu, g, u, need_dx=False, need_dw=False)
