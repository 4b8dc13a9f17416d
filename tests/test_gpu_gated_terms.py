"""The gated backward pass with dG and dU in two terms (M N <= 65536) and in one, in every kernel form.

Every column of the weights and of X holds one value other than zero, so that each result is one element
of dG or dU times a number of two or three bits: a sum's bound hides nothing, and a result without its
remainder is off by more than its own rounding somewhere.

Bounds, u = 2^-23, p = 1 / (1 + exp(-y)): slopes and activations as test_gpu_gated_slope derives them;
two products for dG and one for dU; the remainder's half step, which is step^2 of the value (or dG's own
half step where there is no second term); two additions in the product; the result's half step.
"""
import numpy as np
import pytest
import torch

import pantheon_b200 as pb
from tests import mxfp4_reference as R
from tests import test_gpu_gated as T

ACTS = {"silu": pb.QG_ACT_SILU, "gelu": pb.QG_ACT_GELU_TANH}
UNIT = 2.0 ** -23


def _gradients(dh, g, u, act, kind, terms):
    """dG, dU in 64 bits, and how far what enters the products may be from them."""
    _, step, least, _, _ = T.TYPES[kind]
    y = R.act_arg(g, act)
    p, q = 1 / (1 + np.exp(-y)), 1 / (1 + np.exp(y))
    dy = 1.0 if act == 0 else 1.6 + 0.2141 * g * g
    E = (12 + 6 * np.abs(y)) * UNIT
    slope, a = R.slope(g, act), R.activation(g, act)
    es = E * p + np.abs(g) * p * dy * (2 * q * E + 8 * UNIT) + 2e-38 * (1 + np.abs(g) * dy)
    ea = np.abs(g) * p * (E + UNIT) + 2e-38 * np.abs(g)
    dg, du = dh * u * slope, dh * a
    left = step * step if terms == 2 else step
    out = []
    for d, e in ((dg, np.abs(dh * u) * es + 3 * UNIT * np.abs(dg)), (du, np.abs(dh) * ea + 2 * UNIT * np.abs(du))):
        out += [d, e + np.maximum(left * (np.abs(d) + e), least) * (1 + 2 * step)]
    return out


def _within(have, ref, e, kind):
    return np.abs(have - ref) <= e + T._half_step(np.abs(ref) + e, kind)


def _bounds(dg, edg, du, edu, x, wg, wu):
    """The three gradients and their bounds, of operands with one term to a sum."""
    one = lambda d, e, b: (d @ b, e @ np.abs(b) + 4 * UNIT * (np.abs(d) @ np.abs(b)))
    a, b = one(dg, edg, wg), one(du, edu, wu)
    return (a[0] + b[0], a[1] + b[1]), one(dg.T, edg.T, x), one(du.T, edu.T, x)


def _one_hot(rows, cols, rng, keep):
    """[rows, cols] with one value in the columns where `keep`, at a random row."""
    m = np.zeros((rows, cols))
    at = np.arange(cols)[keep]
    m[rng.integers(0, rows, at.size), at] = rng.choice([0.75, 1.25, 1.5, 1.75, 3.5], at.size) * rng.choice([-1, 1], at.size)
    return m


def _case(shape, kind, seed):
    M, N, K = shape
    rng = np.random.default_rng(seed + M + 3 * N + 7 * K)
    x = _one_hot(M, K, rng, np.ones(K, dtype=bool))
    half = rng.random(K) < 0.5
    wg, wu = _one_hot(N, K, rng, half), _one_hot(N, K, rng, ~half)
    t = lambda a: torch.from_numpy(a).to(T.TYPES[kind][0])
    dense = [t(rng.standard_normal((M, N)) * s) for s in (1.0, 2.0, 1.0)]      # dH, G, U
    return [dense[0], t(x), t(wg), t(wu), dense[1], dense[2]]


# (M, N, K): what computes dX and dW.  dX by the kernel for few rows in tiles of 16, 32, 64, 128; pairs,
# whole; all tiles split with dX's contraction the longer, and with dW's; dX split beside whole dW; dW
# split beside whole dX, and in a launch before it; whole tiles, several to a pair; the last M N with two
# terms, and the first with one
SHAPES = [(10, 264, 136), (20, 1032, 136), (48, 264, 136), (100, 600, 5000), (130, 264, 72), (104, 600, 256),
          (1300, 48, 256), (101, 640, 1536), (1350, 48, 1280), (1350, 48, 2296), (250, 256, 8000), (128, 512, 200),
          (129, 512, 200), (1, 65536, 72), (1, 65544, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(T.TYPES))
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_each_element_of_the_gradients(cuda_device, shape, act, kind):
    M, N, _ = shape
    case = _case(shape, kind, 1)
    got = T.TYPES[kind][4](*(t.to(cuda_device) for t in case), act=ACTS[act])
    dh, x, wg, wu, g, u = (t.double().numpy() for t in case)
    terms = _gradients(dh, g, u, ACTS[act], kind, 2 if M * N <= 65536 else 1)
    for have, (ref, e) in zip(got, _bounds(*terms, x, wg, wu)):
        assert _within(T._np(have), ref, e, kind).all()
    assert pb.device_status(0) == 0


# all tiles split in two terms, and beside them the same in one: sums of many terms
@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(T.TYPES))
@pytest.mark.parametrize("shape", [(104, 600, 256), (1300, 48, 256), (101, 640, 1536), (1350, 48, 1280), (1350, 48, 2296),
                                   (250, 256, 8000), (128, 512, 200), (129, 512, 200), (120, 600, 256)],
                         ids=lambda s: "x".join(map(str, s)))
def test_sums_of_the_split_forms(cuda_device, shape, kind):
    x, wg, wu = T._inputs(shape, kind, cuda_device)
    forward, backward = T.TYPES[kind][3:]
    act = shape[0] % 2
    _, g, u = forward(x, wg, wu, act=act, keep=True)
    dh = torch.randn(g.shape, device=cuda_device, generator=torch.Generator(cuda_device).manual_seed(8)).to(g.dtype)
    got = backward(dh, x, wg, wu, g, u, act=act)
    T._check_backward(dh, x, wg, wu, g, u, act, kind, got)
    assert torch.equal(backward(dh, x, wg, wu, g, u, act=act, need_dw=False)[0], got[0])
    assert all(torch.equal(a, b) for a, b in zip(backward(dh, x, wg, wu, g, u, act=act, need_dx=False)[1:], got[1:]))
    assert all(torch.equal(a, b) for a, b in zip(backward(dh, x, wg, wu, g, u, act=act), got))
    assert pb.device_status(0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", list(ACTS))
def test_differences_without_an_intermediate_rounding(cuda_device, act):
    """Central differences in 64 bits where dG and dU go in two terms: of the gradient's own rounding
    half a step, and of theirs half a step of what half a step leaves."""
    M, N, K = 5, 16, 16
    rng = np.random.default_rng(4)
    x = rng.integers(-1, 2, (M, K)).astype(float)
    wg, wu = (rng.integers(-2, 3, (N, K)) / 2.0 for _ in range(2))
    dh = rng.integers(-4, 5, (M, N)) / 4.0
    d = lambda a: torch.from_numpy(a).to(torch.bfloat16).to(cuda_device)
    _, g, u = pb.gemm_gated_bf16(d(x), d(wg), d(wu), act=ACTS[act], keep=True)
    np.testing.assert_array_equal(T._np(g), x @ wg.T)
    got = pb.gemm_gated_bf16_backward(d(dh), d(x), d(wg), d(wu), g, u, act=ACTS[act])
    # sums of up to 32 terms of up to 30 in magnitude, twice: 64 * 2^-23 of their sum; the activation's
    # units (E of up to 400 units where g is 16 and p is 1 to 4 units); 1e-5 for the differences, as
    # 64-bit losses of a few hundred over 2e-5
    gate, up = x @ wg.T, x @ wu.T
    dg, edg, du, edu = _gradients(dh, gate, up, ACTS[act], "bf16", 2)
    mags = (np.abs(dg) @ np.abs(wg) + np.abs(du) @ np.abs(wu), np.abs(dg).T @ np.abs(x), np.abs(du).T @ np.abs(x))
    errs = (edg @ np.abs(wg) + edu @ np.abs(wu), edg.T @ np.abs(x), edu.T @ np.abs(x))
    step = 1e-5
    for have, var, mag, err in zip(got, (x, wg, wu), mags, errs):
        have = T._np(have)
        for i in np.ndindex(var.shape):
            keep = var[i]
            side = []
            for s in (step, -step):
                var[i] = keep + s
                side.append((dh * R.activation(x @ wg.T, ACTS[act]) * (x @ wu.T)).sum())
            var[i] = keep
            e = err[i] + 64 * UNIT * mag[i] + 1e-5
            diff = (side[0] - side[1]) / (2 * step)
            assert abs(have[i] - diff) <= e + 2.0 ** -8 * (abs(diff) + e)


@pytest.mark.parametrize("kind", list(T.TYPES))
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[0] * s[1] <= 65536], ids=lambda s: "x".join(map(str, s)))
def test_the_bounds_show_a_missing_remainder(shape, act, kind):
    """The oracle with dG (dU) rounded once is outside the two-term bounds of every gradient; with value
    and remainder it is inside."""
    dh, x, wg, wu, g, u = _case(shape, kind, 1)
    t = T.TYPES[kind][0]
    n = lambda v: v.double().numpy()
    terms = _gradients(n(dh), n(g), n(u), ACTS[act], kind, 2)
    bounds = _bounds(*terms, n(x), n(wg), n(wu))
    round_t = lambda a: n(torch.from_numpy(a).to(t))
    dg, du = terms[0], terms[2]
    for whole in (True, False):
        a, b = (round_t(v) + round_t(v - round_t(v)) if whole else round_t(v) for v in (dg, du))
        got = (a @ n(wg) + b @ n(wu), a.T @ n(x), b.T @ n(x))
        for have, (ref, e) in zip(got, bounds):
            assert _within(round_t(have), ref, e, kind).all() == whole
