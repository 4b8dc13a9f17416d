"""MXFP4 quantisation, product and gated product on the GPU against a plain 64-bit statement.

Quantisation is exact arithmetic but for its last rounding, so codes and scale bytes have to be
equal.  Products: mxfp4_reference's bounds, plus half a step of the output type (bf16: 2^-8 of the
value).
"""
import numpy as np
import pytest
import torch

import pantheon_b200 as pb
from tests import mxfp4_reference as R

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ACTS = [pb.QG_ACT_SILU, pb.QG_ACT_GELU_TANH]


def _np(t):
    return t.detach().cpu().double().numpy() if t.is_floating_point() else t.detach().cpu().numpy()


def _values(rows, cols, seed, dtype):
    """Normal values over many magnitudes, with zeros, negative zeros, ties and saturating values."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-6, 7, (rows, 1)).astype(float))
    x[rng.random(x.shape) < 0.05] = 0.0
    x[rng.random(x.shape) < 0.02] = -0.0
    ties = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9], x.shape) * rng.choice([-1, 1], x.shape)
    x = np.where(rng.random(x.shape) < 0.2, ties, x)
    return torch.from_numpy(x).to(dtype)


def _operand(rows, K, seed, dev):
    """A random MXFP4 tensor straight from codes and scale bytes: (device pair, values)."""
    rng = np.random.default_rng(seed)
    q, sf = R.pack(rng.integers(0, 16, (rows, K)).astype(np.uint8), rng.integers(121, 130, (rows, K // 32)).astype(np.uint8))
    return (torch.from_numpy(q).to(dev), torch.from_numpy(sf).to(dev)), R.decode(q, sf)


def _check_quant(x, q, sf):
    rq, rsf = R.pack(*R.quantise(_np(x)))
    np.testing.assert_array_equal(_np(q), rq)
    np.testing.assert_array_equal(_np(sf), rsf)   # the padding of the atoms too


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (4, 8192), (33, 129), (128, 256), (129, 513), (300, 1000)],
                         ids=lambda s: "x".join(map(str, s)))
def test_quant_matches_the_definition(cuda_device, shape, dtype):
    x = _values(*shape, seed=sum(shape), dtype=TYPES[dtype]).to(cuda_device)
    q, sf = pb.quant_mxfp4(x)
    assert q.shape == (shape[0], R.up(shape[1], 32) // 2)
    _check_quant(x, q, sf)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("offset, pad", [(0, 24), (1, 7), (3, 5), (8, 8), (2, 6), (4, 4)])
def test_quant_of_a_slice(cuda_device, dtype, offset, pad):
    """Columns of a wider tensor, rows on and off 16-byte boundaries."""
    base = _values(70, offset + 333 + pad, seed=offset, dtype=TYPES[dtype]).to(cuda_device)
    x = base[:, offset:offset + 333]
    _check_quant(x, *pb.quant_mxfp4(x))


def test_quant_extremes(cuda_device):
    """Subnormals, the largest values, and blocks with NaN or infinity (all NaN afterwards)."""
    x = torch.zeros((8, 96))
    x[0, 0] = 1e-45
    x[1, :] = 2.0 ** -127
    x[1, 5] = 2.0 ** -125
    x[2, 7] = torch.finfo(torch.float32).max
    x[2, 8] = -1.0
    x[3, 40] = float("nan")
    x[3, 0] = 3.0
    x[4, 33] = float("inf")
    x[5, 95] = float("-inf")
    x[6, :] = -0.0
    x[7, :] = torch.linspace(-7.99, 7.99, 96)
    q, sf = pb.quant_mxfp4(x.to(cuda_device))
    _check_quant(x, q, sf)
    for out_type, t in ((pb.QG_OUT_BF16, torch.bfloat16), (pb.QG_OUT_F32, torch.float32)):
        y = pb.dequant_mxfp4(q, sf, out_type)
        assert y.dtype == t
        np.testing.assert_array_equal(_np(y), R.decode(_np(q), _np(sf)))


def test_dequant_of_every_code_and_scale(cuda_device):
    code = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    q, sf = R.pack(code, np.arange(256, dtype=np.uint8)[:, None])
    d = [torch.from_numpy(v).to(cuda_device) for v in (q, sf)]
    ref = R.decode(q, sf)
    assert np.isnan(ref[255]).all()
    with np.errstate(over="ignore"):
        ref32 = ref.astype(np.float32)          # 6 * 2^127 and 4 * 2^127 pass the largest fp32
    for out_type in (pb.QG_OUT_BF16, pb.QG_OUT_F32):
        np.testing.assert_array_equal(_np(pb.dequant_mxfp4(*d, out_type)), ref32.astype(np.float64))


SHAPES = [(1, 1, 32), (1, 17, 64), (2, 200, 96), (5, 128, 1184), (16, 272, 256), (17, 64, 8192), (33, 130, 416),
          (64, 1000, 512), (65, 257, 2048), (128, 256, 256), (130, 200, 544), (255, 511, 1056), (300, 1001, 1024)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_gemm_matches_the_definition(cuda_device, shape):
    M, N, K = shape
    a, av = _operand(M, K, M + K, cuda_device)
    b, bv = _operand(N, K, N + 3 * K, cuda_device)
    y32 = pb.gemm_mxfp4(*a, *b, out_type=pb.QG_OUT_F32)
    ybf = pb.gemm_mxfp4(*a, *b)
    assert y32.dtype == torch.float32 and ybf.dtype == torch.bfloat16
    ref, e = av @ bv.T, R.sum_bound(av, bv)
    assert (np.abs(_np(y32) - ref) <= e).all()
    assert (np.abs(_np(ybf) - ref) <= e + 2.0 ** -8 * np.abs(ref)).all()
    assert pb.device_status(0) == 0


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_gated_matches_the_definition(cuda_device, shape, act):
    M, N, K = shape
    a, av = _operand(M, K, M + K, cuda_device)
    g, gv = _operand(N, K, N + 3 * K, cuda_device)
    u, uv = _operand(N, K, N + 5 * K, cuda_device)
    gate, up = av @ gv.T, av @ uv.T
    eg, eu = R.sum_bound(av, gv), R.sum_bound(av, uv)
    with np.errstate(over="ignore"):
        ref = R.activation(gate, act) * up
        e = R.gated_bound(gate, up, eg, eu, act)
    y32 = pb.gemm_gated_mxfp4(*a, *g, *u, act=act, out_type=pb.QG_OUT_F32)
    ybf = pb.gemm_gated_mxfp4(*a, *g, *u, act=act)
    assert (np.abs(_np(y32) - ref) <= e).all()
    assert (np.abs(_np(ybf) - ref) <= e + 2.0 ** -8 * np.abs(ref)).all()
    if N % 32 == 0:
        q, sf = pb.gemm_gated_mxfp4(*a, *g, *u, act=act, out_type=pb.QG_OUT_MXFP4)
        _check_mx_result(_np(q), _np(sf), ref, e)
    assert pb.device_status(0) == 0


# each kernel and its ways: single CTAs (more than 64, gated 32, rows) with one row tile and with
# several, CTA pairs (more than 148 tiles, or K over 4096) with their last row tile in the first or
# the second CTA and with several tiles each, and the kernel for few rows with K split on many rows
WIDE = [(70, 19001, 288), (130, 10001, 544), (200, 5024, 1056), (513, 9999, 96), (1400, 4320, 800), (130, 9999, 4128),
        (300, 1001, 4128), (130, 257, 8224), (200, 5026, 1056), (520, 5004, 96), (1300, 2050, 224),
        (200, 3091, 4128)]


@pytest.mark.parametrize("out_type", [pb.QG_OUT_BF16, pb.QG_OUT_F32])
@pytest.mark.parametrize("shape", WIDE, ids=lambda s: "x".join(map(str, s)))
def test_wide_gemm_matches_the_definition(cuda_device, shape, out_type):
    M, N, K = shape
    a, av = _operand(M, K, M + K, cuda_device)
    b, bv = _operand(N, K, N + 3 * K, cuda_device)
    ref, e = av @ bv.T, R.sum_bound(av, bv)
    y = _np(pb.gemm_mxfp4(*a, *b, out_type=out_type))
    assert (np.abs(y - ref) <= e + (2.0 ** -8 * np.abs(ref) if out_type == pb.QG_OUT_BF16 else 0)).all()
    assert pb.device_status(0) == 0


@pytest.mark.parametrize("offset", [1, 2, 4])
@pytest.mark.parametrize("out_type", [pb.QG_OUT_BF16, pb.QG_OUT_F32])
@pytest.mark.parametrize("shape", [(3, 264, 128), (130, 10000, 128), (130, 10001, 128), (520, 5000, 128), (520, 5001, 128)],
                         ids=lambda s: "x".join(map(str, s)))
def test_gemm_into_a_tensor_off_16_bytes(cuda_device, shape, out_type, offset):
    """Rows at every place, the elements before and behind the result left as they were."""
    M, N, K = shape
    a, _ = _operand(M, K, M + K, cuda_device)
    b, _ = _operand(N, K, N + 3 * K, cuda_device)
    ref = pb.gemm_mxfp4(*a, *b, out_type=out_type)
    flat = torch.full((offset + M * N + 8,), -7.0, dtype=ref.dtype, device=cuda_device)
    out = flat[offset:offset + M * N].view(M, N)
    assert pb.gemm_mxfp4(*a, *b, out_type=out_type, out=out) is out
    assert torch.equal(out, ref)
    assert (flat[:offset] == -7).all() and (flat[offset + M * N:] == -7).all()


@pytest.mark.parametrize("out_type", [pb.QG_OUT_BF16, pb.QG_OUT_F32, pb.QG_OUT_MXFP4])
@pytest.mark.parametrize("shape", [(40, 9601, 288), (64, 9632, 352), (130, 5001, 544), (200, 4928, 1056), (513, 5024, 96),
                                   (1400, 2176, 416), (200, 4928, 4128), (300, 480, 4128), (200, 5026, 96), (1400, 2179, 416), (100, 96, 512),
                                   (190, 165, 2048)], ids=lambda s: "x".join(map(str, s)))
def test_wide_gated_matches_the_definition(cuda_device, shape, out_type):
    M, N, K = shape
    if out_type == pb.QG_OUT_MXFP4 and N % 32:
        N += 32 - N % 32
    act = ACTS[M % 2]
    a, av = _operand(M, K, M + K, cuda_device)
    g, gv = _operand(N, K, N + 3 * K, cuda_device)
    u, uv = _operand(N, K, N + 5 * K, cuda_device)
    gate, up = av @ gv.T, av @ uv.T
    with np.errstate(over="ignore"):
        ref = R.activation(gate, act) * up
        e = R.gated_bound(gate, up, R.sum_bound(av, gv), R.sum_bound(av, uv), act)
    y = pb.gemm_gated_mxfp4(*a, *g, *u, act=act, out_type=out_type)
    if out_type == pb.QG_OUT_MXFP4:
        _check_mx_result(_np(y[0]), _np(y[1]), ref, e)
    else:
        assert (np.abs(_np(y) - ref) <= e + (2.0 ** -8 * np.abs(ref) if out_type == pb.QG_OUT_BF16 else 0)).all()
    assert pb.device_status(0) == 0


def _check_mx_result(q, sf, ref, e):
    """The conversion of values within e of ref: scales by the block's maximum, values by half a step."""
    M, N = ref.shape
    byte = sf[R.sf_index(M, N)].astype(int)
    hi = (np.abs(ref) + e).reshape(M, -1, 32).max(-1)
    lo = (np.abs(ref) - e).clip(0).reshape(M, -1, 32).max(-1)
    floor2 = lambda v: np.where(v > 0, np.frexp(v)[1] - 1, -200)
    assert (byte <= (floor2(hi) + 125).clip(0)).all() and (byte >= (floor2(lo) + 125).clip(0)).all()
    unit = np.repeat(np.exp2(byte - 127.0), 32, axis=1)
    v = R.decode(q, sf)
    mag = np.abs(v) / unit
    # the half interval that rounds to a level: up to the next level's middle; the last takes all above
    gap = np.array([0.25, 0.25, 0.25, 0.25, 0.5, 0.5, 1.0, 2.0])
    level = np.searchsorted(R.LEVELS, mag)
    assert (R.LEVELS[level] == mag).all()
    assert (np.abs(v - ref) <= gap[level] * unit + e).all()
    pad = np.ones(sf.size, dtype=bool)
    pad[R.sf_index(M, N)] = False
    assert (sf[pad] == 0).all()


def test_nan_scale_reaches_its_row_and_column_only(cuda_device):
    """A block that held a NaN makes its row (A) or column (B) NaN, and nothing else."""
    for M in (3, 200):
        x, w = torch.randn((M, 256), device=cuda_device), torch.randn((300, 256), device=cuda_device)
        x[2, 40] = float("nan")
        w[7, 200] = float("inf")
        y = pb.gemm_mxfp4(*pb.quant_mxfp4(x), *pb.quant_mxfp4(w))
        nan = torch.zeros((M, 300), dtype=torch.bool, device=cuda_device)
        nan[2], nan[:, 7] = True, True
        assert torch.equal(y.isnan(), nan)


@pytest.mark.parametrize("M", [1, 20, 300])
def test_block_as_it_is_used(cuda_device, M):
    """Quantise, gated projections with an MXFP4 result, down projection: the chain against itself
    in 64 bits from the device's own hidden values, and captured in a graph and replayed."""
    K, N = 512, 1056
    x = torch.randn((M, K), device=cuda_device).to(torch.bfloat16)
    w = [pb.quant_mxfp4(torch.randn(s, device=cuda_device) / s[1] ** 0.5) for s in ((N, K), (N, K), (K, N))]

    def block(v):
        return pb.gemm_mxfp4(*pb.gemm_gated_mxfp4(*pb.quant_mxfp4(v), *w[0], *w[1], out_type=pb.QG_OUT_MXFP4), *w[2])

    y = block(x)
    q, sf = pb.quant_mxfp4(x)
    _check_quant(x, q, sf)
    val = lambda p: R.decode(_np(p[0]), _np(p[1]))
    gate, up = val((q, sf)) @ val(w[0]).T, val((q, sf)) @ val(w[1]).T
    e = R.gated_bound(gate, up, R.sum_bound(val((q, sf)), val(w[0])), R.sum_bound(val((q, sf)), val(w[1])), 0)
    h = pb.gemm_gated_mxfp4(q, sf, *w[0], *w[1], out_type=pb.QG_OUT_MXFP4)
    _check_mx_result(_np(h[0]), _np(h[1]), R.activation(gate, 0) * up, e)
    ref = val(h) @ val(w[2]).T
    assert (np.abs(_np(y) - ref) <= R.sum_bound(val(h), val(w[2])) + 2.0 ** -8 * np.abs(ref)).all()

    # captured, and replayed on other inputs
    static = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(static)
    for scale in (1.0, -3.0):
        static.copy_(x * scale)
        graph.replay()
        assert torch.equal(out, block(x * scale))


def test_out_off_16_byte_boundaries_and_nothing_written_past_it(cuda_device):
    for M in (2, 200):
        a, av = _operand(M, 256, 1, cuda_device)
        b, bv = _operand(264, 256, 2, cuda_device)
        buf = torch.full((M * 264 + 64,), 7.0, dtype=torch.bfloat16, device=cuda_device)
        out = buf[1:1 + M * 264].view(M, 264)
        pb.gemm_mxfp4(*a, *b, out=out)
        assert torch.equal(out, pb.gemm_mxfp4(*a, *b))
        assert buf[0] == 7.0 and (buf[1 + M * 264:] == 7.0).all()


def test_two_streams_at_once(cuda_device):
    """Calls on two streams share nothing: each gives what it gives alone."""
    for M in (4, 200):
        a, _ = _operand(M, 2048, 1, cuda_device)
        b = [_operand(1024, 2048, s, cuda_device)[0] for s in (2, 3)]
        ref = [pb.gemm_mxfp4(*a, *x) for x in b]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in b]
        got = [[], []]
        for _ in range(8):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(pb.gemm_mxfp4(*a, *b[i]))
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(y, ref[i]) for y in got[i])


def test_python_refusals(cuda_device):
    q, sf = pb.quant_mxfp4(torch.randn((4, 64), device=cuda_device))
    big = pb.quant_mxfp4(torch.randn((4, 96), device=cuda_device))
    with pytest.raises(ValueError):
        pb.gemm_mxfp4(q, sf, *big)                            # K differs
    with pytest.raises(ValueError):
        pb.gemm_mxfp4(q, sf[:-16], q, sf)                      # scales too short
    with pytest.raises(ValueError):
        pb.gemm_mxfp4(q, sf, q, sf, out_type=pb.QG_OUT_F16)
    with pytest.raises(ValueError):
        pb.gemm_mxfp4(q, sf, q, sf, out=torch.empty((4, 5), dtype=torch.bfloat16, device=cuda_device))
    with pytest.raises(ValueError):
        pb.gemm_mxfp4(q.t().contiguous().t(), sf, q, sf)       # not contiguous
    with pytest.raises(ValueError):
        pb.gemm_gated_mxfp4(q, sf, q, sf, *big)
    with pytest.raises(ValueError):
        pb.gemm_gated_mxfp4(q, sf, q, sf, q, sf, out_type=pb.QG_OUT_MXFP4)   # N = 4
    with pytest.raises(pb.QGError):
        pb.gemm_gated_mxfp4(q, sf, q, sf, q, sf, act=9)
    with pytest.raises(ValueError):
        pb.quant_mxfp4(torch.randn((4, 64), device=cuda_device).t())
    with pytest.raises(ValueError):
        pb.quant_mxfp4(torch.zeros((4, 64), dtype=torch.int32, device=cuda_device))
    with pytest.raises(ValueError):
        pb.quant_mxfp4(torch.zeros((0, 64), device=cuda_device))
    with pytest.raises(ValueError):
        pb.dequant_mxfp4(q, sf, pb.QG_OUT_F16)


def test_first_calls_of_a_process_can_be_captured(cuda_device):
    """Every operator's first call inside a stream capture, in a process of its own."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
import pantheon_b200 as pb
x = torch.randn((200, 256), device="cuda").to(torch.bfloat16)
w = torch.randn((5024, 256), device="cuda").to(torch.bfloat16) / 16
torch.cuda.synchronize()
def run():
    q, p = pb.quant_mxfp4(x), pb.quant_mxfp4(w)
    h, g, u = pb.gemm_gated_bf16(x, w, w, keep=True)
    return (pb.dequant_mxfp4(*q), pb.gemm_mxfp4(*q, *p), pb.gemm_mxfp4(*p, *q), pb.gemm_gated_mxfp4(*q, *p, *p), h,
            *pb.gemm_gated_bf16_backward(h, x, w, w, g, u))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, run()))
print("captured")
"""
    root = Path(__file__).resolve().parent.parent
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


def test_offsets_past_32_bits(cuda_device):
    """Tensors of more than 2^31 values and results of more than 2^31 elements: their last rows."""
    rows, K = 70016, 32768                                    # 2.29e9 values, 1.15 GB of codes
    x = torch.zeros((rows, K), dtype=torch.bfloat16, device=cuda_device)
    last = _values(130, K, seed=9, dtype=torch.bfloat16)
    x[-130:] = last.to(cuda_device)
    q, sf = pb.quant_mxfp4(x)
    code, byte = R.quantise(_np(last))
    np.testing.assert_array_equal(_np(q[-130:]), R.pack(code, byte)[0])
    full = sf.view(-1, K // 128, 512)                         # atoms [row block][K chunk]
    r = np.arange(rows - 130, rows)
    j = np.arange(K // 32)
    at = torch.from_numpy((r % 32)[:, None] * 16 + (r // 32 % 4)[:, None] * 4 + j % 4).to(cuda_device)
    got = full[torch.from_numpy(r // 128).to(cuda_device)[:, None], torch.from_numpy(j // 4).to(cuda_device)[None, :], at]
    np.testing.assert_array_equal(_np(got), byte)
    back = pb.dequant_mxfp4(q, sf)
    np.testing.assert_array_equal(_np(back[-130:]), _np(pb.dequant_mxfp4(*pb.quant_mxfp4(last.to(cuda_device)))))
    assert (back[:-130] == 0).all()
    del x, back
    # as the weights of a product with few rows: code offsets past 32 bits of nibbles and of bytes' bits
    a, av = _operand(2, K, 5, cuda_device)
    wv = _np(pb.dequant_mxfp4(*pb.quant_mxfp4(last.to(cuda_device)), pb.QG_OUT_F32))
    y = pb.gemm_mxfp4(*a, q, sf, out_type=pb.QG_OUT_F32)
    assert (np.abs(_np(y[:, -130:]) - av @ wv.T) <= R.sum_bound(av, wv)).all() and (y[:, :-130] == 0).all()
    del q, sf, y
    # a result of 2.8e9 elements
    M, N = 70000, 40000
    a, av = _operand(M, 64, 6, cuda_device)
    b, bv = _operand(N, 64, 7, cuda_device)
    p, e = av[-65:] @ bv.T, R.sum_bound(av[-65:], bv)
    y = pb.gemm_mxfp4(*a, *b)
    assert (np.abs(_np(y[-65:]) - p) <= e + 2.0 ** -8 * (np.abs(p) + e)).all()
    y = pb.gemm_gated_mxfp4(*a, *b, *b)
    with np.errstate(over="ignore"):
        ref, e = R.activation(p, 0) * p, R.gated_bound(p, p, e, e, 0)
    assert (np.abs(_np(y[-65:]) - ref) <= e + 2.0 ** -8 * (np.abs(ref) + e)).all()
