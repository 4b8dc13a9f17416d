"""The activations' slopes, relative to their own size, where they are small.

With Wg the identity, Wu zero and dH and U one, dX is dG: the slope of each value of G, rounded.  It is
p + g dy p (1 - p), p = 1 / (1 + exp(-y)), in fp32, u = 2^-23:
* p is off by E p, E = (12 + 6 |y|) u: as mxfp4_reference.gated_bound counts it;
* 1 - p by what p is off: E p (1 - p) through exp, and 4 u for the sum, the quotient and the difference;
* so the product by |g| p dy (2 (1 - p) E + 8 u); from |y| = 100 on p is exactly 0 or 1;
* the logistic is cut off below 2^-126: 2e-38 of every factor beside it.
dG is rounded by half a step where M N > 65536, and below that by half a step of what that leaves; the
products' sums have 2 N terms; dX's own half step.
"""
import numpy as np
import pytest
import torch

import pantheon_b200 as pb
from tests import mxfp4_reference as R

pytestmark = pytest.mark.gpu

TYPES = {"bf16": (torch.bfloat16, 2.0 ** -8, 2.0 ** -134, pb.gemm_gated_bf16_backward),
         "f16": (torch.float16, 2.0 ** -11, 2.0 ** -25, pb.gemm_gated_f16_backward)}
# (below -87.3 the logistic is cut off at 2^-126)
GATES = [-85.0, -80.0, -70.0, -60.0, -50.0, -40.0, -35.0, -31.0, -30.0, -29.0, -20.0, -12.0, -10.0, -9.0, -7.0, -5.0,
         -3.0, -2.0, -0.5, 0.0, 0.5, 2.0, 5.0, 9.0, 20.0, 31.0, 60.0, 100.0]


@pytest.mark.parametrize("rows", [len(GATES), 8210], ids=["two terms", "one term"])
@pytest.mark.parametrize("act", [pb.QG_ACT_SILU, pb.QG_ACT_GELU_TANH], ids=["silu", "gelu"])
@pytest.mark.parametrize("kind", list(TYPES))
def test_slopes_are_right_relative_to_themselves(cuda_device, kind, act, rows):
    t, step, least, backward = TYPES[kind]
    N = 8
    vals = torch.tensor(GATES, dtype=torch.float64).repeat(-(-rows // len(GATES)))[:rows]
    g = vals.to(t).to(cuda_device)[:, None].repeat(1, N)
    one = torch.ones_like(g)
    wg, wu = torch.eye(N, dtype=t, device=cuda_device), torch.zeros((N, N), dtype=t, device=cuda_device)
    dx, dwg, dwu = backward(one, one, wg, wu, g, one, act=act)
    gate = g.double().cpu().numpy()
    with np.errstate(over="ignore"):
        slope, y = R.slope(gate, act), R.act_arg(gate, act)
        p, q = 1 / (1 + np.exp(-y)), 1 / (1 + np.exp(y))
    dy = 1.0 if act == 0 else 1.6 + 0.2141 * gate * gate
    unit = 2.0 ** -23
    E = (12 + 6 * np.abs(y)) * unit
    e = np.where(np.abs(y) < 100, E * p + np.abs(gate) * p * dy * (2 * q * E + 8 * unit), 0)
    e += 2e-38 * (1 + np.abs(gate) * dy)
    e += 2 * N * unit * np.abs(slope)
    left = step if rows * N > 65536 else step * step
    e += np.maximum(left * (np.abs(slope) + e), least) * (1 + 2 * step)
    e += np.maximum(step * (np.abs(slope) + e), least)
    assert (np.abs(dx.double().cpu().numpy() - slope) <= e).all()
    assert pb.device_status(0) == 0
