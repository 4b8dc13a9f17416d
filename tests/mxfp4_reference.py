"""Plain 64-bit numpy statement of the MXFP4 format and of the gated products, for the tests.

Blocks of 32 along K share 2^e, e = max(floor(log2 max|x|) - 2, -127), stored as e + 127;
values are rounded to 0, 0.5, 1, 1.5, 2, 3, 4, 6 times 2^e (nearest, ties to even, saturating).
"""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def up(a, b):
    return -(-a // b) * b


def sf_index(rows, K):
    """Byte offsets [rows, K/32] of the scales in their atoms."""
    r = np.arange(rows)[:, None]
    j = np.arange(K // 32)[None, :]
    return ((r // 128) * -(-K // 128) + j // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + j % 4


def quantise(x):
    """x [M, K] -> (code [M, Kp] 0..15, byte [M, Kp/32])."""
    x = np.asarray(x, dtype=np.float64)
    M, K = x.shape
    xp = np.zeros((M, up(K, 32)))
    xp[:, :K] = x
    b = xp.reshape(M, -1, 32)
    bad = ~np.isfinite(b).all(-1)
    amax = np.where(bad, 0.0, np.abs(np.where(np.isfinite(b), b, 0.0)).max(-1))
    e = np.where(amax > 0, np.frexp(amax)[1] - 1 - 2, -127).clip(-127)
    a = np.abs(np.where(bad[..., None], 0.0, b)) * np.exp2(-e.astype(np.float64))[..., None]
    # nearest level; on a tie the level whose code is even
    code = np.zeros(a.shape, dtype=np.uint8)
    for c in range(7):
        mid = (LEVELS[c] + LEVELS[c + 1]) / 2
        code += (a > mid) | ((a == mid) & (c % 2 == 1))
    code |= (np.signbit(b) & ~bad[..., None]).astype(np.uint8) << 3
    return code.reshape(M, -1), np.where(bad, 255, e + 127).astype(np.uint8)


def pack(code, byte):
    """(code, byte) -> (packed codes, atoms with zero padding)."""
    rows, K = code.shape
    atoms = np.zeros(up(rows, 128) * up(K, 128) // 32, dtype=np.uint8)
    atoms[sf_index(rows, K)] = byte
    return code[:, 0::2] | (code[:, 1::2] << 4), atoms


def decode(q, atoms):
    """(packed codes, atoms) -> values [rows, K] in 64 bits."""
    rows, K = q.shape[0], 2 * q.shape[1]
    code = np.stack([q & 15, q >> 4], -1).reshape(rows, K)
    byte = atoms[sf_index(rows, K)]
    scale = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    v = np.where(code >= 8, -1.0, 1.0) * LEVELS[code & 7]
    return (v.reshape(rows, -1, 32) * scale[..., None]).reshape(rows, K)


def act_arg(g, act):
    """The logistic's argument y: act(g) = g / (1 + exp(-y)).  act 0 = silu, 1 = gelu (tanh form)."""
    return g if act == 0 else 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)


def _logistic(g, act):
    """p = 1 / (1 + exp(-y)).  For gelu this is 0.5 (1 + tanh(y / 2)), whose sum would cancel: at
    y = -36 it is 1.6e-16, and 64-bit numbers just below 1 are 1.1e-16 apart."""
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-act_arg(g, act)))


def activation(g, act):
    return g * _logistic(g, act)


def slope(g, act):
    p = _logistic(g, act)
    dy = 1 if act == 0 else 2 * np.sqrt(2 / np.pi) * (1 + 3 * 0.044715 * g ** 2)
    return p + g * p * _logistic(-g, act) * dy


def sum_bound(a, b):
    """How far an fp32 sum of exact products over K may be from a @ b^T: K additions, each at most
    one unit (2^-23, truncation counted) of the sum of magnitudes."""
    return a.shape[1] * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T)


def gated_bound(g, u, eg, eu, act):
    """How far act(g) u in fp32 may be from its 64-bit value, with g and u off by eg and eu: slopes of
    both activations are below 1.13 in magnitude; 2^x and the reciprocal are good to a few units, and
    the argument's own rounding (4 units of |y|) and 2^x's error growth (1.2 units per unit of y)
    count by |y|; two products; the logistic is cut off at exp(87), an absolute 2e-38."""
    rel = (12 + 6 * np.abs(act_arg(g, act))) * 2.0 ** -23
    a = np.abs(activation(g, act))
    return 1.13 * eg * (np.abs(u) + eu) + a * eu + rel * a * np.abs(u) + 2e-38 * (1 + np.abs(g * u))
