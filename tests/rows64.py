"""64-bit restatements of the row operators (linear, mixture, embedding) and how far a result may be off.

UNIT is half a unit in the last place of a type relative to the value (the error of one rounding), TINY half its
smallest subnormal.  A sum of k fp32 terms of total magnitude m is off by at most (k + 2) * 2**-24 * m (1 + o(1)),
whatever its order; SUM adds a tenth for the o(1)."""
import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
DTYPES = (torch.float16, torch.bfloat16, torch.float32)

# what the fp32 evaluation of an activation or its slope may be off by beside its argument's error:
# a few of its own roundings and two library functions of at most 4 units each
EVALUATION = 2.0 ** -20


def sum_error(terms, magnitude):
    return 1.1 * (terms + 2) * 2.0 ** -24 * magnitude


def rounding(dtype, value):
    return UNIT[dtype] * value.abs() * 1.001 + TINY[dtype]


def activation64(z, name):
    """The activation, its slope, and bounds of |slope| and |curvature|."""
    s = torch.sigmoid(z)
    if name == 'none':
        return z, torch.ones_like(z), 1.0, 0.0
    if name == 'relu':
        return z.clamp(min=0), (z > 0).double(), 1.0, 0.0
    if name == 'sigmoid':
        return s, s * torch.sigmoid(-z), 0.25, 0.1
    if name == 'softplus':
        return torch.logaddexp(z, torch.zeros_like(z)), s, 1.0, 0.25
    if name == 'silu':
        return z * s, s * (1 + z * torch.sigmoid(-z)), 1.1, 0.5
    area = torch.special.ndtr(z)
    return z * area, area + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 1.13, 0.8


class Layer64:
    """One layer in 64 bits with the bounds of its results: tensors x, w, b, r, dy of one type."""

    def __init__(self, x, w, b, r, dy, activation):
        dtype = x.dtype
        x, w = x.detach().double(), w.detach().double()
        b = torch.zeros(w.shape[0], dtype=torch.float64, device=x.device) if b is None else b.detach().double()
        r = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device) if r is None \
            else r.detach().double()
        z = x @ w.t() + b
        a, slope, steep, curve = activation64(z, activation)
        z_error = sum_error(x.shape[1] + 1, x.abs() @ w.abs().t() + b.abs())
        a_error = steep * z_error + EVALUATION * (a.abs() + z.abs())
        self.y = a + r
        self.y_error = a_error + 2.0 ** -23 * (a.abs() + r.abs()) + rounding(dtype, self.y)
        self.y_error = self.y_error * (1 + UNIT[dtype])
        if dy is None:
            return
        dy = dy.detach().double()
        dz = dy * slope
        # the backward reads z rounded to the type, and rounds dz to it (neither with no activation)
        dz_error = torch.zeros_like(dz)
        if activation != 'none':
            kept = z_error + rounding(dtype, z)
            dz_error = dy.abs() * (curve * kept + EVALUATION * (1 + z.abs())) + 2.0 ** -23 * dz.abs()
            dz_error = dz_error * (1 + UNIT[dtype]) + rounding(dtype, dz)
        size = dz.abs() + dz_error
        n, outputs = dz.shape
        self.dx = dz @ w
        self.dx_error = dz_error @ w.abs() + sum_error(outputs, size @ w.abs())
        self.dx_error = self.dx_error * (1 + UNIT[dtype]) + rounding(dtype, self.dx)
        self.dw = dz.t() @ x
        self.dw_error = dz_error.t() @ x.abs() + sum_error(n, size.t() @ x.abs())
        self.dw_error = self.dw_error * (1 + UNIT[dtype]) + rounding(dtype, self.dw)
        self.db = dz.sum(0)
        self.db_error = dz_error.sum(0) + sum_error(n, size.sum(0))
        self.db_error = self.db_error * (1 + UNIT[dtype]) + rounding(dtype, self.db)


def check(got, expected, error, what):
    """got within error of expected, entry by entry."""
    got = got.detach().double()
    assert got.shape == expected.shape, (what, got.shape, expected.shape)
    off = (got - expected).abs()
    bad = ~(off <= error)
    if bad.any():
        at = tuple(int(i) for i in torch.nonzero(bad)[0])
        raise AssertionError('%s: %d of %d off, first at %s: %r for %r, %g allowed' % (
            what, int(bad.sum()), bad.numel(), at, float(got[at]), float(expected[at]), float(error[at])))
