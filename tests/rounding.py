"""Values in 64 bits that carry a bound on the error of the same computation in fp32: what the tests
of the row operators compare kernels with.

Running error analysis: every operation adds half a step of fp32 (u = 2^-24, relative to its result)
to what its operands' errors become in it, sums add one such half step per addition on the longest
path of the kernel's order (``depth``), applied to the sum of the magnitudes.  A fused multiply-add
rounds once instead of twice and stays inside the bound.  Storing adds half a step of the type."""
import numpy as np
import torch

U = 2.0 ** -24


class B:
    """v: the value in float64; e: |fp32 result - v| <= e."""

    def __init__(self, v, e=None):
        self.v = v.double() if isinstance(v, torch.Tensor) else torch.tensor(float(v), dtype=torch.float64)
        self.e = torch.zeros_like(self.v) if e is None else e

    def __add__(self, o):
        o = o if isinstance(o, B) else const(o)
        v = self.v + o.v
        return B(v, self.e + o.e + U * (v.abs() + self.e + o.e))

    __radd__ = __add__

    def __neg__(self):
        return B(-self.v, self.e)

    def __sub__(self, o):
        return self + (-(o if isinstance(o, B) else const(o)))

    def __mul__(self, o):
        o = o if isinstance(o, B) else const(o)
        v = self.v * o.v
        e = self.v.abs() * o.e + o.v.abs() * self.e + self.e * o.e
        return B(v, e + U * (v.abs() + e))

    __rmul__ = __mul__

    def sum(self, dim, depth, keepdim=False):
        mag = (self.v.abs() + self.e).sum(dim=dim, keepdim=keepdim)
        return B(self.v.sum(dim=dim, keepdim=keepdim), self.e.sum(dim=dim, keepdim=keepdim) + depth * U * 1.01 * mag)

    def mean(self, dim, depth, keepdim=False):
        """The sum times a rounded 1 / n: two more roundings."""
        s, n = self.sum(dim, depth, keepdim), self.v.shape[dim]
        return B(s.v / n, (s.e + 2.01 * U * (s.v.abs() + s.e)) / n)

    def rsqrt(self):
        """1 / sqrt in two or three roundings."""
        low = (self.v - self.e).clamp(min=1e-300)
        v = self.v.rsqrt()
        return B(v, (low.rsqrt() - v) + 4 * U * low.rsqrt())

    def stored(self, dtype):
        """(value, bound) after rounding to ``dtype`` (half a step; below its smallest normal half of that step)."""
        info = torch.finfo(dtype)
        top = self.v.abs() + self.e
        return self.v, self.e + torch.maximum(info.eps / 2 * top, torch.full_like(top, info.smallest_normal * info.eps / 2))


def const(c):
    """A host number that the kernel holds in fp32."""
    if isinstance(c, torch.Tensor):
        return B(c)
    v = torch.tensor(float(np.float32(c)), dtype=torch.float64)
    return B(v)


def check(got, want, dtype, what):
    """``got`` (any device) against the B ``want`` stored as ``dtype``."""
    v, tol = want.stored(dtype)
    assert got.dtype == dtype, (what, got.dtype)
    assert tuple(got.shape) == tuple(v.shape), (what, tuple(got.shape), tuple(v.shape))
    got = got.detach().double().cpu()
    assert torch.equal(torch.isfinite(got), torch.isfinite(v)), "%s: finite in different places" % what
    err = torch.where(torch.isfinite(v), (got - v).abs(), torch.zeros_like(v))
    tol = torch.where(torch.isfinite(v), tol, torch.ones_like(v))
    bad = err > tol
    if bad.any():
        i = int(torch.argmax(err / tol))
        raise AssertionError("%s: %d of %d off; worst at %d: got %r want %r, bound %.3e"
                             % (what, int(bad.sum()), bad.numel(), i, got.flatten()[i].item(), v.flatten()[i].item(),
                                tol.flatten()[i].item()))
