"""Rows in 8 bits, restated in 64 bits on the host: codes and exponent bytes from the definition, what
they stand for, and the weight gradient with an error bound."""
import torch

from rounding import B, U

GROUP = 128


def scales(x, fmt):
    """Exponent bytes [rows, groups] of float64 rows."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x, (0, -cols % GROUP)).view(rows, -(-cols // GROUP), GROUP)
    top = v.abs().amax(dim=2)
    finite = torch.isfinite(v).all(dim=2)
    top = torch.where(finite, top, torch.ones_like(top))
    k = torch.full_like(top, -111.0)
    for e in range(-111, 128):                           # the smallest exponent with which the top fits
        t = top * 2.0 ** -e
        fits = (torch.round(t) <= 127) if fmt == "int8" else (t <= 448)
        k = torch.where(fits & (k == -111.0) & ~_fits(top, fmt, -111), torch.full_like(k, float(e)), k)
    return torch.where(finite, k + 127, torch.full_like(k, 255.0)).to(torch.uint8)


def _fits(top, fmt, e):
    t = top * 2.0 ** -e
    return (torch.round(t) <= 127) if fmt == "int8" else (t <= 448)


def spread(exps, cols):
    """2^k per column; NaN where the group was not finite."""
    e = exps.double()
    s = torch.where(e == 255, torch.full_like(e, float("nan")), torch.exp2(e - 127))
    return s.repeat_interleave(GROUP, dim=1)[:, :cols]


def pack(x, fmt):
    """(code bytes [rows, pitch], exponent bytes, float64 values)."""
    x = x.double()
    rows, cols = x.shape
    exps = scales(x, fmt)
    s = spread(exps, cols)
    v = torch.where(torch.isnan(s), torch.zeros_like(x), x / s)
    if fmt == "int8":
        q = torch.round(v)
        raw = q.to(torch.int8).view(torch.uint8)
    else:
        step = torch.exp2((torch.frexp(v)[1].double() - 4).clamp(min=-9.0))
        q = torch.round(v / step) * step
        q = torch.copysign(q, v)
        raw = q.float().to(torch.float8_e4m3fn).view(torch.uint8)
        assert torch.equal(raw.view(torch.float8_e4m3fn).double(), q)
    codes = torch.nn.functional.pad(raw, (0, -cols % 16))
    return codes, exps, q * s


def decode(codes, exps, cols, fmt):
    raw = codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).double()[:, :cols]
    return raw * spread(exps, cols)


def weight_grad(a, g, bounds, src=None, dst=None):
    """B [R, K, N].  Products of bf16 parts are exact in fp32 and the parts of a value add up to it (their
    magnitudes to 1 + 2^-7 of its); every row adds up to three products to a sum, each addition off by
    at most one unit (2 U) of what has been added so far, and the chunk sums at most as many more."""
    parts = {torch.float32: 3, torch.bfloat16: 1, torch.float16: 2}[g.dtype]
    g = g.double()
    out, tol = [], []
    for b, e in zip(bounds, bounds[1:]):
        rows = torch.arange(b, e)
        s = rows if src is None else src[rows]
        d = rows if dst is None else dst[rows]
        keep = (s >= 0) & (s < a.shape[0]) & (d >= 0) & (d < g.shape[0])
        x, y = a[s[keep]], g[d[keep]]
        out.append(x.t() @ y)
        depth = parts * x.shape[0] + x.shape[0] // 128 + 2
        tol.append(2 * U * depth * 1.01 * (x.abs().t() @ y.abs()))
    return B(torch.stack(out), torch.stack(tol))


def row_sums(g, bounds, dst=None, keep=None):
    """[B [N]] per segment: sums of the rows of g (at most one rounding per row and chunk), rows with
    ``keep`` False left out."""
    out = []
    for b, e in zip(bounds, bounds[1:]):
        rows = torch.arange(b, e)
        if keep is not None:
            rows = rows[keep[b:e]]
        y = g.double()[rows if dst is None else dst[rows]]
        out.append(B(y.sum(0), U * (y.shape[0] + y.shape[0] // 128 + 2) * 1.01 * y.abs().sum(0)))
    return out
