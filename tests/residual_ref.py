"""Residual norm in 64 bits, forward and backward from the formulas, with error bounds."""
import torch

from rounding import B, const

ROW_DEPTH = 64          # additions on the longest path of a sum over a row: 32 per lane, 6 + 2 across lanes and waves
COL_DEPTH = 160         # ... over up to 4096 rows: 4096 / 256 per team, 4 + 3 in a block, 24 + 5 for partial rows


def normed(v, kind, w, b, eps):
    """(output, normalised rows, 1/std)."""
    if kind == "layer":
        v = v - v.mean(1, ROW_DEPTH, True)
    rstd = ((v * v).mean(1, ROW_DEPTH, True) + eps).rsqrt()
    hat = v * rstd
    out = hat if w is None else hat * B(w)
    return (out if b is None else out + B(b)), hat, rstd


def normed_back(g, hat, rstd, kind):
    out = g - hat * ((g * hat).mean(1, ROW_DEPTH, True))
    if kind == "layer":
        out = out - g.mean(1, ROW_DEPTH, True)
    return out * rstd


def residual_norm(x, f, gate, post, pw, pb, pre, qw, qb, res_scale, branch_scale, eps, dr=None, dy=None):
    """dict of B: r, y and, with dr or dy, the gradients under the arguments' names."""
    out = {}
    a, bs = const(res_scale), const(branch_scale)
    if f is not None:
        f = B(f)
        h, fhat, rstd1 = normed(f, post, pw, pb, eps) if post else (f, f, None)
        gated = h if gate is None else h * B(gate)
        r = B(x) * a + gated * bs
        out["r"] = r
    else:
        r = B(x) * a
    if pre:
        out["y"], rhat, rstd2 = normed(r, pre, qw, qb, eps)
    if dr is None and dy is None:
        return out
    g = B(torch.zeros_like(r.v) if dr is None else dr)
    if dy is not None:
        dy = B(dy)
        t = dy if qw is None else dy * B(qw)
        g = g + normed_back(t, rhat, rstd2, pre)
        out["pre_weight"], out["pre_bias"] = (dy * rhat).sum(0, COL_DEPTH), dy.sum(0, COL_DEPTH)
    elif pre:
        out["pre_weight"] = out["pre_bias"] = B(torch.zeros(r.v.shape[1], dtype=torch.float64))
    out["x"] = g * a
    if f is None:
        return out
    gh = g * h * bs
    if gate is not None:
        if gate.dim() == 1:
            # the kernel sums g * fhat and g and combines them with w and b: bound that order
            s1, s0 = (g * fhat).sum(0, COL_DEPTH), g.sum(0, COL_DEPTH)
            d = s1 if pw is None else s1 * B(pw)
            out["gate"] = (d if pb is None else d + s0 * B(pb)) * bs
        else:
            out["gate"] = gh.sum(1, ROW_DEPTH, True) if gate.shape[1] == 1 and gh.v.shape[1] != 1 else gh
    d = g * bs if gate is None else g * B(gate) * bs
    if post:
        out["post_weight"], out["post_bias"] = (d * fhat).sum(0, COL_DEPTH), d.sum(0, COL_DEPTH)
        d = normed_back(d if pw is None else d * B(pw), fhat, rstd1, post)
    out["f"] = d
    return out
