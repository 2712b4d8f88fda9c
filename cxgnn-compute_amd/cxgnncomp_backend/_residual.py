"""Residual norm on the C ABI (csrc/residual_norm_fwd.hip, csrc/residual_norm_bwd.hip):
argument checks, allocation, workspace and current stream."""
import torch

from . import _lib
from ._ops import _workspace

VALUE_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
NORM_KINDS = {None: 0, "rms": 1, "layer": 2}
GATE_NONE, GATE_CHANNEL, GATE_ROW, GATE_FULL = 0, 1, 2, 3
MAX_COLS = 8192


def rows_of(t, name, device=None):
    """``t`` as a CUDA matrix whose rows are contiguous (their stride is free), copied if they are not."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor" % name)
    if not t.is_cuda:
        raise ValueError("%s must be a CUDA tensor" % name)
    if t.dtype not in VALUE_TYPES:
        raise ValueError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    if t.dim() != 2:
        raise ValueError("%s must have 2 dims, got %d" % (name, t.dim()))
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, expected %s" % (name, t.device, device))
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _vector(t, name, cols, device):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor" % name)
    if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != cols:
        raise ValueError("%s must be float32 [%d], got %s %s" % (name, cols, t.dtype, tuple(t.shape)))
    if t.device != device:
        raise ValueError("%s is on %s, expected %s" % (name, t.device, device))
    return t.contiguous()


class Call:
    """The checked arguments of one residual norm (``x`` and ``f`` as given; ``f`` None: y = pre(x))."""

    __slots__ = ("x", "f", "gate", "gate_kind", "post", "post_w", "post_b", "pre", "pre_w", "pre_b", "res_scale",
                 "branch_scale", "eps", "rows", "cols", "stream_type", "branch_type", "branch_dtype")

    def __init__(self, x, f, gate, post, post_w, post_b, pre, pre_w, pre_b, res_scale, branch_scale, eps):
        self.x = x = rows_of(x, "x")
        dev = x.device
        self.rows, self.cols = rows, cols = x.shape
        if not 1 <= cols <= MAX_COLS:
            raise ValueError("residual_norm takes 1 to %d columns, got %d" % (MAX_COLS, cols))
        if f is not None:
            f = rows_of(f, "f", dev)
            if f.shape != x.shape:
                raise ValueError("f has shape %s, x %s" % (tuple(f.shape), tuple(x.shape)))
            if x.dtype != torch.float32 and f.dtype != x.dtype:
                raise ValueError("f must have x's dtype %s unless x is float32, got %s" % (x.dtype, f.dtype))
        elif gate is not None or post is not None or res_scale != 1.0 or pre is None:
            raise ValueError("without a branch there is the norm of x alone: no gate, post norm or scale, and a pre norm")
        self.f = f
        self.branch_dtype = x.dtype if f is None else f.dtype
        self.stream_type, self.branch_type = VALUE_TYPES[x.dtype], VALUE_TYPES[self.branch_dtype]
        for kind, name in ((post, "post"), (pre, "pre")):
            if kind not in NORM_KINDS:
                raise ValueError("%s must be 'layer', 'rms' or None, got %r" % (name, kind))
        for kind, w, b, name in ((post, post_w, post_b, "post"), (pre, pre_w, pre_b, "pre")):
            if kind is None and not (w is None and b is None):
                raise ValueError("%s_weight / %s_bias without a %s norm" % (name, name, name))
        self.post, self.pre = NORM_KINDS[post], NORM_KINDS[pre]
        self.post_w, self.post_b = _vector(post_w, "post_weight", cols, dev), _vector(post_b, "post_bias", cols, dev)
        self.pre_w, self.pre_b = _vector(pre_w, "pre_weight", cols, dev), _vector(pre_b, "pre_bias", cols, dev)
        if gate is None:
            self.gate_kind = GATE_NONE
        elif isinstance(gate, torch.Tensor) and gate.dim() == 1:
            gate = _vector(gate, "a gate of columns", cols, dev)
            self.gate_kind = GATE_CHANNEL
        else:
            gate = rows_of(gate, "gate", dev)
            if gate.dtype != self.branch_dtype:
                raise ValueError("a gate of rows or elements has f's dtype %s, got %s" % (self.branch_dtype, gate.dtype))
            if tuple(gate.shape) == (rows, 1):
                self.gate_kind = GATE_ROW
            elif tuple(gate.shape) == (rows, cols):
                self.gate_kind = GATE_FULL
            else:
                raise ValueError("gate must be [%d], [%d, 1] or [%d, %d], got %s" % (cols, rows, rows, cols, tuple(gate.shape)))
        self.gate = gate
        self.res_scale, self.branch_scale, self.eps = float(res_scale), float(branch_scale), float(eps)


def _stride(t):
    return 0 if t is None else t.stride(0)


def forward(c, want_stats):
    """(r, y, stats): r None without a branch, y None without a pre norm, stats None unless asked for."""
    dev = c.x.device
    r = None if c.f is None else torch.empty((c.rows, c.cols), dtype=c.x.dtype, device=dev)
    y = torch.empty((c.rows, c.cols), dtype=c.branch_dtype, device=dev) if c.pre else None
    stats = torch.empty((c.rows, 4), dtype=torch.float32, device=dev) if want_stats else None
    p = _lib.ptr
    with torch.cuda.device(dev):
        st = _lib.load().cxg_residual_norm_fwd(
            p(c.x), c.x.stride(0), p(c.f), _stride(c.f), p(c.gate), 0 if c.gate_kind == GATE_CHANNEL else _stride(c.gate),
            c.gate_kind, c.post, p(c.post_w), p(c.post_b), c.pre, p(c.pre_w), p(c.pre_b), c.res_scale, c.branch_scale,
            c.eps, c.rows, c.cols, c.stream_type, c.branch_type, p(r), p(y), p(stats), _lib.current_stream(dev))
    _lib.check(st)
    return r, y, stats


def backward(c, stats, dr, dy, need):
    """Gradients of (x, f, gate, post_weight, post_bias, pre_weight, pre_bias); ``need``: which of them."""
    dev = c.x.device
    shape = (c.rows, c.cols)
    dr = None if dr is None else rows_of(dr, "the gradient of r", dev)
    dy = None if dy is None else rows_of(dy, "the gradient of y", dev)
    lib, p = _lib.load(), _lib.ptr

    def vector(wanted):
        return torch.empty(c.cols, dtype=torch.float32, device=dev) if wanted else None

    dx = torch.empty(shape, dtype=c.x.dtype, device=dev) if need[0] else None
    df = torch.empty(shape, dtype=c.branch_dtype, device=dev) if need[1] else None
    dgate = None
    if need[2]:
        dgate = vector(True) if c.gate_kind == GATE_CHANNEL else torch.empty(c.gate.shape, dtype=c.branch_dtype, device=dev)
    dpost_w, dpost_b, dpre_w, dpre_b = (vector(n) for n in need[3:])
    ws = None
    if any(need[3:]) or (need[2] and c.gate_kind == GATE_CHANNEL):
        ws = _workspace(lib.cxg_residual_norm_workspace_bytes(c.rows, c.cols), dev)
    with torch.cuda.device(dev):
        st = lib.cxg_residual_norm_bwd(
            p(c.x), c.x.stride(0), p(c.f), _stride(c.f), p(c.gate), 0 if c.gate_kind == GATE_CHANNEL else _stride(c.gate),
            c.gate_kind, c.post, p(c.post_w), p(c.post_b), c.pre, p(c.pre_w), c.res_scale, c.branch_scale, c.rows, c.cols,
            c.stream_type, c.branch_type, p(stats), p(dr), _stride(dr), p(dy), _stride(dy), p(dx), p(df), p(dgate),
            p(dpost_w), p(dpost_b), p(dpre_w), p(dpre_b), p(ws), 0 if ws is None else ws.numel(), _lib.current_stream(dev))
    _lib.check(st)
    return dx, df, dgate, dpost_w, dpost_b, dpre_w, dpre_b
