"""Residual connections with norms: what stands between the blocks of a deep model.

``residual_norm`` is the fused operator, ``ResidualNorm`` the module that owns its vectors:

    r = res_scale * x + branch_scale * gate * post(f)      the residual stream after a block
    y = pre(r)                                             what the next block reads

The batch norm of the models (``BatchNorm1d``) stays what it is; these norms work on each row by
itself.  No counterpart upstream.
"""
import torch

from cxgnncomp_backend import residual_norm as _residual_norm

_KINDS = (None, "layer", "rms")


def residual_norm(x, f, gate=None, *, post=None, post_weight=None, post_bias=None, pre="layer", pre_weight=None,
                  pre_bias=None, res_scale=1.0, branch_scale=1.0, eps=1e-5):
    """``r = res_scale * x + branch_scale * gate * post(f)`` and ``y = pre(r)`` from one pass over the
    rows of x and f [N, C] (CUDA, C up to 8192); returns ``(r, y)``.

    ``post`` / ``pre``: "layer", "rms" (over the columns of a row, ``eps`` under the root) or None;
    their weights and biases are fp32 [C], missing ones 1 and 0.  Without a pre norm y is None.
    ``gate``: None, fp32 [C], or of f's dtype [N, 1] or [N, C].  x and r share a dtype, f and y
    another: the same, or x is float32 beside bfloat16 / float16 branches.  Arithmetic is fp32 and
    y is formed from r before r is rounded to its dtype.  Rows may be strided.

    ``f=None`` (the entry of a stack, before any block): ``(x, pre(x))``, x itself.

    One autograd node (csrc_ext/backend_ext.cpp): its backward pass reads x, f, the gate and two
    statistics per norm and row; r and y are not kept.  Gradients of every tensor argument, once (no
    second and no forward-mode derivatives: both raise); the sums over rows behind the
    vectors' gradients are added in a fixed order, so they repeat bit for bit.
    """
    r, y = _residual_norm(x, f, gate, post, post_weight, post_bias, pre, pre_weight, pre_bias, res_scale, branch_scale, eps)
    return (x if f is None else r), y


class ResidualNorm(torch.nn.Module):
    """The vectors of ``residual_norm`` for rows of ``channels`` columns.

    ``post`` / ``pre`` as there (a layer norm has weight and bias, an rms norm a weight);
    ``gate="channel"`` adds a learned gate per column that starts at ``gate_init``; gates of rows or
    elements are passed to ``forward``."""

    def __init__(self, channels, post=None, pre="layer", gate=None, gate_init=1.0, res_scale=1.0, branch_scale=1.0,
                 eps=1e-5):
        super().__init__()
        if gate not in (None, "channel"):
            raise ValueError("gate must be None or 'channel', got %r" % (gate, ))
        for kind, name in ((post, "post"), (pre, "pre")):
            if kind not in _KINDS:
                raise ValueError("%s must be 'layer', 'rms' or None, got %r" % (name, kind))
        self.channels, self.post, self.pre = channels, post, pre
        self.gate_init, self.res_scale, self.branch_scale, self.eps = gate_init, res_scale, branch_scale, eps
        for name, wanted in (("post_weight", post is not None), ("post_bias", post == "layer"),
                             ("pre_weight", pre is not None), ("pre_bias", pre == "layer"), ("gate", gate is not None)):
            self.register_parameter(name, torch.nn.Parameter(torch.empty(channels)) if wanted else None)
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            for p, value in ((self.post_weight, 1.0), (self.post_bias, 0.0), (self.pre_weight, 1.0),
                             (self.pre_bias, 0.0), (self.gate, self.gate_init)):
                if p is not None:
                    p.fill_(value)

    def forward(self, x, f, gate=None):
        if gate is not None and self.gate is not None:
            raise ValueError("the module has a gate of its own")
        return residual_norm(x, f, self.gate if gate is None else gate, post=self.post, post_weight=self.post_weight,
                             post_bias=self.post_bias, pre=self.pre, pre_weight=self.pre_weight, pre_bias=self.pre_bias,
                             res_scale=self.res_scale, branch_scale=self.branch_scale, eps=self.eps)

    def enter(self, x):
        """``(x, pre(x))``: the first block's input, before there is a branch."""
        return residual_norm(x, None, pre=self.pre, pre_weight=self.pre_weight, pre_bias=self.pre_bias, eps=self.eps)

    def extra_repr(self):
        return "%d, post=%r, pre=%r, gate=%s" % (self.channels, self.post, self.pre, self.gate is not None)
