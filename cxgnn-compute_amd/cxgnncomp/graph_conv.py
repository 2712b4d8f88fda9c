"""Aggregation autograd ops and graph convolution layers of the reference
(cxgnncomp/graph_conv.py) on the HIP backend.  Layers take the graph as
``(ptr, idx)`` = CSR by destination plus the number of destination rows.

PyTorch Geometric and torch_scatter are not needed: ``Linear``/``glorot`` are
replaced by torch.nn.Linear with Glorot-uniform weights, and the op-wise edge
softmax is written with core torch ops.
"""
import math

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable
from torch.nn import Parameter

import cxgnncomp_backend
from cxgnncomp_backend import _ops, _typed
from cxgnncomp_backend import (aggr_rel, aggr_rgcn_direct_func, edge_attention, gather,
                               sage_mean_forward, sage_sum_forward, sage_sum_forward_edge_value,
                               selective_aggr, selective_aggr_bwd)

from .graph_kernel import SpMMValOP
from .packed import FORMATS, PackedRows, check_format, pack_rows, packed_weight_grad
from .timer import TimerOP
from .typed_linear import (TypedLinearE2EOP, TypedLinearS2DAggrMMOP, TypedLinearS2DMMAggrOP,
                           TypedLinearS2DPushOP, TypedLinearS2DSort)
from .util import global_tuner, log

for _name in ("edge_attention", "sage_sum_forward_edge_value", "gather", "sage_sum_forward",
              "aggr_rel", "sage_mean_forward"):
    torch.fx.wrap(_name)


def glorot(tensor):
    """Glorot/Xavier uniform over the last two dimensions (what PyG's ``glorot`` does)."""
    if tensor is not None:
        bound = math.sqrt(6.0 / (tensor.size(-2) + tensor.size(-1)))
        tensor.data.uniform_(-bound, bound)


def _num(v):
    return int(v.item()) if isinstance(v, torch.Tensor) else int(v)


class AggrOP(torch.autograd.Function):
    """Sum aggregation through the tuner entry point (upstream :34-77).  Upstream's
    backward re-runs the forward kernel on grad_out, which equals A^T g only for a
    symmetric square graph; the backward here is the true transposed aggregation
    (identical on symmetric graphs)."""

    @staticmethod
    def forward(ctx, x, ptr, idx, num_center):
        n = _num(num_center)
        ctx.save_for_backward(ptr, idx)
        ctx.n, ctx.n_src = n, x.shape[0]
        return global_tuner.tune_graph(n, idx.shape[0], x.shape[-1],
                                       cxgnncomp_backend.run_spmm_configurable,
                                       [ptr, idx, x.contiguous(), n])

    @staticmethod
    def backward(ctx, grad_out):
        ptr, idx = ctx.saved_tensors
        like = grad_out.new_empty((ctx.n_src, 0))
        grad_x = global_tuner.tune_graph(ctx.n, idx.shape[0], grad_out.shape[-1],
                                         cxgnncomp_backend.run_spmm_configurable_bwd,
                                         [ptr, idx, like, grad_out.contiguous(), ctx.n])
        return grad_x, None, None, None


class AggrDirectedOP(AggrOP):
    """Upstream :80-114: forward as AggrOP, backward by run_spmm_configurable_bwd --
    which is what AggrOP does here as well."""


class SeastarRGCNOP(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weights, ptr, idx, rel, num_center):
        if rel.dtype not in (torch.int32, torch.int64):     # integer ids pass as they are: structures built from them are cached per tensor
            rel = rel.to(torch.int64)
        ctx.save_for_backward(x, weights, ptr, idx, rel)
        return cxgnncomp_backend.seastar_forward(x, ptr, idx, weights, rel)

    @staticmethod
    def backward(ctx, grad_out):
        x, weights, ptr, idx, rel = ctx.saved_tensors
        grad_x, grad_weight = cxgnncomp_backend.seastar_backward(x, ptr, idx, weights, rel, grad_out)
        return grad_x, grad_weight, None, None, None, None


class RGCNOP(torch.autograd.Function):
    """Transform all nodes per relation, then masked aggregation (upstream :205-243): one
    product over all nodes and one pass over all edges per relation.  CUDA tensors take the
    same computation in that order as two typed operators -- one typed GEMM over the
    (source, relation) pairs that occur, one aggregation (``TypedLinearS2DMMAggrOP``) -- instead
    of 2 R products and 2 R masked passes over the whole edge array."""

    @classmethod
    def apply(cls, x, weights, ptr, idx, rel, num_center):
        if x.is_cuda and weights.is_cuda and weights.dim() == 3:
            return TypedLinearS2DMMAggrOP.apply(x, weights, ptr, idx, rel, num_center)
        return super().apply(x, weights, ptr, idx, rel, num_center)

    @staticmethod
    def forward(ctx, x, weights, ptr, idx, rel, num_center):
        n = _num(num_center)
        ctx.save_for_backward(x, weights, ptr, idx, rel)
        output = torch.zeros([n, weights.shape[-1]], device=x.device)
        for i in range(weights.shape[0]):
            w = TimerOP.apply(weights[i], f"mm{i}", True)
            t = TimerOP.apply(torch.mm(x, w), f"mm{i}", False)
            t = TimerOP.apply(t, f"selective{i}", True)
            selective_aggr(t, ptr, idx, (rel == i), output, n)
            output = TimerOP.apply(output, f"selective{i}", False)
        return output

    @staticmethod
    def backward(ctx, grad_out):
        x, weights, ptr, idx, rel = ctx.saved_tensors
        grad_out = grad_out.contiguous()
        grad_x = torch.zeros_like(x)
        grad_weights = []
        n = grad_out.shape[0]
        for i in range(weights.shape[0]):
            g_sel = torch.zeros([x.shape[0], grad_out.shape[-1]], device=x.device)
            g_sel = TimerOP.apply(g_sel, f"selective_bwd{i}", True)
            selective_aggr_bwd(grad_out, ptr, idx, (rel == i), g_sel, n)
            g_sel = TimerOP.apply(g_sel, f"selective_bwd{i}", False)
            g_sel = TimerOP.apply(g_sel, f"mm_bwd{i}", True)
            grad_x += torch.mm(g_sel, weights[i].t())
            g_sel = TimerOP.apply(g_sel, f"mm_bwd{i}", False)
            grad_weights.append(torch.mm(x.t(), g_sel))
        return grad_x, torch.stack(grad_weights), None, None, None, None


def RGCNOP_sorted(x, weights, src, dst, num_feat_per_rel, num_center):
    """Edges pre-sorted by relation: per segment gather -> linear -> index_add_ (:246-257)."""
    output = torch.zeros([num_center, weights.shape[-1]], device=x.device)
    start = 0
    for i in range(weights.shape[0]):
        c = int(num_feat_per_rel[i])
        output.index_add_(0, dst[start:start + c], F.linear(x[src[start:start + c]], weights[i].T))
        start += c
    return output


RGCNOP2 = TypedLinearS2DAggrMMOP          # aggregate-then-transform variant (upstream :260-292)


class RGCNOP3(torch.autograd.Function):
    """Fused aggregate+transform (upstream :295-306, whose backward returns random
    tensors); the gradients here are the true ones."""

    @staticmethod
    def forward(ctx, x, weights, ptr, idx, rel, num_center):
        with torch.enable_grad():
            xd = x.detach().requires_grad_(True)
            wd = weights.detach().requires_grad_(True)
            # (no dtype conversion of integer relation ids: a fresh tensor per call would miss the
            # cache of structures built from the index arrays)
            rel_ids = rel if rel.dtype in (torch.int32, torch.int64) else rel.int()
            out = aggr_rgcn_direct_func(xd, ptr, idx, wd, rel_ids, _num(num_center))
        ctx.inner = (xd, wd, out)
        return out.detach()

    @staticmethod
    def backward(ctx, grad_out):
        xd, wd, out = ctx.inner
        gx, gw = torch.autograd.grad(out, (xd, wd), grad_out)
        return gx, gw, None, None, None, None


def run_rgcn4(x, ptr, idx, edge_types, linear, num_center, num_edge, preproccessed):
    """Gather source rows per edge, typed transform edge->edge, sum the consecutive
    edge rows of every destination (upstream :309-326)."""
    x_idxed = x[idx[:num_edge]]
    out = TypedLinearE2EOP.apply(x_idxed, linear, edge_types, preproccessed)
    new_idx = torch.arange(0, num_edge, device=x_idxed.device)
    return AggrDirectedOP.apply(out, ptr, new_idx, num_center)


class MySageConv(torch.nn.Module):

    checkpoint = None                 # (modules saved before there was one)

    def __init__(self, in_channels, hidden_channels, root_weight=True, bias=True, checkpoint=None):
        """``checkpoint`` (not upstream) "int8" or "e4m3": the inputs of the layer's linear maps are kept
        for the backward pass in 8 bits per value (``linear``); where x is wider than the output, x and its
        first rows apart."""
        super().__init__()
        self.checkpoint = check_format(checkpoint)
        self.in_channels = in_channels
        self.hidden_channels = hidden_channels
        self.root_weight = root_weight
        self.lin_l = torch.nn.Linear(in_channels, hidden_channels, bias=bias)
        if root_weight:
            self.lin_r = torch.nn.Linear(in_channels, hidden_channels, bias=False)
        self.reset_parameters()

    def reset_parameters(self):
        self.lin_l.reset_parameters()
        if self.root_weight:
            self.lin_r.reset_parameters()

    def forward(self, x, ptr, idx, num_node):
        if x.is_cuda and x.dim() == 2 and self.checkpoint is None:
            return SageLayerOP.apply(x, self.lin_l.weight, self.lin_l.bias,
                                     self.lin_r.weight if self.root_weight else None, ptr, idx, num_node)
        if self.in_channels > self.hidden_channels:
            out = sage_mean_forward(linear(x, self.lin_l.weight, self.lin_l.bias, checkpoint=self.checkpoint), ptr, idx, num_node)
        else:
            out = linear(sage_mean_forward(x, ptr, idx, num_node), self.lin_l.weight, self.lin_l.bias,
                         checkpoint=self.checkpoint)
        if self.root_weight:
            out = linear(x[:out.shape[0]], self.lin_r.weight, addend=out, checkpoint=self.checkpoint)
        return out


class MyGINConv(torch.nn.Module):

    checkpoint = None                 # (modules saved before there was one)

    def __init__(self, in_channels, hidden_channels, checkpoint=None):
        """``checkpoint`` (not upstream) "int8" or "e4m3": the input of the layer's linear map is kept for
        the backward pass in 8 bits per value (``linear``)."""
        super().__init__()
        self.checkpoint = check_format(checkpoint)
        self.in_channels = in_channels
        self.hidden_channels = hidden_channels
        self.nn = torch.nn.Linear(in_channels, hidden_channels, bias=False)
        self.init_eps = 0.2
        self.eps = torch.nn.Parameter(torch.Tensor([self.init_eps]))
        self.reset_parameters()

    def reset_parameters(self):
        self.nn.reset_parameters()
        self.eps.data.fill_(self.init_eps)

    def forward(self, x, ptr, idx, num_node):
        out = sage_mean_forward(x, ptr, idx, num_node)
        return linear(out + (1 + self.eps) * x[:num_node], self.nn.weight, checkpoint=self.checkpoint)


class MyRGCNConv(torch.nn.Module):

    def __init__(self, in_channels, hidden_channels, num_rel, precision=None):
        """``precision`` (not upstream): how the typed GEMMs of the layer multiply --
        None / "split6" (fp32-accurate), "split3", "fp32", or "bf16" (operands rounded to
        bf16 on the bf16 matrix cores, fp32 accumulation and fp32 aggregation)."""
        super().__init__()
        assert num_rel > 0
        self.in_channels = in_channels
        self.hidden_channels = hidden_channels
        self.num_rel = num_rel
        self.precision = precision
        self.linear = torch.nn.Parameter(torch.randn(num_rel, in_channels, hidden_channels))
        self.register_parameter("rel_weight", self.linear)
        self.single_linear = torch.nn.Linear(in_channels, hidden_channels)
        self.reset_parameters()
        self.preprocessed = []

    def reset_parameters(self):
        glorot(self.linear)
        self.single_linear.reset_parameters()

    def forward(self, x, ptr, idx, edge_types, num_node):
        if idx.shape[0] > 1e8:
            return RGCNOP.apply(x, self.linear, ptr, idx, edge_types, num_node)
        # Upstream gathers x[idx], runs the edge-level typed linear and sums the edge
        # rows of every destination (run_rgcn4, :309-326, :352-378); the same layer as
        # one op that never materialises per-edge rows.  Rows without edges give 0
        # (upstream divides 0 by 0 there).
        return cxgnncomp_backend.aggr_rgcn_mean(x, ptr, idx, self.linear, edge_types, num_node, self.precision)


_ARANGE = {}


def _arange_ptr(n, device):
    key = (int(n), str(device))
    if key not in _ARANGE:
        if len(_ARANGE) > 8:
            _ARANGE.clear()
        _ARANGE[key] = (torch.tensor([0, int(n)], dtype=torch.int64, device=device),
                        torch.arange(int(n), dtype=torch.int64, device=device))
    return _ARANGE[key]


class HeadDotOP(torch.autograd.Function):
    """alpha[n, h] = sum_c x[n, h, c] * att[h, c]: upstream's ``(x * att).sum(dim=-1)``
    (cxgnncomp/graph_conv.py:466-467) without the [N, H, C] temporaries.  On the GPU it is
    the SDDMM of every node row against the single row ``att`` (a one-row CSR over all
    nodes); its weight gradient is a [H, N] x [N, H*C] product on the typed weight-gradient
    kernel.  Host tensors use the upstream expression."""

    @staticmethod
    def forward(ctx, x, att):
        ctx.save_for_backward(x, att)
        if not x.is_cuda:
            return (x * att).sum(dim=-1)
        n, heads, channels = x.shape
        ptr, ar = _arange_ptr(n, x.device)
        return cxgnncomp_backend._ops.sddmm_csr(ptr, ar, x.contiguous(),
                                                att.reshape(1, heads, channels).contiguous(), 1)

    @staticmethod
    def backward(ctx, grad):
        x, att = ctx.saved_tensors
        grad = grad.contiguous()
        gx = gatt = None
        if ctx.needs_input_grad[0]:
            gx = grad.unsqueeze(-1) * att
        if ctx.needs_input_grad[1]:
            gatt = None
            if x.is_cuda:
                # grad^T x on the matrix cores: [H, N] x [N, H*C]; head h's gradient is the
                # h-th diagonal block of the [H, H*C] product
                n, heads, channels = x.shape
                seg = torch.tensor([0, n], dtype=torch.int64, device=x.device)
                full = _typed.typed_gemm_wgrad(grad, x.contiguous().view(n, heads * channels), seg, n, 1)
                if full is not None:
                    full = full.view(heads, heads, channels)
                    gatt = torch.stack([full[h, h] for h in range(heads)]).view_as(att)
            if gatt is None:
                gatt = (grad.unsqueeze(-1) * x).sum(dim=0).view_as(att)
        return gx, gatt


_SEG_CACHE = {}


def _one_segment(m, device):
    """Device tensor [0, m]: the segment table of an untyped weight gradient."""
    key = (m, device)
    seg = _SEG_CACHE.get(key)
    if seg is None:
        if len(_SEG_CACHE) > 64:
            _SEG_CACHE.clear()
        seg = _SEG_CACHE[key] = torch.tensor([0, m], dtype=torch.int64, device=device)
    return seg


def _weight_grad(x, g):
    """g^T x, the weight gradient of ``F.linear(x, w)``: one very long reduction axis, on the
    typed weight-gradient kernel as a single segment."""
    x2, g2 = x.reshape(-1, x.shape[-1]).contiguous(), g.reshape(-1, g.shape[-1]).contiguous()
    if g2.dtype != torch.float32:
        x2 = x2.to(g2.dtype)                                     # (autocast: the output is narrower than the input)
    m = x2.shape[0]
    full = _typed.typed_gemm_wgrad(x2, g2, _one_segment(m, x.device), m, 1) if m > 0 and g2.dtype == torch.float32 else None
    return full[0].t() if full is not None else g2.t() @ x2      # shapes and types that kernel does not take


def _bias_grad(g):
    """The sum of the rows of g, in fp32 in a fixed order (float64 rows: torch's sum, which over many blocks
    does not belong into a captured graph: it clears a buffer by a memory-set node)."""
    g = g.reshape(-1, g.shape[-1])
    return g.sum(dim=0) if g.dtype == torch.float64 else _ops.column_sum(g.float().contiguous())


def _mm(x, w_kn, bias=None, addend=None):
    """x @ w_kn + bias + addend: the typed GEMM as one segment where it takes the shapes
    (bias and addend go into its epilogue), the library GEMM otherwise."""
    out = _typed.dense_linear(x, w_kn, bias, addend)
    if out is not None:
        return out
    if addend is not None:
        out = torch.addmm(addend, x, w_kn)
        return out if bias is None else out.add_(bias)
    return torch.addmm(bias, x, w_kn) if bias is not None else x @ w_kn


def _mm_add_(out, x, w_kn):
    """out += x @ w_kn in place (out may be a leading slice of a larger tensor)."""
    if not _typed.dense_linear_add_(out, x, w_kn):
        out.addmm_(x, w_kn)


class SageLayerOP(torch.autograd.Function):
    """``MySageConv.forward`` on CUDA tensors as one autograd node: mean aggregation and
    ``lin_l`` in the cheaper order, plus the root term ``lin_r(x[:num_node])`` added by the
    GEMM in place.  The backward pass writes the input gradient once (the transposed
    aggregation fills every source row, the root term is added in place on the first
    rows) instead of autograd's zero-padded slice gradient and a full-size add."""

    @staticmethod
    def forward(ctx, x, w_l, b_l, w_r, ptr, idx, num_node):
        n = int(num_node) if int(num_node) != 0 else ptr.shape[0] - 1
        x = x.contiguous()
        mm_first = w_l.shape[1] > w_l.shape[0]
        if ctx.needs_input_grad[0] or mm_first:
            # only a layer whose backward will ask for the reversed graph announces itself: the
            # first layer of a batch with frozen input features does not, and the reversed graphs
            # of the others are then cut out of the largest layer that does need one
            _ops.note_layer(ptr, idx, n, x.shape[0])
        aggr = None
        if mm_first:
            out = _ops.spmm(ptr, idx, _mm(x, w_l.t(), b_l), n, mean=True)
            if w_r is not None:
                _mm_add_(out, x[:n], w_r.t())
        else:
            aggr = _ops.spmm(ptr, idx, x, n, mean=True)
            out = _mm(aggr, w_l.t(), b_l)
            if w_r is not None:
                out = _mm(x[:n], w_r.t(), None, out)
        ctx.n, ctx.mm_first = n, mm_first
        ctx.save_for_backward(x, w_l, w_r, ptr, idx, aggr)
        return out

    @staticmethod
    def backward(ctx, g):
        x, w_l, w_r, ptr, idx, aggr = ctx.saved_tensors
        n, n_src = ctx.n, x.shape[0]
        g = g.contiguous()
        need_x, need_wl, need_bl, need_wr = ctx.needs_input_grad[:4]
        gx = gw_l = gb_l = gw_r = None
        if need_x or ctx.mm_first:
            tg = _ops.transposed(ptr, idx, n, n_src)
            inv = _ops.inv_degree_transposed(tg, ptr, n)
        if ctx.mm_first:
            g_t = _ops.spmm(tg.ptr_t, tg.idx_t, g, n_src, val=inv)
            if need_wl:
                gw_l = _weight_grad(x, g_t)
            if need_bl:
                gb_l = _ops.column_sum(g_t)
            if need_x:
                gx = _mm(g_t, w_l)
        else:
            if need_wl:
                gw_l = _weight_grad(aggr, g)
            if need_bl:
                gb_l = _ops.column_sum(g)
            if need_x:
                gx = _ops.spmm(tg.ptr_t, tg.idx_t, _mm(g, w_l), n_src, val=inv)
        if w_r is not None:
            if need_wr:
                gw_r = _weight_grad(x[:n], g)
            if need_x:
                _mm_add_(gx[:n], g, w_r)
        return gx, gw_l, gb_l, gw_r, None, None, None


class LinearOP(torch.autograd.Function):
    """``F.linear(x, weight, bias) (+ addend)`` on the typed kernels as a single segment: the
    forward product and the input gradient on the split GEMM (bias and addend go into its
    epilogue instead of separate element-wise passes), the weight gradient g^T x -- one very
    long reduction axis (every node), a small output -- on the weight-gradient kernel.  The
    library GEMM serves the shapes those kernels do not take (few rows, wide K)."""

    @staticmethod
    def forward(ctx, x, weight, bias=None, addend=None):
        ctx.save_for_backward(x, weight)
        out = _typed.dense_linear(x, weight.t(), bias, addend)
        if out is not None:
            return out
        if addend is None:
            return F.linear(x, weight, bias)
        out = torch.addmm(addend, x, weight.t())
        return out if bias is None else out.add_(bias)

    @staticmethod
    def backward(ctx, g):
        x, weight = ctx.saved_tensors
        gx = gw = gb = None
        if ctx.needs_input_grad[0]:
            gx = _typed.dense_linear(g, weight) if g.dim() == 2 else None
            if gx is None:
                gx = g @ weight.to(g.dtype)
        if ctx.needs_input_grad[1]:
            gw = _weight_grad(x, g)
        if ctx.needs_input_grad[2]:
            gb = _bias_grad(g)                   # (autograd rounds to the parameters' types)
        grads = (gx, gw, gb, g)              # bias and addend are optional arguments of apply()
        return tuple(grads[i] if need else None for i, need in enumerate(ctx.needs_input_grad))


class PackedLinearOP(torch.autograd.Function):
    """``LinearOP`` whose input is kept for the backward pass in 8 bits (``pack_rows``) instead of as it
    is: a quarter of the memory of fp32 rows, half of bf16.  Output and input gradient are LinearOP's;
    the weight gradient is that of the rows the 8 bits stand for, multiplied from them directly, and
    the bias gradient comes out of the same pass over g (``packed_weight_grad``)."""

    @staticmethod
    def forward(ctx, x, weight, bias, addend, fmt):
        packed = pack_rows(x.reshape(-1, x.shape[-1]), fmt) if ctx.needs_input_grad[1] else None
        ctx.fmt, ctx.shape = fmt, x.shape
        ctx.save_for_backward(weight, *(() if packed is None else (packed.codes, packed.exps)))
        return _linear_product(x, weight, bias, addend)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        weight, codes, exps = (ctx.saved_tensors + (None, None))[:3]
        gx = gw = gb = None
        if ctx.needs_input_grad[0]:
            gx = _typed.dense_linear(g, weight) if g.dim() == 2 else None
            if gx is None:
                gx = g @ weight.to(g.dtype)          # (autocast: the output is narrower than the weight)
        if ctx.needs_input_grad[1]:
            packed = PackedRows(codes, exps, ctx.shape[-1], ctx.fmt)
            gw, gb = packed_weight_grad(packed, g.reshape(-1, g.shape[-1]), want_sums=True)
            gw, gb = gw[0].t(), gb[0] if ctx.needs_input_grad[2] else None      # (autograd rounds to the parameters' types)
        elif ctx.needs_input_grad[2]:
            gb = _bias_grad(g)
        return gx, gw, gb, g if ctx.needs_input_grad[3] else None, None


def _linear_product(x, weight, bias, addend):
    out = _typed.dense_linear(x, weight.t(), bias, addend)
    if out is not None:
        return out
    if addend is None:
        return F.linear(x, weight, bias)
    out = torch.addmm(addend, x, weight.t())
    return out if bias is None else out.add_(bias)


def linear(x, weight, bias=None, addend=None, checkpoint=None):
    """``F.linear(x, weight, bias)``, plus ``addend`` where given, for the conv layers; CUDA
    tensors take LinearOP (types other than float32 the library's products).  ``checkpoint`` "int8" or
    "e4m3": what the weight gradient needs of x is kept in 8 bits per value (PackedLinearOP; CUDA tensors,
    float32 / bfloat16 / float16)."""
    if check_format(checkpoint) is not None and x.is_cuda and torch.is_grad_enabled():     # else nothing is kept
        if addend is not None and x.dim() != 2:
            raise ValueError("an addend goes with x [N, C]")
        rows, (n, k) = x.numel() // max(1, x.shape[-1]), weight.shape
        if not (_typed.dense_linear_shape(rows, k, n, bias is None and addend is None)
                or _typed.dense_linear_shape(rows, n, k, True)):
            return _ops._C.packed_linear(x, weight, bias, addend, FORMATS[checkpoint])     # library products: the compiled node
        return PackedLinearOP.apply(x, weight, bias, addend, checkpoint)
    if not x.is_cuda or (addend is not None and x.dim() != 2):
        out = F.linear(x, weight, bias)
        return out if addend is None else addend + out
    return LinearOP.apply(x, weight, bias, addend)


class AttentionLogitsOP(torch.autograd.Function):
    """Both per-node logits of a GAT layer, ``(x * att_src).sum(-1)`` over every source node
    and ``(x[:num_dst] * att_dst).sum(-1)`` (cxgnncomp/graph_conv.py:466-467), from one
    pass over x; the backward pass reads x once more for grad_x and both parameter
    gradients.  Host tensors use the upstream expressions."""

    @staticmethod
    def forward(ctx, x, att_src, att_dst, num_dst):
        ctx.save_for_backward(x, att_src, att_dst)
        ctx.num_dst = num_dst
        if not x.is_cuda:
            return (x * att_src).sum(dim=-1), (x[:num_dst] * att_dst).sum(dim=-1)
        return cxgnncomp_backend._ops.attention_logits(x.contiguous(), att_src, att_dst, num_dst)

    @staticmethod
    def backward(ctx, g_src, g_dst):
        x, att_src, att_dst = ctx.saved_tensors
        if not x.is_cuda:
            gx = g_src.unsqueeze(-1) * att_src
            gx[:ctx.num_dst] += g_dst.unsqueeze(-1) * att_dst
            ga_src = (g_src.unsqueeze(-1) * x).sum(dim=0).view_as(att_src)
            ga_dst = (g_dst.unsqueeze(-1) * x[:ctx.num_dst]).sum(dim=0).view_as(att_dst)
            return gx, ga_src, ga_dst, None
        gx, ga_src, ga_dst = cxgnncomp_backend._ops.attention_logits_bwd(
            x.contiguous(), att_src, att_dst, g_src.contiguous(), g_dst.contiguous())
        return gx, ga_src.view_as(att_src), ga_dst.view_as(att_dst), None


class GatLayerOP(torch.autograd.Function):
    """``MyGATConv.forward_many`` (several heads) on CUDA tensors as one autograd node: linear
    map, both attention logits, fused edge softmax, edge-weighted aggregation, head
    concatenation or mean, bias.  The backward pass runs the same kernels as the separate
    nodes do, but the two gradients of the transformed features -- from the aggregation
    and from the logits -- meet in one buffer (the logits kernel adds into what the
    transposed aggregation wrote) instead of two tensors and a full-size add, and the
    intermediate views cost no copies.  Where the input is narrower than the transformed
    features (and the kernels take the shape) the logits are read off the input instead,
    ``x @ m.T`` with ``m = att @ W`` per head -- the contraction order of the single-head
    path's einsum (upstream cxgnncomp/graph_conv.py:500-511); their backward pass then adds a
    rank-2H term to the input gradient and returns grad m, from which the shares of the weight
    and attention-vector gradients follow by the chain rule on [2H, in] tensors.  Where the input
    has at most half the columns of the transformed features and the rows have eight edges or
    more on average, the forward aggregation gathers input rows under the H edge weights
    (``sum_e ev[e, h] x[idx[e]]``, [num_dst, H, in]) and transforms per head afterwards -- the
    order "aggregate, then transform" that upstream's single-head path takes when
    in < out (cxgnncomp/graph_conv.py:523-542); the transformed features are then formed in the
    backward pass only, which needs them for the edge-value gradient."""

    @staticmethod
    def _logit_rows(w, att_src, att_dst, H, C):
        w3 = w.view(H, C, -1)
        return torch.cat([torch.bmm(att_src.reshape(H, 1, C), w3), torch.bmm(att_dst.reshape(H, 1, C), w3)]).squeeze(1)

    @staticmethod
    def forward(ctx, x, w, att_src, att_dst, bias, ptr, idx, num_dst, num_src, num_edge, slope, heads, concat):
        H, C = heads, w.shape[0] // heads
        n_in = x.shape[1]
        from_input = (n_in < H * C and _ops.logits_proj_supported(n_in, H) and x.stride(1) == 1
                      and x.stride(0) % 4 == 0 and x.data_ptr() % 16 == 0)
        # aggregate the input rows under the H edge weights, then transform per head: half the gathered
        # bytes or less; pays from about eight edges per destination row on
        aggr_first = (from_input and 2 * n_in <= H * C and _ops.spmm_heads_supported(H, n_in)
                      and num_edge >= 8 * num_dst)
        # one head and a narrower input: the whole layer is "aggregate the input rows, then transform"
        # (the branch upstream's forward_1 takes), forward and backward on rows of `in` floats
        single_first = from_input and H == 1 and x.is_contiguous()
        xs = None if (aggr_first or single_first) else _mm(x[:num_src], w.t()).view(-1, H, C)
        if from_input:
            a_src, a_dst = _ops.attention_logits_proj(x[:num_src], GatLayerOP._logit_rows(w, att_src, att_dst, H, C),
                                                      num_dst, H)
        else:
            a_src, a_dst = _ops.attention_logits(xs, att_src, att_dst, num_dst)
        ev, mask = _ops.edge_softmax_fwd(ptr, idx, a_dst, a_src, num_edge, slope)
        aggr = None
        if single_first:
            aggr = _ops.spmm(ptr, idx, x[:num_src], num_dst, val=ev.view(-1))
            out = _mm(aggr, w.t(), bias)
        elif aggr_first:
            aggr = _ops.spmm_weighted_heads(ptr, idx, ev, x[:num_src], num_dst)
            if concat:
                out = _typed.dense_linear_heads(aggr, w, bias)
            else:
                # mean over heads of aggr[:, h] @ W_h^T = one product over K = H * in
                out = _mm(aggr.view(-1, H * n_in), w.view(H, C, n_in).transpose(1, 2).reshape(H * n_in, C)).div_(H)
                if bias is not None:
                    out.add_(bias)
            aggr = None
        elif concat:
            # the bias goes into the aggregation's row stores
            out = _ops.spmm(ptr, idx, xs, num_dst, val=ev, bias=bias).view(-1, H * C)
        else:
            out = _ops.spmm(ptr, idx, xs, num_dst, val=ev).mean(dim=1)
            if bias is not None:
                out.add_(bias)
        ctx.save_for_backward(x, w, att_src, att_dst, xs, ev, mask, ptr, idx, aggr)
        ctx.dims = (num_dst, num_src, H, C, concat, float(slope), bias is not None, from_input)
        return out

    @staticmethod
    def _backward_single_first(ctx, g, x, w, att_src, att_dst, ev, mask, ptr, idx, aggr):
        """One head, input narrower than the output: out = (sum_e ev x[src]) W^T + bias.  The
        gradient rows g W have `in` columns; they are what the pass over the reversed graph
        aggregates, and their products with the source rows of x are the edge-value gradient."""
        num_dst, num_src, H, C, concat, slope, has_bias, from_input = ctx.dims
        g_bias = _ops.column_sum(g) if has_bias and ctx.needs_input_grad[4] else None
        g_w = _weight_grad(aggr, g) if ctx.needs_input_grad[1] else None
        gw_rows = _mm(g, w)                                       # [num_dst, in]
        xs_rows = x[:num_src]
        n_in = x.shape[1]
        tg = _ops.transposed(ptr, idx, num_dst, num_src)
        g_ev = torch.empty((ev.shape[0], 1), dtype=torch.float32, device=g.device)
        if tg.n_edges < ev.shape[0]:
            g_ev[tg.n_edges:].zero_()
        # (rows under 96 floats: reading the products back through positions costs what the fused pass saves)
        if n_in >= 96 and _ops.spmm_dot_supported(1, n_in, at_edge=True):
            g_x, g_ev = _ops.spmm_dot(tg.ptr_t, tg.idx_t, gw_rows.view(-1, 1, n_in), num_src, ev, tg.perm,
                                      xs_rows.view(-1, 1, n_in), g_ev, dot_at_edge=True)
            g_x = g_x.view(-1, n_in)
            g_adst, t_edge = _ops.edge_softmax_bwd(ptr, ev, mask, g_ev, num_dst, slope,
                                                   grad_pos=_ops.inverse_perm_transposed(tg))
        else:
            g_x = _ops.spmm(tg.ptr_t, tg.idx_t, gw_rows, num_src, val=ev.view(-1), val_perm=tg.perm)
            g_ev = _ops.sddmm_csr(ptr, idx, xs_rows.view(-1, 1, n_in), gw_rows.view(-1, 1, n_in), num_dst, out=g_ev)
            g_adst, t_edge = _ops.edge_softmax_bwd(ptr, ev, mask, g_ev, num_dst, slope)
        g_asrc = _ops.narrow_gather_sum(tg.ptr_t, tg.perm, t_edge, num_src, rows32=_ops.rows32_transposed(tg))
        m = GatLayerOP._logit_rows(w, att_src, att_dst, 1, C)
        need_x = ctx.needs_input_grad[0]
        _, g_m = _ops.attention_logits_proj_bwd(xs_rows, m, g_asrc, g_adst, 1, add_to=g_x if need_x else None,
                                                need_x=False)
        g_att_src, g_att_dst = g_m[0:1] @ w.t(), g_m[1:2] @ w.t()           # [1, C]
        if g_w is not None:
            g_w.addmm_(att_src.reshape(C, 1), g_m[0:1]).addmm_(att_dst.reshape(C, 1), g_m[1:2])
        if not need_x:
            g_x = None
        elif g_x.shape[0] < x.shape[0]:
            g_x = torch.cat([g_x, g_x.new_zeros(x.shape[0] - g_x.shape[0], n_in)])
        return (g_x, g_w, g_att_src.view_as(att_src), g_att_dst.view_as(att_dst), g_bias,
                None, None, None, None, None, None, None, None)

    @staticmethod
    def backward(ctx, g):
        x, w, att_src, att_dst, xs, ev, mask, ptr, idx, aggr = ctx.saved_tensors
        num_dst, num_src, H, C, concat, slope, has_bias, from_input = ctx.dims
        g = g.contiguous()
        if aggr is not None:
            return GatLayerOP._backward_single_first(ctx, g, x, w, att_src, att_dst, ev, mask, ptr, idx, aggr)
        if xs is None:                       # the forward pass aggregated the input rows and never formed them
            xs = _mm(x[:num_src], w.t()).view(-1, H, C)
        g_bias = _ops.column_sum(g) if has_bias and ctx.needs_input_grad[4] else None
        if concat:
            g3 = g.view(-1, H, C)
        else:
            g3 = (g / H).unsqueeze(1).expand(-1, H, -1).contiguous()
        tg = _ops.transposed(ptr, idx, num_dst, xs.shape[0])
        g_ev = torch.empty((ev.shape[0], H), dtype=torch.float32, device=g.device)
        if tg.n_edges < ev.shape[0]:
            g_ev[tg.n_edges:].zero_()
        if H * C >= 96 and _ops.spmm_dot_supported(H, C, at_edge=True):
            # one pass over the reversed graph gathers the rows of g once for both results; the
            # edge-value gradient stays in that pass's edge order (contiguous stores) and the
            # softmax backward reads it through the inverse permutation
            g_xs, g_ev = _ops.spmm_dot(tg.ptr_t, tg.idx_t, g3, xs.shape[0], ev, tg.perm, xs, g_ev, dot_at_edge=True)
            g_adst, t_edge = _ops.edge_softmax_bwd(ptr, ev, mask, g_ev, num_dst, slope,
                                                   grad_pos=_ops.inverse_perm_transposed(tg))
        else:
            g_xs = _ops.spmm(tg.ptr_t, tg.idx_t, g3, xs.shape[0], val=ev, val_perm=tg.perm)
            g_ev = _ops.sddmm_csr(ptr, idx, xs, g3, num_dst, out=g_ev)
            g_adst, t_edge = _ops.edge_softmax_bwd(ptr, ev, mask, g_ev, num_dst, slope)
        g_asrc = _ops.narrow_gather_sum(tg.ptr_t, tg.perm, t_edge, xs.shape[0], rows32=_ops.rows32_transposed(tg))
        if not from_input:
            _, g_att_src, g_att_dst = _ops.attention_logits_bwd(xs, att_src, att_dst, g_asrc, g_adst, add_to=g_xs)
        g_xs2 = g_xs.view(-1, H * C)
        g_x = g_w = None
        if ctx.needs_input_grad[0]:
            g_x = _mm(g_xs2, w)
        if ctx.needs_input_grad[1]:
            g_w = _weight_grad(x[:num_src], g_xs2)
        if from_input:
            # the logits' share: rank 2H into g_x, and through m = att @ W into g_w and g_att
            m = GatLayerOP._logit_rows(w, att_src, att_dst, H, C)
            _, g_m = _ops.attention_logits_proj_bwd(x[:num_src], m, g_asrc, g_adst, H, add_to=g_x, need_x=False)
            g_m = g_m.view(2, H, 1, -1)
            w3t = w.view(H, C, -1).transpose(1, 2)
            g_att_src, g_att_dst = torch.bmm(g_m[0], w3t), torch.bmm(g_m[1], w3t)
            if g_w is not None:
                g_w3 = g_w.view(H, C, -1)
                g_w3.baddbmm_(att_src.reshape(H, C, 1), g_m[0])
                g_w3.baddbmm_(att_dst.reshape(H, C, 1), g_m[1])
        if g_x is not None and g_x.shape[0] < x.shape[0]:
            g_x = torch.cat([g_x, g_x.new_zeros(x.shape[0] - g_x.shape[0], g_x.shape[1])])
        return (g_x, g_w, g_att_src.view_as(att_src), g_att_dst.view_as(att_dst), g_bias,
                None, None, None, None, None, None, None, None)


class MyGATConv(torch.nn.Module):

    def __init__(self, in_channels, out_channels, heads=1, concat=False, negative_slope=0.2,
                 dropout=0.0, bias=True, layer=-1):
        super().__init__()
        assert heads > 0
        self.in_channels = in_channels
        self.out_channels = out_channels
        self.heads = heads
        self.concat = concat
        self.negative_slope = negative_slope
        self.dropout = dropout
        self.layer = layer
        self.lin_src = Parameter(torch.Tensor(heads * out_channels, in_channels))
        self.att_src = Parameter(torch.Tensor(1, heads, out_channels))
        self.att_dst = Parameter(torch.Tensor(1, heads, out_channels))
        if bias:
            self.bias = Parameter(torch.Tensor(heads * out_channels if concat else out_channels))
        else:
            self.bias = None
        self.edge_softmax_schedule = "fused"
        self.reset_parameters()

    def reset_parameters(self):
        glorot(self.lin_src)
        glorot(self.att_src)
        glorot(self.att_dst)
        if self.bias is not None:
            self.bias.data.fill_(0)

    def edge_softmax_fused(self, ptr, idx, att_src, att_dst, num_edge, relu_l):
        return edge_attention(ptr=ptr, idx=idx, att_src=att_src, att_dst=att_dst, num_edge=num_edge,
                              relu_l=relu_l)

    def edge_softmax_opwise(self, ptr, idx, att_src, att_dst, num_edge, relu_l):
        """Op-by-op softmax over each destination's edges (upstream :437-448, there with
        torch_scatter's segment_csr / gather_csr)."""
        n = ptr.shape[0] - 1
        seg = torch.repeat_interleave(torch.arange(n, device=ptr.device), ptr[1:] - ptr[:-1])[:num_edge]
        alpha = F.leaky_relu(att_src.index_select(0, idx[:num_edge]) + att_dst[seg], relu_l)
        segh = seg.unsqueeze(1).expand(-1, alpha.shape[1])
        with torch.no_grad():
            amax = torch.full((n, alpha.shape[1]), -float("inf"), dtype=alpha.dtype, device=alpha.device)
            amax = amax.scatter_reduce(0, segh, alpha, "amax", include_self=True)[seg]
        alpha = torch.exp(alpha - amax)
        total = torch.zeros((n, alpha.shape[1]), dtype=alpha.dtype, device=alpha.device)
        total = total.index_add(0, seg, alpha) + 1e-16
        return alpha / total[seg]

    def edge_softmax(self, ptr, idx, att_src, att_dst, num_edge, relu_l):
        if self.edge_softmax_schedule == "fused":
            return self.edge_softmax_fused(ptr, idx, att_src, att_dst, num_edge, relu_l)
        return self.edge_softmax_opwise(ptr, idx, att_src, att_dst, num_edge, relu_l)

    def forward_many(self, x, ptr, idx, num_dst, num_src, num_edge):
        H, C = self.heads, self.out_channels
        assert x.dim() == 2
        if x.is_cuda and self.edge_softmax_schedule == "fused" and C % 4 == 0:
            x = TimerOP.apply(x, "gat layer", True)
            out = GatLayerOP.apply(x, self.lin_src, self.att_src, self.att_dst, self.bias, ptr, idx, int(num_dst),
                                   int(num_src), int(num_edge), self.negative_slope, H, self.concat)
            return TimerOP.apply(out, "gat layer", False)
        x = TimerOP.apply(x, "linear1", True)
        x_src = x_dst = linear(x[:num_src], self.lin_src).view(-1, H, C)
        x_src = TimerOP.apply(x_src, "linear1", False)
        x_src = TimerOP.apply(x_src, "sum1", True)
        alpha_src, alpha_dst = AttentionLogitsOP.apply(x_src, self.att_src, self.att_dst, num_dst)
        alpha_dst = TimerOP.apply(alpha_dst, "sum1", False)
        alpha_dst = TimerOP.apply(alpha_dst, "softmax1", True)
        edge_value = self.edge_softmax(ptr=ptr, idx=idx, att_src=alpha_src, att_dst=alpha_dst,
                                       num_edge=num_edge, relu_l=self.negative_slope)
        edge_value = TimerOP.apply(edge_value, "softmax1", False)
        edge_value = TimerOP.apply(edge_value, "aggregation", True)
        if self.heads == 1:
            out = sage_sum_forward_edge_value(x_src, ptr, idx, edge_value.squeeze(), num_dst)
        else:
            out = SpMMValOP.apply(x_src, ptr, idx, edge_value, num_dst)
        out = TimerOP.apply(out, "aggregation", False)
        if self.concat:
            out = out.view(-1, H * C)
        elif out.shape[1] == self.heads:
            out = out.mean(dim=1)
        return out + self.bias if self.bias is not None else out

    def forward_1(self, x, ptr, idx, num_dst, num_src, num_edge):
        if x.is_cuda and x.dim() == 2 and self.edge_softmax_schedule == "fused" and self.out_channels % 4 == 0:
            # the same layer node as several heads take; it picks the order of aggregation and
            # transform by the widths, as the expressions below do
            x = TimerOP.apply(x, "gat layer", True)
            out = GatLayerOP.apply(x, self.lin_src, self.att_src, self.att_dst, self.bias, ptr, idx, int(num_dst),
                                   int(num_src), int(num_edge), self.negative_slope, 1, True)
            return TimerOP.apply(out, "gat layer", False)
        w = self.lin_src.T.view(-1, self.heads, self.out_channels)
        x = TimerOP.apply(x, "einsum1", True)
        alpha_src = torch.einsum("mn,nho,ho->mh", x, w, self.att_src.squeeze(0)).view(-1, self.heads)
        alpha_dst = torch.einsum("mn,nho,ho->mh", x[:num_dst], w, self.att_dst.squeeze(0)).view(-1, self.heads)
        alpha_dst = TimerOP.apply(alpha_dst, "einsum1", False)
        alpha_dst = TimerOP.apply(alpha_dst, "softmax1", True)
        edge_value = self.edge_softmax(ptr=ptr, idx=idx, att_src=alpha_src, att_dst=alpha_dst,
                                       num_edge=num_edge, relu_l=self.negative_slope)
        edge_value = TimerOP.apply(edge_value, "softmax1", False)
        if self.out_channels < self.in_channels:
            x = TimerOP.apply(x, "mm1", True)
            t = torch.mm(x, self.lin_src.T).view(-1, self.heads, self.out_channels)
            t = TimerOP.apply(t, "mm1", False)
            t = TimerOP.apply(t, "aggregation", True)
            x = sage_sum_forward_edge_value(t, ptr, idx, edge_value, num_dst).squeeze()
            x = TimerOP.apply(x, "aggregation", False)
        else:
            x = TimerOP.apply(x, "aggregation", True)
            x = sage_sum_forward_edge_value(x, ptr, idx, edge_value.squeeze(), num_dst)
            x = TimerOP.apply(x, "aggregation", False)
            x = TimerOP.apply(x, "mm1", True)
            x = torch.mm(x, self.lin_src.T)
            x = TimerOP.apply(x, "mm1", False)
        return x + self.bias if self.bias is not None else x

    def forward(self, x, ptr, idx, num_dst, num_src, num_edge):
        ptr = ptr[:num_dst + 1]
        idx = idx[:num_edge]
        if self.heads == 1:
            return self.forward_1(x, ptr, idx, num_dst, num_src, num_edge)
        return self.forward_many(x, ptr, idx, num_dst, num_src, num_edge)


class MyGCNConv(torch.nn.Module):

    checkpoint = None                 # (modules saved before there was one)

    def __init__(self, in_channels, out_channels, normalize=False, bias=True, checkpoint=None):
        """``checkpoint`` (not upstream) "int8" or "e4m3": the input of the layer's linear map is kept for
        the backward pass in 8 bits per value (``linear``)."""
        super().__init__()
        self.checkpoint = check_format(checkpoint)
        self.in_channels = in_channels
        self.out_channels = out_channels
        self.normalize = normalize
        self.lin = torch.nn.Linear(in_channels, out_channels, bias=False)
        self.bias = torch.nn.Parameter(torch.Tensor(out_channels)) if bias else None
        self.reset_parameters()

    def reset_parameters(self):
        glorot(self.lin.weight)
        if self.bias is not None:
            self.bias.data.fill_(0)

    def gcn_norm(self, ptr, idx):
        """1 / in-degree per edge, 0 where the degree is 0 (upstream :587-596)."""
        if ptr.is_cuda:
            return cxgnncomp_backend.edge_value_degree(ptr, ptr.shape[0] - 1, idx.shape[0])
        deg = ptr[1:] - ptr[:-1]
        edge_value = deg.repeat_interleave(deg).float().pow(-1)
        edge_value.masked_fill_(edge_value == float("inf"), 0.0)
        return edge_value

    def forward(self, x, ptr, idx, num_node):
        x = TimerOP.apply(x, "linear", True)
        mm_before = self.in_channels > self.out_channels
        out = linear(x, self.lin.weight, checkpoint=self.checkpoint) if mm_before else x
        out = TimerOP.apply(out, "linear", False)
        if self.normalize:
            out = TimerOP.apply(out, "aggregation", True)
            TimerOP.apply(out, "gcn norm", True)
            edge_value = self.gcn_norm(ptr, idx)
            TimerOP.apply(edge_value, "gcn norm", False)
            out = sage_sum_forward_edge_value(out, ptr, idx, edge_value, num_node)
            out = TimerOP.apply(out, "aggregation", False)
        else:
            out = AggrOP.apply(out, ptr, idx, num_node)
        if not mm_before:
            return linear(out, self.lin.weight, self.bias, checkpoint=self.checkpoint)
        return out + self.bias if self.bias is not None else out
