"""Residual stacks and layers that keep their inputs in 8 bits: ``linear(checkpoint=)``,
``TypedLinearE2EOP(checkpoint=)``, the conv layers and ``GNN(residual=, checkpoint=)``, and the operators
behind them used together."""
import copy

import pytest
import torch
import torch.nn.functional as F

import packed_ref
import residual_ref
from conftest import announce
from oracle import pyref
from rounding import check

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _saved_bytes(fn):
    """Result of fn() and the bytes its autograd graph holds, each storage once."""
    held = {}

    def pack(t):
        held[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        out = fn()
    return out, sum(held.values())


# ----------------------------------------- on the CPU ------------------------------------------- #
def test_options_are_checked():
    import cxgnncomp
    lin = torch.nn.Linear(4, 3)
    x = torch.randn(5, 4)
    assert torch.equal(cxgnncomp.linear(x, lin.weight, lin.bias), F.linear(x, lin.weight, lin.bias))
    assert torch.equal(cxgnncomp.linear(x, lin.weight, lin.bias, checkpoint="int8"), F.linear(x, lin.weight, lin.bias))
    with pytest.raises(ValueError):
        cxgnncomp.linear(x, lin.weight, checkpoint="int4")
    for conv in (cxgnncomp.MySageConv, cxgnncomp.MyGCNConv, cxgnncomp.MyGINConv):
        assert conv(4, 3).checkpoint is None and conv(4, 3, checkpoint="e4m3").checkpoint == "e4m3"
        with pytest.raises(ValueError):
            conv(4, 3, checkpoint="fp8")
    with pytest.raises(ValueError):
        cxgnncomp.SAGE(4, 8, 3, 2, 0.0, "CSR", residual="batch")
    with pytest.raises(ValueError):
        cxgnncomp.GAT(4, 8, 3, 2, 0.0, "CSR_Layer", checkpoint="int8", heads=1)
    with pytest.raises(ValueError):
        cxgnncomp.RGCN(4, 8, 3, 2, 0.0, "CSR", checkpoint="int8", num_rel=2)
    plain = cxgnncomp.SAGE(4, 8, 3, 4, 0.0, "CSR")
    assert len(plain.bns) == 3 and not any("norm" in k for k in plain.state_dict())
    deep = cxgnncomp.get_model_from_str("gcn", 4, 8, 3, "CSR", 4, residual="rms", checkpoint="int8")
    assert len(deep.bns) == 0 and len(deep.norms) == 3 and all(c.checkpoint == "int8" for c in deep.convs)
    assert sorted(k for k in deep.state_dict() if k.startswith("norms.0")) == ["norms.0.pre_weight"]
    assert sorted(k for k in deep.state_dict() if k.startswith("norms.2")) == ["norms.2.gate", "norms.2.post_weight",
                                                                              "norms.2.pre_weight"]
    deep.reset_parameters()


# ------------------------------------------ on the GPU ------------------------------------------- #
@gpu
@pytest.mark.parametrize("m,k,n", [(1, 5, 3), (300, 100, 47), (5000, 128, 64), (4097, 47, 256)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("extra", ["plain", "bias", "addend"])
def test_linear_that_keeps_its_input_in_8_bits(m, k, n, fmt, extra):
    """Output, input and addend gradients are those of linear without checkpoint, bit for bit; the weight
    gradient is that of the rows as the 8 bits hold them, the bias gradient the sum of g's rows."""
    import cxgnncomp
    torch.manual_seed(m)
    x, w, g = torch.randn(m, k), torch.randn(n, k) / k ** 0.5, torch.randn(m, n)
    b = torch.randn(n) if extra != "plain" else None
    add = torch.randn(m, n) if extra == "addend" else None
    announce("linear checkpoint %d x %d x %d %s %s" % (m, k, n, fmt, extra))

    def run(checkpoint):
        t = [None if v is None else v.cuda().requires_grad_(True) for v in (x, w, b, add)]
        out = cxgnncomp.linear(*t, checkpoint=checkpoint)
        return [out] + [None if v is None else d for v, d in zip(t, _grads(out, t, g.cuda()))]

    got, plain = run(fmt), run(None)
    for i in (0, 1, 4):
        assert (got[i] is None) == (plain[i] is None) and (got[i] is None or torch.equal(got[i], plain[i])), i
    codes, exps, values = packed_ref.pack(x, fmt)
    want = packed_ref.weight_grad(values, g, [0, m])
    want.v, want.e = want.v[0].t(), want.e[0].t()
    check(got[2], want, F32, "weight gradient")
    if b is not None:
        check(got[3], packed_ref.row_sums(g, [0, m])[0], F32, "bias gradient")


def _grads(out, tensors, g):
    live = [t for t in tensors if t is not None]
    found = dict(zip(map(id, live), torch.autograd.grad(out, live, g)))
    return [None if t is None else found[id(t)] for t in tensors]


@gpu
def test_linear_in_bf16_and_with_frozen_weights():
    import cxgnncomp
    torch.manual_seed(2)
    x, w, g = torch.randn(700, 96).to(BF16), torch.randn(40, 96).to(BF16), torch.randn(700, 40).to(BF16)
    b = torch.randn(40).to(BF16)
    announce("linear checkpoint bf16")
    xc, wc, bc = (t.cuda().requires_grad_(True) for t in (x, w, b))
    (out, held), (_, held_plain) = (_saved_bytes(lambda c=c: cxgnncomp.linear(xc, wc, bc, checkpoint=c)) for c in ("int8", None))
    assert held == held_plain - 700 * 96 * 2 + 700 * 97
    gx, gw, gb = torch.autograd.grad(out, (xc, wc, bc), g.cuda())
    want = packed_ref.weight_grad(packed_ref.pack(x, "int8")[2], g, [0, 700])
    want.v, want.e = want.v[0].t(), want.e[0].t()
    check(gw, want, BF16, "weight gradient")
    check(gb, packed_ref.row_sums(g, [0, 700])[0], BF16, "bias gradient")
    assert torch.equal(gx, g.cuda() @ wc)
    out, held = _saved_bytes(lambda: cxgnncomp.linear(xc, wc.detach(), bc, checkpoint="int8"))
    assert held == 40 * 96 * 2                           # nothing of x where the weight is frozen
    assert torch.equal(torch.autograd.grad(out, xc, g.cuda())[0], gx)
    x3 = xc.detach().view(7, 100, 96).requires_grad_(True)
    out3 = cxgnncomp.linear(x3, wc, bc, checkpoint="int8")
    gx3, gw3 = torch.autograd.grad(out3, (x3, wc), g.cuda().view(7, 100, 40))
    assert torch.equal(gw3, gw) and gx3.shape == x3.shape


@gpu
def test_typed_linear_checkpoint_refuses_second_derivatives():
    import cxgnncomp
    x = torch.randn(90, 64, device="cuda", requires_grad=True)
    w, types = torch.randn(3, 64, 32, device="cuda", requires_grad=True), torch.randint(0, 3, (90, ), device="cuda")
    announce("TypedLinearE2EOP checkpoint create_graph")
    out = cxgnncomp.TypedLinearE2EOP.apply(x, w, types, [], 256, None, "int8")
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(out.sum(), (x, w), create_graph=True)
    out = cxgnncomp.TypedLinearE2EOP.apply(x, w, types, [], 256, None, "int8")
    assert torch.autograd.grad(out.sum(), w)[0].shape == w.shape


@gpu
def test_nothing_is_packed_where_no_backward_pass_follows(monkeypatch):
    """Without gradients (serving) a layer's input is not packed; bad formats are refused all the same."""
    import cxgnncomp
    from cxgnncomp import graph_conv, typed_linear
    from cxgnncomp_backend import _ops

    class NoPacking:
        def __getattr__(self, name):
            assert name not in ("pack_rows", "packed_linear")
            return getattr(_native, name)

    def no_packing(*a):
        raise AssertionError("packed")

    _native = _ops._C
    monkeypatch.setattr(graph_conv, "pack_rows", no_packing)
    monkeypatch.setattr(typed_linear, "pack_rows", no_packing)
    monkeypatch.setattr(_ops, "_C", NoPacking())
    x, w = torch.randn(5000, 64, device="cuda"), torch.randn(32, 64, device="cuda", requires_grad=True)
    w3, types = torch.randn(3, 64, 32, device="cuda", requires_grad=True), torch.randint(0, 3, (5000, ), device="cuda")
    announce("linear checkpoint without gradients")
    with torch.no_grad():
        assert torch.equal(cxgnncomp.linear(x, w, checkpoint="int8"), cxgnncomp.linear(x, w))
        assert torch.equal(cxgnncomp.linear(x[:9], w, checkpoint="int8"), cxgnncomp.linear(x[:9], w))
        a = cxgnncomp.TypedLinearE2EOP.apply(x, w3, types, [], 256, None, "int8")
        assert torch.equal(a, cxgnncomp.TypedLinearE2EOP.apply(x, w3, types))
        with pytest.raises(ValueError):
            cxgnncomp.TypedLinearE2EOP.apply(x, w3, types, [], 256, None, "int4")
    with pytest.raises(AssertionError):
        cxgnncomp.linear(x, w, checkpoint="int8")


@gpu
@pytest.mark.parametrize("m", [300, 5000])
def test_linear_under_autocast_and_without_rows(m):
    import cxgnncomp
    torch.manual_seed(4)
    x, w, b = (torch.randn(s, device="cuda").requires_grad_(True) for s in ((m, 90), (33, 90), (33, )))
    announce("linear checkpoint under autocast")
    with torch.autocast("cuda", dtype=BF16):
        out = cxgnncomp.linear(x, w, b, checkpoint="int8")
    assert out.dtype == BF16
    g = torch.randn(m, 33, device="cuda").to(BF16)
    gx, gw, gb = torch.autograd.grad(out, (x, w, b), g)
    assert gx.dtype == gw.dtype == gb.dtype == F32
    want = packed_ref.weight_grad(packed_ref.pack(x.detach().cpu(), "int8")[2], g.cpu(), [0, m])
    want.v, want.e = want.v[0].t(), want.e[0].t()
    check(gw, want, F32, "weight gradient")
    empty = cxgnncomp.linear(x[:0], w, b, checkpoint="int8")
    gw, gb = torch.autograd.grad(empty.sum(), (w, b))
    assert tuple(empty.shape) == (0, 33) and not gw.any() and not gb.any()


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_typed_linear_that_keeps_its_rows_in_8_bits(fmt):
    import cxgnncomp
    torch.manual_seed(3)
    m, k, n, r = 3000, 64, 96, 7                         # the typed product takes multiples of 32
    x, w, g = torch.randn(m, k), torch.randn(r, k, n) / 8, torch.randn(m, n)
    types = torch.randint(0, r - 1, (m, ))               # the last relation has no rows
    announce("typed linear checkpoint %s" % fmt)

    def run(checkpoint):
        xc, wc = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
        out, held = _saved_bytes(lambda: cxgnncomp.TypedLinearE2EOP.apply(xc, wc, types.cuda(), [], 256, None, checkpoint))
        return (out, held) + torch.autograd.grad(out, (xc, wc), g.cuda())

    out, held, gx, gw = run(fmt)
    out0, held0, gx0, gw0 = run(None)
    assert torch.equal(out, out0) and torch.equal(gx, gx0)
    assert held == held0 - 4 * m * k + m * (k + 1)
    values = packed_ref.pack(x, fmt)[2]
    perm = torch.sort(types, stable=True)[1]
    bounds = [0] + torch.bincount(types, minlength=r).cumsum(0).tolist()
    check(gw, packed_ref.weight_grad(values, g, bounds, perm, perm), F32, "weight gradient")
    assert not gw[r - 1].any()


@pytest.fixture(autouse=True)
def _timers():
    import cxgnncomp
    cxgnncomp.set_timers()            # the conv layers need them


def _graph(n=900, edges=5000, seed=0):
    from cxgnncomp import synthetic as S
    return S.uniform_graph(n, edges, seed=seed)


@gpu
@pytest.mark.parametrize("kind", ["MyGCNConv", "MyGINConv", "MySageConv"])
@pytest.mark.parametrize("widths", [(40, 64), (64, 24)])
def test_conv_layers_that_keep_inputs_in_8_bits(kind, widths):
    """Same output and input gradient as without; weight gradients from the rows that the 8 bits hold: the
    distance to the gradient from the exact rows is that of the rows (|x8 - x| <= max / 127 a group)."""
    import cxgnncomp
    ptr, idx = _graph()
    n = ptr.shape[0] - 1
    torch.manual_seed(5)
    conv = getattr(cxgnncomp, kind)(*widths).cuda()
    packed = getattr(cxgnncomp, kind)(*widths, checkpoint="int8").cuda()
    packed.load_state_dict(conv.state_dict())
    x, g = torch.randn(n, widths[0]), torch.randn(n, widths[1]).cuda()
    announce("%s %s checkpoint" % (kind, widths))
    res = []
    for layer in (conv, packed):
        xc = x.cuda().requires_grad_(True)
        out = layer(xc, ptr.cuda(), idx.cuda(), n)
        params = list(layer.parameters())
        res.append([out] + list(torch.autograd.grad(out, [xc] + params, g)))
    names = ["out", "x"] + [k for k, _ in conv.named_parameters()]
    for name, a, b in zip(names, *res):
        a, b = a.detach(), b.detach()
        scale = float(a.abs().max())
        if name.endswith("weight"):
            # columns of x differ by at most max / 127 of their group: the gradient by that times sum |g|
            assert float((a - b).abs().max()) <= float(g.abs().sum(0).max()) * 60 / 127 and not torch.equal(a, b)
            assert float((a - b).norm() / a.norm()) < 0.02
        else:
            assert float((a - b).abs().max()) <= 2e-5 * scale, name


@gpu
@pytest.mark.parametrize("residual", ["layer", "rms"])
def test_residual_gcn_against_float64(residual):
    """Logits, input and parameter gradients of a four-layer residual GCN against the same stack written out
    in float64 (tolerance 2e-4 of the largest value: the aggregation and GEMM tests' own, four layers)."""
    import cxgnncomp
    ptr, idx = _graph(400, 2500, seed=2)
    n = ptr.shape[0] - 1
    torch.manual_seed(7)
    model = cxgnncomp.GCN(24, 32, 5, 4, 0.0, "CSR", residual=residual)
    with torch.no_grad():
        for p in model.norms.parameters():
            p.add_(0.2 * torch.randn(p.shape))
    ref = copy.deepcopy(model).double()
    x = torch.randn(n, 24)
    g = torch.randn(n, 5)

    def norm(v, kind, w, b):
        if kind == "layer":
            v = v - v.mean(1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5) * w
        return v if b is None else v + b

    x64 = x.double().requires_grad_(True)
    h, stream = x64, None
    ones = torch.ones(idx.shape[0], dtype=torch.float64)
    for i, conv in enumerate(ref.convs):
        h = pyref.spmm_torch(h, ptr, idx, n, ones) @ conv.lin.weight.t() + conv.bias
        if i == 3:
            break
        h, nm = F.relu(h), ref.norms[i]
        stream = h if i == 0 else stream + nm.gate * norm(h, residual, nm.post_weight, nm.post_bias)
        h = norm(stream, residual, nm.pre_weight, nm.pre_bias)
    want = h.log_softmax(-1)
    names = [k for k, _ in ref.named_parameters()]
    wgrads = torch.autograd.grad(want, [x64] + list(ref.parameters()), g.double())
    announce("residual GCN %s" % residual)
    model.cuda()
    batch = cxgnncomp.Batch(x.cuda().requires_grad_(True), ptr.cuda(), idx.cuda(), torch.tensor([n]), torch.tensor([idx.shape[0]]))
    xc = batch.x
    got = model(batch)
    grads = torch.autograd.grad(got, [xc] + list(model.parameters()), g.cuda())
    for name, a, b in [("logits", got, want)] + list(zip(["x"] + names, grads, wgrads)):
        b = b.detach()
        assert float((a.detach().double().cpu() - b).abs().max()) <= 2e-4 * float(b.abs().max()), name


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_residual_stack_with_inputs_in_8_bits(fmt):
    """The checkpoint changes weight gradients of the linear maps (and the order in which their bias
    gradients are added) and what is held, nothing else."""
    import cxgnncomp
    ptr, idx = _graph(6000, 30000, seed=3)
    n = ptr.shape[0] - 1
    torch.manual_seed(1)
    x, g = torch.randn(n, 64).cuda(), torch.randn(n, 7).cuda()
    plain = cxgnncomp.GCN(64, 64, 7, 5, 0.0, "CSR", residual="layer").cuda()
    packed = cxgnncomp.GCN(64, 64, 7, 5, 0.0, "CSR", residual="layer", checkpoint=fmt).cuda()
    packed.load_state_dict(plain.state_dict())
    announce("residual GCN checkpoint %s" % fmt)
    res = []
    for model in (plain, packed):
        xc = x.clone().requires_grad_(True)
        batch = cxgnncomp.Batch(xc, ptr.cuda(), idx.cuda(), torch.tensor([n]), torch.tensor([idx.shape[0]]))
        out, held = _saved_bytes(lambda: model(batch))
        res.append((out, held, torch.autograd.grad(out, [xc] + list(model.parameters()), g)))
    (a, held_a, ga), (b, held_b, gb) = res
    assert torch.equal(a, b)
    assert held_b <= held_a - 4 * n * 64 * (4 - 1.1)     # the aggregated inputs of four layers of 64 columns
    for name, u, v in zip(["x"] + [k for k, _ in plain.named_parameters()], ga, gb):
        if name.endswith("lin.weight"):
            bound = 0.02 if fmt == "int8" else 0.06      # half a step of the rows: 1 / 127 of a group's largest, 1 / 16
            assert 0 < float((u - v).norm() / u.norm()) < bound, name
        elif name.startswith("convs") and name.endswith("bias") and not name.startswith("convs.4"):
            # the same rows of the gradient added in another order (GCN: 64 -> 64, after the aggregation): fp32 sums
            # of 6,000 rows, at most 300 roundings deep in either order, against sums 1 / 80 of their magnitudes
            assert float((u - v).abs().max()) <= 2 * 300 * 2.0 ** -24 * 80 * float(u.abs().max()), name
        else:
            assert torch.equal(u, v), name


@gpu
@pytest.mark.parametrize("kind", ["SAGE", "GIN", "GAT", "RGCN"])
@pytest.mark.parametrize("residual", ["layer", "rms"])
def test_residual_stacks_on_a_sampled_batch(kind, residual):
    """Nested row prefixes: every layer's stream is the prefix of the one before; all parameters that a
    layer uses get a finite gradient, and a step of an optimizer changes them."""
    import cxgnncomp
    from cxgnncomp import synthetic as S
    ptr, idx, nn, ne = S.sampled_batch(num_seeds=64, fanouts=(5, 4, 3), id_space=4000, seed=0)
    torch.manual_seed(0)
    b = cxgnncomp.Batch(torch.randn(nn[-1], 16).cuda(), ptr.cuda(), idx.cuda(), torch.tensor(nn), torch.tensor(ne))
    more = {"GAT": dict(heads=2, concat=True), "RGCN": dict(num_rel=3)}.get(kind, dict(checkpoint="int8"))
    model = getattr(cxgnncomp, kind)(16, 32, 8, 3, 0.1, "CSR_Layer", residual=residual, **more).cuda()
    b.etypes = torch.randint(0, 3, (int(ne[-1]), )).cuda()
    opt = torch.optim.SGD(model.parameters(), lr=0.1)
    announce("residual %s %s on a sampled batch" % (kind, residual))
    for _ in range(2):
        before = {k: p.detach().clone() for k, p in model.named_parameters()}
        out = model(b)
        assert tuple(out.shape) == (nn[0], 8)
        opt.zero_grad()
        F.nll_loss(out, torch.arange(nn[0], device="cuda") % 8).backward()
        opt.step()
        for k, p in model.named_parameters():
            if p.grad is not None:
                assert torch.isfinite(p.grad).all(), k
        moved = [k for k, p in model.named_parameters() if p.grad is not None and not torch.equal(p, before[k])]
        assert any("norms.1.gate" in k for k in moved) and any("norms.0.pre_weight" in k for k in moved)


@gpu
def test_block_captured_and_replayed():
    """Norm, linear map with its input in 8 bits, gate and residual as one captured training step."""
    import cxgnncomp
    torch.manual_seed(0)
    n, c = 6000, 96
    norm = cxgnncomp.ResidualNorm(c, post="rms", pre="layer", gate="channel", gate_init=0.5).cuda()
    w, b = torch.randn(c, c, device="cuda", requires_grad=True), torch.randn(c, device="cuda", requires_grad=True)
    x = torch.randn(n, c, device="cuda").requires_grad_(True)
    f = torch.randn(n, c, device="cuda").requires_grad_(True)
    g = torch.randn(n, c, device="cuda")
    leaves = [x, f, w, b] + list(norm.parameters())

    def step():
        r, y = norm(x, f)
        h = cxgnncomp.linear(y, w, b, checkpoint="int8")
        r, y = norm(r, h)
        grads = torch.autograd.grad((r, y), leaves, (g, g))
        return [r.detach(), y.detach()] + list(grads)

    announce("block eager")
    step()
    torch.cuda.synchronize()
    announce("block captured")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            x.mul_(0.9)
            w.add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in held]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager)), k
        del eager
