"""The residual norm (csrc/residual_norm_fwd.hip, residual_norm_bwd.hip; cxgnncomp.residual_norm,
ResidualNorm) against a 64-bit restatement whose error bounds come from running error analysis
(tests/rounding.py, tests/residual_ref.py)."""
import pytest
import torch

import residual_ref
from conftest import announce
from rounding import check

gpu = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = ["x", "f", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias"]


def _inputs(rows, cols, stream=F32, branch=F32, post="layer", pre="layer", gate="channel", seed=0, shift=0.25):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape, scale=1.0, add=0.0, dtype=F32):
        return (torch.randn(shape, generator=g) * scale + add).to(dtype)

    t = {"x": rand(rows, cols, scale=1.5, add=shift, dtype=stream), "f": rand(rows, cols, scale=0.7, dtype=branch)}
    t["gate"] = {"none": None, "channel": rand(cols, scale=0.3, add=0.5), "row": rand(rows, 1, scale=0.3, add=0.5, dtype=branch),
                 "full": rand(rows, cols, scale=0.3, add=0.5, dtype=branch)}[gate]
    for side, kind in (("post", post), ("pre", pre)):
        t[side + "_weight"] = rand(cols, scale=0.2, add=1.0) if kind else None
        t[side + "_bias"] = rand(cols, scale=0.2) if kind == "layer" else None
    return t, rand(rows, cols, dtype=stream), rand(rows, cols, dtype=branch)


def _reference(t, post, pre, dr, dy, res_scale=0.9, branch_scale=0.5, eps=1e-5):
    return residual_ref.residual_norm(t["x"], t["f"], t["gate"], post, t["post_weight"], t["post_bias"], pre,
                                      t["pre_weight"], t["pre_bias"], res_scale, branch_scale, eps, dr, dy)


def _run(t, post, pre, dr, dy, res_scale=0.9, branch_scale=0.5, eps=1e-5):
    import cxgnncomp
    c = {k: None if v is None else v.cuda().requires_grad_(True) for k, v in t.items()}
    r, y = cxgnncomp.residual_norm(c["x"], c["f"], c["gate"], post=post, post_weight=c["post_weight"],
                                   post_bias=c["post_bias"], pre=pre, pre_weight=c["pre_weight"], pre_bias=c["pre_bias"],
                                   res_scale=res_scale, branch_scale=branch_scale, eps=eps)
    outs = [(o, g.cuda()) for o, g in ((r, dr), (y, dy)) if o is not None and g is not None]
    names = [k for k in NAMES if c[k] is not None]
    grads = torch.autograd.grad([o for o, _ in outs], [c[k] for k in names], [g for _, g in outs], allow_unused=True)
    return r, y, dict(zip(names, grads))


def _compare(t, post, pre, dr, dy, what, **kw):
    announce(what)
    r, y, grads = _run(t, post, pre, dr, dy, **kw)
    want = _reference(t, post, pre, dr, dy, **kw)
    check(r, want["r"], t["x"].dtype, what + " r")
    if pre:
        check(y, want["y"], t["f"].dtype, what + " y")
    for k, g in grads.items():
        if k in ("pre_weight", "pre_bias") and dy is None:
            assert g is None or not g.any()
            continue
        check(g, want[k], t[k].dtype, what + " gradient of " + k)


# ------------------------------- on the CPU: the restatement itself ------------------------------- #
@pytest.mark.parametrize("gate", ["none", "channel", "row", "full"])
@pytest.mark.parametrize("post,pre", [("layer", "rms"), ("rms", "layer"), (None, "layer")])
def test_restatement_against_autograd_and_differences(post, pre, gate):
    """Formulas of the gradients against float64 autograd of the definition and against central differences."""
    t, dr, dy = _inputs(5, 7, post=post, pre=pre, gate=gate, seed=4)
    v = {k: None if x is None else x.double().requires_grad_(True) for k, x in t.items()}

    def loss(v):
        def norm(a, kind, side):
            if kind is None:
                return a
            if kind == "layer":
                a = a - a.mean(dim=1, keepdim=True)
            a = a / torch.sqrt((a * a).mean(dim=1, keepdim=True) + eps) * v[side + "_weight"]
            return a if v[side + "_bias"] is None else a + v[side + "_bias"]
        h = norm(v["f"], post, "post")
        r = a_ * v["x"] + b_ * (h if v["gate"] is None else h * v["gate"])
        return (r * dr.double()).sum() + (norm(r, pre, "pre") * dy.double()).sum()

    a_, b_, eps = (float(torch.tensor(c, dtype=F32)) for c in (0.9, 0.5, 1e-5))
    names = [k for k in NAMES if v[k] is not None]
    grads = torch.autograd.grad(loss(v), [v[k] for k in names])
    want = _reference(t, post, pre, dr, dy)
    for k, g in zip(names, grads):
        assert torch.allclose(want[k].v, g, rtol=1e-9, atol=1e-9), k
        d = torch.randn(v[k].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
        h = 1e-5
        with torch.no_grad():
            up, down = (loss(dict(v, **{k: v[k] + s * h * d})) for s in (1, -1))
        slope = float((up - down) / (2 * h))
        assert abs(slope - float((g * d).sum())) <= 1e-6 * (1 + abs(slope)), k


def test_arguments_are_refused_on_the_host():
    import cxgnncomp
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        cxgnncomp.residual_norm(x, x)
    with pytest.raises(TypeError):
        cxgnncomp.residual_norm([1.0], x)
    with pytest.raises(ValueError):
        cxgnncomp.ResidualNorm(8, post="batch")
    with pytest.raises(ValueError):
        cxgnncomp.ResidualNorm(8, gate="full")


def test_library_refuses_bad_arguments():
    """Refusals of the C entry points: nothing is launched, the message names the argument."""
    from cxgnncomp_backend import _lib
    lib = _lib.load()

    def fwd(rows=1, cols=8, x=256, f=256, gate=None, gate_kind=0, post=0, pre=2, types=(0, 0), r=256, y=256, stats=None, ldx=8):
        return lib.cxg_residual_norm_fwd(x, ldx, f, 8, gate, 8, gate_kind, post, None, None, pre, None, None, 1.0, 1.0, 1e-5,
                                         rows, cols, types[0], types[1], r, y, stats, None)

    for kw, status in ((dict(rows=-1), -1), (dict(cols=0), -1), (dict(cols=8193), -2), (dict(types=(1, 0)), -2),
                       (dict(types=(0, 3)), -1), (dict(gate_kind=1), -1), (dict(gate_kind=4), -1), (dict(post=3), -1),
                       (dict(f=None, post=1), -1), (dict(x=None), -1), (dict(y=None), -1), (dict(r=None), -1),
                       (dict(stats=264), -1), (dict(ldx=-8), -1)):
        assert fwd(**kw) == status, kw
        assert lib.cxg_last_error()
    assert fwd(rows=0, x=None, f=None, r=None, y=None) == 0

    def bwd(rows=1, cols=8, stats=256, f=256, dgate=None, gate_kind=0, df=None, dpre_w=None, ws=None, nbytes=0):
        return lib.cxg_residual_norm_bwd(256, 8, f, 8, None, 0, gate_kind, 0, None, None, 2, None, 1.0, 1.0, rows, cols, 0, 0,
                                         stats, None, 0, None, 0, None, df, dgate, None, None, dpre_w, None, ws, nbytes, None)

    need = lib.cxg_residual_norm_workspace_bytes(1, 8)
    for kw, status in ((dict(stats=None), -1), (dict(stats=260), -1), (dict(f=None, df=256), -1), (dict(dgate=256), -1),
                       (dict(dpre_w=256), -3), (dict(dpre_w=256, ws=256, nbytes=need - 1), -3),
                       (dict(dpre_w=256, ws=264, nbytes=need), -3), (dict(rows=-1), -1)):
        assert bwd(**kw) == status, kw
    assert lib.cxg_residual_norm_workspace_bytes(-1, 8) == 0


# ------------------------------------------ on the GPU ------------------------------------------- #
COLS = [1, 3, 8, 16, 17, 32, 47, 64, 100, 128, 130, 256, 257, 512, 1000, 1025, 1028, 2048, 2050, 4096, 8191, 8192]


@gpu
@pytest.mark.parametrize("cols", COLS)
def test_widths_fp32(cols):
    rows = 37 if cols > 512 else 301
    t, dr, dy = _inputs(rows, cols, seed=cols)
    _compare(t, "layer", "layer", dr, dy, "residual_norm fp32 %d x %d" % (rows, cols))


@gpu
@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("types", [(BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)])
def test_widths_narrow_types(cols, types):
    rows = 9 if cols > 512 else 65
    t, dr, dy = _inputs(rows, cols, types[0], types[1], "rms", "rms", "full", seed=cols)
    _compare(t, "rms", "rms", dr, dy, "residual_norm %s %d x %d" % (types, rows, cols))


@gpu
@pytest.mark.parametrize("gate", ["none", "channel", "row", "full"])
@pytest.mark.parametrize("pre", ["layer", "rms", None])
@pytest.mark.parametrize("post", ["layer", "rms", None])
@pytest.mark.parametrize("cols", [47, 128])
def test_kinds(cols, post, pre, gate):
    t, dr, dy = _inputs(130, cols, post=post, pre=pre, gate=gate, seed=9)
    _compare(t, post, pre, dr, dy if pre else None, "residual_norm %d cols post=%s pre=%s gate=%s" % (cols, post, pre, gate))


@gpu
@pytest.mark.parametrize("rows", [0, 1, 2, 31, 4096])
@pytest.mark.parametrize("cols", [5, 64, 600])
def test_row_counts(rows, cols):
    t, dr, dy = _inputs(rows, cols, seed=rows)
    _compare(t, "layer", "layer", dr, dy, "residual_norm %d x %d" % (rows, cols))


@gpu
@pytest.mark.parametrize("which", ["r", "y"])
def test_one_gradient_alone(which):
    t, dr, dy = _inputs(70, 96, gate="row")
    _compare(t, "layer", "layer", dr if which == "r" else None, dy if which == "y" else None, "residual_norm gradient of %s" % which)


@gpu
def test_missing_weights_are_one_and_biases_zero():
    t, dr, dy = _inputs(40, 33)
    for k in ("post_weight", "post_bias", "pre_weight", "pre_bias"):
        t[k] = None
    _compare(t, "layer", "layer", dr, dy, "residual_norm without vectors")


@gpu
def test_mean_far_from_zero_and_rows_of_one_value():
    """A drift of a hundred standard deviations costs what the rounding of its inputs costs and no more;
    a row of one value has no variance: its normalised values are 0, its factor 1 / sqrt(eps)."""
    t, dr, dy = _inputs(64, 128, shift=150.0)
    t["f"][::7] = 3.0
    t["f"][1::7] = 0.0
    _compare(t, "layer", "layer", dr, dy, "residual_norm far mean")


@gpu
def test_entry_without_a_branch():
    import cxgnncomp
    t, _, dy = _inputs(50, 72)
    announce("residual_norm entry")
    x = t["x"].cuda().requires_grad_(True)
    w, b = t["pre_weight"].cuda().requires_grad_(True), t["pre_bias"].cuda().requires_grad_(True)
    r, y = cxgnncomp.residual_norm(x, None, pre="layer", pre_weight=w, pre_bias=b)
    assert r is x
    want = residual_ref.residual_norm(t["x"], None, None, None, None, None, "layer", t["pre_weight"], t["pre_bias"], 1.0, 1.0,
                                      1e-5, None, dy)
    check(y, want["y"], F32, "y")
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), dy.cuda())
    check(gx, want["x"], F32, "gradient of x")
    check(gw, want["pre_weight"], F32, "gradient of the weight")
    check(gb, want["pre_bias"], F32, "gradient of the bias")


@gpu
def test_strides_alignment_and_expanded_gradients():
    """Rows out of a wider matrix, rows that start off a 16-byte boundary, transposed inputs, one row
    shared by all (stride 0) as input and as gradient."""
    import cxgnncomp
    t, dr, dy = _inputs(48, 64, gate="full")
    want = _reference(t, "layer", "layer", dr, dy)
    for name, lay in (("columns 4..67 of 80", lambda a: torch.nn.functional.pad(a, (4, 12))[:, 4:68]),
                      ("columns 1..64 of 66", lambda a: torch.nn.functional.pad(a, (1, 1))[:, 1:65]),
                      ("transposed", lambda a: a.t().contiguous().t()),
                      ("every other row", lambda a: torch.stack([a, a * 0], 1)[:, 0])):
        announce("residual_norm " + name)
        c = {k: (lay(v.cuda()) if v.dim() == 2 else v.cuda()).requires_grad_(True) for k, v in t.items()}
        r, y = cxgnncomp.residual_norm(c["x"], c["f"], c["gate"], post="layer", post_weight=c["post_weight"],
                                       post_bias=c["post_bias"], pre="layer", pre_weight=c["pre_weight"],
                                       pre_bias=c["pre_bias"], res_scale=0.9, branch_scale=0.5)
        check(r, want["r"], F32, name + " r")
        check(y, want["y"], F32, name + " y")
        for k, g in zip(NAMES, torch.autograd.grad((r, y), [c[k] for k in NAMES], (lay(dr.cuda()), lay(dy.cuda())))):
            check(g, want[k], F32, name + " gradient of " + k)
    announce("residual_norm shared rows")
    one = {k: v[:1].expand(48, 64) if v.dim() == 2 else v for k, v in t.items()}
    ones = torch.ones(1, 1).expand(48, 64)
    want = _reference(one, "layer", "layer", ones, ones * 0.5)
    c = {k: (v[:1].cuda().requires_grad_(True) if v.dim() == 2 else v.cuda()) for k, v in t.items()}
    r, y = cxgnncomp.residual_norm(c["x"].expand(48, 64), c["f"].expand(48, 64), c["gate"].expand(48, 64), post="layer",
                                   post_weight=c["post_weight"], post_bias=c["post_bias"], pre="layer",
                                   pre_weight=c["pre_weight"], pre_bias=c["pre_bias"], res_scale=0.9, branch_scale=0.5)
    check(r, want["r"], F32, "shared r")
    gx, gf = torch.autograd.grad(r.sum() + 0.5 * y.sum(), (c["x"], c["f"]))
    check(gx, want["x"].sum(0, 48, True), F32, "shared gradient of x")
    check(gf, want["f"].sum(0, 48, True), F32, "shared gradient of f")


@gpu
def test_rows_that_are_not_finite_keep_to_themselves():
    import cxgnncomp
    t, dr, dy = _inputs(40, 128, gate="full")
    clean, _, _ = _run(t, "layer", "layer", dr, dy)[0:3]
    t["x"][3, 5], t["f"][11, 0], t["gate"][20, 127] = float("nan"), float("inf"), float("-inf")
    announce("residual_norm rows that are not finite")
    r, y, g = _run(t, "layer", "layer", dr, dy)
    keep = torch.ones(40, dtype=torch.bool)
    keep[[3, 11, 20]] = False
    assert torch.equal(r[keep.cuda()], clean[keep.cuda()])
    for out in (y, g["x"], g["f"]):
        assert torch.isfinite(out[keep.cuda()]).all()
        assert not torch.isfinite(out[~keep.cuda()]).all(dim=1).any()


@gpu
def test_repeats_bit_for_bit_and_rows_do_not_depend_on_their_neighbours():
    t, dr, dy = _inputs(3000, 100, gate="row")
    announce("residual_norm twice")
    a, b = _run(t, "layer", "layer", dr, dy), _run(t, "layer", "layer", dr, dy)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert all(torch.equal(a[2][k], b[2][k]) for k in a[2])
    part = {k: v[1000:1011] if v is not None and v.shape[0] == 3000 else v for k, v in t.items()}
    c = _run(part, "layer", "layer", dr[1000:1011], dy[1000:1011])
    assert torch.equal(c[0], a[0][1000:1011]) and torch.equal(c[1], a[1][1000:1011])
    assert torch.equal(c[2]["f"], a[2]["f"][1000:1011])


@gpu
def test_another_stream_and_a_replayed_graph():
    import cxgnncomp
    t, dr, dy = _inputs(500, 128)
    want_r, want_y, want = _run(t, "layer", "layer", dr, dy)
    torch.cuda.synchronize()
    c = {k: v.cuda().requires_grad_(True) for k, v in t.items()}
    dr, dy = dr.cuda(), dy.cuda()

    def step():
        r, y = cxgnncomp.residual_norm(c["x"], c["f"], c["gate"], post="layer", post_weight=c["post_weight"],
                                       post_bias=c["post_bias"], pre="layer", pre_weight=c["pre_weight"],
                                       pre_bias=c["pre_bias"], res_scale=0.9, branch_scale=0.5)
        return (r.detach(), y.detach()) + torch.autograd.grad((r, y), [c[k] for k in NAMES], (dr, dy))

    announce("residual_norm on a side stream")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want_r) and torch.equal(got[1], want_y)
    assert all(torch.equal(a, want[k]) for k, a in zip(NAMES, got[2:]))
    del got
    announce("residual_norm captured")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            c["x"].mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [h.clone() for h in held]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager)), k
        del eager


@gpu
def test_refusals():
    import cxgnncomp
    x = torch.zeros(4, 8, device="cuda")
    v = torch.ones(8, device="cuda")
    rn = cxgnncomp.residual_norm
    for args, kw in (((x, x[:3]), {}), ((x, x.double()), {}), ((x.double(), x), {}), ((x.bfloat16(), x), {}),
                     ((x, x), dict(pre="batch")), ((x, x), dict(post_weight=v)), ((x, x), dict(pre_weight=v[:7])),
                     ((x, x), dict(pre_weight=v.half())), ((x, x), dict(pre_weight=v.cpu())), ((x, x, v[:7]), {}),
                     ((x, x, v.bfloat16()), {}), ((x, x, x[:, :2]), {}), ((x, x, x[:1]), {}), ((x, x, x.half()), {}),
                     ((x, None, v), {}), ((x, None), dict(res_scale=2.0)), ((x, None), dict(post="rms")), ((x, None), dict(pre=None)),
                     ((x[0], x[0]), {}), ((torch.zeros(4, 8193, device="cuda"), torch.zeros(4, 8193, device="cuda")), {}),
                     ((torch.zeros(4, 0, device="cuda"), torch.zeros(4, 0, device="cuda")), {})):
        with pytest.raises(ValueError):
            rn(*args, **kw)
    m = cxgnncomp.ResidualNorm(8, gate="channel").cuda()
    with pytest.raises(ValueError):
        m(x, x, x)
    r, _ = rn(x.requires_grad_(True), x.detach(), pre=None)
    with pytest.raises(RuntimeError):          # second derivatives are not given
        g = torch.autograd.grad(r.sum(), x, create_graph=True)[0]
        torch.autograd.grad(g.sum(), x)


@gpu
def test_module_and_a_changed_input():
    """ResidualNorm trains its vectors; an input changed between forward and backward is noticed."""
    import cxgnncomp
    torch.manual_seed(0)
    m = cxgnncomp.ResidualNorm(64, post="rms", pre="layer", gate="channel", gate_init=0.1, branch_scale=2.0).cuda()
    assert sorted(m.state_dict()) == ["gate", "post_weight", "pre_bias", "pre_weight"]
    x, f = torch.randn(33, 64), torch.randn(33, 64)
    xc, fc = x.cuda().requires_grad_(True), f.cuda().requires_grad_(True)
    announce("ResidualNorm module")
    stream, y0 = m.enter(xc)
    r, y = m(stream, fc)
    want = residual_ref.residual_norm(x, f, m.gate.detach().cpu(), "rms", m.post_weight.detach().cpu(), None, "layer",
                                      m.pre_weight.detach().cpu(), m.pre_bias.detach().cpu(), 1.0, 2.0, 1e-5, None, torch.ones(33, 64))
    check(y, want["y"], F32, "y")
    y.sum().backward()
    check(m.gate.grad, want["gate"], F32, "gradient of the gate")
    check(m.post_weight.grad, want["post_weight"], F32, "gradient of the post weight")
    check(fc.grad, want["f"], F32, "gradient of f")
    r, y = m(stream, fc)
    with torch.no_grad():
        fc.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@gpu
@pytest.mark.parametrize("eps", [0.0, 1e-42])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_rows_whose_squares_are_below_the_smallest_normal_number(eps, kind):
    """Mean squares near 1e-40 keep some 16 bits: the result is within 2^-10 of the formula in 64 bits."""
    import cxgnncomp
    x = torch.randn(9, 64, generator=torch.Generator().manual_seed(3)) * 1e-20
    announce("residual_norm %s of tiny rows, eps %g" % (kind, eps))
    _, y = cxgnncomp.residual_norm(x.cuda(), None, pre=kind, eps=eps)
    v = x.double()
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    want = v / (v.square().mean(1, keepdim=True) + eps).sqrt()
    assert ((y.cpu().double() - want).abs() <= 2.0 ** -10 * want.abs() + 2.0 ** -12).all()
