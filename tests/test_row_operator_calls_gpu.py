"""Calls of the row operators (residual norm, rows in 8 bits, their weight gradient, linear maps and layers on
them) that the documentation allows or refuses, beside the shapes of the other files."""
import pytest
import torch

import packed_ref
from conftest import announce
from rounding import B, U, check

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _half_step(values, exps, cols, fmt):
    """What a value may be off by: half a step of its code."""
    scale = packed_ref.spread(exps, cols)
    if fmt == "int8":
        return scale / 2
    return torch.maximum(values.abs() / 16, scale * 2.0 ** -10)


def _large_fp16_rows():
    x = torch.zeros(12, 200, dtype=F16)
    large = torch.tensor([65504.0, 65472.0, 65280.0, 65248.0, 65056.0, 65024.0, 64992.0, 63488.0, 63456.0, 61440.0, 40000.0, 1.0], dtype=F16)
    for r in range(12):
        x[r, : 12 - r] = large[r:]                       # every one of them is some row's largest
        x[r, 100:112 - r] = -large[r:]
        x[r, 128 + r:140] = large[r:]
    return x


# ----------------------------------------- on the CPU ------------------------------------------- #
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_large_fp16_values_are_held_within_half_a_step(fmt):
    """The 8-bit form of finite fp16 rows is at most 65536 and off by half a step; 65504 in its place is too."""
    x = _large_fp16_rows()
    _, exps, values = packed_ref.pack(x, fmt)
    assert float(values.abs().max()) == 65536.0
    for v in (values, values.clamp(-65504.0, 65504.0)):
        assert ((v - x.double()).abs() <= _half_step(x.double(), exps, 200, fmt)).all()


def _chunks(m, k, n, segs):
    """Row chunks for which the weight gradient takes workspace."""
    from cxgnncomp_backend import _lib
    return (_lib.load().cxg_packed_wgrad_workspace_bytes(m, k, n, segs) - 256) // (4 * n * (k + 1))


@pytest.mark.parametrize("k,n", [(64, 64), (128, 128), (512, 512), (600, 600), (1024, 1024), (2048, 2048), (4096, 4096)])
def test_rows_per_chunk_with_any_number_of_segments(k, n):
    """What is left of the chunks when every segment but one ends in a ragged one splits a segment of nearly all rows
    at least as finely as one segment is split at most half as finely; no chunk is longer than 65,536 rows."""
    for m in (20000, 400000, 2332486):
        whole = _chunks(m, k, n, 1)
        assert whole * 65536 >= m
        for segs in (2, 7, 33, 40, 65, 129, 200, 237, 1000, 5000):
            left = _chunks(m, k, n, segs) - (segs - 1)
            # (chunks of at least 64 rows; counts are rounded up to a multiple of eight)
            assert left >= min(whole // 2, m // 64) - 8 and left * 65536 >= m, (m, segs, left, whole)
            assert _chunks(m, k, n, segs) <= 2 * whole + segs + 8, (m, segs)


def test_a_weight_gradient_too_large_for_a_launch_is_refused_before_any():
    """(Status -2, not the -4 of a launch that failed; all of it on the host.)"""
    from cxgnncomp_backend import _lib
    lib = _lib.load()
    for k, n, segs in ((1 << 17, 1 << 17, 1), (1 << 22, 1 << 22, 1), (1 << 18, (1 << 16) + 1, 3)):
        need = lib.cxg_packed_wgrad_workspace_bytes(10, k, n, segs)
        assert lib.cxg_packed_wgrad(256, 256, 0, 10, 256, n, 0, 10, None, None, 256, 10, k, n, segs, 256, None, 256, need, None) == -2
        assert b"too large" in lib.cxg_last_error()


# ------------------------------------------ on the GPU ------------------------------------------- #
@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_finite_fp16_rows_read_back_finite(fmt):
    import cxgnncomp
    x = _large_fp16_rows()
    announce("unpack large fp16 rows %s" % fmt)
    for cols in (200, 190, 45, 12):                      # whole and moved-back pieces, every number of lanes
        p = cxgnncomp.pack_rows(x[:, :cols].contiguous().cuda(), fmt)
        codes, exps, values = packed_ref.pack(x[:, :cols], fmt)
        assert torch.equal(p.codes.cpu(), codes) and torch.equal(p.exps.cpu(), exps)
        back = p.unpack()
        assert back.dtype == F16 and torch.equal(back.cpu(), values.clamp(-65504.0, 65504.0).half())
        again = cxgnncomp.pack_rows(back, fmt)           # packing what was unpacked gives the same codes
        assert torch.equal(again.codes, p.codes) and torch.equal(again.exps, p.exps)
        assert torch.equal(p.unpack(F32).cpu().double(), values) and torch.equal(p.unpack(BF16).cpu().double(), values)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_wider_rows_unpacked_to_fp16_overflow_as_a_cast_does(fmt):
    import cxgnncomp
    x = torch.zeros(4, 130)
    x[0, :3] = torch.tensor([1e5, -1e5, 3.0])
    x[1, :2] = torch.tensor([65000.0, -66000.0])
    x[2, 7] = float("nan")
    x[3, 129] = 1e30
    announce("unpack fp32 rows to fp16 %s" % fmt)
    p = cxgnncomp.pack_rows(x.cuda(), fmt)
    _, _, values = packed_ref.pack(x, fmt)
    want = torch.where(values.abs() == 65536, values.sign() * 65504, values).half()
    got = p.unpack(F16).cpu()
    assert torch.isinf(got[0, 0]) and torch.isinf(got[3, 129]) and torch.isnan(got[2, :128]).all()
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want)) and torch.equal(torch.isnan(got), torch.isnan(want))


@gpu
@pytest.mark.parametrize("which", ["x", "f", "gate", "pre_weight"])
@pytest.mark.parametrize("mode", ["no_grad", "grad", "leaf"])
def test_residual_norm_refuses_forward_mode_derivatives(which, mode):
    """An argument with a tangent is refused, whether or not others take part in a backward pass."""
    import cxgnncomp
    from torch.autograd import forward_ad
    t = {"x": torch.randn(5, 8, device="cuda"), "f": torch.randn(5, 8, device="cuda"), "gate": torch.ones(8, device="cuda"),
         "pre_weight": torch.ones(8, device="cuda")}
    if mode == "leaf":
        t["f" if which == "x" else "x"].requires_grad_(True)
    announce("residual_norm of a dual tensor %s %s" % (which, mode))
    with forward_ad.dual_level():
        t[which] = forward_ad.make_dual(t[which].detach(), torch.ones_like(t[which]))
        with torch.set_grad_enabled(mode != "no_grad"):
            with pytest.raises(RuntimeError, match="forward-mode"):
                cxgnncomp.residual_norm(t["x"], t["f"], t["gate"], pre_weight=t["pre_weight"])
            if which in ("x", "pre_weight"):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    cxgnncomp.residual_norm(t["x"], None, pre_weight=t["pre_weight"])
    cxgnncomp.residual_norm(t["x"], t["f"], t["gate"], pre_weight=t["pre_weight"])      # outside the level: no tangents


@gpu
@pytest.mark.parametrize("m,k,n,segs,share", [(100000, 1024, 1024, 40, 0.9), (60000, 512, 512, 200, 0.5), (50000, 300, 200, 700, 0.7), (20000, 64, 40, 3000, 0.3),
                                              (300000, 2048, 2048, 1, 1.0), (400000, 1024, 1024, 1, 1.0)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_weight_grad_of_many_segments_and_of_long_chunks(m, k, n, segs, share, dtype):
    """Skewed segments, more of them than chunks fit the chip at once, and the longest chunks: every segment's 2-norm of
    the error stays where fp32 accumulation of a chunk puts it (random roundings: 2^-24 * sqrt(products of a chunk) of
    the result); the sums of G's rows too; results repeat bit for bit."""
    import cxgnncomp
    torch.manual_seed(0)
    big = int(m * share)
    cuts = [0, big] + (torch.sort(torch.randint(big, m + 1, (segs - 2, )))[0].tolist() + [m] if segs > 1 else [])
    x, g = torch.randn(m, k, device="cuda"), torch.randn(m, n, device="cuda").to(dtype)
    seg = torch.tensor(cuts, device="cuda")
    assert seg.shape[0] == segs + 1
    announce("packed_weight_grad %d x %d x %d, %d segments %s" % (m, k, n, segs, dtype))
    p = cxgnncomp.pack_rows(x)
    gw, gb = cxgnncomp.packed_weight_grad(p, g, seg, want_sums=True)
    again = cxgnncomp.packed_weight_grad(p, g, seg, want_sums=True)
    assert torch.equal(gw, again[0]) and torch.equal(gb, again[1])
    chunk = min(65536, -(-m // (_chunks(m, k, n, segs) - (segs - 1) - 7)))      # rows at most (the count is a multiple of eight)
    bound = 2.0 ** -24 * (chunk * (3 if dtype == F32 else 1)) ** 0.5
    a = p.unpack().double()
    for r in [0] + list(range(1, segs, max(1, segs // 30))):
        b, e = cuts[r], cuts[r + 1]
        want, sums = a[b:e].t() @ g[b:e].double(), g[b:e].double().sum(0)
        if b == e:
            assert not gw[r].any() and not gb[r].any()
            continue
        # (a short segment: one rounding at least)
        assert float((gw[r] - want).norm()) <= max(bound, 2.0 ** -22) * float(want.norm()), r
        assert float((gb[r] - sums).norm()) <= max(bound, 2.0 ** -22) * float(sums.norm()), r


def _product(a, b, dtype):
    """a @ b by a library product of ``dtype`` operands: fp32 sums, rounded once to ``dtype``."""
    a, b = a.to(dtype).double(), b.to(dtype).double()
    v, mag = a @ b, a.abs() @ b.abs()
    return B(v, 2 * U * a.shape[1] * mag + torch.finfo(dtype).eps / 2 * (v.abs() + 2 * U * a.shape[1] * mag))


@gpu
@pytest.mark.parametrize("m,k,n", [(300, 90, 33), (5000, 128, 64), (5000, 90, 64), (1, 16, 8)])
@pytest.mark.parametrize("how", ["bf16", "fp16", "autocast", "bf16 addend", "fp64"])
def test_linear_without_checkpoint_in_other_types(m, k, n, how):
    """Forward and backward where neither the split product nor the weight-gradient kernel takes the types."""
    import cxgnncomp
    torch.manual_seed(k)
    dtype = {"bf16": BF16, "fp16": F16, "autocast": BF16, "bf16 addend": BF16, "fp64": torch.float64}[how]
    held = F32 if how == "autocast" else dtype
    x, w, b = (torch.randn(s).to(held) for s in ((m, k), (n, k), (n, )))
    w = w / 8
    g = torch.randn(m, n).to(dtype)
    t = [v.cuda().requires_grad_(True) for v in ((x, w, b) + ((torch.randn(m, n).to(held), ) if "addend" in how else ()))]
    announce("linear %d x %d x %d %s" % (m, k, n, how))
    with torch.autocast("cuda", dtype=BF16, enabled=how == "autocast"):
        out = cxgnncomp.linear(*t)
    if how == "autocast" and out.dtype == F32:           # fp32 inputs that the split product takes stay fp32
        g, dtype = g.float(), F32
    grads = torch.autograd.grad(out, t, g.cuda())
    if how == "fp64":
        for got, want in zip(grads, (g @ w, g.t() @ x, g.sum(0))):
            assert got.dtype == dtype and torch.allclose(got.cpu(), want, rtol=1e-12, atol=1e-12)
        return
    if dtype == F32:
        assert (m, k, n) == (5000, 128, 64)
        for got, want in zip(grads, (g.double() @ w.double(), g.double().t() @ x.double(), g.double().sum(0))):
            assert float((got.cpu() - want).norm() / want.norm()) < 2.0 ** -20
        return
    check(grads[0], _product(g, w, dtype), held, "gx")
    check(grads[1], _product(g.t(), x, dtype), held, "gw")
    sums = g.double()
    check(grads[2], B(sums.sum(0), U * m * 1.01 * sums.abs().sum(0)), held, "gb")
    if "addend" in how:
        assert torch.equal(grads[3].cpu(), g)


@gpu
@pytest.mark.parametrize("m,k,n", [(5000, 128, 64), (5000, 90, 64), (300, 90, 33)])
def test_linear_that_keeps_8_bits_under_autocast(m, k, n):
    """Output and its type as without checkpoint, on the split product and on the library's; gradients of both."""
    import cxgnncomp
    torch.manual_seed(n)
    x, w, b = (torch.randn(s, device="cuda").requires_grad_(True) for s in ((m, k), (n, k), (n, )))
    announce("linear checkpoint autocast %d x %d x %d" % (m, k, n))
    with torch.autocast("cuda", dtype=BF16):
        out, plain = (cxgnncomp.linear(x, w, b, checkpoint=c) for c in ("int8", None))
    assert out.dtype == plain.dtype and torch.equal(out, plain)
    g = torch.randn(m, n, device="cuda").to(out.dtype)
    got, want = (torch.autograd.grad(o, (x, w, b), g) for o in (out, plain))
    assert torch.equal(got[0], want[0]) and all(v.dtype == F32 for v in got)
    weight = packed_ref.weight_grad(packed_ref.pack(x.detach().cpu(), "int8")[2], g.cpu(), [0, m])
    weight.v, weight.e = weight.v[0].t(), weight.e[0].t()
    check(got[1], weight, F32, "weight gradient")
    check(got[2], packed_ref.row_sums(g.cpu(), [0, m])[0], F32, "bias gradient")


@gpu
@pytest.mark.parametrize("m", [300, 5000])
def test_linear_maps_refuse_forward_mode_derivatives(m):
    import cxgnncomp
    from torch.autograd import forward_ad
    x, w = torch.randn(m, 128, device="cuda"), torch.randn(64, 128, device="cuda")
    announce("linear of a dual tensor")
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for checkpoint in (None, "int8"):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                    cxgnncomp.linear(d, w, checkpoint=checkpoint)


@gpu
@pytest.mark.parametrize("widths", [(16, 24), (24, 16)])
@pytest.mark.parametrize("num_node", [0, 40])
def test_sage_layer_with_8_bits_takes_the_rows_it_takes_without(widths, num_node):
    """More source rows than rows of the graph, all rows asked for as 0, a column slice as input."""
    import cxgnncomp
    from cxgnncomp import synthetic as S
    cxgnncomp.set_timers()
    ptr, idx = S.uniform_graph(60, 300, seed=0)
    ptr, idx = ptr.cuda(), idx.cuda()
    torch.manual_seed(0)
    conv = cxgnncomp.MySageConv(*widths).cuda()
    packed = cxgnncomp.MySageConv(*widths, checkpoint="int8").cuda()
    packed.load_state_dict(conv.state_dict())
    wide = torch.randn(75, widths[0] + 5, device="cuda")
    res = []
    announce("MySageConv %s num_node %d" % (widths, num_node))
    for layer in (conv, packed):
        x = wide[:, 2:widths[0] + 2].detach().requires_grad_(True)
        out = layer(x, ptr, idx, num_node)
        res.append((out, torch.autograd.grad(out.square().sum(), x)[0]))
    assert tuple(res[1][0].shape) == (num_node or 60, widths[1])
    for a, b in zip(*res):
        # the same products of at most 24 values and means of about five rows, in another order
        assert float((a - b).detach().abs().max()) <= 2.0 ** -18 * float(a.detach().abs().max())


@gpu
@pytest.mark.parametrize("empty", ["a", "g", "both"])
@pytest.mark.parametrize("segs", [1, 3, 20])
def test_weight_grad_of_maps_into_matrices_without_rows(empty, segs):
    """Every entry of such a map is outside its matrix and leaves its row out: zeros."""
    import cxgnncomp
    x = torch.randn(0 if empty != "g" else 50, 70, device="cuda")
    g = torch.randn(0 if empty != "a" else 50, 33, device="cuda")
    ids = torch.arange(50, device="cuda")
    seg = torch.linspace(0, 50, segs + 1).long().cuda()
    announce("packed_weight_grad of no rows %s %d" % (empty, segs))
    p = cxgnncomp.pack_rows(x)
    torch.full((1 << 20, ), float("nan"), device="cuda")                # (what the workspace may hold)
    gw, gb = cxgnncomp.packed_weight_grad(p, g, seg, src_idx=ids, dst_idx=ids - (3 if empty == "both" else 0), want_sums=True)
    assert tuple(gw.shape) == (segs, 70, 33) and tuple(gb.shape) == (segs, 33) and not gw.any() and not gb.any()
    with pytest.raises(ValueError):                                     # no map: as many rows as there are entries are needed
        cxgnncomp.packed_weight_grad(p, g, seg, **({"dst_idx": ids} if empty != "g" else {"src_idx": ids}))


@gpu
@pytest.mark.parametrize("m,k,n", [(300, 90, 33), (200000, 90, 33), (200000, 128, 64), (0, 90, 33)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_bias_gradient_beside_a_frozen_weight(m, k, n, dtype):
    """Nothing of x is kept; the sums of g's rows repeat bit for bit, eager and in a graph that is replayed between
    eager passes."""
    import cxgnncomp
    torch.manual_seed(1)
    x, w = torch.randn(m, k, device="cuda").to(dtype), torch.randn(n, k, device="cuda").to(dtype)
    b = torch.randn(n, device="cuda").to(dtype).requires_grad_(True)
    g = torch.randn(m, n, device="cuda").to(dtype)

    def step():
        out = cxgnncomp.linear(x, w, b, checkpoint="int8")
        return torch.autograd.grad(out, b, g)[0]

    def want():
        v = g.double().cpu()
        return B(v.sum(0), U * (m + 2) * 1.01 * v.abs().sum(0))

    announce("linear frozen weight %d x %d x %d %s" % (m, k, n, dtype))
    first = step()
    check(first, want(), dtype, "bias gradient")
    assert torch.equal(first, step())
    if m == 0:
        return
    announce("linear frozen weight captured")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        g.mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        replayed = held.clone()
        eager = step()
        torch.cuda.synchronize()
        assert torch.equal(replayed, eager)
        check(replayed, want(), dtype, "replayed")


@gpu
@pytest.mark.parametrize("m,k,n", [(300, 100, 47), (5000, 256, 47), (1, 64, 8)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("extra", ["bias", "addend"])
def test_linear_on_library_products_captured_and_replayed(m, k, n, dtype, extra):
    """The compiled node as one captured training step, replayed between eager ones with other inputs."""
    import cxgnncomp
    torch.manual_seed(2)
    t = [torch.randn(s, device="cuda").to(dtype).requires_grad_(True) for s in ((m, k), (n, k), (n, ))]
    if extra == "addend":
        t.append(torch.randn(m, n, device="cuda").to(dtype).requires_grad_(True))
    g = torch.randn(m, n, device="cuda").to(dtype)

    def step():
        out = cxgnncomp.linear(*t, checkpoint="e4m3")
        return [out.detach()] + list(torch.autograd.grad(out, t, g))

    announce("linear captured %d x %d x %d %s %s" % (m, k, n, dtype, extra))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            t[0].mul_(-0.9)
            t[1].add_(0.01)
        g.mul_(1.125)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [v.clone() for v in held]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager)), i


@gpu
def test_two_graphs_and_eager_work_keep_apart():
    """Two captured weight gradients of different shapes, many segments in one, replayed in turns with eager work on another
    stream: each has a workspace of its own."""
    import cxgnncomp
    torch.manual_seed(3)
    cases = []
    for m, k, n, segs in ((9000, 130, 70, 40), (4000, 300, 64, 3)):
        p = cxgnncomp.pack_rows(torch.randn(m, k, device="cuda"))
        cases.append((p, torch.randn(m, n, device="cuda"), torch.linspace(0, m, segs + 1).long().cuda()))
    announce("two captured weight gradients")
    want = [cxgnncomp.packed_weight_grad(*c, want_sums=True) for c in cases]
    torch.cuda.synchronize()
    graphs, held = [], []
    for c in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(cxgnncomp.packed_weight_grad(*c, want_sums=True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        with torch.cuda.stream(side):
            other = [cxgnncomp.packed_weight_grad(*c, want_sums=True) for c in cases]
        torch.cuda.synchronize()
        for got in (held, other):
            assert all(torch.equal(a, b) for u, v in zip(got, want) for a, b in zip(u, v))
