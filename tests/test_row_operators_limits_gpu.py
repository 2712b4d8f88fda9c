"""Residual norm, rows in 8 bits and their weight gradient at offsets beyond 32 bits and on two streams at
once: rows have to come out as they do from a call on a slice, bit for bit."""
import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_offsets_beyond_32_bits():
    import cxgnncomp
    rows, cols, tail = (1 << 31) // 128 + 4099, 128, 3000
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(rows, cols, dtype=BF16, device="cuda").normal_(generator=gen)
    assert x.numel() > 1 << 31
    w = torch.rand(cols, device="cuda") + 0.5

    announce("pack_rows %d x %d" % (rows, cols))
    p = cxgnncomp.pack_rows(x)
    q = cxgnncomp.pack_rows(x[-tail:])
    assert torch.equal(p.codes[-tail:], q.codes) and torch.equal(p.exps[-tail:], q.exps)
    announce("unpack %d x %d" % (rows, cols))
    assert torch.equal(p.unpack()[-tail:], q.unpack())

    announce("packed_weight_grad %d x %d" % (rows, cols))
    seg = torch.tensor([rows - tail, rows], device="cuda")
    got = cxgnncomp.packed_weight_grad(p, x, seg, want_sums=True)
    want = q.unpack().double().t() @ x[-tail:].double()
    # 3,000 products of magnitude about 1 per element: 2^-24 of the running sum per addition
    assert float((got[0][0] - want).abs().max()) < 3000 * 2.0 ** -23 * 55
    assert float((got[1][0] - x[-tail:].double().sum(0)).abs().max()) < 3000 * 2.0 ** -24 * 55
    rows_map = torch.arange(rows - tail, rows, device="cuda")
    maps = cxgnncomp.packed_weight_grad(p, x, torch.tensor([0, tail], device="cuda"), rows_map, rows_map)
    assert float((maps[0] - want).abs().max()) < 3000 * 2.0 ** -23 * 55
    del p, got, maps

    announce("residual_norm %d x %d" % (rows, cols))
    x.requires_grad_(True)
    r, y = cxgnncomp.residual_norm(x, x.detach(), x.detach(), post="rms", pre="layer", pre_weight=w)
    gx, = torch.autograd.grad((r, y), x, (x.detach(), x.detach()))
    s = x.detach()[-tail:].clone().requires_grad_(True)
    rs, ys = cxgnncomp.residual_norm(s, s.detach(), s.detach(), post="rms", pre="layer", pre_weight=w)
    gs, = torch.autograd.grad((rs, ys), s, (s.detach(), s.detach()))
    assert torch.equal(r[-tail:], rs) and torch.equal(y[-tail:], ys) and torch.equal(gx[-tail:], gs)


def test_two_streams_at_once():
    """Training passes of one block on two streams, interleaved, each on its own workspace: every result is the
    one that the pass gives alone."""
    import cxgnncomp
    torch.manual_seed(0)

    def make(n, c):
        t = [torch.randn(n, c, device="cuda") for _ in range(4)] + [torch.randn(c, c, device="cuda"), torch.rand(c, device="cuda")]
        return [v.requires_grad_(i != 3) for i, v in enumerate(t)]

    def step(t):
        x, f, _, g, w, v = t
        r, y = cxgnncomp.residual_norm(x, f, v, post="rms", pre="layer", pre_weight=v)
        out = cxgnncomp.linear(y, w, v, checkpoint="e4m3")
        return [r.detach(), out.detach()] + list(torch.autograd.grad((r, out), (x, f, w, v), (g, g)))

    a, b = make(20000, 128), make(3001, 260)
    announce("block alone")
    want = [step(a), step(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    announce("block on two streams")
    got = [[], []]
    for _ in range(5):
        for k, t in enumerate((a, b)):
            with torch.cuda.stream(streams[k]):
                got[k].append(step(t))
    torch.cuda.synchronize()
    for k in range(2):
        for res in got[k]:
            assert all(torch.equal(u, v) for u, v in zip(res, want[k]))
