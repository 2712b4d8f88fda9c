"""Rows held in 8 bits (csrc/packed_rows.hip, csrc/packed_wgrad.hip; cxgnncomp.pack_rows, PackedRows,
packed_weight_grad) against restatements in 64 bits.  Codes, exponents and unpacked values have to be
equal; the weight gradient keeps to a bound that counts its roundings (tests/packed_ref.py)."""
import pytest
import torch

import packed_ref
from conftest import announce
from rounding import B, check

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _rows(rows, cols, dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    if rows > 4:
        x[1] = 0.0
        x[2, : max(1, cols // 2)] *= 1e-4                # a wide range inside a group
        x[3] *= 1e-3
    return x.to(dtype)


# ----------------------------------------- on the CPU ------------------------------------------- #
def test_restatement_rounds_to_the_nearest_code():
    """No other code of the group's scale is nearer, and no smaller scale holds the group."""
    for fmt in ("int8", "e4m3"):
        x = _rows(9, 200, seed=3).double()
        codes, exps, values = packed_ref.pack(x, fmt)
        every = torch.arange(256, dtype=torch.int64).to(torch.uint8)
        grid = (every.view(torch.int8) if fmt == "int8" else every.view(torch.float8_e4m3fn)).double()
        grid = grid[torch.isfinite(grid) & (grid.abs() <= (127 if fmt == "int8" else 448))]
        s = packed_ref.spread(exps, 200)
        best = (x.unsqueeze(2) / s.unsqueeze(2) - grid).abs().min(dim=2).values
        assert torch.equal(best, ((x - values) / s).abs())
        tops = torch.nn.functional.pad(x, (0, 56)).view(9, 2, 128).abs().amax(dim=2)
        k = exps.double() - 127
        low = k > -111
        for top, e in zip(tops[low].tolist(), k[low].tolist()):
            t = torch.tensor([top], dtype=torch.float64)
            assert packed_ref._fits(t, fmt, e).item() and not packed_ref._fits(t, fmt, e - 1).item()


def test_library_refuses_bad_arguments():
    from cxgnncomp_backend import _lib
    lib = _lib.load()
    assert [lib.cxg_packed_pitch(c) for c in (0, 1, 16, 17, 128)] == [0, 16, 16, 32, 128]
    assert [lib.cxg_packed_groups(c) for c in (0, 1, 128, 129)] == [0, 1, 1, 2]

    def pack(x=256, ldx=8, type=0, fmt=0, rows=1, cols=8, codes=256, exps=256):
        return lib.cxg_pack_rows(x, ldx, type, fmt, rows, cols, codes, exps, None)

    for kw, status in ((dict(rows=-1), -1), (dict(cols=0), -1), (dict(type=3), -1), (dict(fmt=2), -1), (dict(x=None), -1),
                       (dict(codes=None), -1), (dict(exps=None), -1), (dict(codes=264), -1), (dict(x=258), -1), (dict(ldx=-1), -1),
                       (dict(cols=(1 << 22) + 1), -2)):
        assert pack(**kw) == status, kw
    assert pack(rows=0, x=None, codes=None, exps=None) == 0

    def unpack(codes=256, exps=256, fmt=0, rows=1, cols=8, out=256, type=0):
        return lib.cxg_unpack_rows(codes, exps, fmt, rows, cols, out, type, None)

    for kw in (dict(codes=None), dict(exps=None), dict(out=None), dict(out=257), dict(codes=257), dict(fmt=-1), dict(type=-1)):
        assert unpack(**kw) == -1, kw

    need = lib.cxg_packed_wgrad_workspace_bytes(10, 8, 8, 1)

    def wgrad(codes=256, a_rows=10, g=256, g_type=0, g_rows=10, src=None, dst=None, seg=None, M=10, K=8, N=8, R=1, gw=256, ws=256,
              nbytes=need, ldg=8, fmt=0):
        return lib.cxg_packed_wgrad(codes, 256, fmt, a_rows, g, ldg, g_type, g_rows, src, dst, seg, M, K, N, R, gw, None, ws, nbytes, None)

    for kw, status in ((dict(M=-1), -1), (dict(K=0), -1), (dict(N=0), -1), (dict(R=0), -1), (dict(R=2), -1), (dict(gw=None), -1),
                       (dict(codes=None), -1), (dict(codes=260), -1), (dict(g=None), -1), (dict(g=258), -1), (dict(a_rows=9), -1),
                       (dict(g_rows=9), -1), (dict(g_type=7), -1), (dict(fmt=5), -1), (dict(ldg=-8), -1), (dict(ws=None), -3),
                       (dict(ws=272), -3), (dict(nbytes=need - 1), -3), (dict(R=70000, seg=256), -2)):
        assert wgrad(**kw) == status, kw
    assert lib.cxg_packed_wgrad_workspace_bytes(-1, 8, 8, 1) == 0


def test_arguments_are_refused_on_the_host():
    import cxgnncomp
    with pytest.raises(ValueError, match="CUDA"):
        cxgnncomp.pack_rows(torch.zeros(3, 4))
    with pytest.raises(ValueError, match="int8"):
        cxgnncomp.pack_rows(torch.zeros(3, 4), "int4")
    with pytest.raises(TypeError):
        cxgnncomp.pack_rows([1.0])


# ------------------------------------------ on the GPU ------------------------------------------- #
@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1, 1), (5, 3), (33, 16), (300, 32), (41, 33), (70, 47), (64, 128), (31, 129), (9, 300), (257, 512), (3, 4100), (0, 8)])
def test_pack_and_unpack(shape, dtype, fmt):
    import cxgnncomp
    x = _rows(*shape, dtype=dtype, seed=shape[1])
    announce("pack_rows %s %s %s" % (shape, dtype, fmt))
    p = cxgnncomp.pack_rows(x.cuda(), fmt)
    codes, exps, values = packed_ref.pack(x, fmt)
    assert torch.equal(p.exps.cpu(), exps)
    assert torch.equal(p.codes.cpu(), codes)
    assert p.shape == x.shape and p.nbytes == codes.numel() + exps.numel()
    announce("unpack %s %s %s" % (shape, dtype, fmt))
    back = p.unpack()
    assert back.dtype == dtype and torch.equal(back.cpu(), values.to(dtype))
    assert torch.equal(p.unpack(F32).cpu().double(), values)
    assert torch.equal(p.unpack(BF16).cpu().double(), values)
    again = cxgnncomp.pack_rows(p.unpack(F32), fmt)
    assert torch.equal(again.unpack(F32).cpu().double(), values)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_borders_of_the_scales_and_codes(fmt):
    """Ties, the largest value that keeps a scale and the next one up, subnormal codes, the smallest and
    largest floats, negative zero."""
    import cxgnncomp
    top = 127.0 if fmt == "int8" else 448.0
    values = [0.5, 1.5, 2.5, -0.5, -1.5, 126.5, 63.5, 3.25, 17.0, 19.0, -17.0, 2 ** -9, 1.5 * 2 ** -9, 2 ** -10, -2 ** -10, 0.0, -0.0]
    x = torch.zeros(14, 130)
    for r in range(14):
        x[r, : len(values)] = torch.tensor(values)
        x[r, 100] = top
    one = torch.tensor(1.0)
    x[1, 100] = 127.5                                    # rounds to 128: the next scale
    x[2, 100] = torch.nextafter(127.5 * one, 0 * one)    # rounds to 127
    x[3, 100] = torch.nextafter(448 * one, 1000 * one)
    x[4] = 0.0
    x[4, 100] = 3.4028234663852886e38
    x[5] = 1e-40
    x[6] = 2.0 ** -111
    x[7] = 2.0 ** -120
    x[8] *= 2.0 ** -100
    x[9] *= 2.0 ** 100
    x[10] = 0.0
    x[11] = -x[11]
    announce("pack_rows borders %s" % fmt)
    p = cxgnncomp.pack_rows(x.cuda(), fmt)
    codes, exps, want = packed_ref.pack(x, fmt)
    assert torch.equal(p.exps.cpu(), exps)
    assert torch.equal(p.codes.cpu(), codes)
    # (the largest float rounds up to 2^128 in either format, which fp32 reads back as an infinity)
    assert torch.isinf(want.float()[4, 100]) and int(torch.isinf(want.float()).sum()) == 1
    assert torch.equal(p.unpack().cpu(), want.float())


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_groups_that_are_not_finite_read_back_as_nan(dtype, fmt):
    import cxgnncomp
    x = _rows(8, 300, dtype=dtype)
    x[0, 5], x[4, 290], x[5, 128] = float("inf"), float("nan"), float("-inf")
    announce("pack_rows not finite %s %s" % (dtype, fmt))
    p = cxgnncomp.pack_rows(x.cuda(), fmt)
    codes, exps, values = packed_ref.pack(x, fmt)
    assert torch.equal(p.exps.cpu(), exps) and torch.equal(p.codes.cpu(), codes)
    back = p.unpack(F32).cpu()
    bad = torch.zeros(8, 300, dtype=torch.bool)
    bad[0, :128] = bad[4, 256:] = bad[5, 128:256] = True
    assert torch.equal(torch.isnan(back), bad)
    assert torch.equal(back[~bad].double(), values[~bad])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pack_strided_rows(dtype):
    import cxgnncomp
    wide = _rows(40, 200, dtype=dtype).cuda()
    for name, x in (("columns 3..132", wide[:, 3:133]), ("every other row", wide[::2]), ("transposed", wide.t()),
                    ("one row for all", wide[:1].expand(12, 200)), ("one column", wide[:, 7:8])):
        announce("pack_rows " + name)
        p, q = cxgnncomp.pack_rows(x), cxgnncomp.pack_rows(x.contiguous())
        assert torch.equal(p.codes, q.codes) and torch.equal(p.exps, q.exps)
        assert torch.equal(p.codes.cpu(), packed_ref.pack(x.cpu(), "int8")[0])


def _wgrad_case(m, k, n, dtype=F32, fmt="int8", segs=1, maps=False, seed=0, rows_a=None, rows_g=None):
    gen = torch.Generator().manual_seed(seed + 7 * k + n)
    rows_a, rows_g = rows_a or m, rows_g or m
    codes, exps, values = packed_ref.pack(_rows(rows_a, k, seed=seed + 1), fmt)
    g = (torch.randn(rows_g, n, generator=gen) * 0.01).to(dtype)
    cuts = torch.sort(torch.randint(0, m + 1, (segs - 1, ), generator=gen)).values.tolist() if segs > 1 else []
    bounds = [0] + cuts + [m]
    src = torch.randint(0, rows_a, (m, ), generator=gen) if maps else None
    dst = torch.randint(0, rows_g, (m, ), generator=gen) if maps else None
    return codes, exps, values, g, bounds, src, dst


def _wgrad(case, k, fmt, with_seg=True):
    import cxgnncomp
    codes, exps, values, g, bounds, src, dst = case
    p = cxgnncomp.PackedRows(codes.cuda(), exps.cuda(), k, fmt)
    seg = torch.tensor(bounds).cuda() if with_seg else None
    return cxgnncomp.packed_weight_grad(p, g.cuda(), seg, src_idx=None if src is None else src.cuda(),
                                        dst_idx=None if dst is None else dst.cuda())


@gpu
@pytest.mark.parametrize("k,n", [(1, 1), (16, 3), (47, 64), (128, 128), (129, 47), (96, 160), (300, 130), (512, 256), (64, 64), (65, 65), (60, 3), (100, 1), (129, 64), (200, 1), (513, 2)])
@pytest.mark.parametrize("fmt,dtype", [("int8", F32), ("int8", BF16), ("int8", F16), ("e4m3", F32), ("e4m3", BF16), ("e4m3", F16)])
def test_weight_grad_shapes(k, n, fmt, dtype):
    for m in (33, 700):
        case = _wgrad_case(m, k, n, dtype, fmt)
        announce("packed_weight_grad %d x %d x %d %s %s" % (m, k, n, fmt, dtype))
        got = _wgrad(case, k, fmt, with_seg=False)
        check(got, packed_ref.weight_grad(case[2], case[3], [0, m]), F32, "gw")


@gpu
@pytest.mark.parametrize("m", [0, 1, 2, 31, 32, 33, 128, 129, 5000])
@pytest.mark.parametrize("segs,maps", [(1, False), (1, True), (5, False), (5, True), (40, True)])
def test_weight_grad_rows_segments_and_maps(m, segs, maps):
    case = _wgrad_case(m, 60, 72, segs=segs, maps=maps and m > 0, seed=m)
    announce("packed_weight_grad %d rows, %d segments, maps %s" % (m, segs, maps))
    got = _wgrad(case, 60, "int8")
    check(got, packed_ref.weight_grad(case[2], case[3], case[4], case[5], case[6]), F32, "gw")


@gpu
@pytest.mark.parametrize("k,n", [(60, 30), (100, 3), (100, 50), (300, 40), (300, 2), (300, 70)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_weight_grad_maps_at_every_tile_shape(k, n, dtype):
    """Row maps with entries outside their matrices, ragged segments and steps, strided rows of g."""
    import cxgnncomp
    m = 1500
    codes, exps, values, g, bounds, src, dst = _wgrad_case(m, k, n, dtype, segs=4, maps=True, seed=k)
    src[::13] = m
    dst[5::17] = -1
    keep = (src < m) & (dst >= 0)
    wide = torch.zeros(m, n + 5, dtype=dtype)
    wide[:, 3:n + 3] = g
    announce("packed_weight_grad maps %d x %d %s" % (k, n, dtype))
    p = cxgnncomp.PackedRows(codes.cuda(), exps.cuda(), k)
    gw, gb = cxgnncomp.packed_weight_grad(p, wide.cuda()[:, 3:n + 3], torch.tensor(bounds).cuda(), src_idx=src.cuda(),
                                          dst_idx=dst.cuda(), want_sums=True)
    rows = [torch.arange(a, b)[keep[a:b]] for a, b in zip(bounds, bounds[1:])]
    cuts = [0]
    for r in rows:
        cuts.append(cuts[-1] + len(r))
    order = torch.cat(rows)
    check(gw, packed_ref.weight_grad(values, g, cuts, src[order], dst[order]), F32, "gw")
    for r, want in enumerate(packed_ref.row_sums(g, cuts, dst[order])):
        check(gb[r], want, F32, "sums of segment %d" % r)


@gpu
@pytest.mark.parametrize("m,n", [(0, 5), (1, 3), (33, 1), (700, 47), (5000, 72), (1300, 300)])
@pytest.mark.parametrize("k", [20, 140])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_row_sums_of_the_gradient(m, n, k, dtype):
    """want_sums: the sums of the rows of g that count, per segment, beside the same weight gradient."""
    import cxgnncomp
    codes, exps, values, g, bounds, src, dst = _wgrad_case(m, k, n, dtype, segs=3, maps=m > 0, seed=m)
    p = cxgnncomp.PackedRows(codes.cuda(), exps.cuda(), k)
    maps = {}
    keep = None
    if m > 0:
        src[::7] = -1
        dst[3::11] = m
        keep = (src >= 0) & (dst < m)
        maps = dict(src_idx=src.cuda(), dst_idx=dst.cuda())
    announce("packed_weight_grad sums %d x %d x %d %s" % (m, k, n, dtype))
    gw, gb = cxgnncomp.packed_weight_grad(p, g.cuda(), torch.tensor(bounds).cuda(), want_sums=True, **maps)
    assert tuple(gb.shape) == (3, n)
    for r, want in enumerate(packed_ref.row_sums(g, bounds, dst, keep)):
        check(gb[r], want, F32, "sums of segment %d" % r)
    assert torch.equal(gw, cxgnncomp.packed_weight_grad(p, g.cuda(), torch.tensor(bounds).cuda(), **maps))
    gw, gb = cxgnncomp.packed_weight_grad(p, g.cuda(), want_sums=True)
    check(gb[0], packed_ref.row_sums(g, [0, m])[0], F32, "sums of all rows")


@gpu
def test_weight_grad_maps_of_other_lengths_and_padding():
    """Maps into matrices of other lengths; entries outside them leave their row out, memory is not
    touched there; rows behind the last segment and before the first do not count."""
    m, k, n = 900, 130, 50
    case = list(_wgrad_case(m, k, n, segs=3, maps=True, rows_a=77, rows_g=41))
    case[5][::9], case[5][4::31], case[6][5::17], case[6][7::41] = -1, 77, 1 << 40, -(1 << 40)
    case[4] = [10] + case[4][1:-1] + [m - 5]
    case[4] = sorted(case[4])
    announce("packed_weight_grad padding")
    got = _wgrad(case, k, "int8")
    check(got, packed_ref.weight_grad(case[2], case[3], case[4], case[5], case[6]), F32, "gw")
    for which in (5, 6):
        one = list(case)
        one[5 if which == 6 else 6] = None
        one[0], one[1], one[2] = (t[:77] for t in one[:3])
        if which == 6:                                   # src missing: row i of 77
            one[6] = one[6][:77]
            one[4] = [0, 30, 77]
        else:
            one[5] = one[5][:41]
            one[4] = [0, 30, 41]
        announce("packed_weight_grad one map")
        check(_wgrad(one, k, "int8"), packed_ref.weight_grad(one[2], one[3], one[4], one[5], one[6]), F32, "gw one map")


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_weight_grad_strided_and_unaligned_gradient(dtype):
    import cxgnncomp
    codes, exps, values, g, bounds, _, _ = _wgrad_case(200, 128, 90, dtype)
    p = cxgnncomp.PackedRows(codes.cuda(), exps.cuda(), 128)
    want = packed_ref.weight_grad(values, g, bounds)
    for name, lay in (("columns 1..90 of 93", lambda a: torch.nn.functional.pad(a, (1, 2))[:, 1:91]),
                      ("transposed", lambda a: a.t().contiguous().t()), ("plain", lambda a: a)):
        announce("packed_weight_grad %s %s" % (name, dtype))
        check(cxgnncomp.packed_weight_grad(p, lay(g.cuda())), want, F32, name)
    announce("packed_weight_grad one row for all")
    one = g[:1].expand(200, 90)
    check(cxgnncomp.packed_weight_grad(p, g[:1].cuda().expand(200, 90)), packed_ref.weight_grad(values, one, bounds), F32, "expanded")


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_weight_grad_over_many_rows(dtype):
    """Long chunks: the 2-norm of the error stays where fp32 accumulation of chunks of a few thousand rows
    puts it (random roundings: U * sqrt(products of a chunk) of the result, here 2^-24 * sqrt(3 * 4096) = 7e-6)."""
    import cxgnncomp
    m, k, n = 400000, 128, 96
    torch.manual_seed(0)
    x = torch.randn(m, k, device="cuda")
    g = torch.randn(m, n, device="cuda").to(dtype)
    announce("packed_weight_grad %d rows %s" % (m, dtype))
    p = cxgnncomp.pack_rows(x)
    got = cxgnncomp.packed_weight_grad(p, g)[0]
    want = p.unpack().double().t() @ g.double()
    assert float((got - want).norm() / want.norm()) < 7e-6
    assert torch.equal(got, cxgnncomp.packed_weight_grad(p, g)[0])
    # the bits of a segment do not depend on other segments' being there
    perm = torch.randperm(m, device="cuda")
    a = cxgnncomp.packed_weight_grad(p, g, torch.tensor([0, 1000, m], device="cuda"), perm, perm)
    assert torch.equal(a, cxgnncomp.packed_weight_grad(p, g, torch.tensor([0, 1000, m], device="cuda"), perm, perm))
    assert float((a.sum(0) - want).norm() / want.norm()) < 1.4e-5


@gpu
def test_weight_grad_of_groups_that_are_not_finite():
    import cxgnncomp
    x = _rows(50, 200)
    x[7, 150] = float("nan")
    g = torch.randn(50, 33)
    announce("packed_weight_grad NaN group")
    got = cxgnncomp.packed_weight_grad(cxgnncomp.pack_rows(x.cuda()), g.cuda())[0].cpu()
    assert torch.isnan(got[128:]).all() and torch.isfinite(got[:128]).all()
    g[3, 4], g[9, 20] = float("nan"), float("inf")
    announce("packed_weight_grad gradient not finite")
    got = cxgnncomp.packed_weight_grad(cxgnncomp.pack_rows(_rows(50, 200).cuda()), g.cuda())[0].cpu()
    bad = ~torch.isfinite(got)
    assert bad[:, 4].all() and bad[:, 20].all() and int(bad.sum()) == 400


@gpu
def test_another_stream_and_a_replayed_graph():
    import cxgnncomp
    m, k, n = 3000, 130, 70
    torch.manual_seed(1)
    x, g = torch.randn(m, k, device="cuda"), torch.randn(m, n, device="cuda")
    seg = torch.tensor([0, 1700, m], device="cuda")
    perm = torch.randperm(m, device="cuda")

    def step():
        p = cxgnncomp.pack_rows(x, "e4m3")
        return p.codes, p.exps, p.unpack(), cxgnncomp.packed_weight_grad(p, g, seg, perm, perm)

    announce("packed rows on a side stream")
    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    announce("packed rows captured")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        x.mul_(1.1)
        g.add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in held]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager))


@gpu
def test_refusals():
    import cxgnncomp
    x = torch.zeros(6, 20, device="cuda")
    p = cxgnncomp.pack_rows(x)
    for bad in (x.double(), x.int(), x[0], x[:, :0]):
        with pytest.raises(ValueError):
            cxgnncomp.pack_rows(bad)
    with pytest.raises(ValueError):
        p.unpack(torch.float64)
    seg, ids = torch.tensor([0, 6], device="cuda"), torch.arange(6, device="cuda")
    wg = cxgnncomp.packed_weight_grad
    for args, kw in (((p, x[:5]), {}), ((p, x.double()), {}), ((p, x.cpu()), {}), ((p, x, seg.int()), {}), ((p, x, seg[:1]), {}),
                     ((p, x, seg.cpu()), {}), ((p, x, seg), dict(src_idx=ids.int())), ((p, x, seg), dict(src_idx=ids, dst_idx=ids[:5])),
                     ((p, x[:3], seg), dict(src_idx=ids)), ((p, x[:, :0]), {}), ((p, x[0]), {}),
                     ((cxgnncomp.PackedRows(p.codes, p.exps, 40), x), {}), ((cxgnncomp.PackedRows(p.codes[:5], p.exps, 20), x), {}),
                     ((cxgnncomp.PackedRows(p.codes.char(), p.exps, 20), x), {}),
                     ((cxgnncomp.PackedRows(p.codes.repeat(1, 2)[:, :32], p.exps, 20), x), {})):
        with pytest.raises(ValueError):
            wg(*args, **kw)
