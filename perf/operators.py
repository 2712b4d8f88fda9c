"""Residual norms, 8-bit rows and the products that read them: what is measured, and each in plain torch.

Four operators of the training path of deep graph models:

  residual_norm       r = res_scale * x + branch_scale * gate * post(f),  y = pre(r); forward and backward
  pack_rows           rows in 8 bits with a power of two per row and 128 columns, and their reading back
  packed_weight_grad  gW[t] = sum over the rows i of type t of A[i]^T (x) G[i], A held in 8 bits
  linear              x W^T + b whose input is kept for the backward pass in 8 bits; forward and backward

A row of a layer or rms norm is normalised over its columns (eps 1e-5 under the root).  In 8 bits, 128 columns of
a row share the scale 2^k, k the smallest exponent (at least -111) with which the largest magnitude fits: at most
127 after rounding (int8) or at most 448 (e4m3).
"""
import math
import os
import sys

import torch
import torch.nn.functional as F

own = False

EPS = 1e-5
GROUP = 128
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}
MIN_EXP = 16                     # smallest biased exponent of a scale: 2^-111


def _framework():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cxgnn-compute_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import cxgnncomp
    return cxgnncomp


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #
def _norm(rows, cols, stream="fp32", branch="fp32", post="layer", pre="layer", gate="channel", train=True):
    return {"op": "norm", "rows": rows, "cols": cols, "stream": stream, "branch": branch, "post": post, "pre": pre,
            "gate": gate, "train": train}


def _pack(rows, cols, dtype="fp32", fmt="int8", back=False):
    return {"op": "pack", "rows": rows, "cols": cols, "dtype": dtype, "fmt": fmt, "back": back}


def _wgrad(rows, cols, outs, types, dtype="fp32", fmt="int8"):
    return {"op": "wgrad", "rows": rows, "cols": cols, "outs": outs, "types": types, "dtype": dtype, "fmt": fmt}


def _linear(rows, cols, outs, fmt="int8"):
    return {"op": "linear", "rows": rows, "cols": cols, "outs": outs, "fmt": fmt}


def listed():
    cases = [
        # one node's embedding is refreshed by a served model: latency of a single row
        ("norm serve 1x128", _norm(1, 128, train=False)),
        # the inner layer of a sampled mini-batch
        ("norm batch 1024x256", _norm(1024, 256)),
        # class-count wide head on a full graph: odd rows, a learned gate for each node
        ("norm ragged 70001x47", _norm(70001, 47, post="rms", gate="row")),
        # hidden layer of the full-graph model with 169,343 nodes
        ("norm full 169343x256", _norm(169343, 256)),
        # layer of the 2.45 M node graph in bf16 with an element-wise gate
        ("norm full 2449029x128 bf16", _norm(2449029, 128, "bf16", "bf16", "rms", "rms", "full")),
        # input of a layer put away for its backward pass on the 2.45 M node graph
        ("pack int8 2449029x128", _pack(2449029, 128)),
        # bf16 rows put away and read back, hidden width of the 169,343 node model
        ("pack e4m3 169343x256 bf16", _pack(169343, 256, "bf16", "e4m3", True)),
        # a small head's input, odd width, put away and read back
        ("pack int8 1000x47", _pack(1000, 47, back=True)),
        # weight gradient of a relational layer: 16 relations over 1 M rows in relation order
        ("wgrad typed 1000000x128x128 bf16", _wgrad(1000000, 128, 128, 16, "bf16", "e4m3")),
        # the wide typed product, an edge list of 2.33 M rows and 7 relations
        ("wgrad typed 2332486x512x512", _wgrad(2332486, 512, 512, 7)),
        # a training step of the full-graph model's first linear layer
        ("linear step 169343x128x256", _linear(169343, 128, 256)),
        # a training step of a mini-batch's output layer
        ("linear step 5000x256x47", _linear(5000, 256, 47, "e4m3")),
    ]
    return [dict(c, name=name) for name, c in cases]


def _spread(rng, low, high):
    """Whole number between low and high, uniform in its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm", "pack", "wgrad", "linear"])
    if op == "norm":
        cols = _spread(rng, 3, 2500)
        if rng.random() < 0.6:
            cols = max(4, cols // 4 * 4)
        rows = _spread(rng, 1, max(1, min(2500000, 200000000 // cols)))
        stream = rng.choice(["fp32", "fp32", "bf16", "fp16"])
        branch = rng.choice(["bf16", "fp32"]) if stream == "fp32" else stream
        return _norm(rows, cols, stream, branch, rng.choice(["layer", "rms", "none"]), rng.choice(["layer", "rms"]),
                     rng.choice(["none", "channel", "row", "full"]), rng.random() < 0.8)
    if op == "pack":
        cols = _spread(rng, 3, 2500)
        rows = _spread(rng, 1, max(1, min(2500000, 300000000 // cols)))
        return _pack(rows, cols, rng.choice(["fp32", "bf16", "fp16"]), rng.choice(["int8", "e4m3"]), True)
    if op == "wgrad":
        cols, outs = _spread(rng, 5, 600), _spread(rng, 5, 600)
        rows = _spread(rng, 1, max(1, min(2000000, 400000000000 // (cols * outs))))
        return _wgrad(rows, cols, outs, rng.choice([1, 3, 7, 16]), rng.choice(["fp32", "bf16", "fp16"]),
                      rng.choice(["int8", "e4m3"]))
    cols, outs = _spread(rng, 5, 600), _spread(rng, 5, 600)
    rows = _spread(rng, 1, max(1, min(1000000, 200000000000 // (cols * outs))))
    return _linear(rows, cols, outs, rng.choice(["int8", "e4m3"]))


def work(case):
    m, c = case["rows"], case["cols"]
    if case["op"] == "norm":
        sx, sf = SIZES[case["stream"]], SIZES[case["branch"]]
        gate = {"none": 0, "channel": 4 * c, "row": m * sf, "full": m * c * sf}[case["gate"]]
        nbytes = m * c * (2 * sx + 2 * sf) + gate + 16 * c
        flops = 16 * m * c
        if case["train"]:
            nbytes += m * c * (2 * sx + 2 * sf) + gate + 16 * c
            flops += 40 * m * c
        return {"bytes": nbytes, "flops": flops}
    held = m * c + m * -(-c // GROUP)
    if case["op"] == "pack":
        s = SIZES[case["dtype"]]
        return {"bytes": m * c * s + held + (m * c * s if case["back"] else 0), "flops": 4 * m * c}
    n = case["outs"]
    if case["op"] == "wgrad":
        index = 8 * m if case["types"] > 1 else 0
        return {"bytes": held + m * n * SIZES[case["dtype"]] + index + 4 * case["types"] * c * n, "flops": 2 * m * c * n}
    # x, g in; out, gx and the held rows out; the weight, its gradient and the bias
    return {"bytes": 4 * m * (2 * c + 2 * n) + held + 8 * c * n + 8 * n, "flops": 6 * m * c * n}


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def rand(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        t = torch.randn(shape, device="cuda", generator=gen)
        return t.mul_(scale).add_(shift).to(dtype)

    m, c = case["rows"], case["cols"]
    s = dict(case)
    if case["op"] == "norm":
        tx, tf = DTYPES[case["stream"]], DTYPES[case["branch"]]
        s["x"] = rand(m, c, dtype=tx, scale=1.5, shift=0.25)          # the stream has a drift
        s["f"] = rand(m, c, dtype=tf, scale=0.7)
        if m > 200:
            s["f"][::193] = 0                                         # nodes without edges aggregate to zero
        s["gate_kind"] = case["gate"]
        s["gate"] = {"none": lambda: None, "channel": lambda: rand(c, scale=0.1, shift=0.5),
                     "row": lambda: rand(m, 1, dtype=tf, scale=0.3, shift=0.5),
                     "full": lambda: rand(m, c, dtype=tf, scale=0.3, shift=0.5)}[case["gate"]]()
        for side in ("post", "pre"):
            kind = case[side]
            s[side + "_weight"] = None if kind == "none" else rand(c, scale=0.1, shift=1.0)
            s[side + "_bias"] = rand(c, scale=0.1) if kind == "layer" else None
        s["res_scale"], s["branch_scale"] = 0.9, 0.5
        if case["train"]:
            s["dr"], s["dy"] = rand(m, c, dtype=tx), rand(m, c, dtype=tf)
            for k in _leaves(s):
                s[k].requires_grad_(True)
        return s
    if case["op"] == "pack":
        spread = torch.exp(torch.randn((m, 1), device="cuda", generator=gen))      # rows of different size
        s["x"] = (rand(m, c) * spread).to(DTYPES[case["dtype"]])
        return s
    n = case["outs"]
    if case["op"] == "wgrad":
        t = case["types"]
        s["codes"], s["exps"] = _to_bits(rand(m, c, scale=2.0), case["fmt"])
        s["g"] = rand(m, n, dtype=DTYPES[case["dtype"]], scale=1e-2)
        s["perm"] = None
        if t > 1:
            types = torch.randint(0, t, (m,), device="cuda", generator=gen)
            s["perm"] = torch.sort(types, stable=True)[1]
            counts = torch.bincount(types, minlength=t)
        else:
            counts = torch.tensor([m], device="cuda")
        s["seg"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
        s["longest"] = int(counts.max())
        return s
    s["x"], s["g"] = rand(m, c).requires_grad_(True), rand(m, n, scale=1e-2)
    s["w"] = rand(n, c, scale=1.0 / math.sqrt(c)).requires_grad_(True)
    s["b"] = rand(n, scale=0.1).requires_grad_(True)
    return s


def _leaves(s):
    names = ["x", "f", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias"]
    return [k for k in names if s[k] is not None]


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #
def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"norm": _plain_norm, "pack": _plain_pack, "wgrad": _plain_wgrad, "linear": _plain_linear}[s["op"]](s)


def _run_own(s):
    fw = _framework()
    if s["op"] == "norm":
        r, y = fw.residual_norm(s["x"], s["f"], s["gate"], post=None if s["post"] == "none" else s["post"],
                                post_weight=s["post_weight"], post_bias=s["post_bias"], pre=s["pre"],
                                pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], res_scale=s["res_scale"],
                                branch_scale=s["branch_scale"], eps=EPS)
        if not s["train"]:
            return {"r": r, "y": y}
        names = _leaves(s)
        grads = torch.autograd.grad((r, y), [s[k] for k in names], (s["dr"], s["dy"]))
        return dict({"d_" + k: g for k, g in zip(names, grads)}, r=r.detach(), y=y.detach())
    if s["op"] == "pack":
        p = fw.pack_rows(s["x"], s["fmt"])
        if s["back"]:
            return {"exps": p.exps, "values": p.unpack()}
        return {"codes": p.codes, "exps": p.exps}
    if s["op"] == "wgrad":
        p = fw.PackedRows(s["codes"], s["exps"], s["cols"], s["fmt"])
        return fw.packed_weight_grad(p, s["g"], s["seg"], src_idx=s["perm"], dst_idx=s["perm"])
    out = fw.linear(s["x"], s["w"], s["b"], checkpoint=s["fmt"])
    gx, gw, gb = torch.autograd.grad(out, (s["x"], s["w"], s["b"]), s["g"])
    return {"out": out.detach(), "gx": gx, "gw": gw, "gb": gb}


# the plain forms ------------------------------------------------------------- #
def _standardise(v, kind):
    """(v - mean) / sqrt(var + eps) (layer) or v / sqrt(mean square + eps) (rms), and the factor."""
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt(v.square().mean(dim=1, keepdim=True) + EPS)
    return v * rstd, rstd


def _affine(v, w, b):
    v = v * w
    return v if b is None else v + b


def _standardise_back(g, xhat, rstd, kind):
    out = g - xhat * (g * xhat).mean(dim=1, keepdim=True)
    if kind == "layer":
        out = out - g.mean(dim=1, keepdim=True)
    return out * rstd


def _plain_norm(s):
    x, f = s["x"].float(), s["f"].float()
    gate = 1.0 if s["gate"] is None else s["gate"].float()
    fhat = rstd_f = None
    h = f
    if s["post"] != "none":
        fhat, rstd_f = _standardise(f, s["post"])
        h = _affine(fhat, s["post_weight"], s["post_bias"])
    r = s["res_scale"] * x + s["branch_scale"] * gate * h
    rhat, rstd_r = _standardise(r, s["pre"])
    y = _affine(rhat, s["pre_weight"], s["pre_bias"])
    out = {"r": r.to(s["x"].dtype), "y": y.to(s["f"].dtype)}
    if not s["train"]:
        return out
    dy = s["dy"].float()
    dr = s["dr"].float() + _standardise_back(dy * s["pre_weight"], rhat, rstd_r, s["pre"])
    out["d_pre_weight"] = (dy * rhat).sum(dim=0)
    if s["pre_bias"] is not None:
        out["d_pre_bias"] = dy.sum(dim=0)
    out["d_x"] = (s["res_scale"] * dr).to(s["x"].dtype)
    dh = s["branch_scale"] * gate * dr
    if s["gate"] is not None:
        dgate = s["branch_scale"] * dr * h
        if s["gate_kind"] == "channel":
            dgate = dgate.sum(dim=0)
        elif s["gate_kind"] == "row":
            dgate = dgate.sum(dim=1, keepdim=True)
        out["d_gate"] = dgate.to(s["gate"].dtype)
    if s["post"] != "none":
        out["d_post_weight"] = (dh * fhat).sum(dim=0)
        if s["post_bias"] is not None:
            out["d_post_bias"] = dh.sum(dim=0)
        dh = _standardise_back(dh * s["post_weight"], fhat, rstd_f, s["post"])
    out["d_f"] = dh.to(s["f"].dtype)
    return out


def _to_bits(x, fmt):
    """The held form of fp32 rows: codes [rows, cols rounded up to 16] and biased exponents [rows, groups], as bytes."""
    m, c = x.shape
    groups = -(-c // GROUP)
    x = F.pad(x, (0, groups * GROUP - c)).view(m, groups, GROUP)
    bits = x.abs().amax(dim=2).view(torch.int32)
    power, mantissa = bits >> 23, bits & 0x7FFFFF
    if fmt == "int8":                                     # 127.5 / 64 and more would round to 128
        exps = power - 6 + (mantissa >= 0x7F0000).int()
    else:                                                 # 448 = 1.75 * 2^8
        exps = power - 8 + (mantissa > 0x600000).int()
    exps = exps.clamp_(min=MIN_EXP)
    exps[power == 255] = 255                              # a group that is not finite
    v = x * ((254 - exps).clamp(min=0) << 23).view(torch.float32).unsqueeze(2)
    v = torch.where((exps == 255).unsqueeze(2), torch.zeros_like(v), v).view(m, groups * GROUP)
    v = v[:, :-(-c // 16) * 16].contiguous()
    codes = v.round_().to(torch.int8) if fmt == "int8" else v.to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), exps.to(torch.uint8)


def _from_bits(codes, exps, cols, fmt):
    v = (codes.view(torch.int8) if fmt == "int8" else codes.view(torch.float8_e4m3fn)).float()
    scale = (exps.int() << 23).view(torch.float32)
    return (v * scale.repeat_interleave(GROUP, dim=1)[:, :v.shape[1]])[:, :cols]


def _plain_pack(s):
    codes, exps = _to_bits(s["x"].float(), s["fmt"])
    if s["back"]:
        return {"exps": exps, "values": _from_bits(codes, exps, s["cols"], s["fmt"]).to(s["x"].dtype)}
    return {"codes": codes, "exps": exps}


def _plain_wgrad(s):
    a = _from_bits(s["codes"], s["exps"], s["cols"], s["fmt"])
    g = s["g"].float()
    if s["perm"] is None:
        return (a.t() @ g).unsqueeze(0)
    # the rows of every type, padded with a row of zeros to the longest type
    at = s["seg"][:-1, None] + torch.arange(s["longest"], device=a.device)
    rows = torch.where(at < s["seg"][1:, None], s["perm"][at.clamp(max=s["perm"].shape[0] - 1)], a.shape[0])
    a, g = F.pad(a, (0, 0, 0, 1))[rows], F.pad(g, (0, 0, 0, 1))[rows]
    return torch.bmm(a.transpose(1, 2), g)


def _plain_linear(s):
    out = s["x"] @ s["w"].t() + s["b"]
    held = _from_bits(*_to_bits(s["x"], s["fmt"]), s["cols"], s["fmt"])
    return {"out": out, "gx": s["g"] @ s["w"], "gw": s["g"].t() @ held, "gb": s["g"].sum(dim=0)}


# --------------------------------------------------------------------------- #
# the definitions in 64 bits
# --------------------------------------------------------------------------- #
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "pack": _exact_pack, "wgrad": _exact_wgrad, "linear": _exact_linear}[case["op"]](s)


def _exact_norm(s):
    names = _leaves(s)
    v = {k: s[k].detach().double().requires_grad_(s["train"]) for k in names}

    def normed(t, side):
        if s[side] == "none":
            return t
        if s[side] == "layer":
            var, mean = torch.var_mean(t, dim=1, unbiased=False, keepdim=True)
        else:
            var, mean = (t * t).sum(dim=1, keepdim=True) / t.shape[1], 0.0
        t = (t - mean) / torch.sqrt(var + EPS) * v[side + "_weight"]
        return t + v[side + "_bias"] if side + "_bias" in v else t

    branch = normed(v["f"], "post")
    if "gate" in v:
        branch = branch * v["gate"]
    r = s["res_scale"] * v["x"] + s["branch_scale"] * branch
    y = normed(r, "pre")
    if not s["train"]:
        return {"r": r, "y": y}
    loss = (r * s["dr"].double()).sum() + (y * s["dy"].double()).sum()
    grads = torch.autograd.grad(loss, [v[k] for k in names])
    return dict({"d_" + k: g for k, g in zip(names, grads)}, r=r.detach(), y=y.detach())


def _held_values(x, fmt):
    """What the 8-bit form of the rows stands for, and the biased exponents, in 64 bits."""
    m, c = x.shape
    v = F.pad(x.double(), (0, -c % GROUP)).view(m, -1, GROUP)
    top = v.abs().amax(dim=2)
    e = torch.frexp(top)[1].double()                       # top = f * 2^e, f in [0.5, 1)
    if fmt == "int8":
        k = e - 7
        k = torch.where(torch.round(top * torch.exp2(-k)) > 127, k + 1, k)
    else:
        k = e - 9
        k = torch.where(top * torch.exp2(-k) > 448, k + 1, k)
    k = k.clamp(min=MIN_EXP - 127.0)
    v = v * torch.exp2(-k).unsqueeze(2)
    if fmt == "int8":
        v = torch.round(v)
    else:                                                  # three bits behind the leading one, steps of 2^-9 at least
        step = torch.exp2((torch.frexp(v)[1].double() - 4).clamp(min=-9.0))
        v = torch.round(v / step) * step
    return (v * torch.exp2(k).unsqueeze(2)).view(m, -1)[:, :c], (k + 127).to(torch.uint8)


def _exact_pack(s):
    values, exps = _held_values(s["x"], s["fmt"])
    return {"exps": exps, "values": values if s["back"] else None, "codes": None}


def _exact_wgrad(s):
    raw = s["codes"].view(torch.int8 if s["fmt"] == "int8" else torch.float8_e4m3fn).float().double()[:, :s["cols"]]
    group = torch.arange(s["cols"], device=raw.device) // GROUP
    raw = raw * torch.exp2(s["exps"].double() - 127.0)[:, group]
    g, bounds = s["g"].double(), s["seg"].tolist()
    if s["perm"] is not None:
        raw, g = raw[s["perm"]], g[s["perm"]]
    return torch.stack([raw[b:e].t() @ g[b:e] for b, e in zip(bounds, bounds[1:])])


def _exact_linear(s):
    x, w, g = s["x"].detach().double(), s["w"].detach().double(), s["g"].double()
    held = _held_values(s["x"].detach(), s["fmt"])[0]
    return {"out": torch.addmm(s["b"].detach().double(), x, w.t()), "gx": g @ w, "gw": g.t() @ held, "gb": g.sum(dim=0)}
