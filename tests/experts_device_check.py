"""Child process of test_gpu_experts.py: runs every case of experts_cases.py (or those whose names
contain argv[1]) and prints a JSON line for each. Not collected by pytest.

Every oracle is plain numpy / torch on the CPU in 64 bits from the operator's formula. U32 is the
largest relative error of one float32 rounding, ROUND[dtype] that of the final one; a sum of n terms
in float32 is off by at most n U32 times the sum of the terms' magnitudes, and the kernels add at
most n / 64 terms to one lane and then join 64 lanes and at most 16 wavefronts."""
import json
import math
import os
import sys
import traceback

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from experts_cases import all_cases  # noqa: E402
from h2o4gpu_amd import codebook4, experts  # noqa: E402
from h2o4gpu_amd.libs import experts_hip, kmeans_hip  # noqa: E402

DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
U32 = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def near(got, want, bound, what):
    """|got - want| <= bound + the last rounding, element by element; NaN and infinities in the same places."""
    u, tiny = ROUND[got.dtype], TINY[got.dtype]
    g, w = got.detach().double().cpu(), want.double()
    assert g.shape == w.shape, "%s: shape %s, expected %s" % (what, tuple(g.shape), tuple(w.shape))
    fine = torch.isfinite(w)
    assert torch.equal(torch.isnan(g), torch.isnan(w)), "%s: NaN in other places" % what
    assert torch.equal(g[~fine & ~torch.isnan(w)], w[~fine & ~torch.isnan(w)]), "%s: infinities" % what
    b = torch.as_tensor(bound, dtype=torch.float64).expand(w.shape)
    off = (g - w).abs()
    allowed = b + u * (w.abs() + b) + tiny
    bad = fine & ~(off <= allowed)
    assert not bad.any(), "%s: %d of %d off, worst %.3g against %.3g allowed" % (
        what, int(bad.sum()), bad.numel(), float(off[bad].max()), float(allowed[bad].min()))


def same(got, want, what):
    assert torch.equal(got.cpu(), want), what


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def laid_out(t, layout):
    """The matrix on the GPU: as it is, in rows with a gap behind, or at an address off by one element."""
    if layout == "strided":
        wide = torch.full((t.shape[0], t.shape[1] + 16), float("nan") if t.is_floating_point() else 77,
                          dtype=t.dtype, device="cuda")
        wide[:, :t.shape[1]] = t.cuda()
        return wide[:, :t.shape[1]]
    if layout == "unaligned":
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.cuda().reshape(-1)
        return flat[1:].view(t.shape)
    return t.cuda()


# ---- route ---------------------------------------------------------------------------------------

def scores_of(c):
    g = gen(c["rows"] * 7 + c["experts"])
    s = torch.randn(c["rows"], c["experts"], generator=g)
    dt, data, worst = DT[c["dtype"]], c["data"], -math.inf if c["largest"] else math.inf
    pick = torch.rand(s.shape, generator=g)
    if data == "ties":
        s = torch.randint(0, 3, s.shape, generator=g).float()
        s[s == 0] = torch.where(pick < 0.5, 0.0, -0.0)[s == 0]
    elif data == "masked":
        s[pick < 0.7] = worst
    elif data == "all_masked":
        s[::2] = worst
        s[1::4, :1] = float("nan")
    elif data == "lowest":  # masks of the type's lowest value count as scores
        low = torch.finfo(dt).min if c["largest"] else torch.finfo(dt).max
        s = s.to(dt)
        s[pick < 0.8] = low
        s[::3] = low
    elif data == "nan":
        s[pick < 0.3] = float("nan")
    elif data == "best_infinity":
        s[pick < 0.2] = -worst
        s[pick > 0.9] = worst
    elif data == "wide":
        s = s * 60
    return s.to(dt)


def route_oracle(s, c, scale):
    """Choice and weights by the definition, and p over everything that shares the weight."""
    key = s.double() if c["largest"] else -s.double()
    key = torch.where(torch.isnan(key), -math.inf, key)
    rows, E, K = s.shape[0], s.shape[1], c["top_k"]
    index = torch.argsort(key, dim=1, descending=True, stable=True)[:, :K]
    picked = key.gather(1, index)
    free = picked > -math.inf
    top = picked[:, :1]
    diff = torch.where(key == top, 0.0, scale * (key - top) if scale else torch.zeros_like(key))
    term = torch.where(key > -math.inf, torch.exp(diff), 0.0)
    term = torch.where(free[:, :1], term, 0.0)
    if not c["over_all"]:
        keep = torch.zeros_like(term).scatter_(1, index, free.double())
        term = term * keep
    total = term.sum(1, keepdim=True)
    p = torch.where(total > 0, term / total, 0.0)
    chosen = torch.where(free, index, -1).to(torch.int32)
    return chosen, torch.where(free, p.gather(1, index), 0.0), p


def check_route(c):
    s = scores_of(c)
    scale = 0.0 if c["data"] == "scale0" else 1.0 if c["rows"] % 2 else 0.3
    if c["strided"] == 1:
        d = s.t().contiguous().cuda().t()
    elif c["strided"] == 2:
        wide = torch.full((2 * s.shape[0], 3 * s.shape[1]), float("nan"), dtype=s.dtype, device="cuda")
        d = wide[::2, ::3]
        d.copy_(s)
    else:
        d = s.cuda()
    d.requires_grad_()
    chosen, weights = experts.route(d, c["top_k"], largest=c["largest"], scale=scale, over_all=c["over_all"])
    want, w, p = route_oracle(s, c, scale)
    same(chosen, want, "experts")
    # a term's exponent is rounded once (|x| U32, and e^x is below 1 where |x| matters: x e^-x <= 0.37),
    # expf is within 2 ulp; sums of E terms; one division
    bound = U32 * (16 + c["experts"] / 32)
    near(weights, w, bound, "weights")
    g = torch.randn(weights.shape, generator=gen(5))
    ds, = torch.autograd.grad(weights, d, g.cuda())
    full = torch.zeros_like(p)
    free = want >= 0
    full.scatter_add_(1, torch.where(free, want, 0).long(), torch.where(free, g.double(), 0.0))
    inner = (p * full).sum(1, keepdim=True)
    sign = scale if c["largest"] else -scale
    dwant = sign * p * (full - inner)
    # p off by `bound` as above (relative to 1), inner by K roundings of sums of |p g|
    gmax = float(g.abs().max())
    near(ds, dwant, scale * gmax * (4 * bound + U32 * (8 + c["top_k"])), "gradient")
    # without a gradient wanted: the same bits
    again, w2 = experts.route(d.detach(), c["top_k"], largest=c["largest"], scale=scale, over_all=c["over_all"])
    assert torch.equal(again, chosen) and torch.equal(w2, weights), "the call without a gradient differs"


# ---- order ---------------------------------------------------------------------------------------

def choices(tokens, top_k, E, data, seed=3):
    rng = np.random.default_rng(seed + tokens + E)
    if data == "skewed":
        e = np.minimum((rng.exponential(0.05, (tokens, top_k)) * E).astype(np.int64), E - 1)
    elif data == "none":
        e = np.where(rng.random((tokens, top_k)) < 0.5, -1, E)
    elif data == "one":
        e = np.full((tokens, top_k), E - 1)
    else:
        e = rng.integers(0, E, (tokens, top_k))
        if data == "dropped":
            bad = rng.random((tokens, top_k))
            e = np.where(bad < 0.1, -1, np.where(bad < 0.2, E, np.where(bad < 0.22, 2 ** 31 - 1,
                                                                        np.where(bad < 0.24, -2 ** 31, e))))
    return e.astype(np.int32)


def order_oracle(e, E):
    flat = e.reshape(-1).astype(np.int64)
    key = np.where((flat >= 0) & (flat < E), flat, E)
    order = np.argsort(key, kind="stable")
    place = np.empty_like(order)
    place[order] = np.arange(order.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])])
    return (order.astype(np.int32), np.where(key < E, place, ~place).astype(np.int32).reshape(e.shape),
            offsets.astype(np.int32))


def check_sort(c):
    e = choices(c["tokens"], c["top_k"], c["experts"], c["data"])
    o = experts.sort_by_expert(torch.from_numpy(e).cuda(), c["experts"])
    order, position, offsets = order_oracle(e, c["experts"])
    same(o.offsets, torch.from_numpy(offsets), "offsets")
    same(o.order, torch.from_numpy(order), "order")
    same(o.position, torch.from_numpy(position), "position")


def _order(c):
    e = choices(c["tokens"], c["top_k"], c["experts"], "uniform")
    rng = np.random.default_rng(9)
    if c.get("dropped"):
        e = np.where(rng.random(e.shape) < c["dropped"], -1, e).astype(np.int32)
    o = experts.sort_by_expert(torch.from_numpy(e).cuda(), c["experts"])
    return e, o, torch.from_numpy(order_oracle(e, c["experts"])[1]).long()


# ---- rows out and back ------------------------------------------------------------------------------

def check_dispatch(c):
    e, o, pos = _order(c)
    T, K, d, dt = c["tokens"], c["top_k"], c["cols"], DT[c["dtype"]]
    x = torch.randn(T, d, generator=gen(1)).to(dt)
    dx = laid_out(x, c["layout"]).requires_grad_()
    rows = experts.dispatch(dx, o)
    want = torch.zeros(T * K, d, dtype=dt)
    kept = pos >= 0
    want[pos[kept]] = x[:, None, :].expand(T, K, d)[kept]
    same(rows, want, "rows")
    g = torch.randn(T * K, d, generator=gen(2)).to(dt)
    got, = torch.autograd.grad(rows, dx, laid_out(g, c["layout"]))
    parts = g.double()[pos.clamp_min(0)] * kept[:, :, None]
    near(got, parts.sum(1), K * U32 * parts.abs().sum(1), "gradient")


def check_combine(c):
    e, o, pos = _order(c)
    T, K, d, dt = c["tokens"], c["top_k"], c["cols"], DT[c["dtype"]]
    y = torch.randn(T * K, d, generator=gen(1)).to(dt)
    w = torch.randn(T, K, generator=gen(4))
    kept = pos >= 0
    # places without an expert hold anything
    held = int(kept.sum())
    y[held:] = float("nan")
    dy, dw = laid_out(y, c["layout"]).requires_grad_(), w.cuda().requires_grad_()
    out = experts.combine(dy, dw, o)
    parts = torch.where(kept[:, :, None], y.double()[pos.clamp_min(0)], 0.0)
    terms = parts * w.double()[:, :, None]
    near(out, terms.sum(1), (K + 1) * U32 * terms.abs().sum(1), "out")
    g = torch.randn(T, d, generator=gen(2)).to(dt)
    gy, gw = torch.autograd.grad(out, (dy, dw), laid_out(g, c["layout"]))
    want = torch.zeros(T * K, d, dtype=torch.float64)
    want[pos[kept]] = (w.double()[:, :, None] * g.double()[:, None, :])[kept]
    near(gy, want, U32 * want.abs(), "gradient of the rows")
    prod = parts * g.double()[:, None, :]
    near(gw, prod.sum(2), (d / 64 + 24) * U32 * prod.abs().sum(2), "gradient of the weights")


# ---- 4-bit products -----------------------------------------------------------------------------------

def matrix(c, lead):
    N, K, group = c["out"], c["cols"], c["group"]
    g = gen(N + K)
    dt, sdt = DT[c["dtype"]], DT[c.get("scale_dtype", c["dtype"])]
    nbytes = (K + 1) // 2
    if c["layout"] == "plain":
        nbytes = (nbytes + 15) // 16 * 16
    codes = torch.randint(0, 256, lead + (N, nbytes), generator=g, dtype=torch.uint8)
    scales = (torch.rand(lead + (N, -(-K // group)), generator=g) - 0.3).to(sdt)
    book = torch.randn((lead if c.get("books") else ()) + (16,), generator=g).to(dt)
    dcodes = codes.cuda()
    if c["layout"] == "unaligned":
        flat = torch.empty(codes.numel() + 3, dtype=torch.uint8, device="cuda")
        flat[3:] = dcodes.reshape(-1)
        dcodes = flat[3:].view(codes.shape)
    w = codebook4.Codebook4(dcodes, scales.cuda(), book.cuda(), K, group)
    k = torch.arange(K)
    code = (codes[..., k // 2].long() >> (4 * (k % 2))) & 15
    if book.dim() == 2:
        values = torch.stack([book[e].double()[code[e]] for e in range(lead[0])])
    else:
        values = book.double()[code]
    return w, values * scales.double()[..., k // group]


def product_bound(x, W):
    """Sum of |w x| times what rounds: w * scale once, the products' sums (at most K / 64 + 32 to a lane or
    matrix instruction, 32 lanes' and 16 wavefronts' joins), twice over for the order inside an instruction."""
    return 2 * U32 * (W.shape[-1] / 64 + 80) * (x.double().abs() @ W.abs().transpose(-1, -2))


def check_product(c):
    w, W = matrix(c, ())
    x = torch.randn(c["rows"], c["cols"], generator=gen(6)).to(DT[c["dtype"]])
    y = codebook4.product(laid_out(x, c["layout"]), w)
    near(y, x.double() @ W.t(), product_bound(x, W), "y")
    deq = w.dequantize().cpu().double()
    assert torch.all((deq - W).abs() <= U32 * W.abs()), "dequantize"


def check_experts_product(c):
    e, o, pos = _order(c)
    w, W = matrix(c, (c["experts"],))
    T, K = c["tokens"], c["top_k"]
    x = torch.randn(T, c["cols"], generator=gen(6)).to(DT[c["dtype"]])
    y = codebook4.experts_product(laid_out(x, c["layout"]), w, o)
    want = torch.zeros(T * K, c["out"], dtype=torch.float64)
    bound = torch.zeros_like(want)
    for t in range(T):
        for j in range(K):
            p = int(pos[t, j])
            if p >= 0:
                want[p] = W[e[t, j]] @ x[t].double()
                bound[p] = product_bound(x[t:t + 1], W[e[t, j]])[0]
    near(y, want, bound, "y")


def check_quantize(c):
    dt, sdt = DT[c["dtype"]], DT[c["scale_dtype"]]
    N, K, group = c["out"], c["cols"], c["group"]
    W = torch.randn(N, K, generator=gen(8))
    if c["data"] == "zeros":
        W[:, : K // 2] = 0
        W[0] = 0
    elif c["data"] == "huge":
        W = W * (3e38 if dt != torch.float16 else 6e4)
        W = W.clamp(-torch.finfo(dt).max, torch.finfo(dt).max)
    elif c["data"] == "nan":
        W[::2, ::3] = float("nan")
    W = W.to(dt)
    book = torch.sort(torch.randn(16, generator=gen(9))).values.to(dt)
    top = 1.0 if c["data"] != "huge" else 2.0
    q = codebook4.quantize(W.cuda(), group, book.cuda(), top=top, scale_dtype=sdt)
    groups = -(-K // group)
    codes, scales = q.codes().cpu(), q.scales().cpu()
    assert q.dtype == dt and scales.dtype == sdt
    for g in range(groups):
        part = W[:, g * group:(g + 1) * group]
        most = torch.nan_to_num(part.double().abs(), nan=0.0, posinf=math.inf).amax(1)
        want = (most.float() / top).to(sdt)
        want = torch.where((want > 0) & torch.isfinite(want), want, torch.ones_like(want))
        same(scales[:, g], want, "scales")
        v = part.float() / want.float()[:, None]
        off = (v[:, :, None] - book.float()).abs()
        off = torch.where(torch.isnan(off), math.inf, off)
        code = torch.argmin(off, 2)
        k = torch.arange(g * group, min(K, (g + 1) * group))
        same(codes[:, k].long(), code, "codes")


# ---- single checks ------------------------------------------------------------------------------------

def check_differences_route(_):
    """(f(s + h v) - f(s - h v)) / 2h against the gradient: f's float32 values are off by U32 (16 + E / 32) a
    weight, the difference's third-order term by h^2 / 6 times a third derivative of at most 6 |v|^3 scale^3."""
    for largest in (True, False):
        for over_all in (True, False):
            E, K, T, h, scale = 24, 4, 6, 2.0 ** -6, 0.7
            s = torch.randn(T, E, generator=gen(11)) * 2
            v = torch.randn(T, E, generator=gen(12))
            g = torch.randn(T, K, generator=gen(13))
            d = s.cuda().requires_grad_()
            e0, w = experts.route(d, K, largest=largest, scale=scale, over_all=over_all)
            ds, = torch.autograd.grad(w, d, g.cuda())
            up, wu = experts.route((s + h * v).cuda(), K, largest=largest, scale=scale, over_all=over_all)
            dn, wd = experts.route((s - h * v).cuda(), K, largest=largest, scale=scale, over_all=over_all)
            fixed = ((up == e0) & (dn == e0)).all(1).cpu()  # the choice held: rows where it did
            assert int(fixed.sum()) >= 2
            est = ((wu - wd).double().cpu() * g.double()).sum(1) / (2 * h)
            want = (ds.double().cpu() * v.double()).sum(1)
            vmax, gsum = float(v.abs().max()), g.abs().sum(1).double()
            tol = gsum * (U32 * (16 + E / 32) * 2 / (2 * h) + h * h * (scale * vmax) ** 3) + 1e-6
            assert ((est - want).abs()[fixed] <= tol[fixed]).all(), (est, want, tol)


def check_differences_rows(_):
    """dispatch and combine are linear: differences have no truncation, only float32 roundings."""
    T, K, E, d = 9, 3, 5, 37
    e = choices(T, K, E, "dropped")
    o = experts.sort_by_expert(torch.from_numpy(e).cuda(), E)
    x, v = torch.randn(T, d, generator=gen(1)), torch.randn(T, d, generator=gen(2))
    g = torch.randn(T * K, d, generator=gen(3))
    dx = x.cuda().requires_grad_()
    grad, = torch.autograd.grad(experts.dispatch(dx, o), dx, g.cuda())
    diff = (experts.dispatch((x + v).cuda(), o) - experts.dispatch((x - v).cuda(), o)).double().cpu() / 2
    est, want = (diff * g.double()).sum(), (grad.double().cpu() * v.double()).sum()
    size = float((g.abs().sum() * (x.abs().max() + v.abs().max())))
    assert abs(est - want) <= 8 * U32 * size, (est, want)
    y, vy = torch.randn(T * K, d, generator=gen(4)), torch.randn(T * K, d, generator=gen(5))
    w, vw = torch.randn(T, K, generator=gen(6)), torch.randn(T, K, generator=gen(7))
    g = torch.randn(T, d, generator=gen(8))
    dy, dw = y.cuda().requires_grad_(), w.cuda().requires_grad_()
    gy, gw = torch.autograd.grad(experts.combine(dy, dw, o), (dy, dw), g.cuda())
    size = float(g.abs().sum() * K * (y.abs().max() + vy.abs().max()) * (w.abs().max() + vw.abs().max()))
    for a, b, c, f, grad, dirn in ((y + vy, y - vy, w, w, gy, vy), (y, y, w + vw, w - vw, gw, vw)):
        diff = (experts.combine(a.cuda(), c.cuda(), o) - experts.combine(b.cuda(), f.cuda(), o)).double().cpu() / 2
        est, want = (diff * g.double()).sum(), (grad.double().cpu() * dirn.double()).sum()
        assert abs(est - want) <= 64 * U32 * size, (est, want)


def refuses(kind, f, *args, **kw):
    try:
        f(*args, **kw)
    except kind:
        return
    raise AssertionError("%s%s was not refused with %s" % (f.__name__, args[1:], kind.__name__))


def check_refusals(_):
    s = torch.randn(4, 8, device="cuda")
    refuses(ValueError, experts.route, s.cpu(), 2)
    refuses(TypeError, experts.route, s.double(), 2)
    refuses(TypeError, experts.route, [[1.0]], 1)
    refuses(ValueError, experts.route, s[0], 2)
    refuses(ValueError, experts.route, s, 0)
    refuses(ValueError, experts.route, s, 9)
    refuses(ValueError, experts.route, torch.zeros(1, 100, device="cuda"), 65)
    refuses(ValueError, experts.route, s[:, :0], 1)
    refuses(ValueError, experts.route, torch.zeros(1, 16385, device="cuda"), 1)
    refuses(ValueError, experts.route, s, 2, scale=-1.0)
    refuses(ValueError, experts.route, s, 2, scale=float("nan"))
    refuses(ValueError, experts.route, s, 2, scale=float("inf"))
    e = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    refuses(TypeError, experts.sort_by_expert, e.long(), 8)
    refuses(ValueError, experts.sort_by_expert, e.cpu(), 8)
    refuses(ValueError, experts.sort_by_expert, e, 0)
    refuses(ValueError, experts.sort_by_expert, e, 16385)
    refuses(ValueError, experts.sort_by_expert, torch.zeros(2, 65, dtype=torch.int32, device="cuda"), 8)
    o = experts.sort_by_expert(e, 8)
    x = torch.randn(4, 16, device="cuda")
    refuses(ValueError, experts.dispatch, x[:3], o)
    refuses(ValueError, experts.dispatch, x[:, :0], o)
    refuses(ValueError, experts.dispatch, torch.randn(4, 32, device="cuda")[:, ::2], o)
    refuses(ValueError, experts.dispatch, x[:1].expand(4, 16), o)
    refuses(TypeError, experts.dispatch, x, e)
    refuses(TypeError, experts.dispatch, x.double(), o)
    y, w = torch.randn(8, 16, device="cuda"), torch.rand(4, 2, device="cuda")
    refuses(ValueError, experts.combine, y[:7], w, o)
    refuses(ValueError, experts.combine, y, w[:3], o)
    refuses(TypeError, experts.combine, y, w.half(), o)
    refuses(ValueError, experts.combine, y, w.cpu(), o)
    codes = torch.zeros(6, 32, dtype=torch.uint8, device="cuda")
    scales, book = torch.ones(6, 2, device="cuda"), torch.randn(16, device="cuda")
    make = codebook4.Codebook4
    m = make(codes, scales, book, 64, 32)
    refuses(TypeError, make, codes.int(), scales, book, 64, 32)
    refuses(ValueError, make, codes, scales, book, 65, 32)
    refuses(ValueError, make, codes, scales, book, 64, 48)
    refuses(ValueError, make, codes, scales, book, 64, 64)
    refuses(ValueError, make, codes, scales, book[:15], 64, 32)
    refuses(ValueError, make, codes, scales.cpu(), book, 64, 32)
    refuses(TypeError, make, codes, scales.double(), book, 64, 32)
    refuses(ValueError, make, codes, scales, torch.zeros(6, 16, device="cuda"), 64, 32)
    x = torch.randn(4, 64, device="cuda")
    refuses(ValueError, codebook4.product, x[:, :63], m)
    refuses(TypeError, codebook4.product, x.half(), m)
    refuses(TypeError, codebook4.product, x, codes)
    refuses(ValueError, codebook4.product, x.clone().requires_grad_(), m)
    refuses(ValueError, codebook4.experts_product, x, m, o)
    many = make(codes.expand(8, 6, 32).contiguous(), scales.expand(8, 6, 2).contiguous(), book, 64, 32)
    refuses(ValueError, codebook4.product, x, many)
    refuses(ValueError, codebook4.experts_product, x[:3], many, o)
    refuses(ValueError, codebook4.experts_product, x, many, experts.sort_by_expert(e, 7))
    W = torch.randn(4, 64, device="cuda")
    refuses(ValueError, codebook4.quantize, W, 33)
    refuses(ValueError, codebook4.quantize, W, 32, book, top=0.0)
    refuses(ValueError, codebook4.quantize, W, 32, book[:3])
    refuses(ValueError, codebook4.quantize, W, 32, None, top=7.0)
    refuses(TypeError, codebook4.quantize, W.double(), 32)


def check_c_refusals(_):
    """The C entry points return EARG and queue nothing (host checks only: no pointer is followed)."""
    L = experts_hip.lib()
    t = torch.zeros(4096, device="cuda")
    p = t.data_ptr()
    bad = kmeans_hip.KMeansHipError("x", -2).code

    def earg(name, *args):
        rc = getattr(L, name)(*args)
        assert rc == bad, "%s%s returned %d" % (name, args, rc)

    earg("h2o4gpu_experts_route", 3, 1, 4, 2, 1, 0, 1.0, p, 4, 1, p, p, None)
    earg("h2o4gpu_experts_route", 0, 1, 4, 2, 1, 0, 1.0, None, 4, 1, p, p, None)
    earg("h2o4gpu_experts_route", 0, 1, 4, 2, 1, 0, 1.0, p + 2, 4, 1, p, p, None)
    earg("h2o4gpu_experts_route", 0, 1, 4, 5, 1, 0, 1.0, p, 4, 1, p, p, None)
    earg("h2o4gpu_experts_route", 0, 2 ** 31, 4, 1, 1, 0, 1.0, p, 4, 1, p, p, None)
    earg("h2o4gpu_experts_route", 0, 1, 4, 2, 1, 0, -1.0, p, 4, 1, p, p, None)
    earg("h2o4gpu_experts_route_backward", 0, 1, 4, 2, 1, 0, 1.0, p, 4, 1, p, p, None, p, 4, 1, None)
    earg("h2o4gpu_experts_sort", 4, 0, p, p, p, p, None, 0, None)
    earg("h2o4gpu_experts_sort", 4, 3, p, p, None, p, None, 0, None)
    need = L.h2o4gpu_experts_sort_workspace(10 ** 6, 64)
    assert need > 0 and L.h2o4gpu_experts_sort_workspace(10, 64) == 0
    earg("h2o4gpu_experts_sort", 10 ** 6, 64, p, p, p, p, p, need - 1, None)
    earg("h2o4gpu_experts_sort", 10 ** 6, 64, p, p, p, p, None, need, None)
    earg("h2o4gpu_experts_dispatch", 0, 1, 2, 8, p, 7, p, p, 8, None)
    earg("h2o4gpu_experts_dispatch", 0, 1, 2, 8, p, 8, p, p, 7, None)
    earg("h2o4gpu_experts_dispatch", 0, 1, 0, 8, p, 8, p, p, 8, None)
    earg("h2o4gpu_experts_dispatch", 0, 1, 2, 0, p, 8, p, p, 8, None)
    earg("h2o4gpu_experts_combine", 0, 1, 2, 8, p, 8, None, p, p, 8, None)
    earg("h2o4gpu_experts_combine_backward", 0, 1, 2, 8, p, 8, p, 8, p, p, p, 8, None, None)
    product = [0, 1, 4, 64, 32, p, 64, p, 0, p, p, p, 4, None]
    for at, value in ((0, 3), (1, 2 ** 31), (2, 0), (3, 0), (3, 2 ** 21), (4, 40), (4, 0), (5, None), (5, p + 2), (6, 63),
                      (7, None), (7, p + 4), (8, 7), (9, None), (9, p + 8), (10, None), (11, None), (12, 3)):
        earg("h2o4gpu_codebook4_product", *(product[:at] + [value] + product[at + 1:]))
    many = [0, 1, 2, 3, 4, 64, 32, p, 64, p, 0, p, p, 0, p, p, p, 4, None]
    for at, value in ((0, -1), (1, 2 ** 31), (2, 0), (2, 65), (3, 0), (3, 16385), (4, 0), (5, 0), (6, 33), (7, None),
                      (8, 2), (9, p + 1), (10, 3), (11, None), (12, p + 1), (13, 8), (14, None), (15, p + 2), (16, None),
                      (17, 1)):
        earg("h2o4gpu_codebook4_experts_product", *(many[:at] + [value] + many[at + 1:]))
    earg("h2o4gpu_codebook4_quantize", 0, 4, 64, 32, 0.0, p, 64, p, p, 32, 0, p, None)
    earg("h2o4gpu_codebook4_quantize", 0, 4, 64, 32, 1.0, p, 64, p, p, 31, 0, p, None)
    earg("h2o4gpu_codebook4_layout", 1, 4, 64, 32, p, 31, 0, p, p, p, None)
    earg("h2o4gpu_codebook4_layout", 1, 4, 64, 32, p, 32, 0, p, p + 4, p, None)
    assert L.h2o4gpu_codebook4_codes_bytes(0, 4, 4) == 0 and L.h2o4gpu_codebook4_scales_bytes(1, 4, 4, 31, 0) == 0
    assert L.h2o4gpu_codebook4_codes_bytes(2, 17, 129) == 2 * 2 * 2 * 1024
    torch.cuda.synchronize()
    assert float(t.abs().sum()) == 0.0


def layer(x, scores, packed, E, K):
    chosen, weights = experts.route(scores, K)
    order = experts.sort_by_expert(chosen, E)
    rows = codebook4.experts_product(x, packed, order)
    back = experts.combine(rows, weights, order)
    return back, experts.dispatch(x, order), order.offsets


def _layer_inputs(T=40, E=6, d=96, N=50):
    x = torch.randn(T, d, generator=gen(21)).bfloat16().cuda()
    s = torch.randn(T, E, generator=gen(22)).cuda()
    W = torch.randn(E, N, d, generator=gen(23)).bfloat16().cuda()
    book = torch.linspace(-1, 1, 16).cuda()
    return x, s, codebook4.quantize(W, 32, book)


def check_graph(_):
    """A captured layer replayed on new inputs equals the eager one, every time."""
    x, s, packed = _layer_inputs()
    for T in (40, 1):
        xs, ss = x[:T].clone(), s[:T].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(xs, ss, packed, 6, 2)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(xs, ss, packed, 6, 2)
        for k in range(4):
            xs.copy_(torch.randn(xs.shape, generator=gen(30 + k)).bfloat16())
            ss.copy_(torch.randn(ss.shape, generator=gen(40 + k)))
            torch.cuda.synchronize()
            want = [t.clone() for t in layer(xs, ss, packed, 6, 2)]
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b), "replay %d differs" % k


def check_other_stream(_):
    """Work queued on another stream than the one the tensors were made on follows that stream's order."""
    x, s, packed = _layer_inputs()
    want = [t.clone() for t in layer(x, s, packed, 6, 2)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = torch.randn(2048, 2048, device="cuda")
        for _ in range(20):  # keeps the side stream busy before the inputs are written
            a = (a @ a).clamp_(-1, 1)
        x2, s2 = x * 0, s * 0
        x2 += x
        s2 += s
        got = layer(x2, s2, packed, 6, 2)
    side.synchronize()
    for p, q in zip(got, want):
        assert torch.equal(p, q)


def check_broadcast_gradients(_):
    """Gradients that autograd hands out expanded or transposed."""
    T, K, E, d = 12, 2, 4, 20
    o = experts.sort_by_expert(torch.from_numpy(choices(T, K, E, "uniform")).cuda(), E)
    x = torch.randn(T, d, device="cuda", requires_grad=True)
    experts.dispatch(x, o).sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, K))
    y = torch.randn(T * K, d, device="cuda", requires_grad=True)
    w = torch.rand(T, K, device="cuda", requires_grad=True)
    g = torch.randn(d, T, device="cuda")
    gy, gw = torch.autograd.grad(experts.combine(y, w, o), (y, w), g.t())
    hy, hw = torch.autograd.grad(experts.combine(y, w, o), (y, w), g.t().contiguous())
    assert torch.equal(gy, hy) and torch.equal(gw, hw)
    s = torch.randn(T, E, device="cuda", requires_grad=True)
    experts.route(s, K)[1].sum().backward()
    assert float(s.grad.abs().max()) <= 8 * U32  # the weights' sum is 1 whatever the scores are
    # one row of weights for all tokens: its gradient is the sum over the tokens
    shared = torch.rand(1, K, device="cuda", requires_grad=True)
    experts.combine(y, shared.expand(T, K), o).sum().backward()
    pos = o.position.long()
    want = y.detach()[pos].double().sum((0, 2))
    assert torch.allclose(shared.grad.double()[0], want, rtol=0, atol=float(64 * U32 * y.detach().abs().sum()))


def check_unwanted_places(_):
    """Rows behind the last expert's are zeros after dispatch and experts_product, and combine reads none of
    them; the product uses nothing behind a row's last column."""
    T, K, E, d = 30, 2, 3, 40
    e = choices(T, K, E, "none")
    o = experts.sort_by_expert(torch.from_numpy(e).cuda(), E)
    x = torch.full((T, d), float("nan"), device="cuda")
    assert int(o.offsets[-1]) == 0
    assert torch.equal(experts.dispatch(x, o), torch.zeros(T * K, d, device="cuda"))
    out = experts.combine(torch.full((T * K, d), float("inf"), device="cuda"),
                          torch.full((T, K), float("nan"), device="cuda"), o)
    assert torch.equal(out, torch.zeros(T, d, device="cuda"))
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        for cols in (1, 31, 33, 127, 129):
            codes = torch.full((20, 80), 0xFF, dtype=torch.uint8, device="cuda")
            wide = torch.full((3, 200), float("nan"), dtype=dt, device="cuda")
            wide[:, :cols] = 1
            book = torch.ones(16, dtype=dt, device="cuda")
            m = codebook4.Codebook4(codes, torch.ones(20, -(-cols // 32), device="cuda"), book, cols, 32)
            y = codebook4.product(wide[:, :cols], m)
            assert torch.equal(y, torch.full((3, 20), cols, dtype=dt, device="cuda")), (dt, cols, y)
            assert not torch.isnan(codebook4.product(torch.zeros(1, cols, dtype=dt, device="cuda"), m)).any()


def check_fitted_codebook(_):
    """A codebook that k-means finds leaves less error than 16 even steps, on weights that are not even."""
    W = torch.randn(256, 512, generator=gen(50)).cuda()
    for dt in (torch.float32, torch.bfloat16):
        fitted = codebook4.quantize(W.to(dt), 128)
        even = codebook4.quantize(W.to(dt), 128, torch.linspace(-1, 1, 16, device="cuda"))
        a = (fitted.dequantize() - W.to(dt).float()).square().mean()
        b = (even.dequantize() - W.to(dt).float()).square().mean()
        assert float(a) < 0.9 * float(b), (a, b)
    q = codebook4.quantize(torch.randn(3, 40, 64, generator=gen(51)).half().cuda(), 32)
    assert q.n_experts == 3 and tuple(q.dequantize().shape) == (3, 40, 64)


def check_far_rows(_):
    """Rows further apart than 2^31 elements."""
    far = torch.empty((2 ** 31 // 2 + 64) * 3, dtype=torch.bfloat16, device="cuda")
    stride = 2 ** 31 // 2 + 64
    x = torch.as_strided(far, (3, 50), (stride, 1))
    vals = torch.randn(3, 50, generator=gen(60)).bfloat16()
    x.copy_(vals)
    e = torch.tensor([[1, 0], [2, 1], [0, 2]], dtype=torch.int32)
    o = experts.sort_by_expert(e.cuda(), 3)
    rows = experts.dispatch(x, o)
    pos = torch.from_numpy(order_oracle(e.numpy(), 3)[1]).long()
    want = torch.zeros(6, 50, dtype=torch.bfloat16)
    want[pos] = vals[:, None, :].expand(3, 2, 50)
    same(rows, want, "rows")
    W = torch.randn(8, 50, generator=gen(61)).bfloat16().cuda()
    q = codebook4.quantize(W, 32, torch.linspace(-1, 1, 16).cuda())
    assert torch.equal(codebook4.product(x, q), codebook4.product(vals.cuda(), q))
    s = torch.as_strided(far, (3, 4), (stride, 5))
    a, b = experts.route(s, 2), experts.route(s.contiguous(), 2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def check_long_cache(_):
    """More rows than a grid dimension of 65535 or 2^24 workgroups of 256 threads hold, and a result beyond
    2^31 elements."""
    T = 17_000_000
    x = torch.arange(T, device="cuda", dtype=torch.float32)[:, None].contiguous()
    e = (torch.arange(T, device="cuda", dtype=torch.int32) % 5)[:, None].contiguous()
    o = experts.sort_by_expert(e, 5)
    rows = experts.dispatch(x, o)
    assert torch.equal(rows, x[o.order.long()])
    assert torch.equal(rows[o.position.long().reshape(-1)], x)
    w = torch.full((T, 1), 2.0, device="cuda")
    out = experts.combine(rows, w, o)
    assert torch.equal(out, 2 * x)
    del rows, out, w, o, e, x
    T, d = 70_000, 16_400
    x = torch.zeros(T, d, device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 1
    x[:, -1] = torch.arange(T, device="cuda").remainder(251).bfloat16()
    e = torch.stack([torch.arange(T, device="cuda", dtype=torch.int32) % 7,
                     torch.arange(T, device="cuda", dtype=torch.int32) % 3], 1).contiguous()
    o = experts.sort_by_expert(e, 7)
    rows = experts.dispatch(x, o)
    assert rows.numel() > 2 ** 31
    token = o.order.long() // 2
    assert torch.equal(rows[:, -1], x[token, -1]) and bool((rows[:, 0] == 1).all())
    out = experts.combine(rows, torch.full((T, 2), 0.5, device="cuda"), o)
    assert torch.equal(out, x)
    book = torch.arange(16, device="cuda").bfloat16()
    codes = torch.full((16, 16), 0x11, dtype=torch.uint8, device="cuda")
    m = codebook4.Codebook4(codes, torch.ones(16, 1, device="cuda"), book, 32, 32)
    x = torch.ones(1_100_000, 32, device="cuda", dtype=torch.bfloat16)
    assert bool((codebook4.product(x, m) == 32).all())
    s = torch.zeros(70_000_000, 2, device="cuda", dtype=torch.bfloat16)
    s[:, 1] = 1
    assert bool((experts.route(s, 1)[0] == 1).all())


def check_repeats(_):
    """The same inputs give the same bits, whatever ran between."""
    x, s, packed = _layer_inputs(T=300)
    first = [t.clone() for t in layer(x, s, packed, 6, 2)]
    for k in range(5):
        other = _layer_inputs(T=17 + k)
        layer(other[0], other[1], other[2], 6, 3)
        for a, b in zip(layer(x, s, packed, 6, 2), first):
            assert torch.equal(a, b)


def check_example(_):
    """The example runs, learns and serves nearly as well with 4 bits."""
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import cluster_experts
    r = cluster_experts.main(["--rows", "4000", "--quiet"])
    assert r["loss_last"] < 0.5 * r["loss_first"], r
    assert r["served_error"] < 0.2, r


def main():
    want = sys.argv[1] if len(sys.argv) > 1 else ""
    bad = 0
    for c in all_cases():
        if want and want not in c["name"]:
            continue
        r = dict(name=c["name"], ok=True, why="")
        print("# " + c["name"], flush=True)
        try:
            globals()["check_" + c["op"]](c)
            torch.cuda.synchronize()
        except Exception as e:  # reported to the collecting test
            r.update(ok=False, why="".join(traceback.format_exception_only(type(e), e))[:1500] +
                     "".join(traceback.format_tb(e.__traceback__)[-2:])[:1000])
            bad += 1
            if "HIP error" in r["why"] or "CUDA error" in r["why"]:
                print(json.dumps(r), flush=True)
                return 1  # nothing more is run on the GPU
        print(json.dumps(r), flush=True)
        if c["op"] in ("far_rows", "long_cache"):
            torch.cuda.empty_cache()
    return 1 if bad else 0


if __name__ == "__main__":
    sys.exit(main())
