"""Child process of test_gpu_products.py: runs every case of products_cases.py (or those whose names
contain argv[1]) and prints a JSON line for each. Not collected by pytest.

Every oracle is plain torch on the CPU in 64 bits from the operator's formula. U32 is the largest
relative error of one float32 rounding, ROUND[dtype] that of the final one. A matrix instruction adds
32 (float32: 4, 4 bits: 128) products to a sum; each is taken to round at most four times at the size of what has been
added up, and the instruction of four products once for each: a sum of n terms is then off by at
most (n / 8 + 16) U32 times the sum of their magnitudes ((n + 16) U32 for float32)."""
import json
import math
import os
import sys
import threading
import traceback

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from products_cases import all_cases  # noqa: E402
from h2o4gpu_amd import experts, microscale4  # noqa: E402
from h2o4gpu_amd.libs import experts_hip, kmeans_hip  # noqa: E402

DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
U32 = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def near(got, want, bound, what):
    """|got - want| <= bound + the last rounding, element by element; NaN and infinities in the same places. A
    number that may be as large as the type's largest and half a step rounds to infinity from there on."""
    u, tiny = ROUND[got.dtype], TINY[got.dtype]
    g, w = got.detach().double().cpu(), want.double()
    assert g.shape == w.shape, "%s: shape %s, expected %s" % (what, tuple(g.shape), tuple(w.shape))
    fine = torch.isfinite(w)
    assert torch.equal(torch.isnan(g), torch.isnan(w)), "%s: NaN in other places" % what
    assert torch.equal(g[~fine & ~torch.isnan(w)], w[~fine & ~torch.isnan(w)]), "%s: infinities" % what
    b = torch.as_tensor(bound, dtype=torch.float64).expand(w.shape)
    off = (g - w).abs()
    allowed = b + u * (w.abs() + b) + tiny
    border = torch.finfo(got.dtype).max * (1 + u / 2)  # (float16: 65504 + 16)
    beyond = (w.abs() + b >= border) & torch.isinf(g) & (torch.sign(g) == torch.sign(w))
    bad = fine & ~(off <= allowed) & ~beyond
    assert not bad.any(), "%s: %d of %d off, worst %.3g against %.3g allowed, first at %s" % (
        what, int(bad.sum()), bad.numel(), float(off[bad].max()), float(allowed[bad].min()), bad.nonzero()[0].tolist())


def same(got, want, what):
    assert torch.equal(got.cpu(), want.cpu()), what


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def laid_out(t, layout):
    """On the GPU: as it is, in rows with a gap behind (of NaN), or at an address off by one element."""
    if layout == "strided":
        wide = torch.full(t.shape[:-1] + (t.shape[-1] + 16,), float("nan"), dtype=t.dtype, device="cuda")
        wide[..., :t.shape[-1]] = t.cuda()
        return wide[..., :t.shape[-1]]
    if layout == "unaligned":
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.cuda().reshape(-1)
        return flat[1:].view(t.shape)
    return t.cuda()


def roundings(n, dt):
    return n + 16 if dt == torch.float32 else n / 8 + 16


def choices(c):
    rng = np.random.default_rng(3 + c["tokens"] + c["experts"])
    T, K, E = c["tokens"], c["top_k"], c["experts"]
    if c.get("data") == "nothing":
        return np.full((T, K), -1, np.int32)
    if c.get("data") == "one_expert":
        return np.full((T, K), E - 1, np.int32)
    e = np.minimum((rng.exponential(0.4, (T, K)) * E).astype(np.int64), E - 1)
    e = np.where(rng.random((T, K)) < c["dropped"], np.where(rng.random((T, K)) < 0.5, -1, E), e)
    return e.astype(np.int32)


def stretches(e, E):
    """(slots in expert order, where each expert's rows begin)."""
    flat = e.reshape(-1).astype(np.int64)
    key = np.where((flat >= 0) & (flat < E), flat, E)
    return np.argsort(key, kind="stable"), np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])])


# ---- products grouped by expert ---------------------------------------------------------------------

def check_product(c):
    e, E, N, K, dt = choices(c), c["experts"], c["out"], c["cols"], DT[c["dtype"]]
    order = experts.sort_by_expert(torch.from_numpy(e).cuda(), E)
    _, at = stretches(e, E)
    S, held = e.size, int(at[-1])
    x = torch.randn(S, K, generator=gen(1)).to(dt)
    W = torch.randn(E, N, K, generator=gen(2)).to(dt)
    g = torch.randn(S, N, generator=gen(3)).to(dt)
    if c["data"] == "infinity":
        x[S // 2, K // 3] = math.inf
        g[S // 3, N // 2] = -math.inf
    if c["data"] == "nan_behind":
        x[held:], g[held:] = math.nan, math.inf
    dx, dW = laid_out(x, c["layout"]).requires_grad_(), laid_out(W, c["layout"]).requires_grad_()
    y = experts.product(dx, dW, order)
    again = experts.product(dx.detach(), dW.detach(), order)
    assert torch.equal(again.nan_to_num(), y.detach().nan_to_num()), "the call without a gradient differs"
    gx, gW = torch.autograd.grad(y, (dx, dW), laid_out(g, c["layout"]))
    wy, my = torch.zeros(S, N, dtype=torch.float64), torch.zeros(S, N, dtype=torch.float64)
    wx, mx = torch.zeros(S, K, dtype=torch.float64), torch.zeros(S, K, dtype=torch.float64)
    wW, mW = torch.zeros(E, N, K, dtype=torch.float64), torch.zeros(E, N, K, dtype=torch.float64)
    most = 0
    for i in range(E):
        lo, hi = int(at[i]), int(at[i + 1])
        if lo == hi:
            continue
        a, b, d = x[lo:hi].double(), W[i].double(), g[lo:hi].double()
        wy[lo:hi], my[lo:hi] = a @ b.t(), a.abs() @ b.t().abs()
        wx[lo:hi], mx[lo:hi] = d @ b, d.abs() @ b.abs()
        wW[i], mW[i] = d.t() @ a, d.t().abs() @ a.abs()
        most = max(most, hi - lo)
    near(y, wy, torch.nan_to_num(roundings(K, dt) * U32 * my), "y")
    near(gx, wx, torch.nan_to_num(roundings(N, dt) * U32 * mx), "gradient of the rows")
    near(gW, wW, torch.nan_to_num(roundings(most, dt) * U32 * mW), "gradient of the matrices")


# ---- microscaled numbers ----------------------------------------------------------------------------

LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def numbers(x):
    """(codes, scales, values) of the rows of x by the definition, in 64 bits; values NaN in a block that is none."""
    rows, K = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -K % 32)).reshape(rows, -1, 32)
    bad = ~torch.isfinite(v).all(2, keepdim=True)
    v = torch.where(bad, torch.zeros_like(v), v)
    most = v.abs().amax(2, keepdim=True)
    power = torch.frexp(most).exponent.double() - 3
    power = torch.where(most > 0, power.clamp(-127, 127), -127.0)
    m = (v / torch.exp2(power)).abs()
    code = torch.zeros_like(m)
    off = m.clone()
    for k in (2, 4, 6, 1, 3, 5, 7):  # even codes first: they win a tie
        far = (m - LEVELS[k]).abs()
        code, off = torch.where(far < off, float(k), code), torch.minimum(far, off)
    value = torch.copysign(LEVELS[code.long()] * torch.exp2(power), v)
    code = torch.where(bad, 0.0, code + 8 * torch.signbit(v))
    scale = torch.where(bad, 255.0, power + 127)
    value = torch.where(bad, math.nan, value)
    return code.reshape(rows, -1)[:, :K].to(torch.uint8), scale[:, :, 0].to(torch.uint8), value.reshape(rows, -1)[:, :K]


def values_of(c):
    g, dt = gen(c["rows"] + 3 * c["cols"]), DT[c["dtype"]]
    x = torch.randn(c["rows"], c["cols"], generator=g)
    pick = torch.rand(x.shape, generator=g)
    if c["data"] == "wide":
        x = x * torch.exp2(torch.randint(-14, 14, x.shape, generator=g).float())
    elif c["data"] == "ties":  # the middles, and numbers next to them
        x = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 4.0, 0.125])[
            torch.randint(0, 11, x.shape, generator=g)] * torch.where(pick < 0.5, 1.0, -1.0)
        x[pick < 0.1] *= 1 + 2.0 ** -7
    elif c["data"] == "tiny":
        x = x * (2.0 ** -24 if dt == torch.float16 else 2.0 ** -126)
    elif c["data"] == "zeros":
        x = torch.where(pick < 0.9, torch.where(pick < 0.4, 0.0, -0.0), x)
        x[0] = 0
    elif c["data"] == "not_finite":
        x[pick < 0.01] = math.nan
        x[(pick > 0.99)] = math.inf
        x[0, 0] = -math.inf
    return x.to(dt)


def check_quantize(c):
    x = values_of(c)
    m = microscale4.quantize(laid_out(x, c["layout"]))
    code, scale, value = numbers(x)
    same(m.scales(), scale, "scales")
    same(m.codes(), code, "codes")
    assert int(m.laid_codes[..., (c["cols"] + 1) // 2:].count_nonzero()) == 0, "codes behind the last column"
    assert int(m.laid_scales.long().sum()) == int(scale.long().sum()), "scales behind the last column"
    near(m.dequantize(), value, 0.0, "values")
    for dt in DT.values():
        got = m.dequantize(dt)
        want = value.to(dt) if dt != torch.float32 else value.float()
        assert torch.equal(got.cpu().nan_to_num(), want.nan_to_num()), "values as %s" % dt
        assert torch.equal(torch.signbit(got.cpu()[~want.isnan()]), torch.signbit(want[~want.isnan()])), "signs"
    again = microscale4.Microscale4(packed(code), scale.cuda(), c["cols"], dtype=x.dtype)
    same(again.laid_codes, m.laid_codes, "codes laid out")
    same(again.laid_scales, m.laid_scales, "scales laid out")


def packed(code):
    code = torch.nn.functional.pad(code, (0, code.shape[-1] % 2))
    return (code[..., 0::2] | (code[..., 1::2] << 4)).cuda()


def matrix(lead, K, seed, made="codes", dt=torch.float32):
    """A Microscale4 and its values in 64 bits (rows flattened)."""
    rows = int(np.prod(lead))
    g = gen(seed)
    if made == "quantize":
        w = (torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-3, 4, (rows, 1), generator=g).float())).to(dt)
        return microscale4.quantize(w.reshape(lead + (K,)).cuda()), numbers(w)[2]
    code = torch.randint(0, 16, (rows, K), generator=g, dtype=torch.uint8)
    scale = torch.randint(118, 136, (rows, -(-K // 32)), generator=g, dtype=torch.uint8)
    value = LEVELS[(code & 7).long()] * torch.where(code >= 8, -1.0, 1.0)
    value = value * torch.exp2(scale.double() - 127).repeat_interleave(32, dim=1)[:, :K]
    # bytes behind the row, and a nibble behind the last column, are anything
    raw = torch.nn.functional.pad(packed(code), (0, 3), value=0xa5)
    if K % 2:
        raw[:, K // 2] |= 0x70
    m = microscale4.Microscale4(raw.reshape(lead + (-1,)), scale.reshape(lead + (-1,)).cuda(), K, dtype=dt)
    return m, value


def check_four(c):
    dt, K = DT[c["dtype"]], c["cols"]
    x, vx = matrix((c["rows"],), K, 1, c["made"], dt)
    w, vw = matrix((c["out"],), K, 2, c["made"], torch.float32)
    y = microscale4.product(x, w)
    assert y.dtype == dt
    near(y, vx @ vw.t(), (K / 8 + 16) * U32 * (vx.abs() @ vw.abs().t()), "y")
    other = microscale4.product(x, w, dtype=torch.float32)
    near(other, vx @ vw.t(), (K / 8 + 16) * U32 * (vx.abs() @ vw.abs().t()), "y in float32")
    same(other.to(dt), y, "one rounding")


def check_four_experts(c):
    e, E, N, K, dt = choices(c), c["experts"], c["out"], c["cols"], DT[c["dtype"]]
    order = experts.sort_by_expert(torch.from_numpy(e).cuda(), E)
    slots, at = stretches(e, E)
    w, vw = matrix((E, N), K, 2, "codes")
    vw = vw.reshape(E, N, K)
    if c["in_order"]:
        held = int(at[-1])
        x = torch.randn(e.size, K, generator=gen(1)).to(dt)
        x[held:] = math.nan
        vx = numbers(x)[2]
        x = microscale4.quantize(x.cuda())
    else:
        x, vx = matrix((c["tokens"],), K, 1, "quantize", dt)
        vx = vx[torch.from_numpy(slots // c["top_k"])]
    y = microscale4.experts_product(x, w, order, in_order=c["in_order"])
    want, size = torch.zeros(e.size, N, dtype=torch.float64), torch.zeros(e.size, N, dtype=torch.float64)
    for i in range(E):
        lo, hi = int(at[i]), int(at[i + 1])
        if lo < hi:
            want[lo:hi], size[lo:hi] = vx[lo:hi] @ vw[i].t(), vx[lo:hi].abs() @ vw[i].abs().t()
    near(y, want, (K / 8 + 16) * U32 * size, "y")


# ---- uses ---------------------------------------------------------------------------------------------

def routed(T, K, E, seed=5, dropped=0.0):
    c = dict(tokens=T, top_k=K, experts=E, dropped=dropped)
    return experts.sort_by_expert(torch.from_numpy(choices(c)).cuda(), E)


def check_differences(_):
    """The product is linear in either operand: a difference quotient is its derivative but for roundings."""
    T, E, N, K = 70, 4, 24, 37
    order = routed(T, 2, E, dropped=0.2)
    x, W = torch.randn(2 * T, K, generator=gen(1)).cuda(), torch.randn(E, N, K, generator=gen(2)).cuda()
    g = torch.randn(2 * T, N, generator=gen(3)).cuda()
    x.requires_grad_(), W.requires_grad_()
    gx, gW = torch.autograd.grad(experts.product(x, W, order), (x, W), g)
    with torch.no_grad():
        for seed in range(4):
            dx, dW = torch.randn(x.shape, generator=gen(10 + seed)).cuda(), torch.randn(W.shape, generator=gen(20 + seed)).cuda()
            for direction, grad, f in ((dx, gx, lambda h: experts.product(x + h * dx, W, order)),
                                       (dW, gW, lambda h: experts.product(x, W + h * dW, order))):
                quotient = ((f(1.0).double() - f(-1.0).double()) * g.double()).sum() / 2
                inner = (direction.double() * grad.double()).sum()
                # each of 2 T N numbers: K + 16 roundings of sums of K products of size about 2 (1.4^2), times g
                # of size 1, of independent signs at best: their plain sum is the bound
                allowed = 2 * T * N * (K + 16) * U32 * K * 3 * 3
                assert abs(float(quotient - inner)) <= allowed, "%g against %g" % (float(quotient), float(inner))


def check_broadcast(_):
    """One matrix for all experts (expanded), an expanded gradient, and their sums."""
    T, E, N, K = 50, 5, 24, 40
    order = routed(T, 2, E)
    for dt in DT.values():
        x = torch.randn(2 * T, K, generator=gen(1)).to(dt).cuda().requires_grad_()
        one = torch.randn(1, N, K, generator=gen(2)).to(dt).cuda().requires_grad_()
        y = experts.product(x, one.expand(E, N, K), order)
        a, b = x.detach().double().cpu(), one.detach()[0].double().cpu()
        near(y, a @ b.t(), roundings(K, dt) * U32 * (a.abs() @ b.abs().t()), "y")
        gx, gW = torch.autograd.grad(y.sum(), (x, one))
        ones = torch.ones(2 * T, N, dtype=torch.float64)
        near(gx, ones @ b, roundings(N, dt) * U32 * (ones @ b.abs()), "gradient of the rows")
        # rounded once for each expert, and again where autograd adds the five up
        size = (ones.t() @ a.abs())[None]
        near(gW, (ones.t() @ a)[None], (roundings(2 * T, dt) * U32 + 6 * ROUND[dt]) * size, "gradient of the matrix")


def check_broadcast_between_words(_):
    """One matrix for all experts whose rows begin between words, in a product that copies such: as three matrices."""
    E, N, K = 3, 3001, 901
    order = experts.sort_by_expert((torch.arange(6000) % E).int().view(-1, 1).cuda(), E)
    x = torch.randn(6000, K, generator=gen(1)).bfloat16().cuda().requires_grad_()
    one = torch.randn(1, N, K, generator=gen(2)).bfloat16().cuda()
    g = torch.randn(6000, N, generator=gen(3)).bfloat16().cuda()
    y, z = experts.product(x, one.expand(E, N, K), order), experts.product(x, one.repeat(E, 1, 1), order)
    same(y, z, "y")
    same(torch.autograd.grad(y, x, g)[0], torch.autograd.grad(z, x, g)[0], "gradient of the rows")
    a, b = x[:50].detach().double().cpu(), one[0].double().cpu()
    near(y[:50], a @ b.t(), roundings(K, x.dtype) * U32 * (a.abs() @ b.abs().t()), "y")


def layer(x, scores, W, packed, top_k):
    chosen, weights = experts.route(scores, top_k)
    order = experts.sort_by_expert(chosen, W.shape[0])
    full = experts.combine(experts.product(experts.dispatch(x, order), W, order), weights, order)
    small = experts.combine(microscale4.experts_product(microscale4.quantize(x), packed, order), weights, order)
    return full, small


def check_graph(_):
    """A captured layer replayed on new inputs equals the eager one, every time."""
    E, N, K = 6, 80, 96
    W = torch.randn(E, N, K, generator=gen(1)).bfloat16().cuda()
    packed = microscale4.quantize(W)
    for T in (1, 40, 700):
        x, s = torch.randn(T, K).bfloat16().cuda(), torch.randn(T, E).cuda()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(x, s, W, packed, 2)
        torch.cuda.current_stream().wait_stream(side)
        graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x, s, W, packed, 2)
        with torch.cuda.graph(second):
            out2 = layer(x, s, W, packed, 2)
        for k in range(4):
            x.copy_(torch.randn(x.shape, generator=gen(30 + k)).bfloat16())
            s.copy_(torch.randn(s.shape, generator=gen(40 + k)))
            torch.cuda.synchronize()
            want = [t.clone() for t in layer(x, s, W, packed, 2)]
            graph.replay()
            second.replay()
            torch.cuda.synchronize()
            for a, b, d in zip(out, want, out2):
                assert torch.equal(a, b) and torch.equal(d, b), "replay %d of %d tokens differs" % (k, T)


def check_graph_of_training(_):
    E, N, K, T = 5, 72, 88, 300
    order = routed(T, 2, E, dropped=0.1)
    for dt in (torch.bfloat16, torch.float32):
        x = torch.randn(2 * T, K, generator=gen(1)).to(dt).cuda().requires_grad_()
        W = torch.randn(E, N, K, generator=gen(2)).to(dt).cuda().requires_grad_()
        g = torch.randn(2 * T, N, generator=gen(3)).to(dt).cuda()

        def step():
            y = experts.product(x, W, order)
            return (y.detach(),) + torch.autograd.grad(y, (x, W), g)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for k in range(4):
            with torch.no_grad():
                x.copy_(torch.randn(x.shape, generator=gen(30 + k)).to(dt))
                W.copy_(torch.randn(W.shape, generator=gen(40 + k)).to(dt))
                g.copy_(torch.randn(g.shape, generator=gen(50 + k)).to(dt))
            torch.cuda.synchronize()
            want = [t.clone() for t in step()]
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b), "replay %d differs" % k


def check_two_at_once(_):
    """Two captured steps with partial sums and aligned copies of their own, and two threads, all at the same time."""
    for E, N, K, T, dt in ((3, 61, 75, 20000, torch.float32), (2, 131, 70, 9000, torch.bfloat16),
                           (3, 1025, 1023, 12000, torch.bfloat16)):
        order = routed(T, 1, E)
        sets = []
        for k in range(2):
            x = torch.randn(T, K, generator=gen(60 + k)).to(dt).cuda().requires_grad_()
            W = torch.randn(E, N, K, generator=gen(70 + k)).to(dt).cuda().requires_grad_()
            sets.append((x, W, torch.randn(T, N, generator=gen(80 + k)).to(dt).cuda()))

        def step(x, W, g):
            y = experts.product(x, W, order)
            return (y.detach(),) + torch.autograd.grad(y, (x, W), g)

        want = [[t.clone() for t in step(*s)] for s in sets]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        graphs, outs = [], []
        torch.cuda.synchronize()
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                step(*s)
            stream.synchronize()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                outs.append(step(*s))
        for k in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            eager = step(*sets[k % 2])
            torch.cuda.synchronize()
            for got, right in zip(outs + [eager], want + [want[k % 2]]):
                for a, b in zip(got, right):
                    assert torch.equal(a, b), "replay %d of %d x %d differs" % (k, N, K)
        found = [None, None]

        def work(k):
            with torch.cuda.stream(streams[k]):
                for _ in range(4):
                    found[k] = step(*sets[k])
            streams[k].synchronize()

        threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for got, right in zip(found, want):
            for a, b in zip(got, right):
                assert torch.equal(a, b), "a thread's %d x %d differs" % (N, K)


def check_other_stream(_):
    E, N, K, T = 4, 64, 128, 200
    order = routed(T, 2, E)
    x, W = torch.randn(2 * T, K, generator=gen(1)).half().cuda(), torch.randn(E, N, K, generator=gen(2)).half().cuda()
    want = experts.product(x, W, order)
    q = microscale4.quantize(x)
    want4 = microscale4.experts_product(q, microscale4.quantize(W), order, in_order=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(2048, 2048, device="cuda")
        for _ in range(20):
            big = big @ big * 0.01
        late = x + 0 * big[0, 0].nan_to_num().half()  # ready only when the stream gets there
        got = experts.product(late, W, order)
        got4 = microscale4.experts_product(microscale4.quantize(late), microscale4.quantize(W), order, in_order=True)
    side.synchronize()
    same(got, want, "product on another stream")
    same(got4, want4, "4-bit product on another stream")


def check_repeats(_):
    E, N, K, T = 3, 200, 300, 2000
    order = routed(T, 2, E)
    x = torch.randn(2 * T, K, generator=gen(1)).bfloat16().cuda().requires_grad_()
    W = torch.randn(E, N, K, generator=gen(2)).bfloat16().cuda().requires_grad_()
    g = torch.randn(2 * T, N, generator=gen(3)).bfloat16().cuda()
    first = None
    for _ in range(5):
        y = experts.product(x, W, order)
        out = (y.detach(),) + torch.autograd.grad(y, (x, W), g)
        first = first or out
        for a, b in zip(out, first):
            assert torch.equal(a, b), "equal calls differ"


def check_two_layers(_):
    """Tokens through two layers of experts in 4 bits: the second takes the first one's rows as they lie."""
    T, E, K, H, N, k = 90, 5, 160, 224, 48, 2
    order = routed(T, k, E, dropped=0.2)
    W1, v1 = matrix((E, H), K, 1)
    W2, v2 = matrix((E, N), H, 2)
    x = torch.randn(T, K, generator=gen(4)).bfloat16()
    hidden = microscale4.experts_product(microscale4.quantize(x.cuda()), W1, order).relu()
    y = microscale4.experts_product(microscale4.quantize(hidden), W2, order, in_order=True)
    h = numbers(hidden.cpu())[2]
    at = order.offsets.tolist()
    want, size = torch.zeros(T * k, N, dtype=torch.float64), torch.zeros(T * k, N, dtype=torch.float64)
    for e in range(E):
        lo, hi = at[e], at[e + 1]
        m = v2.reshape(E, N, H)[e]
        want[lo:hi], size[lo:hi] = h[lo:hi] @ m.t(), h[lo:hi].abs() @ m.abs().t()
    near(y, want, (H / 8 + 16) * U32 * size, "y")


def check_codes_back(_):
    code = torch.randint(0, 16, (3, 5, 700), generator=gen(1), dtype=torch.uint8)
    scale = torch.randint(0, 256, (3, 5, 22), generator=gen(2), dtype=torch.uint8)
    m = microscale4.Microscale4(packed(code), scale.cuda(), 700)
    same(m.codes(), code, "codes")
    same(m.scales(), scale, "scales")
    v = LEVELS[(code & 7).long()] * torch.where(code >= 8, -1.0, 1.0)
    p = torch.where(scale == 255, math.nan, torch.exp2(scale.double() - 127)).repeat_interleave(32, dim=2)[..., :700]
    got, want = m.dequantize(), (v * p).float()
    assert torch.equal(got.cpu().nan_to_num(), want.nan_to_num()) and torch.equal(got.cpu().isnan(), want.isnan())


def check_far_rows(_):
    """Rows whose offsets pass 32 bits: of tokens, of matrices, of results and of gradients."""
    far = (1 << 31) + 4096
    K, N, E = 64, 24, 2
    chosen = torch.tensor([[0], [1], [1]], dtype=torch.int32).cuda()
    order = experts.sort_by_expert(chosen, E)
    buf = torch.zeros(2 * far + K, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, K), (far, 1))
    x.copy_(torch.randn(3, K, generator=gen(1)).bfloat16())
    wbuf = torch.zeros(far + N * K, dtype=torch.bfloat16, device="cuda")
    W = wbuf.as_strided((E, N, K), (far, K, 1))
    W.copy_(torch.randn(E, N, K, generator=gen(2)).bfloat16())
    x.requires_grad_(), W.requires_grad_()
    y = experts.product(x, W, order)
    g = torch.randn(3, N, generator=gen(3)).bfloat16().cuda()
    gx, gW = torch.autograd.grad(y, (x, W), g)
    with torch.no_grad():
        near_x, near_W = x.detach().contiguous().requires_grad_(), W.detach().contiguous().requires_grad_()
    y2 = experts.product(near_x, near_W, order)
    hx, hW = torch.autograd.grad(y2, (near_x, near_W), g)
    same(y, y2, "y"), same(gx, hx, "gradient of the rows"), same(gW, hW, "gradient of the matrices")
    del buf, wbuf, x, W
    # many rows of 4-bit numbers: codes and results beyond 2^32 bytes
    rows, K, N = 17_000_000, 512, 130
    c = torch.randint(0, 256, (rows, K // 2), dtype=torch.uint8, device="cuda")
    s = torch.randint(120, 130, (rows, K // 32), dtype=torch.uint8, device="cuda")
    w, vw = matrix((N,), K, 2)
    m = microscale4.Microscale4(c, s, K)
    y = microscale4.product(m, w)
    for lo in (0, 8_388_600, rows - 100):
        part = microscale4.Microscale4(c[lo:lo + 100], s[lo:lo + 100], K)
        a = part.dequantize().double().cpu()
        near(y[lo:lo + 100], a @ vw.t(), (K / 8 + 16) * U32 * (a.abs() @ vw.abs().t()), "rows from %d on" % lo)


def refuses(kind, f, *args, **kw):
    try:
        f(*args, **kw)
    except kind:
        return
    except Exception as e:  # noqa: BLE001
        raise AssertionError("%s instead of %s: %s" % (type(e).__name__, kind.__name__, e))
    raise AssertionError("%s%s was taken" % (f.__name__, tuple(type(a).__name__ for a in args)))


def check_refusals(_):
    order = routed(4, 2, 3)
    x, W = torch.randn(8, 16, device="cuda"), torch.randn(3, 5, 16, device="cuda")
    p = experts.product
    p(x, W, order)
    refuses(ValueError, p, x[:7], W, order)
    refuses(ValueError, p, x, W[:2], order)
    refuses(ValueError, p, x[:, :8], W, order)
    refuses(ValueError, p, x, W[:, :0], order)
    refuses(ValueError, p, x[:, :0], W[:, :, :0], order)
    refuses(ValueError, p, x, W[0], order)
    refuses(ValueError, p, x.cpu(), W, order)
    refuses(ValueError, p, x, W.cpu(), order)
    refuses(TypeError, p, x.half(), W, order)
    refuses(TypeError, p, x.double(), W.double(), order)
    refuses(TypeError, p, x, W, torch.zeros(8, dtype=torch.int32, device="cuda"))
    refuses(TypeError, p, [[1.0]], W, order)
    refuses(ValueError, p, x.t().contiguous().t(), W, order)
    refuses(ValueError, p, x[:1].expand(8, 16), W, order)
    refuses(ValueError, p, x, W.transpose(1, 2).contiguous().transpose(1, 2), order)
    refuses(ValueError, p, x, W[:, :1].expand(3, 5, 16), order)
    q, make = microscale4.quantize, microscale4.Microscale4
    refuses(TypeError, q, x.double())
    refuses(ValueError, q, x.cpu())
    refuses(ValueError, q, x[0])
    refuses(ValueError, q, x[:, :0])
    refuses(ValueError, q, x.t().contiguous().t())
    refuses(ValueError, q, x.clone().requires_grad_())
    refuses(TypeError, q, [[1.0]])
    codes, scales = torch.zeros(5, 8, dtype=torch.uint8, device="cuda"), torch.zeros(5, 1, dtype=torch.uint8, device="cuda")
    make(codes, scales, 16)
    refuses(ValueError, make, codes, scales, 17)
    refuses(ValueError, make, codes, scales, 0)
    refuses(ValueError, make, codes, scales[:4], 16)
    refuses(TypeError, make, codes.int(), scales, 16)
    refuses(TypeError, make, codes, scales.float(), 16)
    refuses(ValueError, make, codes.cpu(), scales, 16)
    refuses(ValueError, make, codes[0], scales[0], 16)
    refuses(TypeError, make, codes, scales, 16, dtype=torch.float64)
    a, w = q(x), q(W[0])
    many = q(W)
    refuses(TypeError, microscale4.product, x, w)
    refuses(TypeError, microscale4.product, a, W[0])
    refuses(ValueError, microscale4.product, a, many)
    refuses(ValueError, microscale4.product, many, w)
    refuses(ValueError, microscale4.product, q(x[:, :8]), w)
    refuses(TypeError, microscale4.product, a, w, dtype=torch.int32)
    refuses(TypeError, a.dequantize, torch.float64)
    e = microscale4.experts_product
    e(a, many, order, in_order=True)
    refuses(ValueError, e, a, many, order)
    refuses(ValueError, e, q(x[:4]), many, order, in_order=True)
    refuses(ValueError, e, q(x[:4]), w, order)
    refuses(ValueError, e, q(x[:4]), many, routed(4, 2, 4))
    refuses(TypeError, e, q(x[:4]), many, None)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        refuses(NotImplementedError, p, dual, W, order)
        refuses(NotImplementedError, q, dual)


def check_c_refusals(_):
    lib = experts_hip.lib()
    assert lib.h2o4gpu_experts_product(7, 8, 3, 5, 16, 16, 16, 16, 80, 16, 16, 16, 5, None) == -2
    try:
        experts_hip.check("h2o4gpu_experts_product", -2)
    except kmeans_hip.KMeansHipError:
        return
    raise AssertionError("an error status was not raised")


def check_second_derivatives(_):
    order = routed(6, 1, 2)
    x, W = torch.randn(6, 8, device="cuda", requires_grad=True), torch.randn(2, 4, 8, device="cuda", requires_grad=True)
    y = experts.product(x, W, order)
    gx, gW = torch.autograd.grad(y.square().sum(), (x, W), create_graph=True)
    for g in (gx, gW):
        try:
            torch.autograd.grad(g.sum(), (x, W), retain_graph=True, allow_unused=True)
        except RuntimeError as e:
            assert "differentiated again" in str(e), e
        else:
            raise AssertionError("a second derivative was given")


def check_one_gradient(_):
    """Only what is asked for is computed, and it is the same."""
    order = routed(60, 2, 4)
    x, W = torch.randn(120, 40, generator=gen(1)).cuda(), torch.randn(4, 24, 40, generator=gen(2)).cuda()
    g = torch.randn(120, 24, generator=gen(3)).cuda()
    a, b = x.clone().requires_grad_(), W.clone().requires_grad_()
    gx, gW = torch.autograd.grad(experts.product(a, b, order), (a, b), g)
    hx, = torch.autograd.grad(experts.product(a, W, order), a, g)
    hW, = torch.autograd.grad(experts.product(x, b, order), b, g)
    same(hx, gx, "rows"), same(hW, gW, "matrices")


def check_empty(_):
    for dt in DT.values():
        order = experts.sort_by_expert(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 3)
        x = torch.zeros(0, 16, dtype=dt, device="cuda", requires_grad=True)
        W = torch.randn(3, 5, 16, device="cuda").to(dt).requires_grad_()
        y = experts.product(x, W, order)
        assert y.shape == (0, 5)
        gx, gW = torch.autograd.grad(y.sum(), (x, W))
        assert gx.shape == (0, 16) and int(gW.count_nonzero()) == 0 and gW.shape == W.shape
        q = microscale4.quantize(x.detach())
        assert q.dequantize().shape == (0, 16)
        assert microscale4.product(q, microscale4.quantize(W.detach()[0])).shape == (0, 5)
        assert microscale4.experts_product(q, microscale4.quantize(W.detach()), order).shape == (0, 5)


def check_not_finite_products(_):
    """A block that is no number makes its row (of x) or column (of a matrix) of y NaN, and nothing else."""
    for rows, N in ((3, 40), (200, 140)):
        x, w = torch.randn(rows, 300, generator=gen(1)), torch.randn(N, 300, generator=gen(2))
        x[1, 299], w[2, 40] = math.inf, math.nan
        y = microscale4.product(microscale4.quantize(x.cuda()), microscale4.quantize(w.cuda())).cpu()
        want = torch.zeros(rows, N, dtype=torch.bool)
        want[1], want[:, 2] = True, True
        assert torch.equal(y.isnan(), want) and torch.isfinite(y[~want]).all()


def check_labels(_):
    """Labels of rows, as predict gives them, are choices of one expert each."""
    labels = torch.randint(0, 5, (77,), generator=gen(1), dtype=torch.int32)
    order = experts.sort_by_expert(labels.cuda(), 5)
    x, W = torch.randn(77, 20, generator=gen(2)), torch.randn(5, 12, 20, generator=gen(3))
    y = experts.combine(experts.product(experts.dispatch(x.cuda(), order), W.cuda(), order),
                        torch.ones(77, 1, device="cuda"), order)
    want = torch.einsum("tk,tnk->tn", x.double(), W[labels.long()].double())
    near(y, want, 36 * U32 * torch.einsum("tk,tnk->tn", x.double().abs(), W[labels.long()].double().abs()), "y")


def check_example(_):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import cluster_experts
    r = cluster_experts.main(["--rows", "1000", "--clusters", "4", "--steps", "2", "--quiet"])
    assert all(math.isfinite(v) for v in r.values()), r


def main():
    only = sys.argv[1] if len(sys.argv) > 1 else ""
    bad = 0
    for c in all_cases():
        if only not in c["name"]:
            continue
        r = dict(name=c["name"], ok=True, why="")
        print("# " + c["name"], flush=True)
        try:
            globals()["check_" + c["op"]](c)
            torch.cuda.synchronize()
        except Exception:  # reported to the collecting test
            r.update(ok=False, why=traceback.format_exc()[-1500:])
            bad += 1
            if "HIP error" in r["why"] or "CUDA error" in r["why"]:
                print(json.dumps(r), flush=True)
                return 1  # nothing more is run on the GPU
        print(json.dumps(r), flush=True)
        if c["op"] == "far_rows":
            torch.cuda.empty_cache()
    return 1 if bad else 0


if __name__ == "__main__":
    sys.exit(main())
