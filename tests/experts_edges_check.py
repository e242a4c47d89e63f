"""Child process of test_gpu_experts_edges.py: runs the checks named on the command line and prints a JSON
line for each. Not collected by pytest.

Oracles are the formulas in 64 bits; U32 is the largest relative error of one float32 rounding."""
import json
import os
import sys
import traceback

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))
from experts_device_check import _order, choices, matrix, near, order_oracle, product_bound  # noqa: E402
from h2o4gpu_amd import codebook4, experts  # noqa: E402

U32 = 2.0 ** -24


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def codebook_of_all_experts():
    """More rows and more values than a fit takes: the second expert's values are in the sample. Its scaled
    values lie in the outer fifth, where a codebook of the first expert's alone has its entries wide apart."""
    first = torch.randn(4000, 320, generator=gen(70))
    second = 0.8 + 0.2 * torch.rand(4000, 320, generator=gen(71))
    second = torch.where(torch.rand(second.shape, generator=gen(72)) < 0.5, -second, second)
    W = torch.stack([first, second]).cuda()

    def error(book):
        q = codebook4.quantize(W[1], 32, book)
        scale = q.scales().repeat_interleave(32, 1)
        return float(((q.dequantize() - W[1]) / scale).square().mean())

    joint = error(codebook4.quantize(W, 32).codebook)
    alone = error(codebook4.quantize(W[0], 32).codebook)
    # sixteen entries of a mixture by halves: a third of the error at most (about an eighth, were they those of
    # Lloyd's fixed point on the whole matrices)
    assert joint < alone / 3, (joint, alone)


def softmax_over_all(s, K, largest, scale):
    """Choice, softmax over all experts and its exponents in 64 bits; no score is masked."""
    key = s.double() if largest else -s.double()
    chosen = torch.argsort(key, dim=1, descending=True, stable=True)[:, :K]
    x = scale * (key - key.amax(1, keepdim=True))
    return chosen, torch.softmax(x, 1), x


# the largest relative error of a result's last rounding, 2^-(bits of its significand, 24, 8 and 11), and its
# smallest number
LAST = {torch.float32: (2.0 ** -24, 2.0 ** -126), torch.bfloat16: (2.0 ** -8, 2.0 ** -126), torch.float16: (2.0 ** -11, 2.0 ** -24)}


def check_over_all(s, K, largest, scale, place, chain, g, same_rows=None):
    """route over all experts and its gradient, each number against its own size. s: scores on the host, place(s):
    them on the GPU; same_rows: which row of s each row of place(s) is (all of them, one after another).

    Roundings, in U32: an exponent x is the product of two rounded factors and rounded itself, so e^x is off by
    3 |x|, and by 4 for the exponential. A sum over all is off by its terms' errors, each by its share p of the sum,
    and by `chain`, the additions one after another (and what moves the sum to another best score). A weight: its
    term, the sum, a division. A gradient: scale * p * (g - inner), inner a sum of K products."""
    rows, E = s.shape
    chosen, p, x = softmax_over_all(s, K, largest, scale)
    d = place(s).requires_grad_()
    got, weights = experts.route(d, K, largest=largest, scale=scale, over_all=True)
    ds, = torch.autograd.grad(weights, d, g[same_rows].cuda() if same_rows is not None else g.cuda())
    if same_rows is not None:
        for t in (got, weights, ds):
            for lo in range(rows, t.shape[0], rows):
                part = t[lo:lo + rows]
                assert torch.equal(part, t[:part.shape[0]]), "equal rows, other results"
        got, weights, ds = got[:rows], weights[:rows], ds[:rows]
    assert torch.equal(got.cpu().long(), chosen), "choice"
    total = 3 * (p * -x).sum(1, keepdim=True) + 4 + chain
    pick = p.gather(1, chosen)
    c = 3 * -x.gather(1, chosen) + 4 + total + 2
    off = (weights.detach().cpu().double() - pick).abs() / pick / U32
    assert bool((off <= c).all()), "weights off by %.0f, %.0f allowed" % (float((off / c).max() * c.max()), float(c.max()))
    full = torch.zeros_like(p).scatter_(1, chosen, g.double())
    inner = (pick * g.double()).sum(1, keepdim=True)
    sign = scale if largest else -scale
    want = sign * p * (full - inner)
    size = scale * p * (full.abs() + (pick * g.double().abs()).sum(1, keepdim=True))
    u, tiny = LAST[s.dtype]
    bound = U32 * size * (2 * c.amax(1, keepdim=True) + 3 * -x + 4 + K + 6)
    bound += u * (want.abs() + bound) + tiny
    off = (ds.cpu().double() - want).abs()
    assert bool((off <= bound).all()), "gradient off by %.3g times what is allowed" % float((off / bound).max())
    # zeros in place of the gradients of experts that are not chosen would be seen
    others = torch.ones_like(p).scatter_(1, chosen, 0.0).bool()
    held = others & (want.abs() > 64 * tiny)
    assert E == K or float(held.sum()) > 0.5 * float(others.sum())
    assert bool((want.abs() > 8 * bound)[held].all())


def long_sums_of_distances():
    """So many rows that one lane has all of a row's distances. Rows whose other experts all have one term, for
    which roundings do not even out, and rows that get better, or worse, by equal steps."""
    K, scale = 2, 0.7
    for E in (1000, 4096):
        term = torch.linspace(0.01, 0.9, 90, dtype=torch.float64)
        s = (-torch.log(term) / scale)[:, None].repeat(1, E).float() + 1
        s.scatter_(1, torch.randint(0, E, (90, 1), generator=gen(80)), 1.0)
        steps = torch.arange(E).float()[None] * torch.tensor([0.001, 0.01, 0.1])[:, None]
        s = torch.cat([s, steps, steps.flip(1), 3 * torch.rand(30, E, generator=gen(81))])
        at = torch.arange(131072 + 77) % s.shape[0]
        g = 0.5 + torch.rand(s.shape[0], K, generator=gen(82))
        # a lane's sum: pairs of eight (3), an addition (2), moves of the sum (8 each, every one a factor e less)
        check_over_all(s, K, False, scale, lambda s: s.t().cuda()[:, at.cuda()].t(), 3 + 2 + 13 + 5, g, at)


def every_number_by_its_size():
    """Weights and gradients over all experts, each against its own size, in all layouts and through every kernel
    (rows in registers of 4, 16 or 64 lanes, rows of any length, distances in 1 to 16 stretches). Sums: 16 terms of
    a lane and 6 joins, or E / 64 and 6, or as in long_sums_of_distances with 4 joins (each 3 * 0.4 + 3)."""
    for rows, E, K in ((50, 3, 2), (300, 12, 4), (77, 60, 5), (40, 250, 8), (33, 1000, 8), (20, 1024, 64), (12, 1025, 3),
                       (9, 1500, 8), (6, 4099, 5), (3, 16384, 33), (5, 16384, 8), (2000, 40, 1), (9000, 130, 6)):
        for dt in (torch.float32, torch.bfloat16, torch.float16):
            s = torch.randn(rows, E, generator=gen(rows + E)).to(dt)
            # (half a float16 gradient's bits would be lost where a weight is a ten-thousandth)
            g = (0.5 + torch.rand(rows, K, generator=gen(93))) * (1000 if dt == torch.float16 else 1)
            chain = 40 + E / 64

            def gaps(s):
                wide = torch.zeros(2 * rows, 3 * E, dtype=dt, device="cuda")[::2, ::3]
                return wide.copy_(s)

            check_over_all(s, K, True, 1.0, lambda s: s.cuda(), chain, g)
            check_over_all(s, K, False, 0.7, lambda s: s.t().contiguous().cuda().t(), chain, g)
            check_over_all(s, K, True, 0.7, gaps, chain, g)


def small_gradients():
    """Gradients of scores far below the best one, against each other: they are one factor of the row times their
    terms e^x. Scores are multiples of a sixteenth, so that x is exact; a term is off by 4 U32 (exponential) and one
    for each of three products, its neighbour likewise."""
    rows, E, K = 64, 300, 2
    x = -5 - torch.randint(0, 1200, (rows, E), generator=gen(90)).float() / 16
    x[:, :2] = -5
    x[:, 7] = 0
    g = 0.5 + torch.rand(rows, K, generator=gen(91))
    for largest in (True, False):
        s = x if largest else -x
        wide = torch.zeros(2 * rows, 3 * E, device="cuda")[::2, ::3]
        wide.copy_(s)
        for d in (s.cuda(), s.t().contiguous().cuda().t(), wide):
            d = d.detach().requires_grad_()
            chosen, weights = experts.route(d, K, largest=largest, over_all=True)
            assert bool((chosen.cpu()[:, 0] == 7).all() and (chosen.cpu()[:, 1] == 0).all())
            ds, = torch.autograd.grad(weights, d, g.cuda())
            ratio = ds.cpu().double() / ds.cpu().double()[:, 1:2]
            want = torch.exp(x.double() - x.double()[:, 1:2])
            off = (ratio / want - 1).abs() / U32
            off[:, 0] = off[:, 7] = 0  # (the chosen ones)
            assert float(off.max()) <= 14, "strides %s: off by %.1f" % (d.stride(), float(off.max()))


def tokens_that_are_not_finite():
    """A NaN or an infinity in one token's row is in that token's results, as multiplying would have it, and in no
    other's, though few rows share a matrix instruction and are multiplied with more than their own columns."""
    def spoiled(rows, cols, dt, seed):
        x = torch.randn(rows, cols, generator=gen(seed)).to(dt)
        x[0, cols // 2] = float("nan")
        if rows > 1:
            x[1, 0] = float("inf")
        if rows > 3:
            x[2, cols - 1] = -float("inf")
        if rows > 15:
            x[-2, cols // 3] = float("inf")
            x[-2, cols // 2] = -float("inf")
        return x

    for dtype in ("float32", "bfloat16", "float16"):
        for rows in (1, 2, 3, 4, 5, 16, 33, 70):
            for n, cols, group in ((40, 300, 32), (33, 2047, 64), (200, 1024, 128)):
                w, W = matrix(dict(out=n, cols=cols, group=group, dtype=dtype, layout="plain"), ())
                x = spoiled(rows, cols, getattr(torch, dtype), 95)
                near(codebook4.product(x.cuda(), w), x.double() @ W.t(), product_bound(x, W), "y")
        for tokens, top_k, E in ((1, 2, 8), (4, 2, 3), (40, 3, 4)):
            c = dict(tokens=tokens, top_k=top_k, experts=E, out=40, cols=300, group=64, dtype=dtype, layout="plain")
            e, o, pos = _order(c)
            w, W = matrix(c, (E,))
            x = spoiled(tokens, 300, getattr(torch, dtype), 96)
            want, bound = torch.zeros(tokens * top_k, 40, dtype=torch.float64), torch.zeros(tokens * top_k, 40, dtype=torch.float64)
            for t in range(tokens):
                for j in range(top_k):
                    want[pos[t, j]] = W[e[t, j]] @ x[t].double()
                    bound[pos[t, j]] = product_bound(x[t:t + 1], W[e[t, j]])[0]
            near(codebook4.experts_product(x.cuda(), w, o), want, bound, "rows")


def a_token_served_alone():
    """The example's serving path: tokens one by one and all at once, both against the formula."""
    from cluster_experts import serve
    rows, E, K, d, n, scale = 60, 7, 2, 96, 50, 0.3
    x, near_by = torch.randn(rows, d, generator=gen(100)), torch.rand(rows, E, generator=gen(101)) * 9
    distances = near_by.t().contiguous().cuda().t()
    packed = codebook4.quantize(torch.randn(E, n, d, generator=gen(102)).cuda(), 32)
    W = packed.dequantize().cpu().double()
    key = -near_by.double()
    chosen = torch.argsort(key, dim=1, descending=True, stable=True)[:, :K]
    w = torch.softmax(scale * key.gather(1, chosen), 1)
    want, bound = torch.zeros(rows, n, dtype=torch.float64), torch.zeros(rows, n, dtype=torch.float64)
    for t in range(rows):
        for j in range(K):
            e = int(chosen[t, j])
            y = W[e] @ x[t].double()
            want[t] += w[t, j] * y
            # a weight: exponent (2 * 3 at most here), exponential, sum, division; the join
            bound[t] += w[t, j] * (product_bound(x[t:t + 1], W[e])[0] + (2 * 3 + 4 + K + 2 + K + 1) * U32 * y.abs())
    near(serve(x.cuda(), distances, packed, K, scale), want, bound, "all")
    for t in (0, 1, 31, rows - 1):
        near(serve(x[t:t + 1].cuda(), distances[t:t + 1], packed, K, scale), want[t:t + 1], bound[t:t + 1], "token %d" % t)


def labels_in_order():
    """Labels, one a row, in place of choices."""
    for rows, E in ((0, 3), (1, 1), (1000, 7), (70_000, 300)):
        labels = choices(rows, 1, E, "dropped")
        order, position, offsets = order_oracle(labels, E)
        o = experts.sort_by_expert(torch.from_numpy(labels[:, 0].copy()).cuda(), E)
        for got, want in ((o.order, order), (o.position, position), (o.offsets, offsets)):
            assert torch.equal(got.cpu(), torch.from_numpy(want)), (rows, E)


def refuses(kind, f, *args, **kw):
    try:
        f(*args, **kw)
    except kind:
        return
    raise AssertionError("%s was not refused with %s" % (f.__name__, kind.__name__))


def forward_mode_is_refused():
    """A tangent is refused, not dropped; tensors without one are taken inside of a dual level as well."""
    from torch.autograd import forward_ad
    T, K, E, d = 6, 2, 4, 64
    s, x, y = (torch.randn(T, E, device="cuda"), torch.randn(T, d, device="cuda"), torch.randn(T * K, d, device="cuda"))
    w = torch.rand(T, K, device="cuda")
    o = experts.sort_by_expert(experts.route(s, K)[0], E)
    W = torch.randn(E, 20, d, device="cuda")
    book = torch.linspace(-1, 1, 16, device="cuda")
    one, many = codebook4.quantize(W[0], 32, book), codebook4.quantize(W, 32, book)
    calls = ((experts.route, (s, K), 1), (experts.dispatch, (x, o), 1), (experts.combine, (y, w, o), 2),
             (codebook4.product, (x, one), 1), (codebook4.experts_product, (x, many, o), 1))
    for f, args, tensors in calls:
        want = f(*args)
        with forward_ad.dual_level():
            for at in range(tensors):
                for given in (args[at], args[at].clone().requires_grad_()):
                    if f.__module__.endswith("codebook4") and given.requires_grad:
                        continue  # (refused for its gradient)
                    dual = forward_ad.make_dual(given, torch.ones_like(given))
                    refuses(NotImplementedError, f, *(args[:at] + (dual,) + args[at + 1:]))
            got = f(*args)
        for a, b in zip(got, want) if isinstance(got, tuple) else ((got, want),):
            assert torch.equal(a, b)


def second_derivatives():
    """create_graph: gradients come as without it, those of other layers can be differentiated again, and what
    needs a second derivative of an expert layer is an error, also where the incoming gradient is a constant."""
    T, K, E, d = 6, 2, 4, 64
    o = experts.sort_by_expert(experts.route(torch.randn(T, E, device="cuda"), K)[0], E)

    def leaf(*shape):
        return torch.randn(*shape, device="cuda", requires_grad=True)

    s, x, y, w = leaf(T, E), leaf(T, d), leaf(T * K, d), leaf(T, K)
    by = torch.randn(T, K, device="cuda")
    layers = (([s], lambda: (experts.route(s, K)[1] * by).sum(), [True]),
              ([s], lambda: experts.route(s, K, over_all=True)[1].square().sum(), [True]),
              ([x], lambda: experts.dispatch(x, o).square().sum(), [True]),
              ([x], lambda: experts.dispatch(x, o).sum(), [False]),  # (the gradient is top_k, whatever x is)
              ([y, w], lambda: experts.combine(y, w, o).sum(), [True, True]),
              ([y, w], lambda: experts.combine(y, w, o).square().sum(), [True, True]))
    for leaves, f, depends in layers:
        want = torch.autograd.grad(f(), leaves)
        scale = leaf(1)
        got = torch.autograd.grad(f() * 1 + scale.pow(3).sum(), leaves + [scale], create_graph=True)
        for a, b, on in zip(got, want, depends):
            assert torch.equal(a, b) and a.requires_grad == on
            if on:
                refuses(RuntimeError, torch.autograd.grad, a.square().sum(), leaves, retain_graph=True, allow_unused=True)
        # a penalty on another layer's gradient
        second, = torch.autograd.grad(got[-1].square().sum(), scale)
        assert torch.allclose(second, 36 * scale.detach() ** 3)
        # gradients added up in place, twice
        for t in leaves:
            t.grad = None
        for k in (1, 2):
            f().backward(create_graph=True)
            for t, b in zip(leaves, want):
                assert torch.allclose(t.grad, k * b, rtol=1e-6)
        for t in leaves:
            t.grad = None


def groups_longer_than_a_row():
    """One scale a row, with groups of any length; a length that the library's int would cut off is refused (its
    rows of scales would be other ones than those that were allocated)."""
    W = torch.randn(40, 100, generator=gen(110)).cuda()
    book = torch.linspace(-1, 1, 16, device="cuda")
    x = torch.randn(3, 100, generator=gen(111)).cuda()
    want = codebook4.quantize(W, 128, book)
    fitted = codebook4.quantize(W, 128)
    for group in (256, 32 * 1001, 1 << 30):
        q = codebook4.quantize(W, group, book)
        assert torch.equal(q.codes(), want.codes()) and torch.equal(q.scales(), want.scales())
        assert torch.equal(q.dequantize(), want.dequantize())
        near(codebook4.product(x, q), x.cpu().double() @ q.dequantize().cpu().double().t(),
             product_bound(x.cpu(), q.dequantize().cpu().double()), "y")
        # (means of at most 4000 values, whose order of addition is the fit's own)
        assert float((codebook4.quantize(W, group).codebook - fitted.codebook).abs().max()) <= 4000 * U32
    codes, scales = torch.zeros(40, 50, dtype=torch.uint8, device="cuda"), torch.ones(40, 1, device="cuda")
    for group in ((1 << 30) + 32, 2 ** 31 - 32, 2 ** 31, 2 ** 32 + 32, 2 ** 40):
        refuses(ValueError, codebook4.quantize, W, group, book)
        refuses(ValueError, codebook4.Codebook4, codes, scales, book, 100, group)


def main():
    for name in sys.argv[1:]:
        print("# " + name, flush=True)
        r = dict(name=name, ok=True, why="")
        try:
            globals()[name]()
            torch.cuda.synchronize()
        except Exception as e:  # reported to the collecting test
            r.update(ok=False, why="".join(traceback.format_exception_only(type(e), e))[:1500] +
                     "".join(traceback.format_tb(e.__traceback__)[-2:])[:1000])
            if "HIP error" in r["why"] or "CUDA error" in r["why"]:
                print(json.dumps(r), flush=True)
                return 1  # nothing more is run on the GPU
        print(json.dumps(r), flush=True)
        torch.cuda.empty_cache()
    return 0


if __name__ == "__main__":
    sys.exit(main())
