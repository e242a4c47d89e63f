"""Child process of test_gpu_large_products.py: runs every case of large_products_cases.py (or those whose names contain
argv[1]) and prints a JSON line for each. Not collected by pytest.

The oracle is the operator's formula in 64 bits, torch's products of float64 matrices on the GPU, expert by expert; the
bounds are those of products_device_check.py."""
import json
import os
import sys
import traceback

import numpy as np
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.dirname(HERE))
sys.path.insert(0, HERE)
from large_products_cases import DROPPED, all_cases  # noqa: E402
from products_device_check import DT, LEVELS, ROUND, TINY, U32, numbers, roundings, stretches  # noqa: E402
from h2o4gpu_amd import experts, microscale4  # noqa: E402


class Found:
    """Results held against formulas piece by piece, without a wait between them."""

    def __init__(self):
        self.bad = {}

    def add(self, what, got, want, bound):
        """|got - want| <= bound + the last rounding, element by element; all of them numbers."""
        u, tiny = ROUND[got.dtype], TINY[got.dtype]
        assert got.shape == want.shape, "%s: shape %s, expected %s" % (what, tuple(got.shape), tuple(want.shape))
        off = (got.double() - want).abs()
        wrong = ~(off <= bound + u * (want.abs() + bound) + tiny)
        count = wrong.sum() + torch.zeros((), dtype=torch.int64, device="cuda")
        self.bad[what] = self.bad.get(what, 0) + count

    def check(self):
        found = {k: int(v) for k, v in self.bad.items()}
        assert found and not any(found.values()), "numbers off: %s" % found


def chosen(c):
    """Uneven experts, the second without a row; with `most` the last but one has six of ten slots."""
    rng = np.random.default_rng(c["tokens"] + c["experts"])
    T, K, E = c["tokens"], c["top_k"], c["experts"]
    liking = rng.exponential(1.0, E) + 0.3
    liking[1] = 0
    e = rng.choice(E, (T, K), p=liking / liking.sum())
    if c["most"]:
        e = np.where(rng.random((T, K)) < 0.6, E - 2, e)
    return np.where(rng.random((T, K)) < DROPPED, -1, e).astype(np.int32)


def drawn(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def check_large(c):
    E, N, K, dt = c["experts"], c["out"], c["cols"], DT[c["dtype"]]
    e = chosen(c)
    order = experts.sort_by_expert(torch.from_numpy(e).cuda(), E)
    _, at = stretches(e, E)
    S, held = e.size, int(at[-1])
    assert any(at[i] == at[i + 1] for i in range(E)) and held < S
    x = torch.randn(S, K, device="cuda", generator=drawn(1)).to(dt)
    W = torch.randn(E, N, K, device="cuda", generator=drawn(2)).to(dt)
    g = torch.randn(S, N, device="cuda", generator=drawn(3)).to(dt)
    x[held:], g[held:] = float("nan"), float("inf")
    x.requires_grad_(), W.requires_grad_()
    y = experts.product(x, W, order)
    gx, gW = torch.autograd.grad(y, (x, W), g)
    x, W, y = x.detach(), W.detach(), y.detach()
    found, zero = Found(), torch.zeros((), dtype=torch.float64, device="cuda")
    for i in range(E):
        lo, hi = int(at[i]), int(at[i + 1])
        if lo == hi:
            found.add("gradient of unused matrices", gW[i], torch.zeros_like(gW[i], dtype=torch.float64), zero)
            continue
        a, b, d = x[lo:hi].double(), W[i].double(), g[lo:hi].double()
        found.add("y", y[lo:hi], a @ b.t(), roundings(K, dt) * U32 * (a.abs() @ b.t().abs()))
        found.add("gradient of the rows", gx[lo:hi], d @ b, roundings(N, dt) * U32 * (d.abs() @ b.abs()))
        found.add("gradient of the matrices", gW[i], d.t() @ a, roundings(hi - lo, dt) * U32 * (d.t().abs() @ a.abs()))
    for what, t in (("y behind", y), ("gradient of the rows behind", gx)):
        found.add(what, t[held:], torch.zeros_like(t[held:], dtype=torch.float64), zero)
    found.check()


def matrix(lead, K, seed, dt):
    """A Microscale4 of random codes, and a function: the values of some of its rows in 64 bits."""
    rows, g = int(np.prod(lead)), drawn(seed)
    code = torch.randint(0, 16, (rows, K + K % 2), generator=g, dtype=torch.uint8, device="cuda")
    scale = torch.randint(119, 129, (rows, -(-K // 32)), generator=g, dtype=torch.uint8, device="cuda")
    packed = code[:, 0::2] | (code[:, 1::2] << 4)
    m = microscale4.Microscale4(packed.reshape(lead + (-1,)), scale.reshape(lead + (-1,)), K, dtype=dt)

    def values(pick):
        c, s = code[pick, :K], scale[pick]
        v = LEVELS.cuda()[(c & 7).long()] * torch.where(c >= 8, -1.0, 1.0)
        return v * torch.exp2(s.double() - 127).repeat_interleave(32, dim=1)[:, :K]

    return m, values


def check_large_four(c):
    dt, K = DT[c["dtype"]], c["cols"]
    x, vx = matrix((c["rows"],), K, 1, dt)
    w, vw = matrix((c["out"],), K, 2, dt)
    y = microscale4.product(x, w)
    a, b, found = vx(slice(None)), vw(slice(None)), Found()
    found.add("y", y, a @ b.t(), (K / 8 + 16) * U32 * (a.abs() @ b.t().abs()))
    found.check()


def check_large_fours(c):
    E, N, K, dt = c["experts"], c["out"], c["cols"], DT[c["dtype"]]
    e = chosen(c)
    order = experts.sort_by_expert(torch.from_numpy(e).cuda(), E)
    slots, at = stretches(e, E)
    held = int(at[-1])
    w, vw = matrix((E, N), K, 2, dt)
    x, vx = matrix((e.size if c["in_order"] else c["tokens"],), K, 1, dt)
    y = microscale4.experts_product(x, w, order, in_order=c["in_order"])
    token = torch.from_numpy(np.arange(e.size) if c["in_order"] else slots // c["top_k"]).cuda()
    found = Found()
    for i in range(E):
        lo, hi = int(at[i]), int(at[i + 1])
        if lo < hi:
            a, b = vx(token[lo:hi]), vw(slice(i * N, (i + 1) * N))
            found.add("y", y[lo:hi], a @ b.t(), (K / 8 + 16) * U32 * (a.abs() @ b.t().abs()))
    found.add("y behind", y[held:], torch.zeros_like(y[held:], dtype=torch.float64), 0.0 * y.new_zeros((), dtype=torch.float64))
    found.check()


def check_rows_of_any_stride(_):
    """A matrix per expert is copied where its rows are not contiguous, of one row as of several."""
    for E, rows in ((1, 1), (2, 1), (1, 3), (3, 4)):
        for v in (torch.randn(E, rows, 80, generator=drawn(5), device="cuda")[..., ::2],
                  torch.randn(E, 40, rows, generator=drawn(6), device="cuda").transpose(1, 2),
                  torch.randn(E, 1, 40, generator=drawn(7), device="cuda").expand(E, rows, 40)):
            m, (code, scale, _) = microscale4.quantize(v), numbers(v.reshape(-1, 40).cpu())
            assert m.codes().reshape(-1, 40).cpu().equal(code) and m.scales().reshape(-1, 2).cpu().equal(scale)


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
        torch.cuda.empty_cache()
    return 1 if bad else 0


if __name__ == "__main__":
    sys.exit(main())
