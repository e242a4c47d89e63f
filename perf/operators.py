"""Expert layers and 4-bit products as cases that can be timed and compared.

A case is a dict of plain values; prepare() makes what a user's program holds before the call, run()
is one pass through an operator: with `own` through the framework's entry points, without it in a
plain form of elementary torch operations in 32 bits, rounded once at the end. exact() is the
operator's definition in 64 bits. Sizes are this repository's benchmark shapes or generic.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # A serving loop routes a handful of requests by their distances to 8 centres, as
        # transform() leaves them (one centre's distances side by side).
        dict(name="route_serve_1k_e8", op="route", rows=1000, experts=8, top_k=2, dtype="float32",
             distances=True, over_all=False, train=False),
        # Every row of the million-row benchmark table goes to the models of its two nearest centres of 64.
        dict(name="route_1m_e64", op="route", rows=1_000_000, experts=64, top_k=2, dtype="float32",
             distances=True, over_all=False, train=False),
        # A training step of a router: 16k tokens, 256 learned scores each, eight taken, and the
        # gradient with respect to the scores.
        dict(name="route_train_16k_e256", op="route", rows=16_384, experts=256, top_k=8, dtype="bfloat16",
             distances=False, over_all=True, train=True),
        # One batch of a serving loop goes out to its experts: launch latency.
        dict(name="dispatch_serve_16", op="dispatch", rows=16, cols=4096, experts=8, top_k=2, dtype="bfloat16",
             dropped=0.0, train=False),
        # A training step sends 16k tokens to four of 64 experts and brings the gradient back.
        dict(name="dispatch_train_16k", op="dispatch", rows=16_384, cols=2048, experts=64, top_k=4,
             dtype="bfloat16", dropped=0.0, train=True),
        # Odd sizes on every axis, a model per cluster, some slots without an expert.
        dict(name="dispatch_train_100k_d101", op="dispatch", rows=100_003, cols=101, experts=1000, top_k=3,
             dtype="float32", dropped=0.03, train=True),
        # The serving batch's results come back and are joined by weight.
        dict(name="combine_serve_16", op="combine", rows=16, cols=4096, experts=8, top_k=2, dtype="bfloat16",
             dropped=0.0, train=False),
        # The training step's results are joined; gradients of the results and of the weights.
        dict(name="combine_train_16k", op="combine", rows=16_384, cols=2048, experts=64, top_k=4,
             dtype="bfloat16", dropped=0.01, train=True),
        # One new token through one 4-bit layer.
        dict(name="product_1x4096x4096", op="product", rows=1, out=4096, cols=4096, group=128, dtype="bfloat16"),
        # A batch of tokens, odd sizes, the last group cut short.
        dict(name="product_33x11003x8190", op="product", rows=33, out=11_003, cols=8190, group=64, dtype="float16"),
        # One new token through two of 16 experts.
        dict(name="experts_1_e16", op="experts", rows=1, experts=16, top_k=2, out=4096, cols=2048, group=32,
             dtype="bfloat16"),
        # A serving batch through four of 64 experts, some with many tokens and some with none.
        dict(name="experts_64_e64", op="experts", rows=64, experts=64, top_k=4, out=2048, cols=4096, group=128,
             dtype="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges, no dearer than the dearest of them."""
    op = rng.choice(["route", "dispatch", "combine", "product", "product", "experts"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "route":
        distances = rng.random() < 0.5
        experts = _log_int(rng, 2, 1000)
        rows = min(_log_int(rng, 1, 1_000_000), 64_000_000 // experts)
        return dict(op=op, rows=rows, experts=experts, top_k=min(experts, rng.randint(1, 8)),
                    dtype="float32" if distances else dtype, distances=distances,
                    over_all=rng.random() < 0.5, train=rng.random() < 0.5)
    if op in ("dispatch", "combine"):
        cols, top_k, experts = _log_int(rng, 16, 8192), rng.randint(1, 8), _log_int(rng, 2, 1000)
        rows = min(_log_int(rng, 1, 200_000), 128_000_000 // (cols * top_k))
        return dict(op=op, rows=max(1, rows), cols=cols, experts=experts, top_k=min(top_k, experts), dtype=dtype,
                    dropped=rng.choice([0.0, 0.0, 0.05]), train=rng.random() < 0.6)
    group = rng.choice([32, 64, 128, 256])
    cols = _log_int(rng, 64, 8192)
    if op == "product":
        return dict(op=op, rows=_log_int(rng, 1, 64), out=_log_int(rng, 64, 11_000), cols=cols, group=group,
                    dtype=dtype)
    experts = _log_int(rng, 2, 64)
    out = min(_log_int(rng, 64, 4096), 500_000_000 // (experts * cols))
    return dict(op=op, rows=_log_int(rng, 1, 64), experts=experts, top_k=min(experts, rng.randint(1, 4)), out=out,
                cols=cols, group=group, dtype=dtype)


def _choices(case, gen):
    """(rows, top_k) distinct experts a row, some of them more popular than others; `dropped` of the
    slots have none."""
    T, E, k = case["rows"], case["experts"], case["top_k"]
    liking = torch.rand((T, E), device="cuda", generator=gen) + 0.3 * torch.rand((1, E), device="cuda", generator=gen)
    experts = torch.topk(liking, k, dim=1).indices.to(torch.int32)
    if case.get("dropped", 0.0) > 0:
        experts[torch.rand((T, k), device="cuda", generator=gen) < case["dropped"]] = -1
    return experts.contiguous()


def _quantized(case, gen, lead):
    """Codes, group scales and the 16 values of a compressed matrix, as compressing normal weights leaves them."""
    N, K, group, dt = case["out"], case["cols"], case["group"], TYPES[case["dtype"]]
    pitch = (K + 31) // 32 * 16
    codes = torch.randint(0, 256, lead + (N, pitch), device="cuda", generator=gen, dtype=torch.uint8)
    scales = (0.02 + 0.02 * torch.rand(lead + (N, -(-K // group)), device="cuda", generator=gen)).to(
        torch.float32 if case["dtype"] == "float32" else dt)
    at = (torch.arange(16, device="cuda") + 0.5) / 16
    book = torch.erfinv(2 * at - 1)
    book = book / book.abs().max() + 0.01 * torch.randn(16, device="cuda", generator=gen)
    return codes, scales, book.to(dt)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2000 + int(seed))
    dt, op, T = TYPES[case["dtype"]], case["op"], case["rows"]

    def randn(*shape, dtype=dt):
        return torch.randn(shape, device="cuda", generator=gen).to(dtype)

    s = dict(case=case)
    if op == "route":
        E = case["experts"]
        if case["distances"]:  # squared distances in the layout of KMeans.transform, one centre's after another
            s["scores"] = ((randn(E, T) + 3).square_() + 1).t()
        else:
            s["scores"] = randn(T, E)
        if case["train"]:
            s["scores"].requires_grad_()
            s["grad"] = randn(T, case["top_k"], dtype=torch.float32)
        return s
    if op in ("dispatch", "combine"):
        s["experts"] = _choices(case, gen)
        S, d = T * case["top_k"], case["cols"]
        if op == "dispatch":
            s["x"] = randn(T, d)
            if case["train"]:
                s["grad"] = randn(S, d)
                s["x"].requires_grad_()
        else:
            from_order = torch.rand((T, case["top_k"]), device="cuda", generator=gen)
            s["rows"], s["weights"] = randn(S, d), from_order / from_order.sum(1, keepdim=True)
            if case["train"]:
                s["grad"] = randn(T, d)
                s["rows"].requires_grad_()
                s["weights"].requires_grad_()
        return s
    lead = (case["experts"],) if op == "experts" else ()
    s["codes"], s["scales"], s["book"] = _quantized(case, gen, lead)
    s["x"] = randn(T, case["cols"])
    if op == "experts":
        s["experts"] = _choices(case, gen)
    return s


# ---- the framework's operators ----------------------------------------------------------------

def _run_own(s):
    from h2o4gpu_amd import codebook4, experts
    case = s["case"]
    op = case["op"]
    if op == "route":
        scale = -0.25 if case["distances"] else 1.0
        chosen, weights = experts.route(s["scores"], case["top_k"], largest=not case["distances"],
                                        scale=abs(scale), over_all=case["over_all"])
        out = dict(experts=chosen, weights=weights)
        if case["train"]:
            out["dscores"], = torch.autograd.grad(weights, s["scores"], s["grad"])
        return out
    if op == "dispatch":
        order = experts.sort_by_expert(s["experts"], case["experts"])
        rows = experts.dispatch(s["x"], order)
        out = dict(order=order.order, position=order.position, offsets=order.offsets, rows=rows)
        if case["train"]:
            out["dx"], = torch.autograd.grad(rows, s["x"], s["grad"])
        return out
    if op == "combine":
        order = experts.sort_by_expert(s["experts"], case["experts"])
        joined = experts.combine(s["rows"], s["weights"], order)
        out = dict(out=joined)
        if case["train"]:
            out["drows"], out["dweights"] = torch.autograd.grad(joined, (s["rows"], s["weights"]), s["grad"])
        return out
    weights = s.get("laid_out")
    if weights is None:  # weights are laid out once, as a program that serves them does
        weights = s["laid_out"] = codebook4.Codebook4(s["codes"], s["scales"], s["book"], case["cols"], case["group"])
    if op == "product":
        return codebook4.product(s["x"], weights)
    return codebook4.experts_product(s["x"], weights, experts.sort_by_expert(s["experts"], case["experts"]))


# ---- plain forms -------------------------------------------------------------------------------

def _sorted_slots(experts, E):
    """Stable order of the slots by expert, each slot's place in it (~place where it has no expert), and
    where every expert's rows begin."""
    flat = experts.reshape(-1)
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    counts = torch.zeros(E + 1, dtype=torch.int64, device=flat.device)
    ends = torch.cumsum(counts.scatter_add_(0, key.to(torch.int64), torch.ones_like(order))[:E], 0)
    offsets = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    position = torch.where(key < E, place, ~place).to(torch.int32).reshape(experts.shape)
    return order.to(torch.int32), position, offsets


def _dequantized(codes, scales, book, K, group):
    pairs = torch.stack([book[torch.arange(256, device=book.device) & 15],
                         book[torch.arange(256, device=book.device) >> 4]], 1).float()
    values = pairs[codes.to(torch.int32)].flatten(-2)[..., :K]
    return values * scales.float().repeat_interleave(group, dim=-1)[..., :K]


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "route":
        x = s["scores"].float() * (-0.25 if case["distances"] else 1.0)
        best, index = torch.sort(x, dim=1, descending=True, stable=True)
        best, index = best[:, :case["top_k"]], index[:, :case["top_k"]]
        top = torch.exp(best - best[:, :1])
        every = torch.exp(x - best[:, :1]) if case["over_all"] else top
        total = every.sum(1, keepdim=True)
        weights = top / total
        out = dict(experts=index.to(torch.int32), weights=weights)
        if case["train"]:
            inner = (weights * s["grad"]).sum(1, keepdim=True)
            if case["over_all"]:
                d = -inner * every / total
                d.scatter_add_(1, index, weights * s["grad"])
            else:
                d = torch.zeros_like(x).scatter_(1, index, weights * (s["grad"] - inner))
            out["dscores"] = (d * (-0.25 if case["distances"] else 1.0)).to(s["scores"].dtype)
        return out
    if op in ("dispatch", "combine"):
        order, position, offsets = _sorted_slots(s["experts"], case["experts"])
        kept = position >= 0
        at = torch.where(kept, position, 0).to(torch.int64)
        token = order.to(torch.int64) // case["top_k"]
        filled = (torch.arange(order.numel(), device=order.device) < offsets[-1])[:, None]
        if op == "dispatch":
            out = dict(order=order, position=position, offsets=offsets,
                       rows=torch.where(filled, s["x"][token], torch.zeros((), dtype=s["x"].dtype, device="cuda")))
            if case["train"]:
                back = s["grad"].float()[at] * kept[:, :, None]
                out["dx"] = back.sum(1).to(s["x"].dtype)
            return out
        y = s["rows"].float()[at] * kept[:, :, None]
        out = dict(out=(y * s["weights"][:, :, None]).sum(1).to(s["rows"].dtype))
        if case["train"]:
            g = s["grad"].float()
            slot = s["weights"].reshape(-1)[order.to(torch.int64)][:, None]
            out["drows"] = torch.where(filled, g[token] * slot, 0).to(s["rows"].dtype)
            out["dweights"] = (y * g[:, None, :]).sum(2)
        return out
    K, group = case["cols"], case["group"]
    x = s["x"].float()
    if op == "product":
        return torch.matmul(x, _dequantized(s["codes"], s["scales"], s["book"], K, group).t()).to(s["x"].dtype)
    order, position, offsets = _sorted_slots(s["experts"], case["experts"])
    token = order.to(torch.int64) // case["top_k"]
    S, E = order.numel(), case["experts"]
    of_row = s["experts"].reshape(-1)[order.to(torch.int64)].to(torch.int64)
    if S <= E:  # few rows: each takes its own expert's weights
        W = _dequantized(s["codes"][of_row], s["scales"][of_row], s["book"], K, group)
        return (W * x[token][:, None, :]).sum(2).to(s["x"].dtype)
    # rows of each expert padded to the most that one has
    begin = offsets[:-1].to(torch.int64)
    most = int((offsets[1:] - offsets[:-1]).max())
    within = torch.arange(S, device=x.device) - begin[of_row]
    padded = x.new_zeros((E, K, most))
    padded[of_row, :, within] = x[token]
    W = _dequantized(s["codes"], s["scales"], s["book"], K, group)
    return torch.matmul(W, padded)[of_row, :, within].to(s["x"].dtype)


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


# ---- what the cases cannot do without, and the definitions in 64 bits -----------------------------

def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    op, T = case["op"], case["rows"]
    if op == "route":
        E, k, train = case["experts"], case["top_k"], case["train"]
        # the gradient over all experts needs the scores, over the chosen ones only what was given out
        moved = T * E * size + T * k * 8
        if train:
            moved += T * E * size + T * k * 4
        return {"bytes": float(moved), "flops": float(T * E * (4 if case["over_all"] else 2) * (2 if train else 1))}
    S = T * case.get("top_k", 1)
    if op == "dispatch":
        d = case["cols"]
        moved = 4 * S + 8 * S + 4 * (case["experts"] + 1) + (T + S) * d * size
        return {"bytes": float(moved + ((T + S) * d * size if case["train"] else 0)),
                "flops": float(S * d if case["train"] else 0)}
    if op == "combine":
        d = case["cols"]
        moved = 4 * S + 4 * S + (T + S) * d * size
        if case["train"]:
            moved += (T + S) * d * size + 4 * S
        return {"bytes": float(moved), "flops": float(2 * S * d * (3 if case["train"] else 1))}
    N, K = case["out"], case["cols"]
    matrix = N * (K / 2 + -(-K // case["group"]) * size)
    if op == "product":
        return {"bytes": float(matrix + T * (K + N) * size), "flops": 2.0 * T * N * K}
    E = case["experts"]
    read = min(S, E * (1 - (1 - case["top_k"] / E) ** T))  # experts that some row has, about
    return {"bytes": float(read * matrix + (T * K + S * N) * size + 4 * S), "flops": 2.0 * S * N * K}


def exact(case, seed):
    s = prepare(case, seed)
    op, T = case["op"], case["rows"]
    for name in ("scores", "x", "rows", "weights"):
        if name in s:
            s[name] = s[name].detach()
    if op == "route":
        k, E = case["top_k"], case["experts"]
        factor = -0.25 if case["distances"] else 1.0
        weights = torch.empty((T, k), dtype=torch.float64, device="cuda")
        grads = torch.empty((T, E), dtype=torch.float64, device="cuda") if case["train"] else None
        step = max(1, 50_000_000 // E)
        for lo in range(0, T, step):
            z = s["scores"][lo:lo + step].double() * factor
            index = torch.argsort(z, dim=1, descending=True, stable=True)[:, :k]
            chosen = torch.zeros_like(z).scatter_(1, index, 1.0)
            p = torch.softmax(z if case["over_all"] else z.masked_fill(chosen == 0, -math.inf), dim=1)
            weights[lo:lo + step] = p.gather(1, index)
            if case["train"]:
                g = torch.zeros_like(z).scatter_(1, index, s["grad"][lo:lo + step].double())
                grads[lo:lo + step] = factor * p * (g - (p * g).sum(1, keepdim=True))
        out = dict(experts=None, weights=weights)
        if case["train"]:
            out["dscores"] = grads
        return out
    if op == "product":
        out = torch.empty((T, case["out"]), dtype=torch.float64, device="cuda")
        _exact_rows(out, s["x"].double(), s["codes"], s["scales"], s["book"], case)
        return out
    # the order by hand: experts in turn, their slots in turn, then the slots that have none
    flat = s["experts"].reshape(-1)
    slots = [torch.nonzero(flat == e).reshape(-1) for e in range(case["experts"])]
    slots.append(torch.nonzero(flat < 0).reshape(-1))
    order = torch.cat(slots)
    S, k, held = order.numel(), case["top_k"], order.numel() - slots[-1].numel()
    if op == "experts":
        out = torch.zeros((S, case["out"]), dtype=torch.float64, device="cuda")
        at = 0
        for e in range(case["experts"]):
            rows = slots[e].numel()
            if rows:
                _exact_rows(out[at:at + rows], s["x"][slots[e] // k].double(), s["codes"][e], s["scales"][e],
                            s["book"], case)
            at += rows
        return out
    if S * case["cols"] > 400_000_000:
        return None
    token, d = order // k, case["cols"]
    if op == "dispatch":
        rows = torch.zeros((S, d), dtype=torch.float64, device="cuda")
        rows[:held] = s["x"][token[:held]].double()
        out = dict(order=None, position=None, offsets=None, rows=rows)
        if case["train"]:
            out["dx"] = torch.zeros((T, d), dtype=torch.float64, device="cuda").index_add_(
                0, token[:held], s["grad"][:held].double())
        return out
    weight = s["weights"].reshape(-1)[order].double()
    out = dict(out=torch.zeros((T, d), dtype=torch.float64, device="cuda").index_add_(
        0, token[:held], s["rows"][:held].double() * weight[:held, None]))
    if case["train"]:
        g = s["grad"].double()[token[:held]]
        out["drows"] = torch.zeros((S, d), dtype=torch.float64, device="cuda")
        out["drows"][:held] = g * weight[:held, None]
        dw = torch.zeros(S, dtype=torch.float64, device="cuda")
        dw[order[:held]] = (g * s["rows"][:held].double()).sum(1)
        out["dweights"] = dw.reshape(T, k)
    return out


def _exact_rows(out, x, codes, scales, book, case):
    """out = x times the transpose of the matrix, a group at a time: sum of the group times its scale."""
    K, group = case["cols"], case["group"]
    out.zero_()
    values = book.double()
    for g in range(scales.shape[-1]):
        lo, hi = g * group, min(K, (g + 1) * group)
        part = codes[:, lo // 2:(hi + 1) // 2].to(torch.int64)
        w = torch.stack([values[part & 15], values[part >> 4]], 2).reshape(part.shape[0], -1)[:, :hi - lo]
        out += (x[:, lo:hi] @ w.t()) * scales[:, g].double()
