"""Products grouped by expert and products in microscaled 4-bit numbers as cases that can be timed and compared.

A case is a dict of plain values; prepare() makes what a user's program holds before the call, run()
is one pass through an operator: with `own` through the framework's entry points, without it in a
plain form of elementary torch operations in 32 bits, rounded once at the end. exact() is the
operator's definition in 64 bits. Sizes are generic.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # ---- the experts' own products, between dispatch and combine
        # A batch of a serving loop through two of 8 experts: few rows each, the matrices are what is read.
        dict(name="experts_serve_16_e8", op="experts", tokens=16, top_k=2, experts=8, out=4096, cols=4096,
             dtype="bfloat16", dropped=0.0, train=False),
        # A prompt of odd length through two of 8 large experts, some slots without one.
        dict(name="experts_prompt_4099_e8", op="experts", tokens=4099, top_k=2, experts=8, out=11_000, cols=4096,
             dtype="float16", dropped=0.02, train=False),
        # A training step: 16k tokens, four of 64 experts, the gradients of rows and matrices.
        dict(name="experts_train_16k_e64", op="experts", tokens=16_384, top_k=4, experts=64, out=2048, cols=2048,
             dtype="bfloat16", dropped=0.0, train=True),
        # A small model per cluster, odd sizes on every axis, trained in float32.
        dict(name="experts_train_100k_d101", op="experts", tokens=100_003, top_k=3, experts=1000, out=77, cols=101,
             dtype="float32", dropped=0.03, train=True),
        # ---- numbers into 4 bits (and back, which is what they stand for)
        # A serving batch's activations before a layer.
        dict(name="quantize_64x4096", op="quantize", rows=64, cols=4096, dtype="bfloat16"),
        # A weight matrix of odd sizes when a model is compressed.
        dict(name="quantize_11003x8190", op="quantize", rows=11_003, cols=8190, dtype="float16"),
        # ---- a layer in 4 bits: activations are quantized in the call, the matrix was before
        # One new token.
        dict(name="product_1x4096x4096", op="product", rows=1, out=4096, cols=4096, dtype="bfloat16"),
        # A serving batch, odd sizes.
        dict(name="product_33x11003x8190", op="product", rows=33, out=11_003, cols=8190, dtype="float16"),
        # A long prompt: the matrix instructions' rate.
        dict(name="product_8192x8192x8192", op="product", rows=8192, out=8192, cols=8192, dtype="bfloat16"),
        # ---- a layer of experts in 4 bits
        # One new token through two of 16.
        dict(name="experts4_1_e16", op="experts4", tokens=1, top_k=2, experts=16, out=4096, cols=2048,
             dtype="bfloat16", dropped=0.0),
        # A serving batch through four of 64, some with many tokens and some with none.
        dict(name="experts4_64_e64", op="experts4", tokens=64, top_k=4, experts=64, out=2048, cols=4096,
             dtype="bfloat16", dropped=0.0),
        # A prompt's tokens through four of 64.
        dict(name="experts4_16k_e64", op="experts4", tokens=16_384, top_k=4, experts=64, out=4096, cols=2048,
             dtype="bfloat16", dropped=0.01),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size between lo and hi; half of them are multiples of 64, as layers' sizes mostly are."""
    n = _log_int(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    """One more case of the listed ones' ranges, no dearer than the dearest of them."""
    op = rng.choice(["experts", "experts", "experts", "quantize", "product", "product", "experts4"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "quantize":
        cols = _size(rng, 16, 16_384)
        return dict(op=op, rows=min(_log_int(rng, 1, 100_000), 90_000_000 // cols), cols=cols, dtype=dtype)
    if op == "product":
        out, cols = _size(rng, 64, 11_000), _size(rng, 64, 8192)
        rows = min(_log_int(rng, 1, 8192), 500_000_000_000 // (out * cols))
        return dict(op=op, rows=rows, out=out, cols=cols, dtype=dtype)
    out, cols = _size(rng, 64, 8192), _size(rng, 64, 8192)
    experts, top_k = _log_int(rng, 2, 1000), rng.randint(1, 4)
    experts = max(2, min(experts, 360_000_000 // (out * cols)))
    train = op == "experts" and rng.random() < 0.6
    # float32 products run at a twentieth of the 16-bit rate
    flops = 5e11 / (3 if train else 1) / (8 if dtype == "float32" and op == "experts" else 1)
    top_k = min(top_k, experts)
    slots = int(min(flops / (2 * out * cols), 200_000_000 // (out + cols)))
    tokens = max(1, min(_log_int(rng, 1, 100_000), slots // top_k))
    case = dict(op=op, tokens=tokens, top_k=top_k, experts=experts, out=out, cols=cols, dtype=dtype,
                dropped=rng.choice([0.0, 0.0, 0.05]))
    if op == "experts":
        case["train"] = train
    return case


# ---- inputs --------------------------------------------------------------------------------------

def _choices(case, gen):
    """(tokens, top_k) distinct experts a token, some of them more popular than others; `dropped` of the
    slots have none."""
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    liking = torch.rand((T, E), device="cuda", generator=gen) + 0.3 * torch.rand((1, E), device="cuda", generator=gen)
    chosen = torch.topk(liking, k, dim=1).indices.to(torch.int32)
    if case["dropped"] > 0:
        chosen[torch.rand((T, k), device="cuda", generator=gen) < case["dropped"]] = -1
    return chosen.contiguous()


def _plan(chosen, E):
    """The rows in expert order: the slot of each, its expert (E behind the last) and its place among the
    expert's rows, and the most rows that one expert has. A training step and a serving loop make this once
    for all products of a layer."""
    flat = chosen.reshape(-1).to(torch.int64)
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    of_row, slot = torch.sort(key, stable=True)
    counts = torch.bincount(of_row, minlength=E + 1)
    begin = torch.cumsum(counts, 0) - counts
    within = torch.arange(of_row.numel(), device=flat.device) - begin[of_row]
    return dict(slot=slot, of_row=of_row, within=within, most=max(1, int(counts[:E].max())), counts=counts[:E])


_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantized(x):
    """Codes (two to a byte, the even column in the low half) and scales' bytes (exponent + 127) of the rows
    of x, float32: blocks of 32 columns, the last one filled up with zeros."""
    K = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -K % 32))
    blocks = x.reshape(x.shape[:-1] + (-1, 32))
    most = blocks.abs().amax(-1, keepdim=True)
    # floor(log2) is the exponent that frexp gives, less one; 6 = 1.5 * 2^2 is the largest element
    scale = torch.clamp(torch.frexp(most).exponent - 3, -127, 127).to(torch.int32)
    scale = torch.where(most == 0, -127, scale)
    # (2^-scale as a number: its bits)
    scaled = blocks * ((127 - scale) << 23).view(torch.float32) if K else blocks
    m = scaled.abs()
    # the middles between two levels; where it is a tie, the level whose last bit is 0
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
    code = (code + 8 * torch.signbit(blocks)).to(torch.uint8).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), (scale.squeeze(-1) + 127).to(torch.uint8)


def _values(codes, scales, cols):
    """What codes and scales stand for, in float32."""
    levels = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), device=codes.device)
    pairs = torch.stack([levels[torch.arange(256, device=codes.device) & 15],
                         levels[torch.arange(256, device=codes.device) >> 4]], 1)
    values = pairs[codes.to(torch.int32)].flatten(-2)
    power = (scales.to(torch.int32) << 23).view(torch.float32)  # (no block here is as small as 2^-127)
    return (values.reshape(scales.shape + (32,)) * power[..., None]).reshape(values.shape)[..., :cols]


def _matrices(lead, out, cols, gen):
    """Codes and scales of normal matrices, one after another."""
    codes = torch.empty(lead + (out, -(-cols // 32) * 16), dtype=torch.uint8, device="cuda")
    scales = torch.empty(lead + (out, -(-cols // 32)), dtype=torch.uint8, device="cuda")
    flat, flat_scales = codes.reshape(-1, codes.shape[-1]), scales.reshape(-1, scales.shape[-1])
    step = max(1, 32_000_000 // cols)
    for lo in range(0, flat.shape[0], step):
        n = min(step, flat.shape[0] - lo)
        w = torch.randn((n, cols), device="cuda", generator=gen) / math.sqrt(cols)
        flat[lo:lo + n], flat_scales[lo:lo + n] = _quantized(w)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3000 + int(seed))
    dt, op, cols = TYPES[case["dtype"]], case["op"], case["cols"]

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen, dtype=dt)

    s = dict(case=case)
    if op == "quantize":
        # rows of different sizes, as activations and weights have them
        s["x"] = (randn(case["rows"], cols) * torch.exp(randn(case["rows"], 1).float()).to(dt))
        return s
    if op == "product":
        s["x"] = randn(case["rows"], cols)
        s["codes"], s["scales"] = _matrices((), case["out"], cols, gen)
        return s
    E, out = case["experts"], case["out"]
    s["chosen"] = _choices(case, gen)
    s["plan"] = _plan(s["chosen"], E)
    if op == "experts4":
        s["x"] = randn(case["tokens"], cols)
        s["codes"], s["scales"] = _matrices((E,), out, cols, gen)
        return s
    s["rows"] = randn(case["tokens"] * case["top_k"], cols)
    s["weights"] = torch.empty((E, out, cols), dtype=dt, device="cuda")
    for e in range(E):
        s["weights"][e] = randn(out, cols) / math.sqrt(cols)
    if case["train"]:
        s["grad"] = randn(s["rows"].shape[0], out)
        s["rows"].requires_grad_()
        s["weights"].requires_grad_()
    return s


# ---- the framework's operators ---------------------------------------------------------------------

def _run_own(s):
    case, op = s["case"], s["case"]["op"]
    if op == "experts":
        from h2o4gpu_amd import experts
        if "order" not in s:  # made once for a layer's dispatch, products and combination
            s["order"] = experts.sort_by_expert(s["chosen"], case["experts"])
        y = experts.product(s["rows"], s["weights"], s["order"])
        if not case["train"]:
            return y
        drows, dweights = torch.autograd.grad(y, (s["rows"], s["weights"]), s["grad"])
        return dict(y=y, drows=drows, dweights=dweights)
    from h2o4gpu_amd import microscale4
    x = microscale4.quantize(s["x"])
    if op == "quantize":
        return x.dequantize(s["x"].dtype)
    if "laid_out" not in s:  # weights are laid out once, as a program that serves them does
        s["laid_out"] = microscale4.Microscale4(s["codes"], s["scales"], case["cols"])
    if op == "product":
        return microscale4.product(x, s["laid_out"])
    if "order" not in s:
        from h2o4gpu_amd import experts
        s["order"] = experts.sort_by_expert(s["chosen"], case["experts"])
    return microscale4.experts_product(x, s["laid_out"], s["order"])


# ---- plain forms -------------------------------------------------------------------------------------

def _padded(rows, plan, E):
    """(E, most, cols): every expert's rows, filled up with zeros."""
    out = rows.new_zeros((E + 1, plan["most"], rows.shape[1]))
    kept = plan["of_row"] < E
    within = torch.where(kept, plan["within"], 0)
    out[plan["of_row"], within] = torch.where(kept[:, None], rows, 0)
    return out[:E]


def _unpadded(batch, plan, E):
    kept = plan["of_row"] < E
    rows = batch[torch.where(kept, plan["of_row"], 0), torch.where(kept, plan["within"], 0)]
    return torch.where(kept[:, None], rows, 0)


def _run_plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "experts":
        E, dt = case["experts"], s["rows"].dtype
        x, W = _padded(s["rows"].float(), s["plan"], E), s["weights"].float()
        y = _unpadded(torch.matmul(x, W.transpose(1, 2).contiguous()), s["plan"], E).to(dt)
        if not case["train"]:
            return y
        g = _padded(s["grad"].float(), s["plan"], E)
        drows = _unpadded(torch.matmul(g, W), s["plan"], E).to(dt)
        return dict(y=y, drows=drows, dweights=torch.matmul(g.transpose(1, 2).contiguous(), x).to(dt))
    cols = case["cols"]
    x = _values(*_quantized(s["x"].float()), cols)
    if op == "quantize":
        return x.to(s["x"].dtype)
    if op == "product":
        return torch.matmul(x, _values(s["codes"], s["scales"], cols).t()).to(s["x"].dtype)
    plan, E, k = s["plan"], case["experts"], case["top_k"]
    rows = x[plan["slot"] // k]
    if rows.shape[0] <= E:  # few rows: each takes its own expert's matrix
        e = plan["of_row"].clamp_max(E - 1)
        y = (_values(s["codes"][e], s["scales"][e], cols) * rows[:, None, :]).sum(2)
        return torch.where((plan["of_row"] < E)[:, None], y, 0).to(s["x"].dtype)
    W = _values(s["codes"], s["scales"], cols)
    return _unpadded(torch.matmul(_padded(rows, plan, E), W.transpose(1, 2).contiguous()), plan, E).to(s["x"].dtype)


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


# ---- what the cases cannot do without, and the definitions in 64 bits ----------------------------------

def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    op, K = case["op"], case["cols"]
    four = 17 / 32  # bytes of a number in 4 bits and its share of a scale
    if op == "quantize":
        return {"bytes": case["rows"] * K * (2 * size + four), "flops": float(2 * case["rows"] * K)}
    N = case["out"]
    if op == "product":
        return {"bytes": N * K * four + case["rows"] * (K + N) * size, "flops": 2.0 * case["rows"] * N * K}
    T, k, E = case["tokens"], case["top_k"], case["experts"]
    S = T * k
    kept = S * (1 - case["dropped"])
    used = min(S, E * (1 - (1 - k / E) ** T))  # experts that some row has, about
    if op == "experts4":
        return {"bytes": used * N * K * four + (T * K + S * N) * size + 4.0 * S, "flops": 2.0 * kept * N * K}
    moved = (used * N * K + S * (K + N)) * size
    if case["train"]:
        moved += (E * N * K + S * (K + N)) * size
    return {"bytes": float(moved), "flops": 2.0 * kept * N * K * (3 if case["train"] else 1)}


def _exact_values(x):
    """The nearest numbers of a block's grid by trying them all, in 64 bits."""
    K = x.shape[-1]
    x = torch.nn.functional.pad(x.double(), (0, -K % 32))
    blocks = x.reshape(x.shape[0], -1, 32)
    most = blocks.abs().amax(2, keepdim=True)
    step = torch.floor(torch.log2(torch.where(most > 0, most, 1.0))) - 2
    # log2 of a number next to a power of two may round to it: the definition is 2^e <= most < 2^(e + 1)
    step = step - (torch.exp2(step + 2) > most).double() + (torch.exp2(step + 3) <= most).double()
    power = torch.where(most > 0, torch.exp2(step), 1.0)
    scaled = blocks / power
    best, off = torch.zeros_like(scaled), scaled.abs()
    for level in (1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0):  # of two as near, the one whose last bit is 0: it comes first
        far = (scaled.abs() - level).abs()
        nearer = far < off
        best, off = torch.where(nearer, level, best), torch.where(nearer, far, off)
    return (torch.copysign(best, scaled) * power).reshape(x.shape)[:, :K]


def _exact_matrix(codes, scales, cols):
    low, high = (codes & 15).long(), (codes >> 4).long()
    code = torch.stack([low, high], -1).reshape(codes.shape[0], -1)
    levels = torch.tensor(_LEVELS, dtype=torch.float64, device=codes.device)
    value = levels[code & 7] * (1 - 2 * (code >> 3)).double()
    return (value * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1))[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_values(s["x"])
    if op == "product":
        return _exact_values(s["x"]) @ _exact_matrix(s["codes"], s["scales"], case["cols"]).t().contiguous()
    E, N, k = case["experts"], case["out"], case["top_k"]
    flat = s["chosen"].reshape(-1)
    S, at = flat.numel(), 0
    out = torch.zeros((S, N), dtype=torch.float64, device="cuda")
    x = _exact_values(s["x"]) if op == "experts4" else None
    train = case.get("train", False)
    if train:
        drows = torch.zeros((S, case["cols"]), dtype=torch.float64, device="cuda")
        dweights = torch.zeros((E, N, case["cols"]), dtype=torch.float64, device="cuda")
    for e in range(E):
        slots = torch.nonzero(flat == e).reshape(-1)
        lo, at = at, at + slots.numel()
        if at == lo:
            continue
        if op == "experts4":
            out[lo:at] = x[slots // k] @ _exact_matrix(s["codes"][e], s["scales"][e], case["cols"]).t().contiguous()
            continue
        rows, W = s["rows"].detach()[lo:at].double(), s["weights"].detach()[e].double()
        out[lo:at] = rows @ W.t().contiguous()
        if train:
            g = s["grad"][lo:at].double()
            drows[lo:at] = g @ W
            dweights[e] = g.t().contiguous() @ rows
    return dict(y=out, drows=drows, dweights=dweights) if train else out
