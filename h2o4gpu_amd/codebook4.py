"""4-bit matrices whose 16 values are a codebook (as k-means finds it) and whose groups of columns
have a scale each, and their products with tokens.

    from h2o4gpu_amd import codebook4
    packed = codebook4.quantize(W, group=128)      # W (out, cols): the codebook comes from KMeans
    y = codebook4.product(x, packed)               # x (tokens, cols) -> (tokens, out)

Element (n, k) of such a matrix is codebook[code(n, k)] * scales[n, k // group]. A matrix per expert
(a leading axis) is multiplied with the rows that an ExpertOrder gives each expert:

    rows = codebook4.experts_product(x, packed, order)
    y = experts.combine(rows, weights, order)

The products are for serving and have no gradient. Streams and graphs as in h2o4gpu_amd.experts.
"""
import numpy as np
import torch

from .experts import _TYPES, _call, _no_tangents, _order_of, _rows, _tensor, _type_of
from .libs import experts_hip


def _group_of(group):
    group = int(group)
    if group < 32 or group % 32 or group > experts_hip.MAX_GROUP:
        raise ValueError("group must be a multiple of 32, at most %d, got %d" % (experts_hip.MAX_GROUP, group))
    return group


class Codebook4:
    """A 4-bit matrix (out, cols), or one per expert (experts, out, cols).

    codes: uint8 (..., out, bytes), two columns a byte, the even one in the low half; bytes is at least
    cols / 2 rounded up. scales: (..., out, ceil(cols / group)), float32, bfloat16 or float16; group is a
    multiple of 32 (longer than a row: one scale a row). codebook: (16,) or (experts, 16) finite values in
    the type of the tokens.

    Codes and scales are copied once into the order that the products read them in (`laid_codes`,
    `laid_scales`); those passed in are not needed afterwards. `dtype` is that of the tokens.
    """

    __slots__ = ("laid_codes", "laid_scales", "codebook", "cols", "group", "out", "n_experts", "dtype",
                 "device", "_args")

    def __init__(self, codes, scales, codebook, cols, group):
        lead = codes.dim() - 2 if isinstance(codes, torch.Tensor) else 0
        if lead not in (0, 1):
            raise ValueError("codes must be (out, bytes) or (experts, out, bytes), got %s" % (tuple(codes.shape),))
        _tensor("codes", codes, 2 + lead, dtype=torch.uint8)
        _tensor("scales", scales, 2 + lead, codes.device)
        _type_of("scales", scales)
        _tensor("codebook", codebook, codebook.dim() if isinstance(codebook, torch.Tensor) else 1, codes.device)
        _type_of("codebook", codebook)
        cols, group = int(cols), _group_of(group)
        if cols < 1 or codes.shape[-1] < (cols + 1) // 2:
            raise ValueError("%d bytes a row do not hold %d columns" % (codes.shape[-1], cols))
        if codes.shape[-2] < 1 or (lead and not 1 <= codes.shape[0] <= experts_hip.MAX_EXPERTS):
            raise ValueError("codes must have rows (and 1 to %d experts), got %s" % (experts_hip.MAX_EXPERTS,
                                                                                     tuple(codes.shape)))
        groups = -(-cols // group)
        if tuple(scales.shape) != tuple(codes.shape[:-1]) + (groups,):
            raise ValueError("scales must be %s, got %s" % (tuple(codes.shape[:-1]) + (groups,),
                                                            tuple(scales.shape)))
        if tuple(codebook.shape) != (16,) and not (lead and tuple(codebook.shape) == (codes.shape[0], 16)):
            raise ValueError("codebook must have 16 values%s, got shape %s" % (
                " (or 16 for each expert)" if lead else "", tuple(codebook.shape)))
        codes, scales, device = codes.contiguous(), scales.contiguous(), codes.device.index
        self.codebook, self.cols, self.group, self.out = codebook.contiguous(), cols, group, codes.shape[-2]
        self.n_experts = codes.shape[0] if lead else 0
        self.dtype, self.device = codebook.dtype, codes.device
        count, lib = max(1, self.n_experts), experts_hip.lib()
        kind = _TYPES[scales.dtype]
        nbytes = lib.h2o4gpu_codebook4_codes_bytes(count, self.out, cols)
        if nbytes == 0:
            raise ValueError("a matrix of %d x %d is beyond what the products take" % (self.out, cols))
        self.laid_codes = codes.new_empty(nbytes)
        nbytes = lib.h2o4gpu_codebook4_scales_bytes(count, self.out, cols, group, kind)
        self.laid_scales = scales.new_empty(nbytes // scales.element_size())
        _call(device, "h2o4gpu_codebook4_layout", count, self.out, cols, group, codes.data_ptr(), codes.shape[-1],
              kind, scales.data_ptr(), self.laid_codes.data_ptr(), self.laid_scales.data_ptr())
        self._args = (self.laid_codes.data_ptr(), kind, self.laid_scales.data_ptr(), self.codebook.data_ptr())

    def codes(self):
        """The codes, one a byte: uint8 (..., out, cols)."""
        count, tiles, subs = max(1, self.n_experts), -(-self.out // 16), -(-self.cols // 128)
        # (tile, 128 columns, q, row, 32 columns, bytes of 8) -> (tile, row, 128 columns, 32 columns, q, bytes)
        raw = self.laid_codes.view(count, tiles, subs, 4, 16, 4, 4).permute(0, 1, 4, 2, 5, 3, 6)
        raw = raw.reshape(count, tiles * 16, subs * 64)[:, :self.out]
        codes = torch.stack([raw & 15, raw >> 4], -1).flatten(-2)[..., :self.cols]
        return codes if self.n_experts else codes[0]

    def scales(self):
        """The scales, (..., out, ceil(cols / group))."""
        count, tiles, subs = max(1, self.n_experts), -(-self.out // 16), -(-self.cols // 128)
        per = 1 if self.group % 128 == 0 else 2 if self.group % 64 == 0 else 4
        laid = self.laid_scales.view(count, tiles, subs, 16, per).permute(0, 1, 3, 2, 4)
        laid = laid.reshape(count, tiles * 16, subs * per)[:, :self.out]
        laid = laid[..., ::self.group * per // 128].contiguous()[..., :-(-self.cols // self.group)]
        return laid if self.n_experts else laid[0]

    def dequantize(self):
        """The matrix as a float32 tensor (for checks and for training on)."""
        table, codes = self.codebook.float(), self.codes().to(torch.int64)
        if table.dim() == 2:
            values = table[torch.arange(self.n_experts, device=codes.device)[:, None, None], codes]
        else:
            values = table[codes]
        return values * self.scales().float()[..., torch.arange(self.cols, device=codes.device) // self.group]


def _spread(n, m, device=None):
    """m ascending places of n (m <= n), one in each of m equal stretches. Where in its stretch a place lies goes
    by multiples of the golden ratio, so that every column of a matrix is met as often as any other. (A stretch is
    n / m long, no whole number: below 1.6, an end and a start that share a place may both name it.)"""
    i = torch.arange(m, dtype=torch.float64, device=device)
    return ((i + (i * 0.6180339887498949).frac()) * (n / m)).long().clamp_(max=n - 1)


def fit_codebook(values, sample=1 << 20, seed=0):
    """The 16 centroids k-means finds for `values` (a GPU tensor, any shape; of more than `sample`, that many
    spread over all of them), ascending, float32."""
    from .solvers.kmeans import KMeans
    flat = values.reshape(-1)
    if flat.numel() > sample:
        flat = flat[_spread(flat.numel(), sample, flat.device)]
    flat = flat.float()
    flat = flat[torch.isfinite(flat)]
    if flat.numel() < 16:
        raise ValueError("a codebook needs at least 16 finite values, got %d" % flat.numel())
    at = torch.linspace(0.5 / 16, 1 - 0.5 / 16, 16, device=flat.device)
    start = torch.sort(flat).values[(at * (flat.numel() - 1)).long()]
    model = KMeans(n_clusters=16, init=start.cpu().numpy()[:, None], max_iter=100, tol=1e-9, random_state=seed)
    model.fit(flat[:, None].contiguous())
    return torch.from_numpy(np.sort(model.cluster_centers_.reshape(-1))).float().to(flat.device)


def quantize(weights, group=128, codebook=None, top=1.0, scale_dtype=None):
    """Codebook4 of `weights`, (out, cols) or (experts, out, cols).

    A group's scale is its largest magnitude over `top`, and every element gets the code of the entry
    nearest to element / scale. codebook: 16 values (top: the one that a group's largest magnitude
    stands for, e.g. 7 for the integers -8 .. 7); None fits it to the scaled elements with k-means.
    It is rounded to the weights' type before the codes are chosen. scale_dtype defaults to that type; a
    scale that is 0 or no finite number of it (a float32 matrix beyond float16's 65504, say) becomes 1,
    and what is larger than the codebook's largest value then is that value. NaN and infinities get code 0.
    """
    _tensor("weights", weights, weights.dim() if isinstance(weights, torch.Tensor) and weights.dim() == 3 else 2)
    code = _type_of("weights", weights)
    group, top = _group_of(group), float(top)
    if min(weights.shape) < 1:
        raise ValueError("weights are empty: %s" % (tuple(weights.shape),))
    if not 0.0 < top <= 3.4e38:
        raise ValueError("top must be positive and finite, got %r" % top)
    cols = weights.shape[-1]
    flat = weights.detach().reshape(-1, cols)
    if flat.stride(1) != 1 or (flat.shape[0] > 1 and flat.stride(0) < cols):
        flat = flat.contiguous()
    groups, pitch = -(-cols // group), -(-cols // 2)
    if codebook is None:
        if top != 1.0:
            raise ValueError("top goes with a given codebook; one that is fitted has 1")
        part = flat if flat.shape[0] <= 4096 else flat[_spread(flat.shape[0], 4096, flat.device)]
        part = part.float()
        width = min(group, cols)  # (a longer group is a row)
        padded = torch.nn.functional.pad(part, (0, groups * width - cols)).reshape(part.shape[0], groups, width)
        scaled = padded / padded.abs().amax(2, keepdim=True).clamp_min(1e-38)
        codebook = fit_codebook(scaled.reshape(part.shape[0], -1)[:, :cols])
    _tensor("codebook", codebook, 1, weights.device)
    if codebook.shape[0] != 16:
        raise ValueError("codebook must have 16 values, got %d" % codebook.shape[0])
    codebook = codebook.to(weights.dtype).contiguous()
    codes = torch.empty((flat.shape[0], pitch), dtype=torch.uint8, device=flat.device)
    scales = torch.empty((flat.shape[0], groups), dtype=scale_dtype or weights.dtype, device=flat.device)
    ptr, stride = _rows("weights", flat)
    _call(flat.device.index, "h2o4gpu_codebook4_quantize", code, flat.shape[0], cols, group, top, ptr, stride,
          codebook.data_ptr(), codes.data_ptr(), pitch, _type_of("scales", scales), scales.data_ptr())
    lead = tuple(weights.shape[:-1])
    return Codebook4(codes.reshape(lead + (pitch,)), scales.reshape(lead + (groups,)), codebook, cols, group)


def _tokens(x, weights):
    if not isinstance(weights, Codebook4):
        raise TypeError("weights must be a Codebook4, got %s" % type(weights).__name__)
    if not (isinstance(x, torch.Tensor) and x.dim() == 2 and x.dtype == weights.dtype and x.device == weights.device):
        _tensor("x", x, 2, weights.device, weights.dtype)
    if x.shape[1] != weights.cols:
        raise ValueError("x must be (tokens, %d), got %s" % (weights.cols, tuple(x.shape)))
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("products with 4-bit matrices have no gradient: detach x, or multiply with dequantize()")
    _no_tangents(x)
    return _rows("x", x)


def product(x, weights):
    """(tokens, out) = x (tokens, cols) times the transpose of a Codebook4 matrix; products and sums in
    float32, rounded once to the type of x."""
    ptr, stride = _tokens(x, weights)
    if weights.n_experts:
        raise ValueError("weights hold a matrix per expert: experts_product multiplies with those")
    rows, out = x.shape[0], weights.out
    y = x.new_empty((rows, out))
    _call(x.device.index, "h2o4gpu_codebook4_product", _TYPES[x.dtype], rows, out, weights.cols, weights.group, ptr,
          stride, *weights._args, y.data_ptr(), out)
    return y


def experts_product(x, weights, order):
    """(tokens * top_k, out), rows in expert order: the token of every slot of `order` times the
    transpose of its expert's matrix; zeros behind order.offsets[-1]. Only the matrices of experts that
    have a token are read."""
    ptr, stride = _tokens(x, weights)
    _order_of(order, x.device)
    if not weights.n_experts or weights.n_experts != order.n_experts:
        raise ValueError("order has %d experts, weights %d" % (order.n_experts, weights.n_experts))
    if x.shape[0] != order.tokens:
        raise ValueError("x must be (%d, %d), got %s" % (order.tokens, weights.cols, tuple(x.shape)))
    y = x.new_empty((order.tokens * order.top_k, weights.out))
    _call(x.device.index, "h2o4gpu_codebook4_experts_product", _TYPES[x.dtype], order.tokens, order.top_k,
          weights.n_experts, weights.out, weights.cols, weights.group, ptr, stride, *weights._args,
          16 if weights.codebook.dim() == 2 else 0, order._order_ptr, order._offsets_ptr, y.data_ptr(),
          weights.out)
    return y
