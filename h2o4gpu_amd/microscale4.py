"""Microscaled 4-bit matrices, and products in which both operands are such: the serving form of the
expert layers and of single matrices, on the 4-bit matrix instructions.

    from h2o4gpu_amd import microscale4
    packed = microscale4.quantize(W)               # W (out, cols), once
    y = microscale4.product(microscale4.quantize(x), packed)      # x (tokens, cols) -> (tokens, out)

Every 32 columns of a row share a power of two; an element is a sign and one of 0, 0.5, 1, 1.5, 2, 3,
4, 6 times it. A matrix per expert (a leading axis) is multiplied with the rows that an ExpertOrder
gives each expert:

    rows = microscale4.experts_product(microscale4.quantize(x), packed, order)
    y = experts.combine(rows, weights, order)

Nothing here has a gradient: train with experts.product, then quantize. Streams and graphs as in
h2o4gpu_amd.experts. (h2o4gpu_amd.codebook4 keeps the tokens in 16 or 32 bits and takes any 16 values.)
"""
import functools

import torch

from .experts import _TYPES, _call, _no_tangents, _order_of, _rows, _tensor, _type_of
from .libs import experts_hip

BLOCK = 32


@functools.lru_cache(maxsize=256)
def _pitches(cols):
    """Bytes of a row of codes and of a row of scales."""
    lib = experts_hip.lib()
    pitch = lib.h2o4gpu_microscale4_codes_pitch(max(0, cols))
    if pitch == 0:
        raise ValueError("a matrix must have 1 to 2^30 columns, got %d" % cols)
    return pitch, lib.h2o4gpu_microscale4_scales_pitch(cols)


class Microscale4:
    """A matrix (rows, cols) in microscaled 4-bit numbers, or one per expert (experts, rows, cols).

    codes: uint8 (..., rows, bytes), two columns a byte, the even one in the low half; bytes is at least
    cols / 2 rounded up. A code is a sign (8) and the number of one of 0, 0.5, 1, 1.5, 2, 3, 4, 6. scales:
    uint8 (..., rows, ceil(cols / 32)): the power of two plus 127; 255 makes the block not a number.

    Both are copied once into the order that the products read them in; those passed in are not needed
    afterwards. `dtype` is the type of a product whose tokens this matrix is.
    """

    __slots__ = ("rows", "cols", "n_experts", "dtype", "device", "_buffer", "_codes_ptr", "_scales_ptr")

    def __init__(self, codes, scales, cols, dtype=torch.bfloat16):
        lead = codes.dim() - 2 if isinstance(codes, torch.Tensor) else 0
        if lead not in (0, 1):
            raise ValueError("codes must be (rows, bytes) or (experts, rows, bytes), got %s" % (tuple(codes.shape),))
        _tensor("codes", codes, 2 + lead, dtype=torch.uint8)
        _tensor("scales", scales, 2 + lead, codes.device, torch.uint8)
        cols = int(cols)
        if cols < 1 or codes.shape[-1] < (cols + 1) // 2:
            raise ValueError("%d bytes a row do not hold %d columns" % (codes.shape[-1], cols))
        if tuple(scales.shape) != tuple(codes.shape[:-1]) + (-(-cols // BLOCK),):
            raise ValueError("scales must be %s, got %s" % (tuple(codes.shape[:-1]) + (-(-cols // BLOCK),),
                                                            tuple(scales.shape)))
        if dtype not in _TYPES:
            raise TypeError("dtype must be float32, bfloat16 or float16, got %s" % (dtype,))
        self._allocate(codes, codes.shape[:-1], cols, dtype)
        codes, scales = codes.contiguous(), scales.contiguous()
        _call(codes.device.index, "h2o4gpu_microscale4_layout", self.rows * max(1, self.n_experts), cols,
              codes.data_ptr(), codes.shape[-1], scales.data_ptr(), self._codes_ptr, self._scales_ptr)

    def _allocate(self, like, lead, cols, dtype):
        self.rows, self.cols, self.dtype, self.device = lead[-1], cols, dtype, like.device
        rows = self.rows
        if len(lead) == 2:
            if not 1 <= lead[0] <= experts_hip.MAX_EXPERTS:
                raise ValueError("a matrix for each of 1 to %d experts is wanted, got %s" % (
                    experts_hip.MAX_EXPERTS, tuple(lead) + (cols,)))
            rows *= lead[0]
        self.n_experts = lead[0] if len(lead) == 2 else 0
        pitch, scales_pitch = _pitches(cols)
        self._buffer = like.new_empty(rows * (pitch + scales_pitch), dtype=torch.uint8)
        self._codes_ptr = self._buffer.data_ptr()
        self._scales_ptr = self._codes_ptr + rows * pitch

    def _laid(self, which):
        pitch = _pitches(self.cols)[which]
        begin = which * self.rows * max(1, self.n_experts) * _pitches(self.cols)[0]
        shape = ((self.n_experts,) if self.n_experts else ()) + (self.rows, pitch)
        return self._buffer[begin:begin + self.rows * max(1, self.n_experts) * pitch].view(shape)

    @property
    def laid_codes(self):
        """The codes as the products read them: uint8 (..., rows, a multiple of 128 bytes), zeros behind the last column."""
        return self._laid(0)

    @property
    def laid_scales(self):
        """The scales' bytes as the products read them, 16 for 512 columns."""
        return self._laid(1)

    def codes(self):
        """The codes, one a byte: uint8 (..., rows, cols)."""
        return torch.stack([self.laid_codes & 15, self.laid_codes >> 4], -1).flatten(-2)[..., :self.cols]

    def scales(self):
        """The scales' bytes, uint8 (..., rows, ceil(cols / 32))."""
        laid = self.laid_scales.unflatten(-1, (-1, 4, 4)).transpose(-1, -2).flatten(-3)
        return laid[..., :-(-self.cols // BLOCK)].contiguous()

    def dequantize(self, dtype=torch.float32):
        """The numbers that the matrix stands for, (..., rows, cols), rounded to `dtype`."""
        if dtype not in _TYPES:
            raise TypeError("dtype must be float32, bfloat16 or float16, got %s" % (dtype,))
        lead = (self.n_experts,) if self.n_experts else ()
        out = self._buffer.new_empty(lead + (self.rows, self.cols), dtype=dtype)
        _call(self.device.index, "h2o4gpu_microscale4_dequantize", _TYPES[dtype], self.rows * max(1, self.n_experts),
              self.cols, self._codes_ptr, self._scales_ptr, out.data_ptr(), self.cols)
        return out


def quantize(values):
    """Microscale4 of `values`, (rows, cols) with contiguous rows or (experts, rows, cols) of any strides (which are
    copied if need be), float32, bfloat16 or float16.

    The power of two of 32 columns is that of their largest magnitude over 4, at least 2^-127; elements
    are rounded to the nearest number, a tie to the one of even code, and what is then beyond 6 is 6
    (from 7 times the power on that is a step down by up to a quarter). A block that holds a NaN or an infinity is NaN.
    """
    if not (isinstance(values, torch.Tensor) and values.is_cuda and values.dim() in (2, 3) and values.dtype in _TYPES):
        _tensor("values", values, values.dim() if isinstance(values, torch.Tensor) and values.dim() == 3 else 2)
        _type_of("values", values)
    if values.requires_grad and torch.is_grad_enabled():
        raise ValueError("microscaled numbers have no gradient: detach values")
    _no_tangents(values)
    shape = values.shape
    out = object.__new__(Microscale4)
    out._allocate(values, shape[:-1], shape[-1], values.dtype)
    if len(shape) == 3:
        values = values.reshape(-1, shape[-1])
        if not (values.stride(1) == 1 and (values.shape[0] < 2 or values.stride(0) >= shape[-1])):
            values = values.contiguous()
    ptr, stride = _rows("values", values)
    _call(out.device.index, "h2o4gpu_microscale4_quantize", _TYPES[out.dtype], values.shape[0], out.cols, ptr, stride,
          out._codes_ptr, out._scales_ptr)
    return out


def _operands(x, weights, dtype):
    if type(x) is not Microscale4 or type(weights) is not Microscale4:
        name, m = ("x", x) if type(x) is not Microscale4 else ("weights", weights)
        raise TypeError("%s must be a Microscale4 (quantize), got %s" % (name, type(m).__name__))
    if x.n_experts:
        raise ValueError("x must be (tokens, cols), got a matrix per expert")
    if x.device != weights.device:
        raise ValueError("x is on %s, expected %s" % (x.device, weights.device))
    if x.cols != weights.cols or weights.rows < 1:
        raise ValueError("x has %d columns, weights are %d x %d" % (x.cols, weights.rows, weights.cols))
    dtype = x.dtype if dtype is None else dtype
    if dtype not in _TYPES:
        raise TypeError("dtype must be float32, bfloat16 or float16, got %s" % (dtype,))
    return dtype


def product(x, weights, dtype=None):
    """(tokens, out) = x (tokens, cols) times the transpose of weights (out, cols), both Microscale4; sums
    in float32, rounded once to `dtype` (that of the tokens x was made from)."""
    dtype = _operands(x, weights, dtype)
    if weights.n_experts:
        raise ValueError("weights hold a matrix per expert: experts_product multiplies with those")
    out = weights.rows
    y = x._buffer.new_empty((x.rows, out), dtype=dtype)
    _call(x.device.index, "h2o4gpu_microscale4_product", _TYPES[dtype], x.rows, out, x.cols, x._codes_ptr, x._scales_ptr,
          weights._codes_ptr, weights._scales_ptr, y.data_ptr(), out)
    return y


def experts_product(x, weights, order, in_order=False, dtype=None):
    """(tokens * top_k, out), rows in expert order: the token of every slot of `order` times the
    transpose of its expert's matrix; zeros behind order.offsets[-1]. in_order: x holds rows in expert
    order already (tokens * top_k of them), as a second layer's do; those behind offsets[-1] are not read."""
    dtype = _operands(x, weights, dtype)
    _order_of(order, x.device)
    if not weights.n_experts or weights.n_experts != order.n_experts:
        raise ValueError("order has %d experts, weights %d" % (order.n_experts, weights.n_experts))
    slots = order.tokens * order.top_k
    if x.rows != (slots if in_order else order.tokens):
        raise ValueError("x must be (%d, %d), got (%d, %d)" % (slots if in_order else order.tokens, weights.cols,
                                                               x.rows, x.cols))
    out = weights.rows
    y = x._buffer.new_empty((slots, out), dtype=dtype)
    _call(x.device.index, "h2o4gpu_microscale4_experts_product", _TYPES[dtype], order.tokens, order.top_k,
          weights.n_experts, out, x.cols, x._codes_ptr, x._scales_ptr, weights._codes_ptr, weights._scales_ptr,
          None if in_order else order._order_ptr, order._offsets_ptr, y.data_ptr(), out)
    return y
