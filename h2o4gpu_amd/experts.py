"""Expert layers on PyTorch-ROCm tensors: tokens go to the models ("experts") of their best
centroids or scores, and the results come back and are joined by weight.

    from h2o4gpu_amd import KMeans, experts
    model = KMeans(n_clusters=64).fit(X)
    chosen, weights = experts.route(model.transform(X), top_k=2, largest=False)
    order = experts.sort_by_expert(chosen, 64)
    rows = experts.dispatch(X, order)              # rows of expert 0, then of expert 1, ...
    ...                                            # every expert works on its rows
    Y = experts.combine(rows, weights, order)

`route`, `dispatch` and `combine` have gradients (with respect to the scores, the tokens, the rows
and the weights); forward-mode derivatives are refused. All work is queued on the current stream of
the tensors' device, nothing waits for it and nothing is copied to the host, so the calls can be
recorded into a graph (after a call of the same type and sizes outside of one, which may raise a
kernel's limit of shared memory). Tensors are read on that stream: one that another stream writes has
to be waited for, as with any torch operation, and an ExpertOrder used on another stream than it was
made on likewise. Same inputs give the same bits. The kernels are the library's
(include/h2o4gpu_experts.h); there is no CPU path.
"""
import functools

import torch
from torch.autograd import forward_ad

from .libs import experts_hip

_TYPES = {torch.float32: experts_hip.FLOAT32, torch.bfloat16: experts_hip.BFLOAT16,
          torch.float16: experts_hip.FLOAT16}
_functions = {}
# (the raw handle directly where torch offers it: building a Stream object takes longer than queueing a kernel)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(index, name, *args):
    """Calls a function of the library with `args` and the current stream of device `index`."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(experts_hip.lib(), name)
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        experts_hip.check(name, rc)


def _type_of(name, t):
    code = _TYPES.get(t.dtype)
    if code is None:
        raise TypeError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    return code


def _tensor(name, t, dims, device=None, dtype=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor, got %s" % (name, type(t).__name__))
    if not t.is_cuda:
        raise ValueError("%s must be on the GPU" % name)
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, expected %s" % (name, t.device, device))
    if t.dim() != dims:
        raise ValueError("%s must have %d dimensions, got shape %s" % (name, dims, tuple(t.shape)))
    if dtype is not None and t.dtype != dtype:
        raise TypeError("%s must be %s, got %s" % (name, dtype, t.dtype))


def _rows(name, t):
    """(pointer, elements between rows) of a matrix whose rows are contiguous."""
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError("the rows of %s must be contiguous (strides %s)" % (name, t.stride()))
    stride = t.stride(0)
    if t.shape[0] < 2:
        stride = t.shape[1]
    elif stride < t.shape[1]:
        raise ValueError("the rows of %s overlap (strides %s)" % (name, t.stride()))
    return t.data_ptr(), stride


def _no_tangents(*tensors):
    """Refuses tensors of a forward-mode derivative: their tangents would be left out without a word."""
    if getattr(forward_ad, "_current_level", 0) >= 0:  # (outside of any dual_level, this is all that is looked at)
        for t in tensors:
            if forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("expert layers and 4-bit products have no forward-mode derivative")


class _Once(torch.autograd.Function):
    """A gradient as it is, behind which nothing can be differentiated with respect to what it was made of."""

    @staticmethod
    def forward(ctx, gradient, *sources):
        return gradient.view_as(gradient)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("the gradients of expert layers cannot be differentiated again")


def _once(gradient, *sources):
    """What a backward pass returns for a gradient that the kernels made of `sources`. Under create_graph it
    belongs to a graph, in which others' gradients may be differentiated again and this one is an error."""
    if torch.is_grad_enabled() and any(s.requires_grad for s in sources):
        return _Once.apply(gradient, *sources)
    return gradient


def _gradient(t):
    """An incoming gradient with contiguous rows (autograd hands out expanded and transposed ones)."""
    if t.stride(1) == 1 and (t.shape[0] < 2 or t.stride(0) >= t.shape[1]):
        return t
    return t.contiguous()


# ---- routing -----------------------------------------------------------------------------------

class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, top_k, largest, scale, over_all):
        chosen, weights = _route(scores, top_k, largest, scale, over_all)
        ctx.mark_non_differentiable(chosen)
        ctx.set_materialize_grads(False)  # (a tensor of zeros for the choice, otherwise)
        ctx.save_for_backward(scores, chosen, weights)
        ctx.how = (top_k, largest, scale, over_all)
        return chosen, weights

    @staticmethod
    def backward(ctx, _, dweights):
        if dweights is None:
            return None, None, None, None, None
        scores, chosen, weights = ctx.saved_tensors
        top_k, largest, scale, over_all = ctx.how
        dscores = torch.empty_like(scores)
        dweights = _gradient(dweights).contiguous()
        rows, n_experts = scores.shape
        _call(scores.device.index, "h2o4gpu_experts_route_backward", _TYPES[scores.dtype], rows, n_experts, top_k,
              largest, over_all, scale, scores.data_ptr(), *scores.stride(), chosen.data_ptr(), weights.data_ptr(),
              dweights.data_ptr(), dscores.data_ptr(), *dscores.stride())
        return _once(dscores, scores, dweights), None, None, None, None


def _route(scores, top_k, largest, scale, over_all):
    rows, n_experts = scores.shape
    chosen = scores.new_empty((rows, top_k), dtype=torch.int32)
    weights = torch.empty_like(chosen, dtype=torch.float32)
    _call(scores.device.index, "h2o4gpu_experts_route", _TYPES[scores.dtype], rows, n_experts, top_k, largest,
          over_all, scale, scores.data_ptr(), *scores.stride(), chosen.data_ptr(), weights.data_ptr())
    return chosen, weights


def route(scores, top_k, largest=True, scale=1.0, over_all=False):
    """The `top_k` best experts of every row, best first, and their weights.

    scores: (rows, experts), any strides: a model's scores (largest=True) or squared distances as
    KMeans.transform gives them for float32 rows (largest=False: the nearest are the best; up to eight
    of them are found in one pass over the distances, more in one for each). Equal scores go to the
    lowest index. NaN and the worst infinity mark experts that are not available; where none is left
    the expert is -1 and its weight 0. Scores of the best infinity share the weight equally.

    Returns (experts, weights), int32 and float32, both (rows, top_k). The weights are the softmax of
    scale * score (scale * -score for distances) over the chosen experts, or with over_all over every
    available one. They have a gradient with respect to the scores, the choice held fixed.
    """
    if not (isinstance(scores, torch.Tensor) and scores.is_cuda and scores.dim() == 2 and scores.dtype in _TYPES):
        _tensor("scores", scores, 2)
        _type_of("scores", scores)
    top_k, largest, scale, over_all = int(top_k), int(bool(largest)), float(scale), int(bool(over_all))
    if not 1 <= scores.shape[1] <= experts_hip.MAX_EXPERTS:
        raise ValueError("scores must have 1 to %d experts, got %d" % (experts_hip.MAX_EXPERTS, scores.shape[1]))
    if not 1 <= top_k <= min(scores.shape[1], experts_hip.MAX_TOP_K):
        raise ValueError("top_k must be 1 to %d, got %d" % (min(scores.shape[1], experts_hip.MAX_TOP_K), top_k))
    if not 0.0 <= scale <= 3.4e38:
        raise ValueError("scale must be finite and not negative, got %r" % scale)
    _no_tangents(scores)
    if scores.requires_grad and torch.is_grad_enabled():
        return _Route.apply(scores, top_k, largest, scale, over_all)
    return _route(scores, top_k, largest, scale, over_all)


# ---- order by expert ----------------------------------------------------------------------------

class ExpertOrder:
    """Slots ordered by expert, as sort_by_expert makes it; token t's j-th choice is slot t * top_k + j.

    order (tokens * top_k,): the slots of expert 0, then of expert 1, ..., each in ascending order, then
    those without an expert. position (tokens, top_k): a slot's place in it, as ~place (negative) where
    it has no expert. offsets (n_experts + 1,): where each expert's rows begin; the last is how many
    slots have one. All int32, on the GPU, in one allocation.
    """

    __slots__ = ("n_experts", "tokens", "top_k", "device", "_buffer", "_order_ptr", "_position_ptr", "_offsets_ptr")

    def __init__(self, buffer, tokens, top_k, n_experts):
        slots = tokens * top_k
        self.n_experts, self.tokens, self.top_k, self.device, self._buffer = n_experts, tokens, top_k, buffer.device, buffer
        self._order_ptr = buffer.data_ptr()
        self._position_ptr = self._order_ptr + 4 * slots
        self._offsets_ptr = self._position_ptr + 4 * slots

    @property
    def order(self):
        return self._buffer.as_strided((self.tokens * self.top_k,), (1,), 0)

    @property
    def position(self):
        return self._buffer.as_strided((self.tokens, self.top_k), (self.top_k, 1), self.tokens * self.top_k)

    @property
    def offsets(self):
        return self._buffer.as_strided((self.n_experts + 1,), (1,), 2 * self.tokens * self.top_k)


@functools.lru_cache(maxsize=256)
def _workspace(slots, n_experts):
    return experts_hip.lib().h2o4gpu_experts_sort_workspace(slots, n_experts)


def sort_by_expert(experts, n_experts):
    """ExpertOrder of the (tokens, top_k) int32 choices of `route` (or of (tokens,) labels).
    A value that is none of 0 .. n_experts - 1 is a slot without an expert.

    While it runs, many slots take a workspace: n_experts / 512 bytes a slot up to some 3200 experts, and
    as a workgroup then has fewer slots, 20 bytes at 5000 and 256 at 16384."""
    if isinstance(experts, torch.Tensor) and experts.dim() == 1:
        experts = experts.unsqueeze(1)
    _tensor("experts", experts, 2, dtype=torch.int32)
    n_experts = int(n_experts)
    tokens, top_k = experts.shape
    if not 1 <= n_experts <= experts_hip.MAX_EXPERTS:
        raise ValueError("n_experts must be 1 to %d, got %d" % (experts_hip.MAX_EXPERTS, n_experts))
    if not 1 <= top_k <= experts_hip.MAX_TOP_K:
        raise ValueError("experts must have 1 to %d choices a token, got %d" % (experts_hip.MAX_TOP_K, top_k))
    experts = experts.contiguous()
    slots = tokens * top_k
    need = _workspace(slots, n_experts)
    work = experts.new_empty(need // 4) if need else None
    order = ExpertOrder(experts.new_empty(2 * slots + n_experts + 1), tokens, top_k, n_experts)
    _call(order.device.index, "h2o4gpu_experts_sort", slots, n_experts, experts.data_ptr(), order._order_ptr,
          order._position_ptr, order._offsets_ptr, work.data_ptr() if need else None, need)
    return order


def _order_of(order, device):
    if not isinstance(order, ExpertOrder):
        raise TypeError("order must be an ExpertOrder (sort_by_expert), got %s" % type(order).__name__)
    if order.device != device:
        raise ValueError("order is on %s, expected %s" % (order.device, device))


# ---- rows out and back ---------------------------------------------------------------------------

def _dispatch(x, order):
    ptr, stride = _rows("x", x)
    cols = x.shape[1]
    rows = x.new_empty((order.tokens * order.top_k, cols))
    _call(x.device.index, "h2o4gpu_experts_dispatch", _TYPES[x.dtype], order.tokens, order.top_k, cols, ptr, stride,
          order._position_ptr, rows.data_ptr(), cols)
    return rows


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order):
        ctx.order = order
        return _dispatch(x, order)

    @staticmethod
    def backward(ctx, drows):
        order = ctx.order
        drows = _gradient(drows)
        ptr, stride = _rows("drows", drows)
        cols = drows.shape[1]
        dx = drows.new_empty((order.tokens, cols))
        _call(drows.device.index, "h2o4gpu_experts_dispatch_backward", _TYPES[drows.dtype], order.tokens, order.top_k,
              cols, ptr, stride, order._position_ptr, dx.data_ptr(), cols)
        return _once(dx, drows), None


def dispatch(x, order):
    """Rows in expert order, (tokens * top_k, cols): the token of every slot of `order`, zeros in the
    places behind offsets[-1]. x: (tokens, cols) with contiguous rows. Its gradient is the sum of a
    token's rows' gradients."""
    if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dim() == 2 and x.dtype in _TYPES):
        _tensor("x", x, 2)
        _type_of("x", x)
    _order_of(order, x.device)
    if x.shape[0] != order.tokens or x.shape[1] < 1:
        raise ValueError("x must be (%d, cols), got %s" % (order.tokens, tuple(x.shape)))
    _no_tangents(x)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(x, order)
    return _dispatch(x, order)


def _combine(rows, weights, order):
    ptr, stride = _rows("rows", rows)
    cols = rows.shape[1]
    out = rows.new_empty((order.tokens, cols))
    _call(rows.device.index, "h2o4gpu_experts_combine", _TYPES[rows.dtype], order.tokens, order.top_k, cols, ptr,
          stride, weights.data_ptr(), order._position_ptr, out.data_ptr(), cols)
    return out


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, order):
        ctx.order = order
        ctx.save_for_backward(rows, weights)
        return _combine(rows, weights, order)

    @staticmethod
    def backward(ctx, dout):
        order = ctx.order
        rows, weights = ctx.saved_tensors
        dout = _gradient(dout)
        gptr, gstride = _rows("dout", dout)
        rptr, rstride = _rows("rows", rows)
        drows, dweights = rows.new_empty(rows.shape), torch.empty_like(weights)
        _call(rows.device.index, "h2o4gpu_experts_combine_backward", _TYPES[rows.dtype], order.tokens, order.top_k,
              rows.shape[1], gptr, gstride, rptr, rstride, weights.data_ptr(), order._position_ptr,
              drows.data_ptr(), rows.shape[1], dweights.data_ptr())
        return _once(drows, weights, dout), _once(dweights, rows, dout), None


def combine(rows, weights, order):
    """(tokens, cols): the weighted sum of every token's rows, summed in float32 and rounded once.
    rows: (tokens * top_k, cols) in expert order; weights: (tokens, top_k) float32. Slots without an
    expert add nothing, whatever lies in their places. Gradients for rows and weights."""
    if not (isinstance(rows, torch.Tensor) and rows.is_cuda and rows.dim() == 2 and rows.dtype in _TYPES):
        _tensor("rows", rows, 2)
        _type_of("rows", rows)
    _order_of(order, rows.device)
    _tensor("weights", weights, 2, rows.device, torch.float32)
    if rows.shape[0] != order.tokens * order.top_k or rows.shape[1] < 1:
        raise ValueError("rows must be (%d, cols), got %s" % (order.tokens * order.top_k, tuple(rows.shape)))
    if tuple(weights.shape) != (order.tokens, order.top_k):
        raise ValueError("weights must be (%d, %d), got %s" % (order.tokens, order.top_k, tuple(weights.shape)))
    _no_tangents(rows, weights)
    weights = weights.contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or weights.requires_grad):
        return _Combine.apply(rows, weights, order)
    return _combine(rows, weights, order)
