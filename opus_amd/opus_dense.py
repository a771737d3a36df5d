"""The dense operators a decoder layer runs around ``sampling_4d``, as hand-written kernels with gradients.

    linear          y = residual + D(act(x W^T + bias))
    residual_norm   r = residual_scale * x + gate * D(post(block));  y = norm(r)
    dropout         y = residual + D(x)

The reference composes them from library layers (models/opus_transformer.py:225-247, :329-358, :381-448): the
products that make sampling offsets and scale weights, the mixing's parameters and its way back into the query stream,
the feed-forward block, and the norm that follows each of them.

Common to the three: tensors are fp32, bf16 or fp16, all of one type, on one GPU (CPU tensors raise); products, sums,
statistics and the epilogue are in fp32 and every result is rounded once.  A tensor that is not contiguous is copied
first.  The calls are asynchronous on the current stream of the tensors' device, allocate through torch, keep nothing but
the sizes of workspaces and can be captured into a HIP graph.  Results do not depend on the order in which workgroups run:
the same call on the same inputs gives the same bits (asking for other gradients along with one may round that one
otherwise).

Gradients are first-order and reverse-mode only: a tensor with a forward-mode tangent is refused, before or in a backward.
``torch.jit.trace`` records the calls (not their backward, which raises); ``torch.fx``'s tracer at the dispatcher and
``torch.func``'s transforms are refused.

``D`` is dropout with a counter-based generator: whether element (row, column) is kept is computed from
``(seed, offset, row, column)`` - row counting the tensor's last-dimension rows - by Philox 4x32-10, in the forward
and again in the backward; no mask is stored, and the type, the operator and the launch make no difference to it.  The
probability ``p`` is taken to the nearest multiple of 1/65536, kept elements are scaled by the inverse of the
probability so rounded, and a dropped element is exactly 0 (even inf or NaN).  ``seed`` is an int (64 bits are used)
or a one-element int64 tensor on the tensors' device, read when the kernels run: a captured graph draws new masks
when that tensor is changed between replays.  It must not change between a forward and its backward.  Give every
dropout of a step an ``offset`` (0 .. 2**32 - 1) of its own.
"""
import ctypes
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.fx.experimental import proxy_tensor

from . import _lib

_TYPES = {torch.float32: _lib.DENSE_F32, torch.bfloat16: _lib.DENSE_BF16, torch.float16: _lib.DENSE_F16}


# ------------------------------------------------------------------------------------------------
# arguments
# ------------------------------------------------------------------------------------------------
def _check(what, x, names, others):
    """One type, one GPU; ``others`` are tensors or None, ``names`` what they are called."""
    if not x.is_cuda:
        raise RuntimeError(f"{what}: expected CUDA tensors")
    dtype, device = x.dtype, x.device
    if dtype not in _TYPES:
        raise RuntimeError(f"{what}: expected float32, bfloat16 or float16 tensors, got {dtype}")
    if x.dim() < 1:
        raise RuntimeError(f"{what}: expected a tensor of at least one dimension")
    for i, t in enumerate(others):
        if t is not None:
            if t.dtype != dtype:
                raise RuntimeError(f"{what}: {names[i]} is {t.dtype}, expected {dtype}")
            if t.device != device:
                raise RuntimeError(f"{what}: {names[i]} is on {t.device}, expected {device}")


def _threshold(what, p, seed, offset, device):
    """p -> threshold of 65536 (0: no dropout); checks the generator's arguments."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: dropout probability has to be between 0 and 1, got {p}")
    threshold = round(float(p) * 65536)
    if threshold == 0:
        return 0
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise RuntimeError(f"{what}: a seed tensor has to hold one int64 on {device}")
    elif not hasattr(seed, "__index__") or isinstance(seed, bool):
        raise RuntimeError(f"{what}: dropout needs a seed, an int or a one-element int64 tensor")
    if not hasattr(offset, "__index__") or isinstance(offset, (bool, torch.Tensor)):
        raise RuntimeError(f"{what}: offset has to be an int, got {offset!r}")
    if not 0 <= offset < 2 ** 32:
        raise ValueError(f"{what}: offset has to be in [0, 2**32), got {offset}")
    return threshold


def _drop_struct(threshold, seed, offset):
    if threshold == 0:
        return None
    if isinstance(seed, torch.Tensor):
        return _lib.DenseDropout(threshold, int(offset), 0, seed.data_ptr())
    return _lib.DenseDropout(threshold, int(offset), int(seed) & (2 ** 64 - 1), None)


def _seed_tensor(drop, seed):
    """The seed as what autograd keeps an eye on (None for a number): changed in place before the backward, it would
    give another mask there."""
    return seed if drop is not None and isinstance(seed, torch.Tensor) else None


def _drop_again(drop, seed):
    """The forward's dropout for the backward: with the seed tensor autograd hands back, which need not lie where the
    forward's did (saved-tensor hooks may have moved it)."""
    return drop if seed is None else _lib.DenseDropout(drop.threshold, drop.offset, 0, seed.data_ptr())


def _ptr(t):
    return None if t is None else t.data_ptr()


# the current stream's handle: what torch.cuda.current_stream(index).cuda_stream gives, without making a Stream object
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _run(what, fn, device, *args):
    """Calls a C entry, whose last argument is the stream, with ``device`` current."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream(index))
    if rc != 0:
        _lib.check_dense(rc, what)


def _contiguous(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


_is_tracing, _transforms_active = torch._C._is_tracing, torch._C._are_functorch_transforms_active


def _refuse_transforms(what, tensors):
    """A graph tracer at the dispatcher (make_fx) and functionalisation see the allocations of a call but not its kernels:
    what they make of it would return memory nobody wrote."""
    if proxy_tensor._CURRENT_MAKE_FX_TRACER is not None and proxy_tensor.get_proxy_mode() is not None:      # (this thread's)
        raise RuntimeError(f"{what}: cannot be traced by torch.fx")
    if _transforms_active() and any(t is not None and torch._is_functional_tensor(t) for t in tensors):
        raise RuntimeError(f"{what}: cannot be functionalised")


def _needs_autograd(what, tensors):
    """Whether a call has to go through its autograd function: where a gradient is wanted; under ``torch.jit.trace``, which
    records that function and not the kernels inside; and in a forward-mode level, where that function refuses a tensor
    with a tangent, which would otherwise be lost."""
    if proxy_tensor._CURRENT_MAKE_FX_TRACER is not None or _transforms_active():
        _refuse_transforms(what, tensors)
    if _is_tracing() or forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and getattr(t, "requires_grad", False):        # (what is no tensor is refused later)
                return True
    return False


def _first_order(backward):
    """``once_differentiable``, entered only where a graph of the backward is asked for; other ways to look into the
    backward are refused."""
    guarded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        _refuse_transforms("backward", grads)
        if _is_tracing():
            raise RuntimeError("a backward of a dense operator cannot be traced")
        if forward_ad._current_level >= 0 and any(g is not None and forward_ad.unpack_dual(g).tangent is not None for g in grads):
            raise RuntimeError("gradients of a dense operator are first-order only: no tangent goes through its backward")
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return staticmethod(run)


# sizes alone decide these
@functools.lru_cache(maxsize=4096)
def _linear_workspace(kind, M, N, K):
    return _lib.load().opus_dense_linear_workspace_bytes(kind, M, N, K)


@functools.lru_cache(maxsize=4096)
def _linear_backward_workspace(kind, M, N, K):
    return _lib.load().opus_dense_linear_backward_workspace_bytes(kind, M, N, K)


@functools.lru_cache(maxsize=4096)
def _norm_backward_workspace(kind, rows, width, gate_rows):
    return _lib.load().opus_dense_norm_backward_workspace_bytes(kind, rows, width, gate_rows)


# ------------------------------------------------------------------------------------------------
# linear
# ------------------------------------------------------------------------------------------------
def _linear_forward(x, weight, bias, residual, activation, dropout_p, seed, offset, want_z):
    """-> y, z or None, the activation's code, the dropout.  The checks are here, so that a traced call makes them too."""
    _check("linear", x, ("weight", "bias", "residual"), (weight, bias, residual))
    shape, w_shape = x.shape, weight.shape
    if len(w_shape) != 2 or w_shape[1] != shape[-1]:
        raise RuntimeError(f"linear: weight {list(w_shape)} does not fit x {list(shape)}")
    if bias is not None and bias.shape != w_shape[:1]:
        raise RuntimeError(f"linear: bias {list(bias.shape)} does not fit weight {list(w_shape)}")
    if residual is not None and residual.shape != shape[:-1] + w_shape[:1]:
        raise RuntimeError(f"linear: residual {list(residual.shape)} is not of the output's shape")
    code = _lib.DENSE_ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"linear: activation has to be one of {sorted(_lib.DENSE_ACTIVATIONS)}, got {activation!r}")
    threshold = _threshold("linear", dropout_p, seed, offset, x.device) if dropout_p != 0.0 else 0
    drop = _drop_struct(threshold, seed, offset)
    N, K = w_shape
    x, weight, bias, residual = _contiguous(x), _contiguous(weight), _contiguous(bias), _contiguous(residual)
    kind, device = _TYPES[x.dtype], x.device
    y = x.new_empty(shape[:-1] + w_shape[:1])
    M = x.numel() // K if K else y.numel() // max(N, 1)
    z = torch.empty_like(y) if want_z and code else None
    need = _linear_workspace(kind, M, N, K)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _run("linear", _lib.load().opus_dense_linear_forward, device, kind, x.data_ptr(), weight.data_ptr(), _ptr(bias),
         _ptr(residual), M, N, K, code, drop, y.data_ptr(), _ptr(z), _ptr(ws), need)
    return y, z, code, drop


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, dropout_p, seed, offset):
        y, z, code, drop = _linear_forward(x, weight, bias, residual, activation, dropout_p, seed, offset,
                                           any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, weight, z, _seed_tensor(drop, seed))
        ctx.settings = code, drop
        return y

    @_first_order
    def backward(ctx, dy):
        x, weight, z, seed = ctx.saved_tensors
        activation, drop = ctx.settings
        drop = _drop_again(drop, seed)
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            N, K = weight.shape
            kind, device = _TYPES[x.dtype], x.device
            M = x.numel() // K if K else dy.numel() // max(N, 1)
            x, weight, g = _contiguous(x), _contiguous(weight), _contiguous(dy)
            if need_x:
                dx = torch.empty_like(x)
            if need_w:
                dw = torch.empty_like(weight)
            if need_b:
                db = weight.new_empty(N)
            dz = torch.empty_like(g) if activation or drop is not None else None
            need = _linear_backward_workspace(kind, M, N, K)
            ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
            _run("linear backward", _lib.load().opus_dense_linear_backward, device, kind, g.data_ptr(), x.data_ptr(),
                 weight.data_ptr(), _ptr(z), M, N, K, activation, drop, _ptr(dz), _ptr(dx), _ptr(dw), _ptr(db),
                 _ptr(ws), need)
        return dx, dw, db, dy if need_r else None, None, None, None, None


def linear(x, weight, bias=None, activation="none", residual=None, dropout_p=0.0, seed=None, offset=0):
    """``residual + D(act(x @ weight.T + bias))`` in one pass over the product.

    x [..., K], weight [N, K], bias [N] or None, residual [..., N] or None -> [..., N].  ``activation``: "none",
    "relu", "gelu" (with erf), "gelu_tanh" or "silu".  ``dropout_p``, ``seed``, ``offset``: see the module's text.
    Gradients flow to x, weight, bias and residual.  With an activation the backward needs x W^T + bias, which the
    forward then stores in the tensors' type (only where a gradient is wanted; finite values beyond that type as its largest
    number); d act(x W^T + bias) is rounded to that type too before the two products of the backward (the bias' gradient is
    summed before)."""
    args = x, weight, bias, residual, activation, dropout_p, seed, offset
    if _needs_autograd("linear", args[:4]):
        return _Linear.apply(*args)
    return _linear_forward(*args, False)[0]


# ------------------------------------------------------------------------------------------------
# residual_norm
# ------------------------------------------------------------------------------------------------
def _norm_struct(tensors, kind, rows, gate_rows, eps, scale, drop):
    x, block, weight, bias, post_weight, post_bias, gate = tensors
    return _lib.DenseNorm(_TYPES[x.dtype], kind, rows, x.shape[-1], gate_rows, eps, scale, x.data_ptr(),
                          block.data_ptr(), _ptr(weight), _ptr(bias), _ptr(post_weight), _ptr(post_bias), _ptr(gate),
                          None if drop is None else ctypes.addressof(drop))


_NORM_NAMES = ("block", "weight", "bias", "post_weight", "post_bias", "gate")


def _gate_rows(x, gate):
    """How many rows the gate has; row i of x uses gate row i // (rows of x // rows of the gate)."""
    width, lead = x.shape[-1], x.shape[:-1]
    if gate.dim() >= 1 and gate.shape[-1] == width:
        g = gate.shape[:-1]
        if len(g) == 0 or g == lead:
            return g.numel()
        if len(g) == 1 and len(lead) > 0 and g[0] == lead[0]:
            return g[0]
        if len(g) == len(lead):
            n = len(g)
            while n and g[n - 1] == 1:
                n -= 1
            if g[:n] == lead[:n]:
                return g[:n].numel()
    raise RuntimeError(f"residual_norm: gate {list(gate.shape)} does not fit x {list(x.shape)}: expected "
                       f"[{width}], [{lead[0] if len(lead) else 1}, {width}], x's shape, or x's shape with ones for "
                       f"trailing leading dimensions")


def _norm_forward(x, block, weight, bias, post_weight, post_bias, gate, kind, eps, residual_scale, dropout_p, seed, offset,
                  want_stream, want_stats):
    """-> y, r or None, the statistics or None, the settings.  The checks are here, so that a traced call makes them too."""
    tensors = (x, block, weight, bias, post_weight, post_bias, gate)
    _check("residual_norm", x, _NORM_NAMES, tensors[1:])
    shape = x.shape
    width = shape[-1]
    if block.shape != shape:
        raise RuntimeError(f"residual_norm: block {list(block.shape)} is not of x's shape {list(shape)}")
    if not 1 <= width <= _lib.DENSE_MAX_WIDTH:
        raise RuntimeError(f"residual_norm: width has to be in [1, {_lib.DENSE_MAX_WIDTH}], got {width}")
    for i in range(2, 6):
        t = tensors[i]
        if t is not None and (t.dim() != 1 or t.shape[0] != width):
            raise RuntimeError(f"residual_norm: {_NORM_NAMES[i - 1]} {list(t.shape)} has to be [{width}]")
    if post_bias is not None and post_weight is None:
        raise RuntimeError("residual_norm: post_bias without post_weight")
    code = _lib.DENSE_NORMS.get(kind)
    if code is None:
        raise ValueError(f"residual_norm: kind has to be one of {sorted(_lib.DENSE_NORMS)}, got {kind!r}")
    if isinstance(residual_scale, torch.Tensor) or isinstance(eps, torch.Tensor):
        raise RuntimeError("residual_norm: residual_scale and eps are numbers, not tensors (no gradient would reach them)")
    eps, residual_scale = float(eps), float(residual_scale)
    if not eps >= 0.0:
        raise ValueError(f"residual_norm: eps has to be no less than 0, got {eps}")
    gate_rows = 0 if gate is None else _gate_rows(x, gate)
    threshold = _threshold("residual_norm", dropout_p, seed, offset, x.device) if dropout_p != 0.0 else 0
    drop = _drop_struct(threshold, seed, offset)
    tensors = [_contiguous(t) for t in tensors]
    x = tensors[0]
    rows = x.numel() // width
    y = torch.empty_like(x)
    stream = torch.empty_like(x) if want_stream else None
    stats = torch.empty((rows, 4), dtype=torch.float32, device=x.device) if want_stats else None
    args = _norm_struct(tensors, code, rows, gate_rows, eps, residual_scale, drop)
    _run("residual_norm", _lib.load().opus_dense_norm_forward, x.device, args, y.data_ptr(), _ptr(stream), _ptr(stats))
    return y, stream, stats, (code, gate_rows, eps, residual_scale, drop)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, block, weight, bias, post_weight, post_bias, gate, kind, eps, residual_scale, dropout_p, seed, offset,
                want_stream):
        tensors = (x, block, weight, bias, post_weight, post_bias, gate)
        y, stream, stats, ctx.settings = _norm_forward(*tensors, kind, eps, residual_scale, dropout_p, seed, offset,
                                                       want_stream, True)
        ctx.save_for_backward(*tensors, stats, _seed_tensor(ctx.settings[4], seed))
        ctx.set_materialize_grads(False)
        return (y, stream) if want_stream else y

    @_first_order
    def backward(ctx, dy, dstream=None):
        if dy is None and dstream is None:
            return (None,) * 14
        saved = ctx.saved_tensors
        kind, gate_rows, eps, scale, drop = ctx.settings
        drop = _drop_again(drop, saved[8])
        tensors, stats = [_contiguous(t) for t in saved[:7]], saved[7]
        grads = [torch.empty_like(t) if need else None for t, need in zip(tensors, ctx.needs_input_grad)]
        x = tensors[0]
        width = x.shape[-1]
        rows = x.numel() // width
        dy, dstream = _contiguous(dy), _contiguous(dstream)
        args = _norm_struct(tensors, kind, rows, gate_rows, eps, scale, drop)
        need = _norm_backward_workspace(args.type, rows, width, gate_rows)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
        _run("residual_norm backward", _lib.load().opus_dense_norm_backward, x.device, args, _ptr(dy), _ptr(dstream),
             stats.data_ptr(), _lib.DenseNormGrads(*[None if g is None else g.data_ptr() for g in grads]), _ptr(ws),
             need)
        return (*grads, *(None,) * 7)


def residual_norm(x, block, weight=None, bias=None, kind="layer", eps=1e-5, post_weight=None, post_bias=None, gate=None,
                  residual_scale=1.0, dropout_p=0.0, seed=None, offset=0, return_stream=False):
    """The norm between two blocks, with what joins the first block's output to the stream.

        r = residual_scale * x + gate * D(post(block));  y = norm(r)

    x and block [..., width], width at most 16384.  ``kind``: "layer" (mean and variance) or "rms" (mean square), for
    both norms; ``eps`` is added to the variance (mean square).  weight, bias [width] or None (1 and 0).
    ``post_weight`` [width] puts a norm of the block's output before the sum (``post_bias`` [width] or None); None:
    the block's output enters as it is.  ``gate``: [width], one row for each index of x's first dimension
    ([x.shape[0], width]), one for each row (x's shape), or x's shape with ones in place of its last leading
    dimensions; None: 1.  ``residual_scale`` is a number.  ``dropout_p``, ``seed``, ``offset``: see the module's text.

    Returns y, or (y, r) with ``return_stream``.  y is computed from the unrounded r.  Gradients flow to all tensors,
    from either result; the backward computes r again from x and block, so that only two statistics for each norm
    and row are kept."""
    args = (x, block, weight, bias, post_weight, post_bias, gate, kind, eps, residual_scale, dropout_p, seed, offset,
            return_stream)
    if _needs_autograd("residual_norm", args[:7]):
        return _ResidualNorm.apply(*args)
    y, stream, _, _ = _norm_forward(*args, False)
    return (y, stream) if return_stream else y


# ------------------------------------------------------------------------------------------------
# dropout
# ------------------------------------------------------------------------------------------------
def _dropout(x, residual, drop):
    x, residual = _contiguous(x), _contiguous(residual)
    cols = x.shape[-1]
    y = torch.empty_like(x)
    _run("dropout", _lib.load().opus_dense_dropout, x.device, _TYPES[x.dtype], x.data_ptr(), _ptr(residual),
         x.numel() // max(cols, 1), cols, drop, y.data_ptr())
    return y


def _dropout_forward(x, residual, p, seed, offset):
    """-> y, the dropout.  The checks are here, so that a traced call makes them too."""
    _check("dropout", x, ("residual",), (residual,))
    if residual is not None and residual.shape != x.shape:
        raise RuntimeError(f"dropout: residual {list(residual.shape)} is not of x's shape {list(x.shape)}")
    drop = _drop_struct(_threshold("dropout", p, seed, offset, x.device), seed, offset)
    return _dropout(x, residual, drop), drop


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        y, ctx.drop = _dropout_forward(x, residual, p, seed, offset)
        watched = _seed_tensor(ctx.drop, seed)
        if watched is not None:
            ctx.save_for_backward(watched)
        return y

    @_first_order
    def backward(ctx, dy):
        saved = ctx.saved_tensors               # (a seed tensor that was changed since is an error)
        drop = _drop_again(ctx.drop, saved[0]) if saved else ctx.drop
        need_x, need_r = ctx.needs_input_grad[:2]
        return _dropout(dy, None, drop) if need_x else None, dy if need_r else None, None, None, None


def dropout(x, p, seed, offset=0, residual=None):
    """``residual + D(x)``: x [..., columns], residual of x's shape or None.  See the module's text for ``D``.
    Gradients flow to x and residual."""
    if _needs_autograd("dropout", (x, residual)):
        return _Dropout.apply(x, residual, p, seed, offset)
    return _dropout_forward(x, residual, p, seed, offset)[0]
