"""Learned mel inversion: dense layers and group norms on the GPU, and the network made of them.

The reference inverts mel -> linear with one fixed basis, ``np.dot(filterbank.T, mel)`` (griffin_lim.py:18-19).  A
learned inversion takes the log-mel frames (B, T, n_mels) the decoder emits to linear magnitudes (B, T, n_fft/2 + 1)
and is fitted on the pairs that ``analysis.audio_to_mel(..., return_magnitude=True)`` makes.  No counterpart in the
reference.

* :func:`dense`, :func:`group_norm` -- the operators, channels last; differentiable when an input requires a gradient.
* :func:`dense_backward`, :func:`group_norm_backward` -- their gradients as calls of their own.
* :class:`MelInversion` -- a residual network of the two; ``griffin_lim.logmel_to_audio(..., inversion=net)`` runs it
  in place of the fixed basis.

Tensors are float32, bfloat16 or float16 on one GPU; work goes to the current stream of that GPU.  Rows may be views
with a row stride (``h[..., :512]``); anything that is not one row stride over contiguous rows is copied first.  Inside
``Plan.capture()`` nothing may be allocated: pass ``out=`` and ``workspace=`` (a uint8 tensor of at least
:func:`dense_workspace` / ... bytes, not used by anything that may run at the same time).  The differentiable form
refuses to run under a stream capture: autograd's own bookkeeping for leaves that already live in an eager graph ends
the process there; capture the explicit forward and backward calls instead.  Tangents (forward-mode derivatives) and
torch.jit.trace are refused.
"""
import contextlib
import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from .plan import _require_gpu, raw_capture_active

try:
    from . import _calls                 # the plain case of the calls below, compiled; they say None to any other
except ImportError:                      # not built: all cases take the way through this file
    _calls = None

ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3, "tanh": 4, "exp": 5}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


# -- argument plumbing -----------------------------------------------------------------------------------------
# Small calls are bound by the host: the plain case goes through _calls; for the others the checks here are few attribute
# reads each.
def _activation(name):
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {sorted(k for k in ACTIVATIONS if k)} or None, got {name!r}") from None


def _tensor(t, what, device=None, dtype=None, shape=None):
    if device is not None and isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device:
        return t
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what} must be a torch tensor, got {type(t).__name__}")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {t.dtype}")
    if device is None:
        if not t.is_cuda:
            _require_gpu(t.device)
    elif t.device != device:
        raise ValueError(f"{what} is on {t.device}, expected {device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _row_stride(t):
    """Elements between the rows of t (..., cols) when all its rows lie at one stride and are contiguous, else None."""
    cols = t.shape[-1]
    if t.is_contiguous():
        return cols
    if cols > 1 and t.stride(-1) != 1:
        return None
    step, span = None, 1
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if step is None:
            step = stride
        elif stride != step * span:
            return None
        span *= size
    if step is None:
        return cols
    return step if cols <= step <= 2 ** 31 else None


def _rows(t):
    """(tensor, row stride) of an input, copied when its rows do not lie at one stride."""
    stride = _row_stride(t)
    if stride is None:
        t = _copy(t)
        stride = t.shape[-1]
    return t, stride


def _copy(t):
    if raw_capture_active():
        raise RuntimeError("inside Plan.capture() nothing may be copied: pass inputs with contiguous rows at one stride")
    return t.detach().contiguous()


def _vector(t):
    return t if t.is_contiguous() else _copy(t)


def _p(t):
    return None if t is None else t.data_ptr()


def _span(t):
    """Bytes [first, last) a tensor reaches."""
    n, first = t.numel(), t.data_ptr()
    if n and not t.is_contiguous():
        n = 1 + sum((k - 1) * s for k, s in zip(t.shape, t.stride()))
    return first, first + n * t.element_size()


def _apart(out, what, others, same=()):
    """Refuses an output whose memory an input still needs; `same`: inputs it may be, element for element."""
    a0, a1 = _span(out)
    for name, t in others:
        if t is None:
            continue
        b0, b1 = _span(t)
        if a0 < b1 and b0 < a1:
            if b0 == a0 and any(t is s for s in same) and t.stride() == out.stride() and t.dtype == out.dtype:
                continue
            raise ValueError(f"{what} overlaps {name}")


def _new(shape, dtype, device, what):
    if raw_capture_active():
        raise RuntimeError(f"inside Plan.capture() nothing may be allocated: pass {what}=")
    return torch.empty(shape, dtype=dtype, device=device)


def _output(out, shape, dtype, device, what):
    """(tensor, row stride) of an output: new, or the caller's."""
    if out is None:
        return _new(shape, dtype, device, what), shape[-1]
    _tensor(out, what, device, dtype, shape)
    stride = _row_stride(out)
    if stride is None:
        raise ValueError(f"{what} must have contiguous rows at one stride")
    return out, stride


def _written(*tensors):
    """Tells autograd that the caller's own tensors have changed: gradients that need what was in them are then refused."""
    for t in tensors:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


@functools.lru_cache(maxsize=4096)
def _bytes_of(query, *args):
    """What a gl_*_workspace query says: a function of its arguments alone."""
    return _lib.check(getattr(_lib.lib(), query)(*args), query)


def _scratch(workspace, need, device, *others):
    """(workspace, its bytes): new, or the caller's, which none of the other tensors may reach into."""
    if need == 0:
        return None, 0
    if workspace is None:
        return _new((need,), torch.uint8, device, "workspace"), need
    if not isinstance(workspace, torch.Tensor) or workspace.dtype != torch.uint8 or workspace.device != device \
            or not workspace.is_contiguous() or workspace.numel() < need or workspace.data_ptr() % 16:
        raise ValueError(f"workspace must be a contiguous, 16-byte aligned uint8 tensor of at least {need} bytes on {device}")
    _apart(workspace, "workspace", [("an input or an output", t) for t in others])
    return workspace, workspace.numel()


_no_switch = contextlib.nullcontext()


def _on(device):
    """Makes `device` the current one for a launch (a no-op where it is)."""
    return _no_switch if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


_bound = False


def _plain():
    """_calls with the library's addresses, or None where it may not be used: inside Plan.capture() nothing is allocated."""
    global _bound
    if _calls is None or raw_capture_active():
        return None
    if not _bound:
        lib = _lib.lib()
        _calls.bind(torch._C._cuda_getCurrentRawStream, *(ctypes.cast(getattr(lib, f"gl_{name}{query}"), ctypes.c_void_p).value
                                                          for name in ("dense", "dense_backward", "group_norm", "group_norm_backward")
                                                          for query in ("_workspace", "")))
        _bound = True
    return _calls


def _needs_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and getattr(t, "requires_grad", False):
                return True
    return False


def _refuse_transforms(what, *tensors):
    """Refuses what would lose a derivative or the call itself without a word: tangents, and torch.jit.trace."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError(f"{what}() cannot be traced: torch.jit.trace would record its empty result alone")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what}() has no forward-mode derivative: an argument carries a tangent")


def _eager_only(device, what):
    with _on(device):
        capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        raise RuntimeError(f"the differentiable {what}() cannot be captured into a graph: capture {what}() without "
                           f"gradients and {what}_backward()")


# -- dense -----------------------------------------------------------------------------------------------------
def dense_workspace(rows, inputs, outputs, dtype=torch.float32, out_dtype=None):
    """Bytes of workspace :func:`dense` needs for (rows, inputs) @ (outputs, inputs).T."""
    out_dtype = dtype if out_dtype is None else out_dtype
    return _bytes_of("gl_dense_workspace", int(rows), int(inputs), int(outputs), _DTYPES[dtype], _DTYPES[out_dtype])


def dense_backward_workspace(rows, inputs, outputs, dtype=torch.float32, out_dtype=None, activation=None):
    """Bytes of workspace :func:`dense_backward` needs."""
    out_dtype = dtype if out_dtype is None else out_dtype
    return _bytes_of("gl_dense_backward_workspace", int(rows), int(inputs), int(outputs), _DTYPES[dtype],
                     _DTYPES[out_dtype], _activation(activation))


def _dense_args(x, weight, bias, residual, out_dtype):
    """(result's shape, its type, device) of checked arguments."""
    _tensor(x, "x")
    if x.dim() < 1 or not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("x must be (..., inputs) and weight (outputs, inputs)")
    dtype, device, width = x.dtype, x.device, weight.shape
    if out_dtype is None:
        out_dtype = dtype
    elif out_dtype is not dtype and out_dtype is not torch.float32:
        raise ValueError(f"out_dtype must be {dtype} or float32, got {out_dtype}")
    _tensor(weight, "weight", device, dtype, (width[0], x.shape[-1]))
    if width[0] == 0 or width[1] == 0:
        raise ValueError("weight has no elements")
    shape = x.shape[:-1] + width[:1]
    if bias is not None:
        _tensor(bias, "bias", device, dtype, width[:1])
    if residual is not None:
        _tensor(residual, "residual", device, out_dtype, shape)
    return shape, out_dtype, device


def _dense(x, weight, bias, act, residual, out_dtype, out, preactivation, workspace):
    shape, out_dtype, device = _dense_args(x, weight, bias, residual, out_dtype)
    y, y_stride = _output(out, shape, out_dtype, device, "out")
    z, z_stride = None, 0
    if preactivation is not None:
        z, z_stride = _output(preactivation, shape, out_dtype, device, "preactivation")
    if out is not None or z is not None:
        inputs = [("x", x), ("weight", weight), ("bias", bias), ("residual", residual)]
        if out is not None:
            _apart(y, "out", inputs, same=(residual,))
        if z is not None:
            _apart(z, "preactivation", inputs + [("out", y)])
    K, N = x.shape[-1], shape[-1]
    rows = x.numel() // K
    x, x_stride = _rows(x)
    weight, w_stride = _rows(weight)
    r_stride = 0
    if residual is not None:
        residual, r_stride = _rows(residual)
    if bias is not None:
        bias = _vector(bias)
    d, od = _DTYPES[x.dtype], _DTYPES[out_dtype]
    ws, ws_bytes = _scratch(workspace, _bytes_of("gl_dense_workspace", rows, K, N, d, od), device, x, weight, bias,
                            residual, y, z)
    with _on(device):
        _lib.check(_lib.lib().gl_dense(_p(x), x_stride, _p(weight), w_stride, _p(bias), _p(residual), r_stride, _p(y),
                                       y_stride, _p(z), z_stride, rows, K, N, d, od, act, _p(ws), ws_bytes,
                                       _stream(device)), "gl_dense")
    _written(out, preactivation)
    return y


class _Dense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, out_dtype):
        shape, out_dtype, device = _dense_args(x, weight, bias, residual, out_dtype)
        z = torch.empty(shape, dtype=out_dtype, device=device) if act else None
        calls = _plain()
        y = None if calls is None else calls.dense(x, weight, bias, residual, z, out_dtype, act)
        if y is None:
            y = _dense(x, weight, bias, act, residual, out_dtype, None, z, None)
        ctx.act = act
        ctx.save_for_backward(x, weight, z)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = _dense_backward(dy, x, weight, z, ctx.act, need[:3], (None, None, None), None)
        return dx, dw, db, (dy if need[3] else None), None, None


def dense(x, weight, bias=None, *, activation=None, residual=None, out_dtype=None, out=None, preactivation=None,
          workspace=None):
    """``act(x @ weight.T + bias) + residual`` in one kernel, rounded once (gl_dense).

    x: (..., inputs); weight: (outputs, inputs); bias: (outputs,); residual: (..., outputs).  x, weight and bias are of
    one type; residual and result of that type or float32 (``out_dtype``).  activation: None, 'relu', 'silu', 'gelu'
    (z * Phi(z)), 'tanh' or 'exp'.  out: receives the result (may be the residual).  preactivation: a tensor that
    receives the sum with the bias, which :func:`dense_backward` needs unless activation is None.  Differentiable in x,
    weight, bias and residual (without out= and preactivation=)."""
    act = _activation(activation)
    if out is None and workspace is None:
        calls = _plain()
        if calls is not None:
            y = calls.dense(x, weight, bias, residual, preactivation, out_dtype, act)
            if y is not None:
                return y
    _refuse_transforms("dense", x, weight, bias, residual)
    if _needs_grad(x, weight, bias, residual):
        if out is not None or preactivation is not None:
            raise ValueError("out= and preactivation= belong to the form without gradients: use torch.no_grad()")
        _eager_only(x.device, "dense")
        return _Dense.apply(x, weight, bias, residual, act, out_dtype)
    return _dense(x, weight, bias, act, residual, out_dtype, out, preactivation, workspace)


def _apart_from_all(outs, made, inputs, same=()):
    """_apart for the caller's own gradients; made, inputs: (name, tensor)."""
    for k, (name, t) in enumerate(made):
        if t is not None and any(o is t for o in outs):
            _apart(t, name, inputs + made[:k], same if k == 0 else ())


def _dense_backward(dy, x, weight, z, act, need, outs, workspace):
    if workspace is None and outs[0] is None and outs[1] is None and outs[2] is None:
        calls = _plain()
        if calls is not None:
            grads = calls.dense_backward(dy, x, weight, z, act, bool(need[0]), bool(need[1]), bool(need[2]))
            if grads is not None:
                return grads
    _refuse_transforms("dense_backward", dy, x, weight, z)
    _tensor(x, "x")
    if x.dim() < 1 or not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("x must be (..., inputs) and weight (outputs, inputs)")
    dtype, device, width = x.dtype, x.device, weight.shape
    N, K = width
    _tensor(weight, "weight", device, dtype, (N, x.shape[-1]))
    if N == 0 or K == 0:
        raise ValueError("weight has no elements")
    shape = x.shape[:-1] + width[:1]
    dy_dtype = torch.float32 if isinstance(dy, torch.Tensor) and dy.dtype is torch.float32 else dtype
    _tensor(dy, "dy", device, dy_dtype, shape)
    z_stride = dx_stride = dw_stride = 0
    if act:
        if z is None:
            raise ValueError("dense_backward needs the preactivation of an activation's forward pass")
        _tensor(z, "preactivation", device, dy_dtype, shape)
    else:
        z = None
    dx = dw = db = None
    if need[0]:
        dx, dx_stride = _output(outs[0], x.shape, dtype, device, "dx")
    if need[1]:
        dw, dw_stride = _output(outs[1], width, dtype, device, "dweight")
    if need[2]:
        db, _ = _output(outs[2], width[:1], dtype, device, "dbias")
    if outs[0] is not None or outs[1] is not None or outs[2] is not None:
        _apart_from_all(outs, [("dx", dx), ("dweight", dw), ("dbias", db)],
                        [("dy", dy), ("x", x), ("weight", weight), ("preactivation", z)])
    if not any(need):
        return dx, dw, db
    rows = x.numel() // K
    dy, dy_stride = _rows(dy)
    x, x_stride = _rows(x)
    weight, w_stride = _rows(weight)
    if z is not None:
        z, z_stride = _rows(z)
    d, od = _DTYPES[dtype], _DTYPES[dy_dtype]
    ws, ws_bytes = _scratch(workspace, _bytes_of("gl_dense_backward_workspace", rows, K, N, d, od, act), device, dy, x,
                            weight, z, dx, dw, db)
    with _on(device):
        _lib.check(_lib.lib().gl_dense_backward(_p(dy), dy_stride, _p(x), x_stride, _p(weight), w_stride, _p(z), z_stride,
                                                _p(dx), dx_stride, _p(dw), dw_stride, _p(db), rows, K, N, d, od, act,
                                                _p(ws), ws_bytes, _stream(device)), "gl_dense_backward")
    _written(*outs)
    return dx, dw, db


def dense_backward(dy, x, weight, preactivation=None, *, activation=None, needs=(True, True, True), dx=None, dweight=None,
                   dbias=None, workspace=None):
    """Gradients (dx, dweight, dbias) of :func:`dense` (gl_dense_backward); the residual's gradient is dy itself.

    dy, preactivation: (..., outputs), of dense's result type.  dz = dy * act'(preactivation) goes into the products rounded to
    bfloat16 where dy is bfloat16, in two planes (2^-17 of it) where float32 dy meets 16-bit weights, and in float16 in two planes
    that reach far below the type's range: gradients too small for float16 count in sums over frames.  needs: which of the
    three are wanted (None comes back for the others).  dx, dweight, dbias: tensors that receive them."""
    return _dense_backward(dy, x, weight, preactivation, _activation(activation), needs, (dx, dweight, dbias), workspace)


# -- group norm ------------------------------------------------------------------------------------------------
def group_norm_workspace(batch, frames, channels, groups, dtype=torch.float32):
    """Bytes of workspace :func:`group_norm` needs."""
    return _bytes_of("gl_group_norm_workspace", int(batch), int(frames), int(channels), int(groups), _DTYPES[dtype])


def group_norm_backward_workspace(batch, frames, channels, groups, dtype=torch.float32):
    """Bytes of workspace :func:`group_norm_backward` needs."""
    return _bytes_of("gl_group_norm_backward_workspace", int(batch), int(frames), int(channels), int(groups),
                     _DTYPES[dtype])


def _norm_args(x, groups, weight, bias, lengths):
    _tensor(x, "x")
    if x.dim() not in (2, 3) or x.shape[-1] < 1:
        raise ValueError("x must be (B, T, channels) or (T, channels)")
    groups = int(groups)
    C = x.shape[-1]
    if groups < 1 or C % groups:
        raise ValueError(f"{C} channels do not divide into {groups} groups")
    if weight is not None:
        _tensor(weight, "weight", x.device, x.dtype, (C,))
    if bias is not None:
        _tensor(bias, "bias", x.device, x.dtype, (C,))
    B, T = (1, x.shape[0]) if x.dim() == 2 else x.shape[:2]
    lens = None
    if lengths is not None:
        if raw_capture_active() and not (isinstance(lengths, torch.Tensor) and lengths.device == x.device
                                         and lengths.dtype == torch.int32 and lengths.is_contiguous()):
            raise RuntimeError("inside Plan.capture() lengths must be a contiguous int32 tensor on the device")
        lens = lengths
        if not (isinstance(lens, torch.Tensor) and lens.dtype == torch.int32 and lens.device == x.device
                and lens.is_contiguous()):
            lens = torch.as_tensor(lengths, dtype=torch.int32).to(x.device).contiguous()
        if lens.shape != (B,):
            raise ValueError(f"lengths must have shape ({B},)")
    return groups, B, T, C, lens


def _group_norm(x, groups, weight, bias, eps, act, lengths, out, stats, workspace):
    groups, B, T, C, lens = _norm_args(x, groups, weight, bias, lengths)
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    device, dtype = x.device, x.dtype
    y, y_stride = _output(out, x.shape, dtype, device, "out")
    if out is not None or stats is not None:
        inputs = [("weight", weight), ("bias", bias), ("lengths", lens)]
        if out is not None:
            _apart(y, "out", inputs + [("x", x)], same=(x,))
        if stats is not None:
            _tensor(stats, "stats", device, torch.float32, (B, groups, 2))
            if not stats.is_contiguous():
                raise ValueError("stats must be contiguous")
            _apart(stats, "stats", inputs + [("x", x), ("out", y)])
    x, x_stride = _rows(x)
    if weight is not None:
        weight = _vector(weight)
    if bias is not None:
        bias = _vector(bias)
    d = _DTYPES[dtype]
    ws, ws_bytes = _scratch(workspace, _bytes_of("gl_group_norm_workspace", B, T, C, groups, d), device, x, weight,
                            bias, lens, y, stats)
    with _on(device):
        _lib.check(_lib.lib().gl_group_norm(_p(x), x_stride, _p(weight), _p(bias), _p(lens), _p(y), y_stride, _p(stats), B,
                                            T, C, groups, d, act, eps, _p(ws), ws_bytes, _stream(device)),
                   "gl_group_norm")
    _written(out, stats)
    return y


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, lengths):
        groups, B, T, C, lens = _norm_args(x, groups, weight, bias, lengths)
        stats = torch.empty((B, groups, 2), dtype=torch.float32, device=x.device)
        calls = _plain()
        y = None if calls is None else calls.group_norm(x, weight, bias, lens, stats, groups, act, eps)
        if y is None:
            y = _group_norm(x, groups, weight, bias, eps, act, lens, None, stats, None)
        ctx.groups, ctx.act = groups, act
        ctx.save_for_backward(x, weight, bias, stats, lens)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats, lens = ctx.saved_tensors
        dx, dw, db = _group_norm_backward(dy, x, ctx.groups, stats, weight, bias, ctx.act, lens, ctx.needs_input_grad[:3],
                                          (None, None, None), None)
        return dx, dw, db, None, None, None, None


def group_norm(x, groups, weight=None, bias=None, *, eps=1e-5, activation=None, lengths=None, out=None, stats=None,
               workspace=None):
    """``act(groupnorm(x) * weight + bias)`` of x (B, T, channels), channels last (gl_group_norm).

    Mean and variance of every utterance and group of channels, over the frames t < lengths[b] (None: all of them; a
    list or an int32 tensor).  Frames past an utterance's end are not read and come out as zeros.  weight, bias:
    (channels,) of x's type, or None.  out: receives the result (may be x).  stats: (B, groups, 2) float32 tensor that
    receives mean and 1 / sqrt(var + eps) for :func:`group_norm_backward`.  Differentiable in x, weight and bias
    (without out= and stats=)."""
    act = _activation(activation)
    if out is None and workspace is None:
        calls = _plain()
        if calls is not None:
            y = calls.group_norm(x, weight, bias, lengths, stats, int(groups), act, eps)
            if y is not None:
                return y
    _refuse_transforms("group_norm", x, weight, bias)
    if _needs_grad(x, weight, bias):
        if out is not None or stats is not None:
            raise ValueError("out= and stats= belong to the form without gradients: use torch.no_grad()")
        _eager_only(x.device, "group_norm")
        return _GroupNorm.apply(x, weight, bias, groups, eps, act, lengths)
    return _group_norm(x, groups, weight, bias, eps, act, lengths, out, stats, workspace)


def _group_norm_backward(dy, x, groups, stats, weight, bias, act, lengths, need, outs, workspace):
    if workspace is None and outs[0] is None and outs[1] is None and outs[2] is None:
        calls = _plain()
        if calls is not None:
            grads = calls.group_norm_backward(dy, x, stats, weight, bias, lengths, int(groups), act, bool(need[0]), bool(need[1]),
                                              bool(need[2]))
            if grads is not None:
                return grads
    _refuse_transforms("group_norm_backward", dy, x, stats, weight, bias)
    groups, B, T, C, lens = _norm_args(x, groups, weight, bias, lengths)
    device, dtype = x.device, x.dtype
    _tensor(dy, "dy", device, dtype, x.shape)
    _tensor(stats, "stats", device, torch.float32, (B, groups, 2))
    stats = _vector(stats)
    dx = dg = db = None
    dx_stride = 0
    if need[0]:
        dx, dx_stride = _output(outs[0], x.shape, dtype, device, "dx")
    if need[1] and weight is not None:
        dg, _ = _output(outs[1], (C,), dtype, device, "dweight")
    if need[2] and bias is not None:
        db, _ = _output(outs[2], (C,), dtype, device, "dbias")
    if outs[0] is not None or outs[1] is not None or outs[2] is not None:
        _apart_from_all(outs, [("dx", dx), ("dweight", dg), ("dbias", db)],
                        [("x", x), ("stats", stats), ("weight", weight), ("bias", bias), ("lengths", lens), ("dy", dy)], (dy,))
    if dx is None and dg is None and db is None:
        return dx, dg, db
    dy, dy_stride = _rows(dy)
    x, x_stride = _rows(x)
    if weight is not None:
        weight = _vector(weight)
    if bias is not None:
        bias = _vector(bias)
    d = _DTYPES[dtype]
    ws, ws_bytes = _scratch(workspace, _bytes_of("gl_group_norm_backward_workspace", B, T, C, groups, d), device, dy, x, stats,
                            weight, bias, lens, dx, dg, db)
    with _on(device):
        _lib.check(_lib.lib().gl_group_norm_backward(_p(dy), dy_stride, _p(x), x_stride, _p(stats), _p(weight), _p(bias),
                                                     _p(lens), _p(dx), dx_stride, _p(dg), _p(db), B, T, C, groups, d, act,
                                                     _p(ws), ws_bytes, _stream(device)), "gl_group_norm_backward")
    _written(*outs)
    return dx, dg, db


def group_norm_backward(dy, x, groups, stats, weight=None, bias=None, *, activation=None, lengths=None,
                        needs=(True, True, True), dx=None, dweight=None, dbias=None, workspace=None):
    """Gradients (dx, dweight, dbias) of :func:`group_norm` from its input and stats (gl_group_norm_backward).

    dx is zero in frames past an utterance's end and may be dy.  dweight / dbias are None where weight / bias is."""
    return _group_norm_backward(dy, x, groups, stats, weight, bias, _activation(activation), lengths, needs,
                                (dx, dweight, dbias), workspace)


# -- the network -----------------------------------------------------------------------------------------------
class MelInversion(torch.nn.Module):
    """Log-mel frames (B, T, n_mels) -> linear magnitudes (B, T, n_bins), float32 and positive.

        h = dense(logmel)
        h = h + dense(gelu dense(silu group_norm(h)))        `blocks` times, `hidden` wide inside
        mag = exp dense(silu group_norm(h))

    Parameters are of `dtype`; log-mels of another type are cast to it.  lengths (ragged batch): frames past an
    utterance's end do not reach the norms of the others; their magnitudes are for the caller to ignore
    (``logmel_to_audio`` zeroes them).  float16: the gradients between layers are float16 too and vanish below 6e-8, so scale the
    loss (a mean over a batch's magnitudes by some 2**14) and divide the parameters' gradients; float32 and bfloat16 need none.
    A freshly made network starts at magnitudes around exp(out_bias)."""

    def __init__(self, n_mels=80, n_bins=1025, channels=512, hidden=None, blocks=2, groups=32, dtype=torch.float32,
                 device=None, seed=0, out_bias=-3.0):
        super().__init__()
        hidden = 4 * channels if hidden is None else int(hidden)
        if min(n_mels, n_bins, channels, hidden, groups) < 1 or blocks < 0 or channels % groups:
            raise ValueError("widths must be positive and channels a multiple of groups")
        if dtype not in _DTYPES:
            raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
        self.n_mels, self.n_bins, self.groups = int(n_mels), int(n_bins), int(groups)
        g = torch.Generator().manual_seed(int(seed))

        def weight(n, k, gain=1.0):
            return torch.nn.Parameter((torch.randn((n, k), generator=g) * (gain * k ** -0.5)).to(dtype).to(device))

        def vector(n, value):
            return torch.nn.Parameter(torch.full((n,), float(value), dtype=dtype, device=device))

        self.w_in, self.b_in = weight(channels, n_mels), vector(channels, 0)
        self.norm_w = torch.nn.ParameterList([vector(channels, 1) for _ in range(blocks + 1)])
        self.norm_b = torch.nn.ParameterList([vector(channels, 0) for _ in range(blocks + 1)])
        self.w_up = torch.nn.ParameterList([weight(hidden, channels) for _ in range(blocks)])
        self.b_up = torch.nn.ParameterList([vector(hidden, 0) for _ in range(blocks)])
        self.w_down = torch.nn.ParameterList([weight(channels, hidden, 0.5) for _ in range(blocks)])
        self.b_down = torch.nn.ParameterList([vector(channels, 0) for _ in range(blocks)])
        self.w_out, self.b_out = weight(n_bins, channels, 0.1), vector(n_bins, out_bias)

    def forward(self, logmel, lengths=None):
        single = logmel.dim() == 2
        if single:
            logmel = logmel[None]
        if logmel.dim() != 3 or logmel.shape[-1] != self.n_mels:
            raise ValueError(f"logmel must be (T, {self.n_mels}) or (B, T, {self.n_mels}), got {tuple(logmel.shape)}")
        if lengths is not None:
            lengths = torch.as_tensor(lengths, dtype=torch.int32).to(self.w_in.device)
        h = dense(logmel.to(self.w_in.dtype), self.w_in, self.b_in)
        for k in range(len(self.w_up)):
            u = group_norm(h, self.groups, self.norm_w[k], self.norm_b[k], activation="silu", lengths=lengths)
            u = dense(u, self.w_up[k], self.b_up[k], activation="gelu")
            h = dense(u, self.w_down[k], self.b_down[k], residual=h)
        u = group_norm(h, self.groups, self.norm_w[-1], self.norm_b[-1], activation="silu", lengths=lengths)
        mag = dense(u, self.w_out, self.b_out, activation="exp", out_dtype=torch.float32)
        return mag[0] if single else mag
