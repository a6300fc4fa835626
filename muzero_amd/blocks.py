"""Operators of residual feed-forward blocks on this library's HIP kernels, for training and inference: layer norm, the
gated feed-forward projection and dropout.  They stand beside the learner's BatchNorm + ReLU blocks and convolutions
(``muzero_amd.learner``) for trunks and heads whose batches batch statistics do not suit - one state at a time, games of
unequal length.  The reference has no counterpart.

    y = x + dropout(linear(gated_ff(layer_norm(x, w, b), w_gate, w_up)), p, rng)

    h = blocks.gated_ff(blocks.layer_norm(x, w, b), w_gate, w_up)
    y = blocks.dropout(F.linear(h, w_down), p, rng, residual=x)

All take CUDA tensors of any leading shape (the last dimension is the operator's), in bfloat16, float16 or float32,
accumulate in float32, run on the tensors' device and that device's current stream, allocate their outputs and scratch
with torch's allocator per call (so they can be recorded into HIP graphs) and are differentiable once.  Wrong types,
shapes or devices raise ValueError; there is no CPU path.
"""
from typing import Optional

import torch
from torch._C import _cuda_getCurrentRawStream as _raw_stream
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}          # MZ_F32, MZ_BF16, MZ_F16
_ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}
_MAX_COLS = 1 << 24          # columns of layer norm
_MAX_WIDTH = 1 << 20         # input and hidden width of the gated projection
_MAX_STRIDE_BYTES = 1 << 22  # between rows of its input


# The host's part of a call counts: a small training step is a handful of launches, and its backward pass runs on
# autograd's own thread, where every Python operation costs several times what it does in a warm loop.  So entry points
# are looked up once, the stream is read as a plain handle, and nothing is allocated, cast or copied that is there.
_ENTRIES = {}


def _entry(name):
    f = _ENTRIES[name] = getattr(_lib.lib(), name)
    return f


def _run(index, name, *args):
    """Call an entry point on device `index` and its current stream."""
    f = _ENTRIES.get(name) or _entry(name)
    if torch.cuda.current_device() == index:
        rc = f(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _raw_stream(index))
    if rc:
        _lib.fail(name, rc)


def _bytes(name, *args):
    return (_ENTRIES.get(name) or _entry(name))(*args)


def _once(backward):
    """once_differentiable, whose bookkeeping is only needed where a gradient's gradient may be asked for."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


def _like(x):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _checked(x, name):
    """An activation: a CUDA tensor of one of the element types with a last dimension."""
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"{name}: tensor required")
    if not x.is_cuda:
        raise ValueError(f"{name}: must live on the GPU")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name}: dtype {x.dtype}, expected float32, bfloat16 or float16")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{name}: shape {tuple(x.shape)}, expected a last dimension of at least 1")
    return x


def _param(t, name, shape, like, dtypes):
    """Refuse a parameter that is not of the given shape, on the activations' device and of one of the types."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: tensor required")
    if t.device != like.device:
        raise ValueError(f"{name}: on {t.device}, expected {like.device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {' or '.join(str(d) for d in dict.fromkeys(dtypes))}")
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")


def _rows(x):
    """(tensor, elements between rows): x as rows of its last dimension.  Rows may lie apart (a slice of wider rows);
    anything a row stride cannot describe is copied."""
    if x.is_contiguous():
        return x, x.shape[-1]
    x2 = x.reshape(-1, x.shape[-1])
    if (x2.shape[1] > 1 and x2.stride(1) != 1) or (x2.shape[0] > 1 and x2.stride(0) < x2.shape[1]):
        x2 = x2.contiguous()
    return x2, (x2.stride(0) if x2.shape[0] > 1 else x2.shape[1])


def _contiguous(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _address(t):
    return None if t is None else t.data_ptr()


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------------------------------------------- layer norm
def _layer_norm_forward(x, weight, bias, eps, keep):
    xr, ld = _rows(x)
    c = x.shape[-1]
    rows = x.numel() // c
    y = _like(x)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if keep else None
    if rows:
        weight, bias = _contiguous(weight), _contiguous(bias)
        affine = weight if weight is not None else bias
        mean = stats.data_ptr() if keep else None
        _run(x.device.index, "mz_layer_norm_fwd", xr.data_ptr(), ld, _address(weight), _address(bias),
             0 if affine is None else _DTYPES[affine.dtype], eps, rows, c, _DTYPES[x.dtype], y.data_ptr(), mean,
             mean + 4 * rows if keep else None)
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _layer_norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.affine = torch.float32 if weight is None and bias is None else (weight if weight is not None else bias).dtype
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        want_x, want_w, want_b, _ = ctx.needs_input_grad
        c = x.shape[-1]
        rows = x.numel() // c
        device, affine = x.device, ctx.affine
        dx = _like(x) if want_x else None
        fresh = torch.empty if rows else torch.zeros
        dw = fresh(c, dtype=affine, device=device) if want_w else None
        db = fresh(c, dtype=affine, device=device) if want_b else None
        if rows:
            if dy.dtype != x.dtype:
                dy = dy.to(x.dtype)
            (xr, ldx), (gr, ldg) = _rows(x), _rows(dy)
            need = _bytes("mz_layer_norm_workspace_bytes", rows, c) if want_w or want_b else 0
            ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
            mean = stats.data_ptr()
            weight = _contiguous(weight)
            _run(device.index, "mz_layer_norm_bwd", xr.data_ptr(), ldx, gr.data_ptr(), ldg, _address(weight),
                 _DTYPES[affine], mean, mean + 4 * rows, rows, c, _DTYPES[x.dtype], _address(dx), _address(dw), _address(db),
                 _address(ws), need)
        return dx, dw, db, None


def layer_norm(x, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, the biased variance, statistics in float32.

    x: [..., C], C up to 2^24; weight, bias: [C] or None, both float32 or both x's dtype.  Returns x's shape and dtype;
    gradients for x, weight and bias.  Rows that lie apart in memory (a slice of wider rows) are read in place."""
    _checked(x, "layer_norm: x")
    if x.shape[-1] > _MAX_COLS:
        raise ValueError(f"layer_norm: x: at most {_MAX_COLS} columns")
    if weight is not None:
        _param(weight, "layer_norm: weight", x.shape[-1:], x, (torch.float32, x.dtype))
    if bias is not None:
        _param(bias, "layer_norm: bias", x.shape[-1:], x, (torch.float32, x.dtype) if weight is None else (weight.dtype,))
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps {eps}, expected at least 0")
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _layer_norm_forward(x, weight, bias, float(eps), False)[0]


# ------------------------------------------------------------------------------------------- gated feed-forward
def _ff_rows(x):
    """_rows for the matrix kernels: where a row is whole 16-byte units, rows have to start on 16 bytes, and rows lie at
    most 4 MiB apart; what does not is copied."""
    xr, ld = _rows(x)
    size = x.element_size()
    aligned = xr.data_ptr() % 16 == 0 and ld * size % 16 == 0
    if ld * size > _MAX_STRIDE_BYTES or (not aligned and x.shape[-1] * size % 16 == 0):
        xr = xr.clone(memory_format=torch.contiguous_format)
        ld = x.shape[-1]
    return xr, ld


def _ff_weight(w):
    w = _contiguous(w)
    return w.clone() if w.data_ptr() % 16 else w


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _gated_ff_forward(x, w_gate, w_up, b_gate, b_up, activation):
    xr, ld = _ff_rows(x)
    hidden, k = w_gate.shape
    rows = x.numel() // k
    device = x.device
    h = torch.empty(x.shape[:-1] + (hidden,), dtype=x.dtype, device=device)
    if rows:
        w_gate, w_up, b_gate, b_up = _ff_weight(w_gate), _ff_weight(w_up), _contiguous(b_gate), _contiguous(b_up)
        dt = _DTYPES[x.dtype]
        need = _bytes("mz_gated_ff_workspace_bytes", rows, k, hidden, dt, 0)
        ws = _workspace(need, device)
        _run(device.index, "mz_gated_ff_fwd", xr.data_ptr(), ld, w_gate.data_ptr(), w_up.data_ptr(), _address(b_gate),
             _address(b_up), rows, k, hidden, dt, activation, h.data_ptr(), _address(ws), need)
    return h


class _GatedFF(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, activation):
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up)
        ctx.activation = activation
        return _gated_ff_forward(x, w_gate, w_up, b_gate, b_up, activation)

    @staticmethod
    @_once
    def backward(ctx, dh):
        x, w_gate, w_up, b_gate, b_up = ctx.saved_tensors
        hidden, k = w_gate.shape
        rows = x.numel() // k
        want_x, want_g, want_u, want_bg, want_bu, _ = ctx.needs_input_grad
        dtype, device = x.dtype, x.device
        make = torch.empty if rows else torch.zeros
        both = want_g or want_u              # one kernel makes the two weights' gradients
        dx = _like(x) if want_x else None
        dwg = make((hidden, k), dtype=dtype, device=device) if both else None
        dwu = make((hidden, k), dtype=dtype, device=device) if both else None
        dbg = make(hidden, dtype=dtype, device=device) if want_bg else None
        dbu = make(hidden, dtype=dtype, device=device) if want_bu else None
        if rows:
            xr, ld = _ff_rows(x)
            w_gate, w_up, b_gate, b_up = _ff_weight(w_gate), _ff_weight(w_up), _contiguous(b_gate), _contiguous(b_up)
            dt = _DTYPES[dtype]
            if dh.dtype != dtype:
                dh = dh.to(dtype)
            dh = _contiguous(dh)
            need = _bytes("mz_gated_ff_workspace_bytes", rows, k, hidden, dt, 1)
            ws = _workspace(need, device)
            _run(device.index, "mz_gated_ff_bwd", xr.data_ptr(), ld, w_gate.data_ptr(), w_up.data_ptr(), _address(b_gate),
                 _address(b_up), dh.data_ptr(), rows, k, hidden, dt, ctx.activation, _address(dx), _address(dwg),
                 _address(dwu), _address(dbg), _address(dbu), _address(ws), need)
        return dx, dwg if want_g else None, dwu if want_u else None, dbg, dbu, None


def gated_ff(x, w_gate, w_up, b_gate: Optional[torch.Tensor] = None, b_up: Optional[torch.Tensor] = None,
             activation: str = "silu"):
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up) in one kernel - the first half of a gated feed-forward block.

    x: [..., K]; w_gate, w_up: [F, K]; b_gate, b_up: [F] or None; K and F up to 2^20, all of one dtype (under
    ``torch.autocast`` they are cast to its dtype first, as torch's linear does).  activation: "silu", "gelu" (erf),
    "relu" or "sigmoid".  Returns [..., F].  The backward pass computes the two products again from x: nothing of the
    hidden width is kept but the result.  In bfloat16 and float16 it rounds the products' gradients to that type
    (they are matrix operands next); float16 gradients below 6e-5 lose digits as any float16 value does - scale the
    loss."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"gated_ff: activation {activation!r}, expected one of {', '.join(_ACTIVATIONS)}")
    if torch.is_autocast_enabled():
        t = torch.get_autocast_dtype("cuda")
        x, w_gate, w_up, b_gate, b_up = (v.to(t) if isinstance(v, torch.Tensor) and v.is_cuda and v.is_floating_point() else v
                                         for v in (x, w_gate, w_up, b_gate, b_up))
    _checked(x, "gated_ff: x")
    if not isinstance(w_gate, torch.Tensor) or w_gate.dim() != 2 or w_gate.shape[0] == 0:
        raise ValueError("gated_ff: w_gate: [F, K] tensor with F of at least 1 expected")
    hidden, k = w_gate.shape[0], x.shape[-1]
    if k > _MAX_WIDTH or hidden > _MAX_WIDTH:
        raise ValueError(f"gated_ff: widths {k} and {hidden}, expected at most {_MAX_WIDTH}")
    types = (x.dtype,)
    _param(w_gate, "gated_ff: w_gate", (hidden, k), x, types)
    _param(w_up, "gated_ff: w_up", (hidden, k), x, types)
    if b_gate is not None:
        _param(b_gate, "gated_ff: b_gate", (hidden,), x, types)
    if b_up is not None:
        _param(b_up, "gated_ff: b_up", (hidden,), x, types)
    kind = _ACTIVATIONS[activation]
    if _wants_grad(x, w_gate, w_up, b_gate, b_up):
        return _GatedFF.apply(x, w_gate, w_up, b_gate, b_up, kind)
    return _gated_ff_forward(x, w_gate, w_up, b_gate, b_up, kind)


# ---------------------------------------------------------------------------------------------------------- dropout
def _dropout_forward(x, residual, p, rng, call):
    x, residual = _contiguous(x), _contiguous(residual)
    y = torch.empty_like(x)
    n = x.numel()
    if n:
        _run(x.device.index, "mz_dropout", x.data_ptr(), _address(residual), y.data_ptr(), n, p, rng.data_ptr(), call,
             _DTYPES[x.dtype])
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng, call):
        ctx.save_for_backward(rng)
        ctx.p, ctx.call = p, call
        return _dropout_forward(x, residual, p, rng, call)

    @staticmethod
    @_once
    def backward(ctx, dy):
        (rng,) = ctx.saved_tensors
        want_x, want_residual, _, _, _ = ctx.needs_input_grad
        dx = _dropout_forward(dy, None, ctx.p, rng, ctx.call) if want_x else None
        return dx, dy if want_residual else None, None, None, None


def dropout(x, p: float, rng: torch.Tensor, call: int = 0, residual: Optional[torch.Tensor] = None):
    """[residual +] x with elements dropped with probability p and the others divided by 1 - p.

    Which elements go is a function of (seed, offset, call, element index in x's logical order) - Philox4x32-10 - and is
    never stored: the backward pass computes it again.  rng: int64 tensor [2] = (seed, offset) on x's device, read when
    the kernel runs, so a program recorded into a HIP graph draws a new mask when it has changed rng between replays;
    ``call`` (0 .. 2^32 - 1) tells the dropouts of one step apart.  rng must not change between a forward pass and its
    backward pass (autograd raises if it did).  p in [0, 1] is rounded to a multiple of 2^-16 and the scale is that
    value's.  A dropped element counts as zero whatever x holds there.  residual: x's shape and dtype."""
    _checked(x, "dropout: x")
    if x.numel() > 1 << 35:
        raise ValueError("dropout: x: at most 2^35 elements")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: p {p}, expected 0 to 1")
    if not 0 <= call < 1 << 32:
        raise ValueError(f"dropout: call {call}, expected 0 to 2^32 - 1")
    _param(rng, "dropout: rng", (2,), x, (torch.int64,))
    if not rng.is_contiguous():
        raise ValueError("dropout: rng: must be contiguous")
    if residual is not None:
        _param(residual, "dropout: residual", x.shape, x, (x.dtype,))
    if _wants_grad(x, residual):
        return _Dropout.apply(x, residual, float(p), rng, int(call))
    return _dropout_forward(x, residual, float(p), rng, int(call))
