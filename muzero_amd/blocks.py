"""Operators of residual feed-forward blocks on this library's HIP kernels, for training and inference: layer norm, the
gated feed-forward projection and dropout.  They stand beside the learner's BatchNorm + ReLU blocks and convolutions
(``muzero_amd.learner``) for trunks and heads whose batches batch statistics do not suit - one state at a time, games of
unequal length.  The reference has no counterpart.

    y = x + dropout(linear(gated_ff(layer_norm(x, w, b), w_gate, w_up)), p, rng)

    h = blocks.gated_ff(blocks.layer_norm(x, w, b), w_gate, w_up)
    y = blocks.dropout(F.linear(h, w_down), p, rng, residual=x)

All take CUDA tensors of any leading shape (the last dimension is the operator's), in bfloat16, float16 or float32,
accumulate in float32, run on the tensors' device and that device's current stream, allocate their outputs and scratch
with torch's allocator per call (so they can be recorded into HIP graphs) and are differentiable once, in reverse mode.
Wrong types, shapes or devices raise ValueError; there is no CPU path.  While a backward pass is being recorded into a HIP
graph, no eager autograd graph of the same parameters may be alive (as for any torch operator).
"""
import ctypes as C
from typing import Optional

import torch

from . import _lib

_ext = None


def _load():
    """The native module (csrc/blocks_torch.cpp), bound to the entry points of the library that _lib has loaded."""
    global _ext
    handle = _lib.lib()
    try:
        from . import _blocks
    except ImportError as e:
        raise _lib.MuZeroAmdError(f"muzero_amd._blocks not found: build it with `make -C muzero_amd/csrc` ({e})") from e
    names = ("mz_last_error", "mz_layer_norm_fwd", "mz_layer_norm_workspace_bytes", "mz_layer_norm_bwd",
             "mz_gated_ff_workspace_bytes", "mz_gated_ff_fwd", "mz_gated_ff_bwd", "mz_dropout")
    _blocks.bind({n: C.cast(getattr(handle, n), C.c_void_p).value for n in names}, _lib.MuZeroAmdError)
    _ext = _blocks
    return _ext


def layer_norm(x, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, the biased variance, statistics in float32.

    x: [..., C], C up to 2^24; weight, bias: [C] or None, both float32 or both x's dtype.  Returns x's shape and dtype;
    gradients for x, weight and bias.  Rows that lie apart in memory (a slice of wider rows) are read in place."""
    return (_ext or _load()).layer_norm(x, weight, bias, eps)


def gated_ff(x, w_gate, w_up, b_gate: Optional[torch.Tensor] = None, b_up: Optional[torch.Tensor] = None,
             activation: str = "silu"):
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up) in one kernel - the first half of a gated feed-forward block.

    x: [..., K]; w_gate, w_up: [F, K]; b_gate, b_up: [F] or None; K and F up to 2^20, all of one dtype (under
    ``torch.autocast`` they are cast to its dtype first, as torch's linear does).  activation: "silu", "gelu" (erf),
    "relu" or "sigmoid".  Returns [..., F].  The backward pass computes the two products again from x: nothing of the
    hidden width is kept but the result; while it runs it takes scratch of twice the result's size and for the partial
    results of sums that are cut over workgroups.  How they are cut goes by the sizes and by whether x and the weights both want
    gradients: the last bits of one that is asked for alone may differ from those it has beside the other.  In bfloat16 and float16 it rounds the two products' gradients to that
    type, matrix operands as they are next: gradients of x and the weights are then off by sqrt(2) times what rounding the
    result alone costs (relative RMS 2.4e-3 in bfloat16, 2.9e-4 in float16), at any size.  Small problems - rows x F up to
    8192 and K x F up to 2^21 - carry what that rounding left along and are off by the result's rounding alone.
    float16 gradients below 6e-5 lose digits and those above 65504 overflow as any float16 value does - scale the loss."""
    return (_ext or _load()).gated_ff(x, w_gate, w_up, b_gate, b_up, activation)


def dropout(x, p: float, rng: torch.Tensor, call: int = 0, residual: Optional[torch.Tensor] = None):
    """[residual +] x with elements dropped with probability p and the others divided by 1 - p.

    Which elements go is a function of (seed, offset, call, element index in x's logical order) - Philox4x32-10 - and is
    never stored: the backward pass computes it again.  rng: int64 tensor [2] = (seed, offset) on x's device, read when
    the kernel runs, so a program recorded into a HIP graph draws a new mask when it has changed rng between replays;
    ``call`` (0 .. 2^32 - 1) tells the dropouts of one step apart.  rng must not change between a forward pass and its
    backward pass (autograd raises if it did).  p in [0, 1] is rounded to a multiple of 2^-16 and the scale is that
    value's.  A dropped element counts as zero whatever x holds there.  residual: x's shape and dtype."""
    return (_ext or _load()).dropout(x, p, rng, call, residual)
