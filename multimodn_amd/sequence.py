"""Operators that turn a sequence - coded events, tokens, a time series - into features an encoder of the fusion chain can take,
as hand-written HIP kernels (include/mmn_sequence.h): embedding lookup and its gradient, the short causal depthwise convolution, the
selective scan, and the last two for one new step on a kept state.

    embedding, causal_conv, selective_scan          differentiable; what a module's forward calls
    embedding_grad, causal_conv_grad,
    selective_scan_forward + selective_scan_grad    the same passes without autograd, for a caller that keeps its own order
    causal_conv_step, selective_scan_step           one new step for every row; the state moves on in place (no gradient)

Data is float32, bfloat16 or float16, all of one call alike; parameters (`weight`, `bias`, `a`, `d`, `dt_bias`, not the embedding's
table) and the scan's states are float32, and so are all sums inside.  Tensors are [batch, steps, width] with adjacent channels and
any other strides (anything else is copied); results are dense.  `lengths` ([batch], whole numbers) says how many steps of each row
count: what stands behind them is not read, gives 0 and leaves the states as they are.  Results do not change from run to run.

Everything runs on the current stream of the tensors' device, may be captured into a graph (with autograd: once no graph made on another
stream holds the tensors, or the leaves they come from, any more; refused before), and has no CPU or torch-op fallback: off an AMD GPU
these functions raise.  The reference has no counterpart: its recurrent encoders (multimodn/encoders/rnn_encoder.py,
lstm_encoder.py) are torch modules.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from . import hip

MAX_STATES = 32
MAX_TAPS = 4


def _native():
    """The checks and the calls (csrc/binding.cpp)."""
    return hip.load_binding()


def _any_grad(*tensors: Optional[Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _check_capture(*tensors: Optional[Tensor]) -> None:
    """Refuses to record for autograd, inside a graph capture, on what a graph made outside it holds."""
    if tensors[0].is_cuda and torch.cuda.is_current_stream_capturing() and _native().made_elsewhere(tensors):
        raise hip.MmnError("an autograd graph made outside this capture, on another stream, holds these tensors or leaves they come from: drop its "
                           "outputs and losses first (the captured backward pass would go on to that stream), or call under torch.no_grad()")


# ---------------------------------------------------------------------------------------------------------------- embedding
class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale):
        _check_capture(weight)
        ctx.save_for_backward(ids)
        ctx.vocab, ctx.scale = weight.shape[0], scale
        return _native().embed(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        return None, embedding_grad(grad, ids, ctx.vocab, ctx.scale), None


def embedding(ids: Tensor, weight: Tensor, scale: float = 1.0) -> Tensor:
    """scale * weight[ids], [*ids.shape, width] in the table's type.  An id outside [0, vocabulary) - by convention -1 - stands for "no
    token": its output is 0 and it has no part in the gradient.  The gradient sums each table row's contributions in the order of
    their positions, from sorted ids."""
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embedding.apply(ids, weight, float(scale))
    return _native().embed(ids, weight, scale)


def embedding_grad(grad: Tensor, ids: Tensor, num_embeddings: int, scale: float = 1.0) -> Tensor:
    """The table's gradient [num_embeddings, width] in grad's type: row v is scale * the sum of grad over the positions whose id is v."""
    return _native().embed_grad(grad, ids, num_embeddings, scale)


# -------------------------------------------------------------------------------------------------------------- convolution
class ConvGrads(NamedTuple):
    x: Tensor
    weight: Tensor
    bias: Tensor                       # (also where there is no bias: the sum is made anyway)
    state: Optional[Tensor]


def _silu(activation: Optional[str]) -> bool:
    if activation not in ("silu", None):
        raise ValueError("activation must be 'silu' or None")
    return activation == "silu"


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, activation, lengths, return_state):
        _check_capture(x, weight, bias, state)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, lengths, state)
        ctx.activation = activation
        return _native().conv(x, weight, bias, _silu(activation), lengths, state, return_state)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstate=None):
        x, weight, bias, lengths, state = ctx.saved_tensors
        if dy is None and dstate is None:
            return (None,) * 7
        dy = torch.zeros_like(x) if dy is None else dy
        g = causal_conv_grad(dy, x, weight, bias, activation=ctx.activation, lengths=lengths, state=state, state_grad=dstate)
        return g.x, g.weight, None if bias is None else g.bias, g.state, None, None, None


def causal_conv(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: Optional[str] = "silu", lengths: Optional[Tensor] = None,
                state: Optional[Tensor] = None, return_state: bool = False):
    """Each channel of x [batch, steps, width] convolved with its own `weight` [width, taps] (2 to 4 taps) over the steps up to and with
    the present one, plus `bias`, through silu unless `activation` is None.  `state` [batch, taps - 1, width], oldest first, holds
    the inputs in front of the first step (None: zeros); with `return_state` the result is (y, the last taps - 1 inputs)."""
    if _any_grad(x, weight, bias, state):
        y, out = _Conv.apply(x, weight, bias, state, activation, lengths, return_state)
    else:
        y, out = _native().conv(x, weight, bias, _silu(activation), lengths, state, return_state)
    return (y, out) if return_state else y


def causal_conv_grad(dy: Tensor, x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: Optional[str] = "silu",
                     lengths: Optional[Tensor] = None, state: Optional[Tensor] = None, state_grad: Optional[Tensor] = None) -> ConvGrads:
    """The gradients of causal_conv for dy and, where the state it returned was used, `state_grad`."""
    return ConvGrads(*_native().conv_grad(dy, x, weight, bias, _silu(activation), lengths, state, state_grad))


def causal_conv_step(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, state: Tensor, activation: Optional[str] = "silu",
                     out_state: Optional[Tensor] = None) -> Tensor:
    """causal_conv for one new step x [batch, width]; `state` [batch, taps - 1, width] moves on in place, or into `out_state`."""
    return _native().conv_step(x, weight, bias, _silu(activation), state, out_state)


# --------------------------------------------------------------------------------------------------------------------- scan
class ScanGrads(NamedTuple):
    x: Tensor
    dt: Tensor
    a: Tensor
    b: Tensor
    c: Tensor
    d: Tensor                          # (d and dt_bias also where there are none: the sums are made anyway)
    z: Optional[Tensor]
    dt_bias: Tensor
    state: Optional[Tensor]


class ScanSaved(NamedTuple):
    """What selective_scan_grad needs of a forward pass: its inputs, and the states at every 16th step (8th, for small problems)."""
    x: Tensor
    dt: Tensor
    a: Tensor
    b: Tensor
    c: Tensor
    d: Optional[Tensor]
    z: Optional[Tensor]
    dt_bias: Optional[Tensor]
    lengths: Optional[Tensor]
    state: Optional[Tensor]
    marks: Tensor
    softplus: bool


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, a, b, c, d, z, dt_bias, state, softplus, lengths, return_state):
        _check_capture(x, dt, a, b, c, d, z, dt_bias, state)
        ctx.set_materialize_grads(False)
        y, out, *saved = _native().scan(x, dt, a, b, c, d, z, dt_bias, softplus, lengths, state, return_state, True)
        ctx.save_for_backward(*saved)
        ctx.softplus, ctx.shapes = bool(softplus), (b.shape, c.shape)
        return y, out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstate=None):
        if dy is None and dstate is None:
            return (None,) * 12
        saved = ScanSaved(*ctx.saved_tensors, ctx.softplus)
        g = selective_scan_grad(torch.zeros_like(saved.x) if dy is None else dy, saved, dstate)
        return (g.x, g.dt, g.a, g.b.view(ctx.shapes[0]), g.c.view(ctx.shapes[1]), None if saved.d is None else g.d, g.z,
                None if saved.dt_bias is None else g.dt_bias, g.state, None, None, None)


def selective_scan(x: Tensor, dt: Tensor, a: Tensor, b: Tensor, c: Tensor, d: Optional[Tensor] = None, z: Optional[Tensor] = None,
                   dt_bias: Optional[Tensor] = None, *, softplus: bool = True, lengths: Optional[Tensor] = None,
                   state: Optional[Tensor] = None, return_state: bool = False):
    """For every row and channel, step after step: dt' = softplus(dt + dt_bias) (or without softplus), h[n] = exp(dt' a[n]) h[n] + dt' x b[n],
    y = (sum_n c[n] h[n] + d x) silu(z).

    x, dt, z [batch, steps, width]; a [width, states] with 1 to 32 states; b, c [batch, steps, states], or [batch, steps, groups,
    states] where each group serves width / groups neighbouring channels; d, dt_bias [width].  `state` [batch, width, states] is h in
    front of the first step (None: zeros); with `return_state` the result is (y, h behind each row's last step).

    States may grow (dt' a > 0).  Long sequences are walked in segments, whose factors exp(a sum of dt') are 32 bits too: where one
    overflows, so does every state that is not 0 at its beginning."""
    if _any_grad(x, dt, a, b, c, d, z, dt_bias, state):
        y, out = _Scan.apply(x, dt, a, b, c, d, z, dt_bias, state, softplus, lengths, return_state)
    else:
        y, out = _native().scan(x, dt, a, b, c, d, z, dt_bias, softplus, lengths, state, return_state, False)
    return (y, out) if return_state else y


def selective_scan_forward(x: Tensor, dt: Tensor, a: Tensor, b: Tensor, c: Tensor, d: Optional[Tensor] = None, z: Optional[Tensor] = None,
                           dt_bias: Optional[Tensor] = None, *, softplus: bool = True, lengths: Optional[Tensor] = None,
                           state: Optional[Tensor] = None, return_state: bool = False) -> Tuple[Tensor, Optional[Tensor], ScanSaved]:
    """selective_scan without autograd: (y, the state or None, what selective_scan_grad needs).  The inputs must not change in between."""
    y, out, *saved = _native().scan(x, dt, a, b, c, d, z, dt_bias, softplus, lengths, state, return_state, True)
    return y, out, ScanSaved(*saved, bool(softplus))


def selective_scan_grad(dy: Tensor, saved: ScanSaved, state_grad: Optional[Tensor] = None) -> ScanGrads:
    """The gradients of selective_scan_forward for dy and, where the state it returned was used, `state_grad`.  b's and c's come as
    [batch, steps, groups, states]."""
    return ScanGrads(*_native().scan_grad(dy, *saved, state_grad))


def selective_scan_step(x: Tensor, dt: Tensor, a: Tensor, b: Tensor, c: Tensor, d: Optional[Tensor] = None, z: Optional[Tensor] = None,
                        dt_bias: Optional[Tensor] = None, *, state: Tensor, softplus: bool = True, out_state: Optional[Tensor] = None) -> Tensor:
    """selective_scan for one new step: x, dt, z [batch, width], b, c [batch, states] or [batch, groups, states]; `state`
    [batch, width, states] moves on in place, or into `out_state`."""
    return _native().scan_step(x, dt, a, b, c, d, z, dt_bias, softplus, state, out_state)
