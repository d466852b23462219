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

Everything runs on the current stream of the tensors' device, may be captured into a graph, and has no CPU or torch-op fallback: off
an AMD GPU these functions raise.  The reference has no counterpart: its recurrent encoders (multimodn/encoders/rnn_encoder.py,
lstm_encoder.py) are torch modules.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from . import hip

MAX_STATES = 32
MAX_TAPS = 4
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_LIMIT = 2 ** 31 - 1


# ---------------------------------------------------------------------------------------------------------------- arguments
def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _gpu(first: Tensor, **others: Optional[Tensor]) -> int:
    """All tensors on one GPU: its index."""
    if first.device.type != "cuda":
        raise hip.MmnError(f"the sequence operators only run on an AMD GPU (torch device 'cuda' on ROCm), not on {first.device}; "
                           "there is no CPU fallback")
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{name} is on {t.device}, not on {first.device}")
    return first.device.index


def _data(name: str, t: Tensor, dtype: torch.dtype, *shape: int) -> Tensor:
    _need(isinstance(t, Tensor) and t.dtype == dtype, f"{name} must be a {dtype} tensor, as the other data of the call")
    _need(tuple(t.shape) == shape, f"{name} must be {list(shape)}, not {list(t.shape)}")
    # (the kernels address a few steps of a row with 32-bit offsets: steps further apart than 2^23 elements are brought together, steps
    #  that share memory taken apart)
    if t.stride(-1) == 1:
        step = t.stride(1) if len(shape) > 2 else shape[-1]
        if shape[-1] <= step <= 1 << 23 or shape[1] <= 1:
            return t
        return t.clone(memory_format=torch.contiguous_format)
    return t.contiguous()


def _float(name: str, t: Optional[Tensor], *shape: int) -> Optional[Tensor]:
    if t is None:
        return None
    _need(isinstance(t, Tensor) and t.dtype == torch.float32, f"{name} must be a float32 tensor")
    _need(tuple(t.shape) == shape, f"{name} must be {list(shape)}, not {list(t.shape)}")
    return t.contiguous()


def _lengths(lengths: Optional[Tensor], batch: int) -> Optional[Tensor]:
    if lengths is None:
        return None
    _need(isinstance(lengths, Tensor) and lengths.dtype in (torch.int32, torch.int64), "lengths must be an int32 or int64 tensor")
    _need(tuple(lengths.shape) == (batch,), f"lengths must be [{batch}], not {list(lengths.shape)}")
    # (int64 values outside int32 would wrap: the kernels clamp to [0, steps])
    return lengths.contiguous() if lengths.dtype == torch.int32 else lengths.clamp(0, _LIMIT).to(torch.int32)


def _kind(x: Tensor, dims: int) -> int:
    _need(isinstance(x, Tensor) and x.dtype in _TYPES, "data must be float32, bfloat16 or float16")
    _need(x.dim() == dims and x.shape[-1] >= 1, f"x must have {dims} dimensions, the last of at least one channel, not shape {list(x.shape)}")
    _need(max(x.shape) <= 2 ** 30, "sizes above 2^30 are not supported")
    return _TYPES[x.dtype]


def _serving(*tensors: Optional[Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("the one-step forms have no gradient: call them under torch.no_grad(), or the whole sequence's operator")


def _ptr(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


class _On:
    """The device made current for the length of a call (entered only where it is another one)."""

    def __init__(self, index: int):
        self.guard = torch.cuda.device(index) if torch.cuda.current_device() != index else None

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *ex):
        if self.guard is not None:
            self.guard.__exit__(*ex)


def _stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _workspace(n: int, device) -> Tensor:
    return torch.empty(max(int(n), 256), dtype=torch.uint8, device=device)     # (the allocator's blocks begin on 512 bytes)


def _moved(t: Tensor) -> None:
    """A tensor written through its address: autograd's saved copies of it are stale."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _state_pair(state: Tensor, out_state: Optional[Tensor]) -> Tensor:
    out = state if out_state is None else out_state
    _need(out.dtype == state.dtype and out.shape == state.shape and out.device == state.device, "out_state must be like state")
    _need(state.is_contiguous() and out.is_contiguous(), "state and out_state must be contiguous")
    if out is not state:
        a, b, n = state.data_ptr(), out.data_ptr(), state.numel() * state.element_size()
        _need(a == b or a + n <= b or b + n <= a, "out_state overlaps state without being the same memory")
    return out


# ---------------------------------------------------------------------------------------------------------------- embedding
def _ids(ids: Tensor) -> Tensor:
    _need(isinstance(ids, Tensor) and ids.dtype in (torch.int32, torch.int64), "ids must be an int32 or int64 tensor")
    _need(ids.numel() <= _LIMIT, "more than 2^31 - 1 ids")
    return ids.contiguous()


def _embed(ids: Tensor, weight: Tensor, scale: float) -> Tensor:
    index = _gpu(weight, ids=ids)
    out = torch.empty(*ids.shape, weight.shape[1], dtype=weight.dtype, device=weight.device)
    with _On(index):
        hip.check(hip.load().mmn_seq_embed(ids.data_ptr(), int(ids.dtype == torch.int64), weight.data_ptr(), out.data_ptr(), ids.numel(),
                                           weight.shape[0], weight.shape[1], _TYPES[weight.dtype], scale, _stream(index)), "mmn_seq_embed")
    return out


def _table(weight: Tensor) -> Tensor:
    _need(isinstance(weight, Tensor) and weight.dtype in _TYPES, "the table must be float32, bfloat16 or float16")
    _need(weight.dim() == 2 and weight.shape[0] >= 1 and weight.shape[1] >= 1 and max(weight.shape) <= 2 ** 30,
          f"the table must be [vocabulary, width], not {list(weight.shape)}")
    return weight.contiguous()


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale):
        ctx.save_for_backward(ids)
        ctx.vocab, ctx.scale = weight.shape[0], scale
        return _embed(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        return None, embedding_grad(grad, ids, ctx.vocab, ctx.scale), None


def embedding(ids: Tensor, weight: Tensor, scale: float = 1.0) -> Tensor:
    """scale * weight[ids], [*ids.shape, width] in the table's type.  An id outside [0, vocabulary) - by convention -1 - stands for "no
    token": its output is 0 and it has no part in the gradient.  The gradient sums each table row's contributions in the order of
    their positions, from sorted ids."""
    ids, weight = _ids(ids), _table(weight)
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embedding.apply(ids, weight, float(scale))
    return _embed(ids, weight, float(scale))


def embedding_grad(grad: Tensor, ids: Tensor, num_embeddings: int, scale: float = 1.0) -> Tensor:
    """The table's gradient [num_embeddings, width] in grad's type: row v is scale * the sum of grad over the positions whose id is v."""
    ids = _ids(ids)
    _need(isinstance(grad, Tensor) and grad.dtype in _TYPES, "grad must be float32, bfloat16 or float16")
    _need(grad.dim() == ids.dim() + 1 and grad.shape[:-1] == ids.shape and 1 <= grad.shape[-1] <= 2 ** 30,
          f"grad must be [*ids.shape, width], not {list(grad.shape)} for ids {list(ids.shape)}")
    _need(1 <= num_embeddings <= 2 ** 30, "num_embeddings must be in [1, 2^30]")
    index = _gpu(grad, ids=ids)
    grad = grad.contiguous()
    lib, width = hip.load(), grad.shape[-1]
    out = torch.empty(num_embeddings, width, dtype=grad.dtype, device=grad.device)
    n = lib.mmn_seq_embed_grad_bytes(ids.numel(), num_embeddings, width)
    ws = _workspace(n, grad.device)
    with _On(index):
        hip.check(lib.mmn_seq_embed_grad(ids.data_ptr(), int(ids.dtype == torch.int64), grad.data_ptr(), out.data_ptr(), ids.numel(), num_embeddings,
                                         width, _TYPES[grad.dtype], float(scale), ws.data_ptr(), ws.numel(), _stream(index)), "mmn_seq_embed_grad")
    return out


# -------------------------------------------------------------------------------------------------------------- convolution
class ConvGrads(NamedTuple):
    x: Tensor
    weight: Tensor
    bias: Tensor                       # (also where there is no bias: the sum is made anyway)
    state: Optional[Tensor]


def _conv_desc(x, weight, bias, activation, lengths, state, dims=3):
    kind = _kind(x, dims)
    batch, steps, width = x.shape[0], x.shape[1] if dims == 3 else 1, x.shape[-1]
    _need(weight.dim() == 2 and 2 <= weight.shape[1] <= MAX_TAPS, f"weight must be [width, taps] with 2 to {MAX_TAPS} taps")
    taps = weight.shape[1]
    _need(activation in ("silu", None), "activation must be 'silu' or None")
    x = _data("x", x, x.dtype, *x.shape)
    weight, bias, lengths = _float("weight", weight, width, taps), _float("bias", bias, width), _lengths(lengths, batch)
    if state is not None:
        state = _data("state", state, x.dtype, batch, taps - 1, width).contiguous()
    index = _gpu(x, weight=weight, bias=bias, lengths=lengths, state=state)
    d = hip.ConvDesc()
    d.x, d.state, d.weight, d.bias, d.lengths = _ptr(x), _ptr(state), _ptr(weight), _ptr(bias), _ptr(lengths)
    d.batch, d.x_row, d.x_step = batch, x.stride(0), x.stride(1) if dims == 3 else 0
    d.steps, d.width, d.taps, d.silu, d.type = steps, width, taps, int(activation == "silu"), kind
    return d, index, (x, weight, bias, lengths, state)


def _conv(x, weight, bias, activation, lengths, state, return_state):
    d, index, keep = _conv_desc(x, weight, bias, activation, lengths, state)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    out = torch.empty(x.shape[0], d.taps - 1, x.shape[2], dtype=x.dtype, device=x.device) if return_state else None
    d.y, d.state_out = _ptr(y), _ptr(out)
    with _On(index):
        hip.check(hip.load().mmn_seq_conv(C.byref(d), _stream(index)), "mmn_seq_conv")
    return y, out


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, activation, lengths, return_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, lengths, state)
        ctx.activation = activation
        return _conv(x, weight, bias, activation, lengths, state, return_state)

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
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, state)):
        y, out = _Conv.apply(x, weight, bias, state, activation, lengths, return_state)
    else:
        y, out = _conv(x, weight, bias, activation, lengths, state, return_state)
    return (y, out) if return_state else y


def causal_conv_grad(dy: Tensor, x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: Optional[str] = "silu",
                     lengths: Optional[Tensor] = None, state: Optional[Tensor] = None, state_grad: Optional[Tensor] = None) -> ConvGrads:
    """The gradients of causal_conv for dy and, where the state it returned was used, `state_grad`."""
    _kind(x, 3)
    dy = _data("dy", dy, x.dtype, *x.shape)
    d, index, keep = _conv_desc(x, weight, bias, activation, lengths, state)
    batch, steps, width = x.shape
    if state_grad is not None:
        state_grad = _data("state_grad", state_grad, x.dtype, batch, d.taps - 1, width).contiguous()
    _gpu(x, dy=dy, state_grad=state_grad)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dstate = torch.empty(batch, d.taps - 1, width, dtype=x.dtype, device=x.device) if state is not None else None
    params = torch.empty(width * (d.taps + 1), dtype=torch.float32, device=x.device)
    dweight, dbias = params[:width * d.taps].view(width, d.taps), params[width * d.taps:]
    if batch == 0 or steps == 0:
        params.zero_()
        if dstate is not None:
            dstate.zero_() if state_grad is None else dstate.copy_(state_grad)
        return ConvGrads(dx, dweight, dbias, dstate)
    d.dy, d.dstate_out, d.dx, d.dstate = _ptr(dy), _ptr(state_grad), _ptr(dx), _ptr(dstate)
    d.dy_row, d.dy_step = dy.stride(0), dy.stride(1)
    d.dweight, d.dbias = _ptr(dweight), _ptr(dbias)
    lib = hip.load()
    ws = _workspace(lib.mmn_seq_conv_grad_bytes(C.byref(d)), x.device)
    with _On(index):
        hip.check(lib.mmn_seq_conv_grad(C.byref(d), ws.data_ptr(), ws.numel(), _stream(index)), "mmn_seq_conv_grad")
    return ConvGrads(dx, dweight, dbias, dstate)


def causal_conv_step(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, state: Tensor, activation: Optional[str] = "silu",
                     out_state: Optional[Tensor] = None) -> Tensor:
    """causal_conv for one new step x [batch, width]; `state` [batch, taps - 1, width] moves on in place, or into `out_state`."""
    _serving(x, weight, bias, state)
    _need(isinstance(state, Tensor), "state must be a tensor")
    out = _state_pair(state, out_state)
    d, index, keep = _conv_desc(x, weight, bias, activation, None, state, dims=2)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    d.y, d.state_out = _ptr(y), _ptr(out)
    with _On(index):
        hip.check(hip.load().mmn_seq_conv_step(C.byref(d), _stream(index)), "mmn_seq_conv_step")
    _moved(out)
    return y


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
    """What selective_scan_grad needs of a forward pass: its inputs, and the states at every 16th or 32nd step."""
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


def _scan_desc(x, dt, a, b, c, d, z, dt_bias, softplus, lengths, state, dims=3):
    kind = _kind(x, dims)
    lead, width = tuple(x.shape[:-1]), x.shape[-1]
    batch, steps = lead[0], lead[1] if dims == 3 else 1
    _need(isinstance(a, Tensor) and a.dim() == 2 and 1 <= a.shape[1] <= MAX_STATES, f"a must be [width, states] with 1 to {MAX_STATES} states")
    states = a.shape[1]
    both = []
    for name, t in (("b", b), ("c", c)):
        _need(isinstance(t, Tensor) and t.dim() in (dims, dims + 1), f"{name} must be [.., states] or [.., groups, states]")
        t = t.unsqueeze(-2) if t.dim() == dims else t
        both.append(_data(name, t, x.dtype, *lead, t.shape[-2], states))
    b, c = both
    groups = b.shape[-2]
    _need(c.shape[-2] == groups and groups >= 1 and width % groups == 0, "b and c need the same number of groups, which divides the width")
    x, dt = _data("x", x, x.dtype, *x.shape), _data("dt", dt, x.dtype, *x.shape)
    z = _data("z", z, x.dtype, *x.shape) if z is not None else None
    a, d, dt_bias, state = _float("a", a, width, states), _float("d", d, width), _float("dt_bias", dt_bias, width), _float("state", state, batch, width, states)
    lengths = _lengths(lengths, batch)
    index = _gpu(x, dt=dt, a=a, b=b, c=c, d=d, z=z, dt_bias=dt_bias, lengths=lengths, state=state)
    s = hip.ScanDesc()
    s.x, s.dt, s.b, s.c, s.z = x.data_ptr(), dt.data_ptr(), b.data_ptr(), c.data_ptr(), _ptr(z)
    s.a, s.d, s.dt_bias, s.state, s.lengths = a.data_ptr(), _ptr(d), _ptr(dt_bias), _ptr(state), _ptr(lengths)
    s.batch, s.steps, s.width, s.groups, s.states, s.softplus, s.type = batch, steps, width, groups, states, int(bool(softplus)), kind
    s.x_row, s.dt_row, s.b_row, s.c_row = x.stride(0), dt.stride(0), b.stride(0), c.stride(0)
    s.b_group, s.c_group = b.stride(-2), c.stride(-2)
    if dims == 3:
        s.x_step, s.dt_step, s.b_step, s.c_step = x.stride(1), dt.stride(1), b.stride(1), c.stride(1)
    if z is not None:
        s.z_row, s.z_step = z.stride(0), z.stride(1) if dims == 3 else 0
    return s, index, (x, dt, a, b, c, d, z, dt_bias, lengths, state)


def _scan(x, dt, a, b, c, d, z, dt_bias, softplus, lengths, state, return_state, save):
    s, index, keep = _scan_desc(x, dt, a, b, c, d, z, dt_bias, softplus, lengths, state)
    lib = hip.load()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    out = torch.empty(x.shape[0], x.shape[2], s.states, dtype=torch.float32, device=x.device) if return_state else None
    marks = torch.empty(lib.mmn_seq_scan_marks(C.byref(s)), dtype=torch.float32, device=x.device) if save else None
    s.y, s.state_out, s.marks = _ptr(y), _ptr(out), _ptr(marks) if save and marks.numel() else None
    ws = _workspace(lib.mmn_seq_scan_bytes(C.byref(s), 0), x.device)
    with _On(index):
        hip.check(lib.mmn_seq_scan(C.byref(s), ws.data_ptr(), ws.numel(), _stream(index)), "mmn_seq_scan")
    return y, out, ScanSaved(*keep, marks, bool(softplus)) if save else None


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, a, b, c, d, z, dt_bias, state, softplus, lengths, return_state):
        ctx.set_materialize_grads(False)
        y, out, saved = _scan(x, dt, a, b, c, d, z, dt_bias, softplus, lengths, state, return_state, True)
        ctx.save_for_backward(*saved[:-1])
        ctx.softplus, ctx.shapes = saved.softplus, (b.shape, c.shape)
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
    front of the first step (None: zeros); with `return_state` the result is (y, h behind each row's last step)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, dt, a, b, c, d, z, dt_bias, state)):
        y, out = _Scan.apply(x, dt, a, b, c, d, z, dt_bias, state, softplus, lengths, return_state)
    else:
        y, out, _ = _scan(x, dt, a, b, c, d, z, dt_bias, softplus, lengths, state, return_state, False)
    return (y, out) if return_state else y


def selective_scan_forward(x: Tensor, dt: Tensor, a: Tensor, b: Tensor, c: Tensor, d: Optional[Tensor] = None, z: Optional[Tensor] = None,
                           dt_bias: Optional[Tensor] = None, *, softplus: bool = True, lengths: Optional[Tensor] = None,
                           state: Optional[Tensor] = None, return_state: bool = False) -> Tuple[Tensor, Optional[Tensor], ScanSaved]:
    """selective_scan without autograd: (y, the state or None, what selective_scan_grad needs).  The inputs must not change in between."""
    return _scan(x, dt, a, b, c, d, z, dt_bias, softplus, lengths, state, return_state, True)


def selective_scan_grad(dy: Tensor, saved: ScanSaved, state_grad: Optional[Tensor] = None) -> ScanGrads:
    """The gradients of selective_scan_forward for dy and, where the state it returned was used, `state_grad`.  b's and c's come as
    [batch, steps, groups, states]."""
    x = saved.x
    s, index, keep = _scan_desc(x, saved.dt, saved.a, saved.b, saved.c, saved.d, saved.z, saved.dt_bias, saved.softplus, saved.lengths, saved.state)
    batch, steps, width = x.shape
    dy = _data("dy", dy, x.dtype, *x.shape)
    state_grad = _float("state_grad", state_grad, batch, width, s.states)
    _gpu(x, dy=dy, state_grad=state_grad)
    lib = hip.load()
    dx, ddt = torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dz = torch.empty(x.shape, dtype=x.dtype, device=x.device) if saved.z is not None else None
    db, dc = (torch.empty(batch, steps, s.groups, s.states, dtype=x.dtype, device=x.device) for _ in range(2))
    n = width * s.states
    params = torch.empty(n + 2 * width, dtype=torch.float32, device=x.device)
    da, dd, dbias = params[:n].view(width, s.states), params[n:n + width], params[n + width:]
    dstate = torch.empty(batch, width, s.states, dtype=torch.float32, device=x.device) if saved.state is not None else None
    out = ScanGrads(dx, ddt, da, db, dc, dd, dz, dbias, dstate)
    if batch == 0 or steps == 0:
        params.zero_()
        if dstate is not None:
            dstate.zero_() if state_grad is None else dstate.copy_(state_grad)
        return out
    s.marks, s.dy, s.dstate_out = saved.marks.data_ptr(), dy.data_ptr(), _ptr(state_grad)
    s.dy_row, s.dy_step = dy.stride(0), dy.stride(1)
    s.dx, s.ddt, s.db, s.dc, s.dz, s.dparams, s.dstate = _ptr(dx), _ptr(ddt), _ptr(db), _ptr(dc), _ptr(dz), _ptr(params), _ptr(dstate)
    ws = _workspace(lib.mmn_seq_scan_bytes(C.byref(s), 1), x.device)
    with _On(index):
        hip.check(lib.mmn_seq_scan_grad(C.byref(s), ws.data_ptr(), ws.numel(), _stream(index)), "mmn_seq_scan_grad")
    return out


def selective_scan_step(x: Tensor, dt: Tensor, a: Tensor, b: Tensor, c: Tensor, d: Optional[Tensor] = None, z: Optional[Tensor] = None,
                        dt_bias: Optional[Tensor] = None, *, state: Tensor, softplus: bool = True, out_state: Optional[Tensor] = None) -> Tensor:
    """selective_scan for one new step: x, dt, z [batch, width], b, c [batch, states] or [batch, groups, states]; `state`
    [batch, width, states] moves on in place, or into `out_state`."""
    _serving(x, dt, a, b, c, d, z, dt_bias, state)
    _need(isinstance(state, Tensor), "state must be a tensor")
    out = _state_pair(state, out_state)
    s, index, keep = _scan_desc(x, dt, a, b, c, d, z, dt_bias, softplus, None, state, dims=2)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    s.y, s.state_out = _ptr(y), _ptr(out)
    with _On(index):
        hip.check(hip.load().mmn_seq_scan_step(C.byref(s), _stream(index)), "mmn_seq_scan_step")
    _moved(out)
    return y
