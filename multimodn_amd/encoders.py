"""Encoder plugins with the reference's constructor signatures and state_dict keys
(multimodn/encoders/multimod_encoder.py:8-17, mlp_encoder.py:49-80, slp_encoders.py:5-34).

`forward` keeps the module-level contract `encoder(state, x) -> new_state` for users who call a
plugin directly; `MultiModN.train_epoch` does not call it: it hands the parameters to the HIP
chain kernels (multimodn_amd/engine.py)."""
import math
from abc import ABC, abstractmethod
from typing import Callable, NamedTuple, Optional, Tuple

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from . import sequence as seq


class MultiModEncoder(nn.Module, ABC):
    def __init__(self, state_size: int):
        super().__init__()
        self.state_size = state_size

    @abstractmethod
    def forward(self, state: Tensor, x: Tensor) -> Tensor:
        ...


def _identity(x):
    return x


class MLPEncoder(MultiModEncoder):
    """Hidden Linear+activation layers see x only; the state joins the LAST Linear as
    cat([h, state]) and the output has no activation (mlp_encoder.py:64-80)."""

    def __init__(self, state_size: int, n_features: int, hidden_layers: Tuple[int, ...],
                 activation: Callable = F.relu, device: Optional[torch.device] = None):
        super().__init__(state_size)
        self.activation = activation
        self.n_features = n_features
        self.hidden_layers = tuple(hidden_layers)
        widths = [n_features, *self.hidden_layers]
        self.layers = nn.ModuleList()
        for fan_in, fan_out in zip(widths, widths[1:]):
            self.layers.append(nn.Linear(fan_in, fan_out, device=device))
        self.layers.append(nn.Linear(widths[-1] + state_size, state_size, device=device))

    def forward(self, state: Tensor, x: Tensor) -> Tensor:
        h = x
        for lin in list(self.layers)[:-1]:
            h = self.activation(lin(h))
        return self.layers[-1](torch.cat([h, state], dim=1))


class MLPFeatureEncoder(MLPEncoder):
    """One feature through one hidden layer: MLPEncoder(state_size, 1, (hidden_size,)) (mlp_encoder.py:81-94; the
    encoders of pipelines/titanic/titanic_featurewise_pipeline.py:70 and titanic_missingness_pipeline.py:71 over a
    FeatureWiseDataset).  The reference's forward re-wraps x with Tensor(x), which for the [B, 1] float32 batches it is fed
    is the same tensor; here x becomes float32 on the state's device.  On the HIP path it is an MLPEncoder like any other."""

    def __init__(self, state_size: int, hidden_size: int, activation: Callable = F.relu,
                 device: Optional[torch.device] = None):
        super().__init__(state_size, 1, (hidden_size,), activation, device)

    def forward(self, state: Tensor, x) -> Tensor:
        return super().forward(state, torch.as_tensor(x, dtype=torch.float32, device=state.device))


class MIMIC_MLPEncoder(MultiModEncoder):
    """The MIMIC pipelines' encoder (mlp_encoder.py:9-47): Dropout(p) on cat([x, state]) feeds the
    FIRST Linear, the activation follows EVERY Linear including the last one, whose output is the
    new state.  `layers[0]` is the nn.Dropout, so the Linears are layers.1 .. layers.n exactly as in
    the reference's state_dict."""

    def __init__(self, state_size: int, n_features: int, hidden_layers: Tuple[int, ...], dropout: float = .2,
                 activation: Callable = F.relu, device: Optional[torch.device] = None):
        super().__init__(state_size)
        self.activation = activation
        self.dropout = dropout
        self.n_features = n_features
        self.hidden_layers = tuple(hidden_layers)
        widths = [n_features + state_size, *self.hidden_layers, state_size]
        self.layers = nn.ModuleList([nn.Dropout(dropout)])
        for fan_in, fan_out in zip(widths, widths[1:]):
            self.layers.append(nn.Linear(fan_in, fan_out, device=device))

    @property
    def linears(self):
        return list(self.layers)[1:]

    def forward(self, state: Tensor, x: Tensor) -> Tensor:
        h = self.layers[0](torch.cat([x, state], dim=1))
        for lin in self.linears:
            h = self.activation(lin(h))
        return h


class SLPEncoder(MLPEncoder):
    """hidden_layers=() : a single Linear on cat([x, state]); `activation` is never applied
    (slp_encoders.py:5-14)."""

    def __init__(self, state_size: int, n_features: int, activation: Callable = torch.sigmoid):
        super().__init__(state_size, n_features, (), activation)


class LinearEncoder(SLPEncoder):
    def __init__(self, state_size: int, n_features: int):
        super().__init__(state_size, n_features, _identity)


class LogisticEncoder(SLPEncoder):
    def __init__(self, state_size: int, n_features: int):
        super().__init__(state_size, n_features, torch.sigmoid)


class SequenceState(NamedTuple):
    """What SequenceFeatures.step carries from token to token (its tensors move on in place)."""
    conv: Tensor
    scan: Tensor
    total: Tensor
    count: Tensor


class SequenceFeatures(nn.Module):
    """Token ids [batch, steps] to features [batch, width]: embedding, a projection to the scan's input and gate, a short causal
    convolution, the selective scan, the mean over the steps.  Each runs in multimodn_amd.sequence's kernels (the projections in
    torch's), forward and backward; there is no CPU fallback.

    A row ends behind its last id >= 0: pad with -1.  An id outside the vocabulary inside a row is a step without a token (its
    embedding is 0).  A row without any token has the features 0.  The datasets of this package hand every slot over as float32: the
    whole numbers there are the ids, and a row with anything else - a NaN, an infinity, a fraction - has NaN features, so that
    its batch skips the encoder like any other modality's (multimodn/multimodn.py:168).  A floating type that does not hold every id
    of the vocabulary is refused (float16 holds whole numbers to 2048, bfloat16 to 256, float32 to 2^24)."""

    def __init__(self, vocabulary: int, width: int, states: int = 16, taps: int = 4, rank: Optional[int] = None,
                 device: Optional[torch.device] = None):
        super().__init__()
        if not 1 <= states <= seq.MAX_STATES or not 2 <= taps <= seq.MAX_TAPS or vocabulary < 1 or width < 1:
            raise ValueError(f"SequenceFeatures needs 1 to {seq.MAX_STATES} states, 2 to {seq.MAX_TAPS} taps, a vocabulary and a width")
        self.vocabulary, self.width, self.states, self.taps = vocabulary, width, states, taps
        self.rank = rank if rank is not None else max(1, width // 16)
        self.table = nn.Parameter(torch.randn(vocabulary, width, device=device) / math.sqrt(width))
        self.inputs = nn.Linear(width, 2 * width, bias=False, device=device)
        self.conv_weight = nn.Parameter((torch.rand(width, taps, device=device) * 2 - 1) / math.sqrt(taps))
        self.conv_bias = nn.Parameter(torch.zeros(width, device=device))
        self.select = nn.Linear(width, self.rank + 2 * states, bias=False, device=device)
        self.spread = nn.Linear(self.rank, width, bias=False, device=device)
        first = torch.exp(torch.rand(width, device=device) * (math.log(0.1) - math.log(1e-3)) + math.log(1e-3))
        self.dt_bias = nn.Parameter(first + torch.log(-torch.expm1(-first)))            # softplus(dt_bias) = first
        self.a_log = nn.Parameter(torch.log(torch.arange(1, states + 1, dtype=torch.float32, device=device)).repeat(width, 1))
        self.skip = nn.Parameter(torch.ones(width, device=device))

    def _select(self, u: Tensor):
        dt, b, c = self.select(u).split((self.rank, self.states, self.states), dim=-1)
        return self.spread(dt), -torch.exp(self.a_log), b, c

    def forward(self, ids: Tensor) -> Tensor:
        if ids.dim() != 2 or ids.is_complex() or ids.dtype == torch.bool:
            raise ValueError(f"token ids must be a [batch, steps] tensor of whole numbers, not {list(ids.shape)} of {ids.dtype}")
        missing = None
        if ids.is_floating_point():
            if self.vocabulary > 2 / torch.finfo(ids.dtype).eps:
                raise ValueError(f"{ids.dtype} does not hold all {self.vocabulary} token ids: pass them as whole numbers")
            whole = torch.isfinite(ids) & (ids == ids.trunc())
            missing = ~whole.all(1, keepdim=True)
            ids = torch.where(whole, ids, -1.0).clamp(-1, self.vocabulary).long()      # (a whole number of any size, which int64 may not hold)
        elif ids.dtype not in (torch.int32, torch.int64):
            ids = ids.long()
        steps = torch.arange(1, ids.shape[1] + 1, device=ids.device)
        lengths = ((ids >= 0) * steps).amax(1) if ids.shape[1] else torch.zeros(ids.shape[0], dtype=torch.int64, device=ids.device)
        e = seq.embedding(ids, self.table, math.sqrt(self.width))
        x, z = self.inputs(e).chunk(2, dim=-1)
        u = seq.causal_conv(x, self.conv_weight, self.conv_bias, lengths=lengths)
        dt, a, b, c = self._select(u)
        y = seq.selective_scan(u, dt, a, b, c, self.skip, z, self.dt_bias, lengths=lengths)
        features = y.sum(1) / lengths.clamp(min=1).unsqueeze(1)
        return features if missing is None else torch.where(missing, math.nan, features)

    def start(self, batch: int) -> SequenceState:
        """The state in front of the first token of `batch` rows, for `step`."""
        dev = self.table.device
        return SequenceState(torch.zeros(batch, self.taps - 1, self.width, device=dev), torch.zeros(batch, self.width, self.states, device=dev),
                             torch.zeros(batch, self.width, device=dev), torch.zeros(batch, 1, device=dev))

    @torch.no_grad()
    def step(self, ids: Tensor, state: SequenceState) -> Tensor:
        """One more token [batch] for every row: the features of the rows so far, as `forward` gives them for the whole rows.  An id
        below 0 is a step without a token here, also at a row's end.  `state` moves on in place.  No gradient."""
        x, z = self.inputs(seq.embedding(ids, self.table, math.sqrt(self.width))).chunk(2, dim=-1)
        u = seq.causal_conv_step(x, self.conv_weight, self.conv_bias, state=state.conv)
        dt, a, b, c = self._select(u)
        state.total.add_(seq.selective_scan_step(u, dt, a, b, c, self.skip, z, self.dt_bias, state=state.scan))
        state.count.add_(1)
        return state.total / state.count


class SequenceEncoder(MLPEncoder):
    """An MLPEncoder over a token sequence: `front` (SequenceFeatures) makes `width` features of ids [batch, steps], the MLP and the
    state update follow as in MLPEncoder.  MultiModN trains both: the chain kernels hand back the features' gradient, `front`'s own
    kernels take it from there.  The reference's recurrent encoders (rnn_encoder.py, lstm_encoder.py) are torch modules over tabular
    input; a sequence modality has no counterpart there."""

    def __init__(self, state_size: int, vocabulary: int, width: int, hidden_layers: Tuple[int, ...], activation: Callable = F.relu,
                 states: int = 16, taps: int = 4, rank: Optional[int] = None, device: Optional[torch.device] = None):
        if not hidden_layers:
            raise ValueError("SequenceEncoder needs at least one hidden layer")
        super().__init__(state_size, width, hidden_layers, activation, device)
        self.front = SequenceFeatures(vocabulary, width, states, taps, rank, device)

    def forward(self, state: Tensor, x: Tensor) -> Tensor:
        """x: token ids [batch, steps]"""
        return super().forward(state, self.front(x))
