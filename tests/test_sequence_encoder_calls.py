"""Calls of models with a SequenceEncoder that their documentation allows and that once failed, answered wrongly or were not refused."""
import copy

import pytest
import torch

import multimodn_amd as mm
from helpers import rel_err
from test_hip_parity import KERNEL_MODES, set_mode
from test_sequence_encoder import ROWS, STEPS, V, batch, build, plain_step

gpu = pytest.mark.gpu


def incomplete(kind, model):
    """(batch, parameters whose gradient is None in it)"""
    data, y = batch(5)
    if kind == "nan":
        data[1][3, 2] = float("nan")
        return (data, y), list(model.encoders[1].parameters())
    if kind == "nan ids":
        data[0] = data[0].float()
        data[0][3, 2] = float("nan")
        return (data, y), list(model.encoders[0].parameters())
    if kind == "sequence":
        return ([data[2], data[1]], y, torch.tensor([[2, 1]]).expand(ROWS, -1)), list(model.encoders[0].parameters())
    frozen = model.encoders[0].front.table                                    # kind "frozen"
    frozen.requires_grad_(False)
    return (data, y), [frozen]


@gpu
@pytest.mark.parametrize("kind", ["nan", "nan ids", "sequence", "frozen"])
def test_adam_whose_first_batch_is_incomplete(kind):
    """The framework's Adam as torch's: parameters without a gradient stay as they are, and so do their moments; the others take the step,
    and a later, complete batch trains all."""
    models, opts, dropped = [], [], []
    for make in (mm.optim.Adam, torch.optim.Adam):
        model = build(seed=4)
        data, without = incomplete(kind, model)
        before = {n: p.detach().clone() for n, p in model.named_parameters()}
        opt = make(model.parameters(), 1e-3)
        model.train_epoch([data], opt, torch.nn.CrossEntropyLoss())
        ids = {id(p) for p in without}
        for n, p in model.named_parameters():
            if id(p) in ids:
                assert p.grad is None and torch.equal(p, before[n]), n
                assert make is torch.optim.Adam or (not opt.state[p]["exp_avg"].any() and float(opt.state[p]["step"]) == 0), n
            else:
                assert p.grad is not None and float(opt.state[p]["step"]) == 1, n
        models.append(model)
        opts.append(opt)
        dropped.append(ids)
    # The gradients are the same, bit for bit.  The step is lr m / (sqrt(v) + eps) from the moments' few products in 32 bits: under 16 roundings
    # of a step of at most lr on either side, 2 * 16 * 2^-24 * 1e-3 < 2e-9, and one rounding each of a weight under 4: 2 * 2^-24 * 4 < 5e-7
    for p, q in zip(*(m.parameters() for m in models)):
        assert (p.grad is None and q.grad is None) or torch.equal(p.grad, q.grad)
        assert (p - q).abs().max() <= 5e-7 + 2e-9
    later = {n: p.detach().clone() for n, p in models[0].named_parameters()}
    models[0].train_epoch([batch(6)], opts[0], torch.nn.CrossEntropyLoss())
    for n, p in models[0].named_parameters():
        still = id(p) in dropped[0]
        if still and kind == "frozen":
            assert p.grad is None and torch.equal(p, later[n])
        else:
            assert p.grad is not None and float(opts[0].state[p]["step"]) == (1 if still else 2)
            assert not p.grad.any() or not torch.equal(p, later[n]), n


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_a_single_training_step_is_refused(device):
    """It would train the chain alone (the features are made without a graph)."""
    model = build(device)
    data, y = batch()
    eng = model._get_engine(ROWS) if device == "cuda" else None
    with pytest.raises(mm.UnsupportedModelError, match="train_epoch"):
        model._run_step(eng, data, y, None, True)


@gpu
def test_floating_ids_that_are_not_whole_numbers():
    """Rows with a fraction or an infinity have NaN features, the others those of the same ids as whole numbers."""
    front = build(seed=9).encoders[0].front
    ids = torch.tensor([[1.0, 2.0, 3.0], [1.0, 3.7, 2.0], [1.0, float("inf"), 2.0], [-0.5, 1.0, 2.0], [4.0, -1.0, V], [float("nan"), 1.0, 2.0],
                        [2.0, -float("inf"), -1.0], [-1.0, -1.0, -1.0]]).cuda()
    for kind in (torch.float32, torch.float64, torch.float16, torch.bfloat16):
        got = front(ids.to(kind))
        good = [0, 4, 7]
        assert torch.equal(got[good], front(ids[good].long()))
        assert torch.isnan(got[[1, 2, 3, 5, 6]]).all()
    far = torch.tensor([[1.0, 2.0, 1e30], [-1e30, 2.0, 3.0]]).cuda()              # outside the vocabulary; a step without a token
    assert torch.equal(front(far), front(torch.tensor([[1, 2, V], [-1, 2, 3]]).cuda()))
    data, y = batch(5)
    data[0] = data[0].float()
    data[0][3, 2] = 1.5
    model = build(seed=4)
    model.train_epoch([(data, y)], torch.optim.SGD(model.parameters(), 1e-2), torch.nn.CrossEntropyLoss())
    assert all(p.grad is None for p in model.encoders[0].parameters())
    assert all(torch.isfinite(p.grad).all() for e in (1, 2) for p in model.encoders[e].parameters())


def test_floating_types_that_do_not_hold_the_vocabulary_are_refused():
    for vocabulary, kind in ((257, torch.bfloat16), (2049, torch.float16), ((1 << 24) + 1, torch.float32)):
        front = mm.SequenceFeatures(vocabulary, 1, states=1, taps=2)
        with pytest.raises(ValueError, match="token ids"):
            front(torch.zeros(2, 3, dtype=kind))
        with pytest.raises(mm.hip.MmnError):                                  # (ids of a type that holds them go on to the operators)
            front(torch.zeros(2, 3, dtype=torch.float64))


@gpu
@pytest.mark.parametrize("rows", [16, 257])
@pytest.mark.parametrize("mode", list(KERNEL_MODES))
def test_fronts_train_through_every_tier_of_the_chain(mode, rows, monkeypatch):
    """The gradient that leaves the chain at an encoder's input, whichever kernels ran the chain: gradients of all parameters against 64 bits
    at the framework's own sizes (state 128, hidden (32, 32), four encoders).  A sum of n products in 32 bits is off by n 2^-24 of its terms'
    size: an encoder's layers and state update sum 64 + 128, 32 and 32 values and the same backwards, so four encoders some 2100, the front
    3 * STEPS + 60, a weight's gradient rows * STEPS; terms as large as 8 times the largest sum, as in the smaller model's test."""
    set_mode(monkeypatch, mode)
    torch.manual_seed(11)
    size = 128
    encoders = [mm.SequenceEncoder(size, V, 64, (32, 32), states=8, rank=3), mm.MLPEncoder(size, 6, (32, 32)),
                mm.SequenceEncoder(size, V + 5, 24, (32, 32), states=4, rank=2), mm.MLPEncoder(size, 6, (32, 32))]
    model = mm.MultiModN(size, encoders, [mm.LogisticDecoder(size) for _ in range(3)], 0.7, 0.4, device=torch.device("cuda"))
    wide = copy.deepcopy(model).cpu().double()
    data, y = batch(3, rows)
    data, y = data + [data[1].flip(0)], torch.cat([y, y[:, :1].flip(0)], 1)
    hist = mm.MultiModNHistory(["a", "b", "c"])
    model.train_epoch([(data, y)], torch.optim.SGD(model.parameters(), 0.0), torch.nn.CrossEntropyLoss(), hist)
    loss, grid = plain_step(wide, data, y)
    bound = (2100 + 3 * STEPS + 60 + rows * STEPS) * 2.0 ** -24 * 8
    assert rel_err(hist.loss["train"][0], grid.detach().numpy()) < 1e-5
    for (n, p), g in zip(model.named_parameters(), torch.autograd.grad(loss, list(wide.parameters()))):
        assert rel_err(p.grad.cpu().numpy(), g.numpy()) < bound, n
