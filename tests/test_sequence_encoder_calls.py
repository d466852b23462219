"""Calls of models with a SequenceEncoder that their documentation allows and that once failed, answered wrongly or were not refused."""
import pytest
import torch

import multimodn_amd as mm
from test_sequence_encoder import ROWS, S, STEPS, V, WIDTH, batch, build

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
