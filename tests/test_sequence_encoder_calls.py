"""Calls of models with a SequenceEncoder that their documentation allows and that once failed, answered wrongly or were not refused."""
import copy

import pytest
import torch

import multimodn_amd as mm
from helpers import rel_err
from test_hip_parity import KERNEL_MODES, set_mode
from test_sequence_encoder import ROWS, S, STEPS, V, WIDTH, batch, build, plain_features, plain_step

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


@gpu
@pytest.mark.parametrize("split", ["0", "1"])
def test_fronts_beside_encoders_of_another_family(split, monkeypatch):
    """A MIMIC_MLPEncoder (without dropout) and MLPDecoders take the chain through the generic tier's kernels: the front's gradients against 64
    bits.  Bound as in the test of the tiers, with this model's sums (24 + 20, 16, 12 and their backward passes: under 300 for three encoders)."""
    monkeypatch.setenv("MMN_GEN_SPLIT", split)
    torch.manual_seed(12)
    size, rows = 20, 33
    encoders = [mm.SequenceEncoder(size, V, WIDTH, (16,), states=8, rank=3), mm.MIMIC_MLPEncoder(size, 6, (12,), 0.0),
                mm.SequenceEncoder(size, V + 5, 8, (5, 7), torch.sigmoid, states=4, rank=2)]
    model = mm.MultiModN(size, encoders, [mm.MLPDecoder(size, (9,)), mm.LogisticDecoder(size)], 0.7, 0.4, device=torch.device("cuda"))
    wide = copy.deepcopy(model).cpu().double()
    data, y = batch(3, rows)
    model.train_epoch([(data, y)], torch.optim.SGD(model.parameters(), 0.0), torch.nn.CrossEntropyLoss())
    state = wide.init_state.state_value.expand(rows, -1)
    errors, change = [torch.stack([torch.nn.functional.cross_entropy(d(state), y[:, i]) for i, d in enumerate(wide.decoders)])], 0.0
    for enc, x in zip(wide.encoders, data):
        old = state
        state = mm.MLPEncoder.forward(enc, state, plain_features(enc.front, x)) if isinstance(enc, mm.SequenceEncoder) else enc(state, x.double())
        change = change + ((state - old) ** 2).mean()
        errors.append(torch.stack([torch.nn.functional.cross_entropy(d(state), y[:, i]) for i, d in enumerate(wide.decoders)]))
    loss = torch.stack(errors).mean() * wide.err_penalty + change / 3 * wide.state_change_penalty
    bound = (300 + 3 * STEPS + 60 + rows * STEPS) * 2.0 ** -24 * 8
    for (n, p), g in zip(model.named_parameters(), torch.autograd.grad(loss, list(wide.parameters()))):
        assert rel_err(p.grad.cpu().numpy(), g.numpy()) < bound, n


@gpu
def test_fronts_of_no_rows_and_no_steps():
    front = build(seed=4).encoders[0].front
    assert not front(torch.zeros(3, 0, dtype=torch.int64, device="cuda")).any() and front(torch.zeros(0, 5, dtype=torch.int64, device="cuda")).shape == (0, WIDTH)
    assert not front(torch.full((2, 4), -1, device="cuda")).any()
    for ids in (torch.zeros(3, 0, dtype=torch.int64, device="cuda"), torch.full((2, 4), -1, device="cuda")):
        front(ids).sum().backward()
        assert all(p.grad is None or not p.grad.any() for p in front.parameters())


@gpu
def test_missing_ids_in_test_and_predict():
    """test() skips the encoder of a batch with a missing id, as it does another modality's; predict() has no skip: its rows are NaN."""
    model = build(seed=4)
    plain = mm.MultiModN(S, [mm.MLPEncoder(S, e.n_features, e.hidden_layers, e.activation) for e in model.encoders],
                         [mm.LogisticDecoder(S), mm.LogisticDecoder(S)], 0.7, 0.4, device=torch.device("cuda"))
    plain.load_state_dict({k: v for k, v in model.state_dict().items() if ".front." not in k})
    data, y = batch(5)
    data[0] = data[0].float()
    data[0][3, 2] = float("nan")
    with torch.no_grad():
        feats = [e.front(x.cuda()) if isinstance(e, mm.SequenceEncoder) else x.cuda() for e, x in zip(model.encoders, data)]
    assert torch.isnan(feats[0][3]).all() and torch.isfinite(feats[0][[0, 1, 2]]).all()
    crit = torch.nn.CrossEntropyLoss()
    for r, s in zip(model.test([(data, y)], crit), plain.test([(feats, y.cuda())], crit)):
        for a, b in zip(r, s):
            assert torch.allclose(torch.as_tensor(a), torch.as_tensor(b), rtol=0, atol=0, equal_nan=True)
    assert torch.equal(torch.isnan(torch.as_tensor(model.predict(data))), torch.isnan(torch.as_tensor(plain.predict(feats))))


@gpu
def test_autocast():
    """Mixed precision around a front: the projections and what they feed in 16 bits, states and sums in 32."""
    front = build(seed=4).encoders[0].front
    ids = batch(5)[0][0].cuda()
    want = front(ids)
    with torch.autocast("cuda", torch.bfloat16):
        got = front(ids)
        got.sum().backward()
    # x, z, u, dt, b, c and y are rounded to bf16 (2^-8 each, half of that on average): some ten such roundings of values up to 8 times the result
    assert got.dtype == torch.float32 and rel_err(got.detach().cpu(), want.detach().cpu()) < 10 * 2.0 ** -8 * 8
    assert all(torch.isfinite(p.grad).all() and p.grad.dtype == torch.float32 for p in front.parameters())
