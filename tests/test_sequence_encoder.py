"""SequenceEncoder: a token modality in MultiModN, its features' kernels trained through the fusion chain."""
import copy
import math
import pickle

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import multimodn_amd as mm
from helpers import rel_err
from multimodn_amd import hip

gpu = pytest.mark.gpu
S, V, WIDTH, STEPS, ROWS = 20, 30, 24, 12, 16


def build(device="cuda", seed=0, taps=4, states=8, dropout_free=True):
    torch.manual_seed(seed)
    encoders = [mm.SequenceEncoder(S, V, WIDTH, (16,), states=states, taps=taps, rank=3), mm.MLPEncoder(S, 6, (8, 8)),
                mm.SequenceEncoder(S, V + 5, 8, (5, 7), torch.sigmoid, states=4, rank=2)]
    model = mm.MultiModN(S, encoders, [mm.LogisticDecoder(S), mm.LogisticDecoder(S)], 0.7, 0.4, device=torch.device(device))
    return model


def batch(seed=1, rows=ROWS):
    g = torch.Generator().manual_seed(seed)
    a, b = torch.randint(0, V, (rows, STEPS), generator=g), torch.randint(-1, V + 5, (rows, 5), generator=g)
    ends = torch.randint(0, STEPS + 1, (rows,), generator=g)
    ends[0], ends[1] = 0, STEPS
    a[torch.arange(STEPS) >= ends[:, None]] = -1
    return [a, torch.randn(rows, 6, generator=g), b], torch.randint(0, 2, (rows, 2), generator=g)


# ---- the same in 64 bits, step after step on the CPU
def plain_features(front, ids):
    out = []
    silu = F.silu
    for row in ids:
        n = int(((row >= 0) * torch.arange(1, len(row) + 1)).max())
        e = torch.stack([front.table[t] * math.sqrt(front.width) if t >= 0 else torch.zeros_like(front.table[0]) for t in row[:n]]) if n else None
        total = torch.zeros(front.width, dtype=torch.float64)
        if n:
            x, z = (e @ front.inputs.weight.t()).chunk(2, -1)
            line = torch.cat([torch.zeros(front.taps - 1, front.width, dtype=torch.float64), x])
            h = torch.zeros(front.width, front.states, dtype=torch.float64)
            a = -torch.exp(front.a_log)
            for t in range(n):
                u = silu(front.conv_bias + (front.conv_weight.t() * line[t:t + front.taps]).sum(0))
                dt, b, c = (front.select.weight @ u).split((front.rank, front.states, front.states))
                dt = F.softplus(front.spread.weight @ dt + front.dt_bias)
                h = torch.exp(dt[:, None] * a) * h + (dt * u)[:, None] * b
                total = total + ((h * c).sum(-1) + front.skip * u) * silu(z[t])
        out.append(total / max(n, 1))
    return torch.stack(out)


def plain_step(model, data, y):
    """(loss, err_loss grid) of the training step (multimodn/multimodn.py:137-202)."""
    state = model.init_state.state_value.expand(len(y), -1)
    grid, change = [], 0.0

    def errors(s):
        return torch.stack([F.cross_entropy(torch.sigmoid(d.fc(s)), y[:, i]) for i, d in enumerate(model.decoders)])

    grid.append(errors(state))
    for enc, x in zip(model.encoders, data):
        old = state
        state = mm.MLPEncoder.forward(enc, state, plain_features(enc.front, x) if isinstance(enc, mm.SequenceEncoder) else x.double())
        change = change + ((state - old) ** 2).mean()
        grid.append(errors(state))
    grid = torch.stack(grid)
    return grid.mean() * model.err_penalty + change / len(model.encoders) * model.state_change_penalty, grid


@gpu
@pytest.mark.parametrize("kind", ["hip", "torch"])
def test_training_step_against_64_bits(kind):
    """Gradients of every parameter, fronts and chain, and the weights after one Adam step.  A gradient sums at most ROWS * STEPS
    contributions (192), each off by some 3 * STEPS + 60 roundings of terms not over 8 times the largest sum: 300 * 2^-24 * 8 < 1.5e-4."""
    model = build()
    wide = copy.deepcopy(model).cpu().double()
    data, y = batch()
    opt = mm.optim.Adam(model.parameters(), 1e-2) if kind == "hip" else torch.optim.Adam(model.parameters(), 1e-2)
    hist = mm.MultiModNHistory(["a", "b"])
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    model.train_epoch([(data, y)], opt, torch.nn.CrossEntropyLoss(), hist)
    loss, grid = plain_step(wide, data, y)
    assert rel_err(hist.loss["train"][0], grid.detach().numpy()) < 1e-5
    grads = dict(zip((n for n, _ in wide.named_parameters()), torch.autograd.grad(loss, list(wide.parameters()))))
    for n, p in model.named_parameters():
        assert rel_err(p.grad.cpu().numpy(), grads[n].numpy()) < 1.5e-4, n
        # Adam's first step is lr * g / (|g| + 1e-8), whose slope is 1e-8 / (|g| + 1e-8)^2: an error of d = 1.5e-4 G (G the largest) moves it
        # by at most d times the slope at |g| - d, and by 2 at most; the weight's own rounding (2^-24 of a weight under 4) is 2.4e-7
        g, moved = grads[n], (p.detach() - before[n]).cpu().double()
        d = 1.5e-4 * g.abs().max()
        allowed = 1e-2 * (d * 1e-8 / ((g.abs() - d).clamp(min=0) + 1e-8) ** 2).clamp(max=2.0) + 3e-7
        assert ((moved + 1e-2 * g / (g.abs() + 1e-8)).abs() <= allowed).all(), n


@gpu
def test_training_goes_on_and_entry_points_agree():
    model = build(seed=3)
    opt = mm.optim.Adam(model.parameters(), 3e-3)
    crit = torch.nn.CrossEntropyLoss()
    batches = [batch(s, rows) for s, rows in ((1, 16), (2, 33), (3, 7))]
    hist = mm.MultiModNHistory(["a", "b"])
    grads = None
    for _ in range(3):
        model.train_epoch(batches, opt, crit, hist)
        now = [p.grad.data_ptr() for p in model.parameters()]
        fronts = [p.grad.data_ptr() for e in model.encoders if isinstance(e, mm.SequenceEncoder) for p in e.front.parameters()]
        assert grads is None or fronts == grads
        grads = fronts
        assert len(set(now)) == len(now)
    assert np.isfinite(np.array(hist.loss["train"])).all()
    # a model of plain MLPEncoders with the same weights gives the same results on the features
    data, y = batches[1]
    with torch.no_grad():
        feats = [e.front(x.cuda()) if isinstance(e, mm.SequenceEncoder) else x.cuda() for e, x in zip(model.encoders, data)]
    plain = mm.MultiModN(S, [mm.MLPEncoder(S, e.n_features, e.hidden_layers, e.activation) for e in model.encoders],
                         [mm.LogisticDecoder(S), mm.LogisticDecoder(S)], 0.7, 0.4, device=torch.device("cuda"))
    plain.load_state_dict({k: v for k, v in model.state_dict().items() if ".front." not in k})
    assert np.array_equal(model.predict(data), plain.predict(feats))
    for p, q in zip(model.get_states([(data, y)]), plain.get_states([(feats, y.cuda())])):
        assert torch.equal(p, q)
    for r, s in zip(model.test([(data, y)], crit), plain.test([(feats, y.cuda())], crit)):
        for a, b in zip(r, s):
            assert torch.allclose(torch.as_tensor(a), torch.as_tensor(b), rtol=0, atol=0, equal_nan=True)
    again = pickle.loads(pickle.dumps(model))
    assert np.array_equal(again.predict(data), model.predict(data))


@gpu
def test_encoder_sequences():
    """An encoder outside the sequence has no gradient, front and chain."""
    model = build(seed=4)
    opt = torch.optim.SGD(model.parameters(), 1e-2)
    data, y = batch(5)
    order = torch.tensor([[2, 1]]).expand(ROWS, -1)
    model.train_epoch([([data[2], data[1]], y, order)], opt, torch.nn.CrossEntropyLoss())
    assert all(p.grad is None for p in model.encoders[0].parameters())
    assert all(p.grad is not None and p.grad.abs().max() > 0 for p in model.encoders[2].front.parameters())


@gpu
def test_fronts_that_share_a_table():
    """Its gradient is the sum of both encoders' (each sum rounded once: half a step of fp32), or the one's that ran."""
    def twin(tied, encoders):
        torch.manual_seed(8)
        encs = [mm.SequenceEncoder(S, V, WIDTH, (16,), states=8), mm.SequenceEncoder(S, V, WIDTH, (8,), states=4)]
        encs[1].front.table.data.copy_(encs[0].front.table.data)
        if tied:
            encs[1].front.table = encs[0].front.table
        model = mm.MultiModN(S, encs, [mm.LogisticDecoder(S)], 0.7, 0.4, device=torch.device("cuda"))
        data, y = batch(5)
        order = torch.tensor([encoders]).expand(ROWS, -1)
        model.train_epoch([([data[0]] * len(encoders), y[:, :1], order)], torch.optim.SGD(model.parameters(), 0.0), torch.nn.CrossEntropyLoss())
        return [e.front.table.grad for e in encs]

    for order in ([0, 1], [1], [0]):
        apart, tied = twin(False, order), twin(True, order)
        want = sum(g.double() for g in apart if g is not None)
        assert tied[0] is tied[1] and torch.all((tied[0].double() - want).abs() <= 2.0 ** -24 * want.abs())


@gpu
def test_ids_from_the_packages_datasets():
    """PartitionDataset, a stock DataLoader and DeviceResidentLoader hand ids over as float32: the same training as from whole numbers; a NaN
    skips the encoder."""
    (a, x, b), y = batch(5, 32)
    results = []
    packed = mm.PartitionDataset(torch.cat([a.float(), x, b.float()], 1).numpy(), y.numpy(), [STEPS, 6, 5])
    loaders = [[([a[i:i + 16], x[i:i + 16], b[i:i + 16]], y[i:i + 16]) for i in (0, 16)], torch.utils.data.DataLoader(packed, 16),
               mm.DeviceResidentLoader(packed, 16), [([a[i:i + 16].int().cuda(), x[i:i + 16].cuda(), b[i:i + 16].half()], y[i:i + 16]) for i in (0, 16)]]
    for loader in loaders:
        model = build(seed=4)
        model.train_epoch(loader, mm.optim.Adam(model.parameters(), 1e-3), torch.nn.CrossEntropyLoss())
        results.append([p.detach().clone() for p in model.parameters()])
    for other in results[1:]:
        assert all(torch.equal(p, q) for p, q in zip(results[0], other))
    gone = a.float()
    gone[3, 0] = float("nan")
    model.train_epoch([([gone, x, b], y)], torch.optim.SGD(model.parameters(), 1e-2), torch.nn.CrossEntropyLoss())
    assert all(p.grad is None for p in model.encoders[0].parameters())
    assert all(torch.isfinite(p.grad).all() for e in (1, 2) for p in model.encoders[e].parameters())


@gpu
def test_missing_values_in_another_slot():
    """A NaN batch of the tabular modality skips its encoder; the sequence encoders train."""
    model = build(seed=6)
    opt = torch.optim.SGD(model.parameters(), 1e-2)
    data, y = batch(7)
    data[1][3, 2] = float("nan")
    model.train_epoch([(data, y)], opt, torch.nn.CrossEntropyLoss())
    assert all(p.grad is None for p in model.encoders[1].parameters())
    assert all(torch.isfinite(p.grad).all() for e in (0, 2) for p in model.encoders[e].parameters())


@gpu
def test_features_token_by_token():
    """step() after the n-th token = forward() of the first n tokens.  Both round each step's states and outputs alike but the projections are
    other products of the library: 32 bits, sums of 24 terms, 12 steps: under 200 roundings, terms up to 8 times the largest feature."""
    model = build(seed=8)
    front = model.encoders[0].front
    ids = torch.randint(0, V, (5, STEPS), generator=torch.Generator().manual_seed(9)).cuda()
    ids[2, 3] = -1                                                            # a step without a token
    state = front.start(5)
    for t in range(STEPS):
        got = front.step(ids[:, t], state)
        with torch.no_grad():
            want = front(ids[:, :t + 1])
        rows = [0, 1, 3, 4] if t == 3 else slice(None)                        # (forward: a row ends behind its last token)
        assert rel_err(got[rows].cpu(), want[rows].cpu()) < 200 * 2.0 ** -24 * 8, t


@gpu
def test_input_gradient():
    lib = hip.load()
    g = torch.Generator().manual_seed(10)
    for rows, hidden, width in ((1, 1, 1), (33, 128, 65), (100, 7, 300), (4096, 32, 64)):
        d, w = torch.randn(rows, hidden, generator=g).cuda(), torch.randn(hidden, width, generator=g).cuda()
        dx = torch.empty(rows, width, device="cuda")
        assert lib.mmn_seq_input_grad(d.data_ptr(), w.data_ptr(), dx.data_ptr(), rows, hidden, width, torch.cuda.current_stream().cuda_stream) == 0
        want, mag = d.cpu().double() @ w.cpu().double(), d.cpu().double().abs() @ w.cpu().double().abs()
        assert ((dx.cpu().double() - want).abs() <= (hidden + 1) * 2.0 ** -24 * mag).all()
    assert lib.mmn_seq_input_grad(d.data_ptr(), w.data_ptr(), dx.data_ptr(), 4, 129, 4, None) == -1


# ---- refusals (CPU)
def test_refusals():
    with pytest.raises(ValueError):
        mm.SequenceEncoder(8, 10, 4, ())
    for bad in (dict(states=0), dict(states=33), dict(taps=5), dict(taps=1)):
        with pytest.raises(ValueError):
            mm.SequenceFeatures(10, 4, **bad)
    front = mm.SequenceFeatures(10, 4)
    for ids in (torch.zeros(3), torch.zeros(2, 3, dtype=torch.bool), torch.zeros(2, 3, 4, dtype=torch.int64)):
        with pytest.raises(ValueError):
            front(ids)
    with pytest.raises(hip.MmnError):
        front(torch.zeros(2, 3, dtype=torch.int64))
    model = build("cpu")
    model.per_sample = True
    data, y = batch()
    for call in (lambda: model.train_epoch([(data, y)], torch.optim.SGD(model.parameters(), 0.1), torch.nn.CrossEntropyLoss()),
                 lambda: model.test([(data, y)], torch.nn.CrossEntropyLoss()), lambda: model.predict(data), lambda: model.get_states([(data, y)])):
        with pytest.raises(mm.UnsupportedModelError):
            call()


def test_fronts_with_the_chains_parameters_are_refused():
    def attempts(model):
        data, y = batch()
        for call in (lambda: model.train_epoch([(data, y)], torch.optim.SGD(model.parameters(), 0.1), torch.nn.CrossEntropyLoss()),
                     lambda: model.test([(data, y)], torch.nn.CrossEntropyLoss()), lambda: model.predict(data)):
            with pytest.raises(mm.UnsupportedModelError):
                call()

    model = build("cpu")
    model.encoders[0].front.conv_bias = model.encoders[0].front.skip = model.encoders[0].layers[0].bias
    attempts(model)
    model = build("cpu")
    model.encoders[0].front.skip = model.decoders[0].fc.bias
    attempts(model)
    model = build("cpu")
    model.encoders[2].front.half()
    attempts(model)


def test_state_dict_and_arch(capsys):
    enc = mm.SequenceEncoder(S, V, WIDTH, (16,))
    assert {"front.table", "front.conv_weight", "front.a_log", "layers.0.weight"} <= set(enc.state_dict())
    model = build("cpu")
    model.display_arch([np.zeros(STEPS), np.zeros(6), np.zeros(5)])
    assert "Encoder 2:" in capsys.readouterr().out
