"""Calls of the sequence operators that their documentation allows and that once answered wrongly or were refused."""
import os

import pytest
import torch

import sequence_oracle as O
import multimodn_amd as mm
from multimodn_amd import hip, sequence as seq
from test_sequence import normal, rng

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("gated", [True, False])
def test_one_step_of_channels_in_front(dtype, gated):
    """[batch, width, 1] turned to [batch, 1, width]: a step's stride is 1, which no other step uses.  As the dense copies, every gradient."""
    g = rng(40)
    B, W, N = 5, 70, 6
    turned = lambda: normal(g, B, W, 1, dtype=dtype).transpose(1, 2)
    x, dt, dy = turned(), turned(), turned()
    z = turned() if gated else None
    assert x.stride() == (W, 1, 1)
    a, d, bias = -torch.rand(W, N, generator=g).cuda() - 0.1, normal(g, W), normal(g, W)
    b, c, s, ds = normal(g, B, 1, N, dtype=dtype), normal(g, B, 1, N, dtype=dtype), normal(g, B, W, N), normal(g, B, W, N)
    copy = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device="cuda").copy_(t)

    def both(x, dt, z, dy):
        y, out, saved = seq.selective_scan_forward(x, dt, a, b, c, d, z, bias, state=s, return_state=True)
        return (y, out) + tuple(seq.selective_scan_grad(dy, saved, ds))

    dense = [copy(t) for t in (x, dt, z, dy)]
    assert dense[0].stride() == (W, W, 1)
    want = O.scan(x, dt, a, b.unsqueeze(2), c.unsqueeze(2), d, z, bias, True, None, s, dy, ds)
    for got in (both(*dense), both(x, dt, z, dy), both(dense[0], dense[1], dense[2], dy), both(x, dt, z, dense[3])):
        for p, q in zip(got, both(*dense)):
            assert (p is None and q is None) or torch.equal(p, q)
        # d(d) is B products of dy, the gate and x: two roundings each in the gate, one in each product and sum
        O.check(got[7], *want["d"], B + 8, "dd")
    conv = normal(g, W, 4)
    for p, q in zip(seq.causal_conv_grad(dy, x, conv, bias), seq.causal_conv_grad(dense[3], dense[0], conv, bias)):
        assert (p is None and q is None) or torch.equal(p, q)
    leaf = dense[0].clone().requires_grad_(True)                              # a gradient that autograd itself hands over in this layout
    skip = d.clone().requires_grad_(True)
    y = seq.selective_scan(leaf, dense[1], a, b, c, skip, dense[2], bias)
    (grad,) = torch.autograd.grad(y.transpose(1, 2), skip, dy.transpose(1, 2))
    y, _, saved = seq.selective_scan_forward(dense[0], dense[1], a, b, c, d, dense[2], bias)
    assert torch.equal(grad, seq.selective_scan_grad(dense[3], saved).d)


@gpu
def test_one_step_does_not_read_other_channels():
    """An infinity in one channel stays there."""
    g = rng(41)
    x = normal(g, 2, 9, 1)
    x[:, 4] = float("inf")
    x = x.transpose(1, 2)
    dt, b = normal(g, 2, 1, 9), normal(g, 2, 1, 3)
    y, state = seq.selective_scan(x, dt, -torch.ones(9, 3, device="cuda"), b, b, return_state=True)
    others = [0, 1, 2, 3, 5, 6, 7, 8]
    assert torch.isfinite(y[..., others]).all() and torch.isfinite(state[:, others]).all()


@gpu
def test_one_step_or_none_with_any_stride():
    """The stride of a dimension of one step, or of none, is never used: one step of a large time-major batch, no steps of channels in front."""
    g = rng(42)
    B, W = 66000, 128                                                         # B * W > 2^23
    x, dt = normal(g, 1, B, W).transpose(0, 1), normal(g, 1, B, W).transpose(0, 1)
    b = normal(g, B, 1, 2)
    a = -torch.ones(W, 2, device="cuda")
    assert x.stride(1) > 1 << 23
    y, _, saved = seq.selective_scan_forward(x, dt, a, b, b)
    dense = [torch.empty(B, 1, W, device="cuda").copy_(t) for t in (x, dt)]
    y2, _, saved2 = seq.selective_scan_forward(*dense, a, b, b)
    assert torch.equal(y, y2)
    assert all(torch.equal(p, q) for p, q in zip(seq.selective_scan_grad(x, saved), seq.selective_scan_grad(dense[0], saved2)) if p is not None)
    none = torch.zeros(4, W, 0, device="cuda").transpose(1, 2)
    s = normal(g, 4, W, 2)
    y, out = seq.selective_scan(none, none, a, b[:4, :0], b[:4, :0], state=s, return_state=True)
    assert y.shape == (4, 0, W) and torch.equal(out, s)


@gpu
@pytest.mark.parametrize("growth", [0.5, 4.0])
@pytest.mark.parametrize("rows,steps,states", [(1, 2000, 3), (1, 4096, 16), (300, 300, 3), (40, 250, 5), (2, 100, 30)])
def test_states_that_grow_from_zero(rows, steps, states, growth):
    """a > 0: while nothing has come in a state stays 0, in however many segments the steps are walked; the same backwards behind the last
    gradient.  All rows are alike: the statement is made for one."""
    g = rng(43)
    D = 6
    x, dy, dt = torch.zeros(1, steps, D), torch.zeros(1, steps, D), torch.ones(1, steps, D)
    x[:, -3:], dy[:, :3] = torch.randn(1, 3, D, generator=g), torch.randn(1, 3, D, generator=g)
    b, c = torch.randn(1, steps, states, generator=g), torch.randn(1, steps, states, generator=g)
    a = torch.full((D, states), growth)
    want = O.scan(x, dt, a, b.unsqueeze(2), c.unsqueeze(2), None, None, None, False, None, None, dy)
    case = [t.expand(rows, *t.shape[1:]).cuda() for t in (x, dt, b, c, dy)]
    y, state, saved = seq.selective_scan_forward(case[0], case[1], a.cuda(), case[2], case[3], softplus=False, return_state=True)
    grads = seq.selective_scan_grad(case[4], saved)
    n = 3 * 3 + 12 + states + 24                                              # (three steps with anything in them; as scan_terms of the other tests)
    for i in (0, rows - 1):
        O.check(y[i:i + 1], *want["y"], n, "y")
        O.check(state[i:i + 1], *want["state"], n, "state")
        for name in ("x", "dt"):
            O.check(getattr(grads, name)[i:i + 1], *want[name], 2 * n, "d" + name)
        for name in ("b", "c"):
            O.check(getattr(grads, name)[i:i + 1], *want[name], 2 * n + D, "d" + name)
    assert not grads.a.any()                                                  # (every product of a gradient and a state is 0)


fence = pytest.mark.skipif(os.environ.get("MMN_EFENCE", "0") not in ("", "0"), reason="the electric fence's allocator fills new memory, which a capture does not allow")


@gpu
@fence
@pytest.mark.parametrize("where", ["default", "side"])
def test_captures_refuse_what_another_stream_holds(where):
    """A leaf, or a tensor that comes from one, whose autograd graph was made outside the capture: refused before anything is recorded for
    autograd.  Without gradients, and once those graphs are gone, the same calls are captured."""
    g = rng(44)
    B, L, D, N = 2, 9, 16, 4
    source = normal(g, B, L, D).requires_grad_(True)
    w, a = normal(g, D, 3).requires_grad_(True), (-torch.rand(D, N, generator=g).cuda()).requires_grad_(True)
    b = normal(g, B, L, N)
    stream = torch.cuda.Stream() if where == "side" else torch.cuda.current_stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        x = source * 2                                                        # made outside: a node and, behind it, a leaf's accumulator
        held = (w * 1, a * 1)
    torch.cuda.synchronize()
    dense = normal(g, B, L, D)
    for call in (lambda: seq.causal_conv(dense, w), lambda: seq.causal_conv(x, w.detach()), lambda: seq.selective_scan(dense, dense, a, b, b),
                 lambda: seq.selective_scan(dense, x, a.detach(), b, b), lambda: seq.selective_scan(source * 3, dense, a.detach(), b, b),
                 lambda: seq.causal_conv(dense, torch.exp(w))):
        with pytest.raises(hip.MmnError, match="drop its"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        torch.cuda.synchronize()
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = seq.causal_conv(x, w)
        graph.replay()
        assert torch.equal(y, seq.causal_conv(x, w))
    del held, x, graph
    call = lambda: torch.autograd.grad(seq.causal_conv(source * 2, torch.exp(w)), (source, w), dense)
    want = [t.clone() for t in call()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for turn in range(3):
        for t in got:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), turn


@gpu
@fence
def test_captures_of_a_front_refuse_what_another_stream_holds():
    """SequenceFeatures with a frozen table: its projections' weights are the leaves that an eager graph holds."""
    torch.manual_seed(45)
    front = mm.SequenceFeatures(20, 16, states=4, device="cuda")
    front.table.requires_grad_(False)
    ids = torch.randint(0, 20, (3, 9), generator=rng(45)).cuda()
    features = front(ids)
    torch.cuda.synchronize()
    with pytest.raises(hip.MmnError, match="drop its"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            front(ids)
    torch.cuda.synchronize()
    assert torch.equal(features, front(ids))


def test_one_step_forms_refuse_operands_inside_the_state():
    """The step writes the state while other threads read their operands: x, b or a parameter that lies in it would be read before or after."""
    z = torch.zeros
    conv, scan = z(2, 3, 6), z(2, 6, 3)
    w, a, x, b = z(6, 4), z(6, 3), z(2, 6), z(2, 3)
    for call in (lambda: seq.causal_conv_step(conv[:, 2], w, state=conv), lambda: seq.causal_conv_step(x, conv.view(-1)[:24].view(6, 4), state=conv),
                 lambda: seq.causal_conv_step(x, w, conv[0, 0], state=z(2, 3, 6), out_state=conv),
                 lambda: seq.selective_scan_step(scan.view(2, 18)[:, :6], x, a, b, b, state=scan), lambda: seq.selective_scan_step(x, x, a, scan[:, 0], b, state=scan),
                 lambda: seq.selective_scan_step(x, x, scan[0], b, b, state=scan), lambda: seq.selective_scan_step(x, x, a, b, b, state=z(2, 6, 3), out_state=scan, z=scan.view(2, 18)[:, 12:])):
        with pytest.raises(ValueError, match="shares memory"):
            call()
    both = z(36 + 12)                                                         # side by side in one buffer is no overlap: only the CPU is refused
    with pytest.raises(hip.MmnError):
        seq.causal_conv_step(both[36:].view(2, 6), w, state=both[:36].view(2, 3, 6))


@gpu
@pytest.mark.parametrize("rows,steps", [(4, 30), (1, 2000), (1000, 20)])
def test_states_of_one_step(rows, steps):
    """a = -inf: nothing of a state is left at the next step, h = dt' x b.  Rows of every length, in segments and whole, and one step on."""
    g = rng(46)
    D, N = 10, 5
    x, dt, b, c, h0 = normal(g, rows, steps, D), normal(g, rows, steps, D), normal(g, rows, steps, N), normal(g, rows, steps, N), normal(g, rows, D, N)
    lengths = torch.randint(0, steps + 1, (rows,), generator=g)
    lengths[0] = steps // 2 + 1
    a = torch.full((D, N), -float("inf"), device="cuda")
    y, state = seq.selective_scan(x, dt, a, b, c, lengths=lengths.cuda(), state=h0, return_state=True)
    there = torch.arange(steps) < lengths[:, None]
    wide = [t.cpu().double() for t in (x, dt, b, c)]
    step = torch.nn.functional.softplus(wide[1])
    h = (step * wide[0])[..., None] * wide[2][:, :, None]
    want = torch.where(there[..., None], (h * wide[3][:, :, None]).sum(-1), 0.0)
    mag = ((step + torch.sigmoid(wide[1]) * wide[1].abs()) * wide[0].abs())[..., None] * (wide[2] * wide[3]).abs()[:, :, None]
    O.check(y, want, mag.sum(-1), N + 12, "y")
    ends = (lengths - 1).clamp(min=0)
    last = torch.where((lengths > 0)[:, None, None], h[torch.arange(rows), ends], h0.cpu().double())
    last_mag = ((step + torch.sigmoid(wide[1]) * wide[1].abs()) * wide[0].abs())[..., None] * wide[2].abs()[:, :, None]
    O.check(state, last, last_mag[torch.arange(rows), ends], 12, "state")
    for t in (0, 1):
        out = seq.selective_scan_step(x[:, t], dt[:, t], a, b[:, t], c[:, t], state=state)
        O.check(state, h[:, t], last_mag[:, t], 12, "state of a step")
        O.check(out, (h * wide[3][:, :, None]).sum(-1)[:, t], mag.sum(-1)[:, t], N + 12, "y of a step")


@gpu
@pytest.mark.parametrize("rows,steps,growth", [(1000, 300, 1.0), (9000, 200, 1.0), (3, 300, 1.0), (3, 300, 200.0), (1000, 40, 200.0)])
def test_growing_states_of_few_channels(rows, steps, growth):
    """Six channels of a wave's 64 lanes, a > 0 and steps so small that nothing grows much: the lanes without a channel, whose step would be
    softplus(0), add nothing to the gradients of b and c.  All rows are alike."""
    g = rng(47)
    D, N = 6, 3
    x, dy = torch.randn(1, steps, D, generator=g), torch.randn(1, steps, D, generator=g)
    dt = torch.full((1, steps, D), -10.0)
    b, c = torch.randn(1, steps, N, generator=g), torch.randn(1, steps, N, generator=g)
    a, h0, ds = torch.full((D, N), growth), torch.randn(1, D, N, generator=g), torch.randn(1, D, N, generator=g)
    want = O.scan(x, dt, a, b.unsqueeze(2), c.unsqueeze(2), None, None, None, True, None, h0, dy, ds)
    case = [t.expand(rows, *t.shape[1:]).contiguous().cuda() for t in (x, dt, b, c, h0, dy, ds)]
    y, state, saved = seq.selective_scan_forward(case[0], case[1], a.cuda(), case[2], case[3], state=case[4], return_state=True)
    grads = seq.selective_scan_grad(case[5], saved, case[6])
    n = 3 * steps + 12 + N + 24
    for i in (0, rows - 1):
        O.check(y[i:i + 1], *want["y"], n, "y")
        for name in ("x", "dt", "b", "c", "state"):
            O.check(getattr(grads, name)[i:i + 1], *want["dstate" if name == "state" else name], 2 * n + D, "d" + name)
