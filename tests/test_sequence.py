"""The sequence operators (multimodn_amd.sequence) against their 64-bit statements (sequence_oracle), and what they refuse."""
import math
import os

import pytest
import torch

import sequence_oracle as O
from multimodn_amd import hip, sequence as seq

TYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


def rng(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, device="cuda"):
    return torch.randn(*shape, generator=g).to(dtype).to(device)


# ---------------------------------------------------------------------------------------------------------------- embedding
EMBED = [  # ids shape, vocabulary, width
    ((1,), 1, 1), ((16, 1), 1000, 64), ((5, 7), 11, 3), ((33,), 300, 130), ((2, 3, 4), 70000, 66), ((700,), 5, 513), ((4097,), 2000, 8), ((9000,), 300000, 5), ((0,), 9, 4),
    ((8192,), 1501, 203), ((64, 128), 64, 64), ((1025,), 8192, 200), ((8193,), 1501, 66), ((5000,), 60000, 9), ((300,), 500, 4225), ((4000,), 40000, 130),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,vocab,width", EMBED)
def test_embedding_and_its_gradient(shape, vocab, width, dtype):
    g = rng(1)
    scale = math.sqrt(width)
    ids = torch.randint(-2, vocab + 2, shape, generator=g)                  # some outside the vocabulary on both sides
    if len(shape) == 1 and shape[0] > 100:
        ids[: shape[0] // 3] = vocab // 2                                     # one token with a third of the places
    w = normal(g, vocab, width, dtype=dtype)
    dy = normal(g, *shape, width, dtype=dtype)
    for kind in (torch.int64, torch.int32):
        there = ids.to(kind).cuda()
        y = seq.embedding(there, w, scale)
        want = O.embed(ids, w, scale)
        O.check(y, want, want.abs(), 2, "y")                                  # the scale's own rounding and the product's
        dw = seq.embedding_grad(dy, there, vocab, scale)
        want, mag, count = O.embed_grad(dy, ids, vocab, scale)
        O.check(dw, want, mag, (count + 2)[:, None].double(), "gradient")
        assert torch.equal(dw, seq.embedding_grad(dy, there, vocab, scale))


@gpu
def test_embedding_gradient_of_many_places_and_of_one_token():
    """More places than the sort's workgroups hold in one tile each, and every place the same token (all partial sums join)."""
    for n, vocab, same in ((4096 * 130 + 77, 40, False), (300000, 700, True)):
        ids = torch.randint(0, vocab, (n,), generator=rng(2)) if not same else torch.full((n,), 699)
        grad = normal(rng(3), n, 2)
        got = seq.embedding_grad(grad, ids.cuda(), vocab, 0.5)
        want, mag, count = O.embed_grad(grad, ids, vocab, 0.5)
        O.check(got, want, mag, (count + 2)[:, None].double(), f"{n} places")


@gpu
@pytest.mark.parametrize("rows", [1, 63, 1024, 8192, 8193])
def test_embedding_gradient_of_ids_that_name_no_row(rows):
    grad = torch.full((rows, 70), float("nan"), device="cuda")
    for vocab in (3, 700, 60000):
        assert not seq.embedding_grad(grad, torch.full((rows,), -1, device="cuda"), vocab).any()
        ids = torch.full((rows,), vocab, device="cuda")
        ids[rows // 2] = vocab - 1
        grad[rows // 2] = 1.0
        got = seq.embedding_grad(grad, ids, vocab, 2.0)
        assert not got[:-1].any() and torch.equal(got[-1], torch.full((70,), 2.0, device="cuda"))


@gpu
def test_embedding_autograd_and_views():
    g = rng(4)
    base = normal(g, 50, 12)
    w = base[::2, 1:9].clone().requires_grad_(True)                            # (its values; the op takes any table, copied where it is not dense)
    ids = torch.randint(0, 25, (6, 4), generator=g).cuda().t()                # not contiguous
    y = seq.embedding(ids, w, 3.0)
    assert torch.equal(y, seq.embedding(ids.contiguous(), base[::2, 1:9], 3.0))
    dy = normal(g, 4, 6, 8)
    y.backward(dy)
    want, mag, count = O.embed_grad(dy, ids, 25, 3.0)
    O.check(w.grad, want, mag, (count + 2)[:, None].double(), "gradient")
    (grad,) = torch.autograd.grad(seq.embedding(ids, w, 3.0).sum(), w)        # an expanded gradient
    want, mag, count = O.embed_grad(torch.ones(4, 6, 8), ids, 25, 3.0)
    O.check(grad, want, mag, (count + 2)[:, None].double(), "gradient of a sum")


# -------------------------------------------------------------------------------------------------------------- convolution
CONV = [  # batch, steps, width, taps, lengths, state, bias, silu
    (1, 1, 1, 2, None, False, False, True), (3, 2, 5, 4, [2, 0, 1], True, True, True), (2, 17, 64, 3, None, True, True, False),
    (5, 33, 130, 4, [33, 0, 1, 16, 32], True, True, True), (2, 100, 1030, 4, [3, 100], False, True, True), (300, 3, 8, 2, None, False, True, True),
    (2, 50, 12, 4, [99, -5], True, True, True),
]


def conv_case(case, dtype, seed=5):
    B, L, D, K, lengths, state, bias, silu = case
    g = rng(seed)
    x = normal(g, B, L, 2 * D, dtype=dtype)[..., :D]                          # a strided half
    w, b = normal(g, D, K) / K, normal(g, D) if bias else None
    s = normal(g, B, K - 1, D, dtype=dtype) if state else None
    n = torch.tensor(lengths).cuda() if lengths else None
    dy, ds = normal(g, B, L, D, dtype=dtype), normal(g, B, K - 1, D, dtype=dtype)
    return x, w, b, "silu" if silu else None, n, s, dy, ds


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", CONV, ids=str)
def test_conv_and_its_gradients(case, dtype):
    x, w, b, act, n, s, dy, ds = conv_case(case, dtype)
    B, L, D = x.shape
    K = w.shape[1]
    y, out = seq.causal_conv(x, w, b, activation=act, lengths=n, state=s, return_state=True)
    want = O.conv(x, w, b, act is not None, n, s, dy, ds)
    O.check(y, *want["y"], K + 8, "y")
    O.check(out, *want["state"], 0, "state")
    g = seq.causal_conv_grad(dy, x, w, b, activation=act, lengths=n, state=s, state_grad=ds)
    O.check(g.x, *want["x"], 2 * K + 12, "dx")
    O.check(g.weight, *want["weight"], K + 12 + B * L, "dweight")
    O.check(g.bias, *want["bias"], K + 12 + B * L, "dbias")
    if s is not None:
        O.check(g.state, *want["dstate"], 2 * K + 12, "dstate")
    again = seq.causal_conv_grad(dy, x, w, b, activation=act, lengths=n, state=s, state_grad=ds)
    assert all(torch.equal(p, q) for p, q in zip(g, again) if p is not None)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_conv_does_not_read_behind_the_end(dtype):
    x, w, b, act, n, s, dy, ds = conv_case((3, 20, 16, 4, [0, 7, 20], True, True, True), dtype)
    x2, dy2 = x.clone(), dy.clone()
    for i, k in enumerate((0, 7, 20)):
        x2[i, k:], dy2[i, k:] = float("nan"), float("inf")
    for p, q in zip((x, dy), (x2, dy2)):
        assert p.shape == q.shape
    one = seq.causal_conv(x, w, b, lengths=n, state=s, return_state=True) + seq.causal_conv_grad(dy, x, w, b, lengths=n, state=s)
    two = seq.causal_conv(x2, w, b, lengths=n, state=s, return_state=True) + seq.causal_conv_grad(dy2, x2, w, b, lengths=n, state=s)
    assert all(torch.equal(p, q) for p, q in zip(one, two))


@gpu
@pytest.mark.parametrize("taps", [2, 3, 4])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_conv_in_parts_and_steps(taps, dtype):
    """A sequence in one call = its beginning, then the rest from the kept state = step by step."""
    g = rng(6)
    x, w, b = normal(g, 3, 11, 24, dtype=dtype), normal(g, 24, taps), normal(g, 24)
    whole, end = seq.causal_conv(x, w, b, return_state=True)
    first, state = seq.causal_conv(x[:, :1], w, b, return_state=True)
    rest, state2 = seq.causal_conv(x[:, 1:], w, b, state=state, return_state=True)
    assert torch.equal(whole, torch.cat([first, rest], 1)) and torch.equal(end, state2)
    state = torch.zeros(3, taps - 1, 24, dtype=dtype, device="cuda")
    other = torch.empty_like(state)
    for t in range(11):
        if t % 2:
            y = seq.causal_conv_step(x[:, t], w, b, state=state, out_state=other)
            state, other = other, state
        else:
            y = seq.causal_conv_step(x[:, t], w, b, state=state)
        assert torch.equal(y, whole[:, t])
    assert torch.equal(state, end)


# --------------------------------------------------------------------------------------------------------------------- scan
SCAN = [  # batch, steps, width, groups, states, lengths, state, z, d, dt_bias, softplus
    (1, 1, 1, 1, 1, None, False, False, False, False, True), (2, 5, 6, 2, 3, [0, 5], True, True, True, True, True),
    (3, 33, 64, 1, 16, [33, 32, 1], False, True, True, True, True), (2, 70, 130, 1, 16, [70, 37], True, True, True, True, True),
    (1, 129, 72, 3, 8, None, True, True, False, True, True), (2, 64, 320, 2, 20, [64, 40], True, True, True, True, True),
    (2, 40, 66, 1, 32, None, True, False, True, False, True), (1, 200, 300, 1, 4, [150], False, True, True, True, False),
    (40, 9, 65, 1, 16, None, True, True, True, True, True), (1100, 3, 70, 1, 5, "ragged", True, True, True, True, True),
    (2100, 2, 36, 6, 8, None, False, True, True, True, True), (2, 48, 560, 1, 5, [-3, 1000], False, True, True, True, True),
    (90, 100, 64, 1, 16, "ragged", True, True, True, True, True), (60, 250, 40, 2, 6, None, True, False, True, True, True),
    (1, 2049, 30, 1, 4, None, True, True, True, True, True), (3, 1100, 20, 1, 3, [1100, 1, 555], False, True, True, True, True),
]


def scan_case(case, dtype, seed=7):
    B, L, D, G, N, lengths, state, z, d, dt_bias, softplus = case
    g = rng(seed)
    both = normal(g, B, L, 2 * G * N + 3, dtype=dtype)
    b, c = both[..., 3:3 + G * N].unflatten(-1, (G, N)), both[..., 3 + G * N:].unflatten(-1, (G, N))
    dt = (normal(g, B, L, D) * 0.5 if softplus else torch.rand(B, L, D, generator=g).cuda() * 0.1).to(dtype)
    return dict(x=normal(g, B, L, 2 * D, dtype=dtype)[..., D:], dt=dt, a=-(torch.rand(D, N, generator=g) * N + 0.05).cuda(), b=b, c=c,
                d=normal(g, D) if d else None, z=normal(g, B, L, D, dtype=dtype) if z else None,
                dt_bias=(normal(g, D) - 2.5) if dt_bias and softplus else None, softplus=softplus,
                lengths=(torch.randint(0, L + 1, (B,), generator=rng(seed)) if lengths == "ragged" else torch.tensor(lengths)).cuda() if lengths else None, state=normal(g, B, D, N) if state else None), \
        normal(g, B, L, D, dtype=dtype), normal(g, B, D, N)


def scan_terms(case):
    """Roundings on the longest way: a few for each step and state, and the sums over rows, steps and channels."""
    B, L, D, G, N = case[:5]
    state = 3 * L + 12                       # h: an exponential's, a product's and a sum's rounding each step
    return {"y": state + N + 8, "state": state, "one": 2 * state + N + 24, "channels": 2 * state + D // G + 24, "all": 2 * state + N + B * L + 24}


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", SCAN, ids=str)
def test_scan_and_its_gradients(case, dtype):
    args, dy, ds = scan_case(case, dtype)
    y, state = seq.selective_scan(**args, return_state=True)
    want = O.scan(**args, dy=dy, dstate_out=ds)
    n = scan_terms(case)
    O.check(y, *want["y"], n["y"], "y")
    O.check(state, *want["state"], n["state"], "state")
    y2, state2, saved = seq.selective_scan_forward(**args, return_state=True)
    assert torch.equal(y, y2) and torch.equal(state, state2)
    g = seq.selective_scan_grad(dy, saved, ds)
    for name, terms in (("x", "one"), ("dt", "one"), ("b", "channels"), ("c", "channels"), ("a", "all"), ("d", "all"), ("dt_bias", "all")):
        O.check(getattr(g, name), *want[name], n[terms], "d" + name)
    if args["z"] is not None:
        O.check(g.z, *want["z"], n["one"], "dz")
    if args["state"] is not None:
        O.check(g.state, *want["dstate"], n["one"], "dstate")
    again = seq.selective_scan_grad(dy, saved, ds)
    assert all(torch.equal(p, q) for p, q in zip(g, again) if p is not None)


@gpu
def test_scan_of_more_rows_than_fit_at_once():
    """A backward workgroup takes several rows in turn (above 8192 waves): every row as in a batch of its own, sums over all of them."""
    case = (9001, 2, 5, 1, 3, "ragged", True, True, True, True, True)
    args, dy, ds = scan_case(case, torch.float32)
    y, state, saved = seq.selective_scan_forward(**args, return_state=True)
    g = seq.selective_scan_grad(dy, saved, ds)
    n = scan_terms(case)
    rows = torch.tensor([0, 1, 700, 5000, 8191, 8192, 8193, 9000])
    some = {k: (v[rows.cuda()] if k in ("x", "dt", "b", "c", "z", "state", "lengths") else v) for k, v in args.items()}
    want = O.scan(**some, dy=dy[rows.cuda()], dstate_out=ds[rows.cuda()])
    for name in ("x", "dt", "b", "c", "z", "state"):
        O.check(getattr(g, name)[rows.cuda()], *want["dstate" if name == "state" else name], n["one"], "d" + name)
    # sums over the batch from the kernel's own per-row gradients: of d(dt_bias) directly, of the others by parts of 4500 rows
    O.check(g.dt_bias, g.dt.double().sum((0, 1)).cpu(), g.dt.double().abs().sum((0, 1)).cpu(), 2 * 9001 + 24, "d(dt_bias)")
    parts = []
    for part in (slice(0, 4500), slice(4500, 9001)):
        cut = {k: (v[part] if k in ("x", "dt", "b", "c", "z", "state", "lengths") else v) for k, v in args.items()}
        _, _, s = seq.selective_scan_forward(**cut)
        parts.append(seq.selective_scan_grad(dy[part], s, ds[part]))
    mag = O.scan(**some, dy=dy[rows.cuda()], dstate_out=ds[rows.cuda()])           # (the size of one row's terms, from eight of them)
    for name in ("a", "d"):
        total = sum(getattr(p, name).double().cpu() for p in parts)
        O.check(getattr(g, name), total, total.abs() + mag[name][1] * 9001 / 8, 64, "d" + name)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_scan_does_not_read_behind_the_end(dtype):
    case = (3, 70, 40, 1, 16, [0, 33, 70], True, True, True, True, True)
    args, dy, ds = scan_case(case, dtype)
    bad, dy2 = dict(args), dy.clone()
    for name in ("x", "dt", "b", "c", "z"):
        bad[name] = args[name].clone()
        for i, k in enumerate((0, 33, 70)):
            bad[name][i, k:] = float("nan")
            dy2[i, k:] = float("inf")
    y, state, saved = seq.selective_scan_forward(**args, return_state=True)
    y2, state2, saved2 = seq.selective_scan_forward(**bad, return_state=True)
    assert torch.equal(y, y2) and torch.equal(state, state2) and torch.equal(state[0], args["state"][0]) and not y[0].any()
    for p, q in zip(seq.selective_scan_grad(dy, saved, ds), seq.selective_scan_grad(dy2, saved2, ds)):
        assert torch.equal(p, q)


@gpu
@pytest.mark.parametrize("states", [1, 4, 6, 16, 32])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_scan_in_parts_and_steps(states, dtype):
    case = (2, 12, 24, 2, states, None, True, True, True, True, True)
    args, _, _ = scan_case(case, dtype)
    n = scan_terms(case)
    want = O.scan(**args)
    part = lambda lo, hi: {k: v[:, lo:hi] if k in ("x", "dt", "b", "c", "z") else v for k, v in args.items()}
    y1, s1 = seq.selective_scan(**part(0, 5), return_state=True)
    y2, s2 = seq.selective_scan(**{**part(5, 12), "state": s1}, return_state=True)
    O.check(torch.cat([y1, y2], 1), *want["y"], n["y"], "y in two parts")
    O.check(s2, *want["state"], n["state"], "state after two parts")
    state = args["state"].clone()
    other = torch.empty_like(state)
    for t in range(12):
        one = {k: (v[:, t] if k in ("x", "dt", "b", "c", "z") else v) for k, v in args.items() if k not in ("state", "lengths")}
        if t % 2:
            y = seq.selective_scan_step(**one, state=state, out_state=other)
            state, other = other, state
        else:
            y = seq.selective_scan_step(**one, state=state)
        O.check(y, want["y"][0][:, t], want["y"][1][:, t], n["y"], f"step {t}")
    O.check(state, *want["state"], n["state"], "state after the steps")


@gpu
def test_scan_long_and_wide_agree_with_parts():
    """Segments (few rows, many steps) against the same sequence row by row in pieces short enough to need none."""
    case = (1, 1000, 96, 1, 16, None, True, True, True, True, True)
    args, dy, ds = scan_case(case, torch.float32)
    n = scan_terms(case)
    want = O.scan(**args, dy=dy, dstate_out=ds)
    y, state, saved = seq.selective_scan_forward(**args, return_state=True)
    g = seq.selective_scan_grad(dy, saved, ds)
    O.check(y, *want["y"], n["y"], "y")
    O.check(g.x, *want["x"], n["one"], "dx")
    O.check(g.a, *want["a"], n["all"], "da")
    O.check(g.state, *want["dstate"], n["one"], "dstate")


@gpu
def test_layouts():
    """Time-major, expanded, transposed and sliced inputs give what their dense copies give."""
    g = rng(30)
    B, L, D, N = 3, 10, 20, 6
    x = normal(g, L, B, D).transpose(0, 1)                                     # time-major
    dt = normal(g, 1, L, D).expand(B, L, D)                                    # one row's for all
    z = normal(g, B, 1, D).expand(B, L, D)                                     # steps that share memory
    b, c = normal(g, B, N, L).transpose(1, 2), normal(g, B, L, 2 * N)[..., ::2]   # states far apart
    a, d, bias, w = -torch.rand(N, D, generator=g).cuda().t(), normal(g, 2 * D)[::2], normal(g, D), normal(g, 4, D).t()
    dy = normal(g, B, D, L).transpose(1, 2)
    s, cs = normal(g, B, N, D).transpose(1, 2), normal(g, B, D, 3).transpose(1, 2)
    dense = lambda *t: [v.contiguous() for v in t]
    one = seq.selective_scan_forward(x, dt, a, b, c, d, z, bias, state=s, return_state=True)
    two = seq.selective_scan_forward(*dense(x, dt, a, b, c, d, z, bias), state=s.contiguous(), return_state=True)
    assert all(torch.equal(p, q) for p, q in zip(one[:2], two[:2]))
    assert all(torch.equal(p, q) for p, q in zip(seq.selective_scan_grad(dy, one[2]), seq.selective_scan_grad(dy.contiguous(), two[2])))
    one = seq.causal_conv(x, w, bias, state=cs, return_state=True) + seq.causal_conv_grad(dy, x, w, bias, state=cs)
    two = seq.causal_conv(*dense(x, w, bias), state=cs.contiguous(), return_state=True) + seq.causal_conv_grad(*dense(dy, x, w, bias), state=cs.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    step = [x[:, 0], dt[:, 0], a, b[:, 0], c[:, 0], d, z[:, 0], bias]
    h1, h2 = s.contiguous(), s.contiguous().clone()
    assert torch.equal(seq.selective_scan_step(*step, state=h1), seq.selective_scan_step(*dense(*step), state=h2)) and torch.equal(h1, h2)
    c1, c2 = cs.contiguous(), cs.contiguous().clone()
    assert torch.equal(seq.causal_conv_step(x[:, 0], w, bias, state=c1), seq.causal_conv_step(*dense(x[:, 0], w, bias), state=c2)) and torch.equal(c1, c2)
    assert torch.equal(seq.embedding_grad(dy, torch.arange(30).view(3, 10).cuda() % 7, 7), seq.embedding_grad(dy.contiguous(), torch.arange(30).view(3, 10).cuda() % 7, 7))


@gpu
def test_backward_of_another_layout():
    """A forward pass over x whose steps lie 32 MB apart (rows in segments, for 32-bit offsets), the backward over its dense copy."""
    case = (900, 48, 6, 1, 4, "ragged", True, True, True, True, True)
    args, dy, ds = scan_case(case, torch.float32)
    far = torch.zeros(48, 1 << 23, device="cuda")[:, :6]
    far.copy_(args["x"][0])
    args["x"] = far.expand(900, 48, 6)
    y, state, saved = seq.selective_scan_forward(**args, return_state=True)
    g = seq.selective_scan_grad(dy, saved._replace(x=args["x"].contiguous()), ds)
    n = scan_terms(case)
    rows = torch.tensor([0, 1, 450, 899])
    some = {k: (v[rows.cuda()] if k in ("x", "dt", "b", "c", "z", "state", "lengths") else v) for k, v in args.items()}
    want = O.scan(**some, dy=dy[rows.cuda()], dstate_out=ds[rows.cuda()])
    O.check(y[rows.cuda()], *want["y"], n["y"], "y")
    for name in ("x", "dt", "b", "c", "z", "state"):
        O.check(getattr(g, name)[rows.cuda()], *want["dstate" if name == "state" else name], n["one"], "d" + name)
    for one, two in zip(g, seq.selective_scan_grad(dy, saved, ds)):            # and over the same: in segments
        assert torch.allclose(one, two, rtol=1e-3, atol=1e-3 * float(one.abs().max()))


@gpu
@pytest.mark.parametrize("width", [1, 6, 257])
def test_steps_of_odd_widths(width):
    g = rng(31)
    for dtype in TYPES:
        x, w = normal(g, 9, 2, width, dtype=dtype), normal(g, width, 3)
        y, end = seq.causal_conv(x, w, activation=None, return_state=True)
        state = torch.zeros(9, 2, width, dtype=dtype, device="cuda")
        for t in range(2):
            assert torch.equal(seq.causal_conv_step(x[:, t], w, state=state, activation=None), y[:, t])
        assert torch.equal(state, end)


@gpu
def test_offsets_beyond_32_bits():
    """Tensors of over 2^31 elements: the last rows and steps against the same computed on their own."""
    g = torch.Generator(device="cuda").manual_seed(32)
    rows, width = 70000, 32768
    table = torch.randn(rows, width, generator=g, device="cuda", dtype=torch.bfloat16)
    ids = torch.arange(rows, device="cuda").flip(0)
    out = seq.embedding(ids, table)
    assert torch.equal(out[-3:], table[:3].flip(0)) and torch.equal(out[:3], table[-3:].flip(0))
    grad = seq.embedding_grad(out, ids, rows)
    assert torch.equal(grad[-3:], table[-3:]) and torch.equal(grad[:3], table[:3])
    del table, out, grad
    B, L, D = 3, 360000, 2048
    x = torch.randn(B, L, D, generator=g, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(D, 4, generator=g, device="cuda")
    y = seq.causal_conv(x, w)
    tail = seq.causal_conv(x[-1:, -50:], w, state=x[-1:, -53:-50])
    assert torch.equal(y[-1:, -50:], tail)
    # a decay that forgets within a few steps (softplus(5) * 4 = 20: e^-20 a step, 2^-28 of what came before): the end of the last row by itself
    dt, a = torch.full((1, 1, D), 5.0, device="cuda", dtype=torch.bfloat16).expand(B, L, D).contiguous(), torch.full((D, 1), -4.0, device="cuda")
    b = torch.randn(B, L, 1, generator=g, device="cuda", dtype=torch.bfloat16)
    c = torch.ones(B, L, 1, device="cuda", dtype=torch.bfloat16)
    y, _, saved = seq.selective_scan_forward(x, dt, a, b, c)
    short = slice(L - 48, L)
    cut = [t[-1:, short] for t in (x, dt, b, c)]
    y1, _, saved1 = seq.selective_scan_forward(cut[0], cut[1], a, cut[2], cut[3])
    assert torch.allclose(y[-1, -40:].float(), y1[0, -40:].float(), rtol=2.0 ** -7, atol=1e-6)
    g1 = seq.selective_scan_grad(y, saved)
    g2 = seq.selective_scan_grad(y1, saved1)
    assert torch.allclose(g1.x[-1, -40:].float(), g2.x[0, -40:].float(), rtol=2.0 ** -6, atol=1e-6)
    del g1, g2, y, dt


# ------------------------------------------------------------------------------------------------------------------ together
def run_together(ids, table, w, wb, proj, a, dt_bias, d, lengths, dtype):
    """Tokens to features as a sequence encoder makes them: lookup, convolution, the scan's inputs by a projection, the scan."""
    D, N = a.shape
    e = seq.embedding(ids, table, math.sqrt(D))
    u = seq.causal_conv(e, w, wb, lengths=lengths)
    p = (u.float() @ proj).to(dtype)
    y, state = seq.selective_scan(u, p[..., :D], a, p[..., D:D + N], p[..., D + N:D + 2 * N], d, e, dt_bias, lengths=lengths, return_state=True)
    return y, state


def together_inputs(dtype=torch.float32, seed=11):
    g = rng(seed)
    B, L, V, D, N, K = 3, 14, 20, 16, 8, 4
    ids = torch.randint(0, V, (B, L), generator=g)
    lengths = torch.tensor([14, 0, 9])
    ids[torch.arange(L) >= lengths[:, None]] = -1
    leaves = [normal(g, V, D, dtype=dtype) * 0.3, normal(g, D, K) / 2, normal(g, D) * 0.1, normal(g, D, D + 2 * N) * 0.2,
              -(torch.rand(D, N, generator=g) * 4 + 0.1).cuda(), normal(g, D) - 1, normal(g, D)]
    return ids.cuda(), lengths.cuda(), leaves


@gpu
def test_together_gradients_against_differences():
    ids, lengths, leaves = together_inputs()
    g = rng(12)
    cy, cs = normal(g, 3, 14, 16).double(), normal(g, 3, 16, 8).double()

    def loss(values):
        table, w, wb, proj, a, dt_bias, d = values
        y, s = run_together(ids, table, w, wb, proj, a, dt_bias, d, lengths, torch.float32)
        return (y.double() * cy).sum() + (s.double() * cs).sum()

    params = [t.clone().requires_grad_(True) for t in leaves]
    grads = torch.autograd.grad(loss(params), params)
    # Central differences along a random direction of each leaf: off by h^2/6 times the third derivative and by the rounding of the two
    # losses over 2h.  With h = 2^-7 and losses around 100, each off by at most 2^-24 * 100 * (operations on the longest way, under
    # 300), the second part is under 2^-24 * 3e4 * 2^6 = 0.12; Richardson's step removes the first part's leading term.
    with torch.no_grad():
        for i, leaf in enumerate(leaves):
            way = normal(g, *leaf.shape)
            way /= way.norm()
            diff = []
            for h in (2.0 ** -6, 2.0 ** -7):
                up, down = ([t + s * h * way if k == i else t for k, t in enumerate(leaves)] for s in (1, -1))
                diff.append(float((loss(up) - loss(down)) / (2 * h)))
            est = (4 * diff[1] - diff[0]) / 3
            along = float((grads[i] * way).double().sum())
            assert abs(est - along) < 0.12 * 5 / 3 + 1e-2 * abs(along), (i, est, along)


@gpu
@pytest.mark.skipif(os.environ.get("MMN_EFENCE", "0") not in ("", "0"), reason="the electric fence's allocator fills new memory, which a capture does not allow")
def test_together_captured_into_a_graph():
    """Forward and backward captured, replayed several times with eager work between, against the eager result."""
    ids, lengths, leaves = together_inputs()
    dy = normal(rng(13), 3, 14, 16)

    def passes():
        table, w, wb, proj, a, dt_bias, d = leaves
        D, N = a.shape
        e = seq.embedding(ids, table, 4.0)
        u = seq.causal_conv(e, w, wb, lengths=lengths)
        p = u @ proj
        y, _, saved = seq.selective_scan_forward(u, p[..., :D], a, p[..., D:D + N], p[..., D + N:], d, e, dt_bias, lengths=lengths)
        g = seq.selective_scan_grad(dy, saved)
        k = seq.causal_conv_grad(g.x, e, w, wb, lengths=lengths)
        return [y, g.dt, g.a, g.b, g.z, k.x, k.weight, seq.embedding_grad(k.x, ids, table.shape[0], 4.0)]

    with torch.no_grad():
        want = [t.clone() for t in passes()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            passes()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = passes()
            graphs.append((graph, out))
        for turn in range(3):
            for graph, out in graphs:
                for t in out:
                    t.fill_(float("nan"))
                graph.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(p, q) for p, q in zip(out, want)), turn
            again = passes()
            assert all(torch.equal(p, q) for p, q in zip(again, want))


@gpu
@pytest.mark.skipif(os.environ.get("MMN_EFENCE", "0") not in ("", "0"), reason="the electric fence's allocator fills new memory, which a capture does not allow")
def test_autograd_captured_once_no_eager_graph_is_left():
    """While an eager graph holds a leaf the capture is refused at the first call; afterwards forward and backward replay the eager result."""
    ids, lengths, leaves = together_inputs()
    table, w, wb, proj, a, dt_bias, d = [t.clone().requires_grad_(True) for t in leaves]
    params = [table, w, wb, a, dt_bias, d]
    dy = normal(rng(13), 3, 14, 16)
    D, N = a.shape
    dt, bc = normal(rng(14), 3, 14, D), normal(rng(15), 3, 14, N)

    def run():
        e = seq.embedding(ids, table, 4.0)
        u = seq.causal_conv(e, w, wb, lengths=lengths)
        return seq.selective_scan(u, dt, a, bc, bc, d, e, dt_bias, lengths=lengths)

    y = run()
    want = [t.clone() for t in torch.autograd.grad(y, params, dy, retain_graph=True)]
    torch.cuda.synchronize()
    with pytest.raises(hip.MmnError, match="drop its outputs"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            run()
    for call in (lambda: seq.causal_conv(dy, w, wb), lambda: seq.selective_scan(dy, dt, a, bc, bc)):
        with pytest.raises(hip.MmnError, match="drop its outputs"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    del y
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(run(), params, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(run(), params, dy)
    for turn in range(3):
        for t in got:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), turn
        again = torch.autograd.grad(run(), params, dy)
        assert all(torch.equal(p, q) for p, q in zip(again, want))


@gpu
def test_on_another_stream():
    ids, lengths, leaves = together_inputs()
    table, w, wb, proj, a, dt_bias, d = leaves
    want = run_together(ids, table, w, wb, proj, a, dt_bias, d, lengths, torch.float32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run_together(ids, table, w, wb, proj, a, dt_bias, d, lengths, torch.float32)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@gpu
def test_empty_batches_and_no_steps():
    z = lambda *s: torch.zeros(*s, device="cuda")
    w, a = z(8, 4) + 1, z(8, 3) - 1
    for B, L in ((0, 5), (4, 0)):
        s, cs = z(B, 8, 3) + 2, z(B, 3, 8) + 3
        y, out = seq.causal_conv(z(B, L, 8), w, state=cs, return_state=True)
        assert y.shape == (B, L, 8) and torch.equal(out, cs)
        g = seq.causal_conv_grad(z(B, L, 8), z(B, L, 8), w, state=cs, state_grad=cs)
        assert not g.weight.any() and torch.equal(g.state, cs)
        y, out, saved = seq.selective_scan_forward(z(B, L, 8), z(B, L, 8), a, z(B, L, 3), z(B, L, 3), state=s, return_state=True)
        assert y.shape == (B, L, 8) and torch.equal(out, s)
        g = seq.selective_scan_grad(z(B, L, 8), saved, s)
        assert not g.a.any() and torch.equal(g.state, s)
    assert not seq.embedding_grad(z(0, 8), torch.zeros(0, dtype=torch.int64, device="cuda"), 5).any()


# ------------------------------------------------------------------------------------------------------------------ refusals
def test_operators_refuse_the_cpu():
    z = torch.zeros
    with pytest.raises(hip.MmnError):
        seq.embedding(z(3, dtype=torch.int64), z(4, 2))
    with pytest.raises(hip.MmnError):
        seq.embedding_grad(z(3, 2), z(3, dtype=torch.int64), 4)
    with pytest.raises(hip.MmnError):
        seq.causal_conv(z(1, 2, 3), z(3, 4))
    with pytest.raises(hip.MmnError):
        seq.causal_conv_step(z(1, 3), z(3, 4), state=z(1, 3, 3))
    with pytest.raises(hip.MmnError):
        seq.selective_scan(z(1, 2, 3), z(1, 2, 3), z(3, 4), z(1, 2, 4), z(1, 2, 4))
    with pytest.raises(hip.MmnError):
        seq.selective_scan_step(z(1, 3), z(1, 3), z(3, 4), z(1, 4), z(1, 4), state=z(1, 3, 4))


def test_operators_refuse_wrong_arguments():
    z, i64 = torch.zeros, torch.int64
    ids, x, w = z(3, dtype=i64), z(2, 5, 6), z(6, 4)
    bad = [
        lambda: seq.embedding(z(3), z(4, 2)), lambda: seq.embedding(ids, z(4)), lambda: seq.embedding(ids, z(4, 2).double()), lambda: seq.embedding(ids, z(0, 2)),
        lambda: seq.embedding_grad(z(4, 2), ids, 4), lambda: seq.embedding_grad(z(3, 2), ids, 0), lambda: seq.embedding_grad(z(3), ids, 4),
        lambda: seq.causal_conv(x[0], w), lambda: seq.causal_conv(x, z(6, 5)), lambda: seq.causal_conv(x, z(6, 1)), lambda: seq.causal_conv(x, z(5, 4)),
        lambda: seq.causal_conv(x, w.double()), lambda: seq.causal_conv(x, w, z(5)), lambda: seq.causal_conv(x, w, activation="relu"),
        lambda: seq.causal_conv(x, w, lengths=z(3, dtype=i64)), lambda: seq.causal_conv(x, w, lengths=z(2)), lambda: seq.causal_conv(x, w, state=z(2, 4, 6)),
        lambda: seq.causal_conv(x, w, state=z(2, 3, 6).half()), lambda: seq.causal_conv(x.long(), w), lambda: seq.causal_conv_grad(z(2, 5, 7), x, w),
        lambda: seq.causal_conv_step(x[:, 0], w, state=z(2, 4, 6)), lambda: seq.causal_conv_step(x[:, 0], w, state=z(2, 6, 3).transpose(1, 2)),
        lambda: seq.causal_conv_step(x[:, 0], w, state=None),
    ]
    dt, a, b = z(2, 5, 6), z(6, 3), z(2, 5, 3)
    bad += [
        lambda: seq.selective_scan(x, dt[:, :4], a, b, b), lambda: seq.selective_scan(x, dt.half(), a, b, b), lambda: seq.selective_scan(x, dt, z(5, 3), b, b),
        lambda: seq.selective_scan(x, dt, z(6, 33), z(2, 5, 33), z(2, 5, 33)), lambda: seq.selective_scan(x, dt, a, b, z(2, 5, 4)),
        lambda: seq.selective_scan(x, dt, a, z(2, 5, 4, 3), z(2, 5, 4, 3)), lambda: seq.selective_scan(x, dt, a, z(2, 5, 2, 3), b),
        lambda: seq.selective_scan(x, dt, a, b, b, d=z(5)), lambda: seq.selective_scan(x, dt, a, b, b, z=z(2, 5, 5)), lambda: seq.selective_scan(x, dt, a, b, b, dt_bias=z(6).half()),
        lambda: seq.selective_scan(x, dt, a, b, b, state=z(2, 3, 6)), lambda: seq.selective_scan(x, dt, a.half(), b, b),
        lambda: seq.selective_scan_step(x[:, 0], dt[:, 0], a, b[:, 0], b[:, 0], state=z(2, 6, 4)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")


def test_one_step_forms_refuse_gradients_and_overlaps():
    z = torch.zeros
    state = z(2, 3, 6)
    with pytest.raises(ValueError, match="no gradient"):
        seq.causal_conv_step(z(2, 6), z(6, 4).requires_grad_(True), state=state)
    with pytest.raises(ValueError, match="no gradient"):
        seq.selective_scan_step(z(2, 6), z(2, 6), z(6, 3).requires_grad_(True), z(2, 3), z(2, 3), state=z(2, 6, 3))
    big = z(80)
    with pytest.raises(ValueError, match="overlaps"):
        seq.causal_conv_step(z(2, 6), z(6, 4), state=big[:36].view(2, 3, 6), out_state=big[4:40].view(2, 3, 6))
    with pytest.raises(ValueError, match="like state"):
        seq.causal_conv_step(z(2, 6), z(6, 4), state=state, out_state=z(2, 3, 5))


def test_c_entry_points_refuse_without_a_gpu():
    """Argument checks of the C ABI come before any launch."""
    import ctypes as C
    lib = hip.load()
    ARG, UNSUPPORTED, WORKSPACE = -1, -2, -3
    assert lib.mmn_seq_embed(None, 1, None, None, 1, 1, 1, 0, 1.0, None) == ARG
    assert lib.mmn_seq_embed(None, 1, None, None, 0, 1, 1, 0, 1.0, None) == 0
    for rows, vocab, width, kind in ((-1, 1, 1, 0), (1, 0, 1, 0), (1, 1, 0, 0), (1, 1, 1, 3), (2 ** 31, 1, 1, 0)):
        assert lib.mmn_seq_embed(8, 1, 8, 8, rows, vocab, width, kind, 1.0, None) == ARG
        assert lib.mmn_seq_embed_grad(8, 1, 8, 8, rows, vocab, width, kind, 1.0, 256, 1 << 40, None) == ARG
    assert lib.mmn_seq_embed_grad(8, 1, 8, 8, 10, 10, 4, 0, 1.0, 256, 16, None) == WORKSPACE
    assert lib.mmn_seq_embed_grad(8, 1, 8, 8, 10, 10, 4, 0, 1.0, 264, 1 << 40, None) == WORKSPACE
    c = hip.ConvDesc()
    assert lib.mmn_seq_conv(C.byref(c), None) == ARG
    c.batch, c.steps, c.width, c.taps = 2, 3, 4, 5
    assert lib.mmn_seq_conv(C.byref(c), None) == ARG and lib.mmn_seq_conv_grad_bytes(C.byref(c)) == 0
    c.taps = 4
    assert lib.mmn_seq_conv(C.byref(c), None) == ARG and lib.mmn_seq_conv_step(C.byref(c), None) == ARG
    assert lib.mmn_seq_conv_grad(C.byref(c), 256, 1 << 40, None) == ARG
    s = hip.ScanDesc()
    assert lib.mmn_seq_scan(C.byref(s), None, 0, None) == ARG
    s.batch, s.steps, s.width, s.groups, s.states = 2, 3, 6, 4, 16
    assert lib.mmn_seq_scan(C.byref(s), 256, 1 << 40, None) == ARG           # groups do not divide the width
    s.groups = 2
    assert lib.mmn_seq_scan(C.byref(s), 256, 1 << 40, None) == ARG and lib.mmn_seq_scan_step(C.byref(s), None) == ARG
    for name in ("x", "dt", "b", "c", "a", "y"):
        setattr(s, name, 256)
    assert lib.mmn_seq_scan(C.byref(s), 256, 1 << 40, None) == UNSUPPORTED   # steps that share memory
    s.x_step = s.dt_step = 1 << 24
    assert lib.mmn_seq_scan(C.byref(s), 256, 1 << 40, None) == UNSUPPORTED   # steps too far apart
    s.x_step = s.dt_step = 6
    assert lib.mmn_seq_scan(C.byref(s), None, 0, None) == WORKSPACE
    assert lib.mmn_seq_scan_grad(C.byref(s), 256, 1 << 40, None) == ARG
    s.states = 33
    assert lib.mmn_seq_scan(C.byref(s), 256, 1 << 40, None) == ARG and lib.mmn_seq_scan_bytes(C.byref(s), 1) == 0


def test_sequence_symbols_and_structs_match_their_header(tmp_path):
    import ctypes as C
    import os
    import re
    import subprocess
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(repo, "include", "mmn_sequence.h")).read(), flags=re.S)
    assert set(re.findall(r"\b(mmn_seq_[a-z_]+)\s*\(", text)) == set(hip.SEQUENCE_SYMBOLS)
    src = tmp_path / "sz.c"
    fields = [("mmn_seq_conv_desc", f, hip.ConvDesc) for f, _ in hip.ConvDesc._fields_] + [("mmn_seq_scan_desc", f, hip.ScanDesc) for f, _ in hip.ScanDesc._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mmn_sequence.h"\nint main(void){\n'
                   + "".join(f'printf("%zu\\n", offsetof({s}, {f}));\n' for s, f, _ in fields)
                   + 'printf("%zu %zu\\n", sizeof(mmn_seq_conv_desc), sizeof(mmn_seq_scan_desc)); return 0;}\n')
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", os.path.join(repo, "include"), str(src), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in lines[:len(fields)]] == [getattr(t, f).offset for _, f, t in fields]
    assert [int(v) for v in lines[len(fields):]] == [C.sizeof(hip.ConvDesc), C.sizeof(hip.ScanDesc)]


def test_oracle_against_autograd():
    """The oracle's backward formulas against torch's differentiation of its forward formulas, 64 bits."""
    g = rng(20)
    case = (2, 6, 4, 2, 3, [6, 4], True, True, True, True, True)
    cpu = lambda *s: torch.randn(*s, generator=g).double()
    B, L, D, G, N = case[:5]
    leaves = dict(x=cpu(B, L, D), dt=cpu(B, L, D), a=-cpu(D, N).abs(), b=cpu(B, L, G, N), c=cpu(B, L, G, N), d=cpu(D), z=cpu(B, L, D), dt_bias=cpu(D), state=cpu(B, D, N))
    dy, ds = cpu(B, L, D), cpu(B, D, N)
    want = O.scan(**leaves, softplus=True, lengths=torch.tensor(case[5]), dy=dy, dstate_out=ds)
    p = {k: v.clone().requires_grad_(True) for k, v in leaves.items()}
    total = 0.0
    for i, n in enumerate(case[5]):
        h = p["state"][i]
        for t in range(n):
            step = torch.nn.functional.softplus(p["dt"][i, t] + p["dt_bias"])
            bt, ct = (p[k][i, t].repeat_interleave(D // G, 0) for k in ("b", "c"))
            h = torch.exp(step[:, None] * p["a"]) * h + (step * p["x"][i, t])[:, None] * bt
            total = total + (((h * ct).sum(-1) + p["d"] * p["x"][i, t]) * torch.nn.functional.silu(p["z"][i, t]) * dy[i, t]).sum()
        total = total + (h * ds[i]).sum()
    grads = dict(zip(p, torch.autograd.grad(total, list(p.values()))))
    for k, v in grads.items():
        assert torch.allclose(v, want["dstate" if k == "state" else k][0], rtol=1e-10, atol=1e-12), k
    x, w, b, s = cpu(B, L, D), cpu(D, 3), cpu(D), cpu(B, 2, D)
    dy, ds = cpu(B, L, D), cpu(B, 2, D)
    want = O.conv(x, w, b, True, torch.tensor([6, 1]), s, dy, ds)
    p = [v.clone().requires_grad_(True) for v in (x, w, b, s)]
    total = 0.0
    for i, n in enumerate((6, 1)):
        line = torch.cat([p[3][i], p[0][i, :n]])
        for t in range(n):
            total = total + (torch.nn.functional.silu(p[2] + (p[1].t() * line[t:t + 3]).sum(0)) * dy[i, t]).sum()
        total = total + (line[n:] * ds[i]).sum()
    for v, k in zip(torch.autograd.grad(total, p), ("x", "weight", "bias", "dstate")):
        assert torch.allclose(v, want[k][0], rtol=1e-10, atol=1e-12), k
