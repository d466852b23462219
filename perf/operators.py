"""Cases of the operators that turn a sequence into features (multimodn_amd.sequence): embedding lookup and its gradient, the
causal depthwise convolution, the selective scan, and the forms of the last two for one new step.  `run` computes a case with
elementary torch operations (`own` false) or with the framework's kernels (`own` true); `exact` gives its values in 64 bits.

Sizes: batches of 16 to 4096 rows and widths of 64 to 1024 as in the framework's own workloads, sequences from one step to 4096.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new event for each of 16 patients: the lookup in front of a single-token step (latency)
        {"name": "embed_one", "op": "embed", "batch": 16, "steps": 1, "vocab": 1000, "width": 64, "type": "fp32"},
        # looking up a batch of long prompts
        {"name": "embed_prompt", "op": "embed", "batch": 16, "steps": 2048, "vocab": 32000, "width": 1024, "type": "bf16"},
        # a table's gradient: short coded histories with padding, an odd width and vocabulary
        {"name": "embed_grad_odd", "op": "embed_grad", "batch": 37, "steps": 191, "vocab": 1501, "width": 203, "type": "fp32"},
        # a table's gradient in a large training step: frequent tokens hold many of the rows
        {"name": "embed_grad_large", "op": "embed_grad", "batch": 64, "steps": 1024, "vocab": 50000, "width": 512, "type": "bf16"},
        # prompts of unequal length that continue from a kept state
        {"name": "conv_prompt", "op": "conv", "batch": 8, "steps": 2048, "width": 1024, "taps": 4, "type": "bf16",
         "ragged": True, "state": True},
        # training on 48-step stays at the framework's benchmark batch, forward and backward
        {"name": "conv_train", "op": "conv_train", "batch": 4096, "steps": 48, "width": 128, "taps": 4, "type": "fp32",
         "ragged": True, "state": False},
        # one long prompt: little work across, all of it along the sequence
        {"name": "scan_prompt", "op": "scan", "batch": 1, "steps": 4096, "width": 1024, "groups": 1, "states": 16, "type": "bf16",
         "ragged": False, "state": False},
        # training on a few short sequences of odd sizes, two groups (the smallest training step: launches count)
        {"name": "scan_train_odd", "op": "scan_train", "batch": 5, "steps": 117, "width": 90, "groups": 2, "states": 12, "type": "fp32",
         "ragged": True, "state": True},
        # training at the framework's benchmark batch on 48-step stays
        {"name": "scan_train_wide", "op": "scan_train", "batch": 4096, "steps": 48, "width": 64, "groups": 1, "states": 16, "type": "fp32",
         "ragged": True, "state": False},
        # training on long sequences
        {"name": "scan_train_long", "op": "scan_train", "batch": 4, "steps": 2048, "width": 1024, "groups": 1, "states": 16, "type": "bf16",
         "ragged": True, "state": False},
        # one new step for 16 patients: convolution, then scan, each on its kept state (latency)
        {"name": "step_small", "op": "step", "batch": 16, "width": 128, "groups": 1, "states": 16, "taps": 4, "type": "fp32"},
        # one new step for every row of a large batch
        {"name": "step_large", "op": "step", "batch": 2048, "width": 1024, "groups": 1, "states": 16, "taps": 4, "type": "bf16"},
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "conv", "conv_train", "scan", "scan_train", "scan_train", "step"])
    case = {"op": op, "type": rng.choice(["fp32", "bf16", "fp16"])}
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        case["batch"] = _between(rng, 1, 4096)
        if op != "step":
            case["steps"] = _between(rng, 1, 4096)
        case["width"] = _between(rng, 32, 1024)
        if op in ("embed", "embed_grad"):
            case["vocab"] = _between(rng, 50, 60000)
        if op in ("conv", "conv_train", "step"):
            case["taps"] = rng.choice([2, 3, 4, 4])
        if op in ("scan", "scan_train", "step"):
            case["groups"] = rng.choice([1, 1, 1, 2, 4])
            case["width"] -= case["width"] % case["groups"]
            case["states"] = rng.choice([4, 8, 16, 16, 16, 24, 32, _between(rng, 1, 32)])
        if op in ("conv", "conv_train", "scan", "scan_train"):
            case["ragged"], case["state"] = rng.random() < 0.5, rng.random() < 0.5
        if _cost(case) <= most:
            return case


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 16


# --------------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = _TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    op, n, d = case["op"], case["batch"], case["width"]
    steps = case.get("steps", 1)
    s = {"op": op}
    if op in ("embed", "embed_grad"):
        # token frequencies fall with the rank, and a tenth of the rows are padded (-1) behind their end
        ids = (torch.exp(uniform(n, steps) * math.log(case["vocab"])) - 1).long().clamp_(0, case["vocab"] - 1)
        if steps > 1:
            ends = (steps * (0.3 + uniform(n, 1) * 0.7)).long().clamp_(min=1)
            padded = (uniform(n, 1) < 0.1) & (torch.arange(steps, device="cuda") >= ends)
            ids = ids.masked_fill(padded, -1)
        s.update(ids=ids, scale=math.sqrt(d), vocab=case["vocab"])
        if op == "embed":
            s["weight"] = (0.02 * normal(case["vocab"], d)).to(t)
        else:
            s["grad"] = (0.1 * normal(n, steps, d)).to(t)
        return s
    s["lengths"] = (uniform(n) * (steps + 1)).int().clamp_(max=steps) if case.get("ragged") else None
    if op in ("conv", "conv_train", "step"):
        k = case["taps"]
        # x is one half of a projection's output, so its rows are twice as far apart as they are wide
        s["x"] = normal(n, steps, 2 * d).to(t)[..., :d]
        s["taps"] = (2 * uniform(d, k) - 1) / math.sqrt(k)
        s["taps_bias"] = (2 * uniform(d) - 1) / math.sqrt(k)
        s["conv_state"] = normal(n, k - 1, d).to(t) if case.get("state") or op == "step" else None
        if op == "conv_train":
            s["dy"] = normal(n, steps, d).to(t)
    if op in ("scan", "scan_train", "step"):
        groups, states = case["groups"], case["states"]
        s["u"] = torch.nn.functional.silu(normal(n, steps, d)).to(t)
        s["z"] = normal(n, steps, 2 * d).to(t)[..., d:]
        s["dt"] = (0.3 * normal(n, steps, d)).to(t)
        first = torch.exp(math.log(1e-3) + uniform(d) * (math.log(0.1) - math.log(1e-3)))
        s["dt_bias"] = first + torch.log(-torch.expm1(-first))             # softplus(dt_bias) = first
        s["a"] = -(1 + torch.arange(states, device="cuda").float()).repeat(d, 1) * (0.9 + 0.2 * uniform(d, 1))
        both = normal(n, steps, 2 * groups * states).to(t)                   # b and c: parts of one projection's output
        s["b"] = both[..., :groups * states].unflatten(-1, (groups, states))
        s["c"] = both[..., groups * states:].unflatten(-1, (groups, states))
        s["d"] = 0.5 + uniform(d)
        s["state"] = normal(n, d, states) if case.get("state") or op == "step" else None
        if op == "scan_train":
            s["dy"] = normal(n, steps, d).to(t)
    if op == "step":
        for name in ("x", "u", "z", "dt", "b", "c"):
            s[name] = s[name][:, 0]
        s["conv_next"], s["state_next"] = torch.empty_like(s["conv_state"]), torch.empty_like(s["state"])
    return s


# ------------------------------------------------------------------------------------------------------------------ plain form
def _plain_embed(ids, weight, scale):
    rows = weight.float()[ids.clamp(min=0)] if weight.numel() < ids.numel() * weight.shape[1] else weight[ids.clamp(min=0)].float()
    return torch.where((ids >= 0)[..., None], rows * scale, 0.0).to(weight.dtype)


def _plain_embed_grad(grad, ids, vocab, scale):
    out = torch.zeros(vocab, grad.shape[-1], device=grad.device)
    rows = torch.where((ids >= 0)[..., None], grad.float() * scale, 0.0)
    return out.index_add_(0, ids.clamp(min=0).flatten(), rows.flatten(0, -2)).to(grad.dtype)


def _inside(lengths, x):
    """[batch, steps, 1]: the steps that belong to their sequence."""
    at = torch.arange(x.shape[1], device=x.device)
    return (at < lengths[:, None])[..., None] if lengths is not None else torch.ones_like(at, dtype=torch.bool)[None, :, None]


def _window(x, state, k, inside):
    """x in 32 bits behind its k - 1 earlier inputs, [batch, k - 1 + steps, width]."""
    x = torch.where(inside, x.float(), 0.0)
    before = state.float() if state is not None else x.new_zeros(x.shape[0], k - 1, x.shape[2])
    return torch.cat([before, x], 1)


def _kept(w, k, steps, lengths, dtype):
    """The last k - 1 inputs of every sequence."""
    if lengths is None:
        return w[:, steps:].to(dtype)
    at = lengths.long()[:, None, None] + torch.arange(k - 1, device=w.device)[None, :, None]
    return torch.gather(w, 1, at.expand(-1, -1, w.shape[2])).to(dtype)


def _plain_conv(x, taps, bias, lengths, state):
    inside, k, steps = _inside(lengths, x), taps.shape[1], x.shape[1]
    w = _window(x, state, k, inside)
    pre = bias + sum(taps[:, j] * w[:, j:j + steps] for j in range(k))
    y = torch.where(inside, pre * torch.sigmoid(pre), 0.0).to(x.dtype)
    return {"y": y, "state": _kept(w, k, steps, lengths, x.dtype)}


def _plain_conv_grad(dy, x, taps, bias, lengths, state):
    inside, k, steps = _inside(lengths, x), taps.shape[1], x.shape[1]
    w = _window(x, state, k, inside)
    pre = bias + sum(taps[:, j] * w[:, j:j + steps] for j in range(k))
    sig = torch.sigmoid(pre)
    y = torch.where(inside, pre * sig, 0.0).to(x.dtype)
    dpre = torch.where(inside, dy.float() * sig * (1 + pre * (1 - sig)), 0.0)
    late = torch.nn.functional.pad(dpre, (0, 0, k - 1, k - 1))
    dw = sum(taps[:, j] * late[:, k - 1 - j:k - 1 - j + steps + k - 1] for j in range(k))
    out = {"y": y, "dx": torch.where(inside, dw[:, k - 1:], 0.0).to(x.dtype),
           "dtaps": torch.stack([(dpre * w[:, j:j + steps]).sum((0, 1)) for j in range(k)], 1), "dbias": dpre.sum((0, 1))}
    if state is not None:
        out["dstate"] = dw[:, :k - 1].to(x.dtype)
    return out


def _linear_scan(decay, inc):
    """h[t] = decay[t] h[t-1] + inc[t] along dimension 1, by doubling."""
    step = 1
    while step < inc.shape[1]:
        inc = torch.cat([inc[:, :step], inc[:, step:] + decay[:, step:] * inc[:, :-step]], 1)
        decay = torch.cat([decay[:, :step], decay[:, step:] * decay[:, :-step]], 1)
        step *= 2
    return inc


def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


def _per_channel(v, width):
    """b or c, [batch, steps, groups, states], in 32 bits for every channel (a view for one group)."""
    v = v.float()
    return v if v.shape[2] == 1 else v.repeat_interleave(width // v.shape[2], 2)


def _plain_scan_states(s):
    inside = _inside(s["lengths"], s["u"])
    u = torch.where(inside, s["u"].float(), 0.0)
    dt = torch.where(inside, _softplus(s["dt"].float() + s["dt_bias"]), 0.0)
    b, c = (_per_channel(torch.where(inside[..., None], s[k], 0.0), u.shape[2]) for k in ("b", "c"))
    decay = torch.exp(dt[..., None] * s["a"])
    inc = (dt * u)[..., None] * b
    if s["state"] is not None:
        inc[:, 0] += decay[:, 0] * s["state"]
    h = _linear_scan(decay, inc)
    return inside, u, dt, b, c, decay, h


def _plain_scan(s):
    inside, u, dt, b, c, decay, h = _plain_scan_states(s)
    z = s["z"].float()
    out = ((h * c).sum(-1) + s["d"] * u) * z * torch.sigmoid(z)
    return {"y": torch.where(inside, out, 0.0).to(s["u"].dtype), "state": h[:, -1].contiguous()}


def _to_groups(v, groups):
    """Sums the channels of each group: [batch, steps, width, states] to [batch, steps, groups, states]."""
    return v.unflatten(2, (groups, -1)).sum(3)


def _plain_scan_train(s):
    inside, u, dt, b, c, decay, h = _plain_scan_states(s)
    t, groups = s["u"].dtype, s["b"].shape[2]
    z = torch.where(inside, s["z"].float(), 0.0)
    dy = torch.where(inside, s["dy"].float(), 0.0)
    sig = torch.sigmoid(z)
    out = (h * c).sum(-1) + s["d"] * u
    y = torch.where(inside, out * z * sig, 0.0).to(t)
    dout = dy * z * sig
    dz = dy * out * sig * (1 + z * (1 - sig))
    start = s["state"] if s["state"] is not None else torch.zeros_like(h[:, 0])
    before = torch.cat([start[:, None], h[:, :-1]], 1)
    dc = _to_groups(dout[..., None] * h, groups)
    later = torch.cat([decay[:, 1:], torch.ones_like(decay[:, :1])], 1)      # what carries dh[t+1] back to step t
    dh = _linear_scan(later.flip(1), (dout[..., None] * c).flip(1)).flip(1)
    db = _to_groups(dh * (dt * u)[..., None], groups)
    dinc = (dh * b).sum(-1)
    darg = dh * before * decay
    ddt = torch.where(inside, ((darg * s["a"]).sum(-1) + u * dinc) * torch.sigmoid(s["dt"].float() + s["dt_bias"]), 0.0)
    out = {"y": y, "du": (dt * dinc + s["d"] * dout).to(t), "ddt": ddt.to(t), "dz": dz.to(t), "db": db.to(t), "dc": dc.to(t),
           "da": (darg * dt[..., None]).sum((0, 1)), "dd": (dout * u).sum((0, 1)), "ddt_bias": ddt.sum((0, 1))}
    if s["state"] is not None:
        out["dstate"] = dh[:, 0] * decay[:, 0]
    return out


def _plain_step(s):
    w = torch.cat([s["conv_state"].float(), s["x"].float()[:, None]], 1)
    pre = (w * s["taps"].t()).sum(1) + s["taps_bias"]
    u = s["u"].float()
    dt = _softplus(s["dt"].float() + s["dt_bias"])
    b, c = (s[k].float() if s[k].shape[1] == 1 else s[k].float().repeat_interleave(u.shape[1] // s[k].shape[1], 1) for k in ("b", "c"))
    h = torch.exp(dt[..., None] * s["a"]) * s["state"] + (dt * u)[..., None] * b
    z = s["z"].float()
    y = ((h * c).sum(-1) + s["d"] * u) * z * torch.sigmoid(z)
    return {"conv": (pre * torch.sigmoid(pre)).to(s["x"].dtype), "conv_state": w[:, 1:].to(s["x"].dtype), "y": y.to(s["u"].dtype), "state": h}


# ------------------------------------------------------------------------------------------------------------------------ run
def run(s):
    op = s["op"]
    if own:
        from multimodn_amd import sequence as seq
        if op == "embed":
            return seq.embedding(s["ids"], s["weight"], scale=s["scale"])
        if op == "embed_grad":
            return seq.embedding_grad(s["grad"], s["ids"], s["vocab"], scale=s["scale"])
        if op == "conv":
            y, state = seq.causal_conv(s["x"], s["taps"], s["taps_bias"], lengths=s["lengths"], state=s["conv_state"], return_state=True)
            return {"y": y, "state": state}
        if op == "conv_train":
            y = seq.causal_conv(s["x"], s["taps"], s["taps_bias"], lengths=s["lengths"], state=s["conv_state"])
            g = seq.causal_conv_grad(s["dy"], s["x"], s["taps"], s["taps_bias"], lengths=s["lengths"], state=s["conv_state"])
            out = {"y": y, "dx": g.x, "dtaps": g.weight, "dbias": g.bias}
            return out if g.state is None else {**out, "dstate": g.state}
        scan = (s["u"], s["dt"], s["a"], s["b"], s["c"])
        more = {"d": s["d"], "z": s["z"], "dt_bias": s["dt_bias"]}
        if op == "scan":
            y, state = seq.selective_scan(*scan, **more, lengths=s["lengths"], state=s["state"], return_state=True)
            return {"y": y, "state": state}
        if op == "scan_train":
            y, _, saved = seq.selective_scan_forward(*scan, **more, lengths=s["lengths"], state=s["state"])
            g = seq.selective_scan_grad(s["dy"], saved)
            out = {"y": y, "du": g.x, "ddt": g.dt, "dz": g.z, "db": g.b, "dc": g.c, "da": g.a, "dd": g.d, "ddt_bias": g.dt_bias}
            return out if g.state is None else {**out, "dstate": g.state}
        conv = seq.causal_conv_step(s["x"], s["taps"], s["taps_bias"], state=s["conv_state"], out_state=s["conv_next"])
        y = seq.selective_scan_step(*scan, **more, state=s["state"], out_state=s["state_next"])
        return {"conv": conv, "conv_state": s["conv_next"], "y": y, "state": s["state_next"]}
    if op == "embed":
        return _plain_embed(s["ids"], s["weight"], s["scale"])
    if op == "embed_grad":
        return _plain_embed_grad(s["grad"], s["ids"], s["vocab"], s["scale"])
    if op == "conv":
        return _plain_conv(s["x"], s["taps"], s["taps_bias"], s["lengths"], s["conv_state"])
    if op == "conv_train":
        return _plain_conv_grad(s["dy"], s["x"], s["taps"], s["taps_bias"], s["lengths"], s["conv_state"])
    return _plain_scan(s) if op == "scan" else _plain_scan_train(s) if op == "scan_train" else _plain_step(s)


# ----------------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = 4 if case["type"] == "fp32" else 2
    op, n, steps, d = case["op"], case["batch"], case.get("steps", 1), case["width"]
    rows = n * steps
    if op == "embed":                      # ids, the rows looked up (at most the table), the output
        return {"bytes": 8 * rows + size * d * (min(rows, case["vocab"]) + rows), "flops": rows * d}
    if op == "embed_grad":                 # ids, the gradient in, the table's gradient out
        return {"bytes": 8 * rows + size * d * (rows + case["vocab"]), "flops": 2 * rows * d}
    k, nb, fl = case.get("taps", 0), 0, 0
    kept = n * (k - 1) * d * size if k else 0
    if op == "conv":
        nb += 2 * rows * d * size + 4 * d * (k + 1) + (2 if case["state"] else 1) * kept
        fl += rows * d * (2 * k + 6)
    if op == "conv_train":                 # x, y, dy, dx
        nb += 4 * rows * d * size + 12 * d * (k + 1) + (2 * kept if case["state"] else 0)
        fl += rows * d * (6 * k + 16)
    states = case.get("states", 0)
    both = 2 * rows * case.get("groups", 1) * states * size
    if op == "scan":                       # u, dt, z, y; b, c; a; the state
        nb += 4 * rows * d * size + both + 4 * d * (states + 2) + 4 * n * d * states * (2 if case["state"] else 1)
        fl += rows * d * (6 * states + 16)
    if op == "scan_train":                 # u, dt, z, y, dy, du, ddt, dz; b, c, db, dc; a, da; the state and its gradient
        nb += 8 * rows * d * size + 2 * both + 8 * d * (states + 2) + (8 * n * d * states if case["state"] else 0)
        fl += rows * d * (22 * states + 40)
    if op == "step":                       # x, its output, u, dt, z, y; b, c; both states in and out
        nb += 6 * rows * d * size + both + 2 * kept + 4 * d * (k + 1 + states + 2) + 8 * n * d * states
        fl += n * d * (2 * k + 6 * states + 24)
    return {"bytes": nb, "flops": fl}


# ----------------------------------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    op = s["op"]
    if op == "embed":
        table = torch.cat([s["weight"] * s["scale"], s["weight"].new_zeros(1, s["weight"].shape[1])])
        return table[torch.where(s["ids"] < 0, s["weight"].shape[0], s["ids"])]
    if op == "embed_grad":
        flat = s["ids"].flatten()
        there = (flat >= 0).nonzero()[:, 0]
        order = there[torch.argsort(flat[there], stable=True)]
        table = torch.zeros(s["vocab"], s["grad"].shape[-1], dtype=torch.float64, device=flat.device)
        return table.index_add_(0, flat[order], s["grad"].flatten(0, 1)[order]) * s["scale"]
    if op in ("conv", "conv_train"):
        return _exact_conv(s)
    if op == "step":
        conv = _exact_conv({"x": s["x"][:, None], "taps": s["taps"], "taps_bias": s["taps_bias"], "lengths": None,
                            "conv_state": s["conv_state"], "op": "conv"})
        one = {k: s[k][:, None] for k in ("u", "z", "dt", "b", "c")}
        scan = _exact_scan({**one, "a": s["a"], "d": s["d"], "dt_bias": s["dt_bias"], "state": s["state"], "lengths": None, "op": "scan"})
        return {"conv": conv["y"][:, 0], "conv_state": conv["state"], "y": scan["y"][:, 0], "state": scan["state"]}
    return _exact_scan(s)


def _exact_conv(s):
    """One step after another; the gradients go the same way back."""
    x, taps, state = s["x"], s["taps"], s["conv_state"]
    n, steps, d = x.shape
    k = taps.shape[1]
    ends = s["lengths"].long() if s["lengths"] is not None else torch.full((n,), steps, device=x.device)
    last = torch.zeros(n, k - 1, d, dtype=x.dtype, device=x.device) if state is None else state.clone()
    first, y, seen = last.clone(), torch.zeros_like(x), []
    for t in range(steps):
        on = (t < ends)[:, None]
        now = torch.cat([last, x[:, t:t + 1]], 1)
        pre = torch.einsum("nkd,dk->nd", now, taps) + s["taps_bias"]
        y[:, t] = torch.where(on, pre / (1 + torch.exp(-pre)), torch.zeros_like(pre))
        last = torch.where(on[..., None], now[:, 1:], last)
        if s["op"] == "conv_train":
            seen.append((now, pre))
    if s["op"] == "conv":
        return {"y": y, "state": last}
    dx, dtaps, dbias = torch.zeros_like(x), torch.zeros_like(taps), torch.zeros_like(s["taps_bias"])
    dlast = torch.zeros_like(first)
    for t in reversed(range(steps)):
        on = (t < ends)[:, None]
        now, pre = seen[t]
        e = torch.exp(-pre)
        dpre = torch.where(on, s["dy"][:, t] * ((1 + e) + pre * e) / (1 + e) ** 2, torch.zeros_like(pre))
        dtaps += torch.einsum("nd,nkd->dk", dpre, now)
        dbias += dpre.sum(0)
        dnow = torch.cat([torch.zeros_like(dlast[:, :1]), dlast], 1) + torch.einsum("nd,dk->nkd", dpre, taps)
        dx[:, t] = torch.where(on, dnow[:, -1], torch.zeros_like(pre))
        dlast = torch.where(on[..., None], dnow[:, :-1], dlast)
    out = {"y": y, "dx": dx, "dtaps": dtaps, "dbias": dbias}
    return out if state is None else {**out, "dstate": dlast}


def _exact_scan(s):
    """One step after another; the gradients go the same way back over the kept states."""
    u, a = s["u"], s["a"]
    n, steps, d = u.shape
    groups, states = s["b"].shape[2:]
    ends = s["lengths"].long() if s["lengths"] is not None else torch.full((n,), steps, device=u.device)
    h = torch.zeros(n, d, states, dtype=u.dtype, device=u.device) if s["state"] is None else s["state"].clone()
    train = s["op"] == "scan_train"
    kept = torch.empty(steps, n, d, states, dtype=u.dtype, device=u.device) if train else None
    y = torch.zeros_like(u)

    def at(t):
        raw = s["dt"][:, t] + s["dt_bias"]
        dt = torch.logaddexp(raw, torch.zeros_like(raw))
        b, c = (s[k][:, t][:, :, None].expand(n, groups, d // groups, states).reshape(n, d, states) for k in ("b", "c"))
        return raw, dt, b, c, torch.exp(dt[..., None] * a), (t < ends)[:, None]

    for t in range(steps):
        raw, dt, b, c, decay, on = at(t)
        if train:
            kept[t] = h
        h = torch.where(on[..., None], decay * h + (dt * u[:, t])[..., None] * b, h)
        z = s["z"][:, t]
        y[:, t] = torch.where(on, ((h * c).sum(-1) + s["d"] * u[:, t]) * z / (1 + torch.exp(-z)), torch.zeros_like(z))
    if not train:
        return {"y": y, "state": h}
    du, ddt, dz = torch.zeros_like(u), torch.zeros_like(u), torch.zeros_like(u)
    db, dc = torch.zeros_like(s["b"]), torch.zeros_like(s["c"])
    da, dd, dbias = torch.zeros_like(a), torch.zeros_like(s["d"]), torch.zeros_like(s["dt_bias"])
    dh = torch.zeros_like(h)
    for t in reversed(range(steps)):
        raw, dt, b, c, decay, on = at(t)
        old, z, x = kept[t], s["z"][:, t], u[:, t]
        new = decay * old + (dt * x)[..., None] * b
        sig = 1 / (1 + torch.exp(-z))
        dy = torch.where(on, s["dy"][:, t], torch.zeros_like(z))
        inner = (new * c).sum(-1) + s["d"] * x
        dz[:, t] = dy * inner * (sig + z * sig * (1 - sig))
        dinner = dy * z * sig
        dd += (dinner * x).sum(0)
        dc[:, t] = (dinner[..., None] * new).reshape(n, groups, d // groups, states).sum(2)
        live = dh + dinner[..., None] * c
        live = torch.where(on[..., None], live, torch.zeros_like(live))
        db[:, t] = (live * (dt * x)[..., None]).reshape(n, groups, d // groups, states).sum(2)
        push = (live * b).sum(-1)
        turn = live * old * decay
        da += (turn * dt[..., None]).sum(0)
        du[:, t] = dt * push + s["d"] * dinner
        ddt[:, t] = ((turn * a).sum(-1) + x * push) / (1 + torch.exp(-raw))
        dh = torch.where(on[..., None], live * decay, dh)
    dbias = ddt.sum((0, 1))
    out = {"y": y, "du": du, "ddt": ddt, "dz": dz, "db": db, "dc": dc, "da": da, "dd": dd, "ddt_bias": dbias}
    return out if s["state"] is None else {**out, "dstate": dh}
