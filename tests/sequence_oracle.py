"""Plain 64-bit statements of the sequence operators, step after step on the CPU, and beside every result its magnitude: the same
formula over absolute values, which is what a rounding error of the kernels is measured against.

A sum of n products in 32 bits is off by at most (n + 1) u times the sum of the products' magnitudes, u = 2^-24 (Higham, Accuracy and
Stability of Numerical Algorithms, 3.1).  `check` allows `terms` such roundings and one rounding of the result to its own type."""
import torch

U32 = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def f64(t):
    return None if t is None else t.detach().cpu().double()


def check(got, want, mag, terms, what):
    """got: the kernel's; want, mag: 64 bits; terms: roundings in 32 bits on the way, relative to mag."""
    assert got is not None and tuple(got.shape) == tuple(want.shape), (what, None if got is None else got.shape, want.shape)
    half = HALF_STEP[got.dtype]
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 2.0 ** -126       # spacing of the smallest values
    g = got.detach().cpu().double()
    assert torch.isfinite(g).all(), f"{what}: not finite"
    allowed = half * (want.abs() + terms * U32 * mag) + terms * U32 * mag + tiny
    over = (g - want).abs() - allowed
    if over.numel() and float(over.max()) > 0:
        i = int(over.argmax())
        raise AssertionError(f"{what}: {g.flatten()[i]} instead of {want.flatten()[i]}, allowed {allowed.flatten()[i]:.3g}, at {i}")


def embed(ids, weight, scale):
    ids, w = ids.cpu().long(), f64(weight)
    ok = (ids >= 0) & (ids < w.shape[0])
    return torch.where(ok[..., None], w[ids.clamp(0, w.shape[0] - 1)] * scale, torch.zeros((), dtype=torch.float64))


def embed_grad(grad, ids, vocab, scale):
    ids, g = ids.cpu().long().flatten(), f64(grad).reshape(-1, grad.shape[-1])
    out, mag = torch.zeros(vocab, g.shape[1], dtype=torch.float64), torch.zeros(vocab, g.shape[1], dtype=torch.float64)
    ok = (ids >= 0) & (ids < vocab)
    out.index_add_(0, ids[ok], g[ok] * scale)
    mag.index_add_(0, ids[ok], g[ok].abs() * abs(scale))
    return out, mag, torch.bincount(ids[ok], minlength=vocab)


def _ends(lengths, batch, steps):
    return [steps] * batch if lengths is None else [min(max(int(v), 0), steps) for v in lengths]


def conv(x, weight, bias, silu, lengths, state, dy=None, dstate_out=None):
    """{name: (value, magnitude)}."""
    x, w, bias, state, dy, dstate_out = (f64(t) for t in (x, weight, bias, state, dy, dstate_out))
    B, L, D = x.shape
    K = w.shape[1]
    z = torch.zeros
    y, ym = z(B, L, D).double(), z(B, L, D).double()
    last = z(B, K - 1, D).double()
    dx, dxm = z(B, L, D).double(), z(B, L, D).double()
    dst, dstm = z(B, K - 1, D).double(), z(B, K - 1, D).double()
    dw, dwm, db, dbm = z(D, K).double(), z(D, K).double(), z(D).double(), z(D).double()
    b0 = bias if bias is not None else z(D).double()
    for i, n in enumerate(_ends(lengths, B, L)):
        line = torch.cat([state[i] if state is not None else z(K - 1, D).double(), x[i, :n]])
        last[i] = line[n:n + K - 1]
        g, gm = torch.zeros_like(line), torch.zeros_like(line)
        if dstate_out is not None:
            g[n:n + K - 1] += dstate_out[i]
            gm[n:n + K - 1] += dstate_out[i].abs()
        for t in range(n):
            win = line[t:t + K]
            pre = b0 + (w.t() * win).sum(0)
            mag = b0.abs() + (w.t() * win).abs().sum(0)
            s = torch.sigmoid(pre)
            y[i, t] = pre * s if silu else pre
            ym[i, t] = (1.1 * mag + pre.abs() * (pre.abs() + 1)) if silu else mag     # |silu'| < 1.1; s is off by (|pre| + 4) u
            if dy is not None:
                slope = s * (1 + pre * (1 - s)) if silu else torch.ones_like(s)
                # d slope / d pre is under 0.51; its own roundings are relative to s (1 + |pre|), with s off by (|pre| + 4) u
                slope_m = 0.51 * mag + s * (1 + pre.abs()) * (1 + pre.abs()) if silu else slope
                dp, dpm = dy[i, t] * slope, dy[i, t].abs() * torch.maximum(slope_m, slope.abs())
                g[t:t + K] += dp * w.t()
                gm[t:t + K] += dpm * w.t().abs()
                dw += (dp * win).t()
                dwm += (dpm * win.abs()).t()
                db += dp
                dbm += dpm
        dst[i], dstm[i] = g[:K - 1], gm[:K - 1]
        dx[i, :n], dxm[i, :n] = g[K - 1:], gm[K - 1:]
    return {"y": (y, ym), "state": (last, last.abs()), "x": (dx, dxm), "weight": (dw, dwm), "bias": (db, dbm), "dstate": (dst, dstm)}


def scan(x, dt, a, b, c, d, z, dt_bias, softplus, lengths, state, dy=None, dstate_out=None):
    """{name: (value, magnitude)}; b and c [B, L, G, N]."""
    x, dt, a, b, c, d, z, dt_bias, state, dy, dstate_out = (f64(t) for t in (x, dt, a, b, c, d, z, dt_bias, state, dy, dstate_out))
    B, L, D = x.shape
    G, N = b.shape[2:]
    zero = lambda *s: torch.zeros(*s, dtype=torch.float64)
    y, ym, last, lastm = zero(B, L, D), zero(B, L, D), zero(B, D, N), zero(B, D, N)
    out = {k: [torch.zeros_like(v), torch.zeros_like(v)] for k, v in (("x", x), ("dt", x), ("z", x), ("b", b), ("c", c), ("a", a))}
    out.update({k: [zero(D), zero(D)] for k in ("d", "dt_bias")})
    out["dstate"] = [zero(B, D, N), zero(B, D, N)]
    skip = d if d is not None else zero(D)
    for i, n in enumerate(_ends(lengths, B, L)):
        h = state[i].clone() if state is not None else zero(D, N)
        hm = h.abs()
        keep = []
        for t in range(n):
            raw = dt[i, t] + (dt_bias if dt_bias is not None else 0.0)
            step = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
            # softplus is off by its own few u and by the rounding of raw, whose slope is at most 1
            step_m = torch.maximum(step.abs(), raw.abs() + (dt_bias.abs() if dt_bias is not None else 0.0)) if not softplus else step + torch.sigmoid(raw) * (dt[i, t].abs() + (dt_bias.abs() if dt_bias is not None else 0.0))
            bt, ct = (v[i, t][:, None].expand(G, D // G, N).reshape(D, N) for v in (b, c))
            e = torch.exp(step[:, None] * a)
            em = e * (1 + (step_m[:, None] * a.abs()))                        # a decay's error: the exponent's size in roundings
            old, oldm = h, hm
            h = e * h + (step * x[i, t])[:, None] * bt
            hm = em * hm + (step_m * x[i, t].abs())[:, None] * bt.abs()
            zt = z[i, t] if z is not None else None
            gate = zt * torch.sigmoid(zt) if z is not None else torch.ones(D, dtype=torch.float64)
            gate_m = gate.abs() * (1 + zt.abs()) if z is not None else gate
            inner, inner_m = (h * ct).sum(-1) + skip * x[i, t], (hm * ct.abs()).sum(-1) + (skip * x[i, t]).abs()
            y[i, t], ym[i, t] = inner * gate, inner_m * gate_m
            keep.append((raw, step, step_m, bt, ct, e, em, old, oldm, h, hm, gate, gate_m, inner, inner_m))
        last[i], lastm[i] = h, hm
        if dy is None and dstate_out is None:
            continue
        g = dstate_out[i].clone() if dstate_out is not None else zero(D, N)
        gm = g.abs()
        for t in reversed(range(n)):
            raw, step, step_m, bt, ct, e, em, old, oldm, h, hm, gate, gate_m, inner, inner_m = keep[t]
            dyt = dy[i, t] if dy is not None else zero(D)
            xt = x[i, t]
            if z is not None:
                s, zt = torch.sigmoid(z[i, t]), z[i, t]
                out["z"][0][i, t] = dyt * inner * s * (1 + zt * (1 - s))
                out["z"][1][i, t] = dyt.abs() * inner_m * s * (1 + zt.abs()) * (1 + zt.abs())
            do, dom = dyt * gate, dyt.abs() * gate_m
            out["d"][0] += do * xt
            out["d"][1] += dom * xt.abs()
            g, gm = g + do[:, None] * ct, gm + dom[:, None] * ct.abs()
            for k, v in enumerate((do[:, None] * h, dom[:, None] * hm)):
                out["c"][k][i, t] = v.reshape(G, D // G, N).sum(1)
            for k, v in enumerate((g * (step * xt)[:, None], gm * (step_m * xt.abs())[:, None])):
                out["b"][k][i, t] = v.reshape(G, D // G, N).sum(1)
            push, push_m = (g * bt).sum(-1), (gm * bt.abs()).sum(-1)
            q, qm = g * old * e, gm * oldm * em
            out["a"][0] += q * step[:, None]
            out["a"][1] += qm * step_m[:, None]
            out["x"][0][i, t], out["x"][1][i, t] = step * push + skip * do, step_m * push_m + skip.abs() * dom
            rs = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
            rsm = rs * (1 + raw.abs() + (dt_bias.abs() if dt_bias is not None else 0.0)) if softplus else rs
            out["dt"][0][i, t] = ((q * a).sum(-1) + xt * push) * rs
            out["dt"][1][i, t] = ((qm * a.abs()).sum(-1) + xt.abs() * push_m) * rsm
            g, gm = g * e, gm * em
        out["dstate"][0][i], out["dstate"][1][i] = g, gm
    out["dt_bias"] = [out["dt"][0].sum((0, 1)), out["dt"][1].sum((0, 1))]
    return {"y": (y, ym), "state": (last, lastm), **{k: tuple(v) for k, v in out.items()}}
