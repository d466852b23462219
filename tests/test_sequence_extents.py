"""What the sequence kernels rely on, checked on the host over random sizes: every part of a workspace holds the largest index that a kernel
forms in it, segments stay inside 32-bit offsets, LDS inside a compute unit's, and no work is left out.

The plans below restate the host code's (embed_grad_plan, conv_grad_plan, scan_plan); the library's own sizes of the workspaces and marks
pin them: the two have to agree at every size."""
import ctypes as C
import math
import random

import pytest

from multimodn_amd import hip

MAX_GRID, LDS = 0x7fffffff, 160 * 1024
SORT_TILE, SORT_BINS, SMALL_ROWS, FEW_ROWS, FEW_R = 1024, 512, 8192, 8192, 64
CONV_RUN, SUM_COLS = 16, 16


def up(a, b):
    return -(-a // b)


def pad(n):
    return up(n, 256) * 256


def log2_up(n, most):
    k = 0
    while k < most and (1 << k) < n:
        k += 1
    return k


def sum_parts_bytes(parts, n):
    if parts <= 8192:
        return 0
    each = 1024
    while each * 8192 < parts:
        each *= 2
    assert up(parts, each) <= 8192                                            # (the second launch takes what the first leaves)
    return pad(4 * up(parts, each) * n)


def size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def test_embedding_gradient():
    lib, rng = hip.load(), random.Random(1)
    for turn in range(4000):
        rows, vocab, width = size(rng, 1, 2 ** 26), size(rng, 1, 2 ** 30), size(rng, 1, 8192)
        if turn % 3 == 0:
            rows, vocab = size(rng, 1, 9000), size(rng, 1, 40000)
        bits_needed = vocab.bit_length()                                      # keys 0 .. vocab
        passes = up(bits_needed, 9)
        bits = up(bits_needed, passes)
        assert 1 << bits <= SORT_BINS and bits * passes >= bits_needed and (passes - 1) * bits < 32
        run = up(up(rows, SORT_TILE), 128) * SORT_TILE
        nwg = up(rows, run)
        assert nwg <= 128 and run < 2 ** 31 and nwg * run >= rows > (nwg - 1) * run
        chunk = 16
        while chunk < 512 and rows // chunk > 2048:
            chunk *= 2
        nchunk = up(rows, chunk)
        parts = {"hist": 4 * nwg * (1 << bits), "present": 4 * vocab, "keys": 4 * rows, "pos": 4 * rows, "keys2": 4 * rows, "pos2": 4 * rows,
                 "part": 4 * nchunk * 2 * width}
        assert sum(map(pad, parts.values())) == lib.mmn_seq_embed_grad_bytes(rows, vocab, width), (rows, vocab, width)
        assert 4 * (((nchunk - 1) * 2 + 1) * width + width) <= parts["part"]          # the last chunk's tail, its last column
        assert nwg * (1 << bits) < 2 ** 31                                    # hist is read with 32-bit indexes
        assert up(nchunk, 8) <= MAX_GRID and up(width, 64) <= 65535
        # one workgroup's sort: positions in 16 bits, keys of the last pass's digit inside the counts
        assert SMALL_ROWS <= 1 << 16 and FEW_ROWS <= 1 << 16
        # few ids over a small table: every table row has one owner, whose list it fits
        for fv in (1, 2):
            tiles = up(width, 64 * fv)
            if rows > FEW_ROWS or vocab * tiles > 512 * FEW_R:
                continue
            nb = 0
            while 1 << nb < vocab and (tiles << (nb + 1) <= 512 or up(vocab, 1 << nb) > FEW_R):
                nb += 1
            here = up(vocab, 1 << nb)
            assert here <= FEW_R and tiles << nb <= MAX_GRID and log2_up(here, 31) <= 6
            for v in {0, vocab - 1, vocab // 2, rng.randrange(vocab), rng.randrange(vocab)}:
                row, b = v >> nb, (v + (v >> nb)) & ((1 << nb) - 1)
                assert row < here and (row << nb) + ((b - row) & ((1 << nb) - 1)) == v


def test_convolution_gradient():
    lib, rng = hip.load(), random.Random(2)
    for turn in range(4000):
        c = hip.ConvDesc()
        c.batch, c.steps, c.width, c.taps, c.type = size(rng, 1, 2 ** 20), size(rng, 1, 2 ** 20), size(rng, 1, 2 ** 20), rng.choice([2, 3, 4]), rng.randrange(3)
        c.x_row, c.x_step, c.dy_row, c.dy_step = c.width * c.steps, c.width, c.width * c.steps, c.width
        need = []
        for v in {4 if c.width % 4 == 0 else 1, 1}:
            lanes = log2_up(up(c.width, v), 6)
            gy = up(up(c.width, v), 1 << lanes)
            jobs = c.batch * up(c.steps, CONV_RUN)
            per = 256 >> lanes
            parts = max(1, min(up(jobs, per), 1 if gy >= 1024 else 1024 // gy))
            n = (c.taps + 1) * c.width
            assert 4 * (((parts - 1) * (c.taps + 1) + c.taps) * c.width + c.width) <= pad(4 * n * parts)
            assert gy * (1 << lanes) * v >= c.width and parts * gy <= MAX_GRID
            assert (c.taps + 1) * (1 << lanes) * v * 4 <= LDS and 256 * v * 4 <= LDS and (1 << lanes) * per == 256
            need.append(pad(4 * n * parts) + sum_parts_bytes(parts, n))
        assert lib.mmn_seq_conv_grad_bytes(C.byref(c)) == max(need), turn


def scan_plan(s, backward):
    step = lambda v: v if s.steps > 1 else s.width
    per = s.width // s.groups
    tiles = up(per, 64)
    best, waves = 1 << 30, 1
    for w in range(1, 5):
        cost = 4 * up(tiles, w) * w + up(tiles, w)
        if cost < best:
            best, waves = cost, w
    cblocks = up(tiles, waves)
    total = s.batch * s.groups * tiles
    want = 1 if total >= 896 else up(1024 * (3 if s.lengths else 2), max(total, 1))
    ck_log2 = 3 if s.steps <= 2048 and total * up(s.steps, 16) <= 512 else 4
    ck = 1 << ck_log2
    n = min(up(s.steps, ck), want)
    stride = max([s.width, step(s.x_step), step(s.dt_step)] + ([step(s.z_step)] if s.z else []) + ([step(s.dy_step)] if backward else []))
    fits = (1 << 30) // (stride * 4) // ck * ck
    if fits > 0:
        n = max(n, up(s.steps, fits))
    seg = up(up(s.steps, n), ck) * ck if n > 1 else s.steps
    nseg = up(s.steps, seg)
    most = 8192 // (s.groups * tiles)
    slots = max(most, 1) if backward and nseg == 1 and s.batch > most else s.batch
    is_sorted = bool(s.lengths) and total >= 896 and s.batch <= 16384
    order = is_sorted and nseg == 1 and slots == s.batch
    m = {"order": 4 * s.batch if order and not s.marks else 0, "segh": 4 * s.batch * nseg * s.states * s.width if nseg > 1 else 0,
         "segdt": 4 * s.batch * nseg * s.width if nseg > 1 else 0}
    if backward:
        k = (s.states + 2) * s.width
        m.update(part=4 * slots * nseg * k, mid=sum_parts_bytes(slots * nseg, k),
                 bc=4 * cblocks * s.batch * s.steps * s.groups * 2 * s.states if cblocks > 1 else 0)
    return dict(waves=waves, cblocks=cblocks, ck_log2=ck_log2, seg=seg, nseg=nseg, nmark=up(s.steps, ck), slots=slots, sorted=is_sorted, stride=stride, parts=m,
                per=per, step=step)


@pytest.mark.parametrize("backward", [False, True])
def test_scan(backward):
    lib, rng = hip.load(), random.Random(3)
    seen = set()
    for turn in range(6000):
        s = hip.ScanDesc()
        s.groups = rng.choice([1, 1, 1, 2, 3, 8])
        s.width = s.groups * size(rng, 1, rng.choice([300, 4096, 2 ** 20]))
        s.batch, s.steps, s.states, s.type = size(rng, 1, 2 ** 20), size(rng, 1, 2 ** 20), rng.randint(1, 32), rng.randrange(3)
        if s.width > 1 << 23:
            continue
        for name in ("x_step", "dt_step", "z_step", "dy_step"):
            setattr(s, name, rng.choice([s.width, s.width, min(2 * s.width, 1 << 23), rng.randint(s.width, 1 << 23)]))
        s.z, s.lengths, s.marks = rng.choice([None, 256]), rng.choice([None, 256]), (256 if backward else rng.choice([None, 256]))
        p = scan_plan(s, backward)
        assert max(sum(map(pad, p["parts"].values())), 256) == lib.mmn_seq_scan_bytes(C.byref(s), int(backward)), turn
        marks = s.batch * p["nmark"] * s.states * s.width
        assert lib.mmn_seq_scan_marks(C.byref(s)) == marks + (s.batch if p["sorted"] else 0)
        # both passes cut at marks, take all steps and leave no segment empty
        ck, seg, nseg = 1 << p["ck_log2"], p["seg"], p["nseg"]
        assert (nseg == 1 or seg % ck == 0) and nseg * seg >= s.steps > (nseg - 1) * seg
        assert (s.steps - 1) >> p["ck_log2"] < p["nmark"]
        # 32-bit offsets: a segment's bytes, the up to 8 steps that are requested behind it, and lanes without a channel, which start at 2^31
        size_of = 4 if s.type == 0 else 2
        for name, there in (("x_step", True), ("dt_step", True), ("z_step", bool(s.z)), ("dy_step", backward), (None, True)):
            if not there:
                continue
            stride = p["step"](getattr(s, name)) if name else s.width
            n = min(seg, s.steps)
            held, reach = ((n - 1) * stride + s.width) * size_of, (n + 8) * stride * size_of
            assert n * stride * size_of >= held                               # (a step behind the last lies behind the buffer's end)
            assert held <= 1 << 30 and reach + s.width * size_of < 1 << 31 and (1 << 31) - 8 * stride * size_of >= held
            assert (1 << 32) - 8 * stride * size_of >= held                   # a walk backwards that passes the first step
        padded = 4 if s.states <= 4 else 8 if s.states <= 8 else 16 if s.states <= 16 else 32
        assert s.states * s.width * 4 <= 1 << 30 and padded * s.width * 4 < 1 << 31
        # the largest places: states of segments and marks, partial sums, sums of channel blocks
        if nseg > 1:
            assert 4 * (((s.batch - 1) * nseg + nseg - 1) * s.states * s.width + s.states * s.width) <= p["parts"]["segh"]
        if backward:
            assert 4 * ((p["slots"] - 1) * nseg + nseg) * (s.states + 2) * s.width <= p["parts"]["part"]
            if p["cblocks"] > 1:
                last = (p["cblocks"] - 1) * s.batch * s.steps * s.groups * 2 * s.states + ((s.batch * s.steps - 1) * s.groups + s.groups - 1) * 2 * s.states + 2 * s.states - 1
                assert 4 * (last + 1) <= p["parts"]["bc"]
            assert 4 * (2 * 16 * padded + p["waves"] * (16 * 2 * padded + 3 * padded * 64)) <= LDS
            assert 64 * p["waves"] >= 2 * padded                              # (each of the 2 NP sums of a step has a thread)
        assert 64 * p["waves"] * p["cblocks"] >= p["per"]
        seen.add((nseg > 1, nseg > (16 if p["ck_log2"] == 3 else 8), p["sorted"], p["ck_log2"], p["cblocks"] > 1, p["slots"] < s.batch))
    assert len(seen) >= 15                                                    # (the sample reaches most kinds of plans)
