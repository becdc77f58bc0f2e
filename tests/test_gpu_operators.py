"""The device operators against their restatement in 64 bits (tests/operators_ref.py).  Needs an MI355X.

Tolerances: the value's own rounding, half a step of its type, plus c * 2^-24 times what the absolute values of the terms add
up to, c counting the roundings that a term goes through at most.  exp(v) counts |v| + 2 (its argument's rounding and its own)."""
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

import recommendation_amd as ra
from recommendation_amd import ops
from tests import operators_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LEAST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}   # below the type's normal range steps are absolute


def close(got, want, slack, what):
    t = got.dtype
    got, slack = got.double().cpu(), torch.as_tensor(slack, dtype=torch.float64)
    allowed = torch.finfo(t).eps / 2 * (want.abs() + slack) + slack + LEAST[t]
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine].nan_to_num(9e9), want[~fine].nan_to_num(9e9)), what
    assert torch.isfinite(got[fine]).all(), what
    off = ((got - want).abs() - allowed.expand_as(want))[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()), float(allowed.max()))


class Source:
    """Random inputs: a tensor on the GPU and the same values in 64 bits."""

    def __init__(self, seed, t):
        self.gen, self.t = torch.Generator().manual_seed(seed), t

    def __call__(self, *shape, scale=1.0, t=None):
        v = (torch.randn(*shape, generator=self.gen) * scale).to(t or self.t)
        return v.to(DEV), v.double()

    def f32(self, *shape, scale=1.0):
        return self(*shape, scale=scale, t=torch.float32)


def strided(t, pad, shift):
    """The same values as rows of a wider array that starts `shift` elements into its storage."""
    rows, width = t.shape
    store = torch.full((rows * (width + pad) + shift + 8,), float("nan"), dtype=t.dtype, device=t.device)
    v = store[shift:shift + rows * (width + pad)].view(rows, width + pad)[:, :width]
    v.copy_(t)
    return v


def offsets(off):
    return torch.tensor(off, dtype=torch.int64, device=DEV)


# ------------------------------------------------------------------ convolution
CONV = [  # type, channels, taps, offsets, rows, bias, silu, initial
    ("f32", 8, 4, [0, 5], 5, True, True, False),
    ("f32", 1, 2, [0, 1, 1, 2, 2], 2, False, True, True),
    ("bf16", 64, 4, [0, 1, 40, 40, 73, 200], 200, True, True, True),
    ("f16", 24, 3, [0, 100], 100, True, False, False),
    ("bf16", 37, 8, [2, 2, 9, 11, 90], 95, True, True, True),
    ("f32", 260, 5, [0, 33, 64, 65, 66, 67, 96], 96, True, True, True),
    ("f16", 128, 6, [0, 0, 0], 3, True, True, True),
    ("bf16", 16, 7, [0, 31, 32, 33, 64, 97, 129], 129, False, True, False),
]


@pytest.mark.parametrize("layout", ["packed", "strided"])
@pytest.mark.parametrize("case", CONV, ids=[f"{c[0]}-{c[1]}x{c[2]}" for c in CONV])
def test_conv_and_gradient(case, layout):
    tn, ch, W, off, rows, has_bias, silu, has_init = case
    src = Source(ch * 100 + W, TYPES[tn])
    S = len(off) - 1
    (x, x6), (dy, dy6) = src(rows, ch), src(rows, ch)
    if layout == "strided":
        x, dy = strided(x, 5, 1), strided(dy, 3, 2)
    w, w6 = src.f32(ch, W, scale=0.5)
    b, b6 = src.f32(ch) if has_bias else (None, None)
    i, i6 = src(S, W - 1, ch) if has_init else (None, None)
    df, df6 = src(S, W - 1, ch)
    y, fin = ops.history_conv(x, w, b, seq_off=offsets(off), initial=i, silu=silu, want_final=True)
    y6, fin6 = ref.conv(x6, w6, b6, off, i6, silu)
    M, _ = ref.conv(x6, w6, b6, off, i6, silu, absolute=True)
    close(y, y6, U * (1.1 * (W + 2) * M + y6.abs() * (M + 5)), "y")
    assert torch.equal(fin.double().cpu(), fin6)
    g = ops.history_conv_backward(dy, x, w, b, seq_off=offsets(off), initial=i, silu=silu, dfinal=df)
    want = ref.conv_gradient(dy6, x6, w6, b6, off, i6, silu, df6)
    size = ref.conv_gradient(dy6, x6, w6, b6, off, i6, silu, df6, absolute=True)
    c = U * (2 * W + 16 + float(M.max()))
    close(g.dx, want[0], c * size[0], "dx")
    close(g.dweight, want[1], (c + U * rows) * size[1], "dweight")
    if has_bias:
        close(g.dbias, want[2], (c + U * rows) * size[2], "dbias")
    if has_init:
        close(g.dinitial, want[3], c * size[3], "dinitial")
    lo, hi = off[0], off[-1]
    assert not y[:lo].any() and not y[hi:].any() and not g.dx[:lo].any() and not g.dx[hi:].any()


@pytest.mark.parametrize("ch,W,tn", [(128, 4, "bf16"), (64, 3, "f32"), (96, 2, "f16")])
def test_conv_long_strips_against_whole_arrays_in_64_bits(ch, W, tn):
    """Enough rows for the longest strips; the reference shifts whole arrays on the GPU."""
    src = Source(ch, TYPES[tn])
    rows, n = 300001, 3000
    off = torch.cat([torch.zeros(1, dtype=torch.int64), torch.randint(0, rows + 1, (n - 1,), generator=src.gen).sort().values, torch.tensor([rows])]).to(DEV)
    x, dy = src(rows, ch)[0], src(rows, ch)[0]
    w, b = src.f32(ch, W, scale=0.5)[0], src.f32(ch)[0]
    x6, dy6, w6 = x.double(), dy.double(), w.double()
    t = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(off, t, right=True) - 1
    at, left = t - off[seq], off[seq + 1] - 1 - t

    def behind(v, k):   # row t - k of the same history, or 0
        return torch.where((at >= k)[:, None], torch.roll(v, k, 0), torch.zeros((), dtype=torch.float64, device=DEV))

    def ahead(v, k):
        return torch.where((left >= k)[:, None], torch.roll(v, -k, 0), torch.zeros((), dtype=torch.float64, device=DEV))

    v, M = b.double().expand(rows, ch), b.double().abs().expand(rows, ch)
    for j in range(W):
        v, M = v + w6[:, j] * behind(x6, W - 1 - j), M + (w6[:, j] * behind(x6, W - 1 - j)).abs()
    g = torch.sigmoid(v)
    y, _ = ops.history_conv(x, w, b, seq_off=off)
    close(y, (v * g).cpu(), (U * (1.1 * (W + 2) * M + (v * g).abs() * (M + 5))).cpu(), "y")
    d, D = dy6 * g * (1 + v * (1 - g)), dy6.abs() * (1.1 + 0.5 * M)
    got = ops.history_conv_backward(dy, x, w, b, seq_off=off)
    c = U * (2 * W + 16 + float(M.max()))
    want, size = sum(w6[:, W - 1 - k] * ahead(d, k) for k in range(W)), sum(w6[:, W - 1 - k].abs() * ahead(D, k) for k in range(W))
    close(got.dx, want.cpu(), (c * size).cpu(), "dx")
    dw, size = [(d * behind(x6, W - 1 - j)).sum(0) for j in range(W)], [(D * behind(x6, W - 1 - j).abs()).sum(0) for j in range(W)]
    # a thread adds up at most 4 strips of 128 rows one after the other, a block's threads and the blocks after that
    close(got.dweight, torch.stack(dw, 1).cpu(), ((c + U * 600) * torch.stack(size, 1)).cpu(), "dweight")
    close(got.dbias, d.sum(0).cpu(), ((c + U * 600) * D.sum(0)).cpu(), "dbias")


def test_conv_many_rows_over_blocks():
    """More rows than one walk of all blocks takes: the partial sums go around."""
    src = Source(5, torch.float32)
    rows, ch, W = 140000, 8, 2
    off = [0, 3, 70000, 70001, rows]
    x, x6 = src(rows, ch)
    dy, dy6 = src(rows, ch)
    w, w6 = src.f32(ch, W)
    g = ops.history_conv_backward(dy, x, w, seq_off=offsets(off), silu=False)
    back = torch.cat([torch.zeros(1, ch, dtype=torch.float64), x6[:-1]])
    back[off[:-1]] = 0
    want = torch.stack([(dy6 * back).sum(0), (dy6 * x6).sum(0)], 1)
    size = torch.stack([(dy6 * back).abs().sum(0), (dy6 * x6).abs().sum(0)], 1)
    close(g.dweight, want, U * rows * size, "dweight")
    nxt = torch.cat([dy6[1:], torch.zeros(1, ch, dtype=torch.float64)])
    nxt[[o - 1 for o in off[1:]]] = 0
    close(g.dx, dy6 * w6[:, 1] + nxt * w6[:, 0], U * 4 * (dy6.abs() * w6[:, 1].abs() + nxt.abs() * w6[:, 0].abs()), "dx")


@pytest.mark.parametrize("tn,ch,W", [("f32", 5, 2), ("bf16", 128, 4), ("f16", 4104, 3), ("f32", 8, 8)])
def test_conv_step_goes_on_where_the_prompt_ended(tn, ch, W):
    src = Source(ch, TYPES[tn])
    off, rows = [0, 4, 4, 30], 30
    x, x6 = src(rows, ch)
    more, more6 = src(7, ch)
    w, w6 = src.f32(ch, W, scale=0.5)
    b, b6 = src.f32(ch)
    _, pool = ops.history_conv(x, w, b, seq_off=offsets(off), want_final=True)
    # two clicks of history 2, one of 0, three of 1, in this order, and a row without a slot
    order = [2, 0, 1, -1, 2, 1, 1]
    slots = torch.tensor(order, dtype=torch.int32, device=DEV)
    before = pool.clone()
    y = ops.history_conv_step(more, w, b, state=pool, slots=slots)
    whole, at = [], {}
    for s in range(3):
        mine = [r for r, o in enumerate(order) if o == s]
        at.update({r: sum(len(k) for k in whole) + (off[s + 1] - off[s]) + j for j, r in enumerate(mine)})
        whole.append(torch.cat([x6[off[s]:off[s + 1]], more6[mine]]))
    line = torch.cat(whole)
    o2 = np.cumsum([0] + [len(k) for k in whole]).tolist()
    y6, fin6 = ref.conv(line, w6, b6, o2, None, True)
    M, _ = ref.conv(line, w6, b6, o2, None, True, absolute=True)
    rows_of = [at[r] for r in range(7) if order[r] >= 0]
    keep = [r for r in range(7) if order[r] >= 0]
    close(y[keep], y6[rows_of], U * (1.1 * (W + 2) * M[rows_of] + y6[rows_of].abs() * (M[rows_of] + 5)), "y")
    assert not y[3].any()
    assert torch.equal(pool.double().cpu(), fin6)
    # a slot outside the pool moves nothing
    kept = pool.clone()
    z = ops.history_conv_step(more[:2].contiguous(), w, b, state=pool, slots=torch.tensor([3, -7], dtype=torch.int32, device=DEV))
    assert torch.equal(pool, kept) and not z.any() and not torch.equal(before, kept)


# ------------------------------------------------------------------ scan
SCAN = [  # type, channels, groups, states, offsets, rows, gate, D, bias, softplus, initial
    ("f32", 8, 1, 16, [0, 5], 5, True, True, True, True, False),
    ("f32", 1, 1, 1, [0, 1, 1, 2], 2, False, False, False, False, True),
    ("bf16", 64, 1, 16, [0, 1, 40, 40, 73, 200], 200, True, True, True, True, True),
    ("f16", 66, 2, 9, [0, 100, 301], 301, True, True, True, True, True),
    ("f32", 70, 1, 4, [3, 3, 30, 31, 90], 95, True, False, True, True, True),
    ("bf16", 130, 1, 16, [0, 65], 65, False, True, False, True, False),
    ("f32", 36, 3, 32, [0, 16, 32, 33, 64, 130], 130, True, True, True, True, True),
    ("f16", 18, 1, 61, [0, 47, 48], 48, True, True, False, True, False),
    ("f32", 300, 1, 3, [0, 17, 90], 90, True, True, True, True, True),
    ("f32", 12, 2, 7, [0, 0, 0], 4, True, True, True, True, True),
    ("f32", 48, 2, 16, [1, 4, 4, 20, 21, 22, 23, 40, 56, 72, 150], 160, True, True, True, True, False),
    ("bf16", 20, 1, 32, [0, 16, 31, 64, 65, 96], 96, True, True, True, True, False),
    ("f16", 40, 1, 2, [0, 1, 2, 3, 4, 5, 6, 7, 8, 60], 60, True, False, True, True, False),
    ("bf16", 33, 1, 8, [0, 40, 48, 100], 100, False, True, True, True, False),
]


def scan_inputs(case, layout="packed"):
    tn, ch, G, N, off, rows, gate, has_D, has_bias, sp, has_init = case
    src = Source(ch * 7 + N, TYPES[tn])
    S = len(off) - 1
    v = {"u": src(rows, ch), "delta": src(rows, ch, scale=0.5), "B": src(rows, G, N), "C": src(rows, G, N)}
    if not sp:
        v["delta"] = tuple(t.abs() for t in v["delta"])
    a = -(torch.rand(ch, N, generator=src.gen) * 2 + 0.05)
    v["A"] = (a.to(DEV), a.double())
    v["D"] = src.f32(ch) if has_D else (None, None)
    v["z"] = src(rows, ch) if gate else (None, None)
    v["bias"] = src.f32(ch) if has_bias else (None, None)
    v["initial"] = src.f32(S, ch, N) if has_init else (None, None)
    if layout == "strided":
        for k, pad, shift in (("u", 5, 1), ("delta", 2, 3), ("z", 1, 0)):
            if v[k][0] is not None:
                v[k] = (strided(v[k][0], pad, shift), v[k][1])
        for k in ("B", "C"):
            v[k] = (strided(v[k][0].view(rows, G * N), 3, 1).unflatten(1, (G, N)), v[k][1])
    gpu = [v[k][0] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")]
    six = {k: v[k][1] for k in v}
    return src, gpu, six, v["initial"][0]


def scan_count(case, six):
    """Roundings a term of the recurrence goes through at most, over the longest history, and the most of |exponent| a step has."""
    off, rows = case[4], case[5]
    raw = six["delta"] + (six["bias"] if six["bias"] is not None else 0)
    dt = ref.softplus(raw) if case[9] else raw
    most = float(dt.max()) * float(six["A"].abs().max()) if rows else 0.0
    longest = max(b - a for a, b in zip(off, off[1:])) if len(off) > 1 else 0
    # a step: exp's argument (delta off by 8: exp, log1p, addition; A log2e by 2), exp itself, a product and a sum, and a
    # chunk's handing over (the sum of its delta: as many roundings again)
    return longest * (12 * most + 6) + 24


@pytest.mark.parametrize("layout", ["packed", "strided"])
@pytest.mark.parametrize("case", SCAN, ids=[f"{c[0]}-{c[1]}:{c[2]}x{c[3]}" for c in SCAN])
def test_scan_and_gradient(case, layout):
    tn, ch, G, N, off, rows, gate, has_D, has_bias, sp, has_init = case
    src, x, six, init = scan_inputs(case, layout)
    S = len(off) - 1
    (dy, dy6), (df, df6) = src(rows, ch), src.f32(S, ch, N) if has_init else (None, None)   # (states in and out go together or not at all)
    if layout == "strided":
        dy = strided(dy, 7, 1)
    y, fin, kept = ops.history_scan(*x, seq_off=offsets(off), initial=init, softplus=sp, want_final=True, want_checkpoints=True)
    y6, fin6 = ref.scan(**six, off=off, use_softplus=sp)
    ya, fina = ref.scan(**six, off=off, use_softplus=sp, absolute=True)
    c = scan_count(case, six)
    top = float(six["z"].abs().max()) if gate else 0.0
    close(y, y6, U * (c + N + 16 + top) * ya, "y")
    close(fin, fin6, U * c * fina, "final")
    g = ops.history_scan_backward(dy, *x, seq_off=offsets(off), checkpoints=kept, initial=init, softplus=sp, dfinal=df)
    want = ref.scan_gradient(dy6, **six, off=off, dfinal=df6, use_softplus=sp)
    size = ref.scan_gradient(dy6, **six, off=off, dfinal=df6, use_softplus=sp, absolute=True)
    c = U * (2 * c + 2 * N + ch // G + 40 + 2 * top + (8 + float(six["delta"].abs().max() * 2) if rows else 0))
    for name, got in (("u", g.du), ("delta", g.ddelta), ("z", g.dz), ("B", g.dB), ("C", g.dC)):
        if got is not None:
            close(got, want[name], c * size[name], name)
    for name, got in (("A", g.dA), ("D", g.dD), ("bias", g.ddelta_bias)):
        if got is not None:
            close(got, want[name], (c + U * rows) * size[name], name)
    if has_init:
        close(g.dinitial, want["initial"], c * size["initial"], "initial")
    assert (g.dz is None) == (not gate) and (g.dD is None) == (not has_D) and (g.dinitial is None) == (not has_init)
    for t in (y, g.du, g.ddelta, g.dB, g.dC):
        assert not t[:off[0]].any() and not t[off[-1]:].any()


@pytest.mark.parametrize("tn,ch,G,N,longest,states", [("f32", 512, 2, 16, 2100, True), ("bf16", 96, 1, 16, 9000, True), ("f32", 200, 1, 16, 5000, False)])
def test_scan_over_many_chunks_equals_one_row_after_the_other(tn, ch, G, N, longest, states):
    """Histories that cross from chunk to chunk, against a float64 recurrence on the GPU, gradients included."""
    off = [0, 7, longest, longest, longest + 400]
    rows = off[-1]
    case = (tn, ch, G, N, off, rows, True, True, True, True, states)
    src, x, six, init = scan_inputs(case)
    (dy, dy6), (df, df6) = src(rows, ch), src.f32(4, ch, N) if states else (None, None)
    on = {k: t.to(DEV) if t is not None else None for k, t in six.items()}
    y6, fin6 = ref.scan(**on, off=off)
    ya, _ = ref.scan(**on, off=off, absolute=True)
    y, fin, kept = ops.history_scan(*x, seq_off=offsets(off), initial=init, want_final=True, want_checkpoints=True)
    # decays of these inputs forget a term within some hundred rows: 300 steps' roundings bound what is left of it
    few = U * (300 * 12 + N + 64)
    close(y, y6.cpu(), few * ya.cpu(), "y")
    g = ops.history_scan_backward(dy, *x, seq_off=offsets(off), checkpoints=kept, initial=init, dfinal=df)
    df6 = df6.to(DEV) if states else None
    want = ref.scan_gradient(dy6.to(DEV), **on, off=off, dfinal=df6)
    size = ref.scan_gradient(dy6.to(DEV), **on, off=off, dfinal=df6, absolute=True)
    for name, got in (("u", g.du), ("delta", g.ddelta), ("B", g.dB), ("C", g.dC), ("z", g.dz), ("initial", g.dinitial)):
        if got is not None:
            close(got, want[name].cpu(), 2 * few * size[name].cpu(), name)
    for name, got in (("A", g.dA), ("D", g.dD), ("bias", g.ddelta_bias)):
        close(got, want[name].cpu(), (2 * few + U * rows) * size[name].cpu(), name)


@pytest.mark.parametrize("tn,ch,G,N", [("f32", 5, 1, 3), ("bf16", 256, 2, 16), ("f16", 40, 1, 64)])
def test_scan_step_goes_on_where_the_prompt_ended(tn, ch, G, N):
    off, n = [0, 4, 4, 30], 7
    case = (tn, ch, G, N, [0, 37], 37, True, True, True, True, False)
    _, x, six, _ = scan_inputs(case)
    order = [2, 0, 1, -1, 2, 1, 1]
    per_row = (0, 1, 3, 4, 6)
    head = [t[:30].contiguous() if k in per_row else t for k, t in enumerate(x)]
    tail = [t[30:].contiguous() if k in per_row else t for k, t in enumerate(x)]
    _, pool, _ = ops.history_scan(*head, seq_off=offsets(off), want_final=True)
    y = ops.history_scan_step(*tail, state=pool, slots=torch.tensor(order, dtype=torch.int32, device=DEV))
    rows_of, o2 = [], [0]
    for s in range(3):
        rows_of += list(range(off[s], off[s + 1])) + [30 + r for r, o in enumerate(order) if o == s]
        o2.append(len(rows_of))
    line = {k: (t[rows_of] if k in ("u", "delta", "B", "C", "z") else t) for k, t in six.items()}
    y6, fin6 = ref.scan(**line, off=o2)
    ya, fina = ref.scan(**line, off=o2, absolute=True)
    c = scan_count((tn, ch, G, N, o2, len(rows_of), True, True, True, True, False), line) + N + 16 + float(six["z"].abs().max())
    at = {r: k for k, r in enumerate(rows_of)}
    keep = [r for r in range(n) if order[r] >= 0]
    places = [at[30 + r] for r in keep]
    close(y[keep], y6[places], U * c * ya[places], "y")
    close(pool, fin6, U * c * fina, "state")
    assert not y[3].any()


# ------------------------------------------------------------------ losses
def loss_inputs(tn, rows, items, seed, masked=0.1):
    src = Source(seed, TYPES[tn])
    s = torch.randn(rows, items, generator=src.gen) * 3
    s[torch.rand(rows, items, generator=src.gen) < masked] = float("-inf")
    item = torch.randint(0, items, (rows,), generator=src.gen)
    s[torch.arange(rows), item] = torch.randn(rows, generator=src.gen)
    s = s.to(TYPES[tn])
    return src, s, item


def row_slack(s6, scale):
    """What log p of a row may be off by: exp's arguments and values over the scores' range, and the sum's additions."""
    low = torch.where(torch.isfinite(s6), s6, torch.full_like(s6, float("inf"))).amin(1)
    span = (s6.amax(1) - low).clamp(min=0).nan_to_num(0.0, 0.0, 0.0) * scale * 1.45
    return U * (2 * span + s6.shape[1] / 64 + 40)


def check_dscores(got, want, r, slack_coef, row, what):
    """coef (1 - p) and -coef p: p off by the row's roundings, coef by its own."""
    coef = r["coef"].abs()[:, None]
    slack = coef * r["p"].nan_to_num(0.0) * (row[:, None] + 8 * U) + (slack_coef[:, None] + coef * 4 * U) * torch.maximum(r["p"].nan_to_num(0.0), (want != 0) * 1.0)
    close(got, want, slack, what)


PREFERENCE = [  # type, rows, items, offsets, scale, smoothing, beta, reference
    ("f32", 2, 40, [0, 1, 2], 1.0, 0.0, 0.1, True),
    ("bf16", 37, 4001, [0, 5, 9, 9, 37], 1.0, 0.1, 0.1, True),
    ("f16", 12, 2, [2, 4, 4, 4, 4, 5, 10], 0.7, 0.0, 0.5, False),
    ("f32", 9, 1, [0, 3, 9], 1.0, 0.3, 0.2, True),
    ("f32", 5, 70003, [0, 2, 5], 1.5, 1.0, 0.1, True),
    ("bf16", 700, 129, [0, 650, 700], 1.0, 0.0, 0.01, True),
    ("f16", 4, 33, [0], 1.0, 0.0, 0.1, True),
]


@pytest.mark.parametrize("layout", ["packed", "strided", "in place"])
@pytest.mark.parametrize("case", PREFERENCE, ids=[f"{c[0]}-{c[1]}x{c[2]}" for c in PREFERENCE])
def test_preference_loss(case, layout):
    tn, rows, items, off, scale, eps, beta, has_ref = case
    src, s, item = loss_inputs(tn, rows, items, rows * 3 + items)
    item[::7] = -1 if rows > 8 else item[::7]
    pairs = (len(off) - 1) // 2
    (refs, refs6), (w, w6) = src.f32(rows, scale=0.5), src.f32(pairs)
    gpu = s.to(DEV)
    out = None
    if layout == "strided":
        gpu = strided(gpu, 3, 1)
    if layout == "in place":
        out = gpu
    scores6 = s.double()
    r = ops.preference_loss(gpu, item.to(torch.int32).to(DEV), offsets(off), refs if has_ref else None, beta=beta, label_smoothing=eps, scale=scale, grad_weight=w, out=out)
    want = ref.preference(scores6, item, off, refs6 if has_ref else None, beta, eps, float(np.float32(scale)), w6)
    row = row_slack(scores6, scale)
    lo, hi = off[0], off[-1]
    inside = slice(lo, hi)
    close(r.logp[inside], want["logp"][inside], row[inside], "logp")
    total = torch.stack([row[off[2 * p]:off[2 * p + 2]].sum() for p in range(pairs)]) * beta if pairs else torch.zeros(0, dtype=torch.float64)
    # beta and the smoothing arrive as f32
    total = total + (want["margin"].abs() + want["loss"].abs() + 1) * 4 * U
    close(r.margin, want["margin"], total, "margin")
    close(r.loss, want["loss"], total, "loss")
    per_row = torch.zeros(rows, dtype=torch.float64)
    for k in range(len(off) - 1):
        per_row[off[k]:off[k + 1]] = total[k // 2] + 4 * U
    if layout == "in place":
        assert r.dscores is gpu
        assert torch.equal(r.dscores[:lo].cpu(), s[:lo]) and torch.equal(r.dscores[hi:].cpu(), s[hi:])
    else:
        assert not r.dscores[:lo].any() and not r.dscores[hi:].any() and not r.logp[:lo].any() and not r.logp[hi:].any()
    check_dscores(r.dscores[inside], want["dscores"][inside], {k: want[k][inside] for k in ("coef", "p")}, (per_row * (want["coef"].abs() + beta * 4 * U))[inside], row[inside], "dscores")
    again = ops.preference_loss(s.to(DEV), item.to(torch.int32).to(DEV), offsets(off), refs if has_ref else None, beta=beta, label_smoothing=eps, scale=scale)
    assert again.dscores is None and not again.logp[hi:].any()
    if layout != "strided":   # rows that start at another alignment are cut elsewhere
        assert torch.equal(again.loss, r.loss) and torch.equal(again.logp[inside], r.logp[inside])


POLICY = [("f32", 1, 3, 1.0, True), ("f16", 37, 4001, 1.0, True), ("bf16", 300, 257, 0.5, True), ("f32", 3, 100003, 1.0, False), ("bf16", 1100, 64, 2.0, True), ("f32", 5, 1, 1.0, True)]


@pytest.mark.parametrize("layout", ["packed", "strided", "in place"])
@pytest.mark.parametrize("tn,rows,items,scale,has_ref", POLICY)
def test_policy_loss(tn, rows, items, scale, has_ref, layout):
    src, s, item = loss_inputs(tn, rows, items, rows + items)
    item[1::5] = items + 3
    s6 = s.double()
    lp6 = ref.log_probabilities(s6, item, scale)[0]
    old, adv, w = (lp6 + 0.3 * torch.randn(rows, generator=src.gen)).float(), torch.randn(rows, generator=src.gen), torch.rand(rows, generator=src.gen)
    refs = (lp6 + 0.3 * torch.randn(rows, generator=src.gen)).float()
    adv[::6] = 0
    kl = 0.07 if has_ref else 0.0
    gpu = strided(s.to(DEV), 5, 3) if layout == "strided" else s.to(DEV)
    r = ops.policy_loss(gpu, item.to(torch.int32).to(DEV), old.to(DEV), adv.to(DEV), refs.to(DEV) if has_ref else None, clip_low=0.2, clip_high=0.3, kl_coef=kl, scale=scale,
                        grad_weight=w.to(DEV), out=gpu if layout == "in place" else None)
    want = ref.policy(s6, item, old.double(), adv.double(), refs.double() if has_ref else None, float(np.float32(0.2)), float(np.float32(0.3)), float(np.float32(kl)), scale, w.double())
    row = row_slack(s6, scale)
    x = (refs.double() - want["logp"]).abs()
    ratio = torch.exp(want["logp"] - old.double())
    slack = row * (ratio * adv.double().abs() + kl * torch.exp(x)) + 4 * U * want["loss"].abs()
    close(r.logp, want["logp"], row, "logp")
    close(r.loss, want["loss"], slack, "loss")
    if has_ref:
        close(r.kl, want["kl"], row * torch.exp(x) + 2.0 ** -50, "kl")
    else:
        assert r.kl is None
    check_dscores(r.dscores, want["dscores"], want, slack * w.double() + row * kl * w.double() * torch.exp(x), row, "dscores")


def test_rows_whose_mask_leaves_nothing_and_masked_choices():
    inf = float("inf")
    s = torch.tensor([[-inf, -inf, -inf, -inf, -inf], [0.5, -inf, 1.0, -inf, 2.0], [-inf, -inf, 3.0, -inf, -inf], [1.0, 2.0, 3.0, 4.0, 5.0]], device=DEV)
    item = torch.tensor([1, 4, 2, 0], dtype=torch.int32, device=DEV)
    one = torch.ones(4, device=DEV)
    r = ops.policy_loss(s, item, torch.zeros(4, device=DEV), one, grad_weight=one)
    assert r.loss[0] == 0 and r.logp[0] == 0 and not r.dscores[0].any()
    assert r.logp[2] == 0 and not r.dscores[2].any()           # probability 1: nothing left to learn
    assert not r.dscores[1, [1, 3]].any() and r.dscores[1, 0] > 0 and r.dscores[1, 4] < 0
    # a choice that is masked itself has probability 0
    item = torch.tensor([1, 1, 2, 0], dtype=torch.int32, device=DEV)
    off = offsets([0, 2, 4])
    p = ops.preference_loss(s, item, off, grad_weight=torch.ones(1, device=DEV))
    assert p.logp[1] == -inf and p.margin[0] == -inf and p.loss[0] == inf
    assert torch.isfinite(p.dscores).all() and not p.dscores[0].any() and float((p.dscores[1, 1] + 0.1).abs()) < 1e-6
    q = ops.preference_loss(s, item, offsets([2, 3, 3, 3, 4]), grad_weight=torch.ones(2, device=DEV))
    assert torch.isfinite(q.loss).all() and not q.dscores[:2].any()
    # the other way round: the rejected list has probability 0
    v = ops.preference_loss(s[[3, 1]].contiguous(), torch.tensor([0, 1], dtype=torch.int32, device=DEV), offsets([0, 1, 2]), grad_weight=torch.ones(1, device=DEV))
    assert v.margin[0] == inf and v.loss[0] == 0 and not v.dscores.any()


@pytest.mark.parametrize("tn", ["f32", "f16", "bf16"])
def test_rows_that_one_score_decides(tn):
    """The choice stands 32 above 4096 others, at every place within 16 bytes.  The others' part of the sum is below 4096 e^(4.5 - 32),
    5e-9, so log p is between -5e-9 and 0; a sum that starts at 1 loses or gains no more than that part, and what is left
    of the correction for log2(e)'s rounding is 2^-24 of (32 + 4.5) times it."""
    rows, items = 16, 4096
    s = torch.randn(rows, items, generator=torch.Generator().manual_seed(5)).clamp(-4.5, 4.5)
    item = torch.arange(rows) + 1000
    s[torch.arange(rows), item] = 32.0
    s = s.to(TYPES[tn]).to(DEV)
    zero = torch.zeros(rows, device=DEV)
    r = ops.policy_loss(s, item.int().to(DEV), zero, zero + 1)
    assert float(r.logp.abs().max()) <= 1.1e-8 and float((r.loss + 1).abs().max()) <= 2 ** -24
    p = ops.preference_loss(s, item.int().to(DEV), offsets([0, 12, 16]))
    assert float(p.logp.abs().max()) <= 1.1e-8 and float(p.margin.abs().max()) <= 0.1 * 16 * 1.1e-8


def test_values_that_are_not_finite_stay_in_their_rows():
    s = torch.randn(6, 3000, device=DEV)
    s[1, 7], s[3, 2999], s[4, 0] = float("nan"), float("inf"), torch.finfo(torch.float32).min
    item = torch.arange(6, dtype=torch.int32, device=DEV)
    z, one = torch.zeros(6, device=DEV) - 8, torch.ones(6, device=DEV)
    r = ops.policy_loss(s, item, z, one, grad_weight=one)
    bad = torch.tensor([False, True, False, True, False, False], device=DEV)
    assert torch.equal(torch.isnan(r.logp), bad) and torch.equal(torch.isnan(r.dscores).any(1), bad)
    assert r.dscores[4, 0] == 0                                 # a mask of the type's lowest value is as good as -inf
    # a scan and a convolution: what is not finite in one history does not reach its neighbours
    x = torch.randn(40, 16, device=DEV)
    x[12, 3] = float("nan")
    off = offsets([0, 10, 20, 40])
    w = torch.randn(16, 4, device=DEV)
    y, _ = ops.history_conv(x, w, seq_off=off)
    assert torch.equal(torch.isnan(y).any(1).nonzero()[:, 0].cpu(), torch.arange(12, 16))
    g = ops.history_conv_backward(torch.ones_like(x), x, w, seq_off=off)
    assert torch.isnan(g.dx).any(1).nonzero()[:, 0].tolist() == list(range(10, 16))
    B = torch.randn(40, 1, 8, device=DEV)
    A = -torch.rand(16, 8, device=DEV)
    ys, fin, kept = ops.history_scan(x, torch.randn_like(x), A, B, B, seq_off=off, want_final=True, want_checkpoints=True)
    assert torch.isnan(ys).any(1).nonzero()[:, 0].tolist() == list(range(12, 20)) and torch.isnan(ys).any(0).nonzero()[:, 0].tolist() == [3]
    assert torch.isfinite(fin[[0, 2]]).all() and torch.isnan(fin[1]).any()


# ------------------------------------------------------------------ how they are called
def scan_call(seed=3, rows=700, ch=96, t=torch.bfloat16):
    case = ("bf16", ch, 1, 16, [0, 300, rows], rows, True, True, True, True, True)
    _, x, _, init = scan_inputs(case)
    off = offsets(case[4])
    y, fin, kept = ops.history_scan(*x, seq_off=off, initial=init, want_final=True, want_checkpoints=True)
    g = ops.history_scan_backward(y, *x, seq_off=off, checkpoints=kept, initial=init, dfinal=fin)
    return [y, fin, *[v for v in g if v is not None]]


def conv_call():
    src = Source(9, torch.float16)
    x, _ = src(5000, 72)
    w, _ = src.f32(72, 4)
    b, _ = src.f32(72)
    off = offsets([0, 1, 2000, 5000])
    y, fin = ops.history_conv(x, w, b, seq_off=off, want_final=True)
    g = ops.history_conv_backward(y, x, w, b, seq_off=off, dfinal=fin)
    return [y, fin, g.dx, g.dweight, g.dbias]


def loss_call():
    src, s, item = loss_inputs("bf16", 300, 9001, 1)
    gpu, it = s.to(DEV), item.to(torch.int32).to(DEV)
    w, _ = src.f32(300)
    p = ops.preference_loss(gpu, it, offsets([0, 100, 300]), beta=0.1, grad_weight=w[:1].contiguous())
    q = ops.policy_loss(gpu, it, p.logp, w, p.logp, kl_coef=0.1, grad_weight=w)
    return [*p, *q]


@pytest.mark.parametrize("call", [scan_call, conv_call, loss_call])
def test_equal_inputs_give_equal_bits(call):
    a, b = call(), call()
    assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_calls_on_another_stream():
    want = [t.clone() for f in (scan_call, conv_call, loss_call) for t in f()]
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = [t for f in (scan_call, conv_call, loss_call) for t in f()]
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_captured_and_replayed():
    """Forward, gradient, losses and steps in one graph; every replay against the eager result, eager work between the replays."""
    off = offsets([0, 40, 200])
    src = Source(2, torch.bfloat16)
    x, dy = src(200, 32)[0], src(200, 32)[0]
    w, b = src.f32(32, 4)[0], src.f32(32)[0]
    A, Bm = -torch.rand(32, 16, device=DEV), src(200, 1, 16)[0]
    table = src(500, 32)[0]
    item = torch.arange(200, dtype=torch.int32, device=DEV)
    gw = torch.ones(1, device=DEV)
    pool_c, pool_s = torch.zeros(5, 3, 32, dtype=torch.bfloat16, device=DEV), torch.zeros(5, 32, 16, device=DEV)
    slots = torch.tensor([0, 4, 4], dtype=torch.int32, device=DEV)

    def step():
        c, _ = ops.history_conv(x, w, b, seq_off=off)
        y, _, kept = ops.history_scan(c, c, A, Bm, Bm, seq_off=off, want_checkpoints=True)
        scores = y @ table.t()
        p = ops.preference_loss(scores, item, off, grad_weight=gw, out=scores)
        dyy = (p.dscores @ table.contiguous())
        g = ops.history_scan_backward(dyy, c, c, A, Bm, Bm, seq_off=off, checkpoints=kept)
        gc = ops.history_conv_backward(g.du + g.ddelta, x, w, b, seq_off=off)
        s1 = ops.history_conv_step(x[:3], w, b, state=pool_c, slots=slots)
        s2 = ops.history_scan_step(s1, s1, A, Bm[:3], Bm[:3], state=pool_s, slots=slots)
        return [p.loss, p.logp, g.dA, g.dB, gc.dx, gc.dweight, gc.dbias, s2, pool_c, pool_s]

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    pool_c.zero_(), pool_s.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        x.copy_(src(200, 32)[0])
        pool_c.zero_(), pool_s.zero_()
        want = [t.clone() for t in step()]
        pool_c.zero_(), pool_s.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, want)), k
        step()   # eager work between the replays
        torch.cuda.synchronize()


def test_outputs_leave_other_rows_alone():
    x = torch.randn(50, 8, device=DEV)
    off = offsets([3, 20, 41])
    w = torch.randn(8, 3, device=DEV)
    B, A = torch.randn(50, 1, 4, device=DEV), -torch.rand(8, 4, device=DEV)
    s, item = torch.randn(50, 64, device=DEV), torch.zeros(50, dtype=torch.int32, device=DEV)
    outs = []
    for k, shape in ((0, x.shape), (1, x.shape), (2, s.shape)):
        o = torch.full(shape, 7.0, device=DEV)
        if k == 0:
            ops.history_conv(x, w, seq_off=off, out=o)
        elif k == 1:
            ops.history_scan(x, x, A, B, B, seq_off=off, out=o)
        else:
            ops.preference_loss(s, item, off, grad_weight=torch.ones(1, device=DEV), out=o)
        outs.append(o)
    # what is allocated beside the caller's array has zeros there
    r = ops.preference_loss(s, item, off, grad_weight=torch.ones(1, device=DEV), out=s.clone())
    assert not r.logp[:3].any() and not r.logp[41:].any() and r.logp[3:41].all()
    o = torch.full(x.shape, 7.0, device=DEV)
    ops.history_conv_backward(x, x, w, seq_off=off, out=o)
    for o in outs + [o]:
        assert (o[:3] == 7).all() and (o[41:] == 7).all() and not (o[3:41] == 7).all(1).any()


def test_nothing_to_do():
    x, off = torch.zeros(0, 8, device=DEV), offsets([0, 0, 0])
    w, i = torch.randn(8, 4, device=DEV), torch.randn(2, 3, 8, device=DEV)
    y, fin = ops.history_conv(x, w, seq_off=off, initial=i, want_final=True)
    assert y.shape == (0, 8) and torch.equal(fin, i)
    g = ops.history_conv_backward(x, x, w, seq_off=off, initial=i, dfinal=i)
    assert torch.equal(g.dinitial, i) and not g.dweight.any()
    B, A, h = torch.zeros(0, 1, 4, device=DEV), -torch.rand(8, 4, device=DEV), torch.randn(2, 8, 4, device=DEV)
    y, fin, kept = ops.history_scan(x, x, A, B, B, seq_off=off, initial=h, want_final=True, want_checkpoints=True)
    assert y.shape == (0, 8) and torch.equal(fin, h) and kept.shape == (0, 8, 4)
    g = ops.history_scan_backward(x, x, x, A, B, B, seq_off=off, checkpoints=kept, initial=h, dfinal=h)
    assert torch.equal(g.dinitial, h) and not g.dA.any() and g.dB.shape == (0, 1, 4)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert ops.history_conv_step(x, w, state=i.clone(), slots=none).shape == (0, 8)
    assert ops.history_scan_step(x, x, A, B, B, state=h.clone(), slots=none).shape == (0, 8)
    # a pool without slots, and rows that name one all the same
    lost = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert not ops.history_conv_step(torch.ones(3, 8, device=DEV), w, state=i[:0], slots=lost).any()
    assert not ops.history_scan_step(torch.ones(3, 8, device=DEV), torch.ones(3, 8, device=DEV), A, torch.ones(3, 1, 4, device=DEV), torch.ones(3, 1, 4, device=DEV), state=h[:0], slots=lost).any()
    r = ops.policy_loss(torch.zeros(0, 9, device=DEV), none, torch.zeros(0, device=DEV), torch.zeros(0, device=DEV), grad_weight=torch.zeros(0, device=DEV))
    assert r.loss.shape == (0,) and r.dscores.shape == (0, 9)
    r = ops.preference_loss(torch.zeros(0, 9, device=DEV), none, offsets([0, 0, 0]))
    assert float((r.loss - np.log(2)).abs().max()) < 1e-6 and not r.margin.any()
    with pytest.raises(ValueError, match="2 pairs"):
        ops.preference_loss(torch.zeros(4, 9, device=DEV), none, offsets([0, 0]))


def test_rows_of_no_history_alone():
    """No histories at all, though there are rows: zeros, and parameters that learn nothing from what the rows hold."""
    off = offsets([17])
    x = torch.full((40, 8), float("nan"), device=DEV)
    w, A, B = torch.randn(8, 4, device=DEV), -torch.rand(8, 4, device=DEV), x[:, :4].reshape(40, 1, 4)
    y, fin = ops.history_conv(x, w, w[:, 0].contiguous(), seq_off=off, want_final=True)
    g = ops.history_conv_backward(x, x, w, w[:, 0].contiguous(), seq_off=off)
    assert not y.any() and fin.shape == (0, 3, 8) and not g.dx.any() and not g.dweight.any() and not g.dbias.any()
    y, fin, kept = ops.history_scan(x, x, A, B, B, A[:, 0].contiguous(), x, seq_off=off, want_final=True, want_checkpoints=True)
    g = ops.history_scan_backward(x, x, x, A, B, B, A[:, 0].contiguous(), x, seq_off=off, checkpoints=kept)
    assert not y.any() and fin.shape == (0, 8, 4)
    for name in ("du", "ddelta", "dA", "dB", "dC", "dD", "dz"):
        assert not getattr(g, name).any(), name
    r = ops.preference_loss(x, torch.zeros(40, dtype=torch.int32, device=DEV), off, grad_weight=torch.zeros(0, device=DEV))
    assert r.loss.shape == (0,) and not r.logp.any() and not r.dscores.any()


def test_calls_of_two_threads():
    """Each on a stream of its own, over the same inputs, with workspaces of their own."""
    x, A = torch.randn(3000, 32, device=DEV), -torch.rand(32, 16, device=DEV)
    B, off = torch.randn(3000, 1, 16, device=DEV), offsets([0, 1000, 1001, 3000])
    s, item = torch.randn(6, 50000, device=DEV), torch.arange(6, dtype=torch.int32, device=DEV)
    two, one = offsets([0, 2, 6]), torch.ones(1, device=DEV)

    def work():
        y, _, kept = ops.history_scan(x, x, A, B, B, seq_off=off, want_checkpoints=True)
        g = ops.history_scan_backward(x, x, x, A, B, B, seq_off=off, checkpoints=kept)
        return y, g.du, g.dA, g.dB, ops.preference_loss(s, item, two, grad_weight=one).dscores

    want = work()
    torch.cuda.synchronize()
    with ThreadPoolExecutor(2) as pool:
        def run(_):
            with torch.cuda.stream(torch.cuda.Stream()):
                out = [work() for _ in range(10)]
                torch.cuda.current_stream().synchronize()
            return out
        for outs in pool.map(run, range(2)):
            for got in outs:
                assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_element_offsets_beyond_32_bits():
    """Rows that lie more than 2^31 elements into their array, and a slot that does."""
    n, items = 3, 1000
    store = torch.empty((1 << 31) + 4096, dtype=torch.bfloat16, device=DEV)
    s = torch.randn(n, items, device=DEV).bfloat16()
    far = store.as_strided((n, items), (1 << 30, 1))
    far.copy_(s)
    item = torch.arange(n, dtype=torch.int32, device=DEV)
    z, one = torch.zeros(n, device=DEV), torch.ones(n, device=DEV)
    want = ops.policy_loss(s, item, z, one, grad_weight=one)
    got = ops.policy_loss(far, item, z, one, grad_weight=one, out=far)
    assert all(torch.equal(a, b) for a, b in ((want.loss, got.loss), (want.logp, got.logp), (want.dscores, got.dscores)))
    far.copy_(s)
    w, off = torch.randn(items, 3, device=DEV), offsets([0, 3])
    assert torch.equal(ops.history_conv(s, w, seq_off=off)[0], ops.history_conv(far, w, seq_off=off)[0])
    A, B = -torch.rand(items, 4, device=DEV), torch.randn(3, 1, 4, device=DEV).bfloat16()
    assert torch.equal(ops.history_scan(s, s, A, B, B, seq_off=off)[0], ops.history_scan(far, far, A, B, B, seq_off=off)[0])
    del store, far
    slots, ch, N = 560000, 256, 16                  # 2.3e9 values of state
    pool = torch.empty(slots, ch, N, device=DEV)
    pool[slots - 1] = 1
    x, A, B = torch.randn(1, ch, device=DEV), -torch.rand(ch, N, device=DEV), torch.randn(1, 1, N, device=DEV)
    small = torch.ones(1, ch, N, device=DEV)
    a = ops.history_scan_step(x, x, A, B, B, state=pool, slots=torch.tensor([slots - 1], dtype=torch.int32, device=DEV))
    b = ops.history_scan_step(x, x, A, B, B, state=small, slots=torch.tensor([0], dtype=torch.int32, device=DEV))
    assert torch.equal(a, b) and torch.equal(pool[slots - 1], small[0])


def test_long_runs_of_empty_histories():
    """Hundreds of thousands of them between two clicks: what the other histories get is what they get without them."""
    full = [0, 3, 40, 41, 200]
    gaps = [0, 1, 200000, 70001, 1]   # empty histories behind each of the boundaries
    off, at = [], []
    for o, k in zip(full, gaps):
        off += [o] * (1 + k)
        at.append(len(off) - 1)
    at = at[:-1]                      # the histories that have clicks
    off, few, n = offsets(off), offsets(full), len(off) - 1
    x, w = torch.randn(200, 8, device=DEV), torch.randn(8, 4, device=DEV)
    i, df = torch.randn(n, 3, 8, device=DEV), torch.randn(n, 3, 8, device=DEV)
    y, fin = ops.history_conv(x, w, seq_off=off, initial=i, want_final=True)
    y1, fin1 = ops.history_conv(x, w, seq_off=few, initial=i[at], want_final=True)
    assert torch.equal(y, y1) and torch.equal(fin[at], fin1)
    empty = torch.ones(n, dtype=torch.bool, device=DEV)
    empty[at] = False
    assert torch.equal(fin[empty], i[empty])
    g = ops.history_conv_backward(x, x, w, seq_off=off, initial=i, dfinal=df)
    g1 = ops.history_conv_backward(x, x, w, seq_off=few, initial=i[at], dfinal=df[at])
    assert torch.equal(g.dx, g1.dx) and torch.equal(g.dweight, g1.dweight) and torch.equal(g.dinitial[at], g1.dinitial) and torch.equal(g.dinitial[empty], df[empty])
    A, B = -torch.rand(8, 4, device=DEV), torch.randn(200, 1, 4, device=DEV)
    h, dh = torch.randn(n, 8, 4, device=DEV), torch.randn(n, 8, 4, device=DEV)
    y, fin, kept = ops.history_scan(x, x, A, B, B, seq_off=off, initial=h, want_final=True, want_checkpoints=True)
    y1, fin1, kept1 = ops.history_scan(x, x, A, B, B, seq_off=few, initial=h[at], want_final=True, want_checkpoints=True)
    assert torch.equal(y, y1) and torch.equal(fin[at], fin1) and torch.equal(kept, kept1) and torch.equal(fin[empty], h[empty])
    g = ops.history_scan_backward(x, x, x, A, B, B, seq_off=off, checkpoints=kept, initial=h, dfinal=dh)
    g1 = ops.history_scan_backward(x, x, x, A, B, B, seq_off=few, checkpoints=kept, initial=h[at], dfinal=dh[at])
    for name in ("du", "ddelta", "dA", "dB", "dC"):
        assert torch.equal(getattr(g, name), getattr(g1, name)), name
    assert torch.equal(g.dinitial[at], g1.dinitial) and torch.equal(g.dinitial[empty], dh[empty])


def test_steps_of_many_rows_are_steps_one_after_the_other():
    rows, slots = 9001, 5000   # more rows than slots: some name the same one, some none
    slot = torch.randint(-1, slots + 1, (rows,), generator=torch.Generator().manual_seed(3)).to(DEV).int()
    slot[100:4300] = torch.where(torch.arange(4200, device=DEV) % 3 == 0, 7, slot[100:4300])   # one of them 1400 times
    x, w = torch.randn(rows, 12, device=DEV).half(), torch.randn(12, 3, device=DEV)
    pool = torch.randn(slots, 2, 12, device=DEV).half()
    mine = pool.clone()
    y = ops.history_conv_step(x, w, state=pool, slots=slot)
    part = [ops.history_conv_step(x[r:r + 700], w, state=mine, slots=slot[r:r + 700]) for r in range(0, rows, 700)]
    assert torch.equal(y, torch.cat(part)) and torch.equal(pool, mine)
    A, B = -torch.rand(12, 5, device=DEV), torch.randn(rows, 2, 5, device=DEV).half()
    pool = torch.randn(slots, 12, 5, device=DEV)
    mine = pool.clone()
    y = ops.history_scan_step(x, x, A, B, B, z=x, state=pool, slots=slot)
    part = [ops.history_scan_step(*(t[r:r + 700] for t in (x, x)), A, B[r:r + 700], B[r:r + 700], z=x[r:r + 700], state=mine, slots=slot[r:r + 700]) for r in range(0, rows, 700)]
    assert torch.equal(y, torch.cat(part)) and torch.equal(pool, mine)


def test_offsets_that_break_the_rules_touch_nothing_else():
    """Offsets out of order, negative or beyond the rows: meaningless numbers, in the outputs alone."""
    x = torch.randn(64, 8, device=DEV)
    w, B, A = torch.randn(8, 4, device=DEV), torch.randn(64, 1, 4, device=DEV), -torch.rand(8, 4, device=DEV)
    s, item = torch.randn(64, 32, device=DEV), torch.zeros(64, dtype=torch.int32, device=DEV)
    guard = torch.full((1 << 20,), 5.0, device=DEV)
    for off in ([0, 50, 20, 64, 10], [-9, 3, 1 << 40, 64, 64], [70, 80, 90, 1 << 62, -(1 << 62)]):
        o = offsets(off)
        i, h = torch.randn(4, 3, 8, device=DEV), torch.randn(4, 8, 4, device=DEV)
        ops.history_conv(x, w, seq_off=o, initial=i, want_final=True)
        ops.history_conv_backward(x, x, w, seq_off=o, initial=i, dfinal=i)
        _, _, kept = ops.history_scan(x, x, A, B, B, seq_off=o, initial=h, want_final=True, want_checkpoints=True)
        ops.history_scan_backward(x, x, x, A, B, B, seq_off=o, checkpoints=kept, initial=h, dfinal=h)
        ops.preference_loss(s, item, o, grad_weight=torch.ones(2, device=DEV))
        torch.cuda.synchronize()
    assert (guard == 5).all()


def test_refused_tensors():
    x, off = torch.zeros(4, 8, device=DEV), offsets([0, 4])
    w = torch.zeros(8, 4, device=DEV)
    bad = [
        (lambda: ops.history_conv(x.t(), w, seq_off=off), "contiguous"), (lambda: ops.history_conv(x, w.double(), seq_off=off), "float32"),
        (lambda: ops.history_conv(x, w[:7].contiguous(), seq_off=off), "shape"), (lambda: ops.history_conv(x, w, seq_off=off.int()), "int64"),
        (lambda: ops.history_conv(x, w, seq_off=off.cpu()), "int64"), (lambda: ops.history_conv(x.double(), w, seq_off=off), "float32, float16"),
        (lambda: ops.history_conv(x, w, seq_off=off, initial=torch.zeros(2, 3, 8, device=DEV)), "shape"),
        (lambda: ops.history_conv(x, w, seq_off=off, out=torch.zeros(4, 8, device=DEV).half()), "type"),
        (lambda: ops.history_conv(x[:1].expand(4, 8), w, seq_off=off), "overlap"),
        (lambda: ops.history_scan(x, x.half(), -w, x.view(4, 2, 4), x.view(4, 2, 4), seq_off=off), "type"),
        (lambda: ops.history_scan(x, x, -w, x.view(4, 2, 4), x.view(4, 1, 8), seq_off=off), "shape"),
        (lambda: ops.history_scan_backward(x, x, x, -w, x.view(4, 2, 4), x.view(4, 2, 4), seq_off=off, checkpoints=None), "checkpoints"),
        (lambda: ops.history_scan_step(x, x, -w, x.view(4, 2, 4), x.view(4, 2, 4), state=torch.zeros(3, 8, 5, device=DEV), slots=torch.zeros(4, dtype=torch.int32, device=DEV)), "shape"),
        (lambda: ops.policy_loss(x, torch.zeros(4, dtype=torch.int64, device=DEV), x[:, 0], x[:, 0]), "int32"),
        (lambda: ops.policy_loss(x, torch.zeros(4, dtype=torch.int32, device=DEV), x[:, 0], x[:, 0]), "contiguous"),
        (lambda: ops.policy_loss(x, torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(4, device=DEV), torch.zeros(4, device=DEV), out=x), "grad_weight"),
    ]
    for k, (f, words) in enumerate(bad):
        with pytest.raises(ValueError, match=words):
            f()
    with pytest.raises(RuntimeError, match="taps must be"):
        ops.history_conv(x, torch.zeros(8, 9, device=DEV), seq_off=off)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.history_conv(x, w, seq_off=off, out=x)


# ------------------------------------------------------------------ together
def test_from_an_engine_s_corpus_to_the_gradient_of_its_item_table():
    """Clicks of an engine's corpus, its item table's rows, convolution, gated scan, scores against the same table, preferences
    between the histories' next items - loss and every gradient against 64-bit autograd on the CPU."""
    from recommendation_amd.sharded import item_table_tensors
    gen = torch.Generator().manual_seed(11)
    U_, I, K = 6, 50, 16
    lengths = [3, 9, 1, 17, 5, 7]
    seq_off = np.cumsum([0] + lengths).astype(np.int64)
    clicks = torch.randint(0, I, (int(seq_off[-1]),), generator=gen)
    test = torch.randint(0, I, (U_,), generator=gen).numpy().astype(np.int32)
    e = ra.Engine("BPRMF", I, seq_off, clicks.numpy().astype(np.int32), test, test, K=K)
    e.init_params(3)
    e.sync()
    tab = item_table_tensors(e, torch.device(DEV))[1].view(I, K)
    off = torch.tensor(seq_off, device=DEV)
    w, b = torch.randn(K, 4, generator=gen) * 0.5, torch.randn(K, generator=gen) * 0.1
    A, D, bias = -torch.rand(K, 8, generator=gen) - 0.1, torch.randn(K, generator=gen), torch.randn(K, generator=gen) - 2
    proj = torch.randn(K, 2 * K + 16, generator=gen) * 0.3
    target = torch.randint(0, I, (int(seq_off[-1]),), generator=gen)
    gw = torch.tensor([0.3, 0.5, 0.2])
    d = lambda t: t.to(DEV)  # noqa: E731
    # forward
    idx = d(clicks)
    x = tab[idx]
    c, _ = ops.history_conv(x, d(w), d(b), seq_off=off)
    mixed = c @ d(proj)
    delta, z, B, C_ = mixed[:, :K], mixed[:, K:2 * K], mixed[:, 2 * K:2 * K + 8].unflatten(1, (1, 8)), mixed[:, 2 * K + 8:].unflatten(1, (1, 8))
    y, _, kept = ops.history_scan(c, delta, d(A), B, C_, d(D), z, d(bias), seq_off=off, want_checkpoints=True)
    scores = y @ tab.t()
    r = ops.preference_loss(scores, d(target).int(), off, beta=0.5, grad_weight=d(gw))
    # and back
    dy = r.dscores @ tab
    g = ops.history_scan_backward(dy, c, delta, d(A), B, C_, d(D), z, d(bias), seq_off=off, checkpoints=kept)
    dmixed = torch.cat([g.ddelta, g.dz, g.dB.flatten(1), g.dC.flatten(1)], 1)
    gc = ops.history_conv_backward(g.du + dmixed @ d(proj).t(), x, d(w), d(b), seq_off=off)
    dtab = torch.zeros_like(tab).index_add_(0, idx, gc.dx) + r.dscores.t() @ y
    # the same in 64 bits
    leaves = [v.double().requires_grad_() for v in (tab.cpu(), w, b, A, D, bias, proj)]
    T, w6, b6, A6, D6, bias6, proj6 = leaves
    x6 = T[clicks]
    ys = []
    for s in range(U_):
        xs = x6[seq_off[s]:seq_off[s + 1]]
        line = torch.cat([torch.zeros(3, K, dtype=torch.float64), xs])
        cs = torch.nn.functional.silu(sum(line[j:j + len(xs)] * w6[:, j] for j in range(4)) + b6)
        m = cs @ proj6
        h = torch.zeros(K, 8, dtype=torch.float64)
        for t in range(len(xs)):
            dt = torch.nn.functional.softplus(m[t, :K] + bias6)
            h = torch.exp(dt[:, None] * A6) * h + (dt * cs[t])[:, None] * m[t, 2 * K:2 * K + 8]
            ys.append(((h * m[t, 2 * K + 8:]).sum(1) + D6 * cs[t]) * torch.nn.functional.silu(m[t, K:2 * K]))
    lp = torch.log_softmax(torch.stack(ys) @ T.t(), 1).gather(1, target[:, None])[:, 0]
    sums = torch.stack([lp[seq_off[s]:seq_off[s + 1]].sum() for s in range(U_)])
    loss6 = -torch.nn.functional.logsigmoid(0.5 * (sums[0::2] - sums[1::2]))
    grads = torch.autograd.grad((loss6 * gw.double()).sum(), leaves)
    # f32 throughout: a few hundred roundings of 2^-24 on terms of mixed sign
    near = lambda a, q: float((a.double().cpu() - q).norm()) <= 2e-5 * float(q.norm())  # noqa: E731
    assert near(r.loss, loss6.detach())
    dproj = c.t() @ dmixed
    for name, got, want in zip(("table", "weight", "bias", "A", "D", "delta_bias", "projection"), (dtab, gc.dweight, gc.dbias, g.dA, g.dD, g.ddelta_bias, dproj), grads):
        assert near(got, want), name
    e.close()
