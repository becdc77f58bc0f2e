"""The device operators where a call is cut, linked or looped over: values that are not finite and states that grow across the chunks
of a long history, launches whose blocks go around, counts near their limits, and writes beside the outputs.  Needs an MI355X.

Tolerances as in test_gpu_operators: half a step of the value's type, plus a count of roundings times 2^-24 of the terms' size."""
import pytest
import torch

from recommendation_amd import capi, ops
from tests import operators_ref as ref
from tests import test_gpu_operators as base
from tests.test_gpu_operators import DEV, LEAST, TYPES, U, Source, close, offsets

pytestmark = pytest.mark.gpu


def close_on_gpu(got, want, slack, what):
    """`close` for arrays of a gigabyte, all finite."""
    allowed = (want.abs() + slack).mul_(torch.finfo(got.dtype).eps / 2).add_(slack).add_(LEAST[got.dtype])
    off = float(got.double().sub_(want).abs_().sub_(allowed).max())
    assert off <= 0, (what, off, float(allowed.max()))


def scan_arrays(rows, ch, N, histories, seed=1, decay=None):
    src = Source(seed, torch.float32)
    u, delta, dy = (src(rows, ch)[0] for _ in range(3))
    B, Cm = src(rows, 1, N)[0], src(rows, 1, N)[0]
    A = torch.full((ch, N), decay, device=DEV) if decay is not None else -torch.rand(ch, N, generator=src.gen).to(DEV) - 0.05
    return u, delta, dy, B, Cm, A, src(histories, ch, N)[0], src(histories, ch, N)[0]


def same(a, b):
    return int((a.cpu() != b).sum()) == 0


# ------------------------------------------------------------------ values that are not finite, over many chunks
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("states", [True, False])
def test_what_is_not_finite_reaches_the_end_of_a_long_history(value, states):
    """A decay of 8 forgets a finite state within a chunk - its factor is 0 in f32 - but 0 times what is not finite is not 0."""
    rows, ch, N, off = 7000, 16, 8, [0, 500, 6500, 7000]
    u, delta, dy, B, Cm, A, init, dfin = scan_arrays(rows, ch, N, 3, decay=-8.0)
    kw = dict(seq_off=offsets(off), initial=init if states else None)
    bad = u.clone()
    bad[600, 3] = value
    y, fin, _ = ops.history_scan(bad, delta, A, B, Cm, want_final=True, **kw)
    other = [d for d in range(ch) if d != 3]
    assert torch.isfinite(y[:, other]).all() and torch.isfinite(fin[:, other]).all()
    inside = torch.zeros(rows, dtype=torch.bool)
    inside[600:6500] = True
    assert same(~torch.isfinite(y[:, 3]), inside)
    assert not torch.isfinite(fin[1, 3]).any() and torch.isfinite(fin[[0, 2], 3]).all()
    # the gradient, from a row near the end to the history's beginning
    _, _, kept = ops.history_scan(u, delta, A, B, Cm, want_checkpoints=True, **kw)
    dy[6400, 3] = value
    g = ops.history_scan_backward(dy, u, delta, A, B, Cm, checkpoints=kept, dfinal=dfin if states else None, **kw)
    inside[:] = False
    inside[500:6401] = True
    for name in ("du", "ddelta"):
        t = getattr(g, name)
        assert torch.isfinite(t[:, other]).all(), name
        assert same(~torch.isfinite(t[:, 3]), inside), name
    assert same(~torch.isfinite(g.dB[:, 0]).all(1), inside)
    if states:
        assert not torch.isfinite(g.dinitial[1, 3]).any() and torch.isfinite(g.dinitial[[0, 2], 3]).all() and torch.isfinite(g.dinitial[:, other]).all()


@pytest.mark.parametrize("states", [True, False])
def test_a_decay_that_is_not_finite_stays_in_its_history(states):
    """Chunks of 16 rows; a delta of NaN makes the decay of a whole chunk NaN, the next history begins in the chunk behind it (for the
    gradient: ends in the one in front) and runs over fifty more."""
    rows, ch, N, off = 1000, 16, 8, [0, 100, 900, 1000]
    u, delta, dy, B, Cm, A, init, dfin = scan_arrays(rows, ch, N, 3)
    delta[80:96, 3] = delta[912:928, 3] = float("nan")
    kw = dict(seq_off=offsets(off), initial=init if states else None)
    y, fin, kept = ops.history_scan(u, delta, A, B, Cm, want_final=True, want_checkpoints=True, **kw)
    bad = torch.zeros(rows, dtype=torch.bool)
    bad[80:100] = bad[912:1000] = True
    assert same(torch.isnan(y[:, 3]), bad)
    assert torch.isnan(fin[[0, 2], 3]).all() and torch.isfinite(fin[1]).all()
    g = ops.history_scan_backward(dy, u, delta, A, B, Cm, checkpoints=kept, dfinal=dfin if states else None, **kw)
    for name in ("du", "ddelta"):
        assert torch.isfinite(getattr(g, name)[100:900]).all(), name
        assert torch.isnan(getattr(g, name)[900:928, 3]).all(), name
    assert torch.isfinite(g.dB[100:900]).all() and torch.isfinite(g.dC[100:900]).all()
    if states:
        assert torch.isfinite(g.dinitial[1]).all() and torch.isnan(g.dinitial[[0, 2], 3]).all()


# ------------------------------------------------------------------ states that grow
@pytest.mark.parametrize("late", [True, False])
def test_states_that_grow_over_many_chunks(late):
    """exp(delta A) > 1.  late: the factor over the history is e^450, beyond f32, but nothing is there to grow until 100 rows are left; else
    2^-120 grows by e^90, 2^129.8, to some hundreds.  Both are far from the end of f32 in every row."""
    rows, ch, N, off = 2000, 8, 4, [0, 1800, 2000]
    u, _, dy, B, Cm, _, init, dfin = scan_arrays(rows, ch, N, 2, seed=7)
    step = 0.25 if late else 0.05
    A = -torch.ones(ch, N, device=DEV)
    delta = torch.full((rows, ch), -step, device=DEV)
    if late:
        u[:1700], u[1900:] = 0, 0
        init.zero_(), dfin.zero_()
        dy[100:1800], dy[1850:] = 0, 0
    else:
        u.zero_(), dy.zero_()
        init, dfin = init.sign() * 2.0 ** -120, dfin.sign() * 2.0 ** -120
    six = dict(u=u.double(), delta=delta.double(), A=A.double(), B=B.double(), C=Cm.double(), D=None, z=None, bias=None, initial=init.double(), off=off, use_softplus=False)
    y6, fin6 = ref.scan(**six)
    ya, fina = ref.scan(**six, absolute=True)
    kw = dict(seq_off=offsets(off), initial=init, softplus=False)
    y, fin, kept = ops.history_scan(u, delta, A, B, Cm, want_final=True, want_checkpoints=True, **kw)
    # a step's roundings as everywhere, and an exponent of up to 650 (base 2) that some ten additions have made
    c = U * (1800 * (12 * step + 6) + 24 + 10 * 650)
    assert float(fin6.abs().max()) > 1 and float(fin6.abs().max()) < 2.0 ** 100
    close(y, y6.cpu(), (c * ya).cpu(), "y")
    close(fin, fin6.cpu(), (c * fina).cpu(), "final")
    g = ops.history_scan_backward(dy, u, delta, A, B, Cm, checkpoints=kept, dfinal=dfin, **kw)
    want = ref.scan_gradient(dy.double(), **six, dfinal=dfin.double())
    size = ref.scan_gradient(dy.double(), **six, dfinal=dfin.double(), absolute=True)
    for name, got in (("u", g.du), ("initial", g.dinitial)):
        close(got, want[name].cpu(), (2 * c * size[name]).cpu(), name)


# ------------------------------------------------------------------ launches that go around, and strips of the longest kind
@pytest.mark.parametrize("tn,rows,ch,W,longest", [
    ("f32", 60000, 33, 3, 4),          # 15 000 strips of 4 rows, 3750 blocks: two rounds of 1875
    ("bf16", 1100001, 128, 4, 128),    # 8594 strips of 128 rows, 2149 blocks: two rounds of 1075
    ("f16", 34000001, 1, 2, 128),      # one channel: 265 626 strips of 128 rows, 256 a block, one round
])
def test_conv_gradient_over_more_strips_than_blocks(tn, rows, ch, W, longest):
    src = Source(ch, TYPES[tn])
    n = max(4, rows // 100)
    gpu = torch.Generator(device=DEV).manual_seed(ch)
    off = torch.cat([torch.zeros(1, dtype=torch.int64), torch.randint(0, rows + 1, (n - 1,), generator=src.gen).sort().values, torch.tensor([rows])]).to(DEV)
    x, dy = (torch.randn(rows, ch, generator=gpu, device=DEV).to(TYPES[tn]) for _ in range(2))
    w, b = src.f32(ch, W, scale=0.5)[0], src.f32(ch)[0]
    t = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(off, t, right=True) - 1
    at, left = (t - off[seq])[:, None], (off[seq + 1] - 1 - t)[:, None]
    x6, dy6, w6 = x.double(), dy.double(), w.double()
    v, M = b.double().expand(rows, ch), b.double().abs().expand(rows, ch)
    for j in range(W):
        k = W - 1 - j
        term = torch.where(at >= k, torch.roll(x6, k, 0), 0.0) * w6[:, j]
        v, M = v + term, M + term.abs()
    g = torch.sigmoid(v)
    top = float(M.max())
    y, _ = ops.history_conv(x, w, b, seq_off=off)
    close_on_gpu(y, v * g, U * (1.1 * (W + 2) * M + (v * g).abs() * (M + 5)), "y")
    d, D = dy6 * g * (1 + v * (1 - g)), dy6.abs() * (1.1 + 0.5 * M)
    del v, M, g, y
    got = ops.history_conv_backward(dy, x, w, b, seq_off=off)
    c = U * (2 * W + 16 + top)
    want = sum(w6[:, W - 1 - k] * torch.where(left >= k, torch.roll(d, -k, 0), 0.0) for k in range(W))
    size = sum(w6[:, W - 1 - k].abs() * torch.where(left >= k, torch.roll(D, -k, 0), 0.0) for k in range(W))
    close_on_gpu(got.dx, want, c * size, "dx")
    # a thread adds up two strips one after the other at most, a block its 256 threads at most; blocks are added in 64 bits
    few = c + U * (2 * longest + 256)
    for j in range(W):
        k = W - 1 - j
        behind = torch.where(at >= k, torch.roll(x6, k, 0), 0.0)
        close_on_gpu(got.dweight[:, j], (d * behind).sum(0), few * (D * behind.abs()).sum(0), "dweight")
    close_on_gpu(got.dbias, d.sum(0), few * D.sum(0), "dbias")


def test_more_than_a_billion_histories():
    """Histories whose numbers are beyond 2^30: the middle of two of them is beyond an int before it is halved."""
    n = (1 << 30) + 21
    full, at = [0, 40, 120, 200], [3, (1 << 30) + 4, n - 1]
    off = torch.zeros(n + 1, dtype=torch.int64, device=DEV)
    off[at[0] + 1:] = 40
    off[at[1] + 1:] = 120
    off[n:] = 200
    few = offsets(full)
    x, dy, w, B = torch.randn(200, 8, device=DEV), torch.randn(200, 8, device=DEV), torch.randn(8, 4, device=DEV), torch.randn(200, 1, 4, device=DEV)
    A = -torch.rand(8, 4, device=DEV)
    out = []
    for o in (off, few):
        y, _ = ops.history_conv(x, w, seq_off=o)
        g = ops.history_conv_backward(dy, x, w, seq_off=o)
        ys, _, kept = ops.history_scan(x, x, A, B, B, seq_off=o, want_checkpoints=True)
        gs = ops.history_scan_backward(dy, x, x, A, B, B, seq_off=o, checkpoints=kept)
        out.append([y, g.dx, g.dweight, ys, kept, gs.du, gs.ddelta, gs.dA, gs.dB, gs.dC])
    assert all(torch.equal(a, b) for a, b in zip(*out))
    del off
    torch.cuda.empty_cache()


def test_final_states_of_a_million_histories():
    """More than 2^32 values of state, and 2^28 places in windows (two channels each); all but three histories are empty and hand on zeros, or the state they were handed."""
    n, ch, N = 1050000, 256, 16
    at = [5, 700000, n - 1]
    off = torch.zeros(n + 1, dtype=torch.int64, device=DEV)
    for s in at:
        off[s + 1:] += 3
    x, A, B = torch.randn(9, ch, device=DEV), -torch.rand(ch, N, device=DEV), torch.randn(9, 1, N, device=DEV)
    _, want, kept = ops.history_scan(x, x, A, B, B, seq_off=offsets([0, 3, 6, 9]), want_final=True, want_checkpoints=True)
    _, fin, _ = ops.history_scan(x, x, A, B, B, seq_off=off, want_final=True)
    assert fin.shape == (n, ch, N) and torch.equal(fin[at], want)
    fin[at] = 0
    assert int(torch.count_nonzero(fin.view(-1, 4096 * 25).abs().amax(1))) == 0
    fin.fill_(2.0)
    g = ops.history_scan_backward(x, x, x, A, B, B, seq_off=off, checkpoints=kept, initial=fin, dfinal=fin)
    assert g.dinitial.shape == fin.shape
    g.dinitial[at] = 2
    assert float(g.dinitial.min()) == 2 and float(g.dinitial.max()) == 2
    del fin, g
    w = torch.randn(ch, 4, device=DEV)
    _, want = ops.history_conv(x, w, seq_off=offsets([0, 3, 6, 9]), want_final=True)
    _, fin = ops.history_conv(x, w, seq_off=off, want_final=True)
    assert torch.equal(fin[at], want)
    fin[at] = 0
    assert float(fin.abs().max()) == 0
    fin.fill_(3.0)
    g = ops.history_conv_backward(x, x, w, seq_off=off, initial=fin, dfinal=fin)
    g.dinitial[at] = 3
    assert float(g.dinitial.min()) == 3 and float(g.dinitial.max()) == 3
    del fin, g
    torch.cuda.empty_cache()


def test_an_advantage_without_an_end():
    """0 times infinity is not a number, whichever of the two terms of the minimum it stands in."""
    inf = float("inf")
    s = torch.tensor([[0.0, -inf, 1.0]] * 4, device=DEV)
    item = torch.tensor([1, 1, 0, 0], dtype=torch.int32, device=DEV)       # the masked item has probability 0
    adv = torch.tensor([inf, -inf, inf, 1.0], device=DEV)
    zero, one = torch.zeros(4, device=DEV), torch.ones(4, device=DEV)
    r = ops.policy_loss(s, item, zero, adv, grad_weight=one)
    assert torch.isnan(r.loss[:2]).all() and float(r.loss[2]) == -inf and torch.isfinite(r.loss[3])
    assert torch.isnan(r.dscores[:2]).any(1).all() and torch.isfinite(r.dscores[3]).all()


# ------------------------------------------------------------------ writes beside the outputs
class Carved:
    """Outputs and workspace of a call, cut from one buffer of a known pattern with 64 KiB between them."""
    MARGIN, FILL = 1 << 16, 0xA5

    def __init__(self, size=1 << 24):
        self.buf = torch.full((size,), self.FILL, dtype=torch.uint8, device=DEV)
        self.mine = torch.zeros(size, dtype=torch.bool, device=DEV)
        self.at = 0

    def __call__(self, nbytes, rows=1, gap=0):
        """`rows` pieces of nbytes, `gap` bytes of margin behind each."""
        start = self.at + self.MARGIN
        for r in range(rows):
            self.mine[start + r * (nbytes + gap):start + r * (nbytes + gap) + nbytes] = True
        self.at = (start + rows * (nbytes + gap) + 255) // 256 * 256
        assert self.at + self.MARGIN <= self.buf.numel()
        return self.buf.data_ptr() + start

    def check(self):
        torch.cuda.synchronize()
        assert bool((self.buf[~self.mine] == self.FILL).all())


@pytest.mark.parametrize("off", [[0, 50, 20, 64, 10], [-9, 3, 1 << 40, 64, 64], [70, 80, 90, 1 << 60, -(1 << 60)], [400, 300, 200, 100, 0], [0, 130, 130, 350, 400]],
                         ids=["out of order", "beyond", "far", "falling", "in order"])
def test_offsets_that_break_the_rules_write_nothing_beside_the_outputs(off):
    rows, ch, W, N, items = 400, 20, 4, 8, 32
    o = offsets(off)
    x, dy, B = torch.randn(rows, ch, device=DEV), torch.randn(rows, ch, device=DEV), torch.randn(rows, 1, N, device=DEV)
    w, A = torch.randn(ch, W, device=DEV), -torch.rand(ch, N, device=DEV)
    i, df = torch.randn(4, W - 1, ch, device=DEV), torch.randn(4, W - 1, ch, device=DEV)
    h, dh = torch.randn(4, ch, N, device=DEV), torch.randn(4, ch, N, device=DEV)
    kept = torch.randn(-(-rows // 16), ch, N, device=DEV)
    s, item, gw = torch.randn(rows, items, device=DEV), torch.randint(0, items, (rows,), device=DEV).int(), torch.ones(2, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    call = lambda name, *a: capi._check(ops._fn(name)(*a))  # noqa: E731
    for zero_rest in (0, 1):
        c = Carved()
        d = ops._conv_desc(0, 0, rows, 4, ch, W, 1, zero_rest)
        call("rec_history_conv", d, p(x), ch, p(w), None, p(o), p(i), c(4 * ch, rows, 16), ch + 4, c(4 * i.numel()), stream)
        size = ops._fn("rec_history_conv_backward_workspace")(d)
        call("rec_history_conv_backward", d, p(dy), ch, p(x), ch, p(w), None, p(o), p(i), p(df), c(4 * ch, rows, 16), ch + 4, c(4 * w.numel()), c(4 * ch), c(4 * i.numel()),
             c(size), size, stream)
        d = ops._scan_desc(0, 0, rows, 4, ch, 1, N, 1, zero_rest)
        for state in (h, None):
            inputs = ops._scan_inputs(p(x), p(x), 0, p(B), p(B), ch, ch, 0, N, N, p(A), 0, 0, p(state) if state is not None else 0)
            size = ops._fn("rec_history_scan_workspace")(d)
            assert size > 0    # several chunks
            call("rec_history_scan", d, inputs, p(o), c(4 * ch, rows, 16), ch + 4, c(4 * h.numel()), c(4 * kept.numel()), c(size), size, stream)
            size = ops._fn("rec_history_scan_backward_workspace")(d)
            g = ops._scan_gradients(c(4 * rows * ch), c(4 * rows * ch), 0, c(4 * rows * N), c(4 * rows * N), c(4 * A.numel()), c(4 * ch), c(4 * ch), c(4 * h.numel()) if state is not None else 0)
            call("rec_history_scan_backward", d, p(dy), ch, inputs, p(o), p(kept), p(dh) if state is not None else None, g, c(size), size, stream)
        for n in (rows, 40):   # three launches, and one
            d = ops._loss_desc(0, 0, n, items, 1.0, zero_rest)
            size = ops._fn("rec_preference_loss_workspace")(d, 2)
            assert (size > 0) == (n > 64)
            call("rec_preference_loss", d, p(s), items, p(item), p(o), 2, None, 0.1, 0.0, p(gw), c(8), c(8), c(4 * n), c(4 * items, n, 12), items + 3, c(size) if size else None, size, stream)
            call("rec_preference_loss", d, p(s), items, p(item), p(o), 2, None, 0.1, 0.0, None, c(8), c(8), c(4 * n), None, 0, c(size) if size else None, size, stream)
        c.check()


# ------------------------------------------------------------------ preferences on both sides of the one launch's bounds
@pytest.mark.parametrize("case", [
    ("f32", 24, 999, [0, 20, 24], 1.0, 0.1, 0.1, True),                  # one launch, two rounds of a block's wavefronts
    ("bf16", 25, 999, [0, 20, 25], 1.0, 0.1, 0.1, True),                 # three launches
    ("f16", 3, 8000, [1, 2, 3], 1.0, 0.0, 0.1, False), ("f16", 3, 8001, [1, 2, 3], 1.0, 0.0, 0.1, False),
    ("bf16", 64, 700, [0, 1, 30, 31, 60, 60, 64], 1.0, 0.0, 0.1, True),  # one launch for rows that are nearly all one pair's
    ("f32", 64, 40, [64], 1.0, 0.0, 0.1, True),                          # no pairs
], ids=lambda c: f"{c[0]}-{c[1]}x{c[2]}")
@pytest.mark.parametrize("layout", ["packed", "strided", "in place"])
def test_preferences_in_one_launch_and_in_three(case, layout):
    base.test_preference_loss(case, layout)
