"""The device operators' refusals (no GPU needed: an argument is looked at before the device is), and that the 64-bit
references the GPU tests compare with are right: their gradients against differences."""
import ctypes as C

import pytest
import torch

import recommendation_amd as ra
from recommendation_amd import ops
from tests import operators_ref as ref


# the structs of include/recsys_engine.h
class ConvDesc(C.Structure):
    _fields_ = [("device", C.c_int32), ("type", C.c_int32), ("rows", C.c_int64), ("n_seq", C.c_int32), ("channels", C.c_int32),
                ("taps", C.c_int32), ("silu", C.c_int32), ("zero_rest", C.c_int32)]


class ScanDesc(C.Structure):
    _fields_ = [("device", C.c_int32), ("type", C.c_int32), ("rows", C.c_int64), ("n_seq", C.c_int32), ("channels", C.c_int32),
                ("groups", C.c_int32), ("states", C.c_int32), ("softplus", C.c_int32), ("zero_rest", C.c_int32)]


class ScanInputs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("u", "delta", "z", "B", "C")] + \
               [(n + "_stride", C.c_int64) for n in ("u", "delta", "z", "B", "C")] + \
               [(n, C.c_void_p) for n in ("A", "D", "delta_bias", "initial")]


class ScanGradientPointers(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("du", "ddelta", "dz", "dB", "dC", "dA", "dD", "ddelta_bias", "dinitial")]


class LossDesc(C.Structure):
    _fields_ = [("device", C.c_int32), ("type", C.c_int32), ("rows", C.c_int64), ("n_items", C.c_int64), ("scale", C.c_float),
                ("zero_rest", C.c_int32)]


BUF = (C.c_char * (1 << 16))()
AT = (C.addressof(BUF) + 255) // 256 * 256     # host memory: a call that is not refused would be stopped by the missing device


def call(name, *args):
    rc = ops._fn(name)(*args)
    return rc, ra.lib().rec_last_error().decode()


def conv(entry="rec_history_conv", at=AT, out=AT + 8192, stride=8, ws=0, **kw):
    d = ConvDesc(**{**dict(device=0, type=0, rows=4, n_seq=1, channels=8, taps=4, silu=1, zero_rest=0), **kw})
    if entry == "rec_history_conv":
        return call(entry, C.byref(d), at, stride, AT, None, AT, None, out, stride, None, None)
    if entry == "rec_history_conv_step":
        return call(entry, C.byref(d), at, stride, AT, None, AT, AT + 16384, out, stride, None)
    return call(entry, C.byref(d), AT + 4096, stride, at, stride, AT, None, AT, None, None, out, stride, AT + 30000 // 256 * 256, None, None, AT + 40960, ws, None)


CONV_4X8 = ConvDesc(device=0, type=0, rows=4, n_seq=1, channels=8, taps=4, silu=1, zero_rest=0)


def scan(entry="rec_history_scan", in_kw={}, out=AT + 8192, y_stride=8, ws=1 << 20, final=None, **kw):
    d = ScanDesc(**{**dict(device=0, type=0, rows=4, n_seq=1, channels=8, groups=2, states=4, softplus=1, zero_rest=0), **kw})
    i = ScanInputs(**{**dict(u=AT, delta=AT + 256, z=None, B=AT + 512, C=AT + 1024, u_stride=8, delta_stride=8, z_stride=0, B_stride=8, C_stride=8, A=AT), **in_kw})
    if entry == "rec_history_scan":
        return call(entry, C.byref(d), C.byref(i), AT, out, y_stride, final, None, AT, ws, None)
    if entry == "rec_history_scan_step":
        return call(entry, C.byref(d), C.byref(i), AT, AT + 16384, out, y_stride, None)
    o = ScanGradientPointers(du=out, ddelta=out + 1024, dB=out + 2048, dC=out + 3200, dA=out + 4096, dinitial=final)
    return call(entry, C.byref(d), AT + 2048, y_stride, C.byref(i), AT, AT, None, C.byref(o), AT + 32768, ws, None)


def preference(out=None, weight=None, stride=16, ws=1 << 20, n_pairs=1, beta=0.1, smoothing=0.0, out_stride=16, **kw):
    d = LossDesc(**{**dict(device=0, type=0, rows=4, n_items=16, scale=1.0, zero_rest=0), **kw})
    return call("rec_preference_loss", C.byref(d), AT, stride, AT, AT, n_pairs, None, beta, smoothing, weight, AT, AT, AT, out, out_stride, AT + 16384, ws, None)


def policy(out=None, weight=None, clip=(0.2, 0.2), kl=0.0, refs=None, ws=1 << 20, stride=16, **kw):
    d = LossDesc(**{**dict(device=0, type=0, rows=4, n_items=16, scale=1.0, zero_rest=0), **kw})
    return call("rec_policy_loss", C.byref(d), AT, stride, AT, AT, AT, refs, *clip, kl, weight, AT, None, AT, out, 16, AT + 16384, ws, None)


REFUSED = [
    (lambda: conv(type=3), "unknown type"), (lambda: conv(type=-1), "unknown type"), (lambda: conv(rows=-1), "rows must be"), (lambda: conv(rows=1 << 31), "rows must be"),
    (lambda: conv(n_seq=-1), "n_seq"), (lambda: conv(channels=0), "channels must be"), (lambda: conv(taps=1), "taps must be"), (lambda: conv(taps=9), "taps must be"),
    (lambda: conv(stride=7), "stride"), (lambda: conv(stride=1 << 31), "stride"), (lambda: conv(at=None), "null argument"), (lambda: conv(out=None), "null argument"),
    (lambda: conv(out=AT + 64), "overlaps"), (lambda: conv(device=99), "no such HIP device"), (lambda: conv(device=-1), "no such HIP device"),
    (lambda: conv("rec_history_conv_backward"), "workspace is too small"), (lambda: conv("rec_history_conv_backward", out=AT + 64, ws=1 << 20), "overlaps"),
    (lambda: conv("rec_history_conv_step", rows=65537), "at most 65536"), (lambda: conv("rec_history_conv_step", out=AT + 16), "must not overlap"),
    (lambda: conv("rec_history_conv_step", out=AT + 16384), "must not overlap"),
    (lambda: scan(groups=3), "groups must divide"), (lambda: scan(groups=0), "groups must divide"), (lambda: scan(states=0), "states must be"), (lambda: scan(states=65), "states must be"),
    (lambda: scan(type=7), "unknown type"), (lambda: scan(rows=-2), "rows must be"), (lambda: scan(y_stride=4), "stride"), (lambda: scan(in_kw={"u_stride": 7}), "stride"),
    (lambda: scan(in_kw={"B_stride": 7}), "stride"), (lambda: scan(in_kw={"z": AT, "z_stride": 1}), "stride"), (lambda: scan(in_kw={"A": None}), "null argument"),
    (lambda: scan(in_kw={"C": None}), "null argument"), (lambda: scan(out=AT + 16), "overlaps an input"), (lambda: scan(rows=4000, out=AT + (1 << 22), ws=0), "workspace is too small"),
    (lambda: scan("rec_history_scan_backward", ws=0), "workspace is too small"), (lambda: scan("rec_history_scan_backward", out=AT + 256), "overlaps an input"),
    (lambda: scan("rec_history_scan_backward", rows=64, out=AT + 32768, in_kw=dict(u=AT, delta=AT, B=AT, C=AT)), "two outputs overlap"),
    (lambda: scan("rec_history_scan_step", rows=70000), "at most 65536"), (lambda: scan("rec_history_scan_step", out=AT + 16384), "must not overlap"), (lambda: scan(device=5000), "no such HIP device"),
    (lambda: preference(scale=0.0), "scale must be"), (lambda: preference(scale=float("nan")), "scale must be"), (lambda: preference(scale=float("inf")), "scale must be"),
    (lambda: preference(n_items=0), "n_items must be"), (lambda: preference(rows=1 << 22), "rows must be"), (lambda: preference(n_pairs=-1), "n_pairs"),
    (lambda: preference(stride=15), "row stride"), (lambda: preference(beta=float("inf")), "beta"), (lambda: preference(smoothing=1.5), "smoothing"),
    (lambda: preference(smoothing=float("nan")), "smoothing"), (lambda: preference(weight=AT), "come together"), (lambda: preference(out=AT + 8192), "come together"),
    (lambda: preference(out=AT, weight=AT, out_stride=15), "row stride"), (lambda: preference(out=AT + 64, weight=AT), "dscores overlaps"),
    (lambda: preference(out=AT, weight=AT, out_stride=17), "dscores overlaps"), (lambda: preference(ws=0, rows=65, n_items=16), "workspace is too small"), (lambda: preference(device=77), "no such HIP device"),
    (lambda: policy(clip=(-0.1, 0.2)), "clip_low"), (lambda: policy(clip=(0.2, float("nan"))), "clip_low"), (lambda: policy(clip=(1.1, 0.2)), "clip_low"),
    (lambda: policy(kl=0.1), "kl_coef"), (lambda: policy(kl=float("inf"), refs=AT), "kl_coef"), (lambda: policy(out=AT + 8192), "come together"), (lambda: policy(ws=1, rows=2, n_items=16384, stride=16384), "workspace is too small"),
    (lambda: policy(type=4), "unknown type"),
    # the state that a call starts from is not the one that it leaves
    (lambda: call("rec_history_conv", C.byref(CONV_4X8), AT, 8, AT, None, AT, AT + 32768, AT + 8192, 8, AT + 32768 + 64, None), "final_window overlaps"),
    (lambda: call("rec_history_conv_backward", C.byref(CONV_4X8), AT + 4096, 8, AT, 8, AT, None, AT, None, AT + 32768, AT + 8192, 8, AT, None, AT + 32768, AT + 40960, 1 << 20, None), "dinitial overlaps"),
    (lambda: scan(in_kw={"initial": AT + 32768}, final=AT + 32768 + 64), "final_state overlaps"),
    (lambda: scan("rec_history_scan_backward", in_kw={"initial": AT + 32768}, final=AT + 32768), "dinitial overlaps"),
]


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_refused_with_a_reason(case):
    f, words = REFUSED[case]
    rc, said = f()
    assert rc == -1 and words in said, (rc, said)


def test_packed_structs_are_those_of_the_header():
    for pack, cls, few in ((ops._conv_desc, ConvDesc, (1, 2, 3 << 33, 4, 5, 6, 7, 8)), (ops._scan_desc, ScanDesc, (1, 2, 3 << 33, 4, 5, 6, 7, 8, 9)),
                           (ops._scan_inputs, ScanInputs, tuple(k << 40 for k in range(1, 15))), (ops._scan_gradients, ScanGradientPointers, tuple(k << 40 for k in range(1, 10))),
                           (ops._loss_desc, LossDesc, (1, 2, 3 << 33, 4 << 33, 0.5, 6))):
        packed = pack(*few)
        assert len(packed) == C.sizeof(cls)
        back = cls.from_buffer_copy(packed)
        assert tuple(getattr(back, f[0]) for f in cls._fields_) == few


def test_workspace_queries_refuse_what_the_calls_refuse():
    bad = ScanDesc(device=0, type=0, rows=4, n_seq=1, channels=8, groups=3, states=4)
    assert ops._fn("rec_history_scan_workspace")(C.byref(bad)) == -1 and ops._fn("rec_history_scan_backward_workspace")(C.byref(bad)) == -1
    assert ops._fn("rec_history_conv_backward_workspace")(None) == -1 and ops._fn("rec_policy_loss_workspace")(None) == -1
    none = ScanDesc(device=0, type=0, rows=0, n_seq=0, channels=8, groups=1, states=4)
    assert ops._fn("rec_history_scan_workspace")(C.byref(none)) == 0


def test_tensors_that_are_not_on_a_gpu_are_refused():
    x, off = torch.zeros(4, 8), torch.tensor([0, 4])
    with pytest.raises(ValueError, match="on the GPU"):
        ops.history_conv(x, torch.zeros(8, 4), seq_off=off)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.policy_loss(x, torch.zeros(4, dtype=torch.int32), torch.zeros(4), torch.zeros(4))


# ---- the references: gradients against central differences
def differences(f, x, g, h=1e-6):
    """sum(df * direction) along random directions against the gradient."""
    for k in range(3):
        v = torch.randn(x.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(k))
        num = (f(x + h * v) - f(x - h * v)) / (2 * h)
        assert abs(num - (g * v).sum()) < 1e-6 * max(1.0, float((g * v).abs().sum())), (float(num), float((g * v).sum()))


def rnd(gen, *shape):
    return torch.randn(*shape, dtype=torch.float64, generator=gen)


def test_conv_reference_gradient_against_differences():
    gen = torch.Generator().manual_seed(1)
    off = [1, 1, 3, 10, 11]
    x, w, b, init = rnd(gen, 12, 3), rnd(gen, 3, 4), rnd(gen, 3), rnd(gen, 4, 3, 3)
    dy, dfin = rnd(gen, 12, 3), rnd(gen, 4, 3, 3)

    def total(x, w, b, init):
        y, fin = ref.conv(x, w, b, off, init, True)
        return (y[1:11] * dy[1:11]).sum() + (fin * dfin).sum()

    dx, dw, db, di = ref.conv_gradient(dy, x, w, b, off, init, True, dfin)
    differences(lambda v: total(v, w, b, init), x, dx)
    differences(lambda v: total(x, v, b, init), w, dw)
    differences(lambda v: total(x, w, v, init), b, db)
    differences(lambda v: total(x, w, b, v), init, di)


def test_scan_reference_gradient_against_differences():
    gen = torch.Generator().manual_seed(2)
    off = [0, 3, 3, 9]
    v = dict(u=rnd(gen, 10, 4), delta=rnd(gen, 10, 4) - 1, A=-rnd(gen, 4, 3).abs(), B=rnd(gen, 10, 2, 3), C=rnd(gen, 10, 2, 3), D=rnd(gen, 4), z=rnd(gen, 10, 4),
             bias=rnd(gen, 4), initial=rnd(gen, 3, 4, 3))
    dy, dfin = rnd(gen, 10, 4), rnd(gen, 3, 4, 3)

    def total(**k):
        y, fin = ref.scan(off=off, **{**v, **k})
        return (y[:9] * dy[:9]).sum() + (fin * dfin).sum()

    g = ref.scan_gradient(dy, dfinal=dfin, off=off, **v)
    for name in v:
        differences(lambda t: total(**{name: t}), v[name], g[name])


def test_loss_reference_gradients_against_differences():
    gen = torch.Generator().manual_seed(3)
    s, items = rnd(gen, 7, 5), torch.tensor([0, 4, 2, -1, 1, 3, 2])
    refs, w = rnd(gen, 7), rnd(gen, 2)
    off = [0, 2, 4, 4, 7]
    g = ref.preference(s, items, off, refs, 0.7, 0.2, 1.3, w)["dscores"]
    differences(lambda v: (ref.preference(v, items, off, refs, 0.7, 0.2, 1.3, w)["loss"] * w).sum(), s, g)
    old, adv, wr = torch.log_softmax(1.3 * s, 1).gather(1, items.clamp(min=0)[:, None])[:, 0] + 0.3 * rnd(gen, 7), rnd(gen, 7), rnd(gen, 7)
    g = ref.policy(s, items, old, adv, refs, 0.2, 0.3, 0.1, 1.3, wr)["dscores"]
    differences(lambda v: (ref.policy(v, items, old, adv, refs, 0.2, 0.3, 0.1, 1.3, wr)["loss"] * wr).sum(), s, g)


def test_columns_of_one_array_do_not_overlap():
    """An output that is another column slice of the array its input is a slice of passes the check; one column further it does not."""
    d = ConvDesc(device=99, type=0, rows=4, n_seq=1, channels=8, taps=4, silu=1, zero_rest=0)
    for shift, words in ((8 * 4, "no such HIP device"), (7 * 4, "overlaps"), (9 * 4, "overlaps"), (0, "overlaps")):
        rc, said = call("rec_history_conv", C.byref(d), AT, 16, AT + 4096, None, AT + 8192, None, AT + shift, 16, None, None)
        assert rc == -1 and words in said, (shift, said)
        rc, said = call("rec_history_conv", C.byref(d), AT + shift, 16, AT + 4096, None, AT + 8192, None, AT, 16, None, None)
        assert rc == -1 and words in said, (shift, said)
