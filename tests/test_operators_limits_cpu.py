"""More refusals of the device operators (no GPU needed): counts at the ends of their ranges."""
import ctypes as C

import numpy as np
import pytest
import torch

from recommendation_amd import ops

from tests.test_operators_cpu import AT, LossDesc, ScanDesc, ScanGradientPointers, ScanInputs, call, conv, policy, preference, scan

FAR = 1 << 40
WIDE = dict(channels=1 << 20, groups=1, y_stride=1 << 20, ws=1 << 60, out=AT + FAR)   # as wide as a call may be
IN = dict(u_stride=1 << 20, delta_stride=1 << 20, B_stride=64, C_stride=64, B=AT + 2 * FAR, C=AT + 2 * FAR)


def wide_gradient(rows, states, device=0, dA=True):
    """rec_history_scan_backward of 2^20 channels, its arrays far from each other."""
    d = ScanDesc(device=device, type=0, rows=rows, n_seq=1, channels=1 << 20, groups=1, states=states, softplus=1, zero_rest=0)
    i = ScanInputs(u=AT, delta=AT, B=AT + FAR, C=AT + FAR, u_stride=1 << 20, delta_stride=1 << 20, B_stride=states, C_stride=states, A=AT)
    o = ScanGradientPointers(du=AT + 2 * FAR, ddelta=AT + 3 * FAR, dB=AT + 4 * FAR, dC=AT + 5 * FAR, dA=AT if dA else None)
    return call("rec_history_scan_backward", C.byref(d), AT + 6 * FAR, 1 << 20, C.byref(i), AT, AT, None, C.byref(o), AT, 1 << 60, None)


REFUSED = [
    # launches of 2^32 threads: the link of 2^26 states, the sums over 2^26 parameters and more
    (lambda: scan(rows=1024, states=64, in_kw=IN, **WIDE), "too many"), (lambda: scan(rows=1024, states=63, in_kw=IN, device=99, **WIDE), "no such HIP device"),
    (lambda: scan(rows=16, states=64, in_kw=IN, device=99, **WIDE), "no such HIP device"),
    (lambda: wide_gradient(16, 62), "too many"), (lambda: wide_gradient(16, 61, device=99), "no such HIP device"), (lambda: wide_gradient(16, 62, device=99, dA=False), "no such HIP device"),
    (lambda: wide_gradient(1024, 64, dA=False), "too many"),
    (lambda: conv(n_seq=(1 << 31) - 1), "n_seq must be"), (lambda: conv("rec_history_conv_backward", n_seq=(1 << 31) - 1), "n_seq must be"),
    (lambda: scan(n_seq=(1 << 31) - 1), "n_seq must be"), (lambda: scan("rec_history_scan_step", n_seq=(1 << 31) - 1), "n_seq must be"),
    # the exponent's factor, scale * log2(e), is an f32 as well
    (lambda: preference(scale=2.4e38), "scale must be"), (lambda: policy(scale=3.4e38), "scale must be"), (lambda: policy(scale=2.3e38, device=99), "no such HIP device"),
    (lambda: conv(n_seq=(1 << 31) - 2, device=99), "no such HIP device"), (lambda: scan(n_seq=(1 << 31) - 2, device=99), "no such HIP device"),
]


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_refused_with_a_reason(case):
    f, words = REFUSED[case]
    rc, said = f()
    assert rc == -1 and words in said, (rc, said)


def test_what_is_no_tensor_is_refused_as_one():
    """ValueError, as for a tensor of the wrong kind."""
    t, a, off = torch.zeros(4, 8), np.zeros((4, 8), np.float32), torch.tensor([0, 4])
    slots, B = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 1, 2)
    for bad in (None, a, 3.0):
        for f, words in [
            (lambda: ops.history_conv(bad, t, seq_off=off), "x must be"), (lambda: ops.history_conv_backward(t, bad, t, seq_off=off), "x must be"),
            (lambda: ops.history_scan(bad, t, t, B, B, seq_off=off), "u must be"), (lambda: ops.history_scan_backward(t, bad, t, t, B, B, seq_off=off, checkpoints=t), "u must be"),
            (lambda: ops.history_conv(t, t, seq_off=bad), "seq_off must be"), (lambda: ops.history_conv_step(bad, t, state=B, slots=slots), "x must be"),
            (lambda: ops.history_conv_step(t, t, state=bad, slots=slots), "state must be"), (lambda: ops.history_scan_step(t, t, t, B, B, state=bad, slots=slots), "state must be"),
            (lambda: ops.preference_loss(bad, slots, off), "scores must be"), (lambda: ops.policy_loss(bad, slots, t[0], t[0]), "scores must be"),
        ]:
            with pytest.raises(ValueError, match=words):
                f()


def test_numbers_that_no_field_holds_are_refused():
    with pytest.raises(ValueError, match="a count or the scale"):
        ops._desc(ops._conv_desc, 0, 0, 4, 1 << 31, 8, 4, 1, 0)
    with pytest.raises(ValueError, match="a count or the scale"):
        ops._desc(ops._loss_desc, 0, 0, 4, 16, "1", 0)


@pytest.mark.parametrize("rows,items,pairs,one", [(6, 2848, 1, True), (2, 65536, 1, False), (2, 4000, 1, True), (16, 8000, 1, False), (16, 2000, 1, True), (64, 500, 1, False), (64, 500, 32, True),
                                                  (24, 1000, 1, True), (24, 2000, 1, False), (64, 2000, 8, True), (65, 16, 30, False), (4, 33, 0, False)])
def test_long_rows_and_long_lists_are_not_one_block_s(rows, items, pairs, one):
    """A preference call of one launch needs no workspace."""
    d = LossDesc(device=0, type=0, rows=rows, n_items=items, scale=1.0)
    assert (ops._fn("rec_preference_loss_workspace")(C.byref(d), pairs) == 0) == one
