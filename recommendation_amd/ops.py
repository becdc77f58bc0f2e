"""Device operators of sequence models on torch tensors: the entry points of include/recsys_engine.h whose names start with
rec_history_, rec_preference_ and rec_policy_ (same names, same meaning of the arguments).

    history_conv, history_conv_backward, history_conv_step     short causal convolution over packed click histories
    history_scan, history_scan_backward, history_scan_step     selective state space scan over them
    preference_loss, policy_loss                               losses over a catalogue's scores, with their gradient

Histories are packed as in the engine's corpus: the rows of history s are seq_off[s] .. seq_off[s+1]-1 (int64, on the GPU).
Activations and scores are float32, float16 or bfloat16, all of a call of one type, their last dimension contiguous (rows may be
strided); parameters, states and per-row values are contiguous float32.  Every call enqueues on the current stream of its
tensors' GPU, waits for nothing and can be captured into a graph.  Outputs are allocated unless `out` is given; rows that belong
to no history are 0 in an allocated output and left as they were in `out`.  Gradients are explicit calls, as the engine's own
updates are: nothing is recorded for autograd.  Offsets, items and slots are read on the GPU and not checked on the host."""
import ctypes as C
import struct
from collections import namedtuple

import torch

from . import capi

_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
SCAN_CHECKPOINT = 16   # REC_SCAN_CHECKPOINT

ConvGradients = namedtuple("ConvGradients", "dx dweight dbias dinitial")
ScanGradients = namedtuple("ScanGradients", "du ddelta dA dB dC dD dz ddelta_bias dinitial")
PreferenceLoss = namedtuple("PreferenceLoss", "loss margin logp dscores")
PolicyLoss = namedtuple("PolicyLoss", "loss kl logp dscores")


# The structs of the header, packed from their fields (0q: up to the next multiple of 8 bytes).
_conv_desc = struct.Struct("@iiqiiiii0q").pack          # rec_conv_desc
_scan_desc = struct.Struct("@iiqiiiiii0q").pack         # rec_scan_desc
_scan_inputs = struct.Struct("@5P5q4P").pack            # rec_scan_inputs
_scan_gradients = struct.Struct("@9P").pack             # rec_scan_gradients
_loss_desc = struct.Struct("@iiqqfi").pack              # rec_loss_desc

_P, _L, _I, _F = C.c_void_p, C.c_int64, C.c_int32, C.c_float
_SIGNATURES = {
    "rec_history_conv": [_P, _P, _L, _P, _P, _P, _P, _P, _L, _P, _P],
    "rec_history_conv_backward": [_P, _P, _L, _P, _L, _P, _P, _P, _P, _P, _P, _L, _P, _P, _P, _P, _L, _P],
    "rec_history_conv_step": [_P, _P, _L, _P, _P, _P, _P, _P, _L, _P],
    "rec_history_scan": [_P, _P, _P, _P, _L, _P, _P, _P, _L, _P],
    "rec_history_scan_backward": [_P, _P, _L, _P, _P, _P, _P, _P, _P, _L, _P],
    "rec_history_scan_step": [_P, _P, _P, _P, _P, _L, _P],
    "rec_preference_loss": [_P, _P, _L, _P, _P, _I, _P, _F, _F, _P, _P, _P, _P, _P, _L, _P, _L, _P],
    "rec_policy_loss": [_P, _P, _L, _P, _P, _P, _P, _F, _F, _F, _P, _P, _P, _P, _P, _L, _P, _L, _P],
    "rec_history_conv_backward_workspace": [_P],
    "rec_history_scan_workspace": [_P],
    "rec_history_scan_backward_workspace": [_P],
    "rec_preference_loss_workspace": [_P, _I],
    "rec_policy_loss_workspace": [_P],
}
_functions = {}
_raw_stream = torch._C._cuda_getCurrentRawStream   # the handle of the current stream, without an object around it


def _fn(name):
    f = _functions.get(name)
    if f is None:
        f = getattr(capi.lib(), name)
        f.argtypes = _SIGNATURES[name]
        f.restype = _L if name.endswith("_workspace") else C.c_int
        _functions[name] = f
    return f


def _bad(what):
    raise ValueError("recsys operators: " + what)


def _desc(pack, *fields):
    try:
        return pack(*fields)
    except struct.error as e:
        _bad(f"a count or the scale is none that the call takes ({e})")


def _gpu_of(t, name):
    if not isinstance(t, torch.Tensor):
        _bad(f"{name} must be a tensor on the GPU")
    return t.get_device()


def _slots(state):
    if not isinstance(state, torch.Tensor) or state.dim() != 3:
        _bad("state must be a tensor of three dimensions, the slots first")
    return state.shape[0]


# A call of a few microseconds spends most of them here, so the checks take one pass over plain attributes; what is wrong is
# found out in the functions that say so.
def _first(t, name):
    """The array that sets a call's type, GPU and shape: (type, torch type, device, rows, width)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _bad(f"{name} must be a tensor on the GPU")
    dtype = t.dtype
    kind = _TYPE.get(dtype)
    if kind is None:
        _bad(f"{name} must be float32, float16 or bfloat16")
    shape = t.shape
    if len(shape) != 2:
        _bad(f"{name} must have the shape [rows, width]")
    return kind, dtype, t.get_device(), shape[0], shape[1]


def _rows(t, name, dtype, dev, rows, width):
    """A [rows, width] array of activations, its rows anywhere: (pointer, row stride)."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev and t.shape == (rows, width):
        s0, s1 = t.stride()
        if s1 == 1 or width <= 1:
            if rows <= 1 or width == 0:   # the stride of a single row means nothing to torch
                return t.data_ptr(), width
            if s0 >= width:
                return t.data_ptr(), s0
            _bad(f"the rows of {name} overlap")
        _bad(f"the last dimension of {name} must be contiguous")
    _bad_array(t, name, dtype, dev, (rows, width))


def _groups(t, name, dtype, dev, rows, groups, states):
    """A [rows, groups, states] array, the groups of a row contiguous: (pointer, row stride)."""
    width = groups * states
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev and t.shape == (rows, groups, states):
        s0, s1, s2 = t.stride()
        if (s2 == 1 or states <= 1) and (s1 == states or groups <= 1):
            if rows <= 1:
                return t.data_ptr(), width
            if s0 >= width:
                return t.data_ptr(), s0
            _bad(f"the rows of {name} overlap")
        _bad(f"the groups of a row of {name} must be contiguous")
    _bad_array(t, name, dtype, dev, (rows, groups, states))


def _whole(t, name, shape, dtype, dev):
    """A contiguous array of a known shape, or None: its pointer."""
    if t is None:
        return None
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    _bad_array(t, name, dtype, dev, shape)


def _bad_array(t, name, dtype, dev, shape):
    if not isinstance(t, torch.Tensor):
        _bad(f"{name} must be a tensor")
    if t.dtype is not dtype:
        _bad(f"{name} must have the type {dtype}, not {t.dtype}")
    if not t.is_cuda or t.get_device() != dev:
        _bad(f"{name} must be on the GPU of the other arguments")
    if tuple(t.shape) != tuple(shape):
        _bad(f"{name} must have the shape {tuple(shape)}, not {tuple(t.shape)}")
    _bad(f"{name} must be contiguous")


def _offsets(t, dev):
    if isinstance(t, torch.Tensor) and t.dtype is torch.int64 and t.get_device() == dev and t.dim() == 1 and t.is_contiguous() and len(t) >= 1:
        return t.data_ptr(), len(t) - 1
    _bad("seq_off must be a contiguous int64 vector of at least one entry on the GPU of the other arguments")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _space(size, like):
    """A workspace: of the stream's own pool, so it may go back there when the call returns."""
    if size <= 0:
        if size < 0:
            capi._check(-1)
        return None, None
    t = like.new_empty(size, dtype=torch.uint8)
    return t, t.data_ptr()


F32 = torch.float32


def _conv(x, weight, bias, n_seq, silu, zero_rest):
    kind, dtype, dev, rows, ch = _first(x, "x")
    px, sx = _rows(x, "x", dtype, dev, rows, ch)
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        _bad("weight must have the shape [channels, taps]")
    taps = weight.shape[1]
    d = _desc(_conv_desc, dev, kind, rows, n_seq, ch, taps, 1 if silu else 0, zero_rest)
    return d, px, sx, dtype, dev, rows, ch, taps, _whole(weight, "weight", (ch, taps), F32, dev), _whole(bias, "bias", (ch,), F32, dev)


def history_conv(x, weight, bias=None, *, seq_off, initial=None, silu=True, want_final=False, out=None):
    """(y, final window or None): x [rows, channels], weight [channels, taps], initial and final [histories, taps - 1, channels]."""
    off, n = _offsets(seq_off, _gpu_of(x, "x"))
    d, px, sx, dtype, dev, rows, ch, taps, w, b = _conv(x, weight, bias, n, silu, 1 if out is None else 0)
    window = (n, max(0, taps - 1), ch)
    i = _whole(initial, "initial", window, dtype, dev)
    y = torch.empty_like(x) if out is None else out
    py, sy = _rows(y, "out", dtype, dev, rows, ch)
    final = x.new_empty(window) if want_final else None
    capi._check(_fn("rec_history_conv")(d, px, sx, w, b, off, i, py, sy, _ptr(final), _raw_stream(dev)))
    return y, final


def history_conv_backward(dy, x, weight, bias=None, *, seq_off, initial=None, silu=True, dfinal=None, out=None):
    """ConvGradients for dy [rows, channels] and dfinal (the final window's gradient); dbias and dinitial are None without bias / initial."""
    off, n = _offsets(seq_off, _gpu_of(x, "x"))
    d, px, sx, dtype, dev, rows, ch, taps, w, b = _conv(x, weight, bias, n, silu, 1 if out is None else 0)
    pg, sg = _rows(dy, "dy", dtype, dev, rows, ch)
    window = (n, max(0, taps - 1), ch)
    i, df = _whole(initial, "initial", window, dtype, dev), _whole(dfinal, "dfinal", window, dtype, dev)
    dx = torch.empty_like(x) if out is None else out
    pd, sd = _rows(dx, "out", dtype, dev, rows, ch)
    dweight = torch.empty_like(weight)
    dbias = torch.empty_like(bias) if bias is not None else None
    dinitial = torch.empty_like(initial) if initial is not None else None
    size = _fn("rec_history_conv_backward_workspace")(d)
    ws, pw = _space(size, x)
    capi._check(_fn("rec_history_conv_backward")(d, pg, sg, px, sx, w, b, off, i, df, pd, sd, dweight.data_ptr(), _ptr(dbias), _ptr(dinitial), pw, size,
                                                 _raw_stream(dev)))
    return ConvGradients(dx, dweight, dbias, dinitial)


def history_conv_step(x, weight, bias=None, *, state, slots, silu=True, out=None):
    """y [rows, channels] of one click per row; state [slots, taps - 1, channels] (windows, of x's type) is updated in place at
    slots [rows] (int32)."""
    n = _slots(state)
    d, px, sx, dtype, dev, rows, ch, taps, w, b = _conv(x, weight, bias, n, silu, 0)
    ps = _whole(state, "state", (n, taps - 1, ch), dtype, dev)
    y = torch.empty_like(x) if out is None else out
    py, sy = _rows(y, "out", dtype, dev, rows, ch)
    capi._check(_fn("rec_history_conv_step")(d, px, sx, w, b, _whole(slots, "slots", (rows,), torch.int32, dev), ps, py, sy, _raw_stream(dev)))
    return y


def _scan(u, delta, A, B, Cm, D, z, delta_bias, n_seq, initial, softplus, zero_rest):
    kind, dtype, dev, rows, ch = _first(u, "u")
    pu, su = _rows(u, "u", dtype, dev, rows, ch)
    pd, sd = _rows(delta, "delta", dtype, dev, rows, ch)
    pz, sz = _rows(z, "z", dtype, dev, rows, ch) if z is not None else (0, 0)
    if not isinstance(A, torch.Tensor) or A.dim() != 2:
        _bad("A must have the shape [channels, states]")
    states = A.shape[1]
    if not isinstance(B, torch.Tensor) or B.dim() != 3:
        _bad("B must have the shape [rows, groups, states]")
    groups = B.shape[1]
    pB, sB = _groups(B, "B", dtype, dev, rows, groups, states)
    pC, sC = _groups(Cm, "C", dtype, dev, rows, groups, states)
    d = _desc(_scan_desc, dev, kind, rows, n_seq, ch, groups, states, 1 if softplus else 0, zero_rest)
    i = _scan_inputs(pu, pd, pz, pB, pC, su, sd, sz, sB, sC, _whole(A, "A", (ch, states), F32, dev), _whole(D, "D", (ch,), F32, dev) or 0,
                     _whole(delta_bias, "delta_bias", (ch,), F32, dev) or 0, _whole(initial, "initial", (n_seq, ch, states), F32, dev) or 0)
    return d, i, dtype, dev, rows, ch, states


def history_scan(u, delta, A, B, C_, D=None, z=None, delta_bias=None, *, seq_off, initial=None, softplus=True, want_final=False, want_checkpoints=False, out=None):
    """(y, final state or None, checkpoints or None): u, delta, z [rows, channels], A [channels, states], B, C [rows, groups, states],
    D, delta_bias [channels], initial and final [histories, channels, states] float32.  The gradient takes the checkpoints."""
    off, n = _offsets(seq_off, _gpu_of(u, "u"))
    d, i, dtype, dev, rows, ch, states = _scan(u, delta, A, B, C_, D, z, delta_bias, n, initial, softplus, 1 if out is None else 0)
    y = torch.empty_like(u) if out is None else out
    py, sy = _rows(y, "out", dtype, dev, rows, ch)
    final = u.new_empty((n, ch, states), dtype=F32) if want_final else None
    kept = u.new_empty((-(-rows // SCAN_CHECKPOINT), ch, states), dtype=F32) if want_checkpoints else None
    size = _fn("rec_history_scan_workspace")(d)
    ws, pw = _space(size, u)
    capi._check(_fn("rec_history_scan")(d, i, off, py, sy, _ptr(final), _ptr(kept), pw, size, _raw_stream(dev)))
    return y, final, kept


def history_scan_backward(dy, u, delta, A, B, C_, D=None, z=None, delta_bias=None, *, seq_off, checkpoints, initial=None, softplus=True, dfinal=None):
    """ScanGradients for dy [rows, channels] and dfinal (the final state's gradient); dD, dz, ddelta_bias and dinitial are None
    where the call has no D, z, delta_bias or initial."""
    off, n = _offsets(seq_off, _gpu_of(u, "u"))
    d, i, dtype, dev, rows, ch, states = _scan(u, delta, A, B, C_, D, z, delta_bias, n, initial, softplus, 1)
    pg, sg = _rows(dy, "dy", dtype, dev, rows, ch)
    if checkpoints is None:
        _bad("the gradient needs the forward call's checkpoints")
    kept = _whole(checkpoints, "checkpoints", (-(-rows // SCAN_CHECKPOINT), ch, states), F32, dev)
    df = _whole(dfinal, "dfinal", (n, ch, states), F32, dev)
    du, ddelta = u.new_empty((rows, ch)), u.new_empty((rows, ch))
    dz = u.new_empty((rows, ch)) if z is not None else None
    dB, dC = u.new_empty(B.shape), u.new_empty(B.shape)
    dA = torch.empty_like(A)
    dD = torch.empty_like(D) if D is not None else None
    dbias = torch.empty_like(delta_bias) if delta_bias is not None else None
    dinitial = torch.empty_like(initial) if initial is not None else None
    o = _scan_gradients(du.data_ptr(), ddelta.data_ptr(), _ptr(dz) or 0, dB.data_ptr(), dC.data_ptr(), dA.data_ptr(), _ptr(dD) or 0, _ptr(dbias) or 0, _ptr(dinitial) or 0)
    size = _fn("rec_history_scan_backward_workspace")(d)
    ws, pw = _space(size, u)
    capi._check(_fn("rec_history_scan_backward")(d, pg, sg, i, off, kept, df, o, pw, size, _raw_stream(dev)))
    return ScanGradients(du, ddelta, dA, dB, dC, dD, dz, dbias, dinitial)


def history_scan_step(u, delta, A, B, C_, D=None, z=None, delta_bias=None, *, state, slots, softplus=True, out=None):
    """y [rows, channels] of one click per row; state [slots, channels, states] float32 is updated in place at slots [rows] (int32)."""
    n = _slots(state)
    d, i, dtype, dev, rows, ch, states = _scan(u, delta, A, B, C_, D, z, delta_bias, n, None, softplus, 0)
    ps = _whole(state, "state", (n, ch, states), F32, dev)
    y = torch.empty_like(u) if out is None else out
    py, sy = _rows(y, "out", dtype, dev, rows, ch)
    capi._check(_fn("rec_history_scan_step")(d, i, _whole(slots, "slots", (rows,), torch.int32, dev), ps, py, sy, _raw_stream(dev)))
    return y


def _gradient(scores, grad_weight, n, out, dtype, dev, rows, width):
    """(pointer to the weights, dscores or None, its pointer and stride)"""
    if grad_weight is None:
        if out is not None:
            _bad("out is the gradient's: it needs grad_weight")
        return None, None, None, 0
    w = _whole(grad_weight, "grad_weight", (n,), F32, dev)
    ds = torch.empty_like(scores) if out is None else out
    return (w, ds, *_rows(ds, "out", dtype, dev, rows, width))


def preference_loss(scores, items, seq_off, ref_logp=None, *, beta=0.1, label_smoothing=0.0, scale=1.0, grad_weight=None, out=None):
    """PreferenceLoss(loss [pairs], margin [pairs], logp [rows], dscores): scores [rows, catalogue], items [rows] (int32), list 2p of
    seq_off [2 pairs + 1] preferred to list 2p + 1, ref_logp [rows].  With grad_weight [pairs], dscores is the gradient of
    sum(grad_weight * loss); out=scores writes it over the scores."""
    kind, dtype, dev, rows, width = _first(scores, "scores")
    off, n = _offsets(seq_off, dev)
    if n % 2:
        _bad("seq_off must have 2 pairs + 1 entries")
    pairs = n // 2
    p, s = _rows(scores, "scores", dtype, dev, rows, width)
    w, ds, pd, sd = _gradient(scores, grad_weight, pairs, out, dtype, dev, rows, width)
    d = _desc(_loss_desc, dev, kind, rows, width, scale, 1 if out is None else 0)
    i, r = _whole(items, "items", (rows,), torch.int32, dev), _whole(ref_logp, "ref_logp", (rows,), F32, dev)
    logp = scores.new_empty(rows, dtype=F32) if out is None else scores.new_zeros(rows, dtype=F32)   # rows of no list: 0
    loss, margin = scores.new_empty((2, pairs), dtype=F32).unbind()
    size = _fn("rec_preference_loss_workspace")(d, pairs)
    ws, pw = _space(size, scores)
    capi._check(_fn("rec_preference_loss")(d, p, s, i, off, pairs, r, beta, label_smoothing, w, loss.data_ptr(), margin.data_ptr(), logp.data_ptr(), pd, sd, pw, size,
                                           _raw_stream(dev)))
    return PreferenceLoss(loss, margin, logp, ds)


def policy_loss(scores, items, old_logp, advantage, ref_logp=None, *, clip_low=0.2, clip_high=0.2, kl_coef=0.0, scale=1.0, grad_weight=None, out=None):
    """PolicyLoss(loss [rows], kl [rows] or None, logp [rows], dscores): scores [rows, catalogue], items [rows] (int32; a row with an
    item outside the catalogue takes no part), old_logp, advantage and ref_logp [rows].  With grad_weight [rows], dscores is the
    gradient of sum(grad_weight * loss); out=scores writes it over the scores."""
    kind, dtype, dev, rows, width = _first(scores, "scores")
    p, s = _rows(scores, "scores", dtype, dev, rows, width)
    w, ds, pd, sd = _gradient(scores, grad_weight, rows, out, dtype, dev, rows, width)
    d = _desc(_loss_desc, dev, kind, rows, width, scale, 0)
    vec = (rows,)
    i = _whole(items, "items", vec, torch.int32, dev)
    old, adv, ref = _whole(old_logp, "old_logp", vec, F32, dev), _whole(advantage, "advantage", vec, F32, dev), _whole(ref_logp, "ref_logp", vec, F32, dev)
    if ref_logp is None:
        loss, logp = scores.new_empty((2, rows), dtype=F32).unbind()
        kl = None
    else:
        loss, logp, kl = scores.new_empty((3, rows), dtype=F32).unbind()
    size = _fn("rec_policy_loss_workspace")(d)
    ws, pw = _space(size, scores)
    capi._check(_fn("rec_policy_loss")(d, p, s, i, old, adv, ref, clip_low, clip_high, kl_coef, w, loss.data_ptr(), _ptr(kl), logp.data_ptr(), pd, sd, pw, size,
                                       _raw_stream(dev)))
    return PolicyLoss(loss, kl, logp, ds)
