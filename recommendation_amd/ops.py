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
from collections import namedtuple

import torch

from . import capi

_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
SCAN_CHECKPOINT = 16   # REC_SCAN_CHECKPOINT

ConvGradients = namedtuple("ConvGradients", "dx dweight dbias dinitial")
ScanGradients = namedtuple("ScanGradients", "du ddelta dA dB dC dD dz ddelta_bias dinitial")
PreferenceLoss = namedtuple("PreferenceLoss", "loss margin logp dscores")
PolicyLoss = namedtuple("PolicyLoss", "loss kl logp dscores")


class _ConvDesc(C.Structure):
    _fields_ = [("device", C.c_int32), ("type", C.c_int32), ("rows", C.c_int64), ("n_seq", C.c_int32), ("channels", C.c_int32),
                ("taps", C.c_int32), ("silu", C.c_int32), ("zero_rest", C.c_int32)]


class _ScanDesc(C.Structure):
    _fields_ = [("device", C.c_int32), ("type", C.c_int32), ("rows", C.c_int64), ("n_seq", C.c_int32), ("channels", C.c_int32),
                ("groups", C.c_int32), ("states", C.c_int32), ("softplus", C.c_int32), ("zero_rest", C.c_int32)]


class _ScanInputs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("u", "delta", "z", "B", "C")] + \
               [(n + "_stride", C.c_int64) for n in ("u", "delta", "z", "B", "C")] + \
               [(n, C.c_void_p) for n in ("A", "D", "delta_bias", "initial")]


class _ScanGradientPointers(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("du", "ddelta", "dz", "dB", "dC", "dA", "dD", "ddelta_bias", "dinitial")]


class _LossDesc(C.Structure):
    _fields_ = [("device", C.c_int32), ("type", C.c_int32), ("rows", C.c_int64), ("n_items", C.c_int64), ("scale", C.c_float),
                ("zero_rest", C.c_int32)]


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


def _fn(name):
    f = _functions.get(name)
    if f is None:
        f = getattr(capi.lib(), name)
        f.argtypes = _SIGNATURES[name]
        f.restype = _L if name.endswith("_workspace") else C.c_int
        _functions[name] = f
    return f


def _need(ok, what):
    if not ok:
        raise ValueError("recsys operators: " + what)


def _rows(t, name, like=None, shape=None):
    """A [rows, width] array of activations: (pointer, row stride)."""
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a tensor on the GPU")
    _need(t.dim() == 2 if shape is None else tuple(t.shape) == tuple(shape), f"{name} must have the shape {tuple(shape) if shape is not None else '[rows, width]'}")
    _need(t.dtype in _TYPE, f"{name} must be float32, float16 or bfloat16")
    if like is not None:
        _need(t.dtype == like.dtype and t.device == like.device, f"{name} must have the type and the device of the other activations")
    rows, width = t.shape[0], t[0].numel() if t.dim() > 2 and t.shape[0] else (t.shape[1] if t.dim() == 2 else 0)
    s = t.stride()
    if t.dim() == 2:
        _need(t.shape[1] <= 1 or s[1] == 1, f"the last dimension of {name} must be contiguous")
    elif rows:
        _need(t[0].is_contiguous(), f"the groups of a row of {name} must be contiguous")
    # a single row's stride means nothing to torch; the rows of an array must not run into each other
    stride = width if rows <= 1 else s[0]
    _need(stride >= width, f"the rows of {name} overlap")
    return t.data_ptr(), stride


def _f32(t, name, shape, like, dtype=torch.float32):
    """A contiguous array of a known shape, or None: its pointer."""
    if t is None:
        return None
    _need(isinstance(t, torch.Tensor) and t.dtype == dtype and t.device == like.device, f"{name} must be {dtype} on the device of the activations")
    _need(tuple(t.shape) == tuple(shape), f"{name} must have the shape {tuple(shape)}")
    _need(t.is_contiguous(), f"{name} must be contiguous")
    return t.data_ptr()


def _offsets(t, like):
    _need(isinstance(t, torch.Tensor) and t.dtype == torch.int64 and t.device == like.device and t.dim() == 1 and t.shape[0] >= 1 and t.is_contiguous(),
          "seq_off must be a contiguous int64 vector on the device of the activations")
    return t.data_ptr(), t.shape[0] - 1


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _out(out, name, shape, like):
    """The output array, and whether its rows outside all histories are the call's to clear."""
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device), 1
    _rows(out, name, like, shape)
    return out, 0


def _workspace(size, like):
    if size < 0:
        capi._check(-1)
    return torch.empty(size, dtype=torch.uint8, device=like.device) if size else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _conv_desc(x, weight, n_seq, silu, zero_rest):
    _need(isinstance(weight, torch.Tensor) and weight.dim() == 2, "weight must have the shape [channels, taps]")
    return _ConvDesc(x.device.index, _TYPE[x.dtype], x.shape[0], n_seq, x.shape[1], weight.shape[1], 1 if silu else 0, zero_rest)


def history_conv(x, weight, bias=None, *, seq_off, initial=None, silu=True, want_final=False, out=None):
    """(y, final window or None): x [rows, channels], weight [channels, taps], initial and final [histories, taps - 1, channels]."""
    px, sx = _rows(x, "x")
    off, n = _offsets(seq_off, x)
    y, zero = _out(out, "out", x.shape, x)
    d = _conv_desc(x, weight, n, silu, zero)
    window = (n, max(0, d.taps - 1), d.channels)
    args = (_f32(weight, "weight", (d.channels, d.taps), x), _f32(bias, "bias", (d.channels,), x), off, _f32(initial, "initial", window, x, x.dtype))
    final = torch.empty(window, dtype=x.dtype, device=x.device) if want_final else None
    py, sy = _rows(y, "out")
    capi._check(_fn("rec_history_conv")(C.byref(d), px, sx, *args, py, sy, _ptr(final), _stream(x)))
    return y, final


def history_conv_backward(dy, x, weight, bias=None, *, seq_off, initial=None, silu=True, dfinal=None, out=None):
    """ConvGradients for dy [rows, channels] and dfinal (the final window's gradient); dbias and dinitial are None without bias / initial."""
    px, sx = _rows(x, "x")
    pg, sg = _rows(dy, "dy", x, x.shape)
    off, n = _offsets(seq_off, x)
    dx, zero = _out(out, "out", x.shape, x)
    d = _conv_desc(x, weight, n, silu, zero)
    window = (n, max(0, d.taps - 1), d.channels)
    args = (_f32(weight, "weight", (d.channels, d.taps), x), _f32(bias, "bias", (d.channels,), x), off, _f32(initial, "initial", window, x, x.dtype),
            _f32(dfinal, "dfinal", window, x, x.dtype))
    dweight = torch.empty_like(weight)
    dbias = torch.empty_like(bias) if bias is not None else None
    dinitial = torch.empty_like(initial) if initial is not None else None
    size = _fn("rec_history_conv_backward_workspace")(C.byref(d))
    ws = _workspace(size, x)
    pd, sd = _rows(dx, "out")
    capi._check(_fn("rec_history_conv_backward")(C.byref(d), pg, sg, px, sx, *args, pd, sd, _ptr(dweight), _ptr(dbias), _ptr(dinitial), _ptr(ws), size, _stream(x)))
    return ConvGradients(dx, dweight, dbias, dinitial)


def history_conv_step(x, weight, bias=None, *, state, slots, silu=True, out=None):
    """y [rows, channels] of one click per row; state [slots, taps - 1, channels] (windows, of x's type) is updated in place at
    slots [rows] (int32)."""
    px, sx = _rows(x, "x")
    y, _ = _out(out, "out", x.shape, x)
    _need(isinstance(state, torch.Tensor) and state.dim() == 3, "state must have the shape [slots, taps - 1, channels]")
    d = _conv_desc(x, weight, state.shape[0], silu, 0)
    w = _f32(weight, "weight", (d.channels, d.taps), x), _f32(bias, "bias", (d.channels,), x)
    ps = _f32(state, "state", (d.n_seq, d.taps - 1, d.channels), x, x.dtype)
    py, sy = _rows(y, "out")
    capi._check(_fn("rec_history_conv_step")(C.byref(d), px, sx, *w, _f32(slots, "slots", (d.rows,), x, torch.int32), ps, py, sy, _stream(x)))
    return y


def _scan(u, delta, A, B, Cm, D, z, delta_bias, n_seq, initial, softplus, zero_rest):
    pu, su = _rows(u, "u")
    pd, sd = _rows(delta, "delta", u, u.shape)
    pz, sz = _rows(z, "z", u, u.shape) if z is not None else (None, 0)
    _need(isinstance(A, torch.Tensor) and A.dim() == 2, "A must have the shape [channels, states]")
    rows, channels, states = u.shape[0], u.shape[1], A.shape[1]
    _need(isinstance(B, torch.Tensor) and B.dim() == 3 and B.shape[1] >= 1, "B must have the shape [rows, groups, states]")
    groups = B.shape[1]
    pB, sB = _rows(B, "B", u, (rows, groups, states))
    pC, sC = _rows(Cm, "C", u, (rows, groups, states))
    width = groups * states
    d = _ScanDesc(u.device.index, _TYPE[u.dtype], rows, n_seq, channels, groups, states, 1 if softplus else 0, zero_rest)
    i = _ScanInputs(pu, pd, pz, pB, pC, su, sd, sz, max(sB, width), max(sC, width), _f32(A, "A", (channels, states), u), _f32(D, "D", (channels,), u),
                    _f32(delta_bias, "delta_bias", (channels,), u), _f32(initial, "initial", (n_seq, channels, states), u))
    return d, i


def history_scan(u, delta, A, B, C_, D=None, z=None, delta_bias=None, *, seq_off, initial=None, softplus=True, want_final=False, want_checkpoints=False, out=None):
    """(y, final state or None, checkpoints or None): u, delta, z [rows, channels], A [channels, states], B, C [rows, groups, states],
    D, delta_bias [channels], initial and final [histories, channels, states] float32.  The gradient takes the checkpoints."""
    y, zero = _out(out, "out", u.shape, u)
    off, n = _offsets(seq_off, u)
    d, i = _scan(u, delta, A, B, C_, D, z, delta_bias, n, initial, softplus, zero)
    py, sy = _rows(y, "out")
    state = (d.channels, d.states)
    final = torch.empty((n,) + state, dtype=torch.float32, device=u.device) if want_final else None
    kept = torch.empty((-(-d.rows // SCAN_CHECKPOINT),) + state, dtype=torch.float32, device=u.device) if want_checkpoints else None
    size = _fn("rec_history_scan_workspace")(C.byref(d))
    ws = _workspace(size, u)
    capi._check(_fn("rec_history_scan")(C.byref(d), C.byref(i), off, py, sy, _ptr(final), _ptr(kept), _ptr(ws), size, _stream(u)))
    return y, final, kept


def history_scan_backward(dy, u, delta, A, B, C_, D=None, z=None, delta_bias=None, *, seq_off, checkpoints, initial=None, softplus=True, dfinal=None):
    """ScanGradients for dy [rows, channels] and dfinal (the final state's gradient); dD, dz, ddelta_bias and dinitial are None
    where the call has no D, z, delta_bias or initial."""
    off, n = _offsets(seq_off, u)
    d, i = _scan(u, delta, A, B, C_, D, z, delta_bias, n, initial, softplus, 1)
    pg, sg = _rows(dy, "dy", u, u.shape)
    state = (d.channels, d.states)
    kept = _f32(checkpoints, "checkpoints", (-(-d.rows // SCAN_CHECKPOINT),) + state, u)
    _need(kept is not None, "the gradient needs the forward call's checkpoints")
    df = _f32(dfinal, "dfinal", (n,) + state, u)

    def like(t, shape, dtype):
        return torch.empty(shape, dtype=dtype, device=u.device) if t is not None else None

    rows, group = tuple(u.shape), (d.rows, d.groups, d.states)
    du, ddelta, dz = like(u, rows, u.dtype), like(u, rows, u.dtype), like(z, rows, u.dtype)
    dB, dC = like(u, group, u.dtype), like(u, group, u.dtype)
    f = torch.float32
    dA, dD, dbias, dinitial = like(A, state, f), like(D, state[:1], f), like(delta_bias, state[:1], f), like(initial, (n,) + state, f)
    o = _ScanGradientPointers(_ptr(du), _ptr(ddelta), _ptr(dz), _ptr(dB), _ptr(dC), _ptr(dA), _ptr(dD), _ptr(dbias), _ptr(dinitial))
    size = _fn("rec_history_scan_backward_workspace")(C.byref(d))
    ws = _workspace(size, u)
    capi._check(_fn("rec_history_scan_backward")(C.byref(d), pg, sg, C.byref(i), off, kept, df, C.byref(o), _ptr(ws), size, _stream(u)))
    return ScanGradients(du, ddelta, dA, dB, dC, dD, dz, dbias, dinitial)


def history_scan_step(u, delta, A, B, C_, D=None, z=None, delta_bias=None, *, state, slots, softplus=True, out=None):
    """y [rows, channels] of one click per row; state [slots, channels, states] float32 is updated in place at slots [rows] (int32)."""
    y, _ = _out(out, "out", u.shape, u)
    _need(isinstance(state, torch.Tensor) and state.dim() == 3, "state must have the shape [slots, channels, states]")
    d, i = _scan(u, delta, A, B, C_, D, z, delta_bias, state.shape[0], None, softplus, 0)
    ps = _f32(state, "state", (d.n_seq, d.channels, d.states), u)
    py, sy = _rows(y, "out")
    capi._check(_fn("rec_history_scan_step")(C.byref(d), C.byref(i), _f32(slots, "slots", (d.rows,), u, torch.int32), ps, py, sy, _stream(u)))
    return y


def _gradient(scores, grad_weight, n, out):
    """(pointer to the weights, dscores or None, its pointer and stride, whether its rows outside all lists are to be cleared)"""
    _need(grad_weight is not None or out is None, "out is the gradient's: it needs grad_weight")
    if grad_weight is None:
        return None, None, None, 0, 1
    w = _f32(grad_weight, "grad_weight", (n,), scores)
    ds, zero = _out(out, "out", scores.shape, scores)
    return (w, ds, *_rows(ds, "out"), zero)


def preference_loss(scores, items, seq_off, ref_logp=None, *, beta=0.1, label_smoothing=0.0, scale=1.0, grad_weight=None, out=None):
    """PreferenceLoss(loss [pairs], margin [pairs], logp [rows], dscores): scores [rows, catalogue], items [rows] (int32), list 2p of
    seq_off [2 pairs + 1] preferred to list 2p + 1, ref_logp [rows].  With grad_weight [pairs], dscores is the gradient of
    sum(grad_weight * loss); out=scores writes it over the scores."""
    p, s = _rows(scores, "scores")
    off, n = _offsets(seq_off, scores)
    _need(n % 2 == 0, "seq_off must have 2 pairs + 1 entries")
    rows, pairs, dev = scores.shape[0], n // 2, scores.device
    w, ds, pd, sd, zero = _gradient(scores, grad_weight, pairs, out)
    d = _LossDesc(dev.index, _TYPE[scores.dtype], rows, scores.shape[1], scale, zero)
    args = _f32(items, "items", (rows,), scores, torch.int32), off, pairs, _f32(ref_logp, "ref_logp", (rows,), scores), beta, label_smoothing, w
    loss, margin, logp = (torch.empty(k, dtype=torch.float32, device=dev) for k in (pairs, pairs, rows))
    size = _fn("rec_preference_loss_workspace")(C.byref(d), pairs)
    ws = _workspace(size, scores)
    capi._check(_fn("rec_preference_loss")(C.byref(d), p, s, *args, _ptr(loss), _ptr(margin), _ptr(logp), pd, sd, _ptr(ws), size, _stream(scores)))
    return PreferenceLoss(loss, margin, logp, ds)


def policy_loss(scores, items, old_logp, advantage, ref_logp=None, *, clip_low=0.2, clip_high=0.2, kl_coef=0.0, scale=1.0, grad_weight=None, out=None):
    """PolicyLoss(loss [rows], kl [rows] or None, logp [rows], dscores): scores [rows, catalogue], items [rows] (int32; a row with an
    item outside the catalogue takes no part), old_logp, advantage and ref_logp [rows].  With grad_weight [rows], dscores is the
    gradient of sum(grad_weight * loss); out=scores writes it over the scores."""
    p, s = _rows(scores, "scores")
    rows, dev = scores.shape[0], scores.device
    w, ds, pd, sd, _ = _gradient(scores, grad_weight, rows, out)
    d = _LossDesc(dev.index, _TYPE[scores.dtype], rows, scores.shape[1], scale, 0)
    args = (_f32(items, "items", (rows,), scores, torch.int32), _f32(old_logp, "old_logp", (rows,), scores), _f32(advantage, "advantage", (rows,), scores),
            _f32(ref_logp, "ref_logp", (rows,), scores), clip_low, clip_high, kl_coef, w)
    loss, logp = (torch.empty(rows, dtype=torch.float32, device=dev) for _ in range(2))
    kl = torch.empty(rows, dtype=torch.float32, device=dev) if ref_logp is not None else None
    size = _fn("rec_policy_loss_workspace")(C.byref(d))
    ws = _workspace(size, scores)
    capi._check(_fn("rec_policy_loss")(C.byref(d), p, s, *args, _ptr(loss), _ptr(kl), _ptr(logp), pd, sd, _ptr(ws), size, _stream(scores)))
    return PolicyLoss(loss, kl, logp, ds)
