"""Operators of sequence models on the GPU: causal convolution, selective LPV scan, gated feed-forward projections.

Each whole-sequence operator comes in three forms: `op(...)` (differentiable through torch.autograd where an input asks for
it), and the pair `op_fwd(...)` -> outputs and what the gradient needs, `op_bwd(saved, gradients of the outputs)` -> the
gradients, which records no autograd graph and can be captured into a HIP graph.  `*_step` is the form for one sample of
every running sequence and moves its state on in place.  Derivatives are first order and reverse mode: tensors that carry a
forward-mode tangent are refused.

Samples are [batch, steps, channels] (channels contiguous; other layouts are copied) in float32, bfloat16 or float16;
states of the scan and all sums are fp32.  `lengths` [batch] (integers, on the GPU): steps from lengths[b] on are padding -
they are not read, and their outputs and gradients are zero."""
import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import NmpcError, lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {None: 0, "none": 0, "silu": 1, "gelu": 2, "tanh": 3, "sigmoid": 4}
_INTEGERS = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)
_Tensor = torch.Tensor
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)

# The checks below run on every call of a kernel that takes a few microseconds: they test first and build a message only
# where they refuse.


def _fail(what, text, *args):
    raise NmpcError("%s: %s" % (what, text % args if args else text))


def _got(t):
    return list(t.shape) if isinstance(t, _Tensor) else type(t).__name__


def _p(t):
    return None if t is None else t.data_ptr()


def _call(i, what, fn, *args):
    """fn(*args, current stream of GPU i) with that GPU current; an error becomes NmpcError."""
    if i == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _raw_stream(i))
    if rc:
        _lib.check(rc, what)


def _on_gpu(what, x, *others):
    """The number of the GPU that holds x and all others (checked last, after the shapes)."""
    i = x.get_device()
    if i < 0 or not x.is_cuda:
        _lib.require_gpu()
        _fail(what, "tensors must be on the GPU, got %s", x.device)
    for t in others:
        if t is not None and t.get_device() != i:
            _fail(what, "tensors on different devices: %s and %s", x.device, t.device)
    return i


def _samples(what, name, t, shape, dtype):
    """A sample tensor of this shape and type with contiguous channels (a copy only where they are not)."""
    if not isinstance(t, _Tensor) or t.shape != shape:
        _fail(what, "%s must be %s, got %s", name, list(shape), _got(t))
    if t.dtype is not dtype:
        _fail(what, "%s is %s, the samples are %s", name, t.dtype, dtype)
    return t if t.stride(-1) == 1 or shape[-1] == 1 else t.detach().contiguous()


def _param(what, name, t, shape):
    """A parameter as contiguous fp32."""
    if not isinstance(t, _Tensor) or t.shape != shape:
        _fail(what, "%s must be %s, got %s", name, list(shape), _got(t))
    if t.dtype is torch.float32 and t.is_contiguous():
        return t
    if not t.is_floating_point():
        _fail(what, "%s is %s, expected floating point", name, t.dtype)
    return t.detach().to(torch.float32).contiguous()


def _lengths(what, t, nb):
    if t is None:
        return None
    if not isinstance(t, _Tensor) or t.shape != (nb,):
        _fail(what, "lengths must be [%d], got %s", nb, _got(t))
    if t.dtype not in _INTEGERS:
        _fail(what, "lengths are %s, expected integers", t.dtype)
    if t.dtype is torch.int32 and t.is_contiguous():
        return t
    if t.dtype is torch.int64:                                 # values past int32 would wrap around: those above any length are one
        t = t.clamp(-1, 2 ** 31 - 1)
    return t.to(torch.int32).contiguous()


def _no_tangents(what, *tensors):
    """Refuses tensors that carry a forward-mode tangent, which the kernels would drop: there is no form that computes one."""
    if getattr(forward_ad, "_current_level", 0) < 0:           # no forward-mode level is open: nothing to look for
        return
    for t in tensors:
        if isinstance(t, _Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            _fail(what, "has no forward-mode derivative, and an input carries a tangent")


def _records(what, *tensors):
    """Does this call have to be recorded by autograd?  Under graph capture it is refused: autograd's own bookkeeping of
    leaves that an eager graph still holds cannot be captured."""
    _no_tangents(what, *tensors)
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if isinstance(t, _Tensor) and t.requires_grad:
            if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                _fail(what, "autograd is not recorded under graph capture; capture the pair %s_fwd / %s_bwd (or call under torch.no_grad())", what, what)
            return True
    return False


class Saved:
    """What a forward pass leaves for its gradient: `tensors` and plain values."""

    __slots__ = ("what", "tensors", "values")

    def __init__(self, what, tensors, values):
        self.what, self.tensors, self.values = what, tensors, values


def _saved(what, saved):
    if not isinstance(saved, Saved) or saved.what != what:
        _fail(what + "_bwd", "expects what %s_fwd returned last", what)
    return saved.tensors, saved.values


class _Recorded(torch.autograd.Function):
    """An operator's pair as one node of an autograd graph.  fwd() -> (outputs tuple, Saved); bwd(saved, *gradients) ->
    gradients in the order of `inputs`."""

    @staticmethod
    def forward(ctx, fwd, bwd, *inputs):
        outs, saved = fwd()
        ctx.save_for_backward(*saved.tensors)
        ctx.what, ctx.values, ctx.bwd = saved.what, saved.values, bwd
        ctx.set_materialize_grads(False)
        return outs

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        return (None, None) + tuple(ctx.bwd(Saved(ctx.what, ctx.saved_tensors, ctx.values), *grads))


# ---- causal convolution ---------------------------------------------------------------------------------------------
def _conv_args(what, u, w, bias, act, steps):
    if not isinstance(u, _Tensor) or u.dim() != (3 if steps else 2):
        _fail(what, "u must be %s, got %s", "[batch, steps, channels]" if steps else "[batch, channels]", _got(u))
    if u.dtype not in _DTYPES:
        _fail(what, "samples are %s, expected float32, bfloat16 or float16", u.dtype)
    if not isinstance(w, _Tensor) or w.dim() != 2 or not 1 <= w.shape[1] <= 8:
        _fail(what, "w must be [channels, taps] with 1..8 taps, got %s", _got(w))
    if act not in (None, "none", "silu"):
        _fail(what, "activation %r (None or 'silu')", act)
    d = u.shape[-1]
    if d < 1:
        _fail(what, "no channels")
    w = _param(what, "w", w, (d, w.shape[1]))
    bias = None if bias is None else _param(what, "bias", bias, (d,))
    return u if u.stride(-1) == 1 or d == 1 else u.detach().contiguous(), w, bias


def _conv_fwd(what, u, w, bias, act, start, lengths, want_window):
    u, w, bias = _conv_args(what, u, w, bias, act, True)
    nb, steps, d = u.shape
    taps = w.shape[1]
    if start is not None:
        start = _samples(what, "start", start, (nb, taps - 1, d), u.dtype)
        start = start if start.is_contiguous() else start.detach().contiguous()
    lengths = _lengths(what, lengths, nb)
    i = _on_gpu(what, u, w, bias, start, lengths)
    y = torch.empty((nb, steps, d), dtype=u.dtype, device=u.device)
    window = torch.empty((nb, taps - 1, d), dtype=u.dtype, device=u.device) if want_window else None
    _call(i, what, lib().nmpc_causal_conv, _DTYPES[u.dtype], nb, steps, d, taps, u.data_ptr(), u.stride(0), u.stride(1), w.data_ptr(),
          _p(bias), _ACTS[act], _p(start), _p(lengths), y.data_ptr(), _p(window))
    return y, window, (u, w, bias, start, lengths)


def causal_conv_fwd(u, w, bias=None, act=None, start=None, lengths=None):
    """causal_conv that keeps what its gradient needs: (y, window, saved)."""
    _no_tangents("causal_conv_fwd", u, w, bias, start)
    y, window, tensors = _conv_fwd("causal_conv_fwd", u, w, bias, act, start, lengths, True)
    return y, window, Saved("causal_conv", tensors, (act,))


def causal_conv_bwd(saved, dy, dwindow=None):
    """Gradients of causal_conv_fwd's call: {"du", "dw", "dbias", "dstart"} (dw and dbias fp32; None for inputs that were
    not given).  dy [batch, steps, channels] and dwindow [batch, taps-1, channels] (None = zero): gradients of y and window."""
    what = "causal_conv_bwd"
    _no_tangents(what, dy, dwindow)
    (u, w, bias, start, lengths), (act,) = _saved("causal_conv", saved)
    nb, steps, d = u.shape
    taps = w.shape[1]
    dy = torch.zeros_like(u) if dy is None else _samples(what, "dy", dy, u.shape, u.dtype)
    dwindow = None if dwindow is None else _samples(what, "dwindow", dwindow, (nb, taps - 1, d), u.dtype).detach().contiguous()
    i = _on_gpu(what, u, dy, dwindow)
    du = torch.empty((nb, steps, d), dtype=u.dtype, device=u.device)
    dw = torch.empty_like(w)
    dbias = None if bias is None else torch.empty_like(bias)
    dstart = None if start is None else torch.empty_like(start)
    size = lib().nmpc_causal_conv_workspace_bytes(nb, steps, d, taps)
    work = torch.empty(size, dtype=torch.uint8, device=u.device)
    _call(i, what, lib().nmpc_causal_conv_bwd, _DTYPES[u.dtype], nb, steps, d, taps, u.data_ptr(), u.stride(0), u.stride(1), w.data_ptr(),
          _p(bias), _ACTS[act], _p(start), _p(lengths), dy.data_ptr(), dy.stride(0), dy.stride(1), _p(dwindow), du.data_ptr(),
          dw.data_ptr(), _p(dbias), _p(dstart), work.data_ptr(), size)
    return {"du": du, "dw": dw, "dbias": dbias, "dstart": dstart}


def causal_conv(u, w, bias=None, act=None, start=None, lengths=None, return_state=False):
    """y[b,t,c] = act(bias[c] + sum_j w[c,j] line[b,t+j,c]),  line = [start; u] along time.

    u [batch, steps, channels]; w [channels, taps], 1..8 taps; bias [channels]; act None or "silu"; start [batch, taps-1,
    channels]: the samples before the first, oldest first (None = zeros).  Returns y, with return_state also the window
    [batch, taps-1, channels] of the last samples: the start of what follows, and causal_conv_step's state."""
    what = "causal_conv"
    if not _records(what, u, w, bias, start):
        y, window, _ = _conv_fwd(what, u, w, bias, act, start, lengths, return_state)
        return (y, window) if return_state else y

    def fwd():
        y, window, saved = causal_conv_fwd(u, w, bias, act, start, lengths)
        return (y, window), saved

    def bwd(saved, dy, dwindow):
        g = causal_conv_bwd(saved, dy, dwindow)
        return (g["du"], g["dw"].to(w.dtype), None if bias is None else g["dbias"].to(bias.dtype), g["dstart"])
    y, window = _Recorded.apply(fwd, bwd, u, w, bias, start)
    return (y, window) if return_state else y


def causal_conv_step(window, u, w, bias=None, act=None):
    """One sample u [batch, channels] of every sequence: returns y [batch, channels] and moves window [batch, taps-1,
    channels] (contiguous) on by one row in place."""
    what = "causal_conv_step"
    if _records(what, window, u, w, bias):
        _fail(what, "works in place and has no gradient; use causal_conv")
    u, w, bias = _conv_args(what, u, w, bias, act, False)
    nb, d = u.shape
    taps = w.shape[1]
    if isinstance(window, _Tensor) and not window.is_contiguous():
        _fail(what, "window must be a contiguous tensor: it is moved on in place")
    _samples(what, "window", window, (nb, taps - 1, d), u.dtype)
    i = _on_gpu(what, u, w, bias, window)
    y = torch.empty((nb, d), dtype=u.dtype, device=u.device)
    _call(i, what, lib().nmpc_causal_conv_step, _DTYPES[u.dtype], nb, d, taps, window.data_ptr(), u.data_ptr(), u.stride(0),
          w.data_ptr(), _p(bias), _ACTS[act], y.data_ptr())
    return y


# ---- selective LPV scan ---------------------------------------------------------------------------------------------
def _scan_inputs(what, u, dt, A, B, C, D, z, dt_bias, lead):
    """The checked inputs; lead: leading dimensions of the samples (batch, steps)."""
    if not isinstance(u, _Tensor) or u.dim() != lead + 1:
        _fail(what, "u must be %s, got %s", "[batch, steps, channels]" if lead == 2 else "[batch, channels]", _got(u))
    dtype, shape = u.dtype, u.shape
    if dtype not in _DTYPES:
        _fail(what, "samples are %s, expected float32, bfloat16 or float16", dtype)
    d = shape[-1]
    if not isinstance(A, _Tensor) or A.dim() != 2 or A.shape[0] != d or not 1 <= A.shape[1] <= 64:
        _fail(what, "A must be [channels, states] with 1..64 states, got %s", _got(A))
    n = A.shape[1]
    if not isinstance(B, _Tensor) or B.dim() != lead + 2 or B.shape[:lead] != shape[:lead] or B.shape[-1] != n:
        _fail(what, "B must be %s, got %s", list(shape[:lead]) + ["groups", n], _got(B))
    groups = B.shape[-2]
    if d < 1 or groups < 1 or d % groups:
        _fail(what, "%d groups do not divide %d channels", groups, d)
    u = u if u.stride(-1) == 1 or d == 1 else u.detach().contiguous()
    dt = _samples(what, "dt", dt, shape, dtype)
    if z is not None:
        z = _samples(what, "z", z, shape, dtype)
    C = _samples(what, "C", C, B.shape, dtype)
    B = _samples(what, "B", B, B.shape, dtype)
    if groups > 1:
        B = B if B.stride(-2) == n else B.detach().contiguous()
        C = C if C.stride(-2) == n else C.detach().contiguous()
    return (u, dt, _param(what, "A", A, (d, n)), B, C, None if D is None else _param(what, "D", D, (d,)), z,
            None if dt_bias is None else _param(what, "dt_bias", dt_bias, (d,)))


def _scan_struct(u, dt, A, B, C, D, z, dt_bias, softplus):
    """The argument struct with the inputs filled in; unused strides of single steps stay zero."""
    s = _lib.ScanArgs(_SCAN_SIZE, _DTYPES[u.dtype], u.shape[0], 1, u.shape[-1], A.shape[1], B.shape[-2], 1 if softplus else 0,
                      u.data_ptr(), dt.data_ptr(), B.data_ptr(), C.data_ptr(), _p(z), u.stride(0), 0, dt.stride(0), 0, B.stride(0), 0,
                      C.stride(0), 0, 0 if z is None else z.stride(0), 0, A.data_ptr(), _p(D), _p(dt_bias))
    if u.dim() == 3:
        s.L, s.u_ts, s.dt_ts, s.B_ts, s.C_ts = u.shape[1], u.stride(1), dt.stride(1), B.stride(1), C.stride(1)
        if z is not None:
            s.z_ts = z.stride(1)
    return s


_SCAN_SIZE = ctypes.sizeof(_lib.ScanArgs)


def _states(what, name, t, nb, A):
    if t is None:
        return None
    if not isinstance(t, _Tensor) or t.shape != (nb,) + A.shape:
        _fail(what, "%s must be %s, got %s", name, [nb] + list(A.shape), _got(t))
    if t.dtype is not torch.float32:
        _fail(what, "%s is %s, states are float32", name, t.dtype)
    return t if t.is_contiguous() else t.detach().contiguous()


def _scan_work(s, dev, backward):
    size = lib().nmpc_lpv_scan_workspace_bytes(s.nb, s.L, s.D, s.N, s.G, backward)
    if not size:
        return None
    work = torch.empty(size, dtype=torch.uint8, device=dev)
    s.workspace, s.workspace_bytes = work.data_ptr(), size
    return work


def _scan_fwd(what, u, dt, A, B, C, D, z, dt_bias, softplus, start, lengths, want_state, want_saved):
    u, dt, A, B, C, D, z, dt_bias = tensors = _scan_inputs(what, u, dt, A, B, C, D, z, dt_bias, 2)
    nb, steps, d = u.shape
    start, lengths = _states(what, "start", start, nb, A), _lengths(what, lengths, nb)
    i = _on_gpu(what, *tensors, start, lengths)
    s = _scan_struct(*tensors, softplus)
    s.start, s.lengths = _p(start), _p(lengths)
    y = torch.empty((nb, steps, d), dtype=u.dtype, device=u.device)
    last = torch.empty((nb, d, A.shape[1]), dtype=torch.float32, device=u.device) if want_state else None
    saved = None
    if want_saved:
        saved = torch.empty(lib().nmpc_lpv_scan_saved_bytes(nb, steps, d, A.shape[1]), dtype=torch.uint8, device=u.device)
    s.y, s.last, s.saved = y.data_ptr(), _p(last), _p(saved)
    work = _scan_work(s, u.device, 0)  # noqa: F841  (held until the launch)
    _call(i, what, lib().nmpc_lpv_scan, ctypes.addressof(s))
    return y, last, tensors + (start, lengths, saved)


def lpv_scan_fwd(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, start=None, lengths=None):
    """lpv_scan that keeps what its gradient needs: (y, last, saved).  Besides the inputs that is the state before every
    16th step."""
    _no_tangents("lpv_scan_fwd", u, dt, A, B, C, D, z, dt_bias, start)
    y, last, tensors = _scan_fwd("lpv_scan_fwd", u, dt, A, B, C, D, z, dt_bias, softplus, start, lengths, True, True)
    return y, last, Saved("lpv_scan", tensors, (bool(softplus),))


def lpv_scan_bwd(saved, dy, dlast=None):
    """Gradients of lpv_scan_fwd's call: {"du", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dstart"}, those of samples
    in the samples' type, the others fp32; None for inputs that were not given.  dy [batch, steps, channels] and dlast
    [batch, channels, states] (None = zero): gradients of y and of the last state."""
    what = "lpv_scan_bwd"
    _no_tangents(what, dy, dlast)
    (u, dt, A, B, C, D, z, dt_bias, start, lengths, kept), (softplus,) = _saved("lpv_scan", saved)
    dy = torch.zeros_like(u) if dy is None else _samples(what, "dy", dy, u.shape, u.dtype)
    dlast = _states(what, "dlast", dlast, u.shape[0], A)
    i = _on_gpu(what, u, dy, dlast)
    s = _scan_struct(u, dt, A, B, C, D, z, dt_bias, softplus)
    s.lengths, s.saved, s.dy, s.dy_bs, s.dy_ts, s.dlast = _p(lengths), _p(kept), dy.data_ptr(), dy.stride(0), dy.stride(1), _p(dlast)
    like = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
    g = {"du": like(u), "ddt": like(dt), "dA": like(A), "dB": like(B), "dC": like(C), "dD": like(D), "dz": like(z),
         "ddt_bias": like(dt_bias), "dstart": like(start)}
    for name, t in g.items():
        setattr(s, name, _p(t))
    work = _scan_work(s, u.device, 1)  # noqa: F841  (held until the launch)
    _call(i, what, lib().nmpc_lpv_scan_bwd, ctypes.addressof(s))
    return g


def lpv_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, start=None, lengths=None, return_state=False):
    """Selective state-space scan, the diagonal LPV recurrence over a record:
        delta = softplus(dt + dt_bias)   (softplus=False: dt + dt_bias),
        x_t = exp(delta A) x_{t-1} + delta B_t u_t,    y_t = (C_t . x_t + D u_t) silu(z_t).

    u, dt, z [batch, steps, channels]; A [channels, states], 1..64 states; B, C [batch, steps, groups, states], shared by the
    channels / groups neighbouring channels of a group; D, dt_bias [channels]; start [batch, channels, states] fp32 (None =
    zeros).  Returns y, with return_state also the state after the last step, lpv_scan_step's state."""
    what = "lpv_scan"
    if not _records(what, u, dt, A, B, C, D, z, dt_bias, start):
        y, last, _ = _scan_fwd(what, u, dt, A, B, C, D, z, dt_bias, softplus, start, lengths, return_state, False)
        return (y, last) if return_state else y

    def fwd():
        y, last, saved = lpv_scan_fwd(u, dt, A, B, C, D, z, dt_bias, softplus, start, lengths)
        return (y, last), saved

    def bwd(saved, dy, dlast):
        g = lpv_scan_bwd(saved, dy, dlast)
        return (g["du"], g["ddt"], g["dA"].to(A.dtype), g["dB"], g["dC"], None if D is None else g["dD"].to(D.dtype), g["dz"],
                None if dt_bias is None else g["ddt_bias"].to(dt_bias.dtype), g["dstart"])
    y, last = _Recorded.apply(fwd, bwd, u, dt, A, B, C, D, z, dt_bias, start)
    return (y, last) if return_state else y


def lpv_scan_step(state, u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True):
    """One sample of every sequence: u, dt, z [batch, channels], B, C [batch, groups, states].  Returns y [batch, channels];
    state [batch, channels, states] (fp32, contiguous) moves on by one step in place."""
    what = "lpv_scan_step"
    if _records(what, state, u, dt, A, B, C, D, z, dt_bias):
        _fail(what, "works in place and has no gradient; use lpv_scan")
    u, dt, A, B, C, D, z, dt_bias = tensors = _scan_inputs(what, u, dt, A, B, C, D, z, dt_bias, 1)
    if not isinstance(state, _Tensor) or not state.is_contiguous():
        _fail(what, "state must be a contiguous tensor: it is moved on in place")
    _states(what, "state", state, u.shape[0], A)
    i = _on_gpu(what, *tensors, state)
    s = _scan_struct(*tensors, softplus)
    y = torch.empty(u.shape, dtype=u.dtype, device=u.device)
    s.y, s.last = y.data_ptr(), state.data_ptr()
    _call(i, what, lib().nmpc_lpv_scan_step, ctypes.addressof(s))
    return y


# ---- gated feed-forward projections ---------------------------------------------------------------------------------
def _ffn_args(what, x, w_gate, w_up, act):
    if not isinstance(x, _Tensor) or x.dim() < 1:
        _fail(what, "x must be [..., inputs], got %s", _got(x))
    dtype, k = x.dtype, x.shape[-1]
    if dtype not in _DTYPES:
        _fail(what, "x is %s, expected float32, bfloat16 or float16", dtype)
    if not isinstance(w_gate, _Tensor) or w_gate.dim() != 2 or w_gate.shape[1] != k or k < 1 or w_gate.shape[0] < 1:
        _fail(what, "w_gate must be [hidden, %d], got %s", k, _got(w_gate))
    if act not in ("silu", "gelu", "tanh", "sigmoid"):
        _fail(what, "activation %r (silu, gelu, tanh or sigmoid)", act)
    w_up = _samples(what, "w_up", w_up, w_gate.shape, dtype)
    w_gate = _samples(what, "w_gate", w_gate, w_gate.shape, dtype)
    if w_gate.stride(0) != w_up.stride(0):
        w_gate, w_up = w_gate.detach().contiguous(), w_up.detach().contiguous()
    rows = x if x.dim() == 2 else x.detach().reshape(-1, k)
    return rows if rows.stride(-1) == 1 or k == 1 else rows.detach().contiguous(), w_gate, w_up


def _ffn_work(x, w_gate, w_up, backward):
    bits = w_gate.data_ptr() | w_up.data_ptr() | x.data_ptr() | (x.stride(0) | w_gate.stride(0)) * x.element_size()
    size = lib().nmpc_gated_ffn_workspace_bytes(_DTYPES[x.dtype], x.shape[0], x.shape[1], w_gate.shape[0], backward, bits % 16 != 0)
    return (torch.empty(size, dtype=torch.uint8, device=x.device) if size else None), size


def _ffn_fwd(what, x, w_gate, w_up, act, want_saved):
    rows, w_gate, w_up = _ffn_args(what, x, w_gate, w_up, act)
    i = _on_gpu(what, rows, w_gate, w_up)
    (m, k), f = rows.shape, w_gate.shape[0]
    h = torch.empty(x.shape[:-1] + (f,), dtype=x.dtype, device=x.device)
    pre = torch.empty((2, m, f), dtype=torch.float32, device=x.device) if want_saved else None
    work, size = _ffn_work(rows, w_gate, w_up, 0)
    _call(i, what, lib().nmpc_gated_ffn, _DTYPES[x.dtype], m, k, f, rows.data_ptr(), rows.stride(0), w_gate.data_ptr(), w_gate.stride(0),
          w_up.data_ptr(), w_up.stride(0), _ACTS[act], h.data_ptr(), _p(pre), _p(work), size)
    return h, (rows, w_gate, w_up, pre)


def gated_ffn_fwd(x, w_gate, w_up, act="silu"):
    """gated_ffn that keeps what its gradient needs: (h, saved).  Besides the inputs that is both projections in fp32."""
    _no_tangents("gated_ffn_fwd", x, w_gate, w_up)
    h, tensors = _ffn_fwd("gated_ffn_fwd", x, w_gate, w_up, act, True)
    return h, Saved("gated_ffn", tensors, (act, tuple(x.shape)))


def gated_ffn_bwd(saved, dh):
    """Gradients (dx, dw_gate, dw_up) of gated_ffn_fwd's call, in the inputs' type; dh like h."""
    what = "gated_ffn_bwd"
    _no_tangents(what, dh)
    (rows, w_gate, w_up, pre), (act, shape) = _saved("gated_ffn", saved)
    (m, k), f = rows.shape, w_gate.shape[0]
    dh = _samples(what, "dh", dh, shape[:-1] + (f,), rows.dtype).detach().reshape(m, f)
    i = _on_gpu(what, rows, dh)
    dx = torch.empty(shape, dtype=rows.dtype, device=rows.device)
    dwg, dwu = (torch.empty((f, k), dtype=rows.dtype, device=rows.device) for _ in range(2))
    work, size = _ffn_work(rows, w_gate, w_up, 1)
    _call(i, what, lib().nmpc_gated_ffn_bwd, _DTYPES[rows.dtype], m, k, f, rows.data_ptr(), rows.stride(0), w_gate.data_ptr(),
          w_gate.stride(0), w_up.data_ptr(), w_up.stride(0), _ACTS[act], pre.data_ptr(), dh.data_ptr(), dh.stride(0), dx.data_ptr(),
          dwg.data_ptr(), dwu.data_ptr(), _p(work), size)
    return dx, dwg, dwu


def gated_ffn(x, w_gate, w_up, act="silu"):
    """h = act(x w_gate') * (x w_up'): both projections, the activation and the product in one kernel.

    x [..., inputs]; w_gate, w_up [hidden, inputs] of x's type; act "silu", "gelu" (erf), "tanh" or "sigmoid".  One row or a
    few (tokens of running sequences) and many rows (prompts, training) take kernels of their own."""
    what = "gated_ffn"
    if not _records(what, x, w_gate, w_up):
        return _ffn_fwd(what, x, w_gate, w_up, act, False)[0]

    def fwd():
        h, saved = gated_ffn_fwd(x, w_gate, w_up, act)
        return (h,), saved

    def bwd(saved, dh):
        return (None, None, None) if dh is None else gated_ffn_bwd(saved, dh)
    return _Recorded.apply(fwd, bwd, x, w_gate, w_up)[0]
