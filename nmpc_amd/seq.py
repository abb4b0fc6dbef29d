"""Operators of sequence models on the GPU: causal convolution, selective LPV scan, gated feed-forward projections.

Each whole-sequence operator comes in three forms: `op(...)` (differentiable through torch.autograd where an input asks for
it), and the pair `op_fwd(...)` -> outputs and what the gradient needs, `op_bwd(saved, gradients of the outputs)` -> the
gradients, which records no autograd graph and can be captured into a HIP graph.  `*_step` is the form for one sample of
every running sequence and moves its state on in place.

Samples are [batch, steps, channels] (channels contiguous; other layouts are copied) in float32, bfloat16 or float16;
states of the scan and all sums are fp32.  `lengths` [batch] (integers, on the GPU): steps from lengths[b] on are padding -
they are not read, and their outputs and gradients are zero."""
import ctypes

import torch

from . import _lib
from ._lib import NmpcError, lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {None: 0, "none": 0, "silu": 1, "gelu": 2, "tanh": 3, "sigmoid": 4}


def _need(ok, what, text, *args):
    if not ok:
        raise NmpcError("%s: %s" % (what, text % args if args else text))


def _p(t):
    return None if t is None else t.data_ptr()


def _call(dev, what, fn, *args):
    """fn(*args, current stream of dev) with dev current; an error becomes NmpcError."""
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    _lib.check(rc, what)


def _on_gpu(what, x, *others):
    """All tensors on x's GPU (checked last, after the shapes)."""
    _lib.require_gpu()
    _need(x.is_cuda, what, "tensors must be on the GPU, got %s", x.device)
    for t in others:
        _need(t is None or t.device == x.device, what, "tensors on different devices: %s and %s", x.device, getattr(t, "device", None))


def _samples(what, name, t, shape, dtype):
    """A sample tensor of this shape and type with contiguous channels (a copy only where they are not)."""
    _need(torch.is_tensor(t) and tuple(t.shape) == tuple(shape), what, "%s must be %s, got %s", name, list(shape),
          list(t.shape) if torch.is_tensor(t) else type(t).__name__)
    _need(t.dtype == dtype, what, "%s is %s, the samples are %s", name, t.dtype, dtype)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _param(what, name, t, shape):
    """A parameter as contiguous fp32."""
    _need(torch.is_tensor(t) and tuple(t.shape) == tuple(shape), what, "%s must be %s, got %s", name, list(shape),
          list(t.shape) if torch.is_tensor(t) else type(t).__name__)
    _need(t.is_floating_point(), what, "%s is %s, expected floating point", name, t.dtype)
    t = t.detach()
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.to(torch.float32).contiguous()


def _lengths(what, t, nb):
    if t is None:
        return None
    _need(torch.is_tensor(t) and t.dim() == 1 and t.shape[0] == nb, what, "lengths must be [%d]", nb)
    _need(not t.is_floating_point() and not t.is_complex() and t.dtype != torch.bool, what, "lengths are %s, expected integers", t.dtype)
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _records(what, *tensors):
    """Does this call have to be recorded by autograd?  Under graph capture it is refused: autograd's own bookkeeping of
    leaves that an eager graph still holds cannot be captured."""
    if not torch.is_grad_enabled() or not any(torch.is_tensor(t) and t.requires_grad for t in tensors):
        return False
    _need(not (torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()), what,
          "autograd is not recorded under graph capture; capture the pair %s_fwd / %s_bwd (or call under torch.no_grad())", what, what)
    return True


class Saved:
    """What a forward pass leaves for its gradient: `tensors` and plain values."""

    __slots__ = ("what", "tensors", "values")

    def __init__(self, what, tensors, values):
        self.what, self.tensors, self.values = what, tensors, values


def _saved(what, saved):
    _need(isinstance(saved, Saved) and saved.what == what, what + "_bwd", "expects what %s_fwd returned last", what)
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
def _conv_args(what, u, w, bias, act, start, lengths, steps=True):
    _need(torch.is_tensor(u) and u.dim() == (3 if steps else 2), what, "u must be %s", "[batch, steps, channels]" if steps else "[batch, channels]")
    _need(u.dtype in _DTYPES, what, "samples are %s, expected float32, bfloat16 or float16", u.dtype)
    _need(torch.is_tensor(w) and w.dim() == 2 and 1 <= w.shape[1] <= 8, what, "w must be [channels, taps] with 1..8 taps")
    _need(act in (None, "none", "silu"), what, "activation %r (None or 'silu')", act)
    nb, d, taps = u.shape[0], u.shape[-1], w.shape[1]
    _need(d >= 1, what, "no channels")
    w = _param(what, "w", w, (d, taps))
    bias = None if bias is None else _param(what, "bias", bias, (d,))
    if start is not None:
        _need(steps or not torch.is_tensor(start) or start.is_contiguous(), what, "window must be a contiguous tensor: it is moved on in place")
        start = _samples(what, "start" if steps else "window", start, (nb, taps - 1, d), u.dtype).contiguous()
    u = u if u.stride(-1) == 1 or d == 1 else u.contiguous()
    return u, w, bias, start, _lengths(what, lengths, nb)


def _conv_fwd(what, u, w, bias, act, start, lengths, want_window):
    u, w, bias, start, lengths = _conv_args(what, u, w, bias, act, start, lengths)
    _on_gpu(what, u, w, bias, start, lengths)
    nb, steps, d = u.shape
    y = torch.empty((nb, steps, d), dtype=u.dtype, device=u.device)
    window = torch.empty((nb, w.shape[1] - 1, d), dtype=u.dtype, device=u.device) if want_window else None
    _call(u.device, what, lib().nmpc_causal_conv, _DTYPES[u.dtype], nb, steps, d, w.shape[1], _p(u), u.stride(0), u.stride(1), _p(w),
          _p(bias), _ACTS[act], _p(start), _p(lengths), _p(y), _p(window))
    return y, window, (u, w, bias, start, lengths)


def causal_conv_fwd(u, w, bias=None, act=None, start=None, lengths=None):
    """causal_conv that keeps what its gradient needs: (y, window, saved)."""
    with torch.no_grad():
        y, window, tensors = _conv_fwd("causal_conv_fwd", u, w, bias, act, start, lengths, True)
    return y, window, Saved("causal_conv", tensors, (act,))


def causal_conv_bwd(saved, dy, dwindow=None):
    """Gradients of causal_conv_fwd's call: {"du", "dw", "dbias", "dstart"} (dw and dbias fp32; None for inputs that were
    not given).  dy [batch, steps, channels] and dwindow [batch, taps-1, channels] (None = zero): gradients of y and window."""
    what = "causal_conv_bwd"
    (u, w, bias, start, lengths), (act,) = _saved("causal_conv", saved)
    nb, steps, d = u.shape
    taps = w.shape[1]
    dy = torch.zeros_like(u) if dy is None else _samples(what, "dy", dy, u.shape, u.dtype)
    dwindow = None if dwindow is None else _samples(what, "dwindow", dwindow, (nb, taps - 1, d), u.dtype).contiguous()
    _on_gpu(what, u, dy, dwindow)
    du = torch.empty((nb, steps, d), dtype=u.dtype, device=u.device)
    dw = torch.empty_like(w)
    dbias = None if bias is None else torch.empty_like(bias)
    dstart = None if start is None else torch.empty_like(start)
    size = lib().nmpc_causal_conv_workspace_bytes(nb, steps, d, taps)
    work = torch.empty(size, dtype=torch.uint8, device=u.device)
    _call(u.device, what, lib().nmpc_causal_conv_bwd, _DTYPES[u.dtype], nb, steps, d, taps, _p(u), u.stride(0), u.stride(1), _p(w),
          _p(bias), _ACTS[act], _p(start), _p(lengths), _p(dy), dy.stride(0), dy.stride(1), _p(dwindow), _p(du), _p(dw), _p(dbias),
          _p(dstart), _p(work), size)
    return {"du": du, "dw": dw, "dbias": dbias, "dstart": dstart}


def causal_conv(u, w, bias=None, act=None, start=None, lengths=None, return_state=False):
    """y[b,t,c] = act(bias[c] + sum_j w[c,j] line[b,t+j,c]),  line = [start; u] along time.

    u [batch, steps, channels]; w [channels, taps], 1..8 taps; bias [channels]; act None or "silu"; start [batch, taps-1,
    channels]: the samples before the first, oldest first (None = zeros).  Returns y, with return_state also the window
    [batch, taps-1, channels] of the last samples: the start of what follows, and causal_conv_step's state."""
    what = "causal_conv"
    if not _records(what, u, w, bias, start):
        with torch.no_grad():
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
    _need(not _records(what, window, u, w, bias), what, "works in place and has no gradient; use causal_conv")
    u, w, bias, window, _ = _conv_args(what, u, w, bias, act, window, None, steps=False)
    _need(window is not None, what, "needs a window")
    _on_gpu(what, u, w, bias, window)
    y = torch.empty(u.shape, dtype=u.dtype, device=u.device)
    _call(u.device, what, lib().nmpc_causal_conv_step, _DTYPES[u.dtype], u.shape[0], u.shape[1], w.shape[1], _p(window), _p(u),
          u.stride(0), _p(w), _p(bias), _ACTS[act], _p(y))
    return y


# ---- selective LPV scan ---------------------------------------------------------------------------------------------
def _scan_inputs(what, u, dt, A, B, C, D, z, dt_bias, steps=True):
    lead = 2 if steps else 1
    _need(torch.is_tensor(u) and u.dim() == lead + 1, what, "u must be %s", "[batch, steps, channels]" if steps else "[batch, channels]")
    _need(u.dtype in _DTYPES, what, "samples are %s, expected float32, bfloat16 or float16", u.dtype)
    d = u.shape[-1]
    _need(torch.is_tensor(A) and A.dim() == 2 and A.shape[0] == d and 1 <= A.shape[1] <= 64, what, "A must be [channels, states] with 1..64 states")
    n = A.shape[1]
    _need(torch.is_tensor(B) and B.dim() == lead + 2 and B.shape[:lead] == u.shape[:lead] and B.shape[-1] == n, what,
          "B must be %s", list(u.shape[:lead]) + ["groups", n])
    groups = B.shape[-2]
    _need(d >= 1 and groups >= 1 and d % groups == 0, what, "%d groups do not divide %d channels", groups, d)
    u = u if u.stride(-1) == 1 or d == 1 else u.contiguous()
    dt = _samples(what, "dt", dt, u.shape, u.dtype)
    z = None if z is None else _samples(what, "z", z, u.shape, u.dtype)

    def shared(name, t):
        t = _samples(what, name, t, tuple(u.shape[:lead]) + (groups, n), u.dtype)
        return t if groups == 1 or t.stride(-2) == n else t.contiguous()
    return (u, dt, _param(what, "A", A, (d, n)), shared("B", B), shared("C", C), None if D is None else _param(what, "D", D, (d,)), z,
            None if dt_bias is None else _param(what, "dt_bias", dt_bias, (d,)))


def _scan_struct(u, dt, A, B, C, D, z, dt_bias, softplus):
    """The argument struct with the inputs filled in; unused strides of single steps stay zero."""
    s = _lib.ScanArgs()
    s.struct_size, s.dtype, s.nb, s.D, s.softplus = ctypes.sizeof(_lib.ScanArgs), _DTYPES[u.dtype], u.shape[0], u.shape[-1], int(bool(softplus))
    s.N, s.G = A.shape[1], B.shape[-2]
    s.u, s.dt, s.A, s.B, s.C = u.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr()
    s.u_bs, s.dt_bs, s.B_bs, s.C_bs = u.stride(0), dt.stride(0), B.stride(0), C.stride(0)
    if D is not None:
        s.D_skip = D.data_ptr()
    if dt_bias is not None:
        s.dt_bias = dt_bias.data_ptr()
    if z is not None:
        s.z, s.z_bs = z.data_ptr(), z.stride(0)
    if u.dim() == 3:
        s.L, s.u_ts, s.dt_ts, s.B_ts, s.C_ts = u.shape[1], u.stride(1), dt.stride(1), B.stride(1), C.stride(1)
        if z is not None:
            s.z_ts = z.stride(1)
    else:
        s.L = 1
    return s


def _states(what, name, t, nb, A):
    if t is None:
        return None
    _need(torch.is_tensor(t) and tuple(t.shape) == (nb,) + tuple(A.shape), what, "%s must be %s", name, [nb] + list(A.shape))
    _need(t.dtype == torch.float32, what, "%s is %s, states are float32", name, t.dtype)
    return t.contiguous()


def _scan_work(s, dev, backward):
    size = lib().nmpc_lpv_scan_workspace_bytes(s.nb, s.L, s.D, s.N, s.G, backward)
    if not size:
        return None
    work = torch.empty(size, dtype=torch.uint8, device=dev)
    s.workspace, s.workspace_bytes = work.data_ptr(), size
    return work


def _scan_fwd(what, u, dt, A, B, C, D, z, dt_bias, softplus, start, lengths, want_state, want_saved):
    u, dt, A, B, C, D, z, dt_bias = tensors = _scan_inputs(what, u, dt, A, B, C, D, z, dt_bias)
    nb, steps, d = u.shape
    start, lengths = _states(what, "start", start, nb, A), _lengths(what, lengths, nb)
    _on_gpu(what, *tensors, start, lengths)
    s = _scan_struct(*tensors, softplus)
    s.start, s.lengths = _p(start), _p(lengths)
    y = torch.empty((nb, steps, d), dtype=u.dtype, device=u.device)
    last = torch.empty((nb, d, A.shape[1]), dtype=torch.float32, device=u.device) if want_state else None
    saved = None
    if want_saved:
        saved = torch.empty(lib().nmpc_lpv_scan_saved_bytes(nb, steps, d, A.shape[1]), dtype=torch.uint8, device=u.device)
    s.y, s.last, s.saved = y.data_ptr(), _p(last), _p(saved)
    work = _scan_work(s, u.device, 0)  # noqa: F841  (held until the launch)
    _call(u.device, what, lib().nmpc_lpv_scan, ctypes.addressof(s))
    return y, last, tensors + (start, lengths, saved)


def lpv_scan_fwd(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, start=None, lengths=None):
    """lpv_scan that keeps what its gradient needs: (y, last, saved).  Besides the inputs that is the state before every
    32nd step."""
    with torch.no_grad():
        y, last, tensors = _scan_fwd("lpv_scan_fwd", u, dt, A, B, C, D, z, dt_bias, softplus, start, lengths, True, True)
    return y, last, Saved("lpv_scan", tensors, (bool(softplus),))


def lpv_scan_bwd(saved, dy, dlast=None):
    """Gradients of lpv_scan_fwd's call: {"du", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dstart"}, those of samples
    in the samples' type, the others fp32; None for inputs that were not given.  dy [batch, steps, channels] and dlast
    [batch, channels, states] (None = zero): gradients of y and of the last state."""
    what = "lpv_scan_bwd"
    (u, dt, A, B, C, D, z, dt_bias, start, lengths, kept), (softplus,) = _saved("lpv_scan", saved)
    dy = torch.zeros_like(u) if dy is None else _samples(what, "dy", dy, u.shape, u.dtype)
    dlast = _states(what, "dlast", dlast, u.shape[0], A)
    _on_gpu(what, u, dy, dlast)
    s = _scan_struct(u, dt, A, B, C, D, z, dt_bias, softplus)
    s.lengths, s.saved, s.dy, s.dy_bs, s.dy_ts, s.dlast = _p(lengths), _p(kept), dy.data_ptr(), dy.stride(0), dy.stride(1), _p(dlast)
    like = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
    g = {"du": like(u), "ddt": like(dt), "dA": like(A), "dB": like(B), "dC": like(C), "dD": like(D), "dz": like(z),
         "ddt_bias": like(dt_bias), "dstart": like(start)}
    for name, t in g.items():
        setattr(s, name, _p(t))
    work = _scan_work(s, u.device, 1)  # noqa: F841  (held until the launch)
    _call(u.device, what, lib().nmpc_lpv_scan_bwd, ctypes.addressof(s))
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
        with torch.no_grad():
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
    _need(not _records(what, state, u, dt, A, B, C, D, z, dt_bias), what, "works in place and has no gradient; use lpv_scan")
    u, dt, A, B, C, D, z, dt_bias = tensors = _scan_inputs(what, u, dt, A, B, C, D, z, dt_bias, steps=False)
    _need(torch.is_tensor(state) and state.is_contiguous(), what, "state must be a contiguous tensor: it is moved on in place")
    state = _states(what, "state", state, u.shape[0], A)
    _on_gpu(what, *tensors, state)
    s = _scan_struct(*tensors, softplus)
    y = torch.empty(u.shape, dtype=u.dtype, device=u.device)
    s.y, s.last = y.data_ptr(), state.data_ptr()
    _call(u.device, what, lib().nmpc_lpv_scan_step, ctypes.addressof(s))
    return y


# ---- gated feed-forward projections ---------------------------------------------------------------------------------
def _ffn_args(what, x, w_gate, w_up, act):
    _need(torch.is_tensor(x) and x.dim() >= 1, what, "x must be [..., inputs]")
    _need(x.dtype in _DTYPES, what, "x is %s, expected float32, bfloat16 or float16", x.dtype)
    k = x.shape[-1]
    _need(torch.is_tensor(w_gate) and w_gate.dim() == 2 and w_gate.shape[1] == k and k >= 1 and w_gate.shape[0] >= 1, what,
          "w_gate must be [hidden, %d]", k)
    _need(act in ("silu", "gelu", "tanh", "sigmoid"), what, "activation %r (silu, gelu, tanh or sigmoid)", act)
    w_gate = _samples(what, "w_gate", w_gate, w_gate.shape, x.dtype)
    w_up = _samples(what, "w_up", w_up, w_gate.shape, x.dtype)
    if w_gate.stride(0) != w_up.stride(0):
        w_gate, w_up = w_gate.contiguous(), w_up.contiguous()
    rows = x.reshape(-1, k)
    return rows if rows.stride(-1) == 1 or k == 1 else rows.contiguous(), w_gate, w_up


def _ffn_work(x, w_gate, w_up, backward):
    bits = w_gate.data_ptr() | w_up.data_ptr() | x.data_ptr() | (x.stride(0) | w_gate.stride(0)) * x.element_size()
    size = lib().nmpc_gated_ffn_workspace_bytes(_DTYPES[x.dtype], x.shape[0], x.shape[1], w_gate.shape[0], backward, bits % 16 != 0)
    return (torch.empty(size, dtype=torch.uint8, device=x.device) if size else None), size


def _ffn_fwd(what, x, w_gate, w_up, act, want_saved):
    rows, w_gate, w_up = _ffn_args(what, x, w_gate, w_up, act)
    _on_gpu(what, rows, w_gate, w_up)
    (m, k), f = rows.shape, w_gate.shape[0]
    h = torch.empty(x.shape[:-1] + (f,), dtype=x.dtype, device=x.device)
    pre = torch.empty((2, m, f), dtype=torch.float32, device=x.device) if want_saved else None
    work, size = _ffn_work(rows, w_gate, w_up, 0)
    _call(x.device, what, lib().nmpc_gated_ffn, _DTYPES[x.dtype], m, k, f, _p(rows), rows.stride(0), _p(w_gate), w_gate.stride(0),
          _p(w_up), w_up.stride(0), _ACTS[act], _p(h), _p(pre), _p(work), size)
    return h, (rows, w_gate, w_up, pre)


def gated_ffn_fwd(x, w_gate, w_up, act="silu"):
    """gated_ffn that keeps what its gradient needs: (h, saved).  Besides the inputs that is both projections in fp32."""
    with torch.no_grad():
        h, tensors = _ffn_fwd("gated_ffn_fwd", x, w_gate, w_up, act, True)
    return h, Saved("gated_ffn", tensors, (act, tuple(x.shape)))


def gated_ffn_bwd(saved, dh):
    """Gradients (dx, dw_gate, dw_up) of gated_ffn_fwd's call, in the inputs' type; dh like h."""
    what = "gated_ffn_bwd"
    (rows, w_gate, w_up, pre), (act, shape) = _saved("gated_ffn", saved)
    (m, k), f = rows.shape, w_gate.shape[0]
    dh = _samples(what, "dh", dh, shape[:-1] + (f,), rows.dtype).reshape(m, f)
    _on_gpu(what, rows, dh)
    dx = torch.empty(shape, dtype=rows.dtype, device=rows.device)
    dwg, dwu = (torch.empty((f, k), dtype=rows.dtype, device=rows.device) for _ in range(2))
    work, size = _ffn_work(rows, w_gate, w_up, 1)
    _call(rows.device, what, lib().nmpc_gated_ffn_bwd, _DTYPES[rows.dtype], m, k, f, _p(rows), rows.stride(0), _p(w_gate),
          w_gate.stride(0), _p(w_up), w_up.stride(0), _ACTS[act], _p(pre), _p(dh), dh.stride(0), _p(dx), _p(dwg), _p(dwu), _p(work), size)
    return dx, dwg, dwu


def gated_ffn(x, w_gate, w_up, act="silu"):
    """h = act(x w_gate') * (x w_up'): both projections, the activation and the product in one kernel.

    x [..., inputs]; w_gate, w_up [hidden, inputs] of x's type; act "silu", "gelu" (erf), "tanh" or "sigmoid".  One row or a
    few (tokens of running sequences) and many rows (prompts, training) take kernels of their own."""
    what = "gated_ffn"
    if not _records(what, x, w_gate, w_up):
        with torch.no_grad():
            return _ffn_fwd(what, x, w_gate, w_up, act, False)[0]

    def fwd():
        h, saved = gated_ffn_fwd(x, w_gate, w_up, act)
        return (h,), saved

    def bwd(saved, dh):
        return (None, None, None) if dh is None else gated_ffn_bwd(saved, dh)
    return _Recorded.apply(fwd, bwd, x, w_gate, w_up)[0]
