"""CPU tests of the sequence operators: the oracle's gradients against differences, and refusals (Python and C ABI), which
all happen before anything is launched."""
import ctypes

import pytest
import torch

import nmpc_amd
from nmpc_amd import _lib
from oracle import seq as oracle
from seq_util import normal, rng


def _double(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float64).requires_grad_()


def test_oracle_conv_gradient_against_differences():
    g = rng(1)
    u, w, b, s = _double(g, 2, 5, 3), _double(g, 3, 3), _double(g, 3), _double(g, 2, 2, 3)
    for n in (None, [5, 1], [0, 4]):
        assert torch.autograd.gradcheck(lambda *a: oracle.causal_conv(*a[:3], "silu", a[3], n), (u, w, b, s))


def test_conv_refusals():
    u, w = torch.zeros(2, 6, 8), torch.zeros(8, 4)
    bad = [
        (dict(u=torch.zeros(6, 8)), "batch, steps, channels"), (dict(u=u.double()), "float32, bfloat16"),
        (dict(w=torch.zeros(8, 9)), "1..8 taps"), (dict(w=torch.zeros(7, 4)), r"w must be \[8, 4\]"),
        (dict(w=torch.zeros(8, 4, dtype=torch.int32)), "floating"), (dict(bias=torch.zeros(7)), r"bias must be \[8\]"),
        (dict(act="gelu"), "activation"), (dict(start=torch.zeros(2, 4, 8)), "start must be"),
        (dict(start=torch.zeros(2, 3, 8).half()), "the samples are"), (dict(lengths=torch.zeros(3, dtype=torch.int32)), r"lengths must be \[2\]"),
        (dict(lengths=torch.zeros(2)), "integers"), (dict(lengths=torch.zeros(2, dtype=torch.uint32)), "integers"),
    ]
    for change, text in bad:
        args = {**dict(u=u, w=w), **change}
        for fn in (nmpc_amd.causal_conv, nmpc_amd.causal_conv_fwd):
            with pytest.raises(nmpc_amd.NmpcError, match=text):
                fn(**args)
    with pytest.raises(nmpc_amd.NmpcError, match="batch, channels"):
        nmpc_amd.causal_conv_step(torch.zeros(2, 3, 8), u, w)
    with pytest.raises(nmpc_amd.NmpcError, match="contiguous"):
        nmpc_amd.causal_conv_step(torch.zeros(2, 8, 3).transpose(1, 2), u[:, 0], w)
    with pytest.raises(nmpc_amd.NmpcError, match="no gradient"):
        nmpc_amd.causal_conv_step(torch.zeros(2, 3, 8), u[:, 0], w.clone().requires_grad_())
    with pytest.raises(nmpc_amd.NmpcError, match="causal_conv_fwd returned"):
        nmpc_amd.causal_conv_bwd("saved", u)


def test_lengths_keep_their_meaning():
    """Integers of every width mean the same steps; those past 32 bits are above or below every length."""
    from nmpc_amd.seq import _lengths
    for t in (torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64):
        got = _lengths("f", torch.tensor([0, 100, 7], dtype=t), 3)
        assert got.dtype is torch.int32 and got.tolist() == [0, 100, 7]
    got = _lengths("f", torch.tensor([2 ** 40, -2 ** 40, 5]), 3).tolist()
    assert got[0] == 2 ** 31 - 1 and got[1] < 0 and got[2] == 5
    assert _lengths("f", torch.arange(8)[::2], 4).is_contiguous()


def test_conv_abi_refusals():
    L = _lib.lib()
    buf = (ctypes.c_float * 64)()                     # never touched: every call below is refused first
    p = ctypes.addressof(buf)
    def fwd(dtype=0, nb=1, steps=4, d=4, taps=4, u=p, w=p, act=0, y=p):
        return L.nmpc_causal_conv(dtype, nb, steps, d, taps, u, 16, 4, w, None, act, None, None, y, None, None)
    for kw in (dict(dtype=3), dict(nb=-1), dict(steps=-1), dict(d=0), dict(taps=0), dict(taps=9), dict(u=None), dict(w=None),
               dict(act=2), dict(y=None), dict(nb=1 << 30, steps=1 << 10), dict(steps=2 ** 31 - 1, d=1)):
        assert fwd(**kw) != 0 and L.nmpc_last_error(), kw
    assert fwd(nb=0, u=None, y=None) == 0             # nothing to do
    need = L.nmpc_causal_conv_workspace_bytes(2, 40, 8, 4)
    assert need == ((2 * 3 + 7) // 8) * 5 * 8 * 4
    rc = L.nmpc_causal_conv_bwd(0, 2, 40, 8, 4, p, 320, 8, p, None, 0, None, None, p, 320, 8, None, p, p, None, None, p, need - 1, None)
    assert rc != 0 and b"workspace" in L.nmpc_last_error()
    assert L.nmpc_causal_conv_step(0, 1, 4, 4, None, p, 4, p, None, 0, p, None) != 0


def test_seq_operators_need_a_gpu():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    with pytest.raises(nmpc_amd.NmpcError):
        nmpc_amd.causal_conv(torch.zeros(1, 4, 8), torch.zeros(8, 4))


def test_oracle_scan_gradient_against_differences():
    g = rng(2)
    nb, steps, d, n, groups = 2, 4, 4, 2, 2
    leaves = [_double(g, nb, steps, d), _double(g, nb, steps, d), (-torch.rand(d, n, generator=g, dtype=torch.float64)).requires_grad_(),
              _double(g, nb, steps, groups, n), _double(g, nb, steps, groups, n), _double(g, d), _double(g, nb, steps, d), _double(g, d),
              _double(g, nb, d, n)]
    for lengths in (None, [3, 0]):
        assert torch.autograd.gradcheck(lambda *a: oracle.lpv_scan(*a[:8], start=a[8], lengths=lengths), leaves)


def test_scan_refusals():
    u, A, B = torch.zeros(2, 6, 8), torch.zeros(8, 4), torch.zeros(2, 6, 2, 4)
    ok = dict(u=u, dt=u, A=A, B=B, C=B)
    bad = [
        (dict(u=u[0]), "batch, steps, channels"), (dict(u=u.double()), "float32, bfloat16"), (dict(dt=u[:, :5]), "dt must be"),
        (dict(dt=u.half()), "the samples are"), (dict(A=torch.zeros(8, 65)), "1..64 states"), (dict(A=torch.zeros(7, 4)), "A must be"),
        (dict(B=torch.zeros(2, 6, 3, 4), C=torch.zeros(2, 6, 3, 4)), "do not divide"), (dict(B=torch.zeros(2, 6, 4)), "B must be"),
        (dict(C=torch.zeros(2, 6, 1, 4)), "C must be"), (dict(D=torch.zeros(4)), "D must be"), (dict(z=u[..., :4]), "z must be"),
        (dict(dt_bias=torch.zeros(8, 1)), "dt_bias must be"), (dict(start=torch.zeros(2, 8, 5)), "start must be"),
        (dict(start=torch.zeros(2, 8, 4).half()), "states are float32"), (dict(lengths=torch.zeros(2)), "integers"),
    ]
    for change, text in bad:
        for fn in (nmpc_amd.lpv_scan, nmpc_amd.lpv_scan_fwd):
            with pytest.raises(nmpc_amd.NmpcError, match=text):
                fn(**{**ok, **change})
    one = dict(u=u[:, 0], dt=u[:, 0], A=A, B=B[:, 0], C=B[:, 0])
    for state, text in ((torch.zeros(2, 8, 5), "state must be"), (torch.zeros(2, 8, 4).bfloat16(), "states are float32"),
                        (torch.zeros(2, 4, 8).transpose(1, 2), "contiguous")):
        with pytest.raises(nmpc_amd.NmpcError, match=text):
            nmpc_amd.lpv_scan_step(state, **one)
    with pytest.raises(nmpc_amd.NmpcError, match="no gradient"):
        nmpc_amd.lpv_scan_step(torch.zeros(2, 8, 4), **{**one, "A": A.clone().requires_grad_()})


def test_scan_abi(tmp_path):
    """The ctypes mirror has the header's layout; every refusal comes back before anything is launched."""
    import os
    import subprocess
    from conftest import ROOT
    src, exe = tmp_path / "sz.c", tmp_path / "sz"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "nmpc_amd.h"\nint main(void){printf("%zu %zu %zu %zu\\n", sizeof(nmpc_scan_args), '
                   'offsetof(nmpc_scan_args, A), offsetof(nmpc_scan_args, dlast), offsetof(nmpc_scan_args, workspace_bytes));return 0;}\n')
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    S = _lib.ScanArgs
    assert list(map(int, subprocess.check_output([str(exe)]).split())) == [ctypes.sizeof(S), S.A.offset, S.dlast.offset, S.workspace_bytes.offset]
    L = _lib.lib()
    buf = (ctypes.c_float * 64)()
    p = ctypes.addressof(buf)
    def args(**kw):
        s = S()
        s.struct_size, s.nb, s.L, s.D, s.N, s.G = ctypes.sizeof(S), 1, 4, 4, 4, 1
        for k in ("u", "dt", "B", "C", "A", "y", "last", "saved", "dy", "du", "ddt", "dB", "dC", "dA"):
            setattr(s, k, p)
        for k, v in kw.items():
            setattr(s, k, v)
        return ctypes.addressof(s), s
    for kw in (dict(struct_size=8), dict(dtype=7), dict(nb=-1), dict(L=-1), dict(D=0), dict(N=0), dict(N=65), dict(G=3), dict(G=0), dict(A=None),
               dict(u=None), dict(C=None), dict(y=None), dict(nb=1 << 20, D=1 << 12), dict(L=2 ** 31 - 1, D=1)):
        at, hold = args(**kw)
        assert L.nmpc_lpv_scan(at, None) != 0 and L.nmpc_last_error(), kw
    for kw in (dict(saved=None), dict(dy=None), dict(dA=None), dict(dB=None), dict(z=p), dict(D_skip=p), dict(dt_bias=p), dict(workspace=None),
               dict(workspace=p, workspace_bytes=16)):
        at, hold = args(**kw)
        assert L.nmpc_lpv_scan_bwd(at, None) != 0 and L.nmpc_last_error(), kw
    for kw in (dict(saved=p + 4), dict(workspace=p + 8, workspace_bytes=1 << 30), dict(u_ts=-1), dict(z=p, dz=p, z_ts=1 << 25)):
        at, hold = args(**kw)
        assert L.nmpc_lpv_scan_bwd(at, None) != 0 and b"nmpc_lpv_scan_bwd" in L.nmpc_last_error(), kw
    for kw in (dict(last=None), dict(u=None), dict(y=None)):
        at, hold = args(**kw)
        assert L.nmpc_lpv_scan_step(at, None) != 0, kw
    assert L.nmpc_lpv_scan(None, None) != 0
    at, hold = args(nb=0)
    assert L.nmpc_lpv_scan(at, None) == 0 and L.nmpc_lpv_scan_step(at, None) == 0
    assert L.nmpc_lpv_scan_saved_bytes(2, 33, 8, 5) == 2 * 3 * 8 * 8 * 4          # a state of 8 padded values before every 16th step


def test_oracle_ffn_gradient_against_differences():
    g = rng(3)
    for name in ("silu", "gelu", "tanh", "sigmoid"):
        assert torch.autograd.gradcheck(lambda *a: oracle.gated_ffn(*a, name), (_double(g, 3, 4), _double(g, 5, 4), _double(g, 5, 4)))


def test_ffn_refusals():
    x, w = torch.zeros(3, 8), torch.zeros(6, 8)
    bad = [(dict(x=x.double()), "float32, bfloat16"), (dict(w_gate=torch.zeros(6, 7)), r"\[hidden, 8\]"), (dict(w_up=torch.zeros(5, 8)), "w_up must be"),
           (dict(w_up=w.half()), "the samples are"), (dict(w_gate=torch.zeros(8)), "w_gate must be"), (dict(act="relu"), "activation"),
           (dict(act=None), "activation"), (dict(w_gate=torch.zeros(0, 8), w_up=torch.zeros(0, 8)), "w_gate must be")]
    for change, text in bad:
        for fn in (nmpc_amd.gated_ffn, nmpc_amd.gated_ffn_fwd):
            with pytest.raises(nmpc_amd.NmpcError, match=text):
                fn(**{**dict(x=x, w_gate=w, w_up=w), **change})
    with pytest.raises(nmpc_amd.NmpcError, match="gated_ffn_fwd returned"):
        nmpc_amd.gated_ffn_bwd(None, x)


def test_ffn_abi_refusals():
    L = _lib.lib()
    buf = (ctypes.c_float * 64)()
    p = ctypes.addressof(buf)
    def fwd(dtype=0, m=4, k=4, f=4, x=p, wg=p, wu=p, ldu=4, act=1, h=p):
        return L.nmpc_gated_ffn(dtype, m, k, f, x, 4, wg, 4, wu, ldu, act, h, None, None, 0, None)
    for kw in (dict(dtype=-1), dict(m=-1), dict(k=0), dict(f=0), dict(x=None), dict(wg=None), dict(wu=None), dict(h=None), dict(act=0), dict(act=5),
               dict(ldu=8), dict(m=1 << 22)):
        assert fwd(**kw) != 0 and L.nmpc_last_error(), kw
    assert fwd(m=0, x=None, h=None) == 0
    need = L.nmpc_gated_ffn_workspace_bytes(1, 100, 64, 128, 1, 0)
    assert need > 0
    rc = L.nmpc_gated_ffn_bwd(1, 100, 64, 128, p, 64, p, 64, p, 64, 1, p, p, 128, p, p, p, p, need - 1, None)
    assert rc != 0 and b"workspace" in L.nmpc_last_error()
    rc = L.nmpc_gated_ffn_bwd(1, 100, 64, 128, p, 64, p, 64, p, 64, 1, None, p, 128, p, p, p, p, need, None)
    assert rc != 0 and b"null" in L.nmpc_last_error()


def test_forward_mode_tangents_are_refused():
    """A dual tensor does not ask for a gradient, and its tangent would be dropped: every form refuses it, with gradients enabled or not."""
    from torch.autograd import forward_ad
    u, w, A, B, x, wg = torch.zeros(2, 6, 8), torch.zeros(8, 4), torch.zeros(8, 4), torch.zeros(2, 6, 2, 4), torch.zeros(3, 8), torch.zeros(6, 8)
    scan = dict(u=u, dt=u, A=A, B=B, C=B, D=torch.zeros(8), z=u, dt_bias=torch.zeros(8), start=torch.zeros(2, 8, 4))
    one = {k: t[:, 0] if k in ("u", "dt", "B", "C", "z") else t for k, t in scan.items() if k != "start"}
    one["state"] = scan["start"]
    conv = dict(u=u, w=w, bias=torch.zeros(8), start=torch.zeros(2, 3, 8))
    step = dict(window=torch.zeros(2, 3, 8), u=u[:, 0], w=w, bias=torch.zeros(8))
    ffn = dict(x=x, w_gate=wg, w_up=wg)
    calls = [(nmpc_amd.causal_conv, conv), (nmpc_amd.causal_conv_fwd, conv), (nmpc_amd.causal_conv_step, step), (nmpc_amd.lpv_scan, scan),
             (nmpc_amd.lpv_scan_fwd, scan), (nmpc_amd.lpv_scan_step, one), (nmpc_amd.gated_ffn, ffn), (nmpc_amd.gated_ffn_fwd, ffn)]
    with forward_ad.dual_level():
        for fn, args in calls:
            for name in args:
                dual = {**args, name: forward_ad.make_dual(args[name], torch.ones_like(args[name]))}
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(nmpc_amd.NmpcError, match="tangent"):
                        fn(**dual)
        for fn, grads in ((nmpc_amd.causal_conv_bwd, ("dy", "dwindow")), (nmpc_amd.lpv_scan_bwd, ("dy", "dlast")), (nmpc_amd.gated_ffn_bwd, ("dh",))):
            for name in grads:
                with pytest.raises(nmpc_amd.NmpcError, match="tangent"):
                    fn(None, **{**dict.fromkeys(grads, u), name: forward_ad.make_dual(u, u)})
        with pytest.raises(nmpc_amd.NmpcError) as plain:                # a level is open, but nothing carries a tangent
            nmpc_amd.gated_ffn(x.double(), wg, wg)
    assert "tangent" not in str(plain.value)
    with pytest.raises(nmpc_amd.NmpcError, match="tangent"):
        torch.func.jvp(lambda v: nmpc_amd.gated_ffn(v, wg, wg), (x,), (x,))


def test_plan_queries():
    """Which kernels calls take: the refusals, and agreement with the workspaces."""
    L = _lib.lib()
    plan = L.nmpc_lpv_scan_plan
    for bad in ((0, 4, 4, 4, 1), (1, 0, 4, 4, 1), (1, 4, 0, 4, 1), (1, 4, 4, 65, 1), (1, 4, 4, 4, 3), (1, 4, 4, 4, 0)):
        assert plan(*bad, 0) == -1 and plan(*bad, 1) == -1
    for size in ((1, 1, 1, 1, 1), (1, 8192, 2048, 16, 1), (4, 2048, 2048, 16, 1), (120, 40, 1000, 8, 2), (2, 400, 10, 49, 2)):
        parts = plan(*size, 0)                        # parts have a workspace, the others none
        assert parts >= 0 and (parts > 1) == (L.nmpc_lpv_scan_workspace_bytes(*size, 0) > 0), size
        assert plan(*size, 1) >= 1, size
    shape = (ctypes.c_int * 3)()
    at = ctypes.addressof(shape)
    for bad in ((3, 4, 4, 4, 0, 0, at), (0, 0, 4, 4, 0, 0, at), (0, 4, 0, 4, 0, 0, at), (0, 4, 4, 4, 3, 0, at), (0, 4, 4, 4, -1, 0, at), (0, 4, 4, 4, 0, 0, None)):
        assert L.nmpc_gated_ffn_plan(*bad) != 0 and b"nmpc_gated_ffn_plan" in L.nmpc_last_error(), bad
    for product, most in ((0, (64, 32, 16)), (1, (256, 256, 64)), (2, (256, 256, 64))):       # one row: the kernel for few rows forward
        assert L.nmpc_gated_ffn_plan(1, 1, 2048, 8192, product, 0, at) == 0
        assert all(1 <= v <= top for v, top in zip(shape, most)) and (shape[1] == 32) == (product == 0)


def test_sizes_past_one_launch_are_refused_before_anything_runs():
    """The sums of the parameters' gradients take four threads a value: channels whose sums do not fit a launch are refused at the entry, not
    by the runtime after the kernels before them."""
    L = _lib.lib()
    buf = (ctypes.c_float * 64)()
    p = ctypes.addressof(buf)
    many = 1 << 30
    for nb in (0, 1):
        assert L.nmpc_causal_conv_bwd(1, nb, 1, many, 1, p, many, many, p, None, 0, None, None, p, many, many, None, p, p, None, None, p, 1 << 62, None) != 0
        assert b"channels (fewer than 2^30)" in L.nmpc_last_error()
    s = _lib.ScanArgs()
    s.struct_size, s.nb, s.L, s.D, s.N, s.G = ctypes.sizeof(s), 1, 1, 1 << 24, 64, 1
    for k in ("u", "dt", "B", "C", "A", "saved", "dy", "du", "ddt", "dB", "dC", "dA", "workspace"):
        setattr(s, k, (p + 15) // 16 * 16)
    s.workspace_bytes = 1 << 62
    assert L.nmpc_lpv_scan_bwd(ctypes.addressof(s), None) != 0 and b"too many channels and states" in L.nmpc_last_error()
