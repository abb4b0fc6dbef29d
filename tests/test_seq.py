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
        (dict(lengths=torch.zeros(2)), "integers"),
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


def test_conv_abi_refusals():
    L = _lib.lib()
    buf = (ctypes.c_float * 64)()                     # never touched: every call below is refused first
    p = ctypes.addressof(buf)
    def fwd(dtype=0, nb=1, steps=4, d=4, taps=4, u=p, w=p, act=0, y=p):
        return L.nmpc_causal_conv(dtype, nb, steps, d, taps, u, 16, 4, w, None, act, None, None, y, None, None)
    for kw in (dict(dtype=3), dict(nb=-1), dict(steps=-1), dict(d=0), dict(taps=0), dict(taps=9), dict(u=None), dict(w=None),
               dict(act=2), dict(y=None), dict(nb=1 << 30, steps=1 << 10)):
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
