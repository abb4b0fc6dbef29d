"""Sequence operators on tensors of more than 2^31 elements: parts that hold the same numbers give the same bits wherever
they lie, and a few of them are held against the plain formulas."""
import pytest
import torch

import nmpc_amd
from oracle import seq as oracle
from seq_util import U32, assert_close, f64, leaf, normal, rng
from test_gpu_seq_ffn import _bounds
from test_gpu_seq_scan import NAMES, _magnitudes

pytestmark = pytest.mark.gpu


def test_conv_past_32_bit_offsets():
    steps, d = 70000, 16384
    one = torch.randn(1, steps, d, device="cuda", dtype=torch.bfloat16)
    u, dy = one.repeat(2, 1, 1), torch.ones(2, steps, d, device="cuda", dtype=torch.bfloat16)
    assert u.numel() > 2 ** 31
    w, b = normal(rng(1), d, 4).cuda(), normal(rng(2), d).cuda()
    y, window, saved = nmpc_amd.causal_conv_fwd(u, w, b, "silu")
    assert torch.equal(y[0], y[1]) and torch.equal(window[0], u[0, -3:]) and torch.equal(window[1], u[1, -3:])
    part = nmpc_amd.causal_conv(u[1:, -48:], w, b, "silu", u[1:, -51:-48])
    assert torch.equal(y[1:, -48:], part)
    g = nmpc_amd.causal_conv_bwd(saved, dy)
    assert torch.equal(g["du"][0], g["du"][1])
    short = nmpc_amd.causal_conv_bwd(nmpc_amd.causal_conv_fwd(u[1:, -48:], w, b, "silu", u[1:, -51:-48])[2], dy[1:, -48:])
    assert torch.equal(g["du"][1:, -48:], short["du"])


def test_scan_past_32_bit_offsets():
    steps, d, n = 50000, 16384, 16
    gen = rng(3)
    same = lambda t: t.repeat(3, *[1] * (t.dim() - 1))  # noqa: E731
    u, dt, z, dy = (same(torch.randn(1, steps, d, device="cuda", dtype=torch.bfloat16)) for _ in range(4))
    B, C = (same(normal(gen, 1, steps, 1, n, dtype=torch.bfloat16).cuda()) for _ in range(2))
    assert u.numel() > 2 ** 31
    A, D = (-torch.rand(d, n, generator=gen) * 4 - 0.05).cuda(), normal(gen, d).cuda()
    y, last, saved = nmpc_amd.lpv_scan_fwd(u, dt, A, B, C, D, z)
    g = nmpc_amd.lpv_scan_bwd(saved, dy)
    for k, t in {"y": y, "last": last, **{k: g[k] for k in ("du", "ddt", "dB", "dC", "dz")}}.items():
        assert torch.equal(t[0], t[2]), k
        assert torch.isfinite(t[2, -3:].float()).all(), k
    # 16 channels over the last 40 steps, from the state of a run that ends before them
    sel, cut = torch.arange(0, d, d // 16).cuda(), steps - 40
    _, state, _ = nmpc_amd.lpv_scan_fwd(u, dt, A, B, C, D, z, lengths=torch.full((3,), cut, device="cuda"))
    v = dict(u=u[2:, cut:, sel], dt=dt[2:, cut:, sel], A=A[sel], B=B[2:, cut:], C=C[2:, cut:], D=D[sel], z=z[2:, cut:, sel], dt_bias=None, start=state[2:, sel])
    want, end = oracle.lpv_scan(*[f64(v[k]) for k in NAMES[:8]], start=f64(v["start"]))
    m = _magnitudes(v, dy[2:, cut:, sel], torch.zeros_like(v["start"]), True, None)
    r = 52 + n + 3 * 40
    assert_close(y[2:, cut:, sel], want, r, m["y"], "y")
    assert_close(last[2:, sel], end, r, m["last"], "last")


def test_ffn_past_32_bit_offsets():
    m, k, f, few = 300000, 64, 8192, 40
    gen = rng(5)
    x = torch.randn(m, k, device="cuda", dtype=torch.bfloat16)
    x[:few] = x[-few:]
    wg, wu = (normal(gen, f, k, scale=0.1, dtype=torch.bfloat16) for _ in range(2))
    h, saved = nmpc_amd.gated_ffn_fwd(x, wg.cuda(), wu.cuda())
    assert h.numel() > 2 ** 31 and torch.equal(h[:few], h[-few:])
    dh = torch.zeros_like(h)
    dh[-few:] = normal(gen, few, f, dtype=torch.bfloat16).cuda()
    dx, dwg, dwu = nmpc_amd.gated_ffn_bwd(saved, dh)
    assert not dx[:-few].any()
    last, dlast = x[-few:].cpu(), dh[-few:].cpu()
    leaves = [leaf(t) for t in (last, wg, wu)]
    want = oracle.gated_ffn(*leaves, "silu")
    grads = torch.autograd.grad(want, leaves, f64(dlast))
    bound = _bounds(last, wg, wu, dlast, "silu")               # the other rows add zeros to the weights' gradients
    for name, got, ref in (("h", h[-few:], want), ("dx", dx[-few:], grads[0]), ("dwg", dwg, grads[1]), ("dwu", dwu, grads[2])):
        assert_close(got, ref, 1 / U32, bound[name], name)
