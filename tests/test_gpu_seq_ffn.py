"""Gated feed-forward projections against their definition in fp64 (gradients: autograd of it).  Bounds: a product over K
terms is 2 K roundings to fp32 of terms that add up to sum |x| |w|; an activation is 24 roundings of its value and of
min(1, |x|), its slope is below 1.13 and the slope's below 1; dG and dU are rounded to the element type once (half a step)
as operands of the products behind them."""
import pytest
import torch

import nmpc_amd
from oracle import seq as oracle
from seq_util import DTYPES, U32, assert_close, f64, leaf, normal, rng

pytestmark = pytest.mark.gpu


def _inputs(seed, m, k, f, dtype):
    g = rng(seed)
    t = DTYPES[dtype]
    return normal(g, m, k, dtype=t), normal(g, f, k, scale=k ** -0.5, dtype=t), normal(g, f, k, scale=k ** -0.5, dtype=t), normal(g, m, f, dtype=t)


def _bounds(x, wg, wu, dh, name):
    """Absolute error that fp32 arithmetic and the operands' rounding may cause, per output."""
    half = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 0.0
    x, wg, wu, dh = (t.detach().double() for t in (x, wg, wu, dh))
    k, f = x.shape[1], wg.shape[0]
    gate, up = x @ wg.T, x @ wu.T
    eg, eu = (2 * k * U32 * (x.abs() @ w.abs().T) for w in (wg, wu))
    gl = gate.clone().requires_grad_()
    a = oracle.act(gl, name)
    slope = torch.autograd.grad(a.sum(), gl)[0] if a.numel() else gate
    a = a.detach()
    ea = 1.13 * eg + 24 * U32 * (a.abs() + gate.abs().clamp(max=1))
    es = eg + 24 * U32 * (slope.abs() + gate.abs().clamp(max=1))
    eh = ea * (up.abs() + eu) + a.abs() * eu + 2 * U32 * (a * up).abs()
    dg, du = dh * up * slope, dh * a
    edg = dh.abs() * (es * (up.abs() + eu) + slope.abs() * eu) + (4 * U32 + half) * dg.abs()
    edu = dh.abs() * ea + (4 * U32 + half) * du.abs()
    edg, edu = edg * (1 + half), edu * (1 + half)
    edx = edg @ wg.abs() + edu @ wu.abs() + 4 * f * U32 * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    m = x.shape[0]
    edwg, edwu = ((e.T @ x.abs()) + 2 * m * U32 * (d.abs().T @ x.abs()) for e, d in ((edg, dg), (edu, du)))
    return {"h": eh, "dx": edx, "dwg": edwg, "dwu": edwu}


def _run(x, wg, wu, dh, name):
    h, saved = nmpc_amd.gated_ffn_fwd(x.cuda(), wg.cuda(), wu.cuda(), name)
    dx, dwg, dwu = nmpc_amd.gated_ffn_bwd(saved, dh.cuda())
    return {"h": h, "dx": dx, "dwg": dwg, "dwu": dwu}


CASES = [  # rows, inputs, hidden units, dtype, activation
    (1, 1, 1, "f32", "silu"), (1, 8, 16, "bf16", "silu"), (1, 333, 77, "f16", "gelu"), (1, 1024, 200, "bf16", "silu"), (3, 64, 64, "bf16", "tanh"),
    (5, 40, 130, "f32", "sigmoid"), (16, 256, 96, "f16", "silu"), (17, 100, 33, "bf16", "gelu"), (63, 65, 129, "f32", "tanh"),
    (64, 64, 64, "bf16", "silu"), (65, 72, 136, "f16", "sigmoid"), (128, 128, 256, "bf16", "silu"), (200, 96, 520, "bf16", "gelu"),
    (257, 136, 264, "f16", "silu"), (300, 512, 300, "f32", "gelu"), (513, 80, 48, "bf16", "tanh"),
]


@pytest.mark.parametrize("m,k,f,dtype,name", CASES)
def test_forward_and_gradients(m, k, f, dtype, name):
    x, wg, wu, dh = _inputs(m + k, m, k, f, dtype)
    lx, lg, lu = leaf(x), leaf(wg), leaf(wu)
    ho = oracle.gated_ffn(lx, lg, lu, name)
    want = dict(zip(("dx", "dwg", "dwu"), torch.autograd.grad(ho, (lx, lg, lu), f64(dh))), h=ho)
    got = _run(x, wg, wu, dh, name)
    bound = _bounds(x, wg, wu, dh, name)
    for key in ("h", "dx", "dwg", "dwu"):
        assert_close(got[key], want[key], 1 / U32, bound[key], key)
    assert torch.equal(nmpc_amd.gated_ffn(x.cuda(), wg.cuda(), wu.cuda(), name), got["h"])
    again = _run(x, wg, wu, dh, name)
    assert all(torch.equal(got[key], again[key]) for key in got), "the same call gives the same bits"


@pytest.mark.parametrize("m,k,f,dtype,name", [
    (700, 1032, 1500, "bf16", "silu"),        # tiles of 128 x 128, k tail
    (2200, 160, 4104, "f16", "gelu"),         # tiles of 256 x 256, ragged in both directions
    (640, 320, 1800, "f32", "tanh"),
    (2049, 96, 4100, "bf16", "sigmoid"),      # odd rows, hidden units not a multiple of 8
    (150, 72, 9000, "f32", "silu"),           # contraction of the gradients split
])
def test_many_tiles(m, k, f, dtype, name):
    """The same at sizes of many tiles; the definition is evaluated in fp64 on the GPU."""
    x, wg, wu, dh = (t.cuda() for t in _inputs(m, m, k, f, dtype))
    lx, lg, lu = (t.double().requires_grad_() for t in (x, wg, wu))
    ho = oracle.gated_ffn(lx, lg, lu, name)
    want = dict(zip(("dx", "dwg", "dwu"), torch.autograd.grad(ho, (lx, lg, lu), dh.double())), h=ho)
    got = _run(x, wg, wu, dh, name)
    bound = _bounds(x, wg, wu, dh, name)
    for key in ("h", "dx", "dwg", "dwu"):
        assert_close(got[key], want[key], 1 / U32, bound[key].cpu(), key)


def test_no_rows():
    x, wg, wu, dh = _inputs(0, 0, 24, 40, "bf16")
    got = _run(x, wg, wu, dh, "silu")
    assert got["h"].shape == (0, 40) and got["dx"].shape == (0, 24) and not got["dwg"].any() and not got["dwu"].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m", [2, 70, 300])
def test_strides_and_leading_dimensions(dtype, m):
    x, wg, wu, dh = (t.cuda() for t in _inputs(9, 2 * m, 64, 96, dtype))
    want = _run(x, wg, wu, dh, "silu")
    h, saved = nmpc_amd.gated_ffn_fwd(x.view(2, m, 64), wg, wu)
    assert torch.equal(h.view(2 * m, 96), want["h"])
    grads = nmpc_amd.gated_ffn_bwd(saved, dh.view(2, m, 96))
    assert grads[0].shape == (2, m, 64) and torch.equal(grads[0].view(2 * m, 64), want["dx"]) and torch.equal(grads[1], want["dwg"])
    g = rng(4)
    for off, width in ((0, 128), (8, 128), (1, 129)):               # rows of wider tensors, also where no 16-byte access may start
        wide = normal(g, 2 * m, width, dtype=DTYPES[dtype]).cuda()
        both = normal(g, 192, width, dtype=DTYPES[dtype]).cuda()
        wdh = normal(g, 2 * m, 97 + off, dtype=DTYPES[dtype]).cuda()
        p = (wide[:, off:off + 64], both[:96, off:off + 64], both[96:, off:off + 64], wdh[:, off:off + 96])
        a, b = _run(*p, "silu"), _run(*[t.contiguous() for t in p], "silu")
        # aligned and unaligned rows may take different kernels, which add in other orders: each result lies within `bound` of the
        # exact value before its last rounding, so that two of them differ by at most twice that and their roundings
        bound, half = _bounds(*[t.contiguous() for t in p], "silu"), torch.finfo(DTYPES[dtype]).eps / 2 * (1 + 2.0 ** -6)
        for key in a:
            x64, y64 = a[key].double(), b[key].double()
            assert ((x64 - y64).abs() <= 2 * (1 + half) * bound[key] + half * (x64.abs() + y64.abs())).all(), key
    t = x.t().contiguous().t()                                       # columns contiguous: copied
    assert torch.equal(nmpc_amd.gated_ffn(t, wg, wu), want["h"])


@pytest.mark.parametrize("name", ["silu", "gelu", "tanh", "sigmoid"])
def test_far_arguments(name):
    """Saturated activations: finite values and slopes where the definition has them."""
    x = torch.tensor([[-300.0], [-30.0], [-5.0], [-1e-3], [0.0], [1e-3], [5.0], [30.0], [300.0]])
    one = torch.ones(1, 1)
    got = _run(x, one, one, torch.ones(9, 1), name)
    lx, lg, lu = leaf(x), leaf(one), leaf(one)
    ho = oracle.gated_ffn(lx, lg, lu, name)
    want = dict(zip(("dx", "dwg", "dwu"), torch.autograd.grad(ho, (lx, lg, lu), torch.ones(9, 1, dtype=torch.float64))), h=ho)
    bound = _bounds(x, one, one, torch.ones(9, 1), name)
    for key in want:
        # an exponential rounds its argument of up to 300 twice: a relative error of 600 roundings of a result below 2^-40
        assert_close(got[key], want[key], 1 / U32, bound[key] + 1e-7 * 2.0 ** -30, key)


def test_gradient_against_differences():
    x, wg, wu, dh = _inputs(31, 12, 20, 24, "f32")
    got = _run(x, wg, wu, dh, "silu")
    h = 2.0 ** -7
    for i, key in ((0, "dx"), (1, "dwg"), (2, "dwu")):
        base = [x, wg, wu]
        d = normal(rng(50 + i), *base[i].shape)
        d = d / d.norm()
        def loss(s):
            args = [t + s * d if j == i else t for j, t in enumerate(base)]
            return float((f64(nmpc_amd.gated_ffn(*[t.cuda() for t in args], "silu")) * f64(dh)).sum())
        slope = (loss(h) - loss(-h)) / (2 * h)
        # truncation h^2 times a third derivative of order 10, rounding of a loss that adds up 300 terms of order 1
        assert abs(slope - float((f64(got[key]) * f64(d)).sum())) < 10 * h * h + 300 * 40 * U32 / h, key


def test_autograd_is_the_pair_and_capture():
    x, wg, wu, dh = (t.cuda() for t in _inputs(12, 130, 64, 136, "bf16"))
    want = _run(x, wg, wu, dh, "silu")
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    got = torch.autograd.grad(nmpc_amd.gated_ffn(*leaves, "silu"), leaves, dh)
    assert all(torch.equal(a, want[k]) for a, k in zip(got, ("dx", "dwg", "dwu")))
    for m in (1, 130):
        xs, ds = x[:m].clone(), dh[:m].clone()
        step = lambda: list(_run(xs, wg, wu, ds, "silu").values())   # noqa: E731
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for k in range(3):
            xs.copy_(torch.randn(xs.shape, generator=rng(k)).to(xs.dtype))
            graph.replay()
            torch.cuda.synchronize()
            for a, e in zip(outs, step()):
                assert torch.equal(a, e)
