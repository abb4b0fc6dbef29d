"""Causal convolution against the step-by-step definition in fp64.  Bounds: a filter of W taps is W products and W sums in
fp32 (2 W roundings of terms that add up to `scale`), SiLU adds 8 more (the sigmoid's exponential and reciprocal are within
2 steps each, its argument is rounded twice and moves the sigmoid by at most |s|/4 of that) and its slope is below 1.1."""
import pytest
import torch

import nmpc_amd
from oracle import seq as oracle
from seq_util import DTYPES, assert_close, f64, gpu, leaf, normal, rng

pytestmark = pytest.mark.gpu


def _inputs(seed, nb, steps, d, taps, dtype, bias, start, lengths):
    g = rng(seed)
    u = normal(g, nb, steps, d, dtype=dtype)
    w, b = normal(g, d, taps, scale=taps ** -0.5), normal(g, d, scale=0.3) if bias else None
    s = normal(g, nb, taps - 1, d, dtype=dtype) if start else None
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return u, w, b, s, n, normal(g, nb, steps, d, dtype=dtype), normal(g, nb, taps - 1, d, dtype=dtype)


CASES = [  # nb, steps, d, taps, dtype, act, bias, start, lengths
    (1, 1, 1, 1, "f32", None, False, False, None),
    (2, 3, 5, 4, "f32", "silu", True, True, None),              # fewer steps than taps
    (3, 16, 64, 4, "bf16", "silu", True, False, None),          # one run exactly
    (2, 17, 72, 4, "bf16", "silu", True, True, None),           # one step more
    (2, 33, 33, 3, "f16", "silu", True, True, None),            # odd channels: element by element
    (4, 40, 24, 8, "f16", None, False, True, [0, 1, 40, 7]),    # empty sequence, single step, full, shorter than the filter
    (5, 35, 264, 4, "bf16", "silu", True, True, [35, 16, 0, 3, 17]),
    (2, 50, 8, 2, "f32", "silu", False, False, [50, 49]),
    (1, 130, 520, 5, "f32", "silu", True, False, None),
    (2, 19, 40, 7, "bf16", "silu", True, True, [2, 19]),
    (2, 21, 16, 6, "f32", None, True, True, None),
    (3, 0, 8, 4, "f32", "silu", True, True, None),              # no steps
]


def _scale(u, w, b, s, n):
    """Per output: the sum of its terms' magnitudes."""
    a = lambda t: None if t is None else f64(t).abs()
    return oracle.causal_conv(a(u), a(w), a(b), None, a(s), n)[0]


@pytest.mark.parametrize("nb,steps,d,taps,dtype,act,bias,start,lengths", CASES)
def test_forward_and_gradients(nb, steps, d, taps, dtype, act, bias, start, lengths):
    u, w, b, s, n, dy, dwin = _inputs(7, nb, steps, d, taps, DTYPES[dtype], bias, start, lengths)
    lu, lw, lb, ls = leaf(u), leaf(w), leaf(b), leaf(s)
    yo, wo = oracle.causal_conv(lu, lw, lb, act, ls, n)
    y, win, saved = nmpc_amd.causal_conv_fwd(gpu(u), gpu(w), gpu(b), act, gpu(s), gpu(n))
    scale = _scale(u, w, b, s, n)
    assert_close(y, yo, 1.1 * 2 * taps + 8, scale, "y")
    assert torch.equal(f64(win), wo.detach()), "the window is a copy"
    grads = nmpc_amd.causal_conv_bwd(saved, gpu(dy), gpu(dwin))
    if steps == 0:
        want = {"dw": torch.zeros(d, taps), "dbias": torch.zeros(d), "du": torch.zeros(nb, 0, d), "dstart": f64(dwin)}
        for k, v in want.items():
            assert torch.equal(f64(grads[k]), v.double()), k
        return
    leaves = {"du": lu, "dw": lw, "dbias": lb, "dstart": ls}
    named = {k: v for k, v in leaves.items() if v is not None}
    want = dict(zip(named, torch.autograd.grad([yo, wo], list(named.values()), [f64(dy), f64(dwin)], allow_unused=True)))
    # magnitudes: |ds| <= 1.1 |dy|; the slope's own error is 12 roundings plus that of s (2 W roundings of its terms, slope's derivative <= 0.5)
    size = (f64(dy).abs() * (1.1 + scale)).contiguous()
    a = {"u": f64(u).abs(), "w": f64(w).abs(), "s": None if s is None else f64(s).abs()}
    au, aw, asr = a["u"].requires_grad_(), a["w"].requires_grad_(), None if s is None else a["s"].requires_grad_()
    lin, linw = oracle.causal_conv(au, aw, None, None, asr, n)
    ab = torch.autograd.grad([lin, linw], [au, aw] + ([asr] if s is not None else []), [size, f64(dwin).abs()])
    big = {"du": ab[0], "dw": ab[1], "dbias": size.sum((0, 1)), "dstart": ab[2] if s is not None else None}
    count = {"du": 4 * taps + 14, "dw": 2 * taps + 14 + 16 + 40, "dbias": 2 * taps + 14 + 16 + 40, "dstart": 4 * taps + 14}
    for k, v in want.items():
        assert_close(grads[k], torch.zeros_like(named[k]) if v is None else v, count[k], big[k], k)
    for k in grads:
        assert (grads[k] is None) == (k not in named), k


@pytest.mark.parametrize("steps", [15, 17, 27, 28, 29, 31, 32, 55, 56, 57, 59, 85])
@pytest.mark.parametrize("act,cut", [("silu", 0), (None, 9)])
def test_ends_of_runs(steps, act, cut):
    """Either side of the runs of steps that a thread owns, forward (16) and backward (28)."""
    test_forward_and_gradients(2, steps, 20, 4, "f32", act, True, True, [steps, steps - cut])


def test_no_sequences():
    y, window, saved = nmpc_amd.causal_conv_fwd(torch.zeros(0, 5, 8, device="cuda"), torch.ones(8, 3, device="cuda"), torch.ones(8, device="cuda"))
    grads = nmpc_amd.causal_conv_bwd(saved, torch.zeros(0, 5, 8, device="cuda"))
    assert y.shape == (0, 5, 8) and window.shape == (0, 2, 8) and not grads["dw"].any() and not grads["dbias"].any()


def test_padding_is_never_read():
    u, w, b, s, _, dy, dwin = _inputs(3, 3, 40, 64, 4, torch.float32, True, True, None)
    n = torch.tensor([0, 5, 33], dtype=torch.int32)
    clean = nmpc_amd.causal_conv_fwd(u.cuda(), w.cuda(), b.cuda(), "silu", s.cuda(), n.cuda())
    gclean = nmpc_amd.causal_conv_bwd(clean[2], dy.cuda(), dwin.cuda())
    for i, k in enumerate(n.tolist()):
        u[i, k:] = float("nan")
        dy[i, k:] = float("inf")
    dirty = nmpc_amd.causal_conv_fwd(u.cuda(), w.cuda(), b.cuda(), "silu", s.cuda(), n.cuda())
    gdirty = nmpc_amd.causal_conv_bwd(dirty[2], dy.cuda(), dwin.cuda())
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    for k in gclean:
        assert torch.equal(gclean[k], gdirty[k]), k
    for i, k in enumerate(n.tolist()):
        assert not dirty[0][i, k:].any() and not gdirty["du"][i, k:].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_parts_of_a_wider_tensor(dtype):
    g = rng(5)
    both = normal(g, 2, 21, 3 * 64 + 1, dtype=DTYPES[dtype]).cuda()
    w, b = normal(g, 64, 4).cuda(), normal(g, 64).cuda()
    dy = normal(g, 2, 21, 128, dtype=DTYPES[dtype]).cuda()
    for lo in (0, 64, 65):                                     # 65: rows that no 16-byte access may start at
        u, gy = both[..., lo:lo + 64], dy[..., 64:]
        y0, w0, s0 = nmpc_amd.causal_conv_fwd(u.contiguous(), w, b, "silu")
        y1, w1, s1 = nmpc_amd.causal_conv_fwd(u, w, b, "silu")
        assert torch.equal(y0, y1) and torch.equal(w0, w1)
        g0, g1 = nmpc_amd.causal_conv_bwd(s0, gy.contiguous()), nmpc_amd.causal_conv_bwd(s1, gy)
        assert torch.equal(g0["du"], g1["du"])
        assert torch.allclose(g0["dw"], g1["dw"], rtol=1e-5, atol=1e-5)
    flipped = both[..., :64].transpose(1, 2).contiguous().transpose(1, 2)      # channels not contiguous: copied
    assert torch.equal(nmpc_amd.causal_conv(flipped, w, b, "silu"), nmpc_amd.causal_conv(both[..., :64], w, b, "silu"))


@pytest.mark.parametrize("dtype,d,taps", [("bf16", 128, 4), ("f32", 37, 3), ("f16", 64, 1), ("f16", 8, 8)])
def test_steps_continue_a_prompt(dtype, d, taps):
    u, w, b, s, _, _, _ = _inputs(11, 3, 24, d, taps, DTYPES[dtype], True, True, None)
    u, w, b, s = (t.cuda() for t in (u, w, b, s))
    whole, last = nmpc_amd.causal_conv(u, w, b, "silu", start=s, return_state=True)
    y, window = nmpc_amd.causal_conv(u[:, :10], w, b, "silu", start=s, return_state=True)
    assert torch.equal(y, whole[:, :10])
    for t in range(10, 24):
        assert torch.equal(nmpc_amd.causal_conv_step(window, u[:, t], w, b, "silu"), whole[:, t])
    assert torch.equal(window, last)


def test_autograd_is_the_pair():
    u, w, b, s, n, dy, _ = _inputs(2, 2, 20, 16, 4, torch.float32, True, True, [20, 11])
    leaves = [t.cuda().requires_grad_() for t in (u, w, b, s)]
    y = nmpc_amd.causal_conv(*leaves[:3], "silu", start=leaves[3], lengths=n.cuda())
    got = torch.autograd.grad(y, leaves, dy.cuda())
    _, _, saved = nmpc_amd.causal_conv_fwd(*[t.detach() for t in leaves[:3]], "silu", start=leaves[3].detach(), lengths=n.cuda())
    want = nmpc_amd.causal_conv_bwd(saved, dy.cuda())
    for a, k in zip(got, ("du", "dw", "dbias", "dstart")):
        assert torch.equal(a, want[k]), k


def test_captured_pair_replays_as_the_eager_calls():
    u, w, b, s, n, dy, dwin = (t.cuda() for t in _inputs(4, 3, 50, 64, 4, torch.bfloat16, True, True, [50, 0, 31]))
    def step():
        y, win, saved = nmpc_amd.causal_conv_fwd(u, w, b, "silu", s, n)
        return [y, win] + list(nmpc_amd.causal_conv_bwd(saved, dy, dwin).values())
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(3):
        u.copy_(torch.randn(u.shape, generator=rng(k)).to(u.dtype))
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(outs, step()):
            assert torch.equal(a, e)
    leaf_w = w.clone().requires_grad_()
    alive = nmpc_amd.causal_conv(u, leaf_w, b, "silu")         # an eager graph of the leaf lives
    with pytest.raises(nmpc_amd.NmpcError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            nmpc_amd.causal_conv(u, leaf_w, b, "silu")
    alive.float().sum().backward()
    assert torch.isfinite(leaf_w.grad).all()


def test_other_stream():
    u, w, b, _, _, _, _ = _inputs(9, 2, 64, 64, 4, torch.float32, True, False, None)
    want = nmpc_amd.causal_conv(u.cuda(), w.cuda(), b.cuda(), "silu")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = nmpc_amd.causal_conv(u.cuda(), w.cuda(), b.cuda(), "silu")
    side.synchronize()
    assert torch.equal(got, want)


def test_the_pair_records_nothing():
    """Leaves that have to be copied (rows apart, gradients asked for): what a pair keeps and returns hangs on no autograd graph."""
    g = rng(17)
    def apart(*shape):                                         # rows of a wider tensor, a leaf of its own
        t = torch.empty_strided(shape, (shape[1] * (shape[2] + 3), shape[2] + 3, 1), device="cuda")
        return t.copy_(normal(g, *shape)).requires_grad_()
    u, start, dwin, dy = apart(2, 9, 16), apart(2, 3, 16), apart(2, 3, 16), apart(2, 9, 16)
    w, b = normal(g, 16, 4).t().contiguous().t().cuda().requires_grad_(), normal(g, 32).cuda()[::2].detach().requires_grad_()
    y, window, saved = nmpc_amd.causal_conv_fwd(u, w, b, "silu", start)
    grads = nmpc_amd.causal_conv_bwd(saved, dy, dwin)
    wg = normal(g, 24, 16).cuda().requires_grad_()
    h, fsaved = nmpc_amd.gated_ffn_fwd(u, wg, wg)
    dh = apart(2, 9, 24)
    fgrads = nmpc_amd.gated_ffn_bwd(fsaved, dh)
    for t in [y, window, h, *saved.tensors, *fsaved.tensors, *grads.values(), *fgrads]:
        assert t is None or t.grad_fn is None
    plain = lambda t: t.detach().contiguous()                  # noqa: E731
    want = nmpc_amd.causal_conv_bwd(nmpc_amd.causal_conv_fwd(*map(plain, (u, w, b)), "silu", plain(start))[2], plain(dy), plain(dwin))
    assert all(torch.equal(grads[k], want[k]) for k in want)
