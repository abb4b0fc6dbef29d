"""Selective LPV scan against the step-by-step definition in fp64 (gradients: autograd of it).  Bounds count roundings to
fp32 of terms whose magnitudes are followed through the same recurrence (`_magnitudes`).  delta: raw = dt + bias with
|raw| <= 9, its rounding and that of the exponential's argument move softplus by at most 2 |raw| roundings, log1p adds 3: 21.
The exponent delta A carries those and 3 more, times the exponent itself, and x e^-x <= 0.37: 9.  Each step adds a rounding
for the exponential and two for its fma; delta B u adds 23, the sum over N states N, D u and the gate 10: 52 + N + 3 L in
all.  A gradient meets that twice (state and adjoint) and its own sums over steps, sequences and channels."""
import pytest
import torch

import nmpc_amd
from oracle import seq as oracle
from seq_util import DTYPES, assert_close, f64, gpu, leaf, normal, rng

pytestmark = pytest.mark.gpu
NAMES = ("u", "dt", "A", "B", "C", "D", "z", "dt_bias", "start")


def _inputs(seed, nb, steps, d, n, groups, dtype, skip=True, gate=True, bias=True, start=True, softplus=True):
    g = rng(seed)
    t = DTYPES[dtype]
    v = dict(u=normal(g, nb, steps, d, dtype=t), dt=normal(g, nb, steps, d, scale=0.7, dtype=t), A=-torch.rand(d, n, generator=g) * n - 0.05,
             B=normal(g, nb, steps, groups, n, dtype=t), C=normal(g, nb, steps, groups, n, dtype=t), D=normal(g, d) if skip else None,
             z=normal(g, nb, steps, d, dtype=t) if gate else None, dt_bias=-3 + normal(g, d) if bias else None,
             start=normal(g, nb, d, n) if start else None)
    if not softplus:
        v["dt"] = (v["dt"].float().abs() * 0.1).to(t)
        v["dt_bias"] = None if v["dt_bias"] is None else v["dt_bias"].abs() * 0.01
    return v, normal(g, nb, steps, d, dtype=t), normal(g, nb, d, n)


def _magnitudes(v, dy, dlast, softplus, lengths):
    """What every output adds up, with all terms taken positive."""
    a = {k: f64(t) for k, t in v.items()}
    nb, steps, d = a["u"].shape
    groups, n = a["B"].shape[2:]
    raw = a["dt"] if a["dt_bias"] is None else a["dt"] + a["dt_bias"]
    delta = oracle.softplus(raw) if softplus else raw
    u, B, C = a["u"].abs(), a["B"].abs().repeat_interleave(d // groups, 2), a["C"].abs().repeat_interleave(d // groups, 2)
    D = torch.zeros(d, dtype=torch.float64) if a["D"] is None else a["D"].abs()
    gate = torch.ones_like(u) if a["z"] is None else oracle.act(a["z"], "silu").abs()
    m = {k: torch.zeros_like(a[k]) for k in NAMES if a[k] is not None}
    m.update(y=torch.zeros_like(u), last=torch.zeros(nb, d, n, dtype=torch.float64))
    ends = [steps] * nb if lengths is None else [min(max(int(k), 0), steps) for k in lengths]
    for b, end in enumerate(ends):
        x = torch.zeros(d, n, dtype=torch.float64) if a["start"] is None else a["start"][b].abs()
        xs = [x]
        for t in range(end):
            x = torch.exp(delta[b, t, :, None] * a["A"]) * x + (delta[b, t] * u[b, t])[:, None] * B[b, t]
            xs.append(x)
            m["y"][b, t] = ((x * C[b, t]).sum(1) + D * u[b, t]) * gate[b, t]
        m["last"][b] = x
        lam = f64(dlast)[b].abs()
        for t in reversed(range(end)):
            g = f64(dy)[b, t].abs() * gate[b, t]
            lam = lam + C[b, t] * g[:, None]
            s1 = (lam * B[b, t]).sum(1)
            e = torch.exp(delta[b, t, :, None] * a["A"])
            h = lam * e * xs[t]
            m["u"][b, t] = D * g + delta[b, t] * s1
            m["dt"][b, t] = (h * a["A"].abs()).sum(1) + u[b, t] * s1
            m["A"] += h * delta[b, t][:, None]
            m["B"][b, t] = (lam * (delta[b, t] * u[b, t])[:, None]).reshape(groups, -1, n).sum(1)
            m["C"][b, t] = (xs[t + 1] * g[:, None]).reshape(groups, -1, n).sum(1)
            if "D" in m:
                m["D"] += g * u[b, t]
            if "z" in m:
                m["z"][b, t] = f64(dy)[b, t].abs() * 1.1 * ((xs[t + 1] * C[b, t]).sum(1) + D * u[b, t])
            lam = lam * e
        if "start" in m:
            m["start"][b] = lam
    if "dt_bias" in m:
        m["dt_bias"] = m["dt"].sum((0, 1))
    return m


def _check(v, dy, dlast, softplus=True, lengths=None, grads=True):
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    nb, steps, d = v["u"].shape
    states = v["A"].shape[1]
    leaves = {k: leaf(t) for k, t in v.items()}
    yo, lo = oracle.lpv_scan(*[leaves[k] for k in NAMES[:8]], use_softplus=softplus, start=leaves["start"], lengths=n)
    m = _magnitudes(v, dy, dlast, softplus, n)
    args = [gpu(v[k]) for k in NAMES[:8]] + [softplus, gpu(v["start"]), gpu(n)]
    y, last, saved = nmpc_amd.lpv_scan_fwd(*args)
    r = 52 + states + 3 * steps
    assert_close(y, yo, r, m["y"], "y")
    assert_close(last, lo, r, m["last"], "last")
    y2, last2 = nmpc_amd.lpv_scan(*args, return_state=True)
    assert torch.equal(y, y2) and torch.equal(last, last2)
    if not grads:
        return
    got = nmpc_amd.lpv_scan_bwd(saved, gpu(dy), gpu(dlast))
    named = {k: t for k, t in leaves.items() if t is not None}
    want = dict(zip(named, torch.autograd.grad([yo, lo], list(named.values()), [f64(dy), f64(dlast)], allow_unused=True)))
    for k in NAMES:
        key = "d" + k if k != "start" else "dstart"
        if k not in named:
            assert got[key] is None
            continue
        w = torch.zeros_like(named[k]) if want[k] is None else want[k]
        assert_close(got[key], w, 2 * r + 20 + nb * steps + d, m[k], key)
    again = nmpc_amd.lpv_scan_bwd(saved, gpu(dy), gpu(dlast))
    assert all(torch.equal(got[k], again[k]) for k in got if got[k] is not None), "the same call gives the same bits"


CASES = [  # nb, steps, d, n, groups, dtype, skip, gate, bias, start, softplus, lengths
    (1, 1, 1, 1, 1, "f32", False, False, False, False, True, None),
    (2, 1, 3, 5, 1, "f32", True, True, True, True, True, None),
    (1, 31, 8, 4, 2, "f32", True, True, True, False, True, None),
    (2, 32, 64, 16, 1, "bf16", True, True, True, True, True, None),         # one tile, one block of channels
    (2, 33, 65, 16, 1, "bf16", True, True, True, True, True, None),         # one more of each
    (3, 70, 20, 8, 4, "f16", True, False, True, True, True, [70, 0, 33]),
    (2, 40, 24, 24, 2, "f16", False, True, True, True, True, [1, 40]),
    (2, 35, 18, 64, 1, "f32", True, True, True, True, True, [32, 35]),
    (1, 36, 9, 33, 3, "bf16", True, True, False, True, True, None),
    (2, 45, 33, 2, 1, "f32", True, True, True, True, False, None),          # step sizes given directly
    (2, 34, 300, 3, 1, "bf16", True, False, True, False, True, [-3, 99]),   # lengths outside 0 .. L are clamped
]


@pytest.mark.parametrize("nb,steps,d,n,groups,dtype,skip,gate,bias,start,softplus,lengths", CASES)
def test_forward_and_gradients(nb, steps, d, n, groups, dtype, skip, gate, bias, start, softplus, lengths):
    v, dy, dlast = _inputs(steps, nb, steps, d, n, groups, dtype, skip, gate, bias, start, softplus)
    _check(v, dy, dlast, softplus, lengths)


@pytest.mark.parametrize("n", [16, 17, 23, 24, 25, 32, 47, 48, 49])
@pytest.mark.parametrize("steps", [40, 300])
def test_states_per_lane(n, steps):
    """Either side of every change of lanes a channel and states a lane, whole sequences and parts of the time axis."""
    v, dy, dlast = _inputs(n, 2, steps, 10, n, 2, "f32")
    _check(v, dy, dlast, True, [steps, steps - 7])


@pytest.mark.parametrize("nb,steps,d,n,dtype,lengths", [
    (1, 515, 16, 16, "f32", None), (1, 600, 10, 4, "bf16", None), (2, 430, 8, 40, "f32", [430, 129]), (3, 330, 12, 8, "f16", [0, 65, 330])])
def test_long_records(nb, steps, d, n, dtype, lengths):
    """Few channels, many steps: the time axis is worked on in parts."""
    v, dy, dlast = _inputs(steps, nb, steps, d, n, 1, dtype)
    _check(v, dy, dlast, True, lengths)


@pytest.mark.parametrize("steps", [520, 1030])
def test_chunks_of_several_tiles(steps):
    """128 sequences of 17 or 33 tiles are cut into chunks of three or five tiles (the last of fewer) or slots, a sequence alone
    into chunks of one tile."""
    v, dy, dlast = _inputs(2, 128, steps, 4, 4, 1, "f32")
    n = torch.full((128,), steps, dtype=torch.int32)
    n[5], n[77] = 300, 0
    many = _scan_all(v, dy, dlast, n)
    shared = ("A", "D", "dt_bias")
    total = {k: torch.zeros_like(many["d" + k], dtype=torch.float64) for k in shared}
    for b in range(128):
        one = _scan_all({k: t if k in shared else t[b:b + 1] for k, t in v.items()}, dy[b:b + 1], dlast[b:b + 1], n[b:b + 1])
        for k in one:
            if k[1:] in shared:
                total[k[1:]] += one[k].double()
            else:
                # both are within 52 + N + 3 L roundings of the exact states and adjoints, each met at most twice
                assert (many[k][b:b + 1] - one[k]).norm() <= 4 * (56 + 3 * steps) * 2.0 ** -24 * (one[k].norm() + 1e-3), (b, k)
    for k in shared:
        assert (many["d" + k].double() - total[k]).norm() <= 4 * (56 + 3 * steps) * 2.0 ** -24 * total[k].norm(), k


def test_many_sequences_and_channels():
    """Enough of both that whole sequences fill the chip."""
    v, dy, dlast = _inputs(4, 120, 40, 1000, 4, 2, "f16")
    _check(v, dy, dlast, True, [40 - i % 41 for i in range(120)], grads=False)


def test_steep_and_flat_decay():
    """exp(delta A) from 1 (delta = 0: softplus of -200) to 0 (delta A below the range of fp32)."""
    v, dy, dlast = _inputs(1, 2, 40, 16, 8, 1, "f32")
    v["dt_bias"] = None
    v["dt"] = torch.linspace(-200, 60, 40)[None, :, None].expand(2, 40, 16).contiguous()
    v["A"][:, 3], v["A"][:, 4] = -30.0, 0.0
    n = _scan_all(v, dy, dlast)
    leaves = {k: leaf(t) for k, t in v.items()}
    yo, lo = oracle.lpv_scan(*[leaves[k] for k in NAMES[:8]], start=leaves["start"])
    named = {k: t for k, t in leaves.items() if t is not None}
    want = dict(zip(named, torch.autograd.grad([yo, lo], list(named.values()), [f64(dy), f64(dlast)])))
    m = _magnitudes(v, dy, dlast, True, None)
    # |raw| up to 200: where delta is not tiny (raw > -17) the 21 roundings become 40, below that delta is under 4e-8 of the largest
    r = 71 + 8 + 3 * 40
    # the exponential gives zero for results below 2^-126: delta and the decays are off by up to that, times values whose
    # magnitudes add up to less than 2^20 (adjoints and states below 2^10, samples below 2^3, 16 channels, 40 steps, 2 sequences)
    floor = 2.0 ** (-126 + 10 + 3 + 4 + 6 + 1)
    assert_close(n["y"], yo, r, m["y"], "y", floor)
    for k in ("u", "A", "B", "C", "z", "D", "start"):
        assert_close(n["d" + k], want[k], 2 * r + 120, m[k], "d" + k, floor)
    assert all(torch.isfinite(t).all() for t in n.values() if t is not None)


@pytest.mark.parametrize("nb,steps,d", [(2, 70, 8), (2, 1100, 24), (8, 500, 2048)])
def test_growing_modes_at_rest(nb, steps, d):
    """Modes that grow by e^10 a step, past any number within a part of the time axis: a state or an adjoint of zero stays zero."""
    v, dy, dlast = _inputs(3, nb, steps, d, 4, 1, "f32", gate=False, bias=False, start=False)
    v["A"] = torch.full((d, 4), 10.0)
    v["dt"] = torch.full_like(v["dt"], 1.0)
    late = {k: None if t is None else t.clone() for k, t in v.items()}
    late["u"][:, :-3] = 0
    y, last, _ = nmpc_amd.lpv_scan_fwd(*[gpu(late[k]) for k in NAMES[:8]], False)
    want, state = oracle.lpv_scan(*[None if late[k] is None else f64(late[k][:, -3:] if k in ("u", "dt", "B", "C") else late[k]) for k in NAMES[:8]], use_softplus=False)
    assert not y[:, :-3].any()
    m = _magnitudes({k: None if t is None else t[:, -3:] if k in ("u", "dt", "B", "C") else t for k, t in late.items()}, dy[:, -3:], dlast, False, None)
    # the exponent 10 log2(e) is rounded once and meant to a rounding: 2 x 10 a step, three steps; else as above
    assert_close(y[:, -3:], want, 52 + 4 + 9 + 60, m["y"], "y")
    assert_close(last, state, 52 + 4 + 9 + 60, m["last"], "last")
    # the adjoint: gradients of the first steps' outputs only, nothing behind them
    v["u"] = torch.zeros_like(v["u"])
    y, last, saved = nmpc_amd.lpv_scan_fwd(*[gpu(v[k]) for k in NAMES[:8]], False)
    assert not y.any() and not last.any()
    dy[:, 3:] = 0
    got = nmpc_amd.lpv_scan_bwd(saved, gpu(dy))
    assert all(torch.isfinite(t).all() for t in got.values() if t is not None)
    assert not got["du"][:, 3:].any() and not got["dC"].any() and not got["dA"].any()
    few = {k: None if t is None else leaf(t[:, :3] if k in ("u", "dt", "B", "C") else t) for k, t in v.items()}
    yo, _ = oracle.lpv_scan(*[few[k] for k in NAMES[:8]], use_softplus=False)
    du, = torch.autograd.grad([yo], [few["u"]], [f64(dy[:, :3])])
    m = _magnitudes({k: None if t is None else t[:, :3] if k in ("u", "dt", "B", "C") else t for k, t in v.items()}, dy[:, :3], torch.zeros_like(dlast), False, None)
    assert_close(got["du"][:, :3], du, 2 * (52 + 4 + 9 + 60) + 120, m["u"], "du")


def _scan_all(v, dy, dlast, lengths=None):
    y, last, saved = nmpc_amd.lpv_scan_fwd(*[gpu(v[k]) for k in NAMES[:8]], True, gpu(v["start"]), gpu(lengths))
    return {"y": y, "last": last, **nmpc_amd.lpv_scan_bwd(saved, gpu(dy), gpu(dlast))}


@pytest.mark.parametrize("steps", [50, 400])
def test_padding_is_never_read(steps):
    v, dy, dlast = _inputs(8, 3, steps, 12, 16, 2, "f32")
    n = torch.tensor([0, 7, steps - 1], dtype=torch.int32)
    clean = _scan_all(v, dy, dlast, n)
    for i, k in enumerate(n.tolist()):
        for name in ("u", "dt", "B", "C", "z"):
            v[name][i, k:] = float("nan")
        dy[i, k:] = float("inf")
    dirty = _scan_all(v, dy, dlast, n)
    for k in clean:
        if clean[k] is not None:
            assert torch.equal(clean[k], dirty[k]), k
    for i, k in enumerate(n.tolist()):
        for name in ("y", "du", "ddt", "dB", "dC", "dz"):
            assert not dirty[name][i, k:].any(), name
    assert torch.equal(dirty["last"][0].cpu(), v["start"][0]) and torch.equal(dirty["dstart"][0].cpu(), dlast[0])


def test_no_steps():
    v, dy, dlast = _inputs(8, 2, 0, 12, 16, 2, "bf16")
    out = _scan_all(v, dy, dlast)
    assert out["y"].shape == (2, 0, 12) and torch.equal(out["last"].cpu(), v["start"]) and torch.equal(out["dstart"].cpu(), dlast)
    assert not out["dA"].any() and not out["dD"].any() and not out["ddt_bias"].any()


def test_no_sequences():
    v, dy, dlast = _inputs(8, 0, 7, 12, 16, 2, "bf16")
    out = _scan_all(v, dy, dlast)
    assert out["y"].shape == (0, 7, 12) and out["last"].shape == (0, 12, 16) and out["dB"].shape == (0, 7, 2, 16)
    assert not out["dA"].any() and not out["dD"].any() and not out["ddt_bias"].any()


def test_single_step_of_a_far_stride():
    """The stride between steps of a single step means nothing, however large; one that would be used and does not fit is refused."""
    v, dy, dlast = _inputs(8, 2, 1, 8, 4, 1, "f32")
    want = _scan_all(v, dy, dlast)
    far = {k: gpu(t) if t is None or k not in ("u", "dt", "z") else t.cuda().as_strided(t.shape, (8, 1 << 30, 1)) for k, t in v.items()}
    got = _scan_all(far, dy, dlast)
    assert all(torch.equal(want[k], got[k]) for k in want)
    u = torch.zeros(1, device="cuda").as_strided((1, 2, 8), (0, 0, 0))
    far = torch.empty((1 << 24) + 16, device="cuda").as_strided((1, 2, 8), (0, (1 << 24) + 1, 1))
    B = torch.zeros(1, 2, 1, 4, device="cuda")
    with pytest.raises(nmpc_amd.NmpcError, match="strides"):
        nmpc_amd.lpv_scan(far, u, torch.zeros(8, 4, device="cuda"), B, B)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_parts_of_wider_tensors(dtype):
    g = rng(3)
    wide = normal(g, 2, 40, 3 * 72 + 1, dtype=DTYPES[dtype]).cuda()
    bc = normal(g, 2, 40, 1 + 2 * 2 * 8, dtype=DTYPES[dtype]).cuda()
    v, dy, dlast = _inputs(3, 2, 40, 72, 8, 2, dtype)
    v = {k: gpu(t) for k, t in v.items()}
    for lo in (0, 1):
        p = dict(v, u=wide[..., lo:lo + 72], z=wide[..., 72 + lo:144 + lo], dt=wide[..., 144 + lo:216 + lo],
                 B=bc[..., lo:lo + 16].unflatten(-1, (2, 8)), C=bc[..., 16 + lo:32 + lo].unflatten(-1, (2, 8)))
        want = _scan_all({k: None if t is None else t.contiguous() for k, t in p.items()}, dy, dlast)
        got = _scan_all(p, dy, dlast)
        for k in want:
            assert torch.equal(want[k], got[k]), (lo, k)
        flipped = dict(p, B=p["B"].transpose(-1, -2).contiguous().transpose(-1, -2), u=p["u"].transpose(1, 2).contiguous().transpose(1, 2))
        assert torch.equal(_scan_all(flipped, dy, dlast)["y"], want["y"])


@pytest.mark.parametrize("dtype,d,n,groups", [("bf16", 64, 16, 1), ("f32", 37, 5, 1), ("f16", 12, 64, 4)])
def test_steps_continue_a_prompt(dtype, d, n, groups):
    v, _, _ = _inputs(21, 3, 40, d, n, groups, dtype)
    v = {k: gpu(t) for k, t in v.items()}
    whole, last = nmpc_amd.lpv_scan(*[v[k] for k in NAMES[:8]], start=v["start"], return_state=True)
    cut = {k: t[:, :25] if k in ("u", "dt", "B", "C", "z") else t for k, t in v.items()}
    y, state = nmpc_amd.lpv_scan(*[cut[k] for k in NAMES[:8]], start=v["start"], return_state=True)
    assert torch.equal(y, whole[:, :25])
    # the step's sums are the same fp32 operations up to contraction into fma: a few roundings of values of size 1 .. 10
    tol = 64 * 2.0 ** -24 * 10 + (0 if dtype == "f32" else torch.finfo(DTYPES[dtype]).eps)
    for t in range(25, 40):
        at = [v[k][:, t] if k in ("u", "dt", "B", "C", "z") else v[k] for k in NAMES[:8]]
        got = nmpc_amd.lpv_scan_step(state, *at)
        assert torch.all((got.float() - whole[:, t].float()).abs() <= tol * (1 + whole[:, t].float().abs()))
    assert torch.allclose(state, last, rtol=64 * 2.0 ** -24, atol=64 * 2.0 ** -24 * 10)


def test_gradient_against_differences():
    """A directional difference of the GPU's own fp32 forward pass, step 2^-7: truncation h^2 times third derivatives of
    order 10 and rounding 2^-24 / h of a loss of size ~ 50."""
    v, dy, dlast = _inputs(5, 2, 20, 6, 4, 1, "f32")
    got = _scan_all(v, dy, dlast)
    h = 2.0 ** -7
    for k in ("u", "A", "dt", "B", "C", "z"):
        dirn = normal(rng(77), *v[k].shape)
        dirn = dirn / dirn.norm()
        def loss(s):
            y, last, _ = nmpc_amd.lpv_scan_fwd(*[gpu(v[j] + s * dirn if j == k else v[j]) for j in NAMES[:8]], True, gpu(v["start"]))
            return float((f64(y) * f64(dy)).sum() + (f64(last) * f64(dlast)).sum())
        slope = (loss(h) - loss(-h)) / (2 * h)
        assert abs(slope - float((f64(got["d" + k]) * f64(dirn)).sum())) < 10 * h * h + 50 * 64 * 2.0 ** -24 / h, k


def test_autograd_is_the_pair_and_capture():
    v, dy, dlast = _inputs(6, 2, 300, 16, 8, 1, "f32")
    c = {k: gpu(t) for k, t in v.items()}
    leaves = {k: t.clone().requires_grad_() for k, t in c.items()}
    y, last = nmpc_amd.lpv_scan(*[leaves[k] for k in NAMES[:8]], start=leaves["start"], return_state=True)
    got = torch.autograd.grad([y, last], [leaves[k] for k in NAMES], [dy.cuda(), dlast.cuda()])
    want = _scan_all(v, dy, dlast)
    for k, t in zip(NAMES, got):
        assert torch.equal(t, want["d" + k]), k
    dyc, dlc = dy.cuda(), dlast.cuda()
    def step():
        y, last, saved = nmpc_amd.lpv_scan_fwd(*[c[k] for k in NAMES[:8]], True, c["start"])
        return [y, last] + list(nmpc_amd.lpv_scan_bwd(saved, dyc, dlc).values())
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(3):
        c["u"].copy_(torch.randn(c["u"].shape, generator=rng(k)))
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(outs, step()):
            assert torch.equal(a, e)


GROWTH_CASES = [  # nb, steps, d, bits a step, size of the states and of the adjoints
    (2, 40, 8, 8.6, 1e-30),           # the time axis in slots of 16 steps, the gradient whole
    (1, 600, 8, 8.6, 1e-30),          # in parts of 32 steps, both passes
    (2, 1100, 24, 8.6, 1e-30),
    (120, 40, 1000, 8.6, 1e-30),      # whole sequences
    (2, 40, 8, 15.2, 2.0 ** -126),    # growth past the square root of 2^253, from the smallest normal number
    (1, 600, 8, 15.2, 2.0 ** -126),
]


@pytest.mark.parametrize("nb,steps,d,bits,size", GROWTH_CASES)
def test_growing_modes_of_small_states(nb, steps, d, bits, size):
    """Sixteen steps multiply a state, and the adjoint of one, by 2^138 or 2^243: more than a number of fp32 holds, on states so small that
    the results are ordinary numbers.  The steps around them leave a state as it is, so that later parts see what earlier ones did."""
    v, dy, dlast = _inputs(steps, nb, steps, d, 4, 1, "f32", skip=False, gate=False, bias=False)
    growth = bits * 0.6931471805599453
    v["A"] = growth * torch.tensor([1.0, 0.5, -0.01, -1.0]).expand(d, 4).contiguous()
    v["dt"] = torch.zeros_like(v["dt"])
    v["dt"][:, 16:32] = 1.0
    # signs and powers of two: whole parts of the range are left for the growth
    v["start"] = torch.sign(v["start"]) * size
    v["u"], dy, dlast = torch.zeros_like(v["u"]), torch.zeros_like(dy), torch.sign(dlast) * size
    want_y, want_last = oracle.lpv_scan(*[f64(v[k]) for k in NAMES[:8]], use_softplus=False, start=f64(v["start"]))
    y, last, saved = nmpc_amd.lpv_scan_fwd(*[gpu(v[k]) for k in NAMES[:8]], False, gpu(v["start"]))
    m = _magnitudes(v, dy, dlast, False, None)
    # the exponent of a step is rounded twice (A log2 e, its product with delta), of a part likewise: 2 roundings a unit of the
    # exponent of all sixteen steps; two more a step (exponential, product), three factors of two roundings where parts are joined
    r = 52 + 4 + 2 * 16 * growth + 2 * 16 + 6 * 3
    tiny = 2.0 ** -126                 # decaying states may round to multiples of 2^-149, or to zero
    assert_close(last, want_last, r, m["last"], "last", tiny)
    assert_close(y, want_y, r, m["y"], "y", 8 * tiny)
    got = nmpc_amd.lpv_scan_bwd(saved, gpu(dy), gpu(dlast))
    # the adjoint of the state before the first step: the same factors from behind
    decay = torch.exp(16 * f64(v["A"]))[None]
    assert_close(got["dstart"], decay * f64(dlast), r, decay * f64(dlast).abs(), "dstart", tiny)
    # as stepwise: what leaves the range of fp32 does so in every plan
    v["A"][:, 0] = 40.0
    over = nmpc_amd.lpv_scan_fwd(*[gpu(v[k]) for k in NAMES[:8]], False, gpu(v["start"]))[1]
    assert torch.isinf(over[..., 0]).all() and torch.equal(torch.sign(over[..., 0]).cpu(), torch.sign(v["start"][..., 0]))
