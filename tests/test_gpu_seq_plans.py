"""Every kernel that the rules of the scan and of the projections can choose, at sizes that are shown to choose it: the plan is asked
for first.  Definitions and bounds are those of test_gpu_seq_scan.py and test_gpu_seq_ffn.py."""
import ctypes

import pytest
import torch

import nmpc_amd
from nmpc_amd import _lib
from oracle import seq as oracle
from seq_util import U32, assert_close, f64, gpu, leaf
from test_gpu_seq_ffn import DTYPES, _bounds, _run
from test_gpu_seq_ffn import _inputs as _ffn_inputs
from test_gpu_seq_scan import NAMES, _check, _magnitudes
from test_gpu_seq_scan import _inputs as _scan_inputs

pytestmark = pytest.mark.gpu


def _plan(dtype, m, k, f, product):
    """(tile rows, tile columns, parts of the contraction) of contiguous operands; columns 32: the kernel for few rows."""
    shape = (ctypes.c_int * 3)()
    size = 4 if dtype == "f32" else 2
    code = {"f32": 0, "bf16": 1, "f16": 2}[dtype]
    assert _lib.lib().nmpc_gated_ffn_plan(code, m, k, f, product, int(k * size % 16 != 0), ctypes.addressof(shape)) == 0
    return tuple(shape)


FFN = [  # rows, inputs, hidden units, dtype, activation, tile sides of the three products, is the contraction of dx, dW split?
    (65, 72, 72, "bf16", "silu", 32, 64, 128, False, False),
    (65, 72, 136, "f32", "gelu", 32, 64, 128, True, False),
    (65, 520, 6000, "bf16", "gelu", 64, 64, 128, True, False),
    (65, 264, 8200, "f16", "silu", 128, 64, 128, True, False),
    (65, 2056, 2056, "f32", "silu", 32, 128, 256, True, False),
    (65, 2056, 2056, "f16", "silu", 32, 64, 256, True, False),
    (300, 72, 8200, "f32", "sigmoid", 64, 64, 128, True, False),
    (200, 136, 6000, "f32", "silu", 128, 128, 128, True, False),
    (513, 4100, 72, "bf16", "silu", 32, 128, 128, False, False),
    (513, 136, 8200, "f32", "tanh", 64, 128, 256, True, True),
    (700, 72, 6000, "bf16", "silu", 256, 64, 128, True, False),
    (703, 77, 6001, "f16", "tanh", 256, 64, 128, True, False),              # nothing aligned
    (1030, 72, 72, "f16", "silu", 32, 64, 128, False, True),
    (1500, 72, 4104, "f32", "silu", 256, 128, 128, True, True),
    (1501, 75, 4103, "f32", "gelu", 256, 128, 128, True, True),
    (2050, 4100, 72, "bf16", "silu", 32, 256, 128, False, True),
    (2500, 136, 8200, "bf16", "sigmoid", 256, 128, 256, True, True),
    (2501, 133, 8197, "f16", "silu", 256, 128, 256, True, True),
    (3100, 4100, 72, "f32", "silu", 32, 256, 128, False, True),
    (4100, 136, 2056, "f32", "gelu", 64, 256, 256, True, True),
    (4100, 1032, 4104, "bf16", "silu", 256, 256, 256, True, False),
    (4100, 1032, 4101, "f16", "gelu", 256, 256, 256, True, False),
    (4100, 1000, 4104, "f32", "silu", 64, 256, 256, True, True),
]


@pytest.mark.parametrize("m,k,f,dtype,name,fwd,dx,dw,dx_split,dw_split", FFN)
def test_projections(m, k, f, dtype, name, fwd, dx, dw, dx_split, dw_split):
    plans = [_plan(dtype, m, k, f, p) for p in range(3)]
    assert (plans[0][1] if fwd == 32 else plans[0][0], plans[1][0], plans[2][0]) == (fwd, dx, dw), plans
    assert (plans[1][2] > 1, plans[2][2] > 1) == (dx_split, dw_split), plans
    x, wg, wu, dh = (t.cuda() for t in _ffn_inputs(m, m, k, f, dtype))
    lx, lg, lu = (t.double().requires_grad_() for t in (x, wg, wu))
    ho = oracle.gated_ffn(lx, lg, lu, name)
    want = dict(zip(("dx", "dwg", "dwu"), torch.autograd.grad(ho, (lx, lg, lu), dh.double())), h=ho)
    got = _run(x, wg, wu, dh, name)
    bound = _bounds(x, wg, wu, dh, name)
    for key in ("h", "dx", "dwg", "dwu"):
        assert got[key].dtype is DTYPES[dtype]
        assert_close(got[key], want[key], 1 / U32, bound[key].cpu(), key)
    assert torch.equal(nmpc_amd.gated_ffn(x, wg, wu, name), got["h"])


def _scan_plan(nb, steps, d, n, groups, backward):
    return _lib.lib().nmpc_lpv_scan_plan(nb, steps, d, n, groups, backward)


@pytest.mark.parametrize("n", [3, 8, 16, 17, 24, 32, 33, 49, 64])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scan_in_parts(n, dtype):
    """The time axis in parts, forward and backward, for every number of lanes a channel."""
    nb, steps, d, groups = 2, 400, 10, 2
    assert all(_scan_plan(nb, steps, d, n, groups, b) > 1 for b in (0, 1))
    v, dy, dlast = _scan_inputs(n, nb, steps, d, n, groups, dtype)
    _check(v, dy, dlast, True, [steps, steps - 37])


@pytest.mark.parametrize("steps,n", [(4000, 16), (4017, 5)])
def test_scan_in_parts_of_several_tiles(steps, n):
    """Few channels over many steps: parts of more than one tile, so that the join of them stays short."""
    assert all(1 < _scan_plan(1, steps, 6, n, 1, b) < (steps + 31) // 32 for b in (0, 1))
    v, dy, dlast = _scan_inputs(n, 1, steps, 6, n, 1, "f32")
    _check(v, dy, dlast, True, [steps - 5])


@pytest.mark.parametrize("n", [3, 8, 16, 24, 64])
def test_scan_in_slots(n):
    nb, steps, d, groups = 2, 70, 10, 2
    assert _scan_plan(nb, steps, d, n, groups, 0) == 0
    v, dy, dlast = _scan_inputs(n, nb, steps, d, n, groups, "f32")
    _check(v, dy, dlast, True, [steps, steps - 37])


@pytest.mark.parametrize("n", [4, 8, 16, 24, 49])
@pytest.mark.parametrize("dtype,d", [("f32", 1000), ("bf16", 1002)])
def test_scan_whole(n, dtype, d):
    """Whole sequences, with states before them and gradients.  The gradients of three sequences and sixteen channels count, those of the
    others are zero: all sums then run over these alone, which the definition can be evaluated for."""
    nb, steps, groups = 120, 40, 2
    assert all(_scan_plan(nb, steps, d, n, groups, b) == 1 for b in (0, 1))
    v, dy, dlast = _scan_inputs(n, nb, steps, d, n, groups, dtype)
    lengths = torch.tensor([steps - i % (steps + 1) for i in range(nb)], dtype=torch.int32)
    seqs = torch.tensor([0, 17, 101])                                         # 40, 23 and 21 steps
    half = d // 2
    chans = torch.tensor([0, 1, 63, 64, 130, 255, 256, half - 1] + [half, half + 1, half + 31, half + 64, half + 129, half + 300, d - 2, d - 1])
    keep = torch.zeros(nb, d)
    keep[seqs[:, None], chans[None]] = 1
    dy, dlast = (dy * keep[:, None]).to(dy.dtype), dlast * keep[..., None]
    y, last, saved = nmpc_amd.lpv_scan_fwd(*[gpu(v[k]) for k in NAMES[:8]], True, gpu(v["start"]), gpu(lengths))
    got = nmpc_amd.lpv_scan_bwd(saved, gpu(dy), gpu(dlast))
    few = {k: t[seqs] if k in ("B", "C") else t[chans] if k in ("A", "D", "dt_bias") else t[seqs][..., chans, :] if k == "start" else t[seqs][..., chans]
           for k, t in v.items()}
    fdy, fdlast, ends = dy[seqs][..., chans], dlast[seqs][:, chans], lengths[seqs]
    leaves = {k: leaf(t) for k, t in few.items()}
    yo, lo = oracle.lpv_scan(*[leaves[k] for k in NAMES[:8]], start=leaves["start"], lengths=ends)
    m = _magnitudes(few, fdy, fdlast, True, ends)
    r = 52 + n + 3 * steps
    s, c = seqs.cuda(), chans.cuda()
    assert_close(y[s][..., c], yo, r, m["y"], "y")
    assert_close(last[s][:, c], lo, r, m["last"], "last")
    want = dict(zip(NAMES, torch.autograd.grad([yo, lo], [leaves[k] for k in NAMES], [f64(fdy), f64(fdlast)])))
    for k in NAMES:
        g = got["d" + k]
        if k in ("A", "D", "dt_bias"):
            rest = torch.ones(d, dtype=torch.bool)
            rest[chans] = False
            assert not g[rest.cuda()].any(), k
            g = g[c]
        else:
            rest = torch.ones(nb, dtype=torch.bool)
            rest[seqs] = False
            assert not g[rest.cuda()].any(), k
            g = g[s] if k in ("B", "C") else g[s][:, c] if k == "start" else g[s][..., c]
        assert_close(g, want[k], 2 * r + 20 + nb * steps + d, m[k], "d" + k)
