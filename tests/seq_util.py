"""Helpers of the sequence-operator tests: seeded inputs and bounds that count roundings."""
import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24                       # half a step of fp32


def rng(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(g, *shape, scale=1.0, dtype=torch.float32):
    """Values that the type holds exactly, so that both sides start from the same numbers."""
    return (scale * torch.randn(*shape, generator=g)).to(dtype)


def f64(t):
    return None if t is None else t.detach().cpu().double()


def gpu(t):
    return None if t is None else t.cuda()


def leaf(t):
    return None if t is None else t.detach().cpu().double().requires_grad_()


def assert_close(got, want, roundings, scale, name, floor=0.0):
    """|got - want| <= half a step of got's type (one rounding at the end) + `roundings` roundings to fp32 of terms whose
    magnitudes add up to `scale` (a tensor or number), plus `floor` where values leave fp32's normal range."""
    half = torch.finfo(got.dtype).eps / 2
    got64, want = f64(got), f64(want)
    assert got64.shape == want.shape, (name, got64.shape, want.shape)
    slack = roundings * U32 * (scale if torch.is_tensor(scale) else torch.tensor(float(scale), dtype=torch.float64))
    smallest = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    # the final rounding acts on the fp32 value, which is off by the slack itself
    tol = half * (want.abs() + slack) + slack + smallest + floor
    off = (got64 - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), "%s: %d of %d outside; worst %.3g times its bound (got %r, want %r)" % (
        name, int(bad.sum()), off.numel(), float((off / tol).nan_to_num(nan=float("inf")).max()), got64[bad][:3].tolist(), want.expand_as(got64)[bad][:3].tolist())
