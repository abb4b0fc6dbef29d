"""The sequence operators together, as the layers of a learned model of a plant would use them: a causal filter of the samples,
the LPV scan with step sizes and B, C computed from the filtered samples, gated feed-forward projections; as a training step
against the definitions in fp64, and streamed sample by sample behind a prompt."""
import pytest
import torch

import nmpc_amd
from oracle import seq as oracle
from seq_util import f64, normal, rng

pytestmark = pytest.mark.gpu
D, N, G, F, TAPS = 32, 8, 2, 48, 4


def _weights(seed, dtype=torch.float32):
    g = rng(seed)
    w = dict(win=normal(g, 2 * D, D, scale=D ** -0.5), conv_w=normal(g, D, TAPS, scale=0.5), conv_b=normal(g, D, scale=0.1),
             wdt=normal(g, D, D, scale=0.3 * D ** -0.5), dt_bias=-3 + normal(g, D, scale=0.5), wbc=normal(g, 2 * G * N, D, scale=D ** -0.5),
             A=-torch.rand(D, N, generator=g) * N - 0.1, skip=normal(g, D), wg=normal(g, F, D, scale=D ** -0.5), wu=normal(g, F, D, scale=D ** -0.5),
             wout=normal(g, D, F, scale=F ** -0.5))
    fp32 = ("conv_w", "conv_b", "dt_bias", "A", "skip")
    return {k: v if k in fp32 else v.to(dtype) for k, v in w.items()}


def _layer(x, w, ops, lengths=None):
    """x [batch, steps, D] -> [batch, steps, D]"""
    conv, scan, ffn = ops
    u, z = (x @ w["win"].T).split(D, -1)
    u = conv(u, w["conv_w"], w["conv_b"], "silu", lengths)
    B, C = (u @ w["wbc"].T).unflatten(-1, (2 * G, N)).split(G, -2)
    y = scan(u, u @ w["wdt"].T, w["A"], B, C, w["skip"], z, w["dt_bias"], lengths)
    return x + ffn(y, w["wg"], w["wu"], "silu") @ w["wout"].T


OWN = (lambda u, w, b, a, n: nmpc_amd.causal_conv(u, w, b, a, lengths=n),
       lambda u, dt, A, B, C, s, z, b, n: nmpc_amd.lpv_scan(u, dt, A, B, C, s, z, b, lengths=n), nmpc_amd.gated_ffn)
ORACLE = (lambda u, w, b, a, n: oracle.causal_conv(u, w, b, a, lengths=n)[0],
          lambda u, dt, A, B, C, s, z, b, n: oracle.lpv_scan(u, dt, A, B, C, s, z, b, lengths=n)[0], oracle.gated_ffn)


@pytest.mark.parametrize("steps,lengths", [(45, None), (40, [40, 0, 23])])
def test_training_step_of_two_layers(steps, lengths):
    """Two layers, forward and backward through autograd.  Every product and operator is within 52 + N + 3 L + 2 D + 2 F < 500 fp32
    roundings of its terms, ten of them follow one another in each direction, and slopes and norms amplify by less than 16: 80000
    roundings, 5e-3 of a gradient's norm, at the very most; half of that is asked for."""
    w = [_weights(3), _weights(4)]
    x, dy = normal(rng(5), 3, steps, D), normal(rng(6), 3, steps, D)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)

    def run(ops, move, n):
        leaves = [move(x)] + [move(t) for layer in w for t in layer.values()]
        ws = [dict(zip(w[0], leaves[1 + i * len(w[0]):])) for i in range(2)]
        y = leaves[0]
        for layer in ws:
            y = _layer(y, layer, ops, n)
        return [y] + list(torch.autograd.grad(y, leaves, move(dy).detach()))
    want = run(ORACLE, lambda t: t.double().requires_grad_(), n)
    got = run(OWN, lambda t: t.cuda().requires_grad_(), None if n is None else n.cuda())
    for a, b in zip(got, want):
        assert (f64(a) - f64(b)).norm() <= 2.5e-3 * f64(b).norm() + 1e-30


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_streaming_behind_a_prompt(dtype):
    """The whole record at once, and a prompt followed by single samples: the same up to the order of a few sums (bf16: their
    roundings, half a step for each of the seven tensors that one layer rounds, with slopes below 4)."""
    w = {k: v.cuda() for k, v in _weights(8, dtype).items()}
    x = normal(rng(9), 2, 50, D, dtype=dtype).cuda()
    whole = _layer(x, w, OWN)
    cut = 37
    u, z = (x[:, :cut] @ w["win"].T).split(D, -1)
    u, window = nmpc_amd.causal_conv(u, w["conv_w"], w["conv_b"], "silu", return_state=True)
    B, C = (u @ w["wbc"].T).unflatten(-1, (2 * G, N)).split(G, -2)
    y, state = nmpc_amd.lpv_scan(u, u @ w["wdt"].T, w["A"], B, C, w["skip"], z, w["dt_bias"], return_state=True)
    out = [x[:, :cut] + nmpc_amd.gated_ffn(y, w["wg"], w["wu"]) @ w["wout"].T]
    for t in range(cut, 50):
        u, z = (x[:, t] @ w["win"].T).split(D, -1)
        u = nmpc_amd.causal_conv_step(window, u, w["conv_w"], w["conv_b"], "silu")
        B, C = (u @ w["wbc"].T).unflatten(-1, (2 * G, N)).split(G, -2)
        y = nmpc_amd.lpv_scan_step(state, u, u @ w["wdt"].T, w["A"], B, C, w["skip"], z, w["dt_bias"])
        out.append((x[:, t] + nmpc_amd.gated_ffn(y, w["wg"], w["wu"]) @ w["wout"].T)[:, None])
    got = torch.cat(out, 1)
    step = 500 * 2.0 ** -24 if dtype == torch.float32 else 7 * 4 * torch.finfo(dtype).eps / 2
    assert ((got.double() - whole.double()).norm() <= step * whole.double().norm())


def test_padded_batch_is_its_sequences():
    """A padded batch gives what its sequences give one by one (other workgroups, chunks and tiles: the same up to sums' order)."""
    w = {k: v.cuda() for k, v in _weights(11).items()}
    n = [130, 1, 64, 0, 97]
    x = normal(rng(12), len(n), 130, D).cuda()
    got = _layer(x, w, OWN, torch.tensor(n, dtype=torch.int64, device="cuda"))
    for i, k in enumerate(n):
        one = _layer(x[i:i + 1, :k], w, OWN)
        assert (got[i:i + 1, :k] - one).norm() <= 1000 * 2.0 ** -24 * (one.norm() + 1)
