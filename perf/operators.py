"""The sequence-model operators that are measured: causal convolution, selective state-space scan (diagonal LPV
recurrence) and gated feed-forward projections - each for whole sequences, for training and for single tokens.

`run` computes a case in plain torch operations (own = False) or through the public entry points of nmpc_amd
(own = True).  Symbols: b sequences, t steps, d channels, n states per channel, g groups of channels that share B and C,
w convolution taps, m rows (tokens), k inputs, f hidden units."""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new sample for each of 64 running sequences: launch latency
        dict(name="conv_token", op="conv", mode="token", dtype="bfloat16", b=64, t=1, d=4096, w=4, act="silu", ragged=False, start=True),
        # prompts of unequal length in one padded batch, odd sizes, continued from an earlier window
        dict(name="conv_prompt_ragged", op="conv", mode="prompt", dtype="float16", b=6, t=1537, d=1500, w=3, act="silu", ragged=True, start=True),
        # a training step over whole sequences
        dict(name="conv_train", op="conv", mode="train", dtype="bfloat16", b=4, t=2048, d=4096, w=4, act="silu", ragged=False, start=False),
        # one new sample for each of 64 running sequences: the states are read and written once
        dict(name="scan_token", op="scan", mode="token", dtype="bfloat16", b=64, t=1, d=4096, n=16, g=1, gate=True, ragged=False, start=True),
        # one long prompt: few channels in flight, many steps
        dict(name="scan_prompt_long", op="scan", mode="prompt", dtype="bfloat16", b=1, t=8192, d=2048, n=16, g=1, gate=True, ragged=False, start=False),
        # prompts of unequal length, odd sizes, several groups, continued from earlier states
        dict(name="scan_prompt_ragged", op="scan", mode="prompt", dtype="float16", b=5, t=1111, d=1000, n=24, g=4, gate=False, ragged=True, start=True),
        # a training step over whole sequences
        dict(name="scan_train", op="scan", mode="train", dtype="bfloat16", b=4, t=2048, d=2048, n=16, g=1, gate=True, ragged=False, start=False),
        # a training step over short fp32 records, horizon-50 control runs of 64 channels
        dict(name="scan_train_records", op="scan", mode="train", dtype="float32", b=64, t=50, d=64, n=8, g=1, gate=False, ragged=False, start=True),
        # one token: the two weight matrices are read once
        dict(name="ffn_token", op="ffn", mode="token", dtype="bfloat16", m=1, k=2048, f=8192, act="silu"),
        # a short prompt, odd sizes
        dict(name="ffn_prompt_odd", op="ffn", mode="prompt", dtype="float16", m=333, k=1001, f=2731, act="gelu"),
        # a training step in fp32 on the rows of 4096 controllers
        dict(name="ffn_train_f32", op="ffn", mode="train", dtype="float32", m=4096, k=256, f=1024, act="tanh"),
        # a training step: six matrix products
        dict(name="ffn_train", op="ffn", mode="train", dtype="bfloat16", m=4096, k=2048, f=8192, act="silu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "ffn", "ffn"])
    mode = rng.choice(["token", "prompt", "train"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    odd = rng.random() < 0.4
    if op == "ffn":
        m = _log(rng, 1, 16) if mode == "token" else _log(rng, 17, 4096)
        k, f = _log(rng, 64, 2048), _log(rng, 64, 8192)
        if not odd:
            k, f = max(64, k // 64 * 64), max(64, f // 64 * 64)
        return dict(op=op, mode=mode, dtype=dtype, m=m, k=k, f=f, act=rng.choice(["silu", "gelu", "tanh", "sigmoid"]))
    b, d = _log(rng, 1, 64), _log(rng, 64, 4096)
    if not odd:
        d = max(64, d // 64 * 64)
    if op == "conv":
        t = 1 if mode == "token" else _log(rng, 1, max(1, min(8192, 4 * 2048 * 4096 // (b * d))))
        return dict(op=op, mode=mode, dtype=dtype, b=b, t=t, d=d, w=rng.choice([2, 3, 4, 4, 5, 8]), act=rng.choice(["silu", "none"]),
                    ragged=mode != "token" and rng.random() < 0.3, start=mode == "token" or rng.random() < 0.5)
    n = rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 64)])
    g = rng.choice([1, 1, 2, 4])
    d = max(g, d // g * g)
    t = 1 if mode == "token" else _log(rng, 1, max(1, min(8192, 4 * 2048 * 2048 * 16 // (b * d * n))))
    return dict(op=op, mode=mode, dtype=dtype, b=b, t=t, d=d, n=n, g=g, gate=rng.random() < 0.5,
                ragged=mode != "token" and rng.random() < 0.3, start=mode == "token" or rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c, dt = dict(case), DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 1000003 + 17)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda").mul_(scale).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    s = {"case": c}
    if c["op"] == "ffn":
        s["x"] = normal(c["m"], c["k"], dtype=dt)
        s["wg"] = normal(c["f"], c["k"], scale=c["k"] ** -0.5, dtype=dt)
        s["wu"] = normal(c["f"], c["k"], scale=c["k"] ** -0.5, dtype=dt)
        if c["mode"] == "train":
            s["dh"] = normal(c["m"], c["f"], dtype=dt)
        return s
    b, t, d = c["b"], c["t"], c["d"]
    s["lengths"] = None
    if c["ragged"]:
        s["lengths"] = torch.randint(0, t + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
    # u and the gate are the two halves of one projection's output, as B and C are
    both = normal(b, t, 2 * d, dtype=dt)
    s["u"] = both[..., :d] if t > 1 else both[..., :d].contiguous()
    if c["op"] == "conv":
        w = c["w"]
        s["w"], s["bias"] = normal(d, w, scale=w ** -0.5), normal(d, scale=0.1)
        s["start"] = normal(b, w - 1, d, dtype=dt) if c["start"] else None
    else:
        n, g = c["n"], c["g"]
        s["z"] = both[..., d:] if c["gate"] else None
        s["dt"] = normal(b, t, d, scale=0.5, dtype=dt)
        step = torch.exp(uniform(d) * math.log(100.0) + math.log(1e-3))       # step sizes of 1e-3 .. 1e-1
        s["dt_bias"] = torch.log(torch.expm1(step))
        s["A"] = -(torch.arange(1, n + 1, device="cuda", dtype=torch.float32) * torch.exp(0.2 * normal(d, n)))
        bc = normal(b, t, 2 * g * n, dtype=dt)
        s["B"], s["C"] = bc[..., :g * n].unflatten(-1, (g, n)), bc[..., g * n:].unflatten(-1, (g, n))
        s["D"] = 1.0 + 0.1 * normal(d)
        s["start"] = normal(b, d, n, scale=0.5) if c["start"] else None
    if c["mode"] == "token":
        for name in ("u", "z", "dt", "B", "C"):
            if s.get(name) is not None:
                s[name] = s[name][:, 0]
    if c["mode"] == "train":
        s["dy"] = normal(b, t, d, dtype=dt)
        s["dlast"] = normal(*(s["start"].shape if c["start"] else (b, c["w"] - 1, d) if c["op"] == "conv" else (b, d, c["n"])),
                            dtype=dt if c["op"] == "conv" else torch.float32)
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _f(x):
    return None if x is None else x.float()


def _act(x, act):
    """The activation and its derivative."""
    if act == "none":
        return x, torch.ones_like(x)
    if act == "tanh":
        y = torch.tanh(x)
        return y, 1 - y * y
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
        return x * p, p + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))
    p = torch.sigmoid(x)
    return (p, p * (1 - p)) if act == "sigmoid" else (x * p, p * (1 + x * (1 - p)))


def _inside(s, b, t):
    """[b, t, 1]: the steps that belong to their sequence; None where all do."""
    if s["lengths"] is None:
        return None
    return (torch.arange(t, device="cuda")[None] < s["lengths"][:, None])[..., None]


def _only(x, inside):
    return x if inside is None or x is None else torch.where(inside.reshape(inside.shape + (1,) * (x.dim() - 3)), x, torch.zeros_like(x))


def _plain_conv(s):
    c, dt = s["case"], s["u"].dtype
    w, bias = s["w"], s["bias"]
    taps = w.shape[1]
    if c["mode"] == "token":
        full = torch.cat([s["start"], s["u"][:, None]], 1)
        s["start"].copy_(full[:, 1:])
        y = _act((_f(full) * w.T[None]).sum(1) + bias, c["act"])[0]
        return {"y": y.to(dt), "window": s["start"]}
    b, t, d = s["u"].shape
    inside = _inside(s, b, t)
    start = s["start"] if s["start"] is not None else s["u"].new_zeros(b, taps - 1, d)
    full = torch.cat([start, _only(s["u"], inside)], 1)
    seen = _f(full).unfold(1, taps, 1)                                         # [b, t, d, w]
    pre = (seen * w).sum(-1) + bias
    y, slope = _act(pre, c["act"])
    ends = s["lengths"].long() if s["lengths"] is not None else torch.full((b,), t, device="cuda")
    at = (ends[:, None] + torch.arange(taps - 1, device="cuda"))[..., None].expand(-1, -1, d)
    out = {"y": _only(y, inside).to(dt), "window": full.gather(1, at)}
    if c["mode"] == "prompt":
        return out
    dpre = _only(_f(s["dy"]) * slope, inside)
    out["dw"], out["dbias"] = torch.stack([(seen[..., j] * dpre).sum((0, 1)) for j in range(taps)], 1), dpre.sum((0, 1))
    ahead = torch.cat([dpre.new_zeros(b, taps - 1, d), dpre, dpre.new_zeros(b, taps - 1, d)], 1)
    dfull = (ahead.unfold(1, taps, 1) * w.flip(1)).sum(-1).scatter_add(1, at, _f(s["dlast"]))
    out["du"] = _only(dfull[:, taps - 1:], inside).to(dt)
    if s["start"] is not None:
        out["dstart"] = dfull[:, :taps - 1].to(dt)
    return out


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20))))


def _prefix(decay, x):
    """x[:, t] + decay[:, t] * (the same of t - 1), for all t by doubling."""
    step = 1
    while step < x.shape[1]:
        x = torch.cat([x[:, :step], x[:, step:] + decay[:, step:] * x[:, :-step]], 1)
        decay = torch.cat([decay[:, :step], decay[:, step:] * decay[:, :-step]], 1)
        step *= 2
    return x


def _plain_scan(s):
    c, out_type = s["case"], s["u"].dtype
    A, D = s["A"], s["D"]
    per = c["d"] // c["g"]
    u, z = _f(s["u"]), _f(s["z"])
    raw = _f(s["dt"]) + s["dt_bias"]
    if c["mode"] == "token":
        delta = _softplus(raw)
        B, C = _f(s["B"]).repeat_interleave(per, 1), _f(s["C"]).repeat_interleave(per, 1)
        s["start"].copy_(torch.exp(delta[..., None] * A) * s["start"] + (delta * u)[..., None] * B)
        y = (s["start"] * C).sum(-1) + D * u
        return {"y": (y if z is None else y * _act(z, "silu")[0]).to(out_type), "state": s["start"]}
    b, t, d = u.shape
    n = c["n"]
    inside = _inside(s, b, t)
    u, delta = _only(u, inside), _only(_softplus(raw), inside)
    B, C = _only(_f(s["B"]), inside).repeat_interleave(per, 2), _only(_f(s["C"]), inside).repeat_interleave(per, 2)
    start = s["start"] if s["start"] is not None else u.new_zeros(b, d, n)
    decay = torch.exp(delta[..., None] * A)
    x = (delta * u)[..., None] * B
    x[:, :1] += decay[:, :1] * start[:, None]
    x = _prefix(decay, x)                                                      # [b, t, d, n]
    y = (x * C).sum(-1) + D * u
    gate, slope = (None, None) if z is None else _act(z, "silu")
    out = {"y": _only(y if z is None else y * gate, inside).to(out_type), "state": x[:, -1]}
    if c["mode"] == "prompt":
        return out
    dy = _only(_f(s["dy"]), inside)
    if z is not None:
        out["dz"] = _only(dy * y * slope, inside).to(out_type)
        dy = dy * gate
        dy = _only(dy, inside)
    lam = dy[..., None] * C
    lam[:, -1] += s["dlast"]
    after = torch.cat([decay[:, 1:], torch.zeros_like(decay[:, :1])], 1)       # the adjoint runs backwards
    lam = _prefix(after.flip(1), lam.flip(1)).flip(1)
    moved = lam * decay * torch.cat([start[:, None], x[:, :-1]], 1)
    shared = (lam * B).sum(-1)
    ddelta = (moved * A).sum(-1) + u * shared
    draw_ = _only(ddelta * torch.sigmoid(raw), inside)
    out["du"] = _only(D * dy + delta * shared, inside).to(out_type)
    out["ddt"], out["ddt_bias"] = draw_.to(out_type), draw_.sum((0, 1))
    out["dA"], out["dD"] = (moved * delta[..., None]).sum((0, 1)), (dy * u).sum((0, 1))
    out["dB"] = (lam * (delta * u)[..., None]).unflatten(2, (c["g"], per)).sum(3).to(out_type)
    out["dC"] = (x * dy[..., None]).unflatten(2, (c["g"], per)).sum(3).to(out_type)
    if s["start"] is not None:
        out["dstart"] = lam[:, 0] * decay[:, 0]
    return out


def _plain_ffn(s):
    c, dt = s["case"], s["x"].dtype
    x, wg, wu = _f(s["x"]), _f(s["wg"]), _f(s["wu"])
    up = x @ wu.T
    a, slope = _act(x @ wg.T, c["act"])
    out = {"h": (a * up).to(dt)}
    if c["mode"] == "train":
        dh = _f(s["dh"])
        dg, du = dh * up * slope, dh * a
        out["dx"] = (dg @ wg + du @ wu).to(dt)
        out["dwg"], out["dwu"] = (dg.T @ x).to(dt), (du.T @ x).to(dt)
    return out


# ---------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    import nmpc_amd
    c = s["case"]
    if c["op"] == "ffn":
        if c["mode"] != "train":
            return {"h": nmpc_amd.gated_ffn(s["x"], s["wg"], s["wu"], c["act"])}
        h, saved = nmpc_amd.gated_ffn_fwd(s["x"], s["wg"], s["wu"], c["act"])
        dx, dwg, dwu = nmpc_amd.gated_ffn_bwd(saved, s["dh"])
        return {"h": h, "dx": dx, "dwg": dwg, "dwu": dwu}
    if c["op"] == "conv":
        act = None if c["act"] == "none" else c["act"]
        if c["mode"] == "token":
            return {"y": nmpc_amd.causal_conv_step(s["start"], s["u"], s["w"], s["bias"], act), "window": s["start"]}
        if c["mode"] == "prompt":
            y, window = nmpc_amd.causal_conv(s["u"], s["w"], s["bias"], act, start=s["start"], lengths=s["lengths"], return_state=True)
            return {"y": y, "window": window}
        y, window, saved = nmpc_amd.causal_conv_fwd(s["u"], s["w"], s["bias"], act, start=s["start"], lengths=s["lengths"])
        grads = nmpc_amd.causal_conv_bwd(saved, s["dy"], s["dlast"])
        return {"y": y, "window": window, **{k: v for k, v in grads.items() if v is not None}}
    args = dict(D=s["D"], z=s["z"], dt_bias=s["dt_bias"], softplus=True)
    if c["mode"] == "token":
        return {"y": nmpc_amd.lpv_scan_step(s["start"], s["u"], s["dt"], s["A"], s["B"], s["C"], **args), "state": s["start"]}
    args.update(start=s["start"], lengths=s["lengths"])
    if c["mode"] == "prompt":
        y, state = nmpc_amd.lpv_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], return_state=True, **args)
        return {"y": y, "state": state}
    y, state, saved = nmpc_amd.lpv_scan_fwd(s["u"], s["dt"], s["A"], s["B"], s["C"], **args)
    grads = nmpc_amd.lpv_scan_bwd(saved, s["dy"], s["dlast"])
    return {"y": y, "state": state, **{k: v for k, v in grads.items() if v is not None}}


def run(state):
    if own:
        return _own(state)
    return {"conv": _plain_conv, "scan": _plain_scan, "ffn": _plain_ffn}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------- floors
def work(case):
    c, e = case, 4 if case["dtype"] == "float32" else 2
    train = c["mode"] == "train"
    if c["op"] == "ffn":
        m, k, f = c["m"], c["k"], c["f"]
        once = m * k + 2 * f * k + m * f
        return {"bytes": e * (once + (m * f + m * k + 2 * f * k if train else 0)), "flops": (12 if train else 4) * m * k * f}
    seq = c["b"] * c["t"] * c["d"]
    if c["op"] == "conv":
        window = e * c["b"] * (c["w"] - 1) * c["d"]
        small = 4 * c["d"] * (c["w"] + 1)
        return {"bytes": e * seq * (4 if train else 2) + window * (2 if c["start"] else 1) * (2 if train else 1) + small * (2 if train else 1),
                "flops": seq * (2 * c["w"] + 4) * (3 if train else 1)}
    state = 4 * c["b"] * c["d"] * c["n"]
    shared = e * c["b"] * c["t"] * 2 * c["g"] * c["n"]
    streams = 4 if c["gate"] else 3
    small = 4 * c["d"] * (c["n"] + 2)
    fwd = e * seq * streams + shared + small + state * (2 if c["start"] else 1)
    bwd = e * seq * streams + shared + small + state * (2 if c["start"] else 1)    # dy, gradients out, the state's gradient
    return {"bytes": fwd + (bwd if train else 0), "flops": seq * c["n"] * (21 if train else 7)}


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """Step by step, in 64 bits."""
    c, s = dict(case), prepare(case, seed)
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    sig = lambda v: 1 / (1 + torch.exp(-v))                                     # noqa: E731
    phi = lambda v: torch.special.erfc(-v / math.sqrt(2.0)) / 2                 # noqa: E731
    value = {"silu": lambda v: v * sig(v), "gelu": lambda v: v * phi(v), "tanh": torch.tanh, "sigmoid": sig, "none": lambda v: v}
    slope = {"silu": lambda v: sig(v) + v * sig(v) * sig(-v), "gelu": lambda v: phi(v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi),
             "tanh": lambda v: 1 / torch.cosh(v) ** 2, "sigmoid": lambda v: sig(v) * sig(-v), "none": torch.ones_like}
    if c["op"] == "ffn":
        gate, up = s["x"].matmul(s["wg"].t()), s["x"].matmul(s["wu"].t())
        out = {"h": value[c["act"]](gate) * up}
        if c["mode"] == "train":
            dgate, dup = s["dh"] * up * slope[c["act"]](gate), s["dh"] * value[c["act"]](gate)
            out.update(dx=dgate.matmul(s["wg"]) + dup.matmul(s["wu"]), dwg=dgate.t().matmul(s["x"]), dwu=dup.t().matmul(s["x"]))
        return out
    if c["mode"] == "token":
        s["u"], s["lengths"] = s["u"][:, None], None
        for name in ("z", "dt", "B", "C"):
            if s.get(name) is not None:
                s[name] = s[name][:, None]
    b, t, d = s["u"].shape
    ends = s["lengths"].tolist() if s["lengths"] is not None else [t] * b
    live = torch.tensor([[i < e for i in range(t)] for e in ends], device="cuda", dtype=torch.bool).reshape(b, t)
    if c["op"] == "conv":
        taps = c["w"]
        line = torch.zeros(b, taps - 1 + t, d, device="cuda", dtype=torch.float64)
        if s["start"] is not None:
            line[:, :taps - 1] = s["start"]
        line[:, taps - 1:] = s["u"]
        pre = s["bias"].expand(b, t, d).clone()
        for j in range(taps):
            pre += line[:, j:j + t] * s["w"][:, j]
        out = {"y": (value[c["act"]](pre) * live[..., None])}
        out["window"] = torch.stack([line[i, e:e + taps - 1] for i, e in enumerate(ends)])
        if c["mode"] == "token":
            out["y"] = out["y"][:, 0]
        if c["mode"] == "train":
            dpre = s["dy"] * slope[c["act"]](pre) * live[..., None]
            dline, dw = torch.zeros_like(line), torch.zeros(d, taps, device="cuda", dtype=torch.float64)
            for j in range(taps):
                dline[:, j:j + t] += dpre * s["w"][:, j]
                dw[:, j] = (dpre * line[:, j:j + t]).sum((0, 1))
            for i, e in enumerate(ends):
                dline[i, e:e + taps - 1] += s["dlast"][i]
            out.update(dw=dw, dbias=dpre.sum((0, 1)), du=dline[:, taps - 1:] * live[..., None])
            if s["start"] is not None:
                out["dstart"] = dline[:, :taps - 1]
        return out
    n, per = c["n"], c["d"] // c["g"]
    wide = lambda v: v[:, :, None].expand(b, c["g"], per, n).reshape(b, d, n)   # noqa: E731
    raw = s["dt"] + s["dt_bias"]
    delta = torch.logaddexp(raw, torch.zeros_like(raw)) * live[..., None]
    train = c["mode"] == "train"
    x = s["start"] if s["start"] is not None else torch.zeros(b, d, n, device="cuda", dtype=torch.float64)
    xs = [x]
    y = torch.empty(b, t, d, device="cuda", dtype=torch.float64)
    for i in range(t):
        x = torch.exp(delta[:, i, :, None] * s["A"]) * x + (delta[:, i] * s["u"][:, i])[..., None] * wide(s["B"][:, i])
        y[:, i] = (x * wide(s["C"][:, i])).sum(-1) + s["D"] * s["u"][:, i]
        if train:
            xs.append(x)
    gate = value["silu"](s["z"]) if s["z"] is not None else torch.ones_like(y)
    out = {"y": y * gate * live[..., None], "state": x}
    if c["mode"] == "token":
        out["y"] = out["y"][:, 0]
    if train:
        if s["z"] is not None:
            out["dz"] = s["dy"] * y * slope["silu"](s["z"]) * live[..., None]
        dy = s["dy"] * gate * live[..., None]
        lam = s["dlast"].clone()
        du, draw_ = torch.empty_like(y), torch.empty_like(y)
        dA, dB, dC = torch.zeros(d, n, device="cuda", dtype=torch.float64), torch.zeros_like(s["B"]), torch.zeros_like(s["C"])
        for i in reversed(range(t)):
            Bi, e = wide(s["B"][:, i]), torch.exp(delta[:, i, :, None] * s["A"])
            lam = lam + dy[:, i, :, None] * wide(s["C"][:, i])
            along = (lam * Bi).sum(-1)
            grown = lam * e * xs[i]
            du[:, i] = s["D"] * dy[:, i] + delta[:, i] * along
            draw_[:, i] = (grown * s["A"]).sum(-1) + s["u"][:, i] * along
            dA += (grown * delta[:, i, :, None]).sum(0)
            dB[:, i] = (lam * (delta[:, i] * s["u"][:, i])[..., None]).reshape(b, c["g"], per, n).sum(2)
            dC[:, i] = (xs[i + 1] * dy[:, i, :, None]).reshape(b, c["g"], per, n).sum(2)
            lam = lam * e
        draw_ = draw_ * torch.sigmoid(raw) * live[..., None]
        out.update(du=du * live[..., None], ddt=draw_, ddt_bias=draw_.sum((0, 1)), dA=dA, dD=(dy * s["u"]).sum((0, 1)), dB=dB, dC=dC)
        if s["start"] is not None:
            out["dstart"] = lam
    return out
