"""What is measured of the linear half of a hybrid decoder for lines decoded together: the short causal convolution over
each line's own tokens (`lines_conv`), linear attention with a decay for each head, with or without the delta rule, over a
state of each line (`lines_delta`), the norm of its heads with their gate (`gated_norm`), and the join of a block to its
residual with the norms before and after it (`add_norm`).

`run` computes each operator in elementary torch operations in 32 bits where `own` is false, and through
drama3_b200.kernels where it is true."""
import math
import sys

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
CHUNK = 64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _kernels():
    if "comfyui-drama3_b200" not in sys.path:
        sys.path.insert(1, "comfyui-drama3_b200")
    from drama3_b200 import kernels
    return kernels


def listed():
    return [
        # a decode step of 16 lines, one new token each: queries, keys and values of 16 + 16 + 32 heads of 128
        dict(name="conv_decode_16", op="conv", lines=16, new="one", most_new=1, spare=0, channels=8192, taps=4, bias=False,
             dtype="bf16"),
        # a prompt read for the first time
        dict(name="conv_prompt_8192", op="conv", lines=1, new="all", most_new=8192, spare=0, channels=8192, taps=4,
             bias=False, dtype="bf16"),
        # one line alone, one token: latency
        dict(name="delta_step_1", op="delta", lines=1, new="one", most_new=1, spare=0, k_heads=16, v_heads=32, k_dim=128,
             v_dim=128, delta=True, raw=True, norm=True, dtype="bf16"),
        # the decode step of 16 lines
        dict(name="delta_step_16", op="delta", lines=16, new="one", most_new=1, spare=0, k_heads=16, v_heads=32, k_dim=128,
             v_dim=128, delta=True, raw=True, norm=True, dtype="bf16"),
        # the largest batch: a gigabyte of states read and written
        dict(name="delta_step_256", op="delta", lines=256, new="some", most_new=1, spare=3, k_heads=16, v_heads=32, k_dim=128,
             v_dim=128, delta=True, raw=True, norm=True, dtype="bf16"),
        # the lines' own texts, ragged, read behind the shared prompt
        dict(name="delta_texts_16", op="delta", lines=16, new="ragged", most_new=192, spare=0, k_heads=16, v_heads=32,
             k_dim=128, v_dim=128, delta=True, raw=True, norm=True, dtype="bf16"),
        # the shared prompt itself
        dict(name="delta_prompt_8192", op="delta", lines=1, new="all", most_new=8192, spare=0, k_heads=16, v_heads=32,
             k_dim=128, v_dim=128, delta=True, raw=True, norm=True, dtype="bf16"),
        # no delta rule: decays given as logarithms, smaller heads of two sizes, fp16, ragged lines, idle places behind them
        dict(name="decay_ragged_9", op="delta", lines=9, new="ragged", most_new=777, spare=11, k_heads=10, v_heads=10,
             k_dim=64, v_dim=80, delta=False, raw=False, norm=False, dtype="fp16"),
        # the heads' norm and gate: a decode step, a prompt
        dict(name="gated_16", op="gated", tokens=16, heads=32, dim=128, act="silu", unit=False, dtype="bf16"),
        dict(name="gated_8192", op="gated", tokens=8192, heads=32, dim=128, act="silu", unit=False, dtype="bf16"),
        # the join of a block to its residual: a decode step with the next block's norm alone; a clip's rows with a norm
        # after the block too, a gate for each row and a residual scale
        dict(name="join_16", op="join", tokens=16, width=2048, post=False, gate="none", scale=1.0, unit=False, dtype="bf16"),
        dict(name="join_16384", op="join", tokens=16384, width=2048, post=True, gate="row", scale=0.5, unit=True, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("conv", "delta", "gated", "join")}
    while True:
        op = rng.choice(["conv", "delta", "delta", "delta", "gated", "join"])
        new = rng.choice(["one", "some", "ragged", "ragged"])
        if op == "conv":
            case = dict(op=op, lines=_spread(rng, 1, 256), new=new, most_new=_spread(rng, 2, 2048) if new == "ragged" else 1,
                        spare=rng.choice([0, 0, 7]), channels=rng.choice([8192, 4096, 2048, 1000, 777, 96]),
                        taps=rng.choice([4, 4, 2, 3]), bias=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        elif op == "delta":
            k_heads, v_heads, k_dim, v_dim = rng.choice([(16, 32, 128, 128), (16, 16, 128, 128), (4, 8, 128, 256), (8, 8, 64, 64),
                                                         (10, 10, 64, 80), (3, 9, 64, 128), (1, 5, 128, 48)])
            raw = rng.random() < 0.7
            case = dict(op=op, lines=_spread(rng, 1, 256), new=new, most_new=_spread(rng, 2, 1024) if new == "ragged" else 1,
                        spare=rng.choice([0, 0, 5]), k_heads=k_heads, v_heads=v_heads, k_dim=k_dim, v_dim=v_dim,
                        delta=raw or rng.random() < 0.3, raw=raw, norm=True, dtype=rng.choice(["bf16", "bf16", "fp16"]))
            case["norm"] = case["delta"] or rng.random() < 0.5
        elif op == "gated":
            heads, dim = rng.choice([(32, 128), (16, 256), (8, 64), (5, 80), (16, 128), (3, 129)])
            case = dict(op=op, tokens=_spread(rng, 1, 8192), heads=heads, dim=dim, act=rng.choice(["silu", "silu", "sigmoid"]),
                        unit=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        else:
            case = dict(op=op, tokens=_spread(rng, 1, 16384), width=rng.choice([2048, 2048, 4096, 1024, 5120, 1000, 333]),
                        post=rng.random() < 0.5, gate=rng.choice(["none", "row", "channel", "each"]),
                        scale=rng.choice([1.0, 0.5, 0.22]), unit=rng.random() < 0.3,
                        dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        if _cost(case) <= most[op] and (op != "delta" or _padded(case) <= 40000):
            return case


# ---- inputs

def _counts(case):
    """New tokens of each line, on the host: what a scheduler decided. The same lines for every seed, so that a case always
    has the same number of tokens; prepare puts them in an order of the seed's."""
    gen, lines = torch.Generator().manual_seed(1), case["lines"]
    if case["new"] == "all":
        return torch.full((lines,), case["most_new"], dtype=torch.int64)
    if case["new"] == "one":
        return torch.ones(lines, dtype=torch.int64)
    if case["new"] == "some":  # lines that have ended append nothing
        new = (torch.rand(lines, generator=gen) < 0.8).long()
        new[0] = 1
        return new
    new = torch.randint(0, case["most_new"] + 1, (lines,), generator=gen)
    new[-1] = case["most_new"]
    return new


def _padded(case):
    return case["lines"] * case["most_new"]


def _lines(case, seed):
    """The pass's lines: the plan that a program makes once for all its layers, or what the plain form reads of it."""
    new = _counts(case)[torch.randperm(case["lines"], generator=torch.Generator().manual_seed(seed))]
    s = {"new": new.to(torch.int32).to(DEVICE), "tokens": int(new.sum()) + case["spare"], "most": int(new.max())}
    cu = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    s["cu"] = cu.to(DEVICE)
    if own:
        lines, width = case["lines"], -(-s["most"] // 64)
        ints = dict(dtype=torch.int32, device=DEVICE)
        s["plan"] = _kernels().lines_plan(torch.zeros(lines, **ints), s["new"], torch.full((lines, width), -1, **ints),
                                          torch.arange(lines * width, **ints), torch.zeros(1, **ints), 64, s["tokens"])
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, to=dtype, mean=0.0, std=1.0):
        return (mean + std * torch.randn(shape, generator=gen, device=DEVICE)).to(to)

    def uniform(*shape, lo=0.0, hi=1.0):
        return lo + (hi - lo) * torch.rand(shape, generator=gen, device=DEVICE)

    s = {"case": case}
    if case["op"] == "conv":
        s.update(_lines(case, seed))
        C, W = case["channels"], case["taps"]
        # the fused projection's output: these channels and, behind them, the gate's; some channels are louder than others
        gain = torch.exp(0.5 * torch.randn(C, generator=gen, device=DEVICE))
        wide = normal(s["tokens"], C + C // 2, to=torch.float32)
        wide[:, :C] *= gain
        s["x"] = wide.to(dtype)[:, :C]
        s["state"] = (normal(case["lines"], W - 1, C, to=torch.float32) * gain).to(dtype)  # each line's last inputs
        s["weight"] = normal(C, W, std=1 / math.sqrt(W))
        s["bias"] = normal(C, std=0.1) if case["bias"] else None
    elif case["op"] == "delta":
        s.update(_lines(case, seed))
        T, hk, hv, dk, dv = s["tokens"], case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
        # queries, keys and values as the convolution leaves them: one tensor, SiLU of unequal channels
        mixed = normal(T, 2 * hk * dk + hv * dv, to=torch.float32)
        mixed = torch.nn.functional.silu(mixed * torch.exp(0.3 * torch.randn(mixed.shape[1], generator=gen, device=DEVICE)))
        if not case["norm"]:
            mixed[:, :2 * hk * dk] *= dk ** -0.25
        mixed = mixed.to(dtype)
        s["q"] = mixed[:, :hk * dk].view(T, hk, dk)
        s["k"] = mixed[:, hk * dk:2 * hk * dk].view(T, hk, dk)
        s["v"] = mixed[:, 2 * hk * dk:].view(T, hv, dv)
        s["a_log"] = s["dt_bias"] = s["beta"] = None
        if case["raw"]:  # the projections' outputs, and how fast each head forgets
            both = normal(T, 2 * hv)
            s["beta"], s["decay"] = both[:, :hv], both[:, hv:]
            s["a_log"] = torch.log(uniform(hv, lo=1.0, hi=16.0))
            step = torch.exp(uniform(hv, lo=math.log(0.001), hi=math.log(0.1)))
            s["dt_bias"] = step + torch.log(-torch.expm1(-step))  # softplus of it is the step
        else:
            s["decay"] = -torch.exp(uniform(T, hv, lo=math.log(1e-3), hi=math.log(0.5)))
            s["beta"] = uniform(T, hv) if case["delta"] else None
        s["state"] = normal(case["lines"], hv, dv, dk, to=torch.float32, std=0.2)
    elif case["op"] == "gated":
        T, h, d = case["tokens"], case["heads"], case["dim"]
        s["x"] = normal(T, h, d, std=0.3)
        # the gate: the tail of the fused projection's output
        s["gate"] = normal(T, 3 * h * d)[:, 2 * h * d:].view(T, h, d)
        s["weight"] = normal(d, mean=0.0 if case["unit"] else 1.0, std=0.1)
    else:
        T, w = case["tokens"], case["width"]
        s["x"] = normal(T, w, std=0.7)
        s["residual"] = normal(T, w, std=3.0)
        mean = 0.0 if case["unit"] else 1.0
        s["weight"] = normal(w, mean=mean, std=0.1)
        s["post"] = normal(w, mean=mean, std=0.1) if case["post"] else None
        shape = {"none": None, "row": (T, 1), "channel": (1, w), "each": (T, w)}[case["gate"]]
        s["gate"] = None if shape is None else uniform(*shape).to(dtype)
    return s


# ---- the operators in their plain form

def _conv_plain(s):
    c, x, state = s["case"], s["x"], s["state"]
    T, C, W, cu = s["tokens"], c["channels"], c["taps"], s["cu"]
    t = torch.arange(T, device=DEVICE)
    line = torch.searchsorted(cu[1:], t, right=True)
    live = (line < c["lines"])[:, None]
    b = line.clamp(max=c["lines"] - 1)
    i = t - cu[b]
    # row t of `inputs` is the token itself, rows T.. the lines' last inputs of before
    inputs = torch.cat((x, state.flatten(0, 1))).float()
    weight = s["weight"].float()
    y = torch.zeros((T, C), device=DEVICE) if s["bias"] is None else s["bias"].float().expand(T, C)
    for j in range(W):
        back = W - 1 - j
        y = y + inputs[torch.where(i >= back, t - back, T + b * (W - 1) + W - 1 + i - back)] * weight[:, j]
    y = y * torch.sigmoid(y)
    k = torch.arange(W - 1, device=DEVICE)[None]
    n = (cu[1:] - cu[:-1])[:, None]
    at = n - (W - 1) + k  # the input that is k-th of the last, counted in the line's new tokens
    rows = torch.where(at >= 0, cu[:-1, None] + at, T + torch.arange(c["lines"], device=DEVICE)[:, None] * (W - 1) + n + k)
    state.copy_(inputs[rows].to(state.dtype))
    return {"out": torch.where(live, y, torch.zeros_like(y)).to(x.dtype), "state": state}


def _gates(s, wide):
    """(log decay, strength of the delta rule or None) [T, v_heads]."""
    g, beta = s["decay"].to(wide), s["beta"]
    if s["a_log"] is not None:
        g = g + s["dt_bias"].to(wide)
        g = -torch.exp(s["a_log"].to(wide)) * (torch.clamp(g, min=0) + torch.log1p(torch.exp(-g.abs())))
        beta = torch.sigmoid(beta.to(wide))
    return g, None if beta is None else beta.to(wide)


def _delta_plain(s):
    """In chunks of 64 tokens of every line at once, lines padded to the longest: within a chunk the tokens' corrections
    solve a unit lower triangular system, across chunks the state is carried."""
    c, state, cu, T = s["case"], s["state"], s["cu"], s["tokens"]
    B, hv, dk, dv, many = c["lines"], c["v_heads"], c["k_dim"], c["v_dim"], c["v_heads"] // c["k_heads"]
    C = min(CHUNK, s["most"])
    n = -(-s["most"] // C)
    i = torch.arange(n * C, device=DEVICE)[None]
    at = (cu[:-1, None] + i).clamp(max=T - 1)
    here = (i < (cu[1:] - cu[:-1])[:, None])[:, :, None]  # [B, n C, 1]
    g, beta = _gates(s, torch.float32)

    def cut(x):  # [T, heads, d] -> [B, heads, n, C, d]
        return torch.where(here[..., None], x[at], torch.zeros_like(x[:1])).transpose(1, 2).unflatten(2, (n, C))

    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if c["norm"]:
        q, k = (x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS) for x in (q, k))
    q, k, v = cut((q / math.sqrt(dk)).repeat_interleave(many, 1)), cut(k.repeat_interleave(many, 1)), cut(v)
    G = cut(g[..., None]).double().cumsum(3)  # [B, hv, n, C, 1]
    low = torch.ones((C, C), dtype=torch.bool, device=DEVICE).tril()
    ratio = torch.exp((G - G.transpose(3, 4)).masked_fill(~low, -math.inf)).float()
    within = (q @ k.transpose(3, 4)) * ratio
    decay, left = torch.exp(G).float(), torch.exp(G[:, :, :, -1:] - G).float()
    if beta is not None:
        b = cut(beta[..., None])
        A = ((k * b) @ k.transpose(3, 4) * ratio).tril(-1)
        inverse = torch.eye(C, device=DEVICE).expand(A.shape).clone()
        for r in range(1, C):
            inverse[..., r, :r] = -(A[..., r, :r, None] * inverse[..., :r, :r]).sum(-2)
        inverse = inverse * b.transpose(3, 4)
    out = torch.empty_like(v)
    S = state.transpose(2, 3)  # [B, hv, dk, dv]
    for j in range(n):
        u = v[:, :, j]
        if beta is not None:
            u = inverse[:, :, j] @ (u - decay[:, :, j] * (k[:, :, j] @ S))
        out[:, :, j] = decay[:, :, j] * (q[:, :, j] @ S) + within[:, :, j] @ u
        S = S * decay[:, :, j, -1:] + k[:, :, j].transpose(2, 3) @ (left[:, :, j] * u)
    state.copy_(S.transpose(2, 3))
    flat = torch.zeros((T, hv, dv), device=DEVICE)
    keep = here[..., 0]
    flat[at[keep]] = out.flatten(2, 3).transpose(1, 2)[keep]
    return {"out": flat.to(s["v"].dtype), "state": state}


def _normed(x, weight, unit):
    w = weight.float() + 1 if unit else weight.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _gated_plain(s):
    c, z = s["case"], s["gate"].float()
    gate = torch.sigmoid(z) * z if c["act"] == "silu" else torch.sigmoid(z)
    return (_normed(s["x"].float(), s["weight"], c["unit"]) * gate).to(s["x"].dtype)


def _join_plain(s):
    c, x = s["case"], s["x"].float()
    if s["post"] is not None:
        x = _normed(x, s["post"], c["unit"])
    if s["gate"] is not None:
        x = x * s["gate"].float()
    total = s["residual"].float() + c["scale"] * x
    return {"residual": total.to(s["x"].dtype), "normed": _normed(total, s["weight"], c["unit"]).to(s["x"].dtype)}


def run(s):
    c = s["case"]
    if c["op"] == "conv":
        if not own:
            return _conv_plain(s)
        return {"out": _kernels().lines_conv(s["x"], s["weight"], s["state"], s["plan"], bias=s["bias"]), "state": s["state"]}
    if c["op"] == "delta":
        if not own:
            return _delta_plain(s)
        out = _kernels().lines_delta(s["q"], s["k"], s["v"], s["decay"], s["state"], s["plan"], beta=s["beta"],
                                     a_log=s["a_log"], dt_bias=s["dt_bias"], eps=EPS if c["norm"] else None)
        return {"out": out, "state": s["state"]}
    if c["op"] == "gated":
        if not own:
            return _gated_plain(s)
        return _kernels().gated_norm(s["x"], s["gate"], s["weight"], eps=EPS, unit_offset=c["unit"], activation=c["act"])
    if not own:
        return _join_plain(s)
    residual, normed = _kernels().add_norm(s["x"], s["residual"], s["weight"], post_weight=s["post"], gate=s["gate"],
                                           scale=c["scale"], eps=EPS, unit_offset=c["unit"])
    return {"residual": residual, "normed": normed}


# ---- what a pass cannot do without

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "gated":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 3 * n * size, "flops": 10 * n}
    if case["op"] == "join":
        T, w = case["tokens"], case["width"]
        gate = {"none": 0, "row": T, "channel": w, "each": T * w}[case["gate"]]
        return {"bytes": (4 * T * w + gate) * size, "flops": 10 * T * w}
    new = _counts(case)
    T, active = int(new.sum()), int((new > 0).sum())
    if case["op"] == "conv":
        C, W = case["channels"], case["taps"]
        return {"bytes": (2 * T * C + 2 * active * (W - 1) * C + C * W) * size, "flops": 2 * T * C * W}
    hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
    rows = T * (2 * hk * dk + 2 * hv * dv) * size + T * hv * (2 * size if case["raw"] else 8 if case["delta"] else 4)
    # the state decays, is read for the correction, is written to and read for the output
    return {"bytes": rows + 2 * 4 * active * hv * dk * dv, "flops": (7 if case["delta"] else 5) * T * hv * dk * dv}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 250)


# ---- the operators from their definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "delta": _exact_delta, "gated": _exact_gated, "join": _exact_join}[case["op"]](s, case)


def _exact_conv(s, c):
    """Line by line: the line's old and new inputs in a row, a window over each of its tokens."""
    W, cu = c["taps"], s["cu"].tolist()
    out = torch.zeros((s["tokens"], c["channels"]), dtype=torch.float64, device=DEVICE)
    state = s["state"].double()
    for b in range(c["lines"]):
        row = torch.cat((state[b], s["x"][cu[b]:cu[b + 1]].double()))
        if cu[b + 1] > cu[b]:
            y = (row.unfold(0, W, 1) * s["weight"].double()).sum(-1)
            if s["bias"] is not None:
                y = y + s["bias"].double()
            out[cu[b]:cu[b + 1]] = y / (1 + torch.exp(-y))
        state[b] = row[len(row) - (W - 1):]
    return {"out": out, "state": state}


def _exact_delta(s, c):
    """Token by token, all lines that still have one at a time."""
    new = s["new"].tolist()
    if max(new) * sum(1 for n in new if n) > 1 << 18:
        return None
    many, cu = c["v_heads"] // c["k_heads"], s["cu"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    if c["norm"]:
        q, k = (x / torch.sqrt(x.square().sum(-1, keepdim=True) + EPS) for x in (q, k))
    q, k = (x.repeat_interleave(many, 1) for x in (q, k))
    g, beta = _gates(s, torch.float64)
    state = s["state"].double()
    out = torch.zeros((s["tokens"], c["v_heads"], c["v_dim"]), dtype=torch.float64, device=DEVICE)
    order = sorted(range(len(new)), key=lambda b: -new[b])
    S = state[order]  # the lines with most tokens first
    first = cu[:-1][torch.tensor(order, device=DEVICE)]
    for i in range(max(new)):
        m = sum(1 for n in new if n > i)
        t = first[:m] + i
        live = S[:m]
        live *= torch.exp(g[t])[:, :, None, None]
        u = v[t]
        if beta is not None:
            u = (u - (live @ k[t][..., None])[..., 0]) * beta[t][..., None]
        live += u[..., None] * k[t][:, :, None]
        out[t] = (live @ q[t][..., None])[..., 0] / math.sqrt(c["k_dim"])
    state[order] = S
    return {"out": out, "state": state}


def _exact_gated(s, c):
    x, z, w = s["x"].double(), s["gate"].double(), s["weight"].double()
    y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / c["dim"] + EPS) * (w + 1 if c["unit"] else w)
    return y / (1 + torch.exp(-z)) * (z if c["act"] == "silu" else 1)


def _exact_join(s, c):
    def normed(x, w):
        return x / torch.sqrt(x.square().sum(-1, keepdim=True) / c["width"] + EPS) * (w.double() + 1 if c["unit"] else w.double())

    x = s["x"].double()
    if c["post"]:
        x = normed(x, s["post"])
    if s["gate"] is not None:
        x = x * s["gate"].double()
    total = s["residual"].double() + x * c["scale"]
    return {"residual": total, "normed": normed(total, s["weight"])}
