"""What is measured of the attention half of a decoder layer for lines decoded together: the plan of a pass over a
paged key/value cache (`lines_plan`), the per-head norms and the rotation of queries and keys with the cache write
(`qk_norm_rope`), and the attention of every line to the shared prefix and to its own tail (`lines_attention`).

`run` computes each operator in elementary torch operations in 32 bits where `own` is false, and through
drama3_b200.kernels where it is true."""
import math
import sys

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _kernels():
    if "comfyui-drama3_b200" not in sys.path:
        sys.path.insert(1, "comfyui-drama3_b200")
    from drama3_b200 import kernels
    return kernels


def listed():
    return [
        # a decode step of the benchmark's 16 lines, one new token each
        dict(name="plan_decode_16", op="plan", lines=16, new="one", most_new=1, most_kept=4096, page=64, spare=0),
        # the prompts of a thousand lines appended in one pass, ragged, some lines idle, in small pages
        dict(name="plan_prompts_1024", op="plan", lines=1024, new="ragged", most_new=512, most_kept=600, page=16,
             spare=1000),
        # a decode step's queries and keys (the benchmark's 32 / 4 heads of 128), written into the cache
        dict(name="rope_decode_16", op="rope", tokens=16, q_heads=32, kv_heads=4, dim=128, rot=128, axes=1, weave=False,
             pairs=False, cache=True, page=64, dtype="bf16"),
        # a prompt of 16 / 2 heads of 256 with a quarter of each head rotated, by three axes woven together
        dict(name="rope_prompt_2048", op="rope", tokens=2048, q_heads=16, kv_heads=2, dim=256, rot=64, axes=3, weave=True,
             pairs=False, cache=True, page=16, dtype="bf16"),
        # a clip's patches by time, height and width, without a cache
        dict(name="rope_clip_16384", op="rope", tokens=16384, q_heads=32, kv_heads=4, dim=128, rot=128, axes=3, weave=False,
             pairs=False, cache=False, page=0, dtype="bf16"),
        # 32-bit rows of a small head whose size is no power of two, rotated in neighbouring pairs
        dict(name="rope_odd_777", op="rope", tokens=777, q_heads=5, kv_heads=5, dim=80, rot=40, axes=1, weave=False,
             pairs=True, cache=False, page=0, dtype="fp32"),
        # one line alone over its own thousand tokens: latency
        dict(name="attn_line_1", op="attn", lines=1, prefix=0, new="one", most_new=1, most_kept=1000, spare=0, q_heads=32,
             kv_heads=4, dim=128, page=64, dtype="bf16", lse=False),
        # the benchmark's decode step: 16 lines behind a shared prompt of 4096 tokens
        dict(name="attn_decode_16", op="attn", lines=16, prefix=4096, new="one", most_new=1, most_kept=512, spare=0,
             q_heads=32, kv_heads=4, dim=128, page=64, dtype="bf16", lse=False),
        # heads of 256, an odd prefix, small pages, a batch of fixed size with idle rows, fp16, the sums returned too
        dict(name="attn_decode_d256", op="attn", lines=16, prefix=3001, new="some", most_new=1, most_kept=300, spare=3,
             q_heads=16, kv_heads=2, dim=256, page=16, dtype="fp16", lse=True),
        # many lines behind a long shared prompt
        dict(name="attn_decode_64_long", op="attn", lines=64, prefix=32768, new="one", most_new=1, most_kept=2048, spare=0,
             q_heads=32, kv_heads=4, dim=128, page=128, dtype="bf16", lse=False),
        # the lines' own texts, ragged, read behind the shared prompt
        dict(name="attn_texts_16", op="attn", lines=16, prefix=4096, new="ragged", most_new=192, most_kept=0, spare=0,
             q_heads=32, kv_heads=4, dim=128, page=64, dtype="bf16", lse=False),
        # the shared prompt itself, read for the first time
        dict(name="attn_prompt_8192", op="attn", lines=1, prefix=0, new="all", most_new=8192, most_kept=0, spare=0,
             q_heads=32, kv_heads=4, dim=128, page=64, dtype="bf16", lse=False),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("plan", "rope", "attn")}
    while True:
        op = rng.choice(["plan", "rope", "attn", "attn"])
        if op == "plan":
            case = dict(op=op, lines=_spread(rng, 1, 2048), new=rng.choice(["one", "some", "ragged"]), most_new=1,
                        most_kept=_spread(rng, 1, 8192), page=rng.choice([16, 32, 64, 128]), spare=rng.choice([0, 1, 37]))
            if case["new"] == "ragged":
                case["most_new"] = _spread(rng, 2, 512)
        elif op == "rope":
            q_heads, kv_heads, dim = rng.choice([(32, 4, 128), (16, 2, 256), (8, 8, 64), (5, 5, 80), (24, 3, 96), (7, 1, 128)])
            axes = rng.choice([1, 3])
            rot = rng.choice([dim, dim // 2])
            case = dict(op=op, tokens=_spread(rng, 1, 16384), q_heads=q_heads, kv_heads=kv_heads, dim=dim, rot=rot,
                        axes=axes, weave=axes > 1 and rng.random() < 0.5, pairs=rng.random() < 0.3, cache=rng.random() < 0.5,
                        page=rng.choice([16, 64]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        else:
            q_heads, kv_heads, dim = rng.choice([(32, 4, 128), (16, 2, 256), (8, 8, 64), (24, 3, 128), (7, 1, 64), (16, 2, 128)])
            new = rng.choice(["one", "one", "some", "ragged"])
            case = dict(op=op, lines=_spread(rng, 1, 96), prefix=rng.choice([0, _spread(rng, 1, 32768), _spread(rng, 1, 32768)]),
                        new=new, most_new=_spread(rng, 2, 256) if new == "ragged" else 1, most_kept=_spread(rng, 1, 4096),
                        spare=rng.choice([0, 0, 5]), q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                        page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "bf16", "fp16"]), lse=rng.random() < 0.3)
        if _cost(case) <= most[op]:
            return case


# ---- inputs

def _counts(case):
    """(tokens already kept, new tokens) of each line, on the host: what a scheduler decided. The same lines for every
    seed, so that a case always has the same number of tokens; prepare puts them in an order of the seed's."""
    gen, lines = torch.Generator().manual_seed(1), case["lines"]
    if case["new"] == "all":
        return torch.zeros(lines, dtype=torch.int64), torch.full((lines,), case["most_new"], dtype=torch.int64)
    kept = torch.randint(0, case["most_kept"] + 1, (lines,), generator=gen)
    if lines == 1:
        kept[:] = case["most_kept"]
    if case["new"] == "one":
        new = torch.ones(lines, dtype=torch.int64)
    elif case["new"] == "some":  # lines that have ended append nothing
        new = (torch.rand(lines, generator=gen) < 0.8).long()
        new[0] = 1
    else:
        new = torch.randint(0 if case["op"] == "plan" else 1, case["most_new"] + 1, (lines,), generator=gen)
        new[-1] = case["most_new"]
    return kept, new


def _pages(n, page):
    return (n + page - 1) // page


def _lines_state(case, seed, gen):
    """The pass's lengths and the block tables as a running program holds them: kept tokens in pages handed out in a
    scattered order, the free pages behind them."""
    host = torch.Generator().manual_seed(seed)
    kept, new = (t[torch.randperm(case["lines"], generator=torch.Generator().manual_seed(seed))] for t in _counts(case))
    page, prefix = case["page"], case.get("prefix", 0)
    have, width = _pages(kept, page), int(_pages(kept + new, page).max()) + 2
    held = int(have.sum())
    total = held + int((_pages(kept + new, page) - have).sum()) + 8
    shared = _pages(prefix, page)
    order = torch.randperm(total + shared, generator=host).to(torch.int32)
    at = (have.cumsum(0) - have)[:, None] + torch.arange(width)[None]
    table = torch.where(torch.arange(width)[None] < have[:, None], order[at.clamp(max=total - 1)], torch.tensor(-1, dtype=torch.int32))
    put = lambda t: t.to(torch.int32).to(DEVICE)  # noqa: E731
    return dict(kept=put(kept), new=put(new), table=put(table), free=put(order[:total]), used=put(torch.tensor([held])),
                prefix=put(torch.tensor([prefix])), prefix_table=put(order[total:]), pages=total + shared,
                tokens=int(new.sum()) + case["spare"], width=width, most=int(new.max()))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "rope":
        T, hq, hkv, d, dtype = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"], TYPES[case["dtype"]]
        # the fused projection's output; some channels are louder than others, as trained ones are
        gain = torch.exp(0.5 * torch.randn((hq + 2 * hkv) * d, generator=gen, device=DEVICE))
        qkv = (torch.randn((T, (hq + 2 * hkv) * d), generator=gen, device=DEVICE) * gain).to(dtype)
        s["q"] = qkv[:, :hq * d].view(T, hq, d)
        s["k"] = qkv[:, hq * d:(hq + hkv) * d].view(T, hkv, d)
        s["v"] = qkv[:, (hq + hkv) * d:].view(T, hkv, d)
        s["qw"], s["kw"] = ((1 + 0.1 * torch.randn(d, generator=gen, device=DEVICE)).to(dtype) for _ in range(2))
        half = case["rot"] // 2
        angle = torch.arange(8192, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
        s["rotary"] = torch.stack((angle.cos(), angle.sin()), -1).float().to(DEVICE)  # kept by the program, [8192, half, 2]
        if case["axes"] == 1:
            s["axes"] = None
            s["pos"] = torch.randint(0, 8192 - T if T < 8192 else 1, (1,), generator=gen, device=DEVICE) + torch.arange(T, device=DEVICE) % 8192
        else:  # time, height, width of each token; a third of the frequencies each, in runs or woven
            i = torch.arange(half)
            s["axes"] = (i % 3 if case["weave"] else (i * 3) // half).to(torch.uint8).to(DEVICE)
            s["pos"] = torch.stack([torch.randint(0, n, (T,), generator=gen, device=DEVICE) for n in (8192, 64, 96)])
        if case["cache"]:
            pages = _pages(T, case["page"]) + 3
            s["kc"], s["vc"] = (torch.zeros((pages, case["page"], hkv, d), dtype=dtype, device=DEVICE) for _ in range(2))
            s["slots"] = torch.randperm(pages * case["page"], generator=gen, device=DEVICE)[:T]
        return s
    s.update(_lines_state(case, seed, gen))
    if case["op"] == "attn":
        hq, hkv, d, dtype = case["q_heads"], case["kv_heads"], case["dim"], TYPES[case["dtype"]]
        s["q"] = (1.5 * torch.randn((s["tokens"], hq, d), generator=gen, device=DEVICE)).to(dtype)
        s["kc"], s["vc"] = (torch.randn((s["pages"], case["page"], hkv, d), generator=gen, device=DEVICE).to(dtype) for _ in range(2))
        # a program plans once a pass and attends with that plan in every layer; planning is measured by its own cases
        s["plan"] = _plan_own(s) if own else _plan_plain(s)
    return s


# ---- the operators

def _plan_own(s):
    k, c = _kernels(), s["case"]
    return k.lines_plan(s["kept"], s["new"], s["table"], s["free"], s["used"], c["page"], s["tokens"], prefix=s["prefix"],
                        group=c.get("q_heads", 8) // c.get("kv_heads", 1))


def _plan_plain(s):
    kept, new, page = s["kept"].long(), s["new"].long(), s["case"]["page"]
    have, need = (kept + page - 1) // page, (kept + new + page - 1) // page
    more = need - have
    first = more.cumsum(0) - more
    j = torch.arange(s["width"], device=DEVICE)[None]
    fresh = (j >= have[:, None]) & (j < need[:, None])
    at = s["used"].long() + first[:, None] + j - have[:, None]
    table = s["table"]
    table.copy_(torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1)], table))
    cu = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    t = torch.arange(s["tokens"], device=DEVICE)
    line = torch.searchsorted(cu[1:], t, right=True)
    live = line < kept.numel()
    b = line.clamp(max=kept.numel() - 1)
    p = kept[b] + t - cu[b]
    slot = table[b, (p // page).clamp(max=s["width"] - 1)].long() * page + p % page
    gone = torch.full_like(t, -1)
    return {"table": table, "slots": torch.where(live, slot, gone), "positions": torch.where(live, s["prefix"].long() + p, gone + 1),
            "line": torch.where(live, b, gone).int(), "cu": cu.int(), "lengths": (kept + new).int(),
            "used": (s["used"].long() + more.sum()).int()}


def _rope_plain(s):
    c = s["case"]
    half = c["rot"] // 2
    if s["axes"] is None:
        cs = s["rotary"][s["pos"]]
    else:
        cs = s["rotary"][s["pos"][s["axes"].long()], torch.arange(half, device=DEVICE)[:, None]].transpose(0, 1)
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]

    def one(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        r, rest = x[..., :c["rot"]], x[..., c["rot"]:]
        a, b = (r[..., 0::2], r[..., 1::2]) if c["pairs"] else (r[..., :half], r[..., half:])
        a, b = a * cos - b * sin, b * cos + a * sin
        r = torch.stack((a, b), -1).flatten(-2) if c["pairs"] else torch.cat((a, b), -1)
        return torch.cat((r, rest), -1).to(TYPES[c["dtype"]])

    q, k = one(s["q"], s["qw"]), one(s["k"], s["kw"])
    if not c["cache"]:
        return {"q": q, "k": k}
    for cache, rows in ((s["kc"], k), (s["vc"], s["v"])):
        cache.view(-1, c["kv_heads"], c["dim"])[s["slots"]] = rows
    return {"q": q, "kc": s["kc"], "vc": s["vc"]}


def _attn_plain(s):
    """Every line's queries, padded to the pass's longest, against the prefix and the line's own gathered tail."""
    c, plan = s["case"], s["plan"]
    B, hkv, d, page, P = c["lines"], c["kv_heads"], c["dim"], c["page"], c["prefix"]
    g, T, N = c["q_heads"] // hkv, s["tokens"], s["most"]
    scale = 1 / math.sqrt(d)
    q = s["q"].float().view(T, hkv, g, d)
    cu, lengths, new = plan["cu"].long(), plan["lengths"].long(), s["new"].long()
    i = torch.arange(N, device=DEVICE)[None]
    at = (cu[:-1, None] + i).clamp(max=T - 1)  # [B, N] the token of each padded query
    pages = plan["table"].long().clamp(min=0)
    keys, values = (x.float()[pages].flatten(1, 2) for x in (s["kc"], s["vc"]))  # [B, L, hkv, d]
    qb = q[at].permute(0, 2, 3, 1, 4).reshape(B, hkv, g * N, d)
    own_s = (qb @ keys.permute(0, 2, 3, 1)).view(B, hkv, g, N, -1).mul_(scale)
    j = torch.arange(keys.shape[1], device=DEVICE)
    seen = j <= (lengths - new)[:, None, None] + i[:, :, None]  # [B, N, L]
    own_s.masked_fill_(~seen[:, None, None], -math.inf)
    top = own_s.amax(-1)
    shared = s["prefix_table"].long()
    if P:
        pk, pv = (x.float()[shared].flatten(0, 1)[:P] for x in (s["kc"], s["vc"]))  # [P, hkv, d]
        pre_s = torch.matmul(qb.view(B, hkv, g * N, d), pk.permute(1, 2, 0)[None]).view(B, hkv, g, N, P).mul_(scale)
        top = torch.maximum(top, pre_s.amax(-1))
    own_s = own_s.sub_(top[..., None]).exp_()
    total = own_s.sum(-1)
    out = (own_s.view(B, hkv, g * N, -1) @ values.transpose(1, 2)).view(B, hkv, g, N, d)
    if P:
        pre_s = pre_s.sub_(top[..., None]).exp_()
        total = total + pre_s.sum(-1)
        out = out + torch.matmul(pre_s.view(B, hkv, g * N, P), pv.transpose(0, 1)[None]).view(B, hkv, g, N, d)
    out = (out / total[..., None]).permute(0, 3, 1, 2, 4)  # [B, N, hkv, g, d]
    lse = (top + total.log()).permute(0, 3, 1, 2)
    line = plan["line"].long()
    b = line.clamp(min=0)
    row = (torch.arange(T, device=DEVICE) - cu[b]).clamp(0, N - 1)
    live = (line >= 0)[:, None, None]
    res = {"out": (out[b, row] * live[..., None]).reshape(T, -1, d).to(s["q"].dtype)}
    if c["lse"]:
        res["lse"] = torch.where(live, lse[b, row], torch.full_like(lse[:1, :1], -math.inf)[0]).reshape(T, -1)
    return res


def run(s):
    c = s["case"]
    if c["op"] == "plan":
        if not own:
            return _plan_plain(s)
        p = _plan_own(s)
        return {"table": p.table, "slots": p.slots, "positions": p.positions, "line": p.line, "cu": p.cu,
                "lengths": p.lengths, "used": p.used}
    if c["op"] == "rope":
        if not own:
            return _rope_plain(s)
        more = dict(v=s["v"], k_cache=s["kc"], v_cache=s["vc"], slots=s["slots"]) if c["cache"] else {}
        q, k = _kernels().qk_norm_rope(s["q"], s["k"], s["rotary"], s["pos"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                                       axes=s["axes"], pairs=c["pairs"], **more)
        return {"q": q, "kc": s["kc"], "vc": s["vc"]} if c["cache"] else {"q": q, "k": k}
    if not own:
        return _attn_plain(s)
    got = _kernels().lines_attention(s["q"], s["kc"], s["vc"], s["plan"], prefix_table=s["prefix_table"], lse=c["lse"])
    return {"out": got[0], "lse": got[1]} if c["lse"] else {"out": got}


# ---- what a pass cannot do without

def work(case):
    if case["op"] == "rope":
        T, hq, hkv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
        size = 4 if case["dtype"] == "fp32" else 2
        rows = T * (hq + (2 if case["cache"] else 1) * hkv) * d
        return {"bytes": 2 * rows * size + 8 * T * (case["axes"] + case["cache"]), "flops": 8 * T * (hq + hkv) * d}
    kept, new = _counts(case)
    T = int(new.sum()) + case["spare"]
    if case["op"] == "plan":
        fresh = int((_pages(kept + new, case["page"]) - _pages(kept, case["page"])).sum())
        return {"bytes": 16 * case["lines"] + 8 * fresh + 20 * T, "flops": 0}
    hq, hkv, d, P = case["q_heads"], case["kv_heads"], case["dim"], case["prefix"]
    keys = P + int((kept + new)[new > 0].sum())  # each cached key and value once for all that attend to it
    seen = int((new * (P + kept) + new * (new + 1) // 2).sum())
    return {"bytes": 2 * 2 * keys * hkv * d + 2 * 2 * T * hq * d, "flops": 4 * seen * hq * d}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 250)


# ---- the operators from their definitions in 64 bits

def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(s, case)
    return _exact_attn(s, case)


def _exact_rope(s, c):
    """Each rotated pair as a complex number turned by its angle's unit vector."""
    half = c["rot"] // 2
    pos = s["pos"] if s["pos"].dim() == 2 else s["pos"][None]
    axis = s["axes"].long() if s["axes"] is not None else torch.zeros(half, dtype=torch.long, device=DEVICE)
    unit = torch.empty((c["tokens"], half), dtype=torch.complex128, device=DEVICE)
    for f in range(half):
        unit[:, f] = torch.view_as_complex(s["rotary"][pos[axis[f]], f].double())
    out = {}
    for name, x, w in (("q", s["q"], s["qw"]), ("k", s["k"], s["kw"])):
        y = x.double()
        y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / c["dim"] + EPS) * w.double()
        first, second = (slice(0, c["rot"], 2), slice(1, c["rot"], 2)) if c["pairs"] else (slice(0, half), slice(half, c["rot"]))
        z = torch.complex(y[..., first], y[..., second]) * unit[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        out[name] = y
    if not c["cache"]:
        return out
    for name, cache, rows in (("kc", s["kc"], out.pop("k")), ("vc", s["vc"], s["v"].double())):
        whole = cache.double().flatten(0, 1)
        whole[s["slots"]] = rows
        out[name] = whole.view(cache.shape)
    return out


def _exact_attn(s, c):
    """Line by line and KV head by KV head: softmax over the keys that the line's tokens see, in order."""
    kept, new = s["kept"].tolist(), s["new"].tolist()
    plan = s["plan"]
    table = (plan["table"] if isinstance(plan, dict) else plan.table).long()
    hkv, d, page, P = c["kv_heads"], c["dim"], c["page"], c["prefix"]
    g = c["q_heads"] // hkv
    out = torch.zeros((s["tokens"], c["q_heads"], d), dtype=torch.float64, device=DEVICE)
    lse = torch.full((s["tokens"], c["q_heads"]), -math.inf, dtype=torch.float64, device=DEVICE)
    flat_k, flat_v = s["kc"].flatten(0, 1), s["vc"].flatten(0, 1)
    where_p = torch.arange(P, device=DEVICE)
    where_p = s["prefix_table"].long()[where_p // page] * page + where_p % page if P else where_p
    t0 = 0
    for b, (n0, n) in enumerate(zip(kept, new)):
        if not n:
            continue
        own_at = torch.arange(n0 + n, device=DEVICE)
        rows = torch.cat((where_p, table[b][own_at // page] * page + own_at % page))
        hidden = torch.arange(P + n0 + n, device=DEVICE)[None] > P + n0 + torch.arange(n, device=DEVICE)[:, None]
        for h in range(hkv):
            k, v = flat_k[rows, h].double(), flat_v[rows, h].double()
            for x in range(h * g, h * g + g):
                score = (s["q"][t0:t0 + n, x].double() @ k.T) / math.sqrt(d)
                score[hidden] = -math.inf
                lse[t0:t0 + n, x] = torch.logsumexp(score, -1)
                out[t0:t0 + n, x] = torch.exp(score - lse[t0:t0 + n, x, None]) @ v
        t0 += n
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}
