"""Plain restatements, in 64 bits or whole numbers and token by token, of the attention half of a decoder layer: the
plan of a pass over a paged cache, the per-head norm and rotation, and attention over a prefix and a line's own keys."""
import math

import torch


def plan(lengths, counts, table, free, used, page, tokens, prefix=0):
    """lines_plan on Python lists; table is changed in place. Also returns whether a page was missing (`pages`) and
    whether tokens were left out (`tokens`)."""
    slots, positions, line, cu, out_lengths = [], [], [], [0], []
    missing = left_out = False
    for b, (kept, n) in enumerate(zip(lengths, counts)):
        kept, n = max(0, kept), max(0, n)
        fits = min(n, tokens - len(slots))
        left_out |= fits < n
        for s in range(kept, kept + fits):
            j, off = divmod(s, page)
            if off == 0:
                got = free[used] if used < len(free) else -1
                used = min(used + 1, len(free))
                if j < len(table[b]):
                    table[b][j] = got
            p = table[b][j] if j < len(table[b]) else -1
            missing |= p < 0
            slots.append(p * page + off if p >= 0 else -1)
            positions.append(prefix + s)
            line.append(b)
        cu.append(len(slots))
        out_lengths.append(kept + fits)
    spare = tokens - len(slots)
    return dict(slots=slots + [-1] * spare, positions=positions + [0] * spare, line=line + [-1] * spare, cu=cu,
                lengths=out_lengths, used=[used], pages=missing, tokens=left_out)


def norm_rope(x, weight, offset, eps, rotary, positions, axes, pairs):
    """x [T, heads, D] in float64 through the norm and the rotation; weight None: no norm. Positions outside the table
    leave their pair unturned."""
    y = x.double().clone()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * (weight.double() + offset)
    length, n = rotary.shape[:2]
    out = y.clone()
    for f in range(n):
        at = positions if axes is None else positions[int(axes[f])]
        inside = (at >= 0) & (at < length)
        cs = rotary[at.clamp(0, length - 1), f].double()
        c = torch.where(inside, cs[:, 0], torch.ones_like(cs[:, 0]))[:, None]
        s = torch.where(inside, cs[:, 1], torch.zeros_like(cs[:, 1]))[:, None]
        i, j = (2 * f, 2 * f + 1) if pairs else (f, f + n)
        out[..., i] = y[..., i] * c - y[..., j] * s
        out[..., j] = y[..., j] * c + y[..., i] * s
    return out


def attention(q, k_cache, v_cache, kept, counts, table, prefix, prefix_table, scale):
    """(out, lse, bound) in float64: `bound` is softmax @ |V|, the size of what each output sums."""
    T, Hq, D = q.shape
    page, Hkv = k_cache.shape[1:3]
    G = Hq // Hkv
    out = torch.zeros((T, Hq, D), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=q.device)

    def rows(cache, tab, n):
        return torch.cat([cache[p] for p in tab[:(n + page - 1) // page].tolist()] or [cache[0, :0]])[:n]

    t0 = 0
    for b, (kept_b, n) in enumerate(zip(kept, counts)):
        if n == 0:
            continue
        n = min(n, T - t0)
        k, v = (torch.cat((rows(c, prefix_table, prefix), rows(c, table[b], kept_b + n))).double() for c in (k_cache, v_cache))
        seen = torch.arange(prefix + kept_b + n, device=q.device)[None] <= prefix + kept_b + torch.arange(n, device=q.device)[:, None]
        for h in range(Hq):
            s = (q[t0:t0 + n, h].double() @ k[:, h // G].T) * scale
            s = torch.where(seen, s, torch.tensor(-math.inf, dtype=s.dtype, device=s.device))
            lse[t0:t0 + n, h] = torch.logsumexp(s, -1)
            p = torch.exp(s - lse[t0:t0 + n, h, None])
            out[t0:t0 + n, h] = p @ v[:, h // G]
            bound[t0:t0 + n, h] = p @ v[:, h // G].abs()
        t0 += n
    return out, lse, bound
