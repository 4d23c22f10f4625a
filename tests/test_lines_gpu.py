"""The attention half of a decoder layer on the GPU (lines_plan, qk_norm_rope, lines_attention) against its plain
restatements in tests/lines_ref.py.

Tolerances. qk_norm_rope: one rounding to the row's type (half a unit in the last place: at most 2^-8 of the value for
bfloat16's 8 significant bits, 2^-11 for float16's 11) of a 32-bit result whose error is a few 2^-24 of the pair's size; for float32 rows 2^-20 of the pair's size covers the sum of
squares and a dozen operations. lines_attention: an output is a sum of p_j V_j whose p_j are rounded to the values'
type and which is rounded once more at the end, each by at most half a unit in the last place, so |error| <= 2 x that x sum p_j |V_j|; a tenth more stands for everything in 32 bits, and 2^-24 for float16's
smallest steps. lse: the scores' 32-bit sums (2^-22 of sum |q k|, below 2^4 where the scores are ordinary) and the exponentials'
2^-21 make 2e-5; where the scores are large, 2^-21 of the sum's own size is added for the rounding of both."""
import math
import random

import pytest
import torch

import lines_ref as ref

pytestmark = pytest.mark.gpu

HALF_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def fault():
    from drama3_b200._lib import take_fault
    return take_fault()


def i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


# ---- lines_plan

PLANS = [
    # lengths, counts, page, spare token places, prefix
    ([0], [1], 16, 0, None),
    ([0], [0], 16, 2, 5),
    ([15, 16, 17, 0], [1, 1, 1, 1], 16, 0, 100),
    ([0, 5, 64, 3], [0, 70, 0, 200], 16, 3, 7),
    ([1, 2, 3], [4, 0, 1], 1, 1, 0),
    ([6, 7, 8], [1, 1, 30], 7, 0, 3),
    ([-4, 2], [3, -2], 16, 1, 1),
]


def lines_case(lengths, counts, page, spare, seed=0, room=2, extra=5):
    rng = random.Random(seed)
    have = [(max(0, n) + page - 1) // page for n in lengths]
    need = [(max(0, n) + max(0, c) + page - 1) // page for n, c in zip(lengths, counts)]
    width = max(need) + room
    order = list(range(sum(need) + extra))
    rng.shuffle(order)
    table, used = [], 0
    for h in have:
        table.append(order[used:used + h] + [-1] * (width - h))
        used += h
    return table, order, used, sum(max(0, c) for c in counts) + spare


def run_plan(cuda, lengths, counts, table, free, used, page, tokens, prefix, group=1):
    from drama3_b200 import kernels
    t = i32(table, cuda)
    args = (i32(lengths, cuda), i32(counts, cuda), t, i32(free, cuda), i32([used], cuda), page, tokens)
    p = kernels.lines_plan(*args, prefix=None if prefix is None else i32([prefix], cuda), group=group)
    return args, p


def check_plan(p, want, table):
    for name in ("slots", "positions", "line", "cu", "lengths", "used"):
        got = getattr(p, name).tolist()
        assert got == want[name], name
    assert p.table.tolist() == table


@pytest.mark.parametrize("lengths,counts,page,spare,prefix", PLANS)
def test_plan(cuda, lengths, counts, page, spare, prefix):
    table, free, used, tokens = lines_case(lengths, counts, page, spare)
    args, p = run_plan(cuda, lengths, counts, table, free, used, page, tokens, prefix)
    want = ref.plan(lengths, counts, table, free, used, page, tokens, prefix or 0)
    check_plan(p, want, table)
    assert fault() == 0
    # planning the same pass again gives the same plan
    from drama3_b200 import kernels
    again = kernels.lines_plan(*args, prefix=None if prefix is None else i32([prefix], cuda))
    check_plan(again, want, table)


@pytest.mark.parametrize("lines,most", [(1, 5000), (33, 400), (600, 3), (2500, 9), (8192, 2)])
def test_plan_many(cuda, lines, most):
    rng = random.Random(lines)
    lengths = [rng.randrange(0, 300) for _ in range(lines)]
    counts = [rng.randrange(0, most + 1) for _ in range(lines)]
    table, free, used, tokens = lines_case(lengths, counts, 16, 9, seed=lines)
    _, p = run_plan(cuda, lengths, counts, table, free, used, 16, tokens, 1234)
    check_plan(p, ref.plan(lengths, counts, table, free, used, 16, tokens, 1234), table)
    assert fault() == 0


def test_plan_without_room(cuda):
    lengths, counts = [3, 16, 30, 2], [20, 1, 10, 50]
    table, free, used, tokens = lines_case(lengths, counts, 16, 0)
    for cut_free, cut_width, cut_tokens in ((4, 0, 0), (0, 3, 0), (0, 0, 30), (5, 2, 7), (0, 0, tokens)):
        f = free[:len(free) - 5 - cut_free]
        t = [row[:len(row) - cut_width] for row in table]
        _, p = run_plan(cuda, lengths, counts, t, f, used, 16, tokens - cut_tokens, 0)
        want = ref.plan(lengths, counts, t, f, used, 16, tokens - cut_tokens, 0)
        check_plan(p, want, t)
        assert fault() == (32 if want["pages"] else 0) | (64 if want["tokens"] else 0)


def units_of(p):
    work = p.work.tolist()
    at = (16 + p.slots.shape[0] + 3) & ~3
    return work, [tuple(work[at + 8 * u:at + 8 * u + 8]) for u in range(work[1])]


@pytest.mark.parametrize("group", [1, 7, 8, 128])
@pytest.mark.parametrize("lengths,counts,prefix", [
    ([100] * 16, [1] * 16, 300), ([0, 9, 64, 63], [1, 40, 0, 200], 130), ([0], [3000], 0), ([5], [1], 64),
    ([0, 0], [128, 130], 1)])
def test_work_list_covers_every_row_and_key(cuda, group, lengths, counts, prefix):
    table, free, used, tokens = lines_case(lengths, counts, 16, 2)
    _, p = run_plan(cuda, lengths, counts, table, free, used, 16, tokens, prefix, group=group)
    work, units = units_of(p)
    total, tile = sum(counts), 128 // group
    together = work[0] == 1
    assert work[3] == prefix and work[5] == total and work[6] == group
    keys, unit_cost = 128, 3  # of a key tile; what a unit costs besides its tiles
    place, own, shared = 0, [], []
    for line, token0, rows, at, tiles, sees, own_end, lead in units:
        assert at == place + unit_cost and tiles >= 1
        place = at + tiles
        (own if line >= 0 else shared).append((line, token0, rows, tiles, sees, own_end, lead))
    assert place == work[2]
    key_tiles = -(-prefix // keys)
    lead, want, first = key_tiles if together else 0, [], 0
    for b, (kept, n) in enumerate(zip(lengths, counts)):
        for i in range(0, n, tile):
            end = min(i + tile, n)
            assert work[16 + first + i:16 + first + end] == [len(shared) + len(want)] * (end - i)
            want.append((b, first + i, (end - i) * group, lead + -(-(kept + end) // keys), kept + i + 1, kept + end, lead))
        first += n
    assert own == want
    assert shared == ([] if together else [(-1, i, min(tile, total - i) * group, key_tiles, 0, 0, key_tiles)
                                           for i in range(0, total, tile)])
    assert together or prefix


# ---- qk_norm_rope

def rope_inputs(cuda, T, hq, hkv, D, rot, axes, dtype, seed, strided=0):
    from drama3_b200 import kernels
    g = torch.Generator(device=cuda).manual_seed(seed)
    wide = (hq + 2 * hkv) * D + strided
    qkv = (torch.randn((T, wide), generator=g, device=cuda) * 3).to(dtype)[:, strided:]
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split((hq * D, hkv * D, hkv * D), 1))
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g, device=cuda)).to(dtype) for _ in range(2))
    n = rot // 2
    rotary = kernels.rotary_table(10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)), 500, cuda)
    shape = (T,) if axes == 1 else (axes, T)
    pos = torch.randint(0, 500, shape, generator=g, device=cuda)
    amap = None if axes == 1 else kernels.rotary_axes([n - n // 3 * (axes - 1)] + [n // 3] * (axes - 1), woven=n % 2 == 0, device=cuda)
    return q, k, v, qw, kw, rotary, pos, amap


def close_rows(got, want, x, dtype):
    """One rounding of `want` plus 32-bit noise in proportion to the head's largest value."""
    size = want.abs().amax(-1, keepdim=True)
    tol = want.abs() * HALF_UNIT[dtype] + size * 2.0 ** -20 if dtype in HALF_UNIT else size * 2.0 ** -20
    if dtype == torch.float16:
        tol = tol + 2.0 ** -24
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,hq,hkv,D,rot,axes,pairs,strided", [
    (1, 32, 4, 128, 128, 1, False, 0), (16, 16, 2, 256, 64, 3, False, 0), (37, 8, 8, 64, 64, 1, True, 0),
    (5, 5, 5, 80, 40, 1, False, 0), (5, 5, 5, 80, 40, 1, True, 8), (300, 7, 1, 96, 96, 2, False, 16),
    (3, 2, 1, 512, 512, 1, False, 0), (3, 2, 1, 512, 128, 3, True, 0), (4, 3, 3, 1024, 64, 1, False, 0),
    (9, 3, 1, 66, 20, 1, False, 0), (9, 3, 1, 33, 32, 4, True, 0), (6, 4, 2, 128, 128, 1, False, 1),
    (2, 1, 1, 8, 8, 1, False, 0), (2, 1, 1, 2, 2, 1, True, 0), (11, 4, 4, 128, 0, 1, False, 0),
    (1100, 12, 3, 128, 96, 3, False, 0)])
def test_norm_rope(cuda, dtype, T, hq, hkv, D, rot, axes, pairs, strided):
    from drama3_b200 import kernels
    q, k, v, qw, kw, rotary, pos, amap = rope_inputs(cuda, T, hq, hkv, D, rot, axes, dtype, 7 * D + T, strided)
    got = kernels.qk_norm_rope(q, k, rotary, pos, q_weight=qw, k_weight=kw, eps=1e-5, axes=amap, pairs=pairs)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
        close_rows(y, ref.norm_rope(x, w, 0, 1e-5, rotary, pos, amap, pairs), x, dtype)
    assert fault() == 0


@pytest.mark.parametrize("D,strided", [(128, 0), (96, 3)])
def test_norm_rope_weights(cuda, D, strided):
    from drama3_b200 import kernels
    q, k, v, qw, kw, rotary, pos, _ = rope_inputs(cuda, 19, 6, 2, D, D, 1, torch.bfloat16, 3, strided)
    for a, b, off in ((None, None, 0), (qw, None, 0), (None, kw, 1), (qw - 1, kw - 1, 1), (qw.float(), kw.float(), 0)):
        got = kernels.qk_norm_rope(q, k, rotary, pos, q_weight=a, k_weight=b, unit_offset=bool(off))
        for x, w, y in ((q, a, got[0]), (k, b, got[1])):
            close_rows(y, ref.norm_rope(x, w, off, 1e-6, rotary, pos, None, False), x, torch.bfloat16)


def test_norm_rope_rows_of_zeros_and_extremes(cuda):
    from drama3_b200 import kernels
    q, k, v, qw, kw, rotary, pos, _ = rope_inputs(cuda, 4, 4, 4, 128, 128, 1, torch.float32, 5)
    q, k = q.clone(), k.clone()
    q[0], q[1], q[2] = 0, q[1] * 1e15, q[2] * 1e-15
    k[0, 0, 3] = math.nan
    k[1, 1, 5] = math.inf
    out, kk = kernels.qk_norm_rope(q, k, rotary, pos, q_weight=qw, k_weight=kw, eps=1e-6)
    close_rows(out, ref.norm_rope(q, qw, 0, 1e-6, rotary, pos, None, False), q, torch.float32)
    assert (out[0] == 0).all()
    # a head that holds a NaN or an infinity stays its own trouble
    bad = torch.zeros((4, 4), dtype=torch.bool, device=cuda)
    bad[0, 0] = bad[1, 1] = True
    assert torch.equal(kk.isnan().any(-1), bad)


@pytest.mark.parametrize("order", ["plain", "heads_first", "odd"])
@pytest.mark.parametrize("D", [64, 128, 72])
def test_norm_rope_into_cache(cuda, order, D):
    from drama3_b200 import kernels
    T, hq, hkv, page, pages = 41, 6, 3, 16, 9
    q, k, v, qw, kw, rotary, pos, _ = rope_inputs(cuda, T, hq, hkv, D, D, 1, torch.bfloat16, 11)

    def cache(fill):
        if order == "heads_first":  # [pages, heads, page, D]
            return torch.full((pages, hkv, page, D), fill, dtype=torch.bfloat16, device=cuda).transpose(1, 2)
        pad = 1 if order == "odd" else 0
        return torch.full((pages, page, hkv, D + pad), fill, dtype=torch.bfloat16, device=cuda)[..., :D]

    kc, vc = cache(7.0), cache(9.0)
    slots = torch.randperm(pages * page, device=cuda)[:T]
    slots[3], slots[8], slots[20] = -1, pages * page, 1 << 40
    out, none = kernels.qk_norm_rope(q, k, rotary, pos, q_weight=qw, k_weight=kw, v=v, k_cache=kc, v_cache=vc, slots=slots)
    assert none is None and fault() == 4
    plain, k_plain = kernels.qk_norm_rope(q, k, rotary, pos, q_weight=qw, k_weight=kw)
    assert torch.equal(out, plain)
    want_k, want_v = torch.full((pages * page, hkv, D), 7.0, dtype=torch.bfloat16, device=cuda), None
    want_v = torch.full_like(want_k, 9.0)
    ok = (slots >= 0) & (slots < pages * page)
    want_k[slots[ok]], want_v[slots[ok]] = k_plain[ok], v[ok]
    assert torch.equal(kc.reshape(-1, hkv, D), want_k) and torch.equal(vc.reshape(-1, hkv, D), want_v)


def test_norm_rope_positions_outside_the_table(cuda):
    from drama3_b200 import kernels
    for strided in (0, 1):
        q, k, v, qw, kw, rotary, pos, amap = rope_inputs(cuda, 6, 4, 2, 128, 64, 3, torch.bfloat16, 2, strided)
        pos[0, 1], pos[1, 2], pos[2, 5] = -1, 500, 1 << 40
        got = kernels.qk_norm_rope(q, k, rotary, pos, q_weight=qw, k_weight=kw, axes=amap)
        assert fault() == 128
        close_rows(got[0], ref.norm_rope(q, qw, 0, 1e-6, rotary, pos, amap, False), q, torch.bfloat16)
        bad = amap.clone()
        bad[4] = 3
        kernels.qk_norm_rope(q, k, rotary, pos.clamp(0, 499), q_weight=qw, k_weight=kw, axes=bad)
        assert fault() == 128


def test_norm_rope_empty(cuda):
    from drama3_b200 import kernels
    q, k, v, qw, kw, rotary, pos, _ = rope_inputs(cuda, 2, 4, 2, 128, 128, 1, torch.bfloat16, 2)
    got = kernels.qk_norm_rope(q[:0], k[:0], rotary, pos[:0], q_weight=qw, k_weight=kw)
    assert got[0].shape == (0, 4, 128) and got[1].shape == (0, 2, 128)


def test_rotary_helpers(cuda):
    from drama3_b200 import kernels
    t = kernels.rotary_table(torch.tensor([1.0, 0.001]), 200001, cuda)
    for p in (0, 1, 777, 200000):
        for f, w in enumerate((1.0, float(torch.tensor(0.001)))):
            assert abs(float(t[p, f, 0]) - math.cos(p * w)) < 1e-7 and abs(float(t[p, f, 1]) - math.sin(p * w)) < 1e-7
    assert kernels.rotary_axes([3, 2, 1]).tolist() == [0, 0, 0, 1, 1, 2]
    assert kernels.rotary_axes([3, 2, 1], woven=True).tolist() == [0, 1, 2, 0, 1, 0]


# ---- lines_attention

def attn_case(cuda, hq, hkv, D, dtype, page, kept, counts, prefix, spare=0, seed=0, order="plain", poison=True, loud=1.5):
    from drama3_b200 import kernels
    g = torch.Generator(device=cuda).manual_seed(seed)
    table, free, used, tokens = lines_case(kept, counts, page, spare, seed=seed)
    shared = (prefix + page - 1) // page
    pages = len(free) + shared
    names = list(range(pages))
    random.Random(seed + 1).shuffle(names)
    prefix_table = i32(names[len(free):], cuda)
    free = [names[x] for x in free]
    table = [[names[x] if x >= 0 else -1 for x in row] for row in table]
    _, plan = run_plan(cuda, kept, counts, table, free, used, page, tokens, prefix, group=hq // hkv)
    shape = (pages, hkv, page, D) if order == "heads_first" else (pages, page, hkv, D)
    kc, vc = (torch.randn(shape, generator=g, device=cuda).to(dtype) for _ in range(2))
    if order == "heads_first":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    if poison:  # whatever lies past the lengths is never used
        used_slots = torch.zeros(pages * page, dtype=torch.bool, device=cuda)
        for tab, n in [(prefix_table, prefix)] + [(plan.table[b], k + c) for b, (k, c) in enumerate(zip(kept, counts))]:
            for j in range((n + page - 1) // page):
                first = int(tab[j]) * page
                used_slots[first:first + min(page, n - j * page)] = True
        kc.view(pages, -1) if order == "plain" else None
        for c, bad in ((kc, math.nan), (vc, math.inf)):
            c[~used_slots.view(pages, page)] = bad
            c[(~used_slots).view(pages, page) & (torch.arange(page, device=cuda) % 2 == 0)] = math.nan
    q = (loud * torch.randn((tokens, hq, D), generator=g, device=cuda)).to(dtype)
    return q, kc, vc, plan, prefix_table


def check_attn(cuda, case, kept, counts, prefix, scale=None, lse=True):
    from drama3_b200 import kernels
    q, kc, vc, plan, prefix_table = case
    got, sums = kernels.lines_attention(q, kc, vc, plan, prefix_table=prefix_table, scale=scale, lse=True)
    want, want_lse, bound = ref.attention(q, kc, vc, kept, counts, plan.table, prefix, prefix_table,
                                          scale or 1 / math.sqrt(q.shape[2]))
    assert fault() == 0
    tol = 2.2 * HALF_UNIT[q.dtype] * bound + (2.0 ** -24 if q.dtype == torch.float16 else 0)
    err = (got.double() - want).abs()
    assert not got.isnan().any()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-30)).max())
    empty = torch.isinf(want_lse)
    assert torch.equal(empty, torch.isinf(sums)) and (sums[empty] < 0).all()
    assert ((sums.double() - want_lse)[~empty].abs() <= 2e-5 + 2.0 ** -21 * want_lse[~empty].abs()).all()
    return got


SHAPES = [(32, 4, 128), (16, 2, 256), (8, 8, 64), (7, 1, 64), (24, 3, 128), (4, 2, 256), (128, 1, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,D", SHAPES)
@pytest.mark.parametrize("page,prefix", [(16, 0), (16, 200), (32, 63), (64, 64), (128, 1000), (192, 1)])
def test_attention_decode(cuda, dtype, hq, hkv, D, page, prefix):
    kept, counts = [0, 1, 15, 63, 64, 200, 31, 500], [1] * 8
    case = attn_case(cuda, hq, hkv, D, dtype, page, kept, counts, prefix, seed=prefix + D)
    check_attn(cuda, case, kept, counts, prefix)


@pytest.mark.parametrize("hq,hkv,D", SHAPES)
@pytest.mark.parametrize("kept,counts,prefix,spare", [
    ([0], [1], 0, 0), ([0], [300], 0, 0), ([100, 0, 7], [50, 129, 1], 77, 0), ([5, 6, 7, 8], [1, 0, 3, 0], 130, 6),
    ([3] * 20, [2] * 20, 260, 1), ([0, 0], [33, 65], 4, 0), ([64, 1], [64, 16], 64, 0), ([9, 9], [0, 0], 10, 3)])
def test_attention_ragged(cuda, hq, hkv, D, kept, counts, prefix, spare):
    case = attn_case(cuda, hq, hkv, D, torch.bfloat16, 16, kept, counts, prefix, spare=spare, seed=len(kept))
    check_attn(cuda, case, kept, counts, prefix)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_long(cuda, D):
    # runs of many tiles, cut in the middle of units, the maximum growing as they go
    for kept, counts, prefix in (([6000], [1], 0), ([3000] * 3, [1] * 3, 9000), ([0], [2000], 0), ([700, 0], [900, 600], 1500)):
        case = attn_case(cuda, 16, 2, D, torch.bfloat16, 64, kept, counts, prefix, seed=D, loud=4.0)
        check_attn(cuda, case, kept, counts, prefix)


def test_attention_growing_maximum(cuda):
    # every key's score is far above those before it, so each tile moves the maximum, and far below, so none does
    for sign in (1, -1):
        kept, counts, prefix = [400, 90], [1, 40], 300
        q, kc, vc, plan, pt = attn_case(cuda, 8, 1, 128, torch.bfloat16, 16, kept, counts, prefix, poison=False)
        q[:], kc[:] = 1.0, 0.0
        for tab, n, base in ((pt, prefix, 0), (plan.table[0], 401, 300), (plan.table[1], 130, 300)):
            for j in range(n):
                kc[int(tab[j // 16]), j % 16] = sign * (base + j) / 16.0
        check_attn(cuda, (q, kc, vc, plan, pt), kept, counts, prefix)


@pytest.mark.parametrize("order", ["plain", "heads_first"])
def test_attention_strides(cuda, order):
    kept, counts, prefix = [40, 3], [5, 70], 100
    q, kc, vc, plan, pt = attn_case(cuda, 16, 4, 128, torch.bfloat16, 32, kept, counts, prefix, order=order)
    wide = torch.zeros((q.shape[0], 24, 128), dtype=q.dtype, device=cuda)
    wide[:, 8:] = q
    a = check_attn(cuda, (wide[:, 8:], kc, vc, plan, pt), kept, counts, prefix)
    assert torch.equal(a, check_attn(cuda, (q, kc, vc, plan, pt), kept, counts, prefix))
    check_attn(cuda, (q, kc, vc, plan, pt), kept, counts, prefix, scale=0.031)


def test_attention_past_32_bits(cuda):
    # a cache whose last pages lie beyond 2^31 elements and 2^32 bytes
    from drama3_b200 import kernels
    page, hkv, D, pages = 64, 8, 128, 34000
    assert pages * page * hkv * D > 1 << 31
    kc, vc = (torch.zeros((pages, page, hkv, D), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    free = i32(list(range(pages - 1, pages - 12, -1)), cuda)
    table, used = i32([[-1] * 8] * 2, cuda), i32([0], cuda)
    counts = [150, 90]
    plan = kernels.lines_plan(i32([0, 0], cuda), i32(counts, cuda), table, free, used, page, 240, group=2)
    g = torch.Generator(device=cuda).manual_seed(1)
    q, k, v = (torch.randn((240, h, D), generator=g, device=cuda).to(torch.bfloat16) for h in (16, 8, 8))
    rotary = kernels.rotary_table(torch.ones(64), 256, cuda)
    q2, _ = kernels.qk_norm_rope(q, k, rotary, plan.positions, v=v, k_cache=kc, v_cache=vc, slots=plan.slots)
    assert int(plan.slots.min()) * hkv * D > 1 << 31
    small_k, small_v = kc[pages - 12:].clone(), vc[pages - 12:].clone()
    want, _, bound = ref.attention(q2, small_k, small_v, [0, 0], counts, plan.table - (pages - 12), 0, i32([], cuda), 1 / math.sqrt(D))
    got = kernels.lines_attention(q2, kc, vc, plan)
    assert ((got.double() - want).abs() <= 2.2 * HALF_UNIT[torch.bfloat16] * bound).all() and fault() == 0
    assert (bound > 0).any()


def test_attention_bad_page_reads_zeros(cuda):
    from drama3_b200 import kernels
    kept, counts, prefix = [60, 20], [1, 1], 50
    q, kc, vc, plan, pt = attn_case(cuda, 8, 2, 64, torch.bfloat16, 16, kept, counts, prefix, poison=False)
    for bad in (-1, kc.shape[0], 1 << 30):
        table = plan.table.clone()
        table[0, 1] = bad
        got = kernels.lines_attention(q, kc, vc, plan._replace(table=table), prefix_table=pt)
        assert fault() == 32
        # the same with that page there and full of zeros
        kz, vz = (torch.cat((c, torch.zeros_like(c[:1]))) for c in (kc, vc))
        table[0, 1] = kc.shape[0]
        assert torch.equal(got, kernels.lines_attention(q, kz, vz, plan._replace(table=table), prefix_table=pt))
    # a prefix that no table holds
    kernels.lines_attention(q, kc, vc, plan)
    assert fault() == 32


def test_attention_plan_of_another_pass_is_refused(cuda):
    from drama3_b200 import kernels
    kept, counts = [60, 20], [1, 1]
    q, kc, vc, plan, pt = attn_case(cuda, 8, 2, 64, torch.bfloat16, 16, kept, counts, 0)
    other = attn_case(cuda, 8, 2, 64, torch.bfloat16, 16, [3], [2], 0)[3]
    with pytest.raises(ValueError):
        kernels.lines_attention(q, kc, vc, plan._replace(group=2), prefix_table=pt)
    kernels.lines_attention(q, kc, vc, plan._replace(work=other.work), prefix_table=pt)
    assert fault() == 256


def test_attention_twice_is_the_same_and_lines_do_not_mix(cuda):
    # no result depends on the order in which blocks run; a line's rows do not change with what else is decoded
    # beyond the way its keys are cut
    from drama3_b200 import kernels
    kept, counts, prefix = [300, 20, 77], [1, 1, 1], 500
    q, kc, vc, plan, pt = attn_case(cuda, 16, 2, 128, torch.bfloat16, 16, kept, counts, prefix)
    a = kernels.lines_attention(q, kc, vc, plan, prefix_table=pt)
    for _ in range(5):
        assert torch.equal(a, kernels.lines_attention(q, kc, vc, plan, prefix_table=pt))
    q2 = q.clone()
    q2[1] = math.nan
    b = kernels.lines_attention(q2, kc, vc, plan, prefix_table=pt)
    assert torch.equal(a[[0, 2]], b[[0, 2]]) and b[1].isnan().all()


def test_step_on_a_side_stream_and_in_a_graph(cuda):
    """Plan, cache write and attention captured once and replayed as the lines grow, against the same steps alone."""
    from drama3_b200 import kernels
    hq, hkv, D, page, B, prefix = 8, 2, 64, 16, 3, 70
    g = torch.Generator(device=cuda).manual_seed(4)
    pages = 40
    kc, vc = (torch.randn((pages, page, hkv, D), generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
    kc2, vc2 = kc.clone(), vc.clone()
    pt = i32(list(range(35, 40)), cuda)
    rotary = kernels.rotary_table(10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), 400, cuda)
    free = i32(list(range(34, -1, -1)), cuda)
    counts, pre = i32([1, 1, 1], cuda), i32([prefix], cuda)

    def state():
        return [i32([0, 30, 15], cuda), i32([[-1] * 10, [0, 1] + [-1] * 8, [2] + [-1] * 9], cuda), i32([0], cuda)]

    def step(st, kc, vc, qkv):
        q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split((hq * D, hkv * D, hkv * D), 1))
        plan = kernels.lines_plan(st[0], counts, st[1], free, st[2], page, B, prefix=pre, group=hq // hkv)
        qr, _ = kernels.qk_norm_rope(q, k, rotary, plan.positions, v=v, k_cache=kc, v_cache=vc, slots=plan.slots)
        out = kernels.lines_attention(qr, kc, vc, plan, prefix_table=pt)
        st[0].copy_(plan.lengths)
        st[2].copy_(plan.used)
        return out

    xs = [torch.randn((B, (hq + 2 * hkv) * D), generator=g, device=cuda).to(torch.bfloat16) for _ in range(20)]
    st = state()
    want = [step(st, kc, vc, x) for x in xs]
    held, x = state(), xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone() for t in held], kc2.clone(), vc2.clone(), x)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(held, kc2, vc2, x)
        for i, xi in enumerate(xs):
            x.copy_(xi)
            graph.replay()
            side.synchronize()
            assert torch.equal(out, want[i]), i
    assert torch.equal(kc, kc2) and torch.equal(held[0], st[0]) and fault() == 0
    del graph


# ---- refusals that need tensors on a GPU, the ops, the module and the example

def test_wrapper_refusals(cuda):
    from drama3_b200 import kernels
    n = i32([1, 1], cuda)
    t, f, u = i32([[-1], [-1]], cuda), i32([0, 1], cuda), i32([0], cuda)
    for bad in (dict(counts=n[:1]), dict(counts=n.long()), dict(table=i32([[-1]], cuda)), dict(used=n), dict(free=f.float()),
                dict(prefix=n), dict(group=200), dict(table=t.t()), dict(counts=n.cpu())):
        args = dict(lengths=n, counts=n, table=t, free=f, used=u, page=16, tokens=2)
        with pytest.raises(ValueError):
            kernels.lines_plan(**{**args, **bad})
    q, k, v, qw, kw, rotary, pos, amap = rope_inputs(cuda, 4, 4, 2, 64, 64, 3, torch.bfloat16, 1)
    cache = torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16, device=cuda)
    slots = torch.arange(4, device=cuda)
    args = dict(q=q, k=k, rotary=rotary, positions=pos, axes=amap)
    whole = dict(v=v, k_cache=cache, v_cache=cache.clone(), slots=slots)
    for error, bad in ((TypeError, dict(q=q.double())), (TypeError, dict(k=k.half())), (ValueError, dict(k=k[:2])),
                       (ValueError, dict(k=k[..., :32])), (ValueError, dict(q=q.transpose(1, 2))),
                       (ValueError, dict(q_weight=qw[:32])), (ValueError, dict(q_weight=qw, k_weight=kw.float())),
                       (ValueError, dict(rotary=rotary.half())), (ValueError, dict(rotary=rotary.repeat(1, 2, 1))),
                       (ValueError, dict(positions=pos[0])), (ValueError, dict(positions=pos.int())),
                       (ValueError, dict(axes=None)), (ValueError, dict(axes=amap[:8])), (ValueError, dict(axes=amap.long())),
                       (ValueError, dict(v=v)), (ValueError, {**whole, "slots": None}), (ValueError, {**whole, "v": v[:2]}),
                       (ValueError, {**whole, "k_cache": cache.half()}), (ValueError, {**whole, "v_cache": cache[:1]}),
                       (ValueError, {**whole, "slots": slots.int()}), (ValueError, dict(positions=pos.cpu())),
                       (ValueError, {**whole, "k_cache": cache.cpu()})):
        with pytest.raises(error):
            kernels.qk_norm_rope(**{**args, **bad})
    plan = kernels.lines_plan(i32([0] * 4, cuda), i32([1] * 4, cuda), i32([[-1]] * 4, cuda), i32(list(range(4)), cuda), u, 16, 4,
                              group=2)
    kc = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16, device=cuda)
    for error, bad in ((TypeError, dict(q=q.float())), (TypeError, dict(k_cache=kc.half())), (ValueError, dict(v_cache=kc[:3])),
                       (ValueError, dict(k_cache=kc[..., :32], v_cache=kc[..., :32])), (ValueError, dict(q=q[:3])),
                       (ValueError, dict(plan=plan._replace(page=32))), (ValueError, dict(plan=plan._replace(group=4))),
                       (ValueError, dict(prefix_table=i32([0], cuda).long())), (ValueError, dict(v_cache=kc.cpu()))):
        with pytest.raises(error):
            kernels.lines_attention(**{**dict(q=q, k_cache=kc, v_cache=kc, plan=plan), **bad})
    with pytest.raises(ValueError):  # heads of 96: no kernel
        kernels.lines_attention(torch.zeros((4, 4, 96), dtype=torch.bfloat16, device=cuda), *[torch.zeros(
            (4, 16, 2, 96), dtype=torch.bfloat16, device=cuda)] * 2, plan)
    with pytest.raises(_lib_error()):  # a page that no tile is made of
        odd = kernels.lines_plan(i32([0] * 4, cuda), i32([1] * 4, cuda), i32([[-1]] * 4, cuda), i32(list(range(4)), cuda), u, 24,
                                 4, group=2)
        kernels.lines_attention(q, *[torch.zeros((4, 24, 2, 64), dtype=torch.bfloat16, device=cuda)] * 2, odd)
    assert fault() == 0


def _lib_error():
    from drama3_b200._lib import D3Error
    return D3Error


def test_ops_equal_the_kernels(cuda):
    import drama3_b200.ops  # noqa: F401
    from drama3_b200 import kernels
    o = torch.ops.drama3_b200
    kept, counts, prefix = [40, 3], [5, 70], 100
    q, kc, vc, plan, pt = attn_case(cuda, 16, 4, 128, torch.bfloat16, 32, kept, counts, prefix)
    out, lse = kernels.lines_attention(q, kc, vc, plan, prefix_table=pt, lse=True)
    got = o.lines_attention(q, kc, vc, plan.table, plan.work, 4, pt)
    assert torch.equal(out, got[0]) and torch.equal(lse, got[1])
    table, free, used, tokens = lines_case(kept, counts, 32, 3)
    args = lambda: (i32(kept, cuda), i32(counts, cuda), i32(table, cuda), i32(free, cuda), i32([used], cuda), 32, tokens)  # noqa: E731
    a, b = args(), args()
    p = kernels.lines_plan(*a, prefix=i32([9], cuda), group=4)
    r = o.lines_plan(*b, i32([9], cuda), 4)
    assert torch.equal(a[2], b[2])
    for x, y in zip((p.slots, p.positions, p.line, p.cu, p.lengths, p.used), r):
        assert torch.equal(x, y)
    rq, rk, rv, qw, kw, rotary, pos, _ = rope_inputs(cuda, 9, 6, 2, 64, 64, 1, torch.bfloat16, 5)
    for x, y in zip(kernels.qk_norm_rope(rq, rk, rotary, pos, qw, kw), o.qk_norm_rope(rq, rk, rotary, pos, qw, kw)):
        assert torch.equal(x, y)
    caches = [torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16, device=cuda) for _ in range(4)]
    slots = torch.randperm(32, device=cuda)[:9]
    want, _ = kernels.qk_norm_rope(rq, rk, rotary, pos, v=rv, k_cache=caches[0], v_cache=caches[1], slots=slots)
    assert torch.equal(want, o.qk_norm_rope_cached(rq, rk, rv, rotary, pos, caches[2], caches[3], slots))
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


def test_module_reads_a_prefix_and_texts_as_one_sequence(cuda):
    """LinesAttention over a LinesCache: a shared prefix, ragged texts and two steps give each line what torch's layers
    give the whole sequence (bf16 rounds at the same places but inside the attention: 2^-8 of sum p |V| there, and the
    output projection sums 512 such columns; 1.5 % of the output's norm covers both)."""
    from drama3_b200 import kernels
    from drama3_b200.attention import LinesAttention, LinesCache
    torch.manual_seed(3)
    hidden, hq, hkv, D, page = 256, 8, 2, 64, 16
    att = LinesAttention(hidden, hq, hkv, D, device=cuda, dtype=torch.bfloat16)
    with torch.no_grad():
        att.q_norm.mul_(1.3)
        att.k_norm.add_(0.1 * torch.randn(D, device=cuda))
    prefix, texts, steps = 37, [3, 20, 0, 9], 2
    cache = LinesCache(1, 40, page, hkv, D, 4, 64, hq // hkv, cuda)
    rotary = kernels.rotary_table(10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16), 128, cuda)
    x0 = torch.randn((prefix, hidden), device=cuda).bfloat16()
    xs = [torch.randn((n + steps, hidden), device=cuda).bfloat16() for n in texts]

    def layers(x):  # one whole sequence through torch
        q, k, v = (t.unflatten(1, (-1, D)) for t in att.qkv_proj(x).split([hq * D, hkv * D, hkv * D], 1))
        pos = torch.arange(x.shape[0], device=cuda)
        q, k = (ref.norm_rope(t, w, 0, att.eps, rotary, pos, None, False).bfloat16().float() for t, w in
                ((q, att.q_norm), (k, att.k_norm)))
        o = torch.nn.functional.scaled_dot_product_attention(
            q.transpose(0, 1), k.transpose(0, 1).repeat_interleave(hq // hkv, 0),
            v.float().transpose(0, 1).repeat_interleave(hq // hkv, 0), is_causal=True)
        return att.o_proj(o.transpose(0, 1).flatten(1).bfloat16())

    def close(got, want):
        assert float((got.float() - want.float()).norm()) <= 0.015 * float(want.float().norm())

    with torch.no_grad():
        for again in range(2):  # the second time, new lines behind the same prefix
            if again:
                cache.restart()
            else:
                close(att(x0, cache.plan_prefix(prefix), cache.k[0], cache.v[0], rotary), layers(x0))
            want = [layers(torch.cat((x0, x)))[prefix:] for x in xs]
            got = att(torch.cat([x[:n] for x, n in zip(xs, texts)]), cache.plan(i32(texts, cuda), sum(texts)), cache.k[0],
                      cache.v[0], rotary, cache.prefix_table).split(texts)
            for g, w, n in zip(got, want, texts):
                if n:
                    close(g, w[:n])
            for s in range(steps):
                g = att(torch.stack([x[n + s] for x, n in zip(xs, texts)]), cache.plan(i32([1] * 4, cuda), 4), cache.k[0],
                        cache.v[0], rotary, cache.prefix_table)
                close(g, torch.stack([w[n + s] for w, n in zip(want, texts)]))
    assert fault() == 0 and cache.lengths.tolist() == [n + steps for n in texts]


def test_example_runs(cuda):
    import importlib.util
    from pathlib import Path
    spec = importlib.util.spec_from_file_location("lines_decode", Path(__file__).resolve().parents[1] / "examples" / "lines_decode.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    rows, ms = example.decode(lines=3, prompt=70, steps=4, n_layers=2)
    again, _ = example.decode(lines=3, prompt=70, steps=4, n_layers=2)
    assert rows.shape == (3, example.HIDDEN) and rows.isfinite().all() and ms > 0 and fault() == 0
    assert torch.equal(rows, again)
