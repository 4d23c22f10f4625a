"""The attention half of a decoder layer on the GPU at the limits of its arguments, where tests of ordinary sizes say
nothing."""
import math
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import lines_ref as ref
from test_lines_gpu import attn_case, check_attn, fault, lines_case, rope_inputs, run_plan

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


# ---- lines_plan

FRESH = """
import random, sys
sys.path[:0] = [{root!r} + "/tests", {root!r} + "/comfyui-drama3_b200"]
import torch
import lines_ref as ref
from test_lines_gpu import check_plan, fault, lines_case, run_plan
cuda = torch.device("cuda", 0)
for lines in (3007, 3008, 3050, 3071, 3072):
    rng = random.Random(lines)
    lengths = [rng.randrange(0, 40) for _ in range(lines)]
    counts = [rng.randrange(0, 3) for _ in range(lines)]
    table, free, used, tokens = lines_case(lengths, counts, 16, 0, seed=lines)
    _, p = run_plan(cuda, lengths, counts, table, free, used, 16, tokens, 0)
    check_plan(p, ref.plan(lengths, counts, table, free, used, 16, tokens, 0), table)
    assert fault() == 0
print("planned")
"""


def test_plan_of_line_counts_around_48_kb_of_shared_memory(cuda):
    # in a process of its own: a plan of more lines raises the kernel's ceiling for all later ones
    run = subprocess.run([sys.executable, "-c", FRESH.format(root=str(ROOT))], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0 and run.stdout.endswith("planned\n"), run.stderr[-2000:]


@pytest.mark.parametrize("lengths,counts,page,prefix", [
    ([5, 0], [1, 2], 2 ** 31 - 1, 0), ([2 ** 30 - 1], [3], 2 ** 30, 1), ([7], [2], 16, 2 ** 31 - 1),
    ([0, 100], [1, 0], 64, 2 ** 31 - 100)])
def test_plan_of_sums_near_32_bits(cuda, lengths, counts, page, prefix):
    table, free, used, tokens = lines_case(lengths, counts, page, 1)
    _, p = run_plan(cuda, lengths, counts, table, free, used, page, tokens, prefix)
    want = ref.plan(lengths, counts, table, free, used, page, tokens, prefix)
    for name in ("slots", "positions", "line", "cu", "lengths", "used"):
        assert getattr(p, name).tolist() == want[name], name
    assert p.table.tolist() == table and fault() == 0
    work = p.work.tolist()
    at, place = (16 + tokens + 3) & ~3, 0
    assert work[0] == 1 and work[3] == prefix and work[4] == -(-prefix // 128) and work[1] == sum(n > 0 for n in counts)
    live = [b for b, n in enumerate(counts) if n]
    for u, b in enumerate(live):  # a unit per line: few tokens, which see the prefix and their own
        end = lengths[b] + counts[b]
        tiles = work[4] + -(-end // 128)
        assert work[at + 8 * u:at + 8 * u + 8] == [b, want["cu"][b], counts[b], place + 3, tiles, lengths[b] + 1, end, work[4]]
        place += 3 + tiles
    assert work[2] == place


# ---- qk_norm_rope

@pytest.mark.parametrize("strided", [0, 1])
def test_norm_rope_axis_past_the_one_row_of_positions(cuda, strided):
    from drama3_b200 import kernels
    q, k, v, qw, kw, rotary, pos, _ = rope_inputs(cuda, 6, 4, 2, 128, 64, 1, torch.float32, 3, strided)
    axes = torch.zeros(32, dtype=torch.uint8, device=cuda)
    same = kernels.qk_norm_rope(q, k, rotary, pos, q_weight=qw, k_weight=kw)
    got = kernels.qk_norm_rope(q, k, rotary, pos.view(1, -1), q_weight=qw, k_weight=kw, axes=axes)
    assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1]) and fault() == 0
    axes[5], axes[31] = 1, 255  # rows that the positions do not have: these pairs stay as they are
    got = kernels.qk_norm_rope(q, k, rotary, pos.view(1, -1), q_weight=qw, k_weight=kw, axes=axes)
    assert fault() == 128
    unturned = rotary.clone()
    unturned[:, [5, 31]] = torch.tensor([1.0, 0.0], device=cuda)
    want = kernels.qk_norm_rope(q, k, unturned, pos, q_weight=qw, k_weight=kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- lines_attention

@pytest.mark.parametrize("kept,prefix,lines", [(300, 0, 1), (5000, 0, 60), (40, 30000, 3)])
def test_attention_fp16_small_weights_beside_a_large_one(cuda, kept, prefix, lines):
    """The weights of all keys but the first are exp(-17.25), under float16's smallest step beside the first one's 1.
    A weight is rounded by half a unit in the last place, or by half of float16's smallest step, 2^-25, where the largest
    weight is held as 2^7 or more; so to the tolerance of tests/test_lines_gpu.py comes 2^-32 sum |V|."""
    from drama3_b200 import kernels
    D = 64
    q, kc, vc, plan, pt = attn_case(cuda, 4, 1, D, torch.float16, 128, [kept] * lines, [1] * lines, prefix, poison=False)
    q[:], kc[:] = 0.0, 0.0
    q[..., 0] = 17.25
    vc.abs_()
    for b in range(lines):
        first = (pt[0], 0) if prefix else (plan.table[b, 0], 0)
        kc[int(first[0]), 0, :, 0] = 1.0
        vc[int(first[0]), 0] = 0.0
    got, lse = kernels.lines_attention(q, kc, vc, plan, prefix_table=pt, scale=1.0, lse=True)
    args = ([kept] * lines, [1] * lines, plan.table, prefix, pt, 1.0)
    want, want_lse, bound = ref.attention(q, kc, vc, *args)
    total = ref.attention(torch.zeros_like(q), kc, vc, *args)[2] * (prefix + kept + 1)  # equal weights: sum |V| / keys
    tol = 2.2 * 2.0 ** -11 * bound + 2.0 ** -24 + 2.0 ** -32 * total
    err = (got.double() - want).abs()
    assert fault() == 0 and (err <= tol).all(), float((err / tol).max())
    assert ((lse.double() - want_lse).abs() <= 2e-5 + 2.0 ** -21 * want_lse.abs()).all()


def test_attention_op_refuses_a_cache_of_other_pages(cuda):
    """The op is given a work list without the sizes that it was made for, except in the list itself."""
    import drama3_b200.ops  # noqa: F401
    kept, counts, prefix = [40, 3], [5, 70], 100
    q, kc, vc, plan, pt = attn_case(cuda, 16, 4, 128, torch.bfloat16, 32, kept, counts, prefix, poison=False)
    kc, vc = (c.reshape(-1, 16, 4, 128) for c in (kc, vc))  # the same memory as pages of 16
    torch.ops.drama3_b200.lines_attention(q, kc, vc, plan.table, plan.work, 4, pt)
    assert fault() == 256


def test_attention_refused_by_the_kernel_gives_rows_of_nothing(cuda, monkeypatch):
    """A plan that only the GPU can tell to be another pass's: zeros and lse -inf beside the fault bit, not whatever the
    outputs' memory held."""
    from drama3_b200 import kernels
    kept, counts = [60, 20], [1, 1]
    q, kc, vc, plan, pt = attn_case(cuda, 8, 2, 64, torch.bfloat16, 16, kept, counts, 0, spare=3)
    empty, empty_like = torch.empty, torch.empty_like

    def filled(t):
        return t.fill_(math.nan) if t.is_floating_point() else t

    monkeypatch.setattr(torch, "empty", lambda *a, **k: filled(empty(*a, **k)))
    monkeypatch.setattr(torch, "empty_like", lambda *a, **k: filled(empty_like(*a, **k)))
    for work in (torch.zeros_like(plan.work), plan.work.clone()):
        work[2] = 1 << 30  # the cost of a pass that is too long
        out, lse = kernels.lines_attention(q, kc, vc, plan._replace(work=work), prefix_table=pt, lse=True)
        assert fault() == 256 and (out == 0).all() and (lse == -math.inf).all()


def test_attention_from_two_threads_on_one_stream(cuda):
    from drama3_b200 import kernels
    cases, want = [], []
    for seed in range(2):
        q, kc, vc, plan, pt = attn_case(cuda, 16, 2, 128, torch.bfloat16, 16, [300 + seed, 20, 77], [1, 1, 1], 500, seed=seed)
        cases.append((q, kc, vc, plan, pt))
        want.append(kernels.lines_attention(*cases[seed][:4], prefix_table=pt))
    assert not torch.equal(*want)
    got, start = [[], []], threading.Barrier(2, timeout=60)

    def calls(i):
        start.wait()
        for _ in range(500):
            got[i].append(kernels.lines_attention(*cases[i][:4], prefix_table=cases[i][4]))

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert fault() == 0
    for i in range(2):
        assert len(got[i]) == 500 and all(torch.equal(x, want[i]) for x in got[i])


def test_attention_on_two_streams_at_once(cuda):
    from drama3_b200 import kernels
    cases = [attn_case(cuda, 16, 2, 128, torch.bfloat16, 64, [2000 + s] * 8, [1] * 8, 9000, seed=s) for s in range(2)]
    want = [kernels.lines_attention(*c[:4], prefix_table=c[4]) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(kernels.lines_attention(*c[:4], prefix_table=c[4]))
    torch.cuda.synchronize()
    assert fault() == 0
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


# ---- the module

def test_module_reads_the_prefix_that_the_plan_counts(cuda):
    from drama3_b200 import kernels
    from drama3_b200.attention import LinesAttention, LinesCache
    torch.manual_seed(5)
    att = LinesAttention(128, 4, 2, 64, device=cuda, dtype=torch.bfloat16)
    cache = LinesCache(1, 20, 16, 2, 64, 3, 40, 2, cuda)
    rotary = kernels.rotary_table(torch.ones(32), 128, cuda)
    x = torch.randn((50, 128), device=cuda).bfloat16()
    with torch.no_grad():
        # without a prefix, and the prefix itself: there is no table
        plan = cache.plan(torch.ones(3, dtype=torch.int32, device=cuda), 3)
        assert plan.prefix_table is None
        att(x[:3], plan, cache.k[0], cache.v[0], rotary)
        cache.restart()
        att(x, cache.plan_prefix(50), cache.k[0], cache.v[0], rotary)
        plan = cache.plan(torch.ones(3, dtype=torch.int32, device=cuda), 3)
        assert fault() == 0
        want = att(x[:3], plan, cache.k[0], cache.v[0], rotary, cache.prefix_table)
        assert torch.equal(att(x[:3], plan, cache.k[0], cache.v[0], rotary), want) and fault() == 0


# ---- many rows

@pytest.mark.parametrize("spare,together", [(4076, 0), (4077, 1)])
def test_attention_few_lines_in_many_places(cuda, spare, together):
    # 32768 rows of a KV head are the most whose prefix and own units may be apart; one token place more
    kept, counts, prefix = [9 + b for b in range(20)], [1] * 20, 300
    case = attn_case(cuda, 8, 1, 64, torch.bfloat16, 16, kept, counts, prefix, spare=spare)
    assert int(case[3].work[0]) == together
    check_attn(cuda, case, kept, counts, prefix)


@pytest.mark.parametrize("lines,together", [(4096, 0), (4097, 1)])
def test_attention_thousands_of_lines(cuda, lines, together):
    from drama3_b200 import kernels
    prefix, D, hq = 200, 64, 8
    kept = [(7 * b) % 15 for b in range(lines)]
    q, kc, vc, plan, pt = attn_case(cuda, hq, 1, D, torch.bfloat16, 16, kept, [1] * lines, prefix, spare=0)
    work = plan.work[:2].tolist()
    assert work == ([1, lines] if together else [0, lines + lines // 16])  # 16 tokens of 8 heads to a tile of rows
    got, lse = kernels.lines_attention(q, kc, vc, plan, prefix_table=pt, lse=True)
    k, v = (torch.cat((c[pt.long()].flatten(0, 1)[:prefix, 0].expand(lines, -1, -1), c[plan.table[:, 0].long()][:, :, 0]),
                      1).double() for c in (kc, vc))  # the prefix, then the line's one page
    seen = torch.arange(prefix + 16, device=cuda)[None] <= prefix + torch.tensor(kept, device=cuda)[:, None]
    v = torch.where(seen[..., None], v, torch.zeros_like(v))
    s = (q.double() @ k.transpose(1, 2) / math.sqrt(D)).where(seen[:, None], -math.inf)
    p = s.softmax(-1)
    assert fault() == 0
    assert ((got.double() - p @ v).abs() <= 2.2 * 2.0 ** -8 * (p @ v.abs())).all()
    assert ((lse.double() - s.logsumexp(-1)).abs() <= 2e-5 + 2.0 ** -21 * s.logsumexp(-1).abs()).all()


def test_attention_of_no_tokens(cuda):
    from drama3_b200 import kernels
    kept = [20, 3]
    q, kc, vc, plan, pt = attn_case(cuda, 8, 2, 64, torch.bfloat16, 16, kept, [0, 0], 40)
    out, lse = kernels.lines_attention(q, kc, vc, plan, prefix_table=pt, lse=True)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8) and fault() == 0
