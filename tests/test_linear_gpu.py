"""The linear half of a hybrid decoder on the GPU (lines_conv, lines_delta, gated_norm, add_norm) against its plain
restatements in tests/linear_ref.py.

Tolerances, from the sizes that the restatements give; half a step of a type is 2^-8 (bf16), 2^-11 (fp16), 2^-24 (fp32) of
the value. Every output is rounded once: half a step of it. On top of that:
- conv: W + 1 products summed in 32 bits, (W + 2) 2^-24 of the terms' size; SiLU's slope is below 1.1, and its fast form (rows
  of 16 bits) is off by (2 + |y|) 2^-22 of the value, which |y| <= 16 (past that a value is zero or y itself) makes 2^-17.
- delta: with W_t the size of a row of the state, a chunk's products each sum at most 128 terms in 32 bits (128 x 2^-24 =
  2^-17 of the size) of factors held as two fp16 terms (2^-22 each, 2^-21 both); three such products follow one another, so
  3 (2^-17 + 2^-21) < 2^-15 for the state and for what an output takes from it. An output's own two products take the state, what
  is left of the query and the weights of the values rounded to fp16: 2^-11 of each factor, at most two of them in a product,
  2^-10 of the size.
- norms: a mean of D squares in 32 bits is off by (D + 4) 2^-24 of it, its root by half of that, and a dozen operations by
  2^-20: (D / 2 + 16) 2^-24 of the value. The joined sum: 2^-21 of its terms' size plus the norm's share of x's term, and the
  normed row that much of the terms' size over the row's root mean square."""
import threading

import pytest
import torch

import linear_ref as ref

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}  # half of fp16's smallest step
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def fault():
    from drama3_b200._lib import take_fault
    return take_fault()


def plan_of(counts, spare, device):
    """What the operators read of a plan for these tokens and `spare` places behind them."""
    from drama3_b200 import kernels
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    line = [b for b, n in enumerate(counts) for _ in range(n)] + [-1] * spare
    i32 = lambda values: torch.tensor(values, dtype=torch.int32, device=device)  # noqa: E731
    return cu, kernels.LinesPlan(None, None, None, i32(line), i32(cu), None, None, None, 64, 1)


def generator(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def near(got, want, tolerance, what):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - tolerance
    assert not (off > 0).any() and got.isfinite().all(), f"{what}: {int((off > 0).sum())} of {off.numel()} off, worst by {float(off.max())}"


# ---- lines_conv

CONV_LINES = [([1] * 5, 0), ([1], 3), ([0, 2, 0, 3, 1, 4, 0], 1), ([33, 0, 64, 31, 1, 130], 5), ([300], 0), ([0, 0], 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C,W,strided", [(256, 4, False), (264, 4, True), (1048, 3, True), (64, 2, False), (77, 4, False),
                                         (96, 8, True), (8, 5, False)])
@pytest.mark.parametrize("counts,spare", CONV_LINES)
def test_conv(cuda, dtype, C, W, strided, counts, spare):
    from drama3_b200 import kernels
    g = generator(cuda, 1)
    cu, plan = plan_of(counts, spare, cuda)
    T = cu[-1] + spare
    x = torch.randn((T, C + 40 if strided else C), generator=g, device=cuda).to(dtype)[:, 16 if strided else 0:][:, :C]
    w_type = torch.float32 if strided else dtype
    w = torch.randn((C, 1, W) if strided else (C, W), generator=g, device=cuda).to(w_type)
    bias = torch.randn(C, generator=g, device=cuda).to(w_type) if strided else None
    state = torch.randn((len(counts), W - 1, C), generator=g, device=cuda).to(dtype)
    silu = W != 3
    want, after, size = ref.conv(x, w, state, cu, bias, silu)
    out = kernels.lines_conv(x, w, state, plan, bias=bias, silu=silu)
    error = 1.1 * (W + 2) * 2.0 ** -24 * size + 2.0 ** -17 * want.abs() * (dtype != torch.float32) + 2.0 ** -21 * want.abs()
    near(out, want, (1 + HALF[dtype]) * error + HALF[dtype] * want.abs() + TINY[dtype], "out")
    assert torch.equal(state.double(), after)
    assert not out[cu[-1]:].any() and fault() == 0


def test_conv_nothing_of_another_line_or_of_places_behind(cuda):
    from drama3_b200 import kernels
    counts, spare, C = [3, 40, 2, 70, 1], 9, 64
    cu, plan = plan_of(counts, spare, cuda)
    g = generator(cuda, 2)
    x = torch.randn((cu[-1] + spare, C), generator=g, device=cuda).to(torch.bfloat16)
    w = torch.randn((C, 4), generator=g, device=cuda).to(torch.bfloat16)
    state = torch.randn((5, 3, C), generator=g, device=cuda).to(torch.bfloat16)
    bad_x, bad_state = x.clone(), state.clone()
    bad_x[cu[-1]:] = float("nan")
    bad_x[cu[1]:cu[2]] = float("inf")
    bad_state[1] = float("nan")
    good = kernels.lines_conv(x, w, state, plan)
    got = kernels.lines_conv(bad_x, w, bad_state, plan)
    keep = [t for t in range(x.shape[0]) if not cu[1] <= t < cu[2]]
    assert torch.equal(got[keep], good[keep]) and torch.equal(bad_state[[0, 2, 3, 4]], state[[0, 2, 3, 4]])


@pytest.mark.parametrize("cuts", [[5], [1, 2, 3, 4], [31, 33], [64]])
def test_conv_passes_in_pieces_are_one(cuda, cuts):
    from drama3_b200 import kernels
    g = generator(cuda, 3)
    n, C = 100, 128
    x = torch.randn((n, C), generator=g, device=cuda).to(torch.bfloat16)
    w = torch.randn((C, 4), generator=g, device=cuda)
    whole, pieces = (torch.zeros((1, 3, C), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    want = kernels.lines_conv(x, w, whole, plan_of([n], 0, cuda)[1])
    ends = [0, *cuts, n]
    got = torch.cat([kernels.lines_conv(x[a:b], w, pieces, plan_of([b - a], 0, cuda)[1]) for a, b in zip(ends, ends[1:])])
    assert torch.equal(got, want) and torch.equal(whole, pieces)


# ---- lines_delta

HEADS = [(2, 4, 128, 128), (1, 1, 64, 64), (2, 2, 64, 80), (1, 3, 128, 48), (1, 2, 128, 256), (3, 3, 64, 16)]
FORMS = ["raw", "given", "decay only", "rows as they are"]


def delta_case(device, heads, counts, spare, dtype, form, seed, strided=False, slow=False):
    """q, k, v, decay, state and the keywords; the decays spread from nearly none to nearly everything."""
    Hk, Hv, Dk, Dv = heads
    g = generator(device, seed)
    T = sum(counts) + spare

    def normal(*shape):
        return torch.randn(shape, generator=g, device=device)

    wide = normal(T, 2 * Hk * Dk + Hv * Dv + (8 if strided else 0))
    if form == "rows as they are":
        wide *= Dk ** -0.5
    wide = wide.to(dtype)
    q, k, v = (t.unflatten(1, (h, d)) for t, h, d in zip(wide[:, :2 * Hk * Dk + Hv * Dv].split((Hk * Dk, Hk * Dk, Hv * Dv), 1),
                                                        (Hk, Hk, Hv), (Dk, Dk, Dv)))
    state = normal(len(counts), Hv, Dv, Dk)
    more = {}
    if form == "raw":
        both = normal(T, 2 * Hv + 1).to(dtype)
        more["beta"], decay = both[:, :Hv], both[:, Hv:2 * Hv]
        more["a_log"], more["dt_bias"] = normal(Hv), normal(Hv) - (6 if slow else 2)
    else:
        decay = -torch.exp(normal(T, Hv) * 2 - (6 if slow else 2))
        if form != "decay only":
            more["beta"] = torch.rand((T, Hv), generator=g, device=device)
            if form == "rows as they are":
                more["eps"] = None
                # beta |k|^2 stays below 2, where a correction shrinks what it corrects
                more["beta"] = more["beta"] / k.double().square().sum(-1).amax(0).repeat_interleave(Hv // Hk).clamp(min=1).float()
    return (q, k, v, decay, state), more


def check_delta(device, args, more, cu, plan, scale=None):
    from drama3_b200 import kernels
    q, k, v, decay, state = args
    want, after, size, state_size = ref.delta(q, k, v, decay, state, cu, scale=scale, **more)
    out = kernels.lines_delta(q, k, v, decay, state, plan, scale=scale, **more)
    dtype = q.dtype
    error = (2.0 ** -15 + 2.0 ** -10) * size
    near(out, want, (1 + HALF[dtype]) * error + HALF[dtype] * want.abs() + TINY[dtype], "out")
    near(state, after, 2.0 ** -15 * state_size[..., None].expand_as(after), "state")
    # over a head the errors are as many to either side: the 2-norm of the state's is within 2^-18 of the sizes'
    assert (state.double() - after).norm() <= 2.0 ** -18 * state_size.norm() * max(1, q.shape[2] ** 0.5 / 8)
    assert not out[cu[-1]:].any() and fault() == 0
    return out


DELTA_LINES = [([1] * 5, 0), ([1], 2), ([0, 1, 0, 1], 3), ([2, 0, 5, 1, 3], 0), ([63], 0), ([64], 0), ([65], 1), ([128, 1], 0),
               ([17, 0, 1, 46, 64, 3, 90], 4), ([200, 260], 0), ([0, 0], 3)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("counts,spare", DELTA_LINES)
def test_delta(cuda, dtype, heads, counts, spare):
    cu, plan = plan_of(counts, spare, cuda)
    args, more = delta_case(cuda, heads, counts, spare, dtype, "raw", 4)
    check_delta(cuda, args, more, cu, plan)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("slow", [False, True])
@pytest.mark.parametrize("heads", [(2, 4, 128, 128), (1, 2, 64, 80)])
@pytest.mark.parametrize("counts,spare", [([1, 1, 0, 1], 1), ([130, 1, 70, 0, 200], 3)])
def test_delta_forms(cuda, form, slow, heads, counts, spare):
    cu, plan = plan_of(counts, spare, cuda)
    args, more = delta_case(cuda, heads, counts, spare, torch.bfloat16, form, 5, strided=True, slow=slow)
    check_delta(cuda, args, more, cu, plan, scale=0.3)


@pytest.mark.parametrize("counts", [[1], [300]])
def test_delta_rows_off_16_byte_boundaries(cuda, counts):
    from drama3_b200 import kernels
    cu, plan = plan_of(counts, 0, cuda)
    (q, k, v, decay, state), more = delta_case(cuda, (2, 2, 64, 64), counts, 0, torch.bfloat16, "raw", 6)
    odd = [torch.cat((t[..., :1], t), -1)[..., 1:] for t in (q, k, v)]
    again = state.clone()
    assert torch.equal(kernels.lines_delta(q, k, v, decay, state, plan, **more),
                       kernels.lines_delta(*odd, decay, again, plan, **more)) and torch.equal(state, again)
    long = [torch.zeros(t.numel() + 1, dtype=t.dtype, device=cuda)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    assert all(t.data_ptr() % 16 for t in long)
    first, second = state.clone(), state.clone()
    assert torch.equal(kernels.lines_delta(q, k, v, decay, first, plan, **more),
                       kernels.lines_delta(*long, decay, second, plan, **more)) and torch.equal(first, second)


@pytest.mark.parametrize("counts", [[1, 1], [150, 20]])
@pytest.mark.parametrize("over", ["heads", "tokens"])
def test_delta_rows_that_heads_or_tokens_share(cuda, over, counts):
    cu, plan = plan_of(counts, 0, cuda)
    args, more = delta_case(cuda, (2, 4, 64, 64), counts, 0, torch.bfloat16, "raw", 13)
    shared = [(t[:, :1] if over == "heads" else t[:1]).expand_as(t) for t in args[:3]]
    assert all(0 in t.stride() for t in shared)
    check_delta(cuda, (*shared, *args[3:]), more, cu, plan)


@pytest.mark.parametrize("counts", [[1, 1], [150, 200]])
def test_delta_extremes(cuda, counts):
    """Decays of nothing and of everything, above 0 (which count as 0), rows of zeros, strengths of 0 and 1, the same key over
    and over."""
    cu, plan = plan_of(counts, 0, cuda)
    (q, k, v, decay, state), _ = delta_case(cuda, (2, 2, 128, 64), counts, 0, torch.bfloat16, "given", 7)
    T = sum(counts)
    beta = torch.rand(decay.shape, generator=generator(cuda, 8), device=cuda)
    q, k, v = (t.clone() for t in (q, k, v))
    decay[::7], decay[1::7], decay[2::7] = -float("inf"), 0.0, 3.0
    decay[T // 2:, 1] = 0.0
    beta[::5], beta[1::5] = 0.0, 1.0
    k[::9], q[::11], v[::13] = 0, 0, 0
    k[T // 3:T // 2] = k[T // 3]
    check_delta(cuda, (q, k, v, decay, state), dict(beta=beta), cu, plan)


@pytest.mark.parametrize("counts", [[1, 1], [40, 50]])
def test_delta_rows_of_zeros_without_eps(cuda, counts):
    """eps 0: rows of zeros stay zeros, whatever form the call takes."""
    from drama3_b200 import kernels
    cu, plan = plan_of(counts, 0, cuda)
    (q, k, v, decay, state), more = delta_case(cuda, (2, 2, 64, 64), counts, 0, torch.bfloat16, "raw", 26)
    q, k = q.clone(), k.clone()
    q[::3], k[::2] = 0, 0
    out = kernels.lines_delta(q, k, v, decay, state, plan, eps=0.0, **more)
    assert out.isfinite().all() and state.isfinite().all() and not out[::3].any()


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e12, 1e25])
@pytest.mark.parametrize("counts", [[1, 1], [100, 130]])
def test_delta_states_of_any_size(cuda, size, counts):
    """A row of the state far larger or smaller than what is added to it, and rows of all sizes side by side."""
    cu, plan = plan_of(counts, 0, cuda)
    (q, k, v, decay, state), more = delta_case(cuda, (1, 2, 64, 48), counts, 0, torch.bfloat16, "given", 9, slow=True)
    state *= size ** torch.rand((1, 2, 48, 1), generator=generator(cuda, 10), device=cuda)
    from drama3_b200 import kernels
    want, after, out_size, state_size = ref.delta(q, k, v, decay, state, cu, **more)
    out = kernels.lines_delta(q, k, v, decay, state, plan, **more)
    near(state, after, 2.0 ** -15 * state_size[..., None].expand_as(after) + 2.0 ** -126, "state")
    near(out, want, (2.0 ** -15 + 2.0 ** -10) * 1.01 * out_size + HALF[q.dtype] * want.abs() + 2.0 ** -126, "out")


@pytest.mark.parametrize("counts", [[1, 1, 1, 1, 1], [3, 40, 2, 170, 1]])
def test_delta_nothing_of_another_line_or_of_places_behind(cuda, counts):
    from drama3_b200 import kernels
    spare = 9
    cu, plan = plan_of(counts, spare, cuda)
    args, more = delta_case(cuda, (2, 4, 128, 64), counts, spare, torch.bfloat16, "raw", 11)
    more = {name: t.clone() for name, t in more.items()}
    args = tuple(t.clone() for t in args)
    bad = [t.clone() for t in args]
    bad_more = {**more, "beta": more["beta"].clone()}
    for t, value in zip((*bad[:4], bad_more["beta"]), (float("nan"), float("inf"), float("nan"), float("nan"), -float("inf"))):
        t[cu[-1]:] = value
        t[cu[1]:cu[2]] = value
    bad[4][1] = float("nan")
    good = kernels.lines_delta(*args, plan, **more)
    got = kernels.lines_delta(*bad, plan, **bad_more)
    keep = [t for t in range(good.shape[0]) if not cu[1] <= t < cu[2]]
    others = [0, 2, 3, 4]
    assert torch.equal(got[keep], good[keep]) and torch.equal(bad[4][others], args[4][others])
    assert not bad[4][1].isfinite().any() and fault() == 0


def test_delta_lines_without_tokens_keep_their_state(cuda):
    from drama3_b200 import kernels
    for counts in ([0, 1, 0], [0, 90, 0, 0, 70]):
        cu, plan = plan_of(counts, 0, cuda)
        args, more = delta_case(cuda, (1, 2, 64, 64), counts, 0, torch.bfloat16, "raw", 12)
        idle = [b for b, n in enumerate(counts) if n == 0]
        args[4][idle] = float("nan")
        before = args[4].clone()
        out = kernels.lines_delta(*args, plan, **more)
        assert torch.equal(args[4][idle].view(torch.int32), before[idle].view(torch.int32)) and out.isfinite().all()


def test_delta_no_tokens(cuda):
    from drama3_b200 import kernels
    cu, plan = plan_of([0, 0], 0, cuda)
    args, more = delta_case(cuda, (1, 2, 64, 64), [0, 0], 0, torch.bfloat16, "raw", 13)
    before = args[4].clone()
    assert kernels.lines_delta(*args, plan, **more).shape == (0, 2, 64) and torch.equal(args[4], before)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("with_beta", [True, False])
def test_delta_pieces_and_single_tokens_are_one_pass(cuda, dtype, with_beta):
    """A text read at once, in two passes cut anywhere, and a text whose last tokens come one by one: the same up to 32-bit
    rounding, each within the tolerance of the restatement (a state's 2^-15 and an output's 2^-10 and half a step)."""
    from drama3_b200 import kernels
    n, heads = 203, (2, 4, 128, 128)
    (q, k, v, decay, state), more = delta_case(cuda, heads, [n], 0, dtype, "raw" if with_beta else "decay only", 14)
    want, after, size, state_size = ref.delta(q, k, v, decay, state, [0, n], **more)
    for ends in ([0, n], [0, 77, n], [0, 196, *range(197, n + 1)]):
        s, outs = state.clone(), []
        for a, b in zip(ends, ends[1:]):
            cut = {name: t[a:b] if t.dim() == 2 else t for name, t in more.items()}
            outs.append(kernels.lines_delta(q[a:b], k[a:b], v[a:b], decay[a:b], s, plan_of([b - a], 0, cuda)[1], **cut))
        near(torch.cat(outs), want, 1.01 * (2.0 ** -15 + 2.0 ** -10) * size + HALF[dtype] * want.abs() + TINY[dtype], "out")
        near(s, after, 2.0 ** -15 * state_size[..., None].expand_as(after), "state")


@pytest.mark.parametrize("counts", [[1] * 20, [700, 3, 0, 500, 65]])
def test_delta_twice_is_the_same(cuda, counts):
    from drama3_b200 import kernels
    cu, plan = plan_of(counts, 0, cuda)
    args, more = delta_case(cuda, (2, 4, 128, 128), counts, 0, torch.bfloat16, "raw", 15)
    results = []
    for _ in range(3):
        state = args[4].clone()
        results.append((kernels.lines_delta(*args[:4], state, plan, **more), state))
    for out, state in results[1:]:
        assert torch.equal(out, results[0][0]) and torch.equal(state, results[0][1])


def test_delta_long(cuda):
    """Thousands of tokens of a slowly forgetting head, next to short lines."""
    counts = [5000, 1, 0, 333]
    cu, plan = plan_of(counts, 7, cuda)
    args, more = delta_case(cuda, (1, 2, 128, 128), counts, 7, torch.bfloat16, "raw", 16, slow=True)
    check_delta(cuda, args, more, cu, plan)


def test_delta_many_lines(cuda):
    counts = [b % 3 for b in range(1500)]
    cu, plan = plan_of(counts, 2, cuda)
    args, more = delta_case(cuda, (1, 1, 64, 16), counts, 2, torch.float16, "raw", 17)
    check_delta(cuda, args, more, cu, plan)


def test_delta_first_call_of_a_thread(cuda):
    """A thread that has made no CUDA call yet, whose first one encodes a tensor map."""
    from drama3_b200 import kernels
    cu, plan = plan_of([100, 30], 0, cuda)
    args, more = delta_case(cuda, (1, 2, 64, 64), [100, 30], 0, torch.bfloat16, "raw", 27)
    want, got = kernels.lines_delta(*args[:4], args[4].clone(), plan, **more), []
    state = args[4].clone()
    thread = threading.Thread(target=lambda: got.append(kernels.lines_delta(*args[:4], state, plan, **more)))
    thread.start()
    thread.join()
    assert got and torch.equal(got[0], want)


def test_delta_parts_of_a_long_pass_follow_one_another(cuda):
    """A pass of more chunks than the scratch of one part holds: two parts, each from the states that the one before leaves."""
    from drama3_b200 import _lib, kernels
    heads = (16, 64, 64, 16)
    chunk = _lib.lib().d3_lines_delta_workspace(64, 1, 16, 64, 64)
    n = (384 << 20) // chunk * 64 + 100
    assert _lib.lib().d3_lines_delta_workspace(n, 1, 16, 64, 64) <= 384 << 20
    counts = [n - 130, 70]
    cu, plan = plan_of(counts, 60, cuda)
    (q, k, v, decay, state), more = delta_case(cuda, heads, counts, 60, torch.bfloat16, "raw", 28)
    out = kernels.lines_delta(q, k, v, decay, state, plan, **more)
    want = []
    again = delta_case(cuda, heads, counts, 60, torch.bfloat16, "raw", 28)[0][4]
    s0, s1 = again[:1].clone(), again[1:].clone()
    for a, b, s in ((0, 1000, s0), (1000, cu[1], s0), (cu[1], cu[2], s1)):  # the same texts, in other pieces
        cut = {name: t[a:b] if t.dim() == 2 else t for name, t in more.items()}
        want.append(kernels.lines_delta(q[a:b], k[a:b], v[a:b], decay[a:b], s, plan_of([b - a], 0, cuda)[1], **cut))
    want = torch.cat(want)
    # both within the tolerance of the definition: twice its share of the rows' size, which the norms stand for
    size = want.double().norm()
    assert (out[:cu[2]].double() - want.double()).norm() <= 2 * (HALF[torch.bfloat16] + 2.0 ** -10) * size and not out[cu[2]:].any()
    assert (state.double() - torch.cat((s0, s1)).double()).norm() <= 2 * 2.0 ** -15 * state.double().norm() and fault() == 0


def test_delta_from_two_threads_on_one_stream(cuda):
    from drama3_b200 import kernels
    cases = []
    for seed in (18, 19):
        cu, plan = plan_of([300, 41], 0, cuda)
        cases.append((plan, *delta_case(cuda, (2, 4, 64, 64), [300, 41], 0, torch.bfloat16, "raw", seed)))
    wants = [kernels.lines_delta(*args[:4], args[4].clone(), plan, **more) for plan, args, more in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        plan, args, more = cases[i]
        for _ in range(50):
            if not torch.equal(kernels.lines_delta(*args[:4], args[4].clone(), plan, **more), wants[i]):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and fault() == 0


# ---- the norms

NORM_ROWS = [(1, 1, 128), (16, 32, 128), (5, 3, 256), (7, 8, 64), (9, 5, 80), (3, 3, 129), (2, 2, 1024), (2, 1, 1500), (700, 40, 128),
             (4, 2, 1), (90, 8, 512)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,D", NORM_ROWS)
@pytest.mark.parametrize("activation,unit,strided", [("silu", False, True), ("sigmoid", True, False)])
def test_gated_norm(cuda, dtype, T, H, D, activation, unit, strided):
    from drama3_b200 import kernels
    g = generator(cuda, 20)
    x = torch.randn((T, H, D), generator=g, device=cuda).to(dtype)
    z = (3 * torch.randn((T, H, 2 * D if strided else D), generator=g, device=cuda)).to(dtype)[..., -D:]
    w = torch.randn(D, generator=g, device=cuda).to(torch.float32 if strided else dtype)
    if strided:
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    want = ref.gated(x, z, w, 1e-5, int(unit), activation)
    got = kernels.gated_norm(x, z, w, eps=1e-5, unit_offset=unit, activation=activation)
    near(got, want, ((D / 2 + 16) * 2.0 ** -24 * 1.01 + HALF[dtype]) * want.abs() + TINY[dtype], "out")


def test_gated_norm_extremes(cuda):
    from drama3_b200 import kernels
    x = torch.ones((4, 1, 128), dtype=torch.float32, device=cuda)
    x[0], x[1], x[2, 0, 5] = 0, 1e-15, float("nan")
    z = torch.tensor([-200.0, 200.0, 0.0, -1000.0], device=cuda)[:, None, None].expand(4, 1, 128).contiguous()
    w = torch.ones(128, device=cuda)
    got = kernels.gated_norm(x, z, w)
    near(got[:2], ref.gated(x[:2], z[:2], w), 2.0 ** -17 * ref.gated(x[:2], z[:2], w).abs() + 1e-30, "out")
    assert got[2].isnan().all() and got[3].abs().max() == 0


WIDTHS = [(1, 2048), (16, 2048), (300, 2048), (33, 1000), (5, 333), (4, 8192), (3, 12000), (2, 20000), (6, 8), (3, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,W", WIDTHS)
@pytest.mark.parametrize("post,gate,unit", [(False, None, False), (True, "row", True), (True, "channel", False),
                                            (False, "each", True)])
def test_add_norm(cuda, dtype, T, W, post, gate, unit):
    from drama3_b200 import kernels
    g = generator(cuda, 21)
    w_type = torch.float32 if gate == "row" else dtype

    def normal(*shape, to=dtype):
        return torch.randn(shape, generator=g, device=cuda).to(to)

    x, r = normal(T, W + 8)[:, :W], normal(T, W)
    w, p = normal(W, to=w_type), normal(W, to=w_type) if post else None
    z = None if gate is None else normal(*{"row": (T, 1), "channel": (1, W), "each": (T, W)}[gate])
    total, normed, size = ref.join(x, r, w, p, z, 0.5, 1e-5, int(unit))
    got, got_normed = kernels.add_norm(x, r, w, post_weight=p, gate=z, scale=0.5, eps=1e-5, unit_offset=unit)
    part = (W / 2 + 16) * 2.0 ** -24
    error = (2.0 ** -21 + part * post) * size
    near(got, total, 1.01 * error + HALF[dtype] * total.abs() + TINY[dtype], "sum")
    root = torch.sqrt(total.square().mean(-1, keepdim=True) + 1e-5)
    scaled = (error / root + error.norm(dim=-1, keepdim=True) / W ** 0.5 / root ** 2 * total.abs()) * (w.double() + unit).abs()
    near(got_normed, normed, 1.01 * (scaled + part * normed.abs()) + HALF[dtype] * normed.abs() + TINY[dtype], "normed")


def test_add_norm_gate_of_a_view_and_sums_in_float64(cuda):
    """A gate that is a column of another tensor; a sum that cancels; a row of zeros."""
    from drama3_b200 import kernels
    x = torch.randn((4, 256), device=cuda, generator=generator(cuda, 22))
    gate = torch.randn((4, 7), device=cuda, generator=generator(cuda, 23))[:, 3:4]
    r = -(x * gate)
    r[2], x[2] = 0, 0
    w = torch.ones(256, device=cuda)
    got, normed = kernels.add_norm(x, r, w, gate=gate)
    assert (got.abs() <= 2.0 ** -23 * (x * gate).abs()).all() and not normed[2].any() and normed.isfinite().all()


# ---- together

def half_layer(device, lines, tokens, seed):
    """The operators as a layer uses them: the fused projection's output through convolution, attention, gated norm and join."""
    from drama3_b200 import kernels
    Hk, Hv, Dk, Dv = 2, 4, 64, 64
    C, wide = 2 * Hk * Dk + Hv * Dv, Hv * Dv
    g = generator(device, seed)
    normal = lambda *s: torch.randn(s, generator=g, device=device).to(torch.bfloat16)  # noqa: E731
    p = dict(x=normal(tokens, C + wide), residual=normal(tokens, wide), gates=normal(tokens, 2 * Hv), conv=normal(C, 4),
             norm=normal(Dv), join=normal(wide), a_log=normal(Hv).float(), dt=normal(Hv).float() - 3,
             conv_state=normal(lines, 3, C), state=torch.randn((lines, Hv, Dv, Dk), generator=g, device=device))

    def run(plan, p):
        y = kernels.lines_conv(p["x"][:, :C], p["conv"], p["conv_state"], plan)
        q, k, v = (t.unflatten(1, (-1, 64)) for t in y.split((Hk * Dk, Hk * Dk, Hv * Dv), 1))
        o = kernels.lines_delta(q, k, v, p["gates"][:, Hv:], p["state"], plan, beta=p["gates"][:, :Hv], a_log=p["a_log"], dt_bias=p["dt"])
        o = kernels.gated_norm(o, p["x"][:, C:].unflatten(1, (Hv, Dv)), p["norm"])
        return (*kernels.add_norm(o.flatten(1), p["residual"], p["join"]), p["conv_state"], p["state"])

    return p, run


@pytest.mark.parametrize("counts", [[1] * 6, [0, 70, 1, 130]])
def test_together_on_a_side_stream_and_in_a_graph(cuda, counts):
    cu, plan = plan_of(counts, 1, cuda)
    p, run = half_layer(cuda, len(counts), cu[-1] + 1, 24)
    copy = lambda: {name: t.clone() for name, t in p.items()}  # noqa: E731
    first = copy()
    want = [t.clone() for t in run(plan, first)]
    wanted = [want, [t.clone() for t in run(plan, first)]]
    side = copy()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run(plan, side)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    held = copy()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = run(plan, held)
    for expected in wanted:  # the states go on from replay to replay
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, expected))
    del graph
    assert fault() == 0


def test_ops_equal_the_kernels(cuda):
    from drama3_b200 import kernels, ops  # noqa: F401
    o = torch.ops.drama3_b200
    counts = [2, 90, 0]
    cu, plan = plan_of(counts, 1, cuda)
    (q, k, v, decay, state), more = delta_case(cuda, (2, 4, 64, 64), counts, 1, torch.bfloat16, "raw", 25)
    a, b = state.clone(), state.clone()
    assert torch.equal(o.lines_delta(q, k, v, decay, a, plan.cu, plan.line, more["beta"], more["a_log"], more["dt_bias"]),
                       kernels.lines_delta(q, k, v, decay, b, plan, **more)) and torch.equal(a, b)
    x, w = q.flatten(1), torch.ones((128, 4), dtype=torch.bfloat16, device=cuda)
    a, b = (torch.zeros((3, 3, 128), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    assert torch.equal(o.lines_conv(x, w, a, plan.cu, plan.line), kernels.lines_conv(x, w, b, plan)) and torch.equal(a, b)
    ones = torch.ones(64, dtype=torch.bfloat16, device=cuda)
    assert torch.equal(o.gated_norm(q, k, ones), kernels.gated_norm(q, k, ones))
    ones = torch.ones(128, dtype=torch.bfloat16, device=cuda)
    for got, want in zip(o.add_norm(x, k.flatten(1), ones, ones), kernels.add_norm(x, k.flatten(1), ones, ones)):
        assert torch.equal(got, want)
