"""lines_delta over the whole range of its arguments, against the 64-bit restatements of tests/linear_ref.py: corrections that
grow what they correct, token by token and in chunks.

Tolerances. Half a step of a type is 2^-8 (bf16), 2^-11 (fp16) of the value; the multiples of a row's size are those of
tests/test_linear_gpu.py: 2^-15 for the state and what an output takes from it, 2^-10 for factors of an output in 16 bits.
Where a correction grows what it corrects (the token's map of a row of the state, M_t = exp(g) (I - beta k k^T), has a norm
above 1 for beta |k|^2 above 2), it grows what was rounded before as well, and the row of the state may be smaller than what it is
summed from. With M_jt the maps from token j to t, errors are then multiples of
    a row of the state:  N = W_t + |S_0| |M_0t|_F / sqrt(Dk) + sum_j |beta_j v_j| |k_j M_jt|
    an output:           scale (W_t |q_t| + |S_0| |M_0t q_t| + sum_j |beta_j v_j| |k_j M_jt q_t|)
W as in linear_ref.delta, what the row's own sums are; the second terms an error in the first state, of any direction, by the time of
t; the third ones the values' shares. Without growth they are W and W |q| scale but for a factor of about 2. What is below the
smallest normal number of 32 bits, 2^-126, may vanish."""
import pytest
import torch

import linear_ref as ref
from test_linear_gpu import HALF, TINY, delta_case, fault, generator, near, plan_of

pytestmark = pytest.mark.gpu


def sizes(q, k, v, decay, state, cu, beta, eps=1e-6, scale=None):
    """(size of the outputs, of the state's rows) as in the head of this file; the gates given, not raw."""
    Hk, Dk, Hv = q.shape[1], q.shape[2], v.shape[1]
    _, after, out, W = ref.delta(q, k, v, decay, state, cu, beta, eps=eps, scale=scale)
    scale = Dk ** -0.5 if scale is None else scale
    q, k = q.double(), k.double()
    if eps is not None:
        q, k = (x / torch.sqrt(x.square().sum(-1, keepdim=True) + eps) for x in (q, k))
    q, k = (x.repeat_interleave(Hv // Hk, 1) for x in (q, k))
    g, beta = ref.gates(decay, beta)
    out, N, start = out.clone(), W.clone(), state.double().norm(dim=-1)
    for b in range(len(cu) - 1):
        X = torch.eye(Dk, dtype=torch.float64, device=q.device).expand(Hv, Dk, Dk)  # M_0t, and below it the rows k_j M_jt
        values = torch.zeros((Hv, v.shape[2], 0), dtype=torch.float64, device=q.device)
        for t in range(cu[b], cu[b + 1]):
            X = torch.exp(g[t])[:, None, None] * (X - beta[t][:, None, None] * (X @ k[t][..., None]) * k[t][:, None])
            X = torch.cat((X, k[t][:, None]), 1)
            values = torch.cat((values, (beta[t][:, None] * v[t].double()).abs()[..., None]), 2)
            left = (X @ q[t][..., None])[..., 0]
            shares = left[:, :Dk].norm(dim=-1)[:, None] * start[b] + (values @ left[:, Dk:, None].abs())[..., 0]
            out[t] += scale * shares
        if cu[b + 1] > cu[b]:
            N[b] += start[b] * X[:, :Dk].norm(dim=(1, 2))[:, None] / Dk ** 0.5 + (values @ X[:, Dk:].norm(dim=-1)[..., None])[..., 0]
    return out, N


def check(args, cu, plan, **more):
    from drama3_b200 import kernels
    q, k, v, decay, state = args
    dtype = q.dtype
    exact = {**more, "eps": 1e-200} if more.get("eps") == 0 else more  # rows of zeros are zeros
    want, after, _, _ = ref.delta(*args, cu, **exact)
    size, state_size = sizes(*args, cu, **exact)
    assert after.abs().max() < 1e30 and want.abs().max() < (6e4 if dtype == torch.float16 else 1e30)  # the definition's own range
    out = kernels.lines_delta(*args, plan, **more)
    near(out, want, (1 + HALF[dtype]) * (2.0 ** -15 + 2.0 ** -10) * size + HALF[dtype] * want.abs() + TINY[dtype] + 2.0 ** -126, "out")
    near(state, after, 2.0 ** -15 * state_size[..., None].expand_as(after) + 2.0 ** -126, "state")
    # in the 2-norm: a result's own rounding, uniform within half a step (a root of 1/3 of it, a tenth more for the finite sample), and
    # that of two factors to 16 bits, as many errors to either side: sqrt(2 / 3) 2^-12
    assert (out.double() - want).norm() <= HALF[dtype] * 3 ** -0.5 * 1.1 * want.norm() + 2.0 ** -12 * size.norm()
    assert fault() == 0


GROWING = [  # keys, |k|^2, tokens of each line, rows; a line of 16 tokens alone and four a line go token by token, the others in chunks
    ("random", 5.0, [16], torch.bfloat16), ("random", 5.0, [64], torch.bfloat16), ("random", 5.0, [90, 0, 130, 1], torch.bfloat16),
    ("random", 10.0, [4, 1, 3], torch.bfloat16), ("random", 10.0, [64], torch.bfloat16), ("random", 10.0, [30, 33, 2], torch.bfloat16),
    ("repeated", 5.0, [3, 4, 4], torch.bfloat16), ("repeated", 5.0, [17], torch.bfloat16), ("repeated", 5.0, [20, 1, 24], torch.bfloat16),
    ("repeated", 10.0, [16], torch.bfloat16), ("repeated", 10.0, [17], torch.bfloat16), ("repeated", 10.0, [20, 3, 20], torch.bfloat16),
    ("random", 3.0, [8], torch.float16), ("random", 3.0, [40], torch.float16), ("repeated", 2.5, [18], torch.float16)]


@pytest.mark.parametrize("heads", [(2, 4, 128, 128), (1, 2, 64, 48)])
@pytest.mark.parametrize("keys,length2,counts,dtype", GROWING)
def test_delta_corrections_that_grow(cuda, heads, keys, length2, counts, dtype):
    """Keys as they are with beta 1: a correction overshoots by |k|^2 - 1."""
    Hk, Hv, Dk, Dv = heads
    spare = int(len(counts) > 1)
    cu, plan = plan_of(counts, spare, cuda)
    g, T = generator(cuda, 31), sum(counts) + spare
    normal = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    k = normal(1 if keys == "repeated" else T, Hk, Dk).expand(T, Hk, Dk)
    k = (k * (length2 ** 0.5 / k.norm(dim=-1, keepdim=True))).to(dtype)
    q = normal(T, Hk, Dk)
    q = (0.5 * q / q.norm(dim=-1, keepdim=True)).to(dtype) if keys == "random" else (k.float() + 0.05 * q).to(dtype)
    args = (q, k, normal(T, Hv, Dv).to(dtype), -0.01 * torch.rand((T, Hv), generator=g, device=cuda), normal(len(counts), Hv, Dv, Dk))
    check(args, cu, plan, beta=torch.ones((T, Hv), device=cuda), eps=None, scale=0.1 if dtype == torch.bfloat16 else 2.0 ** -6)


@pytest.mark.parametrize("counts", [[12], [20], [40, 0, 50]])
def test_delta_strengths_past_two(cuda, counts):
    """Keys of length 1 and strengths given up to 4."""
    cu, plan = plan_of(counts, 0, cuda)
    g, T = generator(cuda, 32), sum(counts)
    normal = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    q, k, v = (normal(T, 2, 128).bfloat16() for _ in range(3))
    args = (q, k, v, -0.1 * torch.rand((T, 2), generator=g, device=cuda), normal(len(counts), 2, 128, 128))
    check(args, cu, plan, beta=4 * torch.rand((T, 2), generator=g, device=cuda))


@pytest.mark.parametrize("heads", [(2, 4, 64, 48), (2, 2, 128, 64)])
@pytest.mark.parametrize("counts,eps", [([1, 1, 1], 0.0), ([1, 1, 1], 1e-6), ([5, 0, 4, 3], 0.0), ([5, 0, 4, 3], 1e-6), ([100, 130], 0.0),
                                        ([100, 130], 1e-6)])
def test_delta_rows_of_any_size(cuda, heads, counts, eps):
    """Queries and keys whose squares leave 32 bits to either side, next to ordinary ones; rows of zeros."""
    Hk, Hv, Dk, Dv = heads
    cu, plan = plan_of(counts, 0, cuda)
    g, T = generator(cuda, 33), sum(counts)
    normal = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    powers = torch.tensor([20.0, -33.0, 36.0, 0.0, -24.0, 25.0, -12.0, 1.0, -20.0], device=cuda)
    turn = torch.arange(T * Hk, device=cuda).view(T, Hk, 1)
    q, k = ((normal(T, Hk, Dk) * 10.0 ** powers[(turn * step + 1) % 9]).bfloat16() for step in (2, 1))
    k[3::7, 0], q[4::5, 1] = 0, 0
    assert k.float().square().sum(-1).isinf().any() and q.isfinite().all() and k.isfinite().all()
    args = (q, k, normal(T, Hv, Dv).bfloat16(), -torch.exp(normal(T, Hv) - 2), normal(len(counts), Hv, Dv, Dk))
    beta = torch.rand((T, Hv), generator=g, device=cuda)
    check(args, cu, plan, beta=beta, eps=eps)


@pytest.mark.parametrize("heads", [(2, 4, 128, 128), (1, 2, 64, 48)])
@pytest.mark.parametrize("with_beta", [True, False])
@pytest.mark.parametrize("counts", [[3, 2, 4], [14], [100, 130]])
def test_delta_values_far_larger_than_others(cuda, heads, with_beta, counts):
    """Values of 1e9 among ordinary ones: tokens before them keep their bits, tokens after them forget them as the decays say.

    Besides the usual terms, for tokens from a large value on: an entry of P T, which decays may make that small, ends at the second
    term's smallest step, 2^-16 of e5m2, rounded to half of it and held 2^11 times, where the row's largest entry is held as 2^13 at
    least: off by 2^-17 / 2^11 / 2^13 = 2^-41 of that, which is at most scale |q| here (beta and |k| at most 1: corrections
    shrink). It is multiplied by R_j = v_j - S k_j, at most |v_j| + W_j."""
    from drama3_b200 import kernels
    Hk, Hv, Dk, Dv = heads
    cu, plan = plan_of(counts, 0, cuda)
    g, T = generator(cuda, 34), sum(counts)
    normal = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    q, k, v = normal(T, Hk, Dk).bfloat16(), normal(T, Hk, Dk).bfloat16(), normal(T, Hv, Dv)
    large = torch.rand((T, Hv, Dv), generator=g, device=cuda) < 0.02
    args = (q, k, torch.where(large, 1e9 * v, v).bfloat16(), -torch.exp(2 * normal(T, Hv)), normal(len(counts), Hv, Dv, Dk))
    more = dict(beta=torch.rand((T, Hv), generator=g, device=cuda)) if with_beta else {}
    want, after, size, state_size = ref.delta(*args, cu, **more)
    out = kernels.lines_delta(*args, plan, **more)
    half, length = HALF[torch.bfloat16], (q.double() / torch.sqrt(q.double().square().sum(-1, keepdim=True) + 1e-6)).norm(dim=-1)
    length = Dk ** -0.5 * length.repeat_interleave(Hv // Hk, 1)[..., None]  # scale |q|
    left = args[2].double().abs() + size / length
    left = torch.cat([left[a:b].cumsum(0) for a, b in zip(cu, cu[1:])])
    near(out, want, (1 + half) * ((2.0 ** -15 + 2.0 ** -10) * size + 2.0 ** -41 * length * left) + half * want.abs(), "out")
    near(args[4], after, 2.0 ** -15 * state_size[..., None].expand_as(after), "state")
    assert fault() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(2, 4, 128, 128), (1, 2, 64, 64), (8, 16, 128, 256)])
@pytest.mark.parametrize("form", ["raw", "given", "decay only", "raw without beta", "raw without dt_bias"])
@pytest.mark.parametrize("counts", [[1] * 7, [90, 0, 200, 33]])
def test_delta_outputs_are_as_near_as_their_rounding(cuda, dtype, heads, form, counts):
    """Outputs in the 2-norm, over tokens, heads and channels: what rounding the exact ones leaves, and apart from that at most the
    last bit of P T's second terms, 2^-15 of them, of which the root mean square is below 2^-16. A term is a query and a key of
    random directions times a value, so the size over sqrt(Dk), a product's largest being about sqrt(10) of that."""
    from drama3_b200 import kernels
    cu, plan = plan_of(counts, 1, cuda)
    args, more = delta_case(cuda, heads, counts, 1, dtype, form.split(" without")[0], 35)
    if "without" in form:
        del more[form.split()[-1]]
    want, after, size, state_size = ref.delta(*args, cu, **more)
    out = kernels.lines_delta(*args, plan, **more)
    rounding = (want.to(dtype).double() - want).norm()
    other = 2.0 ** -16 * (10 / heads[2]) ** 0.5 * size.norm()
    assert (out.double() - want).norm() <= (rounding ** 2 + other ** 2) ** 0.5
    assert (args[4].double() - after).norm() <= 2.0 ** -18 * state_size.norm() * max(1, heads[2] ** 0.5 / 8)
    assert not out[cu[-1]:].any() and fault() == 0


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("what", ["v", "k", "q", "decay", "beta"])
@pytest.mark.parametrize("counts,line,at", [([2, 9, 3], 1, 4), ([3, 60, 5, 100], 1, 20), ([3, 60, 5, 100], 3, 0), ([150, 20], 0, 63),
                                            ([150, 20], 0, 80), ([150, 20], 0, 149)])
def test_delta_a_value_that_is_not_finite_reaches_nothing_before_it(cuda, value, what, counts, line, at):
    """One value of one token: its line's later tokens and its state, of v those of its column alone, of q nothing but its own token."""
    from drama3_b200 import kernels
    if what == "decay" and value == -float("inf"):
        pytest.skip("a decay of everything is one")
    cu, plan = plan_of(counts, 2, cuda)
    (q, k, v, decay, state), more = delta_case(cuda, (2, 4, 64, 64), counts, 2, torch.bfloat16, "given", 36)
    if what == "decay" and value > 0:
        value = float("nan")  # above 0 counts as 0
    good = {"q": q, "k": k, "v": v, "decay": decay, "beta": more["beta"]}
    bad = {name: t.clone() for name, t in good.items()}
    t = cu[line] + at
    bad[what][(t, 1, 7) if bad[what].dim() == 3 else (t, 1)] = value
    runs = []
    for d in (good, bad):
        s = state.clone()
        runs.append((kernels.lines_delta(d["q"], d["k"], d["v"], d["decay"], s, plan, beta=d["beta"]), s))
    (want, want_state), (got, got_state) = runs
    heads = [2, 3] if what in ("q", "k") else [1]  # of 4, of which two share a key head
    reached = torch.zeros(want.shape, dtype=torch.bool, device=cuda)
    reached_state = torch.zeros(want_state.shape, dtype=torch.bool, device=cuda)
    for h in heads:
        reached[t:t + 1 if what == "q" else cu[line + 1], h, 7 if what == "v" else slice(None)] = True
        if what != "q":
            reached_state[line, h, 7 if what == "v" else slice(None)] = True
    assert not got[reached].isfinite().any() and torch.equal(got[~reached], want[~reached]) and want.isfinite().all()
    assert not got_state[reached_state].isfinite().any() and torch.equal(got_state[~reached_state], want_state[~reached_state])
