"""The linear half of a hybrid decoder without a GPU: what the C ABI and the wrappers refuse before anything is launched, the
custom ops' fake implementations, and the plain restatements that the GPU tests trust, against torch's own convolution and
norms and against the chunks' closed form."""
import math

import pytest
import torch

import linear_ref as ref
from drama3_b200 import _lib, kernels, ops  # noqa: F401


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def strides(*values):
    return kernels._int64s(values)


# ---- refusals of the C ABI: all return before a CUDA call (the pointers are no addresses)

def conv_args(**change):
    args = dict(x=16, x_token=64, type=0, T=4, C=64, weight=16, bias=None, W=4, w_f32=0, state=16, cu=16, line=16, B=2, silu=1,
                out=16, stream=None)
    assert set(change) <= set(args)
    return list({**args, **change}.values())


@pytest.mark.parametrize("change,status", [
    (dict(type=3), 1), (dict(type=-1), 1), (dict(T=-1), 1), (dict(C=0), 1), (dict(W=1), 1), (dict(W=9), 1), (dict(B=0), 1),
    (dict(B=8193), 1), (dict(C=1 << 30, W=4), 1), (dict(x=None), 1), (dict(weight=None), 1), (dict(state=None), 1),
    (dict(cu=None), 1), (dict(line=None), 1), (dict(out=None), 1), (dict(x=17), 2), (dict(state=17), 2), (dict(out=17), 2),
    (dict(weight=17), 2), (dict(weight=18, w_f32=1), 2), (dict(bias=17), 2), (dict(type=2, x=18), 2), (dict(T=0), 0)])
def test_conv_refusals(lib, change, status):
    assert lib.d3_lines_conv(*conv_args(**change)) == status


def delta_args(**change):
    args = dict(q=16, qs=strides(512, 128), k=16, ks=strides(512, 128), v=16, vs=strides(1024, 128), type=0, T=4, Hk=4, Hv=8,
                Dk=128, Dv=128, decay=16, decay_token=8, beta=16, beta_token=8, gates_f32=0, a_log=None, dt_bias=None, eps=1e-6,
                scale=0.1, state=16, cu=16, line=16, B=2, out=16, ws=128, bytes=1 << 40, stream=None)
    assert set(change) <= set(args)
    return list({**args, **change}.values())


@pytest.mark.parametrize("change,status", [
    (dict(type=2), 1), (dict(type=-1), 1), (dict(T=-1), 1), (dict(Hk=0), 1), (dict(Hv=2), 1), (dict(Hv=6), 1),
    (dict(Hv=65536, Hk=1), 1), (dict(Dk=96), 1), (dict(Dk=256), 1), (dict(Dv=0), 1), (dict(Dv=24), 1), (dict(Dv=272), 1),
    (dict(B=0), 1), (dict(B=8193), 1), (dict(scale=0.0), 1), (dict(scale=math.nan), 1), (dict(scale=math.inf), 1),
    (dict(eps=math.nan), 1), *[({name: None}, 1) for name in ("q", "qs", "k", "ks", "v", "vs", "decay", "state", "cu", "line",
                                                             "out")],
    *[({name: 24}, 2) for name in ("q", "k", "v", "state", "out")], (dict(decay=17), 2), (dict(beta=17), 2),
    (dict(decay=18, gates_f32=1), 2), (dict(a_log=18), 2), (dict(dt_bias=18), 2), (dict(qs=strides(516, 128)), 2),
    (dict(ks=strides(512, 132)), 2), (dict(vs=strides(1028, 128)), 2), (dict(ws=64), 2), (dict(T=100, ws=None), 1),
    (dict(T=100, bytes=1000), 5), (dict(qs=strides(-512, 128)), 1), (dict(vs=strides(0, 128)), 1), (dict(T=0), 0)])
def test_delta_refusals(lib, change, status):
    assert lib.d3_lines_delta(*delta_args(**change)) == status


def test_delta_workspace(lib):
    assert lib.d3_lines_delta_workspace(16, 16, 16, 32, 128) == 0 and lib.d3_lines_delta_workspace(0, 1, 1, 1, 64) == 0
    one = 64 * 128 * 2 + 2 * (3 * 64 * 128 * 2 + 64 * 64 * 2 + 5 * 64 * 4)  # a chunk of one key and two value heads
    assert lib.d3_lines_delta_workspace(64, 1, 1, 2, 128) == one and lib.d3_lines_delta_workspace(65, 1, 1, 2, 128) == 2 * one
    # a pass of any length is cut into parts of bounded scratch
    assert lib.d3_lines_delta_workspace(1 << 24, 1, 16, 32, 128) <= 384 << 20


def gated_args(**change):
    args = dict(x=16, xs=strides(512, 128), gate=16, gs=strides(512, 128), type=0, T=4, H=4, D=128, weight=16, w_f32=0,
                w_add=0.0, eps=1e-6, act=0, out=16, stream=None)
    assert set(change) <= set(args)
    return list({**args, **change}.values())


@pytest.mark.parametrize("change,status", [
    (dict(type=3), 1), (dict(T=-1), 1), (dict(H=0), 1), (dict(D=0), 1), (dict(T=1 << 30, H=4), 1), (dict(act=2), 1),
    (dict(act=-1), 1), (dict(eps=-1.0), 1), (dict(eps=math.nan), 1), (dict(x=None), 1), (dict(xs=None), 1), (dict(gate=None), 1),
    (dict(gs=None), 1), (dict(weight=None), 1), (dict(out=None), 1), (dict(x=17), 2), (dict(gate=17), 2), (dict(out=17), 2),
    (dict(weight=18, w_f32=1), 2), (dict(T=0), 0)])
def test_gated_refusals(lib, change, status):
    assert lib.d3_gated_norm(*gated_args(**change)) == status


def join_args(**change):
    args = dict(x=16, x_token=64, residual=16, r_token=64, type=0, T=4, W=64, weight=16, post=None, w_f32=0, w_add=0.0,
                gate=None, gate_token=0, gate_kind=0, scale=1.0, eps=1e-6, sums=16, normed=16, stream=None)
    assert set(change) <= set(args)
    return list({**args, **change}.values())


@pytest.mark.parametrize("change,status", [
    (dict(type=3), 1), (dict(T=-1), 1), (dict(W=0), 1), (dict(gate_kind=3), 1), (dict(gate_kind=-1), 1), (dict(gate_kind=1), 1),
    (dict(eps=-1.0), 1), (dict(eps=math.nan), 1), (dict(x=None), 1), (dict(residual=None), 1), (dict(weight=None), 1),
    (dict(sums=None), 1), (dict(normed=None), 1), (dict(x=17), 2), (dict(residual=17), 2), (dict(gate=17, gate_kind=1), 2),
    (dict(sums=17), 2), (dict(normed=17), 2), (dict(post=18, w_f32=1), 2), (dict(T=0), 0)])
def test_join_refusals(lib, change, status):
    assert lib.d3_add_norm(*join_args(**change)) == status


# ---- refusals of the wrappers

def plan_of(counts, tokens=None):
    cu = torch.tensor([0, *counts], dtype=torch.int32).cumsum(0).to(torch.int32)
    T = int(cu[-1]) if tokens is None else tokens
    line = torch.full((T,), -1, dtype=torch.int32)
    for b in range(len(counts)):
        line[cu[b]:cu[b + 1]] = b
    return kernels.LinesPlan(None, None, None, line, cu, None, None, None, 64, 1)


def test_wrappers_refuse_host_tensors():
    x = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        kernels.lines_conv(x[:, 0], torch.zeros((64, 4)), torch.zeros((1, 3, 64), dtype=torch.bfloat16), plan_of([2]))
    with pytest.raises(ValueError, match="GPU"):
        kernels.lines_delta(x, x, x, x[..., 0], torch.zeros((1, 4, 64, 64)), plan_of([2]))
    with pytest.raises(ValueError, match="GPU"):
        kernels.gated_norm(x, x, torch.zeros(64))
    with pytest.raises(ValueError, match="GPU"):
        kernels.add_norm(x[0], x[0], torch.zeros(64))


@pytest.fixture
def anywhere(monkeypatch):
    """The wrappers' checks of forms, on host tensors."""
    monkeypatch.setattr(kernels, "_gpu_of", lambda t, what: t.device)


def half(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_conv_forms(anywhere):
    x, w, s, plan = half(5, 16), half(16, 4), half(2, 3, 16), plan_of([2, 3])
    plan = (plan.cu, plan.line)
    device, sizes, taps, w_f32, B = kernels._conv_arguments(x, w, s, None, *plan)
    assert sizes == (16, 0, 5, 16) and taps == 4 and w_f32 == 0 and B == 2
    assert kernels._conv_arguments(half(5, 32)[:, 16:], w.view(16, 1, 4).float(), s, torch.zeros(16), *plan)[3] == 1
    for bad in [(x.int(), w, s, None), (half(16, 5).T, w, s, None), (x, half(16, 9), s, None), (x, half(16, 1), s, None),
                (x, half(15, 4), s, None), (x, w.half(), s, None), (x, w, s, torch.zeros(16)), (x, w, s, half(15)),
                (x, w, half(2, 4, 16), None), (x, w, s.float(), None), (x, w, half(2, 3, 32)[..., ::2], None),
                (x, half(4, 16).T, s, None), (x, w, half(3, 3, 16), None), (half(6, 16), w, s, None)]:
        with pytest.raises((TypeError, ValueError)):
            kernels._conv_arguments(*bad, *plan)


def test_delta_forms(anywhere):
    q, k, v, g, s = half(5, 2, 64), half(5, 2, 64), half(5, 4, 48), half(5, 4), torch.zeros((3, 4, 48, 64))
    a, plan = torch.zeros(4), plan_of([2, 0, 3])
    plan = (plan.cu, plan.line)
    device, copies, st, sizes, gates, scale, B, size = kernels._delta_arguments(q, k, v, g, s, g, a, a, *plan)
    assert not copies and sizes == (0, 5, 2, 4, 64, 48) and gates == (4, 4, 0) and list(st[2]) == [192, 48] and B == 3 and size == 0
    wide = half(5, 2 * 64 + 3)
    assert kernels._delta_arguments(wide[:, 3:].view(5, 2, 64), k, v, g.float(), s, None, None, None, *plan)[1]
    for bad in [(q.float(), k.float(), v.float(), g, s), (q, k.half(), v, g, s), (q, half(5, 4, 64), v, g, s),
                (half(5, 3, 64), half(5, 3, 64), v, g, s), (half(5, 2, 96), half(5, 2, 96), v, g, s),
                (q, k, half(5, 4, 40), g, s), (q, k, half(4, 4, 48), g, s), (half(5, 64, 2).transpose(1, 2), k, v, g, s),
                (q, k, v, half(5, 3), s), (q, k, v, half(4, 5).T, s), (q, k, v, g.half(), s), (q, k, v, g, s.to(torch.bfloat16)),
                (q, k, v, g, torch.zeros((3, 4, 64, 48))), (q, k, v, g, torch.zeros((3, 4, 64, 48)).transpose(2, 3)),
                (q, k, v, g, s, g.float()), (q, k, v, g, s, g, None, a), (q, k, v, g, s, g, a.double()),
                (q, k, v, g, s, g, torch.zeros(3)), (q, k, v, g, s, g, a, torch.zeros(8)[::2]),
                (q, k, v, g, torch.zeros((2, 4, 48, 64)))]:
        with pytest.raises((TypeError, ValueError)):
            kernels._delta_arguments(*bad, *[None] * (8 - len(bad)), *plan)


def test_norm_forms(anywhere):
    x, w = half(5, 4, 64), half(64)
    assert kernels._gated_arguments(x, x, w.float())[4] == 1
    for bad in [(x.int(), x.int(), w), (x, x.half(), w), (x, half(5, 4, 32), w), (x[0], x[0], w), (x, x, half(32)),
                (x, half(5, 64, 4).transpose(1, 2), w), (x, x, w.half()), (x, x, half(128)[::2])]:
        with pytest.raises((TypeError, ValueError)):
            kernels._gated_arguments(*bad)
    x = half(5, 64)
    for gate, token, kind in [(None, 0, 0), (half(5, 1), 1, 1), (half(1, 64), 0, 2), (half(64), 0, 2), (half(5, 64), 64, 2),
                              (half(1, 1), 0, 1), (half(5, 128)[:, :64], 128, 2), (half(5, 3)[:, :1], 3, 1)]:
        assert kernels._join_arguments(x, x, w, None, gate)[4:] == (token, kind)
    for bad in [(x.int(), x.int(), w, None, None), (x, x.half(), w, None, None), (x, half(4, 64), w, None, None),
                (half(64, 5).T, x, w, None, None), (x, x, half(32), None, None), (x, x, w, w.float(), None),
                (x, x, w, None, half(4, 1)), (x, x, w, None, half(5, 32)), (x, x, w, None, half(64, 5).T),
                (x, x, w, None, torch.zeros((5, 1)))]:
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            kernels._join_arguments(*bad)


def test_plan_of_another_pass_is_refused():
    device, plan = torch.device("cpu"), plan_of([2, 3])
    kernels._plan_lines("lines_delta", device, plan.cu, plan.line, 5, 2)
    with pytest.raises(ValueError, match="5 tokens"):
        kernels._plan_lines("lines_delta", device, plan.cu, plan.line, 6, 2)
    with pytest.raises(ValueError, match="2 lines"):
        kernels._plan_lines("lines_delta", device, plan.cu, plan.line, 5, 3)
    with pytest.raises(ValueError, match="int32"):
        kernels._plan_lines("lines_delta", device, torch.zeros(3, dtype=torch.int64), plan.line, 5, 2)


def test_state_shapes():
    from drama3_b200.hybrid import LinesDelta, LinesState
    state = LinesState(2, 3, 2, 4, 64, 80, 4, "cpu")
    assert len(state.conv) == 2 and state.conv[0].shape == (3, 3, 2 * 2 * 64 + 4 * 80) and state.delta[1].shape == (3, 4, 80, 64)
    state.prefix_delta[1].fill_(2)
    state.begin()
    assert (state.delta[1] == 2).all() and not state.delta[0].any()
    state.clear()
    assert not state.delta[1].any() and not state.prefix_delta[1].any()
    m = LinesDelta(32, 2, 4, 64, 80)
    assert m.in_proj.weight.shape == (sum(m.sizes), 32) and m.out_proj.weight.shape == (32, 320) and m.a_log.dtype == torch.float32


# ---- restatements

def test_plain_conv_is_torchs():
    g = torch.Generator().manual_seed(1)
    x, w, b = torch.randn((7, 6), generator=g), torch.randn((6, 4), generator=g), torch.randn(6, generator=g)
    state = torch.randn((1, 3, 6), generator=g)
    out, new, size = ref.conv(x, w, state, [0, 7], b)
    rows = torch.cat((state[0], x)).double()
    y = torch.nn.functional.conv1d(rows.T[None], w.double()[:, None], b.double(), groups=6)[0].T
    assert torch.allclose(out, torch.nn.functional.silu(y)) and torch.equal(new[0], rows[-3:]) and (size >= y.abs() - 1e-9).all()
    # two passes are one, the second of fewer tokens than the state holds
    first, middle, _ = ref.conv(x[:5], w, state, [0, 5], b)
    second, last, _ = ref.conv(x[5:], w, middle, [0, 2], b)
    assert torch.allclose(torch.cat((first, second)), out) and torch.equal(last, new)


@pytest.mark.parametrize("with_beta", [True, False])
def test_plain_delta_is_the_closed_form_of_a_chunk(with_beta):
    g = torch.Generator().manual_seed(2)
    T, D, E = 9, 8, 5
    q, k, v = (torch.randn((T, 1, n), generator=g).double() for n in (D, D, E))
    decay, beta = -torch.rand((T, 1), generator=g).double(), torch.rand((T, 1), generator=g).double() if with_beta else None
    S0 = torch.randn((1, 1, E, D), generator=g).double()
    out, S, size, bound = ref.delta(q, k, v, decay, S0, [0, T], beta, eps=None, scale=1.0)
    Q, K, V, G = q[:, 0], k[:, 0], v[:, 0], decay.cumsum(0)
    ratio = torch.exp(G - G.T).tril()
    U = V
    if with_beta:
        A = (beta * (K @ K.T) * ratio).tril(-1)
        U = torch.linalg.solve(torch.eye(T, dtype=torch.float64) + A, beta * (V - torch.exp(G) * (K @ S0[0, 0].T)))
    assert torch.allclose(out[:, 0], torch.exp(G) * (Q @ S0[0, 0].T) + ((Q @ K.T) * ratio) @ U)
    assert torch.allclose(S[0, 0], torch.exp(G[-1]) * S0[0, 0] + (torch.exp(G[-1] - G) * U).T @ K)
    assert (size >= out.abs() - 1e-12).all() and (bound >= S.norm(dim=-1) - 1e-12).all()


def test_plain_norms_are_torchs():
    g = torch.Generator().manual_seed(3)
    x, z, r = (torch.randn((3, 4, 8), generator=g) for _ in range(3))
    w = torch.rand(8, generator=g)
    want = torch.nn.functional.rms_norm(x.double(), (8,), w.double(), 1e-5)
    assert torch.allclose(ref.gated(x, z, w, 1e-5), want * torch.nn.functional.silu(z.double()))
    assert torch.allclose(ref.gated(x, z, w - 1, 1e-5, 1, "sigmoid"), want * torch.sigmoid(z.double()))
    total, normed, size = ref.join(x, r, w, w, z, 0.5, 1e-5)
    assert torch.allclose(total, r.double() + 0.5 * z.double() * want)
    assert torch.allclose(normed, torch.nn.functional.rms_norm(total, (8,), w.double(), 1e-5)) and (size >= total.abs()).all()


# ---- the custom ops on meta tensors

def test_fake_shapes():
    o = torch.ops.drama3_b200
    m = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="meta")  # noqa: E731
    cu, line = m(4, dtype=torch.int32), m(7, dtype=torch.int32)
    assert o.lines_conv(m(7, 64), m(64, 4), m(3, 3, 64), cu, line).shape == (7, 64)
    out = o.lines_delta(m(7, 2, 64), m(7, 2, 64), m(7, 4, 80), m(7, 4), m(3, 4, 80, 64, dtype=torch.float32), cu, line)
    assert out.shape == (7, 4, 80) and out.dtype == torch.bfloat16
    assert o.gated_norm(m(7, 4, 80), m(7, 4, 80), m(80)).shape == (7, 4, 80)
    sums, normed = o.add_norm(m(7, 64), m(7, 64), m(64))
    assert sums.shape == normed.shape == (7, 64) and normed.dtype == torch.bfloat16
    for op in (o.lines_conv, o.lines_delta):
        assert "!) state" in str(op.default._schema)
