"""LinesDelta, LinesState and LinesStack on the GPU: a shared prefix, ragged texts and steps give each line what plain layers
give the whole sequence.

Tolerance. The module rounds to bf16 where the plain layer does (the projections, the convolution, the attention's output, the
gated norm), from sums that differ in 32 bits or, in the attention's outputs, by 2^-10 of their size; where the two round to
different sides a value is off by a whole step, 2^-7 of it at most, and values off by a step at each of four places are off
by 2^-7 sqrt(4) of the norm if they all are: 1.6 %. A stack of two layers, each with two sums whose rows are one of five
comparable terms, stays within twice that."""
import pytest
import torch

import linear_ref as ref

pytestmark = pytest.mark.gpu

HIDDEN, HK, HV, DK, DV, TAPS = 256, 2, 4, 64, 64, 4


def fault():
    from drama3_b200._lib import take_fault
    return take_fault()


def module(cuda, seed):
    from drama3_b200.hybrid import LinesDelta
    torch.manual_seed(seed)
    m = LinesDelta(HIDDEN, HK, HV, DK, DV, TAPS, device=cuda, dtype=torch.bfloat16)
    with torch.no_grad():
        m.conv.add_(0.3 * torch.randn_like(m.conv))
        m.a_log.add_(torch.randn_like(m.a_log))
        m.dt_bias.add_(torch.randn_like(m.dt_bias))
        m.norm.add_(0.1 * torch.randn_like(m.norm))
    return m


def plain(m, x):
    """A whole sequence through the layer, by the 64-bit restatements."""
    n = x.shape[0]
    mixed, gate, beta, decay = m.in_proj(x).split(m.sizes, 1)
    zeros = torch.zeros((1, TAPS - 1, m.sizes[0]), device=x.device)
    mixed = ref.conv(mixed, m.conv, zeros, [0, n])[0].bfloat16()
    q, k, v = (t.unflatten(1, (-1, d)) for t, d in zip(mixed.split((HK * DK, HK * DK, HV * DV), 1), (DK, DK, DV)))
    state = torch.zeros((1, HV, DV, DK), device=x.device)
    out = ref.delta(q, k, v, decay, state, [0, n], beta, m.a_log, m.dt_bias, m.eps)[0].bfloat16()
    out = ref.gated(out, gate.unflatten(1, (HV, DV)), m.norm, m.eps).bfloat16()
    return m.out_proj(out.flatten(1))


def close(got, want, most=0.016):
    assert float((got.float() - want.float()).norm()) <= most * float(want.float().norm())


def test_module_reads_a_prefix_and_texts_as_one_sequence(cuda):
    from drama3_b200.attention import LinesCache
    from drama3_b200.hybrid import LinesState
    m = module(cuda, 1)
    prefix, texts, steps = 77, [3, 90, 0, 9], 2
    cache = LinesCache(0, 40, 16, 1, 64, 4, 128, 1, cuda)
    state = LinesState(1, 4, HK, HV, DK, DV, TAPS, cuda)
    counts = torch.tensor(texts, dtype=torch.int32, device=cuda)
    with torch.no_grad():
        x0 = torch.randn((prefix, HIDDEN), device=cuda).bfloat16()
        xs = [torch.randn((n + steps, HIDDEN), device=cuda).bfloat16() for n in texts]
        close(m(x0, cache.plan_prefix(prefix), state.prefix_conv[0], state.prefix_delta[0]), plain(m, x0))
        for _ in range(2):  # the second time, new lines behind the same prefix
            cache.restart()
            state.begin()
            want = [plain(m, torch.cat((x0, x)))[prefix:] for x in xs]
            got = m(torch.cat([x[:n] for x, n in zip(xs, texts)]), cache.plan(counts, sum(texts)), state.conv[0],
                    state.delta[0]).split(texts)
            for g, w, n in zip(got, want, texts):
                if n:
                    close(g, w[:n])
            for s in range(steps):
                g = m(torch.stack([x[n + s] for x, n in zip(xs, texts)]), cache.plan(torch.ones_like(counts), 4), state.conv[0],
                      state.delta[0])
                close(g, torch.stack([w[n + s] for w, n in zip(want, texts)]))
        state.clear()
        assert not any(t.any() for t in (*state.conv, *state.delta, *state.prefix_conv, *state.prefix_delta))
    assert fault() == 0


def test_stack_joins_attention_and_linear_attention(cuda):
    from drama3_b200 import kernels
    from drama3_b200.attention import LinesAttention, LinesCache
    from drama3_b200.hybrid import LinesStack, LinesState

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.linear = torch.nn.Linear(HIDDEN, HIDDEN, bias=False, device=cuda, dtype=torch.bfloat16)

        def forward(self, x):
            assert x.dim() == 3 and x.shape[1] == 1
            return self.linear(x)

    delta = module(cuda, 2)
    attention = LinesAttention(HIDDEN, 4, 2, 64, device=cuda, dtype=torch.bfloat16)
    stack = LinesStack(HIDDEN, [delta, attention], [Block(), Block()], device=cuda, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="blocks"):
        LinesStack(HIDDEN, [delta], [], device=cuda)
    rotary = kernels.rotary_table(10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), 200, cuda)
    prefix, n, lines = 40, 30, 3

    def new():
        return (LinesCache(1, 60, 16, 2, 64, lines, 64, 2, cuda), LinesState(1, lines, HK, HV, DK, DV, TAPS, cuda))

    def whole(x):  # one sequence, layer by layer, each sum rounded where the stack rounds it
        cache, state = new()
        plan = cache.plan_prefix(x.shape[0])
        norm = lambda t, w: torch.nn.functional.rms_norm(t, (HIDDEN,), w, stack.eps)  # noqa: E731
        for i, (mixer, block) in enumerate(zip(stack.mixers, stack.blocks)):
            y = plain(mixer, norm(x, stack.norms[2 * i])) if i == 0 else mixer(norm(x, stack.norms[2 * i]), plan, cache.k[0], cache.v[0], rotary)
            x = x + y
            x = x + block(norm(x, stack.norms[2 * i + 1]).unsqueeze(1)).squeeze(1)
        return norm(x, stack.norms[4])

    with torch.no_grad():
        x0 = torch.randn((prefix, HIDDEN), device=cuda).bfloat16()
        xs = torch.randn((lines, n + 1, HIDDEN), device=cuda).bfloat16()
        cache, state = new()
        close(stack(x0, cache.plan_prefix(prefix), cache, state, rotary, prefix=True), whole(x0), 0.032)
        state.begin()
        want = torch.stack([whole(torch.cat((x0, x)))[prefix:] for x in xs])
        counts = torch.full((lines,), n, dtype=torch.int32, device=cuda)
        got = stack(xs[:, :n].reshape(-1, HIDDEN), cache.plan(counts, lines * n), cache, state, rotary)
        close(got.view(lines, n, HIDDEN), want[:, :n], 0.032)
        close(stack(xs[:, n].contiguous(), cache.plan(torch.ones_like(counts), lines), cache, state, rotary), want[:, n], 0.032)
    assert fault() == 0


def test_example_runs(cuda):
    import importlib.util
    from pathlib import Path
    spec = importlib.util.spec_from_file_location("hybrid_decode", Path(__file__).resolve().parents[1] / "examples" / "hybrid_decode.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    rows, ms = example.decode(lines=3, prompt=70, steps=4, n_layers=4)
    again, _ = example.decode(lines=3, prompt=70, steps=4, n_layers=4)
    assert rows.shape == (3, example.HIDDEN) and rows.isfinite().all() and ms > 0 and fault() == 0
    assert torch.equal(rows, again)
