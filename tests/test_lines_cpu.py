"""The attention half of a decoder layer without a GPU: what the C ABI and the wrappers refuse before anything is
launched, the rotary helpers, the custom ops' fake implementations, and the plain restatements that the GPU tests trust,
against torch's own attention and a rotation written as complex numbers."""
import math

import pytest
import torch

import lines_ref as ref
from drama3_b200 import _lib, kernels, ops  # noqa: F401


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def strides(*values):
    return kernels._int64s(values)


# ---- refusals of the C ABI: all return before a CUDA call (the pointers are no addresses)

def plan_args(**change):
    args = dict(kept=16, counts=16, B=4, table=16, W=8, free=16, F=8, used=16, prefix=None, page=16, T=4, group=8, slots=16,
                positions=16, line=16, cu=16, lengths=16, used_out=16, work=16, ints=1 << 20, stream=None)
    assert set(change) <= set(args)
    return list({**args, **change}.values())


@pytest.mark.parametrize("change,status", [
    (dict(B=0), 1), (dict(B=8193), 1), (dict(W=0), 1), (dict(F=-1), 1), (dict(page=0), 1), (dict(T=-1), 1),
    (dict(group=0), 1), (dict(group=129), 1), (dict(T=1 << 28, group=8), 1), (dict(kept=None), 1), (dict(counts=None), 1),
    (dict(table=None), 1), (dict(free=None), 1), (dict(used=None), 1), (dict(slots=None), 1), (dict(positions=None), 1),
    (dict(line=None), 1), (dict(cu=None), 1), (dict(lengths=None), 1), (dict(used_out=None), 1), (dict(work=None), 1),
    (dict(work=8), 2), (dict(slots=4), 2), (dict(positions=4), 2), (dict(ints=10), 5)])
def test_plan_refusals(lib, change, status):
    assert lib.d3_lines_plan(*plan_args(**change)) == status


def test_plan_sizes(lib):
    assert lib.d3_lines_plan_ints(0, 4, 8) == 0 and lib.d3_lines_plan_ints(8193, 4, 8) == 0
    assert lib.d3_lines_plan_ints(4, 4, 129) == 0 and lib.d3_lines_plan_ints(4, -1, 1) == 0
    # a header, a unit number per token, and room for a tile per line besides the whole tiles of prefix and lines
    assert lib.d3_lines_plan_ints(16, 16, 8) >= 16 + 16 + 8 * (16 + 1)
    with pytest.raises(ValueError):
        kernels.plan_ints(9000, 4, 8)


def rope_args(**change):
    args = dict(q=16, qs=strides(512, 128, 1), k=16, ks=strides(256, 128, 1), v=None, vs=None, type=0, T=4, Hq=4, Hkv=2,
                D=128, qw=16, kw=16, f32=0, add=0.0, eps=1e-6, rotary=16, rot=128, length=10, pos=16, axes=1, axis=None,
                pairs=0, q_out=16, k_out=16, kc=None, kcs=None, vc=None, vcs=None, pages=0, page=0, slots=None, stream=None)
    assert set(change) <= set(args)
    return list({**args, **change}.values())


CACHE = dict(k_out=None, v=16, vs=strides(256, 128, 1), kc=16, kcs=strides(4096, 256, 128), vc=16,
             vcs=strides(4096, 256, 128), pages=4, page=16, slots=16)


@pytest.mark.parametrize("change,status", [
    (dict(type=3), 1), (dict(T=-1), 1), (dict(Hq=0), 1), (dict(Hkv=0), 1), (dict(D=0), 1), (dict(D=1025), 1),
    (dict(rot=130), 1), (dict(rot=3), 1), (dict(rot=-2), 1), (dict(axes=0), 1), (dict(axes=5, axis=16), 1),
    (dict(axes=3), 1), (dict(length=-1), 1), (dict(eps=-1.0), 1), (dict(eps=math.nan), 1), (dict(q=None), 1),
    (dict(k=None), 1), (dict(q_out=None), 1), (dict(rotary=None), 1), (dict(pos=None), 1), (dict(k_out=None), 1),
    (dict(q=17), 2), (dict(k=17), 2), (dict(q_out=17), 2), (dict(k_out=17), 2), (dict(rotary=4), 2), (dict(pos=4), 2),
    (dict(T=0), 0),
    *[({**CACHE, name: None}, 1) for name in ("v", "vs", "kc", "kcs", "vc", "vcs", "slots")],
    ({**CACHE, "pages": 0}, 1), ({**CACHE, "page": 0}, 1), ({**CACHE, "kc": 17}, 2), ({**CACHE, "v": 17}, 2)])
def test_rope_refusals(lib, change, status):
    assert lib.d3_qk_norm_rope(*rope_args(**change)) == status


def attn_args(**change):
    args = dict(q=16, qs=strides(4096, 128, 1), type=0, T=16, Hq=32, Hkv=4, D=128, kc=16, kcs=strides(32768, 512, 128),
                vc=16, vcs=strides(32768, 512, 128), pages=9, page=64, table=16, W=8, prefix_table=16, PW=2, work=16, B=16,
                scale=0.1, out=16, lse=None, ws=16, bytes=1 << 40, stream=None)
    assert set(change) <= set(args)
    return list({**args, **change}.values())


@pytest.mark.parametrize("change,status", [
    (dict(type=2), 1), (dict(type=-1), 1), (dict(T=-1), 1), (dict(Hkv=3), 1), (dict(Hq=2), 1), (dict(Hkv=0), 1),
    (dict(Hq=516, Hkv=4), 1), (dict(D=96), 1), (dict(D=192), 1), (dict(page=0), 1), (dict(page=8), 1), (dict(page=48), 1),
    (dict(page=100), 1), (dict(pages=0), 1), (dict(pages=1 << 26), 1), (dict(W=0), 1), (dict(PW=-1), 1), (dict(B=0), 1),
    (dict(B=8193), 1), (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=math.nan), 1), (dict(scale=math.inf), 1),
    (dict(q=None), 1), (dict(kc=None), 1), (dict(vc=None), 1), (dict(table=None), 1), (dict(prefix_table=None), 1),
    (dict(work=None), 1), (dict(out=None), 1), (dict(ws=None), 1), (dict(kcs=strides(0, 512, 128)), 1),
    (dict(qs=strides(4096, 0, 1)), 1), (dict(q=8), 2), (dict(kc=8), 2), (dict(out=8), 2), (dict(ws=8), 2),
    (dict(work=8), 2), (dict(qs=strides(4100, 128, 1)), 2), (dict(kcs=strides(32768, 516, 128)), 2), (dict(T=0), 0)])
def test_attention_refusals(lib, change, status):
    assert lib.d3_lines_attention(*attn_args(**change)) == status


def test_wrappers_refuse_host_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        kernels.lines_plan(i, i, i.view(2, 1), i, i[:1], 16, 2)
    x = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        kernels.qk_norm_rope(x, x, torch.zeros((4, 32, 2)), torch.zeros(2, dtype=torch.int64))
    plan = kernels.LinesPlan(i.view(2, 1), i.long(), i.long(), i, i, i, i, i, 16, 1)
    with pytest.raises(ValueError, match="GPU"):
        kernels.lines_attention(x, x.view(1, 2, 4, 64), x.view(1, 2, 4, 64), plan)


# ---- helpers and restatements

def test_rotary_helpers():
    table = kernels.rotary_table(torch.tensor([1.0, 0.25]), 5)
    assert table.shape == (5, 2, 2) and table.dtype == torch.float32
    assert abs(float(table[4, 1, 0]) - math.cos(1.0)) < 1e-7 and abs(float(table[3, 0, 1]) - math.sin(3.0)) < 1e-7
    assert kernels.rotary_axes([2, 1, 1]).tolist() == [0, 0, 1, 2]
    assert kernels.rotary_axes([3, 2, 1], woven=True).tolist() == [0, 1, 2, 0, 1, 0]
    assert kernels.rotary_axes([0, 2], woven=True).tolist() == [1, 1]


def test_plain_norm_rope_is_a_turn_by_complex_numbers():
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn((3, 2, 8), generator=g), torch.rand(8, generator=g)
    table, pos = kernels.rotary_table(torch.tensor([1.0, 0.5, 0.1]), 9), torch.tensor([0, 4, 8])
    got = ref.norm_rope(x, w, 1, 1e-3, table, pos, None, False)
    y = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-3) * (1 + w.double())
    z = torch.complex(y[..., :3], y[..., 3:6]) * torch.view_as_complex(table.double().contiguous())[pos][:, None]
    assert torch.allclose(got, torch.cat((z.real, z.imag, y[..., 6:]), -1))


def test_plain_attention_is_torchs():
    g = torch.Generator().manual_seed(2)
    kc, vc = (torch.randn((9, 4, 2, 8), generator=g) for _ in range(2))
    q = torch.randn((5, 4, 8), generator=g)
    prefix_table, table = torch.tensor([3, 1]), torch.tensor([[0, 2], [5, 8]])
    kept, counts, prefix = [1, 4], [3, 2], 6
    out, lse, bound = ref.attention(q, kc, vc, kept, counts, table, prefix, prefix_table, 0.3)
    t0 = 0
    for b in range(2):
        n, total = counts[b], prefix + kept[b] + counts[b]
        k, v = (torch.cat((c[prefix_table].flatten(0, 1)[:prefix], c[table[b]].flatten(0, 1)[:kept[b] + n])) for c in (kc, vc))
        mask = torch.ones((n, total), dtype=torch.bool).tril(total - n)
        want = torch.nn.functional.scaled_dot_product_attention(
            q[t0:t0 + n].transpose(0, 1).double(), k.transpose(0, 1).repeat_interleave(2, 0).double(),
            v.transpose(0, 1).repeat_interleave(2, 0).double(), attn_mask=mask, scale=0.3).transpose(0, 1)
        assert torch.allclose(out[t0:t0 + n], want)
        t0 += n
    assert (bound >= out.abs() - 1e-12).all() and lse.isfinite().all()


def test_plain_plan_by_hand():
    table = [[7, -1], [4, -1]]
    p = ref.plan([3, 4], [2, 1], table, [9, 8, 7], 1, 4, 4, prefix=10)
    assert table == [[7, 8], [4, 7]] and p["slots"] == [31, 32, 28, -1] and p["used"] == [3] and not p["pages"]
    assert p["lengths"] == [5, 5] and p["cu"] == [0, 2, 3] and p["positions"] == [13, 14, 14, 0]
    assert p["line"] == [0, 0, 1, -1] and not p["tokens"]


# ---- the custom ops on meta tensors

def test_fake_shapes():
    o = torch.ops.drama3_b200
    i32 = lambda *s: torch.empty(s, dtype=torch.int32, device="meta")  # noqa: E731
    slots, positions, line, cu, lengths, used, work = o.lines_plan(i32(3), i32(3), i32(3, 4), i32(9), i32(1), 16, 7, i32(1), 8)
    assert slots.shape == positions.shape == line.shape == (7,) and slots.dtype == torch.int64 and line.dtype == torch.int32
    assert cu.shape == (4,) and lengths.shape == (3,) and used.shape == (1,) and work.shape == (kernels.plan_ints(3, 7, 8),)
    q, k = (torch.empty((7, h, 64), dtype=torch.bfloat16, device="meta") for h in (8, 2))
    table, pos = torch.empty((50, 32, 2), device="meta"), torch.empty(7, dtype=torch.int64, device="meta")
    a, b = o.qk_norm_rope(q, k, table, pos)
    assert a.shape == q.shape and b.shape == k.shape and a.dtype == torch.bfloat16
    cache = torch.empty((5, 16, 2, 64), dtype=torch.bfloat16, device="meta")
    assert o.qk_norm_rope_cached(q, k, k, table, pos, cache, cache, slots).shape == q.shape
    out, lse = o.lines_attention(q, cache, cache, i32(3, 4), work, 4)
    assert out.shape == q.shape and out.dtype == torch.bfloat16 and lse.shape == (7, 8) and lse.dtype == torch.float32
    assert "Tensor(a2!) table" in str(o.lines_plan.default._schema)
    assert "k_cache" in str(o.qk_norm_rope_cached.default._schema) and "!" in str(o.qk_norm_rope_cached.default._schema)
