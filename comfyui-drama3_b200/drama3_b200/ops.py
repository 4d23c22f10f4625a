"""The library's kernels as torch.library custom ops, torch.ops.drama3_b200.<name>, for callers that build graphs
(torch.compile, CUDA graph capture, exported programs): every op takes and returns plain tensors, ints, bools and
strings, writes fresh outputs (shared_expert updates `out` in place and declares it, as lines_plan does its table and
qk_norm_rope_cached its caches and lines_conv and lines_delta their state), and has a fake implementation that gives the output shapes and dtypes without running
anything. Each op calls the matching function of drama3_b200.kernels; there is no CPU or torch fallback, so a call on
tensors that are not on a B200 fails loudly.

Import this module once to register the ops. The expert banks of moe_decode and grouped_mma are passed field by
field: `w` is the bank's weight rows ("weight" for fp8 / fp8c, "_qdata" for the integer layouts), `scale` its scales
and `s_channel` the W4 / W6 per-row factors (None for the other layouts), as drama3/offload.py:72-90 names them."""
from typing import Optional

import torch
from torch import Tensor

from . import _lib, kernels

NAMESPACE = "drama3_b200"
OPS = ("route", "weighted_sum", "rotate", "router", "shared_expert", "moe_decode", "grouped_mma", "prefill_plan",
       "prefill_combine", "lines_plan", "qk_norm_rope", "qk_norm_rope_cached", "lines_attention", "lines_conv", "lines_delta",
       "gated_norm", "add_norm")


def _fields(kind, w, scale, s_channel):
    fields = {_lib.WEIGHT_KEY[kind]: w, "scale": scale}
    if s_channel is not None:
        fields["s_channel"] = s_channel
    return fields


# ---- routing and the per-kernel reference API (drama3/kernels.py:636-661)

@torch.library.custom_op(f"{NAMESPACE}::route", mutates_args=())
def route(logits: Tensor, k: int) -> tuple[Tensor, Tensor]:
    """(ids [rows, k] int64, weights [rows, k] float32) of bfloat16 router logits: kernels.route."""
    return kernels.route(logits, k)


@route.register_fake
def _(logits, k):
    rows = logits.shape[0]
    return logits.new_empty((rows, k), dtype=torch.int64), logits.new_empty((rows, k), dtype=torch.float32)


@torch.library.custom_op(f"{NAMESPACE}::weighted_sum", mutates_args=())
def weighted_sum(parts: Tensor, weights: Tensor) -> Tensor:
    """[rows, H] bfloat16: parts [rows * k, H] float32 summed per row by weights [rows, k], in rank order."""
    return kernels.weighted_sum(parts, weights)


@weighted_sum.register_fake
def _(parts, weights):
    rows = weights.reshape(-1, weights.shape[-1]).shape[0]
    return parts.new_empty((rows, parts.shape[-1]), dtype=torch.bfloat16)


@torch.library.custom_op(f"{NAMESPACE}::rotate", mutates_args=())
def rotate(x: Tensor, only_if: Tensor, swiglu: bool = False) -> Tensor:
    """float32 rows of x in the ConvRot basis (through SiLU(gate) * up first with `swiglu`): kernels.rotate."""
    return kernels.rotate(x, only_if, swiglu)


@rotate.register_fake
def _(x, only_if, swiglu=False):
    rows, width = x.shape
    return x.new_empty((rows, width // 2 if swiglu else width), dtype=torch.float32)


# ---- the fused MoE block pieces (drama3/model.py:40-47,107-123)

@torch.library.custom_op(f"{NAMESPACE}::router", mutates_args=())
def router(x: Tensor, weight: Tensor, k: int) -> tuple[Tensor, Tensor]:
    """(ids, weights) of decode rows through a bf16 router linear and the decode routing: kernels.router."""
    return kernels.router(x, weight, k)


@router.register_fake
def _(x, weight, k):
    rows = x.shape[0]
    return x.new_empty((rows, k), dtype=torch.int64), x.new_empty((rows, k), dtype=torch.float32)


@torch.library.custom_op(f"{NAMESPACE}::shared_expert", mutates_args=("out",))
def shared_expert(x: Tensor, gate_up: Tensor, down: Tensor, gate: Tensor, out: Tensor) -> None:
    """out += the sigmoid-gated shared expert of decode rows x, in place: kernels.shared_expert."""
    kernels.shared_expert(x, gate_up, down, gate, out)


@shared_expert.register_fake
def _(x, gate_up, down, gate, out):
    return None


@torch.library.custom_op(f"{NAMESPACE}::moe_decode", mutates_args=())
def moe_decode(kind: str, x: Tensor, ids: Tensor, weights: Tensor, w13: Tensor, s13: Tensor,
               c13: Optional[Tensor], w2: Tensor, s2: Tensor, c2: Optional[Tensor],
               codebook13: Optional[Tensor] = None, codebook2: Optional[Tensor] = None) -> Tensor:
    """[M, H] bfloat16: rows x through their routed experts, one fused launch (kernels.moe_decode); (w13, s13, c13)
    and (w2, s2, c2) are the gate_up and down banks' weight rows, scales and s_channel."""
    banks = (_fields(kind, w13, s13, c13), _fields(kind, w2, s2, c2))
    return kernels.moe_decode(kind, x, ids, weights, banks, (codebook13, codebook2))


@moe_decode.register_fake
def _(kind, x, ids, weights, w13, s13, c13, w2, s2, c2, codebook13=None, codebook2=None):
    return x.new_empty(x.shape, dtype=torch.bfloat16)


# ---- the prompt pass (drama3/offload.py:126-149)

@torch.library.custom_op(f"{NAMESPACE}::prefill_plan", mutates_args=())
def prefill_plan(topk_idx: Tensor, num_experts: int, drop_invalid: bool = False) -> tuple[Tensor, Tensor, Tensor]:
    """(order, pos, groups) of a prompt's routing sorted by expert on the device: kernels.prefill_plan."""
    return kernels.prefill_plan(topk_idx, num_experts, drop_invalid)


@prefill_plan.register_fake
def _(topk_idx, num_experts, drop_invalid=False):
    P = topk_idx.numel()
    return (topk_idx.new_empty((P,), dtype=torch.int64), topk_idx.new_empty((P,), dtype=torch.int64),
            topk_idx.new_empty((num_experts + 1, 5), dtype=torch.int32))


@torch.library.custom_op(f"{NAMESPACE}::grouped_mma", mutates_args=())
def grouped_mma(kind: str, x: Tensor, groups: Tensor, w: Tensor, scale: Tensor, s_channel: Optional[Tensor],
                codebook: Optional[Tensor], n: int, tiles: int, row_index: Optional[Tensor] = None,
                rotate: bool = False, swiglu: bool = False) -> Tensor:
    """[rows, n] float32: the sorted rows through their experts on the tensor cores (kernels.grouped_mma)."""
    return kernels.grouped_mma(kind, x, groups, _fields(kind, w, scale, s_channel), codebook, n, tiles,
                               row_index=row_index, rotate=rotate, swiglu=swiglu)


@grouped_mma.register_fake
def _(kind, x, groups, w, scale, s_channel, codebook, n, tiles, row_index=None, rotate=False, swiglu=False):
    rows = row_index.shape[0] if row_index is not None else x.shape[0]
    return x.new_empty((rows, n), dtype=torch.float32)


@torch.library.custom_op(f"{NAMESPACE}::prefill_combine", mutates_args=())
def prefill_combine(sorted_out: Tensor, pos: Tensor, weights: Tensor, out_f32: bool = False) -> Tensor:
    """[T, H]: the scatter, routing weights and sum over k of a prompt pass (kernels.prefill_combine), bfloat16 or
    float32 with out_f32."""
    return kernels.prefill_combine(sorted_out, pos, weights, dtype=torch.float32 if out_f32 else torch.bfloat16)


@prefill_combine.register_fake
def _(sorted_out, pos, weights, out_f32=False):
    return sorted_out.new_empty((pos.shape[0], sorted_out.shape[1]),
                                dtype=torch.float32 if out_f32 else torch.bfloat16)


# ---- the attention half of a decoder layer, for lines decoded together

@torch.library.custom_op(f"{NAMESPACE}::lines_plan", mutates_args=("table",))
def lines_plan(lengths: Tensor, counts: Tensor, table: Tensor, free: Tensor, used: Tensor, page: int, tokens: int,
               prefix: Optional[Tensor] = None,
               group: int = 1) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(slots, positions, line, cu, lengths, used, work) of kernels.lines_plan; the block table is updated in place."""
    p = kernels.lines_plan(lengths, counts, table, free, used, page, tokens, prefix=prefix, group=group)
    # outputs of an op share no storage: the plan's are cut from one allocation
    return tuple(t.clone() for t in (p.slots, p.positions, p.line, p.cu, p.lengths, p.used, p.work))


@lines_plan.register_fake
def _(lengths, counts, table, free, used, page, tokens, prefix=None, group=1):
    B = lengths.shape[0]
    i32 = [lengths.new_empty((n,), dtype=torch.int32) for n in (tokens, B + 1, B, 1, kernels.plan_ints(B, tokens, group))]
    return (lengths.new_empty((tokens,), dtype=torch.int64), lengths.new_empty((tokens,), dtype=torch.int64), *i32)


@torch.library.custom_op(f"{NAMESPACE}::qk_norm_rope", mutates_args=())
def qk_norm_rope(q: Tensor, k: Tensor, rotary: Tensor, positions: Tensor, q_weight: Optional[Tensor] = None,
                 k_weight: Optional[Tensor] = None, eps: float = 1e-6, unit_offset: bool = False,
                 axes: Optional[Tensor] = None, pairs: bool = False) -> tuple[Tensor, Tensor]:
    """(q, k) through the norm of each head and the rotation: kernels.qk_norm_rope without a cache."""
    return kernels.qk_norm_rope(q, k, rotary, positions, q_weight, k_weight, eps, unit_offset, axes, pairs)


@qk_norm_rope.register_fake
def _(q, k, rotary, positions, q_weight=None, k_weight=None, eps=1e-6, unit_offset=False, axes=None, pairs=False):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op(f"{NAMESPACE}::qk_norm_rope_cached", mutates_args=("k_cache", "v_cache"))
def qk_norm_rope_cached(q: Tensor, k: Tensor, v: Tensor, rotary: Tensor, positions: Tensor, k_cache: Tensor,
                        v_cache: Tensor, slots: Tensor, q_weight: Optional[Tensor] = None,
                        k_weight: Optional[Tensor] = None, eps: float = 1e-6, unit_offset: bool = False,
                        axes: Optional[Tensor] = None, pairs: bool = False) -> Tensor:
    """q through the norm of each head and the rotation; k (likewise) and v go to their slots of the paged caches."""
    return kernels.qk_norm_rope(q, k, rotary, positions, q_weight, k_weight, eps, unit_offset, axes, pairs, v=v,
                                k_cache=k_cache, v_cache=v_cache, slots=slots)[0]


@qk_norm_rope_cached.register_fake
def _(q, k, v, rotary, positions, k_cache, v_cache, slots, q_weight=None, k_weight=None, eps=1e-6, unit_offset=False,
      axes=None, pairs=False):
    return q.new_empty(q.shape)


@torch.library.custom_op(f"{NAMESPACE}::lines_attention", mutates_args=())
def lines_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, table: Tensor, work: Tensor, group: int,
                    prefix_table: Optional[Tensor] = None, scale: Optional[float] = None) -> tuple[Tensor, Tensor]:
    """(out, lse) of kernels.lines_attention with a plan's block table and work list (made for `group` query heads per
    KV head, q's token places and the cache's pages; what it was made for stands in the list, and the kernel refuses one that
    was made for something else)."""
    plan = kernels.LinesPlan(table, q, None, None, None, None, None, work, k_cache.shape[1], group)
    return kernels.lines_attention(q, k_cache, v_cache, plan, prefix_table=prefix_table, scale=scale, lse=True)


@lines_attention.register_fake
def _(q, k_cache, v_cache, table, work, group, prefix_table=None, scale=None):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


# ---- the linear half of a hybrid decoder, for lines decoded together

def _lines(cu, line):
    """What the operators read of a plan."""
    return kernels.LinesPlan(None, None, None, line, cu, None, None, None, 0, 0)


@torch.library.custom_op(f"{NAMESPACE}::lines_conv", mutates_args=("state",))
def lines_conv(x: Tensor, weight: Tensor, state: Tensor, cu: Tensor, line: Tensor, bias: Optional[Tensor] = None,
               silu: bool = True) -> Tensor:
    """The causal convolution of each line's tokens (cu and line: a plan's), the state updated in place: kernels.lines_conv."""
    return kernels.lines_conv(x, weight, state, _lines(cu, line), bias, silu)


@lines_conv.register_fake
def _(x, weight, state, cu, line, bias=None, silu=True):
    return x.new_empty(x.shape)


@torch.library.custom_op(f"{NAMESPACE}::lines_delta", mutates_args=("state",))
def lines_delta(q: Tensor, k: Tensor, v: Tensor, decay: Tensor, state: Tensor, cu: Tensor, line: Tensor,
                beta: Optional[Tensor] = None, a_log: Optional[Tensor] = None, dt_bias: Optional[Tensor] = None,
                eps: Optional[float] = 1e-6, scale: Optional[float] = None) -> Tensor:
    """Linear attention with decays over a state of each line (cu and line: a plan's), the state updated in place:
    kernels.lines_delta."""
    return kernels.lines_delta(q, k, v, decay, state, _lines(cu, line), beta, a_log, dt_bias, eps, scale)


@lines_delta.register_fake
def _(q, k, v, decay, state, cu, line, beta=None, a_log=None, dt_bias=None, eps=1e-6, scale=None):
    return v.new_empty(v.shape)


@torch.library.custom_op(f"{NAMESPACE}::gated_norm", mutates_args=())
def gated_norm(x: Tensor, gate: Tensor, weight: Tensor, eps: float = 1e-6, unit_offset: bool = False,
               activation: str = "silu") -> Tensor:
    """The norm of each head with its gate: kernels.gated_norm."""
    return kernels.gated_norm(x, gate, weight, eps, unit_offset, activation)


@gated_norm.register_fake
def _(x, gate, weight, eps=1e-6, unit_offset=False, activation="silu"):
    return x.new_empty(x.shape)


@torch.library.custom_op(f"{NAMESPACE}::add_norm", mutates_args=())
def add_norm(x: Tensor, residual: Tensor, weight: Tensor, post_weight: Optional[Tensor] = None,
             gate: Optional[Tensor] = None, scale: float = 1.0, eps: float = 1e-6,
             unit_offset: bool = False) -> tuple[Tensor, Tensor]:
    """(sum, normed): a block joined to its residual with its norms: kernels.add_norm."""
    return kernels.add_norm(x, residual, weight, post_weight, gate, scale, eps, unit_offset)


@add_norm.register_fake
def _(x, residual, weight, post_weight=None, gate=None, scale=1.0, eps=1e-6, unit_offset=False):
    return x.new_empty(x.shape), x.new_empty(x.shape)
