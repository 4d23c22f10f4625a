"""The attention half of a decoder layer for lines decoded together, around kernels.lines_plan, qk_norm_rope and
lines_attention: `LinesCache`, the paged key/value cache of lines that share a prefix, and `LinesAttention`, the module
between a layer's input and its residual. The MoE half is model.SparseMoeBlock; examples/lines_decode.py runs both. (The
reference leaves its attention layers to its host application: drama3/model.py:127-560.)

A pass, for a prompt or a step alike: `cache.plan(counts, tokens)` once, then every layer's attention with that plan. A
decode step is a pass of one token per line; nothing in it waits for the host, so it can be captured in a CUDA graph."""
import torch
import torch.nn as nn

from . import kernels
from .model import OPS


class LinesCache:
    """Keys and values of `layers` layers in pages of `page` tokens ([pages, page, kv_heads, head_dim] each), the
    block tables of `lines` lines of up to `most` tokens of their own, and the pages of the prefix that they share.
    page: 16, 32 or a multiple of 64 (the attention's). group: query heads per KV head. The lengths are on the GPU, so no
    call here can tell that a line outgrows `most` or that the pages run out: such tokens have no place, their keys read
    as zeros, and the fault word says so (_lib.take_fault)."""

    def __init__(self, layers, pages, page, kv_heads, head_dim, lines, most, group, device, dtype=torch.bfloat16):
        self.page, self.group, self.lines, self.width = page, group, lines, -(-most // page)
        shape = (pages, page, kv_heads, head_dim)
        self.k, self.v = ([torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)] for _ in range(2))

        def ints(*shape, fill=0):
            return torch.full(shape, fill, dtype=torch.int32, device=device)

        self.free = torch.arange(pages, dtype=torch.int32, device=device)
        self.used, self.prefix = ints(1), ints(1)
        self.prefix_table = None
        self.lengths, self.table = ints(lines), ints(lines, self.width, fill=-1)

    def plan_prefix(self, tokens):
        """The plan of the pass that reads the shared prefix (on an empty cache): `tokens` tokens of one line, whose
        pages are the lines' prefix from then on."""
        table = torch.full((1, -(-tokens // self.page)), -1, dtype=torch.int32, device=self.free.device)
        plan = kernels.lines_plan(torch.zeros_like(self.used), torch.full_like(self.used, tokens), table, self.free,
                                  self.used, self.page, tokens, group=self.group)
        self.prefix.fill_(tokens)
        self.used.copy_(plan.used)
        self.prefix_table = table.view(-1)
        return plan

    def plan(self, counts, tokens):
        """The plan of a pass that appends counts [lines] (int32, on the GPU) tokens, `tokens` token places in all; the
        cache's lengths and its used pages are those after the pass. It brings the prefix's pages along."""
        plan = kernels.lines_plan(self.lengths, counts, self.table, self.free, self.used, self.page, tokens,
                                  prefix=self.prefix, group=self.group)
        self.lengths.copy_(plan.lengths)
        self.used.copy_(plan.used)
        return plan._replace(prefix_table=self.prefix_table)

    def restart(self):
        """New lines behind the same prefix: the lines' own pages are free again."""
        self.used.fill_(0 if self.prefix_table is None else self.prefix_table.numel())
        self.lengths.zero_()
        self.table.fill_(-1)


class LinesAttention(nn.Module):
    """x [T, hidden] -> [T, hidden]: the fused query/key/value projection, the norms of queries and keys for each head,
    their rotation and the cache write in one launch, attention over the shared prefix and the lines' own tokens, and
    the output projection. `ops` is the factory namespace of the modules of model.py."""

    def __init__(self, hidden, heads, kv_heads, head_dim, eps=1e-6, device=None, dtype=None, ops=None):
        super().__init__()
        ops = ops or OPS
        self.heads, self.kv_heads, self.head_dim, self.eps = heads, kv_heads, head_dim, eps
        self.qkv_proj = ops.Linear(hidden, (heads + 2 * kv_heads) * head_dim, bias=False, device=device, dtype=dtype)
        self.o_proj = ops.Linear(heads * head_dim, hidden, bias=False, device=device, dtype=dtype)
        self.q_norm, self.k_norm = (nn.Parameter(torch.ones(head_dim, device=device, dtype=dtype)) for _ in range(2))

    def forward(self, x, plan, k_cache, v_cache, rotary, prefix_table=None, positions=None, axes=None):
        """rotary: kernels.rotary_table's. positions: of the tokens, where they are not the plan's (with several axes
        [A, T], and `axes` from kernels.rotary_axes). prefix_table: the prefix's pages, where the plan does not bring them
        (LinesCache's do)."""
        T, sizes = x.shape[0], (self.heads, self.kv_heads, self.kv_heads)
        q, k, v = (t.unflatten(1, (-1, self.head_dim)) for t in
                   self.qkv_proj(x).split_with_sizes([n * self.head_dim for n in sizes], 1))
        q, _ = kernels.qk_norm_rope(q, k, rotary, plan.positions if positions is None else positions, q_weight=self.q_norm,
                                    k_weight=self.k_norm, eps=self.eps, axes=axes, v=v, k_cache=k_cache,
                                    v_cache=v_cache, slots=plan.slots)
        out = kernels.lines_attention(q, k_cache, v_cache, plan, prefix_table=prefix_table)
        return self.o_proj(out.view(T, -1))
