"""The linear half of a hybrid decoder for lines decoded together, around kernels.lines_conv, lines_delta, gated_norm and
add_norm: `LinesState`, what linear attention keeps of each line; `LinesDelta`, the module between a layer's input and its
residual; and `LinesStack`, decoder layers of linear attention (`LinesDelta`) and attention (attention.LinesAttention) with
their feed-forward blocks, joined to the residual by add_norm. (Three of four layers of the reference's decoder are linear
attention, drama3/config.py:59-60; it leaves them to its host application.)

A pass is planned by attention.LinesCache (`plan_prefix`, `plan`), whose plans every layer of either kind takes."""
import torch
import torch.nn as nn

from . import kernels
from .attention import LinesAttention
from .model import OPS


class LinesState:
    """What `layers` layers of linear attention keep of `lines` lines: the convolutions' last inputs, conv [lines, taps - 1,
    channels] each, and the heads' states, delta [lines, value_heads, value_dim, key_dim] each (float32); and the same of the
    prefix that the lines share, one line's. A pass over the prefix takes prefix_conv and prefix_delta; `begin` then starts
    the lines behind it, new ones too."""

    def __init__(self, layers, lines, key_heads, value_heads, key_dim, value_dim, taps, device, dtype=torch.bfloat16):
        channels = 2 * key_heads * key_dim + value_heads * value_dim

        def zeros(n):
            return ([torch.zeros((n, taps - 1, channels), dtype=dtype, device=device) for _ in range(layers)],
                    [torch.zeros((n, value_heads, value_dim, key_dim), device=device) for _ in range(layers)])

        self.conv, self.delta = zeros(lines)
        self.prefix_conv, self.prefix_delta = zeros(1)

    def begin(self):
        """Every line at the prefix's end (at nothing, without a prefix)."""
        for mine, prefix in zip((*self.conv, *self.delta), (*self.prefix_conv, *self.prefix_delta)):
            mine.copy_(prefix.expand_as(mine))

    def clear(self):
        """No prefix, and no line has a token."""
        for t in (*self.conv, *self.delta, *self.prefix_conv, *self.prefix_delta):
            t.zero_()


class LinesDelta(nn.Module):
    """x [T, hidden] -> [T, hidden]: one projection to queries, keys and values, the gate, and the raw strengths and decays;
    the short convolution of queries, keys and values over each line's tokens; linear attention with the delta rule; the norm
    of its heads with their gate; and the output projection. `ops` is the factory namespace of the modules of model.py."""

    def __init__(self, hidden, key_heads, value_heads, key_dim, value_dim, taps=4, eps=1e-6, device=None, dtype=None, ops=None):
        super().__init__()
        ops = ops or OPS
        self.key_heads, self.value_heads, self.key_dim, self.value_dim, self.eps = key_heads, value_heads, key_dim, value_dim, eps
        keys, values = key_heads * key_dim, value_heads * value_dim
        self.sizes = (2 * keys + values, values, value_heads, value_heads)  # of the projection: channels, gate, strengths, decays
        self.in_proj = ops.Linear(hidden, sum(self.sizes), bias=False, device=device, dtype=dtype)
        self.out_proj = ops.Linear(values, hidden, bias=False, device=device, dtype=dtype)
        self.conv = nn.Parameter(torch.full((self.sizes[0], taps), 1.0 / taps, device=device, dtype=dtype))
        self.a_log = nn.Parameter(torch.zeros(value_heads, device=device, dtype=torch.float32))
        self.dt_bias = nn.Parameter(torch.full((value_heads,), -3.0, device=device, dtype=torch.float32))
        self.norm = nn.Parameter(torch.ones(value_dim, device=device, dtype=dtype))

    def forward(self, x, plan, conv_state, delta_state):
        """conv_state and delta_state: this layer's of a LinesState, updated in place."""
        mixed, gate, beta, decay = self.in_proj(x).split_with_sizes(self.sizes, 1)
        mixed = kernels.lines_conv(mixed, self.conv, conv_state, plan)
        keys = self.key_heads * self.key_dim
        q, k, v = mixed.split_with_sizes((keys, keys, self.sizes[1]), 1)
        q, k = (t.unflatten(1, (self.key_heads, self.key_dim)) for t in (q, k))
        out = kernels.lines_delta(q, k, v.unflatten(1, (self.value_heads, self.value_dim)), decay, delta_state, plan, beta=beta,
                                  a_log=self.a_log, dt_bias=self.dt_bias, eps=self.eps)
        out = kernels.gated_norm(out, gate.unflatten(1, (self.value_heads, self.value_dim)), self.norm, eps=self.eps)
        return self.out_proj(out.flatten(1))


class LinesStack(nn.Module):
    """Decoder layers: mixers (LinesDelta or LinesAttention) and feed-forward blocks by turns, x + mixer(norm(x)), then x +
    block(norm(x)), and the norm behind the last one. A block takes [T, 1, hidden], as model.SparseMoeBlock does. Each sum and
    the norm that follows it are one launch (kernels.add_norm); the first norm, which follows no sum, is torch's."""

    def __init__(self, hidden, mixers, blocks, eps=1e-6, device=None, dtype=None):
        super().__init__()
        if len(mixers) != len(blocks):
            raise ValueError(f"{len(mixers)} mixers and {len(blocks)} blocks")
        self.mixers, self.blocks, self.eps = nn.ModuleList(mixers), nn.ModuleList(blocks), eps
        self.norms = nn.ParameterList(nn.Parameter(torch.ones(hidden, device=device, dtype=dtype)) for _ in range(2 * len(mixers) + 1))

    def forward(self, x, plan, cache, state, rotary, prefix=False):
        """The normed rows [T, hidden] of a pass's x [T, hidden]. cache: a LinesCache with a layer for each LinesAttention
        among the mixers, state: a LinesState with one for each LinesDelta, in the mixers' order (None where there is
        none); prefix: the pass is the one over the shared prefix (plan_prefix's)."""
        normed = nn.functional.rms_norm(x, (x.shape[1],), self.norms[0], self.eps)
        attention = linear = 0
        for i, (mixer, block) in enumerate(zip(self.mixers, self.blocks)):
            if isinstance(mixer, LinesAttention):
                y = mixer(normed, plan, cache.k[attention], cache.v[attention], rotary)
                attention += 1
            else:
                conv, delta = (state.prefix_conv, state.prefix_delta) if prefix else (state.conv, state.delta)
                y = mixer(normed, plan, conv[linear], delta[linear])
                linear += 1
            x, normed = kernels.add_norm(y, x, self.norms[2 * i + 1], eps=self.eps)
            x, normed = kernels.add_norm(block(normed.unsqueeze(1)).squeeze(1), x, self.norms[2 * i + 2], eps=self.eps)
        return normed
