"""Lines decoded together behind a shared prompt, through whole decoder layers: attention (LinesAttention over a paged
LinesCache) and routed experts (SparseMoeBlock), random weights of a small stack.

    python examples/lines_decode.py [--lines 16] [--prompt 500] [--steps 32] [--layers 4]

The shared prompt is read once, then each line's own text (ragged), then every step appends one token to each line; the
steps are one CUDA graph, replayed. Prints the time of a step."""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "comfyui-drama3_b200"))

from drama3_b200 import kernels  # noqa: E402
from drama3_b200.attention import LinesAttention, LinesCache  # noqa: E402
from drama3_b200.model import SparseMoeBlock, block_config  # noqa: E402

HIDDEN, HEADS, KV_HEADS, HEAD_DIM, EXPERTS, TOP_K, INTERMEDIATE, SHARED = 2048, 32, 4, 128, 32, 8, 512, 512


class Layer(torch.nn.Module):
    """x + attention(norm(x)), then x + experts(norm(x))."""

    def __init__(self, device, dtype, seed):
        super().__init__()
        self.norms = torch.nn.ModuleList(torch.nn.RMSNorm(HIDDEN, eps=1e-6, device=device, dtype=dtype) for _ in range(2))
        self.attention = LinesAttention(HIDDEN, HEADS, KV_HEADS, HEAD_DIM, device=device, dtype=dtype)
        self.moe = SparseMoeBlock(block_config(HIDDEN, EXPERTS, TOP_K, INTERMEDIATE, SHARED, fp8=True, per_channel=True),
                                  device=device, dtype=dtype)
        gen = torch.Generator(device=device).manual_seed(seed)
        for name in ("gate_up", "down"):  # experts of about N(0, 0.02) in float8 with a scale per output channel
            weight, scale = (getattr(self.moe.experts, f"{name}_{part}") for part in ("weight", "scale"))
            scale.data.fill_(0.02)
            weight.data.copy_(torch.randn(weight.shape, generator=gen, device=device).to(weight.dtype))

    def forward(self, x, plan, k, v, rotary, prefix_table):
        x = x + self.attention(self.norms[0](x), plan, k, v, rotary, prefix_table)
        return x + self.moe(self.norms[1](x).unsqueeze(1)).squeeze(1)


def forward(layers, cache, x, plan, rotary, prefix_table):
    for layer, k, v in zip(layers, cache.k, cache.v):
        x = layer(x, plan, k, v, rotary, prefix_table)
    return x


def decode(lines=16, prompt=500, steps=32, n_layers=4, page=64, device="cuda", seed=1):
    """(rows of the last step [lines, hidden], milliseconds per step)."""
    device, dtype = torch.device(device, 0), torch.bfloat16
    torch.manual_seed(seed)
    texts = [5 + 3 * b % 17 for b in range(lines)]
    most = max(texts) + steps + 2
    layers = [Layer(device, dtype, seed + i) for i in range(n_layers)]
    pages = -(-prompt // page) + lines * -(-most // page)
    cache = LinesCache(n_layers, pages, page, KV_HEADS, HEAD_DIM, lines, most, HEADS // KV_HEADS, device)
    rotary = kernels.rotary_table(10000.0 ** (-torch.arange(HEAD_DIM // 2, dtype=torch.float64) / (HEAD_DIM // 2)),
                                  prompt + most, device)
    with torch.no_grad():
        # the shared prompt, then the lines' texts behind it
        forward(layers, cache, torch.randn((prompt, HIDDEN), device=device).to(dtype), cache.plan_prefix(prompt), rotary, None)
        counts = torch.tensor(texts, dtype=torch.int32, device=device)
        x = forward(layers, cache, torch.randn((sum(texts), HIDDEN), device=device).to(dtype),
                    cache.plan(counts, sum(texts)), rotary, cache.prefix_table)
        # each line's last row goes round as its next input: one step, captured and replayed
        row = x[counts.cumsum(0) - 1].clone()
        ones = torch.ones_like(counts)

        def step():
            y = forward(layers, cache, row, cache.plan(ones, lines), rotary, cache.prefix_table)
            row.copy_(torch.nn.functional.rms_norm(y, (HIDDEN,)))

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()  # warm
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step()
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record(stream)
            for _ in range(steps):
                graph.replay()
            end.record(stream)
        stream.synchronize()
    del graph
    return row, start.elapsed_time(end) / steps


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("lines", 16), ("prompt", 500), ("steps", 32), ("layers", 4)):
        ap.add_argument(f"--{name}", type=int, default=value)
    args = ap.parse_args()
    rows, ms = decode(args.lines, args.prompt, args.steps, args.layers)
    print(f"{args.lines} lines behind {args.prompt} shared tokens, {args.layers} layers: {ms:.3f} ms a step, "
          f"rows {tuple(rows.shape)}, norm {float(rows.float().norm()):.3f}")
