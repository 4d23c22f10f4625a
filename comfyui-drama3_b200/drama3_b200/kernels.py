"""The reference's kernel module surface (drama3/kernels.py:604-724), backed by libdrama3_b200.so instead of NVRTC.

Same function names, arguments, output shapes and dtypes; every output is allocated with torch on the input's device
and every launch goes on the device's current stream, so calls can be captured in CUDA graphs. Differences:
  - `available` returns False only for non-CUDA devices (as the reference does); on a CUDA device it raises if the
    library is missing or the device is not an sm_100 GPU: there is no fallback implementation;
  - `route` and `weighted_sum` also take several rows at once;
  - `await_cpu` (the CPU-expert handshake) is not provided: this path has no CPU side;
  - `moe_decode` is new: the whole resident decode (gate_up, SwiGLU, down, combine) for 1..16 rows in one pass;
  - `grouped_mma` is new: the grouped kernels on the tensor cores for banks held whole on the GPU;
  - `lines_plan`, `qk_norm_rope` and `lines_attention` are new: the attention half of a decoder layer for lines decoded
    together, over a paged key/value cache with a prefix that the lines share.
"""
import ctypes
import functools
import math
from typing import NamedTuple

import torch

from . import _lib
from ._lib import check, lib

ROWS_PER_BLOCK = 16


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


@functools.cache
def _device_ok(index):
    with torch.cuda.device(index):
        check(lib().d3_device_check(), f"cuda:{index}")
    return True


def available(device):
    """Whether `device` runs these kernels: a CUDA device that is an sm_100 GPU, with the library built. Raises on a
    CUDA device where that is not so (no fallback); False for other devices."""
    device = torch.device(device)
    if device.type != "cuda":
        return False
    index = device.index if device.index is not None else torch.cuda.current_device()
    return _device_ok(index)


def _on(device):
    available(device)
    return torch.cuda.device(device)


def resolve(ids, layer, layers, num_experts, half_life, cpu, admit, table, owner, score, at, pending, clock, budget,
            reads, step, share):
    """plan [k, 2] int32 for the row's experts `ids` [k] (int64) of `layer` (drama3/kernels.py:618-625)."""
    plan = torch.empty((ids.shape[0], 2), dtype=torch.int32, device=ids.device)
    with _on(ids.device):
        check(lib().d3_resolve(_ptr(ids), ids.shape[0], int(layer), int(layers), int(num_experts), _ptr(table),
                               _ptr(owner), _ptr(score), _ptr(at), _ptr(pending), owner.shape[0], _ptr(clock),
                               _ptr(budget), _ptr(plan), _ptr(reads), _ptr(step), _ptr(share), float(half_life),
                               int(cpu), float(admit), _stream(ids.device)), "resolve")
    return plan


def await_cpu(plan, flag, step, result, timeout_us, took_over):
    raise NotImplementedError("drama3_b200 has no CPU-expert side: every expert runs on the GPU")


def rotate(x, only_if, swiglu=False):
    """Rows of x [rows, K] (float32 or bfloat16; float32 [rows, 2K] gate | up with `swiglu`, SiLU(gate) * up first)
    in the ConvRot basis: float32 [rows, K]; left unset when `only_if` (an int32 on the GPU) is 0
    (drama3/kernels.py:636-644)."""
    rows, width = x.shape
    k = width // 2 if swiglu else width
    mode = 2 if swiglu else (1 if x.dtype == torch.bfloat16 else 0)
    if mode != 1 and x.dtype != torch.float32:
        raise TypeError(f"rotate takes float32 or bfloat16 rows, not {x.dtype}")
    x = x.contiguous()
    out = torch.empty((rows, k), dtype=torch.float32, device=x.device)
    with _on(x.device):
        check(lib().d3_rotate(_ptr(x), mode, rows, k, _ptr(out), _ptr(only_if), _stream(x.device)), "rotate")
    return out


def route(logits, k):
    """(ids [rows, k] int64, weights [rows, k] float32) of router logits [rows, n] (bfloat16): the k largest, by
    descending logit (ties: lower index first), and their softmax weights renormalized over them, rounded to
    bfloat16 (drama3/kernels.py:647-653, for any number of rows)."""
    if logits.dtype != torch.bfloat16:
        raise TypeError("route takes bfloat16 logits")
    logits = logits.contiguous()
    rows, n = logits.shape
    ids = torch.empty((rows, k), dtype=torch.int64, device=logits.device)
    weights = torch.empty((rows, k), dtype=torch.float32, device=logits.device)
    with _on(logits.device):
        check(lib().d3_route(_ptr(logits), rows, n, int(k), _ptr(ids), _ptr(weights), _stream(logits.device)), "route")
    return ids, weights


def _aligned16(t):
    """t, or a copy of it where its data does not start on a 16-byte boundary (the bulk copies' rule)."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def router(x, weight, k, logits=False):
    """(ids [rows, k] int64, weights [rows, k] float32[, logits [rows, E] bfloat16]) of decode rows x [rows, H]
    (bfloat16, rows <= 16) through a bias-free bf16 router linear `weight` [E, H] and the decode routing, in one launch:
    route(x @ weight.T, k) with the logits as the bf16 rounding of fp32 sums of the exact products."""
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError("router takes bfloat16 rows and weight")
    x, weight = _aligned16(x.contiguous()), _aligned16(weight.contiguous())
    rows, H = x.shape
    E = weight.shape[0]
    ids = torch.empty((rows, k), dtype=torch.int64, device=x.device)
    w = torch.empty((rows, k), dtype=torch.float32, device=x.device)
    lg = torch.empty((rows, E), dtype=torch.bfloat16, device=x.device) if logits else None
    with _on(x.device):
        check(lib().d3_router(_ptr(x), rows, H, _ptr(weight), E, int(k), _ptr(ids), _ptr(w), _ptr(lg),
                              _stream(x.device)), "router")
    return (ids, w, lg) if logits else (ids, w)


def router_fits(rows, hidden, experts, k):
    """Whether `router` takes these shapes."""
    return 1 <= rows <= 16 and hidden == 2048 and experts % 64 == 0 and 64 <= experts <= 256 and k <= min(32, experts)


_SHARED_SCRATCH = {}


def shared_expert(x, gate_up, down, gate, out):
    """out [rows, H] bfloat16 += sigmoid(x @ gate.T) * down(SwiGLU(gate_up(x))) for decode rows x [rows, H] (bfloat16,
    rows <= 16), in place, in two launches; gate_up [2I, H], down [H, I], gate [1, H] or [H], all bfloat16 (the
    reference's SharedExpert and shared_expert_gate linears, drama3/model.py:40-47,123). Returns out."""
    for t in (x, gate_up, down, gate, out):
        if t.dtype != torch.bfloat16:
            raise TypeError("shared_expert takes bfloat16 tensors")
    x, gate_up, down, gate = (_aligned16(t.contiguous()) for t in (x, gate_up, down, gate))
    if not out.is_contiguous():
        raise ValueError("out must be contiguous (it is updated in place)")
    rows, H = x.shape
    I = down.shape[1]
    # scratch: the SwiGLU rows [rows, I] bf16, then the gate [rows] fp32
    key = (x.device, torch.cuda.current_stream(x.device).cuda_stream, rows, I)
    if torch.cuda.is_current_stream_capturing():
        scratch = torch.empty(rows * (I + 2), dtype=torch.bfloat16, device=x.device)
    else:
        scratch = _SHARED_SCRATCH.get(key)
        if scratch is None:
            scratch = _SHARED_SCRATCH[key] = torch.empty(rows * (I + 2), dtype=torch.bfloat16, device=x.device)
    with _on(x.device):
        check(lib().d3_shared_expert(_ptr(x), rows, H, _ptr(gate_up), _ptr(down), _ptr(gate), I, _ptr(scratch),
                                     _ptr(out), _stream(x.device)), "shared_expert")
    return out


def shared_expert_fits(rows, hidden, intermediate):
    """Whether `shared_expert` takes these shapes."""
    return 1 <= rows <= 16 and hidden == 2048 and intermediate in (256, 512, 768, 1024)


def prefill_plan(topk_idx, num_experts, drop_invalid=False):
    """(order [P] int64, pos [P] int64, groups [E + 1, 5] int32) of a prompt's routing [T, k] sorted by expert on the
    device in one launch, no host sync: order holds the (token, rank) pairs by expert id, within an expert in index
    order, ids outside [0, E) last; pos its inverse; groups (expert, slot, 0, first, rows) for every expert and one
    last group for the out-of-range ids (0 rows when drop_invalid). num_experts <= 256 (drama3/offload.py:141-145
    sorts on the host)."""
    flat = topk_idx.reshape(-1).to(torch.int64).contiguous()
    P = flat.numel()
    order = torch.empty(P, dtype=torch.int64, device=flat.device)
    pos = torch.empty(P, dtype=torch.int64, device=flat.device)
    groups = torch.empty((num_experts + 1, 5), dtype=torch.int32, device=flat.device)
    with _on(flat.device):
        check(lib().d3_prefill_plan(_ptr(flat), P, int(num_experts), int(bool(drop_invalid)), _ptr(order), _ptr(pos),
                                    _ptr(groups), _stream(flat.device)), "prefill_plan")
    return order, pos, groups


def prefill_plan_fits(num_experts):
    """Whether `prefill_plan` takes this many experts."""
    return 1 <= num_experts <= 256


def weighted_sum(parts, weights):
    """[rows, H] bfloat16: parts [rows * k, H] (float32) summed per row by weights [rows, k] or [k] (float32), in
    rank order (drama3/kernels.py:656-661; there rows == 1)."""
    weights = weights.reshape(-1, weights.shape[-1]).float().contiguous()
    rows, k = weights.shape
    parts = parts.contiguous()
    H = parts.shape[-1]
    if parts.numel() != rows * k * H:
        raise ValueError("parts must hold rows * k rows")
    out = torch.empty((rows, H), dtype=torch.bfloat16, device=parts.device)
    with _on(parts.device):
        check(lib().d3_weighted_sum(_ptr(parts), _ptr(weights), rows, k, H, _ptr(out), _stream(parts.device)),
              "weighted_sum")
    return out


def _bank_rows(fields, key, n):
    return fields[key].shape[0] // n


def gemv_int8(x, ids, plan, took_over, late, slot_fields, host_fields, n):
    """[k, n] float32: each expert's int8 rows against x [1 or k, K] (float32, rotated); fields are
    {"_qdata", "scale"} (drama3/kernels.py:664-671)."""
    k, width = ids.shape[0], x.shape[1]
    out = torch.empty((k, n), dtype=torch.float32, device=x.device)
    with _on(x.device):
        check(lib().d3_gemv_int8(_ptr(x), x.shape[0], _ptr(ids), _ptr(plan), _ptr(took_over), int(late), k,
                                 _ptr(slot_fields["_qdata"]), _ptr(slot_fields["scale"]), _ptr(host_fields["_qdata"]),
                                 _ptr(host_fields["scale"]), _ptr(out), n, width,
                                 _bank_rows(host_fields, "_qdata", n), _bank_rows(slot_fields, "_qdata", n),
                                 _stream(x.device)), "gemv_int8")
    return out


def gemv_fp8(x, ids, plan, slot_fields, host_fields, n):
    """[k, n] float32: each expert's float8 rows against x [1 or k, K] float32; fields are {"weight", "scale"}
    (drama3/kernels.py:674-681)."""
    k, width = ids.shape[0], x.shape[1]
    out = torch.empty((k, n), dtype=torch.float32, device=x.device)
    with _on(x.device):
        check(lib().d3_gemv_fp8(_ptr(x), x.shape[0], _ptr(ids), _ptr(plan), k, _ptr(slot_fields["weight"]),
                                _ptr(slot_fields["scale"]), _ptr(host_fields["weight"]), _ptr(host_fields["scale"]),
                                _ptr(out), n, width, _bank_rows(host_fields, "weight", n),
                                _bank_rows(slot_fields, "weight", n), _stream(x.device)), "gemv_fp8")
    return out


def gemv_codes(x, ids, plan, slot_fields, host_fields, codebook, bits, n):
    """gemv_int8 for W4A8/W6A8 banks; fields are {"_qdata", "scale" (e4m3), "s_channel"}, codebook [16] at 4 bits
    (drama3/kernels.py:703-713)."""
    k, width = ids.shape[0], x.shape[1]
    out = torch.empty((k, n), dtype=torch.float32, device=x.device)
    with _on(x.device):
        check(lib().d3_gemv_codes(_ptr(x), x.shape[0], _ptr(ids), _ptr(plan), k, _ptr(slot_fields["_qdata"]),
                                  _ptr(slot_fields["scale"]), _ptr(slot_fields["s_channel"]),
                                  _ptr(host_fields["_qdata"]), _ptr(host_fields["scale"]),
                                  _ptr(host_fields["s_channel"]), _ptr(codebook), int(bits), _ptr(out), n, width,
                                  _bank_rows(host_fields, "_qdata", n), _bank_rows(slot_fields, "_qdata", n),
                                  _stream(x.device)), "gemv_codes")
    return out


def grouped_int8(x, groups, slot_fields, host_fields, n):
    """[rows, n] float32 for x's rows (float32, rotated, sorted by expert) through their experts; groups [g, 5] int32
    (expert, slot, fill, first, rows). Rows outside every group are left unset (drama3/kernels.py:684-691)."""
    out = torch.empty((x.shape[0], n), dtype=torch.float32, device=x.device)
    with _on(x.device):
        check(lib().d3_grouped_int8(_ptr(x), x.shape[0], _ptr(groups), groups.shape[0], _ptr(slot_fields["_qdata"]),
                                    _ptr(slot_fields["scale"]), _ptr(host_fields["_qdata"]),
                                    _ptr(host_fields["scale"]), _ptr(out), n, x.shape[1],
                                    _bank_rows(host_fields, "_qdata", n), _bank_rows(slot_fields, "_qdata", n),
                                    _stream(x.device)), "grouped_int8")
    return out


def grouped_fp8(x, groups, slot_fields, host_fields, n):
    """grouped_int8 for float8 experts, against float32 rows x (drama3/kernels.py:694-700)."""
    out = torch.empty((x.shape[0], n), dtype=torch.float32, device=x.device)
    with _on(x.device):
        check(lib().d3_grouped_fp8(_ptr(x), x.shape[0], _ptr(groups), groups.shape[0], _ptr(slot_fields["weight"]),
                                   _ptr(slot_fields["scale"]), _ptr(host_fields["weight"]),
                                   _ptr(host_fields["scale"]), _ptr(out), n, x.shape[1],
                                   _bank_rows(host_fields, "weight", n), _bank_rows(slot_fields, "weight", n),
                                   _stream(x.device)), "grouped_fp8")
    return out


def grouped_codes(x, groups, slot_fields, host_fields, codebook, bits, n):
    """grouped_int8 for W4A8/W6A8 banks (drama3/kernels.py:716-724)."""
    out = torch.empty((x.shape[0], n), dtype=torch.float32, device=x.device)
    with _on(x.device):
        check(lib().d3_grouped_codes(_ptr(x), x.shape[0], _ptr(groups), groups.shape[0], _ptr(slot_fields["_qdata"]),
                                     _ptr(slot_fields["scale"]), _ptr(slot_fields["s_channel"]),
                                     _ptr(host_fields["_qdata"]), _ptr(host_fields["scale"]),
                                     _ptr(host_fields["s_channel"]), _ptr(codebook), int(bits), _ptr(out), n,
                                     x.shape[1], _bank_rows(host_fields, "_qdata", n),
                                     _bank_rows(slot_fields, "_qdata", n), _stream(x.device)), "grouped_codes")
    return out


@functools.cache
def grouped_tile_rows():
    """Rows per tile of the tensor-core grouped kernel (its MMA N at most)."""
    return int(lib().d3_grouped_mma_tile_rows())


def grouped_tiles(counts):
    """Row tiles the tensor-core grouped kernel runs for groups of these row counts."""
    t = grouped_tile_rows()
    return sum((int(n) + t - 1) // t for n in counts)


def grouped_mma_fits(n, k):
    """Whether an [n, k] bank runs on the tensor-core grouped kernel (n % 128 == 0, k % 256 == 0)."""
    return n % 128 == 0 and k % 256 == 0 and k >= 256


GM_ROTATE, GM_SWIGLU = 1, 2


def grouped_mma(kind, x, groups, fields, codebook, n, tiles, row_index=None, rotate=False, swiglu=False):
    """[rows, n] float32 for the sorted rows through their experts, on the tensor cores, for a bank held whole on the
    GPU: the grouped_fp8 / grouped_int8 / grouped_codes results with every group's slot = its expert's index in
    `fields` (drama3/offload.py:126-149). groups [g, 5] int32 on the GPU; tiles = grouped_tiles(row counts), or any
    bound on it (the kernels count the tiles the groups need on the device; offload.prefill_plan gives one). Sorted
    row s is x[row_index[s]] (x float32 or bfloat16; row_index int64, or None for x itself), optionally through
    SwiGLU (x holds gate | up) and the ConvRot rotation first, as kernels.rotate would give it. Rows outside every
    group are left unset."""
    fmt = _lib.FORMATS[kind]
    w = fields[_lib.WEIGHT_KEY[kind]]
    scale = fields["scale"]
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"grouped_mma takes float32 or bfloat16 rows, not {x.dtype}")
    x = x.contiguous()
    K = x.shape[1] // 2 if swiglu else x.shape[1]
    rows = row_index.shape[0] if row_index is not None else x.shape[0]
    mode = (GM_ROTATE if rotate else 0) | (GM_SWIGLU if swiglu else 0)
    out = torch.empty((rows, n), dtype=torch.float32, device=x.device)
    size = lib().d3_grouped_mma_workspace(int(tiles), K)
    ws = torch.empty((max(size, 256),), dtype=torch.uint8, device=x.device)
    if row_index is not None:
        row_index = row_index.to(torch.int64).contiguous()
    with _on(x.device):
        check(lib().d3_grouped_mma(fmt, _ptr(x), int(x.dtype == torch.bfloat16), _ptr(row_index), mode, _ptr(groups),
                                   groups.shape[0], int(tiles), _ptr(w), _ptr(scale), _ptr(fields.get("s_channel")),
                                   _ptr(codebook), w.shape[0], _ptr(out), n, K, _ptr(ws), ws.numel(),
                                   _stream(x.device)), "grouped_mma")
    return out


def prefill_combine(sorted_out, pos, weights, dtype=torch.bfloat16):
    """[T, H] `dtype` (bfloat16 or float32): out[t] = sum over k' of weights[t, k'] * sorted_out[pos[t, k']] in rank
    order (the scatter, weighting and sum of drama3/offload.py:146-149 in one launch); pos [T, k] int64, weights
    [T, k] fp32 or bf16."""
    T, k = pos.shape
    H = sorted_out.shape[1]
    if dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"prefill_combine writes bfloat16 or float32, not {dtype}")
    out = torch.empty((T, H), dtype=dtype, device=sorted_out.device)
    weights = weights.contiguous()
    if weights.dtype not in (torch.float32, torch.bfloat16):
        weights = weights.float()
    with _on(sorted_out.device):
        check(lib().d3_prefill_combine(_ptr(sorted_out.contiguous()), _ptr(pos.to(torch.int64).contiguous()),
                                       _ptr(weights), int(weights.dtype == torch.bfloat16), T, k, H, _ptr(out),
                                       int(dtype == torch.float32), _stream(sorted_out.device)), "prefill_combine")
    return out


def moe_decode_ep(kind, x, ids, weights, banks, e_first, num_experts, codebooks=(None, None), workspace=None,
                  partial=None, exchange=None):
    """[M, H] float32: moe_decode over this rank's experts only (expert parallelism). `banks` hold experts
    [e_first, e_first + E_local) of the num_experts routed ones (bank expert 0 = expert e_first); pairs routed to other
    ranks' experts are skipped. The result is the routing-weighted sum over this rank's pairs, in rank order;
    summing the ranks' results and rounding to bf16 gives moe_decode's output. With `exchange` (the device struct
    of an ep.PeerExchange) the partial is pushed into every rank's exchange area instead and None is returned;
    ep_reduce then finishes the layer."""
    fmt = _lib.FORMATS[kind]
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"moe_decode_ep takes bfloat16 or float32 rows, not {x.dtype}")
    gate_up, down = banks
    wkey = _lib.WEIGHT_KEY[kind]
    M, H = x.shape
    k = ids.shape[-1]
    w13, w2 = gate_up[wkey], down[wkey]
    e_local = w2.shape[0] // H
    I = w13.shape[0] // (2 * e_local)
    if partial is None and exchange is None:
        partial = torch.empty((M, H), dtype=torch.float32, device=x.device)
    if workspace is None:
        workspace = _default_workspace(M, k, I, x.device)
    x = x.contiguous()
    ids = ids.reshape(M, k).contiguous()
    weights = weights.reshape(M, k).float().contiguous()
    with _on(x.device):
        check(lib().d3_moe_decode_ep(fmt, _ptr(x), int(x.dtype == torch.bfloat16), M, k, int(num_experts),
                                     int(e_first), e_local, H, I, _ptr(ids), _ptr(weights), _ptr(w13),
                                     _ptr(gate_up["scale"]), _ptr(gate_up.get("s_channel")), _ptr(w2),
                                     _ptr(down["scale"]), _ptr(down.get("s_channel")), _ptr(codebooks[0]),
                                     _ptr(codebooks[1]), _ptr(partial), _ptr(exchange), _ptr(workspace),
                                     workspace.numel(), _stream(x.device)), "moe_decode_ep")
    return partial


def ep_reduce(exchange, M, H, out=None):
    """[M, H] bfloat16: waits (bounded) until every rank has pushed its partial for this call into this rank's
    exchange area, then sums them in rank order. `exchange` is the device struct of an ep.PeerExchange."""
    if out is None:
        out = torch.empty((M, H), dtype=torch.bfloat16, device=exchange.device)
    with _on(exchange.device):
        check(lib().d3_ep_reduce(_ptr(exchange), M, H, _ptr(out), _stream(exchange.device)), "ep_reduce")
    return out


def decode_workspace(rows, k, intermediate, device):
    """The workspace moe_decode needs, allocated once by the caller and reused by every call (graph-captured steps
    included). It must start zeroed: its last bytes are the kernel's grid-barrier ticket counter, which each call
    advances by a whole number of rounds, so it never needs resetting. Calls that share one workspace must not overlap
    on the GPU."""
    size = lib().d3_moe_decode_workspace(rows, k, intermediate)
    return torch.zeros((size,), dtype=torch.uint8, device=device)


_WORKSPACES = {}


def _default_workspace(rows, k, intermediate, device):
    """The workspace of a decode call made without one: one per (device, stream, rows, k, intermediate), made on first
    use and kept, so repeated calls allocate and clear nothing (calls on one stream never overlap; calls on different
    streams get different workspaces). During a CUDA-graph capture a fresh one is made (and zeroed) inside the
    graph instead, which owns it."""
    device = torch.device(device)
    if torch.cuda.is_current_stream_capturing():
        return decode_workspace(rows, k, intermediate, device)
    key = (device, torch.cuda.current_stream(device).cuda_stream, rows, k, intermediate)
    if key not in _WORKSPACES:
        _WORKSPACES[key] = decode_workspace(rows, k, intermediate, device)
    return _WORKSPACES[key]


def moe_decode(kind, x, ids, weights, banks, codebooks=(None, None), workspace=None, out=None):
    """[M, H] bfloat16: rows x [M, H] (bfloat16 or float32, M <= 16) through their routed experts ids [M, k] (int64)
    mixed by weights [M, k], with banks (gate_up, down) held whole on the GPU in the reference layouts:
    fp8 {"weight" uint8 [E*2I, H] / [E*H, I], "scale" fp32 block scales}; int8 {"_qdata", "scale"};
    w4/w6 {"_qdata", "scale" (e4m3 bytes), "s_channel"} and a codebook per bank for w4; the BASELINE layouts fp8c
    {"weight", "scale" fp32 [E*N]} and w4a8 / w6a8 {"_qdata", "scale" bf16 [E*N, K/128]}. Each routed expert is read
    once for all M rows."""
    fmt = _lib.FORMATS[kind]
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"moe_decode takes bfloat16 or float32 rows, not {x.dtype}")
    gate_up, down = banks
    wkey = _lib.WEIGHT_KEY[kind]
    M, H = x.shape
    k = ids.shape[-1]
    w13, w2 = gate_up[wkey], down[wkey]
    E = w2.shape[0] // H
    I = w13.shape[0] // (2 * E)
    if out is None:
        out = torch.empty((M, H), dtype=torch.bfloat16, device=x.device)
    if workspace is None:
        workspace = _default_workspace(M, k, I, x.device)
    x = x.contiguous()
    ids = ids.reshape(M, k).contiguous()
    weights = weights.reshape(M, k).float().contiguous()
    scale13, scale2 = gate_up["scale"], down["scale"]
    with _on(x.device):
        check(lib().d3_moe_decode(fmt, _ptr(x), int(x.dtype == torch.bfloat16), M, k, E, H, I, _ptr(ids),
                                  _ptr(weights), _ptr(w13), _ptr(scale13), _ptr(gate_up.get("s_channel")), _ptr(w2),
                                  _ptr(scale2), _ptr(down.get("s_channel")), _ptr(codebooks[0]), _ptr(codebooks[1]),
                                  _ptr(out), _ptr(workspace), workspace.numel(), _stream(x.device)), "moe_decode")
    return out


# ---- the attention half of a decoder layer, for lines decoded together

ROW_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class LinesPlan(NamedTuple):
    """What `lines_plan` returns: the block tables (the caller's, updated), the new tokens' slots [T] and positions [T]
    (int64) and lines [T] (int32, -1 past the last token), the first token of each line cu [B + 1], the lines' lengths
    [B] and the used part of the free list [1] after the pass (int32), and the attention's work list for `group` query
    heads per KV head. prefix_table: of the prefix that the plan counts, where who made the plan holds it (a LinesCache)."""
    table: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    line: torch.Tensor
    cu: torch.Tensor
    lengths: torch.Tensor
    used: torch.Tensor
    work: torch.Tensor
    page: int
    group: int
    prefix_table: torch.Tensor = None


def _ints(name, t, device, count):
    """Refuses anything but a contiguous int32 tensor of `count` values on `device`."""
    if t.dtype is not torch.int32 or t.numel() != count or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {count} values on {device}, not {t.dtype} "
                         f"{list(t.shape)} on {t.device}")


@functools.lru_cache(maxsize=1024)
def _int64s(values):
    """The strides as the C array that the library takes (kept by value: a step's tensors have the same ones)."""
    return (ctypes.c_int64 * len(values))(*values)


def _launch(device, what, fn, *args):
    """fn(*args, stream) on the device's current stream; raises on a refusal. Made for calls of a few microseconds:
    the device is switched only where it is another than the current one."""
    _device_ok(device.index)
    if device.index == torch.cuda.current_device():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if status:
        check(status, what)


def _gpu_of(t, what):
    """The CUDA device of a tensor; raises where it is on none."""
    device = t.device
    if device.type != "cuda":
        raise ValueError(f"{what} takes tensors on a GPU, not on {device}")
    return device


def lines_plan(lengths, counts, table, free, used, page, tokens, prefix=None, group=1):
    """The plan of a pass that appends counts [B] tokens to lines that hold lengths [B] tokens of their own (int32, on
    the GPU; nothing is read back to the host): a LinesPlan for `tokens` token places (the rows of the pass's tensors;
    places past the lines' last token belong to no line). Each line takes the pages of `page` tokens that it needs
    beyond its own from free[used:] (int32, used [1]) into its row of table [B, W], in line order; table is updated in
    place, lengths and used are not: the plan's are the state after the pass. prefix [1] (int32): tokens of the prefix
    that the lines share, which come first in their positions. group: query heads per KV head of the attention that
    will use the plan. A page that the free list or the table has no room for is -1, as its tokens' slots are, and is
    recorded in the fault word."""
    device = _gpu_of(lengths, "lines_plan")
    if lengths.dim() != 1 or table.dim() != 2 or free.dim() != 1:
        raise ValueError("lines_plan takes lengths and counts [B], a table [B, W], free [F] and used [1]")
    B, T, group = lengths.shape[0], int(tokens), int(group)
    W, F = table.shape[1], free.shape[0]
    _ints("lengths", lengths, device, B)
    _ints("counts", counts, device, B)
    _ints("table", table, device, B * W)
    _ints("free", free, device, F)
    _ints("used", used, device, 1)
    if prefix is not None:
        _ints("prefix", prefix, device, 1)
    size = plan_ints(B, T, group)
    # one allocation for everything, cut up: slots and positions (int64), then the work list (16-byte aligned) and the rest
    ints = (size + T + 2 * B + 3) // 2
    slots, positions, rest = torch.empty(2 * T + ints, dtype=torch.int64, device=device).split_with_sizes((T, T, ints))
    work, line, cu, new_lengths, new_used, _ = rest.view(torch.int32).split_with_sizes(
        (size, T, B + 1, B, 1, 2 * ints - size - T - 2 * B - 2))
    _launch(device, "lines_plan", lib().d3_lines_plan, lengths.data_ptr(), counts.data_ptr(), B, table.data_ptr(), W,
            free.data_ptr(), F, used.data_ptr(), _ptr(prefix), int(page), T, group, slots.data_ptr(),
            positions.data_ptr(), line.data_ptr(), cu.data_ptr(), new_lengths.data_ptr(), new_used.data_ptr(),
            work.data_ptr(), size)
    return LinesPlan(table, slots, positions, line, cu, new_lengths, new_used, work, int(page), group)


@functools.lru_cache(maxsize=4096)
def plan_ints(B, T, group):
    """Ints of a plan's work list, an even number; raises where there is no plan for these sizes."""
    size = lib().d3_lines_plan_ints(B, T, group)
    if size == 0:
        raise ValueError(f"no plan for {B} lines, {T} tokens, {group} query heads per KV head")
    return size + size % 2


def rotary_table(inv_freq, length, device=None):
    """[length, n, 2] float32: cosine and sine of position x inv_freq [n], formed in 64 bits (a 32-bit product of a
    position of many thousands has lost the angle's last digits), for `qk_norm_rope`."""
    angle = torch.arange(length, dtype=torch.float64)[:, None] * torch.as_tensor(inv_freq).detach().double().cpu()[None]
    return torch.stack((angle.cos(), angle.sin()), dim=-1).float().to(device or "cpu")


def rotary_axes(sections, woven=False, device=None):
    """[sum(sections)] uint8: the axis of each rotary frequency, for positions with several axes (time, height,
    width, ...): the first sections[0] frequencies turn by axis 0, the next by axis 1 and so on; with `woven` the axes
    take turns frequency by frequency while they have frequencies left."""
    if woven:
        left, axes = list(sections), []
        while any(left):
            for a, n in enumerate(left):
                if n:
                    axes.append(a)
                    left[a] -= 1
    else:
        axes = [a for a, n in enumerate(sections) for _ in range(n)]
    return torch.tensor(axes, dtype=torch.uint8, device=device or "cpu")


def qk_norm_rope(q, k, rotary, positions, q_weight=None, k_weight=None, eps=1e-6, unit_offset=False, axes=None,
                 pairs=False, v=None, k_cache=None, v_cache=None, slots=None):
    """(q_out [T, Hq, D], k_out [T, Hkv, D]): queries and keys (bfloat16, float16 or float32; any strides with the last
    dimension contiguous, so views of a fused projection's output) through the RMS norm of each head with q_weight /
    k_weight [D] (of the rows' type or float32; 1 + weight with unit_offset; None: no norm) and the rotation of their
    first 2 n columns by rotary [length, n, 2] (`rotary_table`), halves (f, f + n) or, with `pairs`, neighbours (2f,
    2f + 1). positions: [T] int64, or [A, T] with axes [n] uint8 (`rotary_axes`) naming the row that turns each
    frequency (contiguous). With k_cache and v_cache [pages, page, Hkv, D], v [T, Hkv, D] and slots [T] (int64, a LinesPlan's) the
    keys and the values go to their slots of the caches instead (-1: nowhere) and k_out is None. One launch; 32-bit
    arithmetic, rounded once."""
    tensors = (q, k, rotary, positions, q_weight, k_weight, axes, v, k_cache, v_cache, slots)
    forms = tuple([None if t is None else (t.dtype, t.get_device(), t.shape, t.stride()) for t in tensors])
    checked = _ROPE_FORMS.get(forms)
    if checked is None:
        if len(_ROPE_FORMS) >= 4096:
            _ROPE_FORMS.clear()
        checked = _ROPE_FORMS[forms] = _rope_arguments(*tensors)
    device, q_strides, k_strides, v_strides, sizes, w_f32, table, axes_n, cached = checked
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if cached is None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        to = (k_out.data_ptr(), None, None, None, None, 0, 0, None)
    else:
        k_out = None
        kc_strides, vc_strides, pages, page = cached
        to = (None, k_cache.data_ptr(), kc_strides, v_cache.data_ptr(), vc_strides, pages, page, slots.data_ptr())
    _launch(device, "qk_norm_rope", lib().d3_qk_norm_rope, q.data_ptr(), q_strides, k.data_ptr(), k_strides, _ptr(v),
            v_strides, *sizes, _ptr(q_weight), _ptr(k_weight), w_f32, 1.0 if unit_offset else 0.0, eps,
            rotary.data_ptr(), *table, positions.data_ptr(), axes_n, _ptr(axes), 1 if pairs else 0, q_out.data_ptr(), *to)
    return q_out, k_out


# forms (types, devices, shapes and strides) of qk_norm_rope's tensors that were checked -> the arguments they give. A
# step's tensors have the same ones in every layer, and the checks took as long as the launch.
_ROPE_FORMS = {}


def _rope_arguments(q, k, rotary, positions, q_weight, k_weight, axes, v, k_cache, v_cache, slots):
    """Refuses tensors of a form that qk_norm_rope does not take; the arguments that follow from their forms."""
    device = _gpu_of(q, "qk_norm_rope")
    for t in (k, rotary, positions, q_weight, k_weight, axes, v, k_cache, v_cache, slots):
        if t is not None and t.device != device:
            raise ValueError(f"qk_norm_rope: every tensor must be on {device}")
    if q.dtype not in ROW_TYPES or k.dtype != q.dtype:
        raise TypeError(f"qk_norm_rope takes bfloat16, float16 or float32 rows of one type, not {q.dtype} and {k.dtype}")
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("qk_norm_rope takes q [T, Hq, D] and k [T, Hkv, D]")
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    if k.shape != (T, Hkv, D) or q.stride(2) != 1 or k.stride(2) != 1:
        raise ValueError("q [T, Hq, D] and k [T, Hkv, D] must agree in T and D, their last dimension contiguous")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if w.shape != (D,) or not w.is_contiguous() or w.dtype not in (q.dtype, torch.float32) or w.dtype != weights[0].dtype:
            raise ValueError("q_weight and k_weight must be contiguous [D] tensors of the rows' type or float32, alike")
    if rotary.dtype != torch.float32 or rotary.dim() != 3 or rotary.shape[2] != 2 or not rotary.is_contiguous():
        raise ValueError("rotary must be a contiguous float32 [length, n, 2] tensor")
    length, n = rotary.shape[:2]
    if 2 * n > D:
        raise ValueError(f"rotary turns {2 * n} columns of {D}")
    if (positions.dtype != torch.int64 or positions.dim() != (1 if axes is None else 2) or positions.shape[-1] != T
            or not positions.is_contiguous()):
        raise ValueError("positions must be contiguous int64 [T], or [A, T] with axes")
    if axes is not None and (axes.dtype != torch.uint8 or axes.shape != (n,) or not axes.is_contiguous()):
        raise ValueError("axes must be a contiguous uint8 tensor with the axis of each of the n frequencies")
    if any((x is not None) != (k_cache is not None) for x in (v, v_cache, slots)):
        raise ValueError("v, k_cache, v_cache and slots go together")
    cached = v_strides = None
    if k_cache is not None:
        if v.shape != k.shape or v.dtype != q.dtype or v.stride(2) != 1:
            raise ValueError("v must be [T, Hkv, D] of the rows' type, its last dimension contiguous")
        for c in (k_cache, v_cache):
            if c.dim() != 4 or c.shape != k_cache.shape or c.shape[2:] != (Hkv, D) or c.dtype != q.dtype or c.stride(3) != 1:
                raise ValueError("the caches must be [pages, page, Hkv, D] of the rows' type, alike, the last dimension contiguous")
        if slots.dtype != torch.int64 or slots.shape != (T,) or not slots.is_contiguous():
            raise ValueError("slots must be a contiguous int64 [T] tensor")
        cached = (_int64s(k_cache.stride()), _int64s(v_cache.stride()), k_cache.shape[0], k_cache.shape[1])
        v_strides = _int64s(v.stride())
    return (device, _int64s(q.stride()), _int64s(k.stride()), v_strides, (ROW_TYPES[q.dtype], T, Hq, Hkv, D),
            int(bool(weights) and weights[0].dtype == torch.float32), (2 * n, length),
            1 if axes is None else positions.shape[0], cached)


def lines_attention(q, k_cache, v_cache, plan, prefix_table=None, scale=None, lse=False):
    """[T, Hq, D] (and, with `lse`, [T, Hq] float32: the log of each row's sum of exponentials): the attention of the
    plan's tokens q [T, Hq, D] (bfloat16 or float16) over the paged caches [pages, page, Hkv, D] of the same type, whose
    keys of this pass are written (`qk_norm_rope`). A token sees the keys of the shared prefix, in the pages of
    prefix_table [PW] (int32; their number was given to `lines_plan`; None: the plan's, if it has one), and its line's own keys up to its own; query
    head h reads KV head h / (Hq / Hkv), scale defaults to 1 / sqrt(D). D 64, 128 or 256; page 16, 32 or a multiple of
    64. Where the lines bring few tokens, the prefix's keys are read once for all of them (up to T * Hq / Hkv = 32768,
    token places without a token counted too; past that each line reads them for itself). Places of the plan without a
    token get zeros (lse -inf), and all places do where the plan is another pass's or the pass is too long (2^30 key tiles
    over all heads and rows: about a million tokens of a prompt), which the fault word records. What the cache holds past a
    line's length is never used; a value that is not finite reaches the line's own tokens of its tile of 128 keys, earlier
    ones too."""
    T, Hq, D = q.shape
    kind = ROW_TYPES.get(q.dtype)
    if (kind != 0 and kind != 1) or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise TypeError("lines_attention takes bfloat16 or float16 queries and caches of one type")
    device = _gpu_of(q, "lines_attention")
    pages, page, Hkv = k_cache.shape[:3]
    if k_cache.shape != (pages, page, Hkv, D) or v_cache.shape != k_cache.shape:
        raise ValueError("the caches must be [pages, page, Hkv, D], alike")
    q_strides, kc_strides, vc_strides = q.stride(), k_cache.stride(), v_cache.stride()
    if q_strides[2] != 1 or kc_strides[3] != 1 or vc_strides[3] != 1:
        raise ValueError("the last dimension of the queries and the caches must be contiguous")
    table, work = plan.table, plan.work
    B, W = table.shape
    if plan.page != page or plan.slots.shape[0] != T or plan.group * Hkv != Hq:
        raise ValueError(f"the plan is for {plan.slots.shape[0]} tokens, pages of {plan.page} and {plan.group} query heads "
                         f"per KV head, not for {T}, {page} and {Hq} / {Hkv}")
    if k_cache.device != device or v_cache.device != device or work.device != device:
        raise ValueError(f"lines_attention: every tensor must be on {device}")
    _ints("the plan's table", table, device, B * W)
    if work.dtype is not torch.int32 or not work.is_contiguous():
        raise ValueError("the plan's work list must be a contiguous int32 tensor")
    if work.numel() != plan_ints(B, T, plan.group):
        # another pass's list, which the kernel must not read past its end: one of this size that it refuses instead
        work = torch.zeros(plan_ints(B, T, plan.group), dtype=torch.int32, device=device)
    prefix_pages = 0
    if prefix_table is None:
        prefix_table = plan.prefix_table
    if prefix_table is not None:
        prefix_pages = prefix_table.numel()
        _ints("prefix_table", prefix_table, device, prefix_pages)
    size = _attention_workspace(device.index, T, Hq, Hkv, D)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    sums = torch.empty((T, Hq), dtype=torch.float32, device=device) if lse else None
    # scratch of this call alone: it makes two launches, and those of another thread on the same stream may come between
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    _launch(device, "lines_attention", lib().d3_lines_attention, q.data_ptr(), _int64s(q_strides), kind, T, Hq, Hkv, D,
            k_cache.data_ptr(), _int64s(kc_strides), v_cache.data_ptr(), _int64s(vc_strides), pages, page,
            table.data_ptr(), W, _ptr(prefix_table), prefix_pages, work.data_ptr(), B,
            1.0 / math.sqrt(D) if scale is None else scale, out.data_ptr(), _ptr(sums), ws.data_ptr(), size)
    return (out, sums) if lse else out


@functools.lru_cache(maxsize=1024)
def _attention_workspace(index, T, Hq, Hkv, D):
    """Bytes of workspace of an attention of these sizes on cuda:index; raises where there is no kernel for them."""
    _device_ok(index)
    with torch.cuda.device(index):
        size = lib().d3_lines_attention_workspace(T, Hq, Hkv, D)
    if size == 0:
        raise ValueError(f"no attention kernel for {Hq} / {Hkv} heads of {D}")
    return size
