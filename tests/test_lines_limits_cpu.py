"""What kernels.lines_attention gives the library, seen without a GPU: its launch is replaced by one that looks at the
arguments."""
import ctypes
import threading

import pytest
import torch

from drama3_b200 import _lib, kernels

# of d3_lines_attention's arguments
ARGUMENTS = ("q", "q_strides", "type", "T", "Hq", "Hkv", "D", "k_cache", "kc_strides", "v_cache", "vc_strides", "pages", "page",
             "table", "W", "prefix_table", "PW", "work", "B", "scale", "out", "lse", "workspace", "workspace_bytes")


@pytest.fixture
def launches(monkeypatch):
    """The arguments of each launch, by name; tensors on the CPU pass for tensors on a GPU."""
    seen = []
    monkeypatch.setattr(kernels, "_gpu_of", lambda t, what: t.device)
    monkeypatch.setattr(kernels, "_attention_workspace", lambda *sizes: 4096)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    monkeypatch.setattr(kernels, "_launch", lambda device, what, fn, *args: seen.append(dict(zip(ARGUMENTS, args, strict=True))))
    return seen


def a_pass(lines, tokens, group=2, page=16):
    """Queries, caches and a plan of a pass; the work list is of the right size and holds ones."""
    q = torch.zeros((tokens, 2 * group, 64), dtype=torch.bfloat16)
    cache = torch.zeros((3, page, 2, 64), dtype=torch.bfloat16)
    i = torch.zeros(lines, dtype=torch.int32)
    places = torch.zeros(tokens, dtype=torch.int64)
    work = torch.ones(kernels.plan_ints(lines, tokens, group), dtype=torch.int32)
    return q, cache, kernels.LinesPlan(torch.zeros((lines, 2), dtype=torch.int32), places, places, i, i, i, i, work, page, group)


def test_the_work_list_is_as_long_as_the_kernel_reads(launches):
    q, cache, plan = a_pass(3, 200)
    kernels.lines_attention(q, cache, cache, plan)
    assert launches[-1]["work"] == plan.work.data_ptr()
    size = kernels.plan_ints(3, 200, 2)
    assert size >= _lib.lib().d3_lines_plan_ints(3, 200, 2)
    held = []
    zeros = torch.zeros
    torch_zeros = lambda *a, **k: held.append(zeros(*a, **k)) or held[-1]  # noqa: E731
    for work in (a_pass(1, 2)[2].work, plan.work[:20], plan.work[:0], torch.ones(size + 2, dtype=torch.int32)):
        with pytest.MonkeyPatch.context() as m:
            m.setattr(torch, "zeros", torch_zeros)
            kernels.lines_attention(q, cache, cache, plan._replace(work=work))
        # never the list itself: one of the right size, which says that it was made for no tokens
        assert launches[-1]["work"] == held[-1].data_ptr() != work.data_ptr()
        assert held[-1].shape == (size,) and held[-1].dtype == torch.int32 and not held[-1].any()
        assert ctypes.c_int.from_address(launches[-1]["work"] + 4 * 8).value == 0


@pytest.mark.parametrize("spoil", [lambda w: w.long(), lambda w: w.float(), lambda w: torch.stack((w, w), 1)[:, 0]])
def test_a_work_list_of_another_type_is_refused(launches, spoil):
    q, cache, plan = a_pass(3, 200)
    with pytest.raises(ValueError, match="work list"):
        kernels.lines_attention(q, cache, cache, plan._replace(work=spoil(plan.work)))
    assert not launches


def test_calls_of_two_threads_have_workspaces_of_their_own(launches, monkeypatch):
    """A call is two launches, the attention and the joining of its parts, and both threads' may be in the stream in any
    order: neither may write where the other's parts are."""
    both = threading.Barrier(2, timeout=30)
    inner = kernels._launch

    def launch(*args):
        inner(*args)
        both.wait()  # the other thread is between its launches too

    monkeypatch.setattr(kernels, "_launch", launch)
    q, cache, plan = a_pass(3, 200)
    threads = [threading.Thread(target=kernels.lines_attention, args=(q, cache, cache, plan)) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    (a, b), size = (x["workspace"] for x in launches), launches[0]["workspace_bytes"]
    assert a + size <= b or b + size <= a
