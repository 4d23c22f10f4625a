"""Kernels that read by tensor maps, called first of all on a thread that has made no CUDA call yet: encoding a map
needs a current context, which the runtime gives a thread with the first call that needs one."""
import threading

import pytest
import torch

import gpu_data as gd
from test_grouped_mma_gpu import COUNTS, grouped_case
from test_lines_gpu import attn_case, fault

pytestmark = pytest.mark.gpu


def attention(cuda):
    from drama3_b200 import kernels
    q, kc, vc, plan, pt = attn_case(cuda, 16, 2, 128, torch.bfloat16, 16, [300, 20], [1, 1], 500)
    return lambda: kernels.lines_attention(q, kc, vc, plan, prefix_table=pt)


def prompt_pass(cuda):
    from drama3_b200 import kernels
    bank, x, groups = grouped_case("fp8", 1536, 2048, 5, cuda)
    tiles, live = kernels.grouped_tiles(COUNTS), int(sum(COUNTS))
    return lambda: kernels.grouped_mma("fp8", x, groups, bank, None, 1536, tiles)[:live]


def decode(kind):
    def case(cuda):
        from drama3_b200 import kernels
        banks = (gd.rand_bank(kind, 32, 1536, 2048, 5, cuda), gd.rand_bank(kind, 32, 2048, 768, 6, cuda))
        x, (ids, w) = gd.rand_rows(16, 2048, 7, cuda), gd.rand_routing(16, 32, 8, 8, cuda)
        return lambda: kernels.moe_decode(kind, x, ids, w, banks)
    return case


@pytest.mark.parametrize("case", [attention, prompt_pass, decode("fp8c"), decode("w4a8")],
                         ids=["attention", "prompt_pass", "decode_fp8c", "decode_w4a8"])
def test_first_call_of_a_thread(cuda, case, monkeypatch):
    call = case(cuda)
    # asks the runtime, which would give the thread its context before the kernel's own call comes
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    want = call()
    del want  # what a call allocates is held by the allocator from here on, so that the thread's makes no CUDA call for it
    want, got = call(), []

    def run():
        try:
            got.append(call())
        except Exception as e:  # noqa: BLE001
            got.append(e)

    thread = threading.Thread(target=run)
    thread.start()
    thread.join()
    assert isinstance(got[0], torch.Tensor), got[0]
    assert torch.equal(got[0], want) and fault() == 0
