"""The waits of lines_delta's kernels (csrc/lines_delta_chunk.cuh), read from the source: what happens where one runs out cannot
be made to happen from outside, and must neither leave lanes of a warp behind in a full-warp exchange nor end a block whose
copies are still in flight."""
import re
from pathlib import Path

SOURCE = Path(__file__).resolve().parents[1] / "comfyui-drama3_b200" / "csrc" / "lines_delta_chunk.cuh"


def kernel(name):
    """The body of a kernel, without comments."""
    text = re.sub(r"//[^\n]*", "", SOURCE.read_text())
    at = text.index("{", text.index(f"{name}("))
    depth = 0
    for end in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        if depth == 0:
            return text[at:end + 1]
    raise AssertionError(name)


def test_the_scans_loops_end_for_whole_warps():
    """The loops go on while `ok` holds and exchange values with full masks inside: every value that `ok` gets is the same in
    all lanes (ld_wait and __all_sync vote), never one lane's own."""
    body = kernel("lines_delta_scan_kernel")
    assert body.count("&& ok; ++i)") == 2
    given = [m.group(1) for m in re.finditer(r"(?<![\w.])ok\s*=(?!=)\s*([^;]*);", body)]
    assert len(given) >= 6
    for value in given:
        terms = [t.strip() for t in value.split("&&")]
        assert all(re.match(r"(true$|ld_wait\(|__all_sync\(0xffffffffu, )", t) for t in terms), value


def test_no_block_ends_with_copies_in_flight():
    """Where the preparation's wait for its rows ran out, it waits for them once more before it returns; the scan's loading lane
    waits for every stage that it has asked for."""
    body = kernel("lines_delta_prep_kernel")
    bulk = body.index("bulk_g2s(")
    returns = [m.start() for m in re.finditer(r"\breturn;", body)]
    assert len(returns) == 1 and returns[0] > bulk  # no way out before the copies are asked for
    assert body[bulk:returns[0]].count("mbar_wait(&arrived, 0)") == 2
    body = kernel("lines_delta_scan_kernel")
    assert re.search(r"lane == 0 && !ok\)\s*for \(int i = loads - 1; i >= 0 && i >= loads - STAGES; --i\) mbar_wait\(&full", body)
