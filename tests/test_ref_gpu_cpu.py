"""oracle/ref_gpu.py where the reference's kernels were not built: a comparison with them is skipped, not failed."""
import unittest

import pytest

from oracle import ref_gpu


def test_comparisons_without_the_reference_kernels_are_skipped(monkeypatch, tmp_path):
    monkeypatch.setattr(ref_gpu, "CUBIN", tmp_path / "ref_kernels.cubin")
    ref_gpu._driver.cache_clear()
    assert not ref_gpu.available()
    with pytest.raises(unittest.SkipTest, match="build_ref"):
        ref_gpu._driver()
    with pytest.raises(FileNotFoundError):
        ref_gpu._driver()
