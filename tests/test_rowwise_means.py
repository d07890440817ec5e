"""The mean of a row from its sum (``ZpOver``): exact where the sum is a whole multiple of the width.  Host code, run
without a GPU; what the kernels make of it is in test_gpu_rowwise_means.py."""

from __future__ import annotations

import pathlib
import subprocess

import pytest

from zippel_b200.build import CSRC, NVCC_FLAGS, ROOT, nvcc


@pytest.fixture(scope="module")
def means(tmp_path_factory):
    exe = tmp_path_factory.mktemp("means") / "means"
    subprocess.run([nvcc(), *NVCC_FLAGS, "-cudart", "shared", "-I", str(ROOT / "include"), "-I", str(CSRC),
                    str(pathlib.Path(__file__).parent / "native" / "means.cu"), "-o", str(exe)],
                   check=True, capture_output=True)
    return lambda first, last: subprocess.run([str(exe), str(first), str(last)], capture_output=True, text=True).stdout


@pytest.mark.parametrize("first,last", [(1, 4096), (4097, 16384), (16385, 66000)])
def test_means_of_whole_multiples_are_exact(means, first, last):
    assert means(first, last) == "ok\n"
