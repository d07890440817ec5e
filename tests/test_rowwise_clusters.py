"""Rows of more than a block's elements where a device runs few clusters of blocks at a time, or none: every call is
served, by fewer clusters or by the kernels of single blocks.  Host code, run without a GPU."""

from __future__ import annotations

import pathlib
import subprocess

import pytest

from zippel_b200.build import CSRC, NVCC_FLAGS, OBJ, ROOT, build_library, nvcc


@pytest.fixture(scope="module")
def clusters(tmp_path_factory):
    build_library()
    exe = tmp_path_factory.mktemp("clusters") / "clusters"
    objects = [str(OBJ / f"zp_rowwise{part}.o") for part in ("", "_fwd", "_bwd")]
    subprocess.run([nvcc(), *NVCC_FLAGS, "-cudart", "shared", "-I", str(ROOT / "include"), "-I", str(CSRC),
                    str(pathlib.Path(__file__).parent / "native" / "clusters.cpp"), *objects, "-o", str(exe)],
                   check=True, capture_output=True)
    return lambda most: subprocess.run([str(exe), str(most)], capture_output=True, text=True).stdout


@pytest.mark.parametrize("most", [0, 1, 2, 3, 4, 5, 7, 8, 9, 18, 37, 74])
def test_wide_rows_are_served_however_few_clusters_run(clusters, most):
    assert clusters(most) == "ok\n"
