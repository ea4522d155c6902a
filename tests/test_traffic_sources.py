"""The sources that bench.py's measured traffic is stamped with: whatever a listed file includes is listed too, so that a kernel that moves into a
header still invalidates its figure."""
import re
from pathlib import Path

import pytest

import bench

CSRC = Path(bench.ROOT) / "triton_grouped_gemm_amd" / "csrc"
DECLARATIONS = {"launch.hpp"}  # prototypes of host functions: nothing that a kernel's traffic depends on


def included(name):
    return {i for i in re.findall(r'#include "([^"]+)"', (CSRC / name).read_text())}


@pytest.mark.parametrize("source_set", sorted(bench.TRAFFIC_SOURCES))
def test_a_set_holds_what_its_files_include(source_set):
    listed = set(bench.TRAFFIC_SOURCES[source_set])
    missing = {i for name in listed for i in included(name)} - listed - DECLARATIONS
    assert not missing


def test_the_files_left_out_have_no_device_code():
    for name in DECLARATIONS:
        assert not re.search(r"__global__|__device__|TGG_DEV|TGG_HD|constexpr|#define", (CSRC / name).read_text())


@pytest.mark.parametrize("source_set,kernels", [("gemm16", ["gemm_w4_kernel", "gemm_fast_kernel", "gemm_fast_auto_kernel"]), ("wgrad16", ["gemm_wgrad_kernel"]),
                                                ("gemm8", ["gemm_fp8_auto_kernel"]), ("wgrad8", ["fp8_w4_kernel"]), ("permute", ["moe_permute_rows_kernel", "moe_unpermute_kernel"]),
                                                ("quant", ["trans_quant128_kernel", "token_cast128_kernel"])])
def test_a_set_holds_the_kernels_that_were_measured(source_set, kernels):
    text = "".join((CSRC / name).read_text() for name in bench.TRAFFIC_SOURCES[source_set])
    for kernel in kernels:
        assert re.search(r"__global__[^;{]*\b" + kernel + r"\(", text, re.S), kernel
