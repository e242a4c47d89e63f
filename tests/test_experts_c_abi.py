"""The library exports every symbol include/h2o4gpu_experts.h declares, the binding names the same
ones, and bad arguments are refused before any device is touched."""
import ctypes
import os
import re
import subprocess

import pytest

from h2o4gpu_amd.libs import experts_hip

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "h2o4gpu_experts.h")


def test_header_parses_as_c():
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Wextra", "-fsyntax-only", "-x", "c", HEADER])


def test_binding_and_header_name_the_same_symbols(hip):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"^\s*(?:int|size_t)\s+(\w+)\s*\(", text, flags=re.M))
    assert names == set(experts_hip.PROTOTYPES)
    handle = ctypes.CDLL(hip.LIB_PATH)
    for name in names:
        assert hasattr(handle, name), name


def test_limits_match_the_header():
    text = open(HEADER).read()
    for name, value in (("MAX_EXPERTS", experts_hip.MAX_EXPERTS), ("MAX_TOP_K", experts_hip.MAX_TOP_K),
                        ("FLOAT32", experts_hip.FLOAT32), ("BFLOAT16", experts_hip.BFLOAT16),
                        ("FLOAT16", experts_hip.FLOAT16)):
        assert re.search(r"#define H2O4GPU_EXPERTS_%s %d\b" % (name, value), text), name


@pytest.mark.parametrize("slots,experts,blocks_needed", [(0, 4, False), (1000, 4, False), (10 ** 6, 64, True),
                                                         (10 ** 6, 0, False), (2 ** 40, 4, False)])
def test_sort_workspace(slots, experts, blocks_needed):
    need = experts_hip.lib().h2o4gpu_experts_sort_workspace(slots, experts)
    assert (need > 0) == blocks_needed and need % 4 == 0


def test_bad_arguments_are_refused_without_a_device():
    lib = experts_hip.lib()
    assert lib.h2o4gpu_experts_route(9, 1, 4, 2, 1, 0, 1.0, 16, 4, 1, 16, 16, None) == -2
    assert lib.h2o4gpu_experts_route(0, 1, 4, 5, 1, 0, 1.0, 16, 4, 1, 16, 16, None) == -2
    assert lib.h2o4gpu_experts_route(0, 1, 4, 2, 1, 0, 1.0, None, 4, 1, 16, 16, None) == -2
    assert lib.h2o4gpu_experts_route(0, 0, 4, 2, 1, 0, 1.0, None, 4, 1, None, None, None) == 0
    assert lib.h2o4gpu_experts_sort(10, 4, None, 16, 16, 16, None, 0, None) == -2
    assert lib.h2o4gpu_experts_dispatch(0, 3, 2, 8, 16, 4, 16, 16, 8, None) == -2
    assert lib.h2o4gpu_experts_combine(0, 3, 2, 8, 16, 8, None, 16, 16, 8, None) == -2
    assert lib.h2o4gpu_codebook4_product(0, 1, 4, 64, 31, 16, 64, 16, 0, 16, 16, 16, 4, None) == -2
    assert lib.h2o4gpu_codebook4_product(0, 1, 4, 64, 32, 16, 64, 8, 0, 16, 16, 16, 4, None) == -2
    assert lib.h2o4gpu_codebook4_layout(1, 4, 64, 32, 16, 31, 0, 16, 16, 16, None) == -2
