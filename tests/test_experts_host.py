"""Host-side pieces of the expert layers and 4-bit products that need no GPU. They run in a child process:
PyTorch's copy of the HIP runtime is never loaded beside the library's in this one."""
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(code):
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr


# n values (or rows) of which m are taken, and how many neighbours make a row
@pytest.mark.parametrize("n,m,cols", [(5, 5, 1), (8193, 4096, 1), (8000, 4096, 1), (8191, 4096, 1), (4097, 4096, 1),
                                      ((1 << 20) + 1, 1 << 20, 7), (4096 * 320, 1 << 20, 320), (4096 * 640, 1 << 20, 640),
                                      (4096 * 4096, 1 << 20, 4096), (4096 * 1024, 1 << 20, 1024), (10 ** 9, 1000, 64)])
def test_a_sample_is_spread_over_all(n, m, cols):
    run("""
import torch
from h2o4gpu_amd.codebook4 import _spread
n, m, cols = %d, %d, %d
at = _spread(n, m)
stretch = -(-n // m)
assert at.dtype == torch.int64 and at.numel() == m
gaps = at[1:] - at[:-1]
assert int(gaps.min()) >= (1 if n >= 2 * m or n == m else 0) and int(gaps.max()) <= 2 * stretch
assert 0 <= int(at[0]) < stretch and n - stretch <= int(at[-1]) < n
if m >= 64 * cols:  # every column about as often as any other
    share = torch.bincount(at %% cols, minlength=cols).double() * cols / m
    assert 0.8 <= float(share.min()) and float(share.max()) <= 1.2, share
""" % (n, m, cols))


def test_the_library_refuses_groups_that_its_counts_do_not_hold():
    """cols + group is an int in the kernels."""
    run(r"""
from h2o4gpu_amd.libs import experts_hip as e
lib = e.lib()
for group, fine in ((32, True), (e.MAX_GROUP, True), (e.MAX_GROUP + 32, False), (2 ** 31 - 32, False)):
    assert (lib.h2o4gpu_codebook4_scales_bytes(1, 4, 100, group, 0) > 0) == fine, group
    if not fine:
        assert lib.h2o4gpu_codebook4_quantize(0, 4, 100, group, 1.0, 16, 100, 16, 16, 50, 0, 16, None) == -2
        assert lib.h2o4gpu_codebook4_layout(1, 4, 100, group, 16, 50, 0, 16, 16, 16, None) == -2
        assert lib.h2o4gpu_codebook4_product(0, 1, 4, 100, group, 16, 100, 16, 0, 16, 16, 16, 4, None) == -2
import re
assert re.search(r"#define H2O4GPU_CODEBOOK4_MAX_GROUP \(1 << 30\)", open("include/h2o4gpu_experts.h").read())
assert e.MAX_GROUP == 1 << 30
""")


def launches(text):
    """(kernel, bytes of dynamic LDS, what precedes) of every launch in a source."""
    for at in (m.end() for m in re.finditer(r"hipLaunchKernelGGL\(", text)):
        depth, args, start = 0, [], at
        for i in range(at, len(text)):
            if text[i] == "," and depth == 0:
                args.append(text[start:i].strip())
                start = i + 1
            depth += (text[i] in "({[") - (text[i] in ")}]")
            if depth < 0:
                break
        yield args[0], args[3], text[:at]


@pytest.mark.parametrize("name", ["experts_kernels.hip", "codebook4_kernels.hip"])
def test_launches_with_dynamic_lds_raise_their_kernel_s_limit(name):
    """The limit is 64 KB unless it is raised: every launch whose bytes are not a constant goes by the helper."""
    text = open(os.path.join(ROOT, "h2o4gpu_amd", "csrc", name)).read()
    found = list(launches(text))
    assert len(found) >= 4
    for kernel, lds, before in found:
        if lds == "0":
            continue
        asked = "KM_TRY(ensure_dynamic_lds(reinterpret_cast<const void *>(%s), %s));" % (kernel, lds)
        assert asked in before[-1200:], "%s is launched with %s bytes" % (kernel, lds)
