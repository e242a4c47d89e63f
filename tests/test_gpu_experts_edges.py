"""Expert layers and 4-bit products at sizes and uses that take one path of several.

The checks run in one child process (experts_edges_check.py), as those of test_gpu_experts.py do."""
import json
import os
import subprocess
import sys

import pytest

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
HERE = os.path.dirname(os.path.abspath(__file__))

CHECKS = [
    "codebook_of_all_experts",
    "long_sums_of_distances",
    "every_number_by_its_size",
    "small_gradients",
    "tokens_that_are_not_finite",
    "a_token_served_alone",
    "labels_in_order",
    "forward_mode_is_refused",
    "second_derivatives",
    "groups_longer_than_a_row",
]


@pytest.fixture(scope="module")
def results(hip):
    proc = subprocess.run([sys.executable, "-u", os.path.join(HERE, "experts_edges_check.py")] + CHECKS,
                          capture_output=True, text=True, timeout=280)
    found = {}
    for line in proc.stdout.splitlines():
        if line.startswith("{"):
            r = json.loads(line)
            found[r["name"]] = r
    return found, "ended with %s\n%s\n%s" % (proc.returncode, proc.stdout[-1000:], proc.stderr[-3000:])


@pytest.mark.parametrize("name", CHECKS)
def test_check(results, name):
    found, how = results
    assert name in found, how
    assert found[name]["ok"], found[name]["why"]
