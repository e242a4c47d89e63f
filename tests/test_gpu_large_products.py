"""Products in large tiles, of all types and passes, against their formulas in 64 bits, on the GPU.

The cases run in one child process (large_products_check.py), as those of test_gpu_experts.py do."""
import json
import os
import subprocess
import sys

import pytest

from large_products_cases import all_cases

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(600)]
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def results(hip):
    proc = subprocess.run([sys.executable, "-u", os.path.join(HERE, "large_products_check.py")],
                          capture_output=True, text=True, timeout=550)
    found = {}
    for line in proc.stdout.splitlines():
        if line.startswith("{"):
            r = json.loads(line)
            found[r["name"]] = r
    return found, "ended with %s after %d cases\n%s" % (proc.returncode, len(found), proc.stderr[-3000:])


@pytest.mark.parametrize("name", [c["name"] for c in all_cases()])
def test_case(results, name):
    found, how = results
    assert name in found, how
    assert found[name]["ok"], found[name]["why"]
