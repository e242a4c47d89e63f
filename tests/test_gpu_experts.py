"""Expert layers and 4-bit products against plain implementations in 64 bits, on the GPU.

The cases run in one child process (experts_device_check.py), so that PyTorch's copy of the HIP
runtime is loaded before the library there and never into this process."""
import json
import os
import subprocess
import sys

import pytest

from experts_cases import all_cases

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(900)]
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def results(hip):
    proc = subprocess.run([sys.executable, "-u", os.path.join(HERE, "experts_device_check.py")],
                          capture_output=True, text=True, timeout=850)
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
