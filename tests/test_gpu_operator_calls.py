"""The calls of perf/operators.py that go through the backend, used beside torch's own work as a program would: no wait for the device between the two (checks: operator_calls_worker.py)."""
import os
import re
import subprocess
import sys

import pytest

import llama_box_amd as L

WORKER = os.path.join(L.REPO, "tests", "operator_calls_worker.py")
CHECKS = [(c, k) for c in ("result_is_read_at_once", "call_waits", "inputs_changed") for k in ("store", "convert", "read", "product", "experts") if (c, k) != ("call_waits", "store")]


@pytest.fixture(scope="module")
def said(built):
    r = subprocess.run([sys.executable, "-u", WORKER], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    return r.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("check,kind", CHECKS)
def test_calls_beside_torch(said, check, kind):
    begun, done = (re.findall(rf"^{word} ({check}:{kind}-\S+)$", said, re.M) for word in ("CHECK", "OK"))
    assert begun and begun == done, said[-6000:]
