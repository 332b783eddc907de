"""GPU: PageStack and PagedKv4Pool of solidattention/hip_kv.hpp, exercised by the self-checking driver
tests/cpp/kv4_check (built by __graft_entry__.build())."""
import json
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXE = os.path.join(ROOT, "tests", "cpp", "kv4_check")


def test_cpp_kv4_check(hip):
    assert os.path.exists(EXE), "tests/cpp/kv4_check missing: run __graft_entry__.build()"
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=110)
    print(r.stdout[-4000:])
    print(r.stderr[-2000:])
    assert r.returncode == 0, f"kv4_check exit {r.returncode}"
    m = json.loads(r.stdout)
    assert m["counted"] and m["released"] and m["refused"] and m["status"] == 0
    assert m["prompt"] <= 1e-5 and m["decode"] <= 1e-5
