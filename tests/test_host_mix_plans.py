"""How the token mixers' calls are cut into launches, on the host: see tests/host_mix/plan_main.cpp.  The entry
points use the same functions (finchmoe_amd/csrc/fm_mix_index.h)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("what", ["steps", "columns", "windows"])
def test_plans(tmp_path, what):
    exe = str(tmp_path / "plan")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined",
                           "-fno-sanitize-recover=undefined", "-Wall", "-Werror", "-o", exe,
                           os.path.join(ROOT, "tests", "host_mix", "plan_main.cpp")])
    r = subprocess.run([exe, what], capture_output=True, text=True, timeout=600, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"))
    assert r.returncode == 0 and "plans hold" in r.stdout, (r.stdout + r.stderr)[-4000:]
