"""The token mixers' argument checks and the paged cache's address arithmetic on the host: see
tests/host_mix/mix_main.cpp.  The entry points and kernels use the same functions
(finchmoe_amd/csrc/fm_mix_index.h)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_refusals_and_addresses(tmp_path):
    exe = str(tmp_path / "mix")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined",
                           "-fno-sanitize-recover=undefined", "-Wall", "-Werror", "-o", exe,
                           os.path.join(ROOT, "tests", "host_mix", "mix_main.cpp")])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=600, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"))
    assert r.returncode == 0 and "all refusals and addresses hold" in r.stdout, (r.stdout + r.stderr)[-4000:]


def test_descriptors_match_the_header(tmp_path):
    """sizes and field offsets of the ctypes descriptors against the C structs"""
    from finchmoe_amd import binding as fb
    structs = {"fm_gated_delta_args": fb.GatedDeltaArgs, "fm_kv_cache": fb.KvCache, "fm_kv_args": fb.KvArgs,
               "fm_attn_args": fb.AttnArgs}
    lines = ['#include <stdio.h>', '#include "finch_hip.h"', "int main(void) {"]
    for name, cls in structs.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (name, name))
        for f, _ in cls._fields_:
            lines.append('printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (name, f, name, f))
    src, exe = tmp_path / "s.c", str(tmp_path / "s")
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe])
    got = dict(l.split() for l in subprocess.check_output([exe], text=True).splitlines())
    import ctypes as C
    for name, cls in structs.items():
        assert int(got[name]) == C.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got["%s.%s" % (name, f)]) == getattr(cls, f).offset, f
