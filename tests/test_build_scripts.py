"""The scripts that build the library's sources aside (A/B libraries, the projection bench) compile what the library is made of, as
the library is compiled.  The compiler driver is a stand-in that writes down its arguments."""
import importlib.util
import os
import shutil
import subprocess

from conftest import ROOT

spec = importlib.util.spec_from_file_location("mw_build", os.path.join(ROOT, "manual-whisper_amd", "build.py"))
build = importlib.util.module_from_spec(spec)
spec.loader.exec_module(build)


def _run(tmp_path, script, *args):
    root = tmp_path / "tree"                                  # the scripts write beside themselves
    os.makedirs(root / "tools")
    os.makedirs(root / "manual-whisper_amd" / "csrc")
    shutil.copy(os.path.join(ROOT, "manual-whisper_amd", "build.py"), root / "manual-whisper_amd")
    shutil.copy(os.path.join(ROOT, "tools", script), root / "tools")
    fake = tmp_path / "hipcc"
    fake.write_text(f'#!/bin/bash\necho "$@" >> {tmp_path}/calls\nwhile [ "$1" != -o ]; do shift; done\ntouch "$2"\n')
    fake.chmod(0o755)
    subprocess.run(["bash", str(root / "tools" / script), *args], check=True, env=dict(os.environ, HIPCC=str(fake)), timeout=60)
    return [line.split() for line in (tmp_path / "calls").read_text().splitlines()], root


def _has(call, flags):
    return any(call[i:i + len(flags)] == list(flags) for i in range(len(call)))


def test_a_variant_holds_all_sources_under_the_librarys_flags(tmp_path):
    calls, root = _run(tmp_path, "build_variant.sh", "x", "-DSOMETHING=1")
    compiled = {call[call.index("-c") + 1]: call for call in calls if "-c" in call}
    assert set(compiled) == set(build.SOURCES)
    for src, call in compiled.items():
        assert _has(call, build.FLAGS) and "-DSOMETHING=1" in call and all(f in call for f in build.EXTRA_FLAGS.get(src, []))
    link = calls[-1]
    assert "-shared" in link and {os.path.basename(a) for a in link if a.endswith(".o")} == {s.replace(".hip", ".o") for s in build.SOURCES}
    assert (root / "tools" / "ab" / "x" / "libmwhip.so").exists()


def test_the_projection_bench_has_the_device_flags(tmp_path):
    calls, _ = _run(tmp_path, "build_gemv_bench.sh", "-DSOMETHING=1")
    assert len(calls) == 1 and _has(calls[0], build.ARCH_FLAGS) and "-DSOMETHING=1" in calls[0]
