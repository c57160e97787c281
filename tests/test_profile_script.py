"""tools/profile_bench.sh against a stand-in profiler (no GPU needed): a pass that fails, or that runs out of time, is the last one."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("fake,passes", [("exit 3", 1), ("sleep 30", 1), ('case "$*" in *FETCH*) exit 139;; esac', 4)])
def test_a_failing_pass_ends_the_script(tmp_path, fake, passes):
    (tmp_path / "tools").mkdir()
    (tmp_path / "profiles").mkdir()
    (tmp_path / "bin").mkdir()
    shutil.copy(os.path.join(ROOT, "tools", "profile_bench.sh"), tmp_path / "tools")
    shutil.copy(os.path.join(ROOT, "profiles", "summarize_rocprof.py"), tmp_path / "profiles")
    calls = tmp_path / "calls"
    prof = tmp_path / "bin" / "rocprofv3"
    # (a pass that succeeds leaves its result folder, without a database to summarise)
    prof.write_text('#!/bin/bash\necho "$*" >> "%s"\n%s\nwhile [ "$1" != -d ]; do shift; done; mkdir -p "$2"\n' % (calls, fake))
    prof.chmod(0o755)
    env = dict(os.environ, PATH="%s:%s" % (tmp_path / "bin", os.environ["PATH"]), PASS_LIMIT="1")
    r = subprocess.run(["bash", str(tmp_path / "tools" / "profile_bench.sh"), "t_fake"], env=env, capture_output=True, text=True, timeout=60)
    assert r.returncode != 0
    assert len(calls.read_text().splitlines()) == passes, calls.read_text()
