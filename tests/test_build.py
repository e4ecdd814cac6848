"""magicpig_amd/build.py on a tree of its own with a stand-in compiler: what is compiled again after what change (CPU)."""
import importlib.util
import os
import shutil

import pytest

from magicpig_amd import build as B


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A copy of build.py over empty sources, and a compiler that writes down its command and touches its output."""
    pkg = tmp_path / "pkg"
    (pkg / "csrc").mkdir(parents=True)
    (tmp_path / "include").mkdir()
    (tmp_path / "bin").mkdir()
    for f in [pkg / "csrc" / s for s in B.SOURCES] + [pkg / "csrc" / "common.h", tmp_path / "include" / "magicpig_hip.h"]:
        f.write_text("")
    shutil.copyfile(B.__file__, pkg / "build.py")
    log = tmp_path / "log"
    hipcc = tmp_path / "bin" / "hipcc"
    hipcc.write_text('#!/bin/sh\necho "$@" >> %s\nwhile [ "$1" != -o ]; do shift; done\n: > "$2"\n' % log)
    hipcc.chmod(0o755)
    monkeypatch.setenv("PATH", f"{tmp_path / 'bin'}{os.pathsep}{os.environ['PATH']}")
    old = 1.0e9                                            # everything that is there lies in the past
    for root, _, files in os.walk(tmp_path):
        for f in files:
            os.utime(os.path.join(root, f), (old, old))
    spec = importlib.util.spec_from_file_location("build_copy", pkg / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)

    def run(**kw):
        log.write_text("")
        mod.build(**kw)
        lines = log.read_text().splitlines()
        return sorted(os.path.basename(w) for line in lines if " -c " in line for w in line.split() if w.endswith(".hip")), lines
    return pkg, run


def test_what_is_compiled_again(tree):
    pkg, run = tree
    everything = sorted(B.SOURCES)
    made, lines = run()
    assert made == everything
    for line in lines[:-1]:
        assert all(flag in line.split() for flag in B.FLAGS)
    assert run() == ([], [])                               # nothing changed
    now = os.path.getmtime(pkg / "lib" / "libmagicpig_hip.so") + 10
    for path, want in ((pkg / "csrc" / "prompt.hip", ["prompt.hip"]), (pkg / "csrc" / "common.h", everything),
                       (pkg.parent / "include" / "magicpig_hip.h", everything), (pkg / "build.py", everything)):
        os.utime(path, (now, now))
        made, lines = run()
        assert made == want and "-shared" in lines[-1], path
        os.utime(path, (1.0e9, 1.0e9))
    assert run(force=True)[0] == everything
