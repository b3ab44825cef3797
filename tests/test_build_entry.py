"""build() answers "does it build?": it compiles the whole library whenever it is called, also where a built one is there."""
import os
import re
import subprocess

import __graft_entry__ as entry

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join("nanocall_amd", "csrc")


def test_build_compiles_every_object_where_a_built_library_is_there(monkeypatch):
    called = []
    monkeypatch.setattr(entry, "_run", lambda cmd, **kw: called.append(cmd))
    entry.build()
    make = next(c for c in called if CSRC in c)
    # what that command would run, on a tree whose objects are all up to date
    p = subprocess.run(make + ["-n"], cwd=ROOT, check=True, capture_output=True, text=True)
    objs = re.search(r"^OBJS\s*=\s*(.*)$", open(os.path.join(ROOT, CSRC, "Makefile")).read(), re.M).group(1).split()
    assert set(objs) <= set(re.findall(r"-o (\w+\.o)\b", p.stdout))
    assert "-o ../libnanocall_hip.so" in p.stdout and "-o ../bin/nanocall" in p.stdout
