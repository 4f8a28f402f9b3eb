"""CPU-only: what the build compiles again."""
import glob
import os
import subprocess

import __graft_entry__ as entry
from conftest import ROOT

CSRC = os.path.join(ROOT, "diga_amd", "csrc")


def planned(*changed):
    """The commands make would run if these files had just changed."""
    args = [a for name in changed for a in ("-W", name)]
    return subprocess.run(["make", "-n", "-C", CSRC, *args], check=True, capture_output=True, text=True).stdout


def test_a_changed_flag_compiles_everything_again():
    out = planned("Makefile")
    for src in glob.glob(os.path.join(CSRC, "*.hip")):
        assert f"-c {os.path.basename(src)} " in out, src
    assert "-o libdiga_hip.so" in out and "-o ../_calls.so" in out


def test_the_python_side_follows_torch():
    assert "-o ../_calls.so" in planned("torch.stamp")
    import torch
    stamp, make = os.path.join(CSRC, "torch.stamp"), lambda: subprocess.run(["make", "-C", CSRC, "torch.stamp"], check=True, capture_output=True)
    make()
    with open(stamp) as f:
        assert f.read().strip() == torch.__version__
    before = os.stat(stamp).st_mtime_ns
    make()                                    # the same version: left alone
    assert os.stat(stamp).st_mtime_ns == before


def test_build_compiles_whatever_is_there(monkeypatch):
    ran = []
    monkeypatch.setattr(entry.subprocess, "check_call", lambda cmd, **k: ran.append(cmd))
    entry.build()
    assert len(ran) == 1 and ran[0][0] == "make" and "-B" in ran[0]
