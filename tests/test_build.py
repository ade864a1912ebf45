"""What make would do, asked without doing it: objects are older than the flags they were compiled with once the Makefile changes."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "semantic-segmentation_amd", "csrc")


def compiled(*options):
    plan = subprocess.run(["make", "-n", "-C", CSRC, *options], capture_output=True, text=True, check=True).stdout
    return set(re.findall(r"-c (\w+\.hip)", plan))


def test_a_changed_makefile_compiles_every_source_again():
    sources = {f for f in os.listdir(CSRC) if f.endswith(".hip")}
    assert compiled("-B") == sources
    assert compiled("-W", "Makefile") == sources


def test_build_compiles_every_time(monkeypatch):
    import __graft_entry__ as entry
    commands = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, **kw: commands.append(cmd))
    entry.build()
    assert commands and all("-B" in c for c in commands if c[0] == "make")
