"""The library's Makefile rebuilds what it has to (CPU; on a copy of the file with empty sources, nothing is compiled)."""
import os
import re
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _copy(tmp_path):
    src = os.path.join(ROOT, "bournemouth-forced-aligner_amd", "csrc")
    csrc = tmp_path / "package" / "csrc"
    csrc.mkdir(parents=True)
    shutil.copy(os.path.join(src, "Makefile"), csrc)
    text = (csrc / "Makefile").read_text()
    names = re.findall(r"[\w./]+\.(?:hip|cpp|hpp|inc|h|map)\b", text)
    for name in names:
        f = csrc / name
        f.parent.mkdir(parents=True, exist_ok=True)
        f.touch()
    return csrc, set(os.listdir(src))


def _make(csrc, *args):
    return subprocess.run(["make", "-C", str(csrc), *args], capture_output=True, text=True)


def test_a_change_of_the_flags_rebuilds_everything(tmp_path):
    csrc, _ = _copy(tmp_path)
    assert _make(csrc, "-t").returncode == 0  # everything counts as built
    assert _make(csrc, "-q").returncode == 0
    plan = _make(csrc, "-n", "ARCH=gfx942").stdout
    for name in ("bfa_norm.hip", "bfa_backtrace.hip", "bfa_capi.cpp"):
        assert f"-c {name}" in plan


def test_every_header_is_a_prerequisite(tmp_path):
    csrc, there = _copy(tmp_path)
    text = (csrc / "Makefile").read_text()
    for name in sorted(there):
        if name.endswith((".inc", ".hpp")):
            assert re.search(rf"\b{re.escape(name)}\b", text), f"{name} is not a prerequisite of any object"
