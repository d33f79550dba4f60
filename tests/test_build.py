"""CPU-only checks of the build: one set of compiler flags, which every object depends on."""
import glob
import os
import subprocess

from conftest import ROOT

CSRC = os.path.join(ROOT, "stable-diffusion_amd", "csrc")
NO_PACKED_F32 = "-Xclang -target-feature -Xclang -packed-fp32-ops"


def compiled(out):
    """{source: its command} of make's output."""
    return {os.path.basename(w): line for line in out.splitlines() if " -c " in line for w in line.split() if w.endswith(".hip")}


def test_a_change_of_the_flags_builds_everything_again():
    out = subprocess.run(["make", "-n", "-C", CSRC, "-W", "Makefile"], capture_output=True, text=True, check=True).stdout
    lines = compiled(out)
    assert set(lines) == {os.path.basename(f) for f in glob.glob(os.path.join(CSRC, "*.hip"))}
    assert all(NO_PACKED_F32 in line for line in lines.values())


def test_the_timing_build_has_the_flags_of_the_library(tmp_path):
    """The experiment's library differs from the shipped one by its define alone."""
    out = subprocess.run(["bash", os.path.join(ROOT, "experiments", "build_pp_timing.sh"), str(tmp_path)], capture_output=True, text=True,
                         env=dict(os.environ, MAKEFLAGS="n")).stdout
    ours = compiled(subprocess.run(["make", "-n", "-B", "-C", CSRC], capture_output=True, text=True, check=True).stdout)
    theirs = compiled(out)
    assert set(theirs) == set(ours)
    for source, line in theirs.items():
        assert line.replace(" -DSDAMD_PP_TIMING", "").replace(CSRC + "/", "").split() == ours[source].split()


def test_the_build_hook_compiles_what_is_already_built():
    text = open(os.path.join(ROOT, "__graft_entry__.py")).read()
    assert '"make", "-B"' in text
