"""What a change to the build makes stale (make -n: nothing is compiled here)."""
import glob
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lamellar-runtime_amd", "csrc")


@pytest.mark.parametrize("changed,only", [("Makefile", None), ("lmr_internal.hpp", None), ("lmr_rows.hpp", ["lmr_rows.hip"]),
                                          ("lmr_scan.hip", ["lmr_scan.hip"])])
def test_what_is_compiled_again(tmp_path, changed, only):
    """A changed file makes the objects that depend on it stale; the Makefile, which holds the flags, all of them."""
    if shutil.which("make") is None:
        pytest.skip("no make")
    sources = sorted(os.path.basename(p) for p in glob.glob(os.path.join(CSRC, "*.hip")))
    built, out = tmp_path / "objects", tmp_path / "lib.so"
    built.mkdir()
    for s in sources:                                    # stand for a finished build: newer than every source
        (built / (s[:-4] + ".o")).touch()
    out.touch()
    make = ["make", "-n", "-C", CSRC, f"BUILD={built}", f"OUT={out}"]
    assert "-c " not in subprocess.run(make, capture_output=True, text=True, check=True).stdout
    said = subprocess.run(make + ["-W", changed], capture_output=True, text=True, check=True).stdout
    again = sorted(line.split(" -c ")[1].split()[0] for line in said.splitlines() if " -c " in line)
    assert again == (sources if only is None else only)
    assert "-shared" in said
