"""What the Makefile builds again."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rotorquant-vllm_amd", "csrc")


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_another_torch_builds_its_module_again(tmp_path):
    """A Python that says what the Makefile asks it for, first of one torch and then of another."""
    python, target, build = tmp_path / "python", str(tmp_path / "build" / "rq_torch.o"), tmp_path / "build"

    def python_has(torch):
        python.write_text(f"#!/bin/sh\necho /a/torch /a/include 1 {torch} 3.10.12\n")
        python.chmod(0o755)

    def up_to_date():
        run = subprocess.run(["make", "-q", "-C", CSRC, f"BUILD={build}", f"PYTHON={python}", target], capture_output=True, text=True)
        assert run.returncode in (0, 1), run.stderr
        return run.returncode == 0

    build.mkdir()
    python_has("2.10.0")
    assert not up_to_date()
    open(target, "w").close()
    assert up_to_date() and up_to_date()
    python_has("2.11.0")
    assert not up_to_date()
    open(target, "w").close()
    assert up_to_date()
