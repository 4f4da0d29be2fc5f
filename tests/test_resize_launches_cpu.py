"""Resizing is one launch while its warps suffice for the sequences and little can be copied, else two (on the CPU, against a stand-in for the
runtime's launches)."""
import os
import subprocess
import sys

import pytest
from test_more_launches_cpu import CALLS
from test_serving_launches_cpu import LIBRARY, stand_in  # noqa: F401


@pytest.mark.parametrize("page,batch,launches", [("1, 16, 64", 1, 1), ("1, 16, 64", 256, 1), ("1, 16, 64", 257, 2), ("1, 16, 64", 4096, 2),
                                                 ("2, 128, 128", 128, 1), ("2, 128, 128", 129, 2)])
def test_launches_of_a_resize(stand_in, page, batch, launches):  # noqa: F811
    program = CALLS.replace("8, 2, 128, 128, 5", f"8, {page}, 5")
    run = subprocess.run([sys.executable, "-c", program, str(LIBRARY), f"resize{batch}"], env={**os.environ, "LD_PRELOAD": str(stand_in), "FAILING_LAUNCH": "-1"},
                         capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stderr
    assert run.stdout.split()[:2] == ["0", str(launches)], run.stdout
