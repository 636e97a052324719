"""The tests of the microscaled rows on the CPU, through the kernel sources (tests/hip_emu): all but the large products -- refusals, empty
sides and rows behind the last one run here before they run on a GPU."""
import os
import shutil

import pytest

from tests.test_emu_gpu_subset import CLANG, _run


@pytest.mark.skipif(not os.path.exists(CLANG) or not shutil.which("make"), reason="no ROCm clang++ / make")
def test_mx_rows_on_the_emulated_kernels():
    _run(["tests/test_gpu_mx.py"], "not big", 250)
