"""The tests of the microscaled rows on the CPU, through the kernel sources (tests/hip_emu): all but the large products -- refusals, empty
sides and rows behind the last one run here before they run on a GPU."""
import os
import shutil

import pytest

from tests.test_emu_gpu_subset import CLANG, _run


@pytest.mark.skipif(not os.path.exists(CLANG) or not shutil.which("make"), reason="no ROCm clang++ / make")
def test_mx_rows_on_the_emulated_kernels():
    _run(["tests/test_gpu_mx.py"], "not big", 250)


@pytest.mark.skipif(not os.path.exists(CLANG) or not shutil.which("make"), reason="no ROCm clang++ / make")
def test_large_tiles_on_a_chip_of_one_cu(monkeypatch):
    """which form of the product runs goes by the number of CUs: with one, sizes that the emulation can take select the 256 x 256 tiles in two
    phases and the 128 x 128 ones"""
    monkeypatch.setenv("HIPEMU_CUS", "1")
    _run(["tests/test_gpu_mx.py::test_product_large_tiles"], "256-200 or 256-300 or 128-100", 36)
