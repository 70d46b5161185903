"""The example of the int8 expert path: the int8 layer stays near the unquantised one, the training loss falls."""
import importlib.util

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_example_serves_and_trains(cuda_device):
    spec = importlib.util.spec_from_file_location("w8a8_moe_example", ROOT / "examples" / "w8a8_moe.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    error, (first, last) = example.main(["--tokens", "96", "--hidden", "256", "--inter", "128", "--experts", "8",
                                         "--top-k", "2", "--steps", "8"])
    # 8-bit codes of rows and weights: a step of 1/127 of the largest of 256 values (about 3.5 standard
    # deviations) is 0.028 of one, its rounding error 0.028 / sqrt(12) = 0.8 % for each of two operands in
    # each of two products: about 2 % in all
    assert error < 0.04
    assert last < first
