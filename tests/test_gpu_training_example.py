"""The example of a block in training runs, and its gradients are plain torch's."""
import importlib.util

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_example_runs_with_the_gradients_of_plain_torch(cuda_device):
    before = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        spec = importlib.util.spec_from_file_location("moe_training_example", ROOT / "examples" / "moe_training.py")
        example = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(example)
        difference = example.main(["--tokens", "300", "--hidden", "64", "--experts", "6", "--top-k", "2", "--vocabulary", "200",
                                   "--steps", "2"])
    finally:
        torch.backends.cuda.matmul.allow_tf32 = before
    # both sides in fp32: eight steps there and back on each, within 2^-17 of their results' norm (sums of at most
    # 300 products: 300 u = 2^-15.8 at worst), whose errors pass through factors of about one
    assert set(difference) == {"table", "weight", "bias", "router", "experts"}
    assert max(difference.values()) <= 2.0 ** -11
