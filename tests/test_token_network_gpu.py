"""The operators together, as examples/patch_tokens.py uses them."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "patch_tokens.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("patch_tokens", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_trains_and_generates(example, dtype):
    losses, off = example.main(["--steps", "40", "--clouds", "4", "--dtype", dtype])
    assert losses[-1] < 0.5 * losses[0]
    # both passes are fp32: some thousand rounded operations deep
    assert off < 1e-4


def test_inference_mode_and_eval(example):
    tokens, _, lengths, offsets = example.pack(example.make_clouds(3, seed=1))
    net = example.PatchNet().cuda()
    with torch.inference_mode():
        a = net(tokens, offsets)
    assert torch.equal(a, net(tokens, offsets).detach())
