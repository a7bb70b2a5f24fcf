"""The example's training loop, block, clip and step together: the loss falls with every optimizer (by a quarter with
AdamW's), and the 8-bit moments train as the fp32 ones do."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def _train(**kw):
    spec = importlib.util.spec_from_file_location("train_gated_ffn", os.path.join(HERE, "..", "examples", "train_gated_ffn.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod.train(log=lambda line: None, **kw)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_the_loss_falls(dtype):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    last = {}
    for name in ("adamw", "adamw8bit", "came8bit"):
        losses = _train(steps=101, name=name, dtype=dtype)
        last[name] = losses[-1]
        assert losses[-1] < (0.75 if name != "came8bit" else 1.0) * losses[0], (name, losses)
    assert abs(last["adamw8bit"] / last["adamw"] - 1) < 0.05, last
