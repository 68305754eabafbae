"""CPU tests of demo/model.py."""

import os
import pathlib
import subprocess
import sys


DEMO = pathlib.Path(__file__).resolve().parent.parent / "demo"

PLAIN = """
import importlib.util, torch, model
assert importlib.util.find_spec("flash_attention_amd") is None
net = model.TinyGPT(vocab=8, block=8, n_layer=1, n_head=2, n_embd=8)
assert net(torch.zeros(2, 5, dtype=torch.long)).shape == (2, 5, 8)
try:
    model.TinyGPT(vocab=8, block=8, n_layer=1, n_head=2, n_embd=16, rotary=True)
except ModuleNotFoundError as e:
    assert "flash_attention_amd" in str(e)
else:
    raise AssertionError("rotary=True without the package")
"""


def test_the_plain_model_needs_torch_alone():
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    res = subprocess.run([sys.executable, "-c", PLAIN], cwd=DEMO, env=env, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
