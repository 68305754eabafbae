"""CPU tests of demo/model.py."""

import os
import pathlib
import subprocess
import sys

import torch


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


def test_a_rotation_table_made_in_an_evaluation_serves_training(monkeypatch):
    monkeypatch.syspath_prepend(str(DEMO))
    import model

    net = model.TinyGPT(vocab=8, block=8, n_layer=1, n_head=2, n_embd=32, rotary=True)
    with torch.inference_mode():
        table = net.table(torch.device("cpu"))
    assert not table.is_inference() and net.table(torch.device("cpu")) is table
    x = torch.ones(8, 16, requires_grad=True)
    (x * table).sum().backward()                # (saved for the backward, as qk_norm_rope saves it)
    assert torch.equal(x.grad, table)
