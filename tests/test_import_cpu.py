"""The package imports where torch was built without CUDA: only calls need a GPU."""
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent

CODE = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)  # what a torch without CUDA does not have
import deepx_op_gpukernelcompiler_b200 as dx
from deepx_op_gpukernelcompiler_b200 import fusion, kvfunc, workflow
try:
    dx.int8_linear(torch.zeros(1, 16), (torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)))
except ValueError as e:
    print(e)
"""


def test_import_without_cuda():
    proc = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True,
                          timeout=300)
    assert proc.returncode == 0, proc.stderr[-2000:]
    assert "CUDA tensors only" in proc.stdout
