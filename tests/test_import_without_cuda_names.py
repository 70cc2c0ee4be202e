"""The package imports on a torch build without CUDA, whose _C has none of the names of the CUDA runtime."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_import():
    program = ("import torch\n"
               "for name in [n for n in vars(torch._C) if n.startswith('_cuda_get')]:\n"
               "    delattr(torch._C, name)\n"
               "import fufft_b200\n"
               "from fufft_b200 import ops\n"
               "import fufft_b200.torch_ops\n")
    r = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
