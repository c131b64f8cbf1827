"""Block operators without a GPU: what the package needs of torch, and calls that are refused before a launch."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_package_imports_without_cuda_in_torch():
    """A torch built without CUDA has no ``_cuda_getCurrentRawStream``: registries and oracles load there all the same,
    and the stream comes from the public call."""
    code = """
import torch
del torch._C._cuda_getCurrentRawStream
import segment_anything_fast_b200
from segment_anything_fast_b200 import ops
class Stream:
    cuda_stream = 77
torch.cuda.current_device = lambda: 1
torch.cuda.current_stream = lambda dev: Stream if dev == 1 else None
assert ops._stream() == 77
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
