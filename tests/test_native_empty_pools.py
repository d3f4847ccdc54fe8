"""Copies into pools without pages: the native form leaves them to the Python method, which refuses them."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# (a fake mode's CUDA tensors have a device, sizes and strides)
CALL = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from karume_b200 import _kqtorch as native
with FakeTensorMode():
    pairs = torch.empty(3, 2, device="cuda", dtype=torch.int32)
    pools = [torch.empty(*shape, device="cuda") for shape in ((0, 4), (0,), (0, 0, 7))]
for pages in (0, 5):
    book = (4096, 3, 8, 8192, 12288, pages, 16, 16384)
    for pool in pools:
        assert native.pages_copy(8, book, pairs, [pool], 0) is None
print("left")
"""


def test_pools_without_pages():
    # in a process of its own: what goes wrong here ends it
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="", PYTHONPATH=ROOT)
    done = subprocess.run([sys.executable, "-c", CALL], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "left", (done.returncode, done.stderr[-2000:])
