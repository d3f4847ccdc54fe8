"""The native forms of the calls over shared and selected pages (csrc/kq_torch.cpp): an output that cannot be allocated is a Python
exception, an argument that is not of the plain form is left to the Python method, and tensors of another device are refused."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# CUDA tensors of a fake mode have a device, sizes and strides; torch sees no GPU here, so that no output can be allocated.
CALLS = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from karume_b200 import _kqtorch as native
with FakeTensorMode():
    q = torch.empty(3, 4, 64, device="cuda")
    taken = torch.empty(3, 2, 5, device="cuda", dtype=torch.int32)
    each = torch.empty(3, device="cuda", dtype=torch.int32)
    out, places = torch.empty(3, 4, 64, device="cuda:1"), torch.empty(3, 2, 5, device="cuda:1", dtype=torch.int32)
    fewer, one_head, two, long = torch.empty(2, 4, 64, device="cuda"), taken[:, :1], each[:2], torch.empty(3, device="cuda", dtype=torch.int64)
batch, book = (3, 4096, 8, 8192, 0, 3), (4096, 3, 8, 8192, 12288, 40, 16, 16384)
raises = {
    "cache_attention_shared": (8, 1, 64, q, batch, 1, (1, 64, 128, 0), 1.0, 0, None, None, 0),
    "cache_attention_selected": (8, 1, 2, 64, q, batch, taken, 1.0, None, None, 0),
    "cache_select": (8, 1, 2, 64, (16, 32), q, batch, 5, 1, 1, None, None, 0),
    "pages_fork": (8, book, each, None, 0),
    "pages_compact": (8, book, 0),
}
for name, args in raises.items():
    try:
        getattr(native, name)(*args)
    except RuntimeError:
        print("raised", name)
left = {
    "cache_attention_shared": (8, 1, 64, fewer, batch, 1, (1, 64, 128, 0), 1.0, 0, None, None, 0),
    "cache_attention_selected": (8, 1, 2, 64, q, batch, one_head, 1.0, None, None, 0),
    "cache_summarize": (8, 1, (16,), batch),
    "cache_select": (8, 1, 2, 64, (16, 32), q, batch, 1 << 70, 1, 1, None, None, 0),
    "pages_grow": (8, book, two, 0),
    "pages_fork": (8, book, each, long, 0),
    "pages_copy": (8, book, taken, [], 0),
}
for name, args in left.items():
    print("left" if getattr(native, name)(*args) is None else "taken", name)
for name in raises:
    assert getattr(native, name)() is None
# another device than the context's
assert native.pages_grow(8, book, each, 1) is None and native.pages_fork(8, book, each, None, 1) is None
assert native.cache_attention_shared(8, 1, 64, q, batch, 1, (1, 64, 128, 0), 1.0, 0, None, None, 1) is None
assert native.cache_attention_selected(8, 1, 2, 64, q, batch, taken, 1.0, None, None, 1) is None
assert native.cache_select(8, 1, 2, 64, (16, 32), q, batch, 5, 1, 1, None, None, 1) is None
# ... for the output alone
assert native.cache_attention_shared(8, 1, 64, q, batch, 1, (1, 64, 128, 0), 1.0, 0, None, out, 0) is None
assert native.cache_attention_selected(8, 1, 2, 64, q, batch, taken, 1.0, None, out, 0) is None
assert native.cache_select(8, 1, 2, 64, (16, 32), q, batch, 5, 1, 1, None, places, 0) is None
"""


def test_native_calls_without_a_gpu():
    # in a process of its own: an exception that leaves through CPython ends it
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="", PYTHONPATH=ROOT)
    done = subprocess.run([sys.executable, "-c", CALLS], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, (done.returncode, done.stdout, done.stderr[-2000:])
    lines = done.stdout.split("\n")
    assert [x.split()[1] for x in lines if x.startswith("raised")] == ["cache_attention_shared", "cache_attention_selected", "cache_select", "pages_fork", "pages_compact"]
    assert [x.split()[0] for x in lines if x and not x.startswith("raised")] == ["left"] * 7


class OnDevice:
    def __init__(self, index):
        import torch
        self.device = torch.device("cuda", index)


def test_tensors_of_another_device_are_refused():
    from karume_b200.runtime import KqError, _on_device
    _on_device(1, a=OnDevice(1), b=OnDevice(1))
    with pytest.raises(KqError) as e:
        _on_device(0, a=OnDevice(0), b=OnDevice(1))
    assert e.value.status == "KQ_ERR_SHAPE" and "b is on cuda:1" in str(e.value)


def test_batches_and_angles_of_another_device_are_refused():
    from types import SimpleNamespace as Like
    from karume_b200.runtime import CacheSummaries, Gpu, KqError, SharedPrefixes
    gpu, here = object.__new__(Gpu), Like(index=0)
    gpu.index = 0
    cache, summaries, shared = Like(head_dim=64, kv_heads=2, handle=1), object.__new__(CacheSummaries), object.__new__(SharedPrefixes)
    summaries.check = lambda cache, index: None
    elsewhere, mixed, angles = Like(index=1), Like(index=-1), Like(index=1, table=OnDevice(1), args=None)
    for batch, rope, says in ((elsewhere, None, "cuda:1"), (mixed, None, "several devices"), (here, angles, "table is on cuda:1")):
        calls = [lambda: gpu.cache_attention(cache, None, batch, rope=rope, shared=shared), lambda: gpu.cache_attention(cache, None, batch, rope=rope, selected=0),
                 lambda: gpu.cache_select(cache, summaries, None, batch, 4, rope=rope)]
        if rope is None:
            calls.append(lambda: gpu.cache_summarize(cache, summaries, batch))
        for call in calls:
            with pytest.raises(KqError) as e:
                call()
            assert e.value.status == "KQ_ERR_SHAPE" and says in str(e.value)
