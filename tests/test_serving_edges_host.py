"""The serving operators' host side at the edges of what they allow.  No GPU needed: the workspace's size is
computed, and every refusal comes, before the first CUDA call."""
import ctypes as C
import os
import subprocess
import sys

import pytest

from needle_b200 import native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module", autouse=True)
def built():
    import needle_b200.build as b
    return b.build()


def attention_args(**kw):
    a = native.PrefixAttention()
    a.rows, a.heads, a.kv_heads, a.head_dim = 2, 8, 4, 64
    a.slot_count = 2
    for n, v in kw.items():
        setattr(a, n, v)
    a.prefix_capacity = a.prefix_length
    return a


def workspace(**kw):
    n = C.c_size_t(12345)
    native.check(native.lib().needle_cuda_prefix_attention_workspace(C.byref(attention_args(**kw)), C.byref(n)))
    return n.value


def test_workspace_of_an_empty_batch_is_empty():
    """Sizes of every kind, an empty batch and empty caches among them, in a process of its own: a size that is
    divided by would end it."""
    code = """
import itertools, sys
sys.path[:0] = sys.argv[1:]
import __graft_entry__ as entry
entry.load()
import test_serving_edges_host as t
sizes = (0, 1, 16, 31, 100, 160, 256, 4097, 1 << 20)
for rows, prefix, capacity in itertools.product((0, 1, 33, 4096), sizes, sizes):
    for heads, kv_heads, dim in ((8, 4, 64), (1, 1, 128), (40, 2, 64), (4096, 1, 128)):
        n = t.workspace(rows=rows, heads=heads, kv_heads=kv_heads, head_dim=dim, prefix_length=prefix, capacity=capacity)
        assert n % 16 == 0 and (n == 0 or rows > 0), (rows, heads, kv_heads, dim, prefix, capacity, n)
print("sized")
"""
    done = subprocess.run([sys.executable, "-c", code, ROOT, os.path.dirname(os.path.abspath(__file__))],
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "sized" in done.stdout, (done.returncode, done.stderr[-2000:])
