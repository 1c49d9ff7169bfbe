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


def test_workspace_depends_on_what_the_header_names():
    """Each of the six sizes alone changes the workspace; the element type, the slots and their order do not."""
    for sizes in (dict(rows=256, prefix_length=700, capacity=24), dict(rows=2, capacity=20000),
                  dict(rows=2, prefix_length=9000, capacity=500)):
        n = workspace(**sizes)
        assert n > 0
        for other in (dict(type=native.TYPE_BF16), dict(type=native.TYPE_F16), dict(slot_count=77), dict(scale=0.5),
                      dict(slots=P, counts=P, lse=P), dict(q_stride=4096, out_stride=512)):
            assert workspace(**{**sizes, **other}) == n, other
    base = dict(rows=256, prefix_length=700, capacity=24)
    for other in (dict(rows=255), dict(heads=16), dict(head_dim=128), dict(prefix_length=8000)):
        assert workspace(**{**base, **other}) != workspace(**base), other
    assert len({workspace(rows=2, capacity=20000), workspace(rows=2, capacity=2000),
                workspace(rows=2, capacity=20000, kv_heads=1)}) == 3


P = 1 << 20  # an aligned address that nothing reads


@pytest.mark.parametrize("name", ["q", "k", "v"])
@pytest.mark.parametrize("more", [64, -64])
def test_rope_append_in_place_needs_one_row_stride(name, more):
    """A token's output over another token's input: refused, in the order of the tokens or against it."""
    a = native.RopeAppend()
    for n in ("positions", "slots", "entries", "key_codes", "key_scales", "value_codes", "value_scales"):
        setattr(a, n, P)
    for i, n in enumerate(("q", "k", "v")):  # views of one fused buffer, written in place
        setattr(a, n, P + i * 2048)
        setattr(a, n + "_out", P + i * 2048)
        setattr(a, n + "_stride", 2048)
        setattr(a, n + "_out_stride", 2048)
    a.magnitude = 1.0
    a.tokens, a.heads, a.kv_heads, a.head_dim, a.rotary_dim, a.slot_count, a.capacity = 2, 8, 4, 64, 64, 1, 4
    setattr(a, name + "_out_stride", 2048 + more)
    ones = (C.c_double * 32)(*[1.0] * 32)
    with pytest.raises(native.NeedleError, match="same row stride"):
        native.check(native.lib().needle_cuda_rope_append_dev(C.byref(a), ones, None))
