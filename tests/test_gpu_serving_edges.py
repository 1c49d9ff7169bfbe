"""The serving operators on the GPU where values, not sizes, are at the edge: queries that are not finite, scores
that overflow, value scales far apart, logits far from zero, quotients on the border between two codes.  Against
definitions in binary64.

Tolerances.  u = 2^-24 (half a binary32 step), h = half a step of the element type (2^-24, 2^-11, 2^-8).
"""
import math

import pytest

from test_gpu_serving_ops import TYPES, attention_call, dtype_of, random_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import needle_b200.build
    needle_b200.build.build()
    return torch


# ------------------------------------------------------------------ prefix_attention

def attend(torch, name, q, prefix, own, counts, heads, kv_heads, dim, prefix_length):
    """(out [rows, heads, dim], lse [rows, heads]) on the CPU."""
    rows = q.shape[0]
    out = torch.full((rows, heads * dim), 3.0, dtype=dtype_of(torch, name)).cuda()
    lse = torch.full((rows, heads), 4.0).cuda()
    attention_call(torch, name, q.cuda(), out, lse, [t.cuda() for t in prefix], [t.cuda() for t in own], None,
                   torch.tensor(counts, dtype=torch.int32).cuda(), heads, kv_heads, dim, prefix_length)
    torch.cuda.synchronize()
    return out.cpu().view(rows, heads, dim), lse.cpu()


def caches(torch, g, rows, kv_heads, dim, prefix_length, capacity):
    prefix = [*random_cache(torch, g, kv_heads, prefix_length, dim), *random_cache(torch, g, kv_heads, prefix_length, dim)]
    own = [*random_cache(torch, g, rows, kv_heads, capacity, dim), *random_cache(torch, g, rows, kv_heads, capacity, dim)]
    return prefix, own


# rows, heads, kv_heads, dim, prefix, capacity: one part; splits; the prefix as a dense product, beside rows that have
# nothing of their own; both
PLANS = [(5, 8, 4, 64, 37, 20), (2, 8, 4, 64, 5, 5000), (1, 4, 1, 128, 0, 3001), (170, 8, 4, 64, 210, 16),
         (40, 32, 4, 128, 500, 24), (2, 32, 1, 64, 2048, 4000)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,heads,kv_heads,dim,prefix_length,capacity", PLANS)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_queries_that_are_not_finite_give_nan(torch, name, rows, heads, kv_heads, dim, prefix_length, capacity, bad):
    """A query with a NaN or an infinity (its scores are NaN, or infinities of both signs) has no softmax: NaN, and not the
    zeros of a row with nothing to attend to, however the call is split.  The other heads and rows are as without it."""
    g = torch.Generator().manual_seed(rows + dim)
    prefix, own = caches(torch, g, rows, kv_heads, dim, prefix_length, capacity)
    counts = [(capacity - (7 * r) % (capacity + 1)) for r in range(rows)]
    if prefix_length:
        counts[-1] = 0
    q = torch.randn(rows, heads * dim, generator=g).to(dtype_of(torch, name))
    want, want_lse = attend(torch, name, q, prefix, own, counts, heads, kv_heads, dim, prefix_length)
    assert bool(want.isfinite().all()) and bool(want_lse.isfinite().all())
    hit = {(r, (5 * r + 1) % heads) for r in {0, rows // 2, rows - 1}}
    for r, h in hit:
        q[r, h * dim + 11] = bad
    got, lse = attend(torch, name, q, prefix, own, counts, heads, kv_heads, dim, prefix_length)
    for r, h in hit:
        assert bool(got[r, h].isnan().all()) and math.isnan(float(lse[r, h])), (r, h, got[r, h, :4], lse[r, h])
        want[r, h], want_lse[r, h] = 0.0, 0.0
        got[r, h], lse[r, h] = 0.0, 0.0
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
