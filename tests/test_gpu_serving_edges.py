"""The serving operators on the GPU where values, not sizes, are at the edge: queries that are not finite, scores
that overflow, value scales far apart, logits far from zero, quotients on the border between two codes.  Against
definitions in binary64.

Tolerances.  u = 2^-24 (half a binary32 step), h = half a step of the element type (2^-24, 2^-11, 2^-8).
"""
import ctypes as C
import math

import numpy as np
import pytest

from test_gpu_serving_ops import (HALF, TYPES, U, attention_call, attention_reference, dtype_of, random_cache, rope_call,
                                  rules_args, stream_of, to_numpy)

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


def exactly(torch, q, prefix, own, slot, count, heads, kv_heads, dim):
    """One row in binary64: out and lse, the largest sum |q k| scale, sum w |v| (as out), the largest |v| that codes of 127
    would have."""
    sides = [(prefix, slice(None), slice(None)), (own, slot, slice(0, count))]
    k, v = (torch.cat([c[i][at][:, n].double() * c[i + 1][at][:, n, None].double() for c, at, n in sides], 1) for i in (0, 2))
    q = q.double().view(kv_heads, heads // kv_heads, dim)
    s = torch.einsum("kgd,kpd->kgp", q, k) * dim ** -0.5
    big = float((torch.einsum("kgd,kpd->kgp", q.abs(), k.abs()) * dim ** -0.5).max())
    w = torch.softmax(s, -1)
    out, size = (torch.einsum("kgp,kpd->kgd", w, x).reshape(heads, dim) for x in (v, v.abs()))
    vmax = 127 * max(float(prefix[3].max()), float(own[3][slot, :, :count].max()) if count else 0.0)
    return out, torch.logsumexp(s, -1).reshape(heads), big, size, vmax


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


# One position with the whole weight and a score beyond 2^24: the reference maximum, a binary32 number of that size, has
# steps of 2 and more and rounds the exponent of the value scales away that it should cover.  The weight is then not
# some 2^6 but the value scale itself, and its fp16 tail ends at 2^-24: half of that for each of at most 127 steps.
WHOLE_WEIGHT = 127 * 2.0 ** -25


def test_scores_below_the_range_of_binary32_have_no_weight(torch):
    """Prefix scores that overflow to -inf leave the row's own positions, in the dense product and in the stream.
    Tolerance: WHOLE_WEIGHT."""
    for rows in (3, 170):
        g = torch.Generator().manual_seed(rows)
        heads, kv_heads, dim, prefix_length, capacity = 8, 4, 64, 210, 16
        prefix, own = caches(torch, g, rows, kv_heads, dim, prefix_length, capacity)
        q = torch.zeros(rows, heads * dim)
        q[:, ::dim] = 1e30
        prefix[0][..., 0] = torch.randint(-127, -1, (kv_heads, prefix_length), generator=g).to(torch.int8)
        prefix[1][:] = 1e10  # scores of -1e40
        counts = [1 + (5 * r) % capacity for r in range(rows)]
        out, lse = attend(torch, "f32", q, prefix, own, counts, heads, kv_heads, dim, prefix_length)
        for r in range(rows):
            want, want_lse, _, vmax = attention_reference(torch, q[r], prefix, own, r, counts[r], heads, kv_heads, dim, 0, 0.125)
            # neighbouring scores are 1e26 apart and more: one position takes it all
            assert bool((out[r].double() - want).abs().le(4 * U * vmax + WHOLE_WEIGHT).all()), r
            assert bool((lse[r].double() - want_lse).abs().le(16 * U * want_lse.abs()).all()), r


@pytest.mark.parametrize("size", [1e5, 1e7, 3e9, 1e12, 1e30])
def test_scores_of_any_size_choose_their_largest(torch, size):
    """Scores of one product each, five roundings off at most, the largest 5% above the next: it takes all the weight,
    though neighbouring binary32 scores are far more than 1 apart.  In the dense product and in the stream; the largest
    among the prefix, or of the row's own.  Tolerance: WHOLE_WEIGHT."""
    for rows in (3, 170):
        g = torch.Generator().manual_seed(rows)
        heads, kv_heads, dim, prefix_length, capacity = 8, 4, 64, 210, 16
        prefix, own = caches(torch, g, rows, kv_heads, dim, prefix_length, capacity)
        q = torch.zeros(rows, heads * dim)
        q[:, ::dim] = size
        q[1::2] *= -1.0  # (codes are as negative as they are positive)
        for codes, scales in (prefix[:2], own[:2]):
            codes[..., 0] = codes[..., 0].clamp(-100, 100)
            scales[:] = 0.011
        for h in range(kv_heads):
            prefix[0][h, 71 * h % prefix_length, 0], prefix[0][h, (71 * h + 100) % prefix_length, 0] = 110, -110
        own[0][2::3, :, 5, 0], own[0][2::3, :, 4, 0] = 127, -127
        counts = [(5 * r) % capacity for r in range(rows)]
        out, lse = attend(torch, "f32", q, prefix, own, counts, heads, kv_heads, dim, prefix_length)
        for r in range(rows):
            want, want_lse, _, vmax = attention_reference(torch, q[r], prefix, own, r, counts[r], heads, kv_heads, dim, prefix_length,
                                                          0.125)
            assert bool((out[r].double() - want).abs().le(8 * U * vmax + WHOLE_WEIGHT).all()), (r, float((out[r].double() - want).abs().max()))
            assert bool((lse[r].double() - want_lse).abs().le(16 * U * want_lse.abs()).all()), r


def test_positions_whose_values_are_zero_keep_their_weight(torch):
    """Positions with a value scale of 0 count in the softmax beside positions with large ones.  Nothing of their own
    bounds their weights; they are far from binary32's largest all the same."""
    for rows in (3, 170):
        g = torch.Generator().manual_seed(rows)
        heads, kv_heads, dim, prefix_length, capacity = 8, 4, 64, 300, 16
        prefix, own = caches(torch, g, rows, kv_heads, dim, prefix_length, capacity)
        prefix[0][:] = 0
        prefix[1][:] = 0.7
        prefix[0][:, 296:, 0] = 127  # 4 positions whose scores are 11 above the 296 without values
        prefix[3][:, :296] = 0.0
        prefix[3][:, 296:] *= 2.0 ** 17
        q = torch.zeros(rows, heads * dim)
        q[:, ::dim] = 1.0
        counts = [0] * rows
        out, lse = attend(torch, "f32", q, prefix, own, counts, heads, kv_heads, dim, prefix_length)
        for r in (0, rows - 1):
            want, want_lse, big, vmax = attention_reference(torch, q[r], prefix, own, r, 0, heads, kv_heads, dim, prefix_length, 0.125)
            bound = (2 * (dim + 8) * big + prefix_length + 32) * U * vmax + U * want.abs()
            assert bool((out[r].double() - want).abs().le(bound).all()), r
            bound = ((dim + 8) * big + prefix_length) * U + 4 * U * want_lse.abs()
            assert bool((lse[r].double() - want_lse).abs().le(bound).all()), (r, float((lse[r].double() - want_lse).abs().max()))


@pytest.mark.parametrize("name", TYPES)
def test_weights_are_binary32_in_every_type(torch, name):
    """One position of a dense prefix has nearly all the weight: an output is off by what scores, weights and sums in
    binary32 leave, relative to sum w |v|, and half a step of its type (a weight of 11 bits would double fp16's)."""
    g = torch.Generator().manual_seed(12)
    rows, heads, kv_heads, dim, prefix_length, capacity = 170, 16, 4, 64, 300, 8
    prefix, own = caches(torch, g, rows, kv_heads, dim, prefix_length, capacity)
    q = (0.05 * torch.randn(rows, heads * dim, generator=g)).to(dtype_of(torch, name))
    q[:, ::dim] = (8.0 + torch.rand(rows, heads, generator=g)).to(q.dtype)
    prefix[0][..., 0], own[0][..., 0] = 0, 0
    prefix[0][:, 7], prefix[1][:, 7] = 0, 0.1
    prefix[0][:, 7, 0] = 127  # a score of 12.7 and more
    counts = [r % 9 for r in range(rows)]
    out, _ = attend(torch, name, q, prefix, own, counts, heads, kv_heads, dim, prefix_length)
    for r in range(rows):
        want, _, big, size, vmax = exactly(torch, q[r], prefix, own, r, counts[r], heads, kv_heads, dim)
        bound = (2 * (dim + 8) * big + prefix_length + capacity + 32) * U * size + (prefix_length + capacity) * 2.0 ** -30 * vmax
        bound += HALF[name] * want.abs() + 2.0 ** -25
        assert bool((out[r].double() - want).abs().le(bound).all()), (r, float(((out[r].double() - want).abs() / bound).max()))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("small", [2.0 ** -10, 2.0 ** -20, 2.0 ** -30])
def test_small_values_that_dominate(torch, name, small):
    """One position takes nearly all the weight and its values are `small` times the others'.  Weights are held as
    fp16 part(s) of at least 2^-25 next to the largest value scale: a reference M is at most 5 - e below the largest
    score (2^e the largest value scale), so n weights bring an error of n 127 2^-25 2^(e - 5) <= n 2^-30 max |v| on top of
    what binary32 has (relative to sum w |v|)."""
    for rows, prefix_length, capacity in ((3, 37, 40), (170, 300, 16)):
        g = torch.Generator().manual_seed(rows + prefix_length)
        heads, kv_heads, dim = 8, 4, 64
        prefix, own = caches(torch, g, rows, kv_heads, dim, prefix_length, capacity)
        q = torch.randn(rows, heads * dim, generator=g).to(dtype_of(torch, name))
        q[:, ::dim] = 8.0
        prefix[0][:, 7] = 0
        prefix[0][:, 7, 0] = 127
        prefix[1][:, 7] = 0.25  # a score of 8 * 127 * 0.25 / 8 = 32 above the others' order of 1
        prefix[0][:, :7, 0] = 0
        prefix[0][:, 8:, 0] = 0
        own[0][..., 0] = 0
        prefix[3][:, 7] *= small
        counts = [capacity - r % 3 for r in range(rows)]
        out, lse = attend(torch, name, q, prefix, own, counts, heads, kv_heads, dim, prefix_length)
        for r in {0, rows // 2, rows - 1}:
            want, want_lse, big, size, vmax = exactly(torch, q[r], prefix, own, r, counts[r], heads, kv_heads, dim)
            n = prefix_length + counts[r]
            bound = (2 * (dim + 8) * big + n + 32) * U * size + n * 2.0 ** -30 * vmax + HALF[name] * want.abs()
            if name == "f16":
                bound += 2.0 ** -25  # half a step of fp16 below its normal range
            assert bool((out[r].double() - want).abs().le(bound).all()), (r, float(((out[r].double() - want).abs() / bound).max()))
            bound = ((dim + 8) * big + n) * U + 4 * U * want_lse.abs()
            assert bool((lse[r].double() - want_lse).abs().le(bound).all()), r


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,heads,kv_heads,dim,prefix_length,capacity", PLANS)
def test_the_softmax_denominator_is_binary32_in_every_type(torch, name, rows, heads, kv_heads, dim, prefix_length, capacity):
    """lse takes no part in the rounding of weights: (D + 8) u S for the largest score, n u for the sum, 4 u of itself."""
    g = torch.Generator().manual_seed(3 * rows + dim)
    prefix, own = caches(torch, g, rows, kv_heads, dim, prefix_length, capacity)
    counts = [capacity - (3 * r) % (capacity + 1) for r in range(rows)]
    q = torch.randn(rows, heads * dim, generator=g).to(dtype_of(torch, name))
    _, lse = attend(torch, name, q, prefix, own, counts, heads, kv_heads, dim, prefix_length)
    for r in range(rows):
        _, want, big, _ = attention_reference(torch, q[r], prefix, own, r, counts[r], heads, kv_heads, dim, prefix_length, dim ** -0.5)
        bound = ((dim + 8) * big + prefix_length + counts[r]) * U + 4 * U * want.abs()
        assert bool((lse[r].double() - want).abs().le(bound).all()), (r, float(((lse[r].double() - want).abs() / bound).max()))


# ------------------------------------------------------------------ logits_select

@pytest.mark.parametrize("name,offset", [
    ("f32", 0.0), ("f32", 1e3), ("f32", -1e3), ("f32", 1e4), ("f32", -65504.0), ("f32", 1e6), ("f32", 1e8), ("f32", -1e9),
    ("f32", 3e10), ("f32", -1e30), ("f32", 1e38), ("f16", 1e3), ("f16", -2e4), ("f16", 6e4), ("bf16", 1e3), ("bf16", -1e9),
    ("bf16", 1e30)])
@pytest.mark.parametrize("rows,vocab", [(3, 8192), (2, 50001)])
def test_log_probabilities_do_not_depend_on_an_offset(torch, name, offset, rows, vocab):
    """l - max - log sum exp(l - max): an offset of all logits cancels in l - max.  Tolerance: that of logits around zero:
    a thread adds at most ceil(vocab / 4096) * 16 terms, 30 merges follow, every term is off by 2 u relative to the
    sum and its addition by as much; the logarithm makes that absolute; 4 u of the value itself."""
    from needle_b200 import native
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=g)
    # on the grid of the type at the offset: neighbouring values where it is coarse
    x = (offset + (3.0 if abs(offset) < 1e7 else abs(offset) * 2.0 ** -24 * 3) * x).to(dtype_of(torch, name))
    x[-1] = torch.where(torch.arange(vocab) % 3 == 0, x[-1], torch.full((), offset).to(x.dtype))
    d = x.cuda()
    a = rules_args(torch, name, d, {})
    ids, lps = torch.zeros(rows, dtype=torch.int32).cuda(), torch.zeros(rows).cuda()
    native.check(native.lib().needle_cuda_logits_select_dev(C.byref(a), ids.data_ptr(), lps.data_ptr(), stream_of(torch)))
    torch.cuda.synchronize()
    raw = x.double()
    terms = -(-vocab // 4096) * 16 + 30
    for r in range(rows):
        best = int((raw[r] == raw[r].max()).nonzero()[0, 0])
        want = float(torch.log_softmax(raw[r], 0)[best])
        assert int(ids[r]) == best
        assert abs(float(lps[r]) - want) <= (2 * terms + 4 * abs(want)) * U, (r, float(lps[r]), want)


def test_log_probabilities_of_logits_that_climb(torch):
    """Rows whose maximum rises all the way, and a row whose ids but a few are at -1e9 (masked by addition)."""
    from needle_b200 import native
    v = 20000
    x = torch.stack((torch.linspace(-1e5, 1e5, v), torch.linspace(3e4, -3e4, v), torch.full((v,), -1e9)))
    x[0, -40:] = 1e5
    x[2, 777] = -1e9 + 64
    x[2, 9000:9007] = -1e9 + 128
    d = x.cuda()
    a = rules_args(torch, "f32", d, {})
    ids, lps = torch.zeros(3, dtype=torch.int32).cuda(), torch.zeros(3).cuda()
    native.check(native.lib().needle_cuda_logits_select_dev(C.byref(a), ids.data_ptr(), lps.data_ptr(), stream_of(torch)))
    torch.cuda.synchronize()
    want = torch.log_softmax(x.double(), 1)
    best = [v - 40, 0, 9000]
    assert ids.tolist() == best
    for r in range(3):
        w = float(want[r, best[r]])
        assert abs(float(lps[r]) - w) <= (2 * 110 + 4 * abs(w)) * U, (r, float(lps[r]), w)


# ------------------------------------------------------------------ rope_append

def quotients(x):
    """Codes and scales by division, as the engine's append computes them (numpy, binary64)."""
    x = x.astype(np.float64)
    scale = np.maximum(np.abs(x).max(-1), 1e-12) / 127.0
    return np.rint(x / scale[..., None]).astype(np.int8), scale.astype(np.float32)


def products(x):
    x = x.astype(np.float64)
    scale = np.maximum(np.abs(x).max(-1), 1e-12) * (1.0 / 127.0)
    return np.rint(x / scale[..., None]).astype(np.int8), scale.astype(np.float32)


def append(torch, name, rows, dim):
    """Codes and scales of `rows` [tokens, dim] appended as keys and as values, without norm and rotation."""
    t = rows.shape[0]
    d = rows.cuda()
    cache = [torch.zeros(1, 1, t, dim, dtype=torch.int8).cuda(), torch.zeros(1, 1, t).cuda(),
             torch.zeros(1, 1, t, dim, dtype=torch.int8).cuda(), torch.zeros(1, 1, t).cuda()]
    at = torch.arange(t, dtype=torch.int32).cuda()
    rope_call(torch, name, d, d, d, torch.zeros_like(d), None, None, None, None, at, at * 0, at, cache, 1, 1, dim, 0, False, [], 1.0)
    torch.cuda.synchronize()
    return [c[0, 0].cpu().numpy() for c in cache]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_codes_of_half_the_largest_value(torch, name, dim):
    """Half of a row's largest value is 63.5 steps.  Binary32 rows: the code is what dividing by (largest / 127) gives, as
    in the engine.  16-bit rows: what dividing by (largest * (1 / 127)) gives, which on such a border alone is the other
    neighbour of 63.5 in one row of ten."""
    g = torch.Generator().manual_seed(dim)
    x = torch.rand(4000, dim, generator=g) - 0.5
    top = 0.5 + torch.rand(4000, generator=g)
    x = x.to(dtype_of(torch, name))
    x[:, 3] = top.to(x.dtype) * torch.where(torch.arange(4000) % 2 == 0, 1.0, -1.0).to(x.dtype)
    x[:, 9], x[:, 20] = x[:, 3] / 2, -x[:, 3] / 2
    rows = to_numpy(x)
    exact, other = quotients(rows), products(rows)
    assert (exact[0] != other[0]).any(1).mean() > 0.02  # the two definitions are told apart here
    np.testing.assert_array_equal(exact[1], other[1])
    want, scales = exact if name == "f32" else other
    got = append(torch, name, x, dim)
    for codes, stored in (got[:2], got[2:]):
        np.testing.assert_array_equal(codes, want)
        np.testing.assert_array_equal(stored, scales)


def test_codes_and_scales_are_the_engine_s(torch):
    """The keys and values that an engine with a float cache holds, appended by the operator, against an engine with an
    int8 cache that read the same tokens (first layer: nothing before it depends on the cache)."""
    from needle_b200 import synth
    from needle_b200.backend import CudaEngine, StepRequest
    archive = synth.build_archive(3, synth.small_geometry(layers=2, vocab=512), probe_heads=False)
    tokens = np.random.default_rng(5).integers(0, 512, 48)
    held = {}
    for kind in ("float32", "int8"):
        with CudaEngine(archive, device=0, max_seqs=1, max_len=64, max_sink=0, kv_cache=kind) as eng:
            eng.reset(0, 64, 0)
            for t in tokens:
                eng.step([StepRequest(0, int(t), False)])
            held[kind] = eng.read_kv_f32(0, 0) if kind == "float32" else eng.read_kv(0, 0)
    n, dim = len(tokens), held["float32"][0].shape[-1]
    kc, vc, ks, vs = held["int8"]
    for floats, codes, scales in ((held["float32"][0], kc, ks), (held["float32"][1], vc, vs)):
        rows = np.ascontiguousarray(floats[:, :n]).reshape(-1, dim)
        assert np.abs(rows).max() > 0
        got = append(torch, "f32", torch.from_numpy(rows), dim)
        for k in (0, 2):
            np.testing.assert_array_equal(got[k], codes[:, :n].reshape(-1, dim))
            np.testing.assert_array_equal(got[k + 1], scales[:, :n].reshape(-1))


@pytest.mark.parametrize("name,size", [("f32", 1e30), ("f16", 6e4), ("bf16", 1e18), ("bf16", 1e19), ("bf16", 3e38), ("bf16", 1e-30)])
def test_norms_of_large_and_small_queries(torch, name, size):
    """Squares that overflow or vanish in binary32: (1 + s) x / sqrt(mean x^2 + 1e-6) is within its range all the same."""
    g = torch.Generator().manual_seed(6)
    t, dim = 40, 128
    x = ((torch.rand(t, dim, generator=g) - 0.5) * 2 * size).to(dtype_of(torch, name))
    x[1::2] = torch.randn(t // 2, dim, generator=g).to(x.dtype)  # ordinary rows beside them, in the same warp
    norm = 0.2 * torch.randn(dim, generator=g)
    d = x.cuda()
    out = torch.zeros_like(d)
    cache = [torch.zeros(1, 1, t, dim, dtype=torch.int8).cuda(), torch.zeros(1, 1, t).cuda(),
             torch.zeros(1, 1, t, dim, dtype=torch.int8).cuda(), torch.zeros(1, 1, t).cuda()]
    at = torch.arange(t, dtype=torch.int32).cuda()
    small = torch.zeros_like(d)
    rope_call(torch, name, d, small, small, out, None, None, norm.cuda(), None, at, at * 0, at, cache, 1, 1, dim, 0, False, [], 1.0)
    torch.cuda.synchronize()
    y = x.double()
    want = (1.0 + norm.double()) * y / ((y * y).mean(-1, keepdim=True) + 1e-6).sqrt()
    # a sum of 128 squares, a root and two products in binary32, and the rounding to the type
    bound = (200 * U + HALF[name]) * want.abs() + (2.0 ** -25 if name == "f16" else 1e-38)
    assert bool((out.double().cpu() - want).abs().le(bound).all())
