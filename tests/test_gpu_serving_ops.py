"""The serving operators on the GPU against plain implementations in binary64 (torch, on the CPU).

Tolerances.  u = 2^-24 (half a binary32 step), h = half a step of the element type (2^-24, 2^-11, 2^-8).
Codes, ids and scales are compared for equality.  Attention: a score of D products in binary32, a power
and the scale is off by at most (D + 8) u S, S the largest sum |q_i k_i| scale; queries and weights may be
split into two fp16 parts (2^-22 each, 4 u); a weight's relative error is then twice the scores' (its own
and the largest one's), a sum of n weights adds n u, so an output is off by at most
(2 (D + 8) S + n + 32) u max|v|, plus 2^-11 max|v| for 16-bit types, whose weights may be rounded to
fp16 once, plus h |o| for the rounding of the output.  lse: (D + 8) u S + n u + 4 u |lse| (+ 2^-11 for
16-bit types).
"""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16", "bf16"]
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def torch():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import needle_b200.build
    needle_b200.build.build()
    return torch


def dtype_of(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def kind_of(name):
    from needle_b200 import native
    return {"f32": native.TYPE_F32, "f16": native.TYPE_F16, "bf16": native.TYPE_BF16}[name]


def pointer(t):
    return None if t is None else t.data_ptr()


def stream_of(torch):
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ rope_append

def rope_call(torch, name, q, k, v, q_out, k_out, v_out, q_norm, k_norm, positions, slots, entries, cache, heads,
              kv_heads, dim, rotary, interleaved, inverse, magnitude):
    from needle_b200 import native
    kc, ks, vc, vs = cache
    a = native.RopeAppend(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), pointer(k_out), pointer(v_out), q.stride(0),
        k.stride(0), v.stride(0), q_out.stride(0), 0 if k_out is None else k_out.stride(0),
        0 if v_out is None else v_out.stride(0), pointer(q_norm), pointer(k_norm), positions.data_ptr(),
        slots.data_ptr(), entries.data_ptr(), kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), magnitude,
        kind_of(name), q.shape[0], heads, kv_heads, dim, rotary, int(interleaved), kc.shape[0], kc.shape[2])
    w = (C.c_double * max(1, rotary // 2))(*inverse)
    native.check(native.lib().needle_cuda_rope_append_dev(C.byref(a), w, stream_of(torch)))


def turned(x, norm, angle, magnitude, rotary, interleaved):
    """numpy binary64: norm (stored in binary32), rotation (stored in binary32)."""
    x = x.astype(np.float64)
    if norm is not None:
        inverse = 1.0 / np.sqrt((x * x).sum(-1, keepdims=True) / x.shape[-1] + 1e-6)
        x = ((1.0 + norm.astype(np.float64)) * x * inverse).astype(np.float32).astype(np.float64)
    y = x.copy()
    n = rotary // 2
    a = np.arange(n) * 2 if interleaved else np.arange(n)
    b = a + 1 if interleaved else a + n
    c, s = np.cos(angle)[:, None] * magnitude, np.sin(angle)[:, None] * magnitude
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y.astype(np.float32)


def quantised(x):
    x = x.astype(np.float64)
    scale = np.maximum(np.abs(x).max(-1), 1e-12) * (1.0 / 127.0)
    return np.rint(x / scale[..., None]).astype(np.int8), scale.astype(np.float32)


def to_numpy(t):
    return t.detach().float().cpu().numpy()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,interleaved,norm,fused", [
    (1, 8, 4, 64, 64, False, True, True), (5, 8, 4, 64, 64, True, True, False), (33, 6, 2, 128, 64, False, False, True),
    (7, 3, 3, 128, 128, True, True, True), (9, 4, 1, 64, 2, False, False, False), (4, 2, 2, 128, 6, False, True, True),
    (3, 5, 5, 64, 50, False, False, True), (6, 1, 1, 64, 0, False, True, True), (300, 16, 2, 128, 96, False, True, True)])
def test_rope_append(torch, name, tokens, heads, kv_heads, dim, rotary, interleaved, norm, fused):
    g = torch.Generator().manual_seed(tokens * 131 + rotary)
    dt = dtype_of(torch, name)
    width = (heads + 2 * kv_heads) * dim
    extra = 0 if fused else 1  # rows an odd element apart: nothing is aligned past its element
    qkv = torch.randn(tokens, width + extra, generator=g).to(dt)
    qkv[0, :dim] = 0.0            # an all-zero query head
    qkv[-1, heads * dim:(heads + 1) * dim] = 0.0  # and an all-zero key head: the smallest scale
    d = qkv.cuda()
    q, k, v = d[:, :heads * dim], d[:, heads * dim:(heads + kv_heads) * dim], d[:, (heads + kv_heads) * dim:width]
    q_norm = 0.2 * torch.randn(dim, generator=g) if norm else None
    k_norm = 0.2 * torch.randn(dim, generator=g) if norm else None
    positions = torch.randint(0, 1 << 20, (tokens,), generator=g, dtype=torch.int32)
    positions[0] = 0
    slot_count, capacity = 3, tokens + 2
    order = torch.randperm(slot_count * capacity, generator=g)[:tokens]
    slots, entries = (order // capacity).int(), (order % capacity).int()
    if tokens > 4:  # padding and what is out of range is left out
        slots[1], entries[2], slots[3], entries[4] = -1, -7, slot_count, capacity
    cache = [torch.full((slot_count, kv_heads, capacity, dim), 77, dtype=torch.int8).cuda(),
             torch.full((slot_count, kv_heads, capacity), 5.0).cuda(),
             torch.full((slot_count, kv_heads, capacity, dim), 78, dtype=torch.int8).cuda(),
             torch.full((slot_count, kv_heads, capacity), 6.0).cuda()]
    inverse = [10000.0 ** (-2.0 * i / max(rotary, 1)) for i in range(rotary // 2)]
    magnitude = 1.25
    q_out = torch.full((tokens, heads * dim + 2 * extra), 9.0, dtype=dt).cuda()
    k_out = torch.zeros(tokens, kv_heads * dim, dtype=dt).cuda()
    v_out = torch.zeros(tokens, kv_heads * dim, dtype=dt).cuda()
    rope_call(torch, name, q, k, v, q_out[:, :heads * dim], k_out, v_out, None if q_norm is None else q_norm.cuda(),
              None if k_norm is None else k_norm.cuda(), positions.cuda(), slots.cuda(), entries.cuda(), cache, heads,
              kv_heads, dim, rotary, interleaved, inverse, magnitude)
    torch.cuda.synchronize()
    x = to_numpy(qkv)
    angle = positions.numpy().astype(np.float64)[:, None] * np.array(inverse)
    want_q = turned(x[:, :heads * dim].reshape(tokens, heads, dim), None if q_norm is None else q_norm.numpy(), angle,
                    magnitude, rotary, interleaved)
    key = turned(x[:, heads * dim:(heads + kv_heads) * dim].reshape(tokens, kv_heads, dim),
                 None if k_norm is None else k_norm.numpy(), angle, magnitude, rotary, interleaved)
    val = x[:, (heads + kv_heads) * dim:width].reshape(tokens, kv_heads, dim)
    got_q = to_numpy(q_out[:, :heads * dim]).reshape(tokens, heads, dim).astype(np.float64)
    # binary32 arithmetic for 16-bit queries: at most 16 roundings of 2^-24 of the pair's magnitude, and the
    # rounding to the type; binary32 queries: binary64 arithmetic rounded once
    size = np.abs(want_q) + (0 if name == "f32" else 16 * U / HALF[name]) * np.abs(want_q).max(-1, keepdims=True)
    assert np.all(np.abs(got_q - want_q) <= HALF[name] * 1.01 * size + 2.0 ** -25)
    assert extra == 0 or bool((q_out[:, heads * dim:] == 9.0).all())
    for rows, codes, scales, out, fill, fill_scale in ((key, cache[0], cache[1], k_out, 77, 5.0),
                                                       (val, cache[2], cache[3], v_out, 78, 6.0)):
        want_codes, want_scales = quantised(rows)
        whole = np.full(codes.shape, fill, dtype=np.int8)
        whole_scales = np.full(scales.shape, fill_scale, dtype=np.float32)
        for t in range(tokens):
            s, e = int(slots[t]), int(entries[t])
            if 0 <= s < slot_count and 0 <= e < capacity:
                whole[s, :, e], whole_scales[s, :, e] = want_codes[t], want_scales[t]
        np.testing.assert_array_equal(codes.cpu().numpy(), whole)
        np.testing.assert_array_equal(scales.cpu().numpy(), whole_scales)
        stands_for = torch.from_numpy(want_codes.astype(np.float32) * want_scales[..., None]).to(dt)
        assert torch.equal(out.cpu().view(tokens, kv_heads, dim), stands_for)


@pytest.mark.parametrize("tokens", [500, 1000, 1777, 3553])
@pytest.mark.parametrize("name,heads,kv_heads,dim,rotary,interleaved,norm,fused", [
    ("f32", 3, 1, 64, 64, False, True, True), ("bf16", 5, 2, 64, 32, True, False, False), ("f16", 2, 3, 128, 128, False, True, True),
    ("f32", 1, 1, 128, 2, True, True, True), ("bf16", 7, 1, 128, 128, True, True, True)])
def test_rope_append_tokens_shared_by_fewer_warps(torch, name, tokens, heads, kv_heads, dim, rotary, interleaved, norm, fused):
    """Batches from which a token is shared by four warps, two, and one, the last ones not filling a CTA."""
    test_rope_append(torch, name, tokens, heads, kv_heads, dim, rotary, interleaved, norm, fused)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,interleaved", [
    (5, 3, 2, 64, 2, False), (400, 3, 2, 64, 2, False), (9, 2, 1, 128, 2, True), (9, 4, 1, 64, 6, True), (7, 1, 2, 128, 10, True),
    (7, 1, 2, 128, 10, False), (6, 2, 2, 64, 0, True)])
def test_rope_append_few_rotated_dimensions(torch, name, tokens, heads, kv_heads, dim, rotary, interleaved):
    """Rotations that end inside a lane's elements, in rows that allow wide accesses."""
    test_rope_append(torch, name, tokens, heads, kv_heads, dim, rotary, interleaved, True, True)


def test_rope_append_codes_next_to_a_border(torch):
    """Values of half a step and of whole ones: the quotients that binary32 cannot place are divided exactly."""
    d = 128
    x = torch.zeros(3, d)
    x[0] = torch.arange(d) - 63.5   # top 63.5: codes 2 x, and the scale is 0.5
    x[1] = (torch.arange(d) - 64.0) * 0.5
    x[1, 0] = 127.0                 # halves of a step of 1: ties to even
    x[2] = torch.randn(d, generator=torch.Generator().manual_seed(1))
    x[2, 7], x[2, 8], x[2, 9] = 4.0, 2.0, -2.0  # top and half of it: 63.5 steps
    for name in TYPES:
        v = x.to(dtype_of(torch, name)).cuda()
        cache = [torch.zeros(1, 1, 3, d, dtype=torch.int8).cuda(), torch.zeros(1, 1, 3).cuda(),
                 torch.zeros(1, 1, 3, d, dtype=torch.int8).cuda(), torch.zeros(1, 1, 3).cuda()]
        at = torch.arange(3, dtype=torch.int32).cuda()
        rope_call(torch, name, v, v, v, torch.zeros_like(v), None, None, None, None, at * 0, at * 0, at, cache, 1, 1, d, 0,
                  False, [], 1.0)
        torch.cuda.synchronize()
        codes, scales = quantised(to_numpy(v))
        for k in (0, 2):
            np.testing.assert_array_equal(cache[k][0, 0].cpu().numpy(), codes)
            np.testing.assert_array_equal(cache[k + 1][0, 0].cpu().numpy(), scales)


def test_rope_append_in_place_and_next_to_each_other(torch):
    """q_out = q, k_out = k, v_out = v inside one fused buffer give what separate outputs give."""
    g = torch.Generator().manual_seed(4)
    t, h, k, d = 19, 8, 4, 64
    qkv = torch.randn(t, (h + 2 * k) * d, generator=g).cuda()
    inverse = [10000.0 ** (-2.0 * i / d) for i in range(d // 2)]
    positions = torch.arange(t, dtype=torch.int32).cuda()
    slots = torch.zeros(t, dtype=torch.int32).cuda()

    def run(src, outs):
        cache = [torch.zeros(1, k, t, d, dtype=torch.int8).cuda(), torch.zeros(1, k, t).cuda(),
                 torch.zeros(1, k, t, d, dtype=torch.int8).cuda(), torch.zeros(1, k, t).cuda()]
        q, kk, v = src.split([h * d, k * d, k * d], 1)
        o = outs or (q, kk, v)
        rope_call(torch, "f32", q, kk, v, *o, None, None, positions, slots, positions, cache, h, k, d, d, False, inverse,
                  1.0)
        return [*o, *cache]

    apart = run(qkv.clone(), [torch.zeros(t, n * d).cuda() for n in (h, k, k)])
    within = run(qkv.clone(), None)
    torch.cuda.synchronize()
    for a, b in zip(apart, within):
        assert torch.equal(a, b)


def test_rope_append_extreme_values(torch):
    """Rows of the largest and smallest magnitudes, exact halves, infinities and NaN: no code outside
    +-127, and rows beside a bad one are not touched by it."""
    t, k, d = 6, 1, 64
    rows = torch.zeros(t, d)
    rows[0] = 3e38
    rows[1] = 1e-30
    rows[2] = torch.arange(d).float() - 31.5
    rows[3, 0], rows[3, 1], rows[3, 2] = math.inf, 1.0, math.nan
    rows[4, 5] = math.nan
    rows[5] = torch.linspace(-127, 127, d)
    v = rows.cuda()
    cache = [torch.zeros(1, k, t, d, dtype=torch.int8).cuda(), torch.zeros(1, k, t).cuda(),
             torch.zeros(1, k, t, d, dtype=torch.int8).cuda(), torch.zeros(1, k, t).cuda()]
    at = torch.arange(t, dtype=torch.int32).cuda()
    rope_call(torch, "f32", v, v, v, torch.zeros_like(v), None, None, None, None, at, torch.zeros_like(at), at, cache, 1,
              k, d, 0, False, [], 1.0)
    torch.cuda.synchronize()
    for codes, scales in ((cache[0], cache[1]), (cache[2], cache[3])):
        want, want_scales = quantised(rows[[0, 1, 2, 5]].numpy())
        np.testing.assert_array_equal(codes[0, 0, [0, 1, 2, 5]].cpu().numpy(), want)
        np.testing.assert_array_equal(scales[0, 0, [0, 1, 2, 5]].cpu().numpy(), want_scales)
        assert int(codes.abs().max()) <= 127 and bool((codes[0, 0, 3] == 0).all())
        assert scales[0, 0, 3] == math.inf and bool((codes[0, 0, 4] == 0).all())


# ------------------------------------------------------------------ prefix_attention

def attention_call(torch, name, q, out, lse, prefix, own, slots, counts, heads, kv_heads, dim, prefix_length, scale=0.0,
                   workspace=None):
    from needle_b200 import native
    pk, pks, pv, pvs = prefix
    kc, ks, vc, vs = own
    a = native.PrefixAttention(
        q.data_ptr(), out.data_ptr(), pointer(lse), q.stride(0), out.stride(0), pointer(pk), pointer(pks), pointer(pv),
        pointer(pvs), pointer(kc), pointer(ks), pointer(vc), pointer(vs), pointer(slots), counts.data_ptr(), scale,
        kind_of(name), q.shape[0], heads, kv_heads, dim, prefix_length, 0 if pk is None else pk.shape[1],
        0 if kc is None else kc.shape[0], 0 if kc is None else kc.shape[2])
    size = C.c_size_t()
    native.check(native.lib().needle_cuda_prefix_attention_workspace(C.byref(a), C.byref(size)))
    if workspace is None:
        workspace = torch.empty(max(16, size.value), dtype=torch.uint8, device="cuda")
        workspace.fill_(0xff)  # NaN everywhere: nothing may be read before it is written
    assert workspace.numel() >= size.value
    native.check(native.lib().needle_cuda_prefix_attention_dev(C.byref(a), workspace.data_ptr(), workspace.numel(),
                                                               stream_of(torch)))
    return workspace


def random_cache(torch, g, *shape):
    codes = torch.randint(-127, 128, shape, generator=g, dtype=torch.int32).to(torch.int8)
    scales = 0.004 + 0.03 * torch.rand(*shape[:-1], generator=g)
    return codes, scales


def attention_reference(torch, q, prefix, own, slot, count, heads, kv_heads, dim, prefix_length, scale):
    """One row in binary64: (out [heads, dim], lse [heads], largest sum |q k| scale, largest |v|)."""
    group = heads // kv_heads
    q = q.double().view(kv_heads, group, dim)
    keys = (prefix[0][:, :prefix_length].double() * prefix[1][:, :prefix_length, None].double())
    values = (prefix[2][:, :prefix_length].double() * prefix[3][:, :prefix_length, None].double())
    if count:
        keys = torch.cat((keys, own[0][slot, :, :count].double() * own[1][slot, :, :count, None].double()), 1)
        values = torch.cat((values, own[2][slot, :, :count].double() * own[3][slot, :, :count, None].double()), 1)
    if keys.shape[1] == 0:
        return torch.zeros(heads, dim).double(), torch.full((heads,), -math.inf).double(), 0.0, 0.0
    s = torch.einsum("kgd,kpd->kgp", q, keys) * scale
    big = float((torch.einsum("kgd,kpd->kgp", q.abs(), keys.abs()) * scale).max())
    out = torch.einsum("kgp,kpd->kgd", torch.softmax(s, -1), values)
    return out.reshape(heads, dim), torch.logsumexp(s, -1).reshape(heads), big, float(values.abs().max())


def check_attention(torch, name, rows, heads, kv_heads, dim, prefix_length, capacity, counts, slots=None, scale=0.0,
                    seed=0, slot_count=None, spread=1.0, odd=False):
    g = torch.Generator().manual_seed(seed + 7919 * rows + prefix_length)
    dt = dtype_of(torch, name)
    slot_count = slot_count or max(rows, 1)
    q = (spread * torch.randn(rows, heads * dim + (1 if odd else 0), generator=g)).to(dt)[:, :heads * dim]
    prefix = [*random_cache(torch, g, kv_heads, prefix_length + 3, dim), *random_cache(torch, g, kv_heads, prefix_length + 3, dim)]
    own = [*random_cache(torch, g, slot_count, kv_heads, capacity, dim), *random_cache(torch, g, slot_count, kv_heads, capacity, dim)]
    for s in (prefix[1], prefix[3]):  # what lies behind the prefix and behind a row's count is never used
        s[:, prefix_length:] = math.nan
    counts = torch.tensor(counts, dtype=torch.int32)
    named = torch.arange(rows, dtype=torch.int32) if slots is None else torch.tensor(slots, dtype=torch.int32)
    longest = torch.zeros(slot_count, dtype=torch.int64)
    for r in range(rows):
        if 0 <= named[r] < slot_count:
            longest[named[r]] = max(int(longest[named[r]]), min(max(int(counts[r]), 0), capacity))
    for s in range(slot_count):
        own[1][s, :, longest[s]:] = math.inf
        own[3][s, :, longest[s]:] = math.nan
    out = torch.full((rows, heads * dim + 4), 3.0, dtype=dt).cuda()
    lse = torch.full((rows, heads), 4.0).cuda()
    dq = torch.empty(rows, q.stride(0) if rows else heads * dim, dtype=dt, device="cuda")[:, :heads * dim]
    dq.copy_(q)
    attention_call(torch, name, dq, out[:, :heads * dim], lse, [t.cuda() for t in prefix], [t.cuda() for t in own],
                   None if slots is None else named.cuda(), counts.cuda(), heads, kv_heads, dim, prefix_length, scale)
    torch.cuda.synchronize()
    assert bool((out[:, heads * dim:] == 3.0).all())
    out, lse = out[:, :heads * dim].double().cpu().view(rows, heads, dim), lse.double().cpu()
    sc = scale or dim ** -0.5
    extra = 0.0 if name == "f32" else 2.0 ** -11
    for r in range(rows):
        s = int(named[r])
        if not 0 <= s < slot_count:
            assert bool((out[r] == 3.0).all()) and bool((lse[r] == 4.0).all()), r
            continue
        n = min(max(int(counts[r]), 0), capacity)
        want, want_lse, big, vmax = attention_reference(torch, q[r], prefix, own, s, n, heads, kv_heads, dim, prefix_length, sc)
        total = prefix_length + n
        bound = ((2 * (dim + 8) * big + total + 32) * U + extra) * vmax + HALF[name] * want.abs() + 1e-30
        assert bool((out[r] - want).abs().le(bound).all()), (r, float(((out[r] - want).abs() / bound).max()))
        if total == 0:
            assert bool((lse[r] == -math.inf).all())
        else:
            bound = ((dim + 8) * big + total) * U + extra + 4 * U * want_lse.abs()
            assert bool((lse[r] - want_lse).abs().le(bound).all()), r


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 4, 64), (4, 4, 128), (14, 2, 64), (8, 1, 128), (12, 1, 64), (40, 2, 64)])
def test_prefix_attention_head_layouts(torch, name, heads, kv_heads, dim):
    check_attention(torch, name, 3, heads, kv_heads, dim, 37, 20, [0, 1, 20])


@pytest.mark.parametrize("prefix_length", [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
def test_prefix_attention_prefix_lengths(torch, prefix_length):
    check_attention(torch, "f32", 5, 8, 4, 64, prefix_length, 9, [0, 1, 8, 9, 3])
    check_attention(torch, "bf16", 5, 8, 2, 128, prefix_length, 9, [0, 1, 8, 9, 3])


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,heads,kv_heads,dim,prefix_length", [
    (70, 8, 4, 64, 300), (64, 8, 4, 64, 128), (130, 4, 2, 64, 129), (33, 32, 4, 128, 500), (200, 3, 1, 128, 1025),
    (65, 7, 1, 64, 2048)])
def test_prefix_attention_many_rows(torch, name, rows, heads, kv_heads, dim, prefix_length):
    """Batches whose rows share the prefix in tiles, with tiles and prefixes that end raggedly."""
    g = np.random.default_rng(rows)
    check_attention(torch, name, rows, heads, kv_heads, dim, prefix_length, 40, g.integers(0, 41, rows).tolist())


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,heads,kv_heads,dim,prefix_length", [
    (130, 8, 4, 64, 300), (400, 4, 2, 64, 129), (513, 8, 4, 64, 128), (40, 32, 4, 128, 500), (32, 4, 4, 128, 2049),
    (700, 2, 2, 128, 97), (11, 24, 4, 64, 1000)])
def test_prefix_attention_enough_scores_for_the_dense_prefix(torch, name, rows, heads, kv_heads, dim, prefix_length):
    """65536 scores a KV head and more; packed rows that fill a tile, end inside one, or are fewer than one."""
    g = np.random.default_rng(rows)
    check_attention(torch, name, rows, heads, kv_heads, dim, prefix_length, 24, g.integers(0, 25, rows).tolist())


def test_prefix_attention_dense_prefix_padding_scales_and_strides(torch):
    rows = 170
    slots = [(5 * r) % 4 for r in range(rows)]
    slots[1], slots[3], slots[-1] = -1, 4, 1 << 30
    counts = [(7 * r) % 19 - 2 for r in range(rows)]
    counts[2] = 1 << 30
    check_attention(torch, "f32", rows, 8, 4, 64, 210, 16, counts, slots=slots, slot_count=4)
    check_attention(torch, "bf16", rows, 8, 4, 64, 210, 16, [0] * rows, slots=[-1] * rows, slot_count=4)
    for scale in (1e-3, 0.5):
        check_attention(torch, "f16", rows, 8, 4, 64, 200, 12, [5] * rows, scale=scale, odd=True)
    check_attention(torch, "f32", rows, 8, 4, 64, 300, 12, [5] * rows, spread=30.0)
    check_attention(torch, "f32", rows, 8, 4, 64, 300, 12, [5] * rows, spread=1e-4)
    check_attention(torch, "bf16", rows, 8, 4, 64, 300, 12, [5] * rows, spread=1000.0)


@pytest.mark.parametrize("name", TYPES)
def test_prefix_attention_long_own_caches(torch, name):
    check_attention(torch, name, 2, 8, 4, 64, 5, 5000, [4999, 2049])
    check_attention(torch, name, 1, 4, 1, 128, 0, 3001, [3001])


@pytest.mark.parametrize("rows", [6, 90])
def test_prefix_attention_slots_padding_and_counts(torch, rows):
    """Slots in any order, named twice, out of range (rows left as they were); counts out of range."""
    slots = [(5 * r) % 4 for r in range(rows)]
    slots[1], slots[3], slots[-1] = -1, 4, 1 << 30
    counts = [(7 * r) % 19 - 2 for r in range(rows)]
    counts[2] = 1 << 30
    check_attention(torch, "f32", rows, 8, 4, 64, 21, 16, counts, slots=slots, slot_count=4)
    check_attention(torch, "f16", rows, 8, 4, 64, 0, 16, counts, slots=slots, slot_count=4)


def test_prefix_attention_scales_and_strides(torch):
    """Sharp and flat softmaxes; rows an odd number of elements apart."""
    for scale in (1e-3, 0.5):
        check_attention(torch, "f32", 4, 8, 4, 64, 200, 12, [0, 4, 12, 7], scale=scale, odd=True)
        check_attention(torch, "f16", 80, 8, 4, 64, 200, 12, [5] * 80, scale=scale, odd=True)
    check_attention(torch, "f32", 70, 8, 4, 64, 300, 12, [5] * 70, spread=30.0)
    check_attention(torch, "f32", 70, 8, 4, 64, 300, 12, [5] * 70, spread=1e-4)
    check_attention(torch, "bf16", 70, 8, 4, 64, 300, 12, [5] * 70, spread=1000.0)


def test_prefix_attention_without_own_caches(torch):
    g = torch.Generator().manual_seed(3)
    prefix = [*random_cache(torch, g, 2, 50, 64), *random_cache(torch, g, 2, 50, 64)]
    q = torch.randn(3, 4 * 64, generator=g)
    out, lse = torch.zeros(3, 4 * 64).cuda(), torch.zeros(3, 4).cuda()
    own = [torch.zeros(3, 2, 0, 64, dtype=torch.int8).cuda(), torch.zeros(3, 2, 0).cuda()] * 2
    attention_call(torch, "f32", q.cuda(), out, lse, [t.cuda() for t in prefix], own, None,
                   torch.zeros(3, dtype=torch.int32).cuda(), 4, 2, 64, 50)
    torch.cuda.synchronize()
    for r in range(3):
        want, want_lse, big, vmax = attention_reference(torch, q[r], prefix, None, 0, 0, 4, 2, 64, 50, 0.125)
        assert float((out[r].double().cpu().view(4, 64) - want).abs().max()) <= (2 * 72 * big + 82) * U * vmax + U * vmax
        assert float((lse[r].double().cpu() - want_lse).abs().max()) <= (72 * big + 50) * U + 4 * U * float(want_lse.abs().max())


def test_prefix_attention_matches_the_fast_attention_operator(torch):
    """Without a prefix and in the engine's geometry: the values of needle_cuda_attention_dev_fast."""
    from needle_b200 import native
    g = torch.Generator().manual_seed(8)
    batch, cap = 9, 300
    q = torch.randn(batch, 512, generator=g).cuda()
    own = [t.cuda() for t in (*random_cache(torch, g, batch, 4, cap, 64), *random_cache(torch, g, batch, 4, cap, 64))]
    counts = torch.tensor([1, 2, 31, 32, 33, 100, 255, 299, 300], dtype=torch.int32).cuda()
    a, b = torch.zeros(batch, 512).cuda(), torch.zeros(batch, 512).cuda()
    attention_call(torch, "f32", q, a, None, [None] * 4, own, None, counts, 8, 4, 64, 0)
    native.check(native.lib().needle_cuda_attention_dev_fast(
        q.data_ptr(), own[0].data_ptr(), own[1].data_ptr(), own[2].data_ptr(), own[3].data_ptr(), counts.data_ptr(),
        batch, cap, b.data_ptr(), stream_of(torch)))
    torch.cuda.synchronize()
    assert float((a - b).abs().max()) <= 2 * 2e-4 * float(b.abs().max())  # each within 2e-4 of binary64


# ------------------------------------------------------------------ logits_rules, logits_select

def rules_args(torch, name, x, rules):
    from needle_b200 import native
    h, b, m = rules.get("history"), rules.get("bias_ids"), rules.get("masks")
    return native.LogitsRules(
        x.data_ptr(), x.stride(0), pointer(h), 0 if h is None else h.stride(0), pointer(rules.get("history_lengths")),
        pointer(rules.get("prompt_lengths")), pointer(rules.get("repetition")), pointer(rules.get("presence")),
        pointer(rules.get("frequency")), pointer(b), pointer(rules.get("bias_values")), 0 if b is None else b.stride(0),
        pointer(rules.get("bias_counts")), pointer(m), pointer(rules.get("mask_slots")), 0 if m is None else m.shape[0],
        kind_of(name), x.shape[0], x.shape[1])


def rules_reference(x, rules):
    """numpy, binary32 step by step: (ruled logits before the mask, allowed)."""
    x = x.astype(np.float32).copy()
    rows, vocab = x.shape
    r = {k: v.cpu().numpy() for k, v in rules.items()}
    allowed = np.ones((rows, vocab), dtype=bool)
    one = np.float32(1.0)
    for i in range(rows):
        if "history" in r:
            n = int(np.clip(r["history_lengths"][i], 0, r["history"].shape[1]))
            past = r["history"][i, :n]
            p = int(max(r["prompt_lengths"][i], 0)) if "prompt_lengths" in r else 0
            rep = r["repetition"][i] if "repetition" in r else one
            freq = r["frequency"][i] if "frequency" in r else np.float32(0)
            pres = r["presence"][i] if "presence" in r else np.float32(0)
            for v in np.unique(past[(past >= 0) & (past < vocab)]):
                x[i, v] = x[i, v] / rep if x[i, v] > 0 else x[i, v] * rep
                c = int((past[p:] == v).sum())
                if c:
                    x[i, v] = np.float32(x[i, v] - np.float32(freq * np.float32(c)))
                    x[i, v] = np.float32(x[i, v] - pres)
        if "bias_ids" in r:
            last = {}
            for j in range(int(np.clip(r["bias_counts"][i], 0, r["bias_ids"].shape[1]))):
                v = int(r["bias_ids"][i, j])
                if 0 <= v < vocab:
                    last[v] = r["bias_values"][i, j]
            for v, b in last.items():
                x[i, v] = np.float32(x[i, v] + b)
        if "masks" in r:
            s = int(r["mask_slots"][i])
            if s >= r["masks"].shape[0]:
                allowed[i] = False
            elif s >= 0:
                bits = np.unpackbits(r["masks"][s].astype(np.uint32).view(np.uint8), bitorder="little")
                allowed[i] = bits[:vocab] != 0
    return x, allowed


def make_rules(torch, rows, vocab, seed, history=40, biases=6, masks=3):
    g = np.random.default_rng(seed)
    f = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    r = {}
    if history:
        r["history"] = f(g.integers(-2, min(vocab, 30) + 2, (rows, history)).astype(np.int32))  # repeats, some out of range
        r["history_lengths"] = f(g.integers(-1, history + 3, rows).astype(np.int32))
        r["prompt_lengths"] = f(g.integers(-1, history + 3, rows).astype(np.int32))
        r["repetition"] = f(g.uniform(0.8, 1.4, rows).astype(np.float32))
        r["presence"] = f(g.uniform(-0.5, 0.5, rows).astype(np.float32))
        r["frequency"] = f(g.uniform(-0.5, 0.5, rows).astype(np.float32))
    if biases:
        r["bias_ids"] = f(g.integers(-1, min(vocab, 12) + 1, (rows, biases)).astype(np.int32))  # ids twice, out of range
        r["bias_values"] = f(g.standard_normal((rows, biases)).astype(np.float32) * 3)
        r["bias_counts"] = f(g.integers(-1, biases + 2, rows).astype(np.int32))
    if masks:
        words = (vocab + 31) // 32
        m = g.integers(0, 1 << 32, (masks, words), dtype=np.uint32)
        m[0] = 0  # allows nothing
        r["masks"] = f(m.view(np.int32))
        slots = g.integers(-1, masks + 1, rows).astype(np.int32)
        slots[0] = 0
        r["mask_slots"] = f(slots)
    return r


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,vocab,pad", [(1, 1, 0), (3, 7, 0), (4, 8192, 0), (5, 8193, 0), (3, 8191, 1), (9, 500, 3),
                                            (2, 50001, 0), (3, 131072 + 5, 2), (2, 70000, 8)])
def test_logits_rules_and_select(torch, name, rows, vocab, pad):
    """Both operators against the reference: ruled logits bit for bit (one more rounding for 16-bit types),
    ids exactly, log probabilities within the binary32 error of a sum of exponentials: a thread adds at most
    ceil(vocab / 4096) * 16 terms, 30 merges follow, each term's exponential and each addition is off by
    2 u, the logarithm turns that into an absolute error; plus 4 u of the value itself."""
    from needle_b200 import native
    g = torch.Generator().manual_seed(rows + vocab)
    x = (3.0 * torch.randn(rows, vocab + pad, generator=g)).to(dtype_of(torch, name))
    x[:, vocab // 2:vocab // 2 + 3] = x[:, :vocab].amax(1, keepdim=True)  # ties of the largest
    if vocab > 100:
        x[0, 40], x[rows - 1, 41] = -math.inf, -math.inf
    d = x.cuda()[:, :vocab]
    rules = make_rules(torch, rows, vocab, rows * 31 + vocab)
    ruled, allowed = rules_reference(x[:, :vocab].float().numpy(), rules)
    a = rules_args(torch, name, d, rules)
    out = torch.full((rows, vocab + pad), 5.0, dtype=d.dtype).cuda()
    native.check(native.lib().needle_cuda_logits_rules_dev(C.byref(a), out.data_ptr(), out.stride(0), stream_of(torch)))
    ids, lps = torch.zeros(rows, dtype=torch.int32).cuda(), torch.zeros(rows).cuda()
    native.check(native.lib().needle_cuda_logits_select_dev(C.byref(a), ids.data_ptr(), lps.data_ptr(), stream_of(torch)))
    torch.cuda.synchronize()
    masked = np.where(allowed, ruled, -np.inf).astype(np.float32)
    want = torch.from_numpy(masked).to(d.dtype)
    assert torch.equal(out[:, :vocab].cpu(), want)
    assert bool((out[:, vocab:] == 5.0).all())
    raw = x[:, :vocab].double()
    log_all = torch.log_softmax(raw, 1)
    terms = -(-vocab // 4096) * 16 + 30
    for r in range(rows):
        if not allowed[r].any():
            assert int(ids[r]) == -1 and float(lps[r]) == -math.inf
            continue
        best = masked[r][allowed[r]].max()
        want_id = int(np.nonzero(allowed[r] & (masked[r] == best))[0][0])
        assert int(ids[r]) == want_id, r
        lp = float(log_all[r, want_id])
        assert float(lps[r]) == lp or abs(float(lps[r]) - lp) <= 2 * terms * U + 4 * U * (abs(lp) + float(raw[r].abs().max() if math.isfinite(float(raw[r].abs().max())) else 20.0)), r


def test_logits_rules_in_place_and_single_rules(torch):
    from needle_b200 import native
    for only in ((), ("history", "history_lengths", "repetition"), ("history", "history_lengths", "frequency"),
                 ("history", "history_lengths", "prompt_lengths", "presence"), ("bias_ids", "bias_values", "bias_counts"),
                 ("masks", "mask_slots")):
        rules = {k: v for k, v in make_rules(torch, 6, 3001, 5).items() if k in only}
        x = torch.randn(6, 3001, generator=torch.Generator().manual_seed(1))
        ruled, allowed = rules_reference(x.numpy(), rules)
        d = x.cuda()
        a = rules_args(torch, "f32", d, rules)
        native.check(native.lib().needle_cuda_logits_rules_dev(C.byref(a), d.data_ptr(), d.stride(0), stream_of(torch)))
        torch.cuda.synchronize()
        np.testing.assert_array_equal(d.cpu().numpy(), np.where(allowed, ruled, -np.inf).astype(np.float32))


def test_logits_rows_whose_last_part_is_empty_in_some(torch):
    """Rows an odd stride apart begin at every place of a 16-byte unit; with parts of 4096 ids (long lists) a row
    of 4096 ids has a second part only where it does not begin on a boundary.  Several rows a CTA."""
    from needle_b200 import native
    rows, v, stride, listed = 700, 4096, 4097, 5000
    g = torch.Generator().manual_seed(3)
    x = torch.randn(rows, stride, generator=g)
    history = torch.randint(0, v, (rows, listed), generator=g, dtype=torch.int32)
    lengths = torch.randint(0, 40, (rows,), generator=g, dtype=torch.int32)
    lengths[5] = listed
    d = x.cuda()
    rules = {"history": history.cuda(), "history_lengths": lengths.cuda(), "frequency": torch.full((rows,), 0.5).cuda(),
             "presence": torch.full((rows,), 0.25).cuda()}
    ruled = x[:, :v].numpy().copy()
    for r in range(rows):
        ids, times = np.unique(history[r, :lengths[r]].numpy(), return_counts=True)
        ruled[r, ids] = ruled[r, ids] - np.float32(0.5) * times.astype(np.float32) - np.float32(0.25)
    a = rules_args(torch, "f32", d[:, :v], rules)
    ids, lps = torch.zeros(rows, dtype=torch.int32).cuda(), torch.zeros(rows).cuda()
    native.check(native.lib().needle_cuda_logits_select_dev(C.byref(a), ids.data_ptr(), lps.data_ptr(), stream_of(torch)))
    out = torch.zeros(rows, v).cuda()
    native.check(native.lib().needle_cuda_logits_rules_dev(C.byref(a), out.data_ptr(), v, stream_of(torch)))
    torch.cuda.synchronize()
    np.testing.assert_array_equal(out.cpu().numpy(), ruled)
    np.testing.assert_array_equal(ids.cpu().numpy(), ruled.argmax(1))


def test_logits_select_odd_values(torch):
    """NaN never wins, -0 ties with +0, a row of -inf takes the lowest allowed id, the type's lowest value is
    a value like any other."""
    from needle_b200 import native
    v = 9000
    x = torch.full((5, v), -1.0)
    x[0, 8500] = math.nan
    x[0, 8600] = 2.0
    x[1, 10], x[1, 20] = 0.0, -0.0
    x[2, 10], x[2, 20] = -0.0, 0.0
    x[3] = -math.inf
    x[4] = torch.finfo(torch.float32).min
    d = x.cuda()
    words = torch.full((1, (v + 31) // 32), -1, dtype=torch.int32)
    words[0, 0] = ~0xff  # ids 0..7 are not allowed
    rules = {"masks": words.cuda(), "mask_slots": torch.zeros(5, dtype=torch.int32).cuda()}
    a = rules_args(torch, "f32", d, rules)
    ids, lps = torch.zeros(5, dtype=torch.int32).cuda(), torch.zeros(5).cuda()
    native.check(native.lib().needle_cuda_logits_select_dev(C.byref(a), ids.data_ptr(), lps.data_ptr(), stream_of(torch)))
    torch.cuda.synchronize()
    assert ids.tolist() == [8600, 10, 10, 8, 8]
    assert math.isnan(float(lps[0]))  # a NaN among the raw logits leaves no probabilities
    assert abs(float(lps[4]) + math.log(v)) <= 1e-5


def test_logits_select_matches_the_engine(torch, oracle):
    """The engine's own masked selection (needle_cuda_step) and the operator choose the same id from the
    same logits, with the same log probability."""
    from needle_b200 import native, synth
    from needle_b200.backend import CudaEngine, StepRequest
    archive = synth.build_archive(0, synth.small_geometry(layers=2, vocab=512), probe_heads=False)
    rng = np.random.default_rng(2)
    with CudaEngine(archive, device=0, max_seqs=3, max_len=32, max_sink=0) as eng:
        allowed = [np.sort(rng.choice(512, 60, replace=False)).astype(np.uint32), None, np.array([5], dtype=np.uint32)]
        for s in range(3):
            eng.reset(s, 16, 0)
        chosen, logits = eng.step([StepRequest(s, 7 + s, True, allowed[s]) for s in range(3)], want_logits=True)
    masks = np.zeros((2, 16), dtype=np.uint32)
    for slot, ids in ((0, allowed[0]), (1, allowed[2])):
        for i in ids:
            masks[slot, i >> 5] |= np.uint32(1 << (i & 31))
    d = torch.from_numpy(logits).cuda()
    rules = {"masks": torch.from_numpy(masks.view(np.int32)).cuda(),
             "mask_slots": torch.tensor([0, -1, 1], dtype=torch.int32).cuda()}
    a = rules_args(torch, "f32", d, rules)
    ids, lps = torch.zeros(3, dtype=torch.int32).cuda(), torch.zeros(3).cuda()
    native.check(native.lib().needle_cuda_logits_select_dev(C.byref(a), ids.data_ptr(), lps.data_ptr(), stream_of(torch)))
    torch.cuda.synchronize()
    assert ids.tolist() == [c[0] for c in chosen]
    assert np.allclose(lps.cpu().numpy(), [c[1] for c in chosen], rtol=0, atol=(2 * 46 + 4 * 20) * U)


# ------------------------------------------------------------------ together, captured, on other streams

def decode_step(torch, s, name="f32"):
    """One step of the loop: append the step's keys and values, attend, choose."""
    from needle_b200 import native
    rope_call(torch, name, s["q"], s["k"], s["v"], s["q_out"], None, None, s["norm"], s["norm"], s["positions"], s["slots"],
              s["entries"], s["cache"], s["heads"], s["kv_heads"], s["dim"], s["dim"], False, s["inverse"], 1.0)
    s["workspace"] = attention_call(torch, name, s["q_out"], s["out"], s["lse"], s["prefix"], s["cache"], s["slots"],
                                    s["counts"], s["heads"], s["kv_heads"], s["dim"], s["prefix_length"],
                                    workspace=s.get("workspace"))
    a = rules_args(torch, name, s["logits"], s["rules"])
    native.check(native.lib().needle_cuda_logits_select_dev(C.byref(a), s["ids"].data_ptr(), s["lps"].data_ptr(), stream_of(torch)))


def decode_state(torch, rows, seed, prefix_length=150, vocab=512):
    g = torch.Generator().manual_seed(seed)
    heads, kv_heads, dim, cap = 8, 4, 64, 24
    s = dict(heads=heads, kv_heads=kv_heads, dim=dim, prefix_length=prefix_length)
    qkv = torch.randn(rows, 1024, generator=g).cuda()
    s["q"], s["k"], s["v"] = qkv.split([512, 256, 256], 1)
    s["qkv"] = qkv
    s["norm"] = (0.1 * torch.randn(dim, generator=g)).cuda()
    s["inverse"] = [10000.0 ** (-2.0 * i / dim) for i in range(dim // 2)]
    s["counts"] = torch.randint(1, cap + 1, (rows,), generator=g, dtype=torch.int32).cuda()
    s["entries"] = s["counts"] - 1
    s["positions"] = prefix_length + s["entries"]
    s["slots"] = torch.randperm(rows, generator=g).int().cuda()
    if rows > 3:
        s["slots"][-1] = -1  # a batch padded to the graph's size
    c = lambda *shape: [t.cuda() for t in (*random_cache(torch, g, *shape), *random_cache(torch, g, *shape))]  # noqa: E731
    s["cache"], s["prefix"] = c(rows, kv_heads, cap, dim), c(kv_heads, prefix_length, dim)
    s["q_out"], s["out"], s["lse"] = torch.zeros(rows, 512).cuda(), torch.zeros(rows, 512).cuda(), torch.zeros(rows, 8).cuda()
    s["logits"] = torch.randn(rows, vocab, generator=g).cuda()
    s["rules"] = make_rules(torch, rows, vocab, seed)
    s["ids"], s["lps"] = torch.zeros(rows, dtype=torch.int32).cuda(), torch.zeros(rows).cuda()
    return s


OUTPUTS = ("q_out", "out", "lse", "ids", "lps")


@pytest.mark.parametrize("rows", [2, 70])
def test_decode_step_together(torch, rows):
    """The operators in a row, as a decode step uses them: the attention reads what the append of the same
    step has stored."""
    s = decode_state(torch, rows, rows)
    decode_step(torch, s)
    torch.cuda.synchronize()
    x = s["qkv"].cpu().numpy()
    angle = s["positions"].cpu().numpy().astype(np.float64)[:, None] * np.array(s["inverse"])
    norm = s["norm"].cpu().numpy()
    key = turned(x[:, 512:768].reshape(rows, 4, 64), norm, angle, 1.0, 64, False)
    codes, scales = quantised(key)
    vcodes, vscales = quantised(x[:, 768:].reshape(rows, 4, 64))
    prefix, cache = [t.cpu() for t in s["prefix"]], [t.cpu() for t in s["cache"]]
    for r in range(rows):
        slot, n = int(s["slots"][r]), int(s["counts"][r])
        if slot < 0:
            assert bool((s["out"][r] == 0).all())
            continue
        np.testing.assert_array_equal(cache[0][slot, :, n - 1].numpy(), codes[r])
        np.testing.assert_array_equal(cache[1][slot, :, n - 1].numpy(), scales[r])
        np.testing.assert_array_equal(cache[2][slot, :, n - 1].numpy(), vcodes[r])
        np.testing.assert_array_equal(cache[3][slot, :, n - 1].numpy(), vscales[r])
        want, want_lse, big, vmax = attention_reference(torch, s["q_out"][r].cpu(), prefix, cache, slot, n, 8, 4, 64,
                                                        s["prefix_length"], 0.125)
        bound = (2 * 72 * big + s["prefix_length"] + n + 32) * U * vmax + U * want.abs()
        assert bool((s["out"][r].double().cpu().view(8, 64) - want).abs().le(bound).all()), r
    ruled, allowed = rules_reference(s["logits"].cpu().numpy(), s["rules"])
    for r in range(rows):
        want_id = int(np.where(allowed[r], ruled[r], -np.inf).argmax()) if allowed[r].any() else -1
        assert int(s["ids"][r]) == want_id


@pytest.mark.parametrize("rows", [2, 70])
def test_decode_step_captured_and_replayed(torch, rows):
    """A captured step gives what the eager one gives, for inputs written after the capture; two graphs
    with a workspace each run at the same time on two streams."""
    states = [decode_state(torch, rows, 50 + i) for i in range(2)]
    fresh = [decode_state(torch, rows, 60 + i) for i in range(2)]
    graphs = []
    for s in states:
        decode_step(torch, s)  # sizes the workspace
    torch.cuda.synchronize()
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            decode_step(torch, s)
        graphs.append(g)
    wanted = []
    for s, f in zip(states, fresh):
        for k in ("qkv", "counts", "entries", "positions", "slots", "logits"):
            s[k].copy_(f[k])
        for k in ("cache", "prefix"):
            for a, b in zip(s[k], f[k]):
                a.copy_(b)
        for k in f["rules"]:
            s["rules"][k].copy_(f["rules"][k])
        for k in OUTPUTS:
            s[k].zero_()
        f["norm"].copy_(s["norm"])
        decode_step(torch, f)
        wanted.append([f[k].clone() for k in OUTPUTS] + [t.clone() for t in f["cache"]])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, w in zip(states, wanted):
        for a, b in zip([s[k] for k in OUTPUTS] + s["cache"], w):
            assert torch.equal(a, b)


def test_dense_prefix_captured_and_replayed_beside_each_other(torch):
    """Steps whose prefix is long enough for the dense product: two graphs at the same time on two streams,
    and an eager step between them, give what each gives alone."""
    states = [decode_state(torch, 70, 80 + i, prefix_length=700) for i in range(3)]
    wanted = []
    for s in states:
        decode_step(torch, s)
        torch.cuda.synchronize()
        wanted.append([s[k].clone() for k in OUTPUTS])
    graphs = []
    for s in states[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            decode_step(torch, s)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in states:
        for k in OUTPUTS:
            s[k].zero_()
    torch.cuda.synchronize()
    for _ in range(4):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            decode_step(torch, states[2])
    torch.cuda.synchronize()
    for s, w in zip(states, wanted):
        assert all(torch.equal(a, s[k]) for a, k in zip(w, OUTPUTS))


def test_first_calls_of_a_process_captured(torch):
    """The operators' first calls in a process may be captured ones."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = """
import torch, sys
sys.path[:0] = sys.argv[1:]
import __graft_entry__ as entry
entry.load()
import test_gpu_serving_ops as t
s = t.decode_state(torch, 70, 4, prefix_length=700)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    t.decode_step(torch, s)
g.replay()
torch.cuda.synchronize()
first = [s[k].clone() for k in t.OUTPUTS]
t.decode_step(torch, s)
torch.cuda.synchronize()
assert all(torch.equal(a, s[k]) for a, k in zip(first, t.OUTPUTS))
print("captured first")
"""
    done = subprocess.run([sys.executable, "-c", code, os.path.dirname(here), here], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured first" in done.stdout, done.stderr[-2000:]


def test_same_results_every_time(torch):
    """No result depends on the order in which blocks run."""
    s = decode_state(torch, 70, 9, prefix_length=700)
    decode_step(torch, s)
    first = [s[k].clone() for k in OUTPUTS]
    for _ in range(5):
        s["workspace"].fill_(0xff)
        decode_step(torch, s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, s[k]) for a, k in zip(first, OUTPUTS))


def test_host_buffers_are_refused(torch):
    from needle_b200 import native
    x, out = torch.zeros(2, 64), torch.zeros(2, 64).cuda()
    for a, o in ((rules_args(torch, "f32", x, {}), out), (rules_args(torch, "f32", out, {}), x)):
        with pytest.raises(native.NeedleError) as e:
            native.check(native.lib().needle_cuda_logits_rules_dev(C.byref(a), o.data_ptr(), 64, None))
        assert e.value.code == "BACKEND_UNAVAILABLE" and "not device memory" in str(e.value)
    torch.cuda.synchronize()


def test_host_lists_are_refused(torch):
    """A list in host memory is refused before anything is launched, whichever it is."""
    from needle_b200 import native
    s = decode_state(torch, 4, 3, prefix_length=100)
    decode_step(torch, s)
    torch.cuda.synchronize()
    for name in ("positions", "slots", "entries", "norm"):
        with pytest.raises(native.NeedleError, match="not device memory"):
            decode_step(torch, {**s, name: s[name].cpu()})
    for name in ("counts", "slots"):
        bad = {**s, name: s[name].cpu()}
        with pytest.raises(native.NeedleError, match=name + " is not device memory"):
            attention_call(torch, "f32", s["q_out"], s["out"], s["lse"], s["prefix"], s["cache"], bad["slots"], bad["counts"],
                           8, 4, 64, 100, workspace=s["workspace"])
    for name in s["rules"]:
        rules = {**s["rules"], name: s["rules"][name].cpu()}
        a = rules_args(torch, "f32", s["logits"], rules)
        with pytest.raises(native.NeedleError, match=name + " is not device memory"):
            native.check(native.lib().needle_cuda_logits_select_dev(C.byref(a), s["ids"].data_ptr(), s["lps"].data_ptr(),
                                                                    stream_of(torch)))
    torch.cuda.synchronize()


def test_calls_from_two_threads_at_once(torch):
    """Two host threads, each with its own stream and buffers and calls of different sizes, get what one gets."""
    import threading
    states = [[decode_state(torch, rows, seed, prefix_length=p, vocab=v) for rows, seed, p, v in sizes]
              for sizes in (((2, 1, 100, 512), (70, 2, 700, 9000)), ((33, 3, 2000, 3001), (5, 4, 37, 20000)))]
    wanted = []
    for mine in states:
        for s in mine:
            decode_step(torch, s)
            torch.cuda.synchronize()
            wanted.append([s[k].clone() for k in OUTPUTS])
            for k in OUTPUTS:
                s[k].zero_()
    torch.cuda.synchronize()
    failures = []

    def work(mine):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    for s in mine:
                        decode_step(torch, s)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(mine,)) for mine in states]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    for s, w in zip([s for mine in states for s in mine], wanted):
        assert all(torch.equal(a, s[k]) for a, k in zip(w, OUTPUTS))


def test_offsets_past_32_bits(torch):
    """Caches and rows of logits whose elements lie more than 2^32 from the first: what a small copy of the same
    gives.  (Only what is read is written first.)"""
    from needle_b200 import native
    g = torch.Generator().manual_seed(8)
    heads, kv, dim, cap, n = 16, 8, 128, 1 << 21, 40
    small = [t.cuda() for t in (*random_cache(torch, g, 1, kv, n, dim), *random_cache(torch, g, 1, kv, n, dim))]
    large = [torch.empty(3, kv, cap, dim, dtype=torch.int8, device="cuda") if t.dim() == 4 else
             torch.empty(3, kv, cap, device="cuda") for t in small]
    assert large[0][2].data_ptr() - large[0].data_ptr() >= 1 << 32
    for a, b in zip(large, small):
        a[2, :, :n] = b[0]
    x = torch.randn(1, (heads + 2 * kv) * dim, generator=g).cuda()
    q, k, v = x.split([heads * dim, kv * dim, kv * dim], 1)
    inverse = [10000.0 ** (-2.0 * i / dim) for i in range(dim // 2)]
    at = lambda i: torch.tensor([i], dtype=torch.int32).cuda()  # noqa: E731
    results = []
    for cache, slot in ((small, 0), (large, 2)):
        q_out, out, lse = torch.zeros(1, heads * dim).cuda(), torch.zeros(1, heads * dim).cuda(), torch.zeros(1, heads).cuda()
        rope_call(torch, "f32", q, k, v, q_out, None, None, None, None, at(n - 1), at(slot), at(n - 1), cache, heads, kv, dim,
                  dim, False, inverse, 1.0)
        attention_call(torch, "f32", q_out, out, lse, [None] * 4, cache, at(slot), at(n), heads, kv, dim, 0)
        results.append((out, lse))
    rope_call(torch, "f32", q, k, v, torch.zeros_like(q_out), None, None, None, None, at(n - 1), at(2), at(cap - 1), large, heads,
              kv, dim, dim, False, inverse, 1.0)
    torch.cuda.synchronize()
    for a, b in zip(large, small):
        assert torch.equal(a[2, :, :n], b[0]) and torch.equal(a[2, :, cap - 1], b[0, :, n - 1])
    assert all(torch.allclose(a, b, rtol=0, atol=64 * U * float(a.abs().max())) for a, b in zip(*results))
    del large
    rows, vocab, stride = 3, 5000, (1 << 31) + 8
    logits = torch.randn(rows, vocab, generator=g).half().cuda()
    far = torch.empty(rows * stride, dtype=torch.float16, device="cuda").view(rows, stride)
    far[:, :vocab] = logits
    rules = make_rules(torch, rows, vocab, 4)
    chosen, outs = [], []
    for d in (logits, far[:, :vocab]):
        a = rules_args(torch, "f16", d, rules)
        ids, lps = torch.zeros(rows, dtype=torch.int32).cuda(), torch.zeros(rows).cuda()
        native.check(native.lib().needle_cuda_logits_select_dev(C.byref(a), ids.data_ptr(), lps.data_ptr(), stream_of(torch)))
        native.check(native.lib().needle_cuda_logits_rules_dev(C.byref(a), d.data_ptr(), d.stride(0), stream_of(torch)))
        torch.cuda.synchronize()
        chosen.append((ids, lps))
        outs.append(d)
    assert torch.equal(chosen[0][0], chosen[1][0]) and torch.equal(chosen[0][1], chosen[1][1])
    assert torch.equal(*outs)
