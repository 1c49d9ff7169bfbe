"""Measured cases of the serving operators: rope_append, prefix_attention, logits_rules and
logits_select, each with its plain form in elementary torch operations and its definition in 64 bits.

A decode step of a batch whose sequences share a prompt prefix goes through them in this order:
rope_append norms and rotates the step's queries and keys and appends keys and values to each
sequence's int8 cache; prefix_attention attends over the shared prefix and the sequence's own cache;
logits_rules / logits_select apply penalties, biases and grammar masks to the vocabulary's logits.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def listed():
    return [
        # one step of four concurrent sequences of the engine's geometry (latency)
        dict(name="rope decode 4", op="rope", type="f32", tokens=4, heads=8, kv_heads=4, dim=64, rotary=64,
             interleaved=False, norm=True, scaling="plain", capacity=416, base=0, values=False),
        # one step of the engine's largest batch
        dict(name="rope decode 4096", op="rope", type="f32", tokens=4096, heads=8, kv_heads=4, dim=64, rotary=64,
             interleaved=False, norm=True, scaling="plain", capacity=64, base=256, values=True),
        # a long prompt read at once, positions far past the trained length, half of each head rotated
        dict(name="rope prompt 8191", op="rope", type="bf16", tokens=8191, heads=32, kv_heads=8, dim=128, rotary=64,
             interleaved=True, norm=False, scaling="parts", capacity=8192, base=100000, values=True),
        # one tool call over the engine's longest sink (latency)
        dict(name="attend 1 x 160", op="attend", type="f32", rows=1, heads=8, kv_heads=4, dim=64, prefix=160, own=256, pad=0),
        # a serving batch over the longest prompt the engine's positions allow
        dict(name="attend 64 x 2048", op="attend", type="f32", rows=64, heads=8, kv_heads=4, dim=64, prefix=2048, own=256, pad=0),
        # the engine's largest batch: the caches of 4096 sequences behind one sink
        dict(name="attend 4096 x 160", op="attend", type="f32", rows=4096, heads=8, kv_heads=4, dim=64, prefix=160, own=256, pad=0),
        # a long shared document, wider heads, a batch padded to a graph's size
        dict(name="attend 333 x 8191", op="attend", type="bf16", rows=333, heads=32, kv_heads=8, dim=128, prefix=8191, own=500, pad=13),
        # logits of a few sequences whose user samples afterwards (latency)
        dict(name="rules 4 x 8192", op="rules", type="f32", rows=4, vocab=8192, history=100, biases=8, masked=True),
        # a serving batch with an odd, larger vocabulary
        dict(name="rules 512 x 50001", op="rules", type="bf16", rows=512, vocab=50001, history=1000, biases=50, masked=True),
        # greedy choice of one sequence (latency)
        dict(name="select 1 x 8192", op="select", type="f32", rows=1, vocab=8192, history=64, biases=0, masked=True),
        # constrained choice of the engine's largest batch
        dict(name="select 4096 x 8192", op="select", type="f32", rows=4096, vocab=8192, history=256, biases=4, masked=True),
        # large vocabulary, half precision logits, long histories
        dict(name="select 200 x 128000", op="select", type="f16", rows=200, vocab=128000, history=2000, biases=100, masked=False),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "attend", "rules", "select"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op in ("rope", "attend"):
        dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    if op == "rope":
        most = max(2, min(8191, 8191 * 48 * 128 // ((heads + 2 * kv_heads) * dim * SIZES[kind] // 2)))
        return dict(op=op, type=kind, tokens=_spread(rng, 1, most), heads=heads, kv_heads=kv_heads, dim=dim,
                    rotary=rng.choice([2, dim // 4, dim // 2, dim]), interleaved=rng.random() < 0.5,
                    norm=rng.random() < 0.5, scaling=rng.choice(["plain", "linear", "ntk", "parts"]),
                    capacity=rng.randint(40, 300), base=_spread(rng, 1, 120000), values=rng.random() < 0.5)
    if op == "attend":
        prefix, most_own = _spread(rng, 16, 16384), _spread(rng, 1, 700)
        cap = min(4096, int(333 * 32 * 128 * 8191 / (heads * dim * prefix)), int(4096 * 4 * 64 * 256 / (kv_heads * dim * most_own)))
        rows = _spread(rng, 1, max(2, cap))
        return dict(op=op, type=kind, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, prefix=prefix,
                    own=most_own, pad=min(rows - 1, rng.choice([0, 0, 1, 5])))
    vocab = _spread(rng, 400, 130000)
    rows = _spread(rng, 1, max(2, min(4096, 25_000_000 // vocab)))
    return dict(op=op, type=kind, rows=rows, vocab=vocab, history=_spread(rng, 1, 4000 if rows < 500 else 500),
                biases=rng.choice([0, 1, 30, 300]), masked=rng.random() < 0.6)


# ------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _whole(g, low, high, *shape):
    return torch.randint(low, high, shape, generator=g, device="cuda", dtype=torch.int32)


def _frequencies(case):
    """The inverse frequency of each rotated pair in binary64 and the magnitude of the rotation."""
    n, theta = case["rotary"] // 2, 10000.0
    plain = [theta ** (-2.0 * i / case["rotary"]) for i in range(n)]
    factor, trained = 16.0, 8192.0
    if case["scaling"] == "linear":
        return [f / factor for f in plain], 1.0
    if case["scaling"] == "ntk":
        stretched = theta * factor ** (case["rotary"] / max(1.0, case["rotary"] - 2.0))
        return [stretched ** (-2.0 * i / case["rotary"]) for i in range(n)], 1.0
    if case["scaling"] == "parts":  # by parts: turns over the trained length decide (32 and more: kept, 1 and less: interpolated)
        turns = [trained * f / (2 * math.pi) for f in plain]
        keep = [min(1.0, max(0.0, (t - 1.0) / 31.0)) for t in turns]
        return [f * k + f / factor * (1 - k) for f, k in zip(plain, keep)], 0.1 * math.log(factor) + 1.0
    return plain, 1.0


def _cache(g, *shape):
    """int8 codes [..., dim] of normal rows with one scale per row, magnitudes as in a cache in use."""
    x = _normal(g, *shape)
    top = x.abs().amax(-1, keepdim=True)
    codes = (x * (127.0 / top)).round_().to(torch.int8)
    return codes, (top[..., 0] / 127.0).contiguous()


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case=case)
    if case["op"] == "rope":
        t, h, k, d, dtype = case["tokens"], case["heads"], case["kv_heads"], case["dim"], TYPES[case["type"]]
        slots = max(1, min(t, 4096)) if case["capacity"] < 8192 else 1
        # the fused projection's output: queries, keys and values of a token side by side
        s["qkv"] = _normal(g, t, (h + 2 * k) * d).to(dtype)
        s["q"], s["k"], s["v"] = s["qkv"].split([h * d, k * d, k * d], dim=1)
        s["q_norm"] = 0.1 * _normal(g, d) if case["norm"] else None
        s["k_norm"] = 0.1 * _normal(g, d) if case["norm"] else None
        # every token has an entry of its own; the last one of a longer batch is padding and not stored
        order = torch.randperm(slots * case["capacity"], generator=g, device="cuda")[:t]
        s["slots"] = (order // case["capacity"]).to(torch.int32)
        s["entries"] = (order % case["capacity"]).to(torch.int32)
        if t > 4:
            s["slots"][-1] = -1
        s["positions"] = (case["base"] + _whole(g, 0, 2 * case["capacity"], t)).to(torch.int32)
        shape = (slots, k, case["capacity"])
        s["key_codes"] = torch.zeros(*shape, d, dtype=torch.int8, device="cuda")
        s["value_codes"] = torch.zeros(*shape, d, dtype=torch.int8, device="cuda")
        s["key_scales"] = torch.zeros(*shape, device="cuda")
        s["value_scales"] = torch.zeros(*shape, device="cuda")
        s["q_out"] = torch.zeros(t, h * d, dtype=dtype, device="cuda")
        s["k_out"] = torch.zeros(t, k * d, dtype=dtype, device="cuda") if case["values"] else None
        s["v_out"] = torch.zeros(t, k * d, dtype=dtype, device="cuda") if case["values"] else None
        s["frequencies"], s["magnitude"] = _frequencies(case)
        s["inverse"] = torch.tensor(s["frequencies"], dtype=torch.float64, device="cuda")
    elif case["op"] == "attend":
        r, h, k, d, dtype = case["rows"], case["heads"], case["kv_heads"], case["dim"], TYPES[case["type"]]
        s["q"] = (1.5 * _normal(g, r, h * d)).to(dtype)
        s["prefix_key_codes"], s["prefix_key_scales"] = _cache(g, k, case["prefix"], d)
        s["prefix_value_codes"], s["prefix_value_scales"] = _cache(g, k, case["prefix"], d)
        s["key_codes"], s["key_scales"] = _cache(g, r, k, case["own"], d)
        s["value_codes"], s["value_scales"] = _cache(g, r, k, case["own"], d)
        # sequences of every age, the first just admitted (nothing of its own yet), in slots of any order
        s["counts"] = _whole(g, 0, case["own"] + 1, r)
        s["counts"][0] = 0
        s["slots"] = torch.randperm(r, generator=g, device="cuda").to(torch.int32)
        if case["pad"]:
            s["slots"][r - case["pad"]:] = -1
        s["out"] = torch.zeros(r, h * d, dtype=dtype, device="cuda")
        s["lse"] = torch.zeros(r, h, device="cuda")
    else:
        r, v, n = case["rows"], case["vocab"], case["history"]
        s["logits"] = (3.0 * _normal(g, r, v)).to(TYPES[case["type"]])
        # a text repeats itself: ids crowd at the start of the vocabulary
        s["history"] = (torch.rand(r, n, generator=g, device="cuda") ** 3 * v).to(torch.int32)
        s["history_lengths"] = _whole(g, 0, n + 1, r)
        s["prompt_lengths"] = (s["history_lengths"] * torch.rand(r, generator=g, device="cuda")).to(torch.int32)
        s["repetition"] = 1.0 + 0.3 * torch.rand(r, generator=g, device="cuda")
        s["presence"] = 0.6 * torch.rand(r, generator=g, device="cuda")
        s["frequency"] = 0.4 * torch.rand(r, generator=g, device="cuda")
        b = min(case["biases"], v)
        if b:  # ids without repeats, from a random start
            start = _whole(g, 0, v, r, 1).long()  # ids a fixed step apart
            s["bias_ids"] = ((start + torch.arange(b, device="cuda") * max(1, v // b)) % v).to(torch.int32)
            s["bias_values"] = 4.0 * _normal(g, r, b)
            s["bias_counts"] = _whole(g, 0, b + 1, r)
        if case["masked"]:
            slots, words = min(r, 64), (v + 31) // 32
            bits = torch.randint(0, 2 ** 31, (slots, words), generator=g, device="cuda", dtype=torch.int32)
            # half of the grammar states allow few ids, half allow most of the vocabulary
            few = bits & bits.roll(1, 1) & bits.roll(2, 1) & bits.roll(3, 1) & bits.roll(5, 1)
            narrow = torch.arange(slots, device="cuda")[:, None] % 2 == 0
            s["masks"] = torch.where(narrow, few, bits | bits.roll(1, 1))
            s["mask_slots"] = _whole(g, -1, slots, r)  # -1: not constrained
        if case["op"] == "rules":
            s["out"] = torch.zeros(r, v, dtype=TYPES[case["type"]], device="cuda")
        else:
            s["ids"] = torch.zeros(r, dtype=torch.int32, device="cuda")
            s["log_probabilities"] = torch.zeros(r, device="cuda")
    return s


# ------------------------------------------------------------------ plain forms

def _rotate(x, scale, cos, sin, case):
    """x [T, n, D] in binary64: the norm, then the rotation of the first `rotary` dimensions, each stored
    in binary32 as the engine stores them (codes next to a rounding border depend on it)."""
    if scale is not None:
        inverse = 1.0 / ((x * x).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt()
        x = ((1.0 + scale.double()) * x * inverse).float().double()
    part, rest = x[..., :case["rotary"]], x[..., case["rotary"]:]
    if case["interleaved"]:
        first, second = part[..., 0::2], part[..., 1::2]
    else:
        first, second = part.chunk(2, -1)
    a, b = first * cos - second * sin, second * cos + first * sin
    turned = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turned, rest), -1).float()


def _quantise(x):
    x = x.double()
    scale = x.abs().amax(-1).clamp_min(1e-12) / 127.0
    return (x / scale[..., None]).round().to(torch.int8), scale.float()


def _plain_rope(s):
    c = s["case"]
    t, h, k, d, dtype = c["tokens"], c["heads"], c["kv_heads"], c["dim"], TYPES[c["type"]]
    angle = s["positions"].double()[:, None, None] * s["inverse"]
    cos, sin = angle.cos() * s["magnitude"], angle.sin() * s["magnitude"]
    q = _rotate(s["q"].double().view(t, h, d), s["q_norm"], cos, sin, c)
    key = _rotate(s["k"].double().view(t, k, d), s["k_norm"], cos, sin, c)
    key_codes, key_scales = _quantise(key)
    value_codes, value_scales = _quantise(s["v"].float().view(t, k, d))
    s["q_out"].copy_(q.view(t, h * d))
    at = (s["slots"] >= 0).nonzero()[:, 0] if t > 4 else torch.arange(t, device="cuda")
    slot, entry = s["slots"][at].long(), s["entries"][at].long()
    s["key_codes"][slot, :, entry] = key_codes[at]
    s["value_codes"][slot, :, entry] = value_codes[at]
    s["key_scales"][slot, :, entry] = key_scales[at]
    s["value_scales"][slot, :, entry] = value_scales[at]
    if c["values"]:
        s["k_out"].copy_((key_codes * key_scales[..., None]).view(t, k * d))
        s["v_out"].copy_((value_codes * value_scales[..., None]).view(t, k * d))
    return _rope_outputs(s)


def _rope_outputs(s):
    return [s["q_out"], s["k_out"], s["v_out"], s["key_codes"], s["value_codes"], s["key_scales"], s["value_scales"]]


def _plain_attend(s):
    c = s["case"]
    r, h, k, d = c["rows"], c["heads"], c["kv_heads"], c["dim"]
    live = s["slots"] >= 0
    slot = s["slots"].clamp_min(0).long()
    q = s["q"].float().view(r, k, h // k, d) * (1.0 / math.sqrt(d))
    prefix_keys = s["prefix_key_codes"] * s["prefix_key_scales"][..., None]
    prefix_values = s["prefix_value_codes"] * s["prefix_value_scales"][..., None]
    keys = s["key_codes"][slot] * s["key_scales"][slot][..., None]
    values = s["value_codes"][slot] * s["value_scales"][slot][..., None]
    far = torch.einsum("rkgd,kpd->rkgp", q, prefix_keys)
    near = torch.matmul(q, keys.transpose(2, 3))
    hidden = torch.arange(c["own"], device="cuda") >= s["counts"][:, None]
    near = near.masked_fill(hidden[:, None, None], -math.inf)
    top = torch.maximum(far.amax(-1), near.amax(-1))[..., None]
    far, near = (far - top).exp(), (near - top).exp()
    total = far.sum(-1) + near.sum(-1)
    mixed = torch.einsum("rkgp,kpd->rkgd", far, prefix_values) + torch.matmul(near, values)
    out = (mixed / total[..., None]).reshape(r, h * d).to(s["out"].dtype)
    lse = (top[..., 0] + total.log()).reshape(r, h)
    return [torch.where(live[:, None], out, s["out"]), torch.where(live[:, None], lse, s["lse"])]


def _plain_processed(s):
    """The logits after penalties, biases and masks, in binary32, and which ids the mask leaves."""
    c = s["case"]
    r, v = c["rows"], c["vocab"]
    x = s["logits"].float()
    at = torch.arange(c["history"], device="cuda")
    inside = at < s["history_lengths"][:, None]
    answered = inside & (at >= s["prompt_lengths"][:, None])
    ids = s["history"].long()
    seen = torch.zeros(r, v, device="cuda").scatter_add_(1, ids, inside.float()) > 0
    count = torch.zeros(r, v, device="cuda").scatter_add_(1, ids, answered.float())
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count
    x = x - torch.where(count > 0, s["presence"][:, None], 0.0)
    if "bias_ids" in s:
        kept = torch.arange(s["bias_ids"].shape[1], device="cuda") < s["bias_counts"][:, None]
        x = x.scatter_add(1, s["bias_ids"].long(), torch.where(kept, s["bias_values"], 0.0))
    allowed = torch.ones(r, v, dtype=torch.bool, device="cuda")
    if c["masked"]:
        token = torch.arange(v, device="cuda")
        word = s["masks"][s["mask_slots"].clamp_min(0).long()][:, token >> 5]
        allowed = ((word >> (token & 31)) & 1 > 0) | (s["mask_slots"] < 0)[:, None]
    return x, allowed


def _plain_rules(s):
    x, allowed = _plain_processed(s)
    s["out"].copy_(x.masked_fill(~allowed, -math.inf))
    return s["out"]


def _plain_select(s):
    x, allowed = _plain_processed(s)
    x = x.masked_fill(~allowed, -math.inf)
    v = s["case"]["vocab"]
    token = torch.arange(v, device="cuda", dtype=torch.int32)
    best = (allowed & (x == x.amax(1, keepdim=True)))
    ids = torch.where(best, token, v).amin(1)
    ids = torch.where(ids < v, ids, -1)
    raw = s["logits"].float()
    top = raw.amax(1)
    total = (raw - top[:, None]).exp().sum(1)
    chosen = raw.gather(1, ids.clamp_min(0).long()[:, None])[:, 0]
    log_probabilities = torch.where(ids >= 0, (chosen - top) - total.log(), -math.inf)
    return [ids, log_probabilities]


# ------------------------------------------------------------------ the framework's calls

def _native():
    import __graft_entry__
    __graft_entry__.load()
    from needle_b200 import native
    return native


def _pointer(t):
    return None if t is None else t.data_ptr()


def _kind(native, case):
    return {"f32": native.TYPE_F32, "f16": native.TYPE_F16, "bf16": native.TYPE_BF16}[case["type"]]


def _own_rope(s, native, ctypes, stream):
    c = s["case"]
    args = native.RopeAppend(
        s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["q_out"].data_ptr(), _pointer(s["k_out"]),
        _pointer(s["v_out"]), s["q"].stride(0), s["k"].stride(0), s["v"].stride(0), s["q_out"].stride(0),
        c["kv_heads"] * c["dim"], c["kv_heads"] * c["dim"], _pointer(s["q_norm"]), _pointer(s["k_norm"]),
        s["positions"].data_ptr(), s["slots"].data_ptr(), s["entries"].data_ptr(), s["key_codes"].data_ptr(),
        s["key_scales"].data_ptr(), s["value_codes"].data_ptr(), s["value_scales"].data_ptr(),
        s["magnitude"], _kind(native, c), c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["rotary"],
        int(c["interleaved"]), s["key_codes"].shape[0], c["capacity"])
    inverse = (ctypes.c_double * (c["rotary"] // 2))(*s["frequencies"])
    native.check(native.lib().needle_cuda_rope_append_dev(ctypes.byref(args), inverse, stream))
    return _rope_outputs(s)


def _own_attend(s, native, ctypes, stream):
    c = s["case"]
    args = native.PrefixAttention(
        s["q"].data_ptr(), s["out"].data_ptr(), s["lse"].data_ptr(), s["q"].stride(0), s["out"].stride(0),
        s["prefix_key_codes"].data_ptr(), s["prefix_key_scales"].data_ptr(), s["prefix_value_codes"].data_ptr(),
        s["prefix_value_scales"].data_ptr(), s["key_codes"].data_ptr(), s["key_scales"].data_ptr(),
        s["value_codes"].data_ptr(), s["value_scales"].data_ptr(), s["slots"].data_ptr(), s["counts"].data_ptr(),
        0.0, _kind(native, c), c["rows"], c["heads"], c["kv_heads"], c["dim"], c["prefix"], c["prefix"],
        s["key_codes"].shape[0], c["own"])
    if "workspace" not in s:  # kept by the caller from step to step
        size = ctypes.c_size_t()
        native.check(native.lib().needle_cuda_prefix_attention_workspace(ctypes.byref(args), ctypes.byref(size)))
        s["workspace"] = torch.empty(max(16, size.value), dtype=torch.uint8, device="cuda")
    native.check(native.lib().needle_cuda_prefix_attention_dev(
        ctypes.byref(args), s["workspace"].data_ptr(), s["workspace"].numel(), stream))
    return [s["out"], s["lse"]]


def _own_logits(s, native, ctypes, stream):
    c = s["case"]
    args = native.LogitsRules(
        s["logits"].data_ptr(), s["logits"].stride(0), s["history"].data_ptr(), s["history"].stride(0),
        s["history_lengths"].data_ptr(), s["prompt_lengths"].data_ptr(), s["repetition"].data_ptr(),
        s["presence"].data_ptr(), s["frequency"].data_ptr(), _pointer(s.get("bias_ids")),
        _pointer(s.get("bias_values")), s["bias_ids"].stride(0) if "bias_ids" in s else 0,
        _pointer(s.get("bias_counts")), _pointer(s.get("masks")), _pointer(s.get("mask_slots")),
        s["masks"].shape[0] if c["masked"] else 0, _kind(native, c), c["rows"], c["vocab"])
    if c["op"] == "rules":
        native.check(native.lib().needle_cuda_logits_rules_dev(
            ctypes.byref(args), s["out"].data_ptr(), s["out"].stride(0), stream))
        return s["out"]
    native.check(native.lib().needle_cuda_logits_select_dev(
        ctypes.byref(args), s["ids"].data_ptr(), s["log_probabilities"].data_ptr(), stream))
    return [s["ids"], s["log_probabilities"]]


def run(state):
    op = state["case"]["op"]
    if own:
        import ctypes
        call = {"rope": _own_rope, "attend": _own_attend, "rules": _own_logits, "select": _own_logits}[op]
        return call(state, _native(), ctypes, torch.cuda.current_stream().cuda_stream)
    return {"rope": _plain_rope, "attend": _plain_attend, "rules": _plain_rules, "select": _plain_select}[op](state)


# ------------------------------------------------------------------ work

def work(case):
    if case["op"] == "rope":
        t, h, k, d, e = case["tokens"], case["heads"], case["kv_heads"], case["dim"], SIZES[case["type"]]
        moved = t * (2 * h + 2 * k) * d * e + t * k * (2 * d + 8) + 12 * t
        if case["values"]:
            moved += 2 * t * k * d * e
        return {"bytes": moved, "flops": t * (h + k) * (3 * case["rotary"] + (4 * d if case["norm"] else 0)) + 4 * t * k * d}
    if case["op"] == "attend":
        live, h, k, d = case["rows"] - case["pad"], case["heads"], case["kv_heads"], case["dim"]
        seen = live * case["own"] / 2  # counts are uniform in 0 .. own
        row = 2 * d + 8
        return {"bytes": k * case["prefix"] * row + k * seen * row + 2 * live * h * d * SIZES[case["type"]] + live * h * 4,
                "flops": 4 * h * d * (live * case["prefix"] + seen)}
    r, v, e = case["rows"], case["vocab"], SIZES[case["type"]]
    moved = r * v * e * (2 if case["op"] == "rules" else 1) + r * (2 * case["history"] + 4 * case["biases"] + 24)
    if case["masked"]:
        moved += min(r, 64) * ((v + 31) // 32) * 4
    return {"bytes": moved, "flops": r * v * (1 if case["op"] == "rules" else 3)}


# ------------------------------------------------------------------ definitions in 64 bits

def _exact_turn(x, scale, position, case, frequencies, magnitude):
    """One head's rows x [T, D] (binary64), pair by pair as complex numbers."""
    if scale is not None:
        x = x * (1.0 + scale.double()) / torch.sqrt(torch.linalg.vecdot(x, x)[:, None] / x.shape[1] + EPS)
        x = x.float().double()  # stored in binary32 between norm and rotation, by definition
    half = case["rotary"] // 2
    y = x.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
        turn = torch.polar(torch.full_like(position, magnitude), position * frequencies[i])
        z = torch.complex(x[:, a], x[:, b]) * turn
        y[:, a], y[:, b] = z.real, z.imag
    return y


def _exact_rope(case, s):
    t, h, k, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    position = s["positions"].double()
    q = s["q"].double().view(t, h, d)
    q = torch.stack([_exact_turn(q[:, i], s["q_norm"], position, case, s["frequencies"], s["magnitude"]) for i in range(h)], 1)
    stored = s["slots"] >= 0
    slot, entry = s["slots"][stored].long(), s["entries"][stored].long()
    outs, scales = [], []
    for name, norm in (("k", "k_norm"), ("v", None)):
        x = s[name].double().view(t, k, d)
        whole = torch.zeros_like(s["key_scales"], dtype=torch.float64)
        values = []
        for i in range(k):
            y = x[:, i] if norm is None else _exact_turn(x[:, i], s[norm], position, case, s["frequencies"], s["magnitude"])
            y = y.float().double()  # quantised from its binary32 value, by definition
            step = torch.clamp(torch.amax(torch.abs(y), 1), min=1e-12) / 127.0
            values.append(torch.round(y / step[:, None]) * step[:, None])
            whole[slot, i, entry] = step[stored]
        outs.append(torch.stack(values, 1).reshape(t, k * d) if case["values"] else None)
        scales.append(whole)
    return [q.reshape(t, h * d), outs[0], outs[1], None, None, scales[0], scales[1]]


def _exact_attend(case, s):
    r, h, k, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    group = h // k
    out = torch.zeros(r, h, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(r, h, dtype=torch.float64, device="cuda")
    live = (s["slots"] >= 0).nonzero()[:, 0]
    step = max(1, 200_000_000 // (group * (case["prefix"] + case["own"]) + 2 * case["own"] * d) // 8)
    for i in range(k):
        keys = s["prefix_key_codes"][i].double() * s["prefix_key_scales"][i].double()[:, None]
        values = s["prefix_value_codes"][i].double() * s["prefix_value_scales"][i].double()[:, None]
        for rows in live.split(step):
            slot = s["slots"][rows].long()
            q = s["q"][rows].double().view(-1, h, d)[:, i * group:(i + 1) * group] / d ** 0.5
            own_keys = s["key_codes"][slot, i].double() * s["key_scales"][slot, i].double()[..., None]
            own_values = s["value_codes"][slot, i].double() * s["value_scales"][slot, i].double()[..., None]
            scores = torch.cat((q @ keys.T, q @ own_keys.transpose(1, 2)), -1)
            at = torch.arange(scores.shape[-1], device="cuda") - case["prefix"]
            scores = torch.where(at < s["counts"][rows][:, None, None], scores, -math.inf)
            weights = torch.softmax(scores, -1)
            out[rows, i * group:(i + 1) * group] = weights[..., :case["prefix"]] @ values + weights[..., case["prefix"]:] @ own_values
            lse[rows, i * group:(i + 1) * group] = torch.logsumexp(scores, -1)
    return [out.view(r, h * d), lse]


def _exact_logits(case, s):
    r, v = case["rows"], case["vocab"]
    raw = s["logits"].double()
    length, prompt = s["history_lengths"].tolist(), s["prompt_lengths"].tolist()
    biased = s["bias_counts"].tolist() if "bias_ids" in s else [0] * r
    slot = s["mask_slots"].tolist() if case["masked"] else [-1] * r
    ids, chances = torch.full((r,), -1, device="cuda"), torch.full((r,), -math.inf, dtype=torch.float64, device="cuda")
    out = raw.clone()
    bit = torch.arange(32, device="cuda")
    for i in range(r):
        x = out[i]
        rep = s["repetition"][i].double()
        past = s["history"][i, :length[i]].long().unique()
        x[past] = torch.where(x[past] > 0, x[past] / rep, x[past] * rep)
        answered, times = s["history"][i, prompt[i]:length[i]].long().unique(return_counts=True)
        x[answered] -= s["frequency"][i].double() * times + s["presence"][i].double()
        if biased[i]:
            x[s["bias_ids"][i, :biased[i]].long()] += s["bias_values"][i, :biased[i]].double()
        if slot[i] >= 0:
            x[((s["masks"][slot[i]][:, None] >> bit) & 1).flatten()[:v] == 0] = -math.inf
    if case["op"] == "rules":
        return out
    best = out.amax(1)
    some = best > -math.inf
    ids = torch.where(some, (out == best[:, None]).to(torch.int8).argmax(1), ids)
    log_all = torch.log_softmax(raw, 1).gather(1, ids.clamp_min(0)[:, None])[:, 0]
    return [None, torch.where(some, log_all, chances)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, s)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    return _exact_logits(case, s)
