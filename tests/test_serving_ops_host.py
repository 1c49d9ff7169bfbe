"""The serving operators' host side: refusals, the frequency tables, struct layouts.  No GPU needed --
every refusal here comes before the first CUDA call, and the pointers are never followed."""
import ctypes as C
import math
import os
import subprocess

import pytest

from needle_b200 import native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an aligned address that nothing reads


@pytest.fixture(scope="module", autouse=True)
def built():
    import needle_b200.build as b
    return b.build()


def rope_args(**kw):
    a = native.RopeAppend()
    for n in ("q", "k", "v", "q_out", "positions", "slots", "entries", "key_codes", "key_scales", "value_codes",
              "value_scales"):
        setattr(a, n, P)
    a.q_stride = a.q_out_stride = 8 * 64
    a.k_stride = a.v_stride = a.k_out_stride = a.v_out_stride = 4 * 64
    a.magnitude = 1.0
    a.tokens, a.heads, a.kv_heads, a.head_dim, a.rotary_dim = 2, 8, 4, 64, 64
    a.slot_count, a.capacity = 1, 4
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def attention_args(**kw):
    a = native.PrefixAttention()
    for n in ("q", "out", "prefix_key_codes", "prefix_key_scales", "prefix_value_codes", "prefix_value_scales",
              "key_codes", "key_scales", "value_codes", "value_scales", "slots", "counts"):
        setattr(a, n, P)
    a.q_stride = a.out_stride = 512
    a.rows, a.heads, a.kv_heads, a.head_dim = 2, 8, 4, 64
    a.prefix_length = a.prefix_capacity = 100
    a.slot_count, a.capacity = 2, 16
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def logits_args(**kw):
    a = native.LogitsRules()
    a.logits, a.logits_stride, a.rows, a.vocab = P, 100, 2, 100
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def refused(rc, text):
    with pytest.raises(native.NeedleError) as e:
        native.check(rc)
    assert e.value.code == "BACKEND_UNAVAILABLE" and text in str(e.value), str(e.value)


ONES = (C.c_double * 64)(*[1.0] * 64)


@pytest.mark.parametrize("change,text", [
    (dict(type=3), "element type"), (dict(type=-1), "element type"), (dict(head_dim=96), "64 and 128"),
    (dict(tokens=-1), "count"), (dict(heads=0), "count"), (dict(kv_heads=0), "count"), (dict(capacity=-1), "count"),
    (dict(slot_count=-1), "count"), (dict(rotary_dim=66), "rotary_dim"), (dict(rotary_dim=31), "rotary_dim"),
    (dict(rotary_dim=-2), "rotary_dim"), (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"),
    (dict(q_out=None), "null"), (dict(positions=None), "null"), (dict(slots=None), "null"),
    (dict(entries=None), "null"), (dict(key_codes=None), "null"), (dict(value_scales=None), "null"),
    (dict(q_stride=511), "stride"), (dict(k_stride=0), "stride"), (dict(v_stride=-256), "stride"),
    (dict(q_out_stride=0), "stride"), (dict(k_out=P, k_out_stride=255), "stride"), (dict(q=P + 2), "aligned"),
    (dict(type=1, v=P + 1), "aligned"), (dict(key_codes=P + 8), "16-byte"), (dict(value_codes=P + 1), "16-byte"),
    (dict(magnitude=math.inf), "magnitude"), (dict(magnitude=math.nan), "magnitude")])
def test_rope_append_refuses(change, text):
    refused(native.lib().needle_cuda_rope_append_dev(C.byref(rope_args(**change)), ONES, None), text)


def test_rope_append_refuses_frequencies():
    refused(native.lib().needle_cuda_rope_append_dev(C.byref(rope_args()), None, None), "null")
    refused(native.lib().needle_cuda_rope_append_dev(None, ONES, None), "null")
    bad = (C.c_double * 32)(*[1.0] * 31, math.nan)
    refused(native.lib().needle_cuda_rope_append_dev(C.byref(rope_args()), bad, None), "finite")


def test_nothing_to_do_is_not_an_error():
    native.check(native.lib().needle_cuda_rope_append_dev(C.byref(rope_args(tokens=0)), ONES, None))
    native.check(native.lib().needle_cuda_prefix_attention_dev(C.byref(attention_args(rows=0)), None, 0, None))
    native.check(native.lib().needle_cuda_logits_rules_dev(C.byref(logits_args(rows=0)), P, 100, None))
    native.check(native.lib().needle_cuda_logits_select_dev(C.byref(logits_args(rows=0)), P, P, None))


@pytest.mark.parametrize("change,text", [
    (dict(type=7), "element type"), (dict(head_dim=32), "64 and 128"), (dict(heads=6), "multiple"),
    (dict(heads=0), "multiple"), (dict(kv_heads=0), "multiple"), (dict(rows=-1), "count"),
    (dict(prefix_length=-1), "count"), (dict(slot_count=-1), "count"), (dict(capacity=-5), "count"),
    (dict(prefix_length=101), "longer"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(counts=None), "null"),
    (dict(prefix_key_codes=None), "null"), (dict(prefix_value_scales=None), "null"), (dict(key_codes=None), "null"),
    (dict(value_scales=None), "null"), (dict(q_stride=511), "stride"), (dict(out_stride=0), "stride"),
    (dict(q=P + 2), "aligned"), (dict(prefix_key_codes=P + 8), "16-byte"), (dict(value_codes=P + 4), "16-byte")])
def test_prefix_attention_refuses(change, text):
    refused(native.lib().needle_cuda_prefix_attention_dev(C.byref(attention_args(**change)), P, 1 << 40, None), text)


def workspace(a):
    n = C.c_size_t()
    native.check(native.lib().needle_cuda_prefix_attention_workspace(C.byref(a), C.byref(n)))
    return n.value


def test_prefix_attention_workspace_is_checked():
    for a in (attention_args(), attention_args(rows=4096, prefix_length=2000, prefix_capacity=2048),
              attention_args(rows=1, capacity=100000)):
        need = workspace(a)
        if need:
            refused(native.lib().needle_cuda_prefix_attention_dev(C.byref(a), P, need - 1, None), "workspace")
            refused(native.lib().needle_cuda_prefix_attention_dev(C.byref(a), None, need, None), "workspace")
            refused(native.lib().needle_cuda_prefix_attention_dev(C.byref(a), P + 8, need, None), "workspace")
    refused(native.lib().needle_cuda_prefix_attention_workspace(C.byref(attention_args()), None), "null")


@pytest.mark.parametrize("change,text", [
    (dict(type=3), "element type"), (dict(rows=-1), "count"), (dict(vocab=-1), "count"), (dict(rows=65536), "65535"),
    (dict(logits=None), "null"), (dict(logits_stride=99), "stride"), (dict(logits=P + 2), "aligned"),
    (dict(history=P, history_stride=4), "history"), (dict(history=P, history_lengths=P, history_stride=-1), "history"),
    (dict(bias_ids=P, bias_stride=1), "bias"), (dict(bias_ids=P, bias_values=P, bias_stride=1), "bias"),
    (dict(bias_ids=P, bias_values=P, bias_counts=P, bias_stride=-1), "bias"), (dict(masks=P), "masks"),
    (dict(masks=P, mask_slots=P, mask_count=-1), "masks")])
def test_logits_rules_refuse(change, text):
    a = logits_args(**change)
    refused(native.lib().needle_cuda_logits_rules_dev(C.byref(a), P, 100, None), text)
    refused(native.lib().needle_cuda_logits_select_dev(C.byref(a), P, P, None), text)


def test_logits_outputs_are_checked():
    if not _no_gpu():
        pytest.skip("the next check would look the fake pointers up")
    refused(native.lib().needle_cuda_logits_select_dev(C.byref(logits_args(vocab=0)), P, P, None), "empty")
    for rc in (native.lib().needle_cuda_logits_rules_dev(C.byref(logits_args()), None, 100, None),
               native.lib().needle_cuda_logits_select_dev(C.byref(logits_args()), None, P, None)):
        assert rc != 0


@pytest.mark.parametrize("name", ["q_norm", "k_norm", "positions", "slots", "entries", "key_scales", "value_scales", "k_out"])
def test_rope_append_refuses_misaligned_lists(name):
    refused(native.lib().needle_cuda_rope_append_dev(C.byref(rope_args(**{name: P + 2})), ONES, None), name + " is not aligned")


@pytest.mark.parametrize("name", ["lse", "slots", "counts", "prefix_key_scales", "prefix_value_scales", "key_scales", "value_scales"])
def test_prefix_attention_refuses_misaligned_lists(name):
    a = attention_args(**{name: P + 2})
    refused(native.lib().needle_cuda_prefix_attention_dev(C.byref(a), P, 1 << 40, None), name + " is not aligned")


@pytest.mark.parametrize("name", ["history", "history_lengths", "prompt_lengths", "repetition", "presence", "frequency",
                                  "bias_ids", "bias_values", "bias_counts", "masks", "mask_slots"])
def test_logits_operators_refuse_misaligned_lists(name):
    lists = dict.fromkeys(("history", "history_lengths", "bias_ids", "bias_values", "bias_counts", "masks", "mask_slots"), P)
    a = logits_args(**{**lists, "history_stride": 4, "bias_stride": 4, "mask_count": 1, name: P + 1})
    refused(native.lib().needle_cuda_logits_rules_dev(C.byref(a), P, 100, None), name + " is not aligned")
    refused(native.lib().needle_cuda_logits_select_dev(C.byref(a), P, P, None), name + " is not aligned")


def test_logits_operators_refuse_lists_whose_counts_would_not_fit():
    for change in (dict(history=P, history_lengths=P, history_stride=1 << 30),
                   dict(bias_ids=P, bias_values=P, bias_counts=P, bias_stride=1 << 30), dict(vocab=(1 << 30) + 1, logits_stride=1 << 31)):
        a = logits_args(**change)
        refused(native.lib().needle_cuda_logits_rules_dev(C.byref(a), P, 1 << 31, None), "2^30")
        refused(native.lib().needle_cuda_logits_select_dev(C.byref(a), P, P, None), "2^30")


def test_logits_outputs_are_refused():
    a = logits_args(logits=P, logits_stride=120)
    refused(native.lib().needle_cuda_logits_rules_dev(C.byref(a), P, 100, None), "same row stride")
    refused(native.lib().needle_cuda_logits_rules_dev(C.byref(a), P + 2, 100, None), "out is not aligned")
    refused(native.lib().needle_cuda_logits_select_dev(C.byref(a), P + 2, P, None), "ids is not aligned")
    refused(native.lib().needle_cuda_logits_select_dev(C.byref(a), P, P + 1, None), "log_probabilities is not aligned")


def _no_gpu():
    import torch
    return not torch.cuda.is_available()


def frequencies(n, **kw):
    s = native.RopeScaling(**kw)
    w, m = (C.c_double * (n // 2))(), C.c_double()
    native.check(native.lib().needle_cuda_rope_frequencies(C.byref(s), n, w, C.byref(m)))
    return list(w), m.value


@pytest.mark.parametrize("n", [2, 6, 64, 128])
def test_rope_frequencies(n):
    plain, one = frequencies(n, theta=10000.0, kind=native.ROPE_PLAIN)
    assert one == 1.0 and plain == [10000.0 ** (-2.0 * i / n) for i in range(n // 2)]
    linear, one = frequencies(n, theta=10000.0, factor=4.0, kind=native.ROPE_LINEAR)
    assert one == 1.0 and linear == [w / 4.0 for w in plain]
    if n >= 4:
        # the first pair keeps its frequency, the last one is interpolated by the whole factor
        ntk, one = frequencies(n, theta=10000.0, factor=4.0, kind=native.ROPE_NTK)
        assert one == 1.0 and ntk[0] == 1.0 and ntk[-1] == pytest.approx(plain[-1] / 4.0, rel=1e-12)
    parts, m = frequencies(n, theta=10000.0, factor=8.0, trained_length=4096.0, fast_turns=32.0, slow_turns=1.0,
                           kind=native.ROPE_PARTS)
    assert m == pytest.approx(0.1 * math.log(8.0) + 1.0, rel=1e-15)
    for w, p in zip(parts, plain):
        turns = 4096.0 * p / (2 * math.pi)
        if turns >= 32.0:
            assert w == p
        elif turns <= 1.0:
            assert w == pytest.approx(p / 8.0, rel=1e-15)
        else:
            assert p / 8.0 < w < p


@pytest.mark.parametrize("n,kw,text", [
    (3, dict(theta=10.0), "rotary_dim"), (0, dict(theta=10.0), "rotary_dim"), (130, dict(theta=10.0), "rotary_dim"),
    (64, dict(theta=0.0), "theta"), (64, dict(theta=math.nan), "theta"), (64, dict(theta=10.0, kind=4), "scaling"),
    (64, dict(theta=10.0, kind=1), "factor"), (2, dict(theta=10.0, kind=2, factor=2.0), "NTK"),
    (64, dict(theta=10.0, kind=3, factor=2.0), "parts"),
    (64, dict(theta=10.0, kind=3, factor=2.0, trained_length=100.0, fast_turns=1.0, slow_turns=1.0), "parts")])
def test_rope_frequencies_refuse(n, kw, text):
    s = native.RopeScaling(**kw)
    w, m = (C.c_double * 64)(), C.c_double()
    refused(native.lib().needle_cuda_rope_frequencies(C.byref(s), n, w, C.byref(m)), text)


def test_structs_match_the_header(tmp_path):
    """Sizes and offsets of the ctypes structs against the header's, as a C compiler lays them out."""
    pairs = [("needle_rope_append", native.RopeAppend), ("needle_rope_scaling", native.RopeScaling),
             ("needle_prefix_attention", native.PrefixAttention), ("needle_logits_rules", native.LogitsRules)]
    lines = ["#include <stdio.h>", '#include "needle_cuda.h"', "int main(void) {"]
    want = []
    for name, struct in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(struct))
        for field, _ in struct._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(struct, field).offset)
    (tmp_path / "s.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")],
                   check=True)
    got = subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in got] == want
