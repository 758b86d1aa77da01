"""Calls of the operators for many continuations that are refused before
anything reaches a GPU: the pointers here are never read."""
import ctypes as C

import numpy as np
import pytest

from aotk import abi, runtime

P = 1 << 20  # stand-ins for device addresses, far apart
OUT, Q, K, V, KT, VT = (P * (1 << 14) * i for i in range(1, 7))


@pytest.fixture(scope="module")
def lib():
    return abi.load()


def refused(lib, rc, what):
    assert rc == -1
    assert what in lib.aotk_last_error().decode(), lib.aotk_last_error().decode()


SINKS = dict(out=OUT, q=Q, k=K, v=V, kind=0, n_head=8, n_kv_head=2, head_dim=64, ctx=100, layer=0, pos0=10, m=5, window=8,
             n_sink=2)


@pytest.mark.parametrize("change,what", [
    (dict(kind=5), "kind 5"), (dict(kind=-1), "kind -1"), (dict(head_dim=80), "head_dim 80"), (dict(n_head=0), "head counts"),
    (dict(n_kv_head=0), "head counts"), (dict(n_kv_head=3), "head counts"), (dict(n_head=16386), "head counts"),
    (dict(m=0), "no rows"), (dict(pos0=96), "exceed the context"), (dict(pos0=2 ** 64 - 3), "exceed the context"),
    (dict(m=101, pos0=0), "exceed the context"), (dict(out=None), "null"), (dict(q=None), "null"), (dict(k=None), "null"),
    (dict(v=None), "null"), (dict(q=Q + 2), "aligned"), (dict(out=Q), "overlaps"), (dict(out=K + 64), "overlaps"),
    (dict(out=V - 64), "overlaps"), (dict(ctx=2 ** 62), "too large"), (dict(layer=2 ** 60), "too large"),
    (dict(ctx=2 ** 40, m=2 ** 39, pos0=0), "too many"),
], ids=str)
def test_sinks(lib, change, what):
    refused(lib, lib.aotk_attention_sinks(*{**SINKS, **change}.values()), what)


SHARED = dict(out=OUT, q=Q, kp=K, vp=V, kt=KT, vt=VT, kind=0, n_head=8, n_kv_head=2, head_dim=64, prefix_ctx=100, n_prefix=90,
              tail_ctx=20, layer=0, batch=3, tail_len=(5, 20, 0), rows=(1, 4, 1))


def call_shared(lib, change):
    a = {**SHARED, **change}
    for k in ("tail_len", "rows"):
        if a[k] is not None:
            a[k] = (C.c_uint32 * len(a[k]))(*a[k])
    return lib.aotk_attention_shared(*a.values())


@pytest.mark.parametrize("change,what", [
    (dict(kind=4), "kind 4"), (dict(head_dim=96), "head_dim 96"), (dict(n_head=7), "head counts"), (dict(batch=0), "no sequences"),
    (dict(batch=65536), "65536 sequences"), (dict(tail_len=None), "null"), (dict(n_prefix=101), "exceeds"),
    (dict(tail_len=(5, 21, 0)), "tail 1 has 21"), (dict(out=None), "null"), (dict(q=None), "null"), (dict(kp=None), "null"),
    (dict(vp=None), "null"), (dict(kt=None), "null"), (dict(vt=None), "null"), (dict(kt=KT + 1), "aligned"),
    (dict(out=Q + 256), "overlaps"), (dict(out=K), "overlaps"), (dict(out=VT), "overlaps"),
    (dict(rows=(1, 2 ** 31, 1)), "too many"), (dict(prefix_ctx=2 ** 60), "too large"), (dict(tail_ctx=2 ** 59), "too large"),
], ids=str)
def test_shared(lib, change, what):
    refused(lib, call_shared(lib, change), what)


def test_shared_without_rows_succeeds(lib):
    assert call_shared(lib, dict(rows=(0, 0, 0), q=None, out=None)) == 0


RULES = dict(out=OUT, logits=OUT, kind=0, rows=2, vocab=1000, stride=1000, rules=None, hist=Q, n_hist=10, bias_id=K, bias=V,
             n_bias=4, mask=KT, n_mask=1, tokens=VT)


def call_rules(lib, change):
    a = {**RULES, **{k: v for k, v in change.items() if k in RULES}}
    t = np.zeros(2, runtime.LOGITS_RULE_DTYPE)
    t["repetition"], t["mask"] = 1.0, -1
    for k, v in change.items():
        if k not in RULES:
            t[k][1] = v
    if "rules" not in change:
        a["rules"] = t.ctypes.data
    return lib.aotk_logits_rules(*a.values())


@pytest.mark.parametrize("change,what", [
    (dict(kind=3), "kind 3"), (dict(rows=0), "no logits"), (dict(vocab=0), "no logits"), (dict(vocab=2 ** 31, stride=2 ** 31), "too many"),
    (dict(stride=999), "stride"), (dict(rules=None), "null"), (dict(out=None), "null"), (dict(logits=None), "null"),
    (dict(repetition=0.0), "row 1"), (dict(repetition=-1.0), "row 1"), (dict(repetition=np.nan), "row 1"),
    (dict(repetition=np.inf), "row 1"), (dict(presence=np.nan), "not finite"), (dict(frequency=np.inf), "not finite"),
    (dict(hist_off=8, hist_len=3), "history outside"), (dict(hist_off=2 ** 32 - 1, hist_len=2 ** 31 - 1), "history outside"),
    (dict(hist_len=2 ** 31, n_hist=2 ** 40), "more than"), (dict(bias_len=2 ** 32 - 1, n_bias=2 ** 40), "more than"),
    (dict(bias_off=1, bias_len=4), "biases outside"), (dict(mask=1), "null"), (dict(hist=None, hist_len=1), "null"),
    (dict(bias=None, bias_len=1), "null"), (dict(bias_id=None, bias_len=1), "null"), (dict(logits=OUT + 400), "overlaps"),
    (dict(tokens=OUT + 7996), "overlaps"), (dict(hist=OUT + 40), "overlaps"), (dict(tokens=KT), "overlaps"),
    (dict(logits=OUT + 1), "aligned"), (dict(tokens=VT + 2), "aligned"), (dict(stride=2 ** 62), "too large"),
], ids=str)
def test_rules(lib, change, what):
    if change == dict(mask=1):  # the row of masks, not their address
        t = np.zeros(2, runtime.LOGITS_RULE_DTYPE)
        t["repetition"], t["mask"] = 1.0, [-1, 1]
        refused(lib, lib.aotk_logits_rules(*{**RULES, "rules": t.ctypes.data}.values()), "mask 1 of 1")
        t["mask"] = [-1, -2]
        refused(lib, lib.aotk_logits_rules(*{**RULES, "rules": t.ctypes.data}.values()), "mask -2")
        return
    refused(lib, call_rules(lib, change), what)


def test_rules_refuses_a_mask_that_is_not_there(lib):
    t = np.zeros(2, runtime.LOGITS_RULE_DTYPE)
    t["repetition"], t["mask"] = 1.0, 0
    refused(lib, lib.aotk_logits_rules(*{**RULES, "rules": t.ctypes.data, "mask": None}.values()), "null")


def test_the_table_of_rules():
    t, h, i, v = runtime.logits_rules_table([{}, {"history": [4, 5], "bias": {7: 1.5}, "mask": 2}, {"bias": [(1, 2.0), (1, 3.0)]}])
    assert list(t["repetition"]) == [1, 1, 1] and list(t["mask"]) == [-1, 2, -1]
    assert list(t["hist_off"]) == [0, 0, 2] and list(t["hist_len"]) == [0, 2, 0]
    assert list(t["bias_off"]) == [0, 0, 1] and list(t["bias_len"]) == [0, 1, 2]
    assert list(h) == [4, 5] and list(i) == [7, 1, 1] and list(v) == [1.5, 2.0, 3.0]
    with pytest.raises(ValueError, match="temperature"):
        runtime.logits_rules_table([{"temperature": 1.0}])


def test_allowed_mask():
    m = runtime.allowed_mask([0, 31, 32, 69], 70)
    assert list(m) == [0x80000001, 1, 1 << 5]
    assert list(runtime.allowed_mask([], 33)) == [0, 0]
    for outside in (-1, 70, 95):
        with pytest.raises(ValueError, match="outside"):
            runtime.allowed_mask([3, outside], 70)


def test_state_logits_of_no_state(lib):
    assert not lib.aotk_logits_dev(None)
    assert "null state" in lib.aotk_last_error().decode()


def test_the_wrappers_refuse_short_arrays_and_other_types():
    z = np.zeros((1, 4, 1, 64), np.float32)
    with pytest.raises(TypeError, match="float16"):
        runtime.attention_sinks(z[:, 0], z, z, 1, 1, 64, 4, 0, 3, 1, 0, 0, kind=abi.F16)


def f32(*shape):
    return np.zeros(shape, np.float32)


@pytest.mark.parametrize("change,what", [
    (dict(q=f32(4, 4, 64)), "q is smaller"), (dict(k=f32(2, 19, 2, 64)), "a cache is smaller"),
    (dict(v=f32(1, 20, 2, 64)), "a cache is smaller"), (dict(layer=2), "a cache is smaller"), (dict(m=6), "q is smaller"),
], ids=lambda x: None)
def test_sinks_of_short_arrays(change, what):
    a = dict(q=f32(5, 4, 64), k=f32(2, 20, 2, 64), v=f32(2, 20, 2, 64), n_head=4, n_kv_head=2, head_dim=64, ctx=20, layer=1, pos0=10,
             m=5, window=8, n_sink=2)
    with pytest.raises(ValueError, match=what):
        runtime.attention_sinks(*{**a, **change}.values())


@pytest.mark.parametrize("change,what", [
    (dict(q=f32(5, 4, 64)), "q is smaller"), (dict(kp=f32(2, 29, 2, 64)), "a cache is smaller"),
    (dict(vp=f32(1, 30, 2, 64)), "a cache is smaller"), (dict(kt=f32(2, 2, 10, 2, 64)), "a cache is smaller"),
    (dict(vt=f32(2, 3, 9, 2, 64)), "a cache is smaller"), (dict(layer=2), "a cache is smaller"),
    (dict(rows=[1, 2, 4]), "q is smaller"), (dict(rows=[3, 3]), "differ in length"), (dict(rows=[1, 2, 3, 0]), "differ in length"),
], ids=lambda x: None)
def test_shared_of_short_arrays(change, what):
    a = dict(q=f32(6, 4, 64), kp=f32(2, 30, 2, 64), vp=f32(2, 30, 2, 64), kt=f32(2, 3, 10, 2, 64), vt=f32(2, 3, 10, 2, 64), n_head=4,
             n_kv_head=2, head_dim=64, prefix_ctx=30, n_prefix=30, tail_ctx=10, layer=1, tail_len=[5, 10, 3], rows=[1, 2, 3])
    with pytest.raises(ValueError, match=what):
        runtime.attention_shared(*{**a, **change}.values())


def test_rules_of_fewer_dicts_than_rows():
    for n in (2, 4):
        with pytest.raises(ValueError, match="one dict"):
            runtime.logits_rules(f32(3, 100), [{}] * n)


@pytest.mark.parametrize("masks", [np.ones((1, 64), bool), np.ones((2, 64), np.float32), np.ones((1, 64), np.uint8),
                                   np.ones((2, 3), np.uint32), np.ones(4, np.uint32), np.ones((1, 2, 2), np.uint32), [[1, -1]]],
                         ids=lambda m: f"{np.asarray(m).dtype}{np.asarray(m).shape}")
def test_rules_of_masks_that_are_not_rows_of_words(masks):
    """64 tokens are two words: a truth value or a byte per token, or the words
    of another vocabulary, would be read as masks of something else."""
    with pytest.raises((TypeError, ValueError), match="32-bit words|rows of 2 words"):
        runtime.logits_rules(f32(2, 64), [{"mask": 0}] * 2, masks)


def test_rules_of_masks_as_words():
    words = np.array([[1, 2], [0xFFFFFFFF, 0]], np.uint32)
    for masks in (words, words.view(np.int32), words.tolist(), words.astype(np.int64)):
        assert np.array_equal(runtime._rules_host([{}], masks, 1, 64)[4], words)
    assert np.array_equal(runtime._rules_host([{}], words[0], 1, 64)[4], words[:1])
    for none in (None, [], np.zeros((0, 2), np.uint32)):
        assert runtime._rules_host([{}], none, 1, 64)[4].shape == (0, 2)
