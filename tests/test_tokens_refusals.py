"""What the token operators refuse, and the rotation's frequencies: host code
only, nothing reaches a GPU."""

import ctypes as C
import math

import numpy as np
import pytest

import mlvc_hip

A = 1 << 20  # a well-aligned address; nothing here is dereferenced


def rope(**over):
    d = dict(tokens=4, q_heads=8, k_heads=2, head_dim=64, q=A, k=A, q_out=A, k_out=A, q_stride=512, k_stride=128,
             q_out_stride=512, k_out_stride=128, eps=1e-6, positions=A, freqs=A, rot_dim=64, rot_scale=1.0)
    d.update(over)
    return lambda: mlvc_hip.qk_norm_rope(mlvc_hip.QkNormRope(**d))


def cache(**over):
    d = dict(kind=mlvc_hip.KV_INT8, pages=8, page_size=16, heads=2, head_dim=64, k=A, v=A, k_scale=A, v_scale=A)
    d.update(over)
    return mlvc_hip.KvCache(**d)


def rows(op, over_cache=None, **over):
    d = dict(tokens=4, k=A, v=A, k_stride=128, v_stride=128, slots=A)
    d.update(over)
    return lambda: op(cache(**(over_cache or {})), mlvc_hip.KvRows(**d))


def prompt(**over):
    d = dict(sequences=2, q_heads=8, kv_heads=2, head_dim=64, q=A, k=A, v=A, out=A, q_stride=512, k_stride=128,
             v_stride=128, out_stride=512, q_starts=A, k_starts=A, q_tokens=10, k_tokens=10, longest_q=5, causal=1,
             scale=0.125)
    d.update(over)
    return lambda: mlvc_hip.attention_prompt(mlvc_hip.PromptAttention(**d))


def token(over_cache=None, **over):
    c = cache(**(over_cache or {}))
    d = dict(cache=C.pointer(c), streams=3, q_heads=8, q=A, out=A, q_stride=512, out_stride=512, table=A,
             table_stride=4, lengths=A, longest=64, scale=0.125, workspace=A, workspace_bytes=1 << 40)
    d.update(over)
    return lambda: mlvc_hip.attention_token(mlvc_hip.TokenAttention(**d))


NAN = float("nan")


@pytest.mark.parametrize("call,message", [
    (lambda: mlvc_hip.qk_norm_rope(None), "no descriptor"),
    (rope(tokens=-1), "negative token count"),
    (rope(head_dim=0), "head_dim"), (rope(head_dim=513), "head_dim"),
    (rope(q_heads=0, k_heads=0), "head counts"), (rope(q_heads=-1), "head counts"),
    (rope(rot_dim=3), "rot_dim"), (rope(rot_dim=66), "rot_dim"), (rope(rot_dim=-2), "rot_dim"),
    (rope(eps=-1.0), "eps"), (rope(eps=NAN), "eps"), (rope(rot_scale=math.inf), "rot_scale"),
    (rope(q_stride=511), "stride"), (rope(k_out_stride=-128), "stride"),
    (rope(q=None), "null"), (rope(k_out=None), "null"), (rope(positions=None), "positions"),
    (rope(q=A + 1), "aligned"), (rope(k_weight=A + 1), "aligned"),
    (lambda: mlvc_hip.kv_write(None, mlvc_hip.KvRows()), "no cache"),
    (lambda: mlvc_hip.kv_read(cache(), None), "no rows"),
    (rows(mlvc_hip.kv_write, {"kind": 3}), "kind"), (rows(mlvc_hip.kv_read, {"kind": -1}), "kind"),
    (rows(mlvc_hip.kv_write, {"page_size": 24}), "page_size"), (rows(mlvc_hip.kv_read, {"page_size": 0}), "page_size"),
    (rows(mlvc_hip.kv_write, {"head_dim": 60}), "head_dim"), (rows(mlvc_hip.kv_read, {"head_dim": 520}), "head_dim"),
    (rows(mlvc_hip.kv_write, {"heads": 0}), "heads"), (rows(mlvc_hip.kv_write, {"pages": 1 << 27}), "2\\^31"),
    (rows(mlvc_hip.kv_write, {"pages": -1}), "2\\^31"),
    (rows(mlvc_hip.kv_write, {"k": None}), "aligned"), (rows(mlvc_hip.kv_read, {"v": A + 8}), "aligned"),
    (rows(mlvc_hip.kv_write, {"k_scale": None}), "scales"),
    (rows(mlvc_hip.kv_write, tokens=-1), "negative"), (rows(mlvc_hip.kv_read, k_stride=127), "stride"),
    (rows(mlvc_hip.kv_write, slots=None), "null"), (rows(mlvc_hip.kv_read, v=A + 1), "aligned"),
    (lambda: mlvc_hip.attention_prompt(None), "no descriptor"),
    (prompt(sequences=-1), "negative"), (prompt(q_tokens=-1), "negative"), (prompt(longest_q=-1), "negative"),
    (prompt(head_dim=0), "head_dim"), (prompt(head_dim=513), "head_dim"),
    (prompt(q_heads=7), "multiple"), (prompt(kv_heads=0), "multiple"), (prompt(q_heads=0), "multiple"),
    (prompt(scale=NAN), "scale"), (prompt(q_stride=500), "stride"), (prompt(v_stride=0), "stride"),
    (prompt(q=None), "null"), (prompt(k_starts=None), "null"), (prompt(k=None), "null"), (prompt(out=A + 1), "aligned"),
    (lambda: mlvc_hip.attention_token(None), "no descriptor"),
    (token(cache=None), "no cache"), (token({"kind": 9}), "kind"), (token(streams=-1), "negative"),
    (token(longest=-1), "negative"), (token(q_heads=7), "multiple"), (token(scale=math.inf), "scale"),
    (token(q_stride=100), "stride"), (token(lengths=None), "null"), (token(table=None), "null"),
    (token(out=A + 1), "aligned"), (token(longest=1 << 20, table_stride=1 << 16, workspace=None), "workspace"),
    (token(longest=1 << 20, table_stride=1 << 16, workspace_bytes=16), "workspace"),
    (token(longest=1 << 20, table_stride=1 << 16, workspace=A + 4), "workspace"),
    (lambda: mlvc_hip.rope_frequencies(7), "rot_dim"), (lambda: mlvc_hip.rope_frequencies(64, -1.0), "base"),
    (lambda: mlvc_hip.rope_frequencies(64, 1e4, 9), "scaling"),
    (lambda: mlvc_hip.rope_frequencies(64, 1e4, mlvc_hip.ROPE_LINEAR, 0.5), "factor"),
    (lambda: mlvc_hip.rope_frequencies(64, 1e4, mlvc_hip.ROPE_BANDS, 2.0, 0.0), "trained"),
])
def test_refused(call, message):
    with pytest.raises(mlvc_hip.MlvcError, match=message):
        call()


@pytest.mark.parametrize("call", [
    rope(tokens=0, q=None, k=None), rows(mlvc_hip.kv_write, tokens=0), rows(mlvc_hip.kv_read, tokens=0, k=None),
    prompt(sequences=0), prompt(q_tokens=0, q=None), prompt(longest_q=0), token(streams=0, q=None),
])
def test_nothing_to_do(call):
    call()


def test_workspace_of_refused_descriptor_is_zero():
    c = cache(kind=7)
    assert mlvc_hip.attention_token_workspace_bytes(mlvc_hip.TokenAttention(cache=C.pointer(c), streams=1, q_heads=2)) == 0


def test_frequencies():
    i = np.arange(32)
    plain, one = mlvc_hip.rope_frequencies(64)
    assert one == 1.0 and np.allclose(plain, 10000.0 ** (-i / 32), rtol=1e-15)
    linear, one = mlvc_hip.rope_frequencies(64, 10000.0, mlvc_hip.ROPE_LINEAR, 4.0)
    assert one == 1.0 and np.allclose(linear, plain / 4, rtol=1e-15)
    wide, one = mlvc_hip.rope_frequencies(64, 10000.0, mlvc_hip.ROPE_BASE, 4.0)
    assert one == 1.0 and wide[0] == plain[0] and np.isclose(wide[-1], plain[-1] / 4, rtol=1e-12)
    assert np.all(np.diff(wide / plain) < 0)
    bands, scale = mlvc_hip.rope_frequencies(64, 10000.0, mlvc_hip.ROPE_BANDS, 4.0, 4096)
    turns = 4096 * plain / (2 * np.pi)
    assert np.isclose(scale, 0.1 * math.log(4) + 1, rtol=1e-7)
    assert np.array_equal(bands[turns >= 32], plain[turns >= 32])
    assert np.allclose(bands[turns <= 1], plain[turns <= 1] / 4, rtol=1e-15)
    mid = (turns > 1) & (turns < 32)
    kept = (turns[mid] - 1) / 31
    assert mid.any() and np.allclose(bands[mid], plain[mid] * (kept + (1 - kept) / 4), rtol=1e-14)
    assert len(mlvc_hip.rope_frequencies(0)[0]) == 0
