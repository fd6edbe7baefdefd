"""What the operators that decode several tokens a step refuse: host code only,
nothing reaches a GPU."""

import ctypes as C
import math

import pytest

import mlvc_hip

A = 1 << 20  # a well-aligned address; nothing here is dereferenced
NAN = float("nan")


def cache(**over):
    d = dict(kind=mlvc_hip.KV_INT8, pages=8, page_size=16, heads=2, head_dim=64, k=A, v=A, k_scale=A, v_scale=A)
    d.update(over)
    return mlvc_hip.KvCache(**d)


def plan(**over):
    d = dict(streams=3, pages=8, page_size=16, tokens=5, window=0, sinks=0, table=A, table_stride=4, held=A, free_pages=A,
             free_count=A, past=A, fresh=A + 64, seen=A, lengths=A + 128, starts=A, slots=A, positions=A, lacking=A)
    d.update(over)
    return lambda: mlvc_hip.kv_plan(mlvc_hip.KvPlan(**d))


def window(window=16, sinks=4, **over):
    d = dict(sequences=2, q_heads=8, kv_heads=2, head_dim=64, q=A, k=A, v=A, out=A, q_stride=512, k_stride=128,
             v_stride=128, out_stride=512, q_starts=A, k_starts=A, q_tokens=10, k_tokens=10, longest_q=5, causal=1,
             scale=0.125)
    d.update(over)
    return lambda: mlvc_hip.attention_window(mlvc_hip.WindowAttention(prompt=mlvc_hip.PromptAttention(**d), window=window, sinks=sinks))


def drafts(over_cache=None, **over):
    c = cache(**(over_cache or {}))
    d = dict(cache=C.pointer(c), streams=3, q_heads=8, q_tokens=24, longest_q=8, q=A, out=A, q_stride=512, out_stride=512,
             starts=A, seen=A, table=A, table_stride=4, lengths=A, longest=64, window=0, sinks=0, scale=0.125, workspace=A,
             workspace_bytes=1 << 40)
    d.update(over)
    return lambda: mlvc_hip.attention_drafts(mlvc_hip.DraftAttention(**d))


def keep(over_cache=None, **over):
    c = cache(**(over_cache or {}))
    d = dict(cache=C.pointer(c), streams=3, table=A, table_stride=4, starts=A, lengths=A + 64, kept=A, kept_stride=4,
             lengths_out=A + 128)
    d.update(over)
    return lambda: mlvc_hip.kv_keep(mlvc_hip.KvKeep(**d))


@pytest.mark.parametrize("call,message", [
    (lambda: mlvc_hip.kv_plan(None), "no descriptor"),
    (plan(streams=-1), "negative size"), (plan(tokens=-1), "negative size"), (plan(table_stride=-1), "negative size"),
    (plan(window=-1), "window"), (plan(sinks=-1), "sinks"), (plan(page_size=0), "page_size"), (plan(page_size=24), "page_size"),
    (plan(pages=-1), "2\\^31"), (plan(pages=1 << 27), "2\\^31"), (plan(streams=1 << 16, table_stride=1 << 15), "2\\^31"),
    (plan(table=None), "null"), (plan(held=None), "null"), (plan(free_pages=None), "null"), (plan(free_count=None), "null"),
    (plan(past=None), "null"), (plan(fresh=None), "null"), (plan(lengths=None), "null"), (plan(starts=None), "null"),
    (plan(slots=None), "null"), (plan(lacking=None), "null"),
    (plan(lengths=A), "lengths must not be"), (plan(lengths=A + 64), "lengths must not be"),
    (plan(table=A + 2), "aligned"), (plan(positions=A + 1), "aligned"), (plan(held=A + 4), "8-byte"), (plan(seen=A + 4), "8-byte"),
    (lambda: mlvc_hip.attention_window(None), "no descriptor"),
    (window(window=-1), "window"), (window(sinks=-1), "sinks"), (window(sequences=-1), "attention_window: negative"),
    (window(head_dim=0), "head_dim"), (window(q_heads=7), "multiple"), (window(scale=NAN), "scale"),
    (window(q_stride=500), "stride"), (window(k=None), "null"), (window(out=A + 1), "aligned"),
    (lambda: mlvc_hip.attention_drafts(None), "no descriptor"),
    (drafts(cache=None), "no cache"), (drafts({"kind": 9}), "kind"), (drafts({"page_size": 8}), "page_size"),
    (drafts(streams=-1), "negative"), (drafts(longest=-1), "negative"), (drafts(q_tokens=-1), "negative"),
    (drafts(table_stride=-1), "negative"), (drafts(longest_q=0), "longest_q"), (drafts(longest_q=65), "longest_q"),
    (drafts(window=-1), "window"), (drafts(sinks=-1), "sinks"), (drafts(q_heads=7), "multiple"), (drafts(q_heads=0), "multiple"),
    (drafts(scale=math.inf), "scale"), (drafts(q_stride=100), "stride"), (drafts(out_stride=0), "stride"),
    (drafts(q=None), "null"), (drafts(starts=None), "null"), (drafts(lengths=None), "null"), (drafts(table=None), "null"),
    (drafts(out=A + 1), "aligned"), (drafts(seen=A + 4), "aligned"), (drafts(starts=A + 2), "aligned"),
    (drafts(streams=1 << 20, q_heads=64, longest_q=64, longest=1 << 20, q_stride=4096, out_stride=4096), "too many"),
    (lambda: mlvc_hip.kv_keep(None), "no descriptor"),
    (keep(cache=None), "no cache"), (keep({"k": None}), "aligned"), (keep(streams=-1), "negative"), (keep(table_stride=-1), "negative"),
    (keep(kept_stride=-1), "kept_stride"), (keep(kept_stride=65), "kept_stride"), (keep(starts=None), "null"),
    (keep(lengths=None), "null"), (keep(kept=None), "null"), (keep(table=None), "null"), (keep(lengths_out=None), "null"),
    (keep(lengths_out=A + 64), "lengths_out must not be"), (keep(lengths_out=A), "lengths_out must not be"),
    (keep(kept=A + 2), "aligned"), (keep({"heads": 65535}, streams=1 << 20), "too many"),
])
def test_refused(call, message):
    with pytest.raises(mlvc_hip.MlvcError, match=message):
        call()


@pytest.mark.parametrize("call", [
    window(sequences=0), window(q_tokens=0, q=None), window(longest_q=0), drafts(streams=0, q=None), drafts(q_tokens=0, out=None),
    keep(streams=0, starts=None),
])
def test_nothing_to_do(call):
    call()


def test_workspace_of_refused_descriptor_is_zero():
    c = cache(kind=7)
    assert mlvc_hip.attention_drafts_workspace_bytes(mlvc_hip.DraftAttention(cache=C.pointer(c), streams=1, q_heads=2, longest_q=1)) == 0


@pytest.mark.parametrize("call,message", [
    (plan(placed=A), "placed must not be"), (plan(placed=A + 64), "placed must not be"), (plan(placed=A + 128), "placed must not be"),
    (plan(placed=A + 258), "aligned"), (drafts(placed=A + 2), "aligned"), (keep(placed=A + 2), "aligned"),
    (keep(placed=A + 128), "lengths_out must not be"),
])
def test_refused_placed(call, message):
    with pytest.raises(mlvc_hip.MlvcError, match=message):
        call()
