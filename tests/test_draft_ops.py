"""The operators of a drafted-token step (nf_rope_init, nf_kv_write,
nf_tree_attention, nf_token_logprobs, nf_kv_accept) on the CPU: what their
entry points refuse before any CUDA call, and the rotary tables."""
import ctypes
import math

import numpy as np
import pytest

from helpers import nfm

m = nfm()
P = 1 << 12  # a pointer value that no call here may follow (16- and 256-byte aligned)


def cache(**kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, kind=m.KV_E4M3, seqs=4, kv_heads=2, max_context=64, head_dim=128)
    return m.KvDesc(**{**d, **kw})


def rope(head_dim=128, rotary_dim=128, **kw):
    return m.Rope(head_dim, rotary_dim=rotary_dim, **kw)


def call_write(c=None, r=None, **kw):
    a = dict(qkv=P, qkv_type=0, stride=1024, tokens=0, q_heads=4, q_norm=None, k_norm=None, eps=1e-5, pos=P, seq=P, slot=P,
             q=P, status=None)
    a.update(kw)
    c = cache() if c is None else c
    r = rope().desc if r is None else r
    return m.load().nf_kv_write(ctypes.byref(c), ctypes.byref(r), a["qkv"], a["qkv_type"], a["stride"], a["tokens"],
                                a["q_heads"], a["q_norm"], a["k_norm"], a["eps"], a["pos"], a["seq"], a["slot"], a["q"],
                                a["status"], None)


def call_tree(c=None, **kw):
    a = dict(q=P, rows=0, q_heads=4, row_start=P, batch=1, prefix=P, cache_seq=None, mask=None, words=0, scale=0.1, out=P,
             work=P, work_bytes=1 << 40, status=None)
    a.update(kw)
    c = cache() if c is None else c
    return m.load().nf_tree_attention(ctypes.byref(c), a["q"], a["rows"], a["q_heads"], a["row_start"], a["batch"],
                                      a["prefix"], a["cache_seq"], a["mask"], a["words"], a["scale"], a["out"], a["work"],
                                      a["work_bytes"], a["status"], None)


def call_logprobs(**kw):
    a = dict(logits=P, type=0, stride=100, rows=0, vocab=100, target=P, top=0, logprob=P, entropy=P, top_idx=None,
             top_lp=None, work=P, work_bytes=1 << 40)
    a.update(kw)
    return m.load().nf_token_logprobs(a["logits"], a["type"], a["stride"], a["rows"], a["vocab"], a["target"], a["top"],
                                      a["logprob"], a["entropy"], a["top_idx"], a["top_lp"], a["work"], a["work_bytes"], None)


def call_accept(caches=None, layers=None, **kw):
    a = dict(prefix=P, path=P, max_path=0, path_len=P, cache_seq=None, batch=0, status=None)
    a.update(kw)
    caches = [cache()] if caches is None else caches
    arr = (m.KvDesc * max(1, len(caches)))(*caches)
    return m.load().nf_kv_accept(arr, len(caches) if layers is None else layers, a["prefix"], a["path"], a["max_path"],
                                 a["path_len"], a["cache_seq"], a["batch"], a["status"], None)


def message():
    return m.load().nf_kv_last_error().decode()


BAD_CACHES = [(dict(kind=2), "kind", 1), (dict(head_dim=96), "head_dim", 8), (dict(seqs=0), "shape", 2),
              (dict(kv_heads=0), "shape", 2), (dict(max_context=0), "shape", 2), (dict(seqs=1 << 20, kv_heads=1 << 12), "shape", 2),
              (dict(k=None), "null cache pointer", 1), (dict(v=P + 8), "16-byte", 3), (dict(k_scale=None), "needs its scales", 1),
              (dict(v_scale=P + 2), "4-byte", 3), (dict(kind=m.KV_BF16), "no scales", 1)]


@pytest.mark.parametrize("bad, word, status", BAD_CACHES)
def test_every_call_refuses_a_bad_cache(bad, word, status):
    c = cache(**bad)
    for call in (lambda: call_write(c), lambda: call_tree(c), lambda: call_accept([c])):
        assert call() == status and word in message()


def test_empty_calls_do_nothing():
    """No rows: nothing is read, so nothing but the description is checked (and no CUDA call is made: there is no GPU)."""
    assert call_write() == 0 and call_tree() == 0 and call_logprobs() == 0 and call_accept() == 0
    assert call_tree(rows=3, batch=0) == 0 and call_accept(batch=2) == 0 and call_accept([], layers=0, batch=2, max_path=2) == 0
    assert message() == ""


@pytest.mark.parametrize("bad, word, status", [
    (dict(tokens=-1), "tokens", 1), (dict(qkv_type=2), "qkv type", 1), (dict(q_heads=0), "q_heads", 2),
    (dict(stride=1023), "stride", 2), (dict(stride=1026), "aligned", 3), (dict(qkv_type=1, stride=1028), "aligned", 3),
    (dict(qkv=P + 4), "aligned", 3), (dict(q=P + 2), "aligned", 3), (dict(eps=-1.0), "eps", 1), (dict(eps=math.nan), "eps", 1),
    (dict(tokens=1, qkv=None), "null", 1), (dict(tokens=1, pos=None), "null", 1), (dict(tokens=1, q=None), "null", 1),
    (dict(tokens=1 << 30, q_heads=1 << 10, stride=1 << 20), "2\\^31", 10)])
def test_write_refuses(bad, word, status):
    import re

    assert call_write(**bad) == status and re.search(word, message())


def test_write_refuses_other_rotary_tables():
    assert call_write(r=rope(64, 64).desc) == 2 and "head_dim 64" in message()
    r = rope().desc
    r.layout = 5
    assert call_write(r=r) == 1
    r = rope().desc
    r.rotary_dim = 130
    assert call_write(r=r) == 2


@pytest.mark.parametrize("bad, word, status", [
    (dict(rows=-1), "rows", 1), (dict(batch=-1), "batch", 1), (dict(q_heads=3), "multiple", 2), (dict(q_heads=0), "multiple", 2),
    (dict(q_heads=258), "128", 2), (dict(mask=P, words=0), "mask_words", 2), (dict(mask=P, words=65), "mask_words", 2),
    (dict(scale=math.inf), "scale", 1), (dict(rows=1, q=None), "null", 1), (dict(rows=1, out=None), "null", 1),
    (dict(rows=1, prefix=None), "null", 1), (dict(rows=1, row_start=None), "null", 1), (dict(rows=1, q=P + 8), "aligned", 3),
    (dict(rows=1, mask=P + 4, words=1), "aligned", 3), (dict(rows=1, work=None), "workspace", 10),
    (dict(rows=1, work_bytes=1), "workspace", 10), (dict(rows=1, work=P + 16), "256-byte", 3),
    (dict(rows=1 << 30, q_heads=4), "2^31", 10)])
def test_tree_attention_refuses(bad, word, status):
    assert call_tree(**bad) == status and word in message()


@pytest.mark.parametrize("bad, word, status", [
    (dict(type=3), "type", 1), (dict(rows=-1), "rows", 1), (dict(vocab=0), "vocab", 2), (dict(vocab=1 << 31, stride=1 << 32), "vocab", 2),
    (dict(stride=99), "stride", 2), (dict(top=33), "top", 8), (dict(top=-1), "top", 8), (dict(vocab=5, top=6), "top", 8),
    (dict(target=None), "together", 1), (dict(logprob=None), "together", 1), (dict(rows=1, logits=None), "null", 1),
    (dict(rows=1, top=2), "null", 1), (dict(rows=1, logits=P + 2), "aligned", 3), (dict(rows=1, type=1, logits=P + 1), "aligned", 3),
    (dict(rows=1, work=None), "workspace", 10), (dict(rows=1, work_bytes=0), "workspace", 10), (dict(rows=1, work=P + 8), "16-byte", 3)])
def test_logprobs_refuses(bad, word, status):
    assert call_logprobs(**bad) == status and word in message()


def test_accept_refuses():
    for bad in (dict(batch=-1), dict(max_path=-1)):
        assert call_accept(**bad) == 1
    assert call_accept(layers=-1) == 1
    assert call_accept([cache(), cache(max_context=65)]) == 2 and "layer 1" in message()
    assert call_accept([cache(), cache(kind=m.KV_BF16, k_scale=None, v_scale=None)]) == 2
    for bad in (dict(prefix=None), dict(path=None), dict(path_len=None)):
        assert call_accept(batch=1, max_path=1, **bad) == 1 and "null" in message()


@pytest.mark.parametrize("bad", [dict(rotary_dim=3), dict(rotary_dim=130), dict(rotary_dim=-2), dict(theta=0.0), dict(theta=math.inf),
                                 dict(scaling="linear", factor=0.5), dict(scaling="yarn", factor=2.0),
                                 dict(scaling="yarn", factor=2.0, original_context=64, fast=1.0, slow=1.0),
                                 dict(layout="other"), dict(scaling="other")])
def test_rope_refuses(bad):
    with pytest.raises(m.NfError):
        rope(**{**dict(rotary_dim=128), **bad})
    with pytest.raises(m.NfError):
        rope(96, 64)


def frequencies(rd, theta, scaling, factor, original, fast=32.0, slow=1.0):
    f = theta ** (-2.0 * np.arange(rd // 2) / rd)
    if scaling == "linear":
        return f / factor
    if scaling == "yarn":
        g = np.clip((original * f / (2 * np.pi) - slow) / (fast - slow), 0, 1)
        return f * g + f / factor * (1 - g)
    return f


@pytest.mark.parametrize("rd", [2, 62, 64, 128])
@pytest.mark.parametrize("scaling, factor, original", [("none", 1, 0), ("linear", 4, 0), ("yarn", 16, 4096)])
def test_rope_table(rd, scaling, factor, original):
    """The table's turns are the frequencies; a far position's angle from the integer product is the angle to the 2^-33 of a
    turn that the table's 64 bits leave (compared in 64-bit floats, good to position * 2^-53 turns)."""
    theta = 500000.0
    d = rope(128, rd, theta=theta, scaling=scaling, factor=factor, original_context=original).desc
    f = frequencies(rd, theta, scaling, factor, original)
    assert d.rotary_dim == rd and d.magnitude == pytest.approx(0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0)
    for i in range(rd // 2):
        turn = (f[i] / (2 * np.pi)) % 1.0
        assert abs(d.turn[i] / 2.0 ** 64 - turn) < 2.0 ** -50
        pos = 1_000_003
        got = (pos * d.turn[i]) % 2 ** 64 / 2.0 ** 64
        want = (pos * f[i] / (2 * np.pi)) % 1.0
        assert abs((got - want + 0.5) % 1.0 - 0.5) < 2.0 ** -32
    assert all(d.turn[i] == 0 for i in range(rd // 2, 64))


def test_workspace_sizes():
    assert m.tree_attention_workspace(64) > 0 and m.tree_attention_workspace(128) > 0 and m.tree_attention_workspace(96) == 0
    assert m.token_logprobs_workspace(4, 1000, 5) > 0 and m.token_logprobs_workspace(-1, 1000, 5) == 0
    assert m.token_logprobs_workspace(4, 1000, 33) == 0


def test_python_calls_refuse_host_tensors():
    import torch

    x = torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(m.NfError, match="not a CUDA tensor"):
        m.KvCache(x, x)
    with pytest.raises(m.NfError, match="not a CUDA tensor"):
        m.KvCache(np.zeros((2, 1, 8, 64), np.uint16), None)
    with pytest.raises(m.NfError, match="not a CUDA tensor"):
        m.token_logprobs(torch.zeros(2, 8), None, None, None, None, None, None)
    with pytest.raises(m.NfError, match="no caches"):
        m.KvCaches([])


def test_handle_calls_refuse_without_gpu():
    lib = m.load()
    assert lib.nf_stack_verify(None, None, None, None, None, None, 0, 1, 1, None, None, None) == 1
    assert lib.nf_stack_logprobs(None, 1, None, 0, None, None, None, None, None) == 1
    assert lib.nf_stack_accept(None, None, None, 1, None, 1, None) == 1
    assert lib.nf_stack_kv(None, 0, None) == 1
    assert lib.nf_tp_logprobs(None, 1, 10, None, 0, None, None, None, None, None) == 1
    h = ctypes.c_void_p()
    d = m.StackDesc(100, 256, 1, 0, 0, 0, m.Desc(256, 8, 2, 128, 128, 1, 1, 1, 1.0, 10.0, 0, 4), 8, 1, 128, 10000.0, 1e-5, 4, 64)
    assert lib.nf_stack_create_kv(ctypes.byref(d), 7, 0, ctypes.byref(h)) == 1 and not h.value
    assert b"cache kind" in lib.nf_stack_last_error(None)
