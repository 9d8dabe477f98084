"""What the operators on the int8 cache refuse, before anything is launched (no GPU needed)."""
import ctypes as C

import pytest
import torch

from megcc_b200 import _lib, ops

NULL_PTR, OUT_OF_RANGE, DTYPE, LAYOUT = 1, 4, 11, 12
P = 4096  # an address that nothing reads


def cache(change):
    c = dict(k=P, v=P, k_scales=P, v_scales=P, block_table=P, table_stride=4, pages=9, kv_heads=2, page_tokens=32, d=64,
             batch=3, table_pages=4)
    c.update({k: v for k, v in change.items() if k in c})
    return C.byref(_lib.KvCache(*(c[k] for k, _ in _lib.KvCache._fields_)))


def heads(change, name, heads=2):
    return _lib.Heads(*change.get(name, (P, 64 * heads, 64)))


def rest(change, known):
    return {k: v for k, v in change.items() if k in known}


def append(change):
    a = dict(lengths=P, cu=P, tokens=10, heads=4, dtype=2, cosines=P, sines=P, positions=100, rot_dims=64, interleaved=0)
    a.update(rest(change, a))
    p = _lib.KvAppendParam(a["lengths"], a["cu"], a["tokens"], a["heads"], a["dtype"], heads(change, "nk"),
                           heads(change, "nv"), heads(change, "q", 4), heads(change, "q_out", 4), heads(change, "k_out"),
                           a["cosines"], a["sines"], a["positions"], a["rot_dims"], a["interleaved"])
    return _lib.lib().mb200_kv_append_s8(cache(change), C.byref(p), None)


def read(change):
    a = dict(starts=P, cu=P, tokens=10, dtype=1)
    a.update(rest(change, a))
    k, v = heads(change, "nk"), heads(change, "nv")
    return _lib.lib().mb200_kv_read_s8(cache(change), a["starts"], a["cu"], a["tokens"], a["dtype"], C.byref(k), C.byref(v),
                                       None)


def attention_cache(change):
    a = dict(lengths=P, heads=4, queries=1, dtype=1, scale=0.1, ws=P, nbytes=1 << 30)
    a.update(rest(change, a))
    q, out = heads(change, "q", 4), heads(change, "out", 4)
    return _lib.lib().mb200_attention_cache_s8(cache(change), a["lengths"], a["heads"], a["queries"], a["dtype"],
                                               C.byref(q), a["scale"], C.byref(out), a["ws"], a["nbytes"], None)


CACHE = [
    (dict(k=None), NULL_PTR), (dict(v=None), NULL_PTR), (dict(k_scales=None), NULL_PTR), (dict(v_scales=None), NULL_PTR),
    (dict(block_table=None), NULL_PTR), (dict(k=P + 8), LAYOUT), (dict(v=P + 1), LAYOUT), (dict(k_scales=P + 2), LAYOUT),
    (dict(block_table=P + 2), LAYOUT), (dict(pages=0), LAYOUT), (dict(kv_heads=0), LAYOUT), (dict(page_tokens=0), LAYOUT),
    (dict(page_tokens=24), LAYOUT), (dict(batch=-1), LAYOUT), (dict(table_pages=0), LAYOUT), (dict(table_stride=3), LAYOUT),
    (dict(d=0), LAYOUT), (dict(d=72), LAYOUT), (dict(d=144), OUT_OF_RANGE),
    (dict(pages=1 << 30), OUT_OF_RANGE), (dict(dtype=0), DTYPE), (dict(dtype=3), DTYPE)]


@pytest.mark.parametrize("change,status", CACHE)
@pytest.mark.parametrize("call", [append, read, attention_cache])
def test_cache(call, change, status):
    assert call(change) == status


@pytest.mark.parametrize("change,status", [
    (dict(lengths=None), NULL_PTR), (dict(cu=None), LAYOUT), (dict(tokens=-1), LAYOUT), (dict(cosines=None), NULL_PTR),
    (dict(sines=None), NULL_PTR), (dict(cosines=None, sines=None), LAYOUT), (dict(rot_dims=0), LAYOUT),
    (dict(rot_dims=8), LAYOUT), (dict(rot_dims=80), LAYOUT), (dict(positions=0), LAYOUT), (dict(heads=0), LAYOUT),
    (dict(nk=(None, 128, 64)), NULL_PTR), (dict(nv=(None, 128, 64)), NULL_PTR), (dict(q_out=(None, 256, 64)), NULL_PTR),
    (dict(nk=(P + 1, 128, 64)), LAYOUT), (dict(nk=(P, -128, 64)), LAYOUT), (dict(q=(P, 256, -64)), LAYOUT),
    (dict(q_out=(P, 255, 64)), LAYOUT), (dict(q_out=(P, 256, 63)), LAYOUT), (dict(k_out=(P, 0, 64)), LAYOUT),
    (dict(lengths=P + 2), LAYOUT), (dict(cu=P + 1), LAYOUT), (dict(cosines=P + 2), LAYOUT), (dict(sines=P + 2), LAYOUT),
    (dict(tokens=0, lengths=None, nk=(None, 0, 0)), 0), (dict(batch=0, tokens=5), 0),
    (dict(tokens=(1 << 31) - 1), OUT_OF_RANGE), (dict(batch=1 << 30), OUT_OF_RANGE)])
def test_append(change, status):
    assert append(change) == status


@pytest.mark.parametrize("change,status", [
    (dict(cu=None), NULL_PTR), (dict(tokens=-1), LAYOUT), (dict(nk=(None, 128, 64)), NULL_PTR),
    (dict(nv=(P, 128, 60)), LAYOUT), (dict(nk=(P, 100, 64)), LAYOUT), (dict(nk=(P + 1, 128, 64)), LAYOUT),
    (dict(starts=P + 2), LAYOUT), (dict(cu=P + 2), LAYOUT), (dict(tokens=0, cu=None), 0), (dict(batch=0), 0),
    (dict(kv_heads=1 << 24, nk=(P, 1 << 31, 64), nv=(P, 1 << 31, 64)), OUT_OF_RANGE)])
def test_read(change, status):
    assert read(change) == status


FIVE = dict(table_pages=5, table_stride=5)  # (pages, which may be cut)


@pytest.mark.parametrize("change,status", [
    (dict(lengths=None), NULL_PTR), (dict(heads=3), LAYOUT), (dict(heads=0), LAYOUT), (dict(queries=0), LAYOUT),
    (dict(scale=float("nan")), LAYOUT), (dict(scale=float("inf")), LAYOUT),
    (dict(scale=3e38), LAYOUT), (dict(q=(None, 256, 64)), NULL_PTR),
    (dict(out=(None, 256, 64)), NULL_PTR), (dict(q=(P + 1, 256, 64)), LAYOUT), (dict(out=(P, 200, 64)), LAYOUT),
    (dict(out=(P, 256, 0)), LAYOUT), (dict(lengths=P + 1), LAYOUT), (dict(ws=None, **FIVE), NULL_PTR),
    (dict(ws=P + 128, **FIVE), LAYOUT), (dict(nbytes=100, **FIVE), LAYOUT), (dict(queries=1 << 29), OUT_OF_RANGE), (dict(batch=0, q=(None, 0, 0)), 0)])
def test_attention_cache(change, status):
    assert attention_cache(change) == status


def test_nothing_to_ask_for():
    lib = _lib.lib()
    assert lib.mb200_kv_append_s8(cache({}), None, None) == NULL_PTR
    assert lib.mb200_attention_cache_s8_workspace_bytes(None, 4, 1) == 0
    assert lib.mb200_attention_cache_s8_workspace_bytes(cache(dict(d=100)), 4, 1) == 0
    # tables of up to 128 positions: no sequence is cut
    assert lib.mb200_attention_cache_s8_workspace_bytes(cache({}), 4, 1) == 0
    size = lib.mb200_attention_cache_s8_workspace_bytes(cache(dict(table_pages=5, table_stride=5)), 4, 1)
    assert size > 0 and size % 256 == 0


def pool(**change):
    c = ops.kv_cache_s8(3, 2, 32, 64, device="cpu")
    return c._replace(**change)


def test_tensors_that_do_not_fit():
    q, table, lengths = torch.zeros((1, 4, 64), dtype=torch.float16), torch.zeros((1, 2), dtype=torch.int32), None
    for call in (lambda: ops.attention_cache_s8(q, pool(), table, lengths),
                 lambda: ops.kv_read_s8(pool(), table, None, lengths, 3),
                 lambda: ops.kv_append_s8(pool(), table, lengths, q, q),
                 lambda: ops.kv_read_s8(pool(k=q), table, None, lengths, 3),
                 lambda: ops.kv_read_s8(pool(k=None), table, None, lengths, 3)):
        with pytest.raises(ValueError):
            call()


def attention_prompt(change):
    a = dict(batch=3, cu_q=P, cu_k=P, tokens=10, key_tokens=20, heads=4, kv_heads=2, d=64, dtype=1, causal=1, scale=0.1)
    a.update(rest(change, a))
    q, k, v, out = heads(change, "q", 4), heads(change, "nk"), heads(change, "nv"), heads(change, "out", 4)
    return _lib.lib().mb200_attention_prompt(a["batch"], a["cu_q"], a["cu_k"], a["tokens"], a["key_tokens"], a["heads"],
                                             a["kv_heads"], a["d"], a["dtype"], C.byref(q), C.byref(k), C.byref(v),
                                             a["causal"], a["scale"], C.byref(out), None)


@pytest.mark.parametrize("change,status", [
    (dict(batch=-1), LAYOUT), (dict(tokens=-1), LAYOUT), (dict(key_tokens=-1), LAYOUT), (dict(heads=0), LAYOUT),
    (dict(heads=5), LAYOUT), (dict(kv_heads=0), LAYOUT), (dict(cu_k=None), LAYOUT), (dict(d=24), LAYOUT), (dict(d=-16), LAYOUT),
    (dict(d=256), OUT_OF_RANGE), (dict(dtype=0), DTYPE), (dict(scale=float("inf")), LAYOUT), (dict(scale=-3e38), LAYOUT),
    (dict(cu_q=None), NULL_PTR),
    (dict(q=(None, 256, 64)), NULL_PTR), (dict(nk=(None, 128, 64)), NULL_PTR), (dict(nv=(None, 128, 64)), NULL_PTR),
    (dict(out=(None, 256, 64)), NULL_PTR), (dict(q=(P + 2, 256, 64)), LAYOUT), (dict(nk=(P, 130, 64)), LAYOUT),
    (dict(nv=(P, 128, 0)), LAYOUT), (dict(nv=(P, 0, 64)), LAYOUT), (dict(q=(P, 256, 68)), LAYOUT),
    (dict(out=(P, 128, 64)), LAYOUT), (dict(out=(P + 1, 256, 64)), LAYOUT), (dict(cu_q=P + 2), LAYOUT),
    (dict(nk=(P, 1 << 38, 64)), OUT_OF_RANGE), (dict(key_tokens=(1 << 31) - 1), OUT_OF_RANGE),
    (dict(batch=1 << 30), OUT_OF_RANGE), (dict(tokens=0, q=(None, 0, 0)), 0), (dict(batch=0), 0)])
def test_attention_prompt(change, status):
    assert attention_prompt(change) == status
