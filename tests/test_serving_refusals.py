"""Refusals of the operators between the projections, without a GPU: the C entries return their documented codes
before any device work, and the Python ones raise ValueError naming the argument."""

import ctypes

import pytest
import torch

from muse_bf16_proj_b200 import _lib
from muse_bf16_proj_b200.attention import rope_append, rope_table, split_qkv_gate, tree_attention
from muse_bf16_proj_b200.routing import route

INVALID, ALIGN, SHAPE = -1, -2, -3


def rope_args(**kw):
    a = dict(q=16, k=16, v=16, q_out=16, k_pages=16, v_pages=16, rope=16, position=16, slot=16, q_token=64, q_head=64, k_token=64,
             k_head=64, v_token=64, v_head=64, out_token=64, out_head=64, k_page=1024, k_page_head=1024, k_entry=64, v_page=1024,
             v_page_head=1024, v_entry=64, positions=8, pages=4, tokens=1, heads=1, kv_heads=1, dim=64, rotary=64, page_size=16)
    a.update(kw)
    return _lib.MuseRopeAppend(**a)


def attention_args(**kw):
    a = dict(q=16, out=16, k_pages=16, v_pages=16, table=16, context=16, starts=16, scratch=256, scratch_bytes=1 << 40, q_token=64,
             q_head=64, out_token=64, out_head=64, k_page=1024, k_page_head=1024, k_entry=64, v_page=1024, v_page_head=1024, v_entry=64,
             table_row=4, pages=4, tokens=1, requests=1, max_draft=1, table_cols=4, heads=1, kv_heads=1, dim=64, page_size=16, scale=1.0)
    a.update(kw)
    return _lib.MuseTreeAttention(**a)


def route_args(**kw):
    a = dict(logits=16, weights=16, expert_ids=16, row=64, tokens=1, experts=64, top_k=4, groups=1, top_groups=1, type=_lib.TYPE_F32,
             scale=1.0)
    a.update(kw)
    return _lib.MuseRoute(**a)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), INVALID), (dict(slot=None), INVALID), (dict(tokens=-1), INVALID), (dict(type=2), INVALID), (dict(pages=0), INVALID),
    (dict(positions=0), INVALID), (dict(page_size=0), INVALID), (dict(dim=96), SHAPE), (dict(heads=3, kv_heads=2), SHAPE),
    (dict(heads=0), SHAPE), (dict(rotary=7), SHAPE), (dict(rotary=66), SHAPE), (dict(rotary=0), SHAPE), (dict(q=17), ALIGN),
    (dict(slot=20), ALIGN), (dict(rope=18), ALIGN)])
def test_rope_append_codes(change, code):
    assert _lib.load().muse_rope_append(rope_args(**change), None) == code
    assert _lib.load().muse_last_error().startswith(b"rope_append:")


@pytest.mark.parametrize("change,code", [
    (dict(q=None), INVALID), (dict(scratch=None), INVALID), (dict(requests=-1), INVALID), (dict(type=2), INVALID), (dict(pages=0), INVALID),
    (dict(table_cols=0), INVALID), (dict(dim=80), SHAPE), (dict(heads=5, kv_heads=2), SHAPE), (dict(max_draft=0), SHAPE),
    (dict(max_draft=257), SHAPE), (dict(page_size=4), SHAPE), (dict(page_size=24), SHAPE), (dict(page_size=2048), SHAPE),
    (dict(mask=16, mask_words=1, max_draft=33), SHAPE), (dict(q=24), ALIGN), (dict(q_token=60), ALIGN), (dict(v_entry=68), ALIGN),
    (dict(gate=16, gate_token=4, gate_head=64), ALIGN), (dict(context=18), ALIGN), (dict(scale=0.0), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(k_entry=0), SHAPE), (dict(v_page=1 << 40), SHAPE), (dict(kv_heads=2, heads=2, k_page=1544), SHAPE),
    (dict(pages=1 << 31), SHAPE), (dict(table_cols=1 << 28), SHAPE), (dict(requests=1 << 20, table_cols=1 << 16), SHAPE)])
def test_tree_attention_codes(change, code):
    assert _lib.load().muse_tree_attention(attention_args(**change), None) == code
    assert _lib.load().muse_last_error().startswith(b"tree_attention")


@pytest.mark.parametrize("change,code", [
    (dict(logits=None), INVALID), (dict(tokens=-2), INVALID), (dict(type=3), INVALID), (dict(experts=0), SHAPE), (dict(experts=1025), SHAPE),
    (dict(top_k=0), SHAPE), (dict(top_k=33), SHAPE), (dict(top_k=9, groups=8, top_groups=1), SHAPE), (dict(groups=5), SHAPE),
    (dict(groups=64), SHAPE), (dict(groups=4, top_groups=5), SHAPE), (dict(top_groups=0), SHAPE), (dict(logits=18), ALIGN),
    (dict(bias=18), ALIGN)])
def test_route_codes(change, code):
    assert _lib.load().muse_route(route_args(**change), None) == code
    assert _lib.load().muse_last_error().startswith(b"route:")


def test_null_arguments_and_empty_calls():
    lib = _lib.load()
    assert lib.muse_rope_append(None, None) == INVALID and lib.muse_tree_attention(None, None) == INVALID
    assert lib.muse_route(None, None) == INVALID
    assert lib.muse_tree_attention_scratch_bytes(attention_args(), None) == INVALID
    assert lib.muse_rope_append(rope_args(tokens=0, q=None), None) == 0
    assert lib.muse_tree_attention(attention_args(tokens=0), None) == 0
    assert lib.muse_tree_attention(attention_args(requests=0), None) == 0
    assert lib.muse_route(route_args(tokens=0, logits=None), None) == 0


def test_structs_have_the_headers_size():
    # 9 pointers, 16 int64, 8 int32; 10 pointers, 16 int64, 10 int32 and a float; 4 pointers, 1 int64, 8 int32 and a float.
    assert ctypes.sizeof(_lib.MuseRopeAppend) == 8 * 25 + 4 * 8
    assert ctypes.sizeof(_lib.MuseTreeAttention) == 8 * 26 + 4 * 11 + 4
    assert ctypes.sizeof(_lib.MuseRoute) == 8 * 5 + 4 * 9 + 4
    # The packed bytes are the structures.
    for cls, pack in ((_lib.MuseRopeAppend, _lib.PACK_ROPE_APPEND), (_lib.MuseTreeAttention, _lib.PACK_TREE_ATTENTION),
                      (_lib.MuseRoute, _lib.PACK_ROUTE)):
        values = [0.5 if t is ctypes.c_float else i + 1 for i, (_, t) in enumerate(cls._fields_)]
        assert pack(*values) == bytes(cls(*values))


def _attention(**kw):
    bf = torch.bfloat16
    a = dict(q=torch.zeros((2, 4, 64), dtype=bf), k_pages=torch.zeros((3, 2, 16, 64), dtype=bf), v_pages=torch.zeros((3, 2, 16, 64), dtype=bf),
             page_table=torch.zeros((1, 3), dtype=torch.int32), context=torch.zeros(1, dtype=torch.int32),
             starts=torch.zeros(2, dtype=torch.int32), max_draft=2)
    a.update(kw)
    return a


@pytest.mark.parametrize("name,kw", [
    ("q", dict(q=torch.zeros((2, 4, 64)))), ("q", dict(q=torch.zeros((2, 256), dtype=torch.bfloat16))),
    ("k_pages", dict(v_pages=torch.zeros((3, 2, 16, 64)))), ("k_pages", dict(k_pages=torch.zeros((3, 2, 16, 128), dtype=torch.bfloat16))),
    ("context", dict(context=torch.zeros(1, dtype=torch.int64))), ("starts", dict(starts=torch.zeros(3, dtype=torch.int32))),
    ("page_table", dict(page_table=torch.zeros((2, 3), dtype=torch.int32))), ("tree_mask", dict(tree_mask=torch.zeros((3, 1), dtype=torch.int32))),
    ("tree_mask", dict(tree_mask=torch.zeros((2, 1), dtype=torch.int64))), ("gate", dict(gate=torch.zeros((2, 2, 64), dtype=torch.bfloat16))),
    ("out", dict(out=torch.zeros((1, 4, 64), dtype=torch.bfloat16))), ("CUDA", {})])
def test_tree_attention_raises(name, kw):
    with pytest.raises((ValueError, RuntimeError), match=name):
        tree_attention(**_attention(**kw))


def _rope(**kw):
    bf = torch.bfloat16
    a = dict(q=torch.zeros((2, 4, 64), dtype=bf), k=torch.zeros((2, 2, 64), dtype=bf), v=torch.zeros((2, 2, 64), dtype=bf),
             positions=torch.zeros(2, dtype=torch.int32), slots=torch.arange(2), k_pages=torch.zeros((3, 2, 16, 64), dtype=bf),
             v_pages=torch.zeros((3, 2, 16, 64), dtype=bf), rope=torch.zeros((8, 64)))
    a.update(kw)
    return a


@pytest.mark.parametrize("name,kw", [
    ("q", dict(q=torch.zeros((2, 4, 64)))), ("k", dict(k=torch.zeros((3, 2, 64), dtype=torch.bfloat16))),
    ("v", dict(v=torch.zeros((2, 2, 32), dtype=torch.bfloat16))), ("positions", dict(positions=torch.zeros(2, dtype=torch.int64))),
    ("slots", dict(slots=torch.zeros(2, dtype=torch.int32))), ("k_pages", dict(k_pages=torch.zeros((3, 4, 16, 64), dtype=torch.bfloat16))),
    ("rope", dict(rope=torch.zeros((8, 128)))), ("rope", dict(rope=torch.zeros((8, 64), dtype=torch.float64))),
    ("q_out", dict(q_out=torch.zeros((2, 4, 32), dtype=torch.bfloat16))), ("CUDA", {})])
def test_rope_append_raises(name, kw):
    with pytest.raises(ValueError, match=name):
        rope_append(**_rope(**kw))


@pytest.mark.parametrize("name,kw", [
    ("logits", dict(logits=torch.zeros(64))), ("logits", dict(logits=torch.zeros((2, 64), dtype=torch.float64))),
    ("bias", dict(bias=torch.zeros(63))), ("scoring", dict(scoring="tanh")), ("top_k", dict(top_k=0)), ("CUDA", {})])
def test_route_raises(name, kw):
    a = dict(logits=torch.zeros((2, 64)), top_k=4)
    a.update(kw)
    with pytest.raises(ValueError, match=name):
        route(**a)


def test_split_qkv_gate():
    y = torch.arange(2 * 36 * 64, dtype=torch.float32).view(2, -1)
    q, k, v, gate = split_qkv_gate(y, 16, 2, 64)
    assert [tuple(t.shape) for t in (q, k, v, gate)] == [(2, 16, 64), (2, 2, 64), (2, 2, 64), (2, 16, 64)]
    assert torch.equal(torch.cat([t.flatten(1) for t in (q, k, v, gate)], 1), y)
    assert split_qkv_gate(y[:, :20 * 64], 16, 2, 64)[3] is None
    with pytest.raises(ValueError):
        split_qkv_gate(y[:, :-1], 16, 2, 64)


def test_rope_tables():
    """Each scaling against its formula at single entries, in 64 bits."""
    import math

    def entry(table, p, i):
        return table[p, i].item(), table[p, table.shape[1] // 2 + i].item()

    def close(got, angle, magnitude=1.0):
        assert abs(got[0] - magnitude * math.cos(angle)) < 1e-7 and abs(got[1] - magnitude * math.sin(angle)) < 1e-7

    rot, f = 64, 4.0
    freq = [10000.0 ** (-2 * i / rot) for i in range(rot // 2)]
    n = 4000
    for i in (0, 1, 13, 31):
        close(entry(rope_table(rot, n, device="cpu"), 3999, i), 3999 * freq[i])
        close(entry(rope_table(rot, n, scaling="linear", factor=f, device="cpu"), 3999, i), 3999 * freq[i] / f)
        base = 10000.0 * f ** (rot / (rot - 2))
        close(entry(rope_table(rot, n, scaling="ntk", factor=f, device="cpu"), 3999, i), 3999 * base ** (-2 * i / rot))
        turns = 8192 * freq[i] / (2 * math.pi)
        keep = min(max((turns - 1.0) / 3.0, 0.0), 1.0)
        close(entry(rope_table(rot, n, scaling="bands", factor=f, device="cpu"), 3999, i), 3999 * (freq[i] / f * (1 - keep) + freq[i] * keep))
    # The lowest frequency of "ntk" is divided by the factor.
    base = 10000.0 * f ** (rot / (rot - 2))
    assert abs(base ** (-(rot - 2) / rot) - freq[-1] / f) < 1e-12
    yarn = rope_table(rot, n, scaling="yarn", factor=f, device="cpu")
    close(entry(yarn, 3999, 0), 3999 * freq[0], 0.1 * math.log(f) + 1.0)          # turns often: kept
    close(entry(yarn, 3999, 31), 3999 * freq[31] / f, 0.1 * math.log(f) + 1.0)    # hardly turns: divided
    for bad in (dict(rotary=7), dict(rotary=0), dict(positions=0), dict(scaling="cubic"), dict(factor=0.0)):
        with pytest.raises(ValueError):
            rope_table(**{"rotary": 64, "positions": 4, "device": "cpu", **bad})
    with pytest.raises(ValueError):
        rope_table(64, 4, scaling="bands", low=4.0, high=4.0, device="cpu")
