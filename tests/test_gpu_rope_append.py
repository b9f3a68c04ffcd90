"""rope_append on the GPU against a plain 64-bit rotation: both pair layouts, part of the head, both 16-bit
types, aligned and unaligned strides, every cache layout, rows without a slot, in place, on another stream, in a
graph, past 2^31 elements, and positions and slots outside their range. A result is rounded once from FP32, so
it is within u |y| of the exact one plus eight FP32 roundings of what enters it."""

import pytest
import torch

from muse_bf16_proj_b200 import _lib
from muse_bf16_proj_b200.attention import page_slots, rope_append, rope_table, split_qkv_gate
from serving_ref import ROUND, STEP, rope64

pytestmark = pytest.mark.gpu


def device_error() -> int:
    return _lib.device_error(torch.cuda.current_stream().cuda_stream)


def make(m, hq, hk, d, dtype, page, seed, extra=2, column=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    y = torch.randn((m, (hq + 2 * hk) * d + column), generator=g, device="cuda").to(dtype)[:, column:]
    q, k, v, _ = split_qkv_gate(y, hq, hk, d)
    pages = (m + page - 1) // page + extra
    cache = [torch.randn((pages, hk, page, d), generator=g, device="cuda").to(dtype) for _ in range(2)]
    order = torch.randperm(pages * page, generator=g, device="cuda")[:m]
    return q, k, v, cache[0], cache[1], order.long(), g


def check(q, k, v, positions, slots, kp, vp, before_k, before_v, table, interleaved, got):
    dtype = q.dtype
    for x, y in ((q, got), (k, None)):
        want, size = rope64(x, positions, table, interleaved)
        bound = ROUND[dtype] * want.abs() + 8 * 2.0 ** -24 * size + STEP[dtype]
        if y is None:
            live = slots >= 0
            page = kp.shape[2]
            y, want, bound = kp[slots[live] // page, :, slots[live] % page], want[live], bound[live]
        assert ((y.double() - want).abs() <= bound).all()
    live = slots >= 0
    page = kp.shape[2]
    assert torch.equal(vp[slots[live] // page, :, slots[live] % page], v[live])
    # Nothing else of the cache moved.
    keep = torch.ones(kp.shape[0] * page, dtype=torch.bool, device="cuda")
    keep[slots[live]] = False
    for now, old in ((kp, before_k), (vp, before_v)):
        assert torch.equal(now.transpose(1, 2).flatten(0, 1)[keep], old.transpose(1, 2).flatten(0, 1)[keep])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("m,hq,hk,d,rotary,page", [
    (1, 16, 2, 64, 64, 16), (7, 32, 8, 128, 128, 32), (33, 5, 1, 128, 64, 8), (65, 12, 4, 64, 16, 1), (3, 1, 1, 64, 2, 5),
    (19, 8, 8, 128, 36, 64), (257, 64, 8, 128, 126, 128), (2, 3, 3, 64, 62, 1024)])
def test_rope_append(m, hq, hk, d, rotary, page, interleaved, dtype):
    q, k, v, kp, vp, slots, g = make(m, hq, hk, d, dtype, page, 11 + m)
    table = rope_table(rotary, 4096)
    positions = torch.randint(4096, (m,), generator=g, device="cuda", dtype=torch.int32)
    if m > 2:
        slots[1] = -1
        slots[m - 1] = -7
    old = kp.clone(), vp.clone()
    got = rope_append(q, k, v, positions, slots, kp, vp, table, interleaved=interleaved)
    check(q, k, v, positions, slots, kp, vp, *old, table, interleaved, got)
    assert got.is_contiguous() and device_error() == 0


@pytest.mark.parametrize("column", [1, 4, 8])
def test_unaligned_rows_and_cache_layouts(column):
    """Views that rule out 16-byte accesses, a cache with entries outside heads, both halves in one tensor."""
    q, k, v, _, _, slots, g = make(21, 16, 2, 64, torch.bfloat16, 16, 5, column=column)
    both = torch.randn((4, 16, 2, 2, 64), generator=g, device="cuda").to(torch.bfloat16)  # [pages, entry, k / v, heads, dim]
    kp, vp = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    slots = torch.randperm(64, generator=g, device="cuda")[:21]
    positions = torch.arange(100, 121, dtype=torch.int32, device="cuda")
    table = rope_table(64, 200, scaling="yarn", factor=4.0, original=64)
    old = kp.clone(), vp.clone()
    got = rope_append(q, k, v, positions, slots, kp, vp, table)
    check(q, k, v, positions, slots, kp, vp, *old, table, False, got)


def test_in_place_and_other_stream():
    q, k, v, kp, vp, slots, g = make(40, 32, 8, 128, torch.bfloat16, 32, 9)
    table, positions = rope_table(128, 64), torch.arange(40, dtype=torch.int32, device="cuda")
    want = rope_append(q, k, v, positions, slots, kp.clone(), vp.clone(), table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        own = rope_append(q, k, v, positions, slots, kp, vp, table, q_out=q)
    torch.cuda.current_stream().wait_stream(side)
    assert own is q and torch.equal(q, want)


def test_graph_replay_reads_new_inputs():
    q, k, v, kp, vp, slots, g = make(5, 16, 2, 64, torch.bfloat16, 16, 2)
    table, positions = rope_table(64, 64), torch.arange(5, dtype=torch.int32, device="cuda")
    rope_append(q, k, v, positions, slots, kp, vp, table)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rope_append(q, k, v, positions, slots, kp, vp, table)
    positions += 9
    q.mul_(-1.0)
    graph.replay()
    torch.cuda.synchronize()
    old = kp.clone(), vp.clone()
    check(q, k, v, positions, slots, kp, vp, *old, table, False, got)


def test_offsets_past_32_bits():
    """Slots whose element offset passes 2^32: a cache of over 8 GiB each for k and v."""
    pages, page, hk, d = 33000, 128, 8, 128
    kp = torch.zeros((pages, hk, page, d), dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    assert kp.numel() > 2 ** 32
    q, k, v, _, _, _, g = make(3, 8, 8, d, torch.bfloat16, page, 3)
    slots = torch.tensor([pages * page - 1, 0, (pages - 2) * page + 5], device="cuda")
    positions, table = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda"), rope_table(d, 8)
    rope_append(q, k, v, positions, slots, kp, vp, table)
    assert torch.equal(vp[slots // page, :, slots % page], v)
    want, size = rope64(k, positions, table, False)
    assert ((kp[slots // page, :, slots % page].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * size).all()
    assert int(torch.count_nonzero(vp)) == int(torch.count_nonzero(v))
    assert device_error() == 0


def test_no_tokens():
    q, k, v, kp, vp, slots, _ = make(4, 16, 2, 64, torch.bfloat16, 16, 1)
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    got = rope_append(q[:0], k[:0], v[:0], empty, slots[:0], kp, vp, rope_table(64, 8))
    assert got.shape == (0, 16, 64)


@pytest.mark.parametrize("rotary", [64, 36])
def test_out_of_range_is_reported_and_skipped(rotary):
    q, k, v, kp, vp, slots, _ = make(4, 16, 2, 64, torch.bfloat16, 16, 1)
    table = rope_table(rotary, 8)
    good = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    old = kp.clone(), vp.clone()
    with pytest.raises(_lib.MuseError, match="a01"):
        rope_append(q, k, v, torch.tensor([0, 8, 2, -1], dtype=torch.int32, device="cuda"), slots, kp, vp, table)
        _lib.device_error(torch.cuda.current_stream().cuda_stream)
    ok = torch.tensor([0, 2], device="cuda")
    rest = slots.clone()
    rest[1] = rest[3] = -1
    check(q[ok], k[ok], v[ok], good[ok], slots[ok], kp, vp, *old, table, False,
          rope_append(q, k, v, good, rest, kp, vp, table)[ok])
    old = kp.clone(), vp.clone()
    with pytest.raises(_lib.MuseError, match="a02"):
        far = slots.clone()
        far[2] = kp.shape[0] * kp.shape[2]
        rope_append(q, k, v, good, far, kp, vp, table)
        _lib.device_error(torch.cuda.current_stream().cuda_stream)
    far[2] = -1
    check(q, k, v, good, far, kp, vp, *old, table, False, rope_append(q, k, v, good, far, kp, vp, table))
    assert device_error() == 0


def test_page_slots():
    table = torch.tensor([[3, 1], [0, 2]], dtype=torch.int32, device="cuda")
    got = page_slots(table, torch.tensor([0, 0, 1], device="cuda"), torch.tensor([2, 17, 31], device="cuda"), 16)
    assert got.tolist() == [3 * 16 + 2, 16 + 1, 2 * 16 + 15]


def test_a_token_past_its_page_table_is_reported():
    """page_slots gives such a token a slot past every cache; the others are appended, a row without a token nowhere."""
    q, k, v, kp, vp, _, _ = make(4, 16, 2, 64, torch.bfloat16, 16, 1)
    table = torch.tensor([[1, -1]], dtype=torch.int32, device="cuda")
    owner = torch.zeros(4, dtype=torch.int32, device="cuda")
    kp.zero_()
    for index, reported in (([0, 5, -1, 15], False), ([0, 5, 16, 15], True), ([0, 5, 32, 15], True)):
        slots = page_slots(table, owner, torch.tensor(index, dtype=torch.int32, device="cuda"), 16)
        rope_append(q, k, v, owner, slots, kp, vp, rope_table(64, 8))
        if reported:
            with pytest.raises(_lib.MuseError, match="a02"):
                device_error()
        else:
            assert device_error() == 0
        assert torch.nonzero(kp.abs().sum((1, 3)))[:, 1].tolist() == [0, 5, 15] and not kp[0].any() and not kp[2].any()
