"""Between the qkv_gate and o projections: rotary positions with the keys and values appended to a paged
cache (``rope_append``), and attention of each request's drafted tokens over that cache
(``tree_attention``), on this build's own sm_100a kernels (``muse_rope_append``,
``muse_tree_attention``). The reference projects and stops (reference.py:1-8); a step that uses its
projections runs::

    qkvg = project(x, state, "qkv_gate")                     # [M, (2 Hq + 2 Hkv) D]
    q, k, v, gate = split_qkv_gate(qkvg, heads, kv_heads, dim)
    q = rope_append(q, k, v, positions, slots, k_pages, v_pages, rope)
    a = tree_attention(q, k_pages, v_pages, page_table, context, starts, max_draft, tree_mask, gate=gate)
    y = project(a.view(M, Hq * D), state, "o")

The cache is two tensors [pages, kv_heads, page_size, dim] (any order of pages, heads
and entries in memory whose page stride is a multiple of the head stride). Request b
keeps its tokens in the pages of row b of ``page_table``; a token's *slot* is page * page_size + entry
(``page_slots``). Calls launch on torch's current stream, allocate with torch's caching allocator only,
do not synchronise and can be captured in a CUDA graph. A position, slot, page or request size out of
its range is found on the device and recorded in the device error word (``_lib.device_error``).
"""

from __future__ import annotations

import functools
import math

import torch

from . import _lib

_TYPES = {torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}
MAX_DRAFT = 256  # drafted tokens of one request; longer prompts go in pieces over the same pages


def split_qkv_gate(y: torch.Tensor, heads: int, kv_heads: int, dim: int):
    """Views q [M, heads, dim], k, v [M, kv_heads, dim] and gate [M, heads, dim] (None when y has no
    columns for it) of a fused projection's output y [M, (heads + 2 kv_heads (+ heads)) * dim]."""
    m, n = y.shape
    if n not in ((heads + 2 * kv_heads) * dim, (2 * heads + 2 * kv_heads) * dim):
        raise ValueError(f"y has {n} columns, not those of {heads} + 2 x {kv_heads} (+ {heads}) heads of {dim}")
    parts = y.unflatten(1, (n // dim, dim))
    q, k = parts[:, :heads], parts[:, heads:heads + kv_heads]
    v, gate = parts[:, heads + kv_heads:heads + 2 * kv_heads], parts[:, heads + 2 * kv_heads:]
    return q, k, v, gate if gate.shape[1] else None


def rope_table(rotary: int, positions: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
               original: int = 8192, low: float = 1.0, high: float = 4.0, beta_fast: float = 32.0, beta_slow: float = 1.0,
               device="cuda") -> torch.Tensor:
    """The FP32 table [positions, rotary] of ``rope_append``: rotary / 2 cosines, then as many sines of
    position * frequency_i with frequency_i = theta^(-2 i / rotary), computed in 64 bits. ``scaling`` for
    contexts ``factor`` times longer than the ``original`` positions:

    - "linear": every frequency divided by ``factor``;
    - "ntk": theta raised to theta * factor^(rotary / (rotary - 2)), so that the lowest frequency is
      divided by ``factor`` and the highest kept;
    - "bands": by wavelength; frequencies that turn fewer than ``low`` times in ``original`` positions are
      divided by ``factor``, more than ``high`` times kept, between them blended linearly in the turns;
    - "yarn": kept above ``beta_fast`` turns in ``original`` positions, divided by ``factor`` below
      ``beta_slow``, blended linearly in the pair's index between, and cosines and sines multiplied by
      0.1 ln(factor) + 1.
    """
    if rotary < 2 or rotary % 2 or positions < 1:
        raise ValueError(f"rotary must be even and positive and positions positive (got {rotary}, {positions})")
    if scaling not in ("none", "linear", "ntk", "bands", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if not factor > 0 or not theta > 0:
        raise ValueError(f"factor and theta must be positive (got {factor}, {theta})")
    index = torch.arange(0, rotary, 2, dtype=torch.float64, device=device)
    if scaling == "ntk" and rotary > 2:
        theta = theta * factor ** (rotary / (rotary - 2))
    freq = theta ** (-index / rotary)
    magnitude = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "bands":
        if not high > low:
            raise ValueError(f"high must be above low (got {low}, {high})")
        turns = original * freq / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq / factor * (1 - keep) + freq * keep
    elif scaling == "yarn":
        def pair_of(turns: float) -> float:  # the index whose frequency turns that often
            return rotary * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
        first = max(math.floor(pair_of(beta_fast)), 0)
        last = min(math.ceil(pair_of(beta_slow)), rotary - 1)
        ramp = ((index / 2 - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        freq = freq / factor * ramp + freq * (1 - ramp)
        magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return (torch.cat((angle.cos(), angle.sin()), dim=1) * magnitude).float()


def page_slots(page_table: torch.Tensor, request: torch.Tensor, index: torch.Tensor, page_size: int) -> torch.Tensor:
    """int64 slots of the tokens ``index`` (place in the request's sequence) of requests ``request``: -1, nothing
    to append, where the index is negative; past every cache, which ``rope_append`` reports (0xA02) and skips, where
    the page table has no such place (a request outside it, an index past its columns, a negative page)."""
    request, index = request.long(), index.long()
    requests, columns = page_table.shape
    past = torch.iinfo(torch.int64).max
    column = index.clamp(min=0) // page_size
    there = (request >= 0) & (request < requests) & (column < columns)
    if page_table.numel():
        # Indexes are inside the table whatever the lengths say: an indexing kernel's assertion would end the context.
        page = page_table[request.clamp(0, requests - 1), column.clamp(max=columns - 1)].long()
        slot = torch.where(there & (page >= 0), page * page_size + index % page_size, past)
    else:
        slot = torch.full_like(index, past)
    return torch.where(index < 0, -1, slot)


def tree_mask(parents: torch.Tensor, starts: torch.Tensor, max_draft: int) -> torch.Tensor:
    """The mask words [tokens, ceil(max_draft / 32)] int32 of drafted trees: ``parents`` [tokens] is each
    token's parent as an index among its request's drafted tokens (-1 for a root), earlier than the token
    itself; a token sees itself and its ancestors. What is no earlier token of the request counts as no parent, and
    rows that belong to no request (before starts[0], from starts[B] on) see nothing. Made once a step, on the
    tensors' device, in a few launches for each of ``max_draft`` levels."""
    n, size = parents.shape[0], (max_draft + 31) // 32 * 32
    device = parents.device
    token = torch.arange(n, device=device)
    owner = torch.bucketize(token, starts[1:].long(), right=True)
    first = starts.long()[owner]
    place = token - first  # among the request's tokens
    place = torch.where((owner < starts.shape[0] - 1) & (place < size), place, -1)  # negative: of none, or without a bit
    up = torch.where((parents >= 0) & (parents < place), parents.long(), -1)
    bits = torch.zeros((n, size), dtype=torch.bool, device=device)
    at = place
    for _ in range(max_draft):  # the token itself, then one level of ancestors a turn
        # Every index below is inside its tensor whatever the lengths say: an indexing kernel's assertion would end the context.
        live = at >= 0
        bits[token, at.clamp(min=0)] |= live
        at = torch.where(live, up[(first + at).clamp(0, max(n - 1, 0))], -1)
    weight = 1 << torch.arange(32, device=device, dtype=torch.int64)
    packed = (bits.view(n, size // 32, 32).long() * weight).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).int()


def _bad(name: str, wanted: str, t: torch.Tensor) -> ValueError:
    return ValueError(f"{name}: expected {wanted}, got {tuple(t.shape)} {t.dtype} on {t.device} with strides {t.stride()}")


# The checks below ask each tensor for each property once (a call is a few microseconds of host time, as much as a
# small launch) and hand back the strides, which the kernels want too. Devices are compared by index: -1 is the CPU.


def _rows(name: str, t: torch.Tensor, dev: int, dtype, m: int, heads: int, dim: int) -> tuple:
    stride = t.stride()
    if t.shape != (m, heads, dim) or t.dtype != dtype or t.get_device() != dev or stride[2] != 1:
        raise _bad(name, f"[{m}, {heads}, {dim}] {dtype} on device {dev} with contiguous rows", t)
    return stride


def _cache(k_pages: torch.Tensor, v_pages: torch.Tensor, dev: int, dtype, dim: int):
    shape, ck, cv = k_pages.shape, k_pages.stride(), v_pages.stride()
    if (len(shape) != 4 or v_pages.shape != shape or shape[3] != dim or k_pages.dtype != dtype or v_pages.dtype != dtype or
            k_pages.get_device() != dev or v_pages.get_device() != dev or ck[3] != 1 or cv[3] != 1):
        raise ValueError(f"k_pages, v_pages: expected two of [pages, kv_heads, page_size, {dim}] {dtype} on device {dev} with contiguous "
                         f"rows, got {tuple(shape)} {k_pages.dtype} on {k_pages.device} and {tuple(v_pages.shape)} {v_pages.dtype} on "
                         f"{v_pages.device}")
    return shape, ck, cv


def _vector(name: str, t: torch.Tensor, dev: int, dtype, n: int) -> int:
    if t.shape != (n,) or t.dtype != dtype or t.get_device() != dev or (n > 1 and t.stride(0) != 1):
        raise _bad(name, f"contiguous [{n}] {dtype} on device {dev}", t)
    return t.data_ptr()


def _words(name: str, t: torch.Tensor, dev: int, rows: int) -> int:
    shape = t.shape
    if len(shape) != 2 or shape[0] != rows or t.dtype != torch.int32 or t.get_device() != dev or (shape[1] > 1 and t.stride(1) != 1):
        raise _bad(name, f"[{rows}, columns] int32 on device {dev} with contiguous rows", t)
    return t.data_ptr()


def _check_cuda(t: torch.Tensor, dev: int) -> None:
    if dev < 0:
        raise ValueError(f"expected CUDA tensors, got {t.device}")


def _call(dev: int, entry, packed: bytes) -> None:
    """``entry(packed arguments, torch's current stream)`` on the tensors' device, which need not be the current one."""
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if dev == torch.cuda.current_device():
        entry(packed, stream)
    else:
        with torch.cuda.device(dev):
            entry(packed, stream)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                k_pages: torch.Tensor, v_pages: torch.Tensor, rope: torch.Tensor, *, interleaved: bool = False,
                q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Turns q [M, Hq, D] and k [M, Hkv, D] by their tokens' ``positions`` (int32 [M]), writes k and v into the
    cache at ``slots`` (int64 [M], distinct; negative: not appended) and returns the turned q (``q_out``, which
    may be q itself, or a new contiguous tensor). BF16 or FP16, D 64 or 128; q, k, v may be strided views of
    one projection output. ``rope``: FP32 [positions, rotary] (``rope_table``); pairs are (i, i + rotary / 2),
    or (2i, 2i + 1) when ``interleaved``; entries past ``rotary`` are left as they are."""
    dev, dtype = q.get_device(), q.dtype
    kind = _TYPES.get(dtype)
    if q.dim() != 3 or kind is None:
        raise ValueError(f"q: expected [tokens, heads, dim] in bfloat16 or float16, got {tuple(q.shape)} {dtype}")
    m, heads, dim = q.shape
    (pages, kv_heads, page_size, _), ck, cv = _cache(k_pages, v_pages, dev, dtype, dim)
    sq, sk, sv = _rows("q", q, dev, dtype, m, heads, dim), _rows("k", k, dev, dtype, m, kv_heads, dim), _rows("v", v, dev, dtype, m, kv_heads, dim)
    position, slot = _vector("positions", positions, dev, torch.int32, m), _vector("slots", slots, dev, torch.int64, m)
    table = rope.shape
    if len(table) != 2 or table[1] > dim or rope.dtype != torch.float32 or rope.get_device() != dev or not rope.is_contiguous():
        raise _bad("rope", f"contiguous [positions, rotary <= {dim}] float32 on device {dev}", rope)
    if q_out is not None:
        so = _rows("q_out", q_out, dev, dtype, m, heads, dim)
    _check_cuda(q, dev)
    if q_out is None:
        q_out = torch.empty((m, heads, dim), dtype=dtype, device=q.device)
        so = (heads * dim, dim)
    _call(dev, _lib.rope_append, _lib.PACK_ROPE_APPEND(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), rope.data_ptr(), position, slot,
        sq[0], sq[1], sk[0], sk[1], sv[0], sv[1], so[0], so[1], ck[0], ck[1], ck[2], cv[0], cv[1], cv[2], table[0], pages, m, heads, kv_heads,
        dim, table[1], page_size, interleaved, kind))
    return q_out


def tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                   context: torch.Tensor, starts: torch.Tensor, max_draft: int, tree_mask: torch.Tensor | None = None, *,
                   scale: float | None = None, gate: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every request's drafted tokens over its cache: out [M, Hq, D].

    Request b has the tokens starts[b] .. starts[b + 1] - 1 of q [M, Hq, D] (``starts`` int32 [B + 1], rising;
    a request may have none), at most ``max_draft`` (1 .. 256). Rows before starts[0] and from starts[B] on belong
    to no request (a fixed-size step's padding) and are 0. Its sequence is ``context[b]`` (int32
    [B]) cached tokens followed by the drafted ones, already appended, in the pages ``page_table[b]`` (int32
    [B, pages of a request]) of the cache [pages, Hkv, page_size, D] (page_size a power of two, 8 .. 1024).
    Each token sees the context and the drafted tokens whose bits its row of ``tree_mask`` (int32 [M, words],
    see the function of that name) sets; without a mask itself and every earlier one, so ``max_draft`` 1 is
    plain decoding. ``scale`` is 1 / sqrt(D) by default. ``gate`` [M, Hq, D] multiplies the result by its
    sigmoid. A row that sees nothing is 0. BF16 or FP16, D 64 or 128; q and gate may be strided views."""
    dev, dtype = q.get_device(), q.dtype
    kind = _TYPES.get(dtype)
    if q.dim() != 3 or kind is None:
        raise ValueError(f"q: expected [tokens, heads, dim] in bfloat16 or float16, got {tuple(q.shape)} {dtype}")
    m, heads, dim = q.shape
    sq = _rows("q", q, dev, dtype, m, heads, dim)
    (pages, kv_heads, page_size, _), ck, cv = _cache(k_pages, v_pages, dev, dtype, dim)
    requests = context.shape[0] if context.dim() else 0
    lengths, first = _vector("context", context, dev, torch.int32, requests), _vector("starts", starts, dev, torch.int32, requests + 1)
    table = _words("page_table", page_table, dev, requests)
    mask = mask_row = words = 0
    if tree_mask is not None:
        mask = _words("tree_mask", tree_mask, dev, m)
        mask_row, words = tree_mask.stride(0), tree_mask.shape[1]
    gates, sg = 0, (0, 0)
    if gate is not None:
        sg = _rows("gate", gate, dev, dtype, m, heads, dim)
        gates = gate.data_ptr()
    if out is not None:
        so = _rows("out", out, dev, dtype, m, heads, dim)
    _check_cuda(q, dev)
    if out is None:
        out = torch.empty((m, heads, dim), dtype=dtype, device=q.device)
        so = (heads * dim, dim)
    if scale is None:
        scale = dim ** -0.5
    need = _scratch_bytes(dev, max_draft, heads, kv_heads, dim)
    scratch = torch.empty(need, dtype=torch.uint8, device=q.device)
    _call(dev, _lib.tree_attention, _lib.PACK_TREE_ATTENTION(
        q.data_ptr(), gates, out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), table, lengths, first, mask, scratch.data_ptr(), need,
        sq[0], sq[1], sg[0], sg[1], so[0], so[1], ck[0], ck[1], ck[2], cv[0], cv[1], cv[2], page_table.stride(0), mask_row, pages, m, requests,
        max_draft, page_table.shape[1], words, heads, kv_heads, dim, page_size, kind, scale))
    if requests == 0:  # the entry launches nothing: every row is one of no request
        out.zero_()
    return out


@functools.lru_cache(maxsize=None)
def _scratch_bytes(dev: int, max_draft: int, heads: int, kv_heads: int, dim: int) -> int:
    """What the split of the cache needs, by the sizes that decide it."""
    with torch.cuda.device(dev):
        return _lib.tree_attention_scratch_bytes(_lib.MuseTreeAttention(max_draft=max_draft, heads=heads, kv_heads=kv_heads, dim=dim, scale=1.0))
