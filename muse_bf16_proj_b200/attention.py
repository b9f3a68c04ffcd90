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

The cache is two tensors [pages, kv_heads, page_size, dim] (any page, head and entry strides). Request b
keeps its tokens in the pages of row b of ``page_table``; a token's *slot* is page * page_size + entry
(``page_slots``). Calls launch on torch's current stream, allocate with torch's caching allocator only,
do not synchronise and can be captured in a CUDA graph. A position, slot, page or request size out of
its range is found on the device and recorded in the device error word (``_lib.device_error``).
"""

from __future__ import annotations

import math

import torch

from . import _lib

_TYPES = {torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}
MAX_DRAFT = 256  # drafted tokens of one request


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
    """int64 slots of the tokens ``index`` (place in the request's sequence) of requests ``request``."""
    index = index.long()
    return page_table[request.long(), index // page_size].long() * page_size + index % page_size


def tree_mask(parents: torch.Tensor, starts: torch.Tensor, max_draft: int) -> torch.Tensor:
    """The mask words [tokens, ceil(max_draft / 32)] int32 of drafted trees: ``parents`` [tokens] is each
    token's parent as an index among its request's drafted tokens (-1 for a root), earlier than the token
    itself; a token sees itself and its ancestors. Made once a step, on the tensors' device."""
    n, words = parents.shape[0], (max_draft + 31) // 32
    device = parents.device
    token = torch.arange(n, device=device)
    owner = torch.bucketize(token, starts[1:].long(), right=True)
    first = starts.long()[owner]
    bits = torch.zeros((n, words * 32), dtype=torch.bool, device=device)
    bits[token, token - first] = True
    at = parents.long()
    for _ in range(max_draft):  # one level of ancestors a turn
        live = at >= 0
        bits[token, at.clamp(min=0)] |= live
        at = torch.where(live, parents.long()[(first + at.clamp(min=0)).clamp(max=max(n - 1, 0))], -1)
    weight = 1 << torch.arange(32, device=device, dtype=torch.int64)
    packed = (bits.view(n, words, 32).long() * weight).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).int()


def _check_rows(name: str, t: torch.Tensor, device, dtype, dim: int) -> None:
    if t.dim() != 3 or t.dtype != dtype or t.device != device or t.shape[2] != dim or t.stride(2) != 1:
        raise ValueError(f"{name}: expected [tokens, heads, {dim}] {dtype} on {device} with contiguous rows, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device} with strides {t.stride()}")


def _check_cache(k_pages: torch.Tensor, v_pages: torch.Tensor, device, dtype, kv_heads: int | None, dim: int):
    shape = k_pages.shape
    if (k_pages.dim() != 4 or v_pages.shape != shape or shape[3] != dim or (kv_heads is not None and shape[1] != kv_heads) or
            k_pages.dtype != dtype or v_pages.dtype != dtype or k_pages.device != device or v_pages.device != device or
            k_pages.stride(3) != 1 or v_pages.stride(3) != 1):
        raise ValueError(f"k_pages, v_pages: expected [pages, {kv_heads if kv_heads is not None else 'kv_heads'}, page_size, {dim}] "
                         f"{dtype} on {device}, got {tuple(shape)} {k_pages.dtype} on {k_pages.device} and "
                         f"{tuple(v_pages.shape)} {v_pages.dtype} on {v_pages.device}")
    return shape


def _check_vector(name: str, t: torch.Tensor, device, dtype, n: int) -> None:
    if t.dim() != 1 or t.shape[0] != n or t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: expected contiguous [{n}] {dtype} on {device}, got {tuple(t.shape)} {t.dtype} on {t.device}")


def _check_cuda(device: torch.device) -> None:
    if device.type != "cuda":
        raise ValueError(f"expected CUDA tensors, got {device}")


def _on(device: torch.device, call, args) -> None:
    """``call(args, stream)`` on the tensors' device, which need not be the current one."""
    stream = torch.cuda.current_stream(device).cuda_stream
    if device.index == torch.cuda.current_device():
        call(args, stream)
    else:
        with torch.cuda.device(device):
            call(args, stream)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                k_pages: torch.Tensor, v_pages: torch.Tensor, rope: torch.Tensor, *, interleaved: bool = False,
                q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Turns q [M, Hq, D] and k [M, Hkv, D] by their tokens' ``positions`` (int32 [M]), writes k and v into the
    cache at ``slots`` (int64 [M], distinct; negative: not appended) and returns the turned q (``q_out``, which
    may be q itself, or a new contiguous tensor). BF16 or FP16, D 64 or 128; q, k, v may be strided views of
    one projection output. ``rope``: FP32 [positions, rotary] (``rope_table``); pairs are (i, i + rotary / 2),
    or (2i, 2i + 1) when ``interleaved``; entries past ``rotary`` are left as they are."""
    device, dtype = q.device, q.dtype
    if q.dim() != 3 or dtype not in _TYPES:
        raise ValueError(f"q: expected [tokens, heads, dim] in bfloat16 or float16, got {tuple(q.shape)} {dtype}")
    m, heads, dim = q.shape
    _check_rows("q", q, device, dtype, dim)
    _check_rows("k", k, device, dtype, dim)
    _check_rows("v", v, device, dtype, dim)
    kv_heads = k.shape[1]
    if k.shape != v.shape or k.shape[0] != m:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not go with q {tuple(q.shape)}")
    pages, _, page_size, _ = _check_cache(k_pages, v_pages, device, dtype, kv_heads, dim)
    _check_vector("positions", positions, device, torch.int32, m)
    _check_vector("slots", slots, device, torch.int64, m)
    if rope.dim() != 2 or rope.dtype != torch.float32 or rope.device != device or not rope.is_contiguous() or rope.shape[1] > dim:
        raise ValueError(f"rope: expected contiguous [positions, rotary <= {dim}] float32 on {device}, got {tuple(rope.shape)} "
                         f"{rope.dtype} on {rope.device}")
    if q_out is not None:
        _check_rows("q_out", q_out, device, dtype, dim)
        if q_out.shape != q.shape:
            raise ValueError(f"q_out {tuple(q_out.shape)} is not q's shape {tuple(q.shape)}")
    _check_cuda(device)
    if q_out is None:
        q_out = torch.empty((m, heads, dim), dtype=dtype, device=device)
    sq, sk, sv, so, ck, cv = q.stride(), k.stride(), v.stride(), q_out.stride(), k_pages.stride(), v_pages.stride()
    args = _lib.MuseRopeAppend(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), rope.data_ptr(),
        positions.data_ptr(), slots.data_ptr(), sq[0], sq[1], sk[0], sk[1], sv[0], sv[1], so[0], so[1], ck[0], ck[1], ck[2],
        cv[0], cv[1], cv[2], rope.shape[0], pages, m, heads, kv_heads, dim, rope.shape[1], page_size, interleaved,
        _TYPES[dtype])
    _on(device, _lib.rope_append, args)
    return q_out


def tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                   context: torch.Tensor, starts: torch.Tensor, max_draft: int, tree_mask: torch.Tensor | None = None, *,
                   scale: float | None = None, gate: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every request's drafted tokens over its cache: out [M, Hq, D].

    Request b has the tokens starts[b] .. starts[b + 1] - 1 of q [M, Hq, D] (``starts`` int32 [B + 1], from 0
    to M; a request may have none), at most ``max_draft`` (1 .. 256). Its sequence is ``context[b]`` (int32
    [B]) cached tokens followed by the drafted ones, already appended, in the pages ``page_table[b]`` (int32
    [B, pages of a request]) of the cache [pages, Hkv, page_size, D] (page_size a power of two, 8 .. 1024).
    Each token sees the context and the drafted tokens whose bits its row of ``tree_mask`` (int32 [M, words],
    see the function of that name) sets; without a mask itself and every earlier one, so ``max_draft`` 1 is
    plain decoding. ``scale`` is 1 / sqrt(D) by default. ``gate`` [M, Hq, D] multiplies the result by its
    sigmoid. A row that sees nothing is 0. BF16 or FP16, D 64 or 128; q and gate may be strided views."""
    device, dtype = q.device, q.dtype
    if q.dim() != 3 or dtype not in _TYPES:
        raise ValueError(f"q: expected [tokens, heads, dim] in bfloat16 or float16, got {tuple(q.shape)} {dtype}")
    m, heads, dim = q.shape
    _check_rows("q", q, device, dtype, dim)
    pages, kv_heads, page_size, _ = _check_cache(k_pages, v_pages, device, dtype, None, dim)
    requests = context.shape[0]
    _check_vector("context", context, device, torch.int32, requests)
    _check_vector("starts", starts, device, torch.int32, requests + 1)
    if page_table.dim() != 2 or page_table.shape[0] != requests or page_table.dtype != torch.int32 or page_table.device != device or (
            page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError(f"page_table: expected [{requests}, pages] int32 on {device} with contiguous rows, got "
                         f"{tuple(page_table.shape)} {page_table.dtype} on {page_table.device}")
    mask_ptr = mask_row = words = 0
    if tree_mask is not None:
        if tree_mask.dim() != 2 or tree_mask.shape[0] != m or tree_mask.dtype != torch.int32 or tree_mask.device != device or (
                tree_mask.stride(1) != 1 and tree_mask.shape[1] > 1):
            raise ValueError(f"tree_mask: expected [{m}, words] int32 on {device} with contiguous rows, got {tuple(tree_mask.shape)} "
                             f"{tree_mask.dtype} on {tree_mask.device}")
        mask_ptr, mask_row, words = tree_mask.data_ptr(), tree_mask.stride(0), tree_mask.shape[1]
    gate_ptr = gate_token = gate_head = 0
    if gate is not None:
        _check_rows("gate", gate, device, dtype, dim)
        if gate.shape != q.shape:
            raise ValueError(f"gate {tuple(gate.shape)} is not q's shape {tuple(q.shape)}")
        gate_ptr, gate_token, gate_head = gate.data_ptr(), gate.stride(0), gate.stride(1)
    if out is not None:
        _check_rows("out", out, device, dtype, dim)
        if out.shape != q.shape:
            raise ValueError(f"out {tuple(out.shape)} is not q's shape {tuple(q.shape)}")
    _check_cuda(device)
    if out is None:
        out = torch.empty((m, heads, dim), dtype=dtype, device=device)
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    sq, so, ck, cv = q.stride(), out.stride(), k_pages.stride(), v_pages.stride()
    args = _lib.MuseTreeAttention(
        q.data_ptr(), gate_ptr, out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(),
        context.data_ptr(), starts.data_ptr(), mask_ptr, 0, 0, sq[0], sq[1], gate_token, gate_head, so[0], so[1], ck[0],
        ck[1], ck[2], cv[0], cv[1], cv[2], page_table.stride(0), mask_row, pages, m, requests, max_draft,
        page_table.shape[1], words, heads, kv_heads, dim, page_size, _TYPES[dtype], scale)
    scratch = torch.empty(_scratch_bytes(args, device), dtype=torch.uint8, device=device)
    args.scratch, args.scratch_bytes = scratch.data_ptr(), scratch.numel()
    _on(device, _lib.tree_attention, args)
    return out


_scratch_need: dict = {}


def _scratch_bytes(args: _lib.MuseTreeAttention, device: torch.device) -> int:
    """What the split of the cache needs, by the sizes that decide it."""
    key = (device.index, args.requests, args.max_draft, args.heads, args.kv_heads, args.dim)
    need = _scratch_need.get(key)
    if need is None:
        with torch.cuda.device(device):
            need = _lib.tree_attention_scratch_bytes(args)
        _scratch_need[key] = need
    return need
