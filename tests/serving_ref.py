"""Plain 64-bit forms of the operators between the projections, loop by loop, for the tests."""

import math

import torch

# Unit roundoff of the 16-bit types, and the smallest step they keep.
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
STEP = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def rope64(x, positions, table, interleaved):
    """(turned x, sum of the magnitudes that enter each entry) in 64 bits."""
    x = x.double()
    out, size = x.clone(), x.abs()
    half = table.shape[1] // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c = table[positions.long(), i].double()[:, None]
        s = table[positions.long(), half + i].double()[:, None]
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * (c.abs() + s.abs())
    return out, size


def sequence(pages, table_row, n):
    """The first n tokens [n, kv_heads, dim] of a request, from its pages."""
    page = pages.shape[2]
    need = (n + page - 1) // page
    return pages[table_row[:need].long()].transpose(1, 2).reshape(-1, pages.shape[1], pages.shape[3])[:n].double()


def seen_rows(tree_mask, lo, t, context, device):
    """[t, context + t]: what each drafted token sees."""
    seen = torch.ones((t, context + t), dtype=torch.bool, device=device)
    if tree_mask is None:
        seen[:, context:] = torch.tril(torch.ones((t, t), dtype=torch.bool, device=device))
    else:
        words = tree_mask[lo:lo + t].long()
        for j in range(t):
            seen[:, context + j] = (words[:, j // 32] >> (j % 32)) & 1 == 1
    return seen


def attention64(q, k_pages, v_pages, page_table, context, starts, tree_mask=None, scale=None, gate=None):
    """(out, bound on the kernel's error) in 64 bits.

    The kernel's chain: scores with FP32 accumulation (64 or 128 exact 16-bit products: at most 2^-18 of the sum
    of their magnitudes), p = exp2 of them (relative 2^-20), p rounded to 16 bits (u, and in the numerator and
    in the denominator), FP32 sums (2^-16 covers the lengths tested), one rounding of the result (u). Entries of
    16-bit p below the type's normal range are off by an absolute half step, at most 2^-25 of the row's largest."""
    n, hq, d = q.shape
    hk = k_pages.shape[1]
    u = ROUND[q.dtype]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros((n, hq, d), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    starts, contexts = starts.tolist(), context.tolist()
    for b, ctx in enumerate(contexts):
        lo, t = starts[b], starts[b + 1] - starts[b]
        if t == 0:
            continue
        keys, values = sequence(k_pages, page_table[b], ctx + t), sequence(v_pages, page_table[b], ctx + t)
        seen = seen_rows(tree_mask, lo, t, ctx, q.device)
        for h in range(hq):
            k, v = keys[:, h // (hq // hk)], values[:, h // (hq // hk)]
            rows = q[lo:lo + t, h].double()
            for i in range(t):  # row by row: what a row does not see is not even multiplied
                at = torch.nonzero(seen[i])[:, 0]
                if at.numel() == 0:
                    continue
                s = (k[at] @ rows[i]) * scale
                size = (k[at].abs() @ rows[i].abs()).max().item() * abs(scale)
                p = torch.softmax(s, 0)
                out[lo + i, h] = p @ v[at]
                spread = p @ v[at].abs()
                bound[lo + i, h] = (2 * u + 2.0 ** -16 + 2 * size * 2.0 ** -18) * spread
                if q.dtype == torch.float16:
                    bound[lo + i, h] += 2.0 ** -25 * at.numel() * v[at].abs().amax(0) * p.max()
    if gate is not None:
        turn = torch.sigmoid(gate.double())
        out, bound = out * turn, bound * turn + out.abs() * turn * 2.0 ** -20
    return out, bound + u * (out.abs() + bound) + STEP[q.dtype]


def route64(logits, top_k, scoring, bias, groups, top_groups, renormalize, scale):
    """(weights, experts), token by token, in 64 bits with ties to the lowest index."""
    x = logits.double().cpu()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    m, e = x.shape
    add = None if bias is None else bias.double().cpu()
    weights, experts = torch.zeros((m, top_k), dtype=torch.float64), torch.zeros((m, top_k), dtype=torch.int32)
    for t in range(m):
        row = x[t]
        if scoring == "sigmoid":
            score = torch.sigmoid(row)
        else:
            top = row.max()
            raised = torch.exp(row - top) if top > -math.inf else torch.zeros(e, dtype=torch.float64)
            score = raised / raised.sum() if top > -math.inf else raised
        choice = row.clone() if add is None else torch.where(row == -math.inf, row, score + add)
        size = e // groups
        worth = []
        for g in range(groups):
            best = sorted(choice[g * size:(g + 1) * size].tolist(), reverse=True)
            worth.append(best[0] if add is None or size == 1 else best[0] + best[1])
        kept = sorted(range(groups), key=lambda g: (-worth[g], g))[:top_groups]
        open_ = [i for i in range(e) if i // size in kept]
        chosen = sorted(open_, key=lambda i: (-choice[i].item(), i))[:top_k]
        w = score[chosen]
        if renormalize:
            w = w / w.sum() if w.sum() > 0 else torch.zeros_like(w)
        weights[t], experts[t] = w * scale, torch.tensor(chosen, dtype=torch.int32)
    return weights, experts
