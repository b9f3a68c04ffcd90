"""tree_attention on the GPU against a plain 64-bit row-by-row form: single tokens, chains and trees, both head
sizes and 16-bit types, groups of every kind, contexts of 0, 1 and around page and tile edges, requests without
tokens, masks that leave rows empty, values that are infinite or NaN where no row looks, strided views, cache
layouts, streams, graphs, offsets past 32 bits, and out-of-range requests and pages. The bound on the error is
derived in serving_ref.attention64."""

import math

import numpy as np
import pytest
import torch

from muse_bf16_proj_b200 import _lib
from muse_bf16_proj_b200.attention import tree_attention, tree_mask
from serving_ref import attention64

pytestmark = pytest.mark.gpu


def device_error() -> int:
    return _lib.device_error(torch.cuda.current_stream().cuda_stream)


def make(contexts, drafts, hq, hk, d, page, dtype, seed=0, tree="random", gate=False, spread=2.0, spare=2):
    """One batch's arguments; page table entries past a request's need are -1."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    starts = np.concatenate(([0], np.cumsum(drafts)))
    n = int(starts[-1])
    width = (2 * hq + 2 * hk) * d
    y = torch.randn((max(n, 1), width), generator=g, device="cuda")
    y[:, :hq * d] *= spread
    y = y.to(dtype)[:n]
    q, gates = y[:, :hq * d].unflatten(1, (hq, d)), y[:, (hq + 2 * hk) * d:].unflatten(1, (hq, d))
    need = [-(-(c + t) // page) for c, t in zip(contexts, drafts)]
    order = torch.randperm(sum(need) + spare, generator=g, device="cuda").int()
    table = torch.full((len(need), max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    used = 0
    for b, c in enumerate(need):
        table[b, :c] = order[used:used + c]
        used += c
    cache = [torch.randn((sum(need) + spare, hk, page, d), generator=g, device="cuda").to(dtype) for _ in range(2)]
    rng = np.random.RandomState(seed)
    most = max(max(drafts), 1)
    starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
    mask = None
    if tree == "random":
        parents = [rng.randint(-1, i) if i else -1 for t in drafts for i in range(t)]
        mask = tree_mask(torch.tensor(parents, dtype=torch.int32, device="cuda"), starts, most)
    return {"q": q, "k_pages": cache[0], "v_pages": cache[1], "page_table": table,
            "context": torch.tensor(contexts, dtype=torch.int32, device="cuda"), "starts": starts, "max_draft": most,
            "tree_mask": mask, "gate": gates if gate else None}


def want(a, scale=None):
    return attention64(a["q"], a["k_pages"], a["v_pages"], a["page_table"], a["context"], a["starts"], a["tree_mask"], scale, a["gate"])


def check(a, scale=None):
    got = tree_attention(**a, scale=scale)
    out, bound = want(a, scale)
    err = (got.double() - out).abs()
    assert not torch.isnan(got).any()
    assert (err <= bound).all(), f"error {err.max().item():.3e}, {(err / bound.clamp(min=1e-30)).max().item():.2f} of its bound"
    assert device_error() == 0
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,d", [(16, 2, 64), (32, 8, 128), (5, 1, 128), (12, 4, 64), (8, 8, 128)])
def test_single_tokens(hq, hk, d, dtype):
    """Contexts around the edges of pages (16) and of 64, 128 and 256 entries."""
    check(make([0, 1, 15, 16, 17, 63, 64, 127, 128, 129, 255, 256, 700], [1] * 13, hq, hk, d, 16, dtype, seed=hq, tree=None))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,d", [(16, 2, 64), (32, 8, 128), (64, 8, 128), (3, 1, 64)])
@pytest.mark.parametrize("drafts", [[2, 3], [1, 16, 0, 7], [33, 5], [64], [0, 0, 40], [100, 9, 128]])
def test_trees(drafts, hq, hk, d, dtype):
    contexts = [(97 * b + 31) % 300 for b in range(len(drafts))]
    check(make(contexts, drafts, hq, hk, d, 16, dtype, seed=len(drafts) + d, gate=d == 64))


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 1024])
def test_page_sizes(page):
    check(make([3, 200, 511, 0, 1025], [4, 1, 9, 6, 2], 16, 2, 64, page, torch.bfloat16, seed=page))
    check(make([130, 257], [4, 17], 8, 2, 128, page, torch.bfloat16, seed=page))


@pytest.mark.parametrize("d", [64, 128])
def test_chains_without_a_mask(d):
    check(make([5, 0, 126, 1000], [1, 37, 5, 20], 8, 2, d, 32, torch.bfloat16, tree=None, gate=True))


def test_widest_draft():
    check(make([100, 3], [256, 255], 4, 1, 64, 64, torch.bfloat16))
    check(make([100, 3], [256, 255], 8, 2, 128, 64, torch.bfloat16, tree=None))


def test_long_context_is_split_and_joined():
    check(make([20000], [1], 16, 2, 64, 64, torch.bfloat16, tree=None))
    check(make([9000, 11], [3, 40], 8, 1, 128, 16, torch.bfloat16))


def test_many_requests():
    rng = np.random.RandomState(1)
    check(make([int(c) for c in rng.randint(0, 90, 300)], [int(t) for t in rng.randint(0, 4, 300)], 16, 2, 64, 8, torch.bfloat16))


@pytest.mark.parametrize("scale", [0.25, 1e-3, -0.1])
def test_scale(scale):
    check(make([77, 300], [3, 2], 16, 2, 64, 16, torch.bfloat16), scale=scale)


def test_scores_that_grow_along_the_context():
    """The running maximum moves in every tile, by far more than a 16-bit exponent in all."""
    for d, dtype in ((64, torch.bfloat16), (128, torch.float16)):
        a = make([1500], [5], 8, 2, d, 16, dtype, spread=1.0)
        pages = a["page_table"][0, :(1505 + 15) // 16].long()
        ramp = torch.arange(pages.shape[0] * 16, device="cuda", dtype=torch.float32).view(-1, 1, 16, 1) / 1505.0
        a["q"].fill_(1.0)
        for up in (True, False):
            level = ramp if up else 1.0 - ramp
            a["k_pages"][pages] = (level * 40.0).expand(-1, 2, -1, d).to(dtype) / math.sqrt(d)
            check(a)


def test_far_negative_scores():
    """Every score is far below zero: the maximum, not zero, is what they are taken against."""
    a = make([40, 200], [2, 1], 8, 2, 64, 16, torch.bfloat16)
    a["q"].fill_(-4.0)
    a["k_pages"].fill_(9.0)
    check(a)


def test_rows_that_see_nothing_are_zero():
    a = make([0, 0, 50], [3, 70, 2], 16, 2, 64, 16, torch.bfloat16, gate=True)
    a["tree_mask"][:2] = 0
    a["tree_mask"][40] = 0
    got = check(a)
    assert int(torch.count_nonzero(got[:2])) == 0 and int(torch.count_nonzero(got[40])) == 0
    # Mask bits past a request's own tokens mean nothing.
    plain = got.clone()
    a["tree_mask"][2:3] |= -8
    assert torch.equal(tree_attention(**a), plain)


@pytest.mark.parametrize("d,drafts", [(64, [1, 1, 1]), (128, [1, 5, 3]), (64, [9, 30, 17]), (128, [20, 64, 33])])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf"), 3.0e38])
def test_what_no_row_sees_does_not_matter(d, drafts, poison):
    """Pages hold anything past a request's tokens, spare pages too, and drafted tokens that a row's mask
    hides may be anything for that row; a token sees its own."""
    a = make([30, 129, 200], drafts, 8, 2, d, 16, torch.bfloat16)
    for b, (c, t) in enumerate(zip([30, 129, 200], drafts)):
        last = (c + t - 1) // 16
        page = a["page_table"][b, last].long()
        a["k_pages"][page, :, (c + t - 1) % 16 + 1:] = poison
        a["v_pages"][page, :, (c + t - 1) % 16 + 1:] = poison
    used = torch.zeros(a["k_pages"].shape[0], dtype=torch.bool, device="cuda")
    used[a["page_table"][a["page_table"] >= 0].long()] = True
    a["k_pages"][~used], a["v_pages"][~used] = poison, poison
    check(a)
    # Poison one drafted token of the last request: the rows that do not see it keep their values.
    t = drafts[-1]
    if t > 1:
        lo = int(a["starts"][2])
        a["tree_mask"][lo:] = torch.tensor([1 << min(i, 30) for i in range(t)], dtype=torch.int32, device="cuda")[:, None]
        a["tree_mask"][lo + 1:, 1:] = 0
        clean, bound = want(a)
        slot = 200 + 1
        page = a["page_table"][2, slot // 16].long()
        a["k_pages"][page, :, slot % 16], a["v_pages"][page, :, slot % 16] = poison, poison
        got = tree_attention(**a)
        rows = torch.ones(a["q"].shape[0], dtype=torch.bool, device="cuda")
        rows[lo + 1] = False
        assert ((got.double() - clean).abs() <= bound)[rows].all()
        if not math.isfinite(poison):
            assert not torch.isfinite(got[lo + 1]).any()
        assert device_error() == 0


def test_infinite_value_that_is_seen():
    """An infinite value reaches the rows that see it, in its entries alone."""
    a = make([20], [3], 4, 1, 64, 16, torch.bfloat16)
    page = a["page_table"][0, 1].long()
    a["v_pages"][page, 0, 20 + 1 - 16, 5] = float("inf")
    a["tree_mask"][:, 0] = torch.tensor([1, 3, 5], dtype=torch.int32, device="cuda")
    got = tree_attention(**a)
    assert torch.isinf(got[1, :, 5]).all() and torch.isfinite(got[1, :, :5]).all() and torch.isfinite(got[1, :, 6:]).all()
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[2]).all()


def test_cache_layouts_and_strides():
    """Keys and values as halves of one tensor with entries outside heads; q inside a wider row, out strided."""
    a = make([70, 9], [6, 2], 8, 2, 128, 16, torch.bfloat16, gate=True)
    pages = a["k_pages"].shape[0]
    both = torch.empty((pages, 16, 2, 2, 128), dtype=torch.bfloat16, device="cuda")
    both[:, :, 0], both[:, :, 1] = a["k_pages"].transpose(1, 2), a["v_pages"].transpose(1, 2)
    plain = check(a)
    a["k_pages"], a["v_pages"] = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    wide = torch.zeros((8, 3, 8, 128), dtype=torch.bfloat16, device="cuda")
    got = tree_attention(**a, out=wide[:, 1])
    assert got.data_ptr() == wide[:, 1].data_ptr() and torch.equal(wide[:, 1], plain)
    assert int(torch.count_nonzero(wide[:, 0])) == 0 and int(torch.count_nonzero(wide[:, 2])) == 0


def test_same_bits_again_on_another_stream_and_in_a_graph():
    a = make([3000, 17, 600], [8, 1, 30], 16, 2, 64, 16, torch.bfloat16, gate=True)
    first = check(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = tree_attention(**a)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = tree_attention(**a)
    # Other lengths and inputs than those captured: the lengths are read on the device.
    a["context"].copy_(torch.tensor([100, 17, 5], dtype=torch.int32))
    a["q"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    out, bound = want(a)
    assert ((got.double() - out).abs() <= bound).all()


@pytest.mark.parametrize("drafts,d", [([22, 22], 64), ([11, 9, 10], 128), ([1, 1], 128), ([3, 4], 64), ([7, 30], 128)])
def test_same_bits_whatever_ran_before(drafts, d):
    """Rows that a row tile has and the request does not, and what other kernels left in shared and tensor memory,
    have no say in a result."""
    a = make([3000 - 700 * b for b in range(len(drafts))], drafts, 12, 4, d, 64, torch.bfloat16)
    other = make([900, 30], [5, 40], 8, 2, 192 - d, 16, torch.bfloat16, spread=30.0)
    x = torch.randn((2048, 2048), device="cuda").bfloat16()
    first = tree_attention(**a)
    for before in (lambda: tree_attention(**a), lambda: tree_attention(**other), lambda: x @ x, lambda: x.zero_()):
        before()
        assert torch.equal(tree_attention(**a), first)


def test_offsets_past_32_bits():
    pages, page, hk, d = 33000, 128, 8, 128
    kp = torch.empty((pages, hk, page, d), dtype=torch.bfloat16, device="cuda")
    vp = torch.empty_like(kp)
    assert kp.numel() > 2 ** 32
    a = make([250, 100], [3, 1], 16, 8, d, page, torch.bfloat16)
    places = torch.tensor([pages - 1, 17, 32900, 2, 30000], device="cuda")[:a["k_pages"].shape[0]]
    kp[places], vp[places] = a["k_pages"], a["v_pages"]
    a["page_table"] = torch.where(a["page_table"] >= 0, places[a["page_table"].clamp(min=0).long()].int(), -1)
    a["k_pages"], a["v_pages"] = kp, vp
    check(a)


def test_no_tokens_at_all():
    a = make([5, 6], [1, 0], 4, 1, 64, 16, torch.bfloat16, tree=None)
    a["q"], a["starts"] = a["q"][:0], torch.zeros(3, dtype=torch.int32, device="cuda")
    assert tree_attention(**a).shape == (0, 4, 64)


@pytest.mark.parametrize("d", [64, 128])
def test_out_of_range_is_reported(d):
    """A request over max_draft, past its page table, or with a page outside the cache: an error code, and the
    other requests keep their results."""
    a = make([40, 60], [2, 3], 8, 2, d, 16, torch.bfloat16)
    out, bound = want(a)

    def other(got, rows):
        assert ((got.double() - out).abs() <= bound)[rows].all()

    b = dict(a, max_draft=2)
    got = tree_attention(**b)
    with pytest.raises(_lib.MuseError, match="b01"):
        device_error()
    other(got, slice(0, 2))
    b = dict(a, page_table=a["page_table"][:, :3].contiguous())
    got = tree_attention(**b)
    with pytest.raises(_lib.MuseError, match="b02"):
        device_error()
    other(got, slice(0, 2))
    for bad in (-1, a["k_pages"].shape[0]):
        table = a["page_table"].clone()
        table[0, 1] = bad
        got = tree_attention(**dict(a, page_table=table))
        with pytest.raises(_lib.MuseError, match="b03"):
            device_error()
        other(got, slice(2, 5))
    check(a)


def test_tree_mask_words():
    starts = torch.tensor([0, 3, 3, 40], dtype=torch.int32, device="cuda")
    parents = torch.tensor([-1, 0, 0] + [i - 1 for i in range(37)], dtype=torch.int32, device="cuda")
    got = tree_mask(parents, starts, 37)
    assert got.shape == (40, 2) and got[:3, 0].tolist() == [1, 3, 5]
    assert got[3 + 31].tolist() == [-1, 0] and got[39].tolist() == [-1, 31]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("drafts,hq", [([1, 1, 1], 8), ([1, 6, 1], 8), ([1, 12, 1], 8), ([1, 40, 1], 16)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_a_hidden_token_of_one_does_not_matter(drafts, hq, d, poison):
    """A request's only drafted token with an empty mask row: its own entry may hold anything, and over no context
    its row is zero. Row counts of every variant, contexts of 0, inside a tile, and over many runs."""
    a = make([0, 30, 3001], drafts, hq, 2, d, 16, torch.bfloat16, gate=True)
    for b, context in ((0, 0), (2, 3001)):
        a["tree_mask"][int(a["starts"][b])] = 0
        page = a["page_table"][b, context // 16].long()
        a["k_pages"][page, :, context % 16], a["v_pages"][page, :, context % 16] = poison, poison
    got = check(a)
    assert int(torch.count_nonzero(got[0])) == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("drafts,before,after", [([1, 1], 0, 6), ([3, 0, 9], 2, 5), ([40, 33], 3, 0), ([2, 1], 1, 3000)])
def test_rows_outside_every_request_are_zero(drafts, before, after, d):
    """Rows before the first request's and past the last one's, as a fixed-size step's padding leaves them: zero, whatever
    the output held, and the other rows as without them."""
    contexts = [(1900 * b + 5) % 2500 for b in range(len(drafts))]
    a = make(contexts, drafts, 8, 2, d, 16, torch.bfloat16, gate=True)
    plain = check(a)
    n = sum(drafts)
    rows = {name: torch.full((before + n + after,) + tuple(a[name].shape[1:]), float("nan"), dtype=a[name].dtype, device="cuda") for name in ("q", "gate")}
    for name, t in rows.items():
        t[before:before + n] = a[name]
    words = torch.full((before + n + after, a["tree_mask"].shape[1]), -1, dtype=torch.int32, device="cuda")
    words[before:before + n] = a["tree_mask"]
    b = dict(a, **rows, tree_mask=words, starts=a["starts"] + before)
    out = torch.full((before + n + after, 3, 8, d), float("nan"), dtype=torch.bfloat16, device="cuda")
    for to in (out[:, 1], None):
        got = tree_attention(**b, out=to)
        assert torch.equal(got[before:before + n], plain)
        assert int(torch.count_nonzero(got[:before])) == 0 and int(torch.count_nonzero(got[before + n:])) == 0
        assert device_error() == 0
    assert torch.isnan(out[:, 0]).all() and torch.isnan(out[:, 2]).all()


def test_rows_of_no_request_in_a_graph():
    """A captured step of fixed size whose tokens shrink: the rows that are left over become zero."""
    a = make([700, 20], [4, 4], 16, 2, 64, 16, torch.bfloat16)
    out = torch.full((8, 16, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    tree_attention(**a, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tree_attention(**a, out=out)
    a["starts"].copy_(torch.tensor([0, 4, 6], dtype=torch.int32))
    out.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    assert int(torch.count_nonzero(out[6:])) == 0
    want_, bound = want(dict(a, q=a["q"][:6]))
    assert ((out[:6].double() - want_).abs() <= bound).all()
    a["starts"].zero_()
    out.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    assert int(torch.count_nonzero(out)) == 0 and device_error() == 0


def test_starts_out_of_order_keep_the_other_requests():
    """A request whose end is before its start is reported, and rows that another one has keep their results."""
    a = make([40, 60, 9], [5, 0, 0], 8, 2, 64, 16, torch.bfloat16)
    plain = check(a)
    for starts in ([0, 5, 3, 3], [0, 5, 2, 1]):
        got = tree_attention(**dict(a, starts=torch.tensor(starts, dtype=torch.int32, device="cuda")))
        with pytest.raises(_lib.MuseError, match="b01"):
            device_error()
        assert torch.equal(got, plain)


def test_tokens_without_any_request_are_zero():
    a = make([5], [3], 4, 1, 64, 16, torch.bfloat16, tree=None)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    for to in (None, torch.full((3, 4, 64), float("nan"), dtype=torch.bfloat16, device="cuda")):
        got = tree_attention(a["q"], a["k_pages"], a["v_pages"], a["page_table"][:0], none, a["starts"][:1], 1, out=to)
        assert got.shape == (3, 4, 64) and int(torch.count_nonzero(got)) == 0 and (to is None or got is to)
    assert device_error() == 0


@pytest.mark.parametrize("draft,hq,d", [(1, 8, 64), (1, 8, 128), (6, 8, 128), (9, 8, 64), (40, 16, 128)])
@pytest.mark.parametrize("below", [17.0, 18.5, 20.0])
def test_fp16_weights_far_below_the_largest(draft, hq, d, below):
    """One cached token whose score is `below` above every other one's, over a long context: the others' weights, each under
    fp16's normal range against the largest, are a share of the result that must not be lost. (Enough requests over the
    same pages that a CTA walks a whole context by itself.)

    Bound. A weight is held against a reference at least 2^7 below fp16's range above the largest one, so its absolute
    rounding step is 2^-25 / 2^7 of the largest weight: n steps of it times max |V| in the numerator and in the denominator.
    Beside that the chain of attention64: p's relative rounding twice, FP32 sums, the scores, one rounding of the result."""
    n, hk, requests, t, at = 60000, 2, 150, draft, 5
    a = make([n], [t], hq, hk, d, 64, torch.float16, tree=None)
    a["q"] = torch.ones((requests * t, hq, d), dtype=torch.float16, device="cuda")
    a["page_table"] = a["page_table"].expand(requests, -1)
    a["context"] = a["context"].expand(requests).contiguous()
    a["starts"] = torch.arange(requests + 1, dtype=torch.int32, device="cuda") * t
    a["k_pages"].zero_()
    a["v_pages"].fill_(1.0)
    page = a["page_table"][0, 0].long()
    a["k_pages"][page, :, at] = below / math.sqrt(d)
    a["v_pages"][page, :, at] = 0.0
    level = a["k_pages"][page, 0, at, 0].double().item() * d * d ** -0.5  # as fp16 holds it
    got = tree_attention(**a).double().view(requests, t, hq, d)
    u = 2.0 ** -11
    for i in range(t):
        rest = (n + i) * math.exp(-level)  # the token itself and every earlier one but the largest: n + i
        out = rest / (1.0 + rest)
        bound = (2 * u + 2.0 ** -16 + 2 * level * 2.0 ** -18) * out + 2 * (n + i) * 2.0 ** -32
        err = (got[:, i] - out).abs().max().item()
        assert err <= bound + u * (out + bound), (i, err, out)
    assert device_error() == 0


@pytest.mark.parametrize("prompt,context,hq,hk,d", [(600, 100, 8, 2, 64), (513, 0, 4, 1, 128)])
def test_a_prompt_in_pieces(prompt, context, hq, hk, d):
    """A prompt of more than 256 tokens as requests of up to 256 over the same pages, each after the ones before it, against
    the prompt as one request of the 64-bit form."""
    a = make([context], [prompt], hq, hk, d, 16, torch.bfloat16, tree=None, gate=True)
    out, bound = want(a)
    starts = list(range(0, prompt, 256)) + [prompt]
    pieces = len(starts) - 1
    got = tree_attention(a["q"], a["k_pages"], a["v_pages"], a["page_table"].expand(pieces, -1),
                         torch.tensor([context + s for s in starts[:-1]], dtype=torch.int32, device="cuda"),
                         torch.tensor(starts, dtype=torch.int32, device="cuda"), 256, gate=a["gate"])
    assert ((got.double() - out).abs() <= bound).all() and device_error() == 0
