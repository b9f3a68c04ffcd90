"""route on the GPU against a plain 64-bit token-by-token form: both scorings, bias, groups, every logit type,
odd expert counts and strides, ties, masked and NaN logits, a single token. Choices are compared on logits whose
scores lie apart (a shuffled grid), so that the 32-bit and 64-bit orders agree; weights are a few FP32 roundings:
exp and the division (4 of 2^-24 with the argument's), a sum of at most 1024 terms pairwise over lanes and in
order inside one (48 additions at most), so 64 roundings bound them."""

import math

import pytest
import torch

from muse_bf16_proj_b200 import _lib
from muse_bf16_proj_b200.routing import route
from serving_ref import route64

pytestmark = pytest.mark.gpu
REL = 64 * 2.0 ** -24


def grid_logits(m, e, seed, dtype=torch.float32):
    """Shuffled, distinct, evenly spaced logits in [-3, 3) a row (exact in BF16 up to 192 experts)."""
    g = torch.Generator().manual_seed(seed)
    step = 6.0 / 2 ** math.ceil(math.log2(max(e, 2)))
    rows = torch.stack([torch.randperm(e, generator=g) for _ in range(m)])
    return ((rows - e // 2) * step).to(dtype).cuda()


def check(logits, top_k, **kw):
    got_w, got_e = route(logits, top_k, **kw)
    want_w, want_e = route64(logits, top_k, kw.get("scoring", "softmax"), kw.get("bias"), kw.get("groups", 1),
                             kw.get("top_groups", 1), kw.get("renormalize", True), kw.get("scale", 1.0))
    assert got_w.dtype == torch.float32 and got_e.dtype == torch.int32 and got_w.shape == got_e.shape == (logits.shape[0], top_k)
    assert torch.equal(got_e.cpu(), want_e)
    assert ((got_w.cpu().double() - want_w).abs() <= REL * want_w.abs() + 1e-37).all()
    assert _lib.device_error(torch.cuda.current_stream().cuda_stream) == 0
    return got_w, got_e


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("m,e,k", [(1, 256, 8), (5, 256, 1), (3, 8, 8), (7, 60, 6), (130, 64, 2), (2, 1, 1), (9, 129, 32), (4, 1000, 7),
                                   (3, 1024, 16), (6, 384, 6), (2, 31, 31)])
def test_route(m, e, k, scoring, renormalize):
    check(grid_logits(m, e, m + e), k, scoring=scoring, renormalize=renormalize, scale=2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,groups,top_groups,k", [(256, 8, 4, 8), (64, 4, 1, 6), (60, 4, 2, 5), (32, 32, 7, 7), (100, 20, 3, 15),
                                                   (96, 3, 3, 12), (1024, 16, 2, 8), (12, 6, 6, 12)])
def test_groups_and_bias(e, groups, top_groups, k, scoring):
    logits = grid_logits(17, e, e)
    check(logits, k, scoring=scoring, groups=groups, top_groups=top_groups)
    if scoring == "sigmoid":
        # A bias on a grid of its own: scores + bias stay apart by far more than FP32 rounds.
        bias = (torch.arange(e) * 0.37 % 1.0).cuda() * 0.5
        check(logits, k, scoring=scoring, groups=groups, top_groups=top_groups, bias=bias)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("e,pad,shift", [(64, 0, 0), (100, 3, 0), (60, 4, 1), (256, 8, 4)])
def test_types_and_strides(dtype, e, pad, shift):
    wide = torch.zeros((11, e + pad + shift), dtype=dtype, device="cuda")
    view = wide[:, shift:shift + e]
    view.copy_(grid_logits(11, min(e, 192), 3, dtype)[:, :e] if e <= 192 else torch.cat(
        (grid_logits(11, 128, 3, dtype), grid_logits(11, 128, 4, dtype) - 8.0), 1))
    check(view, 5, scoring="sigmoid", groups=2 if e % 2 == 0 else 1, top_groups=1)
    check(view, 5, scoring="softmax", renormalize=False)


def test_ties_go_to_the_lowest_index():
    logits = torch.zeros((3, 100), device="cuda")
    logits[1, 50:] = -0.0
    logits[2, ::7] = 1.0
    _, e = check(logits, 9)
    assert e[0].tolist() == list(range(9)) and e[1].tolist() == list(range(9)) and e[2].tolist() == list(range(0, 63, 7))
    _, e = check(logits, 4, scoring="sigmoid", bias=torch.zeros(100, device="cuda"), groups=4, top_groups=2)
    assert e[0].tolist() == [0, 1, 2, 3]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masked_and_nan_experts(scoring):
    inf = float("inf")
    logits = grid_logits(6, 64, 5)
    logits[0, 10:] = -inf           # ten experts left
    logits[1] = -inf                # none left
    logits[2, 3] = float("nan")
    logits[3, :] = torch.finfo(torch.float32).min
    logits[4, 20:60] = torch.finfo(torch.float32).min
    w, e = check(logits, 12, scoring=scoring)
    assert torch.isfinite(w).all() and (w[1] == 0).all() and e[1].tolist() == list(range(12))
    assert (w[0, 10:] == 0).all() and 3 not in e[2].tolist()
    check(logits, 12, scoring=scoring, bias=torch.full((64,), 5.0, device="cuda"))
    check(logits, 12, scoring=scoring, renormalize=False, groups=8, top_groups=2)


def test_large_logits_do_not_overflow():
    logits = grid_logits(4, 128, 8) * 30.0 + 1000.0
    check(logits, 6)
    check(-logits, 6, renormalize=False)


def test_many_tokens_streams_and_graph():
    logits = grid_logits(64, 256, 9).repeat(130, 1)[:8193]
    bias = (torch.arange(256) * 0.37 % 1.0).cuda() * 0.5
    kw = dict(scoring="sigmoid", bias=bias, groups=8, top_groups=4, scale=2.5)
    w, e = route(logits, 8, **kw)
    w64, e64 = check(logits[:64], 8, **kw)
    assert torch.equal(e, e64.repeat(130, 1)[:8193]) and torch.equal(w, w64.repeat(130, 1)[:8193])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w2, e2 = route(logits, 8, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(w, w2) and torch.equal(e, e2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w3, e3 = route(logits, 8, **kw)
    logits.copy_(logits.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(w3, w.flip(0)) and torch.equal(e3, e.flip(0))


def test_same_bits_as_elementary_operations():
    """score + bias as separate torch operations: the same choices, near ties included."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((20000, 256), generator=g, device="cuda")
    bias = torch.randn(256, generator=g, device="cuda") * 0.05
    _, e = route(x, 8, scoring="sigmoid", bias=bias)
    choice = 1.0 / (1.0 + torch.exp(-x)) + bias
    assert torch.equal(e.long(), choice.sort(dim=-1, descending=True, stable=True)[1][:, :8])


def test_no_tokens():
    w, e = route(torch.zeros((0, 64), device="cuda"), 4)
    assert w.shape == e.shape == (0, 4)


def test_bias_written_just_before():
    """A balance bias that the previous launch wrote counts, another every time."""
    logits = grid_logits(64, 256, 5)
    offsets = (torch.arange(256, device="cuda") % 7 - 3).float() / 4
    bias = torch.zeros(256, device="cuda")
    graph = torch.cuda.CUDAGraph()
    route(logits, 8, scoring="sigmoid", bias=bias, groups=8, top_groups=4)
    with torch.cuda.graph(graph):
        bias.copy_(offsets)
        _, e = route(logits, 8, scoring="sigmoid", bias=bias, groups=8, top_groups=4)
        offsets.copy_(offsets.roll(1))
    for _ in range(5):
        want = route64(logits, 8, "sigmoid", offsets.clone(), 8, 4, True, 1.0)[1]
        graph.replay()
        assert torch.equal(e.cpu(), want)


@pytest.mark.parametrize("experts", [32, 24])
def test_an_infinite_bias_in_a_masked_group(experts):
    """An expert with a bias of +inf whose group is masked but for it: the group is worth +inf (not inf - inf), and no more than
    ``top_groups`` groups take part."""
    size = experts // 4
    g = torch.Generator(device="cuda").manual_seed(experts)
    logits = torch.randn((50, experts), generator=g, device="cuda")
    logits[:, 2 * size:3 * size] = -float("inf")
    forced = 2 * size + 3
    logits[:, forced] = 0.25
    bias = 0.05 * torch.randn(experts, generator=g, device="cuda")
    bias[forced] = float("inf")
    top_k = size + 1
    weights, chosen = route(logits, top_k, scoring="sigmoid", bias=bias, groups=4, top_groups=2, renormalize=False)
    scores = torch.sigmoid(logits.double())
    choice = (scores + bias.double()).cpu()
    worth = choice.view(50, 4, size).topk(2, dim=-1)[0].sum(-1)
    worth[:, 2] = -float("inf")  # the other of the two groups
    best = worth.argmax(1)
    for t in range(50):
        order = choice[t, best[t] * size:(best[t] + 1) * size].argsort(descending=True) + best[t] * size
        assert chosen[t].tolist() == [forced] + order.tolist()
    assert ((weights.double() - torch.gather(scores, 1, chosen.long())).abs() <= 2.0 ** -22).all()
    assert _lib.device_error(torch.cuda.current_stream().cuda_stream) == 0
