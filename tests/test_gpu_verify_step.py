"""The verify step's five operators in a row on the GPU against the same chain in 64 bits, rounded to BF16 where the
step hands BF16 on; the appended cache entries; the experts from the step's own logits; and the step as a graph.

Bounds: a projection rounds once (2^-8) and sums 8192 (or 1024) products in FP32; what differs by a rounding at one
stage spreads through the next with weight at most 1 in norm, so relative norms of 2^-8 a stage add: three stages
(qkv_gate, rotary, attention with its P) to the attention output, four to y, doubled."""

import pytest
import torch

from muse_bf16_proj_b200 import _lib
from muse_bf16_proj_b200.attention import rope_table
from muse_bf16_proj_b200.contract import generate_weights
from muse_bf16_proj_b200.routing import route
from muse_bf16_proj_b200.submission import prepare, project
from muse_bf16_proj_b200.verify_step import DIM, HEADS, KV_HEADS, make_batch, random_trees, verify_step
from serving_ref import attention64, rope64, route64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    weights = {name: w for name, w in generate_weights().items() if name in ("qkv_gate", "o", "router")}
    return weights, prepare(weights, verbose=False)


@pytest.mark.parametrize("contexts,drafts,page", [([300, 17, 1000], [7, 1, 12], 16), ([0, 129], [1, 1], 32), ([64, 2000, 5, 90], [16, 16, 16, 16], 64)])
def test_step_against_64_bits(model, contexts, drafts, page):
    weights, state = model
    batch, pages = make_batch(contexts, random_trees(drafts, seed=page), page)
    g = torch.Generator(device="cuda").manual_seed(page)
    cache = tuple(torch.randn((pages, KV_HEADS, page, DIM), generator=g, device="cuda").bfloat16() for _ in range(2))
    x = torch.randn((sum(drafts), 8192), generator=g, device="cuda").bfloat16()
    balance = 0.05 * torch.randn(256, generator=g, device="cuda")
    rope = rope_table(DIM, max(contexts) + max(drafts) + 1)
    got = verify_step(x, state, cache, batch, rope, balance)
    torch.cuda.synchronize()
    assert _lib.device_error(torch.cuda.current_stream().cuda_stream) == 0

    qkvg = (x.double() @ weights["qkv_gate"].double().T).bfloat16().unflatten(1, (36, DIM))
    q = rope64(qkvg[:, :HEADS], batch["positions"], rope, False)[0].bfloat16()
    k = rope64(qkvg[:, HEADS:HEADS + KV_HEADS], batch["positions"], rope, False)[0].bfloat16()
    v, gate = qkvg[:, HEADS + KV_HEADS:HEADS + 2 * KV_HEADS], qkvg[:, HEADS + 2 * KV_HEADS:]
    at, off = batch["slots"] // page, batch["slots"] % page
    for pages_, new in zip(cache, (k, v)):
        have = pages_[at, :, off].double()
        assert (have - new.double()).norm() <= 2 * 2.0 ** -8 * new.double().norm()
        pages_[at, :, off] = new
    want, _ = attention64(q, *cache, batch["page_table"], batch["context"], batch["starts"], batch["tree_mask"], None, gate)
    assert (got["attention"].double() - want).norm() <= 2 * 3 * 2.0 ** -8 * want.norm()
    y = want.bfloat16().double().flatten(1) @ weights["o"].double().T
    assert (got["y"].double() - y).norm() <= 2 * 4 * 2.0 ** -8 * y.norm()
    w64, e64 = route64(project(x, state, "router"), 8, "sigmoid", balance, 8, 4, True, 1.0)
    same = (got["experts"].cpu() == e64).all(1)
    assert same.float().mean() > 0.9  # 32-bit and 64-bit choices may order a near tie differently
    assert ((got["weights"].cpu().double() - w64)[same].abs() <= 1e-5 * w64[same]).all()


def test_step_as_a_graph(model):
    _, state = model
    batch, pages = make_batch([500, 40], random_trees([8, 3]), 16)
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = tuple(torch.randn((pages, KV_HEADS, 16, DIM), generator=g, device="cuda").bfloat16() for _ in range(2))
    x = torch.randn((11, 8192), generator=g, device="cuda").bfloat16()
    rope = rope_table(DIM, 600)
    eager = verify_step(x, state, cache, batch, rope)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = verify_step(x, state, cache, batch, rope)
    for t in captured.values():
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for name, t in eager.items():
        assert torch.equal(t, captured[name]), name


def test_other_experts_are_near_ties(model):
    """Where the step's choice differs from the 64-bit one of its own logits, the experts (or groups) that changed places are
    worth the same to within 32-bit rounding. A score up to 1 is off by at most 2^-22 (exp 2^-23, its sum with 1 and the
    quotient 2^-24 each), score + bias by 2^-24 more, and two of them are compared: under 2^-20. A group's worth adds two
    with one rounding more: under 2^-19."""
    _, state = model
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((700, 8192), generator=g, device="cuda").bfloat16()
    balance = 0.05 * torch.randn(256, generator=g, device="cuda")
    logits = project(x, state, "router")
    _, experts = route(logits, 8, scoring="sigmoid", bias=balance, groups=8, top_groups=4)
    _, exact = route64(logits, 8, "sigmoid", balance, 8, 4, True, 1.0)
    choice = torch.sigmoid(logits.double().cpu()) + balance.double().cpu()
    worth = choice.view(-1, 8, 32).topk(2, dim=-1)[0].sum(-1)
    for t in torch.nonzero((experts.cpu() != exact).any(1))[:, 0].tolist():
        kept = worth[t].topk(4)
        limit, groups = kept[0][-1].item(), set((experts[t].cpu() // 32).tolist())
        assert all(worth[t, group].item() >= limit - 2.0 ** -19 for group in groups), t
        if groups <= set(kept[1].tolist()) and set((exact[t] // 32).tolist()) <= set(kept[1].tolist()):
            mine, other = choice[t][experts[t].cpu().long()], choice[t][exact[t].long()]
            assert ((mine - other).abs() <= 2.0 ** -20).all(), t
