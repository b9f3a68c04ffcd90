"""One verify step of the layers this library projects, end to end on one GPU's share:

    qkv_gate projection -> rotary positions, keys and values appended to the paged cache -> attention of every
    request's drafted tree over its cache, gated -> o projection;  router projection -> experts and weights.

``python -m muse_bf16_proj_b200.verify_step`` builds random weights of the reference problem's shapes (16 query
heads, 2 key/value heads and a gate of 16 heads, of 64 each; 256 experts), a paged cache with requests of unequal
length and a random tree of drafted tokens for each, runs the step eagerly and as a CUDA graph, checks that both
give the same bits and prints the time of a step. One drafted token a request is plain decoding.
"""

from __future__ import annotations

import argparse

import torch

from . import _lib
from .attention import page_slots, rope_append, rope_table, split_qkv_gate, tree_attention, tree_mask
from .contract import LAYERS, generate_weights
from .routing import route
from .submission import prepare, project

HEADS, KV_HEADS, DIM = 16, 2, 64  # one GPU's share of qkv_gate: (16 + 2 + 2 + 16) x 64 = 2304 rows
TOP_K, GROUPS, TOP_GROUPS = 8, 8, 4


def verify_step(x: torch.Tensor, state: dict, cache: tuple, batch: dict, rope: torch.Tensor,
                balance: torch.Tensor | None = None) -> dict:
    """x [M, 8192] BF16 through the step. ``cache``: (k_pages, v_pages). ``batch``: page_table, context, starts,
    max_draft and tree_mask of ``tree_attention``, and each token's positions and slots (``make_batch``). Returns y
    [M, 8192] (this GPU's o partial), the attention output and the experts with their weights."""
    q, k, v, gate = split_qkv_gate(project(x, state, "qkv_gate"), HEADS, KV_HEADS, DIM)
    q = rope_append(q, k, v, batch["positions"], batch["slots"], *cache, rope)
    a = tree_attention(q, *cache, batch["page_table"], batch["context"], batch["starts"], batch["max_draft"], batch["tree_mask"], gate=gate)
    y = project(a.view(x.shape[0], HEADS * DIM), state, "o")
    weights, experts = route(project(x, state, "router"), TOP_K, scoring="sigmoid", bias=balance, groups=GROUPS, top_groups=TOP_GROUPS)
    return {"y": y, "attention": a, "weights": weights, "experts": experts}


def make_batch(contexts: list, parents: list, page_size: int, device="cuda", seed: int = 0) -> tuple[dict, int]:
    """(batch, pages of the cache it needs). ``parents[b]``: the parent of each drafted token of request b as
    an index among them, -1 for a root; a token's position is its request's context plus its depth."""
    drafts = [len(p) for p in parents]
    need = [-(-(c + t) // page_size) for c, t in zip(contexts, drafts)]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed)).int()
    table = torch.zeros((len(need), max(need)), dtype=torch.int32)
    used = 0
    for b, n in enumerate(need):
        table[b, :n] = order[used:used + n]
        used += n
    starts = torch.zeros(len(drafts) + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(drafts).cumsum(0)
    positions, owner, index = [], [], []
    for b, tree in enumerate(parents):
        depth: list = []
        for i, p in enumerate(tree):
            depth.append(0 if p < 0 else depth[p] + 1)
            positions.append(contexts[b] + depth[i])
            owner.append(b)
            index.append(contexts[b] + i)
    max_draft = max(max(drafts), 1)
    starts, table = starts.to(device), table.to(device)
    flat = torch.tensor([p for tree in parents for p in tree], dtype=torch.int32, device=device)
    return {"page_table": table, "context": torch.tensor(contexts, dtype=torch.int32, device=device), "starts": starts, "max_draft": max_draft,
            "tree_mask": tree_mask(flat, starts, max_draft), "positions": torch.tensor(positions, dtype=torch.int32, device=device),
            "slots": page_slots(table, torch.tensor(owner, device=device), torch.tensor(index, device=device), page_size)}, sum(need)


def random_trees(drafts: list, seed: int = 0) -> list:
    g = torch.Generator().manual_seed(seed)
    return [[-1 if i == 0 else int(torch.randint(-1, i, (1,), generator=g)) for i in range(t)] for t in drafts]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--draft", type=int, default=8, help="drafted tokens a request (1: decoding)")
    ap.add_argument("--context", type=int, default=4096, help="longest cached context")
    ap.add_argument("--page-size", type=int, default=16)
    ap.add_argument("--steps", type=int, default=50)
    args = ap.parse_args()
    weights = {name: w for name, w in generate_weights().items() if name in ("qkv_gate", "o", "router")}
    state = prepare(weights, verbose=False)
    contexts = [max(1, args.context * (b + 1) // args.requests) for b in range(args.requests)]
    batch, pages = make_batch(contexts, random_trees([args.draft] * args.requests), args.page_size)
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = tuple(torch.randn((pages, KV_HEADS, args.page_size, DIM), generator=g, device="cuda").bfloat16() for _ in range(2))
    m = args.requests * args.draft
    x = torch.randn((m, LAYERS["qkv_gate"][1]), generator=g, device="cuda").bfloat16()
    balance = 0.05 * torch.randn(LAYERS["router"][0], generator=g, device="cuda")
    rope = rope_table(DIM, args.context + args.draft, scaling="yarn", factor=4.0, original=max(args.context // 4, 1))
    eager = verify_step(x, state, cache, batch, rope, balance)  # also sizes what a capture must not allocate
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = verify_step(x, state, cache, batch, rope, balance)
    graph.replay()
    torch.cuda.synchronize()
    _lib.device_error(torch.cuda.current_stream().cuda_stream)
    for name, t in eager.items():
        if not torch.equal(t, captured[name]):
            raise RuntimeError(f"{name}: the graph's result differs from the eager one")
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for _ in range(5):
        graph.replay()
    begin.record()
    for _ in range(args.steps):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    print(f"verify step, {args.requests} requests x {args.draft} drafted tokens over up to {args.context} cached: "
          f"{begin.elapsed_time(end) * 1e3 / args.steps:.1f} us a step")


if __name__ == "__main__":
    main()
