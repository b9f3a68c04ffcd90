"""Helpers of the operators between the projections on the CPU: the mask words of drafted trees (``tree_mask``),
the slots of tokens (``page_slots``) and the ramp of a stretched rotary table (``rope_table``)."""

import math

import torch

from muse_bf16_proj_b200.attention import page_slots, rope_table, tree_mask


def _mask_bits(words, draft):
    return [[(int(row[j // 32]) >> (j % 32)) & 1 for j in range(draft)] for row in words.tolist()]


def test_tree_mask_of_a_padded_step():
    """Rows before the first request's tokens and past the last one's, any number of them, see nothing; the others what they
    see without them."""
    starts = torch.tensor([0, 3, 3, 8], dtype=torch.int32)
    parents = torch.tensor([-1, 0, 0, -1, 0, 1, 1, 3], dtype=torch.int32)
    plain = tree_mask(parents, starts, 5)
    assert _mask_bits(plain, 5) == [[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 1, 1, 0, 0],
                                    [1, 1, 0, 1, 0], [1, 1, 0, 1, 1]]
    for before, after in ((0, 1), (0, 70), (40, 2)):
        for fill in (-1, 0):
            padded = torch.cat((torch.full((before,), fill, dtype=torch.int32), parents, torch.full((after,), fill, dtype=torch.int32)))
            got = tree_mask(padded, starts + before, 5)
            assert torch.equal(got[before:before + 8], plain)
            assert int(torch.count_nonzero(got[:before])) == 0 and int(torch.count_nonzero(got[before + 8:])) == 0
    assert tree_mask(parents[:0], torch.zeros(3, dtype=torch.int32), 5).shape == (0, 1)
    none = tree_mask(parents, torch.zeros(1, dtype=torch.int32), 5)
    assert none.shape == (8, 1) and int(torch.count_nonzero(none)) == 0


def test_tree_mask_of_more_tokens_than_max_draft():
    """What tree_attention reports as 0xB01 stays inside the words here, and the other request's rows are right."""
    starts = torch.tensor([0, 40, 42], dtype=torch.int32)
    parents = torch.tensor([-1] + list(range(39)) + [-1, 0], dtype=torch.int32)
    got = tree_mask(parents, starts, 30)
    assert got.shape == (42, 1) and _mask_bits(got[40:], 30) == [[1] + [0] * 29, [1, 1] + [0] * 28]
    assert got[29].tolist() == [(1 << 30) - 1]
    far = torch.tensor([500, -7, 0], dtype=torch.int32)  # no such parent
    assert _mask_bits(tree_mask(far, torch.tensor([0, 3], dtype=torch.int32), 3), 3) == [[1, 0, 0], [0, 1, 0], [1, 0, 1]]


def test_page_slots_without_a_place():
    """A row without a token (negative index) gets no slot. A place that the page table does not have (past its columns, a
    request outside it, an entry that names no page) gets one past every cache, which rope_append reports and skips."""
    table = torch.tensor([[3, 1], [0, -1]], dtype=torch.int32)
    past = torch.iinfo(torch.int64).max
    request = torch.tensor([0, 0, 1, 0, 1, 0, 1, 2, -1, 1], dtype=torch.int32)
    index = torch.tensor([2, 17, 15, -1, -16, 32, 16, 0, 0, 1000], dtype=torch.int32)
    assert page_slots(table, request, index, 16).tolist() == [50, 17, 15, -1, -1, past, past, past, past, past]
    assert page_slots(table, torch.tensor([7]), torch.tensor([-1]), 16).tolist() == [-1]
    for empty in (table[:0], table[:, :0]):
        assert page_slots(empty, torch.tensor([0, 0]), torch.tensor([0, -1]), 16).tolist() == [past, -1]
    assert page_slots(table, request[:0], index[:0], 16).tolist() == []


def test_yarn_blends_by_the_pairs_index():
    """Every entry of the ramp: the share of the divided frequency rises linearly from the pair that turns beta_fast times in
    the original positions to the one that turns beta_slow times."""
    rot, theta, original, f = 64, 10000.0, 8192, 4.0
    table = rope_table(rot, 4000, theta, "yarn", f, original, device="cpu")
    freq = [theta ** (-2 * i / rot) for i in range(rot // 2)]

    def turns(i):
        return original * freq[i] / (2 * math.pi)

    # The last pair that turns at least 32 times, the first that turns at most once.
    first = max(i for i in range(rot // 2) if turns(i) >= 32)
    last = min(i for i in range(rot // 2) if turns(i) <= 1)
    assert 0 < first < last - 1 < rot // 2 - 2  # a ramp with entries inside
    magnitude = 0.1 * math.log(f) + 1.0
    for i in range(rot // 2):
        share = min(max((i - first) / (last - first), 0.0), 1.0)
        angle = 3999 * (freq[i] / f * share + freq[i] * (1 - share))
        for got, exact in ((table[3999, i], math.cos(angle)), (table[3999, rot // 2 + i], math.sin(angle))):
            assert abs(got.item() - magnitude * exact) < 1e-6, (i, share)
