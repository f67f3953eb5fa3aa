"""Edges of the operators of several new rows per sequence: masks and paths that
no tree has, batch sizes at the default shared-memory limit, rows in use counted
by the kernel before, and the attention kernels' values that are not finite, of
very different sizes, or far from 1.

Tolerances of the attention: with A the largest scale * sum |q_i k_i| of a row
and a place, a score is off by at most A 2^-21 (2^-22 for the operands, as much for the
f32 sums) and, where an operand is far below its neighbours, by
scale * 2^-25 * (sum |q_i| + sum |k_i|); a weight by twice that relative to its softmax, and
an output by as much of sum_j p_j |v_j|. Of that sum the products and sums take another
2^-19: 2^-21 each for the weights' 21 bits, the product of the two low parts
that is left out and the f32 sums, 2^-22 each for V's 22 bits and the exponential. An
element of V far below its neighbours keeps 2^-25 (of 1 where the largest of
them lies between 2^-4 and 2^12), the weights' low parts less than that together.
"""
import subprocess
import sys

import numpy as np
import pytest

from test_tree_ops import (ATTN_TOL, ERR_NONFINITE, ERR_POSITION, ERR_TREE, Scene, accept_run, compact_run, dev, p, plan_case,
                           plan_check, plan_run)

pytestmark = pytest.mark.gpu

# shapes that each of the attention's three kernels takes: up to 16 rows of a KV head, blocks of 128, four of them and more
FEW, ROWS, LAID = [(4, 2, 64, 7), (2, 1, 128, 8), (3, 1, 48, 5)], [(4, 2, 64, 20), (8, 2, 128, 24), (4, 1, 48, 64)], [(8, 1, 128, 64), (16, 2, 64, 64)]


@pytest.fixture(scope="module")
def torch():
    import torch
    torch.cuda.init()
    return torch


# ---- b2_kv_plan, b2_rows_append -----------------------------------------------------------------------------


def test_plan_mask_without_a_row(b2, torch):
    """An empty mask is no tree's: reported, and the row's position is not before the new rows."""
    for ctx in ([0, 20], [7, 0]):
        c = plan_case(torch, ctx, [3, 4], 16, True)
        want = plan_run(b2, torch, c)
        c["masks"][1] = c["masks"][5] = 0
        got = plan_run(b2, torch, c)
        assert want["err"][0] == 0 and got["err"][0] == ERR_TREE
        pos = want["pos"].copy()
        pos[1], pos[5] = ctx[0], ctx[1]
        assert (got["pos"] == pos).all()
        for k in ("item", "slot", "start", "table", "mo", "fo"):
            assert (got[k] == want[k]).all()


# ---- b2_tree_accept, b2_kv_compact ----------------------------------------------------------------------------


@pytest.mark.parametrize("masks,count,follow", [
    ([1, 3, 7, 13], 1, 4),          # row 3 below row 2 without row 2's other ancestor; the root's token is nobody's
    ([1, 3, 7, 15], 1, 4),          # the same tokens in a proper chain
    ([1, 3, 5, 11, 31], 1, 4),      # row 4 has two branches' rows
])
def test_accept_masks_that_are_not_their_parents(b2, torch, masks, count, follow):
    tokens, nxt = [9, 5, 6, 7, 8][:len(masks)], [4, 6, 7, 8, 3][:len(masks)]
    r = accept_run(b2, torch, [0, len(masks)], tokens, masks, nxt, [11])
    proper = all(m >> i == 1 and (i == 0 or m ^ 1 << i == masks[(m ^ 1 << i).bit_length() - 1]) for i, m in enumerate(masks))
    assert r["err"][0] == (0 if proper else ERR_TREE)
    assert r["count"][0] == count and r["next"][0] == follow and r["out"][0] == 11 + count
    assert list(r["path"][0][:count + 1]) == [0, -1]


def test_accept_stops_before_a_mask_that_is_not_its_parents(b2, torch):
    """Rows that fit by their tokens: the branch ends before the row whose mask omits an ancestor, here and past row 32; other
    items are as they were."""
    r = accept_run(b2, torch, [0, 4, 6], [0, 1, 2, 3, 0, 1], [1, 3, 7, 13, 1, 3], [1, 2, 3, 4, 1, 2], [0, 5])
    assert r["err"][0] == ERR_TREE
    assert list(r["count"]) == [3, 2] and list(r["next"]) == [3, 2] and list(r["out"]) == [3, 7]
    masks = [(2 << i) - 1 for i in range(64)]
    masks[40] &= ~(1 << 7)
    r = accept_run(b2, torch, [0, 64], list(range(64)), masks, list(range(1, 65)), [0])
    # row 41's mask is no longer its parent's and its own bit either
    assert r["err"][0] == ERR_TREE and r["count"][0] == 40 and r["next"][0] == 40


@pytest.mark.parametrize("path,moved", [([0, 5, 3], [0, 5]), ([0, 5, 5], [0, 5]), ([4, 3, 9], [4, None, 9]), ([0, -1, 7], [0, None, 7])])
def test_compact_paths_that_do_not_ascend(b2, torch, path, moved):
    got, want, err = compact_run(b2, torch, 2, 2, 64, 16, [10], [path], mutate=None)
    assert err == ERR_POSITION
    # the same call without the refused entries: each is left out by naming its own place
    kept = [i if j is None else j for i, j in enumerate(moved)]
    same, want, _ = compact_run(b2, torch, 2, 2, 64, 16, [10], [kept])
    assert (same == want).all() and (got == want).all()


def test_compact_moves_what_lies_32_entries_behind_a_refused_one(b2, torch):
    """A thread looks up entries i and i + 32: each is refused or moved for itself."""
    path = [2 * i for i in range(8)] + list(range(20, 52))   # entry i of 8 and more is 12 + i
    path[5] = path[4]
    got, _, err = compact_run(b2, torch, 2, 2, 64, 16, [10], [path])
    assert err == ERR_POSITION
    path[5] = 5   # its own place: nothing to move
    same, want, _ = compact_run(b2, torch, 2, 2, 64, 16, [10], [path])
    assert (got == want).all()
