"""Drafted trees and selected blocks on the GPU where the inputs are unusual: rows out of any range,
rows of no request, infinities beside tokens that are not there, refused plans, several query rows
of a request, scales that are no powers of two, large batches of scores. References: _steps_ref.py."""
import numpy as np
import pytest
import torch

import ccinfer_amd as cc
from tests import _steps_ref as R
from tests._util import say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(2468)


def i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)


def host(x):
    return x.cpu().numpy()


def check(got, want, tol):
    got = host(got.double())
    assert np.all(np.isfinite(got))
    off = np.abs(got - want)
    assert np.all(off <= tol), (off - tol).max()


def inner(n, fill, dev):
    """(n int32 elements with as many on either side, the whole): all `fill`."""
    whole = torch.full((3 * n,), fill, dtype=torch.int32, device=dev)
    return whole[n:2 * n], whole


# ---- rows out of any range ---------------------------------------------------------------

@pytest.mark.parametrize("qsl,ctx", [([-1, 2 ** 31 - 1], 40), ([-2 ** 31, 2 ** 31 - 1], 40),
                                     ([-2 ** 31, 5], 40), ([5, -2 ** 31], 2 ** 31 - 1),
                                     ([2 ** 31 - 1, -2 ** 31], 1)])
def test_rows_whose_difference_passes_32_bits(gpu, qsl, ctx):
    """Such a request is refused, and nothing outside the rows of the call is written or read."""
    say(f"drafted trees with rows {qsl[0]} to {qsl[1]}")
    total = 8
    here = slice(max(qsl[0], 0), max(max(qsl[0], 0), min(qsl[1], total)))  # its rows that are there
    dq, dc, table = i32(qsl, gpu), i32([ctx], gpu), i32([[0, 1, 2]], gpu)
    parents = i32(np.arange(-1, total - 1), gpu)
    (mask, mask_all), (pos, pos_all), (slots, slots_all) = (inner(total, 7, gpu) for _ in range(3))
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    cc.build_draft_tree(parents, dq, dc, table, 8,
                        out={"tree_mask": mask.view(total, 1), "positions": pos,
                             "slot_mapping": slots, "status": status})
    torch.cuda.synchronize()
    assert status.item() == 6
    for part, whole, none in ((mask, mask_all, 0), (pos, pos_all, -1), (slots, slots_all, -1)):
        assert bool((whole[:total] == 7).all()) and bool((whole[2 * total:] == 7).all())
        assert bool((part[here] == none).all())

    (nodes, nodes_all), (tokens, tokens_all) = (inner(total, 7, gpu) for _ in range(2))
    k, v = torch.randn(2, 48, 1, 64, device=gpu).bfloat16()
    keep = k.clone(), v.clone()
    said = cc.accept_draft_tokens(parents, parents, parents, dq, dc, table, k, v,
                                  out={"accepted": status, "accepted_nodes": nodes,
                                       "tokens": tokens, "context_lens": torch.zeros_like(dc)})
    torch.cuda.synchronize()
    assert status.item() == 0 and said["context_lens"].item() == ctx
    for part, whole in ((nodes, nodes_all), (tokens, tokens_all)):
        want = torch.full((3 * total,), 7, dtype=torch.int32)
        want[total:2 * total][here] = -1
        assert torch.equal(whole.cpu(), want)
    assert torch.equal(k, keep[0]) and torch.equal(v, keep[1])

    q = torch.randn(total, 2, 64, device=gpu).bfloat16()
    out = torch.full_like(q, 7.0)
    cc.tree_attention(q, k, v, table, dq, dc, mask.view(total, 1), output=out)
    torch.cuda.synchronize()
    assert bool((out == 7).all())
