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


# ---- rows of no request --------------------------------------------------------------------

def test_plan_of_a_padded_batch(gpu):
    """Rows before the first request and behind the last one get no mask, position -1 and slot -1,
    whatever an earlier call left there."""
    say("plan of a padded batch")
    qsl, total = np.array([2, 5, 5, 9]), 300
    ctx, table = np.array([20, 7, 33]), np.array([[4, 1, -1], [2, -1, -1], [0, 3, 5]])
    parents = np.zeros(total, np.int32)
    parents[2:9] = [-1, 0, 0, -1, 0, 1, 2]
    out = {"tree_mask": torch.full((total, 2), 7, dtype=torch.int32, device=gpu),
           "positions": torch.full((total,), 7, dtype=torch.int32, device=gpu),
           "slot_mapping": torch.full((total,), 7, dtype=torch.int32, device=gpu),
           "status": torch.full((3,), 7, dtype=torch.int32, device=gpu)}
    cc.build_draft_tree(i32(parents, gpu), i32(qsl, gpu), i32(ctx, gpu), i32(table, gpu), 40,
                        out=out)
    got = {n: host(x) for n, x in out.items()}
    assert got["status"].tolist() == [0, 0, 0]
    assert got["tree_mask"][2:9].tolist() == [[m, 0] for m in (1, 3, 5, 1, 3, 7, 15)]
    assert got["positions"][2:9].tolist() == [17, 18, 18, 29, 30, 31, 32]
    assert got["slot_mapping"][2:9].tolist() == [17, 18, 19, 3 * 16 + 13, 3 * 16 + 14,
                                                 3 * 16 + 15, 5 * 16]
    none = np.r_[0:2, 9:total]
    assert not got["tree_mask"][none].any()
    assert (got["positions"][none] == -1).all() and (got["slot_mapping"][none] == -1).all()


def test_a_replayed_step_of_fewer_nodes_writes_no_old_slots(gpu):
    """A captured step of up to 12 nodes: replays with fewer leave the slots of earlier replays."""
    say("captured plan and cache write, fewer nodes in each replay")
    total, table = 12, i32([[0, 1], [2, 3]], gpu)
    parents = i32(np.tile([-1, 0, 1, 2, 3, 4], 2), gpu)
    qsl, ctx = i32([0, 6, 12], gpu), i32([16, 16], gpu)
    k, v = torch.zeros(2, 64, 1, 64, dtype=torch.bfloat16, device=gpu)
    new = torch.randn(2, total, 1, 64, device=gpu).bfloat16()

    def step():
        plan = cc.build_draft_tree(parents, qsl, ctx, table, 6)
        cc.write_kv_cache(new[0], new[1], k, v, plan["slot_mapping"])
        return plan

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for nodes, lens in (((6, 6), (16, 16)), ((2, 3), (20, 18)), ((1, 0), (21, 18)),
                        ((4, 2), (30, 20))):
        qsl.copy_(i32(np.concatenate([[0], np.cumsum(nodes)]), gpu))
        ctx.copy_(i32(lens, gpu))
        new.copy_(torch.randn(new.shape, device=gpu))
        want = k.clone(), v.clone()
        at = 0
        for b in range(2):
            for i in range(nodes[b]):
                p = lens[b] - nodes[b] + i
                for x in range(2):
                    want[x][(2 * b + p // 16) * 16 + p % 16] = new[x, at]
                at += 1
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(k, want[0]) and torch.equal(v, want[1]), nodes
