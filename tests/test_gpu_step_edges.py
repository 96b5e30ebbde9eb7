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


# ---- infinities beside tokens that are not there ---------------------------------------------

def check_unbounded(got, want, tol):
    """Infinite where the reference is (with its sign), else within its bound."""
    got = host(got.double())
    there = np.isfinite(want)
    assert np.array_equal(got[~there], want[~there])
    assert np.all(np.abs(got[there] - want[there]) <= tol[there])
    assert np.any(~there)


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (8, 2, 128), (4, 2, 80), (4, 1, 256)])
def test_sparse_decode_of_an_infinite_value(gpu, hq, hkv, d):
    """V of one token that a row sees is infinite: the row's result is, in that column alone, also
    where the token's block is not full or has no other beside it in its list."""
    say(f"sparse decode, an infinity in V, {hq}/{hkv} x {d}")
    rng = np.random.default_rng(d)
    ctx = np.array([37])
    table, blocks = R.make_tables(rng, ctx, 4)
    q = torch.randn(1, hq, d).bfloat16()
    for token, lists in ((36, ([2], [0, 2], [2, -1], [-1, 2], [2, 9], [0, 1, 2], [2, 0])),
                         (20, ([1], [1, -1], [-1, 1], [0, 2, 1], [1, 7], [3, 1]))):
        cache = R.Cache(rng, blocks, hkv, d, False, R.held_slots(table, ctx, blocks))
        slot = int(table[0, token // 16]) * 16 + token % 16
        cache.t["v"][slot, 0, 3], cache.t["v"][slot, hkv - 1, d - 2] = np.inf, -np.inf
        cache.t["v64"] = cache.t["v"].double().numpy()
        t = cache.on(gpu)
        for chosen in lists:
            sel = np.broadcast_to(np.array(chosen), (1, hkv, len(chosen)))
            out = cc.sparse_decode_attention(q.to(gpu), t["k"], t["v"], i32(table, gpu),
                                             i32(ctx, gpu), i32(sel, gpu))
            want, tol = R.sparse_decode(q.double().numpy(), cache, table, ctx, sel)
            check_unbounded(out, want, tol)


@pytest.mark.parametrize("d", [64, 80, 128, 256])
@pytest.mark.parametrize("nodes", [3, 14, 30, 60])
def test_tree_attention_of_an_infinite_value_beside_a_hole(gpu, nodes, d):
    """The same in the committed context, beside a block that the table does not have: one, two,
    four and eight wavefronts' rows."""
    say(f"tree attention of {nodes} nodes, an infinity in V beside a hole, d {d}")
    rng = np.random.default_rng(nodes + d)
    hq, hkv, before = 8, 2, 150
    ctx, qsl = np.array([before + nodes]), np.array([0, nodes])
    table, blocks = R.make_tables(rng, ctx, 16)
    table[0, 3] = table[0, 4] = -1
    cache = R.Cache(rng, blocks, hkv, d, False, R.held_slots(table, ctx, blocks))
    for token, column in ((2 * 16 + 5, 3), (5 * 16 + 15, d - 1)):
        cache.t["v"][int(table[0, token // 16]) * 16 + token % 16, :, column] = np.inf
    cache.t["v64"] = cache.t["v"].double().numpy()
    t, see = cache.on(gpu), R.visible(R.random_tree(rng, nodes))
    q = torch.randn(nodes, hq, d).bfloat16()
    words = -(-nodes // 32)
    out = cc.tree_attention(q.to(gpu), t["k"], t["v"], i32(table, gpu), i32(qsl, gpu),
                            i32(ctx, gpu), i32(R.pack_mask(see, words), gpu))
    want, tol = R.tree_attention(q.double().numpy(), cache, table, qsl, ctx, [see], 0.0)
    check_unbounded(out, want, tol)


# ---- requests that the plan refused ------------------------------------------------------------

@pytest.mark.parametrize("fp8", [False, True])
def test_refused_plans_accept_nothing(gpu, fp8):
    """More nodes than planned for, a parent that is no earlier node, a node without a block, fewer
    context tokens than nodes: with the plan's status they accept 0, keep their K and V and lose the
    nodes; the others go on as without it."""
    say(f"acceptance of refused plans, fp8 {fp8}")
    nodes, before = [4, 9, 5, 6, 3, 0, 7], np.array([20, 30, 5, 12, 40, 8, 33])
    trees = [R.random_tree(np.random.default_rng(n), n) for n in nodes]
    ctx, qsl = before + nodes, np.concatenate([[0], np.cumsum(nodes)])
    ctx[4] = 2
    rng = np.random.default_rng(1)
    table, blocks = R.make_tables(rng, ctx, 4)
    parents = np.concatenate([np.array(t, np.int32) for t in trees])
    parents[qsl[2] + 3] = 4
    table[3, (ctx[3] - 1) // 16] = -1
    draft, target = np.zeros((2, int(qsl[-1])), np.int32)     # whole chains are confirmed
    dq, dc, dt = i32(qsl, gpu), i32(ctx, gpu), i32(table, gpu)
    plan = cc.build_draft_tree(i32(parents, gpu), dq, dc, dt, 8)
    refused = [False, True, True, True, True, False, False]
    assert (host(plan["status"]) != 0).tolist() == refused
    start = R.Cache(rng, blocks, 2, 64, fp8).on(gpu)
    args = (i32(draft, gpu), i32(target, gpu), i32(parents, gpu), dq, dc, dt)
    runs = []
    for status in (None, plan["status"]):
        t = {n: None if x is None else x.clone() for n, x in start.items()}
        out = cc.accept_draft_tokens(*args, t["k"], t["v"], k_scale=t["ks"], v_scale=t["vs"],
                                     status=status)
        runs.append({n: host(x) for n, x in out.items()})
    plain, said = runs
    good = ~np.array(refused)
    for n in ("accepted", "context_lens"):
        assert np.array_equal(said[n][good], plain[n][good])
    assert not said["accepted"][~good].any() and plain["accepted"][1] > 0
    assert said["context_lens"][~good].tolist() == [30, 5, 12, 2]
    for b in range(7):
        rows = slice(qsl[b], qsl[b + 1])
        for n in ("accepted_nodes", "tokens"):
            want = np.full(nodes[b], -1) if refused[b] else plain[n][rows]
            assert np.array_equal(said[n][rows], want), (b, n)
    # the refused requests' blocks hold what they held
    for b in np.nonzero(~good)[0]:
        for block in table[b][table[b] >= 0]:
            s = slice(block * 16, block * 16 + 16)
            for n in ("k", "v"):
                assert torch.equal(t[n][s], start[n][s])


def test_a_step_goes_on_after_a_refused_plan(gpu):
    """Contexts of a refused request cut back by update_block_tables: the next step plans it again."""
    say("a step after a refused plan")
    table = torch.full((2, 6), -1, dtype=torch.int32, device=gpu)
    ctx, refs = torch.zeros(2, dtype=torch.int32, device=gpu), \
        torch.zeros(16, dtype=torch.int32, device=gpu)
    rows, none = i32([0, 1], gpu), i32([-1, -1], gpu)
    assert cc.update_block_tables(table, ctx, refs, rows, none, i32([30, 17], gpu)).item() == 0
    qsl, parents = i32([0, 6, 9], gpu), i32([-1, 0, 1, 2, 3, 4, -1, 0, 1], gpu)
    same = torch.zeros(9, dtype=torch.int32, device=gpu)
    for most, want in ((4, [30, 20]), (8, [36, 23])):
        before = host(ctx)
        assert cc.update_block_tables(table, ctx, refs, rows, None,
                                      i32(before + [6, 3], gpu)).item() == 0
        plan = cc.build_draft_tree(parents, qsl, ctx, table, most)
        said = cc.accept_draft_tokens(same, same, parents, qsl, ctx, table, status=plan["status"])
        assert cc.update_block_tables(table, ctx, refs, rows, None,
                                      said["context_lens"]).item() == 0
        assert host(ctx).tolist() == want
        assert int(refs.sum().item()) == sum(-(-c // 16) for c in want)


# ---- rows that share a block -------------------------------------------------------------------

@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hkv,d", [(8, 128), (1, 64), (3, 24), (2, 256)])
def test_bounds_of_several_rows_of_a_request(gpu, fp8, hkv, d):
    """A row for each new token, all with the request's table row: the bounds are of the keys below
    the longest context, in whatever order the rows come."""
    say(f"bounds of rows that share blocks, {hkv} x {d} fp8 {fp8}")
    rng = np.random.default_rng(hkv + d)
    whole = np.array([37, 100, 16, 1, 64, 200])       # contexts after the new tokens
    tokens = np.array([5, 20, 3, 1, 1, 33])
    table, blocks = R.make_tables(rng, whole, 14)
    cache = R.Cache(rng, blocks, hkv, d, fp8, R.held_slots(table, whole, blocks))
    t = cache.on(gpu)
    row = np.repeat(np.arange(6), tokens)
    ctx = np.concatenate([np.arange(c - n + 1, c + 1) for c, n in zip(whole, tokens)])
    start = torch.randn(blocks, hkv, 2, d).bfloat16()
    want = R.key_bounds(cache, table, whole, tokens, start.double().numpy())
    for order in (np.arange(len(row)), np.arange(len(row))[::-1], rng.permutation(len(row))):
        bounds = start.to(gpu)
        cc.update_key_bounds(t["k"], bounds, i32(table[row[order]], gpu), i32(ctx[order], gpu),
                             k_scale=t["ks"])
        assert np.array_equal(host(bounds.double()), want)
    # the same as ranges of new tokens: two rows a request, the first without its last tokens
    both = np.repeat(np.arange(6), 2)
    short = np.maximum(whole - 3, 0)
    ctx = np.stack([short, whole], 1).reshape(-1)
    new = np.stack([np.maximum(tokens - 3, 0), np.minimum(tokens, 3)], 1).reshape(-1)
    bounds = start.to(gpu)
    cc.update_key_bounds(t["k"], bounds, i32(table[both], gpu), i32(ctx, gpu),
                         i32(np.concatenate([[0], np.cumsum(new)]), gpu), k_scale=t["ks"])
    assert np.array_equal(host(bounds.double()), want)


def test_bounds_of_many_rows_that_share_blocks(gpu):
    """More rows than two wavefronts look at together: 300 requests of 2 to 4 rows."""
    say("bounds of 900 rows that share blocks")
    rng = np.random.default_rng(4)
    tokens, whole = rng.integers(2, 5, 300), rng.integers(4, 70, 300)
    table, blocks = R.make_tables(rng, whole, 5)
    cache = R.Cache(rng, blocks, 1, 64, False, R.held_slots(table, whole, blocks))
    row = rng.permutation(np.repeat(np.arange(300), tokens))
    seen, ctx = np.zeros(300, int), np.zeros(len(row), int)
    for x, b in enumerate(row):
        ctx[x] = whole[b] - seen[b]
        seen[b] += 1
    start = torch.zeros(blocks, 1, 2, 64).bfloat16()
    bounds = start.to(gpu)
    cc.update_key_bounds(cache.on(gpu)["k"], bounds, i32(table[row], gpu), i32(ctx, gpu))
    want = R.key_bounds(cache, table, whole, tokens, start.double().numpy())
    assert np.array_equal(host(bounds.double()), want)


def test_a_step_of_several_tokens_a_request(gpu):
    """The whole chain with a row for each of four new tokens of two requests."""
    say("selected blocks, four query rows a request")
    rng = np.random.default_rng(6)
    hkv, hq, d, m = 2, 8, 128, 4
    whole = np.array([503, 81])
    table, blocks = R.make_tables(rng, whole, 34)
    cache = R.Cache(rng, blocks, hkv, d, False, R.held_slots(table, whole, blocks))
    t = cache.on(gpu)
    bounds = torch.full((blocks, hkv, 2, d), float("nan"), dtype=torch.bfloat16, device=gpu)
    before = whole - m
    cc.update_key_bounds(t["k"], bounds, i32(table, gpu), i32(before, gpu),
                         i32(np.concatenate([[0], np.cumsum(before)]), gpu))
    row = np.repeat(np.arange(2), m)
    ctx = np.concatenate([np.arange(c - m + 1, c + 1) for c in whole])
    rows = i32(table[row], gpu), i32(ctx, gpu)
    cc.update_key_bounds(t["k"], bounds, *rows)
    q = torch.randn(2 * m, hq, d).bfloat16()
    sc = cc.score_kv_blocks(q.to(gpu), bounds, *rows)
    got = host(sc.double())
    _, tol = R.scores(q.double().numpy(), host(bounds.double()), table[row], ctx)
    for b in range(2 * m):
        for p in range(ctx[b]):
            s = int(table[row[b], p // 16]) * 16 + p % 16
            for h in range(hkv):
                top = (q[b, 4 * h:4 * h + 4].double().numpy() @ cache.t["k64"][s, h]).max()
                assert top / np.sqrt(d) <= got[b, h, p // 16] + tol[b, h, p // 16]
    chosen = cc.select_kv_blocks(sc, rows[1], 6)
    assert np.array_equal(host(chosen), R.select(host(sc), ctx, 6, 1, 1))
    out = cc.sparse_decode_attention(q.to(gpu), t["k"], t["v"], *rows, chosen)
    want, tol = R.sparse_decode(q.double().numpy(), cache, table[row], ctx, host(chosen))
    check(out, want, tol)


# ---- scores of large batches -------------------------------------------------------------------

def scores_ref(q, bounds, table, ctx):
    """_steps_ref.scores, a row and head at a time."""
    rows, hq, d = q.shape
    hkv, width = bounds.shape[1], table.shape[1]
    out, tol = np.full((rows, hkv, width), -np.inf), np.zeros((rows, hkv, width))
    for b in range(rows):
        n = -(-int(ctx[b]) // 16) if ctx[b] > 0 else 0
        if n > width:
            continue
        for h in range(hkv):
            g = q[b].reshape(hkv, -1, 1, d)[h]
            both = bounds[np.maximum(table[b, :n], 0), h]
            terms = np.maximum(g * both[:, 0], g * both[:, 1])
            there = table[b, :n] >= 0
            out[b, h, :n] = np.where(there, terms.sum(-1).max(0) / np.sqrt(d), -np.inf)
            tol[b, h, :n] = np.abs(terms).sum(-1).max(0) / np.sqrt(d) * (2 * d + 4) * 2.0 ** -24
    return out, tol


@pytest.mark.parametrize("rows,hq,hkv,d,width", [
    (64, 16, 8, 128, 270), (64, 16, 8, 64, 270), (64, 8, 8, 256, 270), (64, 16, 8, 120, 270),
    (64, 16, 8, 80, 257), (205, 40, 2, 64, 270), (256, 17, 1, 128, 500), (300, 34, 2, 40, 255)])
def test_scores_of_large_batches(gpu, rows, hq, hkv, d, width):
    """From 2048 wavefronts on each takes up to four tiles of 16 blocks, copied two ahead: contexts
    that end in each of the tiles, holes, more than 16 query heads a kv head (two rounds)."""
    say(f"scores of {rows} rows, {hq}/{hkv} x {d}, {width} blocks")
    assert -(-width // 64) * rows * hkv >= 2048
    rng = np.random.default_rng(rows + d)
    n = rng.integers(0, width + 1, rows)
    n[:12] = [0, 1, 15, 16, 17, 32, 33, 48, 49, 64, 65, width]
    ctx = np.maximum(n * 16 - rng.integers(0, 16, rows), 0)
    ctx[12] = width * 16 + 1                       # more than the table holds
    blocks = 97
    table = rng.integers(0, blocks, (rows, width))
    table[rng.random(table.shape) < 0.1] = -1
    bounds = torch.randn(blocks, hkv, 2, d).bfloat16().sort(dim=2).values.contiguous()
    q = torch.randn(rows, hq, d).bfloat16()
    out = torch.full((rows, hkv, width), float("nan"), device=gpu)
    want, tol = scores_ref(q.double().numpy(), bounds.double().numpy(), table, ctx)
    for _ in range(3):
        cc.score_kv_blocks(q.to(gpu), bounds.to(gpu), i32(table, gpu), i32(ctx, gpu), out=out)
        got = host(out.double())
        inside = np.isfinite(want)
        assert np.array_equal(np.isneginf(got), ~inside)
        assert np.all(np.abs(got[inside] - want[inside]) <= tol[inside])
        out.fill_(float("nan"))


# ---- fp8 caches with scales that are no powers of two ------------------------------------------

def odd_scales(cache, rng):
    """The cache's scales times numbers in [1, 2), float32."""
    gen = torch.Generator().manual_seed(int(rng.integers(1 << 31)))
    for n in ("k", "v"):
        s = cache.t[n + "s"] * (1 + torch.rand(cache.t[n + "s"].shape, generator=gen))
        cache.t[n + "s"] = s
        rows = s.view(cache.blocks, cache.hkv, 16).permute(0, 2, 1).reshape(-1, cache.hkv)
        values = cache.t[n].view(R.E4M3).double()
        cache.t[n + "64"] = (values * rows.double()[..., None]).numpy()
    return cache


@pytest.mark.parametrize("d", [64, 128])
def test_attention_with_any_scales(gpu, d):
    """Trees and selected blocks. The references' bound holds: a probability times its scale is one
    more float32 rounding, of the 64 that the bound counts beside the sums."""
    say(f"fp8 attention with any scales, d {d}")
    rng = np.random.default_rng(d)
    nodes, before = [26, 3, 64], np.array([300, 0, 95])
    trees = [R.random_tree(rng, n) for n in nodes]
    ctx, qsl = before + nodes, np.concatenate([[0], np.cumsum(nodes)])
    table, blocks = R.make_tables(rng, ctx, 24)
    cache = odd_scales(R.Cache(rng, blocks, 2, d, True, R.held_slots(table, ctx, blocks)), rng)
    t, sees = cache.on(gpu), [R.visible(p) for p in trees]
    q = torch.randn(int(qsl[-1]), 8, d).bfloat16()
    mask = np.concatenate([R.pack_mask(s, 2) for s in sees])
    out = cc.tree_attention(q.to(gpu), t["k"], t["v"], i32(table, gpu), i32(qsl, gpu),
                            i32(ctx, gpu), i32(mask, gpu), k_scale=t["ks"], v_scale=t["vs"])
    want, tol = R.tree_attention(q.double().numpy(), cache, table, qsl, ctx, sees, 0.0)
    check(out, want, tol)
    for take in (3, 20):
        sel = np.stack([[rng.permutation(24)[:take] for _ in range(2)] for _ in ctx])
        out = cc.sparse_decode_attention(q[:3].to(gpu), t["k"], t["v"], i32(table, gpu),
                                         i32(ctx, gpu), i32(sel, gpu), k_scale=t["ks"],
                                         v_scale=t["vs"])
        want, tol = R.sparse_decode(q[:3].double().numpy(), cache, table, ctx, sel)
        check(out, want, tol)


@pytest.mark.parametrize("hkv,d", [(8, 128), (3, 24)])
def test_bounds_and_scores_with_any_scales(gpu, hkv, d):
    """A bound is the product in float32 (2^-24 of it) rounded to bf16 (2^-8 of that): no key passes
    it by more, and no logit its block's score by more than such parts of |q| |bound|."""
    say(f"fp8 bounds with any scales, {hkv} x {d}")
    rng = np.random.default_rng(d)
    ctx = np.array([333, 64, 17])
    table, blocks = R.make_tables(rng, ctx, 22)
    cache = odd_scales(R.Cache(rng, blocks, hkv, d, True, R.held_slots(table, ctx, blocks)), rng)
    t = cache.on(gpu)
    bounds = torch.zeros(blocks, hkv, 2, d, dtype=torch.bfloat16, device=gpu)
    dt, dc = i32(table, gpu), i32(ctx, gpu)
    cc.update_key_bounds(t["k"], bounds, dt, dc, i32(np.cumsum([0, *ctx]), gpu), k_scale=t["ks"])
    want = R.key_bounds(cache, table, ctx, ctx, np.zeros(bounds.shape))
    got = host(bounds.double())
    assert np.all(np.abs(got - want) <= np.abs(want) * (2.0 ** -8 + 2.0 ** -23))
    assert not np.array_equal(got, want)               # (some are rounded)
    q = torch.randn(3, 2 * hkv, d).bfloat16()
    sc = host(cc.score_kv_blocks(q.to(gpu), bounds, dt, dc).double())
    exact, tol = R.scores(q.double().numpy(), got, table, ctx)
    there = np.isfinite(exact)
    assert np.all(np.abs(sc[there] - exact[there]) <= tol[there])
    q = q.double().numpy()
    for b in range(3):
        for p in range(ctx[b]):
            s, j = int(table[b, p // 16]) * 16 + p % 16, p // 16
            for h in range(hkv):
                g = q[b, 2 * h:2 * h + 2]
                top = (g @ cache.t["k64"][s, h]).max() / np.sqrt(d)
                slack = (np.abs(g) @ np.abs(want[table[b, j], h]).max(0)).max() / np.sqrt(d)
                assert top <= sc[b, h, j] + tol[b, h, j] + slack * (2.0 ** -8 + 2.0 ** -23)


def test_plan_of_blocks_whose_slots_pass_32_bits(gpu):
    """Such a table entry is no block: its slots would come out as those of another one."""
    say("plan of blocks of 2^27 and more")
    table = i32([[1 << 27, 3], [1 << 28, 2], [(1 << 27) - 1, 1], [2 ** 31 - 1, 0]], gpu)
    plan = cc.build_draft_tree(i32([-1, 0] * 4, gpu), i32([0, 2, 4, 6, 8], gpu),
                               i32([17] * 4, gpu), table, 2)
    assert host(plan["status"]).tolist() == [6, 6, 0, 6]
    assert host(plan["slot_mapping"]).tolist() == [-1, 48, -1, 32, 2 ** 31 - 1, 16, -1, 0]
