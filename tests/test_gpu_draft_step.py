"""Whole steps with drafted trees on the GPU: pages grown, the tree planned, its K and V written,
attention, acceptance, pages given back, key bounds renewed, and the next drafts' decode over
selected blocks; captured and replayed; and the largest batches."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import ccinfer_amd as cc
from tests import _steps_ref as R
from tests._util import say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(4321)


def i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)


def host(x):
    return x.cpu().numpy()


def check(got, want, tol):
    off = np.abs(got.double().cpu().numpy() - want)
    assert np.all(off <= tol), (off - tol).max()


def view(k, v, blocks, hkv, d):
    """What the references need of a bf16 cache as it is."""
    return SimpleNamespace(fp8=False, hkv=hkv, d=d, blocks=blocks,
                           t={"k64": host(k.double()), "v64": host(v.double())})


def test_steps_of_a_serving_loop(gpu):
    """Three steps of three requests, one of them new in the first (its tree begins at position 0
    of an empty context). Everything that a step computes is checked against the state before it."""
    hkv, hq, d, blocks, width, take = 2, 8, 64, 96, 40, 5
    rng = np.random.default_rng(11)
    say("draft steps: prompts")
    table = torch.full((3, width), -1, dtype=torch.int32, device=gpu)
    ctx = torch.zeros(3, dtype=torch.int32, device=gpu)
    refs = torch.zeros(blocks, dtype=torch.int32, device=gpu)
    rows, none = i32([0, 1, 2], gpu), i32([-1, -1, -1], gpu)
    prompts = np.array([200, 0, 333])
    k = torch.zeros(blocks * 16, hkv, d, dtype=torch.bfloat16, device=gpu)
    v = torch.zeros_like(k)
    bounds = torch.zeros(blocks, hkv, 2, d, dtype=torch.bfloat16, device=gpu)
    assert cc.update_block_tables(table, ctx, refs, rows, none, i32(prompts, gpu)).item() == 0
    held = R.held_slots(host(table), prompts, blocks).to(gpu)
    k[held], v[held] = (torch.randn(2, int(held.sum()), hkv, d, device=gpu).bfloat16())
    cc.update_key_bounds(k, bounds, table, ctx,
                         i32(np.concatenate([[0], np.cumsum(prompts)]), gpu))

    for step, nodes in enumerate(([26, 9, 1], [3, 40, 17], [16, 16, 33])):
        say(f"draft step {step}")
        before = host(ctx).copy()
        trees = [R.random_tree(rng, n, 6) for n in nodes]
        qsl = np.concatenate([[0], np.cumsum(nodes)])
        total, sees = int(qsl[-1]), [R.visible(t) for t in trees]
        parents, dq = i32(np.concatenate(trees), gpu), i32(qsl, gpu)
        assert cc.update_block_tables(table, ctx, refs, rows, None,
                                      i32(before + nodes, gpu)).item() == 0
        assert np.array_equal(host(ctx), before + nodes)
        plan = cc.build_draft_tree(parents, dq, ctx, table, max(nodes))
        t_host = host(table)
        want_slots = np.concatenate([[t_host[b, p // 16] * 16 + p % 16
                                      for p in range(before[b], before[b] + nodes[b])]
                                     for b in range(3)])
        assert np.array_equal(host(plan["slot_mapping"]), want_slots)
        assert not host(plan["status"]).any()
        depth = np.concatenate([s.sum(1) - 1 + before[b] for b, s in enumerate(sees)])
        assert np.array_equal(host(plan["positions"]), depth)

        new = torch.randn(2, total, hkv, d, device=gpu).bfloat16()
        cc.write_kv_cache(new[0], new[1], k, v, plan["slot_mapping"])
        q = torch.randn(total, hq, d, device=gpu).bfloat16()
        out = cc.tree_attention(q, k, v, table, dq, ctx, plan["tree_mask"])
        want, tol = R.tree_attention(host(q.double()), view(k, v, blocks, hkv, d), t_host, qsl,
                                     before + nodes, sees, 0.0)
        check(out, want, tol)

        draft, target = rng.integers(0, 3, total), rng.integers(0, 3, total)
        said = cc.accept_draft_tokens(i32(draft, gpu), i32(target, gpu), parents, dq, ctx, table,
                                      k, v)
        paths, counts, taken, tokens, lengths = R.accept(draft, target, np.concatenate(trees), qsl,
                                                         before + nodes)
        assert np.array_equal(host(said["accepted"]), counts)
        assert np.array_equal(host(said["accepted_nodes"]), taken)
        assert np.array_equal(host(said["tokens"]), tokens)
        assert np.array_equal(host(said["context_lens"]), lengths)
        for b, path in enumerate(paths):
            for x, node in enumerate(path):
                p = before[b] + x
                slot = int(t_host[b, p // 16]) * 16 + p % 16
                assert torch.equal(k[slot], new[0, qsl[b] + node])
                assert torch.equal(v[slot], new[1, qsl[b] + node])

        assert cc.update_block_tables(table, ctx, refs, rows, None,
                                      said["context_lens"]).item() == 0
        assert np.array_equal(host(ctx), lengths)
        assert int(refs.sum().item()) == sum(-(-int(c) // 16) for c in lengths)
        cc.update_key_bounds(k, bounds, table, ctx, dq)
        cache, t_host = view(k, v, blocks, hkv, d), host(table)
        whole = R.key_bounds(cache, t_host, lengths, lengths, host(bounds.double()))
        assert np.array_equal(host(bounds.double()), whole)

        q = torch.randn(3, hq, d, device=gpu).bfloat16()
        sc = cc.score_kv_blocks(q, bounds, table, ctx)
        want, tol = R.scores(host(q.double()), whole, t_host, lengths)
        there = np.isfinite(want)
        assert np.array_equal(np.isfinite(host(sc)), there)
        assert np.all(np.abs(host(sc).astype(float) - want)[there] <= tol[there])
        chosen = cc.select_kv_blocks(sc, ctx, take)
        assert np.array_equal(host(chosen), R.select(host(sc), lengths, take, 1, 1))
        out = cc.sparse_decode_attention(q, k, v, table, ctx, chosen)
        want, tol = R.sparse_decode(host(q.double()), cache, t_host, lengths, host(chosen))
        check(out, want, tol)


def test_two_tree_steps_in_graphs(gpu):
    """Plan, cache write, attention and acceptance of two batches, each captured into a graph of its
    own with a workspace of its own; replayed in turn, and at once on two streams, with eager work
    and synchronizations between, each replay equal to the eager calls on the same state."""
    say("tree steps captured and replayed")
    hkv, hq, d = 2, 8, 128

    def batch(seed, nodes, before):
        rng = np.random.default_rng(seed)
        trees = [R.random_tree(rng, n) for n in nodes]
        ctx = np.array(before) + nodes
        table, blocks = R.make_tables(rng, ctx, int(-(-ctx.max() // 16)))
        cache = R.Cache(rng, blocks, hkv, d, False).on(gpu)
        x = SimpleNamespace(
            nodes=nodes, total=sum(nodes), trees=trees, k=cache["k"], v=cache["v"],
            table=i32(table, gpu), ctx=i32(ctx, gpu),
            qsl=i32(np.concatenate([[0], np.cumsum(nodes)]), gpu),
            parents=i32(np.concatenate(trees), gpu),
            draft=torch.randint(0, 3, (sum(nodes),), dtype=torch.int32, device=gpu),
            target=torch.randint(0, 3, (sum(nodes),), dtype=torch.int32, device=gpu),
            q=torch.randn(sum(nodes), hq, d, device=gpu).bfloat16(),
            new=torch.randn(2, sum(nodes), hkv, d, device=gpu).bfloat16())
        words = -(-max(nodes) // 32)
        x.ws = torch.empty(cc.tree_attention_workspace_size(
            len(nodes), x.total, table.shape[1], words, hq, hkv, d), dtype=torch.uint8, device=gpu)
        return x

    def step(x):
        plan = cc.build_draft_tree(x.parents, x.qsl, x.ctx, x.table, max(x.nodes))
        cc.write_kv_cache(x.new[0], x.new[1], x.k, x.v, plan["slot_mapping"])
        out = cc.tree_attention(x.q, x.k, x.v, x.table, x.qsl, x.ctx, plan["tree_mask"],
                                workspace=x.ws)
        said = cc.accept_draft_tokens(x.draft, x.target, x.parents, x.qsl, x.ctx, x.table, x.k, x.v)
        return [plan["tree_mask"], plan["positions"], plan["slot_mapping"], plan["status"], out,
                said["accepted"], said["accepted_nodes"], said["tokens"], said["context_lens"]]

    xs = [batch(1, [26, 5, 60], [900, 31, 4000]), batch(2, [8, 70], [2500, 16])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in xs:
            step(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for x in xs:
        x.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(x.graph):
            x.outs = step(x)
    streams = [torch.cuda.Stream() for _ in xs]
    for turn in range(5):
        say(f"turn {turn}")
        for x in xs:
            x.q.copy_(torch.randn(x.q.shape, device=gpu))
            x.new.copy_(torch.randn(x.new.shape, device=gpu))
            x.draft.copy_(torch.randint(0, 3, (x.total,), dtype=torch.int32, device=gpu))
        torch.cuda.synchronize()
        if turn % 2:
            for x, s in zip(xs, streams):
                with torch.cuda.stream(s):
                    x.graph.replay()
        else:
            for x in xs:
                x.graph.replay()
        torch.cuda.synchronize()
        for x in xs:
            got, kv = [o.clone() for o in x.outs], (x.k.clone(), x.v.clone())
            want = step(x)
            torch.cuda.synchronize()
            # rows of no request are none here: every element of every output is written
            assert all(torch.equal(g, w) for g, w in zip(got, want))
            assert torch.equal(kv[0], x.k) and torch.equal(kv[1], x.v)


def test_the_most_requests_of_an_attention_call(gpu):
    say("tree attention of 1024 requests")
    rng = np.random.default_rng(5)
    nodes, before = rng.integers(0, 4, 1024), rng.integers(0, 40, 1024)
    trees = [R.random_tree(rng, n) for n in nodes]
    ctx = before + nodes
    table, blocks = R.make_tables(rng, ctx, 3)
    cache = R.Cache(rng, blocks, 1, 64, False)
    t = cache.on(gpu)
    qsl = np.concatenate([[0], np.cumsum(nodes)])
    q = torch.randn(int(qsl[-1]), 2, 64, device=gpu).bfloat16()
    mask = np.concatenate([R.pack_mask(R.visible(p), 1) for p in trees if p])
    out = torch.full_like(q, 7.0)
    args = [t["k"], t["v"], i32(table, gpu), i32(qsl, gpu), i32(ctx, gpu), i32(mask, gpu)]
    cc.tree_attention(q, *args, output=out)
    want, tol = R.tree_attention(host(q.double()), cache, table, qsl, ctx,
                                 [R.visible(p) for p in trees], 7.0)
    check(out, want, tol)
    args[2] = torch.cat([args[2], args[2][:1]])
    args[3] = torch.cat([args[3], args[3][-1:]])
    args[4] = torch.cat([args[4], args[4][:1]])
    with pytest.raises(cc.CcinferError):
        cc.tree_attention(q, *args, output=out)


@pytest.mark.parametrize("nodes,before", [(2048, 0), (2048, 700), (2047, 33)])
def test_the_largest_tree(gpu, nodes, before):
    """64 words of mask; a chain and a random tree: acceptance takes the whole chain."""
    say(f"tree of {nodes} nodes behind {before}")
    rng = np.random.default_rng(nodes + before)
    hkv, hq, d = 1, 2, 64
    for tree in (list(range(-1, nodes - 1)), R.random_tree(rng, nodes, 40)):
        ctx, qsl = np.array([before + nodes]), np.array([0, nodes])
        table, blocks = R.make_tables(rng, ctx, -(-int(ctx[0]) // 16))
        cache = R.Cache(rng, blocks, hkv, d, False)
        t = cache.on(gpu)
        dt, dq, dc = i32(table, gpu), i32(qsl, gpu), i32(ctx, gpu)
        parents = i32(tree, gpu)
        plan = cc.build_draft_tree(parents, dq, dc, dt, 2048)
        see = R.visible(tree)
        assert np.array_equal(host(plan["tree_mask"]), R.pack_mask(see, 64))
        q = torch.randn(nodes, hq, d, device=gpu).bfloat16()
        out = cc.tree_attention(q, t["k"], t["v"], dt, dq, dc, plan["tree_mask"])
        want, tol = R.tree_attention(host(q.double()), cache, table, qsl, ctx, [see], 7.0)
        check(out, want, tol)
        same = np.zeros(nodes, int)
        said = cc.accept_draft_tokens(i32(same, gpu), i32(same, gpu), parents, dq, dc, dt,
                                      t["k"], t["v"])
        _, counts, taken, _, lengths = R.accept(same, same, tree, qsl, ctx)
        assert np.array_equal(host(said["accepted"]), counts)
        assert np.array_equal(host(said["accepted_nodes"]), taken)
        assert np.array_equal(host(said["context_lens"]), lengths)


def test_contexts_far_below_zero(gpu):
    """A context whose difference with the nodes passes 32 bits is one of fewer tokens than nodes."""
    say("drafted trees with contexts of -2^31")
    low = -2 ** 31
    ctx, qsl = i32([low, 20, low + 1], gpu), i32([0, 3, 5, 8], gpu)
    table = i32([[0, 1], [2, 3], [4, 5]], gpu)
    parents = i32([-1, 0, 1, -1, 0, -1, 0, 0], gpu)
    plan = cc.build_draft_tree(parents, qsl, ctx, table, 4)
    assert host(plan["status"]).tolist() == [6, 0, 6]
    assert host(plan["slot_mapping"]).tolist() == [-1] * 3 + [34 + 16, 35 + 16] + [-1] * 3
    k, v = torch.randn(2, 96, 1, 64, device=gpu).bfloat16()
    q = torch.randn(8, 2, 64, device=gpu).bfloat16()
    out = torch.full_like(q, 7.0)
    cc.tree_attention(q, k, v, table, qsl, ctx, plan["tree_mask"], output=out)
    assert bool((out[:3] == 7).all()) and bool((out[5:] == 7).all())
    assert bool((out[3:5] != 7).any())
    bounds = torch.full((6, 1, 2, 64), 5.0, dtype=torch.bfloat16, device=gpu)
    cc.update_key_bounds(k, bounds, table, ctx, qsl)
    assert bool((bounds[[0, 1, 2, 4, 5]] == 5).all()) and bool((bounds[3] != 5).any())
    keep = k.clone()
    said = cc.accept_draft_tokens(parents, parents, parents, qsl, ctx, table, k, v)
    assert host(said["accepted"]).tolist()[::2] == [0, 0]
    assert host(said["context_lens"]).tolist()[::2] == [low, low + 1]
    assert torch.equal(k[:48], keep[:48]) and torch.equal(k[64:], keep[64:])
