"""Trees of drafted tokens on the GPU: plan, attention, acceptance, against the 64-bit and
node-by-node references of tests/_steps_ref.py."""
import numpy as np
import pytest
import torch

import ccinfer_amd as cc
from tests import _steps_ref as R
from tests._util import say

pytestmark = pytest.mark.gpu

NAN = float("nan")


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(1234)


def i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)


class Batch:
    """Requests with trees: parents, tables, contexts."""

    def __init__(self, seed, nodes, before, width=None, back=9, parents=None):
        rng = self.rng = np.random.default_rng(seed)
        self.trees = parents or [R.random_tree(rng, n, back) for n in nodes]
        self.ctx = np.array([b + len(t) for b, t in zip(before, self.trees)])
        self.width = width or int(-(-self.ctx.max() // R.BLOCK)) + 1
        self.table, self.blocks = R.make_tables(rng, self.ctx, self.width)
        self.qsl = np.concatenate([[0], np.cumsum([len(t) for t in self.trees])]).astype(int)
        self.total = int(self.qsl[-1])
        self.sees = [R.visible(t) for t in self.trees]
        self.most = max(1, max(len(t) for t in self.trees))

    def mask(self, words=None):
        words = words or -(-self.most // 32)
        rows = [R.pack_mask(s, words) for s in self.sees if len(s)]
        return np.concatenate(rows) if rows else np.zeros((0, words), np.int32)

    def held(self):
        return R.held_slots(self.table, self.ctx, self.blocks)

    def on(self, dev):
        return dict(block_table=i32(self.table, dev), query_start_loc=i32(self.qsl, dev),
                    context_lens=i32(self.ctx, dev))


def run_attention(dev, b, hq, hkv, d, fp8, mask=None, poison=True, extra_rows=0, cache=None, q=None):
    cache = cache or R.Cache(b.rng, b.blocks, hkv, d, fp8, b.held() if poison else None)
    t = cache.on(dev)
    total = b.total + extra_rows
    if q is None:
        q = torch.randn(total, hq, d, generator=torch.Generator().manual_seed(5)).bfloat16()
    m = b.mask() if mask is None else mask
    if extra_rows:
        m = np.concatenate([m, np.full((extra_rows, m.shape[1]), -1, np.int32)])
    out = torch.full((total, hq, d), 7.0, dtype=torch.bfloat16, device=dev)
    n = cc.tree_attention_workspace_size(len(b.ctx), total, b.width, m.shape[1], hq, hkv, d)
    ws = torch.full((n // 4,), NAN, dtype=torch.float32, device=dev)
    a = b.on(dev)
    got = cc.tree_attention(q.to(dev), t["k"], t["v"], a["block_table"], a["query_start_loc"],
                            a["context_lens"], i32(m, dev), k_scale=t["ks"], v_scale=t["vs"],
                            output=out, workspace=ws)
    torch.cuda.synchronize()
    assert got is out
    return out.double().cpu().numpy(), q.double().numpy(), cache


def check(got, want, tol):
    assert np.all(np.isfinite(got))
    off = np.abs(got - want)
    assert np.all(off <= tol), (off - tol).max()


SHAPES = [(16, 8, 128), (32, 8, 128), (8, 8, 64), (8, 1, 128), (14, 2, 128), (32, 2, 64),
          (4, 4, 256), (10, 5, 64), (6, 3, 120), (16, 8, 80), (4, 1, 32), (8, 4, 192), (4, 2, 8)]


@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("fp8", [False, True])
def test_attention_of_ragged_trees(gpu, hq, hkv, d, fp8):
    if fp8 and d not in (64, 128):
        pytest.skip("fp8 caches: head dims 64 and 128")
    say(f"tree attention {hq}/{hkv} x {d} fp8 {fp8}")
    b = Batch(hq + hkv + d, [1, 26, 7, 33, 16, 2, 64], [300, 0, 17, 95, 15, 1, 700])
    got, q, cache = run_attention(gpu, b, hq, hkv, d, fp8)
    want, tol = R.tree_attention(q, cache, b.table, b.qsl, b.ctx, b.sees, 7.0)
    check(got, want, tol)


@pytest.mark.parametrize("nodes", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 64, 65, 130])
@pytest.mark.parametrize("before", [0, 1, 16, 31, 32, 47])
def test_attention_of_every_edge(gpu, nodes, before):
    """Rows around the edges of tiles and row blocks (G 4), trees that begin anywhere in a chunk."""
    say(f"tree attention {nodes} nodes behind {before}")
    b = Batch(nodes * 100 + before, [nodes, 3], [before, before + 5])
    got, q, cache = run_attention(gpu, b, 8, 2, 64, False)
    want, tol = R.tree_attention(q, cache, b.table, b.qsl, b.ctx, b.sees, 7.0)
    check(got, want, tol)


@pytest.mark.parametrize("fp8", [False, True])
def test_attention_of_long_contexts_that_are_cut(gpu, fp8):
    """One and three requests whose pieces lie in many slots, and one that ends a slot early."""
    for nodes, before in (([26], [9000]), ([5, 40, 12], [6000, 33, 2500]), ([70], [4000])):
        say(f"tree attention {nodes} behind {before} fp8 {fp8}")
        b = Batch(sum(before), nodes, before)
        got, q, cache = run_attention(gpu, b, 4, 2, 128, fp8)
        want, tol = R.tree_attention(q, cache, b.table, b.qsl, b.ctx, b.sees, 7.0)
        check(got, want, tol)


def test_attention_of_many_requests(gpu):
    """More requests than threads of a workgroup, some without nodes."""
    rng = np.random.default_rng(3)
    nodes = rng.integers(0, 6, 700)
    say("tree attention 700 requests")
    b = Batch(4, nodes, rng.integers(0, 60, 700))
    got, q, cache = run_attention(gpu, b, 2, 1, 64, False)
    want, tol = R.tree_attention(q, cache, b.table, b.qsl, b.ctx, b.sees, 7.0)
    check(got, want, tol)


def test_attention_leaves_other_rows_alone(gpu):
    """Requests whose context is shorter than their nodes, holes in the table, a context past the
    table row, and rows behind the last request."""
    say("tree attention of broken requests")
    b = Batch(9, [5, 6, 20, 9], [40, 30, 100, 64])
    b.table[2, 3] = -1                       # a hole in the committed tokens
    b.table[3] = -1                          # nothing to see at all
    b.ctx[1] = 4                             # fewer than its nodes: left alone
    held = b.held()
    cache = R.Cache(b.rng, b.blocks, 2, 64, False, held)
    got, q, _ = run_attention(gpu, b, 4, 2, 64, False, cache=cache, extra_rows=6)
    want, tol = R.tree_attention(q, cache, b.table, b.qsl, b.ctx, b.sees, 7.0)
    check(got, want, tol)
    assert np.all(got[b.qsl[1]:b.qsl[2]] == 7.0) and np.all(got[b.total:] == 7.0)
    assert np.all(got[b.qsl[3]:b.qsl[4]] == 0.0)

    b = Batch(10, [8], [80], width=4)        # 64 of its 88 positions are in the table
    got, q, cache = run_attention(gpu, b, 4, 2, 64, False)
    want, tol = R.tree_attention(q, cache, b.table, b.qsl, b.ctx, b.sees, 7.0)
    check(got, want, tol)


@pytest.mark.parametrize("words", [1, 2, 3])
def test_any_mask(gpu, words):
    """Masks that are no trees, rows that see nothing, nodes past the mask's words."""
    say(f"tree attention, {words} mask words")
    b = Batch(20 + words, [40, 50], [0, 33])
    rng = np.random.default_rng(words)
    b.sees = [rng.random((n, 32 * words)) < 0.4 for n in (40, 50)]
    b.sees[0][3] = False
    mask = np.concatenate([R.pack_mask(s, words) for s in b.sees])
    got, q, cache = run_attention(gpu, b, 4, 1, 128, False, mask=mask)
    want, tol = R.tree_attention(q, cache, b.table, b.qsl, b.ctx, b.sees, 7.0)
    check(got, want, tol)
    assert np.all(got[3] == 0.0)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_unbounded_nodes_reach_only_rows_that_see_them(gpu, fp8, d):
    say(f"tree attention, NaN and infinity in nodes, d {d} fp8 {fp8}")
    b = Batch(31, [40, 12], [50, 7], back=40)
    clean = R.Cache(b.rng, b.blocks, 2, d, fp8, b.held())
    first, q, _ = run_attention(gpu, b, 8, 2, d, fp8, cache=clean)
    for what in ("k", "v"):
        dirty = R.Cache(np.random.default_rng(0), b.blocks, 2, d, fp8, b.held())
        dirty.t = {n: (x.clone() if isinstance(x, torch.Tensor) else x) for n, x in clean.t.items()}
        hit = []
        for r, node in ((0, 5), (0, 33), (1, 11)):
            pos = b.ctx[r] - len(b.trees[r]) + node
            s = int(b.table[r, pos // 16]) * 16 + pos % 16
            if fp8:
                dirty.t[what][s] = 0x7f
            else:
                dirty.t[what][s] = NAN if node != 33 else float("inf")
            hit += [b.qsl[r] + i for i in range(len(b.trees[r])) if b.sees[r][i, node]]
        got, _, _ = run_attention(gpu, b, 8, 2, d, fp8, cache=dirty)
        keep = np.setdiff1d(np.arange(b.total), hit)
        # rows that do not see them: the sums may come in another order (the bound of one result)
        want, tol = R.tree_attention(q, clean, b.table, b.qsl, b.ctx, b.sees, 7.0)
        check(got[keep], want[keep], tol[keep])
        assert np.all(~np.isfinite(got[hit]).all(axis=-1))


def test_unbounded_query_rows_stay_alone(gpu):
    say("tree attention, NaN in one query row")
    b = Batch(32, [30], [90])
    q = torch.randn(30, 8, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    clean, qq, cache = run_attention(gpu, b, 8, 2, 128, False, q=q)
    bad = q.clone()
    bad[4, 3] = NAN
    got, _, _ = run_attention(gpu, b, 8, 2, 128, False, q=bad, cache=cache)
    same = np.ones((30, 8), bool)
    same[4, 3] = False
    assert np.array_equal(got[same], clean[same]) and not np.isfinite(got[4, 3]).any()


@pytest.mark.parametrize("fp8", [False, True])
def test_a_row_that_sees_only_nan_keys_is_nan(gpu, fp8):
    say(f"tree attention, one NaN key alone, fp8 {fp8}")
    b = Batch(33, [1, 2], [0, 0])
    cache = R.Cache(b.rng, b.blocks, 1, 128, fp8)
    slot = int(b.table[0, 0]) * 16
    cache.t["k"][slot] = 0x7f if fp8 else NAN
    got, _, _ = run_attention(gpu, b, 2, 1, 128, fp8, cache=cache)
    assert np.isnan(got[0]).all() and np.isfinite(got[1:]).all()


def test_a_chain_is_a_causal_prefill(gpu):
    """Against the prefill of the same tokens: both within the bound of the reference."""
    say("tree attention of chains and prefill")
    b = Batch(40, None, [100, 5, 0], parents=[list(range(-1, n - 1)) for n in (20, 33, 64)])
    got, q, cache = run_attention(gpu, b, 16, 8, 128, False)
    a, t = b.on(gpu), cache.on(gpu)
    pre = cc.prefill_attention(torch.from_numpy(q).bfloat16().to(gpu), t["k"], t["v"],
                               a["block_table"], a["query_start_loc"], a["context_lens"])
    want, tol = R.tree_attention(q, cache, b.table, b.qsl, b.ctx, b.sees, 7.0)
    check(got, want, tol)
    check(got, pre.double().cpu().numpy(), 2 * tol)


def test_single_nodes_are_a_decode_step(gpu):
    say("tree attention of single nodes and decode")
    b = Batch(41, [1] * 9, [0, 5, 16, 31, 100, 900, 2000, 47, 48])
    got, q, cache = run_attention(gpu, b, 16, 8, 128, False)
    a, t = b.on(gpu), cache.on(gpu)
    dec = cc.decode_attention(torch.from_numpy(q).bfloat16().to(gpu), t["k"], t["v"],
                              a["block_table"], a["context_lens"])
    want, tol = R.tree_attention(q, cache, b.table, b.qsl, b.ctx, b.sees, 7.0)
    check(got, want, tol)
    check(got, dec.double().cpu().numpy(), 2 * tol)


def test_same_bits_every_time_and_on_another_stream(gpu):
    say("tree attention twice, on two streams at once")
    b = Batch(42, [26, 50, 3], [3000, 800, 77])
    first, q, cache = run_attention(gpu, b, 32, 8, 128, False)
    again, _, _ = run_attention(gpu, b, 32, 8, 128, False, cache=cache)
    assert np.array_equal(first, again)
    a, t, m = b.on(gpu), cache.on(gpu), i32(b.mask(), gpu)
    qd = torch.from_numpy(q).bfloat16().to(gpu)
    torch.cuda.synchronize()
    outs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            outs.append(cc.tree_attention(qd, t["k"], t["v"], a["block_table"],
                                          a["query_start_loc"], a["context_lens"], m))
    torch.cuda.synchronize()
    for o in outs:
        assert np.array_equal(o.double().cpu().numpy(), first)


# ---- the plan --------------------------------------------------------------------------

def plan_ref(b, words):
    mask = b.mask(words)
    pos = np.concatenate([c - len(t) + s.sum(1) - 1 for c, t, s in zip(b.ctx, b.trees, b.sees)])
    slots = np.concatenate([[int(b.table[r, p // 16]) * 16 + p % 16
                             for p in range(c - len(t), c)]
                            for r, (c, t) in enumerate(zip(b.ctx, b.trees))])
    return mask, pos.astype(int), slots.astype(int)


@pytest.mark.parametrize("nodes,extra", [([1], 0), ([26], 0), ([0, 5, 64, 1], 0), ([33, 32, 31], 9),
                                         ([257, 3, 100], 0), ([2048], 0)])
def test_plan(gpu, nodes, extra):
    say(f"plan of trees of {nodes}")
    b = Batch(sum(nodes), nodes, [11 * i + 3 for i in range(len(nodes))], back=30)
    a = b.on(gpu)
    flat = np.concatenate([np.array(t, np.int32) for t in b.trees])
    out = cc.build_draft_tree(i32(flat, gpu), a["query_start_loc"], a["context_lens"],
                              a["block_table"], min(2048, b.most + extra))
    mask, pos, slots = plan_ref(b, -(-min(2048, b.most + extra) // 32))
    assert np.array_equal(out["tree_mask"].cpu().numpy(), mask)
    assert np.array_equal(out["positions"].cpu().numpy(), pos)
    assert np.array_equal(out["slot_mapping"].cpu().numpy(), slots)
    assert not out["status"].cpu().numpy().any()


def test_plan_of_broken_requests(gpu):
    say("plan of broken requests")
    b = Batch(50, [4, 5, 6, 7, 3], [20, 30, 40, 10, 0])
    flat = np.concatenate([np.array(t, np.int32) for t in b.trees])
    flat[b.qsl[0] + 2] = 3                    # a later node
    flat[b.qsl[1] + 1] = -5
    b.ctx[2] = 3                              # fewer than its nodes
    b.table[3, (b.ctx[3] - 1) // 16] = -1     # no block for its last node
    a = b.on(gpu)
    out = cc.build_draft_tree(i32(flat, gpu), a["query_start_loc"], a["context_lens"],
                              a["block_table"], 7)
    out = {k: v.cpu().numpy() for k, v in out.items()}
    assert out["status"].tolist() == [6, 6, 6, 6, 0]
    assert out["tree_mask"][b.qsl[0] + 2, 0] == 4  # taken as a root: itself alone
    assert out["positions"][b.qsl[0] + 2] == 20
    assert out["tree_mask"][b.qsl[1] + 1, 0] == 2
    rows = slice(b.qsl[2], b.qsl[3])
    assert not out["tree_mask"][rows].any() and (out["positions"][rows] == -1).all() \
        and (out["slot_mapping"][rows] == -1).all()
    assert out["slot_mapping"][b.qsl[4] - 1] == -1
    # more nodes than the call plans for: this request alone is left out
    out = cc.build_draft_tree(i32(flat, gpu), a["query_start_loc"], a["context_lens"],
                              a["block_table"], 5)
    assert out["status"].tolist() == [6, 6, 6, 6, 0]
    assert not out["tree_mask"][b.qsl[3]:b.qsl[4]].any()


# ---- acceptance ------------------------------------------------------------------------

def accept_case(seed, nodes, before, vocab):
    """Few different tokens: paths of every length."""
    b = Batch(seed, nodes, before, back=6)
    b.parents = np.concatenate([np.array(t, np.int32) for t in b.trees]) if b.total else \
        np.zeros(0, np.int32)
    b.draft, b.target = (b.rng.integers(0, vocab, b.total) for _ in range(2))
    return b


def accept_run(dev, b, layers, hkv, d, fp8, block=16, apart=False):
    """(device results, caches before and after as integers)."""
    gen = torch.Generator().manual_seed(9)
    shape = (layers, b.blocks, block, hkv, d)
    if fp8:
        k, v = (torch.randint(0, 255, shape, generator=gen, dtype=torch.uint8) for _ in range(2))
        ks, vs = (torch.rand(layers, b.blocks * hkv * 16, generator=gen) for _ in range(2))
    else:
        k, v = (torch.randn(shape, generator=gen).bfloat16() for _ in range(2))
        ks = vs = None
    dk, dv = k.to(dev), v.to(dev)
    dks, dvs = (None, None) if not fp8 else (ks.to(dev), vs.to(dev))
    a = b.on(dev)
    out = {"accepted": torch.full((len(b.ctx),), -7, dtype=torch.int32, device=dev),
           "accepted_nodes": torch.full((b.total,), -7, dtype=torch.int32, device=dev),
           "tokens": torch.full((b.total,), -7, dtype=torch.int32, device=dev),
           "context_lens": torch.full((len(b.ctx),), -7, dtype=torch.int32, device=dev)}
    args = (i32(b.draft, dev), i32(b.target, dev), i32(b.parents, dev), a["query_start_loc"],
            a["context_lens"], a["block_table"])
    if apart:
        for x in range(layers):
            cc.accept_draft_tokens(*args, dk[x], dv[x], k_scale=None if not fp8 else dks[x],
                                   v_scale=None if not fp8 else dvs[x], cache_block_size=block,
                                   out=out)
    else:
        cc.accept_draft_tokens(*args, dk, dv, k_scale=dks, v_scale=dvs, cache_block_size=block,
                               out=out)
    torch.cuda.synchronize()
    assert np.array_equal(a["context_lens"].cpu().numpy(), b.ctx)
    return out, (k, v, ks, vs), (dk.cpu(), dv.cpu(), None if not fp8 else dks.cpu(),
                                 None if not fp8 else dvs.cpu())


def accept_check(b, out, old, new, block=16):
    paths, counts, nodes, tokens, lengths = R.accept(b.draft, b.target, b.parents, b.qsl, b.ctx)
    assert np.array_equal(out["accepted"].cpu().numpy(), counts)
    assert np.array_equal(out["accepted_nodes"].cpu().numpy(), nodes)
    assert np.array_equal(out["tokens"].cpu().numpy(), tokens)
    assert np.array_equal(out["context_lens"].cpu().numpy(), lengths)
    for x in range(4):
        if old[x] is None:
            continue
        want = old[x].clone()
        rows = want.view(want.shape[0], -1, *want.shape[3:]) if x < 2 else \
            want.view(want.shape[0], b.blocks, -1, 16)
        src = rows.clone()
        for r, path in enumerate(paths):
            before = int(b.ctx[r]) - len(b.trees[r])
            for k, p in enumerate(path):
                t = [int(b.table[r, (before + y) // block]) for y in (p, k)]
                if min(t) < 0:
                    continue
                s, z = (c * block + (before + y) % block for c, y in zip(t, (p, k)))
                if x < 2:
                    rows[:, z] = src[:, s]
                else:
                    rows[:, z // 16, :, z % 16] = src[:, s // 16, :, s % 16]
        assert torch.equal(new[x].view(torch.uint8), want.view(torch.uint8)), x


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("layers,hkv,d", [(3, 8, 128), (1, 1, 64), (2, 3, 40), (2, 5, 8)])
def test_accept(gpu, fp8, layers, hkv, d):
    say(f"accept {layers} layers {hkv} x {d} fp8 {fp8}")
    for seed, vocab in ((1, 2), (2, 3), (3, 1000), (4, 1)):
        b = accept_case(seed, [26, 1, 64, 0, 7, 130, 2], [40, 0, 15, 9, 33, 16, 7], vocab)
        out, old, new = accept_run(gpu, b, layers, hkv, d, fp8)
        accept_check(b, out, old, new)


def test_accept_a_whole_chain_and_paths_that_step_over_it(gpu):
    """Chains of which all is taken (no row moves), and paths each of whose nodes lies two places
    behind its destination: destinations that are earlier nodes' sources."""
    say("accept chains")
    b = accept_case(7, [300, 5], [3, 12], 1)
    b.parents = np.concatenate([np.arange(-1, 299), [-1, 0, 0, 2, 3]]).astype(np.int32)
    b.target[:] = 0
    b.draft[:] = 0
    b.draft[b.qsl[1] + 1] = 1        # node 2 and its line are taken
    out, old, new = accept_run(gpu, b, 2, 2, 64, False)
    assert out["accepted"].tolist() == [300, 4]
    accept_check(b, out, old, new)
    b = accept_case(8, [200], [5], 1)
    b.parents = np.array([-1, 0, 0] + [i - 1 if i > 3 else 2 for i in range(3, 200)], np.int32)
    b.draft[:], b.target[:] = 0, 0
    b.draft[1] = 1                   # node 1 is wrong: everything behind it moves by one
    out, old, new = accept_run(gpu, b, 2, 2, 64, False)
    assert out["accepted"].tolist() == [199]
    accept_check(b, out, old, new)


def test_accept_of_layers_one_by_one_and_other_blocks(gpu):
    say("accept, layers apart, blocks of 8 and 32")
    b = accept_case(11, [26, 9], [40, 5], 2)
    together = accept_run(gpu, b, 4, 2, 64, True)
    apart = accept_run(gpu, b, 4, 2, 64, True, apart=True)
    for x in range(4):
        assert torch.equal(together[2][x], apart[2][x])
    accept_check(b, apart[0], apart[1], apart[2])
    for block in (8, 32):
        b = accept_case(12, [26, 9], [40, 5], 2)
        b.width = int(-(-b.ctx.max() // block)) + 1
        need = [-(-int(c) // block) for c in b.ctx]
        b.table = np.full((2, b.width), -1, np.int32)
        b.blocks = sum(need) + 2
        ids = b.rng.permutation(b.blocks)
        b.table[0, :need[0]], b.table[1, :need[1]] = ids[:need[0]], ids[need[0]:sum(need)]
        out, old, new = accept_run(gpu, b, 2, 2, 64, False, block=block)
        accept_check(b, out, old, new, block)


def test_accept_of_broken_requests(gpu):
    say("accept of broken requests")
    b = accept_case(13, [6, 5, 2049, 4], [30, 10, 50, 20], 1)
    b.ctx[0] = 5                              # fewer than its nodes
    b.table[3, (b.ctx[3] - 4) // 16] = -1     # its nodes have no block
    b.parents[b.qsl[1] + 2] = 4               # a later node: never a child of an earlier one
    out, old, new = accept_run(gpu, b, 1, 1, 64, False)
    assert out["accepted"].tolist()[0] == 0 and out["accepted"].tolist()[2] == 0
    assert out["context_lens"].tolist()[0] == 5 and out["context_lens"].tolist()[2] == b.ctx[2]
    accept_check(b, out, old, new)
    # without a cache, and blocks outside the pool, which are passed over
    a = b.on(gpu)
    bare = cc.accept_draft_tokens(i32(b.draft, gpu), i32(b.target, gpu), i32(b.parents, gpu),
                                  a["query_start_loc"], a["context_lens"], a["block_table"])
    assert all(torch.equal(bare[k], out[k]) for k in out)
    b.table[1] = b.blocks + 3
    out, old, new = accept_run(gpu, b, 1, 1, 64, False)
    assert torch.equal(new[0].view(torch.uint8), old[0].view(torch.uint8))
