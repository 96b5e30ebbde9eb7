"""Decode over selected blocks on the GPU: bounds, scores, selection, attention, against the 64-bit
references of tests/_steps_ref.py."""
import numpy as np
import pytest
import torch

import ccinfer_amd as cc
from tests import _steps_ref as R
from tests._util import say

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(1234)


def i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)


def rows_of(seed, ctx, width=None):
    rng = np.random.default_rng(seed)
    ctx = np.array(ctx)
    width = width or int(-(-ctx.max() // 16)) + 1
    table, blocks = R.make_tables(rng, ctx, width)
    return rng, ctx, table, blocks


SHAPES = [(16, 8, 128), (32, 8, 128), (8, 8, 64), (14, 2, 128), (32, 1, 128), (40, 2, 64),
          (4, 4, 256), (6, 3, 120), (16, 8, 80), (4, 1, 32), (8, 4, 192), (4, 2, 8)]


# ---- bounds ----------------------------------------------------------------------------

@pytest.mark.parametrize("hkv,d", [(8, 128), (1, 64), (3, 120), (5, 8), (4, 256), (2, 24)])
@pytest.mark.parametrize("fp8", [False, True])
def test_bounds(gpu, hkv, d, fp8):
    say(f"bounds {hkv} x {d} fp8 {fp8}")
    rng, ctx, table, blocks = rows_of(hkv + d, [1, 16, 17, 500, 0, 33, 160])
    table[3, 7] = -1
    cache = R.Cache(rng, blocks, hkv, d, fp8, R.held_slots(table, ctx, blocks))
    t = cache.on(gpu)
    start = torch.randn(blocks, hkv, 2, d).bfloat16()
    for new in (None, [1, 1, 2, 300, 0, 33, 400], [0, 16, 17, 0, 5, 1, 100]):
        bounds = start.to(gpu)
        qsl = None if new is None else i32(np.concatenate([[0], np.cumsum(new)]), gpu)
        cc.update_key_bounds(t["k"], bounds, i32(table, gpu), i32(ctx, gpu), qsl,
                             k_scale=t["ks"])
        want = R.key_bounds(cache, table, ctx, new or [1] * len(ctx), start.double().numpy())
        assert np.array_equal(bounds.double().cpu().numpy(), want), new


def test_bounds_of_nan_keys_and_many_rows(gpu):
    say("bounds, NaN keys; 600 rows")
    rng, ctx, table, blocks = rows_of(3, [40])
    cache = R.Cache(rng, blocks, 2, 64, False)
    k = cache.t["k"].to(gpu)
    slot = int(table[0, 1]) * 16 + 3
    k[slot, 1, 5] = NAN
    k[slot + 1, 1, 6] = -NAN
    k[slot + 2, 0, 7] = INF
    bounds = torch.zeros(blocks, 2, 2, 64, dtype=torch.bfloat16, device=gpu)
    cc.update_key_bounds(k, bounds, i32(table, gpu), i32(ctx, gpu), i32([0, 40], gpu))
    got = bounds.float().cpu().numpy()[table[0, 1]]
    assert np.isnan(got[1, :, 5:7]).all() and np.isnan(got).sum() == 4 and got[0, 1, 7] == INF
    rng, ctx, table, blocks = rows_of(4, rng.integers(0, 90, 600))
    cache = R.Cache(rng, blocks, 1, 64, False, R.held_slots(table, ctx, blocks))
    new = rng.integers(0, 60, 600)
    start = torch.zeros(blocks, 1, 2, 64).bfloat16()
    bounds = start.to(gpu)
    cc.update_key_bounds(cache.on(gpu)["k"], bounds, i32(table, gpu), i32(ctx, gpu),
                         i32(np.concatenate([[0], np.cumsum(new)]), gpu))
    want = R.key_bounds(cache, table, ctx, new, start.double().numpy())
    assert np.array_equal(bounds.double().cpu().numpy(), want)


# ---- scores ----------------------------------------------------------------------------

@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_scores(gpu, hq, hkv, d):
    say(f"scores {hq}/{hkv} x {d}")
    rng, ctx, table, blocks = rows_of(hq + d, [1, 1000, 0, 4100, 257, 90], width=270)
    table[1, 5] = -1
    ctx[5] = 271 * 16 - 3  # more than the table holds
    lo = torch.randn(blocks, hkv, 2, d).bfloat16()
    bounds = lo.sort(dim=2).values.contiguous()
    q = torch.randn(len(ctx), hq, d).bfloat16()
    q[0, :, :3] = 0
    out = torch.full((len(ctx), hkv, 270), NAN, device=gpu)
    cc.score_kv_blocks(q.to(gpu), bounds.to(gpu), i32(table, gpu), i32(ctx, gpu), out=out)
    want, tol = R.scores(q.double().numpy(), bounds.double().numpy(), table, ctx)
    got = out.double().cpu().numpy()
    inside = np.isfinite(want)
    assert np.array_equal(np.isneginf(got), ~inside)
    assert np.all(np.abs(got[inside] - want[inside]) <= tol[inside])


def test_scores_bound_every_logit(gpu):
    """From a cache through its bounds: no key's logit passes its block's score (by more than the
    sum's rounding, which the other test bounds)."""
    say("scores bound logits")
    rng, ctx, table, blocks = rows_of(8, [333, 64])
    cache = R.Cache(rng, blocks, 2, 128, False)
    bounds = torch.zeros(blocks, 2, 2, 128, dtype=torch.bfloat16, device=gpu)
    q = torch.randn(2, 8, 128).bfloat16()
    dt, dc = i32(table, gpu), i32(ctx, gpu)
    cc.update_key_bounds(cache.on(gpu)["k"], bounds, dt, dc, i32(np.cumsum([0, 333, 64]), gpu))
    got = cc.score_kv_blocks(q.to(gpu), bounds, dt, dc).double().cpu().numpy()
    _, tol = R.scores(q.double().numpy(), bounds.double().cpu().numpy(), table, ctx)
    for b in range(2):
        for p in range(ctx[b]):
            s = int(table[b, p // 16]) * 16 + p % 16
            for h in range(2):
                top = (q[b, 4 * h:4 * h + 4].double().numpy() @ cache.t["k64"][s, h]).max()
                assert top / np.sqrt(128) <= got[b, h, p // 16] + tol[b, h, p // 16]


def test_scores_of_nan(gpu):
    say("scores of NaN bounds and queries")
    rng, ctx, table, blocks = rows_of(9, [100, 100])
    bounds = torch.randn(blocks, 1, 2, 64).sort(dim=2).values.bfloat16()
    bounds[table[0, 3], 0, :, 9] = NAN
    bounds[table[0, 4], 0, 1, 9] = INF
    q = torch.randn(2, 4, 64).bfloat16()
    q[1, 2, 7] = NAN
    got = cc.score_kv_blocks(q.to(gpu), bounds.to(gpu), i32(table, gpu), i32(ctx, gpu)).cpu().numpy()
    # 0 x inf in the part of the other sign, or inf
    assert np.isnan(got[0, 0, 3]) and got[0, 0, 4] != -INF and not np.isfinite(got[0, 0, 4])
    assert np.isfinite(got[0, 0, [0, 1, 2, 5, 6]]).all()
    assert np.isnan(got[1, 0, :7]).all() and np.isneginf(got[:, 0, 7:]).all()


# ---- selection -------------------------------------------------------------------------

@pytest.mark.parametrize("width", [1, 7, 300, 1024, 1025, 4097, 9000, 20000])
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "wide", "odd"])
def test_select(gpu, width, kind):
    say(f"select among {width}, {kind}")
    rng = np.random.default_rng(width)
    ctx = np.array([width * 16, max(1, width * 16 - 37), 1, 0, -3, width * 16 + 1, width * 8 + 1])
    shape = (len(ctx), 2, width)
    sc = rng.standard_normal(shape).astype(np.float32)
    if kind == "ties":
        sc = np.round(sc * 2) / 2
    elif kind == "equal":
        sc[:] = 1.5
    elif kind == "wide":
        sc = (sc * 10.0 ** rng.uniform(-38, 37, shape)).astype(np.float32)
    elif kind == "odd":
        for value in (np.inf, -np.inf, np.nan, -0.0, 0.0, 1e-45):
            sc[rng.random(shape) < 0.1] = value
    dev, dc = torch.from_numpy(sc).to(gpu), i32(ctx, gpu)
    for take, first, last in ((1, 0, 0), (1, 0, 1), (5, 2, 3), (64, 1, 2), (128, 0, 0),
                              (max(1, width - 1), 0, 1), (width, 0, 0), (width + 9, 1, 1)):
        if take < first + last:
            continue
        got = cc.select_kv_blocks(dev, dc, take, first, last).cpu().numpy()
        assert np.array_equal(got, R.select(sc, ctx, take, first, last)), (take, first, last)


# ---- attention -------------------------------------------------------------------------

def selections(rng, ctx, hkv, take, width):
    """Distinct blocks in any order, some outside the context, -1 between them."""
    out = np.full((len(ctx), hkv, take), -1, np.int64)
    for b in range(len(ctx)):
        for h in range(hkv):
            ids = rng.permutation(max(width, 1) + 4)[:take]
            ids = np.where(rng.random(len(ids)) < 0.1, -1, ids)
            out[b, h, :len(ids)] = ids
    return out


def run_sparse(dev, q, cache, table, ctx, sel):
    t = cache.on(dev)
    hq, d = q.shape[1:]
    n = cc.sparse_decode_workspace_size(len(ctx), hq, cache.hkv, d, sel.shape[2])
    ws = torch.full((max(1, n // 4),), NAN, dtype=torch.float32, device=dev)
    out = torch.full(q.shape, NAN, dtype=torch.bfloat16, device=dev)
    cc.sparse_decode_attention(q.to(dev), t["k"], t["v"], i32(table, dev), i32(ctx, dev),
                               i32(sel, dev), k_scale=t["ks"], v_scale=t["vs"], output=out,
                               workspace=ws)
    torch.cuda.synchronize()
    return out.double().cpu().numpy()


def check(got, want, tol):
    assert np.all(np.isfinite(got))
    off = np.abs(got - want)
    assert np.all(off <= tol), (off - tol).max()


@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("fp8", [False, True])
def test_sparse_attention(gpu, hq, hkv, d, fp8):
    if fp8 and d not in (64, 128):
        pytest.skip("fp8 caches: head dims 64 and 128")
    say(f"sparse decode {hq}/{hkv} x {d} fp8 {fp8}")
    rng, ctx, table, blocks = rows_of(hq + d, [1, 1000, 0, 333, 16, 40, 700])
    table[1, 5] = -1
    ctx[5] = (table.shape[1] + 1) * 16
    held = R.held_slots(table, np.where(ctx > table.shape[1] * 16, 0, ctx), blocks)
    cache = R.Cache(rng, blocks, hkv, d, fp8, held)
    q = torch.randn(len(ctx), hq, d).bfloat16()
    for take in (1, 2, 3, 16, 41):
        sel = selections(rng, ctx, hkv, take, 30)
        got = run_sparse(gpu, q, cache, table, ctx, sel)
        want, tol = R.sparse_decode(q.double().numpy(), cache, table, ctx, sel)
        check(got, want, tol)
        assert not got[2].any() and not got[5].any()


@pytest.mark.parametrize("take", [64, 300, 1030])
def test_sparse_attention_of_long_lists(gpu, take):
    say(f"sparse decode, lists of {take}")
    rng, ctx, table, blocks = rows_of(take, [take * 16 - 3, 2000])
    cache = R.Cache(rng, blocks, 1, 64, False, R.held_slots(table, ctx, blocks))
    q = torch.randn(2, 4, 64).bfloat16()
    sel = np.full((2, 1, take), -1, np.int64)
    sel[0, 0] = rng.permutation(take)
    sel[1, 0, :min(take, 125)] = rng.permutation(125)[:take]
    got = run_sparse(gpu, q, cache, table, ctx, sel)
    want, tol = R.sparse_decode(q.double().numpy(), cache, table, ctx, sel)
    check(got, want, tol)


def test_everything_selected_is_decode(gpu):
    say("sparse decode over all blocks and decode")
    rng, ctx, table, blocks = rows_of(5, [5, 800, 64, 333])
    q = torch.randn(4, 16, 128).bfloat16()
    for fp8 in (False, True):
        cache = R.Cache(rng, blocks, 8, 128, fp8)
        t = cache.on(gpu)
        sel = np.broadcast_to(np.arange(51), (4, 8, 51))
        got = run_sparse(gpu, q, cache, table, ctx, sel)
        want, tol = R.sparse_decode(q.double().numpy(), cache, table, ctx, sel)
        check(got, want, tol)
        if fp8:
            dec = cc.decode_attention_fp8(q.to(gpu), t["k"], t["v"], t["ks"], t["vs"],
                                          i32(table, gpu), i32(ctx, gpu))
        else:
            dec = cc.decode_attention(q.to(gpu), t["k"], t["v"], i32(table, gpu), i32(ctx, gpu))
        # decode's denominator has 1e-6 more: a 2^-19 of the result
        check(got, dec.double().cpu().numpy(), 2 * tol + 2.0 ** -19 * np.abs(want))


@pytest.mark.parametrize("fp8", [False, True])
def test_a_row_that_sees_only_nan_keys_is_nan(gpu, fp8):
    say(f"sparse decode, one NaN key alone, fp8 {fp8}")
    rng, ctx, table, blocks = rows_of(8, [1, 1])
    cache = R.Cache(rng, blocks, 1, 128, fp8)
    cache.t["k"][int(table[0, 0]) * 16] = 0x7f if fp8 else NAN
    q = torch.randn(2, 2, 128).bfloat16()
    got = run_sparse(gpu, q, cache, table, ctx, np.zeros((2, 1, 200), int))
    assert np.isnan(got[0]).all() and np.isfinite(got[1]).all()


def test_a_block_named_twice_counts_twice(gpu):
    say("sparse decode, a block twice")
    rng, ctx, table, blocks = rows_of(6, [80])
    cache = R.Cache(rng, blocks, 2, 64, False)
    q = torch.randn(1, 4, 64).bfloat16()
    sel = np.array([[[1, 3, 1], [2, 2, 2]]])
    got = run_sparse(gpu, q, cache, table, ctx, sel)
    want, tol = R.sparse_decode(q.double().numpy(), cache, table, ctx, sel)
    check(got, want, tol)


def test_the_whole_chain_in_a_graph(gpu):
    """Token written, bounds renewed, scores, selection, attention: captured once, replayed with
    eager work between the replays, each replay equal to the eager calls on the same state."""
    say("sparse step captured and replayed")
    rng, ctx, table, blocks = rows_of(7, [500, 90, 1300], width=84)
    cache = R.Cache(rng, blocks, 2, 128, False)
    t = cache.on(gpu)
    dt, dc = i32(table, gpu), i32(ctx, gpu)
    bounds = torch.zeros(blocks, 2, 2, 128, dtype=torch.bfloat16, device=gpu)
    cc.update_key_bounds(t["k"], bounds, dt, dc, i32(np.concatenate([[0], np.cumsum(ctx)]), gpu))
    q = torch.randn(3, 8, 128, device=gpu).bfloat16()
    new = torch.randn(2, 3, 2, 128, device=gpu).bfloat16()
    slots = i32([int(table[b, (c - 1) // 16]) * 16 + (c - 1) % 16 for b, c in enumerate(ctx)], gpu)

    def step():
        cc.write_kv_cache(new[0], new[1], t["k"], t["v"], slots)
        cc.update_key_bounds(t["k"], bounds, dt, dc)
        sc = cc.score_kv_blocks(q, bounds, dt, dc)
        sel = cc.select_kv_blocks(sc, dc, 12, 1, 2)
        return sc, sel, cc.sparse_decode_attention(q, t["k"], t["v"], dt, dc, sel)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(4):
        q.copy_(torch.randn(3, 8, 128, device=gpu))
        new.copy_(torch.randn(2, 3, 2, 128, device=gpu))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        held = (t["k"].clone(), bounds.clone())
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))
        assert torch.equal(held[0], t["k"]) and torch.equal(held[1], bounds)
