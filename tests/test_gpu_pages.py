"""Copy, table update and compaction of the paged cache on the GPU, against the same done block by
block (tests/_pages_ref.py): every number and every byte equal."""
import numpy as np
import pytest
import torch

import ccinfer_amd as cc
from tests import _pages_ref as P
from tests._util import say

pytestmark = pytest.mark.gpu


def i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)


class Pool:
    """Caches of all layers as random bits; `apart`: the layers lie apart and start off a 16-byte
    boundary (bf16)."""

    def __init__(self, dev, seed, layers, blocks, h, d, bs=16, fp8=False, apart=False):
        rng = np.random.default_rng(seed)
        self.fp8, self.bs, self.blocks, self.layers = fp8, bs, blocks, layers
        shape = (layers, blocks, bs, h, d)
        n = blocks * bs * h * d
        self.t = []
        for _ in range(2):
            a = torch.from_numpy(rng.integers(0, 256, shape).astype(np.uint8)).to(dev)
            if not fp8:
                a = torch.from_numpy(rng.integers(-2 ** 15, 2 ** 15, shape).astype(np.int16)) \
                    .to(dev).view(torch.bfloat16)
            if apart:
                buf = torch.zeros(layers * (n + 9) + 1, dtype=a.dtype, device=dev)
                v = torch.as_strided(buf, shape, (n + 9, bs * h * d, h * d, d, 1), 1)
                v.copy_(a)
                a = v
            self.t.append(a)
        self.s = [torch.from_numpy(rng.standard_normal((layers, blocks * h * 16))
                                   .astype(np.float32)).to(dev) for _ in range(2)] if fp8 else [None, None]
        self.kw = dict(k_scale=self.s[0], v_scale=self.s[1], cache_block_size=bs)
        self.h = h

    def caches(self):
        return [x.contiguous().view(torch.uint8 if self.fp8 else torch.int16).cpu().numpy()
                .reshape(self.layers, self.blocks, self.bs, -1) for x in self.t]

    def scales(self):
        return [x.cpu().numpy().reshape(self.layers, self.blocks, self.h, 16) for x in self.s] \
            if self.fp8 else []

    def flat(self):
        return self.caches() + [x.reshape(self.layers, self.blocks, -1) for x in self.scales()]


POOLS = [dict(layers=1, blocks=20, h=2, d=64), dict(layers=3, blocks=33, h=1, d=128, fp8=True),
         dict(layers=2, blocks=17, h=3, d=40, apart=True), dict(layers=5, blocks=50, h=8, d=128),
         dict(layers=2, blocks=40, h=1, d=6, bs=5), dict(layers=1, blocks=9, h=1, d=64, fp8=True),
         dict(layers=2, blocks=12, h=1, d=8, bs=1)]


# ---- copy ------------------------------------------------------------------------------

@pytest.mark.parametrize("pool", POOLS)
def test_copy(gpu, pool):
    say(f"copy {pool}")
    p = Pool(gpu, 1, **pool)
    rng = np.random.default_rng(5)
    for n in (1, 2, p.blocks // 2):
        order = rng.permutation(p.blocks)
        dst, src = order[:n].copy(), rng.choice(order[n:], n)
        status = torch.full((1,), 77, dtype=torch.int32, device=gpu)
        want, _ = P.copy(p.flat(), src, dst, p.blocks)
        cc.copy_kv_blocks(*p.t, i32(src, gpu), i32(dst, gpu), status=status, **p.kw)
        assert all(np.array_equal(a, b) for a, b in zip(p.flat(), want))
        assert status.item() == 77  # left alone


def test_copy_one_layer_shapes(gpu):
    say("copy one layer")
    p = Pool(gpu, 2, 1, 10, 2, 64)
    want, _ = P.copy(p.flat(), [3, 4], [9, 0], 10)
    k, v = p.t
    cc.copy_kv_blocks(k[0], v[0], i32([3], gpu), i32([9], gpu))                     # 4 dimensions
    cc.copy_kv_blocks(k.view(160, 2, 64), v.view(160, 2, 64), i32([4], gpu), i32([0], gpu))
    assert all(np.array_equal(a, b) for a, b in zip(p.flat(), want))
    cc.copy_kv_blocks(k, v, i32([], gpu), i32([], gpu))                             # nothing
    assert all(np.array_equal(a, b) for a, b in zip(p.flat(), want))


@pytest.mark.parametrize("pairs", [
    [(1, 2), (3, 2), (4, 5)],             # one destination, two sources
    [(1, 2), (2, 3), (4, 5)],             # a chain
    [(1, 2), (2, 1), (4, 5)],             # a swap
    [(1, 2), (1, 2), (1, 3), (7, 7), (2, 2)],  # twice the same; blocks on themselves
    [(-1, 2), (1, -1), (40, 3), (3, 40), (5, 2 ** 31 - 1), (-2 ** 31, 6), (4, 5)],
    [(0, 9), (9, 9), (1, 8), (8, -1)],
])
def test_copy_pairs_that_depend_on_an_order(gpu, pairs):
    say(f"copy {pairs}")
    p = Pool(gpu, 3, 2, 40, 1, 64)
    src, dst = [a for a, _ in pairs], [b for _, b in pairs]
    want, code = P.copy(p.flat(), src, dst, p.blocks)
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    cc.copy_kv_blocks(*p.t, i32(src, gpu), i32(dst, gpu), status=status)
    assert all(np.array_equal(a, b) for a, b in zip(p.flat(), want))
    assert status.item() == code


# ---- update ----------------------------------------------------------------------------

class Tables:
    def __init__(self, dev, rows, width, blocks):
        self.dev = dev
        self.t = np.full((rows, width), -1, np.int32)
        self.c, self.r = np.zeros(rows, np.int32), np.zeros(blocks, np.int32)
        self.up()

    def up(self):
        self.dt, self.dc, self.dr = (i32(x, self.dev) for x in (self.t, self.c, self.r))

    def step(self, p, dst, src, lengths, caches=True, **kw):
        """One update on both sides; returns the status."""
        dev = lambda x: None if x is None else i32(x, self.dev)  # noqa: E731
        lists = p.caches(), p.scales()
        t, c, r, cs, ss, code = P.update(self.t, self.c, self.r, dst, src, lengths, *lists, p.bs,
                                         have_caches=caches)
        args = p.t if caches else (None, None)
        opts = p.kw if caches else dict(cache_block_size=p.bs)
        status = cc.update_block_tables(self.dt, self.dc, self.dr, i32(dst, self.dev), dev(src),
                                        dev(lengths), *args, **opts, **kw)
        assert status.item() == code
        for got, want in ((self.dt, t), (self.dc, c), (self.dr, r)):
            assert np.array_equal(got.cpu().numpy(), want)
        assert all(np.array_equal(a, b) for a, b in zip(p.caches(), cs))
        assert all(np.array_equal(a, b) for a, b in zip(p.scales(), ss))
        self.t, self.c, self.r = t, c, r
        P.consistent(t, c, r, p.bs)
        return code


@pytest.mark.parametrize("pool", POOLS)
def test_update_random_steps(gpu, pool):
    say(f"update {pool}")
    p = Pool(gpu, 7, **{**pool, "blocks": 60})
    rng = np.random.default_rng(11)
    rows, width = 7, 9
    x = Tables(gpu, rows, width, p.blocks)
    codes = set()
    for k in range(25):
        n = int(rng.integers(1, rows + 1))
        dst = rng.permutation(rows)[:n]
        kind = rng.integers(0, 4, n)
        src = np.where(kind == 0, -1, np.where(kind == 1, dst, rng.integers(0, rows, n)))
        lengths = np.where(rng.random(n) < 0.4, -1, rng.integers(0, width * p.bs + 1, n))
        if k % 5 == 4:
            lengths = None
        codes.add(x.step(p, dst, None if k % 7 == 6 else src, lengths))
    assert 0 in codes


def test_update_each_use(gpu):
    say("update uses")
    p = Pool(gpu, 8, 3, 64, 2, 64)
    x = Tables(gpu, 6, 8, 64)
    assert x.step(p, [0, 1], [-1, -1], [50, 33]) == 0          # admit
    assert x.t[0, :4].tolist() == [0, 1, 2, 3] and x.t[1, :3].tolist() == [4, 5, 6]
    assert x.step(p, [2, 3], [0, 0], None) == 0                # fork: three shared, one own each
    assert x.t[2].tolist() == [0, 1, 2, 7, -1, -1, -1, -1] and x.r[0] == 3 and x.r[3] == 1
    assert x.step(p, [0, 2], None, [64, 65]) == 0              # grow: in the block, into a next
    assert x.step(p, [3], [3], [20]) == 0                      # back into a shared block: copied
    assert x.t[3, 1] not in (1, -1) and x.r[1] == 2
    assert x.step(p, [3], [3], [16]) == 0                      # whole blocks stay shared
    assert x.step(p, [0, 1], [1, 0], None) == 0                # rows change places
    assert x.c.tolist()[:2] == [33, 64]
    assert x.step(p, [0, 1, 2, 3], [-1] * 4, [0] * 4) == 0     # release everything
    assert not x.r.any()
    assert x.step(p, [], [], []) == 0                          # nothing


def test_row_cut_back_into_a_block_that_another_takes_over(gpu):
    # row 0 ends inside block 1 from now on, while row 1 is forked from it with block 1 whole: one
    # of them has to have its own
    say("update cut and fork")
    for fp8 in (False, True):
        p = Pool(gpu, 12, 2, 32, 1, 64, fp8=fp8)
        x = Tables(gpu, 4, 4, 32)
        assert x.step(p, [0], [-1], [50]) == 0
        assert x.step(p, [0, 1], [0, 0], [20, 50]) == 0
        assert x.t[0, 1] != x.t[1, 1] and x.t[0, 0] == x.t[1, 0]
        # the other fork ends in the block too: its tokens are copied, row 0 keeps the block
        b = x.t[0, 1]
        assert x.step(p, [2, 0], [0, 0], [18, 17]) == 0 and x.t[0, 1] == b != x.t[2, 1]
        # ends before the block, or at its start
        assert x.step(p, [2, 0, 3], [0, 0, 0], [7, 18, 16]) == 0 and x.t[0, 1] == b
        assert x.step(p, [0, 2, 3], [1, 1, 1], [32, -1, 33]) == 0
        assert x.step(p, [1, 0, 3], [1, 1, 1], [30, 32, 31]) == 0


def test_update_refused_by_the_device_changes_nothing(gpu):
    say("update refused")
    p = Pool(gpu, 9, 2, 32, 1, 64)
    x = Tables(gpu, 5, 8, 32)
    assert x.step(p, [0, 1], [-1, -1], [40, 17]) == 0
    for dst, src, lengths, code in [
            ([2, 2], [0, 1], None, 6), ([5], [0], None, 6), ([-1], [0], None, 6),
            ([2], [5], None, 6), ([2], [-2], None, 6), ([2], [0], [129], 6), ([2], [0], [-2], 6),
            ([0, 1, 2, 3, 4], [0, 1, -1, -1, -1], [128] * 5, 12),  # 40 blocks of 32
            ([2, 0], [0, 7], None, 6)]:
        assert x.step(p, dst, src, lengths) == code, (dst, src, lengths)
    assert x.step(p, [2], [0], None, caches=False) == 6        # a copy, and nothing to copy in
    assert x.step(p, [2], [0], [32], caches=False) == 0        # whole blocks alone need none
    assert x.step(p, [2], [-1], [0], caches=False) == 0
    keep = x.t.copy(), x.c.copy(), x.r.copy()
    for k, change in enumerate([lambda: x.t.__setitem__((0, 1), 32), lambda: x.t.__setitem__((0, 2), -1),
                                lambda: x.c.__setitem__(0, 129), lambda: x.c.__setitem__(0, -1),
                                lambda: x.r.__setitem__(x.t[0, 0], 0)]):
        change()
        x.up()
        for dst, src in (([2], [0]), ([0], [-1])):
            status = cc.update_block_tables(x.dt, x.dc, x.dr, i32(dst, gpu), i32(src, gpu), None,
                                            *p.t)
            assert status.item() == 14, k
            for got, want in ((x.dt, x.t), (x.dc, x.c), (x.dr, x.r)):
                assert np.array_equal(got.cpu().numpy(), want)
        x.t, x.c, x.r = (a.copy() for a in keep)
    x.up()
    # five blocks are held: the last free one is handed out, then none is left
    assert x.step(p, [2, 3, 4, 0], [-1, -1, -1, 0], [128, 128, 128, 96]) == 0
    assert (x.r > 0).all() and x.step(p, [1], [1], [33]) == 12
    assert x.step(p, [2, 1], [-1, 1], [0, 33]) == 12           # what it releases is free after it
    assert x.step(p, [2], [-1], [0]) == 0 and x.step(p, [1], [1], [33]) == 0


@pytest.mark.parametrize("blocks", [4095, 4096, 4097, 64 * 64 * 5 + 70])
def test_update_over_many_chunks(gpu, blocks):
    say(f"update {blocks} blocks")
    p = Pool(gpu, 10, 1, blocks, 1, 2, bs=2)
    rng = np.random.default_rng(blocks)
    rows, width = 6, blocks // 2
    x = Tables(gpu, rows, width, blocks)
    # most of the pool held by one row, holes scattered by truncating and forking
    assert x.step(p, [0, 1], [-1, -1], [blocks - 40, blocks // 2 - 7]) == 0
    assert x.step(p, [0], [0], [blocks // 2 + 1]) == 0
    assert x.step(p, [2, 3], [1, 0], None) == 0
    assert x.step(p, [1], [-1], [0]) == 0
    held = x.r.copy()
    assert x.step(p, [4], [-1], [(int((held == 0).sum()) // 2) * 2]) == 0
    assert x.step(p, [0, 5], [-1, 4], [0, -1]) == 0
    for _ in range(4):
        x.step(p, rng.permutation(rows)[:3], rng.integers(-1, rows, 3),
               rng.integers(0, blocks // 8, 3))


def test_update_refusals(gpu):
    say("update refusals")
    p = Pool(gpu, 1, 2, 8, 1, 64)
    x = Tables(gpu, 3, 4, 8)
    one = i32([0], gpu)
    ws = torch.empty(64, dtype=torch.uint8, device=gpu)

    def call(table=x.dt, ctx=x.dc, refs=x.dr, dst=one, src=one, lengths=one, k=p.t[0], v=p.t[1],
             **kw):
        return cc.update_block_tables(table, ctx, refs, dst, src, lengths, k, v, **kw)
    call()
    for i, kw in enumerate([dict(table=x.dt.long()), dict(ctx=x.dc[:2]), dict(refs=x.dr[:7]),
                            dict(src=x.dc), dict(lengths=x.dc), dict(v=None), dict(k=None),
                            dict(workspace=ws), dict(status=x.dc), dict(cache_block_size=8),
                            dict(k_scale=torch.zeros(2, 128, device=gpu)), dict(table=x.dt.t()),
                            dict(k=p.t[0].float(), v=p.t[1].float()), dict(v=p.t[1][:1])]):
        with pytest.raises(cc.CcinferError) as e:
            call(**kw)
        assert e.value.code == 6, i


# ---- compact ---------------------------------------------------------------------------

def compact_both(gpu, p, table, refs, in_place=False):
    wt, wr, wm, wn, wc = P.compact(table, refs, p.flat())
    dt, dr = i32(table, gpu), i32(refs, gpu)
    out = None
    if in_place:
        out = {"block_table": dt, "ref_counts": dr, "remap": torch.empty_like(dr),
               "num_live": torch.empty(1, dtype=torch.int32, device=gpu)}
    out = cc.compact_kv_blocks(dt, dr, *p.t, **p.kw, out=out)
    assert out["num_live"].item() == wn
    for name, want in (("block_table", wt), ("ref_counts", wr), ("remap", wm)):
        assert np.array_equal(out[name].cpu().numpy(), want), name
    # every live block's data; what is left behind is free
    for a, b in zip(p.flat(), wc):
        assert np.array_equal(a, b)
    if not in_place:
        assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pool", POOLS)
def test_compact(gpu, pool, in_place):
    say(f"compact {pool} {in_place}")
    rng = np.random.default_rng(21)
    for share in (0.0, 0.2, 0.5, 0.9, 1.0):
        p = Pool(gpu, 22, **pool)
        refs = np.where(rng.random(p.blocks) < share, rng.integers(1, 5, p.blocks), 0)
        table = rng.integers(-3, p.blocks + 4, (4, 6))
        compact_both(gpu, p, table.astype(np.int32), refs.astype(np.int32), in_place)


@pytest.mark.parametrize("blocks,live", [(4096, 4096), (4096, 0), (8192, 4096), (8193, 4097),
                                         (9000, 4095), (20000, 13000), (70000, 300)])
def test_compact_over_many_chunks(gpu, blocks, live):
    say(f"compact {blocks} {live}")
    rng = np.random.default_rng(blocks + live)
    p = Pool(gpu, 23, 1, blocks, 1, 2, bs=1)
    refs = np.zeros(blocks, np.int32)
    refs[rng.permutation(blocks)[:live]] = rng.integers(1, 9, live)
    table = rng.integers(-1, blocks, (50, 301)).astype(np.int32)
    compact_both(gpu, p, table, refs)


def test_compact_without_tables(gpu):
    say("compact no tables")
    p = Pool(gpu, 24, 2, 30, 1, 64)
    refs = np.zeros(30, np.int32)
    refs[[3, 29, 17]] = 1
    compact_both(gpu, p, np.zeros((0, 5), np.int32), refs)


def test_compact_refusals(gpu):
    say("compact refusals")
    p = Pool(gpu, 1, 2, 8, 1, 64)
    t, r = i32(np.zeros((2, 3)), gpu), i32(np.ones(8), gpu)
    ok = cc.compact_kv_blocks(t, r, *p.t)
    for i, call in enumerate([
            lambda: cc.compact_kv_blocks(t, r[:7], *p.t),
            lambda: cc.compact_kv_blocks(t.long(), r, *p.t),
            lambda: cc.compact_kv_blocks(t, r, p.t[0], p.t[1][:1]),
            lambda: cc.compact_kv_blocks(t, r, *p.t, out={**ok, "remap": r[:7]}),
            lambda: cc.compact_kv_blocks(t, r, *p.t, workspace=t),
            lambda: cc.compact_kv_blocks(t[0], r, *p.t)]):
        with pytest.raises(cc.CcinferError) as e:
            call()
        assert e.value.code == 6, i


# ---- far offsets, graphs ----------------------------------------------------------------

def test_blocks_past_two_and_four_gib(gpu):
    # one layer's K of 4.5 GiB: byte offsets past 2^32
    say("pages far offsets")
    blocks, h, d = 147456, 8, 128
    k = torch.zeros(blocks, 16, h, d, dtype=torch.bfloat16, device=gpu)
    v = torch.zeros(blocks, 16, h, d, dtype=torch.bfloat16, device=gpu)
    far = blocks - 1
    k[far], v[far], k[70000] = 3.0, 4.0, 5.0
    cc.copy_kv_blocks(k, v, i32([far, 70000], gpu), i32([far - 1, 2], gpu))
    assert (k[far - 1] == 3).all() and (v[far - 1] == 4).all() and (k[2] == 5).all()
    assert not k[far - 2].any() and not k[3].any()
    refs = torch.zeros(blocks, dtype=torch.int32, device=gpu)
    refs[far], refs[0], refs[1] = 1, 1, 1
    table = i32([[0, 1, far]], gpu)
    out = cc.compact_kv_blocks(table, refs, k, v)
    assert out["block_table"].tolist() == [[0, 1, 2]] and (k[2] == 3).all() and (v[2] == 4).all()
    ctx = i32([40, 0], gpu)
    table = i32([[0, 1, far], [-1, -1, -1]], gpu)
    refs = torch.ones(blocks, dtype=torch.int32, device=gpu)
    refs[far - 5] = 0
    status = cc.update_block_tables(table, ctx, refs, i32([1], gpu), i32([0], gpu), None, k, v)
    assert status.item() == 0 and table.tolist()[1] == [0, 1, far - 5]
    assert (k[far - 5, :8] == 3).all() and not k[far - 5, 8:].any()


def test_update_and_compact_in_replayed_graphs(gpu):
    say("pages graph")
    p, e = (Pool(gpu, 30, 2, 64, 2, 64) for _ in range(2))
    x, y = Tables(gpu, 8, 6, 64), Tables(gpu, 8, 6, 64)
    dst, src, n = i32(np.zeros(3), gpu), i32(np.zeros(3), gpu), i32(np.zeros(3), gpu)
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=gpu)  # both graphs' and the eager calls'
    out = {"block_table": x.dt, "ref_counts": x.dr, "remap": torch.empty_like(x.dr),
           "num_live": torch.empty(1, dtype=torch.int32, device=gpu)}

    def update():
        cc.update_block_tables(x.dt, x.dc, x.dr, dst, src, n, *p.t, workspace=ws, status=status)

    def compact():
        cc.compact_kv_blocks(x.dt, x.dr, *p.t, workspace=ws, out=out)

    dst.copy_(i32([0, 1, 2], gpu)), src.fill_(-1), n.fill_(0)
    update()  # (of empty rows)
    compact()
    torch.cuda.synchronize()
    graphs = []
    for call in (update, compact):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call()
    rng = np.random.default_rng(31)
    for k in range(8):
        a, b, c = rng.permutation(8)[:3], rng.integers(-1, 8, 3), rng.integers(-1, 60, 3)
        for t, v in ((dst, a), (src, b), (n, c)):
            t.copy_(i32(v, gpu))
        graphs[0].replay()
        want = cc.update_block_tables(y.dt, y.dc, y.dr, i32(a, gpu), i32(b, gpu), i32(c, gpu), *e.t)
        assert status.item() == want.item()
        if k % 2:
            graphs[1].replay()
            o = cc.compact_kv_blocks(y.dt, y.dr, *e.t)
            y.dt, y.dr = o["block_table"], o["ref_counts"]
            assert torch.equal(out["remap"], o["remap"])
        for u, w in ((x.dt, y.dt), (x.dc, y.dc), (x.dr, y.dr)):
            assert torch.equal(u, w)
        assert all(np.array_equal(u, w) for u, w in zip(p.flat(), e.flat()))
        P.consistent(y.dt.cpu().numpy(), y.dc.cpu().numpy(), y.dr.cpu().numpy(), 16)


# ---- many items ---------------------------------------------------------------------------

@pytest.mark.parametrize("rows,fp8", [(300, False), (1500, True), (5000, False)])
def test_update_of_many_rows(gpu, rows, fp8):
    # more items than a workgroup has lanes, and more than leave one workgroup for each part
    say(f"update {rows} rows {fp8}")
    p = Pool(gpu, 50, 3, 4 * rows, 1, 32, fp8=fp8)
    rng = np.random.default_rng(rows)
    x = Tables(gpu, rows, 3, p.blocks)
    some = rng.permutation(rows)[:rows // 2]
    assert x.step(p, some, np.full(len(some), -1), rng.integers(1, 20, len(some))) == 0
    rest = np.setdiff1d(np.arange(rows), some)
    assert x.step(p, rest, rng.choice(some, len(rest)), None) == 0      # forks
    assert x.step(p, np.arange(rows), None, x.c + 1) == 0               # a step of every row
    assert x.step(p, rng.permutation(rows), rng.integers(-1, rows, rows), None) == 0  # all change


# ---- layers held one by one ----------------------------------------------------------------

@pytest.mark.parametrize("fp8", [False, True])
def test_copies_told_and_done_layer_by_layer(gpu, fp8):
    say(f"copies told {fp8}")
    p, q = (Pool(gpu, 60, 3, 60, 2, 64, fp8=fp8) for _ in range(2))  # the same bits
    x, y = Tables(gpu, 7, 9, 60), Tables(gpu, 7, 9, 60)
    rng = np.random.default_rng(61)
    told = 0
    for k in range(20):
        n = int(rng.integers(1, 8))
        dst, src = rng.permutation(7)[:n], rng.integers(-1, 7, n)
        lengths = np.where(rng.random(n) < 0.5, -1, rng.integers(0, 9 * 16 + 1, n))
        if k == 10:
            lengths[0] = 9 * 16 + 1  # fails: nothing to copy
        ctx0 = x.c.copy()
        a, b = (torch.full((n,), 77, dtype=torch.int32, device=gpu) for _ in range(2))
        code = x.step(p, dst, src, lengths, copies=(a, b))
        assert (code == 6) == (k == 10)
        c, d = (torch.full((n,), 77, dtype=torch.int32, device=gpu) for _ in range(2))
        status = cc.update_block_tables(y.dt, y.dc, y.dr, i32(dst, gpu), i32(src, gpu),
                                        i32(lengths, gpu), copies=(c, d))
        assert status.item() == code and torch.equal(a, c) and torch.equal(b, d)
        for u, w in ((x.dt, y.dt), (x.dc, y.dc), (x.dr, y.dr)):
            assert torch.equal(u, w)
        if code:
            assert (a == -1).all() and (b == -1).all()
        told += int((a >= 0).sum())
        for layer in range(3):
            s = {} if not fp8 else {"k_scale": q.s[0][layer], "v_scale": q.s[1][layer]}
            cc.copy_kv_blocks(q.t[0][layer], q.t[1][layer], c, d, **s)
        # A whole block is copied there, its held tokens here. The tokens past those are written
        # before they are read, as a server's step does; then what is held is the same.
        table, ctx = x.t, x.c
        for i in range(n if code == 0 else 0):
            kept = min(int(ctx[dst[i]]), int(ctx0[src[i]]) if src[i] >= 0 else 0)
            for pos in range(kept, int(ctx[dst[i]])):
                blk = table[dst[i], pos // 16]
                for u in (*p.t, *q.t):
                    u[:, blk, pos % 16] = pos % 7
                for u in (*p.s, *q.s) if fp8 else ():
                    u.view(3, 60, 2, 16)[:, blk, :, pos % 16] = pos
        for row, n_row in zip(table, ctx):
            for j, blk in enumerate(row[:-(-int(n_row) // 16)]):
                tokens = min(16, int(n_row) - 16 * j)
                for u, w in zip(p.caches(), q.caches()):
                    assert np.array_equal(u[:, blk, :tokens], w[:, blk, :tokens])
                for u, w in zip(p.scales(), q.scales()):
                    assert np.array_equal(u[:, blk, :, :tokens], w[:, blk, :, :tokens])
    assert told > 5
    one = i32([0], gpu)
    for bad in ((one, i32([0, 1], gpu)), (one, one.long())):
        with pytest.raises(cc.CcinferError):
            cc.update_block_tables(y.dt, y.dc, y.dr, one, one, None, copies=bad)


# ---- counts below zero ---------------------------------------------------------------------

@pytest.mark.parametrize("blocks", [24, 30000])
def test_block_given_up_too_often_is_never_handed_out(gpu, blocks):
    # rows 0 and 1 hold block 5, which is counted once: both leave in one call, its count is -1,
    # and no later row may get it. 30000: past the blocks that one workgroup's words cover.
    say(f"count below zero {blocks}")
    p = Pool(gpu, 70, 1, blocks, 1, 8)
    rows = i32([[5, -1, -1, -1], [5, -1, -1, -1], [-1] * 4, [-1] * 4], gpu)
    ctx, refs = i32([16, 16, 0, 0], gpu), i32(np.ones(blocks), gpu)
    refs[[2, 9, blocks - 1]] = 0

    def step(dst, src, lengths):
        return cc.update_block_tables(rows, ctx, refs, i32(dst, gpu), i32(src, gpu),
                                      i32(lengths, gpu), *p.t).item()
    assert step([0, 1], [-1, -1], [0, 0]) == 0
    assert refs[5].item() == -1 and not ctx.any()
    assert step([0], [-1], [16]) == 0 and rows[0].tolist() == [2, -1, -1, -1]
    assert step([1], [-1], [32]) == 0 and rows[1].tolist() == [9, blocks - 1, -1, -1]
    assert step([2], [-1], [16]) == 12                     # nothing is left
    rows[3, 0], ctx[3] = 5, 16                             # a row that holds it all the same
    assert step([3], [3], [10]) == 14 and step([2], [3], [-1]) == 14
    assert refs[5].item() == -1 and rows[3].tolist() == [5, -1, -1, -1]


@pytest.mark.parametrize("blocks", [24, 3000])
def test_compaction_keeps_blocks_of_counts_below_zero(gpu, blocks):
    # such a block is not free: nothing is moved over it, and it goes on with its count
    say(f"compact count below zero {blocks}")
    p = Pool(gpu, 71, 2, blocks, 1, 8)
    refs = np.zeros(blocks, np.int32)
    refs[[1, 4, blocks - 1]], refs[[0, blocks - 3]] = (2, 1, 3), (-1, -2)
    table = np.array([[1, 4, blocks - 1], [0, blocks - 3, 7]], np.int32)
    # the same with the counts' signs aside, which the reference takes as it should
    wt, wr, wm, wn, wc = P.compact(table, np.abs(refs), p.flat())
    out = cc.compact_kv_blocks(i32(table, gpu), i32(refs, gpu), *p.t)
    assert out["num_live"].item() == wn == 5
    assert np.array_equal(out["block_table"].cpu().numpy(), wt)
    assert np.array_equal(out["remap"].cpu().numpy(), wm)
    sign = np.zeros(blocks, np.int32)
    sign[wm[refs != 0]] = np.sign(refs[refs != 0])
    assert np.array_equal(out["ref_counts"].cpu().numpy(), wr * sign)
    for a, b in zip(p.flat(), wc):
        assert np.array_equal(a, b)


# ---- arguments -----------------------------------------------------------------------------

def test_block_size_of_zero_is_refused(gpu):
    say("block size 0")
    p = Pool(gpu, 72, 1, 8, 1, 64)
    k, v = (x.view(8 * 16, 1, 64) for x in p.t)
    x = Tables(gpu, 2, 4, 8)
    one = i32([0], gpu)
    for bs in (0, -16):
        for i, call in enumerate([
                lambda: cc.copy_kv_blocks(k, v, one, one, cache_block_size=bs),
                lambda: cc.compact_kv_blocks(x.dt, x.dr, k, v, cache_block_size=bs),
                lambda: cc.update_block_tables(x.dt, x.dc, x.dr, one, one, one, k, v,
                                               cache_block_size=bs),
                lambda: cc.update_block_tables(x.dt, x.dc, x.dr, one, one, one,
                                               cache_block_size=bs)]):
            with pytest.raises(cc.CcinferError) as e:
                call()
            assert e.value.code == 6, (bs, i)


def test_lists_and_tables_of_more_than_31_bits_are_refused(gpu):
    # lengths that a 32-bit argument would take for 5 elements, 2 rows or 3 columns
    say("past 31 bits")
    p = Pool(gpu, 73, 1, 8, 1, 64)
    x = Tables(gpu, 2, 4, 8)
    one = i32([0], gpu)
    far = torch.zeros(2 ** 32 + 8, dtype=torch.int32, device=gpu)
    long, tall, wide = far[:2 ** 32 + 5], far[:2 ** 32 + 2], far[:2 ** 32 + 3]
    for i, call in enumerate([
            lambda: cc.copy_kv_blocks(*p.t, long, long),
            lambda: cc.update_block_tables(tall.view(-1, 1), tall, x.dr, one, one, one, *p.t),
            lambda: cc.update_block_tables(wide.view(1, -1), one, x.dr, one, one, one, *p.t),
            lambda: cc.update_block_tables(x.dt, x.dc, x.dr, long, long, long, *p.t),
            lambda: cc.update_block_tables(x.dt, x.dc, x.dr, one, one, one,
                                           cache_block_size=2 ** 32 + 16),
            lambda: cc.update_block_tables(x.dt, x.dc, far, one, one, one),
            lambda: cc.compact_kv_blocks(tall.view(-1, 1), x.dr, *p.t,
                                         out={"block_table": tall.view(-1, 1), "ref_counts": x.dr,
                                              "remap": torch.empty_like(x.dr), "num_live": one}),
            lambda: cc.compact_kv_blocks(wide.view(1, -1), x.dr, *p.t,
                                         out={"block_table": wide.view(1, -1), "ref_counts": x.dr,
                                              "remap": torch.empty_like(x.dr), "num_live": one})]):
        with pytest.raises(cc.CcinferError) as e:
            call()
        assert e.value.code == 6, i



def test_caches_of_more_than_31_bits_a_side_are_refused(gpu):
    # 2^32 + 2 elements a head, heads or layers, 2^32 + 16 tokens a block
    say("caches past 31 bits")
    far = torch.zeros(17, 2 ** 32 + 16, dtype=torch.uint8, device=gpu)
    k = far.view(-1)[:16 * (2 ** 32 + 2)].view(torch.bfloat16)
    one, refs, rows = i32([0], gpu), i32([1], gpu), i32([[0]], gpu)
    tokens = far[:2].view(-1).view(torch.bfloat16)
    for i, cache in enumerate([k.view(1, 1, 4, 1, -1), k.view(1, 1, 4, -1, 1),
                               tokens.view(1, 1, -1, 1, 1), k.view(-1, 1, 4, 1, 2)]):
        for call in (lambda: cc.copy_kv_blocks(cache, cache, one, one,
                                               cache_block_size=cache.shape[2]),
                     lambda: cc.update_block_tables(rows, one, refs, one, None, None, cache, cache,
                                                    cache_block_size=cache.shape[2]),
                     lambda: cc.compact_kv_blocks(rows, refs, cache, cache,
                                                  cache_block_size=cache.shape[2])):
            assert max(cache.shape) > 2 ** 32
            with pytest.raises(cc.CcinferError) as e:
                call()
            assert e.value.code == 6, (i, cache.shape)


# ---- blocks of more than one round of loads, scales past a workgroup, single bytes ------------

# Parts of more than 2048 units (a round of a workgroup's loads) of 16, 2 and 1 bytes, more than
# 256 scales a block, and fp8 caches whose tokens or starts are no multiples of 16 bytes.
WIDE_POOLS = [dict(layers=2, blocks=20, h=32, d=128), dict(layers=2, blocks=20, h=32, d=128, fp8=True),
              dict(layers=2, blocks=20, h=8, d=128, bs=32), dict(layers=2, blocks=20, h=8, d=256),
              dict(layers=2, blocks=17, h=9, d=36, apart=True),
              dict(layers=3, blocks=20, h=1, d=72, fp8=True),
              dict(layers=2, blocks=17, h=18, d=68, fp8=True),
              dict(layers=2, blocks=17, h=3, d=40, apart=True, fp8=True)]


@pytest.mark.parametrize("pool", WIDE_POOLS)
def test_copy_of_wide_blocks(gpu, pool):
    test_copy(gpu, pool)


@pytest.mark.parametrize("pool", WIDE_POOLS)
def test_update_of_wide_blocks(gpu, pool):
    test_update_random_steps(gpu, pool)


@pytest.mark.parametrize("pool", WIDE_POOLS)
def test_compact_of_wide_blocks(gpu, pool):
    test_compact(gpu, pool, False)
