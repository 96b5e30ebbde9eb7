"""The operators together, as a server with its block tables on the device uses them: a table of
positions, requests admitted, prompts through norm + rotation + write and prefill, requests
forked, grown and decoded step by step, one released, the pool compacted. Every attention output
against attention in 64 bits over each request's own history."""
import math

import numpy as np
import pytest
import torch

import ccinfer_amd as cc
from tests import _pages_ref as P
from tests import _rotary_ref as R
from tests._util import MAX_ABS, MEAN_ABS, say

pytestmark = pytest.mark.gpu

HQ, HKV, D, ROT, LAYERS, BLOCKS, ROWS, WIDTH = 8, 2, 128, 96, 2, 80, 6, 12
EPS = 1e-6


def stored(x, fp8):
    """x [..., d] as the cache holds it."""
    t = torch.from_numpy(x)
    if not fp8:
        return t.to(torch.bfloat16).double().numpy()
    p = torch.from_numpy(R.row_scale(x))[..., None]
    return ((t / p).float().to(torch.float8_e4m3fn).double() * p).numpy()


class Server:
    def __init__(self, dev, fp8):
        self.dev, self.fp8 = dev, fp8
        self.rng = np.random.default_rng(40 + fp8)
        scaling = {"type": "yarn", "factor": 4.0, "original_max_position": 64}
        self.rope = cc.build_rope_cache(WIDTH * 16, ROT, 1e4, scaling)
        self.tab = self.rope.cpu().numpy()
        shape = (LAYERS, BLOCKS, 16, HKV, D)
        if fp8:
            self.k, self.v = (torch.full(shape, 0x7f, dtype=torch.uint8, device=dev) for _ in "kv")
            n = cc.fp8_scale_numel(BLOCKS * 16, HKV)
            # codes of slots that hold no token may be anything, scales anything finite
            self.ks, self.vs = (torch.full((LAYERS, n), 2.0 ** 100, device=dev) for _ in "kv")
        else:
            self.k, self.v = (torch.full(shape, math.nan, dtype=torch.bfloat16, device=dev)
                              for _ in "kv")
            self.ks = self.vs = None
        i32 = dict(dtype=torch.int32, device=dev)
        self.table = torch.full((ROWS, WIDTH), -1, **i32)
        self.ctx, self.refs = torch.zeros(ROWS, **i32), torch.zeros(BLOCKS, **i32)
        w = lambda: (1 + 0.2 * self.rng.standard_normal((LAYERS, D))).astype(np.float32)  # noqa: E731
        self.qw, self.kw = (torch.from_numpy(w()).to(dev).bfloat16() for _ in "qk")
        # each row's keys and values, layer by layer, as the cache should hold them
        self.past = [[[np.zeros((0, HKV, D))] * 2 for _ in range(LAYERS)] for _ in range(ROWS)]

    def tensor(self, a):
        return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(self.dev)

    def scales(self, layer):
        return dict(k_scale=self.ks[layer], v_scale=self.vs[layer]) if self.fp8 else {}

    def update(self, dst, src, lengths):
        status = cc.update_block_tables(
            self.table, self.ctx, self.refs, self.tensor(dst),
            None if src is None else self.tensor(src),
            None if lengths is None else self.tensor(lengths), self.k, self.v, k_scale=self.ks,
            v_scale=self.vs)
        assert status.item() == 0
        P.consistent(self.table.cpu().numpy(), self.ctx.cpu().numpy(), self.refs.cpu().numpy(), 16)

    def slots(self, rows, pos):
        """Where the tokens of these rows and positions lie, from the table on the device."""
        r, p = self.tensor(rows).long(), self.tensor(pos).long()
        return (self.table[r, p // 16] * 16 + p % 16).int()

    def norm(self, layer, qkv, rows, pos):
        return cc.qkv_norm_rope(qkv, self.qw[layer], self.kw[layer], self.tensor(pos), self.rope,
                                self.slots(rows, pos), self.k[layer], self.v[layer], HQ, EPS,
                                interleaved=True, **self.scales(layer))

    def tokens(self, rows, pos):
        """New tokens' projections, and their rows in 64 bits: q, and k, v into the histories."""
        out = []
        for layer in range(LAYERS):
            x = self.rng.standard_normal((len(rows), (HQ + 2 * HKV) * D)).astype(np.float32)
            qkv = torch.from_numpy(x).to(self.dev).bfloat16()
            y = qkv.double().cpu().numpy().reshape(len(rows), HQ + 2 * HKV, D)
            w = [t[layer].double().cpu().numpy() for t in (self.qw, self.kw)]
            q, _ = R.rotate(R.norm(y[:, :HQ], w[0], EPS), pos, self.tab, True)
            k, _ = R.rotate(R.norm(y[:, HQ:HQ + HKV], w[1], EPS), pos, self.tab, True)
            k, v = stored(k, self.fp8), stored(y[:, HQ + HKV:], self.fp8)
            for i, r in enumerate(rows):
                past = self.past[r][layer]
                assert len(past[0]) == pos[i]
                self.past[r][layer] = [np.concatenate([past[0], k[i:i + 1]]),
                                       np.concatenate([past[1], v[i:i + 1]])]
            out.append((qkv, q))
        return out

    def want(self, layer, row, q, n):
        """Attention of q [hq, d] over the row's first n positions."""
        k, v = (x[:n] for x in self.past[row][layer])
        g = HQ // HKV
        s = np.einsum("hgd,nhd->hgn", q.reshape(HKV, g, D), k) / math.sqrt(D)
        p = np.exp(s - s.max(-1, keepdims=True))
        return np.einsum("hgn,nhd->hgd", p / p.sum(-1, keepdims=True), v).reshape(HQ, D)

    def check(self, got, want, what):
        err = np.abs(got.double().cpu().numpy() - want)
        # an fp8 row can lie a step (2^-3 at most) off its own where float32 and 64 bits round
        # to different codes: rare, so the mean keeps the bf16 bar
        assert np.isfinite(err).all() and err.mean() <= MEAN_ABS, what
        assert err.max() <= (2 * MAX_ABS if self.fp8 else MAX_ABS), (what, err.max())

    def prompts(self, rows, lengths):
        which = np.repeat(rows, lengths)
        pos = np.concatenate([np.arange(n) for n in lengths])
        qsl = self.tensor(np.concatenate([[0], np.cumsum(lengths)]))
        at = self.tensor(rows).long()
        for layer, (qkv, q) in enumerate(self.tokens(which, pos)):
            rotated = self.norm(layer, qkv, which, pos)
            args = [self.k[layer].view(-1, HKV, D), self.v[layer].view(-1, HKV, D)]
            meta = [self.table[at].contiguous(), qsl, self.ctx[at].contiguous()]
            if self.fp8:
                o = cc.prefill_attention_fp8(rotated, *args, self.ks[layer], self.vs[layer], *meta)
            else:
                o = cc.prefill_attention(rotated, *args, *meta)
            want = np.stack([self.want(layer, r, q[i], p + 1)
                             for i, (r, p) in enumerate(zip(which, pos))])
            self.check(o, want, f"prefill layer {layer}")

    def attend(self, layer, q, rows):
        at = self.tensor(rows).long()
        args = [self.k[layer].view(-1, HKV, D), self.v[layer].view(-1, HKV, D)]
        meta = [self.table[at].contiguous(), self.ctx[at].contiguous()]
        if self.fp8:
            return cc.decode_attention_fp8(q, *args, self.ks[layer], self.vs[layer], *meta)
        return cc.decode_attention(q, *args, *meta)

    def step(self, rows):
        """One new token for each of these rows; returns each layer's (q, output)."""
        pos = self.ctx.cpu().numpy()[rows]
        self.update(rows, None, pos + 1)
        out = []
        for layer, (qkv, q) in enumerate(self.tokens(rows, pos)):
            rotated = self.norm(layer, qkv, rows, pos)
            o = self.attend(layer, rotated, rows)
            want = np.stack([self.want(layer, r, q[i], pos[i] + 1) for i, r in enumerate(rows)])
            self.check(o, want, f"decode layer {layer}")
            out.append((rotated, o))
        return out


@pytest.mark.parametrize("fp8", [False, True])
def test_requests_from_admission_to_compaction(gpu, fp8):
    say(f"serving flow fp8={fp8}")
    s = Server(gpu, fp8)
    s.update([0, 1, 5], [-1, -1, -1], [37, 64, 100])
    s.prompts(np.array([0, 1, 5]), [37, 64, 100])
    s.update([2, 3], [0, 1], None)                     # a fork inside a block, one at its end
    s.past[2] = [list(x) for x in s.past[0]]
    s.past[3] = [list(x) for x in s.past[1]]
    for k in range(13):                                # past the ends of blocks
        s.step(np.array([0, 1, 2, 3, 5] if k % 3 else [3, 0, 2]))
    s.update([5], [-1], [0])                           # a request leaves
    s.past[5] = [[np.zeros((0, HKV, D))] * 2 for _ in range(LAYERS)]
    ctx = s.ctx.cpu().numpy()
    s.update([2, 1], [0, 1], [ctx[0], 40])             # a beam takes another's place, one is cut back
    s.past[2] = [list(x) for x in s.past[0]]
    s.past[1] = [[y[:40] for y in x] for x in s.past[1]]
    last = s.step(np.array([0, 1, 2, 3]))
    before = s.refs.cpu().numpy().copy()
    out = {"block_table": s.table, "ref_counts": s.refs, "remap": torch.empty_like(s.refs),
           "num_live": torch.empty(1, dtype=torch.int32, device=gpu)}
    cc.compact_kv_blocks(s.table, s.refs, s.k, s.v, s.ks, s.vs, out=out)
    live = out["num_live"].item()
    assert live == (before > 0).sum() and not s.refs[live:].any()
    P.consistent(s.table.cpu().numpy(), s.ctx.cpu().numpy(), s.refs.cpu().numpy(), 16)
    for layer, (q, o) in enumerate(last):              # the same bits from the other blocks
        assert torch.equal(s.attend(layer, q, np.array([0, 1, 2, 3])), o)
    s.update([4], [-1], [50])                          # and on
    s.prompts(np.array([4]), [50])
    s.step(np.array([4, 0, 2]))


def test_decode_step_in_a_replayed_graph(gpu):
    # grow, norm + rotation + write and decode captured once, replayed over growing contexts
    say("serving graph")
    s, e = Server(gpu, False), Server(gpu, False)
    for x in (s, e):
        x.update([0, 1], [-1, -1], [15, 30])
        x.prompts(np.array([0, 1]), [15, 30])
    rows = s.tensor([0, 1])
    new, pos, slot = (torch.zeros(2, dtype=torch.int32, device=gpu) for _ in range(3))
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    qkv = torch.zeros(LAYERS, 2, (HQ + 2 * HKV) * D, dtype=torch.bfloat16, device=gpu)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=gpu)
    dws = torch.empty(max(16, cc.decode_workspace_size(2, WIDTH, HQ, HKV, D)), dtype=torch.uint8,
                      device=gpu)
    q = torch.empty(LAYERS, 2, HQ, D, dtype=torch.bfloat16, device=gpu)
    o = torch.empty_like(q)

    def step():
        pos.copy_(s.ctx[:2])
        torch.add(pos, 1, out=new)
        cc.update_block_tables(s.table, s.ctx, s.refs, rows, None, new, s.k, s.v, workspace=ws,
                               status=status)
        p = pos.long()
        slot.copy_(s.table[:2].gather(1, (p // 16)[:, None])[:, 0] * 16 + p % 16)
        for layer in range(LAYERS):
            cc.qkv_norm_rope(qkv[layer], s.qw[layer], s.kw[layer], pos, s.rope, slot, s.k[layer],
                             s.v[layer], HQ, EPS, interleaved=True, q_out=q[layer])
            cc.decode_attention(q[layer], s.k[layer].view(-1, HKV, D), s.v[layer].view(-1, HKV, D),
                                s.table[:2], s.ctx[:2], output=o[layer], workspace=dws)

    def both(run):
        p = e.ctx.cpu().numpy()[:2]
        e.update([0, 1], None, p + 1)
        fresh = e.tokens(np.array([0, 1]), p)
        qkv.copy_(torch.stack([x for x, _ in fresh]))
        run()
        assert status.item() == 0 and torch.equal(s.table, e.table) and torch.equal(s.ctx, e.ctx)
        for layer, (x, _) in enumerate(fresh):
            rotated = e.norm(layer, x, np.array([0, 1]), p)
            assert torch.equal(rotated, q[layer])
            assert torch.equal(e.attend(layer, rotated, np.array([0, 1])), o[layer])

    both(step)  # loads what a capture may not
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for _ in range(20):
        both(graph.replay)
