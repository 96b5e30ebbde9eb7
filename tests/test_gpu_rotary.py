"""Rotary table, rotation and norm + rotation + cache write on the GPU against 64 bits
(tests/_rotary_ref.py), over layouts, widths, strides and places where they can go wrong."""
import math

import numpy as np
import pytest
import torch

import ccinfer_amd as cc
from tests import _rotary_ref as R
from tests._util import from_u16, say, u16

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def f64(t):
    return t.detach().double().cpu().numpy()


def i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)


def bits(t):
    return t.contiguous().view(torch.int16).cpu().numpy()


# ---- table -----------------------------------------------------------------------------

@pytest.mark.parametrize("positions,rotary,first,scaling", [
    (1, 2, 0, None), (257, 6, 0, None), (4096, 128, 0, None), (333, 512, 5, None),
    (1000, 64, 1_000_000, None), (100, 128, 2 ** 31 - 101, None), (5000, 80, 0,
    {"type": "linear", "factor": 4.0}), (5000, 96, 77, {"type": "ntk", "factor": 8.0}),
    (9000, 128, 0, {"type": "yarn", "factor": 16.0, "original_max_position": 4096}),
    (9000, 128, 0, {"type": "bands", "factor": 8.0, "original_max_position": 8192}),
    (300, 16, 3, {"type": "factors", "factors": [1, 1.5, 2, 3, 4, 6, 8, 32], "magnitude": 1.19}),
])
def test_table(gpu, positions, rotary, first, scaling):
    say(f"table {positions} x {rotary} from {first} {scaling}")
    freq, m = cc.rope_frequencies(rotary, 5e5, scaling)
    got = f64(cc.build_rope_cache(positions, rotary, 5e5, scaling, first))
    # longdouble angles: the reference's own are exact next to the tolerance
    ang = (np.arange(positions, dtype=np.longdouble) + first)[:, None] * np.array(freq, np.longdouble)
    want = np.stack([np.cos(ang), np.sin(ang)], -1) * m
    # the angle in turns is off by 2^-52 of itself (the frequency's division and the product),
    # the quarter's rest by 2^-24 on its way to float32, the series, its selection and the
    # product with m by 3 more roundings
    bound = m * (np.abs(ang)[..., None] * 2.0 ** -51 + 6 * 2.0 ** -24)
    assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / bound)


def test_table_of_more_than_2_31_entries(gpu):
    say("table 2^31 entries")
    count, rotary = (1 << 23) + 1, 512  # 17.2 GB
    freq, _ = cc.rope_frequencies(rotary, 1e4)
    out = torch.zeros(count, rotary // 2, 2, device=gpu)
    cc.build_rope_cache(count, rotary, 1e4, out=out)
    for n in (0, 1, (1 << 22) - 1, 1 << 22, (1 << 23) - 1, 1 << 23):
        ang = np.longdouble(n) * np.array(freq, np.longdouble)
        bound = np.abs(ang) * 2.0 ** -51 + 6 * 2.0 ** -24
        got = f64(out[n])
        assert np.all(np.abs(got[:, 0] - np.cos(ang)) <= bound)
        assert np.all(np.abs(got[:, 1] - np.sin(ang)) <= bound)
    length = out.view(-1, 2)[:: 9973].double().square().sum(-1)
    assert (length - 1).abs().max().item() < 1e-5  # every entry sampled is a point of the circle


def test_table_quarter_turns(gpu):
    # frequencies of exactly 1 (pair 0): position n is n radians; signs over all quadrants
    got = f64(cc.build_rope_cache(64, 2, 1e4))
    n = np.arange(64)
    assert np.allclose(got[:, 0, 0], np.cos(n), atol=6 * 2.0 ** -24, rtol=0)
    assert np.allclose(got[:, 0, 1], np.sin(n), atol=6 * 2.0 ** -24, rtol=0)


# ---- rotation ---------------------------------------------------------------------------

def make_rotary(dev, seed, t, hq, hkv, d, rotary, max_pos=500, packed=False):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.standard_normal((t, (hq + 2 * hkv) * d)).astype(np.float32)) \
        .to(dev).to(torch.bfloat16)
    q, k = x[:, :hq * d].unflatten(1, (hq, d)), x[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    if not packed:
        q, k = q.contiguous(), k.contiguous()
    pos = rng.integers(0, max_pos, t)
    if t > 3:
        pos[1], pos[2], pos[3] = -1, max_pos, 2 ** 31 - 1  # outside the table: not rotated
    tab = R.table(max_pos, rotary)
    return q, k, pos.astype(np.int32), tab


SHAPES = [  # t, hq, hkv, d, rotary
    (1, 16, 8, 128, 128), (1, 1, 1, 2, 2), (7, 8, 2, 64, 64), (33, 4, 4, 96, 96), (5, 3, 1, 80, 32),
    (9, 5, 5, 112, 56), (6, 4, 2, 120, 120), (6, 4, 2, 192, 64), (11, 2, 1, 256, 256),
    (4, 2, 2, 130, 26), (3, 1, 1, 1024, 1024), (3, 2, 1, 512, 200), (130, 14, 2, 128, 64),
    (700, 32, 8, 128, 128), (2, 64, 8, 32, 16), (5, 7, 3, 72, 24), (4, 6, 2, 40, 20),
    (9, 2, 2, 128, 2), (5, 2, 1, 100, 50), (3000, 16, 8, 128, 96),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,hq,hkv,d,rotary", SHAPES)
def test_rotation(gpu, t, hq, hkv, d, rotary, interleaved):
    say(f"rotary {t} {hq} {hkv} {d} {rotary} {interleaved}")
    q, k, pos, tab = make_rotary(gpu, t + d, t, hq, hkv, d, rotary)
    q0, k0 = bits(q), bits(k)
    table = torch.from_numpy(tab).to(gpu)
    for inverse in (False, True):
        qo, ko = cc.rotary_embedding(q, k, i32(pos, gpu), table, interleaved, inverse)
        for got, x, what in ((qo, q, "q"), (ko, k, "k")):
            want, size = R.rotate(f64(x), pos, tab, interleaved, inverse)
            R.assert_bf16(f64(got), want, size, what)
            x, got = bits(x), bits(got)
            assert np.array_equal(got[..., rotary:], x[..., rotary:])  # copied
            if t > 3:
                assert np.array_equal(got[1:4], x[1:4])
    assert np.array_equal(bits(q), q0) and np.array_equal(bits(k), k0)


@pytest.mark.parametrize("interleaved", [False, True])
def test_views_in_place_and_other_strides(gpu, interleaved):
    say(f"rotary views {interleaved}")
    t, hq, hkv, d, rotary = 37, 8, 2, 128, 96
    q, k, pos, tab = make_rotary(gpu, 5, t, hq, hkv, d, rotary, packed=True)
    table, p = torch.from_numpy(tab).to(gpu), i32(pos, gpu)
    want = cc.rotary_embedding(q.contiguous(), k.contiguous(), p, table, interleaved)
    got = cc.rotary_embedding(q, k, p, table, interleaved)
    for a, b in zip(got, want):
        assert np.array_equal(bits(a), bits(b))
    # [heads, tokens, d] memory, both ways
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty(hq, t, d, dtype=torch.bfloat16, device=gpu).transpose(0, 1)
    got, none = cc.rotary_embedding(qt, None, p, table, interleaved, q_out=out)
    assert none is None and got is out and np.array_equal(bits(got), bits(want[0]))
    # views that start 2 and 8 bytes off a 16-byte boundary, odd row strides
    for off, row in ((1, hq * d + 3), (4, hq * d + 4), (0, hq * d + 8)):
        buf = torch.zeros(off + t * row, dtype=torch.bfloat16, device=gpu)
        view = torch.as_strided(buf, (t, hq, d), (row, d, 1), off)
        view.copy_(q)
        before = bits(buf)
        got, _ = cc.rotary_embedding(view, None, p, table, interleaved)
        assert np.array_equal(bits(got), bits(want[0])), (off, row)
        # in place; what lies between the rows stays
        got, _ = cc.rotary_embedding(view, None, p, table, interleaved, q_out=view)
        assert got is view and np.array_equal(bits(view), bits(want[0]))
        gaps = np.ones(len(before), bool)
        gaps[(off + np.arange(t)[:, None] * row + np.arange(hq * d)).ravel()] = False
        assert np.array_equal(bits(buf)[gaps], before[gaps])
    # the packed projection in place, q and k at once
    qkv = torch.zeros(t, (hq + 2 * hkv) * d, dtype=torch.bfloat16, device=gpu)
    qv, kv = qkv[:, :hq * d].unflatten(1, (hq, d)), qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    qv.copy_(q)
    kv.copy_(k)
    cc.rotary_embedding(qv, kv, p, table, interleaved, q_out=qv, k_out=kv)
    assert np.array_equal(bits(qv), bits(want[0])) and np.array_equal(bits(kv), bits(want[1]))
    assert not qkv[:, (hq + hkv) * d:].any()
    # a broadcast input: one row for every head
    one = q[:, :1].expand(t, hq, d)
    got, _ = cc.rotary_embedding(one, None, p, table, interleaved)
    assert np.array_equal(bits(got), bits(want[0])[:, :1].repeat(hq, 1))


def test_inverse_is_the_gradient(gpu):
    # sum(w * rotate(x)) has the gradient inverse(w); differences of it along single elements
    say("rotary gradient")
    t, h, d, rotary = 5, 2, 32, 24
    rng = np.random.default_rng(3)
    q, _, pos, tab = make_rotary(gpu, 9, t, h, 1, d, rotary)
    w = torch.from_numpy(rng.standard_normal((t, h, d)).astype(np.float32)).to(gpu).bfloat16()
    for inter in (False, True):
        grad, _ = cc.rotary_embedding(w, None, i32(pos, gpu), torch.from_numpy(tab).to(gpu), inter,
                                      inverse=True)
        x, wn = f64(q), f64(w)
        base = (wn * R.rotate(x, pos, tab, inter)[0]).sum()
        _, size = R.rotate(wn, pos, tab, inter, inverse=True)
        got = f64(grad)
        for _ in range(20):
            at = tuple(rng.integers(0, s) for s in x.shape)
            y = x.copy()
            y[at] += 1.0
            diff = (wn * R.rotate(y, pos, tab, inter)[0]).sum() - base
            assert abs(got[at] - diff) <= abs(diff) * R.BF16 + size[at] * R.F32 * 2 + 1e-9


def test_infinities_and_nan_stay_in_their_pairs(gpu):
    say("rotary non-finite")
    t, h, d = 4, 2, 128
    q, _, pos, tab = make_rotary(gpu, 2, t, h, 1, d, d)
    pos[:] = 7
    q[1, 0, 3], q[2, 1, 64] = math.inf, math.nan
    got = f64(cc.rotary_embedding(q, None, i32(pos, gpu), torch.from_numpy(tab).to(gpu))[0])
    want, _ = R.rotate(f64(q), pos, tab)
    assert np.array_equal(np.isfinite(got), np.isfinite(want))
    assert not np.isfinite(got[1, 0, [3, 67]]).any() and np.isnan(got[2, 1, [0, 64]]).all()


def test_rotary_refusals(gpu):
    say("rotary refusals")
    q, k, pos, tab = make_rotary(gpu, 1, 4, 4, 2, 64, 64)
    table, p = torch.from_numpy(tab).to(gpu), i32(pos, gpu)
    wide = torch.zeros(10, 33, 2, device=gpu)
    bad = [
        lambda: cc.rotary_embedding(q, k[:3], p, table),
        lambda: cc.rotary_embedding(q, k, p[:3], table),
        lambda: cc.rotary_embedding(q, k, p.long(), table),
        lambda: cc.rotary_embedding(q.float(), k, p, table),
        lambda: cc.rotary_embedding(q, k, p, wide),                      # wider than the head
        lambda: cc.rotary_embedding(q, k, p, table.double()),
        lambda: cc.rotary_embedding(q[..., ::2], None, p, table[:, :16].contiguous()),
        lambda: cc.rotary_embedding(q, k, p, table, q_out=q[:3]),
        lambda: cc.rotary_embedding(q, None, p, table, q_out=q[:, :1].expand(4, 4, 64)),
        lambda: cc.rotary_embedding(q, None, p, table, k_out=k),
        lambda: cc.rotary_embedding(q[:0], None, p[:0], table),
        lambda: cc.rotary_embedding(q[..., :63], None, p, table[:, :16].contiguous()),
        # where it reads, but on other strides
        lambda: cc.rotary_embedding(q[:, :1], None, p, table,
                                    q_out=torch.as_strided(q, (4, 1, 64), (64, 64, 1))),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(cc.CcinferError) as e:
            call()
        assert e.value.code == 6, i


# ---- norm, rotation and cache write -------------------------------------------------------

def make_norm(dev, seed, t, hq, hkv, d, rotary, fp8, per_head=False, scale=1.0, max_pos=400):
    rng = np.random.default_rng(seed)
    s = {"rng": rng, "tab": R.table(max_pos, rotary)}
    mk = lambda *n: torch.from_numpy(rng.standard_normal(n).astype(np.float32)).to(dev)  # noqa: E731
    s["qkv"] = (mk(t, (hq + 2 * hkv) * d) * scale).bfloat16()
    s["qw"] = (1 + 0.3 * (mk(hq, d) if per_head else mk(d))).bfloat16()
    s["kw"] = (1 + 0.3 * (mk(hkv, d) if per_head else mk(d))).bfloat16()
    pos = rng.integers(0, max_pos, t).astype(np.int32)
    blocks = -(-t // 16) + 2
    slot = rng.permutation(blocks * 16)[:t].astype(np.int32)
    if t > 4:
        pos[0], pos[1] = -5, max_pos
        slot[2], slot[3] = -1, blocks * 16 + 3
    s["pos"], s["slot"], s["slots"] = pos, slot, blocks * 16
    if fp8:
        c = rng.integers(0, 120, (2, s["slots"], hkv, d)).astype(np.uint8)
        s["k"], s["v"] = torch.from_numpy(c[0]).to(dev), torch.from_numpy(c[1]).to(dev)
        n = cc.fp8_scale_numel(s["slots"], hkv)
        s["ks"], s["vs"] = torch.full((n,), 3.0, device=dev), torch.full((n,), 5.0, device=dev)
    else:
        s["k"], s["v"] = mk(s["slots"], hkv, d).bfloat16(), mk(s["slots"], hkv, d).bfloat16()
        s["ks"] = s["vs"] = None
    return s


def run_norm(s, dev, hq, **kw):
    return cc.qkv_norm_rope(s["qkv"], s["qw"], s["kw"], i32(s["pos"], dev),
                            torch.from_numpy(s["tab"]).to(dev), i32(s["slot"], dev), s["k"],
                            s["v"], hq, k_scale=s["ks"], v_scale=s["vs"], **kw)


def want_norm(s, hq, hkv, d, interleaved, eps, offset):
    rows = f64(s["qkv"]).reshape(-1, hq + 2 * hkv, d)
    w = lambda x: None if x is None else f64(x)  # noqa: E731
    out = []
    for x, weight in ((rows[:, :hq], w(s["qw"])), (rows[:, hq:hq + hkv], w(s["kw"]))):
        out.append(R.rotate(R.norm(x, weight, eps, offset), s["pos"], s["tab"], interleaved))
    return out + [(rows[:, hq + hkv:], np.abs(rows[:, hq + hkv:]))]


def check_norm(s, q, hq, hkv, d, interleaved, eps, offset, before, fp8):
    (wq, sq), (wk, sk), (wv, sv) = want_norm(s, hq, hkv, d, interleaved, eps, offset)
    R.assert_bf16(f64(q), wq, sq, "q")
    ok = (s["slot"] >= 0) & (s["slot"] < s["slots"])
    at = s["slot"][ok]
    rest = np.ones(s["slots"], bool)
    rest[at] = False
    for name, scales, want, size in (("k", "ks", wk, sk), ("v", "vs", wv, sv)):
        raw = s[name].view(torch.uint8).cpu().numpy()
        assert np.array_equal(raw[rest], before[name][rest]), f"{name}: slots of no token"
        if not fp8:
            got = f64(s[name])[at]
            R.assert_bf16(got, want[ok], size[ok], name)
            if name == "v":
                assert np.array_equal(got, want[ok])
            continue
        got = s[name].view(E4M3).float().double().cpu().numpy()[at]
        sc = s[scales].cpu().numpy().astype(np.float64).reshape(-1, hkv, 16)
        R.assert_fp8(got, sc[at // 16, :, at % 16], want[ok], size[ok], name)
        left = sc.transpose(0, 2, 1).reshape(-1, hkv)[rest]
        assert np.all(left == (3.0 if name == "k" else 5.0)), f"{name}: scales of no token"


def snap(s):
    return {n: s[n].view(torch.uint8).cpu().numpy() for n in ("k", "v")}


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,hq,hkv,d,rotary", SHAPES)
def test_norm_rope(gpu, t, hq, hkv, d, rotary, interleaved, fp8):
    say(f"norm rope {t} {hq} {hkv} {d} {rotary} {interleaved} fp8={fp8}")
    s = make_norm(gpu, 3 * t + d, t, hq, hkv, d, rotary, fp8)
    before = snap(s)
    q = run_norm(s, gpu, hq, interleaved=interleaved, eps=1e-5)
    check_norm(s, q, hq, hkv, d, interleaved, 1e-5, 0.0, before, fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("which", ["per_head", "offset", "no_q", "no_k", "none"])
def test_norm_weights(gpu, which, fp8):
    say(f"norm weights {which} {fp8}")
    t, hq, hkv, d, rotary = 21, 12, 4, 128, 64
    s = make_norm(gpu, 77, t, hq, hkv, d, rotary, fp8, per_head=which == "per_head")
    offset = 1.0 if which == "offset" else 0.0
    if which in ("no_q", "none"):
        s["qw"] = None
    if which in ("no_k", "none"):
        s["kw"] = None
    before = snap(s)
    q = run_norm(s, gpu, hq, weight_offset=offset)
    check_norm(s, q, hq, hkv, d, False, 1e-6, offset, before, fp8)


def test_without_norm_k_rows_are_those_of_the_rotation(gpu):
    say("norm rope against rotary")
    t, hq, hkv, d, rotary = 50, 8, 8, 128, 96
    for inter in (False, True):
        s = make_norm(gpu, 4, t, hq, hkv, d, rotary, False)
        s["qw"] = s["kw"] = None
        q = run_norm(s, gpu, hq, interleaved=inter)
        rows = s["qkv"].view(t, hq + 2 * hkv, d)
        qo, ko = cc.rotary_embedding(rows[:, :hq], rows[:, hq:hq + hkv], i32(s["pos"], gpu),
                                     torch.from_numpy(s["tab"]).to(gpu), inter)
        assert np.array_equal(bits(q), bits(qo))
        ok = (s["slot"] >= 0) & (s["slot"] < s["slots"])
        assert np.array_equal(bits(s["k"])[s["slot"][ok]], bits(ko)[ok])


@pytest.mark.parametrize("fp8", [False, True])
def test_row_strides_small_and_large_values(gpu, fp8):
    say(f"norm rope strides {fp8}")
    t, hq, hkv, d, rotary = 19, 4, 2, 64, 64
    for scale in (1e-12, 1.0, 1e12):
        s = make_norm(gpu, 8, t, hq, hkv, d, rotary, fp8, scale=scale)
        s["qkv"][5] = 0  # a row of zeros stays one
        before = snap(s)
        q = run_norm(s, gpu, hq, eps=1e-30)
        check_norm(s, q, hq, hkv, d, False, float(np.float32(1e-30)), 0.0, before, fp8)
        want_k, want_v = snap(s)["k"], snap(s)["v"]
        for off, row in ((0, 600), (1, 513), (4, 516)):
            width = s["qkv"].shape[1]
            buf = torch.zeros(off + t * row, dtype=torch.bfloat16, device=gpu)
            view = torch.as_strided(buf, (t, width), (row, 1), off)
            view.copy_(s["qkv"])
            s2 = dict(s, qkv=view, k=s["k"].clone(), v=s["v"].clone())
            q2 = run_norm(s2, gpu, hq, eps=1e-30)
            # other lanes add the squares up: last places may differ, nothing else
            check_norm(s2, q2, hq, hkv, d, False, float(np.float32(1e-30)), 0.0,
                       {"k": want_k, "v": want_v}, fp8)


def test_nan_and_infinity_reach_the_caches(gpu):
    say("norm rope non-finite")
    t, hq, hkv, d = 6, 2, 1, 128
    for fp8 in (False, True):
        s = make_norm(gpu, 6, t, hq, hkv, d, d, fp8)
        s["slot"] = np.arange(t, dtype=np.int32)
        rows = s["qkv"].view(t, hq + 2 * hkv, d)
        rows[1, hq, 5] = math.nan        # k: its whole row (the norm)
        rows[2, hq + 1, 9] = math.nan    # v: the element
        rows[3, hq + 1, 4] = math.inf
        q = run_norm(s, gpu, hq)
        assert torch.isfinite(q).all()
        val = [s[n].view(E4M3).float() if fp8 else s[n].float() for n in ("k", "v")]
        k, v = (x.cpu().numpy()[:, 0] for x in val)
        assert np.isnan(k[1]).all() and np.isfinite(np.delete(k, 1, 0)[:5]).all()
        assert np.isnan(v[2, 9]) and np.isfinite(np.delete(v[2], 9)).all()
        if fp8:
            assert v[3, 4] == 448.0 and f64(s["vs"])[3] == 2.0 ** 126
            assert not np.delete(v[3], 4).any()
        else:
            assert np.isinf(v[3, 4]) and np.isfinite(np.delete(v[3], 4)).all()


def test_norm_rope_refusals(gpu):
    say("norm rope refusals")
    t, hq, hkv, d = 4, 4, 2, 64
    s = make_norm(gpu, 1, t, hq, hkv, d, d, False)
    f = make_norm(gpu, 1, t, hq, hkv, d, d, True)
    tab = torch.from_numpy(s["tab"]).to(gpu)
    p, m = i32(s["pos"], gpu), i32(s["slot"], gpu)

    def call(qkv=s["qkv"], qw=s["qw"], kw=s["kw"], pos=p, table=tab, slot=m, k=s["k"], v=s["v"],
             heads=hq, **kw_):
        return cc.qkv_norm_rope(qkv, qw, kw, pos, table, slot, k, v, heads, **kw_)
    bad = [dict(heads=3), dict(heads=0), dict(pos=p[:3]), dict(slot=m[:3]), dict(qw=s["qw"][:32]),
           dict(kw=s["kw"].expand(3, d).contiguous()), dict(eps=0.0), dict(eps=math.nan),
           dict(weight_offset=math.inf), dict(k_scale=f["ks"]),
           dict(k=f["k"], v=f["v"]), dict(k=f["k"], v=f["v"], k_scale=f["ks"], v_scale=f["vs"][:9]),
           dict(k_scale=f["ks"], v_scale=f["vs"]), dict(max_slots=0),
           dict(max_slots=s["slots"] + 1), dict(qkv=s["qkv"].float()),
           dict(qkv=s["qkv"][:, :-2]), dict(v=s["v"][:16]), dict(q_out=s["qkv"])]
    for i, kw in enumerate(bad):
        with pytest.raises(cc.CcinferError) as e:
            call(**kw)
        assert e.value.code == 6, (i, kw.keys())


def test_skipped_slots_only_and_fewer_slots(gpu):
    say("norm rope skipped")
    t, hq, hkv, d = 9, 4, 2, 128
    s = make_norm(gpu, 12, t, hq, hkv, d, d, False)
    s["slot"] = np.full(t, -1, np.int32)
    before = snap(s)
    q = run_norm(s, gpu, hq)
    check_norm(s, q, hq, hkv, d, False, 1e-6, 0.0, before, False)
    s["slot"] = np.arange(t, dtype=np.int32)
    run_norm(s, gpu, hq, max_slots=5)  # slots 5 .. 8 keep what they held
    after = snap(s)
    assert np.array_equal(after["k"][5:], before["k"][5:])
    assert not np.array_equal(after["k"][:5], before["k"][:5])


# ---- streams and graphs ------------------------------------------------------------------

def test_on_a_side_stream_and_in_a_replayed_graph(gpu):
    say("rotary graph")
    t, hq, hkv, d, rotary = 12, 8, 2, 128, 128
    s = make_norm(gpu, 31, t, hq, hkv, d, rotary, True)
    table = torch.empty(400, rotary // 2, 2, device=gpu)
    pos, slot = i32(np.abs(s["pos"]) % 400, gpu), i32(s["slot"], gpu)
    q_in = s["qkv"].view(t, -1, d)[:, :hq]
    out = [torch.empty(t, hq, d, dtype=torch.bfloat16, device=gpu) for _ in range(2)]

    def step():
        cc.build_rope_cache(400, rotary, 1e4, out=table)
        cc.rotary_embedding(q_in, None, pos, table, q_out=out[0])
        cc.qkv_norm_rope(s["qkv"], s["qw"], s["kw"], pos, table, slot, s["k"], s["v"], hq,
                         k_scale=s["ks"], v_scale=s["vs"], q_out=out[1])

    def results():
        torch.cuda.synchronize()
        return [x.clone() for x in (*out, s["k"], s["v"], s["ks"], s["vs"])]

    step()
    want = results()
    side = torch.cuda.Stream()
    for x in (*out, s["k"], s["v"]):
        x.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    skip = [n for n in range(s["slots"]) if n not in set(s["slot"].tolist())]
    keep = torch.tensor([n for n in range(s["slots"]) if n not in skip], device=gpu)

    def same(got):
        for a, b in zip(got[:2], want[:2]):
            assert torch.equal(a, b)
        for a, b in zip(got[2:4], want[2:4]):
            assert torch.equal(a[keep], b[keep])
        for a, b in zip(got[4:], want[4:]):
            assert torch.equal(a, b)
    same(results())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(4):
        s["qkv"].mul_(1.0 if k < 2 else 2.0)  # other inputs between the replays
        step()
        want = results()
        for x in (*out, s["k"], s["v"]):
            x.zero_()
        table.fill_(7.0)
        graph.replay()
        same(results())


# ---- every width -------------------------------------------------------------------------

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,widths", [(16, range(2, 18, 2)), (18, range(2, 20, 2)),
                                      (128, (2, 14, 16, 18, 110, 112, 118, 120, 122, 124, 126)),
                                      (64, (6, 12, 34, 48, 50, 56, 58, 62)), (14, (2, 8, 14)),
                                      (1024, (1002, 1000, 16, 1022)), (1008, (990,))])
def test_every_width(gpu, d, widths, interleaved):
    # parts of a head shorter than a segment of eight, and parts that end inside one; in place
    # and beside, with the norm into both kinds of cache
    t, hq, hkv = 9, 3, 2
    for rotary in widths:
        say(f"width {d} {rotary} {interleaved}")
        q, k, pos, tab = make_rotary(gpu, d + rotary, t, hq, hkv, d, rotary)
        q[5], k[6] = math.inf, math.nan  # stay in their rows
        q[7, 1, rotary - 1] = math.inf   # stays in its pair
        table = torch.from_numpy(tab).to(gpu)
        with np.errstate(invalid="ignore"):
            wq, sq = R.rotate(f64(q), pos, tab, interleaved)
        qo, ko = cc.rotary_embedding(q, k, i32(pos, gpu), table, interleaved)
        for row in range(t):
            if row not in (5, 7):
                R.assert_bf16(f64(qo)[row], wq[row], sq[row], f"q row {row}")
        assert np.array_equal(np.isfinite(f64(qo)[7]), np.isfinite(wq[7]))
        assert np.array_equal(bits(qo)[..., rotary:], bits(q)[..., rotary:])
        cc.rotary_embedding(q, k, i32(pos, gpu), table, interleaved, q_out=q, k_out=k)
        assert np.array_equal(bits(q), bits(qo)) and np.array_equal(bits(k), bits(ko))
        for fp8 in (False, True):
            s = make_norm(gpu, d + rotary, t, hq, hkv, d, rotary, fp8)
            before = snap(s)
            q2 = run_norm(s, gpu, hq, interleaved=interleaved)
            check_norm(s, q2, hq, hkv, d, interleaved, 1e-6, 0.0, before, fp8)


def test_tensors_of_another_device_are_refused(gpu, monkeypatch):
    say("other device")
    from ccinfer_amd import pages, rope
    s = make_norm(gpu, 3, 4, 4, 2, 64, 64, False)
    table, pos = torch.from_numpy(s["tab"]).to(gpu), i32(s["pos"], gpu)
    k = s["k"].view(-1, 16, 2, 64)
    counts = torch.zeros(len(k), dtype=torch.int32, device=gpu)
    rows = torch.full((2, 3), -1, dtype=torch.int32, device=gpu)
    calls = [lambda: cc.build_rope_cache(len(table), 64, out=table),
             lambda: cc.rotary_embedding(k[0, :4], None, pos, table),
             lambda: run_norm(s, gpu, 4),
             lambda: cc.copy_kv_blocks(k, k, counts[:1], counts[:1]),
             lambda: cc.update_block_tables(rows, counts[:2], counts, counts[:0], None, None),
             lambda: cc.compact_kv_blocks(rows, counts, k, k)]
    for call in calls:
        call()
    for module in (rope, pages):
        monkeypatch.setattr(module, "current_device", lambda: 1)
    for i, call in enumerate(calls):
        with pytest.raises(cc.CcinferError) as e:
            call()
        assert e.value.code == 6, i


def test_copied_elements_keep_their_bits(gpu):
    # every bf16 but the NaNs, subnormal ones among them: past the rotated part, in rows at
    # positions outside the table, and in v rows
    say("copied bits")
    h, d = 4, 128
    every = np.arange(1 << 16, dtype=np.uint16)
    every = every[(every & 0x7fff) <= 0x7f80]
    t = -(-len(every) // (h * d))
    x = np.resize(every, (t, h, d))
    for rotary in (64, 100):
        tab = torch.from_numpy(R.table(8, rotary)).to(gpu)
        for inter in (False, True):
            q = from_u16(x, gpu)
            out, _ = cc.rotary_embedding(q, None, i32(np.arange(t) % 8, gpu), tab, inter)
            assert np.array_equal(u16(out)[..., rotary:], x[..., rotary:])
            out, _ = cc.rotary_embedding(q, None, i32(np.full(t, -1), gpu), tab, inter)
            assert np.array_equal(u16(out), x)
            qkv = from_u16(np.tile(x.reshape(t, h * d), (1, 3)), gpu)
            k, v = (torch.zeros(t, h, d, dtype=torch.bfloat16, device=gpu) for _ in "kv")
            out = cc.qkv_norm_rope(qkv, None, None, i32(np.full(t, -1), gpu), tab,
                                   i32(np.arange(t), gpu), k, v, h, interleaved=inter)
            for got in (out, k, v):
                assert np.array_equal(u16(got), x)


def test_smallest_eps_and_rows_of_zeros(gpu):
    say("smallest eps")
    t, hq, hkv, d = 7, 4, 2, 128
    for fp8 in (False, True):
        s = make_norm(gpu, 14, t, hq, hkv, d, d, fp8)
        s["qkv"][4:6] = 0
        s["qkv"][6] *= 2.0 ** -70  # squares under the smallest normal number
        eps = float(np.float32(2.0 ** -126))
        q = run_norm(s, gpu, hq, eps=eps)
        assert not q[4:6].any()
        s["qkv"][6] = 0  # (float32 squares of the row are no measure for it)
        assert torch.isfinite(q).all()
        (wq, sq), _, _ = want_norm(s, hq, hkv, d, False, eps, 0.0)
        R.assert_bf16(f64(q)[:6], wq[:6], sq[:6], "q")


def test_caches_of_more_than_31_bits_of_slots_are_refused(gpu):
    # 2^32 + 16 slots, which a 32-bit argument would take for 16
    say("slots past 31 bits")
    far = torch.zeros(2 ** 32 + 16, 1, 2, dtype=torch.bfloat16, device=gpu)
    qkv = torch.ones(1, 6, dtype=torch.bfloat16, device=gpu)
    table = torch.from_numpy(R.table(4, 2)).to(gpu)
    pos, slot = i32([-1], gpu), i32([20], gpu)
    for most in (None, 2 ** 32 + 16):
        with pytest.raises(cc.CcinferError) as e:
            cc.qkv_norm_rope(qkv, None, None, pos, table, slot, far, far, 1, max_slots=most)
        assert e.value.code == 6
    cc.qkv_norm_rope(qkv, None, None, pos, table, slot, far, far, 1, max_slots=2 ** 31 - 1)
    assert (far[20] == 1).all()


def test_rows_and_tables_of_more_than_31_bits_are_refused(gpu):
    # lengths that a 32-bit argument would take for 1 head, 64 elements or 5 positions
    say("rows past 31 bits")
    few = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=gpu)
    heads = torch.zeros(1, 2 ** 32 + 1, 2, dtype=torch.bfloat16, device=gpu)
    table, pos = torch.from_numpy(R.table(8, 64)).to(gpu), i32([6], gpu)
    narrow = torch.from_numpy(R.table(8, 2)).to(gpu)
    out = torch.empty_like(heads)
    long = torch.zeros(1, 1, 2 ** 32 + 64, dtype=torch.bfloat16, device=gpu)
    far = torch.zeros(2 ** 32 + 5, 1, 2, device=gpu)
    for i, call in enumerate([
            lambda: cc.rotary_embedding(heads, None, pos, narrow, q_out=out),
            lambda: cc.rotary_embedding(heads[:, :1], heads, pos, narrow, k_out=out),
            lambda: cc.rotary_embedding(long, None, pos, table, q_out=out.view(-1)[:2 ** 32 + 64]
                                        .view(1, 1, -1)),
            lambda: cc.rotary_embedding(few, None, pos, far),
            lambda: cc.rotary_embedding(few, None, pos, far[:2 ** 32 + 4].view(2, -1, 2))]):
        with pytest.raises(cc.CcinferError) as e:
            call()
        assert e.value.code == 6, i


def test_rows_whose_squares_are_under_the_smallest_normal_number(gpu):
    # Elements near 2^-70 beside an eps of 2^-126: float32 squares near 2^-140, which may be lost.
    # Then 1 / sqrt(mean + eps) is too large by a share of mean / (2 eps), 2^-15 here.
    say("tiny rows")
    t, hq, hkv, d = 7, 4, 2, 128
    eps = float(np.float32(2.0 ** -126))
    for rotary in (d, 96, 100):
        s = make_norm(gpu, 15, t, hq, hkv, d, rotary, False)
        s["qkv"] *= 2.0 ** -70
        q = run_norm(s, gpu, hq, eps=eps)
        at = np.flatnonzero((s["slot"] >= 0) & (s["slot"] < s["slots"]))
        x = f64(s["qkv"]).reshape(t, hq + 2 * hkv, d)
        lost = (x ** 2).mean(-1, keepdims=True) / (2 * eps)
        assert lost.max() < 2.0 ** -14
        (wq, sq), (wk, sk), _ = want_norm(s, hq, hkv, d, False, eps, 0.0)
        for got, want, size, share, rows in (
                (f64(q), wq, sq, lost[:, :hq], np.arange(t)),
                (f64(s["k"])[s["slot"][at]], wk[at], sk[at], lost[at, hq:hq + hkv], at)):
            bound = np.abs(want) * R.BF16 + size * (R.F32 + share) * (1 + R.BF16) + 1e-38
            assert np.all(np.abs(got - want) <= bound), rotary
            assert np.abs(got).max(-1).min() > 2.0 ** -9  # (an answer of zeros is none)


def test_rows_whose_sum_of_squares_passes_float32(gpu):
    # stated: such a row comes out as zeros, its neighbours as they should
    say("huge rows")
    t, hq, hkv, d = 6, 2, 1, 64
    s = make_norm(gpu, 16, t, hq, hkv, d, d, False)
    s["qkv"][4] = (s["qkv"][4].float().abs() + 1).bfloat16() * 2.0 ** 64
    q = run_norm(s, gpu, hq)
    assert not q[4].any() and not s["k"][int(s["slot"][4])].any()
    (wq, sq), _, _ = want_norm(s, hq, hkv, d, False, 1e-6, 0.0)
    rest = [0, 1, 2, 3, 5]
    R.assert_bf16(f64(q)[rest], wq[rest], sq[rest], "q")
