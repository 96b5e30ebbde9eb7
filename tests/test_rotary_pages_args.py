"""The rotary and page entries on the CPU: refusals before any device is touched, frequencies of
the scalings against their formulas, and the references of the GPU tests against themselves."""
import ctypes
import math

import numpy as np
import pytest
import torch

import ccinfer_amd as cc
from ccinfer_amd import _lib
from tests import _pages_ref as P
from tests import _rotary_ref as R

INVALID, UNSUPPORTED = 6, 26
FAKE = 0x1000  # never dereferenced: every call fails validation first
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


# ---- frequencies ---------------------------------------------------------------------

def close(got, want):
    assert np.allclose(got, want, rtol=1e-14, atol=0)


def test_plain_linear_ntk_and_factors():
    r, theta = 96, 1e6
    f = theta ** (-np.arange(0, r, 2) / r)
    got, m = cc.rope_frequencies(r, theta)
    close(got, f)
    assert m == 1.0
    close(cc.rope_frequencies(r, theta, {"type": "linear", "factor": 3.5})[0], f / 3.5)
    got, m = cc.rope_frequencies(r, theta, {"type": "ntk", "factor": 8.0})
    close(got, (theta * 8 ** (r / (r - 2))) ** (-np.arange(0, r, 2) / r))
    close(got[-1], f[-1] / 8)          # the slowest pair is stretched by the factor,
    assert got[0] == 1.0 and m == 1.0  # the fastest by nothing
    own = np.linspace(1, 30, r // 2)
    got, m = cc.rope_frequencies(r, theta, {"type": "factors", "factors": list(own),
                                            "magnitude": 1.25})
    close(got, f / own)
    assert m == 1.25


@pytest.mark.parametrize("kind", [{"type": "none"}, {"type": "linear", "factor": 2.0},
                                  {"type": "ntk", "factor": 2.0},
                                  {"type": "yarn", "factor": 2.0, "original_max_position": 4096},
                                  {"type": "bands", "factor": 2.0, "original_max_position": 4096},
                                  {"type": "factors", "factors": [1.5] * 16}])
def test_a_magnitude_is_taken_with_every_scaling(kind):
    f, own = cc.rope_frequencies(32, 1e4, kind)
    got, m = cc.rope_frequencies(32, 1e4, {**kind, "magnitude": 1.25})
    assert got == f and m == 1.25
    assert cc.rope_frequencies(32, 1e4, {**kind, "magnitude": 0.0}) == (f, own)
    for bad in (-1.0, NAN, INF):
        with pytest.raises(cc.CcinferError):
            cc.rope_frequencies(32, 1e4, {**kind, "magnitude": bad})


def test_yarn_and_bands():
    r, theta, n, s = 128, 1e4, 4096, 16.0
    f = theta ** (-np.arange(0, r, 2) / r)
    turns = n * f / (2 * math.pi)
    got, m = cc.rope_frequencies(r, theta, {"type": "yarn", "factor": s,
                                            "original_max_position": n})
    got = np.array(got)
    assert m == 0.1 * math.log(s) + 1
    close(got[turns > 40], f[turns > 40])
    close(got[turns < 0.8], f[turns < 0.8] / s)
    # two libraries' powers, an ulp (2^-52) each at most, and the blend's three roundings
    assert np.all(np.diff(got) < 0)
    assert np.all(got <= f * (1 + 1e-14)) and np.all(got >= f / s * (1 - 1e-14))
    got, m = cc.rope_frequencies(r, theta, {"type": "bands", "factor": s,
                                            "original_max_position": n})
    mix = np.clip((turns - 1) / 3, 0, 1)
    close(got, f / s * (1 - mix) + f * mix)
    assert m == 1.0


@pytest.mark.parametrize("bad", [
    dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=514), dict(theta=1.0),
    dict(theta=NAN), dict(theta=INF), dict(theta=-5.0),
    dict(scaling={"type": "other"}), dict(scaling={"factor": 2.0}),
    dict(scaling={"type": "linear", "factor": 0.5}),
    dict(scaling={"type": "linear", "factor": NAN}),
    dict(scaling={"type": "linear", "factr": 2.0}),
    dict(rotary_dim=2, scaling={"type": "ntk", "factor": 2.0}),
    dict(scaling={"type": "yarn", "factor": 2.0}),
    dict(scaling={"type": "bands", "factor": 2.0, "original_max_position": 99, "fast": 1.0}),
    dict(scaling={"type": "bands", "factor": 2.0, "original_max_position": 99, "slow": 0.0}),
    dict(scaling={"type": "linear", "factor": 2.0, "magnitude": -1.0}),
    dict(scaling={"type": "factors", "factors": [1.0] * 3}),
    dict(scaling={"type": "factors", "factors": [1.0] * 63 + [0.0]}),
])
def test_frequency_refusals(bad):
    args = {"rotary_dim": 128, "theta": 1e4, "scaling": None, **bad}
    with pytest.raises(cc.CcinferError) as e:
        cc.rope_frequencies(**args)
    assert e.value.code == INVALID


def test_rope_cache_refusals(lib):
    f = (ctypes.c_double * 64)(*([0.5] * 64))
    ok = [f, 128, 1.0, 0, 16, FAKE, None]
    for i, bad in [(0, None), (1, 0), (1, 7), (1, 514), (2, NAN), (2, INF), (2, 1e300), (3, -1),
                   (4, 0), (4, -1), (5, None), (5, FAKE + 4)]:
        a = list(ok)
        a[i] = bad
        assert lib.ccinfer_build_rope_cache(*a) == INVALID, (i, bad)
    a = list(ok)
    a[3] = 2 ** 31 - 2  # positions past 2^31
    assert lib.ccinfer_build_rope_cache(*a) == INVALID
    f[5] = 65537.0
    assert lib.ccinfer_build_rope_cache(*ok) == INVALID
    f[5] = INF
    assert lib.ccinfer_build_rope_cache(*ok) == INVALID


# ---- rotary and norm -------------------------------------------------------------------

def test_rotary_refusals(lib):
    fn = lib.ccinfer_rotary_embedding
    ok = [FAKE, 1024, 128, FAKE, 256, 128, FAKE, FAKE, FAKE, 1024, 128, FAKE, 256, 128,
          4, 8, 2, 128, 128, 64, 0, 0, None]
    for i, bad in [(0, None), (3, None), (6, None), (7, None), (7, FAKE + 4), (8, None),
                   (11, None), (14, 0), (15, 0), (16, -1), (16, 0), (17, 0), (17, 127),
                   (17, 1026), (18, 0), (18, 63), (18, 130), (19, 0)]:
        a = list(ok)
        a[i] = bad
        assert fn(*a) == INVALID, (i, bad)
    a = list(ok)
    a[14], a[15] = 2 ** 30, 8  # rows past 2^31
    assert fn(*a) == INVALID


def test_norm_rope_refusals(lib):
    fn = lib.ccinfer_qkv_norm_rope
    ok = [FAKE, 1536, FAKE, 0, FAKE, 0, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, None,
          4, 8, 2, 128, 128, 64, 256, 0, 1e-6, 0.0, None]
    for i, bad in [(0, None), (1, 1535), (6, None), (7, None), (7, FAKE + 4), (8, None), (9, None),
                   (10, None), (11, None), (12, FAKE), (13, FAKE), (14, 0), (15, 0), (16, 0),
                   (17, 0), (17, 127), (17, 1026), (18, 0), (18, 3), (18, 130), (19, 0), (20, 0),
                   (22, 0.0), (22, -1.0), (22, 1e-39), (22, NAN), (22, INF), (23, NAN), (23, INF)]:
        a = list(ok)
        a[i] = bad
        assert fn(*a) == INVALID, (i, bad)


# ---- pages ------------------------------------------------------------------------------

def test_copy_refusals(lib):
    fn = lib.ccinfer_copy_kv_blocks
    layer = 64 * 16 * 8 * 128 * 2
    ok = [FAKE, FAKE, None, None, FAKE, FAKE, 4, 3, layer, 0, 64, 8, 128, 16, None, None]
    for i, bad in [(0, None), (1, None), (2, FAKE), (3, FAKE), (4, None), (5, None), (6, -1),
                   (7, 0), (7, 40000), (8, layer - 2), (8, layer + 1), (10, 0), (11, 0), (12, 0),
                   (13, 0)]:
        a = list(ok)
        a[i] = bad
        assert fn(*a) == INVALID, (i, bad)
    a = list(ok)
    a[6] = (1 << 17) + 1
    assert fn(*a) == UNSUPPORTED
    a = list(ok)
    a[7], a[10], a[11], a[12], a[13] = 1, 1, 4096, 256, 1024  # a block past 2^30 bytes
    assert fn(*a) == INVALID
    fp8 = [FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 4, 3, layer // 2, 64 * 8 * 16, 64, 8, 128, 16, None,
           None]
    for i, bad in [(9, 64 * 8 * 16 - 1), (13, 32), (8, layer // 2 - 1)]:
        a = list(fp8)
        a[i] = bad
        assert fn(*a) == INVALID, (i, bad)
    a = list(ok)
    a[6], a[4], a[5] = 0, None, None  # nothing to copy
    assert fn(*a) == 0


def test_update_refusals(lib):
    fn = lib.ccinfer_update_block_tables
    layer = 64 * 16 * 8 * 128 * 2
    need = lib.ccinfer_update_tables_workspace_size(4, 32, 64)
    assert need > 0
    ok = [FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 4, 8, 32, FAKE, FAKE, None, None, 3, layer, 0, 64, 8,
          128, 16, None, None, FAKE, FAKE, need, None]
    for i, bad in [(0, None), (1, None), (2, None), (3, None), (6, -1), (7, 0), (8, 0), (9, None),
                   (10, None), (11, FAKE), (12, FAKE), (13, 0), (14, layer - 2), (16, 0), (17, 0),
                   (18, 0), (19, 0), (20, FAKE), (21, FAKE), (22, None), (23, None),
                   (23, FAKE + 8), (24, need - 1)]:
        a = list(ok)
        a[i] = bad
        assert fn(*a) == INVALID, (i, bad)
    a = list(ok)
    a[9:16] = [None, None, None, None, 0, 0, 0]
    a[16] = (1 << 24) + 1  # blocks past the bitmap
    a[24] = 1 << 40
    assert fn(*a) == UNSUPPORTED
    a = list(ok)
    a[6], a[24] = (1 << 14) + 1, 1 << 40
    assert fn(*a) == UNSUPPORTED
    assert lib.ccinfer_update_tables_workspace_size(4, 32, (1 << 24) + 1) == 0
    assert lib.ccinfer_update_tables_workspace_size((1 << 14) + 1, 32, 64) == 0
    for bad in [(-1, 32, 64), (4, 0, 64), (4, 32, 0), (1 << 19, 1 << 13, 64)]:
        assert lib.ccinfer_update_tables_workspace_size(*bad) == 0, bad


def test_compact_refusals(lib):
    fn = lib.ccinfer_compact_kv_blocks
    layer = 64 * 16 * 8 * 128 * 2
    need = lib.ccinfer_compact_workspace_size(64)
    ok = [FAKE, FAKE, 8, 32, FAKE, FAKE, None, None, 3, layer, 0, 64, 8, 128, 16, FAKE, FAKE, FAKE,
          FAKE, FAKE, need, None]
    for i, bad in [(0, None), (1, None), (2, -1), (3, 0), (4, None), (5, None), (6, FAKE),
                   (8, 0), (9, layer - 2), (11, 0), (12, 0), (13, 0), (14, 0), (15, None),
                   (16, None), (17, None), (18, None), (19, None), (19, FAKE + 8),
                   (20, need - 1)]:
        a = list(ok)
        a[i] = bad
        assert fn(*a) == INVALID, (i, bad)
    assert lib.ccinfer_compact_workspace_size(0) == 0
    assert lib.ccinfer_compact_workspace_size((1 << 24) + 1) == 0


def test_python_entries_refuse_host_tensors():
    bf = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    i32 = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(4, 32, 2)
    calls = [lambda: cc.rotary_embedding(bf, None, i32, table),
             lambda: cc.build_rope_cache(4, 64, out=table),
             lambda: cc.qkv_norm_rope(bf.view(2, 256), None, None, i32, table, i32, bf, bf, 2)]
    for call in calls:
        with pytest.raises(cc.CcinferError) as e:
            call()
        assert e.value.code == INVALID


# ---- the references -----------------------------------------------------------------------

def test_reference_rotation_turns_back_and_is_its_own_gradient():
    rng = np.random.default_rng(1)
    tab = R.table(50, 24).astype(np.float64)
    pos = np.array([3, 49, 0, 17])
    for inter in (False, True):
        x, w = rng.standard_normal((4, 2, 32)), rng.standard_normal((4, 2, 32))
        y, _ = R.rotate(x, pos, tab, inter)
        back, _ = R.rotate(y, pos, tab, inter, inverse=True)
        assert np.allclose(back, x, atol=1e-6)  # a float32 table: cos^2 + sin^2 is 1 +- 2^-23
        grad, _ = R.rotate(w, pos, tab, inter, inverse=True)
        for _ in range(10):  # differences of the linear map sum(w * rotate(x))
            at = tuple(rng.integers(0, s) for s in x.shape)
            dx = np.zeros_like(x)
            dx[at] = 1.0
            diff = (w * (R.rotate(x + dx, pos, tab, inter)[0] - y)).sum()
            assert abs(diff - grad[at]) < 1e-9


def test_reference_update_keeps_counts():
    rng = np.random.default_rng(2)
    bs, rows, width, blocks = 4, 6, 8, 40
    table, ctx = np.full((rows, width), -1), np.zeros(rows, int)
    refs = np.zeros(blocks, int)
    caches = [rng.integers(0, 99, (2, blocks, bs, 3))]
    for _ in range(60):
        n = rng.integers(1, rows + 1)
        dst = rng.permutation(rows)[:n]
        src = rng.integers(-1, rows, n)
        lengths = rng.integers(-1, width * bs // 2, n)
        table, ctx, refs, caches, _, status = P.update(table, ctx, refs, dst, src, lengths, caches,
                                                       [], bs)
        assert status in (0, 12)
        P.consistent(table, ctx, refs, bs)
