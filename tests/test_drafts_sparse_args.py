"""The entries on drafted trees and selected blocks on the CPU: refusals before any device is
touched, size queries, and the references of the GPU tests against themselves."""
import numpy as np
import pytest
import torch

import ccinfer_amd as cc
from ccinfer_amd import _lib
from tests import _steps_ref as R

INVALID, UNSUPPORTED = 6, 26
FAKE = 0x1000  # never dereferenced: every call fails validation first


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(fn, ok, index, values, code=INVALID):
    for v in values:
        a = list(ok)
        a[index] = v
        assert fn(*a) == code, (index, v)


def test_build_draft_tree_refusals(lib):
    f = lib.ccinfer_build_draft_tree
    ok = [FAKE] * 4 + [2, 8, 4, 33, 2, 16] + [FAKE] * 4 + [None]
    for i in [0, 1, 2, 3, 10, 11, 12, 13]:
        refused(f, ok, i, [None])
    for i in (4, 5, 6, 7, 8):
        refused(f, ok, i, [0, -1])
    refused(f, ok, 9, [8, 0, 32])
    refused(f, ok, 8, [1])                       # 33 nodes in one word
    refused(f, ok, 6, [1 << 28])
    refused(f, ok, 4, [2049], UNSUPPORTED)
    a = list(ok)
    a[7], a[8] = 2049, 65
    assert f(*a) == UNSUPPORTED
    a[7] = 64                                    # more words than the nodes need, past the most
    assert f(*a) == UNSUPPORTED


def test_tree_attention_refusals(lib):
    f = lib.ccinfer_tree_attention
    need = lib.ccinfer_tree_attention_workspace_size(2, 8, 4, 1, 16, 8, 128, 16)
    assert need > 0
    ok = [FAKE] * 3 + [None, None] + [FAKE] * 5 + [2, 8, 4, 1, 16, 8, 128, 16, FAKE, need, None]
    for i in (0, 1, 2, 5, 6, 7, 8, 9):
        refused(f, ok, i, [None])
    for i in (10, 11, 12, 13, 14, 15, 16):
        refused(f, ok, i, [0, -1])
    refused(f, ok, 14, [12])                     # no multiple of the kv heads
    refused(f, ok, 16, [100, 264, 4])
    refused(f, ok, 17, [8, 32])
    refused(f, ok, 18, [None, FAKE + 4])
    refused(f, ok, 19, [need - 1])
    refused(f, ok, 10, [1025], UNSUPPORTED)
    wide = list(ok)
    wide[14] = wide[15] = 1 << 16                # heads of a token: 2^24 bytes
    assert f(*wide) == INVALID
    for i in (0, 1, 2, 9):
        refused(f, ok, i, [FAKE + 8])
    refused(f, ok, 3, [FAKE])                    # one scale alone
    refused(f, ok, 4, [FAKE])
    refused(f, ok, 10, [2049], UNSUPPORTED)
    refused(f, ok, 13, [65], UNSUPPORTED)
    big = list(ok)
    big[11], big[12] = 1 << 20, 1 << 20          # 2^30 units of work and more
    assert f(*big) == UNSUPPORTED
    fp8 = list(ok)
    fp8[3] = fp8[4] = FAKE
    refused(f, fp8, 16, [80, 256, 32], UNSUPPORTED)
    refused(f, fp8, 3, [FAKE + 4])
    refused(f, fp8, 4, [FAKE + 4])


def test_tree_attention_workspace(lib):
    f = lib.ccinfer_tree_attention_workspace_size
    ok = [4, 100, 64, 2, 32, 8, 128, 16]
    base = f(*ok)
    for i, bad in ((0, 0), (0, 2049), (1, 0), (2, 0), (3, 0), (3, 65), (4, 31), (5, 0), (6, 4),
                   (6, 260), (7, 8)):
        a = list(ok)
        a[i] = bad
        assert f(*a) == 0, (i, bad)
    # independent of the lengths and the mask; no more for a longer table
    assert f(1, 100, 64, 1, 32, 8, 128, 16) == f(4, 100, 9000, 2, 32, 8, 128, 16) == base
    assert f(1, 1, 64, 1, 8, 8, 128, 16) < f(1, 8, 64, 1, 8, 8, 128, 16) < base
    assert f(1, 5000, 64, 1, 32, 8, 128, 16) == f(1, 9000, 64, 1, 32, 8, 128, 16)
    assert cc.tree_attention_workspace_size(4, 100, 64, 2, 32, 8, 128) == base


def test_accept_refusals(lib):
    f = lib.ccinfer_accept_draft_tokens
    ok = [FAKE] * 6 + [2, 8, 4, FAKE, FAKE, None, None, 2, 1 << 20, 0, 8, 2, 64, 16] \
        + [FAKE] * 4 + [None]
    for i in [0, 1, 2, 3, 4, 5, 9, 10, 20, 21, 22, 23]:
        refused(f, ok, i, [None])
    for i in (6, 7, 8, 13, 16, 17, 18, 19):
        refused(f, ok, i, [0, -1])
    ok = [FAKE + 64 * i if a == FAKE and i < 6 else a for i, a in enumerate(ok)]
    ok[20:24] = [FAKE + 64 * i for i in range(20, 24)]
    refused(f, ok, 14, [8 * 16 * 2 * 64 * 2 - 2])  # layers that lie inside one another
    for i in range(20, 24):
        refused(f, ok, i, ok[:6])                  # an output that is an input
    refused(f, ok, 11, [FAKE])                     # one scale alone
    refused(f, ok, 6, [2049], UNSUPPORTED)
    bare = list(ok)
    bare[9] = bare[10] = None
    assert f(*bare) == INVALID                     # no caches, but layers
    bare[13], bare[19] = 0, 0
    assert f(*bare) == INVALID


def test_bounds_scores_select_refusals(lib):
    f = lib.ccinfer_update_key_bounds
    ok = [FAKE, None, FAKE, FAKE, FAKE, None, 2, 4, 8, 128, 16, None]
    for i in (0, 2, 3, 4):
        refused(f, ok, i, [None])
    for i in (6, 7, 8, 9):
        refused(f, ok, i, [0, -1])
    refused(f, ok, 9, [100, 264])
    refused(f, ok, 10, [8, 32])
    refused(f, ok, 0, [FAKE + 8])
    refused(f, ok, 2, [FAKE + 8])
    refused(f, ok, 6, [2049], UNSUPPORTED)
    long = list(ok)
    long[6], long[7] = 2048, 1 << 20             # entries of the table: 2^31
    assert f(*long) == INVALID
    fp8 = list(ok)
    fp8[1] = FAKE
    refused(f, fp8, 0, [FAKE + 4])
    refused(f, fp8, 1, [FAKE + 2])

    f = lib.ccinfer_score_kv_blocks
    ok = [FAKE] * 5 + [2, 4, 16, 8, 128, 16, None]
    for i in range(5):
        refused(f, ok, i, [None])
    for i in (5, 6, 7, 8, 9):
        refused(f, ok, i, [0, -1])
    refused(f, ok, 7, [12])
    refused(f, ok, 9, [100, 264])
    refused(f, ok, 10, [8])
    refused(f, ok, 0, [FAKE + 2])
    refused(f, ok, 1, [FAKE + 2])

    f = lib.ccinfer_select_kv_blocks
    ok = [FAKE, FAKE, 2, 4, 8, 16, 1, 2, 16, FAKE, None]
    for i in (0, 1, 9):
        refused(f, ok, i, [None])
    for i in (2, 3, 4, 5):
        refused(f, ok, i, [0, -1])
    refused(f, ok, 6, [-1, 15])
    refused(f, ok, 7, [-1, 16, 2 ** 31 - 1])
    refused(f, ok, 5, [2])
    refused(f, ok, 8, [8])
    refused(f, ok, 3, [(1 << 16) + 1], UNSUPPORTED)


def test_sparse_decode_refusals(lib):
    f = lib.ccinfer_sparse_decode_attention
    ok = [FAKE] * 3 + [None, None] + [FAKE] * 4 + [2, 9, 16, 8, 128, 160, 16, FAKE, 1 << 30, None]
    need = lib.ccinfer_sparse_decode_workspace_size(2, 16, 8, 128, 160, 16)
    assert need > 0
    for i in (0, 1, 2, 5, 6, 7, 8):
        refused(f, ok, i, [None])
    for i in (9, 10, 11, 12, 13, 14):
        refused(f, ok, i, [0, -1])
    refused(f, ok, 11, [12])
    refused(f, ok, 13, [100, 264])
    refused(f, ok, 15, [8])
    refused(f, ok, 16, [None, FAKE + 8])
    refused(f, ok, 17, [need - 1])
    for i in (0, 1, 2, 8):
        refused(f, ok, i, [FAKE + 8])
    refused(f, ok, 3, [FAKE])
    refused(f, ok, 14, [2 ** 31 - 1])
    fp8 = list(ok)
    fp8[3] = fp8[4] = FAKE
    refused(f, fp8, 13, [80, 256], UNSUPPORTED)
    w = lib.ccinfer_sparse_decode_workspace_size
    assert w(64, 32, 8, 128, 4, 16) == 0 and w(0, 32, 8, 128, 4, 16) == 0
    assert w(2, 16, 8, 128, 0, 16) == 0 and w(2, 16, 8, 100, 160, 16) == 0


def test_python_entries_refuse_host_tensors():
    i = torch.zeros(4, dtype=torch.int32)
    q = torch.zeros(4, 8, 64, dtype=torch.bfloat16)
    table, bounds = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(2, 8, 2, 64).bfloat16()
    for call in (lambda: cc.build_draft_tree(i, i, i, table, 4),
                 lambda: cc.tree_attention(q, q, q, table, i, i, table),
                 lambda: cc.accept_draft_tokens(i, i, i, i, i, table),
                 lambda: cc.update_key_bounds(q, bounds, table, i),
                 lambda: cc.score_kv_blocks(q, bounds, table, i),
                 lambda: cc.select_kv_blocks(torch.zeros(4, 8, 2), i, 2),
                 lambda: cc.sparse_decode_attention(q, q, q, table, i, table[:, None])):
        with pytest.raises(cc.CcinferError) as e:
            call()
        assert e.value.code == INVALID


def test_references():
    """The references of the GPU tests against a tree and a row written out by hand."""
    see = R.visible([-1, 0, 0, 1])
    assert see.tolist() == [[True, False, False, False], [True, True, False, False],
                            [True, False, True, False], [True, True, False, True]]
    assert R.pack_mask(see, 2).tolist() == [[1, 0], [3, 0], [5, 0], [11, 0]]
    assert R.pack_mask(np.eye(33, dtype=bool)[31:], 2).tolist() == [[-2 ** 31, 0], [0, 1]]
    paths, counts, nodes, tokens, lengths = R.accept(
        [9, 4, 5, 6], [5, 7, 6, 8], [-1, 0, 0, 2], [0, 4], [14])
    assert paths == [[0, 2, 3]] and counts.tolist() == [3] and lengths.tolist() == [13]
    assert nodes.tolist() == [0, 2, 3, -1] and tokens.tolist() == [5, 6, 8, -1]
    sc = np.array([[[0.0, 3.0, 1.0, 3.0, 2.0, 9.0]]], np.float32)
    assert R.select(sc, [96], 4, 1, 1).tolist() == [[[0, 1, 3, 5]]]
    assert R.select(sc, [33], 4, 1, 1).tolist() == [[[0, 1, 2, -1]]]
    o, tol = R.attend(np.ones((1, 4)), np.zeros((3, 4)), np.arange(6.0).reshape(3, 2))
    assert np.allclose(o, [[2.0, 3.0]]) and (tol > 0).all()
