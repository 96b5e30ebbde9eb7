"""Workspaces that a caller hands in: refused where their elements do not lie one after the other
(an expanded view has less memory than they say), or on another device than the call's tensors."""
import pytest
import torch

import ccinfer_amd as cc
from ccinfer_amd import ops
from tests._util import say

pytestmark = pytest.mark.gpu


def views(dev):
    """Views of 2^26 bytes by their elements."""
    few = torch.zeros(4096, dtype=torch.uint8, device=dev)
    return {"expanded": few[:1].expand(1 << 26), "rows again": few.expand(1 << 14, 4096),
            "every other": torch.zeros(1 << 27, dtype=torch.uint8, device=dev)[::2]}


def calls(dev):
    i32 = dict(dtype=torch.int32, device=dev)
    bf = dict(dtype=torch.bfloat16, device=dev)
    b, hq, hkv, d, blocks, width = 3, 4, 2, 64, 16, 4
    q = torch.ones(b, hq, d, **bf)
    k = torch.ones(blocks * 16, hkv, d, **bf)
    new = torch.ones(b, hkv, d, **bf)
    codes = torch.zeros(blocks * 16, hkv, d, dtype=torch.uint8, device=dev)
    scale = torch.zeros(cc.fp8_scale_numel(blocks * 16, hkv), device=dev)
    rows = torch.arange(b * width, **i32).view(b, width)
    ctx = torch.full((b,), 17, **i32)
    start = torch.arange(b + 1, **i32)
    refs = torch.ones(blocks, **i32)
    none = torch.zeros(0, **i32)
    return {
        "decode": lambda ws: cc.decode_attention(q, k, k, rows, ctx, workspace=ws),
        "decode shared": lambda ws: cc.decode_attention_shared_prefix(q, k, k, rows, ctx,
                                                                      workspace=ws),
        "decode write": lambda ws: cc.decode_attention_write_kv(q, new, new, k, k, rows, ctx,
                                                                workspace=ws),
        "decode fp8": lambda ws: cc.decode_attention_fp8(q, codes, codes, scale, scale, rows, ctx,
                                                         workspace=ws),
        "prefill": lambda ws: cc.prefill_attention(q, k, k, rows, start, ctx, workspace=ws),
        "prefill fp8": lambda ws: cc.prefill_attention_fp8(q, codes, codes, scale, scale, rows,
                                                           start, ctx, workspace=ws),
        "update": lambda ws: cc.update_block_tables(rows, ctx, refs, none, None, None,
                                                    workspace=ws),
        "compact": lambda ws: cc.compact_kv_blocks(rows, refs, k, k, workspace=ws)}


NAMES = ("decode", "decode shared", "decode write", "decode fp8", "prefill", "prefill fp8",
         "update", "compact")


@pytest.mark.parametrize("name", NAMES)
def test_workspace_that_is_no_run_of_memory_is_refused(gpu, name):
    say(f"workspace {name}")
    call = calls(gpu)[name]
    call(None)
    call(torch.empty(1 << 26, dtype=torch.uint8, device=gpu))
    call(torch.empty(1 << 24, 4, dtype=torch.uint8, device=gpu)[:1 << 23])
    for kind, ws in views(gpu).items():
        with pytest.raises(cc.CcinferError) as e:
            call(ws)
        assert e.value.code == 6, kind


def test_workspace_of_another_device_is_refused(gpu):
    say("workspace device")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=gpu)
    for take in (ops._workspace, ops._prefill_workspace):
        assert take(64, gpu, ws)[0] is ws
        with pytest.raises(cc.CcinferError) as e:
            take(64, torch.device("cuda", 1), ws)
        assert e.value.code == 6
        with pytest.raises(cc.CcinferError):
            take(64, gpu, torch.empty(1 << 20, dtype=torch.uint8))
