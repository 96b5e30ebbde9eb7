"""The operators between the QKV projection and the paged attention, and those of the cache's pages.

  table    (cos, sin) table of rotary positions, frequencies scaled for long contexts
  rotary   rotation of q and k by that table: half or interleaved pairs, the whole head or its first part
  norm     RMSNorm of each q and k head, the rotation, and K/V into a paged cache (bf16, or fp8 with row scales)
  copy     blocks of the paged cache copied over all layers
  update   block tables of requests changed at once: forked, admitted, released; counted references,
           the lowest free blocks handed out, a shared last block copied
  compact  live blocks moved to the front of the pool, tables and counts rewritten

Where `own` is false, `run` computes them by elementary torch operations. A case fixes every size and
length; values, positions and which block holds what come from the seed.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 16
EPS = 1e-6
DEVICE = "cuda"
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # The table of an ordinary context length, made when a model is loaded.
        {"op": "table", "positions": 40960, "rotary": 128, "scaling": "none", "name": "table_40960"},
        # A context of a million positions, frequencies stretched, half of the head rotated.
        {"op": "table", "positions": 1048576, "rotary": 64, "scaling": "yarn", "name": "table_1M_yarn"},
        # One new token of one user: latency alone.
        {"op": "rotary", "tokens": 1, "hq": 16, "hkv": 8, "d": 128, "rotary": 128, "interleaved": False,
         "packed": False, "name": "rotary_1"},
        # Prompts of odd total length, interleaved pairs in the first half of each head, q and k
        # still lying in the packed projection.
        {"op": "rotary", "tokens": 8191, "hq": 32, "hkv": 8, "d": 128, "rotary": 64, "interleaved": True,
         "packed": True, "name": "rotary_8191_part"},
        # A decode batch over an fp8 cache, interleaved pairs in part of the head.
        {"op": "norm", "tokens": 48, "hq": 32, "hkv": 8, "d": 128, "rotary": 96, "interleaved": True,
         "fp8": True, "name": "norm_48_fp8"},
        # A prompt batch: eight prompts of 1536 new tokens.
        {"op": "norm", "tokens": 12288, "hq": 16, "hkv": 8, "d": 128, "rotary": 128, "interleaved": False,
         "fp8": False, "name": "norm_12288"},
        # Copy before write of a few blocks, all layers.
        {"op": "copy", "layers": 24, "blocks": 256, "hkv": 8, "d": 128, "pairs": 5, "fp8": False, "name": "copy_5"},
        # A large part of the pool duplicated: the most bytes.
        {"op": "copy", "layers": 24, "blocks": 2048, "hkv": 8, "d": 128, "pairs": 900, "fp8": False,
         "name": "copy_900"},
        # One prompt forked into three more samples while another request leaves.
        {"op": "update", "layers": 24, "rows": 8, "width": 64, "blocks": 300, "hkv": 8, "d": 128, "beam": 0,
         "forks": 3, "admits": 0, "releases": 1, "len_lo": 200, "len_hi": 1000, "lens": 1, "fp8": False,
         "name": "update_fork_3"},
        # Beam search: twelve requests of four beams, each beam continues one of its request's beams.
        {"op": "update", "layers": 8, "rows": 48, "width": 256, "blocks": 8192, "hkv": 8, "d": 128, "beam": 4,
         "forks": 48, "admits": 0, "releases": 0, "len_lo": 100, "len_hi": 4000, "lens": 2, "fp8": False,
         "name": "update_beam_48"},
        # A small pool put in order, an fp8 cache.
        {"op": "compact", "layers": 24, "rows": 12, "width": 40, "blocks": 513, "hkv": 8, "d": 128, "live": 200,
         "fp8": True, "name": "compact_200_of_513"},
        # A pool that a busy day has left full of holes.
        {"op": "compact", "layers": 12, "rows": 64, "width": 128, "blocks": 4096, "hkv": 8, "d": 128, "live": 2400,
         "fp8": False, "name": "compact_2400_of_4096"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(("table", "rotary", "rotary", "norm", "norm", "norm", "copy", "update", "update", "compact"))
    if op == "table":
        return {"op": op, "positions": _log(rng, 2000, 1 << 20), "rotary": 2 * rng.randint(8, 64),
                "scaling": rng.choice(("none", "linear", "ntk", "yarn", "bands"))}
    fp8 = rng.random() < 0.3
    hkv, d = rng.choice(((8, 128), (8, 128), (8, 64), (2, 128), (4, 256), (4, 96), (5, 80), (1, 128)))
    if op in ("rotary", "norm"):
        hq = hkv * rng.choice((1, 2, 4, 7, 8))
        whole = rng.random() < 0.5
        c = {"op": op, "tokens": _log(rng, 1, 1000 if op == "norm" and fp8 else 12288), "hq": hq, "hkv": hkv, "d": d,
             "rotary": d if whole else 2 * rng.randint(d // 8, d // 2), "interleaved": rng.random() < 0.5}
        return {**c, "fp8": fp8} if op == "norm" else {**c, "packed": rng.random() < 0.5}
    layers = rng.randint(1, 36)
    c = {"op": op, "layers": layers, "hkv": hkv, "d": d, "fp8": fp8}
    if op == "copy":
        blocks = _log(rng, 16, 4096)
        return {**c, "blocks": blocks, "pairs": _log(rng, 1, max(1, int(blocks * 0.45)))}
    if op == "compact":
        blocks = _log(rng, 32, 4096)
        width = rng.randint(4, 128)
        return {**c, "rows": rng.randint(2, 64), "width": width, "blocks": blocks,
                "live": max(1, int(blocks * rng.uniform(0.1, 0.9)))}
    beam = rng.choice((0, 0, rng.randint(2, 8)))
    hi = _log(rng, 20, 4000)
    lo = _log(rng, 5, hi)
    if beam:
        rows = beam * rng.randint(1, 16)
        c.update(rows=rows, beam=beam, forks=rows, admits=0, releases=0)
    else:
        forks, admits, releases = _log(rng, 1, 40), rng.randint(0, 8), rng.randint(0, 8)
        c.update(rows=forks + admits + releases + rng.randint(1, 24), beam=0, forks=forks, admits=admits,
                 releases=releases)
    c.update(width=-(-hi // BLOCK) + rng.randint(0, 20), len_lo=lo, len_hi=hi, lens=rng.randrange(1 << 20))
    ctx, fresh = _lengths(c)
    held = int((-(-ctx // BLOCK)).sum()) + c["rows"] + c["releases"]
    again = int((-(-fresh // BLOCK)).sum()) + c["forks"]
    return {**c, "blocks": held + 2 * again + rng.randint(1, 1000)}


def draw(rng):
    """A case of the ranges above that costs no more, and holds no more memory, than the largest listed."""
    while True:
        c = _draw_once(rng)
        if "layers" in c and c["layers"] * c["blocks"] * _block_bytes(c) > 2.2e9:
            continue
        if work(c)["bytes"] <= 2.8e9:
            return c


def _block_bytes(c):
    """Bytes of one block of K (or V) of one layer, its scales included."""
    return BLOCK * c["hkv"] * (c["d"] + 4 if c["fp8"] else 2 * c["d"])


def _lengths(c):
    """(context of every row, lengths of the rows admitted) of an update case."""
    rng = np.random.default_rng(c["lens"])
    ctx = rng.integers(c["len_lo"], c["len_hi"] + 1, c["rows"])
    return ctx, rng.integers(c["len_lo"], c["len_hi"] + 1, c["admits"])


def work(c):
    """Inputs read once and outputs written once; of the cache, what is moved, read and written."""
    op = c["op"]
    if op == "table":
        n = c["positions"] * c["rotary"] // 2
        return {"bytes": 8 * n, "flops": 30 * n}
    if op == "rotary":
        n = c["tokens"] * (c["hq"] + c["hkv"])
        return {"bytes": n * c["d"] * 4 + c["tokens"] * (4 * c["rotary"] + 4), "flops": 3 * n * c["rotary"]}
    if op == "norm":
        rows = c["tokens"] * (c["hq"] + 2 * c["hkv"])
        kv = 2 * c["tokens"] * _block_bytes(c) // BLOCK
        return {"bytes": rows * c["d"] * 2 + c["tokens"] * (c["hq"] * c["d"] * 2 + 4 * c["rotary"] + 8) + kv,
                "flops": c["tokens"] * (c["hq"] + c["hkv"]) * (4 * c["d"] + 3 * c["rotary"])}
    if op == "copy":
        return {"bytes": 4 * c["pairs"] * c["layers"] * _block_bytes(c) + 8 * c["pairs"], "flops": 0}
    if op == "update":
        items = c["forks"] + c["admits"] + c["releases"]
        ctx, fresh = _lengths(c)
        # forks copy the part of a last block that is filled: half a block on the average
        moved = 2 * c["forks"] * c["layers"] * _block_bytes(c)
        return {"bytes": 4 * c["blocks"] + items * (12 + 8 * c["width"]) + moved, "flops": 0}
    n, live = c["blocks"], c["live"]
    moves = live - live * live // n
    return {"bytes": 12 * n + 8 * c["rows"] * c["width"] + 4 * moves * c["layers"] * _block_bytes(c), "flops": 0}


def _gen(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _randn(gen, *shape):
    out = torch.empty(shape, dtype=torch.bfloat16, device=DEVICE)
    flat = out.view(-1)
    for part in flat.split(1 << 27):
        part.copy_(torch.randn(part.shape, generator=gen, device=DEVICE, dtype=torch.float32))
    return out


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEVICE)


def _scaling(c, rng):
    """The frequency scaling of a table case, as a user writes it."""
    kind = c["scaling"]
    if kind == "none":
        return None
    s = {"type": kind, "factor": float(rng.uniform(2.0, 32.0))}
    if kind in ("yarn", "bands"):
        s["original_max_position"] = int(rng.choice((4096, 8192, 32768)))
    return s


def _caches(c, gen, x):
    """All layers' K and V of a pool of blocks, and the scales of an fp8 one."""
    shape = (c["layers"], c["blocks"], BLOCK, c["hkv"], c["d"])
    for name in ("k", "v"):
        if c["fp8"]:
            cache = torch.empty(shape, dtype=torch.uint8, device=DEVICE)
            for part in cache.view(-1).split(1 << 27):
                part.copy_(torch.randn(part.shape, generator=gen, device=DEVICE).mul_(100).clamp_(-448, 448)
                           .to(E4M3).view(torch.uint8))
            scale = torch.randint(-12, 3, (c["layers"], c["blocks"] * c["hkv"] * BLOCK), generator=gen, device=DEVICE)
            x[name], x[name + "s"] = cache, torch.exp2(scale.float())
        else:
            x[name], x[name + "s"] = _randn(gen, *shape), None


def _inputs(c, seed):
    rng, gen, op = np.random.default_rng(seed), _gen(seed), c["op"]
    x = {"op": op, "case": c}
    if op == "table":
        x["theta"] = float(math.exp(rng.uniform(math.log(1e4), math.log(1e6))))
        x["scaling"] = _scaling(c, rng)
    elif op in ("rotary", "norm"):
        t, hq, hkv, d, r = c["tokens"], c["hq"], c["hkv"], c["d"], c["rotary"]
        top = 16384
        ang = torch.arange(top, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, r, 2).double() / r)
        x["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float().to(DEVICE)
        x["pos"] = _i32(rng.integers(0, top, t))
        x["qkv"] = _randn(gen, t, (hq + 2 * hkv) * d)
        if op == "rotary":
            x["q"] = x["qkv"][:, :hq * d].view(t, hq, d)
            x["k"] = x["qkv"][:, hq * d:(hq + hkv) * d].view(t, hkv, d)
            if not c["packed"]:
                x["q"], x["k"] = x["q"].contiguous(), x["k"].contiguous()
        else:
            x["qw"] = (1.0 + 0.3 * torch.randn(d, generator=gen, device=DEVICE)).to(torch.bfloat16)
            x["kw"] = (1.0 + 0.3 * torch.randn(d, generator=gen, device=DEVICE)).to(torch.bfloat16)
            blocks = -(-t * 5 // (4 * BLOCK)) + 4
            x["slot"] = _i32(rng.permutation(blocks * BLOCK)[:t])
            _caches({**c, "layers": 1, "blocks": blocks}, gen, x)
            x["k"], x["v"] = (x[n].view(blocks * BLOCK, hkv, d) for n in ("k", "v"))
            if c["fp8"]:
                x["ks"], x["vs"] = x["ks"].view(-1), x["vs"].view(-1)
    else:
        _caches(c, gen, x)
        {"copy": _copy_inputs, "update": _update_inputs, "compact": _compact_inputs}[op](c, rng, x)
    return x


def _copy_inputs(c, rng, x):
    at = rng.permutation(c["blocks"])
    x["src"], x["dst"] = _i32(rng.choice(at[c["pairs"]:], c["pairs"])), _i32(at[:c["pairs"]])


def _update_inputs(c, rng, x):
    ctx, fresh = _lengths(c)
    rows, forks, admits, releases = c["rows"], c["forks"], c["admits"], c["releases"]
    if c["beam"]:  # every row, from a row of its own group
        dst = rng.permutation(rows)
        src = dst // c["beam"] * c["beam"] + rng.integers(0, c["beam"], rows)
        want = np.full(rows, -1)
    else:  # rows that are empty take parents' blocks, or are admitted; others leave
        order = rng.permutation(rows)
        dst = order[:forks + admits + releases]
        src = np.concatenate([rng.choice(order[forks + admits + releases:], forks), np.full(admits + releases, -1)])
        want = np.concatenate([np.full(forks, -1), fresh, np.zeros(releases, np.int64)])
        ctx[dst[:forks + admits]] = 0
        shuffled = rng.permutation(len(dst))
        dst, src, want = dst[shuffled], src[shuffled], want[shuffled]
    table, refs = np.full((rows, c["width"]), -1), np.zeros(c["blocks"], np.int64)
    free, at = rng.permutation(c["blocks"]), 0
    for b, n in enumerate(-(-ctx // BLOCK)):
        table[b, :n] = free[at:at + n]
        at += n
    refs[free[:at]] = 1
    x.update(table=_i32(table), ctx=_i32(ctx), refs=_i32(refs), dst=_i32(dst), src=_i32(src), want=_i32(want))


def _compact_inputs(c, rng, x):
    live = rng.permutation(c["blocks"])[:c["live"]]
    refs = np.zeros(c["blocks"], np.int64)
    refs[live] = 1
    table = np.full((c["rows"], c["width"]), -1)
    n = min(c["rows"] * c["width"], len(live))
    flat = np.full(c["rows"] * c["width"], -1)
    flat[rng.permutation(len(flat))[:n]] = live[:n]
    table[:] = flat.reshape(table.shape)
    shared = rng.random(c["rows"]) < 0.3  # rows that start with row 0's first block
    table[shared, 0] = table[0, 0]
    held = np.bincount(table[table >= 0], minlength=c["blocks"])
    refs = np.maximum(refs, held)
    x.update(table=_i32(table), refs=_i32(refs))


def prepare(case, seed):
    """The tensors, and the outputs and workspaces that an engine keeps from step to step."""
    x, c, op = _inputs(case, seed), case, case["op"]
    if op == "table":
        x["out"] = torch.empty((c["positions"], c["rotary"] // 2, 2), dtype=torch.float32, device=DEVICE)
    elif op == "rotary":
        x["qo"], x["ko"] = torch.empty(x["q"].shape, dtype=torch.bfloat16, device=DEVICE), torch.empty(
            x["k"].shape, dtype=torch.bfloat16, device=DEVICE)
    elif op == "norm":
        x["qo"] = torch.empty((c["tokens"], c["hq"], c["d"]), dtype=torch.bfloat16, device=DEVICE)
    else:
        x["status"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
        n = 8 * c["blocks"] + (1 << 16)  # scratch of the tables' and counts' size
        if op == "update":
            n += 4 * len(x["dst"]) * (c["width"] + 16)
        x["ws"] = torch.empty(4 * n, dtype=torch.uint8, device=DEVICE)
        if op == "compact":
            x["out"] = {"block_table": torch.empty_like(x["table"]), "ref_counts": torch.empty_like(x["refs"]),
                        "remap": torch.empty_like(x["refs"]),
                        "num_live": torch.empty(1, dtype=torch.int32, device=DEVICE)}
    return x


def run(x):
    return (_run_own if own else _run_plain)(x)


def _held(x):
    """The caches as the values that they hold."""
    if x["ks"] is None:
        return [x["k"], x["v"]]
    return [x["k"].view(E4M3), x["v"].view(E4M3), x["ks"], x["vs"]]


def _run_own(x):
    import ccinfer_amd as cc
    op, c = x["op"], x["case"]
    if op == "table":
        return cc.build_rope_cache(c["positions"], c["rotary"], x["theta"], x["scaling"], out=x["out"])
    if op == "rotary":
        return cc.rotary_embedding(x["q"], x["k"], x["pos"], x["rope"], c["interleaved"], q_out=x["qo"], k_out=x["ko"])
    if op == "norm":
        q = cc.qkv_norm_rope(x["qkv"], x["qw"], x["kw"], x["pos"], x["rope"], x["slot"], x["k"], x["v"], c["hq"], EPS,
                             c["interleaved"], k_scale=x["ks"], v_scale=x["vs"], q_out=x["qo"])
        return [q] + _held(x)
    if op == "copy":
        cc.copy_kv_blocks(x["k"], x["v"], x["src"], x["dst"], k_scale=x["ks"], v_scale=x["vs"], status=x["status"])
        return _held(x) + [x["status"]]
    if op == "update":
        cc.update_block_tables(x["table"], x["ctx"], x["refs"], x["dst"], x["src"], x["want"], x["k"], x["v"],
                               k_scale=x["ks"], v_scale=x["vs"], workspace=x["ws"], status=x["status"])
        return _held(x) + [x["table"], x["ctx"], x["refs"], x["status"]]
    out = cc.compact_kv_blocks(x["table"], x["refs"], x["k"], x["v"], k_scale=x["ks"], v_scale=x["vs"],
                               workspace=x["ws"], out=x["out"])
    return _held(x) + [out["block_table"], out["ref_counts"], out["remap"], out["num_live"]]


def _frequencies(rotary, theta, scaling):
    """(angle per position of every pair, factor of cos and sin), in 64 bits."""
    f = torch.pow(torch.tensor(theta, dtype=torch.float64), -torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    kind, by = (scaling["type"], scaling["factor"]) if scaling else ("none", 1.0)
    if kind == "linear":
        return f / by, 1.0
    if kind == "ntk":
        t = theta * by ** (rotary / (rotary - 2))
        return torch.pow(torch.tensor(t, dtype=torch.float64), -torch.arange(0, rotary, 2).double() / rotary), 1.0
    if kind == "yarn":
        # pairs that turn over 32 times in the original length keep their angle, those under once are stretched
        at = [rotary * math.log(scaling["original_max_position"] / (2 * math.pi * b)) / (2 * math.log(theta))
              for b in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary - 1)
        ramp = ((torch.arange(rotary // 2).double() - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / by * ramp + f * (1 - ramp), 0.1 * math.log(by) + 1
    if kind == "bands":
        # wavelengths up to a quarter of the original length stay, over it are stretched, between them blended
        turns = scaling["original_max_position"] * f / (2 * math.pi)
        mix = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - mix) * f / by + mix * f, 1.0
    return f, 1.0


def _rotate(x, table, rotary, interleaved):
    """x [tokens, heads, d] in 32 bits, its first `rotary` elements rotated by table [tokens, rotary / 2, 2]."""
    cos, sin = table[:, None, :, 0], table[:, None, :, 1]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        y[..., 0:rotary:2], y[..., 1:rotary:2] = a * cos - b * sin, b * cos + a * sin
    else:
        h = rotary // 2
        a, b = x[..., :h], x[..., h:rotary]
        y[..., :h], y[..., h:rotary] = a * cos - b * sin, b * cos + a * sin
    return y


def _quantised(x):
    """(e4m3 bytes, scales) of rows in 32 bits: the smallest power of two that brings the row inside +-448."""
    top = x.abs().amax(-1)
    m, e = torch.frexp(top)
    e = (e - 9 + (m > 0.875).int()).clamp(min=-126)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), e), torch.zeros_like(top))
    y = x / torch.where(top > 0, scale, torch.ones_like(scale))[..., None]
    return y.clamp(-448, 448).to(E4M3).view(torch.uint8), scale


def _scale_at(slot, hkv):
    """Where the scales of the heads of these slots lie: [block][head][16]."""
    return (slot // BLOCK * hkv * BLOCK + slot % BLOCK)[:, None] + torch.arange(hkv, device=slot.device) * BLOCK


def _run_plain(x):
    op, c = x["op"], x["case"]
    if op == "table":
        f, m = _frequencies(c["rotary"], x["theta"], x["scaling"])
        ang = torch.arange(c["positions"], dtype=torch.float64, device=DEVICE)[:, None] * f.to(DEVICE)
        x["out"][..., 0], x["out"][..., 1] = ang.cos() * m, ang.sin() * m
        return x["out"]
    if op == "rotary":
        rows = x["rope"][x["pos"].long()]
        x["qo"].copy_(_rotate(x["q"].float(), rows, c["rotary"], c["interleaved"]))
        x["ko"].copy_(_rotate(x["k"].float(), rows, c["rotary"], c["interleaved"]))
        return x["qo"], x["ko"]
    if op == "norm":
        return _norm_plain(x, c)
    if op == "copy":
        s, d = x["src"].long(), x["dst"].long()
        _move_plain(x, c, s, d)
        return _held(x) + [x["status"]]
    return _update_plain(x, c) if op == "update" else _compact_plain(x, c)


def _norm_plain(x, c):
    hq, hkv = c["hq"], c["hkv"]
    rows = x["qkv"].view(c["tokens"], hq + 2 * hkv, c["d"]).float()
    table, slot = x["rope"][x["pos"].long()], x["slot"].long()
    q, k, v = rows.split((hq, hkv, hkv), 1)
    q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * x["qw"].float()
    k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * x["kw"].float()
    x["qo"].copy_(_rotate(q, table, c["rotary"], c["interleaved"]))
    k = _rotate(k, table, c["rotary"], c["interleaved"])
    if c["fp8"]:
        (x["k"][slot], ks), (x["v"][slot], vs) = _quantised(k), _quantised(v)
        at = _scale_at(slot, hkv)
        x["ks"][at], x["vs"][at] = ks, vs
    else:
        x["k"][slot], x["v"][slot] = k.to(torch.bfloat16), v.to(torch.bfloat16)
    return [x["qo"]] + _held(x)


def _move_plain(x, c, s, d):
    """Blocks s of every layer to d; no d is an s."""
    x["k"][:, d], x["v"][:, d] = x["k"][:, s], x["v"][:, s]
    if c["fp8"]:
        ks, vs = (x[n].view(c["layers"], c["blocks"], -1) for n in ("ks", "vs"))
        ks[:, d], vs[:, d] = ks[:, s], vs[:, s]


def _update_plain(x, c):
    table, ctx, refs = x["table"], x["ctx"], x["refs"]
    d, s = x["dst"].long(), x["src"].long().clamp(min=0)
    have = torch.where(x["src"] < 0, 0, ctx[s])
    want = torch.where(x["want"] < 0, have, x["want"])
    kept = torch.minimum(have, want)
    part, known, total = kept % BLOCK, -(-kept // BLOCK), -(-want // BLOCK)
    rows = table[s]
    last = rows.gather(1, (known - 1).clamp(min=0)[:, None].long())[:, 0].long()
    copied = (part > 0) & ((s != d) | (refs[last.clamp(min=0)] > 1))
    shared = known - copied.int()
    need = total - shared
    first = need.cumsum(0) - need
    free = torch.argsort((refs != 0).int(), stable=True)
    j = torch.arange(c["width"], device=DEVICE)
    fresh = free[(first[:, None] + j - shared[:, None]).clamp(0, c["blocks"] - 1)].int()
    new = torch.where(j < shared[:, None], rows, torch.where(j < total[:, None], fresh, -1))
    old, held = table[d], -(-ctx[d] // BLOCK)
    change = torch.zeros(c["blocks"] + 1, dtype=torch.int32, device=DEVICE)
    one = torch.ones(1, dtype=torch.int32, device=DEVICE).expand(new.numel())
    change.index_add_(0, torch.where(j < total[:, None], new, c["blocks"]).long().view(-1), one)
    change.index_add_(0, torch.where(j < held[:, None], old, c["blocks"]).long().view(-1), -one)
    refs += change[:-1]
    table[d], ctx[d] = new, want.int()
    some = copied.nonzero()[:, 0]
    a, b = last[some], new[some].gather(1, (known[some] - 1)[:, None].long())[:, 0].long()
    filled = (torch.arange(BLOCK, device=DEVICE) < part[some][:, None])
    for name in ("k", "v"):
        cache = x[name]
        cache[:, b] = torch.where(filled[None, :, :, None, None], cache[:, a], cache[:, b])
        if c["fp8"]:
            scale = x[name + "s"].view(c["layers"], c["blocks"], c["hkv"], BLOCK)
            scale[:, b] = torch.where(filled[None, :, None, :], scale[:, a], scale[:, b])
    return _held(x) + [table, ctx, refs, x["status"]]


def _compact_plain(x, c):
    refs, table, out = x["refs"], x["table"], x["out"]
    at = torch.arange(c["blocks"], device=DEVICE)
    live = refs > 0
    n = live.sum()
    s, d = (live & (at >= n)).nonzero()[:, 0], (~live & (at < n)).nonzero()[:, 0]
    remap = torch.where(live, at, -1)
    remap[s] = d
    out["remap"].copy_(remap)
    counts = torch.where(live & (at < n), refs, 0)
    counts[d] = refs[s]
    out["ref_counts"].copy_(counts)
    out["block_table"].copy_(torch.where(table < 0, table, remap[table.clamp(min=0).long()].int()))
    out["num_live"].copy_(n)
    _move_plain(x, c, s, d)
    return _held(x) + [out["block_table"], out["ref_counts"], out["remap"], out["num_live"]]


# The same from the definitions, in 64 bits, on other ways: pairs as complex numbers, tables block by block.

def _turned(x, angle, rotary, interleaved):
    """x [tokens, heads, d] in 64 bits; the pairs as complex numbers times `angle` [tokens, rotary / 2]."""
    head = x[..., :rotary]
    n = x.shape[:-1]
    pairs = head.reshape(*n, rotary // 2, 2) if interleaved else head.reshape(*n, 2, rotary // 2).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * angle[:, None, :])
    z = z if interleaved else z.transpose(-1, -2)
    return torch.cat([z.reshape(*n, rotary), x[..., rotary:]], -1)


def _exact_frequency(p, rotary, theta, scaling):
    """The angle per position of pair p."""
    f = math.exp(-2 * p / rotary * math.log(theta))
    if scaling is None:
        return f
    by = scaling["factor"]
    if scaling["type"] == "linear":
        return f / by
    if scaling["type"] == "ntk":  # the slowest pair is stretched by the whole factor, the fastest by nothing
        return f * math.exp(-2 * p / (rotary - 2) * math.log(by))
    length = scaling["original_max_position"]
    if scaling["type"] == "bands":
        wave = 2 * math.pi / f
        if wave < length / 4:
            return f
        if wave > length:
            return f / by
        part = (length / wave - 1) / 3
        return f * (part + (1 - part) / by)
    edge = [rotary / 2 * (math.log(length) - math.log(2 * math.pi * b)) / math.log(theta) for b in (32, 1)]
    lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rotary - 1)
    part = 0.0 if p <= lo else 1.0 if p >= hi else (p - lo) / (hi - lo)
    return f * ((1 - part) + part / by)


def exact(case, seed):
    x, c, op = _inputs(case, seed), case, case["op"]
    if op == "table":
        s = x["scaling"]
        f = [_exact_frequency(p, c["rotary"], x["theta"], s) for p in range(c["rotary"] // 2)]
        m = 1 + 0.1 * math.log(s["factor"]) if s and s["type"] == "yarn" else 1.0
        ang = torch.outer(torch.arange(c["positions"], device=DEVICE).double(),
                          torch.tensor(f, dtype=torch.float64, device=DEVICE))
        return torch.view_as_real(torch.polar(torch.full_like(ang, m), ang))
    if op in ("rotary", "norm"):
        angle = torch.view_as_complex(x["rope"].double()[x["pos"].long()])
        turn = lambda y: _turned(y, angle, c["rotary"], c["interleaved"])  # noqa: E731
        if op == "rotary":
            return turn(x["q"].double()), turn(x["k"].double())
        rows, hq, hkv = x["qkv"].double().view(c["tokens"], -1, c["d"]), c["hq"], c["hkv"]
        size = torch.sqrt(rows.pow(2).sum(-1, keepdim=True) / c["d"] + EPS)
        q = turn(rows[:, :hq] / size[:, :hq] * x["qw"].double())
        k = turn(rows[:, hq:hq + hkv] / size[:, hq:hq + hkv] * x["kw"].double())
        slot, v = x["slot"].long(), rows[:, hq + hkv:]
        if not c["fp8"]:
            kc, vc = x["k"].double(), x["v"].double()
            kc[slot], vc[slot] = k, v
            return [q, kc, vc]
        answer = [q]
        scales = []
        for cache, scale, y in ((x["k"], x["ks"], k), (x["v"], x["vs"], v)):
            held = cache.view(E4M3).double()
            p = torch.exp2(torch.ceil(torch.log2(y.abs().amax(-1) / 448)).clamp(min=-126))
            held[slot] = y / p[..., None]
            scale = scale.double()
            scale[_scale_at(slot, hkv)] = p
            answer.append(held)
            scales.append(scale)
        return answer + scales
    return _exact_pages(x, c, op)


def _exact_pages(x, c, op):
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)

    def move(a, b, tokens=BLOCK):
        for name in ("k", "v"):
            x[name][:, b, :tokens] = x[name][:, a, :tokens]
            if c["fp8"]:
                scale = x[name + "s"].view(c["layers"], c["blocks"], c["hkv"], BLOCK)
                scale[:, b, :, :tokens] = scale[:, a, :, :tokens]

    if op == "copy":
        for a, b in zip(x["src"].tolist(), x["dst"].tolist()):
            move(a, b)
        return _held(x) + [status]
    table, refs = x["table"].tolist(), x["refs"].tolist()
    if op == "compact":
        live = [b for b, r in enumerate(refs) if r > 0]
        n = len(live)
        to = {b: b for b in live if b < n}
        holes = [b for b in range(n) if refs[b] <= 0]
        for a, b in zip([b for b in live if b >= n], holes):
            move(a, b)
            to[a] = b
        counts = [0] * len(refs)
        for a, b in to.items():
            counts[b] = refs[a]
        table = [[b if b < 0 else to.get(b, -1) for b in row] for row in table]
        return _held(x) + [_i32(table), _i32(counts), _i32([to.get(b, -1) for b in range(len(refs))]), _i32([n])]
    ctx = x["ctx"].tolist()
    free = iter([b for b, r in enumerate(refs) if r == 0])
    new_table, new_ctx, new_refs = [list(r) for r in table], list(ctx), list(refs)
    moves = []
    for d, s, want in zip(x["dst"].tolist(), x["src"].tolist(), x["want"].tolist()):
        have = ctx[s] if s >= 0 else 0
        want = have if want < 0 else want
        kept = min(have, want)
        row = table[s][:-(-kept // BLOCK)] if s >= 0 else []
        if kept % BLOCK and (s != d or refs[row[-1]] > 1):
            fresh = next(free)
            moves.append((row[-1], fresh, kept % BLOCK))
            row[-1] = fresh
        while len(row) * BLOCK < want:
            row.append(next(free))
        for b in row:
            new_refs[b] += 1
        for b in table[d][:-(-ctx[d] // BLOCK)]:
            new_refs[b] -= 1
        new_table[d] = row + [-1] * (c["width"] - len(row))
        new_ctx[d] = want
    for a, b, tokens in moves:
        move(a, b, tokens)
    return _held(x) + [_i32(new_table), _i32(new_ctx), _i32(new_refs), status]
