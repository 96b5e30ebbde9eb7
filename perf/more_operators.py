"""The operators of a decode step that drafts: trees of drafted tokens over the paged cache, and
decode over the blocks of a long context that a cheap score selects.

  plan     what a step needs of its trees: which nodes each one sees, positions, cache slots
  attn     attention of the trees' nodes over their contexts and their own ancestors (bf16 or fp8 cache)
  accept   the drafted tokens that the model confirms, their K and V moved behind the context, all layers
  bounds   smallest and largest key of each block, element by element, after tokens were written
  score    the most that any query head of a group can make of a block, from its bounds
  sparse   blocks selected by scores, and decode attention over them (bf16 or fp8 cache)

Where `own` is false, `run` computes them by elementary torch operations. A case fixes every size, length
and tree; values, tokens and which block holds what come from the seed.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 16
DEVICE = "cuda"
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # One user's step: latency alone.
        {"op": "plan", "rows": 1, "nodes_lo": 26, "nodes_hi": 26, "len_lo": 1187, "len_hi": 1187, "lens": 1,
         "name": "plan_1x26"},
        # A full server, trees of many sizes.
        {"op": "plan", "rows": 192, "nodes_lo": 4, "nodes_hi": 64, "len_lo": 10, "len_hi": 8000, "lens": 2,
         "name": "plan_192"},
        # One user's tree in a conversation of some length.
        {"op": "attn", "rows": 1, "nodes_lo": 26, "nodes_hi": 26, "len_lo": 1187, "len_hi": 1187, "lens": 1,
         "hq": 16, "hkv": 8, "d": 128, "fp8": False, "name": "attn_1x26"},
        # A batch with trees of 8 to 64 nodes and contexts of very different lengths: the most work.
        {"op": "attn", "rows": 48, "nodes_lo": 8, "nodes_hi": 64, "len_lo": 500, "len_hi": 12000, "lens": 3,
         "hq": 32, "hkv": 8, "d": 128, "fp8": False, "name": "attn_48"},
        # The end of one user's step, all layers.
        {"op": "accept", "rows": 1, "nodes_lo": 26, "nodes_hi": 26, "len_lo": 1187, "len_hi": 1187, "lens": 4,
         "layers": 24, "hkv": 8, "d": 128, "fp8": False, "name": "accept_1x26"},
        # The end of a batch's step over an fp8 cache.
        {"op": "accept", "rows": 96, "nodes_lo": 4, "nodes_hi": 64, "len_lo": 20, "len_hi": 300, "lens": 5,
         "layers": 24, "hkv": 8, "d": 128, "fp8": True, "name": "accept_96_fp8"},
        # A decode step's new tokens: one block a request is changed.
        {"op": "bounds", "rows": 48, "new_lo": 0, "new_hi": 0, "len_lo": 3000, "len_hi": 16000, "lens": 6,
         "hkv": 8, "d": 128, "fp8": True, "name": "bounds_step_48_fp8"},
        # Prompts that were just written, some behind a cached prefix.
        {"op": "bounds", "rows": 16, "new_lo": 700, "new_hi": 15000, "len_lo": 15000, "len_hi": 16000, "lens": 7,
         "hkv": 8, "d": 128, "fp8": False, "name": "bounds_prompts_16"},
        # One long conversation: latency.
        {"op": "score", "rows": 1, "len_lo": 20011, "len_hi": 20011, "lens": 8, "hq": 16, "hkv": 8, "d": 128,
         "name": "score_1x20011"},
        # A batch of long contexts.
        {"op": "score", "rows": 48, "len_lo": 4000, "len_hi": 64000, "lens": 9, "hq": 32, "hkv": 8, "d": 128,
         "name": "score_48"},
        # One long conversation, an eighth of it looked at.
        {"op": "sparse", "rows": 1, "len_lo": 20011, "len_hi": 20011, "lens": 8, "hq": 16, "hkv": 8, "d": 128,
         "take": 160, "first": 1, "last": 2, "fp8": False, "name": "sparse_1x20011"},
        # A batch of long contexts over an fp8 cache, 2048 tokens of each looked at.
        {"op": "sparse", "rows": 48, "len_lo": 1000, "len_hi": 32000, "lens": 10, "hq": 32, "hkv": 8, "d": 128,
         "take": 128, "first": 1, "last": 4, "fp8": True, "name": "sparse_48_fp8"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(("plan", "attn", "attn", "attn", "accept", "bounds", "score", "sparse", "sparse"))
    c = {"op": op, "rows": _log(rng, 1, 64 if op != "plan" else 256), "lens": rng.randrange(1 << 20)}
    if op in ("plan", "attn", "accept"):
        hi = _log(rng, 1, 128)
        c.update(nodes_lo=rng.randint(1, hi), nodes_hi=hi)
    hi = _log(rng, 100, {"plan": 100000, "attn": 100000, "accept": 2000, "bounds": 30000}.get(op, 120000))
    c.update(len_lo=_log(rng, 1, hi), len_hi=hi)
    if op == "plan":
        return c
    hkv, d = rng.choice(((8, 128), (8, 128), (4, 128), (8, 64), (1, 128), (2, 128), (5, 64)))
    fp8 = rng.random() < 0.35
    if not fp8:
        hkv, d = rng.choice(((hkv, d), (hkv, d), (hkv, d), (4, 256), (4, 96), (8, 80), (3, 120)))
    c.update(hkv=hkv, d=d)
    if op != "score":
        c["fp8"] = fp8
    if op in ("attn", "score", "sparse"):
        c["hq"] = hkv * rng.choice((1, 2, 4, 4, 5, 7, 8, 16))
    if op == "accept":
        c["layers"] = rng.randint(1, 36)
    if op == "bounds":
        new = rng.choice((0, _log(rng, 1, c["len_hi"])))
        c.update(new_lo=min(new, 1) and rng.randint(1, new), new_hi=new)
    if op == "sparse":
        first, last = rng.randint(0, 4), rng.randint(1, 6)
        c.update(first=first, last=last, take=_log(rng, max(8, first + last), 512))
    return c


def draw(rng):
    """A case of the ranges above that costs no more, and holds no more memory, than the largest listed."""
    while True:
        c = _draw_once(rng)
        w = work(c)
        if c["op"] != "plan" and _pool_bytes(c) > 9e8:
            continue
        if w["bytes"] <= 7.3e8 and w["flops"] <= 1e11:
            return c


def _token_bytes(c):
    """Bytes of one token of K (or V) of one layer, its scales included."""
    return c["hkv"] * (c["d"] + 4 if c.get("fp8") else 2 * c["d"])


def _lengths(c):
    """Committed tokens of every row, spread over their logarithm."""
    rng = np.random.default_rng(c["lens"])
    lo, hi = math.log(c["len_lo"]), math.log(c["len_hi"])
    return np.clip(np.rint(np.exp(rng.uniform(lo, hi, c["rows"]))), c["len_lo"], c["len_hi"]).astype(np.int64)


def _trees(c):
    """(parents of every row's nodes, the node up to which the model confirms them)."""
    rng = np.random.default_rng(c["lens"] + 1)
    trees, goals = [], []
    for _ in range(c["rows"]):
        n = int(rng.integers(c["nodes_lo"], c["nodes_hi"] + 1))
        up = [-1] + [int(rng.integers(max(0, i - 12), i)) for i in range(1, n)]
        trees.append(np.array(up))
        goals.append(int(rng.integers(0, n)))
    return trees, goals


def _path(up, node):
    """The nodes from the root to this one."""
    path = []
    while node >= 0:
        path.append(node)
        node = int(up[node])
    return path[::-1]


def _fresh(c):
    """New tokens of every row of a bounds case: 0 in the case stands for a decode step's one."""
    rng = np.random.default_rng(c["lens"] + 1)
    if c["new_hi"] == 0:
        return np.ones(c["rows"], np.int64)
    return np.minimum(rng.integers(c["new_lo"], c["new_hi"] + 1, c["rows"]), _lengths(c))


def _contexts(c):
    """Tokens of every row that lie in the cache when the operator runs."""
    ctx = _lengths(c)
    if c["op"] in ("plan", "attn", "accept"):
        ctx = ctx + np.array([len(t) for t in _trees(c)[0]])
    return ctx


def _blocks(c):
    return int((-(-_contexts(c) // BLOCK)).sum()) + 3


def _pool_bytes(c):
    n = _blocks(c) * BLOCK * c.get("layers", 1)
    if c["op"] == "score":
        return _blocks(c) * c["hkv"] * c["d"] * 4
    return n * _token_bytes(c) * (1 if c["op"] == "bounds" else 2)


def work(c):
    """Inputs read once and outputs written once; of the cache, what is looked at or moved."""
    op, ctx = c["op"], _contexts(c)
    if op in ("plan", "attn", "accept"):
        trees, goals = _trees(c)
        n = np.array([len(t) for t in trees])
        words = -(-int(n.max()) // 32)
        small = int(n.sum()) * (4 * words + 12) + 8 * c["rows"]
        if op == "plan":
            return {"bytes": small + int(n.sum()) * 4, "flops": int(n.sum()) * words}
        if op == "attn":
            seen = sum(len(t) * int(b - len(t)) + sum(len(_path(t, i)) for i in range(len(t)))
                       for t, b in zip(trees, ctx))
            return {"bytes": int(ctx.sum()) * 2 * _token_bytes(c) + int(n.sum()) * (4 * c["hq"] * c["d"] + 4 * words),
                    "flops": 4 * c["hq"] * c["d"] * seen}
        moved = sum(sum(k != p for k, p in enumerate(_path(t, g))) for t, g in zip(trees, goals))
        return {"bytes": moved * c["layers"] * 4 * _token_bytes(c) + int(n.sum()) * 24 + 16 * c["rows"], "flops": 0}
    if op == "bounds":
        first = (ctx - _fresh(c)) // BLOCK
        touched = -(-ctx // BLOCK) - first
        tokens = int((ctx - first * BLOCK).sum())
        return {"bytes": tokens * _token_bytes(c) + int(touched.sum()) * 4 * c["hkv"] * c["d"],
                "flops": 2 * tokens * c["hkv"] * c["d"]}
    blocks = -(-ctx // BLOCK)
    n, rows = int(blocks.sum()), c["rows"] * c["hq"]
    if op == "score":
        return {"bytes": n * c["hkv"] * (4 * c["d"] + 4) + n * 4 + rows * 2 * c["d"], "flops": 4 * n * c["hq"] * c["d"]}
    tokens = int(np.minimum(blocks, c["take"]).sum()) * BLOCK
    return {"bytes": n * c["hkv"] * 4 + tokens * 2 * _token_bytes(c) + rows * 4 * c["d"]
            + c["rows"] * c["hkv"] * c["take"] * 4, "flops": 4 * tokens * c["hq"] * c["d"]}


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


def _caches(c, gen, x, names, blocks):
    """K and V (or K alone) of a pool of blocks of one or all layers, and the scales of an fp8 one."""
    shape = (c["layers"], blocks, BLOCK) if "layers" in c else (blocks * BLOCK,)
    shape += (c["hkv"], c["d"])
    for name in names:
        if c["fp8"]:
            cache = torch.empty(shape, dtype=torch.uint8, device=DEVICE)
            for part in cache.view(-1).split(1 << 27):
                part.copy_(torch.randn(part.shape, generator=gen, device=DEVICE).mul_(100).clamp_(-448, 448)
                           .to(E4M3).view(torch.uint8))
            scale = torch.randint(-8, -4, (c.get("layers", 1), blocks * c["hkv"] * BLOCK), generator=gen,
                                  device=DEVICE)
            scale = torch.exp2(scale.float())
            x[name], x[name + "s"] = cache, scale if "layers" in c else scale.view(-1)
        else:
            x[name], x[name + "s"] = _randn(gen, *shape), None


def _inputs(c, seed):
    rng, gen, op = np.random.default_rng(seed), _gen(seed), c["op"]
    x = {"op": op, "case": c}
    ctx, blocks = _contexts(c), _blocks(c)
    width = int(-(-ctx.max() // BLOCK)) + 2
    table, pool, at = np.full((c["rows"], width), -1), rng.permutation(blocks), 0
    for b, n in enumerate(-(-ctx // BLOCK)):
        table[b, :n] = pool[at:at + n]
        at += n
    x["table"], x["ctx"] = _i32(table), _i32(ctx)
    if op in ("plan", "attn", "accept"):
        trees, goals = _trees(c)
        sizes = [len(t) for t in trees]
        x["qsl"] = _i32(np.concatenate([[0], np.cumsum(sizes)]))
        x["parents"] = _i32(np.concatenate(trees))
        x["nodes"], x["total"] = max(sizes), sum(sizes)
        x["depth"] = max(len(_path(t, i)) for t in trees for i in range(len(t)))
    if op == "attn":
        x["q"] = _randn(gen, x["total"], c["hq"], c["d"])
        _caches(c, gen, x, ("k", "v"), blocks)
    elif op == "accept":
        draft, target = rng.integers(0, 32000, x["total"]), rng.integers(0, 32000, x["total"])
        at = 0
        for t, g in zip(trees, goals):
            path = _path(t, g)
            for a, b in zip(path, path[1:]):
                target[at + a] = draft[at + b]
            at += len(t)
        x["draft"], x["target"] = _i32(draft), _i32(target)
        _caches(c, gen, x, ("k", "v"), blocks)
    elif op == "bounds":
        x["qsl"] = None if c["new_hi"] == 0 else _i32(np.concatenate([[0], np.cumsum(_fresh(c))]))
        _caches(c, gen, x, ("k",), blocks)
        x["bounds"] = _randn(gen, blocks, c["hkv"], 2, c["d"])
    elif op == "score":
        x["q"] = _randn(gen, c["rows"], c["hq"], c["d"])
        x["bounds"] = _randn(gen, blocks, c["hkv"], 2, c["d"])
        x["bounds"][:, :, 0].sub_(1.8)  # about the smallest and the largest of a block's 16 keys
        x["bounds"][:, :, 1].add_(1.8)
        x["bounds"] = x["bounds"].sort(dim=2).values
    elif op == "sparse":
        x["q"] = _randn(gen, c["rows"], c["hq"], c["d"])
        scores = _randn(gen, c["rows"], c["hkv"], width).float()  # of 16 bits: equal ones are common
        past = torch.arange(width, device=DEVICE) >= ((x["ctx"] + BLOCK - 1) // BLOCK)[:, None]
        x["scores"] = scores.masked_fill_(past[:, None], -math.inf)
        _caches(c, gen, x, ("k", "v"), blocks)
    return x


def prepare(case, seed):
    """The tensors, and the outputs and workspaces that an engine keeps from step to step."""
    x, c, op = _inputs(case, seed), case, case["op"]

    def ints(*shape):
        return torch.empty(shape, dtype=torch.int32, device=DEVICE)

    if op in ("plan", "attn"):
        x["out"] = {"tree_mask": ints(x["total"], -(-x["nodes"] // 32)), "positions": ints(x["total"]),
                    "slot_mapping": ints(x["total"]), "status": ints(c["rows"])}
    if op == "attn":
        x["mask"] = _plan_plain(x)[0]  # made once a step, for all layers
    elif op == "accept":
        x["out"] = {"accepted": ints(c["rows"]), "accepted_nodes": ints(x["total"]), "tokens": ints(x["total"]),
                    "context_lens": ints(c["rows"])}
    elif op == "score":
        x["out"] = torch.empty((c["rows"], c["hkv"], x["table"].shape[1]), dtype=torch.float32, device=DEVICE)
    elif op == "sparse":
        x["selected"] = ints(c["rows"], c["hkv"], c["take"])
    if op in ("attn", "sparse"):
        x["o"] = torch.empty_like(x["q"])
    return x


def run(x):
    return (_run_own if own else _run_plain)(x)


def _held(x, names=("k", "v")):
    """The caches as the values that they hold."""
    if x["ks"] is None:
        return [x[n] for n in names]
    return [x[n].view(E4M3) for n in names] + [x[n + "s"] for n in names]


def _run_own(x):
    import ccinfer_amd as cc
    op, c = x["op"], x["case"]
    if op == "plan":
        out = cc.build_draft_tree(x["parents"], x["qsl"], x["ctx"], x["table"], x["nodes"], out=x["out"])
        return [out["tree_mask"], out["positions"], out["slot_mapping"], out["status"]]
    if op == "attn":
        return cc.tree_attention(x["q"], x["k"], x["v"], x["table"], x["qsl"], x["ctx"], x["mask"],
                                 k_scale=x["ks"], v_scale=x["vs"], output=x["o"])
    if op == "accept":
        out = cc.accept_draft_tokens(x["draft"], x["target"], x["parents"], x["qsl"], x["ctx"], x["table"],
                                     x["k"], x["v"], k_scale=x["ks"], v_scale=x["vs"], out=x["out"])
        return _held(x) + [out["accepted"], out["accepted_nodes"], out["tokens"], out["context_lens"]]
    if op == "bounds":
        cc.update_key_bounds(x["k"], x["bounds"], x["table"], x["ctx"], x["qsl"], k_scale=x["ks"])
        return x["bounds"]
    if op == "score":
        return cc.score_kv_blocks(x["q"], x["bounds"], x["table"], x["ctx"], out=x["out"])
    selected = cc.select_kv_blocks(x["scores"], x["ctx"], c["take"], c["first"], c["last"], out=x["selected"])
    o = cc.sparse_decode_attention(x["q"], x["k"], x["v"], x["table"], x["ctx"], selected, k_scale=x["ks"],
                                   v_scale=x["vs"], output=x["o"])
    return [selected, o]


def _grid(x):
    """(node numbers [rows, most nodes] in the flat arrays, which of them are there, tokens before the trees)."""
    first, size = x["qsl"][:-1].long(), x["qsl"][1:].long() - x["qsl"][:-1].long()
    j = torch.arange(x["nodes"], device=DEVICE)
    there = j < size[:, None]
    return torch.where(there, first[:, None] + j, 0), there, x["ctx"].long() - size


def _slots(x, pos):
    """Cache slots of positions [rows, n] of the rows."""
    return x["table"].long().gather(1, pos // BLOCK) * BLOCK + pos % BLOCK


def _plan_plain(x):
    at, there, before = _grid(x)
    n = x["nodes"]
    up = torch.where(there, x["parents"][at].long(), -1)
    j = torch.arange(n, device=DEVICE)
    # what is reached in any number of steps: (1 + step)^(2^k), as a product of truth values
    reach = ((up[:, :, None] == j) | ((j[:, None] == j) & there[:, :, None])).float()
    for _ in range(max(1, (n - 1).bit_length())):
        reach = (reach @ reach > 0).float()
    depth = reach.sum(-1).long() - 1
    out = x["out"]
    words = out["tree_mask"].shape[1]
    bits = torch.zeros((len(at), n, words * 32), dtype=torch.int64, device=DEVICE)
    bits[:, :, :n] = reach.long()
    word = (bits.view(len(at), n, words, 32) << torch.arange(32, device=DEVICE)).sum(-1)
    word = torch.where(word >= 1 << 31, word - (1 << 32), word).int()
    out["tree_mask"].copy_(word[there])
    out["positions"].copy_((before[:, None] + depth)[there])
    pos = torch.where(there, before[:, None] + j, 0)
    out["slot_mapping"].copy_(_slots(x, pos)[there])
    out["status"].zero_()
    return [out["tree_mask"], out["positions"], out["slot_mapping"], out["status"]]


def _rows_of(x, name, slots, head=slice(None)):
    """Rows of a one-layer cache in 32 bits."""
    y = x[name][slots, head]
    if x["ks"] is None:
        return y.float()
    hkv = x["case"]["hkv"]
    at = (slots // BLOCK * hkv * BLOCK + slots % BLOCK)[..., None] + torch.arange(hkv, device=DEVICE)[head] * BLOCK
    return y.view(E4M3).float() * x[name + "s"][at][..., None]


def _attn_plain(x, c):
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    trees, ctx = _trees(c)[0], _contexts(c)
    at = 0
    for b, t in enumerate(trees):
        n, length = len(t), int(ctx[b])
        pos = torch.arange(length, device=DEVICE)
        slots = _slots({"table": x["table"][b:b + 1]}, pos[None])[0]
        k, v = _rows_of(x, "k", slots), _rows_of(x, "v", slots)
        j = pos - (length - n)
        word = x["mask"][at:at + n].long()[:, j.clamp(min=0) // 32]
        sees = (j < 0) | ((word >> (j.clamp(min=0) % 32)) & 1).bool()
        q = x["q"][at:at + n].float().view(n, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
        s = (q @ k.permute(1, 2, 0)) * d ** -0.5
        s = s.view(hkv, -1, n, length).masked_fill_(~sees, -math.inf).view(hkv, -1, length)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = (p @ v.permute(1, 0, 2)) / p.sum(-1, keepdim=True)
        x["o"][at:at + n] = o.view(hkv, hq // hkv, n, d).permute(2, 0, 1, 3).reshape(n, hq, d).to(torch.bfloat16)
        at += n
    return x["o"]


def _accept_plain(x, c):
    at, there, before = _grid(x)
    up = torch.where(there, x["parents"][at].long(), -1)
    draft, target = x["draft"][at], x["target"][at]
    rows, n = at.shape
    j = torch.arange(n, device=DEVICE)
    path = torch.full((rows, n), -1, dtype=torch.int64, device=DEVICE)
    made = torch.full((rows, n), -1, dtype=torch.int32, device=DEVICE)
    now, live = torch.zeros(rows, dtype=torch.int64, device=DEVICE), torch.ones(rows, dtype=torch.bool, device=DEVICE)
    for step in range(x["depth"]):
        path[:, step] = torch.where(live, now, -1)
        said = target.gather(1, now[:, None])
        made[:, step] = torch.where(live, said[:, 0], -1)
        child = torch.where((up == now[:, None]) & (draft == said) & there & (j > 0), j, n).amin(1)
        live = live & (child < n)
        now = torch.where(live, child, now)
    count = (path >= 0).sum(1)
    some = path >= 0
    s = _slots(x, torch.where(some, before[:, None] + path, 0))[some]
    d = _slots(x, torch.where(some, before[:, None] + j, 0))[some]
    for name in ("k", "v"):
        cache = x[name].view(c["layers"], -1, c["hkv"], c["d"])
        cache[:, d] = cache[:, s]
        if c["fp8"]:
            scale = x[name + "s"].view(c["layers"], -1, c["hkv"], BLOCK)
            scale[:, d // BLOCK, :, d % BLOCK] = scale[:, s // BLOCK, :, s % BLOCK]
    out = x["out"]
    out["accepted"].copy_(count)
    out["accepted_nodes"].copy_(path[there])
    out["tokens"].copy_(made[there])
    out["context_lens"].copy_(before + count)
    return _held(x) + [out["accepted"], out["accepted_nodes"], out["tokens"], out["context_lens"]]


def _bounds_plain(x, c):
    ctx, new = _contexts(c), _fresh(c)
    for b in range(c["rows"]):
        length, start = int(ctx[b]), int(ctx[b] - new[b]) // BLOCK * BLOCK
        blocks = x["table"][b, start // BLOCK:-(-length // BLOCK)].long()
        slots = (blocks[:, None] * BLOCK + torch.arange(BLOCK, device=DEVICE))
        keys = _rows_of(x, "k", slots.view(-1)).view(*slots.shape, c["hkv"], c["d"])
        held = (start + torch.arange(slots.numel(), device=DEVICE).view(slots.shape) < length)[..., None, None]
        x["bounds"][blocks, :, 0] = keys.masked_fill(~held, math.inf).amin(1).to(torch.bfloat16)
        x["bounds"][blocks, :, 1] = keys.masked_fill(~held, -math.inf).amax(1).to(torch.bfloat16)
    return x["bounds"]


def _score_plain(x, c):
    hkv, d = c["hkv"], c["d"]
    ctx = _contexts(c)
    x["out"].fill_(-math.inf)
    for b in range(c["rows"]):
        n = -(-int(ctx[b]) // BLOCK)
        lo, hi = x["bounds"][x["table"][b, :n].long()].float().permute(2, 1, 3, 0)  # [heads, d, blocks] each
        q = x["q"][b].float().view(hkv, -1, d)
        most = q.clamp(min=0) @ hi + q.clamp(max=0) @ lo
        x["out"][b, :, :n] = most.amax(1) * d ** -0.5
    return x["out"]


def _sparse_plain(x, c):
    hq, hkv, d, take = c["hq"], c["hkv"], c["d"], c["take"]
    scores, width = x["scores"], x["table"].shape[1]
    blocks = (x["ctx"].long() + BLOCK - 1) // BLOCK
    j = torch.arange(width, device=DEVICE)
    always = (j < c["first"]) | (j >= (blocks - c["last"])[:, None])
    rank = torch.where(always[:, None], math.inf, scores)
    rank = torch.where((j < blocks[:, None])[:, None], rank, -math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :take]
    best = torch.where(torch.arange(best.shape[-1], device=DEVICE) < blocks[:, None, None], best, width)
    best = best.sort(dim=-1).values
    x["selected"].fill_(-1)
    x["selected"][..., :best.shape[-1]] = torch.where(best < width, best, -1)
    heads = torch.arange(hkv, device=DEVICE)[:, None]
    for b in range(c["rows"]):
        sel = best[b].clamp(max=width - 1)
        pos = (sel[..., None] * BLOCK + torch.arange(BLOCK, device=DEVICE)).view(hkv, -1)
        seen = (pos < x["ctx"][b]) & (best[b] < width).repeat_interleave(BLOCK, 1)
        slots = x["table"][b][sel].long().clamp(min=0).repeat_interleave(BLOCK, 1) * BLOCK + pos % BLOCK
        k, v = x["k"][slots, heads], x["v"][slots, heads]
        if c["fp8"]:
            at = slots // BLOCK * hkv * BLOCK + heads * BLOCK + slots % BLOCK
            k, v = (y.view(E4M3).float() * x[s][at][..., None] for y, s in ((k, "ks"), (v, "vs")))
        q = x["q"][b].float().view(hkv, -1, d)
        s = (q @ k.float().transpose(1, 2) * d ** -0.5).masked_fill(~seen[:, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        x["o"][b] = (p @ v.float() / p.sum(-1, keepdim=True)).view(hq, d).to(torch.bfloat16)
    return [x["selected"], x["o"]]


def _run_plain(x):
    if x["op"] == "plan":
        return _plan_plain(x)
    return {"attn": _attn_plain, "accept": _accept_plain, "bounds": _bounds_plain, "score": _score_plain,
            "sparse": _sparse_plain}[x["op"]](x, x["case"])


# The same from the definitions, in 64 bits, on other ways: trees walked node by node, rows head by head.

def _values(x, name, slots, head):
    """Rows of one head of a one-layer cache, as the values that they stand for."""
    if x["ks"] is None:
        return x[name][slots, head].double()
    scale = x[name + "s"].view(-1, x["case"]["hkv"], BLOCK)[slots // BLOCK, head, slots % BLOCK]
    return x[name].view(E4M3)[slots, head].double() * scale.double()[:, None]


def _softmax_over(q, k, v, hidden=None):
    """q [n, d] against k, v [m, d]; hidden [n, m] or None."""
    s = q @ k.T / math.sqrt(q.shape[-1])
    if hidden is not None:
        s[hidden] = -math.inf
    return torch.exp(s - torch.logsumexp(s, 1, keepdim=True)) @ v


def exact(case, seed):
    x, c, op = _inputs(case, seed), case, case["op"]
    table, ctx = x["table"].tolist(), _contexts(c).tolist()

    def slot(b, p):
        return table[b][p // BLOCK] * BLOCK + p % BLOCK

    if op in ("plan", "accept"):
        return _exact_ints(x, c, slot, ctx)
    if op == "bounds":
        answer = x["bounds"].double()
        for b, new in enumerate(_fresh(c).tolist()):
            slots = [[slot(b, p) for p in range(j * BLOCK, min(ctx[b], (j + 1) * BLOCK))]
                     for j in range((ctx[b] - new) // BLOCK, -(-ctx[b] // BLOCK))]
            for h in range(c["hkv"]):
                keys = _values(x, "k", torch.tensor(sum(slots, []), device=DEVICE), h).split([len(s) for s in slots])
                # every block but the last has 16 tokens
                if len(keys) > 1:
                    at = torch.tensor([s[0] // BLOCK for s in slots[:-1]], device=DEVICE)
                    answer[at, h] = torch.stack(torch.stack(keys[:-1]).aminmax(dim=1), 1)
                answer[slots[-1][0] // BLOCK, h] = torch.stack(keys[-1].aminmax(dim=0))
        return answer
    group = c["hq"] // c["hkv"]
    if op == "score":
        answer = torch.full(x["table"].shape[:1] + (c["hkv"],) + x["table"].shape[1:], -math.inf, dtype=torch.float64,
                            device=DEVICE)
        for b in range(c["rows"]):
            n = -(-ctx[b] // BLOCK)
            both = x["bounds"][x["table"][b, :n].long()].double()
            for h in range(c["hkv"]):
                for g in range(group):
                    s = (x["q"][b, h * group + g].double() * both[:, h]).amax(1).sum(-1) / math.sqrt(c["d"])
                    answer[b, h, :n] = torch.maximum(answer[b, h, :n], s)
        return answer
    answer = torch.zeros(x["q"].shape, dtype=torch.float64, device=DEVICE)
    if op == "attn":
        at = 0
        for b, t in enumerate(_trees(c)[0]):
            n, before = len(t), ctx[b] - len(t)
            hidden = torch.zeros((n, ctx[b]), dtype=torch.bool)
            hidden[:, before:] = True
            for i in range(n):
                hidden[i, [before + a for a in _path(t, i)]] = False
            hidden, slots = hidden.to(DEVICE), torch.tensor([slot(b, p) for p in range(ctx[b])], device=DEVICE)
            for h in range(c["hkv"]):
                k, v = _values(x, "k", slots, h), _values(x, "v", slots, h)
                for g in range(h * group, (h + 1) * group):
                    answer[at:at + n, g] = _softmax_over(x["q"][at:at + n, g].double(), k, v, hidden)
            at += n
        return answer
    scores, chosen = x["scores"].cpu().numpy(), np.full((c["rows"], c["hkv"], c["take"]), -1)
    for b in range(c["rows"]):
        n = -(-ctx[b] // BLOCK)
        for h in range(c["hkv"]):
            must = {j for j in range(n) if j < c["first"] or j >= n - c["last"]}
            rest = sorted((j for j in range(n) if j not in must), key=lambda j: (-scores[b, h, j], j))
            sel = sorted(list(must) + rest[:c["take"] - len(must)])[:c["take"]]
            chosen[b, h, :len(sel)] = sel
            slots = torch.tensor([slot(b, p) for j in sel for p in range(j * BLOCK, min(ctx[b], (j + 1) * BLOCK))],
                                 device=DEVICE)
            rows = slice(h * group, (h + 1) * group)
            answer[b, rows] = _softmax_over(x["q"][b, rows].double(), _values(x, "k", slots, h),
                                            _values(x, "v", slots, h))
    return [_i32(chosen), answer]


def _exact_ints(x, c, slot, ctx):
    up, total = [t.tolist() for t in _trees(c)[0]], x["total"]
    if c["op"] == "plan":
        words = -(-x["nodes"] // 32)
        masks, positions, slots = [], [], []
        for b, t in enumerate(up):
            before = ctx[b] - len(t)
            for i in range(len(t)):
                path = _path(t, i)
                bits = sum(1 << a for a in path)
                masks.append([np.uint32(bits >> 32 * w & 0xffffffff) for w in range(words)])
                positions.append(before + len(path) - 1)
                slots.append(slot(b, before + i))
        return [_i32(np.array(masks, np.uint32).view(np.int32)), _i32(positions), _i32(slots), _i32([0] * c["rows"])]
    draft, target = x["draft"].tolist(), x["target"].tolist()
    counts, nodes, tokens, lengths = [], [], [], []
    shape = (c["layers"], -1, c["hkv"])
    for b, t in enumerate(up):
        at, before, path = len(nodes), ctx[b] - len(t), [0]
        while True:
            good = [i for i in range(1, len(t)) if t[i] == path[-1] and draft[at + i] == target[at + path[-1]]]
            if not good:
                break
            path.append(good[0])
        for k, p in enumerate(path):  # in order: no later node's row lies where an earlier one goes
            a, z = slot(b, before + p), slot(b, before + k)
            for name in ("k", "v"):
                cache = x[name].view(*shape, c["d"])
                cache[:, z] = cache[:, a]
                if c["fp8"]:
                    scale = x[name + "s"].view(*shape, BLOCK)
                    scale[:, z // BLOCK, :, z % BLOCK] = scale[:, a // BLOCK, :, a % BLOCK]
        gap = [-1] * (len(t) - len(path))
        nodes += path + gap
        tokens += [target[at + p] for p in path] + gap
        counts.append(len(path))
        lengths.append(before + len(path))
    assert len(nodes) == total
    return _held(x) + [_i32(counts), _i32(nodes), _i32(tokens), _i32(lengths)]
