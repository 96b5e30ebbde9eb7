"""References in 64 bits (numpy on the CPU) of the operators on drafted trees and selected blocks,
their inputs, and the bounds of what the kernels' arithmetic may be off."""
from __future__ import annotations

import numpy as np
import torch

BLOCK = 16
E4M3 = torch.float8_e4m3fn


def visible(parents):
    """[n, n]: node i sees node j (its ancestors and itself)."""
    n = len(parents)
    see = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while j >= 0:
            see[i, j] = True
            j = parents[j]
    return see


def random_tree(rng, n, back=9):
    return ([-1] + [int(rng.integers(max(0, i - back), i)) for i in range(1, n)])[:n]


def pack_mask(see, words):
    """Rows of truth values -> int32 words, bit j % 32 of word j // 32."""
    bits = np.zeros((see.shape[0], words * 32), np.uint64)
    bits[:, :see.shape[1]] = see
    w = (bits.reshape(-1, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1)
    return w.astype(np.uint32).view(np.int32)


def make_tables(rng, ctx, width, spare=5):
    """Blocks of every row in a shuffled pool: (table int32, number of blocks)."""
    need = [-(-int(c) // BLOCK) if c > 0 else 0 for c in ctx]
    pool = rng.permutation(sum(need) + spare)
    table, at = np.full((len(ctx), width), -1, np.int32), 0
    for b, n in enumerate(need):
        n = min(n, width)
        table[b, :n] = pool[at:at + n]
        at += n
    return table, len(pool)


class Cache:
    """One layer's K and V of `blocks` blocks, bf16 or fp8 with scales; `k64` / `v64` are the
    values. Slots that hold no token are filled with NaN."""

    def __init__(self, rng, blocks, hkv, d, fp8, held=None):
        self.fp8, self.hkv, self.d, self.blocks = fp8, hkv, d, blocks
        shape = (blocks * BLOCK, hkv, d)
        gen = torch.Generator().manual_seed(int(rng.integers(1 << 31)))
        self.t = {}
        for name in ("k", "v"):
            x = torch.randn(shape, generator=gen)
            if fp8:
                q = (x * 100).clamp(-448, 448).to(E4M3)
                s = torch.exp2(torch.randint(-8, -5, shape[:2], generator=gen).float())
                if held is not None:
                    q.view(torch.uint8)[~held] = 0x7f
                    s[~held] = float("nan")
                self.t[name] = q.view(torch.uint8)
                lay = s.view(blocks, BLOCK, hkv).permute(0, 2, 1).contiguous().view(-1)
                self.t[name + "s"] = lay
                self.t[name + "64"] = (q.float().double() * s.double()[..., None]).numpy()
            else:
                y = x.bfloat16()
                if held is not None:
                    y[~held] = float("nan")
                self.t[name], self.t[name + "s"] = y, None
                self.t[name + "64"] = y.double().numpy()

    def on(self, dev):
        return {n: (x.to(dev) if isinstance(x, torch.Tensor) else x)
                for n, x in self.t.items() if not n.endswith("64")}


def held_slots(table, ctx, blocks):
    held = torch.zeros(blocks * BLOCK, dtype=torch.bool)
    for row, c in zip(table, ctx):
        for p in range(min(int(c), table.shape[1] * BLOCK)):
            if row[p // BLOCK] >= 0:
                held[int(row[p // BLOCK]) * BLOCK + p % BLOCK] = True
    return held


def attend(q, k, v, see=None):
    """q [n, d], k / v [m, d], see [n, m]: (output, bound of the kernels' error).

    The bound, with A = sum p |v| / sum p: probabilities are rounded to bf16 once (2^-8 of each);
    a logit's products are summed in float32 (d + 8 roundings of at most 2^-24 of sum |q k|, the
    scale and the exponential among them), which moves a probability by as much and the sum of
    them too; products and sums over m keys, parts and their merge are float32 ((m + 64) 2^-24);
    the result is rounded to bf16 (2^-8 of itself)."""
    n, d = q.shape
    scale = 1 / np.sqrt(d)
    out, tol = np.zeros((n, v.shape[1])), np.zeros((n, v.shape[1]))
    for i in range(n):
        at = np.arange(k.shape[0]) if see is None else np.nonzero(see[i])[0]
        if len(at) == 0:
            continue
        kk, vv = k[at], v[at]
        s = kk @ q[i] * scale
        p = np.exp(s - s.max())
        out[i] = p @ vv / p.sum()
        size = p @ np.abs(vv) / p.sum()
        logit = (d + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[i])).max() * scale
        part = size * (2.0 ** -8 + 2 * logit + (len(at) + 64) * 2.0 ** -24)
        tol[i] = part + 2.0 ** -8 * (np.abs(out[i]) + part) + 2.0 ** -126
    return out, tol


def slots_of(row, ctx, width):
    """(positions that a row holds, their slots)."""
    pos = [p for p in range(min(int(ctx), width * BLOCK)) if row[p // BLOCK] >= 0]
    return np.array(pos, int), np.array([int(row[p // BLOCK]) * BLOCK + p % BLOCK for p in pos], int)


def tree_attention(q, cache, table, qsl, ctx, sees, fill):
    """q float64 [total, hq, d]; sees[b] [n, n]. Rows that are left alone hold `fill`, tolerance 0."""
    total, hq, d = q.shape
    G = hq // cache.hkv
    out, tol = np.full(q.shape, float(fill)), np.zeros(q.shape)
    for b in range(len(ctx)):
        n = qsl[b + 1] - qsl[b]
        before = ctx[b] - n
        if n <= 0 or before < 0:
            continue
        pos, slots = slots_of(table[b], ctx[b], table.shape[1])
        see = np.ones((n, len(pos)), bool)
        for x, p in enumerate(pos):
            if p >= before:
                see[:, x] = sees[b][:, p - before] if p - before < sees[b].shape[1] else False
        rows = slice(qsl[b], min(qsl[b + 1], total))
        for h in range(hq):
            k, v = cache.t["k64"][slots, h // G], cache.t["v64"][slots, h // G]
            o, t = attend(q[rows, h], k, v, see[:rows.stop - rows.start])
            out[rows, h], tol[rows, h] = o, t
    return out, tol


def sparse_decode(q, cache, table, ctx, selected):
    rows, hq, d = q.shape
    G = hq // cache.hkv
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(rows):
        n = -(-int(ctx[b]) // BLOCK) if ctx[b] > 0 else 0
        if n > table.shape[1]:
            continue
        for h in range(cache.hkv):
            slots = []
            for j in selected[b, h]:
                if 0 <= j < n and table[b, j] >= 0:
                    slots += [int(table[b, j]) * BLOCK + x
                              for x in range(min(BLOCK, int(ctx[b]) - int(j) * BLOCK))]
            g = slice(h * G, (h + 1) * G)
            out[b, g], tol[b, g] = attend(q[b, g], cache.t["k64"][slots, h],
                                          cache.t["v64"][slots, h])
    return out, tol


def key_bounds(cache, table, ctx, new, bounds):
    """bounds float64 [blocks, hkv, 2, d], the touched blocks renewed in a copy."""
    bounds = bounds.copy()
    for b, (c, m) in enumerate(zip(ctx, new)):
        if c <= 0 or m <= 0:
            continue
        for j in range(max(c - m, 0) // BLOCK, min(-(-c // BLOCK), table.shape[1])):
            if table[b, j] < 0:
                continue
            s = int(table[b, j]) * BLOCK
            keys = cache.t["k64"][s:s + min(BLOCK, c - j * BLOCK)]
            bounds[table[b, j], :, 0], bounds[table[b, j], :, 1] = keys.min(0), keys.max(0)
    return bounds


def scores(q, bounds, table, ctx):
    """(scores, bound of float32's error): 2 d products and as many sums, the scale."""
    rows, hq, d = q.shape
    hkv, width = bounds.shape[1], table.shape[1]
    out = np.full((rows, hkv, width), -np.inf)
    tol = np.zeros(out.shape)
    for b in range(rows):
        n = -(-int(ctx[b]) // BLOCK) if ctx[b] > 0 else 0
        if n > width:
            continue
        for j in range(n):
            if table[b, j] < 0:
                continue
            for h in range(hkv):
                both = bounds[table[b, j], h]
                g = q[b].reshape(hkv, -1, d)[h]
                terms = np.maximum(g * both[0], g * both[1])
                out[b, h, j] = terms.sum(-1).max() / np.sqrt(d)
                tol[b, h, j] = np.abs(terms).sum(-1).max() / np.sqrt(d) * (2 * d + 4) * 2.0 ** -24
    return out, tol


def select(sc, ctx, take, first, last):
    rows, hkv, width = sc.shape
    out = np.full((rows, hkv, take), -1, np.int32)
    for b in range(rows):
        n = -(-int(ctx[b]) // BLOCK) if ctx[b] > 0 else 0
        n = 0 if n > width else n
        for h in range(hkv):
            if n <= take:
                out[b, h, :n] = np.arange(n)
                continue
            must = [j for j in range(n) if j < first or j >= n - last]
            rest = sorted((j for j in range(first, n - last)),
                          key=lambda j: (0 if np.isnan(sc[b, h, j]) else 1,
                                         0.0 if np.isnan(sc[b, h, j]) else -sc[b, h, j], j))
            out[b, h] = sorted(must + rest[:take - len(must)])
    return out


def accept(draft, target, parents, qsl, ctx):
    """Per request: the path; and accepted, accepted_nodes, tokens, context_lens as the call gives
    them (rows of no request hold -7, as the tests fill the outputs)."""
    total = len(draft)
    nodes, tokens = np.full(total, -7, np.int32), np.full(total, -7, np.int32)
    paths, counts, lengths = [], [], []
    for b in range(len(ctx)):
        a, n = int(qsl[b]), int(qsl[b + 1] - qsl[b])
        before = int(ctx[b]) - n
        nodes[a:a + n], tokens[a:a + n] = -1, -1
        path = []
        if n > 0 and before >= 0 and n <= 2048:
            path = [0]
            while True:
                good = [i for i in range(path[-1] + 1, n)
                        if parents[a + i] == path[-1] and draft[a + i] == target[a + path[-1]]]
                if not good:
                    break
                path.append(good[0])
        nodes[a:a + len(path)] = path
        tokens[a:a + len(path)] = [target[a + i] for i in path]
        paths.append(path)
        counts.append(len(path))
        lengths.append(before + len(path) if path else int(ctx[b]))
    return paths, np.array(counts, np.int32), nodes, tokens, np.array(lengths, np.int32)
