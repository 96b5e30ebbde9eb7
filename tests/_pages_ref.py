"""Block tables, counted references and the pool's order, one block after the other (numpy)."""
from __future__ import annotations

import numpy as np


def copy(caches, src, dst, blocks):
    """(caches after the pairs, status): caches is a list of arrays [layers, blocks, ...]."""
    ok = [(s, d) for s, d in zip(src, dst) if 0 <= s < blocks and 0 <= d < blocks and s != d]
    out, status = [c.copy() for c in caches], 0
    for s, d in ok:
        if any((s, d) != (a, b) and (b == d or b == s or a == d) for a, b in ok):
            status = 6
            continue
        for c, o in zip(caches, out):
            o[:, d] = c[:, s]
    return out, status


def update(table, ctx, refs, dst, src, lengths, caches, scales, bs, have_caches=True):
    """Returns (table, ctx, refs, caches, scales, status); caches [layers, blocks, bs, ...],
    scales [layers, blocks, heads, 16]."""
    rows, width = table.shape
    same = (table.copy(), ctx.copy(), refs.copy(), [c.copy() for c in caches],
            [s.copy() for s in scales])
    n = len(dst)
    src = list(dst) if src is None else list(src)
    lengths = [-1] * n if lengths is None else list(lengths)
    invalid = bad_table = False
    need = []
    for i in range(n):
        d, s, want = dst[i], src[i], lengths[i]
        if not (0 <= d < rows and -1 <= s < rows and -1 <= want <= width * bs) \
                or sum(1 for x in dst if x == d) > 1:
            invalid = True
            continue
        have = int(ctx[s]) if s >= 0 else 0
        if not (0 <= have <= width * bs and 0 <= ctx[d] <= width * bs):
            bad_table = True
            continue
        want = have if want < 0 else want
        kept = min(want, have)
        held = list(table[s][:-(-kept // bs)]) if s >= 0 else []
        old = list(table[d][:-(-int(ctx[d]) // bs)])
        if any(not (0 <= b < len(refs)) or refs[b] <= 0 for b in held + old):
            bad_table = True
            continue
        # rows that take the last block over as a whole block of theirs in the same call
        takers = [j for j in range(n) if src[j] == d and dst[j] != d
                  and min(have, have if lengths[j] < 0 else lengths[j]) >= len(held) * bs]
        copied = kept % bs != 0 and (s != d or refs[held[-1]] > 1 or bool(takers))
        if copied and not have_caches:
            invalid = True
        need.append((d, want, kept, held, old, copied))
    free = [b for b in range(len(refs)) if refs[b] <= 0]
    wanted = sum(-(-w // bs) - len(h) + c for _, w, _, h, _, c in need)
    if invalid or bad_table or wanted > len(free):
        return (*same, 6 if invalid else 14 if bad_table else 12)
    t, c, r, cc, ss = same
    at = 0
    moves = []
    for d, want, kept, held, old, copied in need:
        if copied:
            moves.append((held[-1], free[at], kept % bs))
            held[-1] = free[at]
            at += 1
        more = -(-want // bs) - len(held)
        held += free[at:at + more]
        at += more
        for b in held:
            r[b] += 1
        for b in old:
            r[b] -= 1
        t[d] = held + [-1] * (width - len(held))
        c[d] = want
    for a, b, tokens in moves:
        for x, y in zip(caches, cc):
            y[:, b, :tokens] = x[:, a, :tokens]
        for x, y in zip(scales, ss):
            y[:, b, :, :tokens] = x[:, a, :, :tokens]
    return t, c, r, cc, ss, 0


def compact(table, refs, caches):
    """Returns (table, refs, remap, num_live, caches); caches [layers, blocks, ...]."""
    live = [b for b in range(len(refs)) if refs[b] > 0]
    n = len(live)
    to = {b: b for b in live if b < n}
    out = [c.copy() for c in caches]
    holes = [b for b in range(n) if refs[b] <= 0]
    for a, b in zip([b for b in live if b >= n], holes):
        to[a] = b
        for c, o in zip(caches, out):
            o[:, b] = c[:, a]
    counts = np.zeros_like(refs)
    for a, b in to.items():
        counts[b] = refs[a]
    t = np.array([[b if b < 0 else to.get(int(b), -1) for b in row] for row in table],
                 table.dtype).reshape(table.shape)
    remap = np.array([to.get(b, -1) for b in range(len(refs))], refs.dtype)
    return t, counts, remap, n, out


def consistent(table, ctx, refs, bs):
    """Every block that a row holds is counted once for each row that holds it, and a block that
    a row has filled in part is held by that row alone."""
    count = np.zeros_like(refs)
    for row, n in zip(table, ctx):
        held = row[:-(-int(n) // bs)]
        assert np.all(held >= 0) and np.all(row[len(held):] == -1)
        np.add.at(count, held, 1)
    assert np.array_equal(count, refs)
    for row, n in zip(table, ctx):
        assert n % bs == 0 or refs[row[int(n) // bs]] == 1
