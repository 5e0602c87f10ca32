"""Drafted tokens over a K/V cache in pages, restated plainly in 64 bits (numpy): the definitions that the operators of
``manual_whisper_amd.paged`` are tested against.  Nothing here is shared with the product."""
from __future__ import annotations

import numpy as np


def plan(kept, fresh, page, max_pages, rows, pages, table, free, n_free, parents=None, words=0, target=0, least=64):
    """One step, request by request; returns a dict.  ``table`` and ``free`` (lists of lists / list) are not modified."""
    B = len(kept)
    table = [list(r) for r in table]
    free = list(free)
    out = {"row_start": [0], "admitted": [], "pages": [], "slots": [-1] * rows, "positions": [-1] * rows,
           "mask": [[0] * words for _ in range(rows)]}
    for n in fresh:
        out["row_start"].append(out["row_start"][-1] + max(0, n))
    need = [-(-(kept[b] + fresh[b]) // page) for b in range(B)]
    valid = [kept[b] >= 0 and fresh[b] >= 0 and need[b] <= max_pages and out["row_start"][b + 1] <= rows
             and (parents is None or fresh[b] <= 32 * words) for b in range(B)]
    stack = free[:n_free]
    for b in range(B):
        if valid[b] and need[b] < pages[b]:
            stack += table[b][need[b]:pages[b]]
    supply = len(stack)
    wanted = 0
    for b in range(B):
        grow = max(0, need[b] - pages[b]) if valid[b] else 0
        wanted += grow
        ok = valid[b] and (grow == 0 or wanted <= supply)
        out["admitted"].append(int(ok))
        out["pages"].append(need[b] if ok else pages[b])
        if ok:
            for k in range(grow):
                table[b][pages[b] + k] = stack.pop()
        first = out["row_start"][b]
        for i in range(max(0, fresh[b])):
            r = first + i
            if r >= rows or not valid[b]:
                continue
            at = kept[b] + i
            if ok:
                pg = table[b][at // page]
                out["slots"][r] = pg * page + at % page if pg >= 0 else -1
            if parents is None:
                out["positions"][r] = at
            else:
                line, j = [i], i
                while 0 <= parents[first + j] < j:
                    j = parents[first + j]
                    line.append(j)
                out["positions"][r] = kept[b] + len(line) - 1
                for j in line:
                    out["mask"][r][j // 32] |= 1 << (j % 32)
    out["n_free"] = len(stack)
    out["table"] = table
    lens = [kept[b] + fresh[b] if out["admitted"][b] and fresh[b] > 0 else 0 for b in range(B)]
    up64 = lambda n: -(-n // 64) * 64      # noqa: E731
    most = max(up64(-(-sum(lens) // target) if target else sum(lens)), up64(least))
    out["units"], out["unit_start"] = [], [0]
    for b in range(B):
        n = max(1, -(-lens[b] // most)) if fresh[b] > 0 else 0
        each = up64(-(-lens[b] // n)) if n else 0
        out["units"] += [[b, min(u * each, lens[b]), min((u + 1) * each, lens[b]), n] for u in range(n)]
        out["unit_start"].append(out["unit_start"][-1] + n)
    out["units"] += [[-1] * 4] * (B + target - len(out["units"]))
    return out


def rows_of(cache, table_row, page, n):
    """[heads, n, dim] and which of the n positions exist: cache [pages, heads, page, dim]."""
    got = np.zeros((cache.shape[1], n, cache.shape[3]))
    there = np.zeros(n, bool)
    for j in range(n):
        pg = table_row[j // page] if j // page < len(table_row) else -1
        if 0 <= pg < cache.shape[0]:
            got[:, j], there[j] = cache[pg, :, j % page], True
    return got, there


def attention(q, k, v, table, page, kept, row_start, mask=None, scale=None):
    """q [rows, H, D]; k, v [pages, Hkv, page, D] (values); mask [rows, N] truth values or None (chains).
    -> out, and sum_j p_j |v_j| (what roundings of the weights are relative to), the largest sum |q k| scale, and per row the
    largest |v| it sees."""
    R, H, D = q.shape
    Hkv = k.shape[1]
    scale = 1 / np.sqrt(D) if scale is None else scale
    out, size, big, vmax = np.zeros((R, H, D)), np.zeros((R, H, D)), 0.0, np.zeros((R, H, 1))
    for b in range(len(kept)):
        r0, r1 = row_start[b], row_start[b + 1]
        n = kept[b] + (r1 - r0)
        if r1 <= r0:
            continue
        kk, there = rows_of(k, table[b], page, n)
        vv, _ = rows_of(v, table[b], page, n)
        for i in range(r1 - r0):
            sees = there.copy()
            for j in range(r1 - r0):
                sees[kept[b] + j] &= bool(mask[r0 + i][j]) if mask is not None else j <= i
            if not sees.any():
                continue
            for h in range(H):
                g = h // (H // Hkv)
                with np.errstate(all="ignore"):
                    s = kk[g][sees] @ q[r0 + i, h] * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[r0 + i, h] = p @ vv[g][sees]
                    size[r0 + i, h] = p @ np.abs(vv[g][sees])
                    big = max(big, float((np.abs(kk[g][sees]) @ np.abs(q[r0 + i, h])).max() * scale))
                    vmax[r0 + i, h] = np.abs(vv[g][sees]).max()
    return out, size, big, vmax


def accept(logits, tokens, parents, row_start, depth, suppress=None):
    B = len(row_start) - 1
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    if suppress is not None:
        x[:, np.asarray(suppress) != 0] = -np.inf
    best = x.argmax(1)                                       # the first of equals
    path, ids, count = np.full((B, depth), -1), np.full((B, depth), -1), np.zeros(B, int)
    for b in range(B):
        r0, n = row_start[b], min(row_start[b + 1] - row_start[b], depth)
        at = 0 if n > 0 else None
        while at is not None:
            path[b, count[b]], ids[b, count[b]] = at, best[r0 + at]
            count[b] += 1
            at = next((i for i in range(at + 1, n) if parents[r0 + i] == at and tokens[r0 + i] == best[r0 + at]), None)
    return best, path, count, ids


def compact(cache, table, page, kept, path, count):
    """cache [layers, pages, heads, page, ...] -> a copy with the accepted rows moved."""
    new = cache.copy()
    for b in range(len(kept)):
        for i in range(min(int(count[b]), len(path[b]))):
            src, dst = kept[b] + path[b][i], kept[b] + i
            if path[b][i] <= i or src // page >= len(table[b]):
                continue
            ps, pd = table[b][src // page], table[b][dst // page]
            if 0 <= ps < cache.shape[1] and 0 <= pd < cache.shape[1]:
                new[:, pd, :, dst % page] = cache[:, ps, :, src % page]
    return new


def e4m3_rows(x):
    """float rows [..., D] -> the values their e4m3 codes and scales may stand for: (scale, largest error of a value)."""
    scale = np.abs(x).max(-1, keepdims=True) / 448
    # a code is off by at most half a step: 2^-4 of the value, or half the smallest subnormal step (2^-10) in units of the scale
    return scale, np.maximum(np.abs(x) * 2.0 ** -4, scale * 2.0 ** -10) * (1 + 1e-5)
