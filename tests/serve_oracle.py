"""Plain restatements of the serving operators for the tests: numpy, one
sequence after the other, float64 where the operator computes."""
import numpy as np

TILE = 16


def quantise(x):
    """x fp32 [..., hd] -> numbers [..., G, 32], d, m fp16 [..., G], each operation one rounded fp32 operation."""
    with np.errstate(all="ignore"):
        g = x.astype(np.float32).reshape(*x.shape[:-1], -1, 32)
        lo, hi = g.min(-1), g.max(-1)
        d, m = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16), lo.astype(np.float16)
        bad = ~(np.isfinite(d) & np.isfinite(m))
        d[bad], m[bad] = np.nan, np.nan
        df, mf = d.astype(np.float32)[..., None], m.astype(np.float32)[..., None]
        n = np.clip(np.rint((g - mf) / df), 0, 15)
        n = np.where(df > 0, n, 0)
    return n.astype(np.uint8), d, m


def values(n, d, m, dtype=np.float32):
    v = n.astype(dtype) * d.astype(dtype)[..., None] + m.astype(dtype)[..., None]
    return v.reshape(*n.shape[:-2], -1)


def rotate(x, cs):
    """x fp32 [heads, hd], cs fp32 [hd/2, 2]."""
    h = x.shape[-1] // 2
    x0, x1, c, s = x[..., :h], x[..., h:], cs[:, 0], cs[:, 1]
    return np.concatenate([x0 * c - x1 * s, x0 * s + x1 * c], -1)


def k_nibble(p, i, hd):
    """Index of value i of position p among the keys' numbers of a tile."""
    return ((p * 4 + i % 32 // 8) * (hd // 32) + i // 32) * 8 + i % 8


def v_nibble(p, i, hd):
    j = i % 32
    return ((((p % 4 // 2) * 8 + j % 8) * 4 + p // 4) * 2 + p % 2) * (hd // 32) * 4 + i // 32 * 4 + j // 8


def write_position(tile, p, k, v):
    """Store the vectors k, v (fp32 [hd]) as position p of a tile (uint8 [20 hd], in place)."""
    hd = k.shape[0]
    i = np.arange(hd)
    for which, x in ((0, k), (1, v)):
        n, d, m = quantise(x)
        at = (k_nibble if which == 0 else v_nibble)(p, i, hd)
        for nib, num in zip(at, n.reshape(-1)):
            b = which * 8 * hd + nib // 2
            tile[b] = (tile[b] & 0x0F) | (num << 4) if nib & 1 else (tile[b] & 0xF0) | num
        s = np.stack([d, m], -1).reshape(-1).view(np.uint8)
        o = 16 * hd + which * 2 * hd + p * hd // 8
        tile[o:o + hd // 8] = s


def read_tiles(tiles, hd):
    """tiles uint8 [..., 20 hd] -> k, v float64 [..., 16, hd]."""
    p, i = np.meshgrid(np.arange(TILE), np.arange(hd), indexing="ij")
    out = []
    for which, f in ((0, k_nibble), (1, v_nibble)):
        at = f(p, i, hd)
        byte = tiles[..., which * 8 * hd + at // 2]
        n = np.where(at % 2 == 1, byte >> 4, byte & 15)
        s = np.ascontiguousarray(tiles[..., 16 * hd + which * 2 * hd:16 * hd + (which + 1) * 2 * hd]).view(np.float16)
        s = s.reshape(*tiles.shape[:-1], TILE, hd // 32, 2)
        out.append(values(n.reshape(*tiles.shape[:-1], TILE, hd // 32, 32), s[..., 0], s[..., 1], np.float64))
    return out


def sequence(pages, table_row, n, hd):
    """k, v float64 [kv, n, hd] of a sequence's n positions; pages uint8 [page][kv][tiles][20 hd]."""
    count = -(-n // (pages.shape[2] * TILE))
    t = pages[table_row[:count]]
    k, v = read_tiles(t, hd)
    return [x.transpose(1, 0, 2, 3, 4).reshape(pages.shape[1], -1, hd)[:, :n] for x in (k, v)]


def attention(q, begin, pages, table, lens, hd, scale):
    """(out, lse, tolerance of out, tolerance of lse) in float64; q [rows, heads * hd].

    The tolerances bound fp32 arithmetic: a dot product of hd terms is off by at most hd * 2^-24 of the sum of
    the terms' magnitudes, an exponent that is off by x moves a weight by a factor of 1 + x, and sums of weights
    and of weighted values are off by some 2^-17 of their magnitude."""
    heads, kv = q.shape[1] // hd, pages.shape[1]
    rep = heads // kv
    out = np.zeros((q.shape[0], heads, hd))
    lse = np.full((q.shape[0], heads), -np.inf)
    tol, tol_l = np.zeros((q.shape[0], heads)), np.zeros((q.shape[0], heads))
    for s in range(table.shape[0]):
        n = max(0, int(lens[s]))
        if n == 0 or begin[s + 1] <= begin[s]:
            continue
        k, v = sequence(pages, table[s], n, hd)
        for t in range(begin[s], begin[s + 1]):
            sees = n - (begin[s + 1] - 1 - t)
            if sees <= 0:
                continue
            for h in range(heads):
                qq, kk, vv = q[t, h * hd:(h + 1) * hd].astype(np.float64), k[h // rep, :sees], v[h // rep, :sees]
                x = kk @ qq * scale
                m = x.max()
                e = np.exp(x - m)
                out[t, h] = e @ vv / e.sum()
                lse[t, h] = m + np.log(e.sum())
                ds = hd * 2.0 ** -24 * abs(scale) * (np.abs(kk) @ np.abs(qq)).max()
                tol[t, h] = (2 * ds + 2.0 ** -17) * np.abs(vv).max()
                tol_l[t, h] = ds + 2.0 ** -17 + 2.0 ** -22 * abs(m)
    return out.reshape(q.shape[0], -1), lse, tol, tol_l


def fork(table, lens, source, new_len, n_pages, page_len):
    """(new table, new lengths, copies [(from, to)]) by the header's rules, one sequence after the other."""
    slots = table.shape[1]
    n_new = len(source)
    asked, whole_of, ends_in = [], set(), {}
    for s in range(n_new):
        src, want = int(source[s]), max(0, int(new_len[s]))
        goal = -(-want // page_len)
        if src < -1 or src >= table.shape[0] or goal > slots:
            asked.append(None)
            continue
        kept = 0 if src < 0 else min(want, max(0, int(lens[src])), slots * page_len)
        row = [int(x) for x in table[src][:-(-kept // page_len)]] if src >= 0 else []
        asked.append((row, kept, goal, want))
        whole_of.update(row[:kept // page_len])
        if kept % page_len:
            ends_in.setdefault(row[-1], s)  # the lowest s
    free = [p for p in range(n_pages) if p not in whole_of and p not in ends_in]
    new, out_len, copies = np.full((n_new, slots), -1, np.int32), np.full(n_new, -1, np.int32), []
    at = 0
    for s, a in enumerate(asked):
        if a is None:
            continue
        row, kept, goal, want = a
        held, copy = list(row), None
        if kept % page_len and (row[-1] in whole_of or ends_in[row[-1]] != s):
            copy = held.pop()
        need = goal - len(held)
        given, at = (at, at + need)
        if at > len(free):
            continue
        if copy is not None:
            copies.append((copy, free[given]))
        new[s, :goal] = held + free[given:at]
        out_len[s] = want
    return new, out_len, copies


def compact(table, lens, n_pages, page_len):
    """(new table, pages in use, moves [(from, to)])."""
    rows = [[int(x) for x in table[s][:min(table.shape[1], -(-max(0, int(lens[s])) // page_len))]]
            for s in range(table.shape[0])]
    used = {p for r in rows for p in r}
    n = len(used)
    moves = list(zip(sorted(p for p in used if p >= n), [p for p in range(n) if p not in used]))
    to = dict(moves)
    new = np.full(table.shape, -1, np.int32)
    for s, r in enumerate(rows):
        new[s, :len(r)] = [to.get(p, p) for p in r]
    return new, n, moves


def scores(x, token, k):
    """Of one row (fp32 [vocab]): logprob, rank, entropy, ids, logprobs in float64, and the sum of p * |x - max|."""
    y = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(x.size), -y))
    x64 = x.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x64.max()  # NaN if there is one
        lp = x64 - m - np.log(np.exp(x64 - m).sum()) if np.isfinite(m) else np.full(x.size, np.nan)
        p = np.exp(lp)
        terms = np.where(p > 0, p * lp, 0.0) if np.isfinite(m) else p
        spread = np.where(p > 0, p * np.abs(x64 - m), 0.0).sum() if np.isfinite(m) else 0.0
    known = 0 <= token < x.size
    rank = int(np.nonzero(order == token)[0][0]) if known else -1
    return (lp[token] if known else np.nan), rank, -terms.sum(), order[:k], lp[order[:k]], spread
