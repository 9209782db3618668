"""The serving operators, case by case: their inputs, their plain forms and what they cannot do without.

Many sequences share one cache of pages held in 4 bits.  Four operators work on it:

append   rotates q and k (RoPE) and writes k and v into the pages, quantised
attend   attention of each sequence's newest rows over its pages
pages    fork, reorder, grow, truncate and free sequences; compact the pool
scores   log probability, rank, entropy and best alternatives of sampled tokens

``own`` chooses what ``run`` calls: the plain forms below (elementary torch
operations in fp32), or the framework's kernels.

Page format.  ``pages`` is uint8 [layer][page][kv head][tile][tile bytes]; a
tile holds 16 positions of one head: K nibbles, V nibbles, K scales, V scales.
A head's vector is split into groups of 32 values; a group holds (d, m) in
fp16 and 4-bit numbers n, and stands for d * n + m.

K nibbles  [position 16][t 4][group][n 8]: value 32 group + 8 t + n
V nibbles  [a 2][r 8][t 4][b 2][group][c 4]: position 4 t + 2 a + b, value 32 group + 8 c + r
scales     [position 16][group][d, m]
(two nibbles a byte, the first in the low half)
"""
import math
import random

import numpy as np
import torch

own = False

TILE = 16  # positions of a tile


# ---- cases -----------------------------------------------------------------


def listed():
    return [
        # one generated token of one sequence, heads of an 8B model: latency
        dict(name="append 1 token", op="append", seqs=1, tokens=1, head=32, kv=8, hd=128, page=64, longest=4096,
             rope=True, spread=1),
        # the prompts of a batch of sequences, written in one call
        dict(name="append 2048 tokens", op="append", seqs=7, tokens=2048, head=32, kv=8, hd=128, page=64,
             longest=4096, rope=True, spread=2),
        # the first words of a chat: one sequence, a page that ends inside a tile
        dict(name="attend short", op="attend", seqs=1, rows=1, shortest=37, longest=37, head=32, kv=8, hd=128,
             page=64, spread=3),
        # a serving batch, ragged lengths, heads of a 70B model
        dict(name="attend batch of 64", op="attend", seqs=64, rows=1, shortest=150, longest=8190, head=64, kv=8,
             hd=128, page=64, spread=4),
        # one long document, one generated token: the long axis has to be split
        dict(name="attend 131071", op="attend", seqs=1, rows=1, shortest=131071, longest=131071, head=32, kv=8,
             hd=128, page=64, spread=5),
        # a piece of a prompt against what is cached of it
        dict(name="attend prompt", op="attend", seqs=1, rows=1024, shortest=8000, longest=8000, head=32, kv=8,
             hd=128, page=64, spread=6),
        # heads of 64 without sharing; some sequences decode, some bring rows of a prompt
        dict(name="attend mixed rows", op="attend", seqs=9, rows=300, shortest=5, longest=2500, head=8, kv=8, hd=64,
             page=32, spread=7),
        # eight candidates of one prompt, each with room for its next words
        dict(name="fork best of 8", op="fork", seqs=8, shortest=1001, longest=1001, more=40, layers=8, kv=8, hd=128,
             page=64, pool=64, alike=True, spread=8),
        # one step of a beam search over many requests: most beams change their parent
        dict(name="fork 192 beams", op="fork", seqs=192, shortest=40, longest=500, more=1, layers=4, kv=8, hd=128,
             page=64, pool=2048, alike=False, spread=9),
        # a pool after many requests have left it
        dict(name="compact", op="compact", seqs=96, shortest=100, longest=900, layers=4, kv=8, hd=128, page=64,
             pool=2048, spread=10),
        # the sampled token of one sequence, vocabulary of the 8B model: latency
        dict(name="score 1 row", op="score", rows=1, vocab=128256, top=5, masked=False, spread=11),
        # every token of a prompt
        dict(name="score 512 rows", op="score", rows=512, vocab=128256, top=20, masked=True, spread=12),
    ]


def _log(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm; round ones give way to odd ones."""
    x = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    x = min(hi, max(lo, x))
    return x - 1 if x % 512 == 0 and x > lo else x


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "fork", "compact", "score", "score"])
    kv = rng.choice([1, 2, 4, 8])
    shape = dict(kv=kv, hd=rng.choice([64, 128, 128]), page=rng.choice([16, 32, 48, 64, 128]))
    spread = rng.randrange(1 << 20)
    if op == "append":
        return dict(op=op, seqs=rng.randint(1, 9), tokens=_log(rng, 1, 2048), head=kv * rng.choice([1, 2, 3, 4]),
                    longest=4096, rope=rng.random() < 0.75, spread=spread, **shape)
    if op == "attend":
        head = kv * rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
        if rng.random() < 0.6:  # generated tokens
            longest = _log(rng, 1, 100000)
            seqs = _log(rng, 1, max(1, min(64, 130000 // longest)))
            rows = 1 if rng.random() < 0.8 else rng.randint(2, 6)
        else:  # rows of prompts
            longest, head = _log(rng, 20, 8000), min(head, 32)
            seqs = _log(rng, 1, max(1, min(9, 8000 // longest)))
            rows = _log(rng, 2, min(longest, 900))
        return dict(op=op, seqs=seqs, rows=rows, shortest=max(1, longest // rng.choice([1, 3, 20])), longest=longest,
                    head=head, spread=spread, **shape)
    if op == "fork":
        longest = _log(rng, 10, 500)
        seqs = _log(rng, 2, 160)
        pages = seqs * (longest // shape["page"] + 2) + 7
        return dict(op=op, seqs=seqs, shortest=max(1, longest // 3), longest=longest, more=rng.choice([0, 1, 1, 40]),
                    layers=rng.randint(1, 4), pool=pages, alike=rng.random() < 0.3, spread=spread, **shape)
    if op == "compact":
        longest, seqs = _log(rng, 10, 900), _log(rng, 2, 64)
        pages = int(seqs * (longest // shape["page"] + 1) * rng.uniform(1.0, 2.5)) + 3
        return dict(op=op, seqs=seqs, shortest=max(1, longest // 3), longest=longest, layers=rng.randint(1, 4),
                    pool=pages, spread=spread, **shape)
    vocab = _log(rng, 1000, 152000)
    return dict(op=op, rows=_log(rng, 1, min(512, 40_000_000 // vocab)), vocab=vocab,
                top=rng.choice([0, 1, 5, 20, 32]), masked=rng.random() < 0.5, spread=spread)


# ---- what a case fixes whatever the seed: lengths, rows, the order of pages --


def _lengths(case):
    rng = random.Random(case["spread"])
    lo, hi = case["shortest"], case["longest"]
    got = [int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))) for _ in range(case["seqs"])]
    got[rng.randrange(len(got))] = hi
    return got


def _rows(case):
    """Rows that each sequence brings: all of them, or every third sequence one (it is decoding)."""
    rng = random.Random(case["spread"] + 1)
    lens = _lengths(case)
    if case["rows"] == 1 or case["seqs"] == 1:
        return [min(case["rows"], n) for n in lens]
    return [1 if i % 3 == 2 else min(n, rng.randint(1, case["rows"])) for i, n in enumerate(lens)]


def _append_tokens(case):
    """(sequence, first position, tokens) of what is written."""
    rng = random.Random(case["spread"])
    cut = sorted(rng.randrange(case["tokens"] + 1) for _ in range(case["seqs"] - 1))
    counts = [b - a for a, b in zip([0] + cut, cut + [case["tokens"]])]
    return [(i, rng.randrange(case["longest"] - n + 1), n) for i, n in enumerate(counts)]


def _fork_request(case):
    """Lengths before, source of each new sequence, its new length."""
    rng = random.Random(case["spread"] + 2)
    lens = _lengths(case)
    n = case["seqs"]
    if case["alike"]:  # candidates of the first sequence, which stays
        lens = [lens[0]] + [0] * (n - 1)
        return lens, [0] * n, [lens[0] + case["more"]] * n
    source = [rng.randrange(n) for _ in range(n)]
    ends = [rng.random() < 0.05 for _ in range(n)]  # a finished request leaves
    source = [-1 if e else s for s, e in zip(source, ends)]
    return lens, source, [0 if s < 0 else lens[s] + case["more"] for s in source]


def _fork_copies(case):
    """Pages that the fork has to copy."""
    lens, source, want = _fork_request(case)
    copies, seen = 0, set()
    for s, w in zip(source, want):
        kept = 0 if s < 0 else min(lens[s], w)
        if kept % case["page"]:
            copies += s in seen  # in these cases a page is only ever shared by sequences of one source
            seen.add(s)
    return copies


def _compact_moves(case):
    live = sum(-(-n // case["page"]) for n in _lengths(case))
    ids = _order(case)[:live]
    return sum(i >= live for i in ids), live


def _order(case):
    ids = list(range(case["pool"]))
    random.Random(case["spread"] + 3).shuffle(ids)
    return ids


def work(case):
    if case["op"] == "append":
        n, hd, kv = case["tokens"], case["hd"], case["kv"]
        moved = 2 * case["head"] * hd * 4 + 2 * kv * hd * 4 + kv * (hd + hd // 4) + 2 * kv * hd * 4
        return {"bytes": n * (moved + 8 + (hd * 4 if case["rope"] else 0)), "flops": n * (case["head"] * 3 + kv * 14) * hd}
    if case["op"] == "attend":
        lens, rows = _lengths(case), _rows(case)
        seen = sum(sum(max(0, n - (r - 1 - i)) for i in range(r)) for n, r in zip(lens, rows))
        hd = case["hd"]
        moved = sum(lens) * case["kv"] * (hd + hd // 4) + sum(rows) * case["head"] * (8 * hd + 4)
        return {"bytes": moved, "flops": seen * case["head"] * 4 * hd}
    page = case.get("layers", 0) * case.get("kv", 0) * case.get("page", 0) * (case.get("hd", 0) * 5 // 4)
    if case["op"] == "fork":
        lens, _, want = _fork_request(case)
        entries = sum(-(-n // case["page"]) for n in lens) + sum(-(-n // case["page"]) for n in want)
        return {"bytes": 2 * page * _fork_copies(case) + 4 * entries + 16 * case["seqs"], "flops": 0}
    if case["op"] == "compact":
        moves, live = _compact_moves(case)
        return {"bytes": 2 * page * moves + 8 * live + 4 * case["seqs"], "flops": 0}
    return {"bytes": case["rows"] * (4 * case["vocab"] + 16 + 8 * case["top"]), "flops": case["rows"] * case["vocab"] * 5}


# ---- the page format in plain torch ------------------------------------------


def _tile_bytes(hd):
    return TILE * (hd + hd // 4)


def _quantise(x):
    """x [..., hd] -> numbers [..., group, 32] (uint8), d and m [..., group] (fp16)."""
    g = x.unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1), g.amax(-1)
    d, m = ((hi - lo) * (1.0 / 15.0)).half(), lo.half()
    bad = ~(torch.isfinite(d) & torch.isfinite(m))
    d, m = d.masked_fill(bad, math.nan), m.masked_fill(bad, math.nan)
    n = ((g - m.float().unsqueeze(-1)) / d.float().unsqueeze(-1)).round().clamp(0, 15)
    n = torch.where((d > 0).unsqueeze(-1), n, torch.zeros((), device=x.device))
    return n.to(torch.uint8), d, m


def _values(n, d, m):
    return (n.float() * d.float().unsqueeze(-1) + m.float().unsqueeze(-1)).flatten(-2)


def _pack_tiles(k, v):
    """k, v [..., 16, hd] -> tiles [..., tile bytes]."""
    lead, hd = k.shape[:-2], k.shape[-1]
    g, two = hd // 32, lambda n: n[..., 0::2] | (n[..., 1::2] << 4)
    kn, kd, km = _quantise(k)
    vn, vd, vm = _quantise(v)
    at = len(lead)
    kn = kn.reshape(*lead, 16, g, 4, 8).transpose(at + 1, at + 2)
    vn = vn.reshape(*lead, 4, 2, 2, g, 4, 8).permute(*range(at), at + 1, at + 5, at, at + 2, at + 3, at + 4)
    scales = [torch.stack(s, -1).contiguous().view(torch.uint8).reshape(*lead, -1) for s in ((kd, km), (vd, vm))]
    return torch.cat([two(kn).reshape(*lead, -1), two(vn).reshape(*lead, -1)] + scales, -1)


def _unpack_tiles(tiles, hd):
    """tiles [..., tile bytes] -> k, v [..., 16, hd] fp32."""
    lead, g, at = tiles.shape[:-1], hd // 32, tiles.dim() - 1
    part = 8 * hd
    nib = lambda b: torch.stack((b & 15, b >> 4), -1)  # noqa: E731
    kn = nib(tiles[..., :part]).reshape(*lead, 16, 4, g, 8).transpose(at + 1, at + 2).reshape(*lead, 16, g, 32)
    vn = nib(tiles[..., part:2 * part]).reshape(*lead, 2, 8, 4, 2, g, 4)
    vn = vn.permute(*range(at), at + 2, at, at + 3, at + 4, at + 5, at + 1).reshape(*lead, 16, g, 32)
    s = tiles[..., 2 * part:].contiguous().view(torch.float16).reshape(*lead, 2, 16, g, 2)
    return _values(kn, s[..., 0, :, :, 0], s[..., 0, :, :, 1]), _values(vn, s[..., 1, :, :, 0], s[..., 1, :, :, 1])


# ---- inputs -----------------------------------------------------------------


def _table(case, lens, ids, longest=None):
    """Page table [sequence][slot] (int32), pages given out in the order of `ids`."""
    slots = -(-(longest or max(lens)) // case["page"]) or 1
    table, at = np.full((len(lens), slots), -1, np.int32), 0
    for s, n in enumerate(lens):
        c = -(-n // case["page"])
        table[s, :c] = ids[at:at + c]
        at += c
    return torch.from_numpy(table).cuda()


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _filled_pages(case, count, gen):
    """One layer's pages with keys (some channels far from zero, as keys have them) and values."""
    shape = (count, case["kv"], case["page"] // TILE, TILE, case["hd"])
    bias = torch.randn(case["kv"], 1, 1, case["hd"], device="cuda", generator=gen)
    bias = bias * (torch.rand(bias.shape, device="cuda", generator=gen) < 0.1) * 4
    out = torch.empty((1, *shape[:3], _tile_bytes(case["hd"])), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // math.prod(shape[1:]))
    for a in range(0, count, step):
        n = min(step, count - a)
        k = torch.randn((n, *shape[1:]), device="cuda", generator=gen) + bias
        v = torch.randn((n, *shape[1:]), device="cuda", generator=gen)
        out[0, a:a + n] = _pack_tiles(k, v)
    return out


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed * 7919 + case["spread"])
    s = dict(op=case["op"])
    if case["op"] == "append":
        qd, kd = case["head"] * case["hd"], case["kv"] * case["hd"]
        qkv = torch.randn(case["tokens"], qd + 2 * kd, device="cuda", generator=gen)
        qkv[:, qd:qd + kd] += 2.5 * torch.randn(kd, device="cuda", generator=gen)
        s["q"], s["k"], s["v"] = qkv[:, :qd], qkv[:, qd:qd + kd], qkv[:, qd + kd:]
        parts = _append_tokens(case)
        s["seq"] = _int([i for i, _, n in parts for _ in range(n)])
        s["pos"] = _int([p + j for _, p, n in parts for j in range(n)])
        lens = [p + n for _, p, n in parts]
        pool = sum(-(-n // case["page"]) for n in lens) + 3
        ids = list(range(pool))
        random.Random(case["spread"] + 3).shuffle(ids)
        s["pages"] = torch.zeros((1, pool, case["kv"], case["page"] // TILE, _tile_bytes(case["hd"])),
                                 dtype=torch.uint8, device="cuda")
        s["table"], s["lens"] = _table(case, lens, ids), _int(lens)
        half = case["hd"] // 2
        angle = torch.arange(case["longest"], device="cuda")[:, None] / 500000.0 ** (
            torch.arange(half, device="cuda") / half)
        s["rope"] = torch.stack((angle.cos(), angle.sin()), -1) if case["rope"] else None
    elif case["op"] == "attend":
        lens, rows = _lengths(case), _rows(case)
        pool = sum(-(-n // case["page"]) for n in lens) + 5
        ids = list(range(pool))
        random.Random(case["spread"] + 3).shuffle(ids)
        s["pages"] = _filled_pages(case, pool, gen)
        s["table"], s["lens"] = _table(case, lens, ids), _int(lens)
        s["q"] = 1.5 * torch.randn(sum(rows), case["head"] * case["hd"], device="cuda", generator=gen)
        s["most"], s["hd"] = max(rows), case["hd"]
        s["begin"] = _int(np.concatenate([[0], np.cumsum(rows)]).tolist()) if s["most"] > 1 else None
    elif case["op"] in ("fork", "compact"):
        lens = _fork_request(case)[0] if case["op"] == "fork" else _lengths(case)
        s["pages"] = torch.randint(0, 256, (case["layers"], case["pool"], case["kv"], case["page"] // TILE,
                                            _tile_bytes(case["hd"])), dtype=torch.uint8, device="cuda", generator=gen)
        ids = _order(case)
        if case["op"] == "fork":
            _, source, want = _fork_request(case)
            s["source"], s["want"] = _int(source), _int(want)
            s["table"] = _table(case, lens, ids, max(lens + want))
        else:
            s["table"] = _table(case, lens, ids)
        s["lens"] = _int(lens)
    else:
        x = 2.5 * torch.randn(case["rows"], case["vocab"], device="cuda", generator=gen)
        best = torch.randint(0, case["vocab"], (case["rows"], 6), device="cuda", generator=gen)
        x.scatter_add_(1, best, 9 * torch.rand(best.shape, device="cuda", generator=gen))
        s["tokens"] = best[:, 0].to(torch.int32).contiguous()
        if case["masked"]:  # a grammar allows some of the vocabulary
            x.masked_fill_(torch.rand(x.shape, device="cuda", generator=gen) < 0.3, -math.inf)
            x.scatter_(1, best[:, :1], 4.0)
        s["x"], s["top"] = x, case["top"]
    return s


# ---- plain forms --------------------------------------------------------------


def _plain_rotate(x, heads, hd, cs):
    x = x.unflatten(-1, (heads, hd))
    if cs is None:
        return x
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    x0, x1 = x[..., :hd // 2], x[..., hd // 2:]
    return torch.cat((x0 * c - x1 * s, x0 * s + x1 * c), -1)


def _plain_append(s):
    pages, hd = s["pages"], s["pages"].shape[-1] // 20
    kv, tiles = pages.shape[2], pages.shape[3]
    pos, page_len = s["pos"].long(), tiles * TILE
    cs = None if s["rope"] is None else s["rope"][pos]
    q = _plain_rotate(s["q"], s["q"].shape[1] // hd, hd, cs).flatten(1).contiguous()
    k, v = _plain_rotate(s["k"], kv, hd, cs), s["v"].unflatten(-1, (kv, hd))
    kn, kd, km = _quantise(k)
    vn, vd, vm = _quantise(v)
    g, in_tile = hd // 32, pos % TILE
    two = lambda n: n[..., 0::2] | (n[..., 1::2] << 4)  # noqa: E731
    kb = two(kn.reshape(*kn.shape[:2], g, 4, 8).transpose(2, 3)).flatten(2)
    vb = two(vn.reshape(*vn.shape[:2], g, 4, 8).permute(0, 1, 4, 2, 3)).flatten(2)  # [r][group][c]
    ks, vs = (torch.stack(x, -1).contiguous().view(torch.uint8).flatten(2) for x in ((kd, km), (vd, vm)))
    page = s["table"][s["seq"].long(), pos // page_len].long()
    tile = ((page[:, None] * kv + torch.arange(kv, device=pos.device)) * tiles + (pos % page_len // TILE)[:, None])
    base = (tile * pages.shape[-1])[..., None]
    byte = lambda n: torch.arange(n, device=pos.device)  # noqa: E731
    each = hd // 16  # bytes of one position in one of V's eight columns r
    r, b = byte(hd // 2) // each, byte(hd // 2) % each
    at = in_tile[:, None, None]
    v_at = ((at % 4 // 2 * 8 + r) * 4 + at // 4) * 2 * each + at % 2 * each + b
    flat = pages.view(-1)
    flat[base + at * (hd // 2) + byte(hd // 2)] = kb
    flat[base + 8 * hd + v_at] = vb
    flat[base + 16 * hd + at * (hd // 8) + byte(hd // 8)] = ks
    flat[base + 18 * hd + at * (hd // 8) + byte(hd // 8)] = vs
    return {"q": q, "k": _values(kn, kd, km).flatten(1), "v": _values(vn, vd, vm).flatten(1)}


def _plain_attend(s):
    pages, hd, q = s["pages"], s["hd"], s["q"]
    seqs, slots = s["table"].shape
    kv, rep, most = pages.shape[2], q.shape[1] // hd // pages.shape[2], s["most"]
    k, v = _unpack_tiles(pages[0][s["table"].clamp(min=0).long()], hd)
    k, v = (x.transpose(1, 2).reshape(seqs, kv, -1, hd) for x in (k, v))
    begin = torch.arange(seqs + 1, device=q.device) if s["begin"] is None else s["begin"].long()
    count = begin[1:] - begin[:-1]
    row = torch.arange(most, device=q.device)
    qs = q[(begin[:-1, None] + row).clamp(max=q.shape[0] - 1)]
    qs = qs.reshape(seqs, most, kv, rep, hd).permute(0, 2, 1, 3, 4).reshape(seqs, kv, most * rep, hd)
    x = torch.matmul(qs, k.transpose(2, 3)).mul_(1.0 / math.sqrt(hd))
    sees = s["lens"].long()[:, None] - (count[:, None] - 1 - row)
    sees = sees.repeat_interleave(rep, 1)[:, None, :, None]
    x.masked_fill_(torch.arange(k.shape[2], device=q.device) >= sees, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = x.sub_(top.clamp(min=-3e38)).exp_()
    l = e.sum(-1, keepdim=True)  # noqa: E741
    o = torch.matmul(e, v) / l.clamp(min=1e-30)
    lse = torch.where(l > 0, top + l.log(), top)
    token = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(begin, token, right=True) - 1
    at = token - begin[seq]
    o = o.reshape(seqs, kv, most, rep, hd).transpose(1, 2)[seq, at]
    lse = lse.reshape(seqs, kv, most, rep).transpose(1, 2)[seq, at]
    return {"o": o.reshape(q.shape), "lse": lse.reshape(q.shape[0], -1)}


def _kth_free(used):
    """Ids of the free pages, lowest first (as many as there are pages; the rest is not used), and their number."""
    free = ~used
    rank = free.cumsum(0)
    ids = torch.zeros(used.shape[0] + 1, dtype=torch.long, device=used.device)
    ids[torch.where(free, rank - 1, used.shape[0])] = torch.arange(used.shape[0], device=used.device)
    return ids, rank[-1]


def _plain_fork(s):
    pages, table, source, want = s["pages"], s["table"].long(), s["source"].long(), s["want"].long()
    seqs, slots = table.shape
    pool, page_len = pages.shape[1], pages.shape[3] * TILE
    me, col = torch.arange(seqs, device=table.device), torch.arange(slots, device=table.device)
    rows = table[source.clamp(min=0)]
    kept = torch.where(source >= 0, torch.minimum(s["lens"].long()[source.clamp(min=0)].clamp(min=0), want), 0)
    whole, part, goal = kept // page_len, kept % page_len > 0, -(-want // page_len)
    shared = torch.zeros(pool + 1, dtype=torch.bool, device=table.device)
    shared[torch.where(col < whole[:, None], rows, pool)] = True
    last = torch.where(part, rows.gather(1, whole.clamp(max=slots - 1)[:, None])[:, 0], pool)
    owner = torch.full((pool + 1,), seqs, device=table.device).scatter_reduce(0, last, me, "amin")
    keeps = part & ~shared[last] & (owner[last] == me)
    ids, room = _kth_free((shared | (owner < seqs))[:pool])
    held = whole + keeps
    need = goal - held
    first = need.cumsum(0) - need
    ok = (first + need <= room) & (goal <= slots)
    given = ids[(first[:, None] + col - held[:, None]).clamp(0, pool)]
    new = torch.where(col < held[:, None], rows, torch.where(col < goal[:, None], given, -1))
    new = torch.where(ok[:, None], new, -1)
    at = (part & ~keeps & ok).nonzero()[:, 0]
    pages[:, new[at, whole[at]]] = pages[:, last[at]]
    return {"table": new.int(), "lens": torch.where(ok, want, -1).int(), "pages": pages}


def _plain_compact(s):
    pages, table = s["pages"], s["table"].long()
    pool, page_len = pages.shape[1], pages.shape[3] * TILE
    live = torch.arange(table.shape[1], device=table.device) < -(-s["lens"].long() // page_len)[:, None]
    used = torch.zeros(pool + 1, dtype=torch.bool, device=table.device)
    used[torch.where(live, table, pool)] = True
    used = used[:pool]
    count = used.sum()
    at = torch.arange(pool, device=table.device)
    source, hole = (used & (at >= count)).nonzero()[:, 0], (~used & (at < count)).nonzero()[:, 0]
    at[source] = hole
    pages[:, hole] = pages[:, source]
    return {"table": torch.where(live, at[table.clamp(min=0)], -1).int(), "live": count.int().reshape(1), "pages": pages}


def _plain_score(s):
    x, t, top = s["x"], s["tokens"].long()[:, None], s["top"]
    m = x.amax(-1, keepdim=True)
    c = x - m
    e = c.exp()
    l = e.sum(-1, keepdim=True)  # noqa: E741
    xt = x.gather(1, t)
    at = torch.arange(x.shape[1], device=x.device)
    rank = (x > xt).sum(-1) + ((x == xt) & (at < t)).sum(-1)
    h = l.log() - torch.where(e > 0, e * c, 0).sum(-1, keepdim=True) / l
    out = {"logprob": ((xt - m) - l.log())[:, 0], "entropy": h[:, 0], "rank": rank.int()}
    if top:  # an order of (value, lower index first) in one whole number
        bits = x.view(torch.int32).long()
        key = (torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) << 32) | (0x7FFFFFFF - at)
        ids = 0x7FFFFFFF - (key.topk(top, -1).values & 0x7FFFFFFF)
        out["ids"], out["logprobs"] = ids.int(), (x.gather(1, ids) - m) - l.log()
    return out


_PLAIN = dict(append=_plain_append, attend=_plain_attend, fork=_plain_fork, compact=_plain_compact, score=_plain_score)


# ---- the framework's ------------------------------------------------------------


def _own(s):
    if s["op"] == "score":
        from cllm_inference_b200.scoring import token_scores

        r = token_scores(s["x"], s["tokens"], s["top"])
        out = {"logprob": r.logprob, "entropy": r.entropy, "rank": r.rank}
        return {**out, "ids": r.top_ids, "logprobs": r.top_logprobs} if s["top"] else out
    from cllm_inference_b200.kv4 import KV4Cache

    cache = KV4Cache(s["pages"], s["table"], s["lens"])
    if s["op"] == "append":
        q, k, v = cache.append(0, s["k"], s["v"], s["seq"], s["pos"], q=s["q"], rope=s["rope"], values=True)
        return {"q": q, "k": k, "v": v}
    if s["op"] == "attend":
        o, lse = cache.attention(0, s["q"], begin=s["begin"], lse=True)
        return {"o": o, "lse": lse}
    if s["op"] == "fork":
        new = cache.fork(s["source"], s["want"])
        return {"table": new.table, "lens": new.lens, "pages": new.pages}
    new, live = cache.compact()
    return {"table": new.table, "live": live, "pages": new.pages}


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# ---- the definitions in 64 bits ---------------------------------------------------


def _exact_vector(tile, p, hd, which):
    """Position p of the tiles [..., tile bytes] in float64: which = 0 the key, 1 the value."""
    i = torch.arange(hd, device=tile.device)
    g, j = i // 32, i % 32
    if which == 0:
        nibble = ((p * 4 + j // 8) * (hd // 32) + g) * 8 + j % 8
    else:
        nibble = ((((p % 4 // 2 * 8 + j % 8) * 4 + p // 4) * 2 + p % 2) * (hd // 32) + g) * 4 + j // 8
    byte = tile[..., 8 * hd * which + nibble // 2].long()
    n = torch.where(nibble % 2 == 1, byte // 16, byte % 16).double()
    at = 16 * hd + 2 * hd * which + (p * (hd // 32) + g) * 4
    half = lambda o: (tile[..., at + o].short() | (tile[..., at + o + 1].short() << 8)).view(torch.float16).double()  # noqa: E731
    return half(0) * n + half(2)


def _exact_attend(case, s):
    hd, page_len = case["hd"], case["page"]
    lens, rows = _lengths(case), _rows(case)
    out, lses, at = [], [], 0
    for i, (n, r) in enumerate(zip(lens, rows)):
        tiles = s["pages"][0][s["table"][i, : -(-n // page_len)].long()]  # [page, kv, tile, bytes]
        k, v = (torch.stack([_exact_vector(tiles, p, hd, w) for p in range(TILE)], 3) for w in (0, 1))
        k, v = (x.transpose(0, 1).reshape(case["kv"], -1, hd)[:, :n] for x in (k, v))
        q = s["q"][at:at + r].double().reshape(r, case["kv"], -1, hd)
        for a in range(0, r, 64):  # some rows at a time
            b = min(r, a + 64)
            x = torch.einsum("rkhd,kpd->rkhp", q[a:b], k) / math.sqrt(hd)
            sees = n - (r - 1 - torch.arange(a, b, device=x.device))
            x.masked_fill_((torch.arange(n, device=x.device)[None] >= sees[:, None])[:, None, None], -math.inf)
            w = torch.logsumexp(x, -1)
            out.append(torch.einsum("rkhp,kpd->rkhd", torch.softmax(x, -1), v).reshape(b - a, -1))
            lses.append(w.reshape(b - a, -1))
        at += r
    return {"o": torch.cat(out), "lse": torch.cat(lses)}


def _exact_append(case, s):
    hd = case["hd"]
    out = {}
    for name, heads in (("q", case["head"]), ("k", case["kv"]), ("v", case["kv"])):
        x = s[name].double().reshape(-1, heads, hd)
        if s["rope"] is not None and name != "v":
            cs = torch.view_as_complex(s["rope"][s["pos"].long()].double())[:, None]
            z = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * cs
            x = torch.cat((z.real, z.imag), -1)
        if name != "q":
            x = x.reshape(-1, heads, hd // 32, 32)
            low = x.min(-1, keepdim=True).values
            d, m = ((x.max(-1, keepdim=True).values - low) / 15).half().double(), low.half().double()
            x = torch.where(d > 0, ((x - m) / d).round().clamp(0, 15), 0) * d + m
        out[name] = x.reshape(x.shape[0], -1)
    return out


def _exact_score(case, s):
    x = s["x"].double()
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    out = {"logprob": lp.gather(1, s["tokens"].long()[:, None])[:, 0],
           "entropy": -torch.where(p > 0, p * lp, 0).sum(-1), "rank": None}
    if case["top"]:
        out["ids"], out["logprobs"] = None, lp.sort(-1, descending=True).values[:, :case["top"]]
    return out


def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # whole numbers only
    s = prepare(case, seed)
    return dict(append=_exact_append, attend=_exact_attend, score=_exact_score)[case["op"]](case, s)
