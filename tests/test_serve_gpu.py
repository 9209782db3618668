"""The serving operators (kv4.py, scoring.py) on a GPU against plain numpy
restatements (serve_oracle.py).

Tolerances.  What append stores and every page table are whole numbers and
equal bit for bit.  Attention is compared with float64 on the same stored
numbers, within the bound that serve_oracle.attention derives for fp32
arithmetic.  Scores: sums of up to 2^18 terms in partial sums, off by at most
2^-17 of their magnitude."""
import ctypes

import numpy as np
import pytest
import torch

from cllm_inference_b200 import _lib
from tests import serve_oracle as O

pytestmark = pytest.mark.gpu


def _cache(rng, layers, pages, page_len, kv, hd, lens, max_pages, fill=None):
    """A cache with random contents, pages handed out in random order; unused table entries hold rubbish ids."""
    from cllm_inference_b200.kv4 import KV4Cache

    p = rng.integers(0, 256, (layers, pages, kv, page_len // 16, 20 * hd), dtype=np.uint8)
    s = rng.uniform(0.01, 0.3, (*p.shape[:4], 2, 16, hd // 32, 2)).astype(np.float16)
    s[..., 1] = rng.standard_normal(s.shape[:-1]).astype(np.float16)
    p[..., 16 * hd:] = s.reshape(*p.shape[:4], -1).view(np.uint8)
    ids = rng.permutation(pages)
    table = rng.integers(-5, 10 ** 9, (len(lens), max_pages)).astype(np.int32)
    at = 0
    for i, n in enumerate(lens):
        c = -(-max(0, n) // page_len)
        table[i, :c] = ids[at:at + c]
        at += c
    if fill is not None:  # rubbish where no position lives: unused pages, and the tail of each last page
        p[:, ids[at:]] = fill
        for i, n in enumerate(lens):
            if n > 0:
                _rubbish_tail(p[:, table[i, (n - 1) // page_len]], (n - 1) % page_len + 1, hd, fill)
    c = KV4Cache(torch.from_numpy(p).cuda(), torch.from_numpy(table).cuda(),
                 torch.tensor(lens, dtype=torch.int32, device="cuda"))
    return c, p, table


def _rubbish_tail(page, first, hd, fill):
    """Scales (so: NaN) of the positions from `first` of a page [layer, kv, tiles, bytes]."""
    for pos in range(first, page.shape[2] * 16):
        t, r = pos // 16, pos % 16
        for o in (16 * hd, 18 * hd):
            page[:, :, t, o + r * hd // 8:o + (r + 1) * hd // 8] = fill


def _rope(rng, n_pos, hd):
    a = rng.uniform(0, 6.3, (n_pos, hd // 2)).astype(np.float32)
    return np.stack([np.cos(a), np.sin(a)], -1)


# ---- append -------------------------------------------------------------------


@pytest.mark.parametrize("hd,page_len,heads,kv,n,pad,rope", [
    (128, 64, 32, 8, 1, 0, True), (128, 16, 8, 8, 33, 4, True), (64, 32, 4, 2, 50, 0, True),
    (64, 48, 3, 1, 7, 1, False), (128, 128, 0, 2, 19, 3, True), (64, 16, 7, 7, 130, 0, True)])
def test_append_stores_the_formula_bit_for_bit(cuda, lib, hd, page_len, heads, kv, n, pad, rope):
    rng = np.random.default_rng(n + hd)
    lens = [40, 1, 300]
    cache, pages, table = _cache(rng, 2, 60, page_len, kv, hd, lens, -(-300 // page_len) + 1)
    width = (heads + 2 * kv) * hd
    x = rng.standard_normal((n, width + pad)).astype(np.float32) * 3
    kcol = heads * hd
    x[0, kcol:kcol + 32] = 1.25                      # a constant group
    x[n // 2, kcol:kcol + 32] = 1e-7 * np.arange(32)  # a scale below fp16's normal range
    x[n - 1, kcol + 5] = np.nan
    x[n - 1, kcol + kv * hd + 40] = np.inf
    x[n // 2, kcol + kv * hd:kcol + kv * hd + 32] = 1e6  # outside fp16
    seq = rng.integers(0, 3, n).astype(np.int32)
    pos = np.zeros(n, np.int32)
    for s in range(3):
        at = np.nonzero(seq == s)[0]
        pos[at] = rng.permutation(max(lens[s], at.size))[:at.size] if at.size <= lens[s] else np.arange(at.size)
    for s in range(3):  # room for every position
        c = -(-int(pos[seq == s].max(initial=0) + 1) // page_len)
        table[s, :c] = np.where((table[s, :c] >= 0) & (table[s, :c] < 60), table[s, :c], 0)
    used = {}
    for s in range(3):  # positions of different sequences must not share a page here
        for i in range(-(-int(pos[seq == s].max(initial=0) + 1) // page_len)):
            while table[s, i] in used and used[table[s, i]] != (s, i):
                table[s, i] = (table[s, i] + 1) % 60
            used[table[s, i]] = (s, i)
    if n > 4:
        seq[3] = -1  # padding
    cache.table.copy_(torch.from_numpy(table))
    cs = _rope(rng, 320, hd) if rope else None
    xd = torch.from_numpy(x).cuda()
    q = xd[:, :heads * hd] if heads else None
    got = cache.append(1, xd[:, kcol:kcol + kv * hd], xd[:, kcol + kv * hd:width], torch.from_numpy(seq).cuda(),
                       torch.from_numpy(pos).cuda(), q=q, rope=None if cs is None else torch.from_numpy(cs).cuda(),
                       values=True)
    want = pages.copy()
    for t in range(n):
        k = x[t, kcol:kcol + kv * hd].reshape(kv, hd)
        v = x[t, kcol + kv * hd:width].reshape(kv, hd)
        qq = x[t, :heads * hd].reshape(heads, hd)
        with np.errstate(all="ignore"):
            if cs is not None:
                k, qq = O.rotate(k, cs[pos[t]]), O.rotate(qq, cs[pos[t]])
        kv_want = [O.values(*O.quantise(z)).reshape(-1) for z in (k, v)]
        if seq[t] < 0:
            kv_want, qq = [np.zeros(kv * hd)] * 2, np.zeros((heads, hd))
        else:
            for h in range(kv):
                O.write_position(want[1, table[seq[t], pos[t] // page_len], h, pos[t] % page_len // 16], pos[t] % 16,
                                 k[h], v[h])
        if heads:
            np.testing.assert_array_equal(got[0][t].cpu().numpy(), qq.reshape(-1))
        np.testing.assert_array_equal(got[1][t].cpu().numpy(), kv_want[0])
        np.testing.assert_array_equal(got[2][t].cpu().numpy(), kv_want[1])
    have = cache.pages.cpu().numpy()
    # NaN scales: any NaN pattern
    s, w = have[..., 16 * hd:].view(np.float16), want[..., 16 * hd:].view(np.float16)
    np.testing.assert_array_equal(np.isnan(s), np.isnan(w))
    np.testing.assert_array_equal(np.where(np.isnan(s), 0, s), np.where(np.isnan(w), 0, w))
    np.testing.assert_array_equal(have[..., :16 * hd], want[..., :16 * hd])
    _lib.check(lib.cllm_cuda_check_device_status())


def test_append_never_follows_a_bad_page_or_position(cuda, lib):
    rng = np.random.default_rng(3)
    cache, pages, table = _cache(rng, 1, 8, 16, 2, 64, [20, 20], 2)
    x = torch.randn(4, 2 * 64, device="cuda")
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cache.table[1, 1] = 8  # outside the pool
    for seq, pos in ((ints(0, 1, 0, 0), ints(0, 17, 1, 2)), (ints(2, 0, 0, 0), ints(0, 3, 4, 5)),
                     (ints(0, 0, 0, 0), ints(32, 6, 7, 8)), (ints(0, 0, 0, 0), ints(-1, 9, 10, 11))):
        _, k, _ = cache.append(0, x, x, seq, pos, values=True)
        bad = 1 if int(seq[1]) == 1 else 0
        assert (k[bad] == 0).all() and (k[3] != 0).any()
        assert lib.cllm_cuda_check_device_status() == _lib.ERR_INVALID_ARG
        assert "page table" in _lib.last_error()
    _lib.check(lib.cllm_cuda_check_device_status())  # cleared
    np.testing.assert_array_equal(cache.pages.cpu().numpy()[0, table[1, 0]], pages[0, table[1, 0]])


# ---- attention ------------------------------------------------------------------


def _attend(cache, layer, q, begin, hd, scale=0.0):
    dev_begin = None if begin is None else torch.tensor(begin, dtype=torch.int32, device="cuda")
    o, lse = cache.attention(layer, q, begin=dev_begin, scale=scale, lse=True)
    torch.cuda.synchronize()
    b = list(range(cache.n_seqs + 1)) if begin is None else begin
    want, wl, tol, tol_l = O.attention(q.cpu().numpy(), b, cache.pages[layer].cpu().numpy(), cache.table.cpu().numpy(),
                                       cache.lens.cpu().numpy(), hd, scale or 1 / np.sqrt(hd))
    o, lse = o.cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)
    err = np.abs(o - want).reshape(*tol.shape, hd).max(-1)
    assert not np.isnan(o).any()
    assert (err <= tol + 1e-30).all(), f"worst {np.max(err / (tol + 1e-30)):.3g} of the tolerance"
    none = np.isneginf(wl)
    np.testing.assert_array_equal(np.isneginf(lse), none)
    assert (np.abs(lse[~none] - wl[~none]) <= tol_l[~none]).all()
    return o


EDGE_LENS = [0, 1, 15, 16, 17, 63, 64, 65, 200, -3, 31, 1000]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rep,kv,page_len", [(1, 4, 16), (2, 2, 32), (3, 1, 48), (4, 2, 64), (5, 1, 64), (7, 2, 128),
                                             (8, 1, 64), (12, 1, 32), (16, 1, 64)])
def test_attention_one_row(cuda, lib, hd, rep, kv, page_len):
    rng = np.random.default_rng(rep * 100 + hd)
    cache, _, _ = _cache(rng, 2, 140, page_len, kv, hd, EDGE_LENS, -(-1000 // page_len) + 2, fill=0xFF)
    q = torch.from_numpy(rng.standard_normal((len(EDGE_LENS), rep * kv * hd)).astype(np.float32) * 2).cuda()
    o = _attend(cache, 1, q, None, hd)
    assert (o[0] == 0).all() and (o[9] == 0).all()  # a sequence of no positions
    _lib.check(lib.cllm_cuda_check_device_status())


@pytest.mark.parametrize("hd,rep,kv,page_len,counts", [
    (128, 4, 2, 64, [1, 0, 3, 2, 16, 1, 5, 7, 4, 1, 2, 9]),    # some rows each
    (64, 1, 3, 32, [1, 4, 15, 20, 17, 1, 64, 70, 33, 2, 0, 3]),
    (128, 8, 1, 16, [3, 2, 1, 1, 1, 8, 0, 0, 2, 2, 2, 130]),
    (64, 3, 2, 48, [0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 45]),
    (128, 4, 1, 64, [0, 1, 15, 16, 17, 63, 64, 65, 200, 0, 31, 300]),  # whole prompts
    (64, 8, 2, 128, [0, 1, 15, 16, 17, 63, 64, 65, 200, 0, 31, 129]),
    (128, 1, 2, 32, [0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 400]),
])
def test_attention_many_rows(cuda, lib, hd, rep, kv, page_len, counts):
    rng = np.random.default_rng(sum(counts) + hd)
    cache, _, _ = _cache(rng, 1, 140, page_len, kv, hd, EDGE_LENS, -(-1000 // page_len), fill=0xFF)
    begin = np.concatenate([[0], np.cumsum(counts)]).tolist()
    heads = rep * kv
    x = rng.standard_normal((begin[-1] + 3, heads * hd + 8)).astype(np.float32) * 2  # rows of no sequence, strided
    q = torch.from_numpy(x).cuda()[:, 4:4 + heads * hd]
    o = _attend(cache, 0, q, begin, hd)
    assert (o[begin[-1]:] == 0).all()
    # a first row that does not start at 0
    shifted = [b + 2 for b in begin]
    shifted[0] = 2
    o = _attend(cache, 0, q, shifted, hd)
    assert (o[:2] == 0).all()
    _lib.check(lib.cllm_cuda_check_device_status())


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_extremes(cuda, lib, rows):
    """Large and tiny queries and scales of the cache, a scale of the caller's, equal scores."""
    hd, kv, rep = 128, 2, 4
    rng = np.random.default_rng(rows)
    for q_size, k_size, v_size, scale in ((30.0, 1, 1, 0.0), (1e-6, 1, 1, 0.0), (0.0, 1, 1, 0.0), (1.0, 1, 2000.0, 0.0),
                                          (1.0, 1, 1e-4, 0.0), (1e4, 1e-3, 1, 0.3), (1.0, 1.0, 1.0, -0.5)):
        cache, p, table = _cache(rng, 1, 30, 64, kv, hd, [700, 45], 12)
        s = p[..., 16 * hd:].view(np.float16).reshape(*p.shape[:4], 2, -1)
        s[..., 0, :] *= np.float16(k_size)
        s[..., 1, :] = (s[..., 1, :].astype(np.float32) * v_size).astype(np.float16)
        cache.pages.copy_(torch.from_numpy(p))
        q = torch.from_numpy((rng.standard_normal((2 * rows, kv * rep * hd)) * q_size).astype(np.float32)).cuda()
        _attend(cache, 0, q, [0, rows, 2 * rows], hd, scale)


@pytest.mark.parametrize("rows", [1, 64])
def test_attention_values_that_cancel(cuda, lib, rows):
    """A group of zero scale (all numbers equal), and a page shared by two sequences."""
    hd, kv, rep = 64, 1, 2
    rng = np.random.default_rng(5)
    cache, p, table = _cache(rng, 1, 9, 32, kv, hd, [100, 90], 4)
    s = p[..., 16 * hd:].view(np.float16).reshape(*p.shape[:4], 2, 16, hd // 32, 2)
    s[..., 0, 0] = 0
    cache.pages.copy_(torch.from_numpy(p))
    table[1, :2] = table[0, :2]
    cache.table.copy_(torch.from_numpy(table))
    q = torch.from_numpy(rng.standard_normal((2 * rows, rep * hd)).astype(np.float32)).cuda()
    _attend(cache, 0, q, [0, rows, 2 * rows], hd)


@pytest.mark.parametrize("rows", [1, 50])
def test_attention_a_nan_stays_with_the_rows_that_see_it(cuda, lib, rows):
    hd, page_len = 128, 64
    rng = np.random.default_rng(6)
    cache, p, table = _cache(rng, 1, 12, page_len, 2, hd, [200, 210], 4)
    at = p[0, table[0, 180 // page_len], 0, 180 % page_len // 16]
    at[16 * hd + (180 % 16) * hd // 8:][:hd // 8] = 0xFF  # key of position 180, head 0, sequence 0
    cache.pages.copy_(torch.from_numpy(p))
    q = torch.from_numpy(rng.standard_normal((2 * rows, 4 * hd)).astype(np.float32)).cuda()
    begin = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device="cuda")
    o = cache.attention(0, q, begin=begin).cpu().numpy().reshape(2, rows, 2, 2 * hd)
    sees = 200 - (rows - 1 - np.arange(rows)) > 180
    assert np.isnan(o[0, sees, 0]).all()
    assert not np.isnan(o[0, ~sees]).any() and not np.isnan(o[0, :, 1]).any() and not np.isnan(o[1]).any()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [1, 3, 50])
def test_attention_a_nan_of_the_values_stays_in_its_group(cuda, lib, rows, hd):
    rng = np.random.default_rng(rows + hd)
    cache, p, table = _cache(rng, 1, 12, 64, 2, hd, [200, 210], 4)
    g = hd // 32 - 1
    at = p[0, table[0, 190 // 64], 1, 190 % 64 // 16]
    o = 18 * hd + (190 % 16) * hd // 8 + 4 * g
    at[o:o + 4] = 0xFF  # value of position 190, head 1, last group, sequence 0
    cache.pages.copy_(torch.from_numpy(p))
    q = torch.from_numpy(rng.standard_normal((2 * rows, 4 * hd)).astype(np.float32)).cuda()
    begin = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device="cuda")
    got = cache.attention(0, q, begin=begin).cpu().numpy().reshape(2, rows, 2, 2, hd // 32, 32)
    sees = 200 - (rows - 1 - np.arange(rows)) > 190
    assert np.isnan(got[0, sees, 1, :, g]).all()
    got[0, sees, 1, :, g] = 0
    assert not np.isnan(got).any()


def test_attention_lengths_beyond_the_table_and_bad_pages(cuda, lib):
    hd = 64
    rng = np.random.default_rng(7)
    cache, p, table = _cache(rng, 1, 6, 16, 1, hd, [30, 30], 2)
    q = torch.randn(2, hd, device="cuda")
    cache.lens[0] = 2 ** 31 - 1  # more than two pages: only those are read
    o = cache.attention(0, q)
    assert torch.isfinite(o).all()
    assert lib.cllm_cuda_check_device_status() == _lib.ERR_INVALID_ARG
    cache.lens[0] = 30
    cache.table[0, 1] = 2 ** 30
    cache.attention(0, q)
    assert lib.cllm_cuda_check_device_status() == _lib.ERR_INVALID_ARG
    many = torch.randn(60, hd, device="cuda")
    cache.attention(0, many, begin=torch.tensor([0, 30, 60], dtype=torch.int32, device="cuda"))
    assert lib.cllm_cuda_check_device_status() == _lib.ERR_INVALID_ARG
    _lib.check(lib.cllm_cuda_check_device_status())


def test_attention_a_long_cache_and_offsets_past_32_bits(cuda, lib):
    """40000 positions in the last pages of a pool of 5.4 GB."""
    from cllm_inference_b200.kv4 import KV4Cache

    hd, kv, page_len, n = 128, 8, 64, 40000
    slots = -(-n // page_len)
    pool = 66000
    cache = KV4Cache.empty(1, pool, page_len, kv, hd, 1, slots)
    assert cache.pages.numel() > 2 ** 32
    rng = np.random.default_rng(8)
    small, p, _ = _cache(rng, 1, slots, page_len, kv, hd, [n], slots)
    ids = pool - 1 - torch.randperm(slots, device="cuda")
    cache.pages[0, ids] = small.pages[0]
    cache.table[0] = ids.int()
    cache.lens[0] = n
    q = torch.randn(1, 8 * kv * hd, device="cuda")
    small.table[0] = torch.arange(slots, device="cuda").int()
    a, b = cache.attention(0, q), small.attention(0, q)
    assert torch.equal(a, b)
    q = torch.randn(70, 2 * kv * hd, device="cuda")
    begin = torch.tensor([0, 70], dtype=torch.int32, device="cuda")
    a, b = cache.attention(0, q, begin=begin), small.attention(0, q, begin=begin)
    assert torch.equal(a, b)
    k, v = O.sequence(p[0], np.arange(slots), n, hd)
    sees = n - 69
    x = np.einsum("hpd,hrd->hrp", k[:, :sees], q[0].cpu().numpy().reshape(kv, 2, hd).astype(np.float64)) / np.sqrt(hd)
    w = np.exp(x - x.max(-1, keepdims=True))
    want = np.einsum("hrp,hpd->hrd", w / w.sum(-1, keepdims=True), v[:, :sees])
    np.testing.assert_allclose(a[0].cpu().numpy().reshape(want.shape), want, atol=2.0 ** -16 * np.abs(v).max(), rtol=0)


# The same in calls that are long enough for whole prompts to be worth 128 rows at a time.


@pytest.mark.parametrize("hd,rep,kv,page_len,counts", [
    (128, 4, 4, 64, [0, 1, 15, 16, 17, 63, 64, 65, 200, 0, 31, 300]),
    (64, 8, 3, 128, [0, 1, 15, 16, 17, 63, 64, 65, 200, 0, 31, 200]),
    (128, 1, 16, 32, [0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 300]),
    (64, 3, 12, 48, [0, 0, 0, 0, 0, 0, 0, 41, 0, 0, 0, 130]),
    (128, 16, 3, 16, [3, 2, 1, 1, 1, 8, 0, 0, 2, 2, 2, 130]),
    (64, 1, 40, 64, [0, 0, 0, 0, 0, 0, 0, 0, 129, 0, 0, 128]),
])
def test_attention_prompts(cuda, lib, hd, rep, kv, page_len, counts):
    test_attention_many_rows(cuda, lib, hd, rep, kv, page_len, counts)


def test_attention_prompts_extremes(cuda, lib):
    test_attention_extremes(cuda, lib, 700)
    test_attention_values_that_cancel(cuda, lib, 8100)


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_prompts_a_nan(cuda, lib, hd):
    if hd == 128:
        test_attention_a_nan_stays_with_the_rows_that_see_it(cuda, lib, 2100)
    test_attention_a_nan_of_the_values_stays_in_its_group(cuda, lib, 2100, hd)


def test_attention_prompts_bad_pages_and_repeatable(cuda, lib):
    rng = np.random.default_rng(11)
    cache, p, table = _cache(rng, 1, 30, 16, 2, 64, [130, 250], 18)
    q = torch.randn(9000, 6 * 64, device="cuda")
    begin = torch.tensor([0, 4000, 9000], dtype=torch.int32, device="cuda")
    o = cache.attention(0, q, begin=begin)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = cache.attention(0, q, begin=begin)
    for _ in range(3):
        graph.replay()
        assert torch.equal(cache.attention(0, q, begin=begin), o) and torch.equal(again, o)
    _lib.check(lib.cllm_cuda_check_device_status())
    cache.table[0, 1] = 2 ** 30
    got = cache.attention(0, q, begin=begin)
    assert lib.cllm_cuda_check_device_status() == _lib.ERR_INVALID_ARG
    assert torch.equal(got[4000:], o[4000:])


@pytest.mark.parametrize("rows", [20, 41, 60, 61, 100])
def test_attention_either_kernel_at_the_border(cuda, lib, rows):
    """Calls of about as many rows and steps as the rule between the kernels looks at, in a wide and a tight table."""
    rng = np.random.default_rng(rows)
    for slots in (16, 400):
        cache, _, _ = _cache(rng, 1, 40, 64, 8, 64, [1000, 300, 1000], slots)
        q = torch.from_numpy(rng.standard_normal((2 * rows + 3, 16 * 64)).astype(np.float32)).cuda()
        _attend(cache, 0, q, [0, rows, rows + 3, 2 * rows + 3], 64)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [1, 45])
def test_attention_parts_of_one_item_in_many_ctas(cuda, lib, rows, hd):
    """One KV head and a long sequence: every CTA has a part of the same rows; the next calls find the counts cleared."""
    rng = np.random.default_rng(rows * hd)
    cache, _, _ = _cache(rng, 1, 940, 64, 1, hd, [60000, 33], 938)
    q = torch.from_numpy(rng.standard_normal((2 * rows, 3 * hd)).astype(np.float32)).cuda()
    begin = [0, rows, 2 * rows]
    o = _attend(cache, 0, q, begin, hd)
    short, _, _ = _cache(rng, 1, 9, 64, 1, hd, [130, 300], 5)
    for _ in range(2):
        _attend(short, 0, q, begin, hd)
        again = cache.attention(0, q, begin=torch.tensor(begin, dtype=torch.int32, device="cuda"))
        assert np.array_equal(again.cpu().numpy(), o.astype(np.float32))
    _lib.check(lib.cllm_cuda_check_device_status())


def test_attention_is_repeatable_on_another_stream_and_in_a_graph(cuda, lib):
    hd = 128
    rng = np.random.default_rng(9)
    lens = rng.integers(1, 900, 20).tolist()
    cache, _, _ = _cache(rng, 1, 340, 64, 2, hd, lens, 15)
    q = torch.randn(20, 8 * hd, device="cuda")
    rows = torch.randn(100, 8 * hd, device="cuda")
    begin = torch.arange(0, 101, 5, dtype=torch.int32, device="cuda")
    first, many = cache.attention(0, q), cache.attention(0, rows, begin=begin)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(5):
            assert torch.equal(cache.attention(0, q), first)
            assert torch.equal(cache.attention(0, rows, begin=begin), many)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, m = cache.attention(0, q), cache.attention(0, rows, begin=begin)
    cache.lens += 1  # the graph reads the lengths when it runs
    cache.lens.clamp_(max=900)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, cache.attention(0, q)) and torch.equal(m, cache.attention(0, rows, begin=begin))


# ---- pages ------------------------------------------------------------------------


@pytest.mark.parametrize("seed", range(12))
def test_fork_and_compact_follow_the_rules(cuda, lib, seed):
    rng = np.random.default_rng(seed)
    page_len, hd, kv = int(rng.choice([16, 32, 48, 64])), int(rng.choice([64, 128])), int(rng.choice([1, 3]))
    n_old, layers = int(rng.integers(1, 40)), int(rng.integers(1, 4))
    slots = int(rng.integers(1, 9))
    lens = rng.integers(-1, slots * page_len + 1, n_old)
    lens[rng.random(n_old) < 0.3] //= page_len
    lens[rng.random(n_old) < 0.2] *= page_len
    lens = np.minimum(lens, slots * page_len).astype(np.int32)
    need = int(sum(-(-max(0, int(n)) // page_len) for n in lens))
    pool = need + int(rng.integers(0, 30)) + 1
    cache, _, table = _cache(rng, layers, pool, page_len, kv, hd, lens.tolist(), slots)
    for step in range(3):
        n_new = int(rng.integers(1, 40))
        source = rng.integers(-1, table.shape[0], n_new).astype(np.int32)
        if step == 2:
            source[rng.random(n_new) < 0.2] = table.shape[0] + 7  # there is no such sequence
        base = np.where((source >= 0) & (source < table.shape[0]), lens[np.clip(source, 0, table.shape[0] - 1)], 0)
        new_len = (np.maximum(base, 0) + rng.integers(-page_len, 2 * page_len, n_new)).astype(np.int32)
        want_t, want_l, copies = O.fork(table, lens, source, new_len, pool, page_len)
        pages = cache.pages.cpu().numpy()
        for a, b in copies:
            pages[:, b] = pages[:, a]
        new = cache.fork(torch.from_numpy(source).cuda(), torch.from_numpy(new_len).cuda())
        again = cache.fork(torch.from_numpy(source).cuda(), torch.from_numpy(new_len).cuda())
        for c in (new, again):
            np.testing.assert_array_equal(c.table.cpu().numpy(), want_t)
            np.testing.assert_array_equal(c.lens.cpu().numpy(), want_l)
        np.testing.assert_array_equal(new.pages.cpu().numpy(), pages)
        table, lens, cache = want_t, want_l, new
        want_t, n_live, moves = O.compact(table, lens, pool, page_len)
        for a, b in moves:
            pages[:, b] = pages[:, a]
        new, live = cache.compact()
        assert int(live[0]) == n_live
        np.testing.assert_array_equal(new.table.cpu().numpy(), want_t)
        np.testing.assert_array_equal(new.pages.cpu().numpy(), pages)
        table, cache = want_t, new
        _lib.check(lib.cllm_cuda_check_device_status())


@pytest.mark.parametrize("pool,n_seqs,slots", [(70001, 1500, 40), (33, 1, 33), (32, 32, 1), (100000, 3, 5000)])
def test_fork_and_compact_large_tables(cuda, lib, pool, n_seqs, slots):
    rng = np.random.default_rng(pool)
    page_len = 16
    lens = rng.integers(0, slots * page_len + 1, n_seqs).astype(np.int32)
    while sum(-(-int(n) // page_len) for n in lens) > pool:
        lens //= 2
    cache, pages, table = _cache(rng, 1, pool, page_len, 1, 64, lens.tolist(), slots)
    source = rng.integers(-1, n_seqs, n_seqs).astype(np.int32)
    new_len = np.minimum(np.where(source >= 0, lens[source], 0) + 5, slots * page_len).astype(np.int32)
    want_t, want_l, copies = O.fork(table, lens, source, new_len, pool, page_len)
    for a, b in copies:
        pages[:, b] = pages[:, a]
    new = cache.fork(torch.from_numpy(source).cuda(), torch.from_numpy(new_len).cuda())
    np.testing.assert_array_equal(new.table.cpu().numpy(), want_t)
    np.testing.assert_array_equal(new.lens.cpu().numpy(), want_l)
    want_c, n_live, moves = O.compact(want_t, want_l, pool, page_len)
    for a, b in moves:
        pages[:, b] = pages[:, a]
    new, live = new.compact()
    assert int(live[0]) == n_live
    np.testing.assert_array_equal(new.table.cpu().numpy(), want_c)
    np.testing.assert_array_equal(new.pages.cpu().numpy(), pages)


@pytest.mark.parametrize("pool,n_seqs", [(500, 30), (40000, 30)])
def test_compact_in_place(cuda, lib, pool, n_seqs):
    """The C call may write the table that it reads."""
    rng = np.random.default_rng(n_seqs)
    lens = rng.integers(0, 16 * 8 + 1, n_seqs).astype(np.int32)
    cache, pages, table = _cache(rng, 2, pool, 16, 1, 64, lens.tolist(), 8)
    want, n_live, moves = O.compact(table, lens, pool, 16)
    for a, b in moves:
        pages[:, b] = pages[:, a]
    live = torch.zeros(1, dtype=torch.int32, device="cuda")
    _lib.check(lib.cllm_cuda_kv4_compact(cache.pages.data_ptr(), 2, pool, cache.page_bytes, 16, cache.table.data_ptr(),
                                         cache.lens.data_ptr(), n_seqs, 8, cache.table.data_ptr(), live.data_ptr(),
                                         torch.cuda.current_stream().cuda_stream))
    assert int(live[0]) == n_live
    np.testing.assert_array_equal(cache.table.cpu().numpy(), want)
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), pages)


def test_fork_of_a_bad_page_sets_the_status(cuda, lib):
    rng = np.random.default_rng(1)
    cache, _, table = _cache(rng, 1, 9, 16, 1, 64, [40, 40], 3)
    cache.table[0, 2] = 9
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    new = cache.fork(ints(0, 0, 1), ints(41, 41, 41))
    assert lib.cllm_cuda_check_device_status() == _lib.ERR_INVALID_ARG
    assert (new.table[2].cpu().numpy() == table[1]).all()
    cache.compact()
    assert lib.cllm_cuda_check_device_status() == _lib.ERR_INVALID_ARG


def test_fork_and_compact_in_a_graph(cuda, lib):
    rng = np.random.default_rng(2)
    cache, _, table = _cache(rng, 2, 40, 16, 2, 64, [100, 40, 7], 8)
    source = torch.tensor([0, 0, 1], dtype=torch.int32, device="cuda")
    want = torch.tensor([101, 120, 41], dtype=torch.int32, device="cuda")
    eager = cache.fork(source, want)
    eager.compact()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = cache.fork(source, want)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(new.table, eager.table) and torch.equal(new.lens, eager.lens)


# ---- scores -------------------------------------------------------------------------


def _check_scores(x, tokens, k, got, rows=None):
    for r in (range(x.shape[0]) if rows is None else rows):
        lp, rank, h, ids, lps, spread = O.scores(x[r], int(tokens[r]), k)
        tol = 2.0 ** -17 * (1 + spread)
        g = [t[r].cpu().numpy() for t in (got.logprob, got.rank, got.entropy, got.top_ids, got.top_logprobs)]
        assert g[1] == rank
        np.testing.assert_array_equal(g[3], ids)
        for have, want in ((g[0], lp), (g[2], h), (g[4], lps)):
            with np.errstate(over="ignore"):  # the operator answers in fp32: what overflows there is infinite
                want = np.atleast_1d(want).astype(np.float32).astype(np.float64)
            have = np.atleast_1d(have.astype(np.float64))
            np.testing.assert_array_equal(np.isnan(have), np.isnan(want))
            inf = np.isinf(want)
            np.testing.assert_array_equal(have[inf], want[inf])
            fine = np.isfinite(want)
            assert (np.abs(have[fine] - want[fine]) <= tol + 2.0 ** -22 * np.abs(want[fine])).all()


@pytest.mark.parametrize("rows,vocab,pad,k", [(1, 128256, 0, 5), (3, 1, 0, 1), (2, 7, 1, 7), (5, 32000, 0, 20),
                                              (37, 1023, 1, 32), (2, 151936, 64, 32), (300, 5001, 3, 1), (4, 33, 0, 32),
                                              (700, 257, 0, 0), (160, 50257, 0, 20)])
def test_scores(cuda, lib, rows, vocab, pad, k):
    from cllm_inference_b200.scoring import token_scores

    rng = np.random.default_rng(vocab + rows)
    x = (rng.standard_normal((rows, vocab + pad)) * 4).astype(np.float32)
    tokens = rng.integers(0, vocab, rows).astype(np.int32)
    x[rng.random(x.shape) < 0.2] = -np.inf
    tokens[0] = np.argmax(x[0, :vocab])
    xd = torch.from_numpy(x).cuda()[:, :vocab]
    got = token_scores(xd, torch.from_numpy(tokens).cuda(), k)
    _check_scores(x[:, :vocab], tokens, k, got, rows=range(0, rows, max(1, rows // 40)))
    alone = token_scores(xd, None, k)  # without tokens: the same of what remains
    assert alone.logprob is None and torch.equal(alone.top_ids, got.top_ids)
    np.testing.assert_array_equal(alone.entropy.cpu().numpy(), got.entropy.cpu().numpy())


@pytest.mark.parametrize("vocab", [100, 40000])
def test_scores_of_difficult_rows(cuda, lib, vocab):
    from cllm_inference_b200.scoring import token_scores

    rng = np.random.default_rng(vocab)
    n = np.arange(vocab, dtype=np.float32)
    rows = [np.zeros(vocab), np.sort(rng.standard_normal(vocab)), np.sort(rng.standard_normal(vocab))[::-1],
            np.full(vocab, -np.inf), np.where(n == 17, 3.0, -np.inf), np.where(n < 40, np.floor(n / 8), -np.inf),
            np.where(n % 2, 0.0, -0.0), np.full(vocab, -3.0e38), np.where(n == 5, 3e38, -3e38), np.round(rng.standard_normal(vocab)),
            np.where(n == 50, np.nan, 1.0), np.where(n == 60, np.inf, n), np.full(vocab, np.nan), 1e30 * rng.standard_normal(vocab),
            np.where(n == vocab - 1, 100.0, 0.0), np.floor(n / 50)]
    x = np.stack(rows).astype(np.float32)
    tokens = rng.integers(0, vocab, len(rows)).astype(np.int32)
    tokens[:6] = [vocab, -1, 0, 3, 17, 39]
    got = token_scores(torch.from_numpy(x).cuda(), torch.from_numpy(tokens).cuda(), 32)
    _check_scores(x, tokens, 32, got)


def test_scores_in_a_graph_and_repeatable(cuda, lib):
    from cllm_inference_b200.scoring import token_scores

    x = torch.randn(9, 60001, device="cuda") * 3
    t = torch.arange(9, dtype=torch.int32, device="cuda")
    first = token_scores(x, t, 20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_scores(x, t, 20)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, got))


# ---- refusals that need device tensors -------------------------------------------------


def test_refusals_of_the_front_ends(cuda, lib):
    from cllm_inference_b200.kv4 import KV4Cache, page_bytes
    from cllm_inference_b200.scoring import token_scores

    cache = KV4Cache.empty(2, 4, 16, 2, 64, 3, 2)
    ints = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    bad = [
        lambda: page_bytes(20, 1, 64), lambda: page_bytes(16, 1, 96),
        lambda: KV4Cache(cache.pages.float(), cache.table, cache.lens),
        lambda: KV4Cache(cache.pages, cache.table.long(), cache.lens),
        lambda: KV4Cache(cache.pages, cache.table, cache.lens[:2]),
        lambda: KV4Cache(cache.pages[..., :100].contiguous(), cache.table, cache.lens),
        lambda: cache.append(2, f(1, 128), f(1, 128), ints(1), ints(1)),
        lambda: cache.append(0, f(1, 64), f(1, 64), ints(1), ints(1)),
        lambda: cache.append(0, f(1, 128), f(1, 128), ints(2), ints(1)),
        lambda: cache.append(0, f(1, 128), f(1, 128), ints(1).long(), ints(1)),
        lambda: cache.append(0, f(1, 128).double(), f(1, 128).double(), ints(1), ints(1)),
        lambda: cache.append(0, f(1, 128), f(1, 128), ints(1), ints(1), q=f(1, 100)),
        lambda: cache.attention(0, f(2, 128)),                     # rows, no begin
        lambda: cache.attention(0, f(3, 192)),                     # 3 heads over 2
        lambda: cache.attention(0, f(3, 128), begin=ints(3)),
        lambda: cache.attention(-1, f(3, 128)),
        lambda: cache.attention(0, f(128, 3).t()),                 # rows are not dense
        lambda: cache.attention(0, f(3, 128), scale=float("nan")),
        lambda: cache.fork(ints(2), ints(3)),
        lambda: token_scores(f(4, 10), ints(4), 11), lambda: token_scores(f(4, 100), ints(4), 33),
        lambda: token_scores(f(4, 100), ints(4), -1), lambda: token_scores(f(4, 100), ints(3), 1),
        lambda: token_scores(f(4, 100).half(), ints(4), 1), lambda: token_scores(f(4, 100), ints(4).long(), 1),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(_lib.CudaError) as e:
            call()
        assert e.value.code == _lib.ERR_INVALID_ARG, i
    # nothing to do is no error
    assert cache.attention(0, f(0, 128), begin=ints(4)).shape == (0, 128)
    assert cache.append(0, f(0, 128), f(0, 128), ints(0), ints(0)) is None
    assert cache.fork(ints(0), ints(0)).n_seqs == 0
    assert token_scores(f(0, 50), ints(0), 3).top_ids.shape == (0, 3)
    _lib.check(lib.cllm_cuda_check_device_status())


# ---- together ---------------------------------------------------------------------------


def test_best_of_n_example(cuda, lib):
    """The example's candidates, taken again in one piece each, get the probabilities that they got step by step.

    Rows of a batch are quantized to Q8_0 before every matmul, and a last-bit difference between the batched and
    the one-row kernels can move a value by a whole step: the band is the engine's 5 % of the logits' scale
    (test_engine_gpu.py)."""
    import importlib.util
    import os

    from cllm_inference_b200 import gguf
    from cllm_inference_b200.kv4 import KV4Cache
    from cllm_inference_b200.scoring import token_scores

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "best_of_n.py")
    spec = importlib.util.spec_from_file_location("best_of_n", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    model = ex.Model(gguf.LlamaShape(2, 1024, 8, 2, 2048, 5000, 256))
    prompt = np.random.default_rng(1).integers(0, 5000, 75).tolist()
    steps = 12
    tokens, scores, in_use, cache = ex.best_of_n(model, prompt, n=5, steps=steps, keep=2)
    assert tokens.shape == scores.shape == (2, steps) and cache.n_seqs == 2
    pages = {int(p) for row in cache.table.tolist() for p in row if p >= 0}
    assert in_use == len(pages) and pages == set(range(in_use))
    assert in_use < 2 * -(-(75 + steps) // 16)  # the prompt's whole pages are shared
    for c in range(2):
        text = prompt + tokens[c].tolist()[:-1]
        whole = KV4Cache.empty(2, 8, 16, 2, 128, 1, 8).fork(ex.ints(-1), ex.ints(len(text)))
        n = len(text)
        logits = model.rows(whole, torch.tensor(text, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"),
                            torch.arange(n, dtype=torch.int32, device="cuda"), begin=ex.ints(0, n),
                            last=list(range(74, n)))
        again = token_scores(logits, tokens[c].contiguous()).logprob
        scale = float(logits.std())
        assert float((again - scores[c]).abs().max()) <= 0.05 * scale * 4  # logits within 4 deviations
    _lib.check(lib.cllm_cuda_check_device_status())
