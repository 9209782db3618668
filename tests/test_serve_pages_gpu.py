"""Page tables that name pages which do not exist, and pools that are too small."""
import numpy as np
import pytest
import torch

from cllm_inference_b200 import _lib
from tests import serve_oracle as O
from tests.test_serve_gpu import _cache

pytestmark = pytest.mark.gpu


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# (hd, KV heads, heads a KV head, rows of the first sequence): one row, a few (rows kernel), many (prompt kernel)
@pytest.mark.parametrize("hd,kv,rep,rows", [(128, 2, 4, 1), (64, 1, 3, 1), (128, 1, 2, 30), (64, 2, 2, 30),
                                            (128, 1, 1, 9000), (64, 2, 3, 3000)])
@pytest.mark.parametrize("bad", [12, -1, 2 ** 30])
def test_rows_that_see_a_page_outside_the_pool_are_nan(cuda, lib, hd, kv, rep, rows, bad):
    rng = np.random.default_rng(rows + hd)
    cache, _, _ = _cache(rng, 1, 12, 32, kv, hd, [150, 77], 5)
    q = torch.randn(rows + 3, kv * rep * hd, device="cuda")
    begin = _ints(0, rows, rows + 3)
    want, want_lse = cache.attention(0, q, begin=begin, lse=True)
    cache.table[0, 4] = bad  # positions 128 to 149
    got, lse = cache.attention(0, q, begin=begin, lse=True)
    assert lib.cllm_cuda_check_device_status() == _lib.ERR_INVALID_ARG
    sees = 150 - (rows - 1 - torch.arange(rows, device="cuda")) > 128
    assert torch.isnan(got[:rows][sees]).all() and torch.isnan(lse[:rows][sees]).all()
    assert not torch.isnan(got[:rows][~sees]).any() and torch.equal(got[rows:], want[rows:])
    torch.testing.assert_close(got[:rows][~sees], want[:rows][~sees], rtol=2.0 ** -16, atol=2.0 ** -16)
    torch.testing.assert_close(lse[rows:], want_lse[rows:], rtol=0, atol=0)
    _lib.check(lib.cllm_cuda_check_device_status())


@pytest.mark.parametrize("pool", [9, 20000])  # one launch, four launches
@pytest.mark.parametrize("bad", [20000, -7])
def test_fork_and_compact_carry_a_page_outside_the_pool_along(cuda, lib, pool, bad):
    """A sequence whose unfinished page does not exist gets no other page's content for it."""
    rng = np.random.default_rng(pool)
    cache, _, _ = _cache(rng, 1, pool, 16, 1, 64, [40, 40], 3)
    cache.table[0, 2] = bad  # positions 32 to 39
    new = cache.fork(_ints(0, 0, 1, 0), _ints(41, 48, 41, 32))
    assert lib.cllm_cuda_check_device_status() == _lib.ERR_INVALID_ARG
    assert new.lens.tolist() == [41, 48, 41, 32]
    assert new.table[0, 2] == bad and new.table[1, 2] == bad and new.table[3, 2] == -1
    assert torch.equal(new.table[2], cache.table[1])
    packed, live = new.compact()
    assert lib.cllm_cuda_check_device_status() == _lib.ERR_INVALID_ARG
    assert int(live[0]) == 5 and packed.table[0, 2] == bad and packed.table[1, 2] == bad
    o = packed.attention(0, torch.randn(4, 64, device="cuda"))
    assert lib.cllm_cuda_check_device_status() == _lib.ERR_INVALID_ARG
    assert torch.isnan(o[:2]).all() and torch.isfinite(o[2:]).all()


@pytest.mark.parametrize("slots", [16, 20000])  # one launch, four launches
def test_fork_without_room_for_all_can_be_made_again(cuda, lib, slots):
    """The first request that finds no room takes what comes after it along, even what needs no page; the old
    sequences are still whole and can be forked anew."""
    rng = np.random.default_rng(slots)
    cache, pages, table = _cache(rng, 2, 16, 16, 1, 64, [40, 48, 20, 7], slots)  # 3 + 3 + 2 + 1 pages, 7 free
    lens = [40, 48, 20, 7]
    source, want = [3, 0, 0, 1, 2], [8, 41 + 16 * 5, 41, 48, 21]  # s 1 needs 5, s 2 a copy, the others nothing
    new = cache.fork(_ints(*source), _ints(*want))
    assert new.lens.tolist() == [8, 121, 41, 48, 21]  # 6 of 7
    want[1] += 32
    table_want, lens_want, _ = O.fork(table, lens, source, want, 16, 16)
    new = cache.fork(_ints(*source), _ints(*want))
    assert new.lens.tolist() == lens_want.tolist() == [8, 153, -1, -1, -1]  # all 7: s 2's copy has no page
    want[1] += 16
    table_want, lens_want, _ = O.fork(table, lens, source, want, 16, 16)
    new = cache.fork(_ints(*source), _ints(*want))
    assert new.lens.tolist() == lens_want.tolist() == [8, -1, -1, -1, -1]  # 8
    assert (new.table[1:] == -1).all() and torch.equal(new.table, torch.from_numpy(table_want).cuda())
    # again, the small ones first
    source, want = [0, 3, 2, 1, 0], [41, 8, 21, 48, 41 + 16 * 5]
    table_want, lens_want, copies = O.fork(table, lens, source, want, 16, 16)
    new = cache.fork(_ints(*source), _ints(*want))
    assert new.lens.tolist() == lens_want.tolist() == want
    assert torch.equal(new.table, torch.from_numpy(table_want).cuda())
    have = new.pages.cpu().numpy()
    for s, old in enumerate(source):
        for layer in range(2):
            for x, y in zip(O.sequence(have[layer], table_want[s], lens[old], 64),
                            O.sequence(pages[layer], table[old], lens[old], 64)):
                np.testing.assert_array_equal(x, y)
    _lib.check(lib.cllm_cuda_check_device_status())
