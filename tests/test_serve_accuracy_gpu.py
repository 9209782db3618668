"""Attention over the 4-bit cache where one position takes nearly all of the
weight, as an early position does in trained models: what the many small weights
add must not be lost.

Tolerance.  To first order an output o = sum w v changes by sum w ds (v - o) when
the scores change by ds, which is little where one position dominates.  fp32
arithmetic leaves ds within hd * 2^-24 <= 2^-17 of a score's terms' magnitudes,
a weight (exponent and exponential) within 2^-18 and the sums within 2^-17 of the
magnitudes that they add.  Weights and their products with the values' scales are
pairs of fp16 numbers with a last digit of 2^-24 beside a largest weight of 2^10 and
scales of 2^-3 at least: 2^-24 / sqrt(12) * 4.7 (a number's distance from the
middle) * 8 scales / 2^10 for each position, which add up like a random walk; six
deviations of it."""
import numpy as np
import pytest
import torch

from cllm_inference_b200 import _lib
from tests import serve_oracle as O

pytestmark = pytest.mark.gpu

RAISED = 17.5  # nats by which the position stands out
SINK = 3       # where it is


def _cache(rng, hd, kv, n, size, digits="", raised=RAISED):
    """One sequence of n positions, keys and values with numbers at random; the values (mean 0.1, deviation 0.1, times
    `size`) of the position that dominates are small.  digits "all": the values' scales are whole numbers (the minimum's
    odd) of fp16's last digit instead; "one": those of the position that dominates.  Returns the cache, its pages and table, and the direction of
    queries that the dominating key answers to."""
    from cllm_inference_b200.kv4 import KV4Cache

    slots = -(-n // 64)
    p = rng.integers(0, 256, (1, slots, kv, 4, 20 * hd), dtype=np.uint8)
    s = np.empty((*p.shape[:4], 2, 16, hd // 32, 2), np.float16)
    s[..., 0, :, :, :] = 0.1, -0.75
    s[..., 1, :, :, :] = 0.0217 * size, -0.0625 * size
    table = rng.permutation(slots).astype(np.int32)[None]
    first = p[0, table[0, 0], :, 0]
    side = rng.integers(0, 2, hd)
    size_k = raised / 2 / np.sqrt(hd)
    s[0, table[0, 0], :, 0, 0, SINK] = 2 * size_k / 15, -size_k
    s[0, table[0, 0], :, 0, 1, SINK] = 0.0217 * size / 128, -0.0625 * size / 128
    for at, up in zip(O.k_nibble(SINK, np.arange(hd), hd), side):
        b = first[:, at // 2]
        first[:, at // 2] = (b & 0x0F) | (0xF0 if up else 0) if at & 1 else (b & 0xF0) | (0x0F if up else 0)
    if digits:
        shape = s.shape[:4] + s.shape[5:7]
        few = np.stack([rng.integers(1, 201, shape), rng.integers(-1000, 1001, shape) * 2 + 1], -1) * 2.0 ** -24
        if digits == "all":
            s[..., 1, :, :, :] = few
        else:
            s[0, table[0, 0], :, 0, 1, SINK] = few[0, table[0, 0], :, 0, SINK]
    p[..., 16 * hd:] = s.reshape(*p.shape[:4], -1).view(np.uint8)
    c = KV4Cache(torch.from_numpy(p).cuda(), torch.from_numpy(table).cuda(),
                 torch.tensor([n], dtype=torch.int32, device="cuda"))
    return c, p, table, 2.0 * side - 1.0


def _check(hd, kv, rep, rows, n, size, digits="", raised=RAISED):
    rng = np.random.default_rng(hd + rows + n)
    cache, p, table, side = _cache(rng, hd, kv, n, size, digits, raised)
    heads = kv * rep
    q = (1.5 * rng.standard_normal((rows, heads, hd)) + 2 * side).astype(np.float32)
    begin = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    o, lse = cache.attention(0, torch.from_numpy(q.reshape(rows, -1)).cuda(), begin=begin, lse=True)
    o, lse = o.cpu().numpy().astype(np.float64).reshape(rows, heads, hd), lse.cpu().numpy().astype(np.float64)
    k, v = O.sequence(p[0], table[0], n, hd)
    largest = 200 * 2.0 ** -24 if digits == "all" else 0.0217 * size  # of the values' scales
    worst = 0.0
    for row in sorted({0, rows // 3, rows // 2, rows - 1}):
        sees = n - (rows - 1 - row)
        for h in range(heads):
            qq, kk, vv = q[row, h].astype(np.float64), k[h // rep, :sees], v[h // rep, :sees]
            x = kk @ qq / np.sqrt(hd)
            m = x.max()
            w = np.exp(x - m)
            total = w.sum()
            w /= total
            assert w[SINK] > 0.9
            want = w @ vv
            terms = np.abs(kk) @ np.abs(qq) / np.sqrt(hd)
            tol = (w * (2.0 ** -17 * terms + 2.0 ** -18)) @ np.abs(vv - want) + 2.0 ** -17 * (w @ np.abs(vv))
            tol += 6 * np.sqrt(sees) * 2.0 ** -24 / np.sqrt(12) * 4.7 * 8 * largest / 1024
            worst = max(worst, float((np.abs(o[row, h] - want) / tol).max()))
            assert abs(lse[row, h] - (m + np.log(total))) <= 2.0 ** -17 * (1 + (w * terms).sum())
    assert worst <= 1, f"{worst:.3g} of the tolerance"


@pytest.mark.parametrize("size", [1.0, 2.0 ** -8])
@pytest.mark.parametrize("hd,kv,rep,rows,n", [(128, 2, 2, 160, 8000), (64, 2, 2, 160, 8000), (128, 1, 1, 64, 100000),
                                              (64, 1, 1, 64, 100000)])
def test_small_weights_beside_a_dominating_position_prompts(cuda, lib, hd, kv, rep, rows, n, size):
    _check(hd, kv, rep, rows, n, size)
    _lib.check(lib.cllm_cuda_check_device_status())


@pytest.mark.parametrize("size", [1.0, 2.0 ** -8])
@pytest.mark.parametrize("hd,kv,rep,rows,n", [(128, 1, 4, 1, 8000), (64, 2, 2, 1, 8000), (128, 1, 3, 1, 100000),
                                              (64, 1, 1, 1, 100000)])
def test_small_weights_beside_a_dominating_position_one_row(cuda, lib, hd, kv, rep, rows, n, size):
    _check(hd, kv, rep, rows, n, size)
    _lib.check(lib.cllm_cuda_check_device_status())


@pytest.mark.parametrize("hd,kv,rep,rows,n", [(128, 1, 4, 1, 8000), (64, 2, 2, 1, 8000), (128, 2, 2, 160, 8000),
                                              (64, 2, 2, 160, 8000)])
def test_values_of_a_few_of_fp16s_last_digits(cuda, lib, hd, kv, rep, rows, n):
    _check(hd, kv, rep, rows, n, 1.0, digits="all")
    _lib.check(lib.cllm_cuda_check_device_status())


@pytest.mark.parametrize("hd,kv,rep,rows,n", [(128, 2, 4, 1, 48), (64, 4, 4, 1, 48), (128, 40, 1, 160, 300),
                                              (64, 40, 1, 160, 300)])
def test_a_dominating_value_of_a_few_of_fp16s_last_digits(cuda, lib, hd, kv, rep, rows, n):
    """Beside others with scales of 0.3, so that the cache as a whole needs no power of two."""
    _check(hd, kv, rep, rows, n, 14.0, digits="one", raised=25.0)
    _lib.check(lib.cllm_cuda_check_device_status())
