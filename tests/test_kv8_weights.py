"""Weights and queries of very different size in the 8-bit cache's decode
attention (``wnw_kv8_attn``), against 64 bits over the rows read back.

Tolerances, derived: an output is rounded once (eps / 2 of itself, half the
smallest subnormal number in fp16).  A weight of a full block is held in two
fp16 terms, 2^14 above the largest: off by at most 2^-22 of itself (fp16's
numbers in [1, 2) are 2^-10 apart, twice half of that), and by 2^-39 of the
largest below fp16's normal numbers; of an unfinished block in two terms of the
type (2^-16 in bf16, 2^-22 in fp16).  A score is off by 2^-20 of the sum of its terms'
magnitudes (fp32 sums of up to 128 exact products, three factors), which the
weights carry twice (weight and sum) and the log-sum-exp once.
"""
import math

import pytest
import torch

from oracle import kv8 as O
from wnw_b200.kv8 import KV8Attention, KV8Store

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _filled(k, v, code, page_rows=64):
    """A store with k, v [segments, n, D] in it, and its lengths."""
    S, n, D = k.shape
    pages = -(-n // page_rows)
    s = KV8Store(S, D, S * pages, pages, page_rows, code, k.dtype)
    s.reserve(n)
    s.append(k[:, None].cuda(), v[:, None].cuda(), torch.zeros(S, dtype=torch.int32, device="cuda"))
    return s, torch.full((S,), n, dtype=torch.int32, device="cuda")


def _check(store, q, n, scale, out, lse, segs):
    held = 2.0 ** -16 if store.dtype is BF16 and n % 32 else 2.0 ** -22
    eps = torch.finfo(store.dtype).eps
    tiny = 2.0 ** -25 if store.dtype is F16 else 0.0
    for s in segs:
        k, v = (x.cpu().double() for x in store.dequantize(s, n))
        x = q[s].double()
        want, wl, pv = O.attention(x, k, v, scale)
        ds = 2.0 ** -20 * float((x.abs() @ k.abs().t()).max()) * abs(scale)
        tol = (eps / 2 * want.abs() * (1 + 2.0 ** -7) + (held + 2 * ds + 2.0 ** -20) * pv
               + n * 2.0 ** -39 * float(v.abs().max()) + tiny)
        off = (out[s].cpu().double() - want).abs()
        assert bool((off <= tol).all()), (s, float((off / tol).max()))
        assert bool(((lse[s].cpu().double() - wl).abs() <= ds + 2.0 ** -20 * (wl.abs() + 1)).all())


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("S,n", [(1200, 256), (1, 20), (3, 276)])
@pytest.mark.parametrize("gap", [15.0, 17.5, 22.0, 25.0])
def test_many_small_weights_beside_a_large_one(code, dtype, S, n, gap):
    """One token of value zero, ``gap`` nats above all others: what comes out
    is the others' share, whether blocks or an unfinished one hold them, over
    several blocks a warp and over one."""
    D = 64
    k, v = torch.zeros(S, n, D, dtype=dtype), torch.full((S, n, D), 4096.0, dtype=dtype)
    k[:, 0, 0] = 1.0
    v[:, 0] = 0.0
    store, lens = _filled(k, v, code)
    q = torch.zeros(S, 2, D, dtype=dtype)
    q[..., 0] = 8.0
    out, lse = KV8Attention(store, 2, gap / 8)(q.cuda(), lens, return_lse=True)
    _check(store, q, n, gap / 8, out, lse, range(0, S, max(1, S // 6)))
    store.check()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,G,n", [(64, 3, 96), (128, 4, 900), (128, 8, 41)])
def test_outputs_are_rounded_once(code, dtype, D, G, n):
    """Random rows: nothing but the output's own rounding shows."""
    g = torch.Generator().manual_seed(n)
    k, v = (torch.randn(4, n, D, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(4, G, D, generator=g).to(dtype)
    store, lens = _filled(k, v, code)
    out, lse = KV8Attention(store, G, D ** -0.5)(q.cuda(), lens, return_lse=True)
    _check(store, q, n, D ** -0.5, out, lse, range(4))
    store.check()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,n", [(64, 96), (128, 300), (128, 32)])
def test_small_dimensions_beside_a_large_one(code, dtype, D, n):
    """Queries whose largest dimension meets only zeros: the others, 2^-20 of
    it, are all that the scores are made of."""
    g = torch.Generator().manual_seed(n)
    k, v = (torch.randn(3, n, D, generator=g).to(dtype) for _ in range(2))
    k[..., 0] = 0.0
    bits = 128 if dtype is BF16 else 1024
    q = (1 + torch.randint(0, bits, (3, 4, D), generator=g) / bits) * 2.0 ** -10
    q = (q * (1 - 2 * torch.randint(0, 2, q.shape, generator=g))).to(dtype)
    q[..., 0] = 1024.0
    store, lens = _filled(k, v, code)
    out, lse = KV8Attention(store, 4, 2.0 ** 8)(q.cuda(), lens, return_lse=True)
    _check(store, q, n, 2.0 ** 8, out, lse, range(3))
    store.check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 26, 2.0 ** 30])
def test_equal_scores_of_any_size(dtype, size):
    """Equal keys weigh the same, in blocks and in the unfinished one, however
    large their scores: the output is the values' mean."""
    n, D = 73, 64
    k = torch.zeros(2, n, D, dtype=dtype)
    k[..., :2] = 1.0
    v = torch.zeros(2, n, D, dtype=dtype)
    v[:, :64, 0], v[:, 64:, 1] = 1.0, 1.0
    store, lens = _filled(k, v, "int8")
    store.scales()[..., 0] = 2.0 ** -7  # 127 codes of a key of 127 / 128: scores exact in fp32
    store.tail_k[:, 0, :, :2] = 127 / 128
    q = torch.zeros(2, 1, D, dtype=dtype)
    q[..., 0] = 1.0
    out, _ = KV8Attention(store, 1, size)(q.cuda(), lens, return_lse=True)
    want = torch.zeros(2, 1, D, dtype=torch.float64)
    want[..., 0], want[..., 1] = 64 / n, 9 / n
    eps = torch.finfo(dtype).eps
    # the output's rounding, and the values' scale (2^-20); both keys' scores are the same number
    assert bool(((out.cpu().double() - want).abs() <= (eps / 2 + 2.0 ** -12) * want).all()), out[..., :2]
    store.check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n", [20, 31, 84])
def test_weights_of_values_that_cancel(dtype, n):
    """Values of 1 and -1 whose sum is small beside their number: what the
    weights' own rounding leaves is not hidden behind the output's.  A weight
    is off by 2^-22 of itself however it is held, by its exponential (2^-21)
    and its score (2^-20 of the terms' magnitudes, twice)."""
    g = torch.Generator().manual_seed(n)
    S, G, D = 40, 8, 128
    k = torch.randn(S, n, D, generator=g).to(dtype)
    v = (1 - 2 * torch.randint(0, 2, (S, n, D), generator=g)).to(dtype)
    q = torch.randn(S, G, D, generator=g).to(dtype)
    store, lens = _filled(k, v, "int8")
    out = KV8Attention(store, G, D ** -0.5)(q.cuda(), lens)
    eps, small = torch.finfo(dtype).eps, 0
    for s in range(S):
        kk, vv = (x.cpu().double() for x in store.dequantize(s, n))
        x = q[s].double()
        want, _, pv = O.attention(x, kk, vv, D ** -0.5)
        ds = 2.0 ** -20 * float((x.abs() @ kk.abs().t()).max()) * D ** -0.5
        tol = eps / 2 * want.abs() * (1 + 2.0 ** -7) + (2.0 ** -22 + 2.0 ** -21 + 2 * ds + 2.0 ** -20) * pv + 2.0 ** -25
        small += int((want.abs() < 2.0 ** -9).sum())
        off = (out[s].cpu().double() - want).abs()
        assert bool((off <= tol).all()), (s, float((off / tol).max()))
    assert small > 100
    store.check()
