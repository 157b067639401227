"""Attention over pages and over packed prompts where scores are large, and where values are large or small: steps, drafts, pieces, parts, shared keys, prompts."""
import math

import pytest
import torch

from tests import paged_reference as ref
from tests.test_gpu_packed_prompts import _prompt
from tests.test_gpu_paged import _attention
from tests.test_gpu_paged_parts import _copy_shared

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16

# rows, tokens that the table has room for beyond them (which decides on parts), group, shared; two query heads a cached one
CALLS = {
    "steps": ([(300, 1), (0, 1), (110, 1)], 0, 1, 0),
    "drafts": ([(300, 5), (0, 3), (110, 1)], 0, 1, 0),
    "pieces": ([(300, 70), (0, 130), (110, 20)], 0, 1, 0),
    "steps in parts": ([(1500, 1), (700, 4), (3, 1)], 2100, 1, 0),
    "pieces in parts": ([(1500, 70), (700, 33), (0, 20)], 2100, 1, 0),
    "shared by few rows": ([(700, 1), (900, 1), (650, 2)], 2100, 3, 640),
    "shared by many rows": ([(1450 + 60 * b, 1 + b % 2) for b in range(12)], 2100, 12, 1400),
    "groups of many rows": ([(400 + 40 * b, 1) for b in range(22)], 0, 11, 384),
}
TYPES = [(F16, 64), (BF16, 128), (F16, 256), (BF16, 32)]


def _cached(name, keys_of, dtype, D, g, size=1.0):
    """(rows, group, shared, pool) of a call: keys by their positions, values at random, `size` of them."""
    rows, room, group, shared = CALLS[name]
    pool = ref.new_pool(rows, 64, 1, D, dtype, 3, room=max(2, room // 64), group=group, shared=shared)
    ref.fill(pool, rows, g, size)
    for b, (a, n) in enumerate(rows):
        for i in range(-(-(a + n) // 64)):
            m = min(64, a + n - 64 * i)
            pool[0][int(pool[2][b, i]), 0, :m] = keys_of(torch.arange(64 * i, 64 * i + m))
    _copy_shared(pool, rows, group, shared)
    return rows, group, [shared] if group > 1 else None, pool


def _check(got, want, bound):
    """Within the bound, which neither zeros nor the result with the other sign are."""
    assert not ref.within(torch.zeros_like(want), want, bound) and not ref.within(-want, want, bound)
    assert ref.within(got, want, bound)


def _bound(want, size, dtype, delta):
    """Half a step of each weight and of the output; 2^-20 for sums and the division; what an error `delta` of the scores makes of the weights, above and below the line.
    size: the weighted magnitudes of the values."""
    u = ref.HALF[dtype]
    return u * want.abs() + (u + 2.0 ** -20 + 2 * delta) * size + ref.LEAST[dtype]


def _query(D, dtype, sign):
    q = 1024 * sign
    q[-1] = 256
    return q.to(dtype)


def _keys(D, dtype, sign, side, levels):
    """Keys whose products with the query are side * 2^25 * (1 - 1 / D) + 256 * level, every partial sum a multiple of 256 below 2^26: exact in 32 bits.  Every 97th is one of
    the levels, the others far below them."""
    def of(position):
        k = (side * (32768 // D) * sign).repeat(len(position), 1)
        k[:, -1] = -320
        for i, level in enumerate(levels):
            k[position % (97 * len(levels)) == 97 * i + 5, -1] = level
        return k.to(dtype)

    return of


# Scores of 2^17, whose products with log2(e) and the scale lie beyond 2^16 and are rounded to a step of 2^-6: keys that are alike and keys whose scores differ by 1 and 2.5.  A
# difference of two of them is off by two such roundings, 2^-24 of each.  Beyond that scores that 32 bits hold to no fraction: keys that are alike share the weight.
FAR = [((0.0, -1.0, -2.5), 2.0 ** -8, 2.0 ** -6), ((0.0,), 2.0 ** -8, 0.0), ((0.0,), 2.0 ** 8 + 2.0, 0.0), ((0.0,), 2.0 ** 64, 0.0)]


@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("side", [1, -1])
@pytest.mark.parametrize("levels,scale,delta", FAR)
@pytest.mark.parametrize("name", CALLS)
def test_large_scores_over_pages(name, levels, scale, delta, side, dtype, D):
    g = torch.Generator().manual_seed(51)
    sign = torch.randn(D, generator=g).sign()
    rows, group, shared, pool = _cached(name, _keys(D, dtype, sign, side, levels), dtype, D, g)
    q = _query(D, dtype, sign).expand(ref.offsets_of(rows)[-1], 2, D).contiguous()
    want = ref.paged_attention(q, rows, 0, pool, scale)[0]
    size = ref.paged_attention(q, rows, 0, (pool[0], pool[1].abs(), pool[2]), scale)[0]
    _check(_attention(q, rows, 0, pool, scale, 0, group, shared), want, _bound(want, size, dtype, delta))


@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("side", [1, -1])
@pytest.mark.parametrize("levels,scale,delta", FAR)
@pytest.mark.parametrize("window", [0, 150])
def test_large_scores_of_prompts(window, levels, scale, delta, side, dtype, D):
    g = torch.Generator().manual_seed(52)
    sign, at = torch.randn(D, generator=g).sign(), [0, 1, 260, 900]
    k = torch.cat([_keys(D, dtype, sign, side, levels)(torch.arange(e - a)) for a, e in zip(at, at[1:])])[:, None]
    v = torch.randn(900, 1, D, generator=g).to(dtype)
    q = _query(D, dtype, sign).expand(900, 2, D).contiguous()
    want = ref.prompt_attention(q, k, v, at, at, scale, window)[0]
    size = ref.prompt_attention(q, k, v.abs(), at, at, scale, window)[0]
    _check(_prompt(q, k, v, at, scale, window), want, _bound(want, size, dtype, delta))


# fp16: single steps of the smallest numbers, and the largest ones.  bf16: the largest, and those down to 2^-100: weights begin at 2^-40, so products with these are numbers of
# 2^-140, which lie 2^-149 apart, and a sum of some hundred of them is off by far less than half a step of bf16.
SIZES = [(F16, 64, 2.0 ** -24), (F16, 128, 2.0 ** -17), (F16, 64, 16000.0), (BF16, 128, 2.0 ** -80), (BF16, 64, 2.0 ** -100), (BF16, 64, 2.0 ** -40), (BF16, 64, 2.0 ** 125)]


def _values(g, shape, size, dtype):
    """Up to four times `size`."""
    return ((torch.randn(shape, generator=g) * 1.3).clamp(-3.9, 3.9).round(decimals=1) * size if size > 2.0 ** -24 else torch.randint(-40, 41, shape, generator=g) * size).to(dtype)


@pytest.mark.parametrize("dtype,D,size", SIZES)
@pytest.mark.parametrize("name", CALLS)
def test_sizes_of_values_over_pages(name, dtype, D, size):
    g = torch.Generator().manual_seed(53)
    every = torch.randn(4096, D, generator=g).to(dtype)
    rows, group, shared, pool = _cached(name, lambda p: every[p], dtype, D, g, 0.0)
    seen = pool[1] == 0
    pool[1][seen] = _values(g, pool[1].shape, size, dtype)[seen]
    _copy_shared(pool, rows, group, CALLS[name][3])
    q = torch.randn(ref.offsets_of(rows)[-1], 2, D, generator=g).to(dtype)
    _check(_attention(q, rows, 0, pool, D ** -0.5, 0, group, shared), *ref.paged_attention(q, rows, 0, pool, D ** -0.5))


@pytest.mark.parametrize("dtype,D,size", SIZES)
def test_sizes_of_values_of_prompts(dtype, D, size):
    g = torch.Generator().manual_seed(54)
    at = [0, 1, 260, 900]
    q, k = (torch.randn(900, h, D, generator=g).to(dtype) for h in (2, 1))
    v = _values(g, (900, 1, D), size, dtype)
    _check(_prompt(q, k, v, at, D ** -0.5), *ref.prompt_attention(q, k, v, at, at, D ** -0.5))


@pytest.mark.parametrize("dtype,D", [(F16, 64), (F16, 128), (BF16, 64)])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -13, 2.0 ** -17, 2.0 ** -19])
@pytest.mark.parametrize("name", CALLS)
def test_light_weights_count(name, size, dtype, D):
    """Keys alike whose weights are 1.2 times 2^-13 of the first one's, whose values are zeros: all that is left of the output is theirs.  In fp16 weights have the fewest bits."""
    g = torch.Generator().manual_seed(55)

    def of(position):
        k = torch.zeros(len(position), D)
        k[position == 0, 0] = (13 * math.log(2) - math.log(1.2)) * 8
        return k.to(dtype)

    rows, group, shared, pool = _cached(name, of, dtype, D, g)
    pool[1].copy_(((1 + 0.2 * torch.randn(pool[1].shape, generator=g)) * size).to(dtype))
    for b in range(len(rows)):
        pool[1][int(pool[2][b, 0]), 0, 0] = 0
    _copy_shared(pool, rows, group, CALLS[name][3])
    q = torch.zeros(ref.offsets_of(rows)[-1], 2, D)
    q[..., 0] = 1
    q = q.to(dtype)
    _check(_attention(q, rows, 0, pool, 0.125, 0, group, shared), *ref.paged_attention(q, rows, 0, pool, 0.125))
