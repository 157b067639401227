"""Attention over packed prompts on the GPU, against a plain implementation in 64 bits."""
import math

import pytest
import torch

from tests import paged_reference as ref
from tests.test_gpu_paged import BF16, F16, TYPES, _words

pytestmark = pytest.mark.gpu


def _prompt(q, k, v, at, scale, window=0, k_at=None):
    import flash_gemv

    return flash_gemv.cats_prompt_attention(q.cuda(), k.cuda(), v.cuda(), _words(at), scale, window, None if k_at is None else _words(k_at))


def _check(at, heads, kv, D, dtype, window=0, k_at=None, N=None, M=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    N = at[-1] if N is None else N
    M = N if k_at is None else k_at[-1] if M is None else M
    q = (torch.randn(N, heads, D, generator=g) * 1.5).to(dtype)
    k, v = (torch.randn(M, kv, D, generator=g).to(dtype) for _ in range(2))
    got = _prompt(q, k, v, at, D ** -0.5, window, k_at)
    assert ref.within(got, *ref.prompt_attention(q, k, v, at, k_at or at, D ** -0.5, window))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 2), (6, 2), (7, 1), (8, 1)])
def test_lengths(heads, kv, D, dtype):
    """One token, tiles' ends and what lies on either side of them, prompts without tokens, in one call."""
    _check([0, 1, 17, 17, 80, 144, 209, 209, 338, 600], heads, kv, D, dtype)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
def test_one_prompt(n):
    _check([0, n], 2, 1, 64, F16)
    _check([0, n], 1, 1, 128, BF16)


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64), (F16, 256), (BF16, 32)])
@pytest.mark.parametrize("window", [1, 2, 31, 64, 65, 200, 10000])
def test_windows(window, dtype, D):
    _check([0, 5, 300, 429, 700], 6, 2, D, dtype, window)


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64)])
def test_tokens_of_nobody(dtype, D):
    """Before the first and behind the last: zeros; and a batch of nobody."""
    _check([3, 40, 40, 170], 4, 2, D, dtype, N=400)
    _check([0, 0, 0], 4, 2, D, dtype, N=130)
    _check([130, 130], 4, 2, D, dtype, N=130)


@pytest.mark.parametrize("B", [63, 64, 65, 300, 5000])
def test_many_prompts(B):
    at = [0]
    for b in range(B):
        at.append(at[-1] + (b * 7) % 5)
    _check(at, 2, 1, 32, F16)


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64), (F16, 256), (BF16, 32)])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("at,k_at", [([0, 5, 70, 71, 200], [0, 5, 400, 1000, 1129]), ([0, 100, 230, 231], [0, 20, 150, 150]), ([0, 33], [7, 900])])
def test_more_keys_than_queries_and_fewer(at, k_at, window, dtype, D):
    """Queries are the last tokens of their sequence; those that see no key are zeros."""
    _check(at, 4, 2, D, dtype, window, k_at, M=k_at[-1] + 9)


def test_keys_of_others_and_masked_ones_may_be_anything():
    """NaN and infinities in keys and values reach the queries behind them in their own prompt, and no other."""
    g = torch.Generator().manual_seed(1)
    at = [0, 70, 270, 300]
    for dtype in TYPES:
        for bad in (70, 133, 200, 269):
            for value in (math.nan, math.inf):
                q, k, v = (torch.randn(310, h, 64, generator=g).to(dtype) for h in (4, 2, 2))
                v[bad, 0, 9] = value
                k[bad, 1, 3] = math.nan
                assert ref.within(_prompt(q, k, v, at, 0.125), *ref.prompt_attention(q, k, v, at, at, 0.125))


def test_strides():
    """Queries, keys and values as slices of one projection's output, heads outermost, and a layout that is copied."""
    g = torch.Generator().manual_seed(2)
    at = [0, 90, 200]
    f = torch.randn(200, 8 * 64, generator=g).bfloat16()
    q, k, v = (x.reshape(200, -1, 64) for x in f.split([256, 128, 128], 1))
    want = ref.prompt_attention(q, k, v, at, at, 0.125)
    c = f.cuda()
    assert ref.within(_prompt(c[:, :256].view(200, 4, 64), c[:, 256:384].view(200, 2, 64), c[:, 384:].view(200, 2, 64), at, 0.125), *want)
    turned = lambda t: t.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    assert ref.within(_prompt(turned(q), turned(k), turned(v), at, 0.125), *want)
    odd = lambda t: torch.cat([t[..., :1], t], -1).cuda()[..., 1:]
    assert ref.within(_prompt(odd(q), odd(k), odd(v), at, 0.125), *want)
    one = torch.randn(1, 1, 64, generator=g).bfloat16()  # expanded: a stride of 0
    assert ref.within(_prompt(q, one.expand(200, 2, 64), v, at, 0.125), *ref.prompt_attention(q, one.expand(200, 2, 64), v, at, at, 0.125))


@pytest.mark.parametrize("scale", [2.0 ** -64, 1e-4, 3.0, 40.0])
def test_scales(scale):
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(200, h, 64, generator=g).half() for h in (2, 1, 1))
    assert ref.within(_prompt(q, k, v, [0, 200], scale), *ref.prompt_attention(q, k, v, [0, 200], [0, 200], scale))
