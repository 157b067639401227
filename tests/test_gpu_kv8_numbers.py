"""Attention over a cache in 8 bits where the numbers are large, small or far apart, by the step's kernel and by the one for many tokens."""
import math

import pytest
import torch

from cats_amd import capi
from tests import cache_reference as ref
from tests.test_gpu_kv8 import BF16, F16, _attention, _filled, _tokens

pytestmark = pytest.mark.gpu

KERNELS = [(1, 0), (5, 0), (1, 130), (70, 0)]  # T, tokens further back than which nothing is seen; the last takes the kernel for many tokens
ROOM = 600  # blocks, of which few are used


def _call(cache, q, start, window=0, scale=None):
    T, heads, kv, blocks = q.shape[1], q.shape[2], *cache["k8"].shape[1:3]
    assert capi.kv8_attention_plan(q.shape[0], T, heads, kv, q.shape[3], blocks, window)[0] == (T == 70)
    return _attention(ref.to(cache, "cuda"), q.cuda(), start, scale=scale, window=window).cpu().double()


def _room(k, v, blocks=ROOM):
    return ref.append(ref.new_cache(k.shape[0], k.shape[2], blocks, k.shape[3], k.dtype), k, v, [0] * k.shape[0], None)


def _scores(cache, q, start, scale, window):
    """Of one row and one cached head, in double: (T, heads, keys), -infinity for keys that are not seen, and the largest sum of magnitudes."""
    T, n = q.shape[1], start + q.shape[1]
    full = (n - 1) // 64
    k = torch.cat([(cache["k8"][0, 0, :full].double() * cache["k_scale"][0, 0, :full, None, None].double()).flatten(0, 1), cache["k_tail"][0, 0, : n - full * 64].double()])
    x = (q[0].double() @ k.t()) * scale
    back = torch.arange(start, n)[:, None] - torch.arange(n)
    return x.masked_fill(((back < 0) | (back >= (window or n)))[:, None], -math.inf), float((q[0].double().abs() @ k.abs().t()).max()) * scale


@pytest.mark.parametrize("T,window", KERNELS)
@pytest.mark.parametrize("dtype,size,scale", [(F16, 1024.0, None), (F16, 2500.0, None), (F16, 1.0, 2.0 ** 40), (F16, 1.0, 2.0 ** 64), (BF16, 2500.0, None), (BF16, 1.0, 2.0 ** 64),
                                               (BF16, 2.0 ** 30, None)])
@pytest.mark.parametrize("lean", [0.0, 3.0, -3.0])
def test_scores_that_32_bits_hold_to_no_fraction(dtype, size, scale, lean, T, window):
    """Where the two best scores of a query lie further apart than what 32 bits make of them (a sum of D products, a scaling) by more than 2^6, which is nearly
    always, one key has all the weight and no other reaches 2^-60: what is left is half a step each of that weight and of the output.  Elsewhere the result
    lies among the values.  lean: all scores moved up or down."""
    D = 128
    g = torch.Generator().manual_seed(int(size) % 1000 + T)
    scale = D ** -0.5 if scale is None else scale
    along = torch.randn(D, generator=g).sign() * size  # what queries and keys have in common
    k, v = ((_tokens(g, 1, 300, 1, D, torch.float32, 0.0) * size + 0.3 * lean * along).to(dtype), _tokens(g, 1, 300, 1, D, dtype))
    q = (torch.randn(1, T, 8, D, generator=g) * size + 0.3 * abs(lean) * along).to(dtype)
    cache = _room(k, v)
    x, most = _scores(cache, q, 300 - T, scale, window)
    best = x.topk(2, -1).values
    clear = best[..., 0] - best[..., 1] > 64 + 2 * (D + 8) * most * 2.0 ** -24
    assert clear.double().mean() > 0.9
    want, _ = ref.attention(cache, q, [300 - T], None, scale, window)
    out, u, least = _call(cache, q, [300 - T], window, scale), ref.HALF[dtype], 2.0 ** -25 * (dtype == F16)
    assert float(out.abs().max()) <= (1 + 2 * u) * float(v.abs().max()) * (1 + 2.0 ** -4)  # v as it was before it was stored
    assert ref.within(out[0][clear], want[0][clear], (2 * u * want.abs() + 2.0 ** -50 * float(v.abs().max()) + least)[0][clear])


@pytest.mark.parametrize("T,window", [(1, 0), (5, 0), (70, 0)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scale", [128 ** -0.5, 2.0 ** 20 + 2.0 ** 3, 2.0 ** 64])
def test_equal_scores_that_are_large_share_the_weight(dtype, scale, T, window):
    """The same key in two complete blocks and in the tail, all its products exact: they share the weight, whatever the score.  Everybody else's score is half
    of theirs or less."""
    D, at = 128, [20, 150, 260]
    g = torch.Generator().manual_seed(3)
    sign = torch.randn(D, generator=g).sign()
    k, v = (512 * sign).expand(1, 300, 1, D).clone().to(dtype), _tokens(g, 1, 300, 1, D, dtype)
    k[0, at, 0] = (1024 * sign).to(dtype)
    k[0, 140, 0] = 0
    k[0, 140, 0, 5] = 4096 * sign[5]  # its block has another scale
    q = (1024 * sign).expand(1, T, 2, D).to(dtype).contiguous()
    cache = _room(k, v)
    assert cache["k_scale"][0, 0, 0] != cache["k_scale"][0, 0, 2]
    for p in at[:2]:
        assert ref.same(cache["k8"][0, 0, p // 64, p % 64].float() * cache["k_scale"][0, 0, p // 64], k[0, p, 0])
    vv = torch.cat([(cache["v8"][0, 0, :4].double() * cache["v_scale"][0, 0, :4, None, None].double()).transpose(1, 2).flatten(0, 1), cache["v_tail"][0, 0].double().t()])
    want, bound = torch.empty(2, 1, T, 2, D, dtype=torch.float64).unbind(0)
    for i in range(T):
        x = vv[[p for p in at if p <= 300 - T + i]]
        want[0, i] = x.mean(0)
        # half a step of each weight and of the output, 2^-20 for the sums and the division
        bound[0, i] = (ref.HALF[dtype] + 2.0 ** -20) * (x.mean(0).abs() + x.abs().mean(0)) + 2.0 ** -25 * (dtype == F16)
    assert ref.within(_call(cache, q, [300 - T], window, scale), want, bound)


@pytest.mark.parametrize("T,blocks", [(1, 16), (5, 16), (70, ROOM)])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -13, 2.0 ** -17, 2.0 ** -19])
def test_light_weights_of_small_values_count(size, T, blocks):
    """A thousand tokens alike whose weights are 1.2 times 2^-13 of a key's in the tail: a seventh of the whole together, whatever the values' size and with
    a block of zeros (whose scale is 1) among them.  fp16, where weights have the fewest bits; one split, so that waves have the tail and blocks."""
    D, n = 64, 1010
    g = torch.Generator().manual_seed(11)
    k = torch.zeros(1, n, 1, D)
    v = (1 + 0.2 * torch.randn(1, n, 1, D, generator=g)) * size
    v[:, 640:704] = 0
    q = torch.zeros(1, T, 2, D)
    q[..., 0] = 1.0
    k[0, n - T, 0, 0] = (13 * math.log(2) - math.log(1.2)) / 0.125
    k, v, q = k.half(), v.half(), q.half()
    cache = _room(k, v, blocks)
    assert capi.kv8_attention_plan(1, T, 2, 1, D, blocks, 0)[0] or capi.kv8_attention_plan(1, T, 2, 1, D, blocks, 0)[1] == 1
    want, bound = ref.attention(cache, q, [n - T], None, 0.125)
    assert ref.within(_call(cache, q, [n - T]), want, bound)


@pytest.mark.parametrize("T,window", [(1, 0), (5, 0), (70, 0)])
@pytest.mark.parametrize("large,small", [(2.0 ** 100, 1.0), (2.0 ** 126, 1.0), (2.0 ** 126, 2.0 ** -40), (2.0 ** 126, 0.0), (2.0 ** 66, 2.0 ** 60)])
def test_values_of_all_sizes_count_in_the_sum_of_weights(large, small, T, window):
    """bf16 blocks whose scales lie up to 2^167 apart: the keys of the small values weigh as much as those of the large ones."""
    g = torch.Generator().manual_seed(12)
    k, v = _tokens(g, 1, 300, 1, 64, BF16), torch.randn(1, 300, 1, 64, generator=g).clamp(-1.9, 1.9) * small
    v[:, 64:128] = torch.randn(1, 64, 1, 64, generator=g).clamp(-1.9, 1.9) * large
    q = torch.randn(1, T, 2, 64, generator=g).bfloat16()
    cache = _room(k, v.bfloat16())
    want, bound = ref.attention(cache, q, [300 - T], None, 0.125)
    out = _call(cache, q, [300 - T], window)
    assert out.isfinite().all() and ref.within(out, want, bound)


@pytest.mark.parametrize("T,window", [(1, 0), (5, 0), (70, 0)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("size", ["largest", "smallest"])
def test_values_at_the_ends_of_the_type(dtype, size, T, window):
    """Values up to the largest number, whose block rounds to 256 times its scale, and fp16's down to single steps of 2^-24; in blocks and in the tail."""
    g = torch.Generator().manual_seed(13)
    k, v = _tokens(g, 1, 300, 1, 64, dtype), torch.rand(1, 300, 1, 64, generator=g) * 2 - 1
    if size == "largest":
        v = v * torch.finfo(dtype).max
        v[0, 3, 0, 9], v[0, 290, 0, 11] = torch.finfo(dtype).max, -torch.finfo(dtype).max
    else:
        v = torch.randint(-40, 41, v.shape, generator=g) * (2.0 ** -24 if dtype == F16 else 2.0 ** -62)
        v[0, 64:128] = v[0, 64:128].sign() * (2.0 ** -24 if dtype == F16 else 2.0 ** -62)
    q = torch.randn(1, T, 2, 64, generator=g).to(dtype)
    cache = _room(k, v.to(dtype))
    want, bound = ref.attention(cache, q, [300 - T], None, 0.125)
    assert ref.within(_call(cache, q, [300 - T], window), want, bound)
