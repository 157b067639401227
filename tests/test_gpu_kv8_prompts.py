"""Attention over a cache in 8 bits by the kernel for many tokens, at the sizes and masks where it can go wrong.  Which kernel a call takes goes by its
work, so the caches have room for more than they hold; each test asks which one it was."""
import math

import pytest
import torch

from cats_amd import capi
from tests import cache_reference as ref
from tests.test_gpu_kv8 import BF16, F16, _args, _attention, _check, _filled, _tokens, _words

pytestmark = pytest.mark.gpu


def _many(B, T, heads, kv, D, blocks, window=0, splits=None):
    """Asserts that such a call is for this kernel (and how many splits it has)."""
    prompt, n = capi.kv8_attention_plan(B, T, heads, kv, D, blocks, window)
    assert prompt and (splits is None or (n > 1) == (splits > 1))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("T,heads,kv,lengths,blocks", [
    (150, 3, 1, [150, 400], 90), (129, 2, 2, [129, 193], 145), (21, 7, 1, [21, 300], 260), (65, 1, 1, [65, 128], 520), (33, 1, 1, [64, 1100], 850), (17, 1, 1, [17, 18], 1300)])
def test_prompts(T, heads, kv, lengths, blocks, D, dtype):
    """Tiles of rows that end inside a token's heads, waves without a row, rows that end in the tail and before it, odd numbers of tiles."""
    _many(2, T, heads, kv, D, blocks, splits=2)
    _check(2, T, heads, kv, D, dtype, lengths, blocks)


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64), (F16, 32), (BF16, 256)])
@pytest.mark.parametrize("lengths", [[63, 1250], [64, 1280], [127, 129]])
def test_prompts_that_are_not_split(lengths, dtype, D):
    _many(2, 63, 32, 4, D, 20, splits=1)
    _check(2, 63, 32, 4, D, dtype, lengths, 20)


@pytest.mark.parametrize("T,heads,kv,window,D,dtype,lengths", [
    (80, 32, 4, 1000, 128, F16, [1250, 700]), (160, 64, 8, 77, 64, BF16, [700, 160]), (210, 64, 8, 1, 32, F16, [300, 210]), (210, 64, 8, 64, 128, BF16, [1000, 257]),
    (40, 64, 8, 900, 256, BF16, [1250, 41])])
def test_windows(T, heads, kv, window, D, dtype, lengths):
    """Tiles that a window cuts and tiles that it hides, before and in the tail."""
    _many(2, T, heads, kv, D, 20, window)
    _check(2, T, heads, kv, D, dtype, lengths, 20, window)


@pytest.mark.parametrize("dtype,D,T,heads,kv,lengths,blocks,window,count", [
    (F16, 128, 40, 2, 1, [4000, 100], 520, 0, [40, 40]), (BF16, 64, 70, 32, 4, [6000, 3000], 96, 2500, [70, 3]), (BF16, 256, 33, 2, 1, [3000, 2900], 520, 0, [0, 33]),
    (F16, 32, 90, 2, 1, [3000, 2999], 230, 0, [90, 90]), (F16, 64, 40, 2, 1, [2048, 1024], 520, 0, [40, 17])])
def test_pieces_behind_long_caches(dtype, D, T, heads, kv, lengths, blocks, window, count):
    """Splits of which a short row, a window or an empty row leaves some without a tile."""
    _many(2, T, heads, kv, D, blocks, window, splits=2)
    _check(2, T, heads, kv, D, dtype, lengths, blocks, window, count)


@pytest.mark.parametrize("count,lengths", [([40, 1, 17, 99], [140, 65, 128, 192]), ([0, -4, 40, 2], [50, 60, 40, 130])])
@pytest.mark.parametrize("D", [64, 128])
def test_padded_batches(count, lengths, D):
    _many(4, 40, 4, 2, D, 140)
    _check(4, 40, 4, 2, D, BF16, lengths, 140, count=count)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("bad_at", [10, 131, 140, 150, 191, 192, 199])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite(bad_at, value, D, dtype):
    """They reach the queries that see them, and no other: in tiles that all see, in the queries' own, and in the tail."""
    g = torch.Generator().manual_seed(7)
    k, v = _tokens(g, 1, 200, 2, D, dtype), _tokens(g, 1, 200, 2, D, dtype)
    v[0, bad_at, 0, 17] = value
    k[0, bad_at, 1, 5] = value
    q = torch.randn(1, 70, 4, D, generator=g).to(dtype)
    cache = ref.append(ref.new_cache(1, 2, 300, D, dtype), k, v, [0], None)
    _many(1, 70, 4, 2, D, 300)
    out = _attention(ref.to(cache, "cuda"), q.cuda(), [130])
    assert ref.within(out, *ref.attention(cache, q, [130], None, D ** -0.5))


@pytest.mark.parametrize("bad_at", [20, 70, 140, 199])
def test_values_that_are_not_finite_and_windows(bad_at):
    g = torch.Generator().manual_seed(7)
    k, v, q = _tokens(g, 1, 330, 16, 64, F16), _tokens(g, 1, 330, 16, 64, F16), torch.randn(1, 210, 128, 64, generator=g).half()
    v[0, bad_at, 3, 17] = math.nan
    k[0, bad_at, 5, 5] = math.inf
    cache = ref.append(ref.new_cache(1, 16, 6, 64, F16), k, v, [0], None)
    _many(1, 210, 128, 16, 64, 6, 45)
    out = _attention(ref.to(cache, "cuda"), q.cuda(), [120], window=45)
    heads = torch.tensor([0, 24, 31, 40, 47, 127])  # of cached heads 0, 3, 5 and 15
    part = {f: t[:, [0, 3, 3, 5, 5, 15]] for f, t in cache.items()}
    assert ref.within(out[:, :, heads.cuda()], *ref.attention(part, q[:, :, heads], [120], None, 0.125, 45))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_queries_that_are_not_finite(value):
    g = torch.Generator().manual_seed(8)
    cache = _filled(g, 1, 1, 600, 64, F16, [300])
    q = torch.randn(1, 70, 2, 64, generator=g).half()
    q[0, 69, 1, 9] = value
    _many(1, 70, 2, 1, 64, 600)
    out = _attention(ref.to(cache, "cuda"), q.cuda(), [230])
    assert ref.within(out, *ref.attention(cache, q, [230], None, 0.125)) and out[0, 69, 1].isnan().all()


def test_tails_behind_the_last_token_hold_anything():
    g = torch.Generator().manual_seed(13)
    cache = _filled(g, 1, 1, 1100, 128, F16, [140])
    q = torch.randn(1, 80, 1, 128, generator=g).half()
    want, bound = ref.attention(cache, q, [60], None, 0.1)
    _many(1, 80, 1, 1, 128, 1100)
    for value in (math.inf, -math.inf, 65504.0):
        c = {f: t.clone() for f, t in cache.items()}
        c["k_tail"][:, :, 12:], c["v_tail"][..., 12:] = value, value
        assert ref.within(_attention(ref.to(c, "cuda"), q.cuda(), [60], scale=0.1), want, bound)


@pytest.mark.parametrize("scale", [2.0 ** -64, 1e-4, 3.0, 40.0, 2.0 ** 64])
def test_scales(scale):
    """Weights that are all alike and weights of which one is left; keys of the smallest block scale."""
    g = torch.Generator().manual_seed(5)
    k, v, q = _tokens(g, 1, 200, 1, 64, BF16), _tokens(g, 1, 200, 1, 64, BF16), _tokens(g, 1, 70, 2, 64, BF16)
    if not 1e-5 < scale < 100:
        k = k * 2.0 ** -58
    cache = ref.append(ref.new_cache(1, 1, 600, 64, BF16), k, v, [0], None)
    _many(1, 70, 2, 1, 64, 600)
    out = _attention(ref.to(cache, "cuda"), q.cuda(), [130], scale=scale)
    want, bound = ref.attention(cache, q, [130], None, scale)
    assert out.isfinite().all() and ref.within(out, want, bound)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_blocks_of_very_different_sizes(dtype):
    """Maxima that grow and fall by 2^20 from block to block, keys' scales the one way and values' the other."""
    g = torch.Generator().manual_seed(9)
    size = torch.tensor([1.0, 2.0 ** -10, 2.0 ** 8, 2.0 ** -12, 1.0]).repeat_interleave(64)[:290, None, None]
    k, v = (_tokens(g, 1, 290, 1, 64, torch.float32) * size).to(dtype), (_tokens(g, 1, 290, 1, 64, torch.float32) / size.clamp_min(2.0 ** -7)).to(dtype)
    q = (torch.randn(1, 80, 2, 64, generator=g) * 0.01).to(dtype)
    cache = ref.append(ref.new_cache(1, 1, 600, 64, dtype), k, v, [0], None)
    _many(1, 80, 2, 1, 64, 600)
    out = _attention(ref.to(cache, "cuda"), q.cuda(), [210])
    assert ref.within(out, *ref.attention(cache, q, [210], None, 0.125))


def test_outside_the_cache_and_from_call_to_call_and_in_a_graph():
    """NaN where the tokens do not lie in the cache; the same bits each time, eagerly, replayed, and from strided queries."""
    import flash_gemv

    g = torch.Generator().manual_seed(10)
    cache = ref.to(_filled(g, 2, 2, 600, 128, F16, [3000, 2000]), "cuda")
    wide = torch.randn(2, 90, 4, 136, generator=g).half().cuda()
    q = wide[..., :128]
    _many(2, 90, 4, 2, 128, 600, splits=2)
    first = _attention(cache, q.contiguous(), [2910, 1910])
    out = _attention(cache, q, [2910, 600 * 64 - 89])
    assert torch.equal(out[0], first[0]) and out[1].isnan().all()
    start = _words([2910, 1910])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = flash_gemv.cats_kv8_attention(q, start, None, *_args(cache), 128 ** -0.5)
        for _ in range(4):
            captured.fill_(7.0)
            graph.replay()
            (q @ q.transpose(2, 3).contiguous()).sum()
            assert torch.equal(captured, first)
            assert torch.equal(_attention(cache, q, [2910, 1910]), first)
    side.synchronize()


@pytest.mark.parametrize("blocks,lengths", [(20, [1200, 80]), (600, [5000, 900])])
def test_replayed_on_other_tokens(blocks, lengths):
    """A captured call of the kernel for many tokens without splits and with them, replayed on other queries, starts and counts, with other work between."""
    import flash_gemv

    g = torch.Generator().manual_seed(17)
    heads, kv = (32, 4) if blocks == 20 else (2, 1)
    _many(2, 63, heads, kv, 64, blocks, splits=1 if blocks == 20 else 2)
    cache = ref.to(_filled(g, 2, kv, blocks, 64, F16, lengths), "cuda")
    q, start, count = torch.zeros(2, 63, heads, 64, dtype=F16, device="cuda"), _words([0, 0]), _words([63, 63])
    call = lambda: flash_gemv.cats_kv8_attention(q, start, count, *_args(cache), 0.125)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call()
    torch.cuda.current_stream().wait_stream(side)
    for n in ([63, 63], [63, 1], [0, 40], [5, 63]):
        q.copy_(torch.randn(2, 63, heads, 64, generator=g).half())
        start.copy_(torch.tensor([a - b for a, b in zip(lengths, n)]))
        count.copy_(torch.tensor(n))
        out.fill_(7.0)
        graph.replay()
        got = out.clone()
        (q.float() ** 2).sum()
        assert torch.equal(got, call())
        for b in range(2):
            assert not got[b, n[b]:].any() and got[b, : n[b]].isfinite().all()
