"""The cache in 8 bits: what is stored, to the bit, and attention over it, against plain implementations in 64 bits."""
import math

import pytest
import torch

from tests import cache_reference as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _args(cache):
    return [cache[f] for f in ref.FIELDS]


def _words(v):
    return None if v is None else torch.tensor(v, device="cuda")


def _append(cache, k, v, start, count=None):
    import flash_gemv

    flash_gemv.cats_kv8_append(k, v, _words(start), _words(count), *_args(cache))


def _attention(cache, q, start, count=None, scale=None, window=0):
    import flash_gemv

    return flash_gemv.cats_kv8_attention(q, _words(start), _words(count), *_args(cache), q.shape[-1] ** -0.5 if scale is None else scale, window)


def _tokens(g, B, T, heads, D, dtype, spread=0.5):
    return (torch.randn(B, T, heads, D, generator=g) * torch.exp(spread * torch.randn(heads, D, generator=g))).to(dtype)


def _filled(g, B, heads, blocks, D, dtype, lengths):
    """A cache on the CPU that holds `lengths` tokens a row, NaN behind them."""
    cache = ref.new_cache(B, heads, blocks, D, dtype)
    T = max(lengths)
    return ref.append(cache, _tokens(g, B, T, heads, D, dtype), _tokens(g, B, T, heads, D, dtype), [0] * B, lengths)


# ---- storing ----

@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("pieces", [
    [[1, 1]], [[63, 64]], [[65, 1], [1, 64], [1, 1]], [[130, 200], [62, 56], [1, 1], [64, 64]], [[0, 5], [-3, 59], [1, 0]], [[256, 1]]])
def test_append_in_pieces(D, dtype, pieces):
    """Row by row: blocks that are completed, blocks that are not, tokens that a piece of one row has and another's has not, counts of 0 and
    below; every byte that is not written stays."""
    g = torch.Generator().manual_seed(D + len(pieces))
    B, heads, blocks = 2, 3, 5
    want = ref.new_cache(B, heads, blocks, D, dtype)
    got = ref.to(want, "cuda")
    at = [0, 0]
    for counts in pieces:
        T = max(max(counts), 1)
        k, v = _tokens(g, B, T, heads, D, dtype), _tokens(g, B, T, heads, D, dtype)
        want = ref.append(want, k, v, at, counts)
        _append(got, k.cuda(), v.cuda(), at, counts)
        for f in ref.FIELDS:
            assert ref.same(got[f], want[f]), (f, counts)
        at = [a + max(c, 0) for a, c in zip(at, counts)]


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_gives_the_same_whatever_the_pieces(dtype):
    g = torch.Generator().manual_seed(1)
    k, v = _tokens(g, 1, 300, 2, 64, dtype).cuda(), _tokens(g, 1, 300, 2, 64, dtype).cuda()
    caches = []
    for step in (300, 1, 37, 64, 128):
        c = ref.new_cache(1, 2, 5, 64, dtype, fill=0.0, device="cuda")
        for at in range(0, 300, step):
            _append(c, k[:, at:at + step], v[:, at:at + step], [at])
        caches.append(c)
    last = 300 // 64 * 64
    for c in caches[1:]:
        for f in ref.FIELDS:
            a, b = c[f].cpu().float(), caches[0][f].cpu().float()
            if f == "k_tail":
                a, b = a[:, :, : 300 - last], b[:, :, : 300 - last]
            if f == "v_tail":
                a, b = a[..., : 300 - last], b[..., : 300 - last]
            assert torch.equal(a, b), f


@pytest.mark.parametrize("start", [128, 129, 150, 64, 0])
def test_tokens_taken_back(start):
    """150 tokens, of which those from `start` on are replaced: within the last block, and from the start of an earlier one."""
    g = torch.Generator().manual_seed(start)
    k, v, k2, v2, q = (_tokens(g, 1, 150, n, 64, F16) for n in (2, 2, 2, 2, 4))
    c = ref.new_cache(1, 2, 4, 64, F16, device="cuda")
    _append(c, k.cuda(), v.cuda(), [0])
    _append(c, k2[:, :40].cuda(), v2[:, :40].cuda(), [start])
    both = [torch.cat((a[:, :start], b[:, :40]), 1) for a, b in ((k, k2), (v, v2))]
    want = ref.append(ref.new_cache(1, 2, 4, 64, F16), *both, [0], None)
    out = _attention(c, q[:, :40].cuda(), [start])
    assert ref.within(out, *ref.attention(want, q[:, :40], [start], None, 0.125))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_values_at_the_edges(dtype):
    """Zeros, the largest and the smallest numbers, maxima on a power of two and on 448 times one, one step above it, ties between two
    e4m3 numbers, infinities and NaN."""
    tiny, big = torch.finfo(dtype).smallest_normal, torch.finfo(dtype).max
    above = 448 * (1 + torch.finfo(dtype).eps)
    rows = [torch.zeros(64, 64), torch.full((64, 64), big), torch.full((64, 64), tiny), torch.linspace(-448, 448, 64 * 64).view(64, 64),
            torch.linspace(-1, 1, 64 * 64).view(64, 64) * above, torch.linspace(0, 2, 64 * 64).view(64, 64), torch.arange(64 * 64).view(64, 64) / 16.0 % 36]
    odd = torch.randn(64, 64, generator=torch.Generator().manual_seed(3))
    odd[3, 5], odd[9, 5], odd[63, 63] = math.inf, -math.inf, math.nan
    rows += [odd, torch.full((64, 64), math.nan), torch.full((64, 64), tiny / 8), torch.full((64, 64), 2.0 ** -62)]
    k = torch.stack(rows).to(dtype)[:, :, None].contiguous()  # (rows, 64, 1, 64)
    v = -k.flip(0)
    want = ref.append(ref.new_cache(len(rows), 1, 2, 64, dtype), k, v, [0] * len(rows), None)
    got = ref.new_cache(len(rows), 1, 2, 64, dtype, device="cuda")
    _append(got, k.cuda(), v.cuda(), [0])
    for f in ref.FIELDS:
        assert ref.same(got[f], want[f]), f


def test_append_outside_the_cache_leaves_it():
    g = torch.Generator().manual_seed(2)
    k = _tokens(g, 4, 3, 1, 64, F16).cuda()
    c = ref.new_cache(4, 1, 1, 64, F16, fill=1.0, device="cuda")
    before = {f: t.clone() for f, t in c.items()}
    _append(c, k, k, [-1, 62, 64, 1 << 40])
    for f in ref.FIELDS:
        assert ref.same(c[f], before[f]), f
    _append(c, k, k, [61])  # just inside
    assert ref.same(c["k_tail"][:, 0, 61:], k[:, :, 0])


def test_append_strides():
    """Tokens as a projection leaves them, heads in front of tokens, every second head, and elements that no vector reads."""
    g = torch.Generator().manual_seed(4)
    base = _tokens(g, 2, 70, 6, 64, BF16).cuda()
    want = ref.append(ref.new_cache(2, 3, 2, 64, BF16), base[:, :, ::2].cpu(), base[:, :, 1::2].cpu(), [0, 0], None)
    fronted = base.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.empty(2, 70, 6, 65, dtype=BF16, device="cuda")
    odd[..., 1:] = base
    reversed_elements = base.flip(-1).contiguous()
    for x in (base, fronted, odd[..., 1:], torch.empty(2, 70, 6, 128, dtype=BF16, device="cuda")[..., ::2].copy_(base)):
        c = ref.new_cache(2, 3, 2, 64, BF16, device="cuda")
        _append(c, x[:, :, ::2], x[:, :, 1::2], [0])
        for f in ref.FIELDS:
            assert ref.same(c[f], want[f]), f
    assert not torch.equal(reversed_elements, base)


# ---- attention ----

def _check(B, T, heads, kv, D, dtype, lengths, blocks, window=0, count=None, seed=0, scale=None):
    """lengths: tokens of each row with the new ones."""
    g = torch.Generator().manual_seed(seed + D + T)
    cache = _filled(g, B, kv, blocks, D, dtype, lengths)
    q = (torch.randn(B, T, heads, D, generator=g) * 1.5).to(dtype)
    n = [T] * B if count is None else [min(max(c, 0), T) for c in count]
    start = [a - c for a, c in zip(lengths, n)]
    out = _attention(ref.to(cache, "cuda"), q.cuda(), start, count, scale, window)
    want, bound = ref.attention(cache, q, start, count, D ** -0.5 if scale is None else scale, window)
    assert out.dtype == dtype and out.shape == q.shape
    worst = float(((out.cpu().double() - want).abs() / bound.clamp_min(1e-30)).nan_to_num().max())
    assert ref.within(out, want, bound), worst


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 128, 129, 300])
def test_attention_of_one_token(D, length, dtype):
    _check(1, 1, 2, 2, D, dtype, [length], 6)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (6, 2), (7, 1), (8, 1), (16, 1), (17, 1), (34, 2)])
def test_attention_of_grouped_heads(heads, kv, dtype):
    _check(2, 1, heads, kv, 64, dtype, [200, 77], 4)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,heads,kv,lengths,window", [
    (2, 3, 1, [2, 65], 0), (5, 14, 2, [130, 66], 0), (5, 14, 2, [130, 260], 70), (16, 1, 1, [16, 79], 0), (17, 1, 1, [64, 100], 0), (33, 2, 1, [33, 150], 20),
    (64, 1, 1, [64, 192], 0), (100, 3, 3, [100, 228], 64), (130, 2, 1, [130, 300], 1), (3, 4, 4, [300, 129], 129), (1, 4, 2, [300, 257], 128), (1, 4, 2, [300, 257], 1),
    (1, 4, 2, [300, 257], 1000)])
def test_attention_of_several_tokens(T, heads, kv, lengths, window, dtype):
    """Queries of one call that see different keys, in the tail, in the block before it and across windows."""
    _check(2, T, heads, kv, 64, dtype, lengths, 5, window)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("T,heads,kv,lengths,window", [(150, 3, 1, [150, 400], 0), (150, 3, 1, [400, 192], 77), (129, 2, 2, [129, 193], 0), (21, 7, 1, [21, 300], 0), (65, 1, 1, [65, 128], 0)])
def test_attention_of_prompts(T, heads, kv, lengths, window, D, dtype):
    """Many rows a workgroup: tiles of rows that end inside a token's heads, waves without a row, rows that end in the tail and before it."""
    _check(2, T, heads, kv, D, dtype, lengths, 8, window)


@pytest.mark.parametrize("dtype,D,T,lengths,window,count", [
    (F16, 128, 40, [4000, 100], 0, [40, 40]), (BF16, 64, 70, [6000, 3000], 2500, [70, 3]), (BF16, 256, 33, [1700, 1600], 0, [0, 33]), (F16, 32, 90, [3000, 2999], 64, [90, 90])])
def test_attention_of_pieces_behind_long_caches(dtype, D, T, lengths, window, count):
    """Many rows and a cache in splits, of which a short row, a window or an empty row leaves some without a tile."""
    _check(2, T, 2, 1, D, dtype, lengths, max(lengths) // 64 + 3, window, count)


@pytest.mark.parametrize("T,count,lengths", [(5, [5, 2, 0, -4], [130, 64, 70, 65]), (40, [40, 1, 17, 99], [140, 65, 128, 192]), (1, [1, 0, 1, 2], [64, 10, 1, 130])])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_of_ragged_rows(T, count, lengths, D):
    """Rows of a padded batch: those behind a row's count are zeros."""
    _check(4, T, 4, 2, D, BF16, lengths, 4, count=count)


@pytest.mark.parametrize("dtype,D,length,heads,kv", [(F16, 128, 5000, 4, 1), (BF16, 64, 20000, 2, 2), (F16, 256, 2500, 1, 1), (BF16, 32, 9001, 3, 1)])
def test_attention_over_long_caches(dtype, D, length, heads, kv):
    """Many splits of a row's cache, some rows with one, and room behind them that holds NaN."""
    _check(2, 1, heads, kv, D, dtype, [length, 70], length // 64 + 40)


def test_attention_of_a_draft_over_a_long_cache():
    _check(1, 6, 8, 2, 64, BF16, [6000], 120, window=5000)


@pytest.mark.parametrize("scale", [1e-4, 3.0, 40.0])
def test_attention_scales(scale):
    """Weights that are all alike and weights of which one is left."""
    _check(1, 3, 2, 1, 64, F16, [200], 4, scale=scale)


@pytest.mark.parametrize("T", [3, 70])
@pytest.mark.parametrize("scale", [2.0 ** -64, 2.0 ** 64])
def test_attention_scales_at_the_limits(scale, T):
    """Keys of the smallest block scale: masked weights are 0 all the same."""
    g = torch.Generator().manual_seed(T)
    k, v, q = _tokens(g, 1, 200, 1, 64, BF16) * 2.0 ** -58, _tokens(g, 1, 200, 1, 64, BF16), _tokens(g, 1, T, 2, 64, BF16)
    cache = ref.append(ref.new_cache(1, 1, 4, 64, BF16), k, v, [0], None)
    assert cache["k_scale"][0, 0, 0] == 2.0 ** -60
    out = _attention(ref.to(cache, "cuda"), q.cuda(), [200 - T], scale=scale, window=90)
    want, bound = ref.attention(cache, q, [200 - T], None, scale, 90)
    assert out.isfinite().all() and ref.within(out, want, bound)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_blocks_of_very_different_sizes(dtype):
    """The scales of the blocks lie 2^20 apart, keys' the one way and values' the other."""
    g = torch.Generator().manual_seed(9)
    size = torch.tensor([1.0, 2.0 ** -10, 2.0 ** 8, 2.0 ** -12, 1.0]).repeat_interleave(64)[:290, None, None]
    k, v = (_tokens(g, 1, 290, 1, 64, torch.float32) * size).to(dtype), (_tokens(g, 1, 290, 1, 64, torch.float32) / size.clamp_min(2.0 ** -7)).to(dtype)
    q = (torch.randn(1, 1, 2, 64, generator=g) * 0.01).to(dtype)
    cache = ref.append(ref.new_cache(1, 1, 5, 64, dtype), k, v, [0], None)
    out = _attention(ref.to(cache, "cuda"), q.cuda(), [289])
    want, bound = ref.attention(cache, q, [289], None, 0.125)
    assert ref.within(out, want, bound)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,bad_at", [(1, 10), (1, 199), (70, 10), (70, 140), (70, 150), (70, 199), (20, 150)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_attention_values_that_are_not_finite(T, bad_at, value, dtype):
    """They reach the queries that see them, in their own element (values) or all (keys), and no other query; in a complete block (200 tokens: up
    to 191) and in the tail."""
    g = torch.Generator().manual_seed(7)
    k, v = _tokens(g, 1, 200, 2, 64, dtype), _tokens(g, 1, 200, 2, 64, dtype)
    v[0, bad_at, 0, 17] = value
    k[0, bad_at, 1, 5] = value
    q = torch.randn(1, T, 4, 64, generator=g).to(dtype)
    for window in (0, 45):
        cache = ref.append(ref.new_cache(1, 2, 4, 64, dtype), k, v, [0], None)
        out = _attention(ref.to(cache, "cuda"), q.cuda(), [200 - T], window=window)
        want, bound = ref.attention(cache, q, [200 - T], None, 0.125, window)
        assert ref.within(out, want, bound), window


@pytest.mark.parametrize("T", [1, 5, 70])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_attention_of_queries_that_are_not_finite(T, value):
    """They spoil their own outputs alone."""
    g = torch.Generator().manual_seed(8)
    cache = _filled(g, 1, 1, 5, 64, F16, [300])
    q = torch.randn(1, T, 2, 64, generator=g).half()
    q[0, T - 1, 1, 9] = value
    out = _attention(ref.to(cache, "cuda"), q.cuda(), [300 - T])
    want, bound = ref.attention(cache, q, [300 - T], None, 0.125)
    assert ref.within(out, want, bound) and out[0, T - 1, 1].isnan().all()


@pytest.mark.parametrize("T", [1, 3, 70])
@pytest.mark.parametrize("window", [319, 320, 321, 2 ** 31 - 1])
def test_attention_windows_as_long_as_the_cache(T, window):
    """319 of the 320 tokens that five blocks hold, and windows that hide nothing."""
    _check(2, T, 2, 1, 64, BF16, [320, 100], 5, window)


def test_attention_tails_behind_the_last_token_hold_anything():
    """Infinities and the largest numbers where the tails have not been written."""
    g = torch.Generator().manual_seed(13)
    cache = _filled(g, 1, 1, 3, 128, F16, [140])
    q = torch.randn(1, 80, 1, 128, generator=g).half()
    want, bound = ref.attention(cache, q, [60], None, 0.1)
    for value in (math.inf, -math.inf, 65504.0):
        c = {f: t.clone() for f, t in cache.items()}
        c["k_tail"][:, :, 12:], c["v_tail"][..., 12:] = value, value
        c = ref.to(c, "cuda")
        assert ref.within(_attention(c, q.cuda(), [60], scale=0.1), want, bound)
        assert ref.within(_attention(c, q[:, 79:].cuda(), [139], scale=0.1), want[:, 79:], bound[:, 79:])


def test_two_streams_at_once():
    """Calls of two caches of one shape side by side: nothing is shared."""
    g = torch.Generator().manual_seed(14)
    caches = [ref.to(_filled(g, 1, 2, 60, 64, BF16, [3000]), "cuda") for _ in range(2)]
    q = [torch.randn(1, 1, 8, 64, generator=g).bfloat16().cuda() for _ in range(2)]
    alone = [_attention(c, x, [2999]) for c, x in zip(caches, q)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    start = _words([2999])
    import flash_gemv

    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(flash_gemv.cats_kv8_attention(q[i], start, None, *_args(caches[i]), 0.125))
    torch.cuda.synchronize()
    for a, o in zip(alone, outs):
        assert all(torch.equal(a, x) for x in o)


def test_prompt_in_a_graph():
    """A captured prompt, replayed on other tokens and another start, with splits and without."""
    import flash_gemv

    g = torch.Generator().manual_seed(15)
    for lengths in ([70, 200], [4000, 4000]):
        cache = ref.to(_filled(g, 2, 1, 70, 64, F16, lengths), "cuda")
        q, start, count = torch.zeros(2, 70, 2, 64, dtype=F16, device="cuda"), torch.tensor([0, 0], device="cuda"), torch.tensor([70], device="cuda")
        call = lambda: flash_gemv.cats_kv8_attention(q, start, count, *_args(cache), 0.125)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = call()
        torch.cuda.current_stream().wait_stream(side)
        for n in (70, 65, 70):
            q.copy_(torch.randn(2, 70, 2, 64, generator=g).half())
            start.copy_(torch.tensor([x - n for x in lengths]))
            count.fill_(n)
            graph.replay()
            got = out.clone()
            assert torch.equal(got, call()) and not got[:, :n].isnan().any()
            (q.float() ** 2).sum()


def test_what_the_operators_refuse():
    """Types, shapes and devices that do not belong together, before anything is launched."""
    import flash_gemv

    c = ref.new_cache(2, 2, 3, 128, F16, fill=0.0, device="cuda")
    x, at = torch.zeros(2, 1, 2, 128, dtype=F16, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    append = lambda k=x, v=x, start=at, count=None, **o: flash_gemv.cats_kv8_append(k, v, start, count, *(o.get(f, c[f]) for f in ref.FIELDS))
    attend = lambda q=x, start=at, count=None, scale=0.1, window=0, **o: flash_gemv.cats_kv8_attention(q, start, count, *(o.get(f, c[f]) for f in ref.FIELDS), scale, window)
    append(), attend()
    three = torch.zeros(3, dtype=torch.int64, device="cuda")
    for call in (append, attend):
        for wrong in (dict(start=at.int()), dict(start=at.cpu()), dict(start=three), dict(count=three), dict(k8=c["k8"].view(torch.uint8)), dict(v8=c["k8"]),
                      dict(k_scale=c["k_scale"].double()), dict(v_scale=c["v_scale"][:, :, :2]), dict(k_tail=c["k_tail"].bfloat16()), dict(v_tail=c["k_tail"]),
                      dict(k8=c["k8"][:, :, :2])):
            with pytest.raises(RuntimeError):
                call(**wrong)
    for wrong in (x.float(), x[0], x[..., :32], x.double(), x[:1], x.cpu()):
        with pytest.raises(RuntimeError):
            append(wrong, wrong)
        with pytest.raises(RuntimeError):
            attend(wrong)
    with pytest.raises(RuntimeError):
        append(x, x.bfloat16())
    with pytest.raises(RuntimeError):
        append(x[:, :, :1], x[:, :, :1])
    with pytest.raises(RuntimeError):
        attend(torch.zeros(2, 1, 3, 128, dtype=F16, device="cuda"))
    for wrong in (dict(window=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=1e39)):
        with pytest.raises(RuntimeError):
            attend(**wrong)
    long = torch.zeros(2, 193, 2, 128, dtype=F16, device="cuda")  # more tokens than the cache has room for
    with pytest.raises(RuntimeError):
        append(long, long)


def test_attention_outside_the_cache_is_nan():
    g = torch.Generator().manual_seed(2)
    cache = ref.to(_filled(g, 3, 1, 2, 64, F16, [100, 100, 100]), "cuda")
    q = torch.randn(3, 2, 1, 64, generator=g).half()
    out = _attention(cache, q.cuda(), [127, -1, 98], [2, 1, 2]).cpu()
    assert out[0].isnan().all() and out[1, 0].isnan().all() and (out[1, 1] == 0).all() and not out[2].isnan().any()


def test_attention_strides_and_one_start_for_all():
    g = torch.Generator().manual_seed(12)
    cache = _filled(g, 3, 2, 3, 64, BF16, [150] * 3)
    q = torch.randn(3, 4, 8, 64, generator=g).bfloat16()
    want, bound = ref.attention(cache, q[:, :, ::2], [146] * 3, None, 0.125)
    on = ref.to(cache, "cuda")
    odd = torch.empty(3, 4, 8, 65, dtype=BF16, device="cuda")
    odd[..., 1:] = q.cuda()
    for x in (q.cuda(), q.transpose(1, 2).contiguous().cuda().transpose(1, 2), odd[..., 1:]):
        assert ref.within(_attention(on, x[:, :, ::2], [146]), want, bound)
    one = _attention(on, q[:1, :1].cuda().expand(3, 4, 8, 64)[:, :, ::2], [146])  # a stride of nothing
    want, bound = ref.attention(cache, q[:1, :1].expand(3, 4, 8, 64)[:, :, ::2], [146] * 3, None, 0.125)
    assert ref.within(one, want, bound)


def test_empty_calls():
    import flash_gemv

    c = ref.new_cache(2, 1, 1, 64, F16, fill=0.0, device="cuda")
    z = torch.empty(2, 0, 1, 64, dtype=F16, device="cuda")
    flash_gemv.cats_kv8_append(z, z, _words([0]), None, *_args(c))
    assert flash_gemv.cats_kv8_attention(z, _words([0]), None, *_args(c), 0.125).shape == (2, 0, 1, 64)


def test_steps_on_another_stream_and_in_a_graph():
    """A row that grows over the end of a block, eagerly on a stream of its own and replayed from a graph, with other work between."""
    import flash_gemv

    g = torch.Generator().manual_seed(5)
    k, v, q = (_tokens(g, 2, 140, n, 64, F16).cuda() for n in (2, 2, 4))
    states = []
    for graph in (False, True):
        c = ref.new_cache(2, 2, 40, 64, F16, fill=0.0, device="cuda")
        _append(c, k[:, :120], v[:, :120], [0])
        kk, vv, qq, at = k[:, 0:1].clone(), v[:, 0:1].clone(), q[:, 0:1].clone(), torch.tensor([120], device="cuda")
        outs = []
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            def step():
                flash_gemv.cats_kv8_append(kk, vv, at, None, *_args(c))
                return flash_gemv.cats_kv8_attention(qq, at, None, *_args(c), 0.125)

            if graph:
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured, stream=side):
                    out = step()
            for p in range(120, 140):
                kk.copy_(k[:, p:p + 1]), vv.copy_(v[:, p:p + 1]), qq.copy_(q[:, p:p + 1]), at.fill_(p)
                if graph:
                    captured.replay()
                else:
                    out = step()
                outs.append(out.clone())
                (qq @ qq.transpose(2, 3).contiguous()).sum()
        side.synchronize()
        states.append((outs, c))
    for a, b in zip(*(s[0] for s in states)):
        assert torch.equal(a, b)
    for f in ref.FIELDS:
        assert ref.same(states[0][1][f], states[1][1][f])
    cpu = {f: t.cpu() for f, t in states[0][1].items()}
    want, bound = ref.attention(cpu, q[:, 139:140].cpu(), [139, 139], None, 0.125)
    assert ref.within(states[0][0][-1], want, bound)


def test_results_do_not_change_from_call_to_call():
    g = torch.Generator().manual_seed(6)
    c = ref.to(_filled(g, 2, 2, 60, 64, BF16, [3500, 900]), "cuda")
    q = torch.randn(2, 1, 8, 64, generator=g).bfloat16().cuda()
    first = _attention(c, q, [3499, 899])
    for _ in range(5):
        assert torch.equal(_attention(c, q, [3499, 899]), first)


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes of keys and of values, its last tokens, by the step's and the prompt's kernel."""
    from cats_amd import capi
    from cats_amd.kv8 import Kv8Cache

    g = torch.Generator().manual_seed(12)
    blocks, behind = 70000, 192  # zeros in front of the new tokens, as many as the window reaches back
    c = Kv8Cache(1, 8, blocks * 64, 128, BF16)
    small = ref.new_cache(1, 8, 20, 128, BF16, fill=0.0)
    small["k_scale"].fill_(1.0), small["v_scale"].fill_(1.0)
    start = blocks * 64 - 1024
    for T, at in ((700, 0), (1, 700)):
        assert capi.kv8_attention_plan(1, T, 32, 8, 128, blocks, 150)[0] == (T > 1)
        k, v, q = (_tokens(g, 1, T, n, 128, BF16) for n in (8, 8, 32))
        small = ref.append(small, k, v, [behind + at], None)
        c.append(k.cuda(), v.cuda(), _words([start + at]))
        out = c.attend(q.cuda(), _words([start + at]), window=150)
        assert ref.within(out, *ref.attention(small, q, [behind + at], None, 128 ** -0.5, 150))
    assert torch.equal(c.k8[0, :, start // 64:start // 64 + 10].cpu().float(), small["k8"][0, :, 3:13].float())
    assert torch.equal(c.v8[0, :, start // 64:start // 64 + 10].cpu().float(), small["v8"][0, :, 3:13].float())


def test_gradients_are_refused():
    """What records a gradient would be cut off from it; under no_grad, and detached, the same tensors are taken."""
    from cats_amd.kv8 import Kv8Cache

    c = Kv8Cache(1, 1, 64, 64, F16)
    x, at = torch.randn(1, 2, 1, 64, dtype=F16, device="cuda"), _words([0])
    w = x.clone().requires_grad_()
    for call in (lambda: c.append(w, x, at), lambda: c.append(x, w, at), lambda: c.attend(w, at), lambda: c.attend(w * 2, at)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    assert not c.k_tail.any() and not c.v_tail.any()
    c.append(w.detach(), x, at)
    with torch.no_grad():
        c.append(w, w, at)
        out = c.attend(w, at)
    assert torch.equal(out, c.attend(x, at)) and not out.requires_grad


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("accepted", [[0, 0, 0], [1, 2, 5], [4, 3, 1]])
def test_drafts_past_the_end_of_a_block_are_taken_back(accepted, dtype):
    """Rows at 62, 60 and 127 tokens, five drafted ones, fewer kept: with the tails put back and the accepted tokens stored again a cache is what it
    would be without the draft, and goes on over the block's end to the same bytes."""
    from cats_amd.kv8 import Kv8Cache

    g = torch.Generator().manual_seed(sum(accepted))
    at = [62, 60, 127]
    k, v, draft_k, draft_v, more_k, more_v, q = (_tokens(g, 3, n, h, 64, dtype).cuda() for n, h in ((127, 2), (127, 2), (5, 2), (5, 2), (70, 2), (70, 2), (70, 4)))
    caches = [Kv8Cache(3, 2, 256, 64, dtype) for _ in range(2)]
    start, end = _words(at), _words([a + n for a, n in zip(at, accepted)])
    for c in caches:
        c.append(k, v, _words([0]), start)
    drafted, plain = caches
    kept = drafted.k_tail.clone(), drafted.v_tail.clone()
    drafted.append(draft_k, draft_v, start)
    assert drafted.attend(q[:, :5], start).isfinite().all()
    drafted.k_tail.copy_(kept[0]), drafted.v_tail.copy_(kept[1])
    for c in caches:
        c.append(draft_k, draft_v, start, _words(accepted))
    one = more_k[:, :1], more_v[:, :1]
    for c in caches:
        c.append(*one, end)
    assert torch.equal(drafted.attend(q[:, :1], end), plain.attend(q[:, :1], end))
    for c in caches:
        c.append(more_k[:, 1:], more_v[:, 1:], end + 1)
    assert torch.equal(drafted.attend(q[:, 1:], end + 1), plain.attend(q[:, 1:], end + 1))
    for b, e in enumerate((end + 70).tolist()):
        full = (e - 1) // 64
        for f in ("k8", "v8", "k_scale", "v_scale"):
            assert ref.same(getattr(drafted, f)[b, :, :full], getattr(plain, f)[b, :, :full]), f
        assert ref.same(drafted.k_tail[b, :, : e - full * 64], plain.k_tail[b, :, : e - full * 64])
        assert ref.same(drafted.v_tail[b, ..., : e - full * 64], plain.v_tail[b, ..., : e - full * 64])


def test_elements_in_any_order():
    """Strides that no vector reads: every second element, elements in front of heads, a transposed batch; the same as of a copy."""
    g = torch.Generator().manual_seed(16)
    wide = _tokens(g, 3, 70, 2, 128, F16).cuda()
    turned = _tokens(g, 3, 70, 64, 2, F16).cuda().transpose(2, 3)
    batch = _tokens(g, 70, 3, 2, 64, F16).cuda().transpose(0, 1)
    for x in (wide[..., ::2], wide[..., 1::2], turned, batch, batch[:, ::7], wide.flip(-1)[..., 64:]):
        T = x.shape[1]
        want = ref.append(ref.new_cache(3, 2, 2, 64, F16), x.cpu(), x.cpu(), [0] * 3, None)
        c = ref.new_cache(3, 2, 2, 64, F16, device="cuda")
        _append(c, x, x, [0])
        for f in ref.FIELDS:
            assert ref.same(c[f], want[f]), f
        assert torch.equal(_attention(c, x, [0]), _attention(c, x.contiguous(), [0])) and x.shape == (3, T, 2, 64)
