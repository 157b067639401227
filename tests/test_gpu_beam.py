"""Beam search's selection and the moving of caches, against plain implementations in 64 bits."""
import math

import pytest
import torch

from tests import cache_reference as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _check(logits, scores, finished=None, eos=-1, keep=0):
    import flash_gemv

    n = keep or logits.shape[1]
    got = flash_gemv.cats_beam_select(logits.cuda(), scores.cuda(), None if finished is None else finished.cuda(), eos, keep)
    want = ref.select(logits, scores, finished, eos, n)
    best, parents, tokens, done = (t.cpu() for t in got)
    assert best.shape == (logits.shape[0], n) and best.dtype == F32 and parents.dtype == tokens.dtype == torch.int64 and done.dtype == torch.bool
    assert parents.tolist() == [[w[1] for w in g] for g in want]
    assert tokens.tolist() == [[w[2] for w in g] for g in want]
    assert done.tolist() == [[w[3] for w in g] for g in want]
    # the score is rounded once; the logarithm's sum is one of 32-bit exponentials
    w = torch.tensor([[x[0] for x in g] for g in want], dtype=torch.float64)
    near = (best.double() - w).abs() <= 2.0 ** -24 * w.abs() + 4 * 2.0 ** -23
    assert bool((near | ((best == -math.inf) & (w == -math.inf))).all())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("G,n,V,keep", [
    (1, 1, 1, 0), (1, 1, 2, 2), (1, 2, 1, 0), (2, 3, 5, 0), (1, 4, 32000, 0), (3, 4, 2047, 0), (2, 8, 2048, 3), (1, 16, 2049, 0), (5, 16, 70, 16), (1, 1, 100003, 16),
    (40, 8, 8193, 0), (70, 16, 3001, 0), (2, 5, 50257, 7)])
def test_select(G, n, V, keep, dtype):
    """Rows of one word and of many pieces, whole and not, in both sizes of a piece; fewer and more beams kept than there are."""
    g = torch.Generator().manual_seed(V + G)
    # far from ties between rows: totals of different rows differ by more than the logarithm's error unless the draw is unlucky
    _check((torch.randn(G, n, V, generator=g) * 3).to(dtype), -5 * torch.rand(G, n, generator=g), keep=keep)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("V", [3, 64, 3000, 40000, 180000])
def test_ties_go_to_the_lowest(V, dtype):
    """All logits equal, few values, zeros of both signs, and rows with the same score: more equal values than a wave gathers."""
    g = torch.Generator().manual_seed(V)
    zero = torch.zeros(2, 3, V, dtype=dtype)
    s = torch.tensor([[0.0, 0.0, -1.0], [-2.0, -1.0, -1.0]])
    _check(zero, s)
    _check(torch.where(torch.rand(2, 3, V, generator=g) < 0.5, zero, -zero), s)
    _check(torch.randint(0, 3, (1, 1, V), generator=g).to(dtype), torch.zeros(1, 1), keep=3)
    up = torch.arange(V).float().expand(1, 2, V).div(V / 4).to(dtype)  # ascending: every wave's last lanes hold the best
    _check(up, torch.tensor([[0.0, -0.3]]))
    _check(up.flip(-1).contiguous(), torch.tensor([[0.0, -0.3]]))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,V", [(1, 2000), (256, 8100), (256, 20001)])
def test_more_candidates_than_are_gathered(rows, V, dtype):
    """Equal best values spread over the waves of a workgroup, or in one of them, and few words left side by side, in both sizes of a piece."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(rows // min(rows, 16), min(rows, 16), V, generator=g).to(dtype)
    s = -torch.arange(min(rows, 16)).float().expand(x.shape[:2]).contiguous()
    spread = x.clone()
    spread[..., torch.randperm(min(V, 8000), generator=g)[:100]] = 10.0
    _check(spread, s)
    one = x.clone()
    one[..., 300:400] = 10.0
    one[..., torch.randperm(V, generator=g)[:3]] = 11.0
    _check(one, s)
    left = torch.full_like(x, -math.inf)
    left[..., 200:300] = x[..., 200:300]
    _check(left, s)


@pytest.mark.parametrize("V", [40, 9000, 140000])
def test_select_at_the_start_and_where_words_are_masked(V):
    """Beams that take no part yet, words at -infinity and at the type's lowest value, fewer words left than beams, rows with a NaN or +infinity."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(2, 4, V, generator=g)
    none = -math.inf
    _check(x, torch.tensor([[0.0, none, none, none], [none, none, -1.0, none]]))
    masked = x.clone()
    masked[:, :, 2:] = none
    _check(masked, torch.zeros(2, 4) - torch.arange(4))
    masked[0, :, :] = none
    _check(masked, torch.zeros(2, 4) - torch.arange(4))
    low = x.clone()
    low[:, :, ::2] = torch.finfo(F32).min
    _check(low, torch.zeros(2, 4) - torch.arange(4) * 0.1)
    odd = x.clone()
    odd[0, 0, 7], odd[0, 1, 3], odd[1, 2, 11] = math.nan, math.inf, -math.inf
    _check(odd, torch.zeros(2, 4) - torch.arange(4) * 0.1)
    _check(x, torch.tensor([[math.nan, 0.0, math.inf, -1.0], [none, none, none, none]]))


@pytest.mark.parametrize("V,eos", [(50, 0), (50, 49), (50, 3), (20000, 2), (140000, 100000)])
def test_finished_beams_go_on_alone(V, eos):
    g = torch.Generator().manual_seed(V + eos)
    x = torch.randn(4, 4, V, generator=g).half()
    s = -torch.rand(4, 4, generator=g) * 4
    done = torch.tensor([[True, False, False, True], [True, True, True, True], [False] * 4, [False, True, True, True]])
    x[1, 0] = math.nan  # a finished beam's logits are not read
    _check(x, s, done, eos)
    _check(x, s, done, eos, keep=6)  # more than four finished beams offer: the rest at -infinity
    s[0, 0] = -math.inf
    _check(x, s, done, eos)
    x[1, 0] = 0
    _check(x, s, None, eos)


def test_select_reads_the_last_position_in_place():
    import flash_gemv

    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, 5, 1001, generator=g)
    s = -torch.rand(2, 3, generator=g)
    for part in (x[:, -1].view(2, 3, 1001), x[:, 1].unflatten(0, (2, 3)), x.permute(2, 0, 1)[:700, :, 2].t().unflatten(0, (2, 3))):
        _check(part, s)
    out = flash_gemv.cats_beam_select(x.cuda()[:, -1].unflatten(0, (2, 3)), s.cuda())
    assert out[1].tolist() == [[w[1] for w in g] for g in ref.select(x[:, -1].view(2, 3, 1001), s, None, -1, 3)]


def _caches(g, rows, length):
    """One of each kind: 16-byte entries, 4-byte entries, blocks, whole tails; odd numbers of heads and entries."""
    r = lambda *s: torch.randint(-2 ** 31, 2 ** 31 - 1, s, generator=g, dtype=torch.int32)
    return [r(rows, 3, 77, 8), r(rows, 2, 5, 16, 8), r(rows, 2, 5), r(rows, 1, 64, 4), r(rows, 5, 301, 3), r(rows, 1, 1, 4)], [1, 64, 64, 0, 1, 0]


@pytest.mark.parametrize("G,n", [(1, 2), (3, 4), (2, 5), (1, 8), (2, 16), (1, 1)])
@pytest.mark.parametrize("length", [[0], [1], [64], [65], [77], [1000], None])
def test_reorder(G, n, length):
    import flash_gemv

    g = torch.Generator().manual_seed(G * 100 + n)
    if length is None:  # a length for each row
        length = torch.randint(-2, 400, (G * n,), generator=g).tolist()
    caches, slots = _caches(g, G * n, length)
    parents = torch.randint(0, n, (G, n), generator=g)
    got = [c.cuda() for c in caches]
    flash_gemv.cats_cache_reorder(got, slots, parents.cuda(), torch.tensor(length, device="cuda"))
    for c, s, x in zip(caches, slots, got):
        assert torch.equal(x.cpu(), ref.reorder(c, s, parents, length))


@pytest.mark.parametrize("parents", [[[1, 0, 3, 2]], [[3, 3, 3, 3]], [[0, 1, 2, 3]], [[1, 2, 3, 0]], [[-1, 0, 4, 1 << 40]]])
def test_reorder_cycles_and_parents_that_are_none(parents):
    import flash_gemv

    g = torch.Generator().manual_seed(1)
    caches, slots = _caches(g, 4, 70)
    got = [c.cuda() for c in caches]
    flash_gemv.cats_cache_reorder(got, slots, torch.tensor(parents, device="cuda"), torch.tensor([70], device="cuda"))
    for c, s, x in zip(caches, slots, got):
        assert torch.equal(x.cpu(), ref.reorder(c, s, torch.tensor(parents), [70]))


def test_reorder_of_many_caches_and_off_a_boundary():
    """More caches than a launch holds; views that start inside 16 bytes; 16-bit, 8-bit and empty ones."""
    import flash_gemv

    g = torch.Generator().manual_seed(8)
    parents = torch.tensor([[2, 0, 1], [0, 0, 2]])
    caches = [torch.randint(0, 100, (6, 2, 9 + i, 4), generator=g, dtype=torch.int16) for i in range(70)]
    caches += [torch.randint(0, 100, (6, 1, 40, 8), generator=g, dtype=torch.uint8), torch.empty(6, 0, 4, 4, dtype=torch.int16)]
    buf = torch.zeros(6 * 33 * 4 + 1, dtype=torch.int32, device="cuda")
    off = buf[1:].view(6, 1, 33, 4)
    off.copy_(torch.randint(0, 100, (6, 1, 33, 4), generator=g))
    want = [ref.reorder(c, 1, parents, [12]) for c in caches] + [ref.reorder(off.cpu(), 1, parents, [12])]
    got = [c.cuda() for c in caches] + [off]
    flash_gemv.cats_cache_reorder(got, [1] * len(got), parents.cuda(), torch.tensor([12], device="cuda"))
    for x, w in zip(got, want):
        assert torch.equal(x.cpu(), w)
    flash_gemv.cats_cache_reorder([torch.zeros(6, 1, 3, 4, device="cuda")], [0], parents.cuda())  # no lengths are needed


def test_large_reorder():
    import flash_gemv

    g = torch.Generator(device="cuda").manual_seed(8)
    c = torch.randint(0, 1 << 30, (8, 4, 4096, 64), generator=g, device="cuda", dtype=torch.int32)
    parents = torch.tensor([[1, 1, 0, 3], [2, 3, 1, 0]], device="cuda")
    rows = (parents + torch.tensor([[0], [4]], device="cuda")).view(-1)
    want = c.clone()
    want[:, :, :3001] = c[rows][:, :, :3001]
    flash_gemv.cats_cache_reorder([c], [1], parents, torch.tensor([3001], device="cuda"))
    assert torch.equal(c, want)


def test_a_step_in_a_graph():
    """Selection and moving, replayed on new logits, against the same calls made eagerly."""
    import flash_gemv

    g = torch.Generator(device="cuda").manual_seed(4)
    x = [torch.randn(2, 4, 5000, generator=g, device="cuda") for _ in range(4)]
    cache = torch.randn(8, 2, 50, 8, generator=g, device="cuda")
    results = []
    for graph in (False, True):
        c, scores, done, logits = cache.clone(), torch.zeros(2, 4, device="cuda"), torch.zeros(2, 4, dtype=torch.bool, device="cuda"), x[0].clone()
        length = torch.tensor([20], device="cuda")

        def step():
            s, p, t, d = flash_gemv.cats_beam_select(logits, scores, done, 17)
            flash_gemv.cats_cache_reorder([c], [1], p, length)
            scores.copy_(s), done.copy_(d)
            return p, t

        if graph:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured, stream=side):
                out = step()
            torch.cuda.current_stream().wait_stream(side)
        seen = []
        for i in range(4):
            logits.copy_(x[i])
            if graph:
                captured.replay()
            else:
                out = step()
            seen += [o.clone() for o in out] + [scores.clone(), done.clone(), c.clone()]
            torch.randn(100, device="cuda").sum()
        torch.cuda.synchronize()
        results.append(seen)
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_what_the_operators_refuse():
    import flash_gemv

    x, s = torch.zeros(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    done = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    flash_gemv.cats_beam_select(x, s, done, 4)
    for args in ((x[0], s), (x.double(), s), (x, s.double()), (x, s[:1]), (x, s.cpu()), (x, s, done[:1], 4), (x, s, done.int(), 4), (x, s, done), (x, s, None, 50),
                 (x, s, None, -1, 17), (x, s, None, -1, -1), (x[:, :1, :2], s[:, :1].contiguous(), None, -1, 3), (torch.zeros(1, 17, 50, device="cuda"), torch.zeros(1, 17, device="cuda"))):
        with pytest.raises(RuntimeError):
            flash_gemv.cats_beam_select(*args)
    c, p, n = torch.zeros(6, 2, 5, 4, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.tensor([3], device="cuda")
    flash_gemv.cats_cache_reorder([c], [1], p, n)
    for args in (([c], [1], p), ([c], [1, 1], p, n), ([], [], p, n), ([c], [-1], p, n), ([c[:5]], [1], p, n), ([c[0]], [1], p, n), ([c], [1], p.int(), n),
                 ([c], [1], p[0], n), ([c], [1], p, n.int()), ([c], [1], p, torch.zeros(2, dtype=torch.int64, device="cuda")), ([c.transpose(1, 2)], [1], p, n),
                 ([c.to(torch.uint8)[..., :3].contiguous()], [1], p, n), ([c.cpu()], [1], p, n), ([c], [1], p.cpu(), n)):
        with pytest.raises(RuntimeError):
            flash_gemv.cats_cache_reorder(*args)


def test_reorder_with_a_length_that_no_cache_has():
    import flash_gemv

    c = torch.arange(2 * 5 * 4, dtype=torch.int32).view(2, 1, 5, 4)
    got = c.cuda()
    flash_gemv.cats_cache_reorder([got], [64], torch.tensor([[1, 0]], device="cuda"), torch.tensor([2 ** 63 - 1], device="cuda"))
    assert torch.equal(got.cpu(), c.flip(0))


def test_offsets_beyond_32_bits():
    """Logits whose rows lie 2^32 bytes apart, and a row of a cache of more than 2^32 bytes."""
    import flash_gemv

    g = torch.Generator().manual_seed(6)
    x, s = torch.randn(1, 3, 1000, generator=g).half(), -torch.rand(1, 3, generator=g)
    far = torch.empty(2 ** 32 + 2000, dtype=F16, device="cuda").as_strided((1, 3, 1000), (0, 2 ** 31 + 8, 1))
    far.copy_(x)
    _check(x, s)
    for a, b in zip(flash_gemv.cats_beam_select(far, s.cuda()), flash_gemv.cats_beam_select(x.cuda(), s.cuda())):
        assert torch.equal(a, b)
    del far
    torch.cuda.empty_cache()
    entries = 2 ** 28 + 1000
    c = torch.zeros(2, 1, entries, 4, dtype=torch.int32, device="cuda")
    last = torch.randint(1, 1 << 30, (2, 1, 2000, 4), generator=g, dtype=torch.int32)
    c[:, :, -2000:] = last.cuda()
    flash_gemv.cats_cache_reorder([c], [1], torch.tensor([[1, 0]], device="cuda"), torch.tensor([entries - 3], device="cuda"))
    assert torch.equal(c[:, :, -2000:-3].cpu(), last.flip(0)[:, :, :-3]) and torch.equal(c[:, :, -3:].cpu(), last[:, :, -3:])
    assert int(c[:, :, :-2000].max()) == 0


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("G,n,V", [(1, 2, 50257), (3, 8, 50257), (2, 4, 1001), (1, 16, 100003), (40, 8, 8193), (2, 2, 7)])
def test_rows_that_are_the_same_tie(G, n, V, dtype):
    """The same logits and scores in every beam, in rows that start at every offset within 16 bytes: their totals are the same to the bit, so each word's beams
    come in order."""
    g = torch.Generator().manual_seed(V + n)
    x = (torch.randn(G, 1, V, generator=g) * 3).to(dtype).expand(G, n, V).contiguous()
    s = torch.full((G, n), -1.25)
    _check(x, s)
    import flash_gemv

    for pitch in (V + 1, V + 3, V + 8):
        far = torch.zeros(G * n * pitch + 5, dtype=dtype, device="cuda")[5:].as_strided((G, n, V), (n * pitch, pitch, 1))
        far.copy_(x)
        for a, b in zip(flash_gemv.cats_beam_select(far, s.cuda()), flash_gemv.cats_beam_select(x.cuda(), s.cuda())):
            assert torch.equal(a, b)
