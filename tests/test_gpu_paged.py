"""The cache of pages on the GPU, against plain implementations in 64 bits: storing with the rotation, attention of steps, drafts and pieces, shared prefixes."""
import math

import pytest
import torch

from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
TYPES = [F16, BF16]


def _words(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


def _tables(positions, rot, dtype=torch.float32):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.cat([a, a], 1)
    return a.cos().to(dtype), a.sin().to(dtype)


def _append(q, k, v, rows, lead, cos, sin, pool):
    """The op on copies of the pool; (q', k_pages, v_pages) on the CPU."""
    import flash_gemv

    dev = lambda t: None if t is None else t.cuda()
    kp, vp, table = (t.cuda() for t in pool)
    out = flash_gemv.cats_paged_append(dev(q), dev(k), dev(v), _words(ref.offsets_of(rows, lead)), _words([a for a, _ in rows]), dev(cos), dev(sin), kp, vp, table)
    assert torch.equal(table.cpu(), pool[2])
    return None if out is None else out.cpu(), kp.cpu(), vp.cpu()


def _same(a, b):
    return bool(((a.double() == b.double()) | (a.isnan() & b.isnan())).all())


def _check_append(rows, page, heads, kv, D, dtype, rot, lead=0, behind=0, table_dtype=torch.float32, positions=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    N = ref.offsets_of(rows, lead)[-1] + behind
    pool = ref.new_pool(rows, page, kv, D, dtype, seed)
    k, v = (torch.randn(N, kv, D, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(N, heads, D, generator=g).to(dtype) if heads else None
    cos, sin = _tables(positions or max(a + n for a, n in rows) + 1, rot, table_dtype) if rot else (None, None)
    got = _append(q, k, v, rows, lead, cos, sin, pool)
    (wq, bq), (wk, bk), (wv, bv) = ref.append(q, k, v, rows, lead, cos, sin, pool)
    if heads:
        assert ref.within(got[0], wq, bq)
    else:
        assert got[0] is None
    assert ref.within(got[1], wk, bk) and _same(got[2], wv)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,rot", [(32, 32), (64, 16), (64, 64), (128, 128), (128, 64), (128, 0), (256, 256), (256, 48)])
def test_append(D, rot, dtype):
    """Prompts, pieces and steps in one call, a sequence without tokens, tokens that are nobody's."""
    _check_append([(0, 37), (100, 1), (15, 0), (31, 2), (63, 70)], 32, 6, 2, D, dtype, rot, lead=2, behind=3)


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("heads,kv", [(0, 1), (1, 1), (7, 1), (32, 8), (3, 3)])
def test_append_heads_and_pages(heads, kv, page):
    _check_append([(1000, 1), (0, 1), (page - 1, 2)], page, heads, kv, 64, BF16, 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_tables_in_the_type(dtype):
    _check_append([(5, 20), (0, 3)], 16, 4, 2, 128, dtype, 128, table_dtype=dtype)


def test_append_many_tokens():
    """More tokens than a workgroup a CU has: several a workgroup; more sequences than a wave has lanes."""
    _check_append([(7 * b, 1 + b % 5) for b in range(1500)], 16, 2, 1, 32, F16, 32, lead=1, behind=5)


@pytest.mark.parametrize("B", [1, 63, 64, 65, 4095, 4097])
def test_append_finds_its_sequence(B):
    _check_append([(b % 16, (b % 3 == 1) + 2 * (b == B - 1)) for b in range(B)], 16, 1, 1, 32, F16, 32)


def test_append_without_a_place():
    """Positions outside the rotary tables or the table, entries that are no page: not stored, the query NaN, and nothing else."""
    rows, page = [(10, 4), (2 ** 40, 2), (-3, 2), (0, 40), (30, 8)], 16
    g = torch.Generator().manual_seed(3)
    pool = ref.new_pool([(10, 4), (0, 2), (0, 2), (0, 40), (30, 8)], page, 2, 64, F16, room=0)
    pool[2][3, 1] = -1
    pool[2][4, 2] = pool[0].shape[0]
    N = sum(n for _, n in rows)
    q, k, v = (torch.randn(N, h, 64, generator=g).half() for h in (4, 2, 2))
    cos, sin = _tables(34, 64)
    got = _append(q, k, v, rows, 0, cos, sin, pool)
    (wq, bq), (wk, bk), (wv, bv) = ref.append(q, k, v, rows, 0, cos, sin, pool)
    assert wq.isnan().any() and ref.within(got[0], wq, bq) and ref.within(got[1], wk, bk) and _same(got[2], wv)


def test_append_strides():
    """Heads that are slices of one projection's output, tokens apart, and strides that no vector reads."""
    import flash_gemv

    g = torch.Generator().manual_seed(4)
    rows, page = [(3, 9), (40, 1)], 16
    pool = ref.new_pool(rows, page, 2, 64, BF16)
    cos, sin = _tables(60, 64)
    fused = torch.randn(10, (4 + 2 + 2) * 64, generator=g).bfloat16()
    q, k, v = (x.reshape(10, -1, 64) for x in fused.split([256, 128, 128], 1))
    (wq, bq), (wk, bk), (wv, _) = ref.append(q, k, v, rows, 0, cos, sin, pool)
    odd = torch.randn(10, 2, 65, generator=g).bfloat16().cuda()
    odd[..., 1:] = k.cuda()
    f = fused.cuda()
    turned = lambda t: t.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    for qq, kk, vv in ((f[:, :256].view(10, 4, 64), f[:, 256:384].view(10, 2, 64), f[:, 384:].view(10, 2, 64)), (turned(q), turned(k), turned(v)),
                       (q.cuda(), odd[..., 1:], v.cuda())):
        kp, vp, table = (t.cuda() for t in pool)
        out = flash_gemv.cats_paged_append(qq, kk, vv, _words(ref.offsets_of(rows)), _words([3, 40]), cos.cuda(), sin.cuda(), kp, vp, table)
        assert ref.within(out, wq, bq) and ref.within(kp, wk, bk) and _same(vp.cpu(), wv)


def _attention(q, rows, lead, pool, scale, window=0, group=1, shared=None):
    import flash_gemv

    kp, vp, table = (t.cuda() for t in pool)
    return flash_gemv.cats_paged_attention(q.cuda(), _words(ref.offsets_of(rows, lead)), _words([a for a, _ in rows]), kp, vp, table, scale, window, group,
                                           None if shared is None else _words(shared))


def _check(rows, page, heads, kv, D, dtype, window=0, lead=0, behind=0, group=1, shared=None, seed=0, scale=None):
    g = torch.Generator().manual_seed(seed)
    N = ref.offsets_of(rows, lead)[-1] + behind
    pool = ref.new_pool(rows, page, kv, D, dtype, seed, group=group, shared=min(shared) if shared else 0)
    ref.fill(pool, rows, g)
    if shared:  # what the pages do not share is copied
        for b in range(len(rows)):
            first, n = b - b % group, min(rows[b][0], rows[b - b % group][0], shared[b // group if len(shared) > 1 else 0])
            for i in range(-(-n // page)):
                m = min(page, n - i * page)
                for x in pool[:2]:
                    x[int(pool[2][b, i]), :, :m] = x[int(pool[2][first, i]), :, :m]
    q = (torch.randn(N, heads, D, generator=g) * 1.5).to(dtype)
    scale = D ** -0.5 if scale is None else scale
    got = _attention(q, rows, lead, pool, scale, window, group, shared)
    assert ref.within(got, *ref.paged_attention(q, rows, lead, pool, scale, window))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (8, 2), (7, 1), (32, 2), (20, 1)])
def test_steps(heads, kv, D, dtype):
    """A token each: the first one, page and tile ends, long ones."""
    _check([(0, 1), (15, 1), (16, 1), (31, 1), (127, 1), (128, 1), (700, 1)], 16, heads, kv, D, dtype)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
def test_pages(page):
    _check([(300, 1), (1023, 3), (1024, 1), (5, 2)], page, 8, 2, 64, BF16)


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64), (F16, 256), (BF16, 32)])
@pytest.mark.parametrize("rows", [[(50, 5), (0, 0), (129, 2), (0, 3), (1000, 1)], [(0, 40), (333, 17), (64, 64), (0, 1)], [(513, 150), (0, 129), (2000, 33)]])
@pytest.mark.parametrize("window", [0, 1, 40, 500])
def test_drafts_and_pieces(rows, window, dtype, D):
    """Several tokens a sequence, of different numbers, windows, tokens that are nobody's."""
    _check(rows, 16, 6, 2, D, dtype, window, lead=3, behind=70)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_one_long_sequence(D, dtype):
    _check([(9999, 1)], 64, 4, 1, D, dtype)
    _check([(9990, 5), (20, 1)], 16, 2, 1, D, dtype, window=6000)


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 128), (F16, 64), (BF16, 256), (F16, 32)])
@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 2), (7, 1)])
@pytest.mark.parametrize("rows,group,shared", [
    ([(300, 1), (256, 1), (411, 1)], 3, [256]),                        # whole pages, one sequence ends with them
    ([(130 + 17 * b, 1) for b in range(8)], 4, [100, 64]),             # a part of a page, groups that share differently
    ([(500 + b, 1 + b % 3) for b in range(12)], 12, [500]),            # drafts
    ([(200, 1), (90, 1), (0, 4), (150, 0)], 2, [160, 170]),            # sequences that are shorter than what is shared, and none
    ([(70 + b, 1) for b in range(40)], 20, [0, 64]),
    ([(1200, 40), (1100, 30)], 2, [1024])])
def test_shared_prefixes(rows, group, shared, heads, kv, dtype, D):
    _check(rows, 16, heads, kv, D, dtype, group=group, shared=shared, behind=2)


@pytest.mark.parametrize("window", [30, 128, 400])
def test_shared_prefixes_and_windows(window):
    _check([(300, 1), (256, 2), (411, 1), (500, 1)], 16, 8, 2, 64, BF16, window, group=4, shared=[256])


def test_shared_is_read_through_the_first_one():
    """The others' entries of whole pages that are shared are not looked at; shared beyond 2^31 and below 0 are all and none."""
    g = torch.Generator().manual_seed(9)
    rows = [(256, 1), (256, 1), (270, 1)]
    pool = ref.new_pool(rows, 64, 2, 64, F16, group=3, shared=256)
    ref.fill(pool, rows, g)
    q = torch.randn(3, 4, 64, generator=g).half()
    want = ref.paged_attention(q, rows, 0, pool, 0.125)
    assert ref.within(_attention(q, rows, 0, pool, 0.125, 0, 3, [-5]), *want)
    short = [rows[0], rows[1]]
    assert ref.within(_attention(q[:2], short, 0, (*pool[:2], pool[2][:2]), 0.125, 0, 2, [2 ** 40]), *ref.paged_attention(q[:2], short, 0, pool, 0.125))
    pool[2][1:, :4] = -1  # a page of nobody's
    assert ref.within(_attention(q, rows, 0, pool, 0.125, 0, 3, [256]), *want)


@pytest.mark.parametrize("T", [1, 3, 40])
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
def test_pages_that_are_none(bad, T):
    """Queries that see a token of such an entry are NaN, the others are not; entries that a window hides, and those behind the last token, may be anything."""
    g = torch.Generator().manual_seed(5)
    rows = [(200, T), (90, T), (300, T)]
    pool = ref.new_pool(rows, 32, 2, 64, F16)
    ref.fill(pool, rows, g)
    q = torch.randn(3 * T, 4, 64, generator=g).half()
    pool[2][0, 3] = bad
    pool[2][2, 0:2] = bad
    want = ref.paged_attention(q, rows, 0, pool, 0.125)
    assert want[0][:T].isnan().all() and want[0][2 * T:].isnan().all() and ref.within(_attention(q, rows, 0, pool, 0.125), *want)
    want = ref.paged_attention(q, rows, 0, pool, 0.125, 100)
    assert want[0][0].isnan().all() and not want[0][2 * T:].isnan().any() and ref.within(_attention(q, rows, 0, pool, 0.125, 100), *want)


def test_positions_outside_the_table():
    rows = [(20, 1), (2 ** 62, 1), (-1, 1), (2 ** 31, 2), (60, 4), (60, 5)]
    g = torch.Generator().manual_seed(6)
    pool = ref.new_pool([(20, 1), (0, 1), (0, 1), (0, 1), (60, 4), (59, 5)], 32, 1, 64, BF16, room=0)
    ref.fill(pool, [(20, 1), (0, 1), (0, 1), (0, 1), (60, 4), (59, 5)], g)
    q = torch.randn(14, 2, 64, generator=g).bfloat16()
    want = ref.paged_attention(q, rows, 0, pool, 0.125)
    assert want[0].isnan().any(-1).any(-1).tolist() == [False] + [True] * 4 + [False] * 4 + [True] * 5
    assert ref.within(_attention(q, rows, 0, pool, 0.125), *want)


@pytest.mark.parametrize("n", [1, 60])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("at", [3, 120, 190, 200, 205, 259])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite(value, at, dtype, n):
    """They reach the queries that see them, and no other: keys all elements, values their own."""
    g = torch.Generator().manual_seed(7)
    rows = [(200, n), (30, n)]
    pool = ref.new_pool(rows, 64, 2, 64, dtype)
    ref.fill(pool, rows, g)
    q = torch.randn(2 * n, 4, 64, generator=g).to(dtype)
    if at < 200 + n:
        i, j = int(pool[2][0, at // 64]), at % 64
        pool[1][i, 0, j, 17] = value
        pool[0][i, 1, j, 5] = math.nan
    q[-1, 3, 2] = value
    assert ref.within(_attention(q, rows, 0, pool, 0.125), *ref.paged_attention(q, rows, 0, pool, 0.125))


@pytest.mark.parametrize("scale", [2.0 ** -64, 1e-4, 3.0, 40.0, 2.0 ** 20])
@pytest.mark.parametrize("n", [1, 40])
def test_scales(scale, n):
    """Weights that are all alike and weights of which one is left."""
    g = torch.Generator().manual_seed(5)
    rows = [(300, n)]
    pool = ref.new_pool(rows, 64, 1, 64, F16)
    ref.fill(pool, rows, g)
    if scale > 1000:  # a key that is far ahead of the others, or the order of the two largest is a matter of rounding
        pool[0][int(pool[2][0, 1]), 0, 7] = 0
        q = torch.randn(1, 2, 64, generator=g).half().expand(n, 2, 64).contiguous()
        pool[0][int(pool[2][0, 1]), 0, 7] = (q[0, 0] * 8).half()
        q[:, 1] = q[:, 0]
    else:
        q = torch.randn(n, 2, 64, generator=g).half()
    assert ref.within(_attention(q, rows, 0, pool, scale), *ref.paged_attention(q, rows, 0, pool, scale))
