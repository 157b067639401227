"""Attention over pages whose keys are split into parts, and shared ones that many rows read: against the plain implementation in 64 bits."""
import math

import pytest
import torch

from tests import paged_reference as ref
from tests.test_gpu_paged import _attention

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _pool(rows, page, kv, D, dtype, g, **shared):
    """With a table of more than 2000 tokens whoever needs them: what the parts go by."""
    pool = ref.new_pool(rows, page, kv, D, dtype, 3, room=2100 // page, **shared)
    ref.fill(pool, rows, g)
    return pool


def _copy_shared(pool, rows, group, shared):
    """The page in which the shared tokens end is each one's own, and holds the same."""
    page = pool[0].shape[2]
    for b in range(len(rows)):
        first = b - b % group
        i, m = shared // page, shared % page
        if b != first and m:
            for x in pool[:2]:
                x[int(pool[2][b, i]), :, :m] = x[int(pool[2][first, i]), :, :m]


MANY = [(3000, 70), (500, 33), (0, 129), (1279, 1), (5, 0)]
FEW = [(3000, 3), (0, 1), (1279, 1), (64, 2), (2047, 4)]


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 128), (BF16, 64), (F16, 256), (F16, 32)])
@pytest.mark.parametrize("heads,kv", [(4, 2), (5, 5), (6, 1)])
@pytest.mark.parametrize("rows", [MANY, FEW])
def test_parts(rows, heads, kv, dtype, D):
    g = torch.Generator().manual_seed(11)
    pool = _pool(rows, 64, kv, D, dtype, g)
    N = ref.offsets_of(rows, 2)[-1] + 5
    q = torch.randn(N, heads, D, generator=g).to(dtype)
    assert ref.within(_attention(q, rows, 2, pool, D ** -0.5), *ref.paged_attention(q, rows, 2, pool, D ** -0.5))


@pytest.mark.parametrize("window", [1000, 1300, 2900])
@pytest.mark.parametrize("rows", [MANY, FEW])
def test_parts_of_a_window(rows, window):
    g = torch.Generator().manual_seed(12)
    pool = _pool(rows, 16, 2, 64, BF16, g)
    q = torch.randn(ref.offsets_of(rows)[-1], 4, 64, generator=g).bfloat16()
    assert ref.within(_attention(q, rows, 0, pool, 0.125, window), *ref.paged_attention(q, rows, 0, pool, 0.125, window))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows,at", [(MANY, 0), (MANY, 1500), (MANY, 3060), (FEW, 0), (FEW, 1500), (FEW, 3001)])
def test_values_that_are_not_finite(rows, at, value, dtype):
    g = torch.Generator().manual_seed(13)
    pool = _pool(rows, 32, 2, 64, dtype, g)
    q = torch.randn(ref.offsets_of(rows)[-1], 4, 64, generator=g).to(dtype)
    i, j = int(pool[2][0, at // 32]), at % 32
    pool[1][i, 0, j, 17] = value
    pool[0][i, 1, j, 5] = math.nan
    assert ref.within(_attention(q, rows, 0, pool, 0.125), *ref.paged_attention(q, rows, 0, pool, 0.125))


@pytest.mark.parametrize("bad", [-1, 10 ** 6])
@pytest.mark.parametrize("rows", [MANY, FEW])
def test_pages_that_are_none(rows, bad):
    g = torch.Generator().manual_seed(14)
    pool = _pool(rows, 32, 2, 64, F16, g)
    q = torch.randn(ref.offsets_of(rows)[-1], 4, 64, generator=g).half()
    pool[2][0, 50] = bad
    pool[2][3, 39] = bad
    want = ref.paged_attention(q, rows, 0, pool, 0.125)
    assert want[0].isnan().any() and not want[0].isnan().all() and ref.within(_attention(q, rows, 0, pool, 0.125), *want)


@pytest.mark.parametrize("scale", [2.0 ** -64, 3.0, 40.0, 2.0 ** 20])
@pytest.mark.parametrize("rows", [MANY, FEW])
def test_scales(rows, scale):
    """Weights that are all alike, and one key that is far ahead of the others of each sequence, in the last part or the first."""
    g = torch.Generator().manual_seed(15)
    pool = _pool(rows, 64, 1, 64, F16, g)
    q = torch.randn(ref.offsets_of(rows)[-1], 2, 64, generator=g).half()
    if scale > 2:  # or the order of the two largest is a matter of rounding
        q = q.abs() + 0.5
        for b, (a, n) in enumerate(rows):
            for at in ([a] if n and a % 2 else [0]):
                pool[0][int(pool[2][b, at // 64]), 0, at % 64] = 24.0
    assert ref.within(_attention(q, rows, 0, pool, scale), *ref.paged_attention(q, rows, 0, pool, scale))


GROUPS = [([(1500 + b, 1) for b in range(20)], 10, 1450), ([(1400 + 3 * b, 2 + b % 2) for b in range(16)], 8, 1400), ([(300 + b, 1) for b in range(9)], 9, 290),
          ([(1100, 4), (1100, 0), (1300, 4), (1101, 1)], 4, 1024), ([(2100 + b, 1) for b in range(70)], 70, 2080)]


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64), (F16, 256), (BF16, 32)])
@pytest.mark.parametrize("heads,kv", [(4, 2), (3, 3)])
@pytest.mark.parametrize("rows,group,shared", GROUPS)
def test_shared_by_many_rows(rows, group, shared, heads, kv, dtype, D):
    g = torch.Generator().manual_seed(16)
    pool = _pool(rows, 16, kv, D, dtype, g, group=group, shared=shared)
    _copy_shared(pool, rows, group, shared)
    q = torch.randn(ref.offsets_of(rows, 1)[-1] + 3, heads, D, generator=g).to(dtype)
    want = ref.paged_attention(q, rows, 1, pool, D ** -0.5)
    assert ref.within(_attention(q, rows, 1, pool, D ** -0.5, 0, group, [shared]), *want)
    assert ref.within(_attention(q, rows, 1, pool, D ** -0.5), *want)


@pytest.mark.parametrize("window", [600, 1200])
@pytest.mark.parametrize("rows,group,shared", GROUPS[:2])
def test_shared_by_many_rows_in_a_window(rows, group, shared, window):
    g = torch.Generator().manual_seed(17)
    pool = _pool(rows, 64, 2, 128, F16, g, group=group, shared=shared)
    _copy_shared(pool, rows, group, shared)
    q = torch.randn(ref.offsets_of(rows)[-1], 4, 128, generator=g).half()
    assert ref.within(_attention(q, rows, 0, pool, 0.1, window, group, [shared]), *ref.paged_attention(q, rows, 0, pool, 0.1, window))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,group,shared", GROUPS[:2])
def test_shared_ones_that_are_not_finite_or_none(rows, group, shared, dtype):
    g = torch.Generator().manual_seed(18)
    pool = _pool(rows, 64, 2, 128, dtype, g, group=group, shared=shared)
    _copy_shared(pool, rows, group, shared)
    q = torch.randn(ref.offsets_of(rows)[-1], 4, 128, generator=g).to(dtype)
    pool[1][int(pool[2][0, 9]), 0, 7, 33] = math.inf
    pool[0][int(pool[2][group, 3]), 1, 60, 3] = math.nan
    want = ref.paged_attention(q, rows, 0, pool, 0.1)
    assert ref.within(_attention(q, rows, 0, pool, 0.1, 0, group, [shared]), *want)
    pool[2][:group, 5] = -1
    want = ref.paged_attention(q, rows, 0, pool, 0.1)
    assert ref.within(_attention(q, rows, 0, pool, 0.1, 0, group, [shared]), *want)


@pytest.mark.parametrize("B", [60, 61, 62, 63, 125, 126, 190, 253, 254, 255, 520])
@pytest.mark.parametrize("n", [1, 9])
def test_workgroups_find_their_sequence(B, n):
    """Some without tokens, some with many: of one workgroup's rows and of several."""
    rows = [(7 * b % 50, (b * 5 % 4 != 0) * (n + b % 3) + 70 * (b % 40 == 17)) for b in range(B)]
    g = torch.Generator().manual_seed(19)
    pool = ref.new_pool(rows, 16, 1, 32, F16)
    ref.fill(pool, rows, g)
    q = torch.randn(ref.offsets_of(rows, 3)[-1] + 40, 2, 32, generator=g).half()
    assert ref.within(_attention(q, rows, 3, pool, 0.2), *ref.paged_attention(q, rows, 3, pool, 0.2))


@pytest.mark.parametrize("B,group", [(120, 2), (126, 2), (504, 2), (600, 2), (600, 3), (900, 300)])
@pytest.mark.parametrize("n", [1, 4])
def test_workgroups_find_their_group(B, group, n):
    """Groups of which some have no tokens, some of one workgroup's rows and some of several."""
    rows = [(40 + b % 5, (b // group % 7 != 3) * (n + (b % 11 == 0) * 5)) for b in range(B)]
    g = torch.Generator().manual_seed(20)
    pool = ref.new_pool(rows, 16, 1, 32, BF16, group=group, shared=32)
    ref.fill(pool, rows, g)
    q = torch.randn(ref.offsets_of(rows, 2)[-1] + 9, 3, 32, generator=g).bfloat16()
    assert ref.within(_attention(q, rows, 2, pool, 0.2, 0, group, [32]), *ref.paged_attention(q, rows, 2, pool, 0.2))


@pytest.mark.parametrize("heads,kv", [(130, 1), (96, 1), (64, 64)])
@pytest.mark.parametrize("rows", [[(30, 1), (200, 2)], [(1500, 1)]])
def test_many_heads(heads, kv, rows):
    """More rows a token than a workgroup has."""
    g = torch.Generator().manual_seed(22)
    pool = _pool(rows, 64, kv, 64, F16, g)
    q = torch.randn(ref.offsets_of(rows)[-1], heads, 64, generator=g).half()
    assert ref.within(_attention(q, rows, 0, pool, 0.125), *ref.paged_attention(q, rows, 0, pool, 0.125))
