"""Storing in pages where a token's heads take several workgroups, and queries that are rotated in place."""
import ctypes

import pytest
import torch

from cats_amd import capi
from tests import paged_reference as ref
from tests.test_gpu_paged import BF16, F16, _append, _check_append, _same, _tables, _words

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv,D,rot", [(32, 32, 128, 128), (32, 32, 128, 64), (33, 32, 256, 256), (0, 40, 128, 128), (65, 32, 64, 16), (511, 1, 32, 32), (512, 1, 32, 0)])
def test_more_heads_than_a_workgroup_has_threads(heads, kv, D, rot, dtype):
    """Two to four workgroups a token, the last of them full or in part."""
    _check_append([(0, 37), (100, 1), (15, 0), (31, 2)], 32, heads, kv, D, dtype, rot, lead=1, behind=2)


@pytest.mark.parametrize("n", [4093, 4096, 4101])
def test_many_heads_of_many_tokens(n):
    """Eight tokens a workgroup, as many as it has, or fewer in the last one."""
    assert n + 3 >= 16 * torch.cuda.get_device_properties(0).multi_processor_count
    _check_append([(0, n - 100), (7, 100)], 64, 65, 32, 64, BF16, 64, lead=1, behind=2)


@pytest.mark.parametrize("heads,kv,D", [(4, 2, 64), (32, 32, 128)])
@pytest.mark.parametrize("per", [1, 8])
def test_queries_in_place(per, heads, kv, D):
    """q_out is q: as beside it, with queries of nobody and of tokens without a place among them."""
    rows = [(3, 9), (20, 70), (5, 2)] if per == 1 else [(0, 4100), (40, 30)]
    g = torch.Generator().manual_seed(61)
    pool = ref.new_pool(rows, 16, kv, D, F16, room=0)
    pool[2][1, 2] = -1
    N = ref.offsets_of(rows, 2)[-1] + 1
    q, k, v = (torch.randn(N, h, D, generator=g).half() for h in (heads, kv, kv))
    cos, sin = _tables(max(a + n for a, n in rows), D)
    want = _append(q, k, v, rows, 2, cos, sin, pool)
    qq, kk, vv, c, s, kp, vp, table = (t.cuda() for t in (q, k, v, cos, sin, *pool))
    offsets, start = _words(ref.offsets_of(rows, 2)), _words([a for a, _ in rows])
    strides = lambda t: (ctypes.c_int64 * 2)(t.stride(0), t.stride(1))
    status = capi.lib().cats_paged_append(qq.data_ptr(), strides(qq), kk.data_ptr(), strides(kk), vv.data_ptr(), strides(vv), offsets.data_ptr(), start.data_ptr(), c.data_ptr(),
                                          s.data_ptr(), D, c.shape[0], 2, qq.data_ptr(), kp.data_ptr(), vp.data_ptr(), table.data_ptr(), table.stride(0), N, len(rows), heads, kv, D,
                                          16, kp.shape[0], table.shape[1], 0, torch.cuda.current_stream().cuda_stream)
    assert status == 0 and want[0].isnan().any() and not want[0].isnan().all()
    assert _same(qq.cpu(), want[0]) and _same(kp.cpu(), want[1]) and _same(vp.cpu(), want[2])
