"""What the cache of pages and packed attention refuse, before anything is launched: the pointers are never read.  Needs no GPU."""
import ctypes

import pytest
import torch

OK, DTYPE, SHAPE, ALIGN, BATCH, NULL, WORKSPACE = 0, 1, 2, 3, 4, 5, 6


@pytest.fixture(scope="module")
def L():
    from cats_amd import capi

    return capi.lib()


def _p(offset=0):
    buf = (ctypes.c_char * 4096)()
    _p.keep = getattr(_p, "keep", []) + [buf]
    return ctypes.c_void_p((ctypes.addressof(buf) + 255) // 256 * 256 + offset)


def _s(token, head):
    a = (ctypes.c_int64 * 2)(token, head)
    _p.keep.append(a)
    return ctypes.cast(a, ctypes.c_void_p)


def _append(L, **change):  # as it stands: a call that is fine but for its batch
    a = dict(q=_p(), qs=_s(128, 64), k=_p(), ks=_s(64, 64), v=_p(), vs=_s(64, 64), offsets=_p(), start=_p(), cos=_p(), sin=_p(), rot=64, positions=10, table_dtype=2,
             q_out=_p(), k_pages=_p(), v_pages=_p(), table=_p(), stride=4, N=3, B=0, heads=2, kv=1, D=64, page=16, pages=8, width=4, dtype=0)
    a.update(change)
    return L.cats_paged_append(*a.values(), None)


def _attention(L, **change):  # ends at its scratch
    a = dict(q=_p(), qs=_s(128, 64), offsets=_p(), start=_p(), k_pages=_p(), v_pages=_p(), table=_p(), stride=4000, scale=0.125, window=0, group=1, shared=None,
             step=0, out=_p(), N=1, B=1, heads=2, kv=1, D=64, page=16, pages=8, width=4000, dtype=1, scratch=None, bytes=0)
    a.update(change)
    return L.cats_paged_attention(*a.values(), None)


def _prompt(L, **change):
    a = dict(q=_p(), qs=_s(128, 64), k=_p(), ks=_s(64, 64), v=_p(), vs=_s(64, 64), offsets=_p(), k_offsets=None, scale=0.125, window=0, out=_p(), N=3, M=3, B=0,
             heads=2, kv=1, D=64, dtype=0)
    a.update(change)
    return L.cats_prompt_attention(*a.values(), None)


POOL = [(dict(page=8), SHAPE), (dict(page=48), SHAPE), (dict(page=2048), SHAPE), (dict(pages=0), SHAPE), (dict(width=0), SHAPE), (dict(page=1024, width=(1 << 20) + 1), SHAPE),
        (dict(k_pages=None), NULL), (dict(v_pages=None), NULL), (dict(table=None), NULL), (dict(k_pages=_p(8)), ALIGN), (dict(v_pages=_p(2)), ALIGN), (dict(table=_p(2)), ALIGN),
        (dict(stride=-1), SHAPE)]
TOKENS = [(dict(dtype=2), DTYPE), (dict(dtype=9), DTYPE), (dict(B=-1), BATCH), (dict(B=(1 << 20) + 1), BATCH), (dict(N=0), SHAPE), (dict(N=-1), SHAPE), (dict(N=(1 << 24) + 1), SHAPE),
          (dict(kv=0), SHAPE), (dict(kv=65536, heads=65536), SHAPE), (dict(D=48), SHAPE), (dict(D=512), SHAPE), (dict(q=_p(8)), ALIGN), (dict(qs=None), NULL),
          (dict(qs=_s(128, 4)), ALIGN), (dict(qs=_s(-128, 64)), ALIGN), (dict(qs=_s((1 << 23) + 8, 64)), SHAPE), (dict(offsets=None), NULL), (dict(offsets=_p(4)), ALIGN)]
ATTENTION = [(dict(heads=3, kv=2), SHAPE), (dict(heads=1, kv=2), SHAPE), (dict(heads=0), SHAPE), (dict(window=-1), SHAPE), (dict(scale=2.0 ** -65), SHAPE), (dict(scale=2.0 ** 65), SHAPE),
             (dict(scale=0.0), SHAPE), (dict(scale=-1.0), SHAPE), (dict(scale=float("nan")), SHAPE), (dict(scale=float("inf")), SHAPE), (dict(q=None), NULL), (dict(out=None), NULL),
             (dict(out=_p(8)), ALIGN), (dict(N=1 << 24, heads=32), SHAPE)]


@pytest.mark.parametrize("change,status", POOL + TOKENS + [
    (dict(rot=-16), SHAPE), (dict(rot=24), SHAPE), (dict(rot=80), SHAPE), (dict(positions=0), SHAPE), (dict(table_dtype=1), DTYPE), (dict(cos=None), NULL), (dict(sin=None), NULL),
    (dict(cos=_p(4)), ALIGN), (dict(q_out=None), NULL), (dict(q=None), NULL), (dict(q=None, q_out=None), NULL), (dict(heads=0), NULL), (dict(q_out=_p(8)), ALIGN), (dict(k=None), NULL),
    (dict(v=_p(4)), ALIGN), (dict(ks=_s(64, 1)), ALIGN), (dict(start=None), NULL), (dict(start=_p(4)), ALIGN)])
def test_append_refuses(L, change, status):
    assert _append(L, **{"B": 1, **change}) == status


def test_batches_of_none(L):
    assert _append(L) == BATCH and _prompt(L) == BATCH and _attention(L, B=0) == BATCH


@pytest.mark.parametrize("change,status", POOL + TOKENS + ATTENTION + [
    (dict(), WORKSPACE), (dict(scratch=_p(8), bytes=1 << 30), WORKSPACE), (dict(scratch=_p(), bytes=64), WORKSPACE), (dict(group=0), SHAPE), (dict(group=2), SHAPE),
    (dict(B=2, group=2), NULL), (dict(B=2, group=2, shared=_p(4)), ALIGN), (dict(step=2), SHAPE), (dict(start=None), NULL), (dict(B=2, group=2, shared=_p(), N=1 << 20, heads=32), SHAPE)])
def test_attention_refuses(L, change, status):
    """The plain call ends at its scratch, which a table of 64000 tokens needs."""
    assert _attention(L, **change) == status


@pytest.mark.parametrize("change,status", TOKENS + ATTENTION + [
    (dict(M=0), SHAPE), (dict(M=4), SHAPE), (dict(M=(1 << 24) + 1, k_offsets=_p()), SHAPE), (dict(k=None), NULL), (dict(v=_p(4)), ALIGN), (dict(vs=_s(64, 63)), ALIGN), (dict(k_offsets=_p(4)), ALIGN)])
def test_prompt_refuses(L, change, status):
    assert _prompt(L, **{"B": 1, "M": change.get("N", 3), **change}) == status


def test_scratch(L):
    f = L.cats_paged_attention_scratch_bytes  # N, B, heads, kv_heads, D, page, width, window, group
    assert f(1, 1, 32, 8, 128, 64, 1000, 0, 1) > 0 and f(1, 1, 32, 8, 128, 64, 16, 0, 1) == 0
    assert f(1, 1, 32, 8, 128, 64, 1000, 500, 1) == 0  # a window of few keys
    assert f(4, 4, 32, 8, 128, 64, 4, 0, 4) >= 4 * 32 * 2 * 130 * 4  # a part of what is shared, and one of what is not
    for bad in ((0, 1, 32, 8, 128, 64, 1000, 0, 1), (1, 0, 32, 8, 128, 64, 1000, 0, 1), (1, 1, 32, 5, 128, 64, 1000, 0, 1), (1, 1, 4, 8, 128, 64, 1000, 0, 1), (1, 1, 32, 8, 100, 64, 1000, 0, 1),
                (1, 1, 32, 8, 128, 60, 1000, 0, 1), (1, 1, 32, 8, 128, 64, 0, 0, 1), (1, 1, 32, 8, 128, 64, 1000, -1, 1), (3, 3, 32, 8, 128, 64, 1000, 0, 2), (1, 1, 32, 8, 128, 64, 1000, 0, 0)):
        assert f(*bad) == 0


def test_tensors_of_the_host_are_refused():
    import flash_gemv

    x, w, pool = torch.zeros(2, 2, 64).half(), torch.tensor([0, 2]), torch.zeros(2, 2, 16, 64).half()
    table = torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: flash_gemv.cats_paged_append(x, x, x, w, w[:1], None, None, pool, pool, table), lambda: flash_gemv.cats_paged_attention(x, w, w[:1], pool, pool, table, 0.1),
                 lambda: flash_gemv.cats_prompt_attention(x, x, x, w, 0.1)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def _ops():
    """Each op of torch on tensors of the host, and those of its tensors that hold numbers."""
    import flash_gemv

    x, w, pool, turn = (torch.zeros(2, 2, 64).half() for _ in range(3)), torch.tensor([0, 2]), [torch.zeros(2, 2, 16, 64).half() for _ in range(2)], [torch.zeros(4, 64) for _ in range(2)]
    a, table = dict(zip(("q", "k", "v", "k_pages", "v_pages", "cos", "sin"), (*x, *pool, *turn))), torch.zeros(1, 2, dtype=torch.int32)
    append = lambda q, k, v, k_pages, v_pages, cos, sin: flash_gemv.cats_paged_append(q, k, v, w, w[:1], cos, sin, k_pages, v_pages, table)
    attention = lambda q, k_pages, v_pages: flash_gemv.cats_paged_attention(q, w, w[:1], k_pages, v_pages, table, 0.1)
    prompt = lambda q, k, v: flash_gemv.cats_prompt_attention(q, k, v, w, 0.1)
    return [(append, a), (attention, {n: a[n] for n in ("q", "k_pages", "v_pages")}), (prompt, {n: a[n] for n in "qkv"})]


@pytest.mark.parametrize("op,name", [(0, n) for n in ("q", "k", "v", "k_pages", "v_pages", "cos", "sin")] + [(1, n) for n in ("q", "k_pages", "v_pages")] + [(2, n) for n in "qkv"])
def test_what_records_a_gradient_is_refused(op, name):
    """Tokens, pages and rotary tables alike.  Where nothing is recorded they are as any others, and what is wrong with these is that they are not on the GPU."""
    call, args = _ops()[op]
    args[name].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        call(**args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        call(**args)


@pytest.mark.parametrize("op,name", [(0, "q"), (0, "k"), (0, "v_pages"), (0, "sin"), (1, "q"), (1, "k_pages"), (2, "q"), (2, "v")])
def test_tangents_are_refused(op, name):
    """Of forward differentiation, which no_grad does not end."""
    from torch.autograd import forward_ad

    call, args = _ops()[op]
    with forward_ad.dual_level():
        args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(RuntimeError, match="no gradient"):
            call(**args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
            call(**args)
        with torch.inference_mode(), pytest.raises(RuntimeError, match="GPU"):
            call(**args)
    with pytest.raises(RuntimeError, match="GPU"):  # it has none any more
        call(**args)


def test_tangents_of_a_cache_in_8_bits_are_refused():
    """The ops of the other cache look at their tokens in the same way."""
    import flash_gemv
    from torch.autograd import forward_ad
    from cats_amd.kv8 import Kv8Cache

    c, x, w = Kv8Cache(1, 2, 64, 64, device="cpu"), torch.zeros(1, 1, 2, 64).half(), torch.tensor([0])
    t = [getattr(c, n) for n in Kv8Cache.FIELDS]
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: flash_gemv.cats_kv8_append(d, x, w, None, *t), lambda: flash_gemv.cats_kv8_append(x, d, w, None, *t), lambda: flash_gemv.cats_kv8_attention(d, w, None, *t, 0.125)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
