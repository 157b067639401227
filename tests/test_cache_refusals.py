"""What the cache in 8 bits and beam search refuse, before anything is launched: the pointers are never read.  Needs no GPU."""
import ctypes

import pytest
import torch

OK_STRIDES = (64, 64, 64)


@pytest.fixture(scope="module")
def L():
    from cats_amd import capi

    return capi.lib()


def _p(offset=0):
    buf = (ctypes.c_char * 4096)()
    _p.keep = getattr(_p, "keep", []) + [buf]
    return ctypes.c_void_p((ctypes.addressof(buf) + 255) // 256 * 256 + offset)


def _strides(*s):
    a = (ctypes.c_int64 * 3)(*s)
    _p.keep.append(a)
    return ctypes.cast(a, ctypes.c_void_p)


def _append(L, **change):
    a = dict(k=_p(), ks=_strides(*OK_STRIDES), v=_p(), vs=_strides(*OK_STRIDES), start=_p(), ss=0, count=None, cs=0, k8=_p(), v8=_p(), k_scale=_p(),
             v_scale=_p(), k_tail=_p(), v_tail=_p(), B=0, T=1, heads=1, D=64, blocks=2, dtype=0)  # B = 0: a call that is fine but for its batch
    a.update(change)
    return L.cats_kv8_append(*a.values(), None)


def _attention(L, **change):
    a = dict(q=_p(), qs=_strides(*OK_STRIDES), start=_p(), ss=0, count=None, cs=0, k8=_p(), v8=_p(), k_scale=_p(), v_scale=_p(), k_tail=_p(), v_tail=_p(),
             scale=0.125, window=0, out=_p(), B=1, T=1, heads=2, kv=1, D=64, blocks=4000, dtype=1, scratch=None, bytes=0)
    a.update(change)
    return L.cats_kv8_attention(*a.values(), None)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), 1), (dict(dtype=7), 1), (dict(B=-1), 4), (dict(B=65536), 4), (dict(B=1, T=0), 2), (dict(B=1, T=129), 2), (dict(B=1, heads=0), 2),
    (dict(B=1, D=48), 2), (dict(B=1, D=512), 2), (dict(B=1, blocks=0), 2), (dict(B=1, blocks=(1 << 24) + 1), 2), (dict(B=65535, heads=65535), 2),
    (dict(B=1, k=None), 5), (dict(B=1, v=None), 5), (dict(B=1, ks=None), 5), (dict(B=1, start=None), 5), (dict(B=1, k8=None), 5), (dict(B=1, v_scale=None), 5),
    (dict(B=1, v_tail=None), 5), (dict(B=1, k=_p(8)), 3), (dict(B=1, v8=_p(8)), 3), (dict(B=1, k_tail=_p(2)), 3), (dict(B=1, k_scale=_p(2)), 3),
    (dict(B=1, start=_p(4)), 3), (dict(B=1, count=_p(4)), 3), (dict(B=1, ss=2), 2), (dict(B=1, cs=-1), 2), (dict(), 4)])
def test_append_refuses(L, change, status):
    assert _append(L, **change) == status


@pytest.mark.parametrize("strides", [(64, 4, 64), (64, 64, 1), (-64, 64, 64), (7, 64, 64)])
def test_strides_that_no_vector_reads(L, strides):
    assert _append(L, B=1, vs=_strides(*strides)) == 3
    assert _attention(L, qs=_strides(*strides)) == 3


@pytest.mark.parametrize("change,status", [
    (dict(), 6), (dict(scratch=_p(), bytes=64), 6), (dict(dtype=2), 1), (dict(B=0), 4), (dict(heads=3, kv=2), 2), (dict(heads=1, kv=2), 2), (dict(window=-1), 2),
    (dict(scale=2.0 ** -65), 2), (dict(scale=2.0 ** 65), 2), (dict(scale=0.0), 2), (dict(scale=-1.0), 2), (dict(scale=float("nan")), 2), (dict(scale=float("inf")), 2), (dict(q=None), 5), (dict(out=None), 5), (dict(out=_p(8)), 3),
    (dict(q=_p(2)), 3), (dict(T=4000 * 64 + 1), 2), (dict(T=100000, heads=64), 2), (dict(k8=None), 5)])
def test_attention_refuses(L, change, status):
    """The plain call ends at its scratch, which a cache of 4000 blocks needs."""
    assert _attention(L, **change) == status


def test_attention_scratch(L):
    f = L.cats_kv8_attention_scratch_bytes
    assert f(1, 1, 32, 8, 128, 4000, 0) > 0 and f(1, 1, 32, 8, 128, 1, 0) == 0
    assert f(0, 1, 32, 8, 128, 4000, 0) == 0 and f(1, 1, 32, 5, 128, 4000, 0) == 0


@pytest.mark.parametrize("change,status", [
    (dict(), 6), (dict(scratch=_p(8), bytes=1 << 30), 6), (dict(dtype=2), 1), (dict(B=0), 4), (dict(B=9), 4), (dict(H=8192 * 9, heads=576), 2), (dict(heads=3), 2), (dict(heads=8), 2),
    (dict(blocks=0), 2), (dict(max_len=129), 2), (dict(max_len=0), 2), (dict(h=None), 5), (dict(wo=None), 5), (dict(v_tail=None), 5), (dict(position=None), 5), (dict(x=_p(8)), 3),
    (dict(wk=_p(8)), 3), (dict(v8=_p(4)), 3)])
def test_step_refuses(L, change, status):
    a = dict(h=_p(), x=_p(), norm=None, eps=1e-5, wq=_p(), wk=_p(), wv=_p(), wo=_p(), k8=_p(), v8=_p(), k_scale=_p(), v_scale=_p(), k_tail=_p(), v_tail=_p(), cos=_p(),
             sin=_p(), position=_p(), out=_p(), B=1, H=128, heads=2, blocks=2, max_len=128, dtype=0, scratch=None, bytes=0)
    a.update(change)
    assert L.cats_kv8_attention_step(*a.values(), None) == status


@pytest.mark.parametrize("change,status", [
    (dict(), 6), (dict(dtype=3), 1), (dict(beams=17), 2), (dict(keep=17), 2), (dict(keep=0), 2), (dict(groups=0), 2), (dict(V=0), 2), (dict(beams=1, V=2, keep=3), 2),
    (dict(eos=100), 2), (dict(finished=_p(), eos=-1), 2), (dict(stride=-1), 2), (dict(groups=65536, beams=1), 2), (dict(logits=None), 5), (dict(parents=None), 5),
    (dict(finished_out=None), 5), (dict(logits=_p(1)), 3), (dict(dtype=2, logits=_p(2)), 3), (dict(scores=_p(2)), 3), (dict(tokens=_p(4)), 3), (dict(scratch=_p(8), bytes=1 << 30), 6)])
def test_select_refuses(L, change, status):
    a = dict(logits=_p(), stride=100, scores=_p(), finished=None, eos=5, best=_p(), parents=_p(), tokens=_p(), finished_out=_p(), groups=2, beams=4, V=100, keep=4,
             dtype=0, scratch=None, bytes=0)
    a.update(change)
    assert L.cats_beam_select(*a.values(), None) == status


class Cache(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("entry_bytes", ctypes.c_int64), ("heads", ctypes.c_int), ("entries", ctypes.c_int), ("slots", ctypes.c_int)]


@pytest.mark.parametrize("cache,change,status", [
    ({}, dict(beams=17), 2), ({}, dict(beams=0), 2), ({}, dict(groups=0), 2), ({}, dict(n=0), 2), ({}, dict(step=2), 2), ({}, dict(parents=None), 5), ({}, dict(caches=None), 5),
    ({}, dict(lengths=None), 5), ({}, dict(parents=_p(4)), 3), ({}, dict(lengths=_p(4)), 3), (dict(data=None), {}, 5), (dict(data=_p(2).value), {}, 3), (dict(entry_bytes=6), {}, 3),
    (dict(entry_bytes=0), {}, 2), (dict(heads=0), {}, 2), (dict(entries=0), {}, 2), (dict(slots=-1), {}, 2), (dict(entry_bytes=1 << 41), {}, 2),
    ({}, dict(beams=1), 0)])
def test_reorder_refuses(L, cache, change, status):
    c = dict(data=_p().value, entry_bytes=16, heads=1, entries=4, slots=1)
    c.update(cache)
    a = dict(caches=ctypes.byref(Cache(**c)), n=1, parents=_p(), lengths=_p(), step=0, groups=1, beams=2)
    a.update(change)
    assert L.cats_cache_reorder(*a.values(), None) == status


def test_operators_refuse_cpu_tensors():
    import flash_gemv
    from tests import cache_reference as ref

    c = [t for t in ref.new_cache(1, 1, 1, 64, torch.float16).values()]
    x, at = torch.zeros(1, 1, 1, 64, dtype=torch.float16), torch.zeros(1, dtype=torch.int64)
    for call in (lambda: flash_gemv.cats_kv8_append(x, x, at, None, *c), lambda: flash_gemv.cats_kv8_attention(x, at, None, *c, 0.1),
                 lambda: flash_gemv.cats_beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2)), lambda: flash_gemv.cats_cache_reorder([x], [0], torch.zeros(1, 1, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_plan_refusals():
    from cats_amd import capi

    out = (ctypes.c_int * 2)()
    plan = capi.lib().cats_kv8_attention_plan
    assert plan(1, 1, 2, 1, 64, 4, 0, out) == 0 and out[0] == 0 and out[1] == 1
    assert plan(1, 1, 2, 1, 64, 4, 0, None) == 5
    for bad in ((1, 1, 3, 2, 64, 4, 0), (1, 1, 2, 1, 48, 4, 0), (1, 0, 2, 1, 64, 4, 0), (1, 1, 2, 1, 64, 4, -1), (1, 300, 2, 1, 64, 4, 0)):
        assert plan(*bad, out) == 2
