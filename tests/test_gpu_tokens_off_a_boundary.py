"""Tokens whose elements stand side by side but begin off a 16-byte boundary, as a slice of a larger buffer may: the results are those of tokens that begin on one."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _moved(x, by):
    buffer = torch.empty(x.numel() + by, dtype=x.dtype, device=x.device)
    y = buffer[by:].view(x.shape)
    assert y.copy_(x).is_contiguous() and y.data_ptr() % 16
    return y


def _words(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("by", [1, 4])
def test_packed_tokens(by, dtype):
    import flash_gemv

    g = torch.Generator(device="cuda").manual_seed(71)
    q, k, v = (torch.randn(60, h, 64, generator=g, device="cuda").to(dtype) for h in (4, 2, 2))
    at, start, table = _words([0, 20, 60]), _words([3, 0]), torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    cos, sin = (torch.randn(64, 64, generator=g, device="cuda") for _ in range(2))

    def calls(q, k, v):
        pages = [torch.zeros(8, 2, 16, 64, dtype=dtype, device="cuda") for _ in range(2)]
        turned = flash_gemv.cats_paged_append(q, k, v, at, start, cos, sin, *pages, table)
        return turned, *pages, flash_gemv.cats_paged_attention(q, at, start, *pages, table, 0.125), flash_gemv.cats_prompt_attention(q, k, v, at, 0.125)

    want = calls(q, k, v)
    for moved in ((_moved(q, by), k, v), (q, _moved(k, by), v), (q, k, _moved(v, by)), tuple(_moved(x, by) for x in (q, k, v))):
        assert all(torch.equal(a, b) for a, b in zip(calls(*moved), want))


@pytest.mark.parametrize("by", [1, 4])
def test_tokens_of_a_cache_in_8_bits(by):
    from cats_amd.kv8 import Kv8Cache

    g = torch.Generator(device="cuda").manual_seed(72)
    q, k, v = (torch.randn(2, 100, h, 64, generator=g, device="cuda").half() for h in (4, 2, 2))

    def calls(q, k, v):
        cache = Kv8Cache(2, 2, 200, 64, F16)
        cache.append(k, v, _words([0]))
        return cache.k8.float(), cache.v8.float(), cache.k_tail, cache.v_tail, cache.attend(q, _words([0]))

    want = calls(q, k, v)
    for moved in ((_moved(q, by), k, v), (q, _moved(k, by), v), (q, k, _moved(v, by))):
        assert all(torch.equal(a, b) for a, b in zip(calls(*moved), want))
