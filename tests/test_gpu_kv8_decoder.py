"""A decode step over a cache in 8 bits, and the decoder with such a cache and with beam search."""
import math

import pytest
import torch

from cats_amd import decoder as dec
from tests import cache_reference as ref
from tests.test_gpu_decode_step import _check, _randn

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _step(B, heads, hd, blocks, max_len, pos, dtype, norm=False):
    """One step behind `pos` tokens against the same products in 64 bits."""
    import flash_gemv  # noqa: F401

    H = heads * hd
    g = torch.Generator().manual_seed(H + pos)
    h, x = _randn(g, B, 1, H, dtype=dtype, scale=2.0), _randn(g, B, 1, H, dtype=dtype)
    ws = [_randn(g, H, H, dtype=dtype, scale=1 / math.sqrt(H)) for _ in range(4)]
    cache = ref.new_cache(B, heads, blocks, hd, dtype)
    if pos > 0:
        k, v = _randn(g, B, pos, heads, hd, dtype=dtype), _randn(g, B, pos, heads, hd, dtype=dtype)
        cache = ref.append(cache, k, v, [0] * B, None)
    ang = torch.outer(torch.arange(max_len).float(), 1.0 / (10000.0 ** (torch.arange(0, hd, 2).float() / hd)))
    emb = torch.cat((ang, 0.7 * ang + 0.3), -1)
    cos, sin = emb.cos().to(dtype), emb.sin().to(dtype)
    nw = (1 + 0.1 * torch.randn(H, generator=g)).to(dtype) if norm else None
    on = ref.to(cache, "cuda")
    args = (h.cuda(), x.cuda(), nw.cuda() if norm else None, 1e-5, *(w.cuda() for w in ws), *(on[f] for f in ref.FIELDS), cos.cuda(), sin.cuda())
    out = torch.ops.flash_gemv.cats_kv8_attention_step(*args, torch.tensor([pos], device="cuda"))
    xr = x
    if norm:
        xr = (x.double() * torch.rsqrt(x.double().pow(2).mean(-1, keepdim=True) + 1e-5)).to(dtype)
        xr = (nw.double() * xr.double()).to(dtype)
    q, k, v = (xr.double().view(B, -1) @ w.double().t() for w in ws[:3])
    q, k, v = (t.view(B, heads, hd) for t in (q, k, v))
    half = lambda t: torch.cat((-t[..., hd // 2:], t[..., : hd // 2]), -1)
    q, k = (t * cos.double()[pos] + half(t) * sin.double()[pos] for t in (q, k))
    # what the kernel stored in the tails is what attention reads and what the block is quantised from
    got_k, got_v = on["k_tail"][:, :, pos % 64].cpu(), on["v_tail"][..., pos % 64].cpu()
    _check(got_k, k, dtype, 2 * H)
    _check(got_v, v, dtype, 2 * H)
    want_cache = ref.append(cache, got_k.view(B, 1, heads, hd), got_v.view(B, 1, heads, hd), [pos] * B, None)
    for f in ref.FIELDS:
        assert ref.same(on[f], want_cache[f]), f
    att, _ = ref.attention(want_cache, q.to(dtype).view(B, 1, heads, hd), [pos] * B, None, 1 / math.sqrt(hd))
    # attention and q are rounded before the products that follow: half a step of each of the H terms, added as random signs
    _check(out.view(B, H), h.double().view(B, H) + att.view(B, H) @ ws[3].double().t(), dtype, 8 * H)
    for bad in (-1, max_len):
        before = {f: t.clone() for f, t in on.items()}
        out = torch.ops.flash_gemv.cats_kv8_attention_step(*args, torch.tensor([bad], device="cuda"))
        assert out.isnan().all()
        for f in ref.FIELDS:
            assert ref.same(on[f], before[f]), f


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,heads,hd,pos", [(1, 4, 64, 0), (1, 4, 64, 63), (2, 2, 128, 64), (3, 4, 32, 127), (8, 1, 256, 200), (4, 8, 64, 255), (1, 2, 256, 130)])
@pytest.mark.parametrize("norm", [False, True])
def test_step(B, heads, hd, pos, dtype, norm):
    """Blocks that the token opens, fills and completes; projections a wave a row and on the matrix cores."""
    _step(B, heads, hd, 5, 300, pos, dtype, norm)


def test_step_over_a_long_cache():
    """Attention in splits, one of which completes a block."""
    _step(1, 2, 64, 100, 6400, 4095, F16)
    _step(1, 2, 64, 100, 6399, 4200, BF16)


def _model(dtype, kv_cache, max_len=200, device="cuda", layers=3, heads=4, hidden=256):
    cfg = dec.DecoderConfig(hidden_size=hidden, intermediate_size=384, num_layers=layers, num_heads=heads, vocab_size=120, max_len=max_len, kv_cache=kv_cache)
    return dec.LlamaDecoder(cfg, dtype, device, seed=0, init_std=0.1).eval()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decoder_with_a_cache_in_8_bits(dtype):
    """A prompt in pieces, then single tokens with torch's projections: every layer's cache to the bit and its attention, given the layer's own
    projections."""
    m = _model(dtype, "e4m3")
    toks = torch.randint(0, 120, (2, 135), generator=torch.Generator().manual_seed(1)).cuda()
    seen = [dict(x=[], out=[]) for _ in m.layers]
    hooks = []
    for l, s in zip(m.layers, seen):
        hooks.append(l.self_attn.q_proj.register_forward_pre_hook(lambda mod, a, s=s: s["x"].append(a[0].clone())))
        hooks.append(l.self_attn.o_proj.register_forward_pre_hook(lambda mod, a, s=s: s["out"].append(a[0].clone())))
    pieces = [(0, 100), (100, 127), (127, 128), (128, 129), (129, 135)]
    with torch.no_grad():
        m.reset_cache(2)
        for a, b in pieces:
            m(toks[:, a:b], torch.arange(a, b, device="cuda"))
        for h in hooks:
            h.remove()
        for l, s in zip(m.layers, seen):
            at, cache = l.self_attn, ref.new_cache(2, 4, 4, 64, dtype, fill=0.0)
            cache["k_scale"].fill_(1.0), cache["v_scale"].fill_(1.0)  # as a new cache has them
            for (a, b), x, out in zip(pieces, s["x"], s["out"]):
                cos, sin = m.cos_table[a:b], m.sin_table[a:b]
                q, k, v = (p(x).view(2, b - a, 4, 64).transpose(1, 2) for p in (at.q_proj, at.k_proj, at.v_proj))
                q, k = (t * cos + dec.rotate_half(t) * sin for t in (q, k))
                q, k, v = (t.transpose(1, 2).cpu() for t in (q, k, v))
                cache = ref.append(cache, k, v, [a, a], None)
                want, bound = ref.attention(cache, q, [a, a], None, 0.125)
                assert ref.within(out.view(2, b - a, 4, 64), want, bound), (a, b)
            for f, t in zip(ref.FIELDS, at.kv8.tensors()):
                assert ref.same(t, cache[f]), f


@pytest.mark.parametrize("T", [1, 40])
def test_tokens_that_were_never_stored_are_zeros(T):
    from cats_amd.kv8 import Kv8Cache

    c = Kv8Cache(2, 1, 256, 64, F16)
    q = _randn(torch.Generator().manual_seed(3), 2, T, 4, 64, dtype=F16).cuda()
    assert (c.attend(q, torch.tensor([200, 7], device="cuda")) == 0).all()


def test_greedy_with_a_cache_in_8_bits_replays_its_graph():
    m = _model(F16, "e4m3")
    prompt = torch.randint(0, 120, (1, 60), generator=torch.Generator().manual_seed(2)).cuda()
    eager, _ = m.generate_greedy(prompt, 80, use_graph=False)
    caches = [t.clone() for l in m.layers for t in l.self_attn.caches()[0]]
    graph, _ = m.generate_greedy(prompt, 80, use_graph=True)
    assert torch.equal(eager, graph)
    for a, b in zip(caches, (t for l in m.layers for t in l.self_attn.caches()[0])):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("positions", [[40, 41, 43], [40, 40, 41], [42, 41, 40], [41, 40, 42], [2, 3, 40]])
def test_positions_that_are_no_row_give_nan(positions):
    """A cache in 8 bits stores a call's tokens one behind the other: any other positions leave it as it is, and no logits come of them."""
    m = _model(F16, "e4m3", 70)
    toks = torch.randint(0, 120, (2, 43), generator=torch.Generator().manual_seed(6)).cuda()
    with torch.no_grad():
        m.reset_cache(2)
        m(toks[:, :40], torch.arange(40, device="cuda"))
        kept = [t.clone() for l in m.layers for t in l.self_attn.caches()[0]]
        assert m(toks[:, 40:], torch.tensor(positions, device="cuda")).isnan().all()
        for a, l in zip(kept, (t for l in m.layers for t in l.self_attn.caches()[0])):
            assert torch.equal(a.view(torch.uint8), l.view(torch.uint8))
        with pytest.raises(ValueError, match="one position"):
            m(toks[:, 40:], torch.tensor([40], device="cuda"))
        assert m(toks[:, 40:], torch.arange(40, 43, device="cuda")).isfinite().all()


@pytest.mark.parametrize("kv_cache", ["dtype", "e4m3"])
def test_one_token_has_no_step_to_capture(kv_cache):
    """The only token comes from the prompt: a step made for the capture alone would store its token behind the output."""
    m = _model(F16, kv_cache, 40)
    prompt = torch.randint(0, 120, (1, 39), generator=torch.Generator().manual_seed(4)).cuda()
    eager, _ = m.generate_greedy(prompt, 1, use_graph=False)
    graph, _ = m.generate_greedy(prompt, 1, use_graph=True)
    assert eager.shape == (1,) and torch.equal(eager, graph)


def _search(m, prompt, beams, gen_len, eos):
    """Beam search that computes every beam from its first token at every step."""
    G, P = prompt.shape
    hyps = [[([], 0.0, False)] for _ in range(G)]
    for _ in range(gen_len):
        rows = [prompt[g].tolist() + h[0] for g in range(G) for h in hyps[g]]
        m.reset_cache(len(rows))
        lg = m(torch.tensor(rows), torch.arange(len(rows[0])))[:, -1].double()
        n = len(hyps[0])
        done = torch.tensor([[h[2] for h in hs] for hs in hyps])
        found = ref.select(lg.view(G, n, -1), torch.tensor([[h[1] for h in hs] for hs in hyps], dtype=torch.float64), done, eos, beams)
        hyps = [[(hyps[g][b][0] + [t], s, d) for s, b, t, d in found[g]] for g in range(G)]
    return [[h[0] for h in hs] for hs in hyps], [[h[1] for h in hs] for hs in hyps]


@pytest.mark.parametrize("G,beams,gen_len,eos", [(1, 4, 12, -1), (2, 3, 12, 7), (2, 8, 6, 100), (1, 1, 5, -1), (1, 5, 1, -1)])
@pytest.mark.parametrize("graph", [False, True])
def test_beams_are_those_of_a_search_that_keeps_no_cache(G, beams, gen_len, eos, graph):
    """float32 models, up to eight rows a step (the step's kernels) and sixteen (torch's)."""
    prompt = torch.randint(0, 120, (G, 9), generator=torch.Generator().manual_seed(G + beams))
    with torch.no_grad():
        model, plain = _model(F32, "dtype", 40), _model(F32, "dtype", 40, "cpu")
        plain.load_state_dict(model.state_dict())  # the devices draw other weights from one seed
        want, scores = _search(plain, prompt, beams, gen_len, eos)
        tokens, got = model.generate_beams(prompt.cuda(), beams, gen_len, eos, use_graph=graph)
    assert tokens.shape == (G, beams, gen_len) and tokens.tolist() == want
    torch.testing.assert_close(got.cpu().double(), torch.tensor(scores, dtype=torch.float64), rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("G,beams", [(1, 4), (2, 4), (3, 4)])
def test_beams_over_caches_in_8_bits(dtype, G, beams):
    """Past the end of a block, with beams that move: the same from a graph, and every beam's score is that of its own tokens fed one by one."""
    m = _model(dtype, "e4m3")
    prompt = torch.randint(0, 120, (G, 50), generator=torch.Generator().manual_seed(G)).cuda()
    tokens, scores = m.generate_beams(prompt, beams, 40, use_graph=False)
    again, scores2 = m.generate_beams(prompt, beams, 40, use_graph=True)
    assert torch.equal(tokens, again) and torch.equal(scores, scores2)
    assert bool((scores[:, :-1] >= scores[:, 1:]).all())
    with torch.no_grad():
        rows = torch.cat([prompt.repeat_interleave(beams, 0), tokens.view(G * beams, 40)], 1)
        m.reset_cache(G)
        lg = [m(prompt, torch.arange(50, device="cuda"))[:, -1].repeat_interleave(beams, 0)]
        for layer in m.layers:
            layer.self_attn.repeat_cache(beams)
        for i in range(50, 89):
            lg.append(m(rows[:, i:i + 1], torch.tensor([i], device="cuda"))[:, -1])
        lp = torch.log_softmax(torch.stack(lg, 1).double(), -1).gather(2, rows[:, 50:, None]).sum((1, 2)).view(G, beams)
    # the same kernels on the same values row by row: only the score's 40 roundings to float and the logarithms' sums differ
    torch.testing.assert_close(scores.double(), lp, rtol=40 * 2.0 ** -23, atol=40 * 2.0 ** -21)


def test_what_the_decoder_refuses():
    m = _model(F16, "e4m3", 40)
    m.reset_cache(1)
    toks = torch.zeros(1, 3, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="no gradient"):
        m(toks, torch.arange(3, device="cuda"))
    for beams, n in ((17, 2), (0, 2), (2, 0), (2, 38)):
        with pytest.raises(ValueError):
            m.generate_beams(toks, beams, n)
    with pytest.raises(ValueError):
        _model(F32, "e4m3", 40).reset_cache(1)
    with pytest.raises(ValueError):
        _model(F16, "int4", 40).reset_cache(1)
