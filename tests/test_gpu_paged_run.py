"""The cache of pages in use: prompts, their continuations by several sequences, captured steps, other streams, and pools beyond 32 bits."""
import pytest
import torch

from cats_amd.paged import PagedCache
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _words(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


def _tables(positions, rot):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.cat([a, a], 1)
    return a.cos().float(), a.sin().float()


class _Run:
    """Sequences over a PagedCache beside what each of them should hold."""

    def __init__(self, layers, pages, heads, kv, D, page, dtype):
        self.g = torch.Generator().manual_seed(21)
        self.cache = PagedCache(layers, pages, kv, D, page, dtype)
        self.layers, self.heads, self.kv, self.D, self.dtype = layers, heads, kv, D, dtype
        self.cos, self.sin = _tables(600, D)
        self.held = {}  # (layer, sequence): k, v, in double, and the bound of k

    def call(self, ids, starts, counts, group=1, shared=None):
        """New tokens of the sequences through all layers; the outputs are checked."""
        cache = self.cache
        cache.reserve(ids, [s + n for s, n in zip(starts, counts)])
        rows = list(zip(starts, counts))
        at = ref.offsets_of(rows)
        table = cache.table(ids)
        offsets, start = _words(at), _words(starts)
        for layer in range(self.layers):
            q, k, v = (torch.randn(at[-1], h, self.D, generator=self.g).to(self.dtype) for h in (self.heads, self.kv, self.kv))
            turned = cache.append(layer, q.cuda(), k.cuda(), v.cuda(), offsets, start, table, self.cos.cuda(), self.sin.cuda())
            out = cache.attend(layer, turned, offsets, start, table, group=group, shared=None if shared is None else _words([shared]))
            for b, i in enumerate(ids):
                old = self.held.get((layer, i), tuple(torch.zeros(0, self.kv, self.D, dtype=torch.float64) for _ in range(3)))
                a, e, p = at[b], at[b + 1], slice(starts[b], starts[b] + counts[b])
                new, bound = ref.rotate(k[a:e], self.cos[p], self.sin[p])
                self.held[layer, i] = tuple(torch.cat([x[: starts[b]], y]) for x, y in zip(old, (new, v[a:e].double(), bound)))
                want, far = ref.rotate(q[a:e], self.cos[p], self.sin[p])
                assert ref.within(turned[a:e], want, far)
            pool = cache.k[layer].cpu(), cache.v[layer].cpu(), table.cpu()
            for b, i in enumerate(ids):
                kk, vv = ref.tokens(pool, b, starts[b] + counts[b])
                want = self.held[layer, i]
                assert ref.within(kk, want[0], want[2]) and torch.equal(vv.double(), want[1])
            assert ref.within(out, *ref.paged_attention(turned.cpu(), rows, 0, pool, self.D ** -0.5))
        return out

    def fork(self, i, count, length):
        new = self.cache.fork(i, count, length)
        for layer in range(self.layers):
            for j in new:
                self.held[layer, j] = tuple(x[:length] for x in self.held[layer, i])
        return new


@pytest.mark.parametrize("dtype,heads,kv,D,page", [(F16, 8, 2, 64, 16), (BF16, 4, 4, 128, 64)])
def test_from_prompts_to_steps(dtype, heads, kv, D, page):
    """Two prompts, one in pieces; four continuations of the first that share its pages, drafts that are taken back, and a sequence that ends and another in its pages."""
    r = _Run(2, 60, heads, kv, D, page, dtype)
    a, b = r.cache.open(), r.cache.open()
    r.call([a, b], [0, 0], [150, 37])
    r.call([b], [37], [61])
    beams = r.fork(a, 4, 150)
    for t in range(3):
        r.call(beams + [b], [150 + t] * 4 + [98 + t], [1] * 5)
        r.call(beams, [151 + t] * 4, [1] * 4, group=4, shared=150)  # the next token, which is given again
    r.call(beams, [153] * 4, [5] * 4, group=4, shared=150)
    for i in beams:
        r.cache.trim(i, 155)
    r.call(beams, [155, 155, 155, 155], [1, 3, 0, 1], group=4, shared=150)
    r.cache.close(a)
    r.cache.close(b)
    c = r.cache.open()
    r.call([c] + beams[:2], [0, 156, 158], [200, 1, 1])
    for i in [c] + beams:
        r.cache.close(i)
    assert r.cache.free == 60


def test_a_prompt_by_both():
    """A prompt over its own keys and over the pages that hold them: the same within both bounds."""
    import flash_gemv

    r = _Run(1, 40, 4, 2, 128, 32, BF16)
    ids = [r.cache.open() for _ in range(3)]
    g = torch.Generator().manual_seed(5)
    at = [0, 257, 258, 500]
    q, k, v = (torch.randn(500, h, 128, generator=g).bfloat16() for h in (4, 2, 2))
    r.cache.reserve(ids, [257, 1, 242])
    table, offsets, start = r.cache.table(ids), _words(at), _words([0, 0, 0])
    assert torch.equal(r.cache.append(0, q.cuda(), k.cuda(), v.cuda(), offsets, start, table).cpu(), q)  # without a rotation
    want, bound = ref.prompt_attention(q, k, v, at, at, 128 ** -0.5)
    assert ref.within(r.cache.attend(0, q.cuda(), offsets, start, table), want, bound)
    assert ref.within(flash_gemv.cats_prompt_attention(q.cuda(), k.cuda(), v.cuda(), offsets, 128 ** -0.5), want, bound)


def _step_state(B, group, shared, length, dtype=F16, heads=8, kv=2, D=64, page=16):
    """Tensors of a step of B sequences, in groups that share their first tokens, and of a call of prompts; the calls on them."""
    import flash_gemv

    g = torch.Generator().manual_seed(31)
    rows = [(length + 3 * b, 1) for b in range(B)]
    pool = ref.new_pool([(a, 8) for a, _ in rows], page, kv, D, dtype, group=group, shared=shared, room=2000 // page)
    ref.fill(pool, rows, g)
    s = {"kp": pool[0].cuda(), "vp": pool[1].cuda(), "table": pool[2].cuda(), "start": _words([a for a, _ in rows]), "offsets": _words(list(range(B + 1))),
         "at": _words([0, 40, 41, 41, 100]), "shared": _words([shared])}
    for n, h in (("q", heads), ("k", kv), ("v", kv)):
        s[n] = torch.randn(B, h, D, generator=g).to(dtype).cuda()
        s["p" + n] = torch.randn(100, h, D, generator=g).to(dtype).cuda()
    s["cos"], s["sin"] = (x.cuda() for x in _tables(length + 3 * B + 10, D))

    def calls():
        q = flash_gemv.cats_paged_append(s["q"], s["k"], s["v"], s["offsets"], s["start"], s["cos"], s["sin"], s["kp"], s["vp"], s["table"])
        return (q, flash_gemv.cats_paged_attention(q, s["offsets"], s["start"], s["kp"], s["vp"], s["table"], 0.125, 0, group, s["shared"] if group > 1 else None),
                flash_gemv.cats_prompt_attention(s["pq"], s["pk"], s["pv"], s["at"], 0.125, 30))

    return s, calls


def _same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("B,group,shared,length", [(3, 1, 0, 60), (2, 1, 0, 3000), (4, 4, 200, 200), (24, 24, 1100, 1100)])
def test_captured_steps(B, group, shared, length):
    """A captured step follows its tensors: new tokens, positions, lengths of prompts and tables.  The result is the eager one's, whatever runs between."""
    s, calls = _step_state(B, group, shared, length)
    for _ in range(2):
        calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = calls()
    for t in range(5):
        for n in ("q", "k", "v", "pq", "pk", "pv"):
            s[n].normal_()
        s["start"] += 1
        s["at"].copy_(_words([[0, 40, 41, 41, 100], [5, 10, 80, 80, 90], [0, 100, 100, 100, 100], [0, 1, 2, 3, 4], [0, 0, 0, 0, 0]][t]))
        if t == 3 and group == 1:  # sequences change places: an entry may be no page now, and the query that sees it NaN
            s["table"].copy_(s["table"].roll(1, 0))
        table = s["table"].clone()
        want = [x.clone() for x in calls()]
        pages = s["kp"].clone(), s["vp"].clone()
        graph.replay()
        assert all(_same(a, b) for a, b in zip([*outs, s["kp"], s["vp"]], [*want, *pages])) and torch.equal(s["table"], table)
        torch.randn(1000, 1000, device="cuda").sum().item()


def test_two_graphs_and_eager_calls_on_other_streams():
    """Each has scratch memory of its own."""
    states = [_step_state(2, 1, 0, 3000), _step_state(24, 24, 1100, 1100), _step_state(5, 1, 0, 2000, BF16, 4, 4, 128)]
    want = [[x.clone() for x in calls()] for _, calls in states]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _, calls in states[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(calls())
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        eager = []
        for i, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                for _ in range(4):
                    if i < 2:
                        graphs[i].replay()
                    else:
                        eager.append(states[2][1]())
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        for got, to in [*zip(outs, want), *((e, want[2]) for e in eager)]:
            assert all(torch.equal(a, b) for a, b in zip(got, to))
        torch.cuda.synchronize()


def test_pools_beyond_32_bits():
    """Pages whose numbers lie more than 2^32 elements from the first: as in a small pool."""
    import flash_gemv

    g = torch.Generator().manual_seed(41)
    B, heads, kv, D, page, pages = 3, 16, 8, 128, 64, 70000
    far = torch.tensor([[69999, 65536, 1, -1], [33000, 69998, 65537, -1], [40000, 32768, 68000, -1]], dtype=torch.int32)
    near = torch.tensor([[0, 1, 2, -1], [3, 4, 5, -1], [6, 7, 8, -1]], dtype=torch.int32)
    counts = [150, 100, 191]
    at = ref.offsets_of([(0, n) for n in counts])
    q, k, v = (torch.randn(at[-1], h, D, generator=g).half().cuda() for h in (heads, kv, kv))
    steps = [torch.randn(B, h, D, generator=g).half().cuda() for h in (heads, kv, kv)]
    outs = []
    for table, n in ((near, 9), (far, pages)):
        kp, vp = (torch.empty(n, kv, page, D, dtype=F16, device="cuda") for _ in range(2))
        t = table.cuda()
        flash_gemv.cats_paged_append(None, k, v, _words(at), _words([0] * B), None, None, kp, vp, t)
        prompt = flash_gemv.cats_paged_attention(q, _words(at), _words([0] * B), kp, vp, t, 0.1)
        flash_gemv.cats_paged_append(None, steps[1], steps[2], _words([0, 1, 2, 3]), _words(counts), None, None, kp, vp, t)
        step = flash_gemv.cats_paged_attention(steps[0], _words([0, 1, 2, 3]), _words(counts), kp, vp, t, 0.1)
        parts = flash_gemv.cats_paged_attention(steps[0], _words([0, 1, 2, 3]), _words(counts), kp, vp, torch.cat([t, t.new_full((B, 40), -1)], 1), 0.1)
        outs.append((prompt.cpu(), step.cpu(), parts.cpu()))
        del kp, vp
    torch.cuda.empty_cache()
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert not any(x.isnan().any() for x in outs[0])


def test_strides_beyond_32_bits():
    """Tokens that lie 2^23 elements apart."""
    import flash_gemv

    n, apart = 300, 1 << 23
    g = torch.Generator().manual_seed(42)
    room = torch.empty(n * apart, dtype=BF16, device="cuda")
    near = [torch.randn(n, h, 64, generator=g).bfloat16().cuda() for h in (4, 2, 2)]
    far = [room.as_strided((n, h, 64), (apart, 64, 1), 1024 * i) for i, h in enumerate((4, 2, 2))]
    for a, b in zip(far, near):
        a.copy_(b)
    at = _words([0, 280, 300])
    assert torch.equal(flash_gemv.cats_prompt_attention(*far, at, 0.125), flash_gemv.cats_prompt_attention(*near, at, 0.125))
    outs = []
    table = torch.arange(40, dtype=torch.int32, device="cuda").reshape(2, 20)
    for q, k, v in (far, near):
        kp, vp = (torch.zeros(40, 2, 16, 64, dtype=BF16, device="cuda") for _ in range(2))
        flash_gemv.cats_paged_append(None, k, v, at, _words([0, 0]), None, None, kp, vp, table)
        outs.append((kp, vp, flash_gemv.cats_paged_attention(q, at, _words([0, 0]), kp, vp, table, 0.125)))
    del room, far
    torch.cuda.empty_cache()
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_a_row_of_the_table_for_all():
    """Tables whose rows lie apart, or are one and the same."""
    import flash_gemv

    g = torch.Generator().manual_seed(43)
    rows = [(200, 1)] * 6
    pool = ref.new_pool(rows[:1], 32, 2, 64, F16)
    ref.fill(pool, rows[:1], g)
    q = torch.randn(6, 4, 64, generator=g).half()
    all_alike = pool[2].expand(6, -1)
    want = ref.paged_attention(q, rows, 0, (*pool[:2], all_alike), 0.125)
    kp, vp, t = (x.cuda() for x in pool)
    wide = torch.cat([t.expand(6, -1), torch.full((6, 5), -1, dtype=torch.int32, device="cuda")], 1)
    args = q.cuda(), _words(list(range(7))), _words([200] * 6), kp, vp
    for table in (t.expand(6, -1), wide[:, : t.shape[1]], wide):
        assert ref.within(flash_gemv.cats_paged_attention(*args, table, 0.125), *want)
    assert ref.within(flash_gemv.cats_paged_attention(*args, t.expand(6, -1), 0.125, 0, 6, _words([192])), *want)


def test_calls_that_are_refused():
    import flash_gemv

    x, w = torch.zeros(2, 2, 64, dtype=F16, device="cuda"), _words([0, 2])
    pool = torch.zeros(2, 2, 16, 64, dtype=F16, device="cuda")
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    paged = lambda q=x, offsets=w, start=w[:1], kp=pool, vp=pool, table=table, scale=0.1, **more: flash_gemv.cats_paged_attention(q, offsets, start, kp, vp, table, scale, **more)
    append = lambda q=x, k=x, v=x, offsets=w, start=w[:1], cos=None, sin=None, kp=pool, vp=pool, table=table: flash_gemv.cats_paged_append(q, k, v, offsets, start, cos, sin, kp, vp, table)
    prompt = lambda q=x, k=x, v=x, offsets=w, scale=0.1, **more: flash_gemv.cats_prompt_attention(q, k, v, offsets, scale, **more)
    grad, cos = x.clone().requires_grad_(), torch.zeros(4, 64, device="cuda")
    for call in (lambda: paged(grad), lambda: append(grad), lambda: append(k=grad), lambda: prompt(grad), lambda: prompt(v=grad),
                 lambda: paged(x.float()), lambda: paged(x.bfloat16()), lambda: paged(x[:, :, :48]), lambda: paged(x[0]), lambda: paged(torch.zeros(2, 3, 64, dtype=F16, device="cuda")),
                 lambda: paged(offsets=w.int()), lambda: paged(offsets=w[:1]), lambda: paged(start=w), lambda: paged(table=table.long()), lambda: paged(table=table.expand(2, -1)),
                 lambda: paged(table=table[:, :0]), lambda: paged(kp=pool[0]), lambda: paged(vp=pool[:1]), lambda: paged(kp=pool[:, :, :15]), lambda: paged(window=-1),
                 lambda: paged(scale=0.0), lambda: paged(group=2), lambda: paged(group=0), lambda: paged(shared=_words([1, 2])), lambda: paged(shared=w[:1].int()),
                 lambda: append(v=x[:1]), lambda: append(q=x[:1]), lambda: append(k=x[:, :1], v=x[:, :1]), lambda: append(cos=cos), lambda: append(cos=cos[:, :24], sin=cos[:, :24]),
                 lambda: append(cos=cos.double(), sin=cos.double()), lambda: prompt(k=x[:1], v=x[:1]), lambda: prompt(k=x[:, :1]), lambda: prompt(offsets=w[:1]),
                 lambda: prompt(scale=float("nan")), lambda: prompt(window=2 ** 31), lambda: paged(offsets=w.cpu()), lambda: paged(table=table.cpu())):
        with pytest.raises(RuntimeError):
            call()


def test_none_of_them():
    """No tokens, or no keys."""
    import flash_gemv

    x, pool = torch.zeros(0, 2, 64, dtype=F16, device="cuda"), torch.ones(2, 2, 16, 64, dtype=F16, device="cuda")
    table, w = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), _words([0, 0, 0, 0])
    assert flash_gemv.cats_paged_append(x, x, x, w, w[:3], None, None, pool, pool, table).shape == x.shape
    assert flash_gemv.cats_paged_attention(x, w, w[:3], pool, pool, table, 0.1).shape == x.shape
    assert flash_gemv.cats_prompt_attention(x, x, x, w, 0.1).shape == x.shape
    y = torch.ones(4, 2, 64, dtype=F16, device="cuda")
    assert flash_gemv.cats_prompt_attention(y, x, x, w[:2], 0.1, k_offsets=w[:2]).eq(0).all()
    assert flash_gemv.cats_paged_attention(y, w, w[:3], pool, pool, table, 0.1).eq(0).all()
