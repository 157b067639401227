"""What the operators of a cache in 8 bits and of beam search are measured on: the calls a decode program makes around its key / value caches.

A case is one call of ``flash_gemv`` on tensors that such a program keeps.  ``listed()`` names twelve of them, ``draw()`` gives others of
the same ranges.  Fields: ``op`` (below), ``dtype`` of the model, and the sizes of the operator.

  attention  flash_gemv.cats_kv8_attention   T new tokens of each of B rows over its cache: ``heads`` query and ``kv_heads`` cached heads of D
  append     flash_gemv.cats_kv8_append      stores T new tokens of each of B rows, quantising the blocks that are complete
  select     flash_gemv.cats_beam_select     the best ``beams`` continuations of ``groups`` searches over V words
  reorder    flash_gemv.cats_cache_reorder   the caches of ``layers`` layers moved to the beams that go on

The cache in 8 bits: blocks of 64 tokens, each with one power of two as its scale for a head's keys and one for its values.  ``k8`` (B, kv_heads,
blocks, 64, D) and ``v8`` (B, kv_heads, blocks, D, 64) hold e4m3 numbers, the scales (B, kv_heads, blocks) are float32, and a row's last
block, complete or not, is read as it was given from ``k_tail`` (B, kv_heads, 64, D) and ``v_tail`` (B, kv_heads, D, 64).
"""
import math

import torch

own = False  # False: the operators in elementary torch operations; True: the framework's kernels

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
BLOCK = 64


def listed():
    def attention(name, B, T, heads, kv_heads, D, length, dtype, window=0, ragged=False):
        return {"name": name, "op": "attention", "B": B, "T": T, "heads": heads, "kv_heads": kv_heads, "D": D, "length": length, "dtype": dtype,
                "window": window, "ragged": ragged}

    return [
        # single-stream decoding of a 7B model, early in the answer: launches and dependent trips are all there is
        attention("step - 1 row - 100 tokens", 1, 1, 32, 32, 128, 100, "fp16"),
        # a server's batch of sequences of all lengths, grouped heads
        attention("step - 16 rows - to 4096", 16, 1, 32, 8, 128, 4096, "bf16", ragged=True),
        # one very long document: the cache is all there is to read
        attention("step - 1 row - 131072 tokens", 1, 1, 32, 8, 128, 131072, "fp16"),
        # five drafted tokens to be checked, an odd number of heads a group, a sliding window
        attention("draft of 5 - window 4096", 4, 5, 14, 2, 64, 20001, "bf16", window=4096, ragged=True),
        # a prompt of a 7B model
        attention("prompt - 2048 tokens", 1, 2048, 32, 32, 128, 2048, "fp16"),
        # the next piece of two long prompts that are taken in pieces, the shorter one padded
        attention("piece of 512 behind 7680", 2, 512, 32, 8, 128, 8192, "bf16", ragged=True),
        # eight prompts' keys and values go into a fresh cache
        {"name": "append - 8 prompts of 2048", "op": "append", "B": 8, "T": 2048, "kv_heads": 32, "D": 128, "length": 2048, "dtype": "fp16"},
        # one token for each of many streams; some of them complete a block
        {"name": "append - 64 rows", "op": "append", "B": 64, "T": 1, "kv_heads": 8, "D": 128, "length": 1088, "dtype": "bf16"},
        # four beams of one search over a 7B model's vocabulary
        {"name": "select - 4 beams", "op": "select", "groups": 1, "beams": 4, "V": 32000, "dtype": "fp16", "finished": False},
        # many searches of sixteen beams over a large, odd vocabulary, some beams finished
        {"name": "select - 16 x 16 beams", "op": "select", "groups": 16, "beams": 16, "V": 100003, "dtype": "fp32", "finished": True},
        # four beams' 16-bit caches of a few layers
        {"name": "reorder - 4 beams", "op": "reorder", "groups": 1, "beams": 4, "kv_heads": 32, "D": 128, "length": 300, "layers": 4, "dtype": "fp16", "e4m3": False},
        # a batch of searches over caches in 8 bits
        {"name": "reorder - 8 x 4 beams - e4m3", "op": "reorder", "groups": 8, "beams": 4, "kv_heads": 8, "D": 128, "length": 4000, "layers": 2,
         "dtype": "bf16", "e4m3": True},
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))

    dtype = rng.choice(["fp16", "bf16"])
    op = rng.choice(["attention", "attention", "append", "select", "reorder"])
    D, kv_heads = rng.choice([32, 64, 128, 128, 256]), rng.choice([1, 2, 4, 8, 8, 16, 32])
    if op == "attention":
        group = rng.choice([1, 1, 2, 3, 4, 7, 8])
        if rng.random() < 0.6:  # a step, or a few drafted tokens
            T = rng.choice([1, 1, 1, rng.randint(2, 16)])
            B, length = log(1, 32), log(T, 65536)
            while B * length * kv_heads * D > 1 << 27:
                length = max(T, length // 2)
        else:  # a prompt or a piece of one
            T = log(17, 2048)
            B, length = log(1, 4), T + rng.choice([0, log(1, 8192)])
            while B * T * length * kv_heads * group * D > 1 << 34:
                B, T, length = max(1, B // 2), max(1, T // 2), max(1, length // 2)
        return {"op": op, "B": B, "T": T, "heads": kv_heads * group, "kv_heads": kv_heads, "D": D, "length": length, "dtype": dtype,
                "window": rng.choice([0, 0, log(16, 8192)]), "ragged": rng.random() < 0.5}
    if op == "append":
        T = rng.choice([1, log(2, 4096)])
        B = log(1, 64)
        while B * T * kv_heads * D > 1 << 25:
            T = max(1, T // 2)
        return {"op": op, "B": B, "T": T, "kv_heads": kv_heads, "D": D, "length": T if T > 1 else log(1, 4000), "dtype": dtype}
    if op == "select":
        groups, beams = log(1, 32), rng.randint(1, 16)
        return {"op": op, "groups": groups, "beams": beams, "V": log(beams + 1, 160000 if groups * beams <= 160 else 50000), "dtype": rng.choice(["fp16", "bf16", "fp32"]),
                "finished": rng.random() < 0.5}
    groups, beams, layers, length = log(1, 8), rng.randint(2, 8), rng.randint(1, 4), log(1, 4000)
    while groups * beams * layers * kv_heads * D * length > 1 << 27:
        length = max(1, length // 2)
    return {"op": op, "groups": groups, "beams": beams, "kv_heads": kv_heads, "D": D, "length": length, "layers": layers, "dtype": dtype, "e4m3": rng.random() < 0.5}


# ---- sizes that follow from a case --------------------------------------------------------------------------------------------------

def blocks_of(length):
    """Blocks of a cache that has room for a quarter more than `length` tokens."""
    return -(-(length + length // 4 + 1) // BLOCK)


def rows_of(case):
    """(start, count) of each row: where its new tokens go, and how many of the T they are."""
    B, T, length = case["B"], case["T"], case["length"]
    if case["op"] == "append":  # whole prompts, or one token each at positions of their own
        return [(0, T)] * B if T > 1 else [(length - 1 - 7 * b % length, 1) for b in range(B)]
    if not case["ragged"]:
        return [(length - T, T)] * B
    count = [max(1, T - b * T // (2 * B)) for b in range(B)]
    return [(max(n, length - b * length // (2 * B)) - n, n) for b, n in enumerate(count)]


def pairs_of(case):
    """Query-key pairs of one head, and keys that any query of a row sees, over all rows."""
    pairs = keys = 0
    w = case["window"]
    for start, n in rows_of(case):
        first = start + 1  # keys that the first query sees
        pairs += n * first + n * (n - 1) // 2
        keys += start + n
        if w:
            lost = max(0, first - w)  # of the first query; the others lose one more each
            gone = max(0, start + n - w)
            pairs -= (lost + gone) * (gone - lost + 1) // 2 if lost else gone * (gone + 1) // 2
            keys -= lost
    return pairs, keys


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "attention":
        pairs, keys = pairs_of(case)
        return {"bytes": 2 * keys * case["kv_heads"] * case["D"] + 2 * e * case["heads"] * case["D"] * sum(n for _, n in rows_of(case)),
                "flops": 4 * pairs * case["heads"] * case["D"]}
    if case["op"] == "append":
        tokens, D = case["B"] * case["T"], case["kv_heads"] * case["D"]
        return {"bytes": 2 * tokens * D * (e + (1 if case["T"] > 1 else e)), "flops": 0}
    if case["op"] == "select":
        n = case["groups"] * case["beams"] * case["V"]
        return {"bytes": n * e, "flops": 2 * n}
    # the rows that are read, and those that are written, of keys and values
    moved = sum(len({p for j, p in enumerate(g) if p != j}) + sum(p != j for j, p in enumerate(g)) for g in parents_of(case))
    tail = BLOCK * e if case["e4m3"] else 0
    return {"bytes": 2 * moved * case["layers"] * case["kv_heads"] * case["D"] * (case["length"] * (1 if case["e4m3"] else e) + tail), "flops": 0}


def parents_of(case):
    """The beam that each beam of a group goes on from: about half of them move."""
    n = case["beams"]
    return [[max(0, j - 1 - (j + g) % 2) if (j + g) % 2 else j for j in range(n)] for g in range(case["groups"])]


# ---- inputs --------------------------------------------------------------------------------------------------------------------------

def _cache(case, B, g):
    """A cache in 8 bits that holds `length` tokens a row (and, behind them, what an earlier sequence left)."""
    kv, D, dt = case["kv_heads"], case["D"], DTYPES[case["dtype"]]
    n = blocks_of(case["length"])

    def codes(*shape):  # a block's largest number is near 448
        out = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
        for row in range(shape[0]):
            out[row] = (torch.randn(shape[1:], generator=g, device="cuda") * 110).clamp_(-448, 448).to(torch.float8_e4m3fn)
        return out

    def scales():
        return torch.exp2(torch.randint(-8, -5, (B, kv, n), generator=g, device="cuda").float())

    return {"k8": codes(B, kv, n, BLOCK, D), "v8": codes(B, kv, n, D, BLOCK), "k_scale": scales(), "v_scale": scales(),
            "k_tail": torch.randn(B, kv, BLOCK, D, generator=g, device="cuda").to(dt), "v_tail": torch.randn(B, kv, D, BLOCK, generator=g, device="cuda").to(dt)}


CACHE = ("k8", "v8", "k_scale", "v_scale", "k_tail", "v_tail")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] in ("attention", "append"):
        B, T, D = case["B"], case["T"], case["D"]
        s.update(_cache(case, B, g))
        rows = rows_of(case)
        s["start"] = torch.tensor([a for a, _ in rows], device="cuda")
        s["count"] = torch.tensor([n for _, n in rows], device="cuda")
        if case["op"] == "attention":
            s["q"] = (torch.randn(B, T, case["heads"], D, generator=g, device="cuda") * 2).to(dt)
            s["scale"] = 1 / math.sqrt(D)
        else:
            channel = torch.exp(torch.randn(case["kv_heads"], D, generator=g, device="cuda") * 0.5)  # keys have channels of their own size
            s["k"] = (torch.randn(B, T, case["kv_heads"], D, generator=g, device="cuda") * channel).to(dt)
            s["v"] = torch.randn(B, T, case["kv_heads"], D, generator=g, device="cuda").to(dt)
    elif case["op"] == "select":
        G, n, V = case["groups"], case["beams"], case["V"]
        s["logits"] = (torch.randn(G, n, V, generator=g, device="cuda") * 3).to(dt)
        s["scores"] = -torch.rand(G, n, generator=g, device="cuda") * 5
        s["finished"] = torch.rand(G, n, generator=g, device="cuda") < (0.25 if case["finished"] else -1.0)
        s["eos"] = V // 2
    else:
        B = case["groups"] * case["beams"]
        s["caches"], s["slots"] = [], []
        for _ in range(case["layers"]):
            if case["e4m3"]:
                c = _cache(case, B, g)
                s["caches"] += [c[k] for k in CACHE]
                s["slots"] += [BLOCK, BLOCK, BLOCK, BLOCK, 0, 0]
            else:
                shape = (B, case["kv_heads"], blocks_of(case["length"]) * BLOCK, case["D"])
                s["caches"] += [torch.randn(shape, generator=g, device="cuda", dtype=dt) for _ in range(2)]
                s["slots"] += [1, 1]
        s["parents"] = torch.tensor(parents_of(case), device="cuda")
        s["lengths"] = torch.tensor([case["length"]], device="cuda")
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        import flash_gemv

        if op == "attention":
            return flash_gemv.cats_kv8_attention(s["q"], s["start"], s["count"], *(s[k] for k in CACHE), s["scale"], s["case"]["window"])
        if op == "append":
            flash_gemv.cats_kv8_append(s["k"], s["v"], s["start"], s["count"], *(s[k] for k in CACHE))
            return {k: s[k] for k in CACHE}
        if op == "select":
            return flash_gemv.cats_beam_select(s["logits"], s["scores"], s["finished"], s["eos"])
        flash_gemv.cats_cache_reorder(s["caches"], s["slots"], s["parents"], s["lengths"])
        return s["caches"]
    return {"attention": _attention, "append": _append, "select": _select, "reorder": _reorder}[op](s)


def _attention(s):
    """softmax(scale q . k) v over the tokens up to each query, at most `window` of them; rows behind a sequence's last query are zeros."""
    q, start, count, w = s["q"], s["start"], s["count"], s["case"]["window"]
    B, T, heads, D = q.shape
    kv, n = s["k8"].shape[1], s["k8"].shape[2]
    k = (s["k8"].float() * s["k_scale"][..., None, None]).view(B, kv, n * BLOCK, D)
    v = (s["v8"].float() * s["v_scale"][..., None, None]).transpose(3, 4).reshape(B, kv, n * BLOCK, D)
    row = torch.arange(B, device=q.device)[:, None]
    end = start + count
    at = (end - 1)[:, None] // BLOCK * BLOCK + torch.arange(BLOCK, device=q.device)  # the tokens of each row's last block
    k[row, :, at], v[row, :, at] = s["k_tail"].float().transpose(1, 2), s["v_tail"].float().permute(0, 3, 1, 2)
    keys = int(s["case"]["length"])
    k, v = k[:, :, :keys], v[:, :, :keys]
    qs = q.float().view(B, T, kv, heads // kv, D).permute(0, 2, 3, 1, 4).reshape(B, kv, -1, D)  # (B, kv, group * T, D)
    score = torch.matmul(qs, k.transpose(2, 3)) * s["scale"]
    i, j = start[:, None, None] + torch.arange(T, device=q.device)[:, None], torch.arange(keys, device=q.device)
    seen = j <= i
    if w:
        seen = seen & (j > i - w)
    score = score.view(B, kv, -1, T, keys).masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(e.view(B, kv, -1, keys), v).view(B, kv, -1, T, D) / e.sum(-1)[..., None]
    o = o.permute(0, 3, 1, 2, 4).reshape(B, T, heads, D)
    return o.masked_fill((torch.arange(T, device=q.device) >= count[:, None])[:, :, None, None], 0).to(q.dtype)


def _quantised(x):
    """x (..., 64, D) -> e4m3 numbers and the smallest power of two that brings the block within 448."""
    m, e = torch.frexp(x.abs().amax((-2, -1)))  # m in [1/2, 1): up to 448 = 0.875 * 2^9
    scale = torch.where(m > 0, torch.ldexp(torch.ones_like(m), e - 9 + (m > 0.875)), torch.ones_like(m))
    return (x / scale[..., None, None]).to(torch.float8_e4m3fn), scale


def _append(s):
    k, v, start = s["k"].float(), s["v"].float(), s["start"]
    B, T, kv, D = k.shape
    dev = k.device
    # each row's tokens from the start of the block that `start` lies in: what its tail holds, then the new ones
    n = (T + BLOCK - 1) // BLOCK + (1 if T == 1 or T % BLOCK == 0 else 0)
    row = torch.arange(B, device=dev)[:, None]
    inside = start % BLOCK
    buf_k, buf_v = torch.zeros(2, B, n * BLOCK, kv, D, device=dev).unbind(0)
    buf_k[:, :BLOCK], buf_v[:, :BLOCK] = s["k_tail"].float().transpose(1, 2), s["v_tail"].float().permute(0, 3, 1, 2)
    at = inside[:, None] + torch.arange(T, device=dev)
    buf_k[row, at], buf_v[row, at] = k, v
    buf_k, buf_v = (b.view(B, n, BLOCK, kv, D).permute(0, 3, 1, 2, 4) for b in (buf_k, buf_v))  # (B, kv, n, 64, D)
    k8, ks = _quantised(buf_k)
    v8, vs = _quantised(buf_v)
    end = inside + s["count"]
    block = torch.arange(n, device=dev)
    whole = ((block + 1) * BLOCK <= end[:, None])  # (B, n)
    to = (start // BLOCK)[:, None] + block
    r, b = torch.nonzero(whole, as_tuple=True)
    slot = to[r, b]
    bits = torch.uint8
    s["k8"].view(bits)[r, :, slot] = k8.view(bits)[r, :, b]
    s["v8"].view(bits)[r, :, slot] = v8.transpose(3, 4).contiguous().view(bits)[r, :, b]
    s["k_scale"][r, :, slot], s["v_scale"][r, :, slot] = ks[r, :, b], vs[r, :, b]
    # the last block's tokens, as they were given
    last = (end - 1) // BLOCK
    live = (torch.arange(BLOCK, device=dev) < (end - last * BLOCK)[:, None])[:, None, :, None]
    tail_k, tail_v = buf_k[row[:, 0], :, last], buf_v[row[:, 0], :, last]  # (B, kv, 64, D)
    s["k_tail"].copy_(torch.where(live, tail_k, s["k_tail"].float()))
    s["v_tail"].copy_(torch.where(live.transpose(2, 3), tail_v.transpose(2, 3), s["v_tail"].float()))
    return {key: s[key] for key in CACHE}


def _select(s):
    x, scores, finished, eos = s["logits"].double(), s["scores"].double(), s["finished"], s["eos"]
    G, n, V = x.shape
    top = x.amax(-1, keepdim=True)
    total = scores[..., None] + (x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    ended = torch.full_like(total, -math.inf)
    ended[..., eos] = scores
    total = torch.where(finished[..., None], ended, total).view(G, n * V)
    best, at = torch.sort(total, dim=-1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    parents, tokens = at // V, at % V
    return best.float(), parents, tokens, finished.gather(1, parents) | (tokens == eos)


def _reorder(s):
    G, n = s["parents"].shape
    rows = (s["parents"] + torch.arange(G, device=s["parents"].device)[:, None] * n).view(-1)
    for c, slots in zip(s["caches"], s["slots"]):
        bits = c.view(torch.uint8) if c.element_size() == 1 else c
        moved = bits[rows]
        if slots:
            live = torch.arange(c.shape[2], device=c.device) * slots < s["lengths"]
            moved = torch.where(live.view(-1, *[1] * (c.dim() - 3)), moved, bits)
        bits.copy_(moved)
    return s["caches"]


# ---- the operators' definitions in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "select": _exact_select, "reorder": _exact_reorder}[case["op"]](s)


def _exact_attention(s):
    q, w = s["q"].double(), s["case"]["window"]
    B, T, heads, D = q.shape
    group = heads // s["k8"].shape[1]
    out = torch.zeros_like(q)
    for b in range(B):
        a, n = int(s["start"][b]), int(s["count"][b])
        end = a + n
        full = (end - 1) // BLOCK
        for h in range(heads):
            c = h // group
            k = torch.cat([(s["k8"][b, c, :full].double() * s["k_scale"][b, c, :full, None, None].double()).reshape(-1, D),
                           s["k_tail"][b, c, : end - full * BLOCK].double()])
            v = torch.cat([(s["v8"][b, c, :full].double() * s["v_scale"][b, c, :full, None, None].double()).transpose(1, 2).reshape(-1, D),
                           s["v_tail"][b, c, :, : end - full * BLOCK].double().t()])
            x = q[b, :n, h] @ k.t() * s["scale"]
            at = torch.arange(a, end, device=q.device)[:, None] - torch.arange(end, device=q.device)  # how far back a key lies
            x[(at < 0) | (at >= w if w else at < 0)] = -math.inf
            out[b, :n, h] = torch.softmax(x, -1) @ v
    return out


def _exact_append(s):
    out = {key: s[key].double() for key in CACHE}
    for b in range(s["k"].shape[0]):
        a, n = int(s["start"][b]), int(s["count"][b])
        first, end = a // BLOCK, a + n
        old = a - first * BLOCK
        k = torch.cat([s["k_tail"][b, :, :old], s["k"][b, :n].transpose(0, 1)], 1).double()  # (kv, tokens, D)
        v = torch.cat([s["v_tail"][b, :, :, :old].transpose(1, 2), s["v"][b, :n].transpose(0, 1)], 1).double()
        whole = k.shape[1] // BLOCK
        for x, key, turn in ((k, "k", False), (v, "v", True)):
            blocks = x[:, : whole * BLOCK].reshape(x.shape[0], whole, BLOCK, x.shape[2])
            scale = torch.exp2(torch.ceil(torch.log2(blocks.abs().amax((2, 3)) / 448)))
            y = blocks / scale[..., None, None]
            step = torch.exp2(torch.clamp(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20))), min=-6) - 3)  # between neighbours of e4m3
            y = torch.round(y / step) * step
            out[key + "8"][b, :, first:first + whole] = y.transpose(2, 3) if turn else y
            out[key + "_scale"][b, :, first:first + whole] = scale
        last = (k.shape[1] - 1) // BLOCK
        live = k.shape[1] - last * BLOCK
        out["k_tail"][b, :, :live], out["v_tail"][b, :, :, :live] = k[:, last * BLOCK:], v[:, last * BLOCK:].transpose(1, 2)
    return out


def _exact_select(s):
    G, n, V = s["logits"].shape
    lp = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None]
    found = [[], [], [], []]
    for g in range(G):
        best = []
        for b in range(n):
            if s["finished"][g, b]:
                best.append((-float(s["scores"][g, b]), b, s["eos"]))
            else:
                v, i = torch.topk(lp[g, b], min(V, n))
                best += [(-x, b, t) for x, t in zip(v.tolist(), i.tolist())]
        best = sorted(best)[:n]
        for to, x in zip(found, ([-x for x, _, _ in best], [b for _, b, _ in best], [t for _, _, t in best],
                                 [bool(s["finished"][g, b]) or t == s["eos"] for _, b, t in best])):
            to.append(x)
    dev = s["logits"].device
    return (torch.tensor(found[0], dtype=torch.float64, device=dev), torch.tensor(found[1], device=dev), torch.tensor(found[2], device=dev),
            torch.tensor(found[3], device=dev))


def _exact_reorder(s):
    out = [c.double() for c in s["caches"]]
    n = s["parents"].shape[1]
    for c, o, slots in zip(s["caches"], out, s["slots"]):
        live = min(c.shape[2], -(-int(s["lengths"]) // slots)) if slots else c.shape[2]
        for g, parents in enumerate(s["parents"].tolist()):
            for j, p in enumerate(parents):
                o[g * n + j, :, :live] = c[g * n + p, :, :live].double()
    return out
