"""What the operators of a paged cache and of packed prompts are measured on: the calls that a server makes around attention.

A case is one call of ``flash_gemv`` on tensors that such a program keeps.  ``listed()`` names twelve of them, ``draw()`` gives others of
the same ranges.  Fields: ``op`` (below), ``dtype`` of the model, and the sizes of the operator.

  append     flash_gemv.cats_paged_append      rotates new queries and keys at their positions and stores keys and values in pages
  attention  flash_gemv.cats_paged_attention   new tokens over the pages of their sequences; ``group`` sequences share their first ``shared`` tokens
  prompt     flash_gemv.cats_prompt_attention  whole prompts, causal, without a cache

Tokens are packed: sequence s has the tokens ``offsets[s]`` to ``offsets[s + 1] - 1`` of (N, heads, D), at the positions ``start[s]`` onwards.  Pages are
(pages, kv_heads, page, D) in the model's type, and token p of sequence s lies in page ``table[s, p // page]``, place ``p % page``.
"""
import math

import torch

own = False  # False: the operators in elementary torch operations; True: the framework's kernels

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    def append(name, B, T, heads, kv_heads, D, page, length, dtype, rot, ragged=False):
        return {"name": name, "op": "append", "B": B, "T": T, "heads": heads, "kv_heads": kv_heads, "D": D, "page": page, "length": length, "dtype": dtype,
                "rot": rot, "ragged": ragged}

    def attention(name, B, T, heads, kv_heads, D, page, length, dtype, window=0, ragged=False, group=1, shared=0):
        return {"name": name, "op": "attention", "B": B, "T": T, "heads": heads, "kv_heads": kv_heads, "D": D, "page": page, "length": length, "dtype": dtype,
                "window": window, "ragged": ragged, "group": group, "shared": shared}

    def prompt(name, B, T, heads, kv_heads, D, dtype, window=0, ragged=False):
        return {"name": name, "op": "prompt", "B": B, "T": T, "heads": heads, "kv_heads": kv_heads, "D": D, "dtype": dtype, "window": window, "ragged": ragged}

    return [
        # a token of a single stream of a 7B model: a launch is all there is
        append("append - 1 token", 1, 1, 32, 32, 128, 16, 100, "fp16", 128),
        # a decode step of a server's batch, grouped heads
        append("append - 64 tokens", 64, 1, 32, 8, 128, 64, 4000, "bf16", 128),
        # prompts of all lengths enter the cache, half of each head rotated
        append("append - 8 prompts to 2048", 8, 2048, 32, 32, 128, 64, 2048, "fp16", 64, ragged=True),
        # single-stream decoding, early in the answer: launches and dependent trips
        attention("step - 1 row - 100 tokens", 1, 1, 32, 32, 128, 16, 100, "fp16"),
        # a server's batch of sequences of all lengths, small pages
        attention("step - 32 rows - to 4096", 32, 1, 32, 8, 128, 16, 4096, "bf16", ragged=True),
        # beam search: the eight beams of a prompt share it
        attention("step - 4 x 8 beams on 2000", 32, 1, 32, 32, 128, 64, 2120, "fp16", ragged=True, group=8, shared=2000),
        # many conversations behind one long system prompt
        attention("step - 64 rows share 16384", 64, 1, 32, 8, 128, 64, 16384 + 500, "bf16", ragged=True, group=64, shared=16384),
        # the next piece of two long prompts that are taken in pieces
        attention("piece of 512 behind 7680", 2, 512, 32, 8, 128, 64, 8192, "bf16", ragged=True),
        # small prompts of a small model, a window, an odd number of heads a group
        prompt("prompts - 24 to 300 - window", 24, 300, 14, 2, 64, "bf16", window=100, ragged=True),
        # a prompt of a 7B model
        prompt("prompt - 2048 tokens", 1, 2048, 32, 32, 128, "fp16"),
        # a server's batch of prompts, packed
        prompt("prompts - 16 to 1500", 16, 1500, 32, 8, 128, "bf16", ragged=True),
        # a long document
        prompt("prompt - 8192 tokens", 1, 8192, 32, 8, 128, "bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))

    case = {"op": rng.choice(["append", "attention", "attention", "attention", "prompt", "prompt"]), "D": rng.choice([32, 64, 128, 128, 256]),
            "kv_heads": rng.choice([1, 2, 4, 8, 8, 16, 32]), "dtype": rng.choice(["fp16", "bf16"]), "ragged": rng.random() < 0.7}
    group_heads = rng.choice([1, 1, 2, 3, 4, 7, 8])
    case["heads"] = case["kv_heads"] * group_heads
    width = case["kv_heads"] * case["D"]
    if case["op"] == "prompt":
        B, T = log(1, 32), log(17, 8192)
        while B * T * T * case["heads"] > 1 << 31 or B * T * case["heads"] * case["D"] > 1 << 25:
            B, T = max(1, B // 2), max(1, T * 2 // 3)
        return {**case, "B": B, "T": T, "window": rng.choice([0, 0, log(16, 4096)])}
    case["page"] = rng.choice([16, 16, 32, 64, 64, 128, 256])
    if case["op"] == "append":
        T, B = rng.choice([1, log(2, 4096)]), log(1, 64)
        while B * T * (case["heads"] + 2 * case["kv_heads"]) * case["D"] > 1 << 26:
            T = max(1, T // 2)
        return {**case, "B": B, "T": T, "length": T + rng.choice([0, log(1, 3000)]), "rot": rng.choice([case["D"], case["D"], max(16, case["D"] // 4)])}
    case.update(window=rng.choice([0, 0, 0, log(16, 8192)]), group=1, shared=0)
    kind = rng.random()
    if kind < 0.4:  # a step, or a few drafted tokens
        T, B, length = rng.choice([1, 1, 1, rng.randint(2, 16)]), log(1, 64), log(16, 65536)
    elif kind < 0.75:  # sequences that share a prefix
        T, case["window"] = rng.choice([1, 1, 1, rng.randint(2, 5)]), 0
        case["group"], case["shared"] = rng.randint(2, 32), log(100, 32768)
        B, length = case["group"] * rng.randint(1, 4), case["shared"] + T + log(1, 2000)
    else:  # a piece of a prompt
        T, B = log(17, 2048), log(1, 4)
        length = T + rng.choice([0, log(1, 8192)])
    while B * T * length * case["heads"] > 1 << 30 or B * length * width > 1 << 29:
        if T > 32:
            T, length = T // 2, max(T // 2, length * 3 // 4)
        else:
            case["shared"] //= 2
            length = case["shared"] + T + max(1, (length - T) // 2)
    return {**case, "B": B, "T": T, "length": max(length, case["shared"] + T)}


# ---- sizes that follow from a case --------------------------------------------------------------------------------------------------

def rows_of(case):
    """(start, count) of each sequence: how many tokens it has already, and how many it gets."""
    B, T = case["B"], case["T"]
    if case["op"] == "prompt":
        return [(0, max(1, T - b * T // B) if case["ragged"] else T) for b in range(B)]
    length = case["length"]
    shared = case.get("shared", 0)
    rows = []
    for b in range(B):
        n = max(1, T - b * T // (2 * B)) if case["ragged"] else T
        least = shared + n
        rows.append((max(least, length - b * (length - shared) // (2 * B)) - n if case["ragged"] else length - n, n))
    return rows


def shared_of(case):
    """Tokens of whole pages among those that a group shares."""
    return case["shared"] // case["page"] * case["page"] if case["op"] == "attention" else 0


def seen_of(case, start, n):
    """Query-key pairs of one head of a sequence, and its first key that is seen."""
    w = case["window"] or start + n
    return sum(min(start + i + 1, w) for i in range(n)), max(0, start + 1 - w)


def work(case):
    heads, kv, D = case["heads"], case["kv_heads"], case["D"]
    rows = rows_of(case)
    tokens = sum(n for _, n in rows)
    if case["op"] == "append":
        positions = len({p for a, n in rows for p in range(a, a + n)})
        return {"bytes": 2 * 2 * tokens * (heads + 2 * kv) * D + 8 * positions * case["rot"], "flops": 3 * tokens * (heads + kv) * case["rot"]}
    pairs = keys = 0
    shared = shared_of(case)
    for b, (start, n) in enumerate(rows):
        more, first = seen_of(case, start, n)
        pairs += more
        keys += start + n - first
        if shared and b % case["group"]:
            keys -= max(0, shared - first)
    return {"bytes": 2 * 2 * D * (keys * kv + tokens * heads), "flops": 4 * pairs * heads * D}


# ---- inputs --------------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    B, heads, kv, D = case["B"], case["heads"], case["kv_heads"], case["D"]
    rows = rows_of(case)
    N = sum(n for _, n in rows)
    channel = torch.exp(torch.randn(kv, 1, D, generator=g, device="cuda") * 0.4)  # keys have channels of their own size
    s = {"case": case, "scale": 1 / math.sqrt(D)}
    ends = [0]
    for _, n in rows:
        ends.append(ends[-1] + n)
    s["offsets"] = torch.tensor(ends, device="cuda")
    s["q"] = (torch.randn(N, heads, D, generator=g, device="cuda") * 1.5).to(dt)
    if case["op"] != "attention":
        s["k"] = (torch.randn(N, kv, D, generator=g, device="cuda") * channel[:, 0]).to(dt)
        s["v"] = torch.randn(N, kv, D, generator=g, device="cuda").to(dt)
    if case["op"] == "prompt":
        return s
    s["start"] = torch.tensor([a for a, _ in rows], device="cuda")
    # the table: pages in no order, room for a quarter more tokens, -1 where a sequence has no page yet
    P, longest = case["page"], max(a + n for a, n in rows)
    width = -(-(longest + longest // 4 + 1) // P)
    common = shared_of(case) // P
    used = [-(-(a + n) // P) for a, n in rows]
    fresh = [u - (common if b % case.get("group", 1) else 0) for b, u in enumerate(used)]
    pages = sum(fresh) + 8
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        first = u - fresh[b]
        if first:
            table[b, :first] = table[b - b % case["group"], :first]
        table[b, first:u] = order[at:at + fresh[b]]
        at += fresh[b]
    s["table"] = table.cuda()
    s["shared"] = torch.tensor([shared_of(case)], device="cuda") if case.get("group", 1) > 1 else None
    for name in ("k_pages", "v_pages"):
        t = torch.empty(pages, kv, P, D, dtype=dt, device="cuda")
        for i in range(0, pages, 1024):
            x = torch.randn(t[i:i + 1024].shape, generator=g, device="cuda")
            t[i:i + 1024] = x * channel if name == "k_pages" else x
        s[name] = t
    if case["op"] == "append":
        R = case["rot"]
        angle = torch.arange(longest + 1, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
        angle = torch.cat([angle, angle], 1)
        s["cos"], s["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        import flash_gemv

        if case["op"] == "append":
            q = flash_gemv.cats_paged_append(s["q"], s["k"], s["v"], s["offsets"], s["start"], s["cos"], s["sin"], s["k_pages"], s["v_pages"], s["table"])
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if case["op"] == "attention":
            return flash_gemv.cats_paged_attention(s["q"], s["offsets"], s["start"], s["k_pages"], s["v_pages"], s["table"], s["scale"], case["window"],
                                                   case["group"], s["shared"])
        return flash_gemv.cats_prompt_attention(s["q"], s["k"], s["v"], s["offsets"], s["scale"], case["window"])
    return {"append": _append, "attention": _paged, "prompt": _prompt}[case["op"]](s)


def _places(s):
    """Sequence and index in it of each packed token."""
    token = torch.arange(s["q"].shape[0], device=s["q"].device)
    row = torch.searchsorted(s["offsets"], token, right=True) - 1
    return row, token - s["offsets"][row]


def _append(s):
    row, index = _places(s)
    position = s["start"][row] + index
    R = s["cos"].shape[1]
    cos, sin = s["cos"][position][:, None], s["sin"][position][:, None]

    def rotated(x):
        x = x.float()
        a = x[..., :R]
        turned = a * cos + torch.cat([-a[..., R // 2:], a[..., :R // 2]], -1) * sin
        return torch.cat([turned, x[..., R:]], -1)

    P = s["k_pages"].shape[2]
    page = s["table"][row, position // P].long()
    s["k_pages"][page, :, position % P] = rotated(s["k"]).to(s["k"].dtype)
    s["v_pages"][page, :, position % P] = s["v"]
    return {"q": rotated(s["q"]).to(s["q"].dtype), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attend(s, k, v, start, T):
    """softmax(scale q . k) v of each sequence's tokens over k, v (B, kv, keys, D) in 32 bits, up to each token's own position."""
    q, w = s["q"], s["case"]["window"]
    N, heads, D = q.shape
    B, kv, keys, _ = k.shape
    row, index = _places(s)
    qs = torch.zeros(B, T, kv, heads // kv, D, device=q.device)
    qs[row, index] = q.float().view(N, kv, heads // kv, D)
    qs = qs.permute(0, 2, 3, 1, 4).reshape(B, kv, -1, D)  # (B, kv, group * T, D)
    score = torch.matmul(qs, k.transpose(2, 3)) * s["scale"]
    i, j = start[:, None, None] + torch.arange(T, device=q.device)[:, None], torch.arange(keys, device=q.device)
    seen = j <= i
    if w:
        seen = seen & (j > i - w)
    score = score.view(B, kv, -1, T, keys).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = score.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    o = torch.matmul(e.view(B, kv, -1, keys), v).view(B, kv, -1, T, D) / e.sum(-1)[..., None]
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, heads, D)[row, index].to(q.dtype)


def _paged(s):
    case = s["case"]
    P = case["page"]
    table = s["table"][:, :-(-case["length"] // P)].long().clamp(min=0)
    B, n = table.shape

    def rows(pages):
        return pages[table].float().permute(0, 2, 1, 3, 4).reshape(B, pages.shape[1], n * P, pages.shape[3])

    v = rows(s["v_pages"])
    end = s["start"] + s["offsets"].diff()
    v.masked_fill_((torch.arange(n * P, device=v.device) >= end[:, None])[:, None, :, None], 0)  # nobody's yet: their weight is 0
    return _attend(s, rows(s["k_pages"]), v, s["start"], case["T"])


def _prompt(s):
    case = s["case"]
    row, index = _places(s)
    B, T = case["B"], case["T"]

    def rows(x):
        out = torch.zeros(B, T, x.shape[1], x.shape[2], device=x.device)
        out[row, index] = x.float()
        return out.transpose(1, 2).contiguous()

    return _attend(s, rows(s["k"]), rows(s["v"]), torch.zeros(B, dtype=torch.int64, device=row.device), T)


# ---- in 64 bits, a sequence and a cached head at a time ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    rows = rows_of(case)
    dev = s["q"].device
    if case["op"] == "append":
        P, half = case["page"], case["rot"] // 2
        out = {"q": s["q"].double(), "k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double()}
        turn = torch.complex(s["cos"][:, :half].double(), s["sin"][:, :half].double())  # a rotation is a product of complex numbers
        at = 0
        for b, (start, n) in enumerate(rows):
            place = torch.arange(start, start + n, device=dev)
            page = s["table"][b, place // P].long()
            for name, x in (("q", s["q"]), ("k", s["k"])):
                x = x[at:at + n].double()
                z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn[place][:, None]
                x = torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)
                if name == "q":
                    out["q"][at:at + n] = x
                else:
                    out["k_pages"][page, :, place % P] = x
            out["v_pages"][page, :, place % P] = s["v"][at:at + n].double()
            at += n
        return out
    heads, kv, D = case["heads"], case["kv_heads"], case["D"]
    group = heads // kv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=dev)
    at = 0
    for b, (start, n) in enumerate(rows):
        for c in range(kv):
            if case["op"] == "prompt":
                k, v = s["k"][at:at + n, c].double(), s["v"][at:at + n, c].double()
            else:
                P = case["page"]
                page = s["table"][b, :-(-(start + n) // P)].long()
                k, v = (s[name][page, c].double().reshape(-1, D)[:start + n] for name in ("k_pages", "v_pages"))
            for i in range(0, n, 1024):
                m = min(1024, n - i)
                q = s["q"][at + i:at + i + m, c * group:(c + 1) * group].double().transpose(0, 1)  # (group, m, D)
                last = start + i + torch.arange(m, device=dev)
                key = torch.arange(start + n, device=dev)
                hidden = key[None] > last[:, None]
                if case["window"]:
                    hidden |= key[None] <= last[:, None] - case["window"]
                score = (q.reshape(-1, D) @ k.t() * s["scale"]).view(group, m, -1).masked_fill_(hidden, -math.inf)
                o = torch.softmax(score, -1).view(group * m, -1) @ v
                out[at + i:at + i + m, c * group:(c + 1) * group] = o.view(group, m, D).transpose(0, 1)
        at += n
    return out
