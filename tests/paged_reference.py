"""Plain implementations, in 64 bits on the CPU, of the cache of pages and of attention over packed sequences: a sequence and a head at a time."""
import math

import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # of a rounding to the type, relative to the value
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # and of the smallest numbers, absolute


def offsets_of(rows, lead=0):
    """rows: (start, count) of each sequence; lead: tokens before the first."""
    at = [lead]
    for _, n in rows:
        at.append(at[-1] + n)
    return at


def new_pool(rows, page, kv, D, dtype, seed=0, spare=3, room=2, group=1, shared=0):
    """(k_pages, v_pages, table) with room for the rows' tokens: pages in no order, every number NaN, entries of the table that nobody needs anything.
    Whole pages of the first `shared` tokens are the same for the sequences of a group."""
    g = torch.Generator().manual_seed(seed)
    used = [-(-(a + n) // page) for a, n in rows]
    common = shared // page
    fresh = [u - min(u, common, used[b - b % group]) * (b % group != 0) for b, u in enumerate(used)]
    pages = sum(fresh) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.randint(-2 ** 31, 2 ** 31 - 1, (len(rows), max(1, *used) + room), generator=g, dtype=torch.int64).to(torch.int32)
    at = 0
    for b, u in enumerate(used):
        old = u - fresh[b]
        table[b, :old] = table[b - b % group, :old]
        table[b, old:u] = order[at:at + fresh[b]]
        at += fresh[b]
    k, v = (torch.full((pages, kv, page, D), math.nan, dtype=dtype) for _ in range(2))
    return k, v, table


def fill(pool, rows, g, scale=1.0):
    """Random tokens in all places that the rows have, up to the end of their new ones.  Shared pages are written again by each of a group."""
    k, v, table = pool
    _, kv, page, D = k.shape
    for b, (a, n) in enumerate(rows):
        for i in range(-(-(a + n) // page)):
            m = min(page, a + n - i * page)
            for x in (k, v):
                x[int(table[b, i]), :, :m] = (torch.randn(kv, m, D, generator=g) * scale).to(x.dtype)


def tokens(pool, b, n):
    """The first n tokens of sequence b: k, v (n, kv, D)."""
    k, v, table = pool
    page = k.shape[2]
    ids = table[b, : -(-n // page)].long()
    return tuple(x[ids].transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:n] for x in (k, v))


def rotate(x, cos, sin):
    """x (n, heads, D), tables (n, R) -> the rotation in double, and how far a kernel's may be from it: half a step of the type, and three roundings in 32
    bits (one product, the second product with the sum, which rounds once) relative to the two products."""
    R = cos.shape[1]
    y = x.double()
    a, c, s = y[..., :R], cos.double()[:, None], sin.double()[:, None]
    turned = torch.cat([-a[..., R // 2:], a[..., : R // 2]], -1)
    out, size = y.clone(), torch.zeros_like(y)
    out[..., :R] = a * c + turned * s
    size[..., :R] = (a * c).abs() + (turned * s).abs()
    return out, HALF[x.dtype] * out.abs() * (size > 0) + 3 * 2.0 ** -24 * size + LEAST[x.dtype] * (size > 0)


def append(q, k, v, rows, lead, cos, sin, pool):
    """((q', bound), (k_pages, bound), (v_pages, bound)) in double.  cos None: nothing is rotated."""
    kp, vp, table = pool
    pages, _, page, _ = kp.shape
    want_q = torch.zeros(q.shape, dtype=torch.float64) if q is not None else None
    want_k, want_v = kp.double(), vp.double()
    bound_q = torch.zeros_like(want_q) if q is not None else None
    bound_k = torch.zeros_like(want_k)
    t = lead
    for b, (start, n) in enumerate(rows):
        for i in range(n):
            p = start + i
            ok = 0 <= p < table.shape[1] * page and (cos is None or p < cos.shape[0])
            at = int(table[b, p // page]) if ok else -1
            if not 0 <= at < pages:
                if q is not None:
                    want_q[t] = math.nan
                t += 1
                continue
            turn = (lambda x: rotate(x[t:t + 1], cos[p:p + 1], sin[p:p + 1])) if cos is not None else (lambda x: (x[t:t + 1].double(), torch.zeros_like(x[t:t + 1].double())))
            if q is not None:
                (want_q[t],), (bound_q[t],) = turn(q)
            (want_k[at, :, p % page],), (bound_k[at, :, p % page],) = turn(k)
            want_v[at, :, p % page] = v[t].double()
            t += 1
    return (want_q, bound_q), (want_k, bound_k), (want_v, torch.zeros_like(want_v))


def attend(q, k, v, last, scale, window):
    """One sequence: q (n, heads, D) over k, v (m, kv, D), query i sees the keys up to last + i.  (out, bound) in double: the bound is half a step of the output; half
    a step of each weight, which is held in q's type (in relation to the weighted magnitudes A of the values); and what an error of the scores makes of the
    weights, above and below the line: a sum of D products in 32 bits, their scaling, the exponential (two units) and the sums over the keys, all
    relative to A."""
    n, heads, D = q.shape
    kv, m = k.shape[1], k.shape[0]
    u = HALF[q.dtype]
    out, bound = torch.zeros(n, heads, D, dtype=torch.float64), torch.zeros(n, heads, D, dtype=torch.float64)
    if n == 0 or m == 0:
        return out, bound
    at = last + torch.arange(n)[:, None]
    key = torch.arange(m)[None]
    seen = (key <= at) & ((key > at - window) if window else True)
    some = seen.any(1)
    for h in range(heads):
        c = h // (heads // kv)
        kk, vv, x = k[:, c].double(), v[:, c].double(), q[:, h].double()
        bad_k, bad_v, bad_q = ~torch.isfinite(kk).all(1), ~torch.isfinite(vv), ~torch.isfinite(x).all(1)
        kk, vv, x = (torch.nan_to_num(z, posinf=0.0, neginf=0.0) for z in (kk, vv, x))
        w = torch.softmax((x @ kk.t() * scale).masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
        o, A = w @ vv, w @ vv.abs()
        products = (x.abs() @ kk.abs().t()).masked_fill(~seen, 0).amax(1, keepdim=True) * scale
        delta = ((D + 8) * products + 8 + m) * 2.0 ** -24
        o = torch.where((seen.double() @ bad_v.double()) > 0, math.nan, o)  # not finite: an infinity or NaN
        o[((seen & bad_k).any(1) | bad_q) & some] = math.nan
        out[:, h] = o
        bound[:, h] = u * o.abs() + u * A + 2 * delta * A + LEAST[q.dtype]
    return out, bound


def paged_attention(q, rows, lead, pool, scale, window=0):
    """Every sequence over its own row of the table (whatever is shared is the same there).  A token whose page is none is as a key that is not finite."""
    kp, vp, table = pool
    pages, _, page, _ = kp.shape
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    t = lead
    for b, (start, n) in enumerate(rows):
        if n:
            ids = table[b, : -(-(start + n) // page)].long()
            if start < 0 or start + n > table.shape[1] * page:
                out[t:t + n] = math.nan
            else:
                none = (ids < 0) | (ids >= pages)
                k, v = tokens((kp, vp, torch.where(none, 0, ids)[None]), 0, start + n)
                k[none.repeat_interleave(page)[: start + n]] = math.nan
                out[t:t + n], bound[t:t + n] = attend(q[t:t + n], k, v, start, scale, window)
        t += n
    return out, bound


def prompt_attention(q, k, v, at, k_at, scale, window=0):
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for s in range(len(at) - 1):
        a, e, ka, ke = at[s], at[s + 1], k_at[s], k_at[s + 1]
        out[a:e], bound[a:e] = attend(q[a:e], k[ka:ke], v[ka:ke], (ke - ka) - (e - a), scale, window)
    return out, bound


def within(got, want, bound):
    """Within the bound, and not finite where it is to be so."""
    got = got.cpu().double()
    if not torch.equal(~torch.isfinite(got), want.isnan()):
        return False
    return bool((((got - want).abs() <= bound) | want.isnan()).all())
