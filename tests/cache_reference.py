"""Plain implementations, in 64 bits on the CPU, of the cache in 8 bits and of beam search: a token, a row and a beam at a time."""
import math

import torch

BLOCK = 64
FIELDS = ("k8", "v8", "k_scale", "v_scale", "k_tail", "v_tail")
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # of a rounding to the type, relative to the value


def new_cache(B, heads, blocks, D, dtype, fill=None, device="cpu"):
    """A cache whose every byte is something else before it is written: NaN by default, or zeros."""
    bad = math.nan if fill is None else fill
    shapes = {"k8": (blocks, BLOCK, D), "v8": (blocks, D, BLOCK), "k_scale": (blocks,), "v_scale": (blocks,), "k_tail": (BLOCK, D), "v_tail": (D, BLOCK)}
    types = {"k8": torch.float8_e4m3fn, "v8": torch.float8_e4m3fn, "k_scale": torch.float32, "v_scale": torch.float32, "k_tail": dtype, "v_tail": dtype}
    return {f: torch.full((B, heads, *shapes[f]), bad, dtype=torch.float32).to(types[f]).to(device) for f in FIELDS}


def to(cache, device):
    return {f: t.to(device) for f, t in cache.items()}


def same(a, b):
    """Equal bit for bit, but for the sign and payload of a NaN."""
    a, b = a.cpu().float(), b.cpu().float()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def quantise(x):
    """x (64, D) in double -> (numbers in double, scale)."""
    finite = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs()
    amax = float(finite.max())
    scale = 1.0
    if amax > 0:
        e = -60
        while amax > 448 * 2.0 ** e:
            e += 1
        scale = 2.0 ** e
    y = torch.where(torch.isfinite(x), x / scale, torch.full_like(x, math.nan))
    m, e = torch.frexp(y.abs())  # m in [1/2, 1): four significant bits, and none below 2^-9
    step = torch.ldexp(torch.ones_like(y), torch.clamp(e, min=-5) - 4)
    y = torch.where(y.isnan(), y, torch.round(y / step) * step)
    return y, scale


def append(cache, k, v, start, count):
    """cache (on the CPU) after k, v (B, T, heads, D) have been stored; start and count lists of ints, count None: all."""
    cache = {f: t.clone() for f, t in cache.items()}
    B, T, heads, D = k.shape
    blocks = cache["k8"].shape[2]
    for b in range(B):
        n = T if count is None else min(max(count[b], 0), T)
        if n == 0 or start[b] < 0 or start[b] + n > blocks * BLOCK:
            continue
        for h in range(heads):
            at = start[b] // BLOCK * BLOCK
            ks = {at + i: cache["k_tail"][b, h, i].double() for i in range(start[b] - at)}
            vs = {at + i: cache["v_tail"][b, h, :, i].double() for i in range(start[b] - at)}
            for i in range(n):
                ks[start[b] + i], vs[start[b] + i] = k[b, i, h].double(), v[b, i, h].double()
            end = start[b] + n
            for blk in range(at // BLOCK, end // BLOCK):
                for x, f, turn in ((ks, "k", False), (vs, "v", True)):
                    y, s = quantise(torch.stack([x[blk * BLOCK + i] for i in range(BLOCK)]))
                    cache[f + "8"][b, h, blk] = (y.t() if turn else y).float().to(torch.float8_e4m3fn)
                    cache[f + "_scale"][b, h, blk] = s
            last = (end - 1) // BLOCK * BLOCK
            for p in range(max(last, start[b]), end):
                cache["k_tail"][b, h, p - last] = ks[p].to(k.dtype)
                cache["v_tail"][b, h, :, p - last] = vs[p].to(v.dtype)
    return cache


def attention(cache, q, start, count, scale, window=0):
    """(out, bound) in double: what the queries of q (B, T, heads, D) see, and how far a kernel may be from it.

    The bound: half a step of the output; half a step of each weight, which is held in q's type (in relation to the weighted magnitudes A of the
    values); and what an error of the scores makes of the weights, above and below the line: a sum of D products in 32 bits, their scaling, the
    exponential (two units) and the sums over the keys, all relative to A."""
    B, T, heads, D = q.shape
    kv, blocks = cache["k8"].shape[1:3]
    out, bound = torch.zeros(B, T, heads, D, dtype=torch.float64), torch.zeros(B, T, heads, D, dtype=torch.float64)
    u = HALF[q.dtype]
    for b in range(B):
        n = T if count is None else min(max(count[b], 0), T)
        if n == 0:
            continue
        if start[b] < 0 or start[b] + n > blocks * BLOCK:
            out[b, :n] = math.nan
            continue
        end = start[b] + n
        full = (end - 1) // BLOCK
        for c in range(kv):
            k = torch.cat([(cache["k8"][b, c, :full].double() * cache["k_scale"][b, c, :full, None, None].double()).reshape(-1, D),
                           cache["k_tail"][b, c, : end - full * BLOCK].double()])
            v = torch.cat([(cache["v8"][b, c, :full].double() * cache["v_scale"][b, c, :full, None, None].double()).transpose(1, 2).reshape(-1, D),
                           cache["v_tail"][b, c, :, : end - full * BLOCK].double().t()])
            for i in range(n):
                p = start[b] + i
                lo = max(0, p - window + 1) if window else 0
                kk, vv = k[lo:p + 1], v[lo:p + 1]
                bad_k, bad_v = ~torch.isfinite(kk).all(), ~torch.isfinite(vv).all(0)
                kk, vv = torch.nan_to_num(kk, posinf=0.0, neginf=0.0), torch.nan_to_num(vv, posinf=0.0, neginf=0.0)
                for g in range(heads // kv):
                    x = q[b, i, c * (heads // kv) + g].double()
                    w = torch.softmax(kk @ x * scale, 0)
                    o = w @ vv
                    A = w @ vv.abs()
                    products = float((kk.abs() @ x.abs()).max()) * scale
                    delta = ((D + 8) * products + 8 + kk.shape[0]) * 2.0 ** -24
                    o[bad_v] = math.nan
                    if bad_k or not torch.isfinite(x).all():
                        o[:] = math.nan
                    out[b, i, c * (heads // kv) + g] = o
                    bound[b, i, c * (heads // kv) + g] = u * o.abs() + u * A + 2 * delta * A + 2.0 ** -25 * (q.dtype == torch.float16)
    return out, bound


def within(got, want, bound):
    got = got.cpu().double()
    if not torch.equal(got.isnan(), want.isnan()):
        return False
    near = (got - want).abs() <= bound
    return bool((near | want.isnan()).all())


def select(logits, scores, finished, eos, keep):
    """Per group lists of (score, parent, token, finished); every beam and word is a candidate."""
    G, n, V = logits.shape
    found = []
    for g in range(G):
        total = torch.full((n, V), -math.inf, dtype=torch.float64)
        for b in range(n):
            if finished is not None and finished[g, b]:
                total[b, eos] = float(scores[g, b])
            else:
                total[b] = float(scores[g, b]) + torch.log_softmax(logits[g, b].double(), -1)
        total = torch.where(torch.isfinite(total), total, torch.full_like(total, -math.inf)).flatten()
        order = torch.sort(-total, stable=True).indices[:keep].tolist()
        found.append([(float(total[i]), i // V, i % V, bool(i % V == eos or (finished is not None and finished[g, i // V]))) for i in order])
    return found


def reorder(cache, slots, parents, lengths):
    out = cache.clone()
    n = parents.shape[1]
    for g in range(parents.shape[0]):
        for j in range(n):
            p = int(parents[g, j])
            if not 0 <= p < n:
                continue
            live = cache.shape[2]
            if slots:
                length = int(lengths[0] if len(lengths) == 1 else lengths[g * n + p])
                live = min(live, max(0, -(-length // slots)))
            out[g * n + j, :, :live] = cache[g * n + p, :, :live]
    return out
