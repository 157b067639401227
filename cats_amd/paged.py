"""A cache of keys and values in pages, for many sequences of different lengths: the tensors that ``flash_gemv.cats_paged_append`` and ``cats_paged_attention``
share, and who has which of them.

A page holds ``page`` tokens of one layer; a sequence has as many as its tokens need, anywhere in the pool, and its row of a table says which.  So no
sequence takes the memory of the longest one, and sequences that begin alike (beams, answers to one prompt) share the pages of what they have in common.

    cache = PagedCache(layers, pages, kv_heads, head_dim, dtype=torch.float16)
    ids = [cache.open() for _ in prompts]
    cache.reserve(ids, lengths)                        # room for that many tokens each
    table = cache.table(ids)                           # (B, entries) int32 on the GPU: one for all layers, until somebody's pages change
    q = cache.append(layer, q, k, v, offsets, start, table, cos, sin)     # packed tokens; offsets, start: int64 on the GPU
    out = cache.attend(layer, q, offsets, start, table)
    beams = cache.fork(ids[0], 4, length)              # four more sequences that begin with its first `length` tokens
    cache.close(ids[0])

Which pages are whose is kept on the host.  A sequence goes on from behind its last token, or from where ``trim`` put its end: what lies before may be others' too.
Pages that come free are given to the next who asks: work that still reads them must have been launched on the same
stream before, or be over.  Pages are not cleared.  A table that a captured graph reads is filled in place with ``table(ids, out=...)``.

For fp16 and bf16 on the GPU, heads of 32, 64, 128 or 256 elements, pages of 16 to 1024 tokens (a power of two), without gradients.
"""
from __future__ import annotations

import torch


class PagedCache:
    def __init__(self, layers, pages, kv_heads, head_dim, page=64, dtype=torch.float16, device="cuda"):
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"a cache of pages is for float16 and bfloat16 models, not {dtype}")
        if head_dim not in (32, 64, 128, 256):
            raise ValueError(f"heads of 32, 64, 128 or 256 elements, not {head_dim}")
        if page not in (16, 32, 64, 128, 256, 512, 1024):
            raise ValueError(f"pages of 16 to 1024 tokens, a power of two, not {page}")
        if min(layers, pages, kv_heads) < 1:
            raise ValueError("a cache needs at least one layer, one page and one head")
        self.page = page
        self.k, self.v = (torch.zeros(layers, pages, kv_heads, page, head_dim, dtype=dtype, device=device) for _ in range(2))
        self._free = list(range(pages - 1, -1, -1))
        self._users = [0] * pages
        self._pages = {}  # of each sequence
        self._next = 0

    @property
    def free(self):
        """Pages that nobody has."""
        return len(self._free)

    def pages_of(self, seq):
        return list(self._pages[seq])

    def open(self):
        """A new sequence, without pages."""
        self._pages[self._next] = []
        self._next += 1
        return self._next - 1

    def reserve(self, seqs, lengths):
        """Pages for the first `lengths` tokens (an int, or one a sequence) of each; what a sequence has more stays.  Takes none if there are not enough."""
        seqs = list(seqs)
        lengths = [lengths] * len(seqs) if isinstance(lengths, int) else list(lengths)
        if len(seqs) != len(lengths) or len(set(seqs)) != len(seqs):
            raise ValueError(f"{len(seqs)} sequences, each once, with {len(lengths)} lengths")
        need = [max(0, -(-n // self.page) - len(self._pages[s])) for s, n in zip(seqs, lengths)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"{sum(need)} pages are needed and {len(self._free)} are free")
        for s, n in zip(seqs, need):
            self._pages[s] += [self._take() for _ in range(n)]

    def trim(self, seq, length):
        """Gives back the pages behind the first `length` tokens, from where the sequence may go on.  The page in which they end becomes its own: where others have
        it too, it is copied, and if there is no page for the copy, nor one among those that come free, the sequence stays as it is."""
        pages = self._pages[seq]
        if not 0 <= length <= len(pages) * self.page:
            raise ValueError(f"the first {length} tokens of a sequence with {len(pages)} pages of {self.page}")
        whole, rest = divmod(length, self.page)
        kept = whole + (rest > 0)
        copied = rest > 0 and self._users[pages[whole]] > 1
        if copied and not self._free and all(self._users[p] > 1 for p in pages[kept:]):
            raise RuntimeError("1 page is needed and 0 are free")
        for p in pages[kept:]:
            self._give(p)
        del pages[kept:]
        if copied:
            pages[whole] = self._copy(pages[whole], rest)

    def fork(self, seq, count, length):
        """`count` new sequences that begin with the first `length` tokens of this one.  Whole pages are shared, the page in which they end is copied, in all
        layers.  Sequences that stand together in a call and were forked at `length` may be attended as a group with `shared` = length: of that the whole
        pages count, and the first one's are read, so it may not have been cut within them."""
        pages = self._pages[seq]
        if not 0 <= length <= len(pages) * self.page:
            raise ValueError(f"the first {length} tokens of a sequence with {len(pages)} pages of {self.page}")
        whole, rest = divmod(length, self.page)
        if rest and count > len(self._free):
            raise RuntimeError(f"{count} pages are needed and {len(self._free)} are free")
        new = []
        for _ in range(count):
            s = self.open()
            self._pages[s] = pages[:whole] + ([self._copy(pages[whole], rest, give=False)] if rest else [])
            for p in pages[:whole]:
                self._users[p] += 1
            new.append(s)
        return new

    def close(self, seq):
        """The sequence ends; pages that nobody else has come free."""
        for p in self._pages.pop(seq):
            self._give(p)

    def table(self, seqs, out=None):
        """(sequences, entries) int32 on the cache's device: each one's pages in order, -1 behind them.  out: filled in place, with as many entries as it has."""
        rows = [self._pages[s] for s in seqs]
        most = max([1] + [len(r) for r in rows])
        width = most if out is None else out.shape[1]
        if out is not None and (most > width or out.shape[0] != len(rows)):
            raise ValueError(f"a table of {tuple(out.shape)} for {len(rows)} sequences with up to {most} pages")
        t = torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32).reshape(len(rows), width)
        if out is None:
            return t.to(self.k.device)
        out.copy_(t)
        return out

    def append(self, layer, q, k, v, offsets, start, table, cos=None, sin=None):
        """Rotate the queries and keys of packed tokens (no tables: not) and store keys and values; the queries, rotated."""
        import flash_gemv

        return flash_gemv.cats_paged_append(q, k, v, offsets, start, cos, sin, self.k[layer], self.v[layer], table)

    def attend(self, layer, q, offsets, start, table, scale=None, window=0, group=1, shared=None):
        """Causal attention of packed tokens that have been appended at start."""
        import flash_gemv

        scale = q.shape[-1] ** -0.5 if scale is None else scale
        return flash_gemv.cats_paged_attention(q, offsets, start, self.k[layer], self.v[layer], table, scale, window, group, shared)

    def _take(self):
        if not self._free:
            raise RuntimeError("1 page is needed and 0 are free")
        p = self._free.pop()
        self._users[p] = 1
        return p

    def _give(self, p):
        self._users[p] -= 1
        if self._users[p] == 0:
            self._free.append(p)

    def _copy(self, old, tokens, give=True):
        p = self._take()
        for x in (self.k, self.v):
            x[:, p, :, :tokens] = x[:, old, :, :tokens]
        if give:
            self._give(old)
        return p
