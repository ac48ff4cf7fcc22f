"""Plain models of the paged cache for the tests: the pages' rules on host integers, attention and
the rotation in 64 bits."""

import numpy as np
import torch

from llm_accelerator_amd._lib import STATUS_BAD_PAGE, STATUS_BAD_POSITION, STATUS_BAD_SEQUENCE, STATUS_NOT_RESERVED, STATUS_NO_PAGES


class Pages:
    """table, lengths and refs as lists, by the rules of include/q4dec.h; ``rows[page]`` is what the
    page's rows hold (any list of page_size values)."""

    def __init__(self, num_pages, page_size, num_seqs, max_pages):
        self.ps, self.max_pages = page_size, max_pages
        self.table = [[-1] * max_pages for _ in range(num_seqs)]
        self.lengths, self.refs = [0] * num_seqs, [0] * num_pages
        self.rows = [[None] * page_size for _ in range(num_pages)]
        self.status = 0

    def held(self, n):
        return -(-n // self.ps)

    def reserve(self, seqs, counts):
        err = self.status & STATUS_NOT_RESERVED
        grow = [(s, c) for s, c in zip(seqs, counts) if c != 0]
        for i, (s, c) in enumerate(grow):
            if c < 0 or not 0 <= s < len(self.lengths) or s in [g[0] for g in grow[:i]]:
                err |= STATUS_BAD_SEQUENCE
            elif self.lengths[s] + c > self.max_pages * self.ps:
                err |= STATUS_BAD_POSITION
            elif self.lengths[s] % self.ps and not 0 <= self.table[s][self.lengths[s] // self.ps] < len(self.refs):
                err |= STATUS_BAD_PAGE
        if err:
            self.status |= err | STATUS_NOT_RESERVED
            return
        last = {s: self.table[s][self.lengths[s] // self.ps] if self.lengths[s] % self.ps else None for s, _ in grow}
        shared = {}
        for s, _ in grow:
            if last[s] is not None:
                shared.setdefault(last[s], []).append(s)
        copies = [s for s, _ in grow if last[s] is not None and self.refs[last[s]] > 1
                  and not (len(shared[last[s]]) == self.refs[last[s]] and shared[last[s]][-1] == s)]
        need = [(s, s in copies, self.held(self.lengths[s] + c) - self.held(self.lengths[s])) for s, c in grow]
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if sum(c + k for _, c, k in need) > len(free):
            self.status |= STATUS_NO_PAGES | STATUS_NOT_RESERVED
            return
        for s, copy, more in need:
            have = self.held(self.lengths[s])
            if copy:
                page, old = free.pop(0), last[s]
                n = self.lengths[s] % self.ps
                self.rows[page][:n] = self.rows[old][:n]
                self.table[s][have - 1] = page
                self.refs[old] -= 1
                self.refs[page] = 1
            for i in range(more):
                page = free.pop(0)
                self.table[s][have + i] = page
                self.refs[page] = 1
        for s, c in grow:
            self.lengths[s] += c

    def fork(self, src, dst):
        n = len(self.lengths)
        lengths = list(self.lengths)
        for i, (s, d) in enumerate(zip(src, dst)):
            if not (0 <= s < n and 0 <= d < n) or d in src or d in dst[:i] or lengths[d] != 0:
                self.status |= STATUS_BAD_SEQUENCE
                continue
            pages = self.table[s][:self.held(lengths[s])]
            if any(not 0 <= p < len(self.refs) for p in pages):
                self.status |= STATUS_BAD_PAGE
                continue
            self.table[d][:len(pages)] = pages
            self.lengths[d] = lengths[s]
            for p in pages:
                self.refs[p] += 1

    def truncate(self, seqs, lengths=None):
        for i, s in enumerate(seqs):
            keep = lengths[i] if lengths is not None else 0
            if not 0 <= s < len(self.lengths) or s in seqs[:i] or not 0 <= keep <= self.lengths[s]:
                self.status |= STATUS_BAD_SEQUENCE
                continue
            for k in range(self.held(keep), self.held(self.lengths[s])):
                p = self.table[s][k]
                if 0 <= p < len(self.refs):
                    self.refs[p] -= 1
                else:
                    self.status |= STATUS_BAD_PAGE
                self.table[s][k] = -1
            self.lengths[s] = keep

    def compact(self):
        used = sum(r != 0 for r in self.refs)
        movers = [p for p, r in enumerate(self.refs) if r and p >= used]
        holes = [p for p, r in enumerate(self.refs) if not r and p < used]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.rows[b] = list(self.rows[a])
        for s, n in enumerate(self.lengths):
            for k in range(self.held(n)):
                self.table[s][k] = to.get(self.table[s][k], self.table[s][k])
        return used


def attend(cache, layer, batch, q, scaling):
    """(64-bit output, sum of p |v|, the largest |v| a subnormal probability may lose) per token row,
    NaN where a row is of no sequence.  Bad pages' positions are not there."""
    t, qh, d = q.shape
    out = torch.full((t, qh, d), float("nan"), dtype=torch.float64, device=q.device)
    size, tiny = out.clone(), out.clone()
    starts = batch.starts.tolist()
    seqs = batch.seqs.tolist() if batch.seqs is not None else list(range(batch.n))
    table, lengths, ps, kvh = cache.table.cpu(), cache.lengths.tolist(), cache.page_size, cache.num_kv_heads
    for b, row in enumerate(seqs):
        lo, hi = starts[b], starts[b + 1]
        if lo == hi:
            continue
        n = lengths[row]
        slots = np.arange(n)
        page = table[row].numpy()[slots // ps] if n else np.zeros(0, int)
        ok = (page >= 0) & (page < cache.num_pages)
        slots, page = torch.from_numpy(slots[ok]).to(q.device), torch.from_numpy(page[ok].astype(np.int64)).to(q.device)
        k, v = (cache.data[layer, i][page, :, slots % ps].double().repeat_interleave(qh // kvh, 1) for i in range(2))
        for i in range(lo, hi):
            seen = slots <= n - (hi - lo) + (i - lo)
            if not bool(seen.any()):
                out[i] = size[i] = tiny[i] = 0
                continue
            z = (k[seen] * q[i].double()).sum(-1) * scaling         # [s, qh]
            p = torch.softmax(z, 0)
            out[i] = (p[..., None] * v[seen]).sum(0)
            size[i] = (p[..., None] * v[seen].abs()).sum(0)
            tiny[i] = v[seen].abs().sum(0) * p.amax(0)[:, None]
    return out, size, tiny


def attend_bound(out, size, tiny, dtype):
    """The output rounded once and every probability rounded once to the cache's type (half a step
    each), scores and sums in fp32 (2^-14 of the weighted size: 32768 positions, exponents of scores up
    to 2^6); an fp16 probability below 2^-14 of the largest is off by up to 2^-25 of it, and the largest
    may be taken up to 2^8 low."""
    half = torch.finfo(dtype).eps / 2
    bound = half * out.abs() + (half + 2.0 ** -14) * size + 1e-30
    return bound + (2.0 ** -25 * tiny + 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)


def turn(x, gamma, eps, cos, sin, interleaved):
    """Head norm and rotation in 64 bits of x [tokens, heads, dim]; cos, sin [tokens, r / 2] or None."""
    y = x.double().clone()
    if gamma is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * gamma.double()
    if cos is None:
        return y
    half = cos.shape[1]
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cos.double()[:, None], sin.double()[:, None]
    ya, yb = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = ya * c - yb * s, yb * c + ya * s
    return y
