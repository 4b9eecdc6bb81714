"""Helpers of the tests of the paged 16-bit cache."""
import math

import torch

import llmx_b200
from oracle import paged as opaged

DEV = "cuda"


def table_of(lens_max, page, extra, gen, unused=-7):
    """A block table of shuffled pages for sequences of up to lens_max tokens;
    entries behind a sequence are never read."""
    need = [-(-n // page) for n in lens_max]
    order = torch.randperm(sum(need) + extra, generator=gen).int()
    table = torch.full((len(need), max(max(need), 1)), unused, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(need) + extra


def empty_cache(n_pages, hkv, page, d, dtype, order="hnd", fill=math.nan):
    """K, V of garbage; order "nhd": tokens outside, heads inside."""
    shape = (n_pages, hkv, page, d) if order == "hnd" else (n_pages, page, hkv, d)
    both = [torch.full(shape, fill, dtype=dtype, device=DEV) for _ in range(2)]
    return tuple(c if order == "hnd" else c.transpose(1, 2) for c in both)


def rows(gen, n, hkv, d, dtype):
    return torch.randn(n, hkv, d, generator=gen).to(dtype)


def place(cache, table, b, x):
    """Writes x [n, hkv, d] as tokens 0 .. of sequence b (plain indexing)."""
    page = cache.shape[2]
    j = torch.arange(x.shape[0])
    cache[table[b, j // page].long().to(DEV), :, (j % page).to(DEV)] = x.to(DEV)


def read(cache, table, b, n):
    page = cache.shape[2]
    j = torch.arange(n)
    return cache[table[b, j // page].long().to(DEV), :, (j % page).to(DEV)].cpu()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def check_attention(out, lse, weights, want, dtype, what="", old=None):
    """out [S, H, D], lse [H, S], weights [H_kv, N] of one sequence against the
    oracle's tuple; `old` is added to the weights' expectation."""
    o, le, w, bo, bl, bw = want
    half = torch.finfo(dtype).eps / 2
    out = out.double().cpu()
    room = bo * (1 + 2 ** -10) + (o.abs() + bo) * half + torch.finfo(dtype).smallest_normal * half
    off = ~((out - o).abs() <= room)
    assert not off.any(), (f"{what}: {int(off.sum())} of {off.numel()} outputs off, worst "
                           f"{float(((out - o).abs() / room.clamp_min(1e-300)).nan_to_num(1e9).max()):.3g} of the bound")
    if lse is not None:
        lse = lse.double().cpu()
        empty = le == -math.inf
        assert torch.equal(lse == -math.inf, empty), f"{what}: empty rows"
        assert ((lse - le).abs()[~empty] <= bl[~empty]).all(), f"{what}: lse"
    if weights is not None:
        weights = weights.double().cpu()
        if old is not None:
            w = w + old
        # Each of a token's terms, one for each row and head of its kv head, may be
        # below the normal range of fp32 and then counts as 0.
        terms = le.numel() // w.shape[0] if le.numel() else 64
        room = bw + 2.0 ** -23 * w.abs() + terms * 2.0 ** -126
        off = ~((weights - w).abs() <= room)
        assert not off.any(), (f"{what}: {int(off.sum())} of {off.numel()} weights off, worst "
                               f"{float(((weights - w).abs() / room).nan_to_num(1e9).max()):.3g} of the bound")


class Case:
    """Sequences in a garbage cache, with queries."""

    def __init__(self, dtype, d, heads, hkv, page, q_len, lens, *, q_lens=None, order="hnd", seed=0, extra=2):
        gen = torch.Generator().manual_seed(seed)
        self.dtype, self.d, self.heads, self.hkv, self.page, self.q_len = dtype, d, heads, hkv, page, q_len
        self.lens, self.q_lens = lens, q_lens
        self.table, n_pages = table_of(lens, page, extra, gen)
        self.k_cache, self.v_cache = empty_cache(n_pages, hkv, page, d, dtype, order)
        self.k = [rows(gen, n, hkv, d, dtype) for n in lens]
        self.v = [rows(gen, n, hkv, d, dtype) for n in lens]
        for b in range(len(lens)):
            self.put(b)
        self.q = torch.randn(len(lens), q_len, heads, d, generator=gen).to(dtype)
        self.gen = gen

    def put(self, b):
        place(self.k_cache, self.table, b, self.k[b])
        place(self.v_cache, self.table, b, self.v[b])

    def run(self, *, weights=None, algo="auto", call=None, **kw):
        out = torch.full_like(self.q, math.nan, device=DEV)
        lse = torch.full((len(self.lens), self.heads, self.q_len), math.nan, device=DEV)
        (call or llmx_b200.paged_attention)(
            out, self.q.to(DEV), self.k_cache, self.v_cache, kw.pop("sm_scale", self.d ** -0.5), kw.pop("window", -1),
            kw.pop("cap", 0.0), kv_lens=ints(self.lens), block_table=self.table.to(DEV),
            q_lens=None if self.q_lens is None else ints(self.q_lens), lse=lse, key_weights=weights, algo=algo, **kw)
        torch.cuda.synchronize()
        return out, lse

    def want(self, b, **kw):
        kw.setdefault("sm_scale", self.d ** -0.5)
        return opaged.attention(self.q[b], self.k[b], self.v[b], self.q_len if self.q_lens is None else self.q_lens[b],
                                self.lens[b], **kw)

    def check(self, *, weights=False, algo="auto", what="", call=None, slopes=None, **kw):
        w = torch.full(self.k_cache.shape[:3], math.nan, device=DEV) if weights else None
        dev = {} if slopes is None else {"alibi_slopes": slopes.to(DEV)}
        out, lse = self.run(weights=w, algo=algo, call=call, **dev, **kw, **({"decay": 0.0} if weights else {}))
        for name in ("decay", "max_kv_len"):
            kw.pop(name, None)
        for b, n in enumerate(self.lens):
            got = None
            if weights:
                got = read(w.unsqueeze(-1), self.table, b, n)[..., 0].T
            check_attention(out[b], lse[b], got, self.want(b, slopes=slopes, **kw), self.dtype, f"{what} sequence {b}")
        if weights:  # places that hold no token keep what they had
            held = torch.zeros(w.shape[0], w.shape[2], dtype=torch.bool)
            for b, n in enumerate(self.lens):
                j = torch.arange(n)
                held[self.table[b, j // self.page].long(), j % self.page] = True
            assert torch.equal(~w.isnan().any(1).cpu(), held), f"{what}: weights outside the sequences"
        return out, lse
