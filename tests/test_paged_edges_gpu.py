"""The paged 16-bit cache on the GPU where a value, a length or a page is at the edge of
what a call may hold: infinities and NaN beside masks, padded rows, pages outside the
cache, sizes near 2^31, soft-caps of any size."""
import math

import pytest
import torch

import llmx_b200
from gpu_helpers import needs_cuda
from llmx_b200 import LlmxError, paged
from oracle import paged as opaged
from paged_helpers import DEV, Case, check_attention, ints, place, read, table_of

pytestmark = [pytest.mark.gpu, needs_cuda]

DTYPES = [torch.float16, torch.bfloat16]


def rows_that_see(c, b, tokens, window=-1):
    """Which query rows of sequence b see one of the tokens (causal)."""
    ql = c.q_len if c.q_lens is None else c.q_lens[b]
    i = torch.arange(c.q_len)
    diag = i + c.lens[b] - ql
    hit = torch.zeros(c.q_len, dtype=torch.bool)
    for t in tokens:
        hit |= (t <= diag) & (i < ql) & ((diag - t <= window) if window >= 0 else True)
    return hit


def check_spread(c, poison, value, where="v", **kw):
    """`value` in channel 7 of kv head 1 of the tokens poison[b] of sequence b:
    rows that do not see one of them, and the other heads, keep their bits; with a
    NaN the rows that do become NaN."""
    clean, _ = c.run(**kw)
    assert clean.isfinite().all()
    group = c.heads // c.hkv
    for b, tokens in poison.items():
        for t in tokens:
            (c.k if where == "k" else c.v)[b][t, 1, 7] = value
        c.put(b)
    for _ in range(3):
        out, _ = c.run(**kw)
        for b in range(len(c.lens)):
            hit = rows_that_see(c, b, poison.get(b, ()), kw.get("window", -1))
            keep = torch.ones(c.q_len, c.heads, dtype=torch.bool)
            keep[hit, group:2 * group] = False
            assert torch.equal(out[b, keep], clean[b, keep]), f"sequence {b}"
            if math.isnan(value):
                assert out[b, hit.to(DEV), group:2 * group].isnan().flatten(2).any(-1).all(), f"sequence {b}"
    llmx_b200.device_status(0)


# Tiles: several items a CTA (160 of them and more), contexts of several blocks before
# the diagonal, so that the products of a block may be behind the next one's scores.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_non_finite_v_in_tiles(dtype, d, value):
    lens = [900 - 7 * i for i in range(40)]
    for kw in (dict(), dict(window=200)):
        c = Case(dtype, d, 4, 2, 32, 150, lens, seed=d)
        poison = {b: (lens[b] - 1, lens[b] - 77, lens[b] - 140, 300) for b in range(0, 40, 3)}
        check_spread(c, poison, value, algo="tcgen05", **kw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tiles_of_head_dim_256_without_anything_non_finite(dtype):
    c = Case(dtype, 256, 4, 2, 64, 200, [1500 - 31 * i for i in range(30)], seed=1)
    first, _ = c.check(algo="tcgen05", weights=True)
    for _ in range(5):
        out, lse = c.run(algo="tcgen05")
        assert torch.equal(out, first) and lse.isfinite().all()
    llmx_b200.device_status(0)


# Few rows at head_dim 256, whose ring holds fewer than three blocks: the new rows lie
# across a border of 128 tokens, so that the last block but one is partly seen while V
# of the block before it may still be on its way.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,q_len", [(16, 3), (16, 4), (16, 7), (6, 8), (6, 20)])
@pytest.mark.parametrize("value", [math.nan, -math.inf])
def test_non_finite_v_of_few_rows_across_a_block(dtype, heads, q_len, value):
    for lens in ([1025, 898, 385, 257], [129 + 128 * (i % 9) for i in range(90)]):
        c = Case(dtype, 256, heads, 2, 64, q_len, lens, seed=heads + q_len)
        poison = {b: (n // 128 * 128 - 1, n - 1, n // 128 * 128 - 2) for b, n in enumerate(lens) if b % 3 != 1}
        check_spread(c, poison, value, algo="decode")
        check_spread(Case(dtype, 256, heads, 2, 64, q_len, lens, seed=3), poison, value, algo="decode", window=150)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("algo", ["decode", "tcgen05"])
def test_padded_rows_beside_non_finite_tokens_are_zero(dtype, d, algo):
    """Rows at or past q_lens see no token: they are 0 (lse -inf) whatever the cache holds,
    in short sequences, which one CTA has whole, and in long ones."""
    for lens in ([200, 130, 256, 9], [2000, 130, 700, 9]):
        for where, value in (("v", math.nan), ("v", math.inf), ("k", math.nan), ("k", -math.inf)):
            c = Case(dtype, d, 4, 2, 32, 4, lens, q_lens=[1, 3, 0, 2], seed=d)
            check_spread(c, {0: (5,), 1: (0, 40), 2: (100,)}, value, where=where, algo=algo)
            out, lse = c.run(algo=algo)
            for b, n in enumerate(c.q_lens):
                assert not out[b, n:].any() and (lse[b, :, n:] == -math.inf).all(), (where, value, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_weights_of_a_chunk_with_a_negative_scale_and_a_cap(dtype, d):
    """Scores to well past the cap on both sides."""
    c = Case(dtype, d, 4, 2, 32, 40, [333, 77], seed=d)
    for cap in (3.0, 40.0):
        c.check(algo="decode", sm_scale=-4.0 * d ** -0.5, cap=cap, weights=True, what=f"cap {cap}")
        c.check(algo="decode", sm_scale=-4.0 * d ** -0.5, cap=cap, weights=True, slopes=torch.tensor([0.5, 0.1, 0.02, 0.004]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("algo,q_len", [("decode", 1), ("decode", 5), ("decode", 40), ("tcgen05", 5), ("tcgen05", 150)])
def test_weights_and_lse_do_not_depend_on_v(dtype, d, algo, q_len):
    """Key weights and lse come from q and K: an infinity or NaN in V does not show in them,
    in blocks that all rows see and in blocks that some do."""
    for lens in ([250, 190], [1500, 600]):
        for window in (-1, 100):
            c = Case(dtype, d, 4, 2, 32, q_len, lens, seed=d)
            w0, w1 = (torch.zeros(c.k_cache.shape[:3], device=DEV) for _ in range(2))
            _, lse0 = c.run(algo=algo, weights=w0, decay=0.0, window=window)
            c.v[0][[3, lens[0] - 1, lens[0] - 2, lens[0] - 80], 0, 9] = math.nan
            c.v[1][[lens[1] - 1, lens[1] - 30], 1, 1] = math.inf
            c.put(0), c.put(1)
            out, lse1 = c.run(algo=algo, weights=w1, decay=0.0, window=window)
            assert torch.equal(w0, w1) and torch.equal(lse0, lse1)
            assert out[0, -1, :2].isnan().flatten(1).any(-1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("algo,q_len", [("decode", 1), ("decode", 4), ("decode", 40), ("tcgen05", 70)])
@pytest.mark.parametrize("cap", [0.5, 50.0, 1e3, 1e4, 1e6])
def test_a_soft_cap_keeps_the_bits_of_the_scores(dtype, algo, q_len, cap):
    """A capped score is right to 2^-20 of itself, whatever the cap: its argument, the product
    with the cap and the fit or the special functions each cost a few 2^-24 of it."""
    for d, scale in ((64, 0.25), (128, 3.0)):  # scores of spread 2, and of 34, past a cap of 50
        c = Case(dtype, d, 4, 2, 32, q_len, [300, 90], seed=q_len)
        kw = dict(cap=cap, sm_scale=scale)
        for slopes in (None, torch.tensor([0.1, 0.03, 0.01, 0.002])):
            w = torch.zeros(c.k_cache.shape[:3], device=DEV)
            out, lse = c.run(algo=algo, weights=w, decay=0.0, alibi_slopes=None if slopes is None else slopes.to(DEV), **kw)
            for b, n in enumerate(c.lens):
                want = c.want(b, slopes=slopes, cap_relative=True, **kw)
                check_attention(out[b], lse[b], read(w.unsqueeze(-1), c.table, b, n)[..., 0].T, want, dtype, f"{b} {scale}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,heads", [(64, 14), (128, 14), (256, 6), (128, 8)])
@pytest.mark.parametrize("scale", [1.0, -1.0])
def test_soft_capped_bits_do_not_depend_on_what_no_row_sees(dtype, d, heads, scale):
    """Padded rows of q, the rest of a sequence's last page and whatever ran before:
    groups that do not divide 128 leave rows of a tile unused."""
    c = Case(dtype, d, heads, 2, 64, 50, [333, 70, 50], q_lens=[50, 33, 7], seed=heads)
    algos = ("auto", "tcgen05") if scale > 0 else ("decode",)
    for algo in algos:
        for kw in (dict(cap=8.0), dict(cap=30.0, window=90), dict(cap=4.0, causal=False)):
            first = None
            for junk in (0.0, 3.0, -1000.0, math.nan, math.inf):
                for b, n in enumerate(c.q_lens):
                    c.q[b, n:] = junk
                c.k_cache.fill_(junk), c.v_cache.fill_(junk)
                for b in range(3):
                    c.put(b)
                w = torch.zeros(c.k_cache.shape[:3], device=DEV)
                out, lse = c.run(algo=algo, weights=w, decay=0.0, sm_scale=scale * d ** -0.5, **kw)
                if first is None:
                    first = out, lse, w
                for x, y in zip(first, (out, lse, w)):
                    assert torch.equal(x, y), (algo, kw, junk)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 256)])
def test_evicted_tokens_of_pages_outside_the_cache_are_zeros(in_place, dtype, d):
    """A kept token whose page lies outside the cache becomes a row of zeros with weight 0."""
    page, lens, budget, recent, sinks = 16, [100, 40, 70], 50, 20, 18
    gen = torch.Generator().manual_seed(d)
    table, n_pages = table_of(lens, page, 1, gen)
    need = -(-budget // page)
    kc, vc = (torch.full((n_pages + 3 * need, 2, page, d), 7.0, dtype=dtype, device=DEV) for _ in range(2))
    w = torch.full(kc.shape[:3], 7.0, device=DEV)
    data = []
    for b, n in enumerate(lens):
        k, v = (torch.randn(n, 2, d, generator=gen).to(dtype) for _ in range(2))
        x = torch.rand(n, 2, 1, generator=gen) + 1
        place(kc, table, b, k), place(vc, table, b, v), place(w.unsqueeze(-1), table, b, x)
        data.append((k, v, x[..., 0]))
    # the second page of the first sequence (sinks), its fifth (recent), one of a
    # sequence that is kept whole, and one of neither in the third
    table[0, 1], table[0, 5], table[1, 2], table[2, 1] = n_pages + 999, -1, 2 ** 31 - 1, -2 ** 31
    out = (n_pages + torch.randperm(3 * need, generator=gen)).view(3, need).int()
    kept, new = llmx_b200.paged_evict(kc, vc, w, budget, kv_lens=ints(lens), block_table=table.to(DEV), recent=recent, sinks=sinks,
                                      **({} if in_place else {"out_table": out.to(DEV)}))
    with pytest.raises(LlmxError):
        llmx_b200.device_status(0)
    llmx_b200.device_status(0)
    for b, n in enumerate(lens):
        k, v, x = data[b]
        outside = torch.tensor([not 0 <= int(p) < kc.shape[0] for p in table[b]])
        gone = outside[torch.arange(n) // page]
        ranked = torch.where(gone[:, None], torch.tensor(-math.inf), x)
        m = min(n, budget)
        assert int(new[b]) == m
        for h in range(2):
            want = opaged.kept(ranked[:, h], n, budget, recent, sinks)
            assert kept[b, h, :m].tolist() == want
            for r, j in enumerate(want):
                to = int((table if in_place else out)[b, r // page])
                if not 0 <= to < kc.shape[0]:
                    continue  # the place itself lies outside
                for got, src in ((kc, k), (vc, v), (w, x)):
                    expect = torch.zeros_like(src[j, h]) if gone[j] else src[j, h]
                    assert torch.equal(got[to, h, r % page].cpu(), expect), (b, h, r, j)


@pytest.mark.parametrize("seqs", [1, 2])
def test_the_largest_budget_stays_inside_kept(seqs):
    """-1 behind the kept positions up to a budget of 2^31 - 1, and nothing in front of it."""
    page, budget, front = 16, 2 ** 31 - 1, 65536
    kc, vc = (torch.zeros(4 * seqs, 1, page, 64, dtype=torch.float16, device=DEV) for _ in range(2))
    w = torch.zeros(4 * seqs, 1, page, device=DEV)
    buf = torch.full((front + seqs * budget,), 5, dtype=torch.int32, device=DEV)
    kept = buf[front:].view(seqs, 1, budget)
    lens = [50, 3][:seqs]
    llmx_b200.paged_evict(kc, vc, w, budget, kv_lens=ints(lens), kept=kept)
    assert (buf[:front] == 5).all()
    for b, n in enumerate(lens):
        assert kept[b, 0, :n].tolist() == list(range(n))
        assert int(kept[b, 0, n:].max()) == -1 and int(kept[b, 0, n:].min()) == -1
    llmx_b200.device_status(0)


@pytest.mark.parametrize("rows", [2 ** 31 - 1, 2 ** 31 - 64, 2 ** 31 - 65])
def test_store_of_row_counts_near_2_31(rows):
    """Rows that are all one row (stride 0), of which lens takes a few."""
    kc, vc = (torch.zeros(4, 1, 16, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    k = torch.randn(1, 1, 1, 64, device=DEV).bfloat16()
    for call in (llmx_b200.paged_store, paged.paged_store_ctypes):
        kc.zero_(), vc.zero_()
        call(kc, vc, k.expand(1, rows, 1, 64), (-k).expand(1, rows, 1, 64), start=ints([3]), lens=ints([40]))
        got = kc.view(64, 64)
        assert (got[3:43] == k.view(64)).all() and not got[:3].any() and not got[43:].any() and torch.equal(vc, -kc)
    llmx_b200.device_status(0)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("algo,q_len", [("decode", 4), ("tcgen05", 150)])
def test_non_finite_v_with_alibi_and_padded_rows(d, algo, q_len):
    """ALiBi takes a sequence's blocks last to first."""
    slopes = torch.tensor([0.3, -0.1, 0.02, 0.004], device=DEV)
    lens = [900 - 23 * i for i in range(12)]
    c = Case(torch.bfloat16, d, 4, 2, 48, q_len, lens, q_lens=[q_len - i % 4 for i in range(12)], seed=d)
    poison = {b: (n - 1, n - 90, n // 128 * 128 - 1, 200) for b, n in enumerate(lens) if b % 2}
    check_spread(c, poison, math.nan, algo=algo, alibi_slopes=slopes)
