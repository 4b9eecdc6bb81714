"""The paged 16-bit cache on the GPU: store and eviction bit by bit, attention and
key weights element by element against the oracle's bounds (oracle/paged.py)."""
import ctypes
import math

import pytest
import torch

import llmx_b200
from gpu_helpers import needs_cuda
from llmx_b200 import LlmxError, _lib, paged
from oracle import paged as opaged
from paged_helpers import DEV, Case, check_attention, empty_cache, ints, place, read, rows, table_of

pytestmark = [pytest.mark.gpu, needs_cuda]

DTYPES = [torch.float16, torch.bfloat16]


def slopes_of(heads):
    return torch.pow(2.0, -8.0 * torch.arange(1, heads + 1, dtype=torch.float64) / heads).float()


# ------------------------------------------------------------------- store
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,hkv,page,order", [(64, 1, 16, "hnd"), (128, 3, 48, "nhd"), (256, 2, 64, "hnd")])
def test_store_writes_its_rows_and_nothing_else(dtype, d, hkv, page, order):
    gen = torch.Generator().manual_seed(1)
    starts, lens, S = [0, 5, page - 1, 7, 3 * page], [33, 0, 2, 70, 1], 70
    table, n_pages = table_of([s + n for s, n in zip(starts, lens)], page, 2, gen)
    kc, vc = empty_cache(n_pages, hkv, page, d, dtype, order, fill=3.0)
    k = torch.randn(5, S, hkv, d, generator=gen).to(dtype)
    v = torch.randn(5, S, hkv, d, generator=gen).to(dtype)
    want_k, want_v = kc.cpu().clone(), vc.cpu().clone()
    for b in range(5):
        for i in range(lens[b]):
            p, o = divmod(starts[b] + i, page)
            want_k[table[b, p], :, o] = k[b, i]
            want_v[table[b, p], :, o] = v[b, i]
    for call in (llmx_b200.paged_store, paged.paged_store_ctypes):
        kc.fill_(3.0), vc.fill_(3.0)
        call(kc, vc, k.to(DEV), v.to(DEV), start=ints(starts), lens=ints(lens), block_table=table.to(DEV))
        assert torch.equal(kc.cpu(), want_k) and torch.equal(vc.cpu(), want_v)
    # rows by other strides: heads outside, and rows that are not 16-byte aligned
    for view in (lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda x: torch.nn.functional.pad(x, (1, 2))[..., 1:-2]):
        kc.fill_(3.0), vc.fill_(3.0)
        llmx_b200.paged_store(kc, vc, view(k.to(DEV)), view(v.to(DEV)), start=ints(starts), lens=ints(lens),
                              block_table=table.to(DEV))
        assert torch.equal(kc.cpu(), want_k) and torch.equal(vc.cpu(), want_v)


def test_store_without_table_start_and_lens():
    kc, vc = empty_cache(6, 2, 16, 64, torch.float16, fill=0.0)
    k = torch.randn(3, 20, 2, 64, device=DEV).half()
    llmx_b200.paged_store(kc, vc, k, -k)
    got = kc.view(3, 2, 2, 16, 64).transpose(2, 3).reshape(3, 32, 2, 64)
    assert torch.equal(got[:, :20], k) and not got[:, 20:].any()
    assert torch.equal(vc, -kc)


def test_store_drops_rows_outside_the_cache():
    kc, vc = empty_cache(4, 1, 16, 64, torch.bfloat16, fill=0.0)
    k = torch.randn(3, 4, 1, 64, device=DEV).bfloat16()
    table = ints([[0, 9], [-1, 1], [2, 3]])
    llmx_b200.paged_store(kc, vc, k, k, start=ints([14, 14, -2]), block_table=table)
    with pytest.raises(LlmxError):
        llmx_b200.device_status(0)
    llmx_b200.device_status(0)
    want = torch.zeros_like(kc)
    want[0, :, 14:] = k[0, :2].transpose(0, 1)
    want[1, :, :2] = k[1, 2:].transpose(0, 1)
    want[2, :, :2] = k[2, 2:].transpose(0, 1)
    assert torch.equal(kc, want)


# --------------------------------------------------------------- attention
SHAPES = [
    # d, heads, hkv, page, q_len, lens, q_lens
    (64, 8, 2, 16, 1, [77], None),
    (64, 3, 3, 16, 1, [1, 15, 16, 17, 64, 65, 0, 300], None),
    (128, 8, 2, 64, 1, [1000, 5, 0, 257, 64], None),
    (128, 32, 1, 32, 1, [333, 90], None),
    (128, 7, 1, 48, 1, [130, 1, 999], None),
    (256, 4, 2, 16, 1, [500, 31], None),
    (128, 8, 2, 64, 5, [300, 3, 5, 0, 640], [5, 5, 4, 2, 0]),
    (64, 16, 1, 32, 3, [200, 77], None),
    (128, 4, 4, 16, 16, [16, 500], [16, 3]),
    (256, 16, 2, 64, 7, [129, 70], [7, 1]),
    (64, 2, 1, 16, 150, [150, 400], [150, 31]),
    (128, 6, 2, 112, 100, [100, 613, 90], [100, 77, 90]),
    (256, 4, 1, 32, 80, [81, 260], None),
    (256, 3, 3, 16, 300, [300, 700, 512], [300, 299, 1]),
]
MASKS = [dict(), dict(causal=False), dict(window=20), dict(window=0), dict(cap=5.0), dict(alibi=True),
         dict(causal=False, window=33, cap=3.0), dict(window=100, alibi=True)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "d%d_h%d_%d_p%d_q%d" % s[:5])
@pytest.mark.parametrize("algo", ["auto", "decode"])
def test_attention(dtype, shape, algo):
    d, heads, hkv, page, q_len, lens, q_lens = shape
    c = Case(dtype, d, heads, hkv, page, q_len, lens, q_lens=q_lens, seed=d + heads + q_len)
    for mask in MASKS:
        kw = dict(mask)
        if kw.pop("alibi", False):
            kw["slopes"] = slopes_of(heads)
        c.check(algo=algo, what=str(mask), **kw)
        c.check(algo=algo, what=str(mask) + " weights", weights=True, **kw)


TC_SHAPES = [
    # d, heads, hkv, page, q_len, lens, q_lens
    (64, 8, 2, 16, 1, [77, 0, 300], None),
    (128, 8, 2, 64, 5, [300, 3, 5, 0, 640], [5, 5, 4, 2, 0]),
    (64, 2, 2, 16, 150, [150, 400], [150, 31]),
    (128, 6, 2, 112, 100, [100, 613, 90], [100, 77, 90]),
    (128, 1, 1, 128, 300, [300], None),
    (128, 7, 1, 32, 40, [1000, 40, 41], None),
    (64, 128, 1, 256, 3, [513, 2], None),
    (128, 4, 4, 48, 257, [700, 257, 128, 0], [257, 200, 1, 0]),
    (64, 16, 8, 64, 33, [5000, 33], None),
    (128, 32, 8, 64, 130, [900] * 5, None),
    (256, 4, 2, 32, 70, [600, 0, 71, 128], [70, 3, 69, 1]),
    (256, 5, 1, 16, 60, [300], None),
    (256, 2, 2, 128, 290, [1000, 290], None),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", TC_SHAPES, ids=lambda s: "d%d_h%d_%d_p%d_q%d" % s[:5])
def test_attention_in_tiles(dtype, shape):
    d, heads, hkv, page, q_len, lens, q_lens = shape
    c = Case(dtype, d, heads, hkv, page, q_len, lens, q_lens=q_lens, seed=d + heads + q_len)
    for mask in MASKS:
        kw = dict(mask)
        if kw.pop("alibi", False):
            kw["slopes"] = slopes_of(heads)
        c.check(algo="tcgen05", what=str(mask), **kw)
        c.check(algo="tcgen05", what=str(mask) + " weights", weights=True, **kw)
    llmx_b200.device_status(0)


@pytest.mark.parametrize("algo", ["auto", "decode"])
@pytest.mark.parametrize("q_len", [1, 3, 40])
def test_other_layouts_and_scales(q_len, algo):
    c = Case(torch.bfloat16, 128, 8, 2, 48, q_len, [400, 41, 0], order="nhd")
    c.check(what="tokens outside", weights=True, algo=algo)
    c.check(what="ctypes", call=paged.paged_attention_ctypes, weights=True, algo=algo)
    c.check(what="bound", max_kv_len=400, algo=algo)
    c.check(what="negative slopes", slopes=-slopes_of(8), weights=True, algo=algo)
    if algo == "decode":
        c.check(what="negative scale", sm_scale=-0.1, algo=algo)
        c.check(what="zero scale", sm_scale=0.0, algo=algo)


@pytest.mark.parametrize("q_len", [1, 6, 70])
def test_strided_q_and_output(q_len):
    c = Case(torch.float16, 64, 6, 2, 32, q_len, [300, 90])
    want, _ = c.run()
    q = torch.empty(2, 6, q_len, 128, dtype=c.dtype, device=DEV)[..., 64:].transpose(1, 2)
    q.copy_(c.q)
    out = torch.full((q_len, 2, 6, 72), 9.0, dtype=c.dtype, device=DEV).transpose(0, 1)
    llmx_b200.paged_attention(out[..., :64], q, c.k_cache, c.v_cache, 64 ** -0.5, kv_lens=ints(c.lens),
                              block_table=c.table.to(DEV))
    assert torch.equal(out[..., :64], want) and (out[..., 64:] == 9.0).all()


def test_without_a_table():
    c = Case(torch.bfloat16, 64, 4, 2, 16, 1, [60, 33], seed=3)
    kc, vc = empty_cache(8, 2, 16, 64, c.dtype)
    table = torch.arange(8).view(2, 4).int()
    for b in range(2):
        place(kc, table, b, c.k[b])
        place(vc, table, b, c.v[b])
    out = torch.empty_like(c.q, device=DEV)
    llmx_b200.paged_attention(out, c.q.to(DEV), kc, vc, 64 ** -0.5, kv_lens=ints(c.lens))
    assert torch.equal(out, c.run()[0])


@pytest.mark.parametrize("algo", ["auto", "decode", "tcgen05"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len", [1, 4, 90])
def test_non_finite_tokens_reach_the_rows_that_see_them_only(dtype, q_len, algo):
    d, heads, hkv, lens = 128, 4, 2, [300, 200]
    for where in ("k", "v"):
        for value in (math.nan, math.inf, -math.inf):
            c = Case(dtype, d, heads, hkv, 32, q_len, lens, seed=5)
            clean = {w: c.run(window=w, algo=algo) for w in (-1, 50)}
            # tokens 299 (the last row's own), 210 and 5 of sequence 0, kv head 1
            for tok in (299, 210, 5):
                (c.k if where == "k" else c.v)[0][tok, 1, 7] = value
            c.put(0)
            for window in (-1, 50):
                out, lse = c.run(window=window, algo=algo)
                diag = torch.arange(q_len) + 300 - q_len
                hit = torch.zeros(q_len, dtype=torch.bool)
                for tok in (299, 210, 5):
                    hit |= (tok <= diag) & ((diag - tok <= window) if window >= 0 else True)
                o, l = clean[window]
                assert torch.equal(out[1], o[1]) and torch.equal(lse[1], l[1])
                assert torch.equal(out[0, :, :2], o[0, :, :2])  # heads of the other kv head
                rows_ok = out[0, ~hit][:, 2:]
                assert torch.equal(rows_ok, o[0, ~hit][:, 2:]), (where, value, window)
                if math.isnan(value):
                    bad = out[0, hit.to(DEV)][:, 2:]
                    assert bad.isnan().flatten(2).any(-1).all()


def test_infinite_query_rows_keep_to_themselves():
    c = Case(torch.bfloat16, 64, 4, 1, 16, 20, [100])
    want, _ = c.run()
    c.q[0, 3, 2, 5] = math.inf
    c.q[0, 7, 0, 0] = math.nan
    for algo in ("auto", "decode"):
        out, _ = c.run(algo=algo)
        ref, _ = Case(torch.bfloat16, 64, 4, 1, 16, 20, [100]).run(algo=algo)
        keep = torch.ones(20, 4, dtype=torch.bool)
        keep[3, 2] = keep[7, 0] = False
        assert torch.equal(out[0, keep], ref[0, keep])
        assert out[0, 7, 0].isnan().all()


@pytest.mark.parametrize("q_len", [1, 100])
def test_alibi_far_into_a_sequence_keeps_its_bits(q_len):
    c = Case(torch.float16, 64, 2, 1, 128, q_len, [40000], seed=9)
    for s in (torch.tensor([0.84, 0.01]), torch.tensor([-0.84, -0.001])):
        c.check(slopes=s, what="alibi", weights=True)


def test_long_sequence_among_short_ones():
    c = Case(torch.bfloat16, 128, 8, 2, 64, 1, [9000, 1, 64, 0, 700, 3, 2500, 65] * 3, seed=2)
    c.check(weights=True)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens,q_lens", [([4200, 4200, 4200], None), ([6000, 40, 0, 4100], [50, 40, 0, 7]), ([9, 1, 5000], [9, 1, 50])])
def test_tiles_cut_by_the_lengths_on_the_device(d, lens, q_lens):
    c = Case(torch.bfloat16, d, 8, 2, 64, 50, lens, q_lens=q_lens, seed=d + len(lens))
    for kw in (dict(), dict(causal=False), dict(window=4500, cap=20.0), dict(slopes=slopes_of(8))):
        c.check(algo="tcgen05", what=str(list(kw)), **kw)
    c.check(algo="tcgen05", weights=True)
    llmx_b200.device_status(0)


def test_many_sequences():
    lens = [(37 * i) % 200 for i in range(300)]
    c = Case(torch.float16, 64, 2, 1, 16, 1, lens, seed=4)
    c.check(weights=True)


def test_weights_accumulate_and_decay():
    c = Case(torch.bfloat16, 128, 4, 2, 16, 3, [100, 40])
    w = torch.full(c.k_cache.shape[:3], 2.0, device=DEV)
    c.run(weights=w, decay=0.5)
    for b, n in enumerate(c.lens):
        got = read(w.unsqueeze(-1), c.table, b, n)[..., 0].T
        old = torch.where(torch.arange(n) < n - 3, 1.0, 0.0).double()
        want = c.want(b)
        check_attention(torch.zeros(0), None, got, (torch.zeros(0),) * 2 + want[2:3] + (torch.zeros(0),) * 2 + want[5:], c.dtype,
                        old=old)
    w.fill_(2.0)
    c.run(weights=w, causal=False)  # decay 1, and no token is the call's own
    got = read(w.unsqueeze(-1), c.table, 0, 100)[..., 0].T
    want = c.want(0, causal=False)
    assert ((got.double() - want[2] - 2.0).abs() <= want[5] + 2.0 ** -22 * (want[2] + 2)).all()


def test_weights_sum_to_the_rows():
    c = Case(torch.float16, 64, 8, 2, 32, 9, [500, 20])
    w = torch.zeros(c.k_cache.shape[:3], device=DEV)
    c.run(weights=w)
    for b, n in enumerate(c.lens):
        got = read(w.unsqueeze(-1), c.table, b, n)[..., 0].sum(0)
        assert (got - 9 * 4).abs().max() < 1e-3


def test_pages_outside_the_cache_read_as_zeros():
    c = Case(torch.bfloat16, 64, 2, 1, 16, 1, [40])
    good = c.table.clone()
    c.table[0, 1] = 99
    c.k[0][16:32] = 0
    c.v[0][16:32] = 0
    out, lse = c.run()
    with pytest.raises(LlmxError):
        llmx_b200.device_status(0)
    check_attention(out[0], lse[0], None, c.want(0), c.dtype)
    c.table = good
    c.run()
    llmx_b200.device_status(0)


@pytest.mark.parametrize("algo", ["decode", "tcgen05"])
def test_pages_outside_the_cache_in_each_form(algo):
    c = Case(torch.float16, 128, 4, 2, 32, 30, [200, 90])
    c.table[0, 2], c.table[1, 0] = 2 ** 31 - 1, -5
    c.k[0][64:96] = 0
    c.v[0][64:96] = 0
    c.k[1][:32] = 0
    c.v[1][:32] = 0
    w = torch.zeros(c.k_cache.shape[:3], device=DEV)
    out, lse = c.run(algo=algo, weights=w)
    with pytest.raises(LlmxError):
        llmx_b200.device_status(0)
    for b in range(2):
        check_attention(out[b], lse[b], None, c.want(b), c.dtype)
    llmx_b200.device_status(0)


@pytest.mark.parametrize("algo", ["decode", "tcgen05"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_garbage_in_padded_rows_stays_there(d, algo):
    """Rows at or past q_lens hold NaN: they are written as 0 and reach nothing."""
    c = Case(torch.bfloat16, d, 6, 2, 32, 40, [300, 77, 40], q_lens=[33, 0, 7])
    for b, n in enumerate(c.q_lens):
        c.q[b, n:] = math.nan
    for weights in (False, True):
        out, _ = c.check(algo=algo, weights=weights)
        for b, n in enumerate(c.q_lens):
            assert not out[b, n:].any()


def test_lengths_past_the_bounds_are_clamped():
    c = Case(torch.float16, 64, 2, 1, 16, 4, [64, 10])
    out, lse = c.run()
    args = dict(kv_lens=torch.tensor([2 ** 40, 10], device=DEV), q_lens=torch.tensor([99, 2 ** 33], device=DEV))
    o2 = torch.empty_like(out)
    llmx_b200.paged_attention(o2, c.q.to(DEV), c.k_cache, c.v_cache, 64 ** -0.5, block_table=c.table.to(DEV), **args)
    assert torch.equal(o2, out)  # the table holds 64 tokens a sequence
    llmx_b200.paged_attention(o2, c.q.to(DEV), c.k_cache, c.v_cache, 64 ** -0.5, block_table=c.table.to(DEV),
                              kv_lens=ints([-3, 0]))
    assert not o2.any()


def test_strides_of_extents_of_one_do_not_matter():
    c = Case(torch.bfloat16, 64, 2, 1, 16, 1, [40], extra=0)
    q = c.q.to(DEV).as_strided((1, 1, 2, 64), (3, 5, 64, 1))
    kc, vc = (x.as_strided(x.shape, (x.stride(0), 7, 64, 1)) for x in (c.k_cache, c.v_cache))
    out = torch.empty_like(c.q, device=DEV)
    w = torch.zeros(c.k_cache.shape[:3], device=DEV)
    llmx_b200.paged_attention(out, q, kc, vc, 64 ** -0.5, kv_lens=ints([40]), block_table=c.table.to(DEV),
                              key_weights=w.as_strided(w.shape, (w.stride(0), 3, 1)))
    check_attention(out[0], None, None, c.want(0), c.dtype)
    assert abs(float(w.sum()) - 2) < 1e-4


def test_output_over_q_is_refused_with_weights():
    c = Case(torch.bfloat16, 64, 2, 1, 16, 3, [40])
    want, _ = c.run()
    q = c.q.to(DEV)
    args = dict(kv_lens=ints([40]), block_table=c.table.to(DEV))
    with pytest.raises(LlmxError):
        llmx_b200.paged_attention(q, q, c.k_cache, c.v_cache, 64 ** -0.5, key_weights=torch.zeros(c.k_cache.shape[:3], device=DEV), **args)
    llmx_b200.paged_attention(q, q, c.k_cache, c.v_cache, 64 ** -0.5, **args)
    assert torch.equal(q, want)


def test_calls_at_once_on_two_streams():
    cases = [Case(torch.bfloat16, 128, 8, 2, 64, q, [900, 333], seed=q) for q in (1, 9, 64)]
    want = [c.run()[0] for c in cases]
    args = [(c.q.to(DEV), c.k_cache, c.v_cache, ints(c.lens), c.table.to(DEV)) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [torch.empty_like(w) for w in want]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, (q, k, v, lens, table), o in zip(streams, args, outs):
            with torch.cuda.stream(s):
                llmx_b200.paged_attention(o, q, k, v, 128 ** -0.5, kv_lens=lens, block_table=table)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


@pytest.mark.parametrize("q_len,lens", [(1, [3000, 100]), (33, [500, 90]), (200, [700, 300])])
def test_same_bits_again_on_other_streams_and_in_graphs(q_len, lens):
    c = Case(torch.bfloat16, 128, 8, 2, 64, q_len, lens)
    w = torch.zeros(c.k_cache.shape[:3], device=DEV)
    out, lse = c.run(weights=w, decay=0.0)
    w0 = w.clone()
    q, kl, table = c.q.to(DEV), ints(c.lens), c.table.to(DEV)
    o2, w2 = torch.empty_like(out), torch.zeros_like(w)

    def call():
        llmx_b200.paged_attention(o2, q, c.k_cache, c.v_cache, 128 ** -0.5, kv_lens=kl, block_table=table, key_weights=w2,
                                  decay=0.0)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    s.synchronize()
    assert torch.equal(o2, out) and torch.equal(w2, w0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(3):
        o2.zero_(), w2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o2, out) and torch.equal(w2, w0)
    kl.copy_(ints([n // 2 + q_len // 2 for n in lens]))  # a replay follows the lengths
    graph.replay()
    c.lens = kl.tolist()
    c.k, c.v = [k[:n] for k, n in zip(c.k, c.lens)], [v[:n] for v, n in zip(c.v, c.lens)]
    assert torch.equal(c.run(max_kv_len=table.shape[1] * 64)[0], o2)


def test_without_workspace_runs_unsplit_and_weights_are_refused():
    c = Case(torch.bfloat16, 128, 4, 2, 16, 1, [700, 20])
    lib = _lib.load()
    p = _lib.AttnParams()
    lib.llmx_attn_params_init(ctypes.byref(p))
    keep = []
    cc = paged._cache_arg(c.k_cache, c.v_cache, 2, c.table.to(DEV), None, keep)
    q, out = c.q.to(DEV), torch.empty_like(c.q, device=DEV)
    lens = ints(c.lens)
    p.dtype, p.batch, p.n_heads, p.n_kv_heads, p.head_dim, p.max_q_len, p.max_kv_len = 2, 2, 4, 2, 128, 1, 704
    p.q, p.o, p.sm_scale, p.kv_lens = q.data_ptr(), out.data_ptr(), 128 ** -0.5, lens.data_ptr()
    lib.llmx_attn_set_contiguous_strides(ctypes.byref(p))
    assert lib.llmx_paged_attn_fwd(ctypes.byref(p), ctypes.byref(cc), 1.0, None) == 0
    torch.cuda.synchronize()
    for b in range(2):
        check_attention(out[b], None, None, c.want(b), c.dtype)
    w = torch.zeros(c.k_cache.shape[:3], device=DEV)
    cc.key_weights, cc.w_stride[0], cc.w_stride[1] = w.data_ptr(), w.stride(0), w.stride(1)
    assert lib.llmx_paged_attn_fwd(ctypes.byref(p), ctypes.byref(cc), 1.0, None) == 3


# ---------------------------------------------------------------- eviction
def evict_case(dtype, d, hkv, page, lens, seed=0, order="hnd", ties=True):
    gen = torch.Generator().manual_seed(seed)
    table, n_pages = table_of(lens, page, 1, gen)
    kc, vc = empty_cache(n_pages, hkv, page, d, dtype, order)
    w = torch.full((n_pages, hkv, page), math.nan, device=DEV)
    data = []
    for b, n in enumerate(lens):
        k, v = rows(gen, n, hkv, d, dtype), rows(gen, n, hkv, d, dtype)
        x = torch.exp(3 * torch.randn(n, hkv, generator=gen))
        if ties:
            x = torch.where(torch.rand(n, hkv, generator=gen) < 0.5, (x * 2).round() / 2, x)
        place(kc, table, b, k), place(vc, table, b, v)
        place(w.unsqueeze(-1), table, b, x.unsqueeze(-1))
        data.append((k, v, x))
    return kc, vc, w, table, data


def check_evicted(kc, vc, w, table, data, lens, kept, new_lens, budget, recent, sinks):
    for b, n in enumerate(lens):
        m = min(n, budget)
        assert int(new_lens[b]) == m
        k, v, x = data[b]
        gk, gv, gw = read(kc, table, b, m), read(vc, table, b, m), read(w.unsqueeze(-1), table, b, m)[..., 0]
        for h in range(k.shape[1]):
            want = opaged.kept(x[:, h], n, budget, recent, sinks)
            assert kept[b, h].tolist() == want + [-1] * (budget - m), (b, h)
            assert torch.equal(gk[:, h], k[want, h]) and torch.equal(gv[:, h], v[want, h])
            assert torch.equal(gw[:, h].nan_to_num(-5.0), x[want, h].nan_to_num(-5.0))


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dtype,d,hkv,page,lens,budget,recent,sinks,order", [
    (torch.bfloat16, 128, 2, 64, [1000, 100, 99, 0, 1, 101], 100, 20, 4, "hnd"),
    (torch.float16, 64, 3, 16, [77, 300], 33, 0, 0, "nhd"),
    (torch.float16, 256, 1, 48, [500], 499, 100, 3, "hnd"),
    (torch.bfloat16, 64, 1, 32, [5000, 4999], 1, 0, 0, "hnd"),
    (torch.bfloat16, 64, 2, 32, [700], 40, 40, 0, "hnd"),
    (torch.bfloat16, 64, 2, 32, [700], 40, 30, 10, "nhd"),
    (torch.float16, 64, 8, 16, [129] * 40, 64, 8, 1, "hnd"),
    (torch.float16, 64, 2, 128, [20000, 17000], 9000, 500, 4, "hnd"),
])
def test_evict(in_place, dtype, d, hkv, page, lens, budget, recent, sinks, order):
    for call in (llmx_b200.paged_evict, paged.paged_evict_ctypes):
        kc, vc, w, table, data = evict_case(dtype, d, hkv, page, lens, seed=len(lens) + d, order=order)
        out_table, extra = table, {}
        if not in_place:
            need = -(-min(budget, max(lens)) // page)
            first = kc.shape[0]
            kc, vc = (torch.cat([c, torch.full_like(c[:1], 7.0).expand(need * len(lens), -1, -1, -1)]) for c in (kc, vc))
            w = torch.cat([w, torch.full_like(w[:1], 7.0).expand(need * len(lens), -1, -1)])
            out_table = (first + torch.randperm(need * len(lens))).view(len(lens), need).int()
            extra["out_table"] = out_table.to(DEV)
            before = kc[:first].clone(), vc[:first].clone(), w[:first].clone()
        kept, new_lens = call(kc, vc, w, budget, kv_lens=ints(lens), block_table=table.to(DEV), recent=recent, sinks=sinks,
                              **extra)
        torch.cuda.synchronize()
        check_evicted(kc, vc, w, out_table, data, lens, kept.cpu(), new_lens.cpu(), budget, recent, sinks)
        if not in_place:
            for x, y in zip(before, (kc, vc, w)):
                assert torch.equal(x.nan_to_num(5.0), y[:first].nan_to_num(5.0))
    llmx_b200.device_status(0)


def test_evict_order_of_special_weights():
    lens = [300]
    kc, vc, w, table, data = evict_case(torch.float16, 64, 1, 16, lens, ties=False)
    x = data[0][2]
    x[:, 0] = 0.0
    x[10:20] = -0.0
    x[20] = math.inf
    x[30] = -math.inf
    x[40:45] = math.nan
    x[50] = -1.0
    x[60] = 1e-45
    place(w.unsqueeze(-1), table, 0, x.unsqueeze(-1))
    for budget in (1, 2, 3, 40, 293, 294, 295, 299):
        c = [t.clone() for t in (kc, vc, w)]
        kept, n = llmx_b200.paged_evict(*c, budget, kv_lens=ints(lens), block_table=table.to(DEV))
        check_evicted(*c, table, data, lens, kept.cpu(), n.cpu(), budget, 0, 0)


@pytest.mark.parametrize("n", [140000, 16385, 1024])
def test_evict_long_and_equal_weights(n):
    """Several CTAs a sequence (beyond 131072 candidates some are read again), and only ties."""
    kc, vc, w, table, data = evict_case(torch.float16, 64, 1, 64, [n], ties=True)
    kept, lens = llmx_b200.paged_evict(kc, vc, w, n // 3, kv_lens=ints([n]), block_table=table.to(DEV), recent=7, sinks=2)
    check_evicted(kc, vc, w, table, data, [n], kept.cpu(), lens.cpu(), n // 3, 7, 2)
    w.fill_(0.25)
    kept, lens = llmx_b200.paged_evict(kc, vc, w, 100, kv_lens=lens, block_table=table.to(DEV), recent=10)
    assert kept[0, 0].tolist() == list(range(90)) + list(range(n // 3 - 10, n // 3))


def test_evict_new_lens_may_be_kv_lens_and_graphs_replay():
    lens = [500, 90]
    kc, vc, w, table, data = evict_case(torch.bfloat16, 128, 2, 16, lens)
    kl, t = ints(lens), table.to(DEV)
    kept, out = llmx_b200.paged_evict(kc, vc, w, 64, kv_lens=kl, block_table=t, recent=4, new_lens=kl)
    assert out.data_ptr() == kl.data_ptr()
    check_evicted(kc, vc, w, table, data, lens, kept.cpu(), kl.cpu(), 64, 4, 0)
    kc2, vc2, w2, _, _ = evict_case(torch.bfloat16, 128, 2, 16, lens)
    saved = [x.clone() for x in (kc2, vc2, w2)]
    kl2, kept2 = ints(lens), torch.empty_like(kept)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        llmx_b200.paged_evict(kc2, vc2, w2, 64, kv_lens=kl2, block_table=t, recent=4, new_lens=kl2, kept=kept2)
    for _ in range(2):
        for x, y in zip((kc2, vc2, w2), saved):
            x.copy_(y)
        kl2.copy_(ints(lens))
        graph.replay()
        torch.cuda.synchronize()
        check_evicted(kc2, vc2, w2, table, data, lens, kept2.cpu(), kl2.cpu(), 64, 4, 0)


# ------------------------------------------------- a run of them together
@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_chunks_steps_eviction_steps(dtype):
    """A prompt in chunks, decode steps that note the weights, eviction, more steps."""
    gen = torch.Generator().manual_seed(11)
    B, H, Hkv, D, page = 2, 4, 2, 64, 16
    kc, vc = empty_cache(64, Hkv, page, D, dtype)
    weights = llmx_b200.paged_weights(kc)
    table = torch.randperm(64, generator=gen).view(B, 32).int()
    seqs = [[torch.zeros(0, Hkv, D, dtype=dtype)] * 2 for _ in range(B)]
    noted = [torch.zeros(Hkv, 0, dtype=torch.float64) for _ in range(B)]
    slack = [torch.zeros(Hkv, 0, dtype=torch.float64) for _ in range(B)]
    lens = [0, 0]

    def step(q_lens):
        S = max(q_lens)
        k, v = (torch.randn(B, S, Hkv, D, generator=gen).to(dtype) for _ in range(2))
        q = torch.randn(B, S, H, D, generator=gen).to(dtype)
        llmx_b200.paged_store(kc, vc, k.to(DEV), v.to(DEV), start=ints(lens), lens=ints(q_lens), block_table=table.to(DEV))
        for b in range(B):
            lens[b] += q_lens[b]
            seqs[b] = [torch.cat([x, y[b, :q_lens[b]]]) for x, y in zip(seqs[b], (k, v))]
        out = torch.empty_like(q, device=DEV)
        llmx_b200.paged_attention(out, q.to(DEV), kc, vc, D ** -0.5, kv_lens=ints(lens), q_lens=ints(q_lens),
                                  block_table=table.to(DEV), key_weights=weights)
        for b in range(B):
            want = opaged.attention(q[b], *seqs[b], q_lens[b], lens[b], sm_scale=D ** -0.5)
            check_attention(out[b], None, None, want, dtype)
            pad = (0, q_lens[b])
            noted[b] = torch.nn.functional.pad(noted[b], pad) + want[2]
            slack[b] = torch.nn.functional.pad(slack[b], pad) + want[5] + 2.0 ** -23 * noted[b]
            got = read(weights.unsqueeze(-1), table, b, lens[b])[..., 0].T.double()
            assert ((got - noted[b]).abs() <= slack[b]).all()

    for q_lens in ([100, 37], [90, 150], [1, 1], [1, 1], [3, 2]):
        step(q_lens)
    old = list(lens)
    held = [read(weights.unsqueeze(-1), table, b, n)[..., 0] for b, n in enumerate(lens)]
    kept, new = llmx_b200.paged_evict(kc, vc, weights, 64, kv_lens=ints(lens), block_table=table.to(DEV), recent=16, sinks=2)
    lens = new.tolist()
    for b in range(B):
        pick = [opaged.kept(held[b][:, h], old[b], 64, 16, 2) for h in range(Hkv)]
        assert kept[b].tolist() == pick
        seqs[b] = [torch.stack([x[p, h] for h, p in enumerate(pick)], 1) for x in seqs[b]]
        noted[b] = torch.stack([noted[b][h, p] for h, p in enumerate(pick)])
        slack[b] = torch.stack([slack[b][h, p] for h, p in enumerate(pick)])
    for q_lens in ([1, 1], [5, 1], [80, 3]):
        step(q_lens)
    llmx_b200.device_status(0)
