"""The 4-bit key/value cache on the GPU against its oracle in 64 bits.

The store and the load are held to the oracle bit by bit.  The attention is
held, element by element, to the oracle's bound (oracle/kv4.py: the fp16
rounding of p s, fp32 sums and scores) plus half a step of the output's type.
"""
import ctypes
import math

import pytest
import torch

import llmx_b200
from gpu_helpers import HALF_MAX_ABS, HALF_MEAN_REL, needs_cuda
from llmx_b200 import LlmxError, _lib, kv4
from oracle import kv4 as okv4

pytestmark = [pytest.mark.gpu, needs_cuda]

DEV = "cuda"


def table_of(lens_max, page, extra, gen):
    """A block table of shuffled pages for sequences of up to lens_max tokens."""
    need = [max(1, -(-n // page)) for n in lens_max]
    order = torch.randperm(sum(need) + extra, generator=gen).int()
    table = torch.full((len(need), max(need)), -7, dtype=torch.int32)  # entries behind a sequence are never read
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(need) + extra


def garbage(n_pages, hkv, d, page):
    """A cache whose every byte is 0xff: all its steps and minima are NaN."""
    c = llmx_b200.kv4_empty(n_pages, hkv, d, page, device=DEV)
    c.fill_(255)
    return c


def rows(gen, n, hkv, d, dtype, offset=0.0):
    return (torch.randn(n, hkv, d, generator=gen) + offset).to(dtype)


def filled(gen, lens, hkv, d, dtype, page, offset=0.0):
    """(cache, table, k, v): sequences of the given lengths stored by kv4_store into a garbage cache."""
    S = max(max(lens), 1)
    table, n_pages = table_of(lens, page, 2, gen)
    cache = garbage(n_pages, hkv, d, page)
    k = torch.stack([rows(gen, S, hkv, d, dtype, offset) for _ in lens])
    v = torch.stack([rows(gen, S, hkv, d, dtype) for _ in lens])
    llmx_b200.kv4_store(cache, k.to(DEV), v.to(DEV), lens=torch.tensor(lens, device=DEV, dtype=torch.int32),
                        block_table=table.to(DEV))
    return cache, table.to(DEV), k, v


def check(out, lse, q, k, v, q_lens, kv_lens, dtype, *, sm_scale, causal=True, window=-1, cap=0.0, slopes=None, what=""):
    out, lse = out.double().cpu(), None if lse is None else lse.double().cpu()
    half_step = torch.finfo(dtype).eps / 2
    for b in range(q.shape[0]):
        o, le, bound, le_bound = okv4.attention(q[b], k[b], v[b], q_lens[b], kv_lens[b], sm_scale=sm_scale, causal=causal,
                                      window=window, cap=cap, slopes=slopes)
        # The second term is the output's own rounding (below the normal range: half its smallest number).
        room = bound * (1 + 2 ** -10) + (o.abs() + bound) * half_step + torch.finfo(dtype).smallest_normal * half_step
        bad = ~((out[b] - o).abs() <= room)
        assert not bad.any(), (f"{what} sequence {b}: {int(bad.sum())} of {bad.numel()} off, worst "
                               f"{float(((out[b] - o).abs() / room).nan_to_num(1e9).max()):.3g} of the bound")
        if lse is not None:
            empty = le == -math.inf
            assert torch.equal(lse[b] == -math.inf, empty), f"{what}: empty rows"
            assert ((lse[b] - le).abs()[~empty] <= le_bound[~empty]).all(), f"{what}: lse"


def expect_tile_bytes(table, starts, lens, k, v, hkv, d, page):
    """{(page id, kv head, tile): uint8 tile, written mask} the oracle writes."""
    tiles = {}
    for b in range(k.shape[0]):
        for i in range(lens[b]):
            pos = starts[b] + i
            pid = int(table[b, pos // page])
            for h in range(hkv):
                key = (pid, h, pos % page // 16)
                if key not in tiles:
                    tiles[key] = torch.full((18 * d,), 255, dtype=torch.uint8)
                okv4.write_token(tiles[key], pos % 16, k[b, i, h], v[b, i, h])
    return tiles


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,hkv,page,starts,lens,S", [
    (64, 1, 16, [0], [1], 1),
    (128, 2, 64, [0, 15, 63, 40], [33, 2, 1, 0], 33),
    (256, 1, 32, [5, 31], [17, 20], 20),
    (64, 3, 48, [47, 16, 1], [3, 16, 47], 47),
    (128, 1, 128, [7], [150], 150),
])
def test_store_writes_exactly_the_oracles_bytes(dtype, d, hkv, page, starts, lens, S):
    gen = torch.Generator().manual_seed(d + S)
    table, n_pages = table_of([s + n for s, n in zip(starts, lens)], page, 2, gen)
    cache = garbage(n_pages, hkv, d, page)
    k = torch.stack([rows(gen, S, hkv, d, dtype, 0.5) for _ in lens])
    v = torch.stack([rows(gen, S, hkv, d, dtype) * 3 for _ in lens])
    k[0, 0, 0, :64] = 2.5  # a constant group
    if S > 1:
        k[0, 1, 0, 3] = 1e4  # an outlier
        v[0, 1, 0, :] = 0.0
    llmx_b200.kv4_store(cache, k.to(DEV), v.to(DEV), start=torch.tensor(starts, device=DEV),
                        lens=torch.tensor(lens, device=DEV), block_table=table.to(DEV))
    llmx_b200.device_status(0)
    got = cache.cpu()
    want = torch.full_like(got, 255)
    for (pid, h, t), tile in expect_tile_bytes(table, starts, lens, k, v, hkv, d, page).items():
        want[pid, h, t] = tile
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,hkv,page,B,S", [(64, 2, 16, 3, 37), (128, 8, 64, 2, 130), (256, 1, 32, 1, 1), (128, 3, 80, 4, 257)])
def test_load_returns_the_stored_values(dtype, d, hkv, page, B, S):
    gen = torch.Generator().manual_seed(S)
    lens = [max(0, S - 11 * b) for b in range(B)]
    starts = [(5 * b) % 19 for b in range(B)]
    table, n_pages = table_of([s + n for s, n in zip(starts, lens)], page, 0, gen)
    cache = garbage(n_pages, hkv, d, page)
    k = torch.stack([rows(gen, S, hkv, d, dtype, 1.0) for _ in lens])
    v = torch.stack([rows(gen, S, hkv, d, dtype) for _ in lens])
    kw = dict(start=torch.tensor(starts, device=DEV), lens=torch.tensor(lens, device=DEV), block_table=table.to(DEV))
    llmx_b200.kv4_store(cache, k.to(DEV), v.to(DEV), **kw)
    ko, vo = torch.full_like(k, 9.0, device=DEV), torch.full_like(v, 9.0, device=DEV)
    llmx_b200.kv4_load(cache, ko, vo, **kw)
    for b in range(B):
        for got, x in ((ko, k), (vo, v)):
            want = okv4.values(x[b])[1]
            want[lens[b]:] = 0
            assert torch.equal(got[b].cpu(), want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_non_finite_inputs_poison_their_group_only(bad, dtype):
    gen = torch.Generator().manual_seed(3)
    k, v = rows(gen, 20, 2, 128, dtype)[None], rows(gen, 20, 2, 128, dtype)[None]
    k[0, 7, 1, 70], v[0, 9, 0, 3] = bad, bad
    cache = garbage(2, 2, 128, 16)
    llmx_b200.kv4_store(cache, k.to(DEV), v.to(DEV))
    ko, vo = torch.empty_like(k, device=DEV), torch.empty_like(v, device=DEV)
    llmx_b200.kv4_load(cache, ko, vo)
    wk, wv = okv4.values(k)[1], okv4.values(v)[1]
    assert wk[0, 7, 1, 64:].isnan().all() and wv[0, 9, 0, :64].isnan().all()
    for got, want in ((ko, wk), (vo, wv)):
        assert torch.equal(got.cpu().nan_to_num(-77.0), want.nan_to_num(-77.0))
    # A row that sees the poisoned tokens is NaN where the formula says so, one that does not is not:
    # query row i of 20 sees tokens 0 .. i.
    q = torch.randn(1, 20, 2, 128, generator=gen).to(dtype)
    out = torch.empty_like(q, device=DEV)
    llmx_b200.kv4_attention(out, q.to(DEV), cache, 128 ** -0.5, max_kv_len=20)
    out = out.cpu()
    assert out[0, :7].isfinite().all() and out[0, 7:, 1].isnan().all()
    assert out[0, :9, 0].isfinite().all() and out[0, 9:, 0, :64].isnan().all() and out[0, 9:, 0, 64:].isfinite().all()


def test_extreme_values():
    """Ranges near the ends of bf16, subnormal ones, and offsets far above the range."""
    dtype = torch.bfloat16
    gen = torch.Generator().manual_seed(5)
    base = torch.randn(1, 16, 1, 64, generator=gen)
    scales = torch.tensor([1e37, 1e30, 1e-30, 1e-37, 1e-39, 1.0, 1e4, 1e-4] * 2)[None, :, None, None]
    k = (base * scales).to(dtype)
    v = (base + 1000.0).to(dtype)
    cache = garbage(1, 1, 64, 16)
    llmx_b200.kv4_store(cache, k.to(DEV), v.to(DEV))
    ko, vo = torch.empty_like(k, device=DEV), torch.empty_like(v, device=DEV)
    llmx_b200.kv4_load(cache, ko, vo)
    assert torch.equal(ko.cpu(), okv4.values(k)[1]) and torch.equal(vo.cpu(), okv4.values(v)[1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_strided_rows_and_caches(dtype):
    """Rows cut out of a fused QKV tensor, unaligned rows, broadcast rows, a cache that is one layer of a larger one."""
    gen = torch.Generator().manual_seed(11)
    B, S, hkv, d = 2, 21, 2, 128
    layers = torch.full((4, 3, hkv, 2, 18 * d), 255, dtype=torch.uint8, device=DEV)  # [pages, layers, ...]
    cache = layers[:, 1]
    fused = torch.randn(B, S, 3 * hkv, d + 1, generator=gen).to(dtype).to(DEV)
    for k, v in ((fused[:, :, :hkv, :d], fused[:, :, hkv:2 * hkv, :d]), (fused[:, :, :hkv, 1:], fused[:, :, hkv:2 * hkv, 1:]),
                 (fused[:1, :, :hkv, :d].expand(B, -1, -1, -1), fused[:, :1, :hkv, :d].expand(-1, S, -1, -1)),
                 (fused[:, :, :hkv, :d].transpose(1, 2).contiguous().transpose(1, 2), fused[:, :, :hkv, :d].flip(-1))):
        layers.fill_(255)
        llmx_b200.kv4_store(cache, k, v)
        out = torch.full((B, S, 2 * hkv, d + 8), 5.0, dtype=dtype, device=DEV)
        ko, vo = out[:, :, :hkv, 3:d + 3], out[:, :, hkv:, 8:]  # one side unaligned
        llmx_b200.kv4_load(cache, ko, vo)
        assert torch.equal(ko.cpu(), okv4.values(k.cpu())[1]) and torch.equal(vo.cpu(), okv4.values(v.cpu())[1])
        assert (out[:, :, :hkv, :3] == 5).all() and (out[:, :, :hkv, d + 3:] == 5).all() and (out[:, :, hkv:, :8] == 5).all()
        assert (layers[:, 0] == 255).all() and (layers[:, 2] == 255).all()


def test_sizes_of_zero_do_nothing():
    cache = garbage(2, 2, 64, 16)
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64)):
        k = torch.empty(shape, dtype=torch.float16, device=DEV)
        llmx_b200.kv4_store(cache, k, k)
        llmx_b200.kv4_load(cache, k, k)
    q = torch.empty(2, 0, 4, 64, dtype=torch.float16, device=DEV)
    llmx_b200.kv4_attention(q.clone(), q, cache, 1.0)
    assert (cache == 255).all()


ATTENTION_CASES = [
    # d, heads, kv_heads, q_len, kv_lens, page
    (64, 1, 1, 1, [1], 16),
    (64, 8, 2, 1, [0, 1, 15, 16, 17, 77], 16),
    (128, 4, 4, 1, [64, 65, 300], 64),
    (128, 8, 1, 1, [1000, 3], 32),
    (128, 12, 4, 3, [5, 100, 2, 0], 48),
    (128, 16, 2, 5, [257, 31], 128),
    (256, 4, 2, 1, [130, 16], 64),
    (256, 7, 1, 2, [200, 1], 16),
    (64, 6, 2, 13, [100, 13, 7], 32),
    (128, 32, 1, 1, [513], 64),
    (64, 40, 1, 1, [90, 33], 16),
    (128, 2, 2, 40, [70, 40], 64),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,H,hkv,sq,lens,page", ATTENTION_CASES)
def test_attention_against_the_oracle(dtype, d, H, hkv, sq, lens, page):
    gen = torch.Generator().manual_seed(d + H + sq)
    cache, table, k, v = filled(gen, lens, hkv, d, dtype, page, offset=0.3)
    B = len(lens)
    q = torch.randn(B, sq, H, d, generator=gen).to(dtype)
    slopes = torch.pow(2.0, -8.0 * torch.arange(1, H + 1) / H).float()
    q_lens = [1 + (sq + b) % sq for b in range(B)]
    kv_lens = torch.tensor(lens, device=DEV)
    scale = d ** -0.5
    for opts in (dict(), dict(window=9), dict(cap=3.0), dict(slopes=slopes), dict(causal=False),
                 dict(causal=False, window=4, slopes=slopes, cap=20.0), dict(window=0)):
        out = torch.full_like(q, 7.0, device=DEV)
        lse = torch.full((B, H, sq), 7.0, device=DEV)
        ragged = "window" in opts
        llmx_b200.kv4_attention(out, q.to(DEV), cache, scale, opts.get("window", -1), opts.get("cap", 0.0),
                                kv_lens=kv_lens, block_table=table, causal=opts.get("causal", True), lse=lse, algo="decode",
                                q_lens=torch.tensor(q_lens, device=DEV) if ragged else None,
                                alibi_slopes=None if "slopes" not in opts else slopes.to(DEV))
        check(out, lse, q, k, v, q_lens if ragged else [sq] * B, lens, dtype, sm_scale=scale, what=str(opts), **opts)
    llmx_b200.device_status(0)


@pytest.mark.parametrize("dtype,d,H,hkv,n,page", [(torch.bfloat16, 128, 8, 2, 20000, 64), (torch.float16, 64, 4, 4, 9001, 16),
                                                  (torch.float16, 256, 2, 1, 5003, 128)])
def test_long_sequences_split_and_unsplit(dtype, d, H, hkv, n, page):
    """Many splits against the oracle, and the same request without a workspace (one split)."""
    gen = torch.Generator().manual_seed(n)
    lens = [n, 17]
    cache, table, k, v = filled(gen, lens, hkv, d, dtype, page)
    q = (2 * torch.randn(2, 1, H, d, generator=gen)).to(dtype)
    qd = q.to(DEV)
    for window in (-1, n // 3):
        out, lse = torch.empty_like(qd), torch.empty(2, H, 1, device=DEV)
        llmx_b200.kv4_attention(out, qd, cache, d ** -0.5, window, kv_lens=torch.tensor(lens, device=DEV), block_table=table, lse=lse)
        check(out, lse, q, k, v, [1, 1], lens, dtype, sm_scale=d ** -0.5, window=window, what=f"split, window {window}")
    keep = []
    c = kv4._cache_arg(cache, 2, dtype, d, table, keep)
    p = _lib.AttnParams()
    lib = _lib.load()
    lib.llmx_attn_params_init(ctypes.byref(p))
    one = torch.empty_like(qd)
    kv = torch.tensor(lens, device=DEV, dtype=torch.int32)
    p.dtype, p.batch, p.n_heads, p.n_kv_heads, p.head_dim, p.max_q_len = c.dtype, 2, H, hkv, d, 1
    p.max_kv_len, p.q, p.o, p.kv_lens, p.sm_scale = c.max_pages * page, qd.data_ptr(), one.data_ptr(), kv.data_ptr(), d ** -0.5
    lib.llmx_attn_set_contiguous_strides(ctypes.byref(p))
    _lib.check(lib.llmx_kv4_attn_fwd(ctypes.byref(p), ctypes.byref(c), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    torch.cuda.synchronize()
    check(one, None, q, k, v, [1, 1], lens, dtype, sm_scale=d ** -0.5, what="one split")


@pytest.mark.parametrize("d,H,hkv,sq", [(128, 8, 2, 5), (64, 4, 4, 2), (256, 4, 2, 3), (128, 8, 8, 1), (64, 32, 2, 3)])
def test_rows_and_sequences_that_are_empty(d, H, hkv, sq):
    """Query rows past their length next to long caches, sequences with no row, with no key, with neither."""
    dtype = torch.bfloat16
    gen = torch.Generator().manual_seed(sq)
    lens, q_lens = [900, 0, 333, 2000, 70, 0, 1], [1, sq, 0, sq, max(sq - 1, 1), 0, sq]
    cache, table, k, v = filled(gen, lens, hkv, d, dtype, 32)
    q = torch.randn(len(lens), sq, H, d, generator=gen).to(dtype)
    for causal in (True, False):
        out, lse = torch.full_like(q, 7.0, device=DEV), torch.full((len(lens), H, sq), 7.0, device=DEV)
        llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, kv_lens=torch.tensor(lens, device=DEV), block_table=table,
                                q_lens=torch.tensor(q_lens, device=DEV), lse=lse, causal=causal)
        check(out, lse, q, k, v, q_lens, lens, dtype, sm_scale=d ** -0.5, causal=causal, what=f"causal {causal}")


def test_batch_of_many_sequences():
    """More sequences than one launch takes, most of them short."""
    dtype, d, H, hkv = torch.float16, 64, 2, 1
    gen = torch.Generator().manual_seed(77)
    lens = torch.randint(0, 40, (1201,), generator=gen).tolist()
    lens[600], lens[1200] = 700, 300
    cache, table, k, v = filled(gen, lens, hkv, d, dtype, 16)
    q = torch.randn(len(lens), 1, H, d, generator=gen).to(dtype)
    out, lse = torch.full_like(q, 7.0, device=DEV), torch.full((len(lens), H, 1), 7.0, device=DEV)
    llmx_b200.kv4_attention(out, q.to(DEV), cache, 0.125, kv_lens=torch.tensor(lens, device=DEV), block_table=table, lse=lse)
    check(out, lse, q, k, v, [1] * len(lens), lens, dtype, sm_scale=0.125)


@pytest.mark.parametrize("d,group,sq,opts", [(128, 1, 1, "alibi"), (64, 1, 2, ""), (128, 4, 1, ""), (128, 3, 2, "window"), (256, 2, 1, ""),
                                             (64, 7, 1, "alibi")])
def test_more_units_than_the_gpu_holds(d, group, sq, opts):
    """Units enough that every warp has shares of its own: whole units, units shared by two warps, empty sequences."""
    dtype, hkv, B = torch.bfloat16, 4, 153
    gen = torch.Generator().manual_seed(d + group)
    lens = torch.randint(0, 150, (B,), generator=gen).tolist()
    lens[3], lens[77], lens[B - 1] = 1100, 0, 400
    cache, table, k, v = filled(gen, lens, hkv, d, dtype, 32)
    H = hkv * group
    q = torch.randn(B, sq, H, d, generator=gen).to(dtype)
    slopes = torch.pow(2.0, -8.0 * torch.arange(1, H + 1) / H).float() if opts == "alibi" else None
    window = 40 if opts == "window" else -1
    out, lse = torch.full_like(q, 7.0, device=DEV), torch.full((B, H, sq), 7.0, device=DEV)
    call = dict(kv_lens=torch.tensor(lens, device=DEV), block_table=table, algo="decode",
                alibi_slopes=None if slopes is None else slopes.to(DEV))
    llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, window, lse=lse, **call)
    check(out, lse, q, k, v, [sq] * B, lens, dtype, sm_scale=d ** -0.5, window=window, slopes=slopes)
    again = torch.empty_like(out)
    llmx_b200.kv4_attention(again, q.to(DEV), cache, d ** -0.5, window, **call)
    assert torch.equal(again, out)
    llmx_b200.device_status(0)


def test_non_finite_queries_poison_their_row_only():
    dtype, d = torch.bfloat16, 128
    gen = torch.Generator().manual_seed(6)
    cache, table, k, v = filled(gen, [300], 2, d, dtype, 64)
    q = torch.randn(1, 1, 8, d, generator=gen).to(dtype)
    ref = torch.empty_like(q, device=DEV)
    args = dict(kv_lens=torch.tensor([300], device=DEV), block_table=table)
    llmx_b200.kv4_attention(ref, q.to(DEV), cache, 0.1, **args)
    q[0, 0, 1, 5], q[0, 0, 2, 77], q[0, 0, 6, 0] = float("inf"), float("nan"), float("-inf")
    out = torch.empty_like(q, device=DEV)
    llmx_b200.kv4_attention(out, q.to(DEV), cache, 0.1, **args)
    hit = [1, 2, 6]
    assert out[0, 0, hit].isnan().all()
    rest = [h for h in range(8) if h not in hit]
    assert torch.equal(out[0, 0, rest], ref[0, 0, rest])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,hkv,B,S,page", [(64, 30, 3, 190, 48), (128, 40, 3, 150, 64), (256, 33, 2, 270, 16)])
def test_whole_tiles_and_single_rows_write_the_same(dtype, d, hkv, B, S, page):
    """Rows enough for the kernels that take a tile a warp, against the oracle and against the same rows stored a few at a time."""
    gen = torch.Generator().manual_seed(S)
    starts, lens = [3 + 9 * b for b in range(B)], [S - 21 * b for b in range(B)]
    table, n_pages = table_of([s + n for s, n in zip(starts, lens)], page, 1, gen)
    k, v = (torch.randn(B, S, hkv, d, generator=gen).to(dtype) for _ in range(2))
    k[0, :40] *= torch.pow(10.0, torch.linspace(-7, 3, 40))[:, None, None].to(dtype)
    v[0, 50:60] = 1.25  # steps of 0
    k[1, 20, 3, 7], v[1, 33, 2, 5], v[1, 34, 1, 1] = float("nan"), float("inf"), float("-inf")
    if dtype == torch.bfloat16:
        v[0, 60] *= 1e36
        v[0, 61] *= 1e-38
    st, ln = torch.tensor(starts, device=DEV), torch.tensor(lens, device=DEV)
    kw = dict(block_table=table.to(DEV))
    big, small = garbage(n_pages, hkv, d, page), garbage(n_pages, hkv, d, page)
    kd, vd = k.to(DEV), v.to(DEV)
    llmx_b200.kv4_store(big, kd, vd, start=st, lens=ln, **kw)
    for i in range(0, S, 13):
        llmx_b200.kv4_store(small, kd[:, i:i + 13], vd[:, i:i + 13], start=st + i, lens=(ln - i).clamp(0, 13), **kw)
    assert torch.equal(big, small)
    ko, vo = torch.full_like(kd, 9.0), torch.full_like(vd, 9.0)
    llmx_b200.kv4_load(big, ko, vo, start=st, lens=ln, **kw)
    for b in range(B):
        for got, x in ((ko, k), (vo, v)):
            want = okv4.values(x[b])[1]
            want[lens[b]:] = 0
            assert torch.equal(got[b].cpu().nan_to_num(-77.0), want.nan_to_num(-77.0))
    # Unaligned rows take the same kernels element by element.
    wide = torch.zeros(B, S, hkv, d + 1, dtype=dtype, device=DEV)
    wide[..., 1:] = kd
    other = garbage(n_pages, hkv, d, page)
    llmx_b200.kv4_store(other, wide[..., 1:], vd, start=st, lens=ln, **kw)
    assert torch.equal(big, other)
    wide.fill_(5.0)
    llmx_b200.kv4_load(big, wide[..., 1:], vo, start=st, lens=ln, **kw)
    assert torch.equal(wide[..., 1:].nan_to_num(-77.0), ko.nan_to_num(-77.0)) and (wide[..., 0] == 5).all()
    llmx_b200.device_status(0)


def test_scores_that_move_the_maximum():
    """Rising and falling scores, a weight that underflows everything before it, steps of very different sizes."""
    dtype, d, n = torch.bfloat16, 128, 700
    gen = torch.Generator().manual_seed(2)
    k, v = rows(gen, n, 1, d, dtype), rows(gen, n, 1, d, dtype)
    ramp = torch.linspace(0.0, 8.0, n)[:, None, None]
    size = torch.pow(10.0, torch.linspace(-6, 6, n))[torch.randperm(n, generator=gen)][:, None, None]
    for kk, vv in (((k * ramp).to(dtype), v), ((k * ramp.flip(0)).to(dtype), v), (k, (v * size).to(dtype)),
                   ((k * ramp).to(dtype), (v * ramp * 1e-3).to(dtype))):
        cache = garbage(-(-n // 64), 1, d, 64)
        llmx_b200.kv4_store(cache, kk[None].to(DEV), vv[None].to(DEV))
        q = (torch.randn(1, 1, 8, d, generator=gen) * torch.tensor([1e-20, 1e-3, 1, 1, 2, 4, 8, 30])[None, None, :, None]).to(dtype)
        out, lse = torch.empty_like(q, device=DEV), torch.empty(1, 8, 1, device=DEV)
        llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, max_kv_len=n, lse=lse)
        check(out, None, q, kk[None], vv[None], [1], [n], dtype, sm_scale=d ** -0.5, what="moving maxima")


def test_q_and_output_views_and_lse():
    """Unaligned q, outputs with their own strides: only the output's elements change."""
    dtype, d, H, hkv = torch.float16, 64, 6, 2
    gen = torch.Generator().manual_seed(8)
    lens = [50, 20]
    cache, table, k, v = filled(gen, lens, hkv, d, dtype, 16)
    base = torch.randn(2, 4, H, 3 * d + 1, generator=gen).to(dtype)
    room = torch.full((2, 4, H + 1, 2 * d), 3.0, dtype=dtype, device=DEV)
    for q in (base[..., 1:d + 1], base[..., :d], base[:, :, :, 2 * d:3 * d].transpose(1, 2).contiguous().transpose(1, 2),
              base[..., :2 * d:2]):
        room.fill_(3.0)
        out = room[:, :, 1:, 5:d + 5]
        qd = torch.empty_strided(q.shape, q.stride(), dtype=dtype, device=DEV).copy_(q) if q.stride(-1) == 1 else q.to(DEV)
        llmx_b200.kv4_attention(out, qd, cache, 0.2, kv_lens=torch.tensor(lens, device=DEV), block_table=table)
        check(out, None, q, k, v, [4, 4], lens, dtype, sm_scale=0.2)
        assert (room[:, :, 0] == 3).all() and (room[..., :5] == 3).all() and (room[..., d + 5:] == 3).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,H,hkv,sq,lens", [(128, 8, 2, 200, [1000, 300, 200]), (64, 4, 4, 130, [513, 130]), (256, 2, 1, 260, [700])])
def test_expanded_form(dtype, d, H, hkv, sq, lens):
    """Long query blocks through the expanded form, held like the framework's
    prefill: against attention over the values that kv4_load returns."""
    import oracle

    gen = torch.Generator().manual_seed(sq)
    cache, table, k, v = filled(gen, lens, hkv, d, dtype, 64)
    B = len(lens)
    q = torch.randn(B, sq, H, d, generator=gen).to(dtype)
    ref = oracle.attention_ref_padded(q.float(), okv4.values(k)[1].float(), okv4.values(v)[1].float(), kv_lens=lens,
                                      sm_scale=d ** -0.5)
    for algo in ("auto", "tcgen05"):
        # A workspace full of NaN must not reach the output.
        poison = torch.full((64 << 20,), float("nan"), device=DEV)
        del poison
        out = torch.empty_like(q, device=DEV)
        llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, kv_lens=torch.tensor(lens, device=DEV), block_table=table, algo=algo)
        err = (out.float().cpu() - ref).abs()
        assert err.max() <= HALF_MAX_ABS and err.mean() <= HALF_MEAN_REL * ref.abs().mean(), (algo, float(err.max()))
    llmx_b200.device_status(0)


def test_generation_run():
    """A prompt stored in two chunks, then decode steps of one token: store, then attend, as a server does."""
    dtype, d, H, hkv, page = torch.bfloat16, 128, 8, 2, 16
    gen = torch.Generator().manual_seed(21)
    lens = [37, 5, 16]
    B, steps = len(lens), 6
    table, n_pages = table_of([n + steps for n in lens], page, 0, gen)
    table = table.to(DEV)
    cache = garbage(n_pages, hkv, d, page)
    S = max(lens) + steps
    k = torch.stack([rows(gen, S, hkv, d, dtype) for _ in lens])
    v = torch.stack([rows(gen, S, hkv, d, dtype) for _ in lens])
    first = torch.tensor([n // 2 for n in lens], device=DEV)
    llmx_b200.kv4_store(cache, k.to(DEV), v.to(DEV), lens=first, block_table=table)
    rest = torch.zeros(B, S, hkv, d, dtype=dtype)
    rest_v = torch.zeros_like(rest)
    for b, n in enumerate(lens):
        rest[b, :n - n // 2], rest_v[b, :n - n // 2] = k[b, n // 2:n], v[b, n // 2:n]
    llmx_b200.kv4_store(cache, rest.to(DEV), rest_v.to(DEV), start=first, lens=torch.tensor([n - n // 2 for n in lens], device=DEV),
                        block_table=table)
    pos = torch.tensor(lens, device=DEV, dtype=torch.int32)
    for step in range(steps):
        at = [n + step for n in lens]
        kt = torch.stack([k[b, at[b]] for b in range(B)])[:, None]
        vt = torch.stack([v[b, at[b]] for b in range(B)])[:, None]
        llmx_b200.kv4_store(cache, kt.to(DEV), vt.to(DEV), start=pos, block_table=table)
        pos += 1
        q = torch.randn(B, 1, H, d, generator=gen).to(dtype)
        out = torch.empty_like(q, device=DEV)
        llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, kv_lens=pos, block_table=table)
        check(out, None, q, k, v, [1] * B, [n + 1 for n in at], dtype, sm_scale=d ** -0.5, what=f"step {step}")
    # The prefill over the expanded cache agrees with the attention over it.
    ko, vo = torch.empty_like(k, device=DEV), torch.empty_like(v, device=DEV)
    llmx_b200.kv4_load(cache, ko, vo, lens=pos, block_table=table)
    dense = llmx_b200.attention(q.to(DEV), ko, vo, kv_lens=pos)
    assert (dense.float() - out.float()).abs().max() <= HALF_MAX_ABS


def test_bad_pages_and_positions_are_skipped_and_reported():
    """Entries outside the cache are not followed (both kernels bound them before any access)."""
    dtype, d, hkv, page = torch.float16, 64, 1, 16
    gen = torch.Generator().manual_seed(4)
    cache = garbage(3, hkv, d, page)
    k, v = rows(gen, 48, hkv, d, dtype)[None].to(DEV), rows(gen, 48, hkv, d, dtype)[None].to(DEV)
    table = torch.tensor([[2, 3, 0]], dtype=torch.int32, device=DEV)  # page 3 does not exist
    llmx_b200.kv4_store(cache, k, v, block_table=table)
    with pytest.raises(LlmxError, match="page"):
        llmx_b200.device_status(0)
    llmx_b200.device_status(0)  # cleared
    assert (cache[1] == 255).all() and not (cache[0] == 255).all() and not (cache[2] == 255).all()
    ko, vo = torch.full_like(k, 4.0), torch.full_like(v, 4.0)
    table[0, 1] = -1
    llmx_b200.kv4_load(cache, ko, vo, block_table=table)
    with pytest.raises(LlmxError, match="page"):
        llmx_b200.device_status(0)
    want = okv4.values(k.cpu())[1]
    want[:, 16:32] = 0
    assert torch.equal(ko.cpu(), want)
    # The attention sees the other 32 tokens only.
    q = torch.randn(1, 1, 2, d, generator=gen).to(dtype)
    out = torch.empty_like(q, device=DEV)
    llmx_b200.kv4_attention(out, q.to(DEV), cache, 0.125, block_table=table)
    with pytest.raises(LlmxError, match="page"):
        llmx_b200.device_status(0)
    kept = torch.cat([torch.arange(16), torch.arange(32, 48)])
    check(out, None, q, k.cpu()[:, kept], v.cpu()[:, kept], [1], [32], dtype, sm_scale=0.125)
    # Positions outside the table: before its begin and behind its end.
    cache.fill_(255)
    table[0, 1] = 1
    for start, live in ((-5, range(5, 48)), (40, range(0, 8)), (2 ** 31 - 1, range(0))):
        llmx_b200.kv4_store(cache, k, v, start=torch.tensor([start], device=DEV, dtype=torch.int32), block_table=table)
        with pytest.raises(LlmxError, match="position"):
            llmx_b200.device_status(0)
        if len(live):
            n = len(live)
            ko, vo = torch.empty_like(k[:, :n]), torch.empty_like(v[:, :n])
            llmx_b200.kv4_load(cache, ko, vo, start=torch.tensor([start + live[0]], device=DEV, dtype=torch.int32), block_table=table)
            assert torch.equal(ko.cpu(), okv4.values(k.cpu()[:, live[0]:live[0] + n])[1])
        llmx_b200.device_status(0)


def test_python_refusals():
    cache = garbage(4, 2, 128, 16)
    q = torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(2, 3, 2, 128, dtype=torch.bfloat16, device=DEV)
    table = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    for call in (llmx_b200.kv4_attention, kv4.kv4_attention_ctypes):
        for args, kw, match in [
            ((q[0], q[0], cache, 1.0), {}, "batch"), ((q, q.half(), cache, 1.0), {}, "dtype"),
            ((q.float(), q.float(), cache, 1.0), {}, "float16 and bfloat16"), ((q, q, cache.int(), 1.0), {}, "uint8"),
            ((q, q, cache[..., :64], 1.0), {}, "18"), ((q, q, cache, 1.0), {"block_table": table[:1]}, "block_table"),
            ((q, q, cache, 1.0), {"block_table": table.long()}, "block_table"), ((q, q, cache, 1.0), {"kv_lens": table}, "kv_lens"),
            ((q, q, cache, 1.0), {"kv_lens": table[:, 0].cpu()}, "kv_lens"), ((q, q, cache, 1.0), {"max_kv_len": 33}, "max_kv_len"),
            ((q, q, cache, 1.0), {"algo": "simt"}, "algo"), ((q, q, cache, float("nan")), {}, "sm_scale"),
            ((q, q, cache, 1.0), {"lse": torch.zeros(2, 4, 2, device=DEV)}, "lse"),
            ((q[:, :, :3].contiguous(), q[:, :, :3].contiguous(), cache, 1.0), {}, "n_kv_heads"),
            ((q, q, cache, 1.0), {"algo": "tcgen05"}, "TCGEN05"),
        ]:
            with pytest.raises(RuntimeError, match=match):
                call(*args, **kw)
    rows_calls = [(llmx_b200.kv4_store, llmx_b200.kv4_load),
                  (lambda *a, **w: kv4._rows_call("llmx_kv4_store", *a, w.get("start"), w.get("lens"), w.get("block_table")),
                   lambda *a, **w: kv4._rows_call("llmx_kv4_load", *a, w.get("start"), w.get("lens"), w.get("block_table")))]
    for store, load in rows_calls:
        for fn in (store, load):
            for args, kw, match in [
                ((cache, k, k[:, :2]), {}, "same shape"), ((cache, k, k.half()), {}, "same shape and dtype"),
                ((cache, k[:, :, :1], k[:, :, :1]), {}, "n_kv_heads"), ((cache, k.float(), k.float()), {}, "float16 and bfloat16"),
                ((cache, k, k), {"start": table}, "start"), ((cache, k, k), {"lens": table[0, :1]}, "lens"),
                ((cache, k.repeat(3, 1, 1, 1), k.repeat(3, 1, 1, 1)), {}, "page per sequence"),
            ]:
                with pytest.raises(RuntimeError, match=match):
                    fn(*args, **kw)
        with pytest.raises(RuntimeError, match="unit stride"):
            load(cache, torch.zeros(2, 3, 2, 256, dtype=torch.bfloat16, device=DEV)[..., ::2], k)


def test_ctypes_form_agrees_with_the_binding():
    gen = torch.Generator().manual_seed(31)
    dtype, d, H, hkv = torch.bfloat16, 128, 8, 2
    lens = [300, 45]
    cache, table, k, v = filled(gen, lens, hkv, d, dtype, 32)
    other = garbage(cache.shape[0], hkv, d, 32)
    kv = torch.tensor(lens, device=DEV, dtype=torch.int32)
    kv4._rows_call("llmx_kv4_store", other, k.to(DEV), v.to(DEV), None, kv, table)
    assert torch.equal(cache, other)
    q = torch.randn(2, 2, H, d, generator=gen).to(dtype).to(DEV)
    a, b = torch.empty_like(q), torch.empty_like(q)
    la, lb = torch.empty(2, H, 2, device=DEV), torch.empty(2, H, 2, device=DEV)
    slopes = torch.rand(H, device=DEV)
    kw = dict(kv_lens=kv, block_table=table, alibi_slopes=slopes)
    llmx_b200.kv4_attention(a, q, cache, 0.1, 100, 5.0, lse=la, **kw)
    kv4.kv4_attention_ctypes(b, q, cache, 0.1, 100, 5.0, lse=lb, **kw)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_other_stream_graphs_and_repeats():
    """A non-default stream, captured and replayed calls (two graphs with their own workspaces), bit-identical repeats."""
    gen = torch.Generator().manual_seed(41)
    dtype, d, H, hkv = torch.float16, 128, 8, 2
    lens = [3000, 700]
    cache, table, k, v = filled(gen, lens, hkv, d, dtype, 64)
    kv = torch.tensor(lens, device=DEV, dtype=torch.int32)
    q = torch.randn(2, 1, H, d, generator=gen).to(dtype).to(DEV)
    ref = torch.empty_like(q)
    llmx_b200.kv4_attention(ref, q, cache, 0.1, kv_lens=kv, block_table=table)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = [torch.empty_like(q) for _ in range(3)]
    with torch.cuda.stream(side):
        llmx_b200.kv4_attention(outs[0], q, cache, 0.1, kv_lens=kv, block_table=table)
    side.synchronize()
    assert torch.equal(outs[0], ref)
    kn = torch.randn(2, 1, hkv, d, generator=gen).to(dtype).to(DEV)
    graphs = []
    for out in outs[1:]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            llmx_b200.kv4_store(cache, kn, kn, start=kv - 1, block_table=table)
            llmx_b200.kv4_attention(out, q, cache, 0.1, kv_lens=kv, block_table=table)
        graphs.append(g)
    kn.copy_(torch.stack([k[b, n - 1] for b, n in enumerate(lens)])[:, None])  # the same token again
    vn = torch.stack([v[b, n - 1] for b, n in enumerate(lens)])[:, None].to(DEV)
    for g, out in zip(graphs, outs[1:]):
        out.fill_(9.0)
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[1], outs[2])
    llmx_b200.kv4_store(cache, kn, vn, start=kv - 1, block_table=table)
    for _ in range(3):
        llmx_b200.kv4_attention(outs[0], q, cache, 0.1, kv_lens=kv, block_table=table)
        assert torch.equal(outs[0], ref)
    # Two streams at once, each with its own output and workspace.
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, out in zip(streams, outs):
            with torch.cuda.stream(s):
                llmx_b200.kv4_attention(out, q, cache, 0.1, kv_lens=kv, block_table=table)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref)


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.get_device_properties(0).total_memory < 60 << 30, reason="needs 30 GB")
def test_offsets_past_32_bits():
    """A cache of 5 GB: pages whose byte offset passes 2^32."""
    dtype, d, hkv, page = torch.float16, 256, 8, 128
    page_bytes = hkv * 8 * 18 * d
    n_pages = (5 << 30) // page_bytes
    cache = torch.empty(n_pages, hkv, 8, 18 * d, dtype=torch.uint8, device=DEV)
    gen = torch.Generator().manual_seed(51)
    k, v = rows(gen, 200, hkv, d, dtype)[None], rows(gen, 200, hkv, d, dtype)[None]
    table = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32, device=DEV)
    llmx_b200.kv4_store(cache, k.to(DEV), v.to(DEV), block_table=table)
    ko, vo = torch.empty_like(k, device=DEV), torch.empty_like(v, device=DEV)
    llmx_b200.kv4_load(cache, ko, vo, block_table=table)
    assert torch.equal(ko.cpu(), okv4.values(k)[1]) and torch.equal(vo.cpu(), okv4.values(v)[1])
    q = torch.randn(1, 1, 8, d, generator=gen).to(dtype)
    out = torch.empty_like(q, device=DEV)
    llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, block_table=table, max_kv_len=200)
    check(out, None, q, k, v, [1], [200], dtype, sm_scale=d ** -0.5)


def test_offsets_past_32_bits_inside_a_page():
    """One page of 7.7 million tokens (2.2 GB): offsets of tiles in their page pass 2^31."""
    dtype, d = torch.bfloat16, 256
    tiles = 482000
    cache = torch.empty(1, 1, tiles, 18 * d, dtype=torch.uint8, device=DEV)
    n = 16 * tiles
    gen = torch.Generator().manual_seed(52)
    k, v = rows(gen, 150, 1, d, dtype)[None], rows(gen, 150, 1, d, dtype)[None]
    start = torch.tensor([n - 150], device=DEV, dtype=torch.int32)
    llmx_b200.kv4_store(cache, k.to(DEV), v.to(DEV), start=start)
    ko, vo = torch.empty_like(k, device=DEV), torch.empty_like(v, device=DEV)
    llmx_b200.kv4_load(cache, ko, vo, start=start)
    assert torch.equal(ko.cpu(), okv4.values(k)[1]) and torch.equal(vo.cpu(), okv4.values(v)[1])
    q = torch.randn(1, 1, 4, d, generator=gen).to(dtype)
    out = torch.empty_like(q, device=DEV)
    llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, 149)  # a window of the last 150 tokens
    check(out, None, q, k, v, [1], [150], dtype, sm_scale=d ** -0.5)


def test_expanded_form_with_empty_and_tiny_sequences():
    dtype, d, H, hkv, sq = torch.float16, 128, 4, 2, 33
    gen = torch.Generator().manual_seed(61)
    lens = [0, 1, 200, 33]
    cache, table, k, v = filled(gen, lens, hkv, d, dtype, 64)
    q = torch.randn(len(lens), sq, H, d, generator=gen).to(dtype)
    q_lens = [33, 1, 0, 20]
    import oracle

    ref = oracle.attention_ref_padded(q.float(), okv4.values(k)[1].float(), okv4.values(v)[1].float(), kv_lens=lens,
                                      q_lens=q_lens, sm_scale=d ** -0.5)
    for algo in ("tcgen05", "decode"):
        poison = torch.full((1 << 20,), float("nan"), device=DEV)
        del poison
        out = torch.full_like(q, 3.0, device=DEV)
        llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, kv_lens=torch.tensor(lens, device=DEV), block_table=table,
                                q_lens=torch.tensor(q_lens, device=DEV), algo=algo)
        assert (out.float().cpu() - ref).abs().max() <= HALF_MAX_ABS, algo


def test_overlapping_outputs_are_refused():
    cache = garbage(2, 2, 64, 16)
    k = torch.zeros(1, 1, 1, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(LlmxError, match="overlap"):
        llmx_b200.kv4_load(cache, k.expand(2, 4, 2, 64), torch.empty(2, 4, 2, 64, dtype=torch.float16, device=DEV))
    with pytest.raises(LlmxError, match="overlap"):
        llmx_b200.kv4_attention(k.expand(2, 1, 4, 64), torch.zeros(2, 1, 4, 64, dtype=torch.float16, device=DEV), cache, 1.0)


def test_pages_shared_by_sequences():
    """Two sequences with a common prefix: their tables name the same pages."""
    dtype, d, H, hkv, page = torch.bfloat16, 64, 4, 1, 16
    gen = torch.Generator().manual_seed(71)
    k, v = rows(gen, 60, hkv, d, dtype), rows(gen, 60, hkv, d, dtype)
    cache = garbage(6, hkv, d, page)
    # tokens 0 .. 31 in pages 4, 2; the tails 32 .. of the sequences in 0 and 5
    llmx_b200.kv4_store(cache, k[None, :44].to(DEV), v[None, :44].to(DEV), block_table=torch.tensor([[4, 2, 0]], dtype=torch.int32, device=DEV))
    tail = torch.tensor([32], device=DEV, dtype=torch.int32)
    table = torch.tensor([[4, 2, 0], [4, 2, 5]], dtype=torch.int32, device=DEV)
    llmx_b200.kv4_store(cache, k[None, 44:].to(DEV), v[None, 44:].to(DEV), start=tail, block_table=table[1:])
    lens = [44, 48]
    kk = torch.stack([torch.nn.functional.pad(k[:44], (0, 0, 0, 0, 0, 4)), torch.cat([k[:32], k[44:60]])])
    vv = torch.stack([torch.nn.functional.pad(v[:44], (0, 0, 0, 0, 0, 4)), torch.cat([v[:32], v[44:60]])])
    q = torch.randn(2, 2, H, d, generator=gen).to(dtype)
    out = torch.empty_like(q, device=DEV)
    llmx_b200.kv4_attention(out, q.to(DEV), cache, 0.125, kv_lens=torch.tensor(lens, device=DEV), block_table=table)
    check(out, None, q, kk, vv, [2, 2], lens, dtype, sm_scale=0.125)


@pytest.mark.parametrize("opts", ["causal", "alibi", "window"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,H,hkv,sq,n", [(128, 8, 2, 4, 40), (64, 4, 4, 2, 16), (256, 4, 2, 3, 700), (128, 8, 8, 4, 90), (128, 2, 2, 2, 1300)])
def test_large_values_that_a_row_does_not_see(d, H, hkv, sq, n, dtype, opts):
    """Values far above the others in the last tokens, which only the last row sees, and with a window in the first
    one, which only the first row sees: the other rows' weights keep their bits."""
    gen = torch.Generator().manual_seed(d + n)
    k, v = rows(gen, n, hkv, d, dtype), rows(gen, n, hkv, d, dtype)
    small, large = (1e-2, 3e4 / 8) if dtype == torch.float16 else (1.0, 1e25)
    v = (v * small).to(dtype)
    window = n - sq if opts == "window" else -1
    far = 0 if opts == "window" else n - 1
    v[far] = (rows(gen, 1, hkv, d, dtype)[0].float() * large).to(dtype)
    slopes = torch.linspace(0.01, 0.2, H) if opts == "alibi" else None
    cache = garbage(-(-n // 16), hkv, d, 16)
    table = torch.arange(-(-n // 16), dtype=torch.int32, device=DEV)[None]
    llmx_b200.kv4_store(cache, k[None].to(DEV), v[None].to(DEV), block_table=table)
    q = torch.randn(1, sq, H, d, generator=gen).to(dtype)
    out, lse = torch.empty_like(q, device=DEV), torch.empty(1, H, sq, device=DEV)
    llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, window, max_kv_len=n, block_table=table, lse=lse, algo="decode",
                            alibi_slopes=None if slopes is None else slopes.to(DEV))
    check(out, lse, q, k[None], v[None], [sq], [n], dtype, sm_scale=d ** -0.5, window=window, slopes=slopes, what=opts)


@pytest.mark.parametrize("d,H", [(64, 1), (128, 4), (128, 8), (256, 2)])
@pytest.mark.parametrize("n", [30, 400])
def test_values_far_apart(d, H, n):
    """Constant groups of large values (steps of 0), and steps 2^150 apart whose tokens count alike in the sums."""
    dtype = torch.bfloat16
    gen = torch.Generator().manual_seed(n + d)
    k, base = rows(gen, n, 1, d, dtype), rows(gen, n, 1, d, dtype)
    first = (torch.arange(n) < n // 2)[:, None, None]
    constant = torch.full_like(base, 1e30)
    for v in (constant, -constant, torch.where(first, constant, base), torch.where(first, base, constant),
              torch.where(first, base * 1e-10, base * 1e36), torch.where(first, base * 1e36, base * 1e-10)):
        v = v.to(dtype)
        cache = garbage(-(-n // 64), 1, d, 64)
        table = torch.arange(-(-n // 64), dtype=torch.int32, device=DEV)[None]
        llmx_b200.kv4_store(cache, k[None].to(DEV), v[None].to(DEV), block_table=table)
        q = torch.randn(1, 1, H, d, generator=gen).to(dtype)
        out, lse = torch.empty_like(q, device=DEV), torch.empty(1, H, 1, device=DEV)
        llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, max_kv_len=n, block_table=table, lse=lse)
        check(out, lse, q, k[None], v[None], [1], [n], dtype, sm_scale=d ** -0.5, what="far apart")


@pytest.mark.parametrize("d,H,hkv,sq,B,top", [
    (128, 8, 2, 1, 120, 1200),  # a CTA for a unit, long ones too
    (128, 8, 2, 2, 120, 2600),  # units shared by warps, fewer units than CTAs
    (64, 8, 2, 1, 120, 2600),   # units shared by CTAs
    (256, 4, 2, 1, 120, 1300),
    (64, 4, 4, 1, 700, 90),     # a warp for a unit, in two launches
    (128, 10, 5, 1, 520, 90),   # more units than warps
    (128, 5, 5, 3, 520, 700),   # units shared by warps, in two launches
])
def test_each_way_of_dealing_units(d, H, hkv, sq, B, top):
    dtype = torch.float16 if B == 120 else torch.bfloat16
    gen = torch.Generator().manual_seed(B + top)
    lens = torch.randint(0, 40, (B,), generator=gen).tolist()
    lens[0], lens[B // 2], lens[B - 2] = top, 0, top // 2
    cache, table, k, v = filled(gen, lens, hkv, d, dtype, 16)
    q = torch.randn(B, sq, H, d, generator=gen).to(dtype)
    q_lens = [sq] * B
    q_lens[1] = 0
    for slopes in (None, torch.linspace(0.01, 0.3, H)):
        out, lse = torch.full_like(q, 7.0, device=DEV), torch.full((B, H, sq), 7.0, device=DEV)
        llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, kv_lens=torch.tensor(lens, device=DEV), block_table=table, lse=lse,
                                q_lens=torch.tensor(q_lens, device=DEV), algo="decode",
                                alibi_slopes=None if slopes is None else slopes.to(DEV))
        check(out, lse, q, k, v, q_lens, lens, dtype, sm_scale=d ** -0.5, slopes=slopes)
    llmx_b200.device_status(0)
