"""The 4-bit key/value cache on the GPU at its edges: host threads at once,
empty sequences, numbers at the ends of their types, tokens that a row must not
see, sizes near 31 bits, workspaces that are missing."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

import llmx_b200
from gpu_helpers import needs_cuda
from llmx_b200 import _lib, kv4
from oracle import kv4 as okv4

pytestmark = [pytest.mark.gpu, needs_cuda]

DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# Host threads that call the C entry at the same moment, step by step; each has
# its own requests (of growing batches), stream and results.
GATE_C = r"""
#include <pthread.h>
#include <stdatomic.h>
#include <stddef.h>
#include "llmx_attn.h"
struct job { const llmx_attn_params *p; const llmx_kv4_cache *c; void *stream; int n, threads; int *status; atomic_int *gate; };
static void *work(void *arg) {
  struct job *j = arg;
  for (int i = 0; i < j->n; ++i) {
    atomic_fetch_add(j->gate, 1);
    while (atomic_load(j->gate) < j->threads * (i + 1)) {}
    j->status[i] = llmx_kv4_attn_fwd(j->p + i, j->c + i, j->stream);
  }
  return NULL;
}
int run(int threads, int n, const llmx_attn_params **p, const llmx_kv4_cache **c, void **streams, int *status) {
  pthread_t t[16];
  struct job j[16];
  atomic_int gate = 0;
  for (int i = 0; i < threads; ++i) {
    j[i] = (struct job){p[i], c[i], streams[i], n, threads, status + i * n, &gate};
    if (pthread_create(&t[i], NULL, work, &j[i]) != 0) return 1;
  }
  for (int i = 0; i < threads; ++i) pthread_join(t[i], NULL);
  return 0;
}
"""
THREADS = r"""
import ctypes, sys
import torch
from llmx_b200 import _lib, kv4

lib, gate = _lib.load(), ctypes.CDLL(sys.argv[1])
THREADS, failed = 4, []
for dtype in (torch.bfloat16, torch.float16):
    for d, heads, most in ((256, 1, 440), (256, 9, 440), (128, 1, 440), (128, 4, 440), (128, 8, 512), (64, 2, 512)):
        cache = torch.zeros(most, 1, 1, 18 * d, dtype=torch.uint8, device="cuda")
        n, keep, streams = most // THREADS, [], [torch.cuda.Stream() for _ in range(THREADS)]
        ps, cs = [(_lib.AttnParams * n)() for _ in range(THREADS)], [(_lib.Kv4Cache * n)() for _ in range(THREADS)]
        for t in range(THREADS):
            q = torch.zeros(most, 1, heads, d, dtype=dtype, device="cuda")
            out = torch.empty_like(q)
            keep += [q, out]
            for i in range(n):
                b, p, c = THREADS * i + t + 1, ps[t][i], kv4._cache_arg(cache, THREADS * i + t + 1, dtype, d, None, keep)
                c.max_pages = 1
                cs[t][i] = c
                lib.llmx_attn_params_init(ctypes.byref(p))
                p.dtype, p.batch, p.n_heads, p.n_kv_heads, p.head_dim, p.max_q_len, p.max_kv_len = c.dtype, b, heads, 1, d, 1, 16
                p.q, p.o, p.sm_scale = q.data_ptr(), out.data_ptr(), 1.0
                lib.llmx_attn_set_contiguous_strides(ctypes.byref(p))
        torch.cuda.synchronize()
        status = (ctypes.c_int * (n * THREADS))()
        ptrs = lambda xs: (ctypes.c_void_p * THREADS)(*xs)
        assert gate.run(THREADS, n, ptrs(map(ctypes.addressof, ps)), ptrs(map(ctypes.addressof, cs)),
                        ptrs(s.cuda_stream for s in streams), status) == 0
        torch.cuda.synchronize()
        failed += [(str(dtype), d, heads, i) for i, s in enumerate(status) if s != 0]
print("failed", len(failed), failed[:5], lib.llmx_attn_last_error())
sys.exit(1 if failed else 0)
"""


def test_host_threads_with_different_batches(tmp_path):
    """A fresh process: each kernel's shared-memory limit is set by its first calls."""
    src, so = tmp_path / "gate.c", tmp_path / "gate.so"
    src.write_text(GATE_C)
    lib = os.path.join(ROOT, "llmx_b200")
    subprocess.run(["gcc", "-O2", "-shared", "-fPIC", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(so), "-L", lib,
                    "-lllmx_attn", "-Wl,-rpath," + lib, "-lpthread"], check=True)
    r = subprocess.run([sys.executable, "-c", THREADS, str(so)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr[-2000:]


def request(cache, table, q, out, lens, *, scale, algo="auto", lse=None, slopes=None, max_kv_len=0):
    """(params, cache, what they point to) of a call of the C entry; the caller sets the workspace."""
    lib, keep = _lib.load(), [q, out, lens, table, lse, slopes]
    B, sq, H, d = q.shape
    c = kv4._cache_arg(cache, B, q.dtype, d, table, keep)
    p = _lib.AttnParams()
    lib.llmx_attn_params_init(ctypes.byref(p))
    p.dtype, p.batch, p.n_heads, p.n_kv_heads, p.head_dim, p.max_q_len = c.dtype, B, H, c.n_kv_heads, d, sq
    p.max_kv_len = max_kv_len or c.max_pages * c.page_size
    p.q, p.o, p.kv_lens, p.sm_scale, p.algo = q.data_ptr(), out.data_ptr(), lens.data_ptr(), scale, _lib.ALGO[algo]
    p.lse = None if lse is None else lse.data_ptr()
    p.alibi_slopes = None if slopes is None else slopes.data_ptr()
    lib.llmx_attn_set_contiguous_strides(ctypes.byref(p))
    return p, c, keep


def stored(k, v, page=64):
    """A cache without a table that holds k, v [B, S, Hkv, D]."""
    B, S, hkv, d = k.shape
    cache = llmx_b200.kv4_empty(B * -(-S // page), hkv, d, page, device=DEV)
    cache.fill_(255)
    llmx_b200.kv4_store(cache, k.to(DEV), v.to(DEV))
    return cache


def check(out, lse, q, k, v, kv_len, dtype, *, sm_scale, slopes=None, causal=True, window=-1, what=""):
    """One sequence, element by element, to the oracle's bound and half a step of the output's type."""
    o, le, bound, le_bound = okv4.attention(q, k, v, q.shape[0], kv_len, sm_scale=sm_scale, slopes=slopes, causal=causal,
                                            window=window)
    half = torch.finfo(dtype).eps / 2
    room = bound * (1 + 2 ** -10) + (o.abs() + bound) * half + torch.finfo(dtype).smallest_normal * half
    off = (out.double().cpu() - o).abs()
    assert (off <= room).all(), f"{what}: worst {float((off / room).nan_to_num(1e9).max()):.3g} of the bound"
    if lse is not None:
        off = (lse.double().cpu() - le).abs()
        seen = le != -math.inf
        assert (off <= le_bound)[seen].all(), f"{what}: lse, worst {float((off / le_bound)[seen].nan_to_num(1e9).max()):.3g} of the bound"


@pytest.mark.parametrize("start", [5, 63, 10 ** 6 + 3])
def test_an_empty_sequence_reads_no_page(start):
    """Rows enough for a tile a warp; the first sequence has none of them, and nothing valid in its table."""
    dtype, d, hkv, S = torch.bfloat16, 128, 16, 600
    gen = torch.Generator().manual_seed(start)
    k, v = (torch.randn(2, S, hkv, d, generator=gen).to(dtype).to(DEV) for _ in range(2))
    table = torch.tensor([[-1] * 10, list(range(10))], dtype=torch.int32, device=DEV)
    cache = llmx_b200.kv4_empty(10, hkv, d, 64, device=DEV)
    kw = dict(start=torch.tensor([start, 0], device=DEV), lens=torch.tensor([0, S], device=DEV), block_table=table)
    llmx_b200.device_status(0)
    llmx_b200.kv4_store(cache, k, v, **kw)
    llmx_b200.device_status(0)
    ko, vo = torch.full_like(k, 9.0), torch.full_like(v, 9.0)
    llmx_b200.kv4_load(cache, ko, vo, **kw)
    llmx_b200.device_status(0)
    assert (ko[0] == 0).all() and (vo[0] == 0).all()
    assert torch.equal(ko[1].cpu(), okv4.values(k[1].cpu())[1]) and torch.equal(vo[1].cpu(), okv4.values(v[1].cpu())[1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,hkv,S", [(64, 1, 5), (128, 24, 700), (256, 2, 40)])
def test_finite_values_at_the_ends_of_the_type(dtype, d, hkv, S):
    """Groups that reach the type's largest numbers read back finite, each value within half a step."""
    top = torch.finfo(dtype).max
    gen = torch.Generator().manual_seed(d)
    x = (torch.rand(1, S, hkv, d, generator=gen, dtype=torch.float64) * top).to(dtype)
    x[..., 0], x[..., 1] = 0.0, top
    x[:, 1::4] = -x[:, 1::4]
    if dtype == torch.float16:  # (for bf16 this range passes fp32)
        x[:, 2::4, :, 0] = -top
    x[:, 3::4, :, 0] = 0.01 * top
    cache = stored(x, x)
    n, s, m = okv4.quantise(x)
    ko, vo = torch.empty_like(x, device=DEV), torch.empty_like(x, device=DEV)
    llmx_b200.kv4_load(cache, ko, vo)
    want = okv4.values(x)[1]
    assert want.isfinite().all() and torch.equal(ko.cpu(), want) and torch.equal(vo.cpu(), want)
    # Half a step, fp32's rounding of the difference, and the read-back's own rounding.
    room = okv4.spread(s) * 0.5 * (1 + 2.0 ** -20) + want.double().abs() * torch.finfo(dtype).eps
    assert ((ko.double().cpu() - x.double()).abs() <= room).all()
    # A row that sees one token gets its values.
    for b in range(4):
        q = torch.zeros(1, 1, hkv, d, dtype=dtype, device=DEV)
        out = torch.empty_like(q)
        one = torch.zeros(1, 1, hkv, d, dtype=dtype)
        llmx_b200.kv4_attention(out, q, stored(one, x[:, b:b + 1]), 1.0, max_kv_len=1)
        check(out[0], None, q[0].cpu(), one[0], x[0, b:b + 1], 1, dtype, sm_scale=1.0, what=f"token {b}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,H,hkv,sq,lens", [(128, 8, 2, 160, [900, 400]), (64, 4, 4, 200, [513, 200]), (256, 3, 1, 140, [700, 140])])
def test_nan_tokens_reach_only_the_rows_that_see_them(dtype, d, H, hkv, sq, lens):
    """A NaN in K makes the rows that see the token NaN, one in V their channels of its group (expanded: the whole rows)."""
    import oracle

    gen = torch.Generator().manual_seed(sq)
    B, S, page = len(lens), max(lens), 64
    k, v = (torch.randn(B, S, hkv, d, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(B, sq, H, d, generator=gen).to(dtype)
    bad_v = [(0, lens[0] - 3, 0, d - 1), (0, lens[0] - sq // 2, hkv - 1, 5), (0, 11, hkv - 1, 3), (1, lens[1] - 40, 0, 7),
             (1, lens[1] - 41, hkv - 1, d - 2), (1, lens[1] - 1, 0, 0)]
    bad_k = [(0, lens[0] - 20, 0), (1, lens[1] - 30, hkv - 1)]
    kx, vx = k.clone(), v.clone()
    for b, j, h, c in bad_v:
        vx[b, j, h, c] = math.nan
        v[b, j, h, c // 64 * 64:c // 64 * 64 + 64] = 0.0  # what the others of the reference see
    for b, j, h in bad_k:
        kx[b, j, h, 1] = math.inf
        k[b, j, h] = 0.0
    cache = stored(kx, vx, page)
    slopes = torch.pow(2.0, -8.0 * torch.arange(1, H + 1) / H).float()
    kv = torch.tensor(lens, device=DEV, dtype=torch.int32)
    kd, vd = okv4.values(k)[1].float(), okv4.values(v)[1].float()
    for opts in (dict(), dict(window=25), dict(causal=False, window=30), dict(alibi=slopes), dict(cap=5.0)):
        causal, window = opts.get("causal", True), opts.get("window", -1)
        ref = oracle.attention_ref_padded(q.float(), kd, vd, kv_lens=lens, sm_scale=d ** -0.5, causal=causal,
                                          **({"sliding_window": window} if window >= 0 else {}),
                                          **({"alibi": slopes} if "alibi" in opts else {}),
                                          **({"logits_soft_cap": 5.0} if "cap" in opts else {}))
        nan, nan_lse = torch.zeros(B, sq, H, d, dtype=torch.bool), torch.zeros(B, H, sq, dtype=torch.bool)
        group = H // hkv

        def rows_that_see(b, j):
            diag = torch.arange(sq) + lens[b] - sq
            return ((j <= diag) | (not causal)) & ((diag - j <= window) | (window < 0))

        for b, j, h, c in bad_v:
            nan[b, rows_that_see(b, j), h * group:(h + 1) * group, c // 64 * 64:c // 64 * 64 + 64] = True
        for b, j, h in bad_k:
            nan[b, rows_that_see(b, j), h * group:(h + 1) * group] = True
            nan_lse[b, h * group:(h + 1) * group, rows_that_see(b, j)] = True
        for algo in ("decode", "tcgen05"):
            out, lse = torch.full_like(q, 7.0, device=DEV), torch.zeros(B, H, sq, device=DEV)
            llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, window, opts.get("cap", 0.0), kv_lens=kv, causal=causal,
                                    alibi_slopes=slopes.to(DEV) if "alibi" in opts else None, lse=lse, algo=algo)
            what, want = f"{algo} {opts}", nan
            if algo == "tcgen05":
                want = nan.any(-1, keepdim=True).expand_as(nan)
                nan_lse = want[..., 0].transpose(1, 2)
            assert torch.equal(lse.cpu().isnan(), nan_lse), what
            assert torch.equal(out.cpu().isnan(), want), f"{what}: {int((out.cpu().isnan() != want).sum())} differ"
            err = (out.float().cpu() - ref).abs()[~want]
            assert err.numel() == 0 or err.max() <= 2e-2, f"{what}: {float(err.max())}"
    llmx_b200.device_status(0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,H,hkv,sq,n", [(128, 8, 2, 160, 400), (64, 4, 4, 200, 200), (256, 3, 1, 140, 130)])
def test_infinities_and_nan_in_q_make_their_rows_nan(dtype, d, H, hkv, sq, n):
    """Both forms; rows above the keys' begin stay 0, also with such a q.  (The first rows see few keys: all scores -inf is one outcome.)"""
    gen = torch.Generator().manual_seed(n)
    k, v = (torch.randn(1, n, hkv, d, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(1, sq, H, d, generator=gen).to(dtype)
    bad = torch.zeros(sq, H, dtype=torch.bool)
    bad[torch.randperm(sq, generator=gen)[:40], torch.randint(0, H, (40,), generator=gen)] = True
    bad[max(0, sq - n):max(0, sq - n) + 4] = True
    for i, h in bad.nonzero().tolist():
        q[0, i, h, (7 * i + h) % d] = [math.inf, -math.inf, math.nan][(i + h) % 3]
    cache = stored(k, v)
    only_nan = torch.where(q.isinf(), torch.full_like(q, math.nan), q)  # (a soft-cap makes finite scores of infinite ones)
    for opts in (dict(), dict(sliding_window=20), dict(causal=False), dict(logits_soft_cap=4.0), dict(alibi_slopes=torch.rand(H, device=DEV))):
        qd = (only_nan if "logits_soft_cap" in opts else q).to(DEV)
        seen = (torch.arange(sq) + n - sq >= 0) | (not opts.get("causal", True))
        for algo in ("decode", "tcgen05"):
            out, lse = torch.full_like(q, 7.0, device=DEV), torch.zeros(1, H, sq, device=DEV)
            llmx_b200.kv4_attention(out, qd, cache, d ** -0.5, max_kv_len=n, lse=lse, algo=algo, **opts)
            o, nan, what = out[0].cpu(), bad & seen[:, None], f"{algo} {opts}"
            assert torch.equal(o.isnan(), nan[..., None].expand_as(o)), what
            assert torch.equal(lse[0].cpu().isnan(), nan.T), what
            assert (o[~seen] == 0).all() and (lse[0].cpu()[:, ~seen] == -math.inf).all(), what
    llmx_b200.device_status(0)


def test_a_cache_full_of_nan():
    """Every V group NaN: all rows that see a key are NaN, rows without one are 0."""
    dtype, d, H, hkv, sq = torch.bfloat16, 128, 4, 2, 300
    cache = llmx_b200.kv4_empty(2 * 8, hkv, d, 64, device=DEV)
    x = torch.full((2, 512, hkv, d), math.nan, dtype=dtype, device=DEV)
    llmx_b200.kv4_store(cache, torch.zeros_like(x), x)
    q = torch.randn(2, sq, H, d, device=DEV, dtype=dtype)
    for algo in ("decode", "tcgen05"):
        out = torch.full_like(q, 7.0)
        llmx_b200.kv4_attention(out, q, cache, 0.1, kv_lens=torch.tensor([500, 100], device=DEV), algo=algo)
        seen = torch.ones(2, sq, dtype=torch.bool)
        seen[1, :200] = False
        assert torch.equal(out.isnan().all(-1).all(-1).cpu(), seen) and (out[~seen.to(DEV)] == 0).all(), algo


@pytest.mark.parametrize("H,hkv,sq", [(8, 2, 1024), (16, 4, 700)])
def test_auto_without_its_workspace_runs_the_direct_form(H, hkv, sq):
    dtype, d, n = torch.bfloat16, 128, 1500
    gen = torch.Generator().manual_seed(sq)
    k, v = (torch.randn(1, n, hkv, d, generator=gen).to(dtype) for _ in range(2))
    cache, q = stored(k, v), torch.randn(1, sq, H, d, generator=gen).to(dtype)
    qd, lens = q.to(DEV), torch.tensor([n], device=DEV, dtype=torch.int32)
    out, lib = torch.empty_like(qd), _lib.load()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    ws = ctypes.c_size_t(0)
    need = {}
    for algo in ("auto", "tcgen05", "decode"):
        p, c, keep = request(cache, None, qd, out, lens, scale=d ** -0.5, algo=algo)
        _lib.check(lib.llmx_kv4_attn_workspace_size(ctypes.byref(p), ctypes.byref(c), ctypes.byref(ws)))
        need[algo] = ws.value
    assert need["auto"] == need["tcgen05"]  # a request that AUTO expands
    p, c, keep = request(cache, None, qd, out, lens, scale=d ** -0.5, algo="tcgen05")
    assert lib.llmx_kv4_attn_fwd(ctypes.byref(p), ctypes.byref(c), stream) == 3, lib.llmx_attn_last_error()
    small = torch.empty(need["decode"] + 16, dtype=torch.uint8, device=DEV)
    for ptr, size in ((None, 0), (small.data_ptr(), small.numel())):
        p, c, keep = request(cache, None, qd, out, lens, scale=d ** -0.5)
        p.workspace, p.workspace_bytes = ptr, size
        out.fill_(7.0)
        _lib.check(lib.llmx_kv4_attn_fwd(ctypes.byref(p), ctypes.byref(c), stream))
        torch.cuda.synchronize()
        check(out[0], None, q[0], k[0], v[0], n, dtype, sm_scale=d ** -0.5)


@pytest.mark.parametrize("H,hkv,d", [(1, 1, 64), (4, 1, 128), (8, 1, 128), (8, 8, 128), (2, 1, 256), (6, 2, 64)])
@pytest.mark.parametrize("batch", [1, 40])
def test_many_small_weights_beside_large_steps(H, hkv, d, batch):
    """One token at the maximum and 8192 that weigh 2^-12 of it each, V near bf16's end: the small ones are two thirds of the sum."""
    dtype, n = torch.bfloat16, 8193
    gen = torch.Generator().manual_seed(d + H)
    v = ((torch.rand(1, n, hkv, d, generator=gen) * 2 - 1) * 1e38).to(dtype)
    k = torch.zeros(1, n, hkv, d, dtype=dtype)
    k[:, 100] = 1.0  # a score of 12 ln 2 over the rest
    q = torch.full((1, 1, H, d), 12 * math.log(2.0) / d, dtype=torch.float32).to(dtype)
    cache = stored(k.expand(batch, -1, -1, -1), v.expand(batch, -1, -1, -1))
    out, lse = torch.empty(batch, 1, H, d, dtype=dtype, device=DEV), torch.empty(batch, H, 1, device=DEV)
    llmx_b200.kv4_attention(out, q.to(DEV).expand(batch, -1, -1, -1), cache, 1.0, max_kv_len=n, lse=lse, algo="decode")
    for b in {0, batch // 2, batch - 1}:
        check(out[b], lse[b], q[0], k[0], v[0], n, dtype, sm_scale=1.0, what=f"sequence {b}")


def test_the_log_sum_exp_of_scores_that_move_the_maximum():
    """Rising and falling scores, steps of very different sizes: the log-sum-exp beside the output."""
    dtype, d, n = torch.bfloat16, 128, 700
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn(n, 1, d, generator=gen).to(dtype) for _ in range(2))
    ramp = torch.linspace(0.0, 8.0, n)[:, None, None]
    size = torch.pow(10.0, torch.linspace(-6, 6, n))[torch.randperm(n, generator=gen)][:, None, None]
    for kk, vv in (((k * ramp).to(dtype), v), ((k * ramp.flip(0)).to(dtype), v), (k, (v * size).to(dtype)),
                   ((k * ramp).to(dtype), (v * ramp * 1e-3).to(dtype)), (k, (v * size * 1e30).to(dtype))):
        cache = stored(kk[None], vv[None])
        q = (torch.randn(1, 1, 8, d, generator=gen) * torch.tensor([1e-20, 1e-3, 1, 1, 2, 4, 8, 30])[None, None, :, None]).to(dtype)
        out, lse = torch.empty_like(q, device=DEV), torch.empty(1, 8, 1, device=DEV)
        llmx_b200.kv4_attention(out, q.to(DEV), cache, d ** -0.5, max_kv_len=n, lse=lse)
        check(out[0], lse[0], q[0], kk, vv, n, dtype, sm_scale=d ** -0.5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,H,hkv,sq", [(64, 8, 2, 1), (128, 4, 4, 1), (64, 8, 1, 3), (256, 4, 2, 1), (128, 8, 1, 2)])
@pytest.mark.parametrize("batch", [1, 150])
def test_alibi_goes_by_distance_however_far(dtype, d, H, hkv, sq, batch):
    """The same tokens behind windows that end early and late in a sequence: the biases differ by a constant, which a softmax does
    not see.  Steep and flat slopes of both signs; the pages before the window are one page, never read."""
    gen = torch.Generator().manual_seed(d + H + sq)
    page, n, window = 2 ** 14, 1000, 800
    k, v = (torch.randn(1, n, hkv, d, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(1, sq, H, d, generator=gen).to(dtype)
    slopes = torch.tensor([0.84, -0.5, 0.25, 0.003, -0.01, 0.0, 0.71, 1.0])[:H]
    cache = llmx_b200.kv4_empty(2, hkv, d, page, device=DEV)
    cache.fill_(255)
    got = []
    for far in (0, 2 ** 17, 2 ** 20, 2 ** 25):
        table = torch.ones(batch, far // page + 1, dtype=torch.int32, device=DEV)
        table[:, -1] = 0
        at = torch.full((batch,), far, dtype=torch.int32, device=DEV)
        llmx_b200.kv4_store(cache, k.to(DEV), v.to(DEV), start=at[:1], block_table=table[:1])
        out, lse = torch.empty(batch, sq, H, d, dtype=dtype, device=DEV), torch.empty(batch, H, sq, device=DEV)
        llmx_b200.kv4_attention(out, q.to(DEV).expand(batch, -1, -1, -1), cache, d ** -0.5, window, kv_lens=at + n, block_table=table,
                                alibi_slopes=slopes.to(DEV), lse=lse, algo="decode")
        got.append((far, out.double().cpu(), lse.double().cpu()))
    o, le, _, _ = okv4.attention(q[0], k[0], v[0], sq, n, sm_scale=d ** -0.5, slopes=slopes, window=window)
    half = torch.finfo(dtype).eps / 2
    # What differs from call to call: each p s is rounded to fp16 (2^-11) from another reference, at most 8 steps (half the range) of V
    # each; sums in fp32 (1000 terms of at most 2^-24, over outputs of at most 8 steps) and the output's own rounding.
    steps = okv4.quantise(v)[1].double().max()
    for far, out, lse in got[1:]:
        room = 2 * (8 * steps * (2 ** -11 + 2 ** -14) + half * o.abs() + half * 8 * steps * 2 ** -8)
        off = (out - got[0][1]).abs()
        assert (off <= room).all(), f"{far}: worst {float((off / room).max()):.3g} of the room"
        # fp32 numbers of the size of the log-sum-exp: three roundings each, and the sum's.
        want = got[0][2] + (slopes.double() * far)[None, :, None]
        assert ((lse - want).abs() <= (lse.abs() + le.abs()) * 2 ** -22 + 2 ** -12).all(), f"{far}: lse"


def test_a_row_count_near_31_bits():
    """max_rows as the largest integer, over rows of stride 0, with a length of a few."""
    dtype, d, hkv = torch.float16, 256, 15
    gen = torch.Generator().manual_seed(7)
    x = torch.randn(1, 1, hkv, d, generator=gen).to(dtype)
    cache = llmx_b200.kv4_empty(1, hkv, d, 16, device=DEV)
    cache.fill_(255)
    wide = x.to(DEV).expand(1, 2 ** 31 - 1, hkv, d)
    llmx_b200.kv4_store(cache, wide, wide, lens=torch.tensor([3], device=DEV, dtype=torch.int32))
    want = torch.full((hkv, 18 * d), 255, dtype=torch.uint8)
    for h in range(hkv):
        for tok in range(3):
            okv4.write_token(want[h], tok, x[0, 0, h], x[0, 0, h])
    assert torch.equal(cache[0, :, 0].cpu(), want)
    llmx_b200.device_status(0)


@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("start", [2 ** 32 + 3, -2 ** 32 + 3, 2 ** 40])
def test_positions_past_32_bits_are_reported(binding, start):
    """int64 positions whose low halves are inside the cache: dropped and reported, like any other outside it."""
    dtype, d, hkv = torch.bfloat16, 64, 2
    cache = llmx_b200.kv4_empty(1, hkv, d, 16, device=DEV)
    cache.fill_(255)
    k = torch.randn(1, 2, hkv, d, device=DEV).to(dtype)
    at = torch.tensor([start], device=DEV, dtype=torch.int64)
    llmx_b200.device_status(0)
    if binding:
        llmx_b200.kv4_store(cache, k, k, start=at)
    else:
        kv4._rows_call("llmx_kv4_store", cache, k, k, at, None, None)
    with pytest.raises(_lib.LlmxError, match="position"):
        llmx_b200.device_status(0)
    assert (cache == 255).all()
    # Lengths too: past the cache means all of it.
    q = torch.randn(1, 1, hkv, d, device=DEV).to(dtype)
    x = torch.randn(1, 16, hkv, d, device=DEV).to(dtype)
    llmx_b200.kv4_store(cache, x, x)
    a, b = torch.empty_like(q), torch.empty_like(q)
    call = llmx_b200.kv4_attention if binding else kv4.kv4_attention_ctypes
    call(a, q, cache, 0.1, kv_lens=torch.tensor([2 ** 32 + 3], device=DEV))
    call(b, q, cache, 0.1)
    assert torch.equal(a, b)
    # Narrow types have nothing to lose.
    for t in (torch.int16, torch.uint8):
        call(a, q, cache, 0.1, kv_lens=torch.tensor([7], device=DEV, dtype=t))
        call(b, q, cache, 0.1, kv_lens=torch.tensor([7], device=DEV, dtype=torch.int32))
        assert torch.equal(a, b)
