"""Key/value cache held in 4 bits: writing, reading back, and attention over it.

The cache is one uint8 CUDA tensor [n_pages, n_kv_heads, page_size / 16,
18 * head_dim] (``kv4_empty``): pages of tiles of 16 tokens, each with the
codes of K, the codes of V and their parameters in the layout that
include/llmx_attn.h describes.  K and V are fp16 or bf16 with head_dim 64, 128
or 256, quantised in groups of 64 channels to n s + m with n in 0 .. 15 and s,
m in the type of K and V: 4.5 bits a value.  ``block_table`` (CUDA int32
[batch, max_pages]) names the pages of each sequence; without one sequence b
owns pages b * max_pages .., max_pages = n_pages / batch.

    cache = kv4_empty(n_pages, n_kv_heads, head_dim, page_size)
    kv4_store(cache, k, v, start=lens_before, block_table=table)      # [B, S, H_kv, D], S = 1 per decode step
    kv4_attention(out, q, cache, sm_scale, kv_lens=lens, block_table=table)
    kv4_load(cache, k, v, lens=lens, block_table=table)               # back to dense rows

Everything runs on torch's current stream of the tensors' device.  Zeroed or
uninitialised pages are never read behind a sequence's length.  A table entry
or position outside the cache is skipped and reported by ``device_status``.
The calls go through the C++ torch binding (llmx_b200.llmx_bind) when it is
built, else through ctypes.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib, ops
from .ops import _TORCH_DTYPE, _req

TILE_TOKENS = 16


def kv4_empty(n_pages: int, n_kv_heads: int, head_dim: int, page_size: int = 64, device="cuda") -> torch.Tensor:
    """An uninitialised cache of ``n_pages`` pages of ``page_size`` tokens."""
    _req(head_dim in (64, 128, 256), "kv4: head_dim must be 64, 128 or 256")
    _req(page_size >= TILE_TOKENS and page_size % TILE_TOKENS == 0, "kv4: page_size must be a multiple of 16")
    _req(n_pages >= 1 and n_kv_heads >= 1, "kv4: n_pages and n_kv_heads must be >= 1")
    return torch.empty(n_pages, n_kv_heads, page_size // TILE_TOKENS, 18 * head_dim, dtype=torch.uint8, device=device)


def _int_arg(name: str, t: Optional[torch.Tensor], batch: int, device, keep):
    if t is None:
        return None
    _req(t.is_cuda and t.device == device, f"{name} must be on the cache's device")
    if t.dtype == torch.int64:  # what 32 bits do not hold becomes the nearest number that they do, not its low half
        t = t.clamp(-2 ** 31, 2 ** 31 - 1)
    t = t.to(torch.int32).contiguous()
    _req(t.numel() == batch, f"{name} must have batch elements")
    keep.append(t)
    return t.data_ptr()


def _cache_arg(cache: torch.Tensor, batch: int, dtype: torch.dtype, head_dim: int, block_table, keep):
    _req(cache.dtype == torch.uint8 and cache.dim() == 4,
         "kv4: cache must be uint8 [n_pages, n_kv_heads, page_size / 16, 18 * head_dim]")
    _req(cache.is_cuda, "kv4: cache must be a CUDA tensor")
    _req(dtype in (torch.float16, torch.bfloat16), "kv4: only float16 and bfloat16 are supported")
    _req(cache.shape[3] == 18 * head_dim, f"kv4: cache tiles must have 18 * head_dim = {18 * head_dim} bytes")
    _req(cache.stride(3) == 1 and (cache.shape[2] == 1 or cache.stride(2) == cache.shape[3]),
         "kv4: the tiles of a page must be contiguous")
    c = _lib.Kv4Cache()
    c.dtype, c.n_kv_heads, c.head_dim = _lib.DTYPE[_TORCH_DTYPE[dtype]], cache.shape[1], head_dim
    c.page_size, c.n_pages = cache.shape[2] * TILE_TOKENS, cache.shape[0]
    c.data, c.page_stride, c.head_stride = cache.data_ptr(), cache.stride(0), cache.stride(1)
    if block_table is None:
        _req(batch == 0 or cache.shape[0] >= batch, "kv4: without a block_table the cache needs a page per sequence")
        c.max_pages = cache.shape[0] // max(batch, 1)
    else:
        _req(block_table.is_cuda and block_table.device == cache.device, "kv4: block_table must be on the cache's device")
        _req(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == batch
             and block_table.shape[1] >= 1, "kv4: block_table must be int32 [batch, max_pages]")
        if block_table.stride(1) != 1:
            block_table = block_table.contiguous()
        keep.append(block_table)
        c.max_pages = block_table.shape[1]
        c.block_table, c.table_stride = block_table.data_ptr(), block_table.stride(0)
    return c


def _rows_call(fn: str, cache, k, v, start, lens, block_table) -> None:
    _req(k.dim() == 4 and v.dim() == 4, "kv4: k and v must be [batch, rows, n_kv_heads, head_dim]")
    _req(tuple(k.shape) == tuple(v.shape) and k.dtype == v.dtype, "kv4: k and v must have the same shape and dtype")
    _req(k.is_cuda and v.is_cuda and k.device == v.device == cache.device, "kv4: k, v and cache must be on one CUDA device")
    _req(k.shape[2] == cache.shape[1], "kv4: k and v must have the cache's n_kv_heads")
    if fn == "llmx_kv4_store":
        k, v = (x if x.stride(-1) == 1 else x.contiguous() for x in (k, v))
    else:
        _req(k.stride(-1) == 1 and v.stride(-1) == 1, "kv4: k and v must have a unit stride on head_dim")
    keep = [k, v]
    c = _cache_arg(cache, k.shape[0], k.dtype, k.shape[3], block_table, keep)
    r = _lib.Kv4Rows()
    r.batch, r.max_rows = k.shape[0], k.shape[1]
    r.k, r.v = k.data_ptr(), v.data_ptr()
    r.k_stride[:], r.v_stride[:] = k.stride()[:3], v.stride()[:3]
    r.start = _int_arg("start", start, k.shape[0], k.device, keep)
    r.lens = _int_arg("lens", lens, k.shape[0], k.device, keep)
    with torch.cuda.device(k.device):
        stream = torch.cuda.current_stream(k.device).cuda_stream
        _lib.check(getattr(_lib.load(), fn)(ctypes.byref(c), ctypes.byref(r), ctypes.c_void_p(stream)))


def kv4_store(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, start: Optional[torch.Tensor] = None,
              lens: Optional[torch.Tensor] = None, block_table: Optional[torch.Tensor] = None) -> None:
    """Quantises k, v [batch, rows, n_kv_heads, head_dim] into the cache: row
    i < lens[b] (all rows without ``lens``) becomes token start[b] + i of
    sequence b (i without ``start``).  Other tokens are left as they were.
    Rows that one call sends to the same place leave an undefined mix there."""
    ext = ops._extension()
    if ext is not None:
        ext.kv4_store(cache, k, v, start=start, lens=lens, block_table=block_table)
    else:
        _rows_call("llmx_kv4_store", cache, k, v, start, lens, block_table)


def kv4_load(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, start: Optional[torch.Tensor] = None,
             lens: Optional[torch.Tensor] = None, block_table: Optional[torch.Tensor] = None) -> None:
    """Reads tokens back into k, v [batch, rows, n_kv_heads, head_dim]: row i <
    lens[b] gets token start[b] + i of sequence b (n s + m in fp32, rounded to
    the dtype), the rows behind get 0."""
    ext = ops._extension()
    if ext is not None:
        ext.kv4_load(cache, k, v, start=start, lens=lens, block_table=block_table)
    else:
        _rows_call("llmx_kv4_load", cache, k, v, start, lens, block_table)


def kv4_attention(output: torch.Tensor, q: torch.Tensor, cache: torch.Tensor, sm_scale: float, sliding_window: int = -1,
                  logits_soft_cap: float = 0.0, *, kv_lens: Optional[torch.Tensor] = None,
                  block_table: Optional[torch.Tensor] = None, q_lens: Optional[torch.Tensor] = None,
                  alibi_slopes: Optional[torch.Tensor] = None, causal: bool = True, lse: Optional[torch.Tensor] = None,
                  algo: str = "auto", max_kv_len: int = 0) -> None:
    """Writes attention of q [batch, q_len, n_heads, head_dim] over the cached
    sequences into ``output``, with the masks, ALiBi, soft-cap and lse of
    ``single_mha_attention_half``.

    ``max_kv_len`` (0: all the table can hold) bounds kv_lens where the caller
    knows a bound: the work is split by it.  ``algo``: "decode" reads the 4-bit
    tiles directly (any q_len), "tcgen05" expands the sequences to 16 bits in
    a workspace and runs the tensor-core prefill, "auto" takes the latter for
    long query blocks."""
    ext = ops._extension()
    if ext is not None:
        ext.kv4_attention(output, q, cache, float(sm_scale), int(sliding_window), float(logits_soft_cap), kv_lens=kv_lens,
                          block_table=block_table, q_lens=q_lens, alibi_slopes=alibi_slopes, causal=bool(causal), lse=lse,
                          algo=algo, max_kv_len=int(max_kv_len))
        return
    kv4_attention_ctypes(output, q, cache, sm_scale, sliding_window, logits_soft_cap, kv_lens=kv_lens,
                         block_table=block_table, q_lens=q_lens, alibi_slopes=alibi_slopes, causal=causal, lse=lse,
                         algo=algo, max_kv_len=max_kv_len)


def kv4_attention_ctypes(output, q, cache, sm_scale, sliding_window=-1, logits_soft_cap=0.0, *, kv_lens=None,
                         block_table=None, q_lens=None, alibi_slopes=None, causal=True, lse=None, algo="auto",
                         max_kv_len=0) -> None:
    """The same op through ctypes over the C ABI (no compiled binding needed)."""
    _req(q.dim() == 4 and output.dim() == 4, "kv4: q must be [batch, q_len, n_heads, head_dim]")
    _req(output.dtype == q.dtype and tuple(output.shape) == tuple(q.shape), "output must have the shape and dtype of q")
    _req(q.is_cuda and output.is_cuda and q.device == output.device == cache.device,
         "q, output and cache must be on one CUDA device")
    _req(output.stride(-1) == 1, "output must have a unit stride on head_dim")
    if q.stride(-1) != 1:
        q = q.contiguous()
    B, Sq, H, D = q.shape
    if q.numel() == 0:
        return
    keep = [q, output]
    c = _cache_arg(cache, B, q.dtype, D, block_table, keep)
    p = _lib.AttnParams()
    _lib.check(_lib.load().llmx_attn_params_init(ctypes.byref(p)))
    p.dtype = c.dtype
    p.batch, p.n_heads, p.n_kv_heads, p.head_dim = B, H, c.n_kv_heads, D
    p.max_q_len, p.max_kv_len = Sq, int(max_kv_len) if max_kv_len > 0 else c.max_pages * c.page_size
    p.algo = _lib.ALGO[algo]
    p.q, p.o = q.data_ptr(), output.data_ptr()
    p.q_stride[:], p.o_stride[:] = q.stride()[:3], output.stride()[:3]
    p.q_lens = _int_arg("q_lens", q_lens, B, q.device, keep)
    p.kv_lens = _int_arg("kv_lens", kv_lens, B, q.device, keep)
    if alibi_slopes is not None:
        _req(alibi_slopes.is_cuda and alibi_slopes.device == q.device, "alibi_slopes must be on q's device")
        a = alibi_slopes.to(torch.float32).contiguous()
        _req(a.numel() == H, "alibi_slopes must have n_heads elements")
        keep.append(a)
        p.alibi_slopes = a.data_ptr()
    if lse is not None:
        _req(lse.dtype == torch.float32 and lse.is_contiguous() and tuple(lse.shape) == (B, H, Sq)
             and lse.device == q.device, "lse must be contiguous fp32 [batch, n_heads, max_q_len] on q's device")
        p.lse = lse.data_ptr()
    p.sm_scale, p.causal = float(sm_scale), 1 if causal else 0
    p.sliding_window, p.logits_soft_cap = int(sliding_window), float(logits_soft_cap)
    lib = _lib.load()
    with torch.cuda.device(q.device):
        ws = ctypes.c_size_t(0)
        _lib.check(lib.llmx_kv4_attn_workspace_size(ctypes.byref(p), ctypes.byref(c), ctypes.byref(ws)))
        if ws.value:
            buf = torch.empty(ws.value, dtype=torch.uint8, device=q.device)
            keep.append(buf)
            p.workspace, p.workspace_bytes = buf.data_ptr(), ws.value
        stream = torch.cuda.current_stream(q.device).cuda_stream
        _lib.check(lib.llmx_kv4_attn_fwd(ctypes.byref(p), ctypes.byref(c), ctypes.c_void_p(stream)))
