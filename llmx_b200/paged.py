"""Paged key/value cache in 16 bits: storing rows, attention of new tokens over
it, the weight that each cached token gets, and eviction by that weight.

K and V are two CUDA tensors [n_pages, n_kv_heads, page_size, head_dim]
(``paged_empty``; any strides with a unit one on head_dim, so a cache kept as
[n_pages, page_size, n_kv_heads, head_dim] is passed transposed), fp16 or bf16,
head_dim 64, 128 or 256, page_size a multiple of 16.  ``block_table`` (CUDA
int32 [batch, max_pages]) names the pages of each sequence; without one sequence
b owns pages b * max_pages .., max_pages = n_pages / batch.

    k_cache, v_cache = paged_empty(n_pages, n_kv_heads, head_dim, page_size)
    paged_store(k_cache, v_cache, k, v, start=lens_before, block_table=table)   # [B, S, H_kv, D]
    paged_attention(out, q, k_cache, v_cache, sm_scale, kv_lens=lens, block_table=table)

The new tokens' rows are stored first; q [B, S, H, D] are their queries, S = 1
for a decode step, a few for proposed tokens, a chunk of a prompt.

    weights = paged_weights(k_cache)                                            # fp32, in the same pages
    paged_attention(..., key_weights=weights)                                   # adds each token's attention
    kept, lens = paged_evict(k_cache, v_cache, weights, budget, kv_lens=lens, block_table=table, recent=64)

Everything runs on torch's current stream of the tensors' device.  What a page
holds behind a sequence's length is never used.  A table entry or position
outside the cache is not followed (it reads as zeros and is not written) and is
reported by ``device_status``.  The calls go through the C++ torch binding
(llmx_b200.llmx_bind) when it is built, else through ctypes.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib, ops
from .kv4 import _int_arg
from .ops import _TORCH_DTYPE, _req


def paged_empty(n_pages: int, n_kv_heads: int, head_dim: int, page_size: int = 64, dtype: torch.dtype = torch.bfloat16,
                device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """Uninitialised K and V of ``n_pages`` pages of ``page_size`` tokens."""
    _req(head_dim in (64, 128, 256), "paged: head_dim must be 64, 128 or 256")
    _req(page_size >= 16 and page_size % 16 == 0, "paged: page_size must be a multiple of 16")
    _req(n_pages >= 1 and n_kv_heads >= 1, "paged: n_pages and n_kv_heads must be >= 1")
    _req(dtype in (torch.float16, torch.bfloat16), "paged: only float16 and bfloat16 are supported")
    shape = (n_pages, n_kv_heads, page_size, head_dim)
    return torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)


def paged_weights(k_cache: torch.Tensor) -> torch.Tensor:
    """Key weights of 0 for every place of a cache."""
    return torch.zeros(k_cache.shape[:3], dtype=torch.float32, device=k_cache.device)


def _cache_arg(k: torch.Tensor, v: torch.Tensor, batch: int, block_table, key_weights, keep):
    _req(k.dim() == 4 and v.dim() == 4 and tuple(k.shape) == tuple(v.shape),
         "paged: the cache must be two tensors [n_pages, n_kv_heads, page_size, head_dim]")
    _req(k.is_cuda and k.device == v.device, "paged: the cache must be on one CUDA device")
    _req(k.dtype == v.dtype and k.dtype in (torch.float16, torch.bfloat16),
         "paged: only float16 and bfloat16 are supported")
    _req(k.stride(3) == 1 and v.stride(3) == 1, "paged: the cache must have a unit stride on head_dim")
    c = _lib.PagedCache()
    c.dtype = _lib.DTYPE[_TORCH_DTYPE[k.dtype]]
    c.n_pages, c.n_kv_heads, c.page_size, c.head_dim = k.shape
    c.k, c.v = k.data_ptr(), v.data_ptr()
    c.k_stride[:], c.v_stride[:] = k.stride()[:3], v.stride()[:3]
    if block_table is None:
        _req(batch == 0 or k.shape[0] >= batch, "paged: without a block_table the cache needs a page per sequence")
        c.max_pages = k.shape[0] // max(batch, 1)
    else:
        block_table = _table_arg("block_table", block_table, batch, k.device, keep)
        c.max_pages = block_table.shape[1]
        c.block_table, c.table_stride = block_table.data_ptr(), block_table.stride(0)
    if key_weights is not None:
        _req(key_weights.dtype == torch.float32 and tuple(key_weights.shape) == tuple(k.shape[:3])
             and key_weights.device == k.device and key_weights.stride(2) == 1,
             "paged: key_weights must be fp32 [n_pages, n_kv_heads, page_size] on the cache's device, unit stride on tokens")
        c.key_weights = key_weights.data_ptr()
        c.w_stride[:] = key_weights.stride()[:2]
    return c


def _table_arg(name, table, batch, device, keep):
    _req(table.is_cuda and table.device == device, f"paged: {name} must be on the cache's device")
    _req(table.dtype == torch.int32 and table.dim() == 2 and table.shape[0] == batch and table.shape[1] >= 1,
         f"paged: {name} must be int32 [batch, max_pages]")
    if table.stride(1) != 1:
        table = table.contiguous()
    keep.append(table)
    return table


def paged_store(k_cache: torch.Tensor, v_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                start: Optional[torch.Tensor] = None, lens: Optional[torch.Tensor] = None,
                block_table: Optional[torch.Tensor] = None) -> None:
    """Copies k, v [batch, rows, n_kv_heads, head_dim] into the cache: row i <
    lens[b] (all rows without ``lens``) becomes token start[b] + i of sequence b
    (i without ``start``).  Other tokens are left as they were.  Rows that one
    call sends to the same place leave an undefined mix there."""
    ext = ops._extension()
    if ext is not None:
        ext.paged_store(k_cache, v_cache, k, v, start=start, lens=lens, block_table=block_table)
    else:
        paged_store_ctypes(k_cache, v_cache, k, v, start=start, lens=lens, block_table=block_table)


def paged_store_ctypes(k_cache, v_cache, k, v, *, start=None, lens=None, block_table=None) -> None:
    """The same op through ctypes over the C ABI (no compiled binding needed)."""
    _req(k.dim() == 4 and tuple(k.shape) == tuple(v.shape), "paged: k and v must be [batch, rows, n_kv_heads, head_dim]")
    _req(k.dtype == v.dtype == k_cache.dtype, "paged: k and v must have the cache's dtype")
    _req(k.device == v.device == k_cache.device, "paged: k, v and the cache must be on one CUDA device")
    _req(k_cache.dim() == 4 and k.shape[2] == k_cache.shape[1] and k.shape[3] == k_cache.shape[3],
         "paged: k and v must have the cache's n_kv_heads and head_dim")
    k, v = (x if x.stride(-1) == 1 else x.contiguous() for x in (k, v))
    keep = [k, v]
    c = _cache_arg(k_cache, v_cache, k.shape[0], block_table, None, keep)
    r = _lib.Kv4Rows()
    r.batch, r.max_rows = k.shape[0], k.shape[1]
    r.k, r.v = k.data_ptr(), v.data_ptr()
    r.k_stride[:], r.v_stride[:] = k.stride()[:3], v.stride()[:3]
    r.start = _int_arg("start", start, k.shape[0], k.device, keep)
    r.lens = _int_arg("lens", lens, k.shape[0], k.device, keep)
    with torch.cuda.device(k.device):
        stream = torch.cuda.current_stream(k.device).cuda_stream
        _lib.check(_lib.load().llmx_paged_store(ctypes.byref(c), ctypes.byref(r), ctypes.c_void_p(stream)))


def paged_attention(output: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, sm_scale: float,
                    sliding_window: int = -1, logits_soft_cap: float = 0.0, *, kv_lens: Optional[torch.Tensor] = None,
                    block_table: Optional[torch.Tensor] = None, q_lens: Optional[torch.Tensor] = None,
                    alibi_slopes: Optional[torch.Tensor] = None, causal: bool = True, lse: Optional[torch.Tensor] = None,
                    key_weights: Optional[torch.Tensor] = None, decay: float = 1.0, algo: str = "auto",
                    max_kv_len: int = 0) -> None:
    """Writes attention of q [batch, q_len, n_heads, head_dim] over the cached
    sequences into ``output``, with the masks, ALiBi, soft-cap and lse of
    ``single_mha_attention_half``.

    With ``key_weights`` (fp32 [n_pages, n_kv_heads, page_size]) the weight of
    every token of the sequences becomes ``decay`` times what it was plus the
    softmax weights that the call's query rows, over the query heads of the kv
    head, give it.  The call's own tokens (causal: the last q_lens) had 0
    before, and with ``decay`` 0 all had.

    ``max_kv_len`` (0: all the table can hold) bounds kv_lens where the caller
    knows a bound: the work is split by it.  ``algo``: "decode" streams the cache
    once for every 16 to 64 (row, head) pairs of a kv head, "tcgen05" takes tiles
    of 128, "auto" chooses by the pairs.  ``output`` must not overlap the cache,
    and with ``key_weights`` not q."""
    ext = ops._extension()
    call = ext.paged_attention if ext is not None else paged_attention_ctypes
    call(output, q, k_cache, v_cache, float(sm_scale), int(sliding_window), float(logits_soft_cap), kv_lens=kv_lens,
         block_table=block_table, q_lens=q_lens, alibi_slopes=alibi_slopes, causal=bool(causal), lse=lse,
         key_weights=key_weights, decay=float(decay), algo=algo, max_kv_len=int(max_kv_len))


def paged_attention_ctypes(output, q, k_cache, v_cache, sm_scale, sliding_window=-1, logits_soft_cap=0.0, *, kv_lens=None,
                           block_table=None, q_lens=None, alibi_slopes=None, causal=True, lse=None, key_weights=None,
                           decay=1.0, algo="auto", max_kv_len=0) -> None:
    """The same op through ctypes over the C ABI (no compiled binding needed)."""
    _req(q.dim() == 4 and output.dim() == 4, "paged: q must be [batch, q_len, n_heads, head_dim]")
    _req(output.dtype == q.dtype and tuple(output.shape) == tuple(q.shape), "output must have the shape and dtype of q")
    _req(q.is_cuda and output.is_cuda and q.device == output.device == k_cache.device,
         "q, output and the cache must be on one CUDA device")
    _req(output.stride(-1) == 1, "output must have a unit stride on head_dim")
    _req(k_cache.dim() == 4 and q.dtype == k_cache.dtype and q.shape[3] == k_cache.shape[3],
         "paged: q must have the cache's dtype and head_dim")
    if q.stride(-1) != 1:
        q = q.contiguous()
    B, Sq, H, D = q.shape
    if q.numel() == 0:
        _req(key_weights is None, "paged: key_weights need query rows")
        return
    keep = [q, output]
    c = _cache_arg(k_cache, v_cache, B, block_table, key_weights, keep)
    p = _lib.AttnParams()
    _lib.check(_lib.load().llmx_attn_params_init(ctypes.byref(p)))
    p.dtype = c.dtype
    p.batch, p.n_heads, p.n_kv_heads, p.head_dim = B, H, c.n_kv_heads, D
    room = c.max_pages * c.page_size
    _req(max_kv_len <= room, "max_kv_len must be at most max_pages * page_size")
    p.max_q_len, p.max_kv_len = Sq, int(max_kv_len) if max_kv_len > 0 else min(room, 2 ** 31 - 1)
    _req(algo in ("auto", "decode", "tcgen05"), "paged: algo must be one of auto, decode, tcgen05")
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
    p.sliding_window, p.logits_soft_cap = max(-1, min(int(sliding_window), 2 ** 30)), float(logits_soft_cap)
    lib = _lib.load()
    with torch.cuda.device(q.device):
        ws = ctypes.c_size_t(0)
        _lib.check(lib.llmx_paged_attn_workspace_size(ctypes.byref(p), ctypes.byref(c), ctypes.byref(ws)))
        if ws.value:
            buf = torch.empty(ws.value, dtype=torch.uint8, device=q.device)
            keep.append(buf)
            p.workspace, p.workspace_bytes = buf.data_ptr(), ws.value
        stream = torch.cuda.current_stream(q.device).cuda_stream
        _lib.check(lib.llmx_paged_attn_fwd(ctypes.byref(p), ctypes.byref(c), ctypes.c_float(decay),
                                           ctypes.c_void_p(stream)))


def paged_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, key_weights: torch.Tensor, budget: int, *,
                kv_lens: torch.Tensor, block_table: Optional[torch.Tensor] = None, recent: int = 0, sinks: int = 0,
                out_table: Optional[torch.Tensor] = None, kept: Optional[torch.Tensor] = None,
                new_lens: Optional[torch.Tensor] = None, max_kv_len: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keeps min(kv_lens[b], ``budget``) tokens of each sequence and kv head: the
    first ``sinks``, the last ``recent``, and of the others those of the largest
    ``key_weights`` (of equal ones the earliest; NaN as -inf), in their order.
    Their rows of K, V and weights become tokens 0, 1, .. of the pages of
    ``out_table`` (int32 [batch, pages]; the pages then hold nothing that the
    call reads), or without one of the sequence's own pages (which no other
    sequence may share).

    A token whose page lies outside the cache ranks last and, if kept, becomes
    zeros with weight 0.

    Returns (kept, new_lens): int32 [batch, n_kv_heads, budget], the former
    positions (-1 behind the kept ones), and int32 [batch].  Both may be given;
    ``new_lens`` may be ``kv_lens``."""
    ext = ops._extension()
    call = ext.paged_evict if ext is not None else paged_evict_ctypes
    return call(k_cache, v_cache, key_weights, int(budget), kv_lens=kv_lens, block_table=block_table, recent=int(recent),
                sinks=int(sinks), out_table=out_table, kept=kept, new_lens=new_lens, max_kv_len=int(max_kv_len))


def paged_evict_ctypes(k_cache, v_cache, key_weights, budget, *, kv_lens, block_table=None, recent=0, sinks=0,
                       out_table=None, kept=None, new_lens=None, max_kv_len=0):
    """The same op through ctypes over the C ABI (no compiled binding needed)."""
    _req(1 <= budget < 2 ** 31 and 0 <= recent < 2 ** 31 and 0 <= sinks < 2 ** 31,
         "paged: budget must be >= 1, recent and sinks >= 0")
    _req(kv_lens.dim() == 1, "kv_lens must be [batch]")
    B = kv_lens.numel()
    keep = []
    c = _cache_arg(k_cache, v_cache, B, block_table, key_weights, keep)
    dev = k_cache.device
    if kept is None:
        kept = torch.empty(B, c.n_kv_heads, budget, dtype=torch.int32, device=dev)
    if new_lens is None:
        new_lens = torch.empty(B, dtype=torch.int32, device=dev)
    _req(kept.dtype == torch.int32 and tuple(kept.shape) == (B, c.n_kv_heads, budget) and kept.is_contiguous()
         and kept.device == dev, "paged: kept must be contiguous int32 [batch, n_kv_heads, budget] on the cache's device")
    _req(new_lens.dtype == torch.int32 and tuple(new_lens.shape) == (B,) and new_lens.is_contiguous()
         and new_lens.device == dev, "paged: new_lens must be contiguous int32 [batch] on the cache's device")
    e = _lib.PagedEvictParams()
    room = c.max_pages * c.page_size
    _req(max_kv_len <= room, "max_kv_len must be at most max_pages * page_size")
    e.batch, e.budget, e.recent, e.sinks = B, budget, recent, sinks
    e.max_kv_len = int(max_kv_len) if max_kv_len > 0 else min(room, 2 ** 31 - 1)
    e.kv_lens = _int_arg("kv_lens", kv_lens, B, dev, keep)
    if out_table is not None:
        out_table = _table_arg("out_table", out_table, B, dev, keep)
        e.out_table, e.out_table_stride, e.out_pages = out_table.data_ptr(), out_table.stride(0), out_table.shape[1]
    e.kept, e.new_lens = kept.data_ptr(), new_lens.data_ptr()
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        _lib.check(_lib.load().llmx_paged_evict(ctypes.byref(c), ctypes.byref(e), ctypes.c_void_p(stream)))
    return kept, new_lens
