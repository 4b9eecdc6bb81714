"""The paged 16-bit cache without a GPU: host-side checks of its entry points
(nothing is launched: a refused call returns before any device work) and the C
structures."""
import ctypes
import shutil
import subprocess
import os

import pytest
import torch

import llmx_b200
from llmx_b200 import _lib
from oracle import paged as opaged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def cache(**over):
    c = _lib.PagedCache()
    c.dtype, c.n_kv_heads, c.head_dim, c.page_size, c.n_pages, c.max_pages = 2, 2, 128, 64, 10, 4
    c.k, c.v = 0x10000, 0x20000  # never dereferenced on the host
    c.k_stride[:] = c.v_stride[:] = [2 * 64 * 128, 64 * 128, 128]
    c.block_table, c.table_stride = 0x30000, 4
    for k, v in over.items():
        if k in ("k_stride", "v_stride", "w_stride"):
            getattr(c, k)[:] = v
        else:
            setattr(c, k, v)
    return c


def request(**over):
    p = _lib.AttnParams()
    assert _lib.load().llmx_attn_params_init(ctypes.byref(p)) == 0
    p.dtype, p.batch, p.n_heads, p.n_kv_heads, p.head_dim, p.max_q_len, p.max_kv_len = 2, 2, 8, 2, 128, 1, 256
    p.q, p.o, p.sm_scale = 0x40000, 0x50000, 0.1
    assert _lib.load().llmx_attn_set_contiguous_strides(ctypes.byref(p)) == 0
    for k, v in over.items():
        if k in ("q_stride", "o_stride"):
            getattr(p, k)[:] = v
        else:
            setattr(p, k, v)
    return p


def rows(**over):
    r = _lib.Kv4Rows()
    r.batch, r.max_rows, r.k, r.v = 2, 3, 0x60000, 0x70000
    r.k_stride[:] = r.v_stride[:] = [3 * 256, 256, 128]
    for k, v in over.items():
        setattr(r, k, v)
    return r


def evict(**over):
    e = _lib.PagedEvictParams()
    e.batch, e.budget, e.recent, e.sinks, e.max_kv_len = 2, 64, 8, 2, 256
    e.kv_lens, e.kept, e.new_lens = 0x80000, 0x90000, 0xa0000
    for k, v in over.items():
        setattr(e, k, v)
    return e


def message():
    return _lib.load().llmx_attn_last_error().decode()


BAD_CACHES = [
    (dict(dtype=0), 2, "fp16 or bf16"), (dict(head_dim=96), 2, "head_dim"), (dict(n_kv_heads=0), 1, "n_kv_heads"),
    (dict(page_size=24), 1, "multiple of 16"), (dict(page_size=0), 1, "multiple of 16"), (dict(n_pages=0), 1, "n_pages"),
    (dict(max_pages=0), 1, "max_pages"), (dict(max_pages=1 << 28), 1, "2^30"), (dict(k=0), 1, "aligned"),
    (dict(v=0x20008), 1, "aligned"), (dict(k_stride=[2 * 64 * 128, 64 * 128, 124]), 1, "multiples of 8"),
    (dict(v_stride=[-16384, 64 * 128, 128]), 1, ">= 0"), (dict(k_stride=[2 * 64 * 128, 64 * 128, 120]), 1, "overlap"),
    (dict(k_stride=[0, 64 * 128, 128]), 1, "overlap"), (dict(v_stride=[64 * 128, 64 * 128, 128]), 1, "overlap"),
    (dict(v_stride=[1 << 60, 64 * 128, 128]), 1, "strides"), (dict(table_stride=-1), 1, "table_stride"),
    (dict(block_table=0, max_pages=6), 1, "without a block table"),
    (dict(key_weights=0xb0008, w_stride=[128, 64]), 1, "key_weights"),
    (dict(key_weights=0xb0000, w_stride=[126, 64]), 1, "multiples of 4"),
    (dict(key_weights=0xb0000, w_stride=[64, 64]), 1, "key_weights"),
]


@pytest.mark.parametrize("over,status,text", BAD_CACHES, ids=lambda x: str(x)[:40])
def test_bad_caches_are_refused_by_every_entry_point(over, status, text):
    lib, c = _lib.load(), cache(**over)
    n = ctypes.c_size_t(0)
    p = request(dtype=over.get("dtype", 2), head_dim=over.get("head_dim", 128), max_kv_len=64)
    if "n_kv_heads" not in over:
        for call in (lambda: lib.llmx_paged_attn_fwd(ctypes.byref(p), ctypes.byref(c), 1.0, None),
                     lambda: lib.llmx_paged_attn_workspace_size(ctypes.byref(p), ctypes.byref(c), ctypes.byref(n))):
            assert call() == status and text in message()
    assert lib.llmx_paged_store(ctypes.byref(c), ctypes.byref(rows()), None) == status and text in message()
    assert lib.llmx_paged_evict(ctypes.byref(c), ctypes.byref(evict()), None) == status and text in message()


@pytest.mark.parametrize("over,status,text", [
    (dict(n_kv_heads=4), 1, "cache's"), (dict(dtype=1), 1, "cache's"), (dict(head_dim=64), 1, "cache's"),
    (dict(kv_offset=1), 1, "kv_offset"), (dict(kv_total=9), 1, "kv_offset"), (dict(max_kv_len=257), 1, "max_kv_len"),
    (dict(algo=1), 2, "algo"), (dict(algo=7), 1, "algo"), (dict(q=0x40008), 2, "aligned"), (dict(o=0x50002), 2, "aligned"),
    (dict(q_stride=[1024, 1024, 132]), 2, "multiples of 8"), (dict(o_stride=[0, 1024, 128]), 1, "overlap"),
    (dict(o_stride=[1024, 1024, 0]), 1, "overlap"), (dict(max_q_len=1 << 29), 1, "2^30"), (dict(q=0), 1, "NULL"),
    (dict(sm_scale=float("inf")), 1, "sm_scale"), (dict(workspace=0xc0008, workspace_bytes=16), 1, "workspace"),
    (dict(algo=3, sm_scale=-1.0), 2, "sm_scale"),
])
def test_bad_requests_are_refused(over, status, text):
    lib = _lib.load()
    p, c = request(**over), cache()
    assert lib.llmx_paged_attn_fwd(ctypes.byref(p), ctypes.byref(c), 1.0, None) == status
    assert text in message()


def test_null_arguments_are_refused():
    lib = _lib.load()
    n = ctypes.c_size_t(0)
    p, c = request(), cache()
    assert lib.llmx_paged_attn_fwd(None, ctypes.byref(c), 1.0, None) == 1
    assert lib.llmx_paged_attn_fwd(ctypes.byref(p), None, 1.0, None) == 1
    assert lib.llmx_paged_attn_workspace_size(ctypes.byref(p), ctypes.byref(c), None) == 1
    assert lib.llmx_paged_attn_workspace_size(ctypes.byref(p), None, ctypes.byref(n)) == 1
    assert lib.llmx_paged_store(None, ctypes.byref(rows()), None) == 1
    assert lib.llmx_paged_store(ctypes.byref(c), None, None) == 1
    assert lib.llmx_paged_evict(ctypes.byref(c), None, None) == 1


@pytest.mark.parametrize("decay", [float("nan"), float("inf"), -1.0])
def test_bad_decay_is_refused(decay):
    p, c = request(), cache(key_weights=0xb0000, w_stride=[128, 64])
    assert _lib.load().llmx_paged_attn_fwd(ctypes.byref(p), ctypes.byref(c), decay, None) == 1
    assert "decay" in message()


def test_output_over_q_is_refused_with_weights():
    p, c = request(o=0x40000), cache(key_weights=0xb0000, w_stride=[128, 64])
    assert _lib.load().llmx_paged_attn_fwd(ctypes.byref(p), ctypes.byref(c), 1.0, None) == 1
    assert "read again" in message()


@pytest.mark.parametrize("over", [dict(batch=-1), dict(max_rows=-1), dict(k=0), dict(v=0)])
def test_bad_rows_are_refused(over):
    assert _lib.load().llmx_paged_store(ctypes.byref(cache()), ctypes.byref(rows(**over)), None) == 1


def test_nothing_to_store_or_evict_is_no_error():
    lib = _lib.load()
    assert lib.llmx_paged_store(ctypes.byref(cache()), ctypes.byref(rows(batch=0)), None) == 0
    assert lib.llmx_paged_store(ctypes.byref(cache()), ctypes.byref(rows(max_rows=0)), None) == 0
    c = cache(key_weights=0xb0000, w_stride=[128, 64])
    assert lib.llmx_paged_evict(ctypes.byref(c), ctypes.byref(evict(batch=0)), None) == 0


@pytest.mark.parametrize("over,text", [
    (dict(batch=-1), "batch"), (dict(budget=0), "budget"), (dict(recent=-1), "budget"), (dict(sinks=-1), "budget"),
    (dict(recent=40, sinks=25), "budget"), (dict(max_kv_len=0), "max_kv_len"), (dict(max_kv_len=257), "max_kv_len"),
    (dict(kv_lens=0), "kv_lens"), (dict(kept=0), "kept"), (dict(new_lens=0), "new_lens"),
    (dict(out_table=0xd0000, out_pages=0), "out_pages"), (dict(out_table=0xd0000, out_pages=1, out_table_stride=-1), "stride"),
    (dict(out_table=0xd0000, out_pages=1, budget=65), "out_table must hold"),
])
def test_bad_evictions_are_refused(over, text):
    c = cache(key_weights=0xb0000, w_stride=[128, 64])
    assert _lib.load().llmx_paged_evict(ctypes.byref(c), ctypes.byref(evict(**over)), None) == 1
    assert text in message()


def test_eviction_needs_weights():
    assert _lib.load().llmx_paged_evict(ctypes.byref(cache()), ctypes.byref(evict()), None) == 1
    assert "key_weights" in message()


def test_struct_layouts_match_c(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    cases = {"llmx_paged_cache": _lib.PagedCache, "llmx_paged_evict_params": _lib.PagedEvictParams}
    lines = []
    for name, cls in cases.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "llmx_attn.h"\nint main(void){' + "".join(lines)
                   + "return 0;}\n")
    subprocess.run([gcc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    for line in filter(None, out):
        name, field, value = line.split()
        cls = cases[name]
        assert (ctypes.sizeof(cls) if field == "size" else getattr(cls, field).offset) == int(value), line


@pytest.mark.parametrize("kw", [dict(page_size=8), dict(page_size=24), dict(head_dim=80), dict(n_pages=0), dict(n_kv_heads=0),
                                dict(dtype=torch.float32)])
def test_empty_refuses_bad_caches(kw):
    args = dict(n_pages=4, n_kv_heads=2, head_dim=64, device="cpu")
    args.update(kw)
    with pytest.raises(RuntimeError):
        llmx_b200.paged_empty(**args)


def test_cpu_tensors_are_refused():
    k, v = llmx_b200.paged_empty(4, 2, 64, device="cpu")
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        llmx_b200.paged_store(k, v, torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        llmx_b200.paged_attention(torch.empty_like(q), q, k, v, 1.0)
    with pytest.raises(RuntimeError):
        llmx_b200.paged_evict(k, v, llmx_b200.paged_weights(k), 4, kv_lens=torch.tensor([3], dtype=torch.int32))


def test_oracle_attention_agrees_with_torch():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h, 64, generator=g).half() for n, h in ((5, 4), (9, 2), (9, 2)))
    out, lse, w, *_ = opaged.attention(q, k, v, 5, 9, sm_scale=0.125)
    mask = torch.arange(9) <= torch.arange(5)[:, None] + 4
    kk, vv = (x.double().repeat_interleave(2, 1).transpose(0, 1) for x in (k, v))
    ref = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), kk, vv, attn_mask=mask, scale=0.125)
    assert (out.transpose(0, 1) - ref).abs().max() < 1e-12
    assert (w.sum(-1) - 10).abs().max() < 1e-12 and w.shape == (2, 9)


def test_oracle_keeps_sinks_recent_and_the_heaviest():
    assert opaged.kept([5, 1, 3, 3, 0, 2, 9, 1], 8, 5, 2, 1) == [0, 2, 3, 6, 7]
    assert opaged.kept([1.0] * 6, 6, 3, 1, 0) == [0, 1, 5]
    assert opaged.kept([1.0] * 3, 3, 3, 0, 0) == [0, 1, 2]
