"""The 4-bit key/value cache without a GPU: its oracle's own properties, the
host-side checks of its entry points, and the C structures."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import llmx_b200
from llmx_b200 import _lib
from oracle import kv4 as okv4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantiser_properties(dtype):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, 128, generator=g).to(dtype)
    x[0] = 3.0
    x[1] = 0.0
    x[2, 0] = 60000.0 if dtype == torch.float16 else 1e30
    n, s, m = okv4.quantise(x)
    assert int(n.min()) >= 0 and int(n.max()) <= 15
    v, back = okv4.values(x)
    # Every value is within half a step, and one rounding to fp32 of the difference.
    err = (v - x.double()).abs()
    assert (err <= okv4.spread(s) * 0.5 * (1 + 2.0 ** -20)).all()
    # Equal channels come back as they are, and so does each group's minimum.
    assert torch.equal(back[0], x[0]) and torch.equal(back[1], x[1])
    low = x.reshape(200, 2, 64).argmin(-1)
    assert torch.equal(back.reshape(200, 2, 64).gather(-1, low[..., None]), x.reshape(200, 2, 64).gather(-1, low[..., None]))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_group_reads_back_as_nan(bad):
    x = torch.randn(1, 128).to(torch.bfloat16)
    x[0, 5] = bad
    _, back = okv4.values(x)
    assert back[0, :64].isnan().all() and back[0, 64:].isfinite().all()


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_layout_covers_every_byte_of_a_tile_once(head_dim):
    used = torch.zeros(okv4.tile_bytes(head_dim), dtype=torch.int64)
    for tok in range(16):
        for is_v in (False, True):
            for chunk in range(head_dim // 8):
                at = okv4.word_offsets(head_dim, tok, chunk, is_v)
                used[at:at + 4] += 1
            for h in range(head_dim // 64):
                at = okv4.param_offset(head_dim, tok, is_v, h)
                used[at:at + 4] += 1
    assert (used == 1).all()


def test_page_bytes():
    lib = _lib.load()
    n = ctypes.c_int64(0)
    for d in (64, 128, 256):
        assert lib.llmx_kv4_page_bytes(d, 64, ctypes.byref(n)) == 0 and n.value == 4 * 18 * d
    assert lib.llmx_kv4_page_bytes(96, 64, ctypes.byref(n)) == 2
    assert lib.llmx_kv4_page_bytes(128, 24, ctypes.byref(n)) == 1
    assert lib.llmx_kv4_page_bytes(128, 64, None) == 1


def test_struct_layouts_match_c(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    cases = {"llmx_kv4_cache": _lib.Kv4Cache, "llmx_kv4_rows": _lib.Kv4Rows}
    lines = []
    for name, cls in cases.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "llmx_attn.h"\nint main(void){' + "".join(lines)
                   + "return 0;}\n")
    subprocess.run([gcc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        name, field, off = line.split()
        cls = cases[name]
        assert (ctypes.sizeof(cls) if field == "size" else getattr(cls, field).offset) == int(off), line


def _cache(**over):
    c = _lib.Kv4Cache()
    c.dtype, c.n_kv_heads, c.head_dim, c.page_size, c.n_pages, c.max_pages = 2, 2, 128, 64, 8, 4
    c.data, c.page_stride, c.head_stride = 0x10000, 2 * 4 * 18 * 128, 4 * 18 * 128
    c.block_table, c.table_stride = 0x20000, 4
    for k, v in over.items():
        setattr(c, k, v)
    return c


def _rows(**over):
    r = _lib.Kv4Rows()
    r.batch, r.max_rows, r.k, r.v = 2, 5, 0x30000, 0x40000
    r.k_stride[:] = r.v_stride[:] = (5 * 2 * 128, 2 * 128, 128)
    for k, v in over.items():
        setattr(r, k, v)
    return r


def _params(**over):
    p = _lib.AttnParams()
    lib = _lib.load()
    lib.llmx_attn_params_init(ctypes.byref(p))
    p.dtype, p.batch, p.n_heads, p.n_kv_heads, p.head_dim = 2, 2, 8, 2, 128
    p.max_q_len, p.max_kv_len = 1, 256
    p.q, p.o, p.sm_scale = 0x50000, 0x60000, 128 ** -0.5
    lib.llmx_attn_set_contiguous_strides(ctypes.byref(p))
    for k, v in over.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("field,value,status", [
    ("dtype", 0, 2), ("head_dim", 96, 2), ("n_kv_heads", 0, 1), ("page_size", 8, 1), ("page_size", 40, 1),
    ("n_pages", 0, 1), ("max_pages", 0, 1), ("max_pages", 1 << 25, 1), ("data", 0, 1), ("data", 0x10008, 1),
    ("page_stride", -16, 1), ("page_stride", 8, 1), ("page_stride", 16, 1), ("head_stride", 4 * 18 * 128 + 4, 1),
    ("head_stride", 16, 1), ("table_stride", -1, 1),
])
def test_cache_arguments_rejected(field, value, status):
    lib = _lib.load()
    c = _cache(**{field: value})
    for fn in (lib.llmx_kv4_store, lib.llmx_kv4_load):
        assert fn(ctypes.byref(c), ctypes.byref(_rows()), None) == status
        assert lib.llmx_attn_last_error()
    if field not in ("dtype", "n_kv_heads", "head_dim"):
        assert lib.llmx_kv4_attn_fwd(ctypes.byref(_params()), ctypes.byref(c), None) == status


def test_cache_without_a_table_must_hold_every_sequence():
    lib = _lib.load()
    c = _cache(block_table=None, max_pages=5)
    assert lib.llmx_kv4_store(ctypes.byref(c), ctypes.byref(_rows()), None) == 1
    assert b"batch * max_pages" in lib.llmx_attn_last_error()


@pytest.mark.parametrize("field,value", [("batch", -1), ("batch", 70000), ("max_rows", -1), ("k", 0), ("v", 0), ("k", 0x30001)])
def test_row_arguments_rejected(field, value):
    lib = _lib.load()
    for fn in (lib.llmx_kv4_store, lib.llmx_kv4_load):
        assert fn(ctypes.byref(_cache()), ctypes.byref(_rows(**{field: value})), None) == 1
    r = _rows()
    r.v_stride[1] = -1
    assert lib.llmx_kv4_load(ctypes.byref(_cache()), ctypes.byref(r), None) == 1
    assert lib.llmx_kv4_store(None, ctypes.byref(_rows()), None) == 1
    assert lib.llmx_kv4_store(ctypes.byref(_cache()), None, None) == 1


@pytest.mark.parametrize("field,value,status", [
    ("dtype", 1, 1), ("n_kv_heads", 4, 1), ("head_dim", 64, 1), ("max_kv_len", 257, 1), ("max_kv_len", 0, 1),
    ("kv_offset", 4, 1), ("kv_total", 4, 1), ("algo", 1, 2), ("algo", 3, 2), ("algo", 9, 1), ("q", 0x50001, 1), ("q", 0, 1),
    ("sm_scale", float("inf"), 1), ("batch", 0, 1),
])
def test_attention_arguments_rejected(field, value, status):
    lib = _lib.load()
    ws = ctypes.c_size_t(0)
    assert lib.llmx_kv4_attn_workspace_size(ctypes.byref(_params(**{field: value})), ctypes.byref(_cache()), ctypes.byref(ws)) == status
    assert lib.llmx_attn_last_error()


def test_workspace_sizes():
    lib = _lib.load()
    ws = ctypes.c_size_t(0)
    p, c = _params(), _cache()
    assert lib.llmx_kv4_attn_workspace_size(ctypes.byref(p), ctypes.byref(c), ctypes.byref(ws)) == 0
    assert ws.value % (2 * 8 * (128 + 1) * 4) == 0  # whole splits of 2 sequences x 8 heads
    # The expanded form wants both tensors, rounded up to 256 bytes, and the prefill's counter.
    p = _params(max_q_len=8, algo=_lib.ALGO["tcgen05"])
    assert lib.llmx_kv4_attn_workspace_size(ctypes.byref(p), ctypes.byref(c), ctypes.byref(ws)) == 0
    assert ws.value == 2 * 2 * 256 * 2 * 128 * 2 + 256
    assert lib.llmx_kv4_attn_workspace_size(ctypes.byref(p), ctypes.byref(c), None) == 1


def test_auto_form_follows_work_and_room():
    """AUTO expands long query blocks, never into more than 4 GiB; DECODE and short blocks do not."""
    lib = _lib.load()
    ws = ctypes.c_size_t(0)

    def size(algo, q_len, pages):
        p = _params(max_q_len=q_len, algo=_lib.ALGO[algo], n_heads=32, n_kv_heads=8, max_kv_len=pages * 64)
        lib.llmx_attn_set_contiguous_strides(ctypes.byref(p))
        c = _cache(n_kv_heads=8, max_pages=pages, n_pages=2 * pages, page_stride=8 * 4 * 18 * 128)
        assert lib.llmx_kv4_attn_workspace_size(ctypes.byref(p), ctypes.byref(c), ctypes.byref(ws)) == 0
        return ws.value

    expanded = 2 * 2 * 8192 * 8 * 128 * 2 + 256
    assert size("tcgen05", 512, 128) == expanded and size("auto", 512, 128) == expanded
    assert size("auto", 8, 128) == size("decode", 8, 128) < expanded
    assert size("decode", 512, 128) < expanded
    assert size("tcgen05", 512, 16384) > 4 << 30 > size("auto", 512, 16384)
    # More query rows than the direct form counts: AUTO expands whatever it takes, DECODE refuses.
    p = _params(max_q_len=1 << 16, algo=_lib.ALGO["decode"], n_heads=32, n_kv_heads=8, max_kv_len=16384 * 64)
    lib.llmx_attn_set_contiguous_strides(ctypes.byref(p))
    c = _cache(n_kv_heads=8, max_pages=16384, n_pages=32768, page_stride=8 * 4 * 18 * 128)
    assert lib.llmx_kv4_attn_workspace_size(ctypes.byref(p), ctypes.byref(c), ctypes.byref(ws)) == 2
    assert b"too many query rows" in lib.llmx_attn_last_error()
    p.algo = _lib.ALGO["auto"]
    assert lib.llmx_kv4_attn_workspace_size(ctypes.byref(p), ctypes.byref(c), ctypes.byref(ws)) == 0 and ws.value > 4 << 30


def test_python_checks():
    with pytest.raises(RuntimeError, match="head_dim"):
        llmx_b200.kv4_empty(4, 2, 96, device="cpu")
    with pytest.raises(RuntimeError, match="page_size"):
        llmx_b200.kv4_empty(4, 2, 64, page_size=24, device="cpu")
    cache = llmx_b200.kv4_empty(4, 2, 128, device="cpu")
    assert cache.shape == (4, 2, 4, 18 * 128)
    k = torch.zeros(2, 3, 2, 128, dtype=torch.bfloat16)
    for fn in (llmx_b200.kv4_store, llmx_b200.kv4_load):
        with pytest.raises(RuntimeError, match="CUDA"):
            fn(cache, k, k)
        with pytest.raises(RuntimeError, match="batch, rows"):
            fn(cache, k[0], k[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        llmx_b200.kv4_attention(k, k, cache, 1.0)
    from llmx_b200 import kv4

    with pytest.raises(RuntimeError, match="CUDA"):
        kv4.kv4_attention_ctypes(k, k, cache, 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv4._rows_call("llmx_kv4_store", cache, k, k, None, None, None)


def test_sizes_that_the_launches_cannot_number():
    """Tiles of one sequence's rows past 31 bits are refused."""
    lib = _lib.load()
    c = _cache(n_kv_heads=60000, page_stride=60000 * 4 * 18 * 128)
    r = _rows(max_rows=(1 << 31) - 1)
    for fn in (lib.llmx_kv4_store, lib.llmx_kv4_load):
        assert fn(ctypes.byref(c), ctypes.byref(r), None) == 1
        assert b"max_rows" in lib.llmx_attn_last_error()
