"""Refusals and workspace sizes of the paged 16-bit cache at the ends of its ranges, without
a GPU (nothing is launched)."""
import ctypes

import pytest

from llmx_b200 import _lib
from test_paged import cache, message, request


def workspace(p, c):
    n = ctypes.c_size_t(0)
    status = _lib.load().llmx_paged_attn_workspace_size(ctypes.byref(p), ctypes.byref(c), ctypes.byref(n))
    return status, n.value


WEIGHTS = dict(key_weights=0xb0000, w_stride=[128, 64])


@pytest.mark.parametrize("q_len,kv_len", [(4096, 65536), (1 << 22, 1 << 30), (1 << 21, 1 << 30), (1 << 10, 1 << 14)])
def test_kept_scores_are_bounded(q_len, kv_len):
    """256 query heads a kv head: every score is kept, 4 bytes each; the product of the sizes may
    pass 64 bits, and is refused, not wrapped."""
    p = request(n_heads=512, max_q_len=q_len, max_kv_len=kv_len, algo=2)
    c = cache(max_pages=max(4, kv_len // 64), table_stride=1 << 24, **WEIGHTS)
    need = 4 * 2 * 2 * 256 * q_len * kv_len
    status, size = workspace(p, c)
    if need > 16 << 30:
        assert status == 2 and "16 GiB" in message()
        assert _lib.load().llmx_paged_attn_fwd(ctypes.byref(p), ctypes.byref(c), 1.0, None) == 2
    else:
        assert status == 0 and need <= size < need + (1 << 30)


def test_scores_are_not_kept_where_they_can_be_computed_again():
    c = cache(max_pages=1 << 10, table_stride=1 << 24, **WEIGHTS)
    p = request(n_heads=256, max_q_len=4096, max_kv_len=65536)  # 128 query heads a kv head
    assert workspace(p, c)[0] == 0 and workspace(p, c)[1] < 1 << 30
    p.algo = 2
    assert workspace(p, c)[0] == 0 and workspace(p, c)[1] < 1 << 30
    p.q_stride[1] = 0  # one row of q for all positions
    assert workspace(p, c)[0] == 2
