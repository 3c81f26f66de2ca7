"""Sizes of a paged batch whose products pass 64 bits are refused like other sizes out of range."""
import ctypes

import pytest

from test_paged_cpu import PagedAppendArgs, PagedAttentionArgs, base, batch_of, lib  # noqa: F401 (fixtures)


@pytest.mark.parametrize("change", [dict(num_pages=1 << 60), dict(num_pages=1 << 62), dict(table_width=1 << 60, table_stride=1 << 60),
                                    dict(table_width=(1 << 63) - 1, table_stride=(1 << 63) - 1)])
def test_products_beyond_64_bits_are_refused(lib, base, change):  # noqa: F811
    b = batch_of(base, **change)
    att = PagedAttentionArgs(q=base, ld_q=256, q_heads=4, max_kv_len=64, out=base, out_kind=0)  # (no valid call: none may launch)
    app = PagedAppendArgs(k=base, v=base, ld_k=128, ld_v=128, dtype=4)
    assert lib.ti_paged_attention(ctypes.byref(b), ctypes.byref(att), None) == -1 and b"out of range" in lib.ti_last_error()
    assert lib.ti_paged_append(ctypes.byref(b), ctypes.byref(app), None) == -1 and b"out of range" in lib.ti_last_error()
