"""Host side of the paged int8 cache operators, without a GPU: argument checks of the C ABI and of the Python entry
points, the workspace query, the rotary table, and the oracle against a direct formula."""
import ctypes
import math
import os

import pytest
import torch

from oracle import paged as P
from torch_int import _CUDA as C
from torch_int.functional import paged as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "torch-int_b200", "torch_int", "lib", "libtorch_int_b200.so")


I_, F_, P_ = ctypes.c_int64, ctypes.c_float, ctypes.c_void_p


class PagedBatch(ctypes.Structure):
    # struct ti_paged_batch
    _fields_ = [
        ("k_pages", P_), ("v_pages", P_), ("block_table", P_), ("query_starts", P_), ("kv_lens", P_),
        ("num_pages", I_), ("kv_heads", I_), ("page_size", I_), ("head_dim", I_),
        ("table_stride", I_), ("table_width", I_), ("batch", I_), ("tokens", I_), ("max_query_len", I_),
    ]


class PagedAppendArgs(ctypes.Structure):
    # struct ti_paged_append_args
    _fields_ = [
        ("q", P_), ("k", P_), ("v", P_), ("ld_q", I_), ("ld_k", I_), ("ld_v", I_), ("q_heads", I_),
        ("rotary", P_), ("rotary_rows", I_), ("rotary_dim", I_), ("q_out", P_),
        ("q_alpha", F_), ("k_alpha", F_), ("v_alpha", F_), ("dtype", ctypes.c_int32), ("interleaved", ctypes.c_int32),
    ]


class PagedAttentionArgs(ctypes.Structure):
    # struct ti_paged_attention_args
    _fields_ = [
        ("q", P_), ("ld_q", I_), ("q_heads", I_), ("max_kv_len", I_), ("out", P_), ("workspace", P_),
        ("workspace_bytes", I_), ("alpha_qk", F_), ("alpha_pv", F_), ("out_kind", ctypes.c_int32),
    ]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    lib.ti_last_error.restype = ctypes.c_char_p
    return lib


@pytest.fixture(scope="module")
def base():
    buf = ctypes.create_string_buffer(1 << 16)
    base.keep = buf
    return (ctypes.addressof(buf) + 63) & ~63


def batch_of(base, **kw):
    b = dict(k_pages=base, v_pages=base, block_table=base, query_starts=base, kv_lens=base, num_pages=4, kv_heads=2,
             page_size=16, head_dim=64, table_stride=4, table_width=4, batch=2, tokens=3, max_query_len=2)
    b.update(kw)
    return PagedBatch(**b)


@pytest.mark.parametrize("change,words", [
    (dict(head_dim=96), b"head_dim"), (dict(page_size=24), b"page_size"), (dict(page_size=8), b"page_size"),
    (dict(kv_heads=0), b"out of range"), (dict(num_pages=0), b"out of range"), (dict(num_pages=1 << 31), b"out of range"),
    (dict(table_width=0), b"out of range"), (dict(table_stride=3), b"out of range"), (dict(batch=70000), b"out of range"),
    (dict(tokens=-1), b"out of range"), (dict(max_query_len=-1), b"out of range"), (dict(k_pages=None), b"null pointer"),
    (dict(kv_lens=None), b"null pointer"), (dict(v_pages=8), b"aligned"), (dict(query_starts=2), b"aligned"),
])
def test_bad_batches_are_refused(lib, base, change, words):
    """Before any CUDA call, by both entry points."""
    b = batch_of(base, **{k: (base + v if k in ("v_pages", "query_starts") else v) for k, v in change.items()})
    att = PagedAttentionArgs(q=base, ld_q=256, q_heads=4, max_kv_len=64, out=base, out_kind=1)
    app = PagedAppendArgs(k=base, v=base, ld_k=128, ld_v=128, dtype=3)
    assert lib.ti_paged_attention(ctypes.byref(b), ctypes.byref(att), None) == -1 and words in lib.ti_last_error()
    assert lib.ti_paged_append(ctypes.byref(b), ctypes.byref(app), None) == -1 and words in lib.ti_last_error()


@pytest.mark.parametrize("change,words", [
    (dict(q_heads=3), b"multiple of the key heads"), (dict(q_heads=0), b"multiple of the key heads"),
    (dict(out_kind=0), b"int8, fp16 or bf16"), (dict(out_kind=4), b"int8, fp16 or bf16"), (dict(q=None), b"null"),
    (dict(out=None), b"null"), (dict(ld_q=250), b"aligned"), (dict(ld_q=128), b"aligned"), (dict(max_kv_len=-1), b"max_kv_len"),
    (dict(max_kv_len=1 << 20), b"workspace"), (dict(max_kv_len=1 << 30), b"max_kv_len"),
    (dict(alpha_qk=float("nan")), b"finite"), (dict(alpha_qk=-1e21), b"finite"), (dict(alpha_pv=float("inf")), b"finite"),
])
def test_bad_attention_arguments_are_refused(lib, base, change, words):
    a = dict(q=base, ld_q=256, q_heads=4, max_kv_len=64, out=base, out_kind=1, alpha_qk=1.0, alpha_pv=1.0)
    a.update(change)
    args = PagedAttentionArgs(**a)
    rc = lib.ti_paged_attention(ctypes.byref(batch_of(base)), ctypes.byref(args), None)
    assert rc == (-4 if words == b"workspace" else -1) and words in lib.ti_last_error()


@pytest.mark.parametrize("change,words", [
    (dict(dtype=4), b"input type"), (dict(k=None), b"null"), (dict(q="base", q_heads=4), b"null"), (dict(ld_k=120), b"aligned"),
    (dict(ld_v=64), b"aligned"), (dict(rotary="base", rotary_dim=72, rotary_rows=9), b"rotary_dim"),
    (dict(rotary="base", rotary_dim=80, rotary_rows=9), b"rotary_dim"), (dict(rotary="base", rotary_dim=64), b"rotary"),
])
def test_bad_append_arguments_are_refused(lib, base, change, words):
    a = dict(k=base, v=base, ld_k=128, ld_v=128, dtype=3, k_alpha=1.0, v_alpha=1.0)
    a.update({k: (base if v == "base" else v) for k, v in change.items()})
    args = PagedAppendArgs(**a)
    assert lib.ti_paged_append(ctypes.byref(batch_of(base)), ctypes.byref(args), None) == -1
    assert words in lib.ti_last_error()


def test_null_descriptors_and_empty_calls(lib, base):
    att = PagedAttentionArgs(q=base, ld_q=256, q_heads=4, max_kv_len=64, out=base, out_kind=1)
    app = PagedAppendArgs(k=base, v=base, ld_k=128, ld_v=128, dtype=3)
    assert lib.ti_paged_attention(None, ctypes.byref(att), None) == -1
    assert lib.ti_paged_append(ctypes.byref(batch_of(base)), None, None) == -1
    for kw in (dict(tokens=0), dict(batch=0), dict(max_query_len=0)):  # accepted, nothing launched
        b = batch_of(base, **kw)
        assert lib.ti_paged_attention(ctypes.byref(b), ctypes.byref(att), None) == 0
        assert lib.ti_paged_append(ctypes.byref(b), ctypes.byref(app), None) == 0


def test_packed_descriptors_match_the_structs():
    """The bytes that the Python entry points pass are those of the C structs, field by field."""
    n = range(1, 15)
    assert C._pack_paged_batch(*n) == bytes(PagedBatch(*n))
    a = (1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 0.5, 0.25, 0.125, 2, 1)
    assert C._pack_paged_append(*a) == bytes(PagedAppendArgs(*a))
    a = (1, 2, 3, 4, 5, 6, 7, 0.5, 0.25, 3)
    assert C._pack_paged_attention(*a) == bytes(PagedAttentionArgs(*a))


def test_workspace_query():
    f = C._c_paged_workspace
    assert f(0, 0, 8, 8, 128, 1, 100) == 0 and f(1, 1, 8, 8, 128, 1, 16) == 0
    one = f(1, 1, 8, 8, 128, 1, 100000)  # one long sequence: split
    assert one > 0 and one % (8 * (128 * 4 + 8)) == 0
    assert f(1, 1, 8, 8, 128, 5, 100000) == one  # the bound is cut to the tokens
    # bounds far above the lengths: at most 512 MB
    for batch, tokens, longest, keys in [(64, 2111, 2048, 131072), (1, 4096, 4096, 1 << 19), (256, 256, 1, 1 << 20), (512, 9000, 64, 1 << 29)]:
        assert 0 <= f(batch, tokens, 64, 8, 128, longest, keys) <= 512 << 20


def test_python_entry_points_refuse_cpu_tensors():
    k = torch.zeros((1, 2, 64), dtype=torch.int8)
    pages = torch.zeros((3, 2, 16, 64), dtype=torch.int8)
    idx = torch.zeros((1, 3), dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), torch.tensor([1], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        C.paged_append(k, k, pages, pages, *idx)
    with pytest.raises(RuntimeError, match="CUDA"):
        C.paged_attention(k, pages, pages, *idx, alpha_qk=1.0, alpha_pv=1.0)
    with pytest.raises(RuntimeError, match="k must be"):
        C.paged_append(k[0], k, pages, pages, *idx)
    with pytest.raises(RuntimeError, match="q must be"):
        C.paged_attention(None, pages, pages, *idx, alpha_qk=1.0, alpha_pv=1.0)


def test_rotary_table():
    t = F.rotary_table(32, 100000, base=10000.0)
    assert t.shape == (100000, 32) and t.dtype == torch.float32
    for p, i in ((0, 0), (7, 3), (99999, 0), (99999, 15)):
        angle = p * 10000.0 ** (-2 * i / 32)
        assert abs(float(t[p, i]) - math.cos(angle)) < 1e-7 and abs(float(t[p, 16 + i]) - math.sin(angle)) < 1e-7
    for bad in (0, 24, -16):
        with pytest.raises(ValueError, match="rotary_dim"):
            F.rotary_table(bad, 10)
    with pytest.raises(ValueError, match="positions"):
        F.rotary_table(16, 0)


def test_oracle_against_a_direct_sum():
    g = torch.Generator().manual_seed(3)
    pages = [torch.randint(-127, 128, (5, 2, 16, 64), generator=g, dtype=torch.int8) for _ in range(2)]
    table = torch.tensor([[4, 1], [2, 0]], dtype=torch.int32)
    q = torch.randint(-127, 128, (3, 4, 64), generator=g, dtype=torch.int8)
    ctx, spread = P.paged_attention(q, *pages, table, [0, 2, 3], [20, 5], 1e-3, 0.5)
    k = lambda b, h, j: pages[0][table[b, j // 16], h, j % 16].double()  # noqa: E731
    v = lambda b, h, j: pages[1][table[b, j // 16], h, j % 16].double()  # noqa: E731
    for b, tok, last in ((0, 0, 18), (0, 1, 19), (1, 2, 4)):
        for h in range(4):
            w = [math.exp(1e-3 * float(q[tok, h].double() @ k(b, h // 2, j))) for j in range(last + 1)]
            want = sum(x * v(b, h // 2, j) for j, x in enumerate(w)) / sum(w) * 0.5
            assert torch.allclose(ctx[tok, h], want, rtol=1e-12, atol=1e-12)
    assert bool((spread >= ctx.abs() - 1e-12).all())


def test_oracle_rotation_preserves_length_and_is_relative():
    """A rotation keeps a pair's length, and products of rotated vectors depend on the difference of positions."""
    table = F.rotary_table(64, 64)
    g = torch.Generator().manual_seed(4)
    x, y = torch.randn((1, 1, 64), generator=g), torch.randn((1, 1, 64), generator=g)
    for inter in (False, True):
        a = [P.rotate(x, table[p:p + 1], inter) for p in (3, 23)]
        c = [P.rotate(y, table[p:p + 1], inter) for p in (10, 30)]
        assert abs(float(a[0].norm() - x.norm())) < 1e-5
        assert abs(float((a[0] * c[0]).sum() - (a[1] * c[1]).sum())) < 1e-4
