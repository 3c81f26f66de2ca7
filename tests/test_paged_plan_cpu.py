"""How paged_attention cuts a call (csrc/paged_plan.h), compiled by itself for the host and swept over sizes and bounds:
every launch that a plan leads to has blocks, and every kernel of it has rows to serve."""
import ctypes
import itertools
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-int_b200", "csrc")
FIELDS = ("rows tiles few nt warps row_tiles chunk row_splits cluster tokens_per_tile pairs tile_chunk tile_splits splits "
          "join_blocks bytes").split()
WRAPPER = """
#include "paged_plan.h"
using namespace ti;
extern "C" void plan(int64_t batch, int64_t tokens, int64_t group, int64_t kv_heads, int head_dim, int64_t max_query_len,
                     int64_t max_kv_len, float scale_log2, int64_t* o) {
  const PagedPlan p = make_plan_for_scale(batch, tokens, group, kv_heads, head_dim, max_query_len, max_kv_len, scale_log2);
  const int64_t join = p.splits > 1 ? plan_join(p, batch, tokens, group * kv_heads, group, max_query_len).blocks : -1;
  const int64_t v[] = {p.rows, p.tiles, p.few, p.nt, p.warps, p.row_tiles, p.chunk, p.row_splits, p.cluster, p.tile.tokens_per_tile,
                       p.tile.pairs, p.tile.chunk, p.tile.splits, p.splits, join, partial_bytes(p, tokens, group * kv_heads, head_dim)};
  for (unsigned i = 0; i < sizeof(v) / sizeof(v[0]); ++i) o[i] = v[i];
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(WRAPPER)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, "-o", str(d / "plan.so"), str(d / "plan.cpp")])
    fn = ctypes.CDLL(str(d / "plan.so")).plan
    i64 = ctypes.c_int64
    fn.argtypes = [i64, i64, i64, i64, ctypes.c_int, i64, i64, ctypes.c_float, ctypes.POINTER(i64)]
    fn.restype = None

    def call(*sizes, scale_log2=1e-3):
        out = (i64 * len(FIELDS))()
        fn(*sizes, scale_log2, out)
        return dict(zip(FIELDS, out))
    return call


def calls(max_kv_lens):
    """(batch, tokens, group, kv_heads, head_dim, max_query_len, max_kv_len): single tokens, drafts, prompts, and one prompt
    among single tokens."""
    for batch, group, kv_heads, dim, keys in itertools.product((1, 2, 8, 16, 33, 64, 300, 600), (1, 3, 8, 16, 17, 32, 40, 71, 128, 129),
                                                               (1, 2, 8, 40), (64, 128), max_kv_lens):
        for new in (1, 5, 100, 512, 2048):
            yield batch, batch * new, group, kv_heads, dim, new, keys
            if new > 1:
                yield batch, batch - 1 + new, group, kv_heads, dim, new, keys


def test_every_launch_has_blocks_and_every_kernel_has_rows(plan):
    for sizes in calls((1, 16, 300, 2000, 4000, 8000, 131072)):
        p = plan(*sizes)
        group, new = sizes[2], sizes[5]
        assert p["rows"] or p["tiles"], sizes
        if p["splits"] > 1:
            assert 0 < p["join_blocks"] <= 0x7FFFFFFF, (sizes, p)
        if p["rows"]:
            assert group <= p["few"], (sizes, p)  # a sequence with a single token has `group` rows
            assert p["row_tiles"] >= 1 and p["row_splits"] >= 1, (sizes, p)
        if p["tiles"]:
            assert p["tokens_per_tile"] >= 1 and p["pairs"] >= 1 and p["tile_splits"] >= 1, (sizes, p)
            assert group * new > p["few"], (sizes, p)
        assert p["bytes"] <= 512 << 20, (sizes, p)


def test_the_pieces_cover_the_keys(plan):
    """Bounds from no key at all on (a step whose sequences hold none gives zeros)."""
    for sizes in calls((0, 1, 31, 300, 4000, 131072)):
        p = plan(*sizes)
        keys = sizes[6]
        if p["rows"]:
            assert p["chunk"] > 0 and p["chunk"] % 32 == 0 and p["chunk"] * p["row_splits"] >= keys, (sizes, p)
        if p["tiles"]:
            assert p["tile_chunk"] > 0 and p["tile_chunk"] % 128 == 0 and p["tile_chunk"] * p["tile_splits"] >= keys, (sizes, p)


def test_kernels_read_the_index_arrays_behind_their_wait():
    """A kernel that is launched as a programmatic dependent may start before the writer of query_starts, kv_lens or the
    block table is done; only griddepcontrol.wait orders its reads behind those writes."""
    for name, kernels in (("paged_attention.cu", ("paged_rows_kernel", "paged_combine_kernel")), ("paged_append.cu", ("paged_append_kernel",))):
        with open(os.path.join(CSRC, name)) as f:
            source = f.read()
        for kernel in kernels:
            start = source.index("__global__", source.rindex("template", 0, source.index(kernel + "(const")))
            body = source[start:source.index("\n}\n", start)]
            wait = body.index("grid_dep_wait()")
            for read in ("query_starts[", "kv_lens[", "paged_sequence(", "paged_page(", "rows_of_a_cta<"):
                assert read not in body[:wait], (kernel, read)


def test_steep_scores_are_the_rows_kernels(plan):
    """Factors that the tile kernel's fp32 offset cannot carry: its sequences go to the rows kernel, without more workspace
    than ti_paged_attention_workspace_bytes, which does not know the factor, gives for the sizes."""
    for sizes in calls((0, 300, 4000, 131072)):
        flat = plan(*sizes)
        assert plan(*sizes, scale_log2=4.0) == plan(*sizes, scale_log2=-4.0) == flat
        for scale in (4.1, -23.0, 1.4e20):
            p = plan(*sizes, scale_log2=scale)
            assert p["rows"] and not p["tiles"] and p["bytes"] <= flat["bytes"], (sizes, scale, p)
            assert p["chunk"] > 0 and p["chunk"] * p["row_splits"] >= sizes[6], (sizes, scale, p)
            assert p["row_tiles"] * 8 * p["nt"] >= sizes[2] * sizes[5], (sizes, scale, p)
            assert p["splits"] == 1 or 0 < p["join_blocks"] <= 0x7FFFFFFF, (sizes, scale, p)


def test_workspace_query_of_sizes_that_no_call_accepts():
    """Sizes that ti_paged_attention refuses need no workspace, and no arithmetic on them may end the process."""
    from torch_int import _CUDA as C
    ask = C._c_paged_workspace
    good = dict(batch=2, tokens=2, q_heads=64, kv_heads=8, head_dim=128, max_query_len=1, max_kv_len=131072)
    assert ask(*good.values()) > 0
    huge = (1 << 62, (1 << 63) - 1, -(1 << 63), -1, 0)
    for field in good:
        for bad in huge + {"head_dim": (-2, 72), "q_heads": (63, 65536), "kv_heads": (65536, 3), "batch": (65536,),
                           "tokens": (1 << 31,), "max_kv_len": (1 << 30,)}.get(field, ()):
            if field == "max_query_len" and bad > 0:
                continue  # a bound: cut to the tokens
            assert ask(*{**good, field: bad}.values()) == 0, (field, bad)
    for sizes in itertools.product((1 << 62, 1 << 32), repeat=7):
        assert ask(*sizes) == 0
