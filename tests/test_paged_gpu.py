"""The paged int8 cache operators on the GPU against their 64-bit restatement (oracle/paged.py).

Tolerance of a context, per element.  A probability carries a relative error of at most
  2^-11            its rounding to fp16 (kernel for many rows; the one for few rows splits it and has 2^-21),
  |s| * 2^-22      two roundings of the score s in the log2 domain (|s| < 32 here: 2^-17),
  2^-20            exp2 to 2 ulp, fp32 sums of at most a few thousand terms in tree-like order,
in the numerator, and without the first in the denominator; so the context is off by at most
spread * (2^-11 + 2^-15), spread = |alpha_pv| sum_j p_j |v_j|, before it is rounded once to the output type, which
adds half a step: |value| * finfo.eps / 2 (plus half the smallest subnormal in fp16), or 1/2 for int8."""
import pytest
import torch

from helpers import rand_s8, randn
from oracle import paged as P

pytestmark = pytest.mark.gpu

DT = {"int8": torch.int8, "fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def make_batch(new, keys, kv_heads, page, dim, seed, extra_tokens=0, spare_pages=2):
    """CPU tensors of a ragged batch whose pages are dealt out in random order."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in keys]
    pages = sum(need) + spare_pages
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(keys), max(max(need), 1) + 1), -7, dtype=torch.int32)  # unused entries are never read
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[:n], dtype=torch.int32)
        del order[:n]
    starts = [0]
    for t in new:
        starts.append(starts[-1] + t)
    return {"k_pages": rand_s8((pages, kv_heads, page, dim), seed + 1), "v_pages": rand_s8((pages, kv_heads, page, dim), seed + 2),
            "block_table": table, "query_starts": torch.tensor(starts, dtype=torch.int32),
            "kv_lens": torch.tensor(keys, dtype=torch.int32), "tokens": starts[-1] + extra_tokens}


def cuda(b):
    return {k: (x.cuda() if isinstance(x, torch.Tensor) else x) for k, x in b.items()}


def index_args(b):
    return b["k_pages"], b["v_pages"], b["block_table"], b["query_starts"], b["kv_lens"]


def assert_context(out, ctx, spread, tokens):
    """`out` (GPU) against the 64-bit context by the bound above, for the first `tokens` rows."""
    got, ctx, spread = out[:tokens].double().cpu(), ctx[:tokens], spread[:tokens]
    tol = spread * (2.0 ** -11 + 2.0 ** -15)
    if out.dtype == torch.int8:
        ctx = ctx.clamp(-128, 127)
        tol = tol + 0.5
    else:
        tol = tol + ctx.abs() * (torch.finfo(out.dtype).eps / 2 * 1.001) + 2.0 ** -25
    err = (got - ctx).abs()
    assert bool((err <= tol).all()), f"{int((err > tol).sum())} of {err.numel()} off, worst {float((err / tol.clamp_min(1e-30)).max()):.3g} x the bound"


def run_attention(C, new, keys, heads, kv_heads, page, dim, out_dtype, seed, alpha_qk=None, alpha_pv=0.02, bounds=True):
    b = make_batch(new, keys, kv_heads, page, dim, seed)
    q = rand_s8((b["tokens"], heads, dim), seed + 3)
    alpha_qk = 2.5 / (127 * 127 * dim ** 0.5) if alpha_qk is None else alpha_qk
    want, spread = P.paged_attention(q, *index_args(b), alpha_qk, alpha_pv)
    g = cuda(b)
    limits = {"max_query_len": max(new), "max_kv_len": max(keys)} if bounds else {}
    out = C.paged_attention(q.cuda(), *index_args(g), alpha_qk=alpha_qk, alpha_pv=alpha_pv, out_dtype=out_dtype, **limits)
    assert C.device_status() == 0
    assert_context(out, want, spread, b["tokens"])
    return out, want


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (8, 1), (10, 2), (12, 1)])
@pytest.mark.parametrize("page", [16, 64])
def test_decode(cuda_ops, dim, heads, kv_heads, page):
    """One new token per sequence; lengths of one, around a page's end, odd and split over CTAs."""
    keys = [1, 15, 16, 17, 63, 65, 127, 128, 129, 333, 1000]
    run_attention(cuda_ops, [1] * len(keys), keys, heads, kv_heads, page, dim, torch.float16, 11)


@pytest.mark.parametrize("out", ["int8", "fp16", "bf16"])
@pytest.mark.parametrize("dim", [64, 80, 128])
def test_output_types(cuda_ops, out, dim):
    alpha_pv = 1.5 if out == "int8" else 0.02
    run_attention(cuda_ops, [1, 3, 2], [200, 77, 431], 4, 2, 32, dim, DT[out], 21, alpha_pv=alpha_pv)
    run_attention(cuda_ops, [40, 200, 129], [200, 200, 431], 4, 2, 32, dim, DT[out], 22, alpha_pv=alpha_pv)


@pytest.mark.parametrize("new,keys", [
    ([1], [4099]),                         # one long context: many splits
    ([5, 1, 4, 2], [5, 77, 1029, 2]),      # drafts, some with nothing before them
    ([8, 8, 7], [100, 9, 300]),
    ([17, 16, 9], [17, 500, 260]),         # around a tile of rows
    ([128], [128]), ([127], [255]), ([129], [1000]),
    ([300, 1, 1, 64, 2], [300, 900, 5, 700, 2]),   # a chunk among single tokens
    ([1, 260], [3000, 260]),
])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(2, 2, 128, 16), (8, 2, 64, 128), (5, 1, 80, 32)])
def test_ragged_batches(cuda_ops, new, keys, heads, kv_heads, dim, page):
    run_attention(cuda_ops, new, keys, heads, kv_heads, page, dim, torch.bfloat16, 31)


@pytest.mark.parametrize("heads,kv_heads", [(3, 1), (6, 1), (7, 1), (24, 2), (16, 1), (40, 1), (64, 1)])
def test_groups_of_query_heads(cuda_ops, heads, kv_heads):
    """Shared key heads, groups that divide a tile of rows and groups that do not."""
    run_attention(cuda_ops, [1, 2, 30], [50, 300, 200], heads, kv_heads, 16, 64, torch.float16, 41)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_page_sizes(cuda_ops, page):
    run_attention(cuda_ops, [1, 150, 3], [700, 513, 3], 4, 2, page, 128, torch.float16, 51)


def test_rows_that_see_no_key_give_zero(cuda_ops):
    """Fewer keys than new tokens: the first tokens see nothing; sequences without keys, without tokens."""
    new, keys = [6, 4, 0, 1, 200, 3], [2, 0, 5, 1, 150, 3]
    out, want = run_attention(cuda_ops, new, keys, 4, 2, 16, 64, torch.float16, 61)
    first = torch.cat([out[0:4], out[6:10], out[11:61]])
    assert bool((first == 0).all())


def test_default_bounds_and_tight_bounds_agree(cuda_ops):
    a, _ = run_attention(cuda_ops, [1, 1], [300, 41], 4, 4, 16, 64, torch.float16, 71, bounds=False)
    b, _ = run_attention(cuda_ops, [1, 1], [300, 41], 4, 4, 16, 64, torch.float16, 71, bounds=True)
    assert bool(((a - b).abs() <= a.abs() * 2.0 ** -9 + 1e-3).all())


def test_repeated_calls_are_identical(cuda_ops):
    outs = [run_attention(cuda_ops, [1, 70, 2], [2000, 900, 1500], 8, 2, 16, 128, torch.bfloat16, 81)[0] for _ in range(2)]
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("new", [1, 150])
@pytest.mark.parametrize("alpha", [0.0, 1e-9, 0.02, -0.01])
def test_flat_and_peaked_scores(cuda_ops, new, alpha):
    """All scores equal, and scores that differ by hundreds (one key has nearly all the weight); a negative factor.
    |s| reaches 127 * 127 * 64 * 0.02 here, so the bound takes the score term from the formula itself."""
    dim, keys = 64, 700
    b = make_batch([new], [keys], 1, 32, dim, 91)
    q = rand_s8((new, 2, dim), 92)
    want, spread = P.paged_attention(q, *index_args(b), alpha, 0.02)
    out = cuda_ops.paged_attention(q.cuda(), *index_args(cuda(b)), alpha_qk=alpha, alpha_pv=0.02, out_dtype=torch.float16)
    s_max = abs(alpha) * 127 * 127 * dim * 1.4427
    tol = spread * (2.0 ** -11 + 2.0 ** -15 + 2 * s_max * 2.0 ** -23) + want.abs() * 2.0 ** -11 * 1.001 + 2.0 ** -25
    assert bool(((out.double().cpu() - want).abs() <= tol).all())


@pytest.mark.parametrize("new,keys", [(1, 300), (150, 300), (150, 2000)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_far_from_zero(cuda_ops, new, keys, sign):
    """All scores near +1800 or -1800 (in powers of two): only their differences count."""
    dim = 64
    b = make_batch([new], [keys], 1, 16, dim, 93)
    b["k_pages"] = rand_s8(tuple(b["k_pages"].shape), 94, 90, 110)
    q = torch.full((new, 2, dim), 100 * sign, dtype=torch.int8)
    alpha = 2e-3
    want, spread = P.paged_attention(q, *index_args(b), alpha, 0.02)
    out = cuda_ops.paged_attention(q.cuda(), *index_args(cuda(b)), alpha_qk=alpha, alpha_pv=0.02, out_dtype=torch.float16)
    s_max = alpha * 100 * 110 * dim * 1.4427
    tol = spread * (2.0 ** -11 + 2.0 ** -15 + 2 * s_max * 2.0 ** -23) + want.abs() * 2.0 ** -11 * 1.001 + 2.0 ** -25
    assert bool(((out.double().cpu() - want).abs() <= tol).all())


def test_long_tail_of_small_weights(cuda_ops):
    """One key far above 4095 others (weights near 2^-20 each): the tail must not be rounded away."""
    dim, keys = 64, 4096
    for new in (1, 20):
        b = make_batch([new], [keys], 1, 64, dim, 95)
        b["k_pages"].zero_()
        b["v_pages"].fill_(100)
        at = b["block_table"][0, 0]
        b["k_pages"][at, 0, 0] = 100
        b["v_pages"][at, 0, 0] = 0
        q = torch.full((new, 1, dim), 100, dtype=torch.int8)
        alpha = 13.8 / (100 * 100 * dim)
        want, spread = P.paged_attention(q, *index_args(b), alpha, 1.0)
        assert 0.1 < float(want.min()) < 1.0
        out = cuda_ops.paged_attention(q.cuda(), *index_args(cuda(b)), alpha_qk=alpha, alpha_pv=1.0, out_dtype=torch.float16)
        tol = spread * (2.0 ** -11 + 2.0 ** -15) + want.abs() * 2.0 ** -11 * 1.001
        assert bool(((out.double().cpu() - want).abs() <= tol).all()), float((out.double().cpu() - want).abs().max())


def test_strided_queries_and_given_output(cuda_ops):
    """Queries as a column block of a fused projection; rows behind the last sequence keep what they held."""
    heads, dim, new, keys = 4, 64, [3, 1, 150], [90, 33, 400]
    b = make_batch(new, keys, heads, 16, dim, 101, extra_tokens=5)
    rows = rand_s8((b["tokens"], 3 * heads, dim), 102)
    q = rows[:, :heads]
    want, spread = P.paged_attention(q, *index_args(b), 1e-4, 0.02)
    out = torch.full((b["tokens"], heads, dim), 7.0, dtype=torch.float16, device="cuda")
    res = cuda_ops.paged_attention(rows.cuda()[:, :heads], *index_args(cuda(b)), alpha_qk=1e-4, alpha_pv=0.02, out=out)
    assert res is out and cuda_ops.device_status() == 0
    assert_context(out, want, spread, sum(new))
    assert bool((out[sum(new):] == 7.0).all())


def test_the_stride_of_a_single_token_is_not_used(cuda_ops):
    """One token with 64 heads on one key head (a tile), the distance to a next token given as 7."""
    b = make_batch([1], [300], 1, 16, 64, 105)
    q = rand_s8((1, 64, 64), 106)
    want, spread = P.paged_attention(q, *index_args(b), 1e-4, 0.02)
    g, x = cuda(b), q.cuda()
    out = torch.empty((1, 64, 64), dtype=torch.float16, device="cuda")
    batch = cuda_ops._paged_batch(*index_args(g), 1, 1)[0]
    args = cuda_ops._pack_paged_attention(x.data_ptr(), 7, 64, 300, out.data_ptr(), 0, 0, 1e-4, 0.02, 1)
    rc = cuda_ops._c_paged_attention(batch, args, torch.cuda.current_stream().cuda_stream)
    if rc == -4:
        ws = torch.empty(cuda_ops._c_paged_workspace(1, 1, 64, 1, 64, 1, 300), dtype=torch.int8, device="cuda")
        args = cuda_ops._pack_paged_attention(x.data_ptr(), 7, 64, 300, out.data_ptr(), ws.data_ptr(), ws.numel(), 1e-4, 0.02, 1)
        rc = cuda_ops._c_paged_attention(batch, args, torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and cuda_ops.device_status() == 0
    assert_context(out, want, spread, 1)


def test_wide_block_table_view(cuda_ops):
    """A block table that is a view of a wider one (row stride beyond its width)."""
    b = make_batch([1, 2], [50, 200], 2, 16, 64, 111)
    wide = torch.full((2, 64), -1, dtype=torch.int32)
    wide[:, :b["block_table"].shape[1]] = b["block_table"]
    q = rand_s8((3, 2, 64), 112)
    want, spread = P.paged_attention(q, *index_args(b), 1e-4, 0.02)
    g = cuda(b)
    g["block_table"] = wide.cuda()[:, :b["block_table"].shape[1]]
    out = cuda_ops.paged_attention(q.cuda(), *index_args(g), alpha_qk=1e-4, alpha_pv=0.02, out_dtype=torch.bfloat16)
    assert_context(out, want, spread, 3)


@pytest.mark.parametrize("dim,batch,heads,kv_heads,keys", [
    (128, 8, 56, 56, 90),     # 448 units: three warps
    (64, 20, 32, 32, 70),     # 640
    (128, 32, 16, 8, 300),    # two CTAs of six warps per SM
    (64, 8, 32, 32, 200),     # of eight
    (80, 16, 32, 32, 300),    # of eight, two rounds
    (128, 16, 32, 8, 500),    # a CTA of eight warps per SM
    (128, 4, 32, 8, 1000),    # four of them in a cluster
    (80, 1, 16, 2, 9000),     # many, joined through the workspace
    (128, 6, 56, 56, 200),    # 336: four warps
    (64, 5, 64, 64, 900),     # pieces of 256 and more, clusters of four warps
    (128, 2, 32, 8, 2000),    # clusters of eight
])
def test_ways_of_cutting_a_decode_step(cuda_ops, dim, batch, heads, kv_heads, keys):
    """Single tokens, contexts of unequal lengths up to `keys`, one of them a single key and one of the whole length."""
    lens = [1 + (i * 7919) % keys for i in range(batch - 1)] + [keys]
    run_attention(cuda_ops, [1] * batch, lens, heads, kv_heads, 16, dim, torch.float16, 113)


@pytest.mark.parametrize("dim,batch,new,heads,kv_heads,keys", [
    (128, 4, 8, 32, 8, 700), (64, 1, 24, 16, 16, 1000), (80, 2, 5, 32, 8, 500), (128, 16, 5, 32, 8, 400), (64, 3, 33, 4, 4, 300),
    (128, 1, 5, 32, 8, 2000),
])
def test_drafts_of_shared_key_heads(cuda_ops, dim, batch, new, heads, kv_heads, keys):
    """9 to 32 rows per key head (tiles of 16), and 33."""
    lens = [max(new, 1 + (i * 7919) % keys) for i in range(batch - 1)] + [keys]
    run_attention(cuda_ops, [new - (i % 3) for i in range(batch)], lens, heads, kv_heads, 16, dim, torch.bfloat16, 114)


def test_more_sequences_than_the_tile_kernel_takes_at_once(cuda_ops):
    """600 sequences, two thirds of them with enough new tokens for the tile kernel."""
    new = [20 + i % 7 if i % 3 else 1 for i in range(600)]
    keys = [t + (7 * i) % 50 for i, t in enumerate(new)]
    run_attention(cuda_ops, new, keys, 1, 1, 16, 64, torch.float16, 115)


@pytest.mark.parametrize("new,keys", [([1, 5, 2], [40, 300, 1500]), ([30], [64])])
def test_more_query_heads_than_a_tile_has_rows(cuda_ops, new, keys):
    run_attention(cuda_ops, new, keys, 160, 1, 16, 64, torch.bfloat16, 116)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 80), (12, 1, 64)])
def test_prompt_among_decoding_sequences(cuda_ops, heads, kv_heads, dim):
    """One prompt and many single tokens, all with several splits: both kernels and the joining of both."""
    new, keys = [1] * 7 + [300] + [1, 0, 3, 1] * 2, [50, 5000, 2900, 1, 4096, 7000, 33, 4000, 6000, 12, 900, 6500, 4, 3, 3, 3333]
    run_attention(cuda_ops, new, keys, heads, kv_heads, 32, dim, torch.float16, 117)


def test_bad_sequence_beside_a_prompt(cuda_ops):
    """A sequence with bad lengths in such a batch: its rows stay, the others are served."""
    new, keys = [1, 1, 200] + [1] * 9, [300, 5000, 4200] + [2000 + 300 * i for i in range(9)]
    b = make_batch(new, keys, 1, 16, 64, 118)
    q = rand_s8((b["tokens"], 2, 64), 119)
    want, spread = P.paged_attention(q, *index_args(b), 1e-4, 0.02)
    b["kv_lens"][1] = 1 << 20
    g = cuda(b)
    out = torch.full((b["tokens"], 2, 64), 9.0, dtype=torch.float16, device="cuda")
    cuda_ops.paged_attention(q.cuda(), *index_args(g), alpha_qk=1e-4, alpha_pv=0.02, max_query_len=200, max_kv_len=5000, out=out)
    assert cuda_ops.device_status() == 211
    assert bool((out[1] == 9.0).all())
    assert_context(out, want, spread, 1)
    assert_context(out[2:], want[2:], spread[2:], b["tokens"] - 2)


@pytest.mark.parametrize("new", [1, 150])
def test_pages_beyond_four_gigabytes(cuda_ops, new):
    """Pages whose offset in the pool does not fit 32 bits, appended to and read."""
    b = make_batch([new, 1], [400, 300], 8, 128, 128, 125)
    rows = rand_s8((new + 1, 24, 128), 126)
    kp, vp = b["k_pages"].clone(), b["v_pages"].clone()
    P.paged_append(rows[:, 8:16], rows[:, 16:], kp, vp, b["block_table"], b["query_starts"], b["kv_lens"])
    want, spread = P.paged_attention(rows[:, :8], kp, vp, *index_args(b)[2:], 1e-4, 0.02)
    pages, total = kp.shape[0], 33000  # of 128 KB
    g = cuda(b)
    for name in ("k_pages", "v_pages"):
        far = torch.empty((total, 8, 128, 128), dtype=torch.int8, device="cuda")
        far[total - pages:] = g[name]
        g[name] = far
    used = g["block_table"] >= 0
    g["block_table"] = torch.where(used, g["block_table"] + (total - pages), g["block_table"])
    r = rows.cuda()
    cuda_ops.paged_append(r[:, 8:16], r[:, 16:], *index_args(g))
    out = cuda_ops.paged_attention(r[:, :8], *index_args(g), alpha_qk=1e-4, alpha_pv=0.02, out_dtype=torch.float16)
    assert cuda_ops.device_status() == 0
    assert torch.equal(g["k_pages"][total - pages:].cpu(), kp) and torch.equal(g["v_pages"][total - pages:].cpu(), vp)
    assert_context(out, want, spread, new + 1)


def test_bad_lengths_and_pages_are_reported(cuda_ops):
    """Lengths beyond the bounds or the table, tokens beyond N, pages outside the pool: a status, no fault, and the
    other sequences are served."""
    new, keys = [1, 1, 1], [40, 60, 20]
    b = make_batch(new, keys, 2, 16, 64, 121)
    q = rand_s8((3, 2, 64), 122)
    want, spread = P.paged_attention(q, *index_args(b), 1e-4, 0.02)

    def run(change, **kw):
        g = {k: (x.clone() if isinstance(x, torch.Tensor) else x) for k, x in b.items()}
        change(g)
        out = torch.full((3, 2, 64), 9.0, dtype=torch.float16, device="cuda")
        cuda_ops.paged_attention(q.cuda(), *index_args(cuda(g)), alpha_qk=1e-4, alpha_pv=0.02, out=out, **kw)
        status = cuda_ops.device_status()
        assert_context(out[2:], want[2:], spread[2:], 1)
        return status, out

    status, out = run(lambda g: g["kv_lens"].__setitem__(0, 10000))
    assert status == 211 and bool((out[0] == 9.0).all())
    status, out = run(lambda g: None, max_kv_len=50)
    assert status == 211 and bool((out[1] == 9.0).all())
    assert run(lambda g: g["kv_lens"].__setitem__(1, -3))[0] == 211
    assert run(lambda g: g["block_table"].__setitem__((0, 1), 1 << 20))[0] == 212
    assert run(lambda g: g["block_table"].__setitem__((1, 2), -1))[0] == 212
    b2 = dict(b)
    b2["query_starts"] = torch.tensor([0, 1, 2, 9], dtype=torch.int32)  # tokens 3..8 do not exist
    out = cuda_ops.paged_attention(q.cuda(), *index_args(cuda(b2)), alpha_qk=1e-4, alpha_pv=0.02, out_dtype=torch.float16)
    assert cuda_ops.device_status() == 211
    assert_context(out, want, spread, 2)
    assert cuda_ops.device_status() == 0


def test_empty_calls(cuda_ops):
    b = cuda(make_batch([0, 0], [5, 9], 2, 16, 64, 131))
    q = torch.empty((0, 2, 64), dtype=torch.int8, device="cuda")
    out = cuda_ops.paged_attention(q, *index_args(b), alpha_qk=1.0, alpha_pv=1.0)
    assert out.shape == (0, 2, 64)
    none = torch.empty((0, 2, 64), dtype=torch.int8, device="cuda")
    assert cuda_ops.paged_append(none, none, *index_args(b)) is None
    assert cuda_ops.device_status() == 0


# --------------------------------------------------------------------------------------------------- append
def run_append(C, new, keys, heads, kv_heads, page, dim, dtype, rotary_dim, interleaved, seed, values=None):
    b = make_batch(new, keys, kv_heads, page, dim, seed)
    n = b["tokens"]
    if dtype == torch.int8:
        rows = rand_s8((n, heads + 2 * kv_heads, dim), seed + 4, lo=-128)
    else:
        rows = (randn((n, heads + 2 * kv_heads, dim), seed + 4) * 3).to(dtype)
    if values is not None:
        values(rows)
    q = rows[:, :heads] if heads else None
    k, v = rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
    from torch_int.functional.paged import rotary_table
    table = rotary_table(rotary_dim, max(keys)) if rotary_dim else None
    alpha = {"q_alpha": 11.25, "k_alpha": 30.5, "v_alpha": 25.0} if dtype != torch.int8 else \
        {"q_alpha": 0.75, "k_alpha": 1.0, "v_alpha": 1.0}
    alpha = {a: torch.tensor(x, dtype=torch.float32).item() for a, x in alpha.items()}
    kp, vp = b["k_pages"].clone(), b["v_pages"].clone()
    want_q = P.paged_append(k, v, kp, vp, b["block_table"], b["query_starts"], b["kv_lens"], q=q, rotary=table,
                            interleaved=interleaved, **alpha)
    g, r = cuda(b), rows.cuda()
    got_q = C.paged_append(r[:, heads:heads + kv_heads], r[:, heads + kv_heads:], *index_args(g), max_query_len=max(new),
                           q=r[:, :heads] if heads else None, rotary=None if table is None else table.cuda(),
                           interleaved=interleaved, **alpha)
    assert C.device_status() == 0
    assert torch.equal(g["k_pages"].cpu(), kp) and torch.equal(g["v_pages"].cpu(), vp)  # every other row as it was
    if heads:
        assert torch.equal(got_q.cpu(), want_q)
    else:
        assert got_q is None


@pytest.mark.parametrize("dtype", ["int8", "fp16", "bf16", "fp32"])
@pytest.mark.parametrize("dim,rotary_dim", [(64, 64), (80, 80), (80, 32), (128, 128), (128, 16), (128, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(cuda_ops, dtype, dim, rotary_dim, interleaved):
    """Bit for bit: the arithmetic up to the rounding is fixed operation by operation."""
    run_append(cuda_ops, [1, 7, 40, 3], [1, 100, 40, 333], 6, 2, 16, dim, DT[dtype], rotary_dim, interleaved, 201)


@pytest.mark.parametrize("heads,kv_heads,page", [(0, 1, 16), (1, 1, 256), (56, 56, 16), (5, 1, 64), (0, 40, 128)])
def test_append_heads_and_pages(cuda_ops, heads, kv_heads, page):
    run_append(cuda_ops, [1, 33, 0, 2], [70, 33, 5, 517], heads, kv_heads, page, 64, torch.bfloat16, 64, False, 211)
    run_append(cuda_ops, [300], [301], heads, kv_heads, page, 128, torch.int8, 0, False, 212)


def test_append_saturates_and_zeroes_nan(cuda_ops):
    def values(rows):
        flat = rows.view(-1)
        flat[0:6] = torch.tensor([float("nan"), float("inf"), float("-inf"), 1e30, -1e30, 0.5 / 30.5])
        rows[-1, -1, :4] = torch.tensor([float("nan"), float("inf"), float("-inf"), 5e4], dtype=rows.dtype)
    run_append(cuda_ops, [9], [20], 0, 2, 16, 64, torch.float32, 0, False, 221, values)


def test_append_skips_bad_sequences(cuda_ops):
    """A sequence with fewer keys than new tokens, a page outside the pool, a position beyond the rotary table."""
    from torch_int.functional.paged import rotary_table
    b = make_batch([2, 2], [20, 40], 1, 16, 64, 231)
    rows = rand_s8((4, 2, 64), 232)

    def run(change, rotary=None):
        g = {k: (x.clone() if isinstance(x, torch.Tensor) else x) for k, x in b.items()}
        change(g)
        c = cuda(g)
        r = rows.cuda()
        cuda_ops.paged_append(r[:, :1], r[:, 1:], *index_args(c), rotary=rotary)
        return cuda_ops.device_status(), c["k_pages"].cpu()

    keep = b["k_pages"]
    for change, code in ((lambda g: g["kv_lens"].__setitem__(0, 1), 211), (lambda g: g["kv_lens"].__setitem__(0, 1 << 28), 211),
                         (lambda g: g["block_table"].__setitem__((0, 1), -5), 212)):
        status, k = run(change)
        assert status == code
        t = b["block_table"]
        assert torch.equal(k[t[1, 2], 0, 6], rows[2, 0]) and torch.equal(k[t[1, 2], 0, 7], rows[3, 0])
        assert torch.equal(k[t[0, 1]], keep[t[0, 1]])
    status, k = run(lambda g: None, rotary_table(64, 39).cuda())  # position 39 has no angle
    assert status == 211 and torch.equal(k[b["block_table"][1, 2], 0, 7], keep[b["block_table"][1, 2], 0, 7])
    assert cuda_ops.device_status() == 0


# ------------------------------------------------------------------------------------------------ together
def test_append_then_attend_as_a_sequence_grows(cuda_ops):
    """A prompt in two chunks, then single tokens: each step's context equals attention over everything appended."""
    C = cuda_ops
    from torch_int.functional.paged import rotary_table
    heads, kv_heads, dim, page = 4, 2, 64, 16
    steps = [[37, 5], [20, 1], [1, 1], [1, 1], [3, 1]]
    total = [sum(s[b] for s in steps) for b in range(2)]
    b = make_batch([0, 0], total, kv_heads, page, dim, 301)
    g = cuda(b)
    table = rotary_table(dim, 128)
    kp, vp = b["k_pages"].clone(), b["v_pages"].clone()
    lens = [0, 0]
    for i, new in enumerate(steps):
        lens = [l + t for l, t in zip(lens, new)]
        starts = torch.tensor([0, new[0], sum(new)], dtype=torch.int32)
        kv = torch.tensor(lens, dtype=torch.int32)
        rows = randn((sum(new), heads + 2 * kv_heads, dim), 310 + i)
        q, k, v = rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
        q8 = P.paged_append(k, v, kp, vp, b["block_table"], starts, kv, q=q, k_alpha=40.0, v_alpha=40.0, q_alpha=40.0, rotary=table)
        r = rows.cuda()
        got = C.paged_append(r[:, heads:heads + kv_heads], r[:, heads + kv_heads:], g["k_pages"], g["v_pages"], g["block_table"],
                             starts.cuda(), kv.cuda(), q=r[:, :heads], k_alpha=40.0, v_alpha=40.0, q_alpha=40.0, rotary=table.cuda())
        assert torch.equal(got.cpu(), q8) and torch.equal(g["k_pages"].cpu(), kp) and torch.equal(g["v_pages"].cpu(), vp)
        want, spread = P.paged_attention(q8, kp, vp, b["block_table"], starts, kv, 2e-4, 1 / 40)
        out = C.paged_attention(got, g["k_pages"], g["v_pages"], g["block_table"], starts.cuda(), kv.cuda(), alpha_qk=2e-4,
                                alpha_pv=1 / 40, out_dtype=torch.float16)
        assert C.device_status() == 0
        assert_context(out, want, spread, sum(new))


@pytest.mark.parametrize("new", [1, 40])
def test_captured_step_follows_the_lengths(cuda_ops, new):
    """Append and attention captured once and replayed while lengths, tokens and pages change in place; two graphs,
    replayed in turn, do not disturb each other."""
    C = cuda_ops
    heads, dim, page, cap = 4, 64, 16, 640
    graphs = []
    for which in range(2):
        b = make_batch([new, new], [cap, cap], heads, page, dim, 401 + which)
        g = cuda(b)
        rows = rand_s8((2 * new, 3 * heads, dim), 403 + which).cuda()
        out = torch.empty((2 * new, heads, dim), dtype=torch.float16, device="cuda")

        def step(rows=rows, g=g, out=out):
            C.paged_append(rows[:, heads:2 * heads], rows[:, 2 * heads:], *index_args(g), max_query_len=new)
            C.paged_attention(rows[:, :heads], *index_args(g), alpha_qk=2e-4, alpha_pv=0.02, max_query_len=new, max_kv_len=cap, out=out)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append((graph, b, g, rows, out, b["k_pages"].clone(), b["v_pages"].clone()))
    for graph, b, g, rows, out, kp, vp in graphs:  # undo what the first steps stored
        g["k_pages"].copy_(kp)
        g["v_pages"].copy_(vp)
    for i, lens in enumerate([[new, 600], [200, 50], [cap, 77]]):
        for graph, b, g, rows, out, kp, vp in graphs:
            fresh = rand_s8(tuple(rows.shape), 500 + i)
            rows.copy_(fresh)
            kv = torch.tensor(lens, dtype=torch.int32)
            g["kv_lens"].copy_(kv)
            P.paged_append(fresh[:, heads:2 * heads], fresh[:, 2 * heads:], kp, vp, b["block_table"], b["query_starts"], kv)
            graph.replay()
        for graph, b, g, rows, out, kp, vp in graphs:
            want, spread = P.paged_attention(rows[:, :heads].cpu(), kp, vp, b["block_table"], b["query_starts"],
                                             torch.tensor(lens, dtype=torch.int32), 2e-4, 0.02)
            assert torch.equal(g["k_pages"].cpu(), kp)
            assert_context(out, want, spread, 2 * new)
    assert C.device_status() == 0


def test_captured_mixed_batch_follows_the_lengths(cuda_ops):
    """Both attention kernels and the join of their splits in one graph; afterwards the lengths move between them."""
    C = cuda_ops
    heads, kv_heads, dim, cap, n = 8, 2, 128, 5000, 170
    b = make_batch([160, 1, 1, 8], [cap] * 4, kv_heads, 64, dim, 411)
    g = cuda(b)
    q = rand_s8((n, heads, dim), 412).cuda()
    out = torch.empty((n, heads, dim), dtype=torch.float16, device="cuda")

    def step():
        C.paged_attention(q, *index_args(g), alpha_qk=1e-4, alpha_pv=0.02, max_query_len=160, max_kv_len=cap, out=out)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for starts, lens in [([0, 160, 161, 162, 170], [cap] * 4), ([0, 1, 161, 162, 170], [4800, 160, 1, 3000]), ([0, 1, 2, 3, 4], [4999, 1, 700, 64])]:
        b["query_starts"], b["kv_lens"] = torch.tensor(starts, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32)
        g["query_starts"].copy_(b["query_starts"])
        g["kv_lens"].copy_(b["kv_lens"])
        out.fill_(7.0)
        graph.replay()
        assert C.device_status() == 0
        want, spread = P.paged_attention(q.cpu(), *index_args(b), 1e-4, 0.02)
        assert_context(out, want, spread, starts[-1])
        assert bool((out[starts[-1]:] == 7.0).all())


def test_calls_on_two_streams_at_once(cuda_ops):
    """The same cache read by calls on two streams: each call has its own scratch."""
    C = cuda_ops
    b = make_batch([1] * 4, [3000, 2500, 2999, 64], 4, 16, 128, 601)
    q = [rand_s8((4, 8, 128), 602 + i) for i in range(2)]
    want = [P.paged_attention(x, *index_args(b), 2e-4, 0.02) for x in q]
    g, gq = cuda(b), [x.cuda() for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for st, x in zip(streams, gq):
            with torch.cuda.stream(st):
                outs.append(C.paged_attention(x, *index_args(g), alpha_qk=2e-4, alpha_pv=0.02, out_dtype=torch.float16))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert_context(out, *want[i % 2], 4)
        assert torch.equal(out, outs[i % 2])


def test_refusals_on_gpu_tensors(cuda_ops):
    C = cuda_ops
    b = cuda(make_batch([1], [20], 2, 16, 64, 701))
    q = rand_s8((1, 4, 64), 702).cuda()
    k = rand_s8((1, 2, 64), 703).cuda()
    ok = dict(alpha_qk=1e-4, alpha_pv=0.02)
    with pytest.raises(RuntimeError, match="multiple of the key heads"):
        C.paged_attention(q[:, :3], *index_args(b), **ok)
    with pytest.raises(RuntimeError, match="int8, float16 or bfloat16"):
        C.paged_attention(q, *index_args(b), out_dtype=torch.float32, **ok)
    with pytest.raises(RuntimeError, match="int8"):
        C.paged_attention(q.half(), *index_args(b), **ok)
    with pytest.raises(RuntimeError, match="int32"):
        C.paged_attention(q, b["k_pages"], b["v_pages"], b["block_table"].long(), b["query_starts"], b["kv_lens"], **ok)
    with pytest.raises(RuntimeError, match="int32"):
        C.paged_attention(q, b["k_pages"], b["v_pages"], b["block_table"], b["query_starts"], b["kv_lens"].cpu(), **ok)
    with pytest.raises(RuntimeError, match=r"\[B \+ 1\]"):
        C.paged_attention(q, b["k_pages"], b["v_pages"], b["block_table"], b["query_starts"][:1], b["kv_lens"], **ok)
    with pytest.raises(RuntimeError, match="contiguous"):
        C.paged_attention(q, b["k_pages"].transpose(1, 2), b["v_pages"].transpose(1, 2), b["block_table"], b["query_starts"], b["kv_lens"], **ok)
    with pytest.raises(RuntimeError, match="page_size"):
        odd = torch.zeros((3, 2, 24, 64), dtype=torch.int8, device="cuda")
        C.paged_attention(q, odd, odd, b["block_table"], b["query_starts"], b["kv_lens"], **ok)
    with pytest.raises(RuntimeError, match="head_dim"):
        odd = torch.zeros((3, 2, 16, 72), dtype=torch.int8, device="cuda")
        C.paged_attention(torch.zeros((1, 2, 72), dtype=torch.int8, device="cuda"), odd, odd, b["block_table"], b["query_starts"], b["kv_lens"], **ok)
    with pytest.raises(RuntimeError, match="packed heads"):
        C.paged_attention(rand_s8((1, 4, 128), 1).cuda()[:, :, ::2], *index_args(b), **ok)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        wide = rand_s8((2, 4 * 64 + 8), 1).cuda()
        C.paged_append(k, k, *index_args(b), q=wide.view(-1)[8:8 + 256].view(1, 4, 64))
    with pytest.raises(RuntimeError, match="out must be"):
        C.paged_attention(q, *index_args(b), out=torch.empty((1, 2, 64), dtype=torch.int8, device="cuda"), **ok)
    with pytest.raises(RuntimeError, match="heads, the cache"):
        C.paged_append(q, q, *index_args(b))
    with pytest.raises(RuntimeError, match="rotary"):
        C.paged_append(k, k, *index_args(b), rotary=torch.zeros((40, 64), device="cuda", dtype=torch.float64))
    with pytest.raises(RuntimeError, match="rotary_dim"):
        C.paged_append(k, k, *index_args(b), rotary=torch.zeros((40, 72), device="cuda"))
    with pytest.raises(RuntimeError, match="v must be"):
        C.paged_append(k, k.half(), *index_args(b))
    assert C.device_status() == 0


# ----------------------------------------------------------------------------------------------- in the model
@pytest.fixture(scope="module")
def opt_model():
    from torch_int.models.opt import Int8OPTConfig
    from torch_int.models.random_init import random_int8_opt
    cfg = Int8OPTConfig(vocab_size=512, hidden_size=256, num_hidden_layers=2, ffn_dim=512, num_attention_heads=4,
                        max_position_embeddings=512)
    return random_int8_opt(cfg, seed=5, device="cuda")


def prompts_of(*lens):
    g = torch.Generator().manual_seed(9)
    return [torch.randint(2, 512, (n,), generator=g).cuda() for n in lens]


def close(a, b, tol=2e-2):
    """A batch and a sequence alone may be cut differently, so an int8 context may differ by a unit where it lies near a
    half: by the operator's bound (2^-11 of a spread of about 10 units, to both sides) in at most 2 * 2^-11 * 10 = 1 % of
    the 256 columns, 2.6 of them.  A unit is 1 / (10 * sqrt(256)) = 0.6 % of a context of 10 units per column, so a
    layer's attention output is off by about sqrt(2.6) * 0.6 % = 1 %, two layers' by 1.4 % at most of the residual."""
    return float((a - b).norm() / b.norm()) < tol


def test_model_batch_agrees_with_its_sequences_alone(cuda_ops, opt_model):
    prompts = prompts_of(200, 1, 37, 64)
    cache = opt_model.new_paged_cache(40)
    seqs = [cache.open() for _ in prompts]
    got = opt_model.forward_paged(torch.cat(prompts), cache, cache.step(seqs, [len(p) for p in prompts]))
    for i, p in enumerate(prompts):
        alone = opt_model.new_paged_cache(20, page_size=32)
        want = opt_model.forward_paged(p, alone, alone.step([alone.open()], [len(p)]))
        assert close(got[i:i + 1], want)
    # a chunk for one sequence, single tokens for two others
    new = prompts_of(90, 1, 1)
    step = cache.step([seqs[3], seqs[0], seqs[1]], [90, 1, 1])
    got = opt_model.forward_paged(torch.cat(new), cache, step)
    for i, s in enumerate((3, 0, 1)):
        alone = opt_model.new_paged_cache(30)
        h = alone.open()
        opt_model.forward_paged(prompts[s], alone, alone.step([h], [len(prompts[s])]))
        want = opt_model.forward_paged(new[i], alone, alone.step([h], [len(new[i])]))
        assert close(got[i:i + 1], want)
    assert cuda_ops.device_status() == 0


def test_model_generates_the_same_eagerly_and_from_a_graph(cuda_ops, opt_model):
    prompts = prompts_of(30, 5, 100)
    eager = opt_model.generate_paged(prompts, 12, use_cuda_graph=False)
    graph = opt_model.generate_paged(prompts, 12)
    assert all(torch.equal(a, b) for a, b in zip(eager, graph))
    assert [len(x) for x in graph] == [42, 17, 112] and all(torch.equal(x[:len(p)], p) for x, p in zip(graph, prompts))
    one = opt_model.generate_paged(prompts[:1], 1)
    assert torch.equal(one[0], graph[0][:31])
    assert cuda_ops.device_status() == 0
