"""The paged int8 cache operators at the edges of what their entry points accept, on the GPU against oracle/paged.py with
the bound that test_paged_gpu.py derives."""
import pytest
import torch

from helpers import rand_s8
from oracle import paged as P
from test_paged_gpu import assert_context, cuda, index_args, make_batch, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 1, 128), (71, 1, 64), (48, 1, 128), (40, 2, 80), (34, 2, 64), (128, 1, 64)])
@pytest.mark.parametrize("batch,prompt,longest", [(16, 500, 4000), (8, 1024, 4096), (4, 40, 8000)])
def test_prompt_among_tokens_of_many_heads_per_key_head(cuda_ops, heads, kv_heads, dim, batch, prompt, longest):
    """17 to 128 query heads on a key head: a single token has more rows than the rows kernel takes beside a prompt."""
    new = [1] * (batch - 1) + [prompt]
    keys = [1 + (i * 7919) % longest for i in range(batch - 2)] + [longest, max(prompt, longest // 2)]
    run_attention(cuda_ops, new, keys, heads, kv_heads, 16, dim, torch.float16, 803)


@pytest.mark.parametrize("new,batch,heads,kv_heads,dim", [(1, 300, 1, 1, 64), (1, 32, 32, 8, 128), (1, 32, 32, 8, 64), (3, 3, 4, 2, 80),
                                                          (1, 8, 56, 56, 128), (40, 2, 8, 2, 128)])
def test_a_step_without_any_key_gives_zeros(cuda_ops, new, batch, heads, kv_heads, dim):
    """Every sequence holds no key, and the bound says so: max_kv_len = 0."""
    out, _ = run_attention(cuda_ops, [new] * batch, [0] * batch, heads, kv_heads, 16, dim, torch.float16, 811)
    assert bool((out == 0).all())


def test_lengths_written_by_the_kernel_before(cuda_ops):
    """Lengths and starts that change on the stream right before each call, joined through the workspace."""
    b = make_batch([1] * 3, [9000] * 3, 2, 16, 128, 821)
    q = rand_s8((3, 16, 128), 822)
    lens = [torch.tensor(x, dtype=torch.int32) for x in ([9000, 30, 4000], [2, 9000, 8999], [5000, 7000, 1], [900, 1800, 2700])]
    want = [P.paged_attention(q, *index_args(b)[:4], x, 2e-4, 0.02) for x in lens]
    g, gq, glens = cuda(b), q.cuda(), [x.cuda() for x in lens]
    outs = [torch.empty((3, 16, 128), dtype=torch.float16, device="cuda") for _ in range(200)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        g["kv_lens"].copy_(glens[i % 4])
        cuda_ops.paged_attention(gq, *index_args(g), alpha_qk=2e-4, alpha_pv=0.02, max_query_len=1, max_kv_len=9000, out=out)
    assert cuda_ops.device_status() == 0
    for i in range(4):
        assert_context(outs[i], *want[i], 3)
        assert all(torch.equal(outs[i], x) for x in outs[i::4])


@pytest.mark.parametrize("new,keys", [(1, 300), (20, 300), (150, 300), (150, 3000), (300, 300)])
@pytest.mark.parametrize("alpha", [2.7, -2.7, 4.0, 16.0, -16.0, 1000.0, 1e20])
def test_steep_scores(cuda_ops, new, keys, alpha):
    """Factors at which one unit of q . k decides, for one token and for prompts.  q . k is within 64, so to the bound of
    assert_context comes the rounding of a score of up to 64 * alpha powers of e to fp32, twice: 2 s 2^-23 of a weight.  From
    alpha = 16 on only the keys with the largest q . k count (the others have 2^-23 of their weight or less, 3000 keys 2^-11,
    and that rounding of it): their scores are equal numbers, so the term falls away."""
    dim = 64
    b = make_batch([new, 1], [keys, 40], 2, 16, dim, 831)
    b["k_pages"] = rand_s8(tuple(b["k_pages"].shape), 832, -1, 1)
    q = rand_s8((new + 1, 4, dim), 833, -1, 1)
    want, spread = P.paged_attention(q, *index_args(b), alpha, 0.02)
    out = cuda_ops.paged_attention(q.cuda(), *index_args(cuda(b)), alpha_qk=alpha, alpha_pv=0.02, out_dtype=torch.float16)
    assert cuda_ops.device_status() == 0 and bool(out.isfinite().all())
    term = 2 * 64 * abs(alpha) * 1.4427 * 2.0 ** -23 if abs(alpha) < 16 else 0.0
    tol = spread * (2.0 ** -11 + 2.0 ** -15 + term) + want.abs() * 2.0 ** -11 * 1.001 + 2.0 ** -25
    err = (out.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("new,keys", [(1, 300), (150, 300), (150, 3000)])
@pytest.mark.parametrize("alpha", [2.7, -2.7, 16.0, 1e20])
def test_steep_scores_far_from_zero(cuda_ops, new, keys, alpha):
    """The largest q . k there is, the same for every key: every context is the mean of the values it sees."""
    dim = 128
    b = make_batch([new], [keys], 1, 16, dim, 841)
    b["k_pages"].fill_(-128)
    q = torch.full((new, 2, dim), -128, dtype=torch.int8)
    want, spread = P.paged_attention(q, *index_args(b), 0.0, 0.02)
    out = cuda_ops.paged_attention(q.cuda(), *index_args(cuda(b)), alpha_qk=alpha, alpha_pv=0.02, out_dtype=torch.float16)
    assert cuda_ops.device_status() == 0
    assert_context(out, want, spread, new)


@pytest.mark.parametrize("alpha,unit", [(5.6, -115), (5.63, -128), (5.67, -128), (5.7, -122)])
@pytest.mark.parametrize("new,batch,heads", [(1, 64, 8), (5, 64, 32), (150, 2, 8)])
def test_scores_that_rise_by_just_what_the_maximum_may_lag_behind(cuda_ops, alpha, unit, new, batch, heads):
    """Scores near 2^24 are 2 apart in fp32.  Here later keys are 8 above the first ones: not more than a running maximum
    may lag behind, but one more than that once 7 minus the maximum is rounded.  All values are equal, and so is each
    context, whatever the weights."""
    dim, kv_heads, keys = 128, 8, 1024
    b = make_batch([new] * batch, [keys] * batch, kv_heads, 64, dim, 851)
    b["k_pages"].fill_(-128)
    row = torch.arange(64)
    for s in range(batch):
        for i in range(keys // 64):  # 256 keys with `unit` in the last column, 256 with one more
            b["k_pages"][b["block_table"][s, i], :, row, dim - 1] = unit + (i // 4) % 2
    b["v_pages"].fill_(50)
    q = torch.full((new * batch, heads, dim), -128, dtype=torch.int8)
    q[..., dim - 1] = 1
    out = cuda_ops.paged_attention(q.cuda(), *index_args(cuda(b)), alpha_qk=alpha, alpha_pv=0.02, max_query_len=new, max_kv_len=keys,
                                   out_dtype=torch.float16)
    assert cuda_ops.device_status() == 0
    want = torch.full(out.shape, 50 * 0.02, dtype=torch.float64)
    assert_context(out, want, want, new * batch)


@pytest.mark.parametrize("bound", [1 << 31, 1 << 32, (1 << 32) + 1, (1 << 63) - 1])
def test_a_bound_of_the_new_tokens_beyond_32_bits(cuda_ops, bound):
    """max_query_len of the C entry points is 64 bits wide: any value from the longest sequence's on serves the batch."""
    C = cuda_ops
    new, keys = [3, 1], [40, 33]
    b = make_batch(new, keys, 2, 16, 64, 861)
    rows = rand_s8((4, 6, 64), 862)
    kp, vp = b["k_pages"].clone(), b["v_pages"].clone()
    P.paged_append(rows[:, 2:4], rows[:, 4:], kp, vp, *index_args(b)[2:])
    want, spread = P.paged_attention(rows[:, :2], kp, vp, *index_args(b)[2:], 1e-4, 0.02)
    g, r = cuda(b), rows.cuda()
    out = torch.empty((4, 2, 64), dtype=torch.float16, device="cuda")
    pages, table = b["k_pages"].shape[0], b["block_table"].shape[1]
    batch = C._pack_paged_batch(*(t.data_ptr() for t in index_args(g)), pages, 2, 16, 64, table, table, 2, 4, bound)
    stream = torch.cuda.current_stream().cuda_stream
    base = r.data_ptr()
    append = C._pack_paged_append(0, base + 128, base + 256, 0, 384, 384, 0, 0, 0, 0, 0, 1.0, 1.0, 1.0, 3, 0)
    assert C._c_paged_append(batch, append, stream) == 0
    assert C._c_paged_attention(batch, C._pack_paged_attention(base, 384, 2, 40, out.data_ptr(), 0, 0, 1e-4, 0.02, 1), stream) == 0
    assert C.device_status() == 0
    assert torch.equal(g["k_pages"].cpu(), kp) and torch.equal(g["v_pages"].cpu(), vp)
    assert_context(out, want, spread, 4)


@pytest.mark.parametrize("batch,new,heads,alpha", [(33000, 2, 10, 1e-4), (70, 1900, 8, 16.0)])
def test_more_row_tiles_than_a_grid_is_high(cuda_ops, batch, new, heads, alpha):
    """33000 sequences with two row tiles each, and 70 whose bound of 1900 tokens of 8 heads asks for 950 each (a steep factor:
    the rows kernel's), the first and the last of them longer than the rest.  The sequences share their pages."""
    keys = 40
    short = 2
    b = make_batch([0], [keys], 1, 16, 64, 871)
    b["k_pages"] = rand_s8(tuple(b["k_pages"].shape), 872, -1, 1)
    news = [new if i in (0, batch - 1) else short for i in range(batch)]
    starts = torch.tensor([0] + news, dtype=torch.int32).cumsum(0).to(torch.int32)
    lens = torch.full((batch,), keys, dtype=torch.int32)
    lens[-1] = keys - 3
    n = int(starts[-1])
    q = rand_s8((short, heads, 64), 873, -1, 1).repeat(-(-n // short), 1, 1)[:n].contiguous()
    g = cuda(b)
    out = cuda_ops.paged_attention(q.cuda(), g["k_pages"], g["v_pages"], g["block_table"].expand(batch, -1).contiguous(), starts.cuda(),
                                   lens.cuda(), alpha_qk=alpha, alpha_pv=0.02, max_query_len=new, max_kv_len=keys, out_dtype=torch.float16)
    assert cuda_ops.device_status() == 0
    seen = {}
    for i in {0, 1, batch // 2, batch - 2, batch - 1}:
        at, t = int(starts[i]), news[i]
        want, spread = P.paged_attention(q[at:at + t], *index_args(b)[:3], [0, t], [int(lens[i])], alpha, 0.02)
        assert_context(out[at:at + t], want, spread, t)
        seen[i] = out[at:at + t]
    middle = out[int(starts[1]):int(starts[batch - 1])].view(batch - 2, short, heads, 64)
    assert bool((middle == seen[1]).all())


def test_queries_of_tokens_that_are_not_stored_keep_their_rows(cuda_ops):
    """A sequence with bad lengths, a page outside the pool and tokens of no sequence: their rows of q_out stay."""
    C = cuda_ops
    b = make_batch([2, 1, 2], [20, 9, 40], 2, 16, 64, 881, extra_tokens=2)
    b["kv_lens"][1] = -1
    b["block_table"][2, 2] = -1  # positions 38 and 39
    rows = rand_s8((7, 6, 64), 882)
    g, r = cuda(b), rows.cuda()
    q_out = torch.full((7, 2, 64), 77, dtype=torch.int8, device="cuda")
    pages, table = b["k_pages"].shape[0], b["block_table"].shape[1]
    batch = C._pack_paged_batch(*(t.data_ptr() for t in index_args(g)), pages, 2, 16, 64, table, table, 3, 7, 2)
    base = r.data_ptr()
    append = C._pack_paged_append(base, base + 128, base + 256, 384, 384, 384, 2, 0, 0, 0, q_out.data_ptr(), 1.0, 1.0, 1.0, 3, 0)
    assert C._c_paged_append(batch, append, torch.cuda.current_stream().cuda_stream) == 0
    assert C.device_status() in (211, 212)
    assert torch.equal(q_out[:2].cpu(), rows[:2, :2]) and bool((q_out[2:] == 77).all())
