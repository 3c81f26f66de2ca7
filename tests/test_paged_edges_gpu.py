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
