"""The paged cache's bookkeeping and the paged model path on CPU: the model's own Python with the extension replaced by
the stand-ins of cpu_ops_stub.py plus the 64-bit oracle of the paged operators."""
import pytest
import torch

import cpu_ops_stub as stub
from oracle import paged as P
from torch_int.models.paged_cache import PagedInt8KVCache


def _append(k, v, k_pages, v_pages, block_table, query_starts, kv_lens, *, max_query_len=None, q=None, k_alpha=1.0,
            v_alpha=1.0, q_alpha=1.0, rotary=None, interleaved=False):
    t = query_starts[1:] - query_starts[:-1]
    assert int(t.max()) <= max_query_len and int(query_starts[-1]) == k.shape[0] and bool((kv_lens >= t).all())
    return P.paged_append(k, v, k_pages, v_pages, block_table, query_starts, kv_lens, q, k_alpha, v_alpha, q_alpha, rotary, interleaved)


def _attention(q, k_pages, v_pages, block_table, query_starts, kv_lens, *, alpha_qk, alpha_pv, max_query_len=None,
               max_kv_len=None, out=None, out_dtype=torch.int8):
    assert int(kv_lens.max()) <= max_kv_len
    ctx, _ = P.paged_attention(q, k_pages, v_pages, block_table, query_starts, kv_lens, alpha_qk, alpha_pv)
    return ctx.round().clamp(-128, 127).to(out_dtype)


@pytest.fixture()
def cpu_model(monkeypatch):
    from torch_int.models.opt import Int8OPTConfig
    from torch_int.models.random_init import random_int8_opt
    monkeypatch.setattr(stub, "paged_append", _append, raising=False)
    monkeypatch.setattr(stub, "paged_attention", _attention, raising=False)
    stub.install(monkeypatch.setattr)
    cfg = Int8OPTConfig(vocab_size=96, hidden_size=128, num_hidden_layers=2, ffn_dim=256, num_attention_heads=2,
                        max_position_embeddings=64)
    return random_int8_opt(cfg, seed=7, device="cpu")


def prompts_of(*lens, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(2, 96, (n,), generator=g) for n in lens]


def test_pages_are_handed_out_and_given_back():
    c = PagedInt8KVCache(1, 6, 2, 64, "cpu", page_size=16)
    a, b = c.open(), c.open()
    s = c.step([a, b], [17, 1])
    assert s.query_starts.tolist() == [0, 17, 18] and s.kv_lens.tolist() == [17, 1] and s.last.tolist() == [16, 17]
    assert s.positions.tolist() == list(range(17)) + [0] and s.max_query_len == 17 and s.max_kv_len == 17
    assert c.free_pages == 3 and s.block_table.shape == (2, 2)
    used = set(s.block_table[0].tolist()) | {int(s.block_table[1, 0])}
    assert len(used) == 3
    s = c.step([b, a], [16, 1])  # any order, any subset; b crosses a page
    assert s.kv_lens.tolist() == [17, 18] and s.positions.tolist() == list(range(1, 17)) + [17]
    with pytest.raises(RuntimeError, match="free pages"):
        c.step([a, b], [60, 1])
    assert c.length(a) == 18 and c.length(b) == 17 and c.free_pages == 2  # nothing changed
    c.rewind(a, 16)
    s = c.step([a], [1])
    assert s.positions.tolist() == [16]
    c.close(b)
    assert c.free_pages == 4
    c.close(a)
    assert c.free_pages == 6


@pytest.mark.parametrize("call,words", [
    (lambda c, a: c.step([a], []), "one number"), (lambda c, a: c.step([], []), "a sequence"),
    (lambda c, a: c.step([a, a], [1, 1]), "once"), (lambda c, a: c.step([a], [0]), "at least one"),
    (lambda c, a: c.rewind(a, 1), "rewound"),
])
def test_bad_steps_are_refused(call, words):
    c = PagedInt8KVCache(1, 2, 2, 64, "cpu")
    with pytest.raises(ValueError, match=words):
        call(c, c.open())


def test_bad_caches_are_refused():
    with pytest.raises(ValueError, match="page_size"):
        PagedInt8KVCache(1, 2, 2, 64, "cpu", page_size=20)
    with pytest.raises(ValueError, match="num_pages"):
        PagedInt8KVCache(1, 0, 2, 64, "cpu")


def test_a_batch_gives_what_its_sequences_give_alone(cpu_model):
    dec = cpu_model.model.decoder
    prompts = prompts_of(5, 23, 1)
    together = dec.new_paged_cache(8)
    seqs = [together.open() for _ in prompts]
    hidden = dec.forward_paged(torch.cat(prompts), together, together.step(seqs, [5, 23, 1]))
    assert hidden.shape == (29, 128)
    at = 0
    for p in prompts:
        alone = dec.new_paged_cache(2)
        h = dec.forward_paged(p, alone, alone.step([alone.open()], [len(p)]))
        assert torch.allclose(hidden[at:at + len(p)], h, rtol=1e-5, atol=1e-5)
        at += len(p)


def test_chunks_and_single_tokens_give_what_one_step_gives(cpu_model):
    dec = cpu_model.model.decoder
    x = prompts_of(30)[0]
    c = dec.new_paged_cache(4)
    whole = dec.forward_paged(x, c, c.step([c.open()], [30]))
    c = dec.new_paged_cache(4)
    s = c.open()
    parts, at = [], 0
    for n in (13, 9, 1, 1, 6):
        parts.append(dec.forward_paged(x[at:at + n], c, c.step([s], [n])))
        at += n
    assert torch.allclose(torch.cat(parts), whole, rtol=1e-5, atol=1e-5)


def test_advanced_steps_and_their_counts(cpu_model):
    """Steps advanced in place give what new steps give; the cache is told afterwards; what has no page is never 0."""
    dec = cpu_model.model.decoder
    x = prompts_of(12)[0]
    c = dec.new_paged_cache(6)
    a, b = c.open(), c.open()
    s = c.step([a, b], [17, 1])
    assert s.block_table[1, 1] == -1
    with pytest.raises(ValueError, match="single tokens"):
        s.advance()
    c = dec.new_paged_cache(2)
    whole = dec.forward_paged(x, c, c.step([c.open()], [12]))
    c = dec.new_paged_cache(2)
    a = c.open()
    c.reserve({a: 20})
    parts = [dec.forward_paged(x[:9], c, c.step([a], [9]))]
    s = c.step([a], [1])
    for i in (9, 10, 11):
        if i > 9:
            s.advance()
        parts.append(dec.forward_paged(x[i:i + 1], c, s))
    assert torch.allclose(torch.cat(parts), whole, rtol=1e-5, atol=1e-5)
    assert c.length(a) == 10 and s.max_kv_len == 12
    c.fill(a, 12)
    assert c.step([a], [1]).positions.tolist() == [12]
    for bad in (12, 33):
        with pytest.raises(ValueError, match="filled"):
            c.fill(a, bad)


def test_model_limits_are_refused(cpu_model):
    dec = cpu_model.model.decoder
    c = dec.new_paged_cache(8)
    s = c.step([c.open()], [3])
    with pytest.raises(ValueError, match="2 tokens given"):
        dec.forward_paged(torch.tensor([5, 6]), c, s)
    with pytest.raises(ValueError, match="beyond the model"):
        dec.forward_paged(torch.full((65,), 5), c, c.step([c.open()], [65]))
    with pytest.raises(ValueError, match="exceed the model"):
        cpu_model.generate_paged(prompts_of(60), 6)
    assert cpu_model.generate_paged(prompts_of(60), 5, use_cuda_graph=False)[0].shape == (65,)


def test_generation_agrees_with_teacher_forcing_and_leaves_the_cache(cpu_model):
    prompts = prompts_of(4, 17, 9)
    cache = cpu_model.new_paged_cache(12)
    other = cache.open()
    cache.step([other], [20])
    outs = cpu_model.generate_paged(prompts, 6, cache=cache, use_cuda_graph=False)
    assert cache.free_pages == 10 and cache.length(other) == 20
    for p, out in zip(prompts, outs):
        assert out.shape == (len(p) + 6,) and torch.equal(out[:len(p)], p)
        c = cpu_model.new_paged_cache(3)
        logits = cpu_model.forward_paged(out[:-1], c, c.step([c.open()], [len(out) - 1]), last_token_only=False)
        assert torch.equal(logits[len(p) - 1:].argmax(-1), out[len(p):])
    with pytest.raises(RuntimeError, match="free pages"):
        cpu_model.generate_paged(prompts_of(200), 1, cache=cache)
    assert cache.free_pages == 10
    for bad in ([], [torch.empty(0, dtype=torch.long)]):
        with pytest.raises(ValueError, match="prompt"):
            cpu_model.generate_paged(bad, 2)
