"""The paged model path on CPU against what it has to equal: the static path where both round alike, the reference model's
dataflow with unrounded probabilities (oracle/paged.py, oracle/opt_model.py) everywhere, and, on gloo ranks, itself on one.
The extension is replaced by the stand-ins of cpu_ops_stub.py and the 64-bit oracle of the paged operators."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import cpu_ops_stub as stub
from oracle import opt_model as OM
from oracle import paged as P
from test_paged_model_cpu import _append, _attention, cpu_model, prompts_of  # noqa: F401 (a fixture)
from test_tensor_parallel_cpu import _free_port


def dataflow(model, ids):
    """Logits [T, vocab] of one sequence."""
    sd = {k: v.detach() for k, v in model.state_dict().items()}
    kept = OM.attention
    OM.attention = P.model_attention
    try:
        return OM.causal_lm_logits(sd, model.model.decoder.config, ids.view(1, -1))[0][0]
    finally:
        OM.attention = kept


def test_a_single_token_gives_the_static_paths_logits(cpu_model):  # noqa: F811
    """The only probability is 1, which the static path's rounding keeps."""
    for token in (5, 40, 95):
        x = torch.tensor([token])
        c = cpu_model.new_paged_cache(1)
        got = cpu_model.forward_paged(x, c, c.step([c.open()], [1]))
        assert torch.equal(got, cpu_model(x.view(1, 1)).logits[0])


def test_prompts_and_single_tokens_follow_the_unrounded_dataflow(cpu_model):  # noqa: F811
    """(1e-5 as in the other wiring tests: a product of other sizes may round differently in the CPU BLAS of lm_head.)"""
    prompts = prompts_of(23, 1, 40)
    c = cpu_model.new_paged_cache(8)
    seqs = [c.open() for _ in prompts]
    got = cpu_model.forward_paged(torch.cat(prompts), c, c.step(seqs, [23, 1, 40]), last_token_only=False)
    assert torch.allclose(got, torch.cat([dataflow(cpu_model, p) for p in prompts]), rtol=1e-5, atol=1e-5)
    more = prompts_of(3, 1, 1, seed=4)  # a chunk behind the longest, single tokens behind the others
    got = cpu_model.forward_paged(torch.cat(more), c, c.step([seqs[2], seqs[0], seqs[1]], [3, 1, 1]), last_token_only=False)
    want = [dataflow(cpu_model, torch.cat((prompts[s], new)))[len(prompts[s]):] for s, new in zip((2, 0, 1), more)]
    assert torch.allclose(got, torch.cat(want), rtol=1e-5, atol=1e-5)


def _rank_main(rank, world, port, ret):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from torch_int.models.opt import Int8OPTConfig
        from torch_int.models.random_init import random_int8_opt
        from torch_int.models.tensor_parallel import TensorParallel
        torch.set_num_threads(1)
        stub.paged_append, stub.paged_attention = _append, _attention
        stub.install()
        cfg = Int8OPTConfig(vocab_size=96, hidden_size=256, num_hidden_layers=2, ffn_dim=512, num_attention_heads=4,
                            max_position_embeddings=64)
        whole = random_int8_opt(cfg, seed=5, device="cpu")
        tp = TensorParallel.from_world()
        tp.use_peer_memory = False
        model = random_int8_opt(cfg, seed=5, device="cpu", tp=tp)
        prompts = prompts_of(21, 1, 9)
        steps = []
        for m in (whole, model):
            c = m.new_paged_cache(8)
            seqs = [c.open() for _ in prompts]
            assert c.k_pages[0].shape[1] == (4 if m is whole else 4 // world)
            first = m.forward_paged(torch.cat(prompts), c, c.step(seqs, [21, 1, 9]))
            steps.append((first, m.forward_paged(torch.tensor([7, 8]), c, c.step([seqs[2], seqs[0]], [1, 1]))))
        checks = {"prompts": torch.equal(steps[0][0], steps[1][0]), "single_tokens": torch.equal(steps[0][1], steps[1][1])}
        outs = [m.generate_paged(prompts, 5, use_cuda_graph=False) for m in (whole, model)]
        checks["generate"] = all(torch.equal(a, b) for a, b in zip(*outs))
        ret[rank] = checks
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 4])
def test_paged_path_on_cpu_ranks(world):
    """The ranks exchange integers: the sharded model's logits are the whole one's bit for bit."""
    ctx = mp.get_context("spawn")
    ret = ctx.Manager().dict()
    port = _free_port()
    procs = [ctx.Process(target=_rank_main, args=(r, world, port, ret)) for r in range(world)]
    for pr in procs:
        pr.start()
    for pr in procs:
        pr.join(timeout=240)
        assert pr.exitcode == 0, f"rank exited with {pr.exitcode}"
    for r in range(world):
        assert all(ret[r].values()), f"rank {r}: {ret[r]}"
