"""The paged model path on the GPU against the reference model's dataflow with unrounded probabilities (oracle/paged.py)."""
import pytest
import torch

from oracle import opt_model as OM
from oracle import paged as P
from test_paged_gpu import close, opt_model, prompts_of  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def test_logits_follow_the_unrounded_dataflow(cuda_ops, opt_model, monkeypatch):  # noqa: F811
    """A batch of prompts, then a chunk and a single token; the bound is that of close(): contexts may differ by a unit where
    they lie near a half."""
    sd = {k: v.detach().cpu() for k, v in opt_model.state_dict().items()}
    monkeypatch.setattr(OM, "attention", P.model_attention)

    def want(*parts):
        return OM.causal_lm_logits(sd, opt_model.model.decoder.config, torch.cat(parts).view(1, -1).cpu())[0][0, -1:].cuda()
    prompts = prompts_of(200, 1, 37)
    cache = opt_model.new_paged_cache(24)
    seqs = [cache.open() for _ in prompts]
    got = opt_model.forward_paged(torch.cat(prompts), cache, cache.step(seqs, [200, 1, 37]))
    for i, p in enumerate(prompts):
        assert close(got[i:i + 1], want(p))
    new = prompts_of(60, 1)
    got = opt_model.forward_paged(torch.cat(new), cache, cache.step([seqs[2], seqs[0]], [60, 1]))
    assert close(got[0:1], want(prompts[2], new[0])) and close(got[1:2], want(prompts[0], new[1]))
    assert cuda_ops.device_status() == 0


def test_a_single_token_agrees_with_the_static_path(cuda_ops, opt_model):  # noqa: F811
    """The only probability is 1 on both paths."""
    x = prompts_of(1)[0]
    cache = opt_model.new_paged_cache(1)
    got = opt_model.forward_paged(x, cache, cache.step([cache.open()], [1]))
    assert close(got, opt_model(x.view(1, 1)).logits[0])
    assert cuda_ops.device_status() == 0
