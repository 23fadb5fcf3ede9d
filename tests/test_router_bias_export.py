"""A router's balance bias travels with the model: ``state_dict`` and the ``torch_dist`` checkpoint."""
import pytest
import torch

from mlperf_training_b200.checkpoint import megatron as MG
from mlperf_training_b200.models.gpt import GPT, tiny_moe


def model(seed, rate=0.01, **over):
    cfg = tiny_moe(**dict(dict(n_layers=2, hidden=32, n_heads=2, n_kv_heads=1, head_dim=16, vocab_size=50, seq_len=16, moe_ffn_hidden=32, n_experts=8, top_k=2,
                               router_score="sigmoid", router_bias_rate=rate), **over))
    m = GPT(cfg, seed=seed)
    g = torch.Generator().manual_seed(seed)
    for r in m.routers():
        r.router_bias.copy_(torch.randn(8, generator=g))
        r.router_load.fill_(3)
    return m


def logits_loss(m):
    t = torch.arange(16)[None] % 50
    with torch.no_grad():
        return float(m(t, t.roll(1)))


def same(a, b):
    return len(a) > 0 and all(torch.equal(x, y) for x, y in zip(a, b, strict=True))


def test_state_dict():
    a, b = model(1), model(2)
    sd = a.state_dict()
    assert [n for n in sd if n.endswith("router_bias")] == [f"blocks.{i}.mlp.router_bias" for i in range(2)]
    assert not any("router_load" in n for n in sd)
    b.load_state_dict(sd)
    assert same(a.router_state(), b.router_state()) and logits_loss(a) == logits_loss(b)
    assert not any("router_bias" in n for n in model(1, rate=0.0).state_dict())


def test_torch_dist(tmp_path):
    a, b = model(1), model(2)
    names = MG.to_megatron_state(a)
    assert torch.equal(names["decoder.layers.1.mlp.router.expert_bias"], a.router_state()[1])
    assert MG.local_name("decoder.layers.1.mlp.router.expert_bias") == "blocks.1.mlp.router_bias"
    MG.save_torch_dist(a, str(tmp_path))
    assert MG.load_torch_dist(b, str(tmp_path))["missing"] == []
    assert same(a.router_state(), b.router_state()) and logits_loss(a) == logits_loss(b)
    c = model(3)
    assert MG.load_megatron_state(c, names) == [] and same(a.router_state(), c.router_state())


def test_a_checkpoint_without_one(tmp_path):
    """A model without a balance bias goes into one with it, whose bias starts at 0."""
    a, b = model(1, rate=0.0), model(2)
    MG.save_torch_dist(a, str(tmp_path))
    info = MG.load_torch_dist(b, str(tmp_path))
    assert info["missing"] == [f"blocks.{i}.mlp.router_bias" for i in range(2)]
    assert all((s == 0).all() for s in b.router_state()) and logits_loss(a) == logits_loss(b)


def test_a_model_without_a_place_for_it(tmp_path):
    a, b = model(1), model(2, rate=0.0)
    MG.save_torch_dist(a, str(tmp_path))
    with pytest.warns(UserWarning, match="balance bias"):
        MG.load_torch_dist(b, str(tmp_path))
    with pytest.warns(UserWarning, match="balance bias"):
        MG.load_megatron_state(b, MG.to_megatron_state(a))
