"""The operators of post-training on packed documents together, on the GPU's kernels: a packed sample against its documents one by one, against the
CPU's bodies, and training steps with a balance bias and a teacher."""
import pytest
import torch

from mlperf_training_b200.models.gpt import GPT, GPTConfig
from mlperf_training_b200.ops import _lib
from mlperf_training_b200.parallel.engine import OptimConfig
from mlperf_training_b200.trainer.pretrain import PretrainTrainer, TrainConfig

pytestmark = pytest.mark.gpu

LENGTHS = (130, 1, 77, 200, 60)


def config(**over):
    base = dict(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn_hidden=256, vocab_size=1000, seq_len=512, n_experts=8, top_k=3,
                moe_ffn_hidden=192, window=96, window_layers="even", sink=True, router_score="sigmoid", router_groups=4, router_top_groups=2,
                router_scale=1.5, attn_softcap=5.0)
    base.update(over)
    return GPTConfig(**base)


def sample(cfg, K=9, pad=44, seed=0, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    S, V = sum(LENGTHS) + pad, cfg.vocab_size
    tokens, labels = (torch.randint(0, V, (1, S), generator=g) for _ in range(2))
    labels[:, sum(LENGTHS):] = -100
    docs = torch.cat([torch.full((n,), i) for i, n in enumerate(LENGTHS)] + [torch.full((pad,), -1)])[None]
    prefix = torch.zeros(1, S, dtype=torch.bool)
    at = 0
    for n in LENGTHS:
        prefix[0, at:at + n // 3] = True
        at += n
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(S)])[None]
    t = (ids.to(dev), (3 * torch.randn(1, S, K, generator=g)).to(dev))
    return tokens.to(dev), labels.to(dev), docs.to(dev), prefix.to(dev), t


@pytest.mark.parametrize("over", [dict(), dict(attn_alibi=True, n_experts=0, ffn_hidden=384)], ids=["capped", "alibi-dense"])
def test_a_packed_sample_is_its_documents(over):
    cfg = config(**over)
    tokens, labels, docs, prefix, teacher = sample(cfg)
    distil = dict(alpha=0.6, temperature=2.0)
    model = GPT(cfg, device="cuda", seed=3)
    with torch.no_grad():
        whole = float(model(tokens, labels, n_valid=1, documents=docs, prefix=prefix, teacher=teacher, distill=distil))
        total, at = 0.0, 0
        for n in LENGTHS:
            rows = slice(at, at + n)
            total += float(model(tokens[:, rows], labels[:, rows], n_valid=1, prefix=prefix[:, rows], teacher=tuple(t[:, rows] for t in teacher),
                                 distill=distil))
            at += n
    # bf16 activations: roundings of other rotary angles; a token's loss moves by a few 2^-8, and 468 of them average out
    assert abs(whole - total) <= 2 ** -8 * abs(total)
    _lib.check_status("packed")


def test_against_the_cpu():
    cfg = config(n_layers=1)
    out = []
    for dev in ("cpu", "cuda"):
        model = GPT(cfg, device="cpu", seed=3).to(dev)
        tokens, labels, docs, prefix, teacher = sample(cfg, dev=dev)
        loss = model(tokens, labels, documents=docs, prefix=prefix, teacher=teacher, distill=dict(alpha=0.6, temperature=2.0))
        loss.backward()
        out.append((float(loss.detach()), {n: p.grad.float().cpu() for n, p in model.named_parameters()}))
    assert abs(out[0][0] - out[1][0]) <= 2 ** -8 * abs(out[0][0])
    for n, g in out[0][1].items():
        # bf16 in every product on both sides, in another order; a token whose router is near a tie goes elsewhere
        assert (g - out[1][1][n]).norm() <= 0.1 * g.norm() + 1e-6, n
    _lib.check_status("model")


def test_training_steps():
    cfg = config(router_bias_rate=0.01)
    tr = PretrainTrainer(cfg, OptimConfig(lr=1e-3), TrainConfig(micro_batch=1, local_batch=2, warmup_steps=0, distill=dict(alpha=0.8)), "cuda")
    parts = [sample(cfg, seed=i) for i in range(2)]
    tokens, labels, docs, _ = (torch.cat([p[i] for p in parts]) for i in range(4))
    teacher = tuple(torch.cat([p[4][i] for p in parts]) for i in range(2))
    losses = [float(tr.train_step_device(tokens, labels, docs, teacher)) for _ in range(3)]
    assert all(x == x and abs(x) < 1e4 for x in losses)
    for b in tr.model.router_state():
        assert 0 < float(b.abs().max()) <= 0.03 + 1e-6
    _lib.check_status("steps")
