"""The operators of post-training on packed documents as a decoder runs them together, on the CPU: a packed sample against its documents
one by one, training steps, the run loop with a document mask, the balance bias over steps, checkpoints and a resumed run."""
import io

import numpy as np
import pytest
import torch

from mlperf_training_b200.data.indexed import PackedSFTDataset, write_packed_sft
from mlperf_training_b200.models.gpt import GPT, GPTConfig, tiny_moe
from mlperf_training_b200.parallel.engine import OptimConfig
from mlperf_training_b200.trainer import loop
from mlperf_training_b200.trainer.pretrain import PretrainTrainer, TrainConfig

LENGTHS = (9, 1, 14, 7)


def config(**over):
    base = dict(n_layers=2, hidden=64, n_heads=4, n_kv_heads=2, head_dim=16, vocab_size=97, seq_len=40, moe_ffn_hidden=48, n_experts=8, top_k=3,
                window=8, router_score="sigmoid", router_groups=4, router_top_groups=2, router_scale=1.5, attn_softcap=3.0)
    base.update(over)
    return tiny_moe(**base)


def sample(cfg, K=5, pad=3, seed=0):
    """Tokens, labels, documents, prefix flags, teacher of one packed row, padded at its end."""
    g = torch.Generator().manual_seed(seed)
    S, V = sum(LENGTHS) + pad, cfg.vocab_size
    tokens = torch.randint(0, V, (1, S), generator=g)
    labels = torch.randint(0, V, (1, S), generator=g)
    labels[:, sum(LENGTHS):] = -100
    labels[:, 4] = -100
    docs = torch.cat([torch.full((n,), i) for i, n in enumerate(LENGTHS)] + [torch.full((pad,), -1)])[None]
    prefix = torch.zeros(1, S, dtype=torch.bool)
    at = 0
    for n in LENGTHS:
        prefix[0, at:at + n // 3] = True
        at += n
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(S)])[None]
    return tokens, labels, docs, prefix, (ids, 3 * torch.randn(1, S, K, generator=g))


@pytest.mark.parametrize("over", [dict(), dict(attn_alibi=True), dict(attn_softcap=0.0, router_score="softmax", router_groups=1, router_top_groups=0, router_scale=1.0)],
                         ids=["capped", "alibi", "plain"])
@pytest.mark.parametrize("distil", [None, dict(alpha=0.6, temperature=2.0)], ids=["labels", "teacher"])
def test_a_packed_sample_is_its_documents(over, distil):
    cfg = config(**over)
    tokens, labels, docs, prefix, teacher = sample(cfg)
    more = dict(teacher=teacher, distill=distil) if distil else {}
    model = GPT(cfg, seed=3)
    loss = model(tokens, labels, n_valid=1, documents=docs, prefix=prefix, **more)
    loss.backward()
    grads = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    total, at = 0.0, 0
    for n in LENGTHS:
        rows = slice(at, at + n)
        m = dict(teacher=tuple(t[:, rows] for t in teacher), distill=distil) if distil else {}
        part = model(tokens[:, rows], labels[:, rows], n_valid=1, prefix=prefix[:, rows], **m)
        part.backward()
        total += float(part.detach())
        at += n
    # fp32 throughout: sums in another order, rotary angles of other positions (the same differences)
    assert abs(float(loss.detach()) - total) <= 1e-4 * abs(total)
    for name, p in model.named_parameters():
        assert (p.grad - grads[name]).norm() <= 1e-3 * grads[name].norm() + 1e-6, name


def test_padding_gets_and_gives_nothing():
    cfg = config()
    tokens, labels, docs, prefix, teacher = sample(cfg)
    model = GPT(cfg, seed=3)
    run = lambda t: model(t, labels, n_valid=1, documents=docs, teacher=teacher, distill=dict(alpha=0.5))  # noqa: E731
    other = tokens.clone()
    other[:, sum(LENGTHS):] = 11
    assert float(run(tokens).detach()) == float(run(other).detach())


def test_without_documents_nothing_changes():
    cfg = config(attn_softcap=0.0, router_score="softmax", router_groups=1, router_scale=1.0, router_top_groups=0)
    tokens, labels, *_ = sample(cfg)
    assert cfg.plain_router and cfg.plain_scores
    model = GPT(cfg, seed=3)
    # one document that is everything: the masked path against the framework's own
    a = model(tokens, labels)
    b = model(tokens, labels, documents=torch.zeros_like(tokens))
    assert abs(float(a) - float(b)) <= 1e-5 * abs(float(a))


def trainer(cfg, **over):
    return PretrainTrainer(cfg, OptimConfig(lr=1e-3), TrainConfig(micro_batch=1, local_batch=2, warmup_steps=0, seed=5, **over), "cpu")


def batch(cfg, seed=0):
    parts = [sample(cfg, seed=seed + i) for i in range(2)]
    tokens, labels, docs, _ = (torch.cat([p[i] for p in parts]) for i in range(4))
    return tokens, labels, docs, tuple(torch.cat([p[4][i] for p in parts]) for i in range(2))


def test_training_steps_with_a_teacher_and_a_balance_bias():
    cfg = config(router_bias_rate=0.01)
    tr = trainer(cfg, distill=dict(alpha=0.8, temperature=2.0))
    tokens, labels, docs, teacher = batch(cfg)
    before = [b.clone() for b in tr.model.router_state()]
    first = float(tr.train_step_device(tokens, labels, docs, teacher))
    for b, a in zip(tr.model.router_state(), before):
        assert set(torch.unique((b - a).abs() * 100).round(decimals=3).tolist()) <= {0.0, 1.0} and (b != a).any()
    assert all(int(m.router_load.sum()) == 0 for m in tr.model.routers())
    second = float(tr.train_step_device(tokens, labels, docs, teacher))
    assert np.isfinite([first, second]).all()
    # the load is what moved the bias: experts below the mean went up
    with torch.enable_grad():
        tr.model(tokens, labels, documents=docs)
    load = tr.model.routers()[0].router_load.clone()
    old = tr.model.router_state()[0]
    tr.model.balance_routers()
    moved = tr.model.router_state()[0] - old
    assert torch.equal(torch.sign(moved), torch.sign(load.float().mean() - load.float()))
    with torch.no_grad():
        tr.model(tokens, labels)
    assert int(tr.model.routers()[0].router_load.sum()) == 0          # evaluation does not count


def test_recomputed_blocks_take_the_mask():
    tokens, labels, docs, prefix, teacher = sample(config())
    out = []
    for rc in ("none", "full"):
        model = GPT(config(recompute=rc), seed=3)
        loss = model(tokens, labels, documents=docs, prefix=prefix, teacher=teacher, distill=dict(alpha=0.5))
        loss.backward()
        out.append((float(loss), [p.grad.clone() for p in model.parameters()]))
    assert out[0][0] == out[1][0] and all(torch.equal(a, b) for a, b in zip(out[0][1], out[1][1]))


def test_packed_dataset_names_its_documents(tmp_path):
    f = str(tmp_path / "p.npy")
    write_packed_sft(f, [dict(input_ids=np.arange(12), seq_start_id=[0, 4, 9]), dict(input_ids=np.arange(7), seq_start_id=[0]),
                         dict(input_ids=np.arange(3))])
    ds = PackedSFTDataset(f, 10)
    assert ds.documents(0, 0, 1, 3).tolist() == [[1] * 4 + [2] * 5 + [3], [1] * 7 + [-1] * 3, [1] * 3 + [-1] * 7]
    assert ds.batch(0, 0, 1, 3)[0].shape == (3, 10)


def test_documents_of_a_token_stream():
    x = torch.tensor([[5, 9, 1, 9, 9, 2]])
    assert loop.document_ids(x, 9).tolist() == [[0, 0, 1, 1, 2, 3]]


def experiment(tmp_path, **over):
    model = dict(n_layers=2, hidden=32, n_heads=2, n_kv_heads=1, head_dim=16, ffn_hidden=64, vocab_size=50, seq_len=24, dtype="fp32")
    return {**dict(benchmark="t", model=model, train_iters=3, global_batch=2, micro_batch=1, warmup_train_steps=1, lr=1e-3, lr_warmup_iters=0,
                   eod_token=7), **over}


def test_run_loop_with_a_document_mask(tmp_path):
    kw = dict(eval_interval=3, eval_iters=1)
    plain = loop.run(experiment(tmp_path, **kw), device="cpu", stream=io.StringIO())
    masked = loop.run(experiment(tmp_path, document_mask=True, **kw), device="cpu", stream=io.StringIO())
    none = loop.run(experiment(tmp_path, document_mask=True, eod_token=49999, **kw), device="cpu", stream=io.StringIO())
    # no document ends: the same run
    assert np.allclose(none["losses"], plain["losses"], rtol=1e-4) and abs(none["eval_loss"] - plain["eval_loss"]) < 1e-3
    assert masked["losses"] != plain["losses"]
    f = str(tmp_path / "p.npy")
    rng = np.random.default_rng(0)
    write_packed_sft(f, [dict(input_ids=rng.integers(0, 50, 20 + i), seq_start_id=[0, 6, 11]) for i in range(8)])
    packed = loop.run(experiment(tmp_path, document_mask=True, data=dict(kind="packed_sft", path=f), **kw), device="cpu", stream=io.StringIO())
    assert np.isfinite(packed["losses"]).all()


def test_a_resumed_run_keeps_its_balance_bias(tmp_path):
    model = dict(preset="tiny-moe", n_layers=1, hidden=32, n_heads=2, n_kv_heads=1, head_dim=16, vocab_size=50, seq_len=24, moe_ffn_hidden=32,
                 router_score="sigmoid", router_bias_rate=0.01)
    kw = dict(model=model, train_iters=4)
    whole = loop.run(experiment(tmp_path, **kw), device="cpu", stream=io.StringIO())
    d = str(tmp_path / "ck")
    with pytest.raises(SystemExit):
        loop.run(experiment(tmp_path, checkpoint_dir=d, die_at_step=2, **kw), device="cpu", stream=io.StringIO())
    rest = loop.run(experiment(tmp_path, checkpoint_dir=d, **kw), device="cpu", stream=io.StringIO())
    assert rest["losses"] == whole["losses"][2:]
    bias = [r["trainer"].model.router_state() for r in (whole, rest)]
    assert len(bias[0]) == 1 and bias[0][0].abs().max() > 0 and torch.equal(bias[0][0], bias[1][0])


def test_refusals(tmp_path):
    with pytest.raises(NotImplementedError):
        loop.run(experiment(tmp_path, document_mask=True, pipeline_parallel=2), device="cpu", stream=io.StringIO())
    model = GPT(config(), seed=3)
    with pytest.raises(ValueError):
        model(torch.zeros(1, 8, dtype=torch.long), torch.zeros(1, 8, dtype=torch.long), documents=torch.zeros(1, 9, dtype=torch.long))
    with pytest.raises(ValueError):
        model.load_router_state([torch.zeros(8)])
