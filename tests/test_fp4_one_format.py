"""The fp4 recipe multiplies a weight in one format, whatever the number of tokens is."""
import pytest
import torch

from mlperf_training_b200.ops import functional as F


def devices():
    return ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def operands(dev, T, D=256, N=384):
    torch.manual_seed(T)
    dtype = torch.bfloat16 if dev == "cuda" else torch.float32
    x, nw, w = torch.randn(T, D), 1 + 0.1 * torch.randn(D), torch.randn(N, D) * D ** -0.5
    return x.to(dev, dtype), nw.to(dev, dtype), w.to(dev, dtype)


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("T", [1, 127, 129, 255, 300])
def test_rows_do_not_depend_on_how_many_there_are(dev, T):
    """The same operands: fp32 sums in another order, and at most a step of the result's type (2^-7) where that changes its rounding."""
    x, nw, w = operands(dev, 384)
    full = F.norm_linear(x, nw, w, precision="fp4").float()
    part, h = F.norm_linear(x[:T], nw, w, precision="fp4", pass_x=True)
    assert getattr(w, "_mx4_cache", None) is None and torch.equal(h, x[:T])
    assert float((part.float() - full[:T]).norm()) <= 2 ** -7 * float(full[:T].norm())
    alone, _ = F.add_norm_linear(x[:T], None, nw, w)
    assert torch.equal(alone, part)


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("T", [1, 100, 128, 131, 257])
def test_gradients_of_any_number_of_tokens(dev, T):
    """As for whole tiles of tokens: two operands of 8 bits in each product, 2^-5 of a value each at worst, a quarter of that in the mean."""
    x, nw, w = operands(dev, T)
    r = torch.randn_like(x)
    t = [v.requires_grad_() for v in (x, r, nw, w)]
    y, h = F.add_norm_linear(*t)
    dy, dh = torch.randn_like(y), torch.randn_like(h)
    dx, dr, dnw, dw = torch.autograd.grad([y, h], t, [dy, dh])
    assert torch.equal(dx, dr) and dx.shape == x.shape and dw.shape == w.shape
    hd, nd, wd = (v.detach().double().requires_grad_() for v in (h, nw.bfloat16(), w))
    yd = (hd * (hd.square().mean(1, keepdim=True) + 1e-5).rsqrt() * nd) @ wd.t()
    ref = torch.autograd.grad([yd, hd * 1.0], [hd, nd, wd], [dy.double(), dh.double()])
    for got, want in ((y, yd), (dx, ref[0]), (dnw, ref[1]), (dw, ref[2])):
        assert float((got.detach().double() - want.detach()).norm() / want.detach().norm()) < 2 ** -4


@pytest.mark.parametrize("dev", devices())
def test_no_tokens(dev):
    x, nw, w = (v.requires_grad_() for v in operands(dev, 1))
    e = x[:0].detach().requires_grad_()
    y, h = F.add_norm_linear(e, None, nw, w)
    assert y.shape == (0, 384) and h.shape == (0, 256)
    dx, dnw, dw = torch.autograd.grad(y.sum() + h.sum(), [e, nw, w])
    assert dx.shape == (0, 256) and not dnw.any() and not dw.any()
    assert F.norm_linear(e, nw, w, precision="fp4").shape == (0, 384)


@pytest.mark.parametrize("dev", devices())
def test_a_ragged_evaluation_leaves_no_4_bit_copies_behind_a_norm(dev):
    from mlperf_training_b200.models.gpt import GPT, GPTConfig
    m = GPT(GPTConfig(n_layers=2, hidden=128, n_heads=2, n_kv_heads=2, head_dim=64, ffn_hidden=128, vocab_size=256, seq_len=128,
                      dtype="bf16" if dev == "cuda" else "fp32", precision="fp4"), device=dev)
    t = torch.randint(0, 256, (1, 101), generator=torch.Generator().manual_seed(0)).to(dev)
    with torch.no_grad():
        loss = m(t[:, :-1], t[:, 1:])
    assert bool(loss.isfinite())
    for b in m.blocks:
        assert getattr(b.w_qkv, "_mx4_cache", None) is None and getattr(b.mlp.w_gate_up, "_mx4_cache", None) is None
        assert b.w_qkv._mx_cache is not None and b.w_proj._mx4_cache is not None


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("T", [1, 100, 256])
def test_vocabulary_projection_is_a_linear_behind_a_norm(dev, T):
    """Loss and gradients of the last norm and projection against 64 bits; the weight has 8-bit copies and no others.  (A logit is a sum
    of products off by 2^-4 at worst; the softmax hands that on, so the gradients get twice the bound of a product.)"""
    x, nw, w = operands(dev, T)
    labels = torch.randint(0, w.shape[0], (T,), generator=torch.Generator().manual_seed(T)).to(dev)
    t = [v.requires_grad_() for v in (x, nw, w)]
    loss = F.lm_head_loss(*t, labels, precision="fp4")
    got = torch.autograd.grad(loss, t)
    assert getattr(w, "_mx4_cache", None) is None and getattr(w, "_mx_cache", None) is not None
    td = [v.detach().double().requires_grad_() for v in (x, nw.bfloat16(), w)]
    yd = (td[0] * (td[0].square().mean(1, keepdim=True) + 1e-5).rsqrt() * td[1]) @ td[2].t()
    ref = torch.nn.functional.cross_entropy(yd, labels)
    assert abs(float(loss.detach()) - float(ref.detach())) < 2 ** -4
    for a, b in zip(got, torch.autograd.grad(ref, td)):
        assert float((a.double() - b).norm() / b.norm()) < 2 ** -3


@pytest.mark.parametrize("dev", devices())
def test_a_model_step_leaves_8_bit_copies_behind_every_norm(dev):
    from mlperf_training_b200.models.gpt import GPT, GPTConfig
    m = GPT(GPTConfig(n_layers=2, hidden=128, n_heads=2, n_kv_heads=2, head_dim=64, ffn_hidden=128, vocab_size=256, seq_len=128,
                      dtype="bf16" if dev == "cuda" else "fp32", precision="fp4"), device=dev)
    t = torch.randint(0, 256, (1, 129), generator=torch.Generator().manual_seed(0)).to(dev)
    m(t[:, :-1], t[:, 1:]).backward()
    for w in [m.lm_head] + [w for b in m.blocks for w in (b.w_qkv, b.mlp.w_gate_up)]:
        assert w._mx_cache is not None and getattr(w, "_mx4_cache", None) is None and bool(w.grad.isfinite().all())
    for w in [w for b in m.blocks for w in (b.w_proj, b.mlp.w_down)]:
        assert w._mx4_cache is not None and getattr(w, "_mx_cache", None) is None


def test_deoscillation_goes_by_the_copies_of_the_last_step():
    """4-bit copies that something made of a weight before the last step (an evaluation, an earlier recipe) do not put it on the grid."""
    from mlperf_training_b200.ops import linear as L
    from mlperf_training_b200.ops.recipe import DeoscConfig, Deoscillator
    from mlperf_training_b200.parallel.engine import OptimConfig, ZeroEngine
    torch.manual_seed(0)
    w4, w8 = torch.nn.Parameter(torch.randn(32, 64)), torch.nn.Parameter(torch.randn(32, 64))
    engine = ZeroEngine(torch.nn.ParameterList([w4, w8]), OptimConfig())
    d = Deoscillator(engine, DeoscConfig(enabled=True, start_step=0, period=100, ratio=2.0))
    tracked = lambda: {p.data_ptr(): bool(d._keys(b, "fp4")[0][o - b.lo]) for b in engine.buckets for (_, p), o in zip(b.params, b.offsets)}
    x = torch.randn(1, 64)
    with torch.no_grad():
        F.mxfp4_linear(x, w8)
        for step in range(3):
            F.mxfp4_linear(x, w4)                # the forward of a step
            L.bump_weight_epoch()                # and its update
            t = tracked()
            d.after_step(step, "fp4")
    assert t[w4.data_ptr()] and not t[w8.data_ptr()]


def test_experts_stay_in_bf16_and_say_so():
    """A mixture-of-experts decoder in the recipe: the experts are as the bf16 model has them, the attention's weights are not, and a warning
    tells the two apart."""
    from mlperf_training_b200.models.gpt import GPT, GPTConfig
    from mlperf_training_b200.ops import moe_ops as M
    cfg = dict(n_layers=1, hidden=128, n_heads=2, n_kv_heads=2, head_dim=64, ffn_hidden=128, vocab_size=256, seq_len=128, n_experts=4, top_k=2)
    m = GPT(GPTConfig(**cfg, precision="fp4"))
    moe = m.blocks[0].mlp
    M._say_experts_in_bf16.cache_clear()
    with pytest.warns(UserWarning, match="experts.*bf16"):
        assert M.expert_precision("fp4", moe.w1, moe.w2) == "bf16"
    t = torch.randint(0, 256, (1, 129), generator=torch.Generator().manual_seed(0))
    m(t[:, :-1], t[:, 1:]).backward()
    assert getattr(moe.w1, "_mx_stack", None) is None and getattr(m.blocks[0].w_proj, "_mx4_cache", None) is not None
    assert bool(moe.w1.grad.isfinite().all())
