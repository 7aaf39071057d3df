"""Per-head norms, the head without logits and Muon inside the model and the trainer (B200)."""

import dataclasses
import json

import pytest
import torch

pytestmark = pytest.mark.gpu

CFG = dict(vocab_size=1000, context_length=256, d_model=128, num_layers=2, num_heads=2, d_ff=344,
           rope_theta=10000.0, attention_backend="sdpa")


@pytest.fixture(scope="module")
def dev():
    from systems_for_llms_b200.ops import lib
    if not lib.available():
        pytest.skip("kernels need a compute-capability 10.x device")
    return torch.device("cuda", torch.cuda.current_device())


def build(dev, **overrides):
    from systems_for_llms_b200.models.transformer import TransformerLM
    torch.manual_seed(0)
    model = TransformerLM(**{**CFG, **overrides}, device=dev, dtype=torch.float32)
    if model.qk_norm:       # weights of one would hide a swapped or missing product
        gen = torch.Generator(device=dev).manual_seed(5)
        for layer in model.layers:
            for norm in (layer.attn.q_norm, layer.attn.k_norm):
                norm.weight.data += 0.2 * torch.randn(norm.weight.shape, device=dev, generator=gen)
    return model


def batch(dev, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    draw = lambda: torch.randint(0, 1000, (3, 256), device=dev, generator=gen)
    return draw(), draw()


def relative(a, b):
    return ((a - b).norm() / (b.norm() + 1e-12)).item()


@pytest.mark.parametrize("ckpt", ["none", "block"])
@pytest.mark.parametrize("head_loss", ["logits", "pieces"])
@pytest.mark.parametrize("d_model", [128, 256])        # head dimensions 64 and 128
def test_qk_norm_model_matches_portable(dev, ckpt, head_loss, d_model):
    """The fused engine rounds activations to bf16 where the portable path under autocast does;
    gradients of two bf16 paths agree to a few percent (the bound of the model without options)."""
    from systems_for_llms_b200.ops.gemm import check_status
    options = dict(qk_norm=True, head_loss=head_loss, activation_checkpointing=ckpt, d_model=d_model)
    fused, plain = build(dev, **options), build(dev, **options)
    plain.disable_fused()
    x, y = batch(dev)
    for _ in range(2):      # the second pass accumulates
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss_f, loss_p = fused.loss(x, y, 0.5), plain.loss(x, y, 0.5)
        loss_f.backward()
        loss_p.backward()
    torch.cuda.synchronize()
    check_status()
    assert fused._fused is not None
    assert loss_f.item() == pytest.approx(loss_p.item(), rel=2e-3)
    for (name, a), (_, b) in zip(fused.named_parameters(), plain.named_parameters()):
        assert relative(a.grad, b.grad) < 0.03, name
        assert a.grad.data_ptr() == fused._fused.grad_view(a).data_ptr()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert relative(fused(x).float(), plain(x).float()) < 0.02


def test_head_without_logits_agrees_with_the_one_that_keeps_them(dev):
    """The two heads share everything up to the final norm.  Keeping the logits rounds each to
    bf16 (2^-8 of logits of size below 4 here): losses agree to 0.02, and to a few percent the
    gradients, whose probabilities that rounding moves."""
    kept, pieces = build(dev), build(dev, head_loss="pieces")
    x, y = batch(dev)
    for model in (kept, pieces):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            model.loss(x, y, 0.5).backward()
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.no_grad():
        a, b = kept.loss(x, y).item(), pieces.loss(x, y).item()
    assert abs(a - b) < 0.02
    for (name, p), (_, q) in zip(kept.named_parameters(), pieces.named_parameters()):
        assert relative(q.grad, p.grad) < 0.03, name
    # a factor on the loss reaches every gradient, exactly for a power of two
    first = [p.grad.clone() for p in pieces.parameters()]
    pieces.zero_grad(set_to_none=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        (pieces.loss(x, y, 0.5) * -4.0).backward()
    for g, p in zip(first, pieces.parameters()):
        assert relative(p.grad, -4.0 * g) < 1e-6


def test_head_gradient_against_64_bits(dev):
    """The head alone: 64-bit gradients of the mean cross entropy of the same bf16 operands."""
    from systems_for_llms_b200.models import fused as F
    model = build(dev, head_loss="pieces")
    x, y = batch(dev)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        model.loss(x, y).backward()
    engine = model._fused
    hidden = torch.randn(3 * 256, 128, device=dev)
    loss, saved = F.head_loss_pieces(engine, hidden, y.reshape(-1))
    model.zero_grad(set_to_none=True)
    F.head_loss_pieces_backward(engine, saved, torch.ones((), device=dev))
    h = saved[1].double()
    w = engine.shadow(model.lm_head.weight).double().requires_grad_()
    want = torch.nn.functional.cross_entropy(h @ w.t(), y.reshape(-1))
    (dw,) = torch.autograd.grad(want, w)
    assert loss.item() == pytest.approx(want.item(), rel=1e-5)
    # dl is rounded to bf16 (2^-8 at most, rms 2^-8 / sqrt(3)), everything else is fp32
    assert relative(model.lm_head.weight.grad.double(), dw) < 2.0 ** -8


def test_muon_step_matches_the_portable_one(dev):
    """Same gradients on both paths: the matrices' steps differ by the kernel's error (below 0.0025
    of the direction's norm, doubled for small matrices), the others by fp32 rounding."""
    from systems_for_llms_b200.ops.gemm import check_status
    from systems_for_llms_b200.optim import FusedMuon
    fused, plain = build(dev, qk_norm=True), build(dev, qk_norm=True)
    plain.disable_fused()
    x, y = batch(dev)
    kw = dict(lr=0.01, momentum=0.9, weight_decay=0.1)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        fused.loss(x, y).backward()
    opt_f = FusedMuon.from_model(fused, engine=fused._fused, **kw)
    opt_p = FusedMuon.from_model(plain, **kw)
    assert opt_f._fused_ready() and not opt_p._fused_ready()
    for step in range(3):
        for p, q in zip(fused.parameters(), plain.parameters()):
            q.grad = p.grad.clone()
            q.data.copy_(p.data)
        norm_f = opt_f.clip_and_step(0.5)
        norm_p = opt_p.clip_and_step(0.5)
        check_status()
        assert norm_f.item() == pytest.approx(norm_p.item(), rel=1e-4)
        matrices = {id(p) for layer in fused.layers for p in layer.parameters() if p.dim() == 2}
        for (name, p), q in zip(fused.named_parameters(), plain.parameters()):
            bound = 5e-3 if id(p) in matrices else 1e-4
            state_f, state_p = opt_f.state[p], opt_p.state[q]
            for key in state_f:
                if key != "step":
                    assert relative(state_f[key], state_p[key]) < 1e-5, (name, key)
            assert float(state_f["step"]) == float(state_p["step"]) == step + 1
            change = (p.detach() - q.detach()).norm().item()
            size = 0.01 * 0.2 * max(p.shape) ** 0.5 * min(p.shape) ** 0.5 if id(p) in matrices \
                else 0.01 * p.numel() ** 0.5
            assert change <= bound * size, name
        # the shadow the kernels read is the updated parameter in bf16
        engine = fused._fused
        assert torch.equal(engine.flat_shadow, engine.flat_param.bfloat16())
        fused.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            fused.loss(*batch(dev, seed=step + 1)).backward()


def test_muon_skips_a_step_with_infinite_gradients(dev):
    from systems_for_llms_b200.optim import FusedMuon
    model = build(dev)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        model.loss(*batch(dev)).backward()
    optimizer = FusedMuon.from_model(model, engine=model._fused, lr=0.01)
    optimizer.clip_and_step(1.0)
    before = [p.detach().clone() for p in model.parameters()]
    held = [{k: v.clone() for k, v in optimizer.state[p].items() if k != "step"}
            for p in model.parameters()]
    model.layers[0].ffn.w2.weight.grad[0, 0] = float("inf")
    assert not torch.isfinite(optimizer.clip_and_step(1.0))
    for p, q, h in zip(model.parameters(), before, held):
        assert torch.equal(p, q)
        assert all(torch.equal(optimizer.state[p][k], v) for k, v in h.items())


def test_muon_state_survives_a_checkpoint(dev):
    from systems_for_llms_b200.optim import FusedMuon
    model = build(dev)

    def step(m, o, seed):
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            m.loss(*batch(dev, seed)).backward()
        o.engine = m._fused
        o.clip_and_step(1.0)

    optimizer = FusedMuon.from_model(model, lr=0.01)
    step(model, optimizer, 1)
    weights = {k: v.clone() for k, v in model.state_dict().items()}
    saved = torch.load(_roundtrip(optimizer.state_dict()), weights_only=True)
    step(model, optimizer, 2)
    other = build(dev)
    other.load_state_dict(weights)
    resumed = FusedMuon.from_model(other, lr=0.01)
    resumed.load_state_dict(saved)
    step(other, resumed, 2)
    for p, q in zip(model.parameters(), other.parameters()):
        assert torch.equal(p, q)


def _roundtrip(state):
    import io
    buffer = io.BytesIO()
    torch.save(state, buffer)
    buffer.seek(0)
    return buffer


def test_trainer_runs_with_every_option(dev, tmp_path):
    from systems_for_llms_b200 import train as trainer
    from systems_for_llms_b200.config import DataConfig, ModelConfig, TrainConfig
    config = TrainConfig(
        model=ModelConfig(**{k: v for k, v in CFG.items() if k != "rope_theta"}, qk_norm=True,
                          head_loss="pieces"),
        data=DataConfig(kind="synthetic", synthetic_tokens=20000), device="cuda", precision="bf16",
        batch_size=2, grad_accum_steps=2, max_steps=6, warmup_steps=1, learning_rate=1e-3,
        min_learning_rate=1e-4, eval_interval=3, eval_batches=2, eval_batch_size=2,
        checkpoint_interval=3, optimizer="muon")
    summary = trainer.run(config, tmp_path / "run")
    assert summary["status"] == "completed" and summary["execution_path"] == "sm_100a fused engine"
    rows = [json.loads(line) for line in (tmp_path / "run" / "metrics.jsonl").read_text().splitlines()]
    assert all(r["loss"] > 0 and r["gradient_norm"] > 0 for r in rows if r["event"] == "train")
    trainer.run(config, tmp_path / "a", stop_after=3)
    resumed = trainer.run(config, tmp_path / "b", resume=tmp_path / "a" / "checkpoint.pt")
    # the same operations on the same numbers, in a fixed order
    assert resumed["valid_loss"] == summary["valid_loss"]
    with pytest.raises(ValueError, match="resume configuration"):
        trainer.run(dataclasses.replace(config, optimizer="adamw"), tmp_path / "c",
                    resume=tmp_path / "a" / "checkpoint.pt")


def test_runner_strategy_steps_with_muon(dev):
    """The runner's single mode drives the same optimizer through clip_and_step."""
    from systems_for_llms_b200.config import ModelConfig, TrainConfig
    from systems_for_llms_b200.optim import FusedMuon
    from systems_for_llms_b200.parallel.train import Strategy
    config = TrainConfig(model=ModelConfig(**CFG), device="cuda", precision="bf16", optimizer="muon")
    model = build(dev)
    strategy = Strategy("single", model, config, dev, world=1, rank=0, sync_policy="last",
                        bucket_cap_mb=25)
    assert isinstance(strategy.optimizer, FusedMuon) and strategy.optimizer.engine is model._fused
    with torch.autocast("cuda", dtype=torch.bfloat16):
        model.loss(*batch(dev)).backward()
    before = model.layers[0].attn.q_proj.weight.detach().clone()
    norm = strategy.reduce_and_update()
    assert norm.item() > 0 and not torch.equal(before, model.layers[0].attn.q_proj.weight)
