"""Options beyond the reference's schema on the CPU: configuration, portable model, Muon, refusals."""

import copy
import dataclasses
import json

import pytest
import torch

from systems_for_llms_b200.config import DataConfig, ModelConfig, TrainConfig, load_config
from systems_for_llms_b200.models.attention import MultiHeadSelfAttention
from systems_for_llms_b200.models.transformer import TransformerLM
from systems_for_llms_b200.optim import FusedMuon
from systems_for_llms_b200.ops.newton_schulz import newton_schulz_portable
from systems_for_llms_b200.parallel.train import check_extensions

TINY = dict(vocab_size=32, context_length=8, d_model=16, num_layers=2, num_heads=4, d_ff=24,
            rope_theta=10000.0)


def test_defaults_keep_the_old_form_of_a_configuration():
    plain = TrainConfig().to_dict()
    assert not {"optimizer", "muon_momentum"} & set(plain)
    assert not {"qk_norm", "head_loss"} & set(plain["model"])
    config = TrainConfig(model=ModelConfig(qk_norm=True, head_loss="pieces"), optimizer="muon",
                         muon_momentum=0.9)
    chosen = config.to_dict()
    assert chosen["model"]["qk_norm"] is True and chosen["model"]["head_loss"] == "pieces"
    assert chosen["optimizer"] == "muon" and chosen["muon_momentum"] == 0.9


def test_options_load_from_json(tmp_path):
    document = {"model": {"vocab_size": 64, "qk_norm": True, "head_loss": "pieces"},
                "data": {"kind": "synthetic"}, "max_steps": 5, "warmup_steps": 1,
                "optimizer": "muon", "muon_momentum": 0.8}
    path = tmp_path / "c.json"
    path.write_text(json.dumps(document))
    config = load_config(path)
    assert config.model.qk_norm and config.optimizer == "muon" and config.muon_momentum == 0.8


@pytest.mark.parametrize("change", [dict(optimizer="sgd"), dict(muon_momentum=1.0),
                                    dict(muon_momentum=-0.1), dict(muon_momentum=float("nan"))])
def test_bad_top_level_options_are_refused(change):
    with pytest.raises(ValueError):
        dataclasses.replace(TrainConfig(), **change).validate()


@pytest.mark.parametrize("change", [dict(qk_norm=1), dict(qk_norm="yes"), dict(head_loss="fp8")])
def test_bad_model_options_are_refused(change):
    with pytest.raises(ValueError):
        TrainConfig(model=ModelConfig(**change)).validate()
    if "head_loss" in change:
        with pytest.raises(ValueError):
            TransformerLM(**TINY, **change)


@pytest.mark.parametrize("mode", ["single", "naive", "ddp", "zero1", "fsdp", "tp"])
def test_sharded_modes_refuse_what_they_do_not_cover(mode):
    base = TrainConfig()
    check_extensions(base, mode)
    for config, refused in (
            (dataclasses.replace(base, optimizer="muon"), ("zero1", "fsdp", "tp")),
            (dataclasses.replace(base, model=ModelConfig(qk_norm=True)), ("fsdp", "tp")),
            (dataclasses.replace(base, model=ModelConfig(head_loss="pieces")), ("fsdp", "tp"))):
        if mode in refused:
            with pytest.raises(ValueError, match=mode):
                check_extensions(config, mode)
        else:
            check_extensions(config, mode)


def test_tensor_parallel_surgery_refuses_per_head_norms():
    from systems_for_llms_b200.parallel.tensor_parallel import parallelize_model
    with pytest.raises(ValueError, match="norms"):
        parallelize_model(TransformerLM(**TINY, qk_norm=True))


@pytest.mark.parametrize("option", [dict(qk_norm=True), dict(head_loss="pieces")])
def test_fused_sharded_model_refuses_what_it_does_not_cover(option):
    from systems_for_llms_b200.parallel.fsdp_fused import FusedShardedTransformer
    with pytest.raises(ValueError, match="not supported"):
        FusedShardedTransformer(TransformerLM(**TINY, **option), None)


def test_qk_norm_leaves_the_random_stream_alone_and_adds_two_weights_per_layer():
    torch.manual_seed(3)
    plain = TransformerLM(**TINY)
    torch.manual_seed(3)
    normed = TransformerLM(**TINY, qk_norm=True)
    extra = set(normed.state_dict()) - set(plain.state_dict())
    assert extra == {f"layers.{i}.attn.{n}.weight" for i in range(2) for n in ("q_norm", "k_norm")}
    for name, value in plain.state_dict().items():
        assert torch.equal(value, normed.state_dict()[name])


def test_qk_norm_attention_matches_its_definition():
    torch.manual_seed(0)
    attention = MultiHeadSelfAttention(16, 2, theta=100.0, max_seq_len=6, qk_norm=True).double()
    attention.q_norm.weight.data.uniform_(0.5, 1.5)
    attention.k_norm.weight.data.uniform_(0.5, 1.5)
    x = torch.randn(2, 6, 16, dtype=torch.float64)
    heads = lambda t: t.view(2, 6, 2, 8).transpose(1, 2)
    q, k, v = (heads(p(x)) for p in (attention.q_proj, attention.k_proj, attention.v_proj))
    # RMSNorm works in fp32: its results are known to fp32
    norm = lambda t, w: t / (t.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w
    positions = torch.arange(6)
    q = attention.rope(norm(q, attention.q_norm.weight), positions)
    k = attention.rope(norm(k, attention.k_norm.weight), positions)
    scores = (q @ k.transpose(-1, -2) / 8 ** 0.5).masked_fill(
        ~torch.ones(6, 6, dtype=torch.bool).tril(), float("-inf"))
    want = attention.output_proj((scores.softmax(-1) @ v).transpose(1, 2).flatten(-2))
    assert torch.allclose(attention(x), want, rtol=1e-5, atol=1e-6)


def test_portable_newton_schulz_against_64_bits():
    for shape in ((5, 9), (9, 5), (2, 3, 8, 8)):
        u = torch.randn(*shape, generator=torch.Generator().manual_seed(1))
        left, s, right = torch.linalg.svd(u.double(), full_matrices=False)
        s = s / (s.square().sum(-1, keepdim=True).sqrt() + 1e-7)
        for _ in range(5):
            s = s * (3.4445 + s ** 2 * (-4.7750 + 2.0315 * s ** 2))
        want = left * s[..., None, :] @ right
        # five steps multiply fp32 roundings by at most 4 each, of matrices of norm below 3
        assert (newton_schulz_portable(u).double() - want).norm() < 4 ** 5 * 3 * 2.0 ** -24 * 10


def test_muon_on_the_cpu_follows_its_definition():
    torch.manual_seed(0)
    model = TransformerLM(**TINY, qk_norm=True)
    optimizer = FusedMuon.from_model(model, lr=0.02, momentum=0.9, weight_decay=0.1)
    matrices = [p for layer in model.layers for p in layer.parameters() if p.dim() == 2]
    others = [p for p in model.parameters() if all(p is not q for q in matrices)]
    assert len(matrices) == 14 and len(others) == 2 + 1 + 2 * 4
    adamw = torch.optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in others], lr=0.02,
                              betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    momentum = [torch.zeros_like(p) for p in matrices]
    expect = [p.detach().clone() for p in matrices]
    for step in range(3):
        x = torch.randint(0, 32, (2, 8))
        optimizer.zero_grad(set_to_none=True)
        model.loss(x, x).backward()
        for v, w, p in zip(momentum, expect, matrices):
            v.mul_(0.9).add_(p.grad)
            direction = newton_schulz_portable(p.grad + 0.9 * v)
            w.mul_(1 - 0.02 * 0.1).add_(direction, alpha=-0.02 * 0.2 * max(w.shape) ** 0.5)
        for q, p in zip(adamw.param_groups[0]["params"], others):
            q.grad = p.grad.clone()
        optimizer.step()
        adamw.step()
        for w, p in zip(expect, matrices):
            assert torch.allclose(p, w, rtol=1e-6, atol=1e-7)
        for q, p in zip(adamw.param_groups[0]["params"], others):
            assert torch.allclose(p, q, rtol=1e-5, atol=1e-7)
    # state round trip
    state = copy.deepcopy(optimizer.state_dict())
    again = FusedMuon.from_model(model, lr=0.5)
    again.load_state_dict(state)
    assert again.param_groups[0]["lr"] == 0.02
    held = again.state[matrices[0]]
    assert torch.equal(held["momentum_buffer"], optimizer.state[matrices[0]]["momentum_buffer"])
    assert float(held["step"]) == 3


def test_muon_refuses_bad_arguments():
    matrix, vector = torch.nn.Parameter(torch.zeros(4, 4)), torch.nn.Parameter(torch.zeros(4))
    for args, kw in ((([vector], []), {}), (([matrix], []), dict(momentum=1.0)),
                     (([matrix], []), dict(steps=0)), (([matrix], []), dict(lr=-1.0)),
                     (([matrix], []), dict(weight_decay=-0.1)), (([], []), {})):
        with pytest.raises(ValueError):
            FusedMuon(*args, **kw)
    FusedMuon([matrix], [vector])


def test_trainer_runs_on_the_cpu_with_the_options(tmp_path):
    from systems_for_llms_b200 import train as trainer
    config = TrainConfig(model=ModelConfig(**TINY, qk_norm=True, head_loss="pieces"),
                         data=DataConfig(kind="synthetic", synthetic_tokens=256), batch_size=2,
                         max_steps=4, learning_rate=1e-3, min_learning_rate=1e-4, warmup_steps=1,
                         eval_interval=2, eval_batches=2, eval_batch_size=1, checkpoint_interval=2,
                         optimizer="muon")
    whole = trainer.run(config, tmp_path / "whole")
    trainer.run(config, tmp_path / "a", stop_after=2)
    resumed = trainer.run(config, tmp_path / "b", resume=tmp_path / "a" / "checkpoint.pt")
    assert whole["status"] == "completed" and resumed["valid_loss"] == whole["valid_loss"]
