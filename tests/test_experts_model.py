"""GPT with a mixture of experts: configuration and parameter accounting (CPU),
the whole layer's gradients against a 64-bit restatement with autograd, and the
trainer's ways of running a step (GPU)."""
import pytest

CONFIG = dict(layers=2, hidden=256, ffn=512, heads=2, sequence=128, micro_batch=2, accumulation_steps=2, vocab=512,
              chunk_rows=128, experts=8, experts_per_token=2)


def test_configuration_and_counts():
    from tempname_dcu_b200.models.config import parameter_counts, train_flops_per_step, validate_config
    from tempname_dcu_b200.models.params import FlatParams, gpt_param_specs
    c = validate_config(CONFIG, 1)
    flat = FlatParams(gpt_param_specs(c, 1), "cpu")
    counts = parameter_counts(c, 1)
    assert flat.numel_logical() == counts["logical_parameters"] == counts["parameters_per_rank"]
    assert flat.p("layers.1.fc1_weight").shape == (8, 512, 256)
    dense = {k: v for k, v in CONFIG.items() if not k.startswith("experts")}
    assert "experts" not in validate_config(dense, 1) and "experts_per_token" not in validate_config(dense, 1)
    # two experts per token double the feed-forward products and add the router's
    extra = 6.0 * 512 * 2 * (2 * 256 * 512 + 8 * 256)
    assert train_flops_per_step(CONFIG) == pytest.approx(train_flops_per_step(dense) + extra)


@pytest.mark.parametrize("changes", [{"experts": 0}, {"experts": 12}, {"experts": 520}, {"experts": True},
                                     {"experts_per_token": 0}, {"experts_per_token": 9}, {"experts_per_token": 2.0}])
def test_configuration_refusals(changes):
    from tempname_dcu_b200.models.config import validate_config
    with pytest.raises(ValueError):
        validate_config(dict(CONFIG, **changes), 1)
    with pytest.raises(ValueError):
        validate_config(CONFIG, 2)
    with pytest.raises(ValueError):
        validate_config({"experts_per_token": 2}, 1)


def test_baseline_refuses_experts():
    from tempname_dcu_b200.models.torch_baseline import BaselineTrainer
    with pytest.raises(ValueError):
        BaselineTrainer(CONFIG, device="cpu")


def _reference(model, tokens, targets, chosen):
    """Loss and gradients in 64 bits from the model's bf16 parameters, with the
    experts that the model chose (a near tie may fall differently in 64 bits)."""
    import torch
    import torch.nn.functional as F
    c = model.config
    P = {n: model.P(n).double().requires_grad_(True) for n in model.params.order}
    seq, mb, h = c["sequence"], c["micro_batch"], c["hidden"]
    x = P["embedding"][tokens] + P["position"].repeat(mb, 1)
    for i in range(c["layers"]):
        p = f"layers.{i}."
        a = F.layer_norm(x, (h,), P[p + "ln1_weight"], P[p + "ln1_bias"], c["layer_norm_epsilon"])
        q, k, v = (a @ P[p + "qkv_weight"].t() + P[p + "qkv_bias"]).view(mb, seq, 3, c["heads"], 128).permute(2, 0, 3, 1, 4)
        s = q @ k.transpose(-1, -2) / 128 ** 0.5
        s = s.masked_fill(torch.ones(seq, seq, device=s.device).triu(1).bool(), float("-inf"))
        o = (s.softmax(-1) @ v).transpose(1, 2).reshape(mb * seq, h)
        x = x + o @ P[p + "attn_weight"].t() + P[p + "attn_bias"]
        b = F.layer_norm(x, (h,), P[p + "ln2_weight"], P[p + "ln2_bias"], c["layer_norm_epsilon"])
        ids = chosen[i].long()
        w = (b @ P[p + "router_weight"].t()).gather(1, ids).softmax(1)
        y = torch.zeros_like(x)
        for e in range(c["experts"]):
            t, j = (ids == e).nonzero(as_tuple=True)
            u = F.gelu(b[t] @ P[p + "fc1_weight"][e].t() + P[p + "fc1_bias"][e])
            y = y.index_add(0, t, w[t, j][:, None] * (u @ P[p + "fc2_weight"][e].t() + P[p + "fc2_bias"][e]))
        x = x + y
    x = F.layer_norm(x, (h,), P["final_weight"], P["final_bias"], c["layer_norm_epsilon"])
    loss = F.cross_entropy((x @ P["embedding"].t())[:, : c["vocab"]], targets)
    loss.backward()
    return loss.detach(), {n: t.grad for n, t in P.items()}


@pytest.mark.gpu
def test_gradients_against_64_bits(cuda):
    """bf16 activations round by 2^-9 of their size at some 30 places between a
    parameter and the loss; independent roundings add in squares, sqrt(30) 2^-9
    = 1.1 %, taken three times for what the layers amplify."""
    import torch
    from tempname_dcu_b200.models.gpt import GPT
    from tempname_dcu_b200.ops import moe, native
    from tempname_dcu_b200.train import synthetic_batches
    model = GPT(dict(CONFIG), "flux", None, device="cuda")
    (tokens, labels), = synthetic_batches(model.config, 1, seed=3)
    tokens, labels = tokens.cuda(), labels.cuda()
    chosen, route = [], moe.route

    def spy(*args, **kwargs):
        chosen.append(route(*args, **kwargs))
        return chosen[-1]
    moe.route = spy
    try:
        model.params.grad.fill_(float("nan"))
        loss = model.forward_backward(tokens[0], labels[0], grad_scale=1.0 / 256, loss_scale=1.0 / 256,
                                      overwrite_grads=True)
    finally:
        moe.route = route
    ref_loss, ref = _reference(model, tokens[0], labels[0], [r.ids for r in chosen])
    assert abs(loss.item() - ref_loss.item()) < 0.01
    for name, g in ref.items():
        got = model.Gr(name).double()
        assert torch.isfinite(got).all(), name
        err = (got - g).norm() / g.norm().clamp_min(1e-12)
        assert err < 0.034, (name, err.item())
    native.raise_on_status()


@pytest.mark.gpu
def test_trainer_eager_graph_and_checkpoint(cuda, tmp_path):
    import torch
    from tempname_dcu_b200.ops import native
    from tempname_dcu_b200.train import Trainer, synthetic_batches
    eager = Trainer(dict(CONFIG), "flux", None, device="cuda")
    graph = Trainer(dict(CONFIG), "flux", None, device="cuda", cuda_graph=True, graph_warmup=1)
    batches = synthetic_batches(eager.config, 4, seed=5)
    for tokens, labels in batches[:3]:
        a, _ = eager.step(tokens, labels)
        b, _ = graph.step(tokens, labels)
        assert torch.equal(a, b) and torch.isfinite(a)
    assert torch.equal(eager.model.params.master, graph.model.params.master)
    eager.save_checkpoint(str(tmp_path / "ckpt"))
    other = Trainer(dict(CONFIG), "flux", None, device="cuda", seed=99)
    assert other.load_checkpoint(str(tmp_path / "ckpt")) == 3
    a, _ = eager.step(*batches[3])
    b, _ = other.step(*batches[3])
    assert torch.equal(a, b) and torch.equal(eager.model.params.master, other.model.params.master)
    graph.release_graph()
    native.raise_on_status()
