"""Query / key norms, partial interleaved scaled rotation, the general router and the fused output layer in the training
core on gloo ranks: the loss and the gradient norm depend neither on the layout nor on switches, and the fused output
layer gives the losses of the unfused one."""
import numpy as np
import pytest

from dist_utils import run_distributed


def _cfg(moe):
    from elasticmegatron_b200.config import ModelConfig, RopeScaling

    kw = dict(num_experts=4, moe_router_topk=2, moe_ffn_hidden_size=32, moe_router_score_function="sigmoid",
              moe_router_num_groups=2, moe_router_group_topk=1, moe_router_topk_scaling_factor=1.5) if moe else {}
    return ModelConfig(num_layers=2, hidden_size=64, num_attention_heads=4, num_query_groups=2, ffn_hidden_size=128,
                       vocab_size=500, seq_length=32, params_dtype="fp32", max_tensor_parallel_size=2,
                       make_vocab_size_divisible_by=8, qk_layernorm=True, rotary_percent=0.5, rotary_interleaved=True,
                       rope_scaling=RopeScaling("yarn", 4.0, 16), **kw)


def _run(rank, world, specs, moe, fused):
    from elasticmegatron_b200.config import Args, TrainConfig, set_args
    from elasticmegatron_b200.parallel.process_groups import create_all_groups
    from elasticmegatron_b200.parallel.strategy import ParallelStrategy
    from elasticmegatron_b200.runtime.manager import ElasticMegatronManager
    from elasticmegatron_b200.runtime.train import train_step
    from elasticmegatron_b200.runtime.training_state import TrainingState

    set_args(Args(model=_cfg(moe), train=TrainConfig(micro_batch_size=2, global_batch_size=8, lr=1e-3,
                                                     overlap_grad_reduce=True, ddp_bucket_size=20000,
                                                     fuse_linear_cross_entropy=fused)))
    S = [ParallelStrategy.parse(x) for x in dict.fromkeys(specs)]
    create_all_groups(S)
    ts = TrainingState(S[0])
    ts.init_weights(0)
    mgr = ElasticMegatronManager(S, training_state=ts, engine="torch")
    consumed, losses, norms = 0, [], []
    it = mgr.build_iterators(consumed)[0]
    for i, spec in enumerate(specs):
        if i and spec != specs[i - 1]:
            ts = mgr.reshard(spec)
            it = mgr.build_iterators(consumed)[0]
        out = train_step(ts, it)
        losses.append(out["loss"])
        norms.append(float(out["grad_norm"]))
        consumed += 8
    ws = [p for n, p in ts.stage.params_by_name.items() if n.endswith(("q_layernorm.weight", "k_layernorm.weight"))]
    trained = bool(ws) and all(float((p.detach() - 1).abs().max()) > 0 for p in ws)
    return losses, norms, trained


@pytest.mark.parametrize("moe", [False, True])
def test_losses_do_not_depend_on_layout(moe):
    base = run_distributed(_run, 2, ["ws2"] * 4, moe, False)
    assert all(t for _, _, t in base)  # every head norm left 1 after training
    tp = "ws2-tp2-etp1" if moe else "ws2-tp2"
    runs = [(["ws2"] * 4, True), (["ws2", tp, "ws2-pp2", "ws2"], True), ([tp] * 4, False)]
    runs += [(["ws2-ep2-etp1"] * 4, True)] if moe else [(["ws2-tp2-nosp"] * 4, True), (["ws2-cp2"] * 4, True)]
    for specs, fused in runs:
        res = run_distributed(_run, 2, specs, moe, fused)
        # (the auxiliary loss of a layout sees its own micro-batch of tokens, so an MoE's later losses move a little)
        rtol = 2e-4 if moe else 1e-5
        np.testing.assert_allclose(res[0][0], base[0][0], rtol=rtol, err_msg=str(specs))
        np.testing.assert_allclose(res[0][1][0], base[0][1][0], rtol=1e-3 if moe else 1e-4, err_msg=str(specs))
        assert all(t for _, _, t in res), specs


def test_expert_bias_moves_the_choice_only():
    """A selection bias changes which experts are chosen; the weights stay the scores of the chosen."""
    import torch

    from elasticmegatron_b200.config import Args, TrainConfig, set_args
    from elasticmegatron_b200.parallel.strategy import ParallelStrategy
    from elasticmegatron_b200.runtime.training_state import TrainingState

    set_args(Args(model=_cfg(True), train=TrainConfig(micro_batch_size=2, global_batch_size=8)))
    ts = TrainingState(ParallelStrategy(world_size=1, tensor_model_parallel_size=1, pipeline_model_parallel_size=1))
    ts.init_weights(0)
    layer = ts.stage.moe[0]
    h = torch.randn(64, 64)
    layer(h)
    before = layer.last_counts.clone()
    layer.expert_bias = torch.tensor([10.0, 9.0, -5.0, -5.0])
    layer(h)
    assert layer.last_counts.tolist() == [64, 64, 0, 0] and before.tolist() != [64, 64, 0, 0]
    logits = torch.randn(5, 4)
    w, e, _, _ = layer._route(logits)
    s = torch.sigmoid(logits)[:, :2]
    torch.testing.assert_close(w, 1.5 * s / s.sum(-1, keepdim=True), atol=1e-6, rtol=1e-5)
    assert e.tolist() == [[0, 1]] * 5


def test_config_refusals():
    from elasticmegatron_b200.config import ModelConfig

    for kw in (dict(rotary_percent=0.0), dict(rotary_percent=1.5), dict(hidden_size=64, rotary_percent=0.4),
               dict(moe_router_score_function="relu"), dict(moe_router_num_groups=2),
               dict(num_experts=8, moe_router_num_groups=3, moe_router_group_topk=1),
               dict(num_experts=8, moe_router_num_groups=8, moe_router_group_topk=1)):
        with pytest.raises(ValueError):
            ModelConfig(**kw)
