"""A training step with the decoder options on one GPU: head norms, partial interleaved rotation, the general router and
the fused output layer on the native kernels."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _train(fused, moe, steps=4, recompute=False):
    from elasticmegatron_b200.config import Args, ModelConfig, RopeScaling, TrainConfig, set_args
    from elasticmegatron_b200.ops.native import check_device_errors
    from elasticmegatron_b200.parallel.strategy import ParallelStrategy
    from elasticmegatron_b200.runtime.data import DataloaderState
    from elasticmegatron_b200.runtime.train import train_step
    from elasticmegatron_b200.runtime.training_state import TrainingState

    kw = dict(num_experts=16, moe_router_topk=4, moe_ffn_hidden_size=128, moe_router_score_function="sigmoid",
              moe_router_num_groups=4, moe_router_group_topk=2, moe_router_topk_scaling_factor=2.5) if moe else {}
    cfg = ModelConfig(num_layers=2, hidden_size=512, num_attention_heads=8, num_query_groups=4, ffn_hidden_size=1376,
                      vocab_size=5000, seq_length=256, params_dtype="bf16", qk_layernorm=True, rotary_percent=0.5,
                      rotary_interleaved=True, rope_scaling=RopeScaling("llama3", 8.0, 64), **kw)
    set_args(Args(model=cfg, train=TrainConfig(micro_batch_size=2, global_batch_size=4, lr=2e-3, recompute=recompute,
                                               fuse_linear_cross_entropy=fused)))
    ts = TrainingState(ParallelStrategy(world_size=1, tensor_model_parallel_size=1, pipeline_model_parallel_size=1))
    ts.init_weights(0, method="local")
    it = DataloaderState.build_iterators(ts, 0)[0]
    batch = [next(it) for _ in range(2)]
    losses = [train_step(ts, iter(batch))["loss"] for _ in range(steps)]
    check_device_errors()
    ws = [p for n, p in ts.stage.params_by_name.items() if "_layernorm.weight" in n and "self_attention" in n
          and n.split(".")[-2] in ("q_layernorm", "k_layernorm")]
    assert len(ws) == 4 and all(float((p.detach().float() - 1).abs().max()) > 0 for p in ws)
    return losses


@pytest.mark.parametrize("moe", [False, True])
def test_train_step(moe):
    plain, fused = _train(False, moe), _train(True, moe)
    assert plain[-1] < plain[0] - 0.5  # the same batch again and again
    # the unfused loss goes over bf16 logits (2^-9 of logits of a few units, averaged over 1024 tokens)
    for a, b in zip(plain, fused):
        assert abs(a - b) < 2e-2
    again = _train(True, moe, recompute=True)
    for a, b in zip(fused, again):
        assert abs(a - b) < (2e-2 if moe else 5e-3)
