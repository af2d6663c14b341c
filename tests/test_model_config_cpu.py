"""Positional arguments of the model configuration keep their meaning."""
from elasticmegatron_b200.config import ModelConfig


def test_positional_arguments():
    names = ["num_layers", "hidden_size", "num_attention_heads", "num_query_groups", "ffn_hidden_size", "vocab_size",
             "make_vocab_size_divisible_by", "max_tensor_parallel_size", "seq_length", "rotary_base", "norm_epsilon",
             "normalization", "init_method_std", "untie_embeddings_and_output_weights", "num_experts", "moe_router_topk",
             "moe_aux_loss_coeff", "moe_ffn_hidden_size", "params_dtype"]
    values = [2, 64, 4, 2, 128, 500, 8, 2, 32, 5000.0, 1e-6, "LayerNorm", 0.01, False, 4, 1, 0.0, 32, "fp32"]
    assert ModelConfig(*values) == ModelConfig(**dict(zip(names, values)))
