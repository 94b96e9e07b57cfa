"""Gradients through frozen 4-bit matrices of any size."""
import pytest
import torch

from flex_shard_b200.models.deepseek_v3 import DeepSeekV3, DeepSeekV3Config
from flex_shard_b200.ops.gemm import linear
from flex_shard_b200.quant import BlockwiseMxfp4Weight, FlexShardMxfp4BlockwiseLinear, freeze_mxfp4_weights_

SIZES = [(1, 576, 256), (5, 40, 128), (3, 36, 96), (130, 1, 32), (17, 257, 160), (2, 128, 96)]


def check_input_gradient(T, N, K, device):
    """Products of bf16 numbers are exact in fp32, a sum of N of them good to N 2^-24 of the magnitudes' sum; rounded to bf16 once."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(T, K, generator=g).bfloat16().to(device).requires_grad_()
    w = BlockwiseMxfp4Weight.from_float(torch.randn(N, K, generator=g).bfloat16().to(device))
    dy = torch.randn(T, N, generator=g).bfloat16().to(device)
    y = linear(x, torch.nn.Parameter(w, requires_grad=False))
    with torch.no_grad():
        assert torch.equal(y, linear(x, w))
    (dx,) = torch.autograd.grad(y, x, dy)
    a, b = dy.double(), w.dequantize().double()
    want = a @ b
    assert dx.shape == x.shape and dx.dtype == torch.bfloat16
    assert ((dx.double() - want).abs() <= (a.abs() @ b.abs()) * (N * 2.0 ** -24) + want.abs() * 2.0 ** -8).all()


@pytest.mark.parametrize("T,N,K", SIZES)
def test_matrices_of_any_size_pass_gradients_on(T, N, K):
    check_input_gradient(T, N, K, "cpu")


def test_a_frozen_layer_of_any_size():
    layer = FlexShardMxfp4BlockwiseLinear(96, 40)
    torch.nn.init.normal_(layer.weight)
    x = torch.randn(2, 3, 96).bfloat16().requires_grad_()
    with pytest.raises(ValueError, match="multiples of 128"):
        layer(x)                                            # a trained one keeps to the 8-bit products
    layer.freeze_()(x).sum().backward()
    assert x.grad.shape == x.shape and x.grad.any()


def test_a_decoder_with_frozen_latent_projections():
    """Compressed key and value projections have rows that are no multiple of 128 at the usual sizes."""
    cfg = DeepSeekV3Config(vocab_size=128, d_model=64, n_layers=2, n_heads=2, q_lora_rank=32, kv_lora_rank=32, qk_nope_dim=16,
                           qk_rope_dim=8, v_dim=16, dense_hidden=64, n_experts=4, expert_hidden=32, top_k=2, max_seq_len=16)
    model = DeepSeekV3(cfg, dtype=torch.bfloat16, device="cpu")
    model.init_weights(0)
    names = [n for n, p in model.named_parameters() if p.dim() == 2 and n.split(".")[-1] in ("wq_a", "wq_b", "wkv_a", "wkv_b", "wo")]
    assert len(names) == 10 and model.get_parameter([n for n in names if n.endswith("wkv_a")][0]).shape[0] % 128
    freeze_mxfp4_weights_(model, names)
    tokens = torch.randint(0, 128, (2, 8), generator=torch.Generator().manual_seed(0))
    model.token_logprobs(tokens, tokens).logprob.sum().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters() if p.requires_grad and p.dim() == 2)
    experts = [n for n, p in model.named_parameters() if p.dim() == 3]
    with pytest.raises(ValueError, match="not a matrix"):
        freeze_mxfp4_weights_(model, experts)
