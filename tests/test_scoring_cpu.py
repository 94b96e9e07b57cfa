"""A frozen 4-bit teacher and a trained policy scoring the same tokens, on CPU tensors."""
import pytest
import torch

from flex_shard_b200 import flex_shard
from flex_shard_b200.models.deepseek_v3 import DeepSeekV3, DeepSeekV3Config
from flex_shard_b200.models.llama import Llama, LlamaConfig, llama_buckets
from flex_shard_b200.quant import BlockwiseMxfp4Weight, freeze_mxfp4_weights_
from tests.logprobs_common import definition

TINY = dict(vocab_size=384, d_model=256, n_layers=2, n_heads=2, n_kv_heads=1, ffn_hidden=256, max_seq_len=32)


def tiny(seed=0):
    model = Llama(LlamaConfig(**TINY), dtype=torch.bfloat16, device="cpu")
    model.init_weights(seed)
    return model


def test_frozen_teacher_scores_and_policy_takes_gradients():
    teacher, policy = tiny(), tiny()
    freeze_mxfp4_weights_(teacher, ["layers.*.w*", "head.output"])
    frozen = [n for n, p in teacher.named_parameters() if isinstance(p, BlockwiseMxfp4Weight)]
    assert len(frozen) == 2 * 4 + 1 and "tok_embeddings.weight" not in frozen
    tokens = torch.randint(0, 384, (2, 9), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        ref = teacher.token_logprobs(tokens[:, :-1], tokens[:, 1:], top_k=4)
    out = policy.token_logprobs(tokens[:, :-1], tokens[:, 1:], temperature=0.9, top_k=4)
    assert out.logprob.shape == (2, 8) and ref.top_index.shape == (2, 8, 4)
    with torch.no_grad():
        _, want = definition(teacher(tokens[:, :-1]), tokens[:, 1:].reshape(-1), 1.0, 4)
    torch.testing.assert_close(ref.logprob.reshape(-1).double(), want["logprob"], rtol=0, atol=1e-5)
    assert torch.equal(ref.top_index.reshape(-1, 4), want["top_index"])
    loss = -(out.logprob * torch.sign(ref.logprob - ref.logprob.mean())).mean() - 0.01 * out.entropy.mean() \
        + 0.1 * (out.logprob - ref.logprob).mean()
    loss.backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in policy.parameters())


def test_gradients_pass_through_frozen_weights():
    model = tiny()
    freeze_mxfp4_weights_(model, ["layers.*.w*"])
    tokens = torch.randint(0, 384, (1, 8))
    model.token_logprobs(tokens, tokens).logprob.sum().backward()
    assert model.tok_embeddings.weight.grad.abs().sum() > 0 and model.head.output.grad is not None


def test_expert_decoder_scores():
    cfg = DeepSeekV3Config(vocab_size=256, d_model=64, n_layers=2, n_heads=2, q_lora_rank=32, kv_lora_rank=32, qk_nope_dim=16,
                           qk_rope_dim=8, v_dim=16, dense_hidden=64, n_experts=4, expert_hidden=32, top_k=2, max_seq_len=16)
    model = DeepSeekV3(cfg, dtype=torch.bfloat16, device="cpu")
    model.init_weights(0)
    tokens = torch.randint(0, 256, (2, 8))
    out = model.token_logprobs(tokens, tokens, top_k=3, ignore_index=int(tokens[0, 0]))
    assert out.top_logprob.shape == (2, 8, 3) and out.logprob[0, 0] == 0
    out.entropy.sum().backward()
    assert model.output.grad.isfinite().all()


def test_refusals():
    model = tiny()
    with pytest.raises(ValueError, match="no parameter"):
        freeze_mxfp4_weights_(model, ["nothing.*"])
    with pytest.raises(ValueError, match="attention_norm"):
        freeze_mxfp4_weights_(model, ["layers.0.*"])
    freeze_mxfp4_weights_(model, ["layers.0.w2"])
    with pytest.raises(ValueError, match="layers.0.w2"):
        freeze_mxfp4_weights_(model, ["layers.*.w2"])
    sharded = tiny()
    flex_shard(sharded, llama_buckets(sharded))
    with pytest.raises(ValueError, match="not sharded"):
        freeze_mxfp4_weights_(sharded, ["layers.*.w*"])
