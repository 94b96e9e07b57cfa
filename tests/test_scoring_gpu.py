"""A frozen 4-bit teacher and a trained, sharded policy that score the same tokens on one GPU."""
import pytest
import torch

from flex_shard_b200 import flex_shard, ops
from flex_shard_b200.models.llama import Llama, LlamaConfig, llama_buckets
from flex_shard_b200.ops import mxfp4 as m4
from flex_shard_b200.ops.gemm import linear
from flex_shard_b200.quant import freeze_mxfp4_weights_
from tests.logprobs_common import definition, gradient, value_tolerance

pytestmark = pytest.mark.gpu
CFG = dict(vocab_size=4096, d_model=512, n_layers=2, n_heads=4, n_kv_heads=2, ffn_hidden=1024, max_seq_len=256)


def model(seed):
    m = Llama(LlamaConfig(**CFG), dtype=torch.bfloat16, device="cuda")
    m.init_weights(seed)
    return m


def test_teacher_and_policy():
    teacher, policy = model(0), model(0)
    with torch.no_grad():
        x = torch.randn(2, 256, 512, device="cuda").bfloat16()
        full = linear(x, teacher.layers[0].w13)
        freeze_mxfp4_weights_(teacher, ["layers.*.w*", "head.output"])
        w = teacher.layers[0].w13
        y = linear(x, w)
        xv = m4.mx4_dequantize(*m4.mx4_quantize_act(x.view(-1, 512)), torch.float32).double()
        ref = xv @ w.dequantize().double().t()
        size = xv.abs() @ w.dequantize().double().abs().t()
        assert ((y.view(-1, 2048).double() - ref).abs() <= size * (512 * 2.0 ** -24) + ref.abs() * 2.0 ** -8).all()
        # two operands off by up to a quarter of a value each, at random: their product by about a seventh of its size
        assert 0 < float((y - full).float().norm() / full.float().norm()) < 0.35
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, 4096, (2, 257), generator=g, device="cuda")
    inputs, targets = tokens[:, :-1], tokens[:, 1:].clone()
    targets[:, :40] = -100                                   # the prompt
    with torch.no_grad():
        t = teacher.token_logprobs(inputs, targets, top_k=8)
        logits = teacher(inputs)
    _, want = definition(logits, targets.reshape(-1), 1.0, 8)
    torch.testing.assert_close(t.logprob.reshape(-1).double(), want["logprob"], rtol=0, atol=value_tolerance(logits, 1.0))
    assert torch.equal(t.top_index.reshape(-1, 8), want["top_index"])

    flex_shard(policy, llama_buckets(policy))
    out = policy.token_logprobs(inputs, targets, temperature=0.8, top_k=8)
    advantage = torch.randn(2, 256, generator=g, device="cuda")
    n = (targets != -100).sum()
    loss = -(advantage * out.logprob).sum() / n - 0.01 * out.entropy.sum() / n + 0.1 * (t.top_logprob.exp() * -out.top_logprob).sum() / n
    loss.backward()
    got = [p.grad.float().clone() for p in policy.parameters()]
    ops.check_status()
    # the same gradient of the logits from the formula in 64 bits, rounded to bf16, through the same model: what differs is
    # single roundings of the logits' gradient, half a step (2^-8) of their values at most
    for p in policy.parameters():
        p.grad = None
    logits = policy(inputs)
    d, _ = gradient(logits.detach(), targets.reshape(-1), 0.8, 8, (-advantage / n).reshape(-1), torch.full((512,), -0.01, device="cuda") / n,
                    (-0.1 * t.top_logprob.exp() / n).reshape(-1, 8))
    logits.backward(d.to(torch.bfloat16))
    for a, p in zip(got, policy.parameters()):
        b = p.grad.float()
        assert b.abs().sum() > 0 and float((a - b).norm() / b.norm()) <= 2.0 ** -7


def test_scoring_repeats_bit_for_bit_and_in_a_graph():
    teacher = freeze_mxfp4_weights_(model(3), ["layers.*.w*", "head.output"])
    tokens = torch.randint(0, 4096, (1, 257), device="cuda")
    with torch.no_grad():
        first = teacher.token_logprobs(tokens[:, :-1], tokens[:, 1:], top_k=5)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            teacher.token_logprobs(tokens[:, :-1], tokens[:, 1:], top_k=5)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = teacher.token_logprobs(tokens[:, :-1], tokens[:, 1:], top_k=5)
        torch.cuda.current_stream().wait_stream(side)
        graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, out))
    ops.check_status()
