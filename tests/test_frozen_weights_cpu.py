"""A frozen 4-bit model is kept: copied, moved, saved and loaded."""
import copy
import io

import pytest
import torch

from flex_shard_b200.models.llama import Llama, LlamaConfig
from flex_shard_b200.quant import BlockwiseMxfp4Weight, FlexShardMxfp4BlockwiseLinear, freeze_mxfp4_weights_

PATTERNS = ["layers.*.w*", "head.output"]
TOKENS = torch.arange(12).view(2, 6) * 7 % 128


def model(seed=0):
    m = Llama(LlamaConfig(vocab_size=128, d_model=256, n_layers=1, n_heads=2, n_kv_heads=1, ffn_hidden=256, max_seq_len=256),
              dtype=torch.bfloat16, device="cpu")
    m.init_weights(seed)
    return m


def frozen(seed=0):
    return freeze_mxfp4_weights_(model(seed), PATTERNS)


def score(m):
    with torch.no_grad():
        return m.token_logprobs(TOKENS, TOKENS).logprob


def payload(m):
    return [t for p in m.parameters() if isinstance(p, BlockwiseMxfp4Weight) for t in (p.qdata, p.scale, p.dgrad_scale, p.extra["tile_exp"])]


def test_a_deep_copy_is_the_same_model_in_memory_of_its_own():
    a = frozen()
    b = copy.deepcopy(a)
    assert [type(p) for p in a.parameters()] == [type(p) for p in b.parameters()]
    assert all(torch.equal(p, q) and p.data_ptr() != q.data_ptr() for p, q in zip(payload(a), payload(b)))
    assert not any(p.requires_grad for p in b.parameters() if isinstance(p, BlockwiseMxfp4Weight))
    want = score(a)
    assert torch.equal(score(b), want)
    for t in payload(b):
        t.zero_()
    assert torch.equal(score(a), want)


def test_a_copy_of_a_layer_still_passes_gradients_on():
    layer = FlexShardMxfp4BlockwiseLinear(128, 256)
    torch.nn.init.normal_(layer.weight, std=0.1)
    layer = copy.deepcopy(layer.freeze_())
    x = torch.randn(3, 128).bfloat16().requires_grad_()
    layer(x).sum().backward()
    assert x.grad.any() and isinstance(layer.weight, torch.nn.Parameter)


def test_moves_keep_the_payload():
    a = frozen()
    want, before = score(a), [t.clone() for t in payload(a)]
    a.to("cpu").bfloat16()
    assert torch.equal(score(a), want)
    a.to(torch.float32)
    weights = [p for p in a.parameters() if isinstance(p, BlockwiseMxfp4Weight)]
    assert len(weights) == 5 and all(p.dtype == torch.float32 for p in weights)
    assert all(torch.equal(p, q) for p, q in zip(payload(a), before))
    a.bfloat16()
    assert torch.equal(score(a), want)
    w = weights[0].detach()
    assert torch.equal(w.clone().qdata, w.qdata) and w.to(torch.float16).dtype == torch.float16
    with pytest.raises(NotImplementedError):
        w.to(torch.int32)
    with pytest.raises(NotImplementedError):
        w + w


def test_meta_and_back():
    a, b = frozen(1), frozen(0).to("meta")
    assert all(t.is_meta for t in payload(b)) and all(p.device.type == "meta" for p in b.parameters())
    b.to_empty(device="cpu")
    assert all(not t.is_meta for t in payload(b))
    b.load_state_dict(a.state_dict())
    for (n, p), q in zip(a.named_buffers(), b.buffers()):
        q.copy_(p)
    assert torch.equal(score(a), score(b))


@pytest.mark.parametrize("assign", [False, True])
@pytest.mark.parametrize("file", [False, True])
def test_state_dicts(assign, file):
    a, b = frozen(1), frozen(2)
    state = a.state_dict()
    if file:
        f = io.BytesIO()
        torch.save(state, f)
        f.seek(0)
        state = torch.load(f, weights_only=True)
        assert all(type(state[n]) is type(p) or not isinstance(p, BlockwiseMxfp4Weight) for n, p in a.named_parameters())
    assert not torch.equal(score(a), score(b))
    b.load_state_dict(state, assign=assign)
    assert torch.equal(score(a), score(b))
    assert all(torch.equal(p, q) for p, q in zip(payload(a), payload(b)))
    assert (payload(b)[0].data_ptr() == payload(a)[0].data_ptr()) == (assign and not file)


def test_a_high_precision_checkpoint_is_quantised_on_the_way_in():
    b = frozen(2)
    b.load_state_dict(model(1).state_dict())
    assert torch.equal(score(b), score(frozen(1)))


def test_refusals():
    a = frozen()
    with pytest.raises((NotImplementedError, RuntimeError), match="prequantised|detach"):
        model().load_state_dict(a.state_dict())                 # a master weight does not become a payload unnoticed
    w = a.head.output.detach()
    with pytest.raises(ValueError, match="does not fit"):
        w.copy_(torch.zeros(1, 128).bfloat16())


def test_weights_that_only_score():
    """Payloads without the input gradient's scales and without tile exponents, as a user may put them together."""
    full = frozen().head.output.detach()
    lean = BlockwiseMxfp4Weight(full.qdata.clone(), full.scale.clone(), full.shape)
    for w in (lean.clone(), lean.to(torch.float32), copy.deepcopy(torch.nn.Parameter(lean, requires_grad=False)), lean.to("meta")):
        assert w.dgrad_scale is None and w.extra == {} and w.shape == full.shape
    lean.qdata.zero_()
    lean.copy_(full)
    assert torch.equal(lean.qdata, full.qdata)
    with pytest.raises(ValueError, match="cannot be loaded"):
        full.copy_(lean)
