"""A frozen 4-bit model moved to the GPU, copied there, loaded in place under a captured graph, and moved back."""
import copy

import pytest
import torch

from flex_shard_b200 import ops
from flex_shard_b200.quant import BlockwiseMxfp4Weight, freeze_mxfp4_weights_
from tests.test_frozen_weights_cpu import PATTERNS, frozen, model, payload

pytestmark = pytest.mark.gpu


def score(m):
    tokens = torch.arange(256, device="cuda")[None] * 7 % 128
    with torch.no_grad():
        return m.token_logprobs(tokens, tokens, top_k=3)


def test_moves_and_copies():
    a = frozen().cuda()                                             # quantised on the CPU, then moved
    b = freeze_mxfp4_weights_(model().cuda(), PATTERNS)             # moved, then quantised
    assert all(p.is_cuda and torch.equal(p, q) for p, q in zip(payload(a), payload(b)))
    c = copy.deepcopy(a)
    want = score(b)
    for m in (a, c):
        assert all(torch.equal(x, y) for x, y in zip(score(m), want))
    ops.check_status()
    a.cpu()
    assert all(torch.equal(p, q.cpu()) and not p.is_cuda for p, q in zip(payload(a), payload(b)))
    assert all(isinstance(p, BlockwiseMxfp4Weight) == isinstance(q, BlockwiseMxfp4Weight) for p, q in zip(a.parameters(), b.parameters()))


def test_loading_in_place_under_a_captured_graph():
    a, b = frozen(1).cuda(), frozen(2).cuda()
    want = score(b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        x = torch.randn(5, 256, device="cuda").bfloat16()
        layer = lambda m: ops.linear(x, m.layers[0].w13)  # noqa: E731
        layer(a)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = layer(a)
    torch.cuda.current_stream().wait_stream(side)
    a.load_state_dict(b.state_dict())                               # the payload's memory stays where it is
    graph.replay()
    assert torch.equal(y, layer(b)) and all(torch.equal(p, q) for p, q in zip(score(a), want))
    ops.check_status()
